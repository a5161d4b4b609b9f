"""Trees of drafts end to end: a small GQA decoder whose tree step is projection,
Rotate, Append, AttendTree and KeepPath, under TreeSpeculativeDecoder; and the
operators of one step together in a graph."""
import math
import random

import numpy as np
import pytest
import torch

from oracle import tree as ref

pytestmark = pytest.mark.gpu


class _Decoder:
    """Two layers, 4 heads over 2 kv heads of 32 dims, f32 activations, bf16 cache."""
    V, DM, H, KVH, D, L = 60, 64, 4, 2, 32, 2

    def __init__(self, gpu, seed, near=None, layout="halves"):
        from relux_amd import KVCache, rope_frequencies
        g = torch.Generator(device=gpu).manual_seed(seed)
        shapes = dict(e=(self.V, self.DM), o=(self.DM, self.V))
        for i in range(self.L):
            shapes.update({f"qkv{i}": (self.DM, (self.H + 2 * self.KVH) * self.D), f"wo{i}": (self.H * self.D, self.DM),
                           f"up{i}": (self.DM, 2 * self.DM), f"down{i}": (2 * self.DM, self.DM)})
        self.w = {}
        for k, s in shapes.items():
            w = torch.randn(*s, device=gpu, generator=g) * (1.0 if k == "e" else 3.0 if k == "o" else 1.5) / math.sqrt(s[0] if k != "e" else 1)
            self.w[k] = w if near is None else near.w[k] + 0.05 * w
        self.cache = KVCache(num_layers=self.L, max_len=600, num_kv_heads=self.KVH, head_dim=self.D, device=gpu.index)
        self.inv, self.scale = rope_frequencies(self.D, 10000.0, dict(type="linear", factor=2.0), gpu)
        self.gpu, self.layout, self.tree = gpu, layout, 0

    def reset(self):
        self.cache.Reset()
        self.tree = 0

    def _run(self, ids, pos, attend):
        x = self.w["e"][torch.tensor(ids, device=self.gpu)]
        pos = torch.tensor(pos, dtype=torch.int32, device=self.gpu)
        H, KVH, D = self.H, self.KVH, self.D
        for i in range(self.L):
            y = torch.nn.functional.layer_norm(x, (self.DM,))
            qkv = (y @ self.w[f"qkv{i}"]).view(len(ids), H + 2 * KVH, D)
            qk = qkv[:, :H + KVH]  # q and k heads in one call, in place
            self.cache.Rotate(qk, pos, self.inv, layout=self.layout, scale=self.scale, out=qk)
            self.cache.Append(i, qkv[:, H:H + KVH].contiguous(), qkv[:, H + KVH:].contiguous(), n_tok=[len(ids)],
                              layout="SHD")
            x = x + attend(i, qkv[:, :H].contiguous()).view(len(ids), H * D) @ self.w[f"wo{i}"]
            y = torch.nn.functional.layer_norm(x, (self.DM,))
            x = x + torch.nn.functional.gelu(y @ self.w[f"up{i}"]) @ self.w[f"down{i}"]
        return torch.nn.functional.layer_norm(x, (self.DM,)) @ self.w["o"]

    def forward(self, ids):
        n = self.cache.TotalLen(0)
        # (a chain is a tree without branches: the same attention, so the same rounding)
        chain = torch.arange(-1, len(ids) - 1, dtype=torch.int32, device=self.gpu)
        return self._run(ids, [n + j for j in range(len(ids))],
                         lambda i, q: self.cache.AttendTree(i, q, self.H, chain))

    def forward_tree(self, ids, parents, depths, n_new):
        n = self.cache.TotalLen(0) - self.tree
        assert self.tree == len(ids) - n_new
        self.tree = len(ids)
        up = torch.tensor(parents, dtype=torch.int32, device=self.gpu)
        return self._run(ids[-n_new:], [n + k for k in depths[-n_new:]],
                         lambda i, q: self.cache.AttendTree(i, q, self.H, up, n_nodes=[len(ids)], n_q=[n_new]))

    def keep_path(self, n_nodes, path):
        self.cache.KeepPath(0, n_nodes, path)
        self.tree = 0


@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_tree_logits_are_the_path_s(gpu, layout):
    """Every node's logits are those of its path fed token by token; after a kept path the next token's are too."""
    m, plain = _Decoder(gpu, 1, layout=layout), _Decoder(gpu, 1, layout=layout)
    prompt, rng = [5, 9, 2, 40, 7, 7, 3], random.Random(2)
    parents = [-1] + [rng.randint(max(0, j - 5), j - 1) for j in range(1, 20)]
    depths = [len(ref.ancestors(parents, j)) - 1 for j in range(20)]
    ids = [rng.randrange(60) for _ in range(20)]
    m.forward(prompt)
    first = m.forward_tree(ids[:8], parents[:8], depths[:8], 8)
    got = torch.cat([first, m.forward_tree(ids, parents, depths, 12)])  # level by level
    for j in (0, 3, 11, 19):
        plain.reset()
        path = [ids[a] for a in ref.ancestors(parents, j)[::-1]]
        want = plain.forward(prompt + path)[-1]
        # f32 throughout, the same bf16 keys and values but where an activation's last bits round one over
        assert (got[j] - want).abs().max() <= 0.05 * want.abs().max()
    path = ref.ancestors(parents, 19)[::-1]
    m.keep_path(20, path)
    plain.reset()
    plain.forward(prompt + [ids[a] for a in path])
    a, b = m.forward([11])[-1], plain.forward([11])[-1]
    assert (a - b).abs().max() <= 0.05 * b.abs().max()
    for layer in range(2):
        for x, y in zip(m.cache.View(layer), plain.cache.View(layer)):
            assert (x.float() - y.float()).abs().max() <= 2.0 ** -5 * y.float().abs().max()


@pytest.mark.parametrize("widths,branch", [((4, 4, 4, 2), 2), ((8,), 8), ((1, 1, 1, 1, 1), 1)])
def test_decoder_greedy_is_the_target_s(gpu, widths, branch):
    from relux_amd import Draws, Sampler, TreeSpeculativeDecoder
    t = _Decoder(gpu, 3)
    d = _Decoder(gpu, 4, near=t)
    dec = TreeSpeculativeDecoder(d, t, widths=widths, branch=branch,
                                 sampling=Sampler(temperature=1e-4, rand=Draws(seed=5)))
    got, rate = dec.Generate([1, 2, 3], 60)
    plain = _Decoder(gpu, 3)
    logits = plain.forward([1, 2, 3])[-1]
    for k, x in enumerate(got):
        best = torch.topk(logits, 2).values
        # the target's own choice, unless its two best are within the rounding of their logits
        assert int(logits.argmax()) == x or float(best[0] - best[1]) <= 0.02 * float(logits.abs().max()), k
        logits = plain.forward([x])[-1]
    # a step takes at most one node of each level, len(widths) of its sum(widths)
    assert rate > 0.2 * len(widths) / sum(widths)
    assert t.cache.TotalLen(0) == t.cache.TotalLen(1) == d.cache.TotalLen(1) >= 3 + 60 - 1


def test_one_step_in_a_graph(gpu):
    """Rotate, AttendTree and tree_accept_async of a batch captured once, replayed on other rows, trees and
    draws; each replay's results are the eager ones, and KeepPath goes on from them."""
    from relux_amd import KVCache, Sampler, rope_frequencies, tree_accept_async
    g, rng = torch.Generator(device=gpu).manual_seed(7), random.Random(8)
    B, H, KVH, D, V, n = 3, 8, 2, 64, 500, [12, 20, 7]
    T = [300, 41, 900]
    c = KVCache(num_layers=1, max_len=1100, num_kv_heads=KVH, head_dim=D, max_seqs=B, device=gpu.index)
    seqs, rows = list(range(B)), sum(n)
    K, V_ = (torch.randn(sum(T), KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c.Append(0, K, V_, seq_ids=seqs, n_tok=T, layout="SHD")
    inv, scale = rope_frequencies(D, 10000.0, None, gpu)
    w = torch.randn(H * D, V, device=gpu, generator=g) * 0.3
    x, draft = torch.zeros(rows, H, D, device=gpu), torch.zeros(rows, V, device=gpu)
    pos, tok, par = (torch.zeros(rows, dtype=torch.int32, device=gpu) for _ in range(3))
    u, smp = torch.zeros(rows, device=gpu), Sampler(temperature=0.9)

    def step(out):
        q = c.Rotate(x, pos, inv, scale=scale, out=out[0])
        o = c.AttendTree(0, q, H, par, seq_ids=seqs, n_nodes=n, out=out[1])
        torch.mm(o.view(rows, H * D), w, out=out[2])
        return tree_accept_async(c, out[2], tok, par, n, u, smp, draft_logits=draft, path=out[3], n_acc=out[4],
                                 next_tok=out[5])

    def buffers():
        i32 = dict(dtype=torch.int32, device=gpu)
        return [torch.zeros(rows, H, D, device=gpu), torch.zeros(rows, H, D, device=gpu),
                torch.zeros(rows, V, device=gpu), torch.zeros(B, 20, **i32), torch.zeros(B, **i32), torch.zeros(B, **i32)]

    kn, vn = (torch.randn(rows, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c.Append(0, kn, vn, seq_ids=seqs, n_tok=n, layout="SHD")
    held, eager = buffers(), buffers()
    step(held)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    c.use_stream(stream)
    with torch.cuda.graph(graph, stream=stream):
        step(held)
    c.use_stream(torch.cuda.current_stream())
    for _ in range(4):
        trees = [[-1] + [rng.randint(max(0, j - 4), j - 1) for j in range(1, k)] for k in n]
        flat = sum(trees, [])
        par.copy_(torch.tensor(flat, dtype=torch.int32))
        pos.copy_(torch.tensor(sum([[a + len(ref.ancestors(p, j)) - 1 for j in range(len(p))] for a, p in zip(T, trees)], []),
                               dtype=torch.int32))
        x.copy_(torch.randn(rows, H, D, device=gpu, generator=g))
        u.copy_(torch.rand(rows, device=gpu, generator=g))
        draft.copy_(torch.randn(rows, V, device=gpu, generator=g) * 2)
        tok.copy_(torch.randint(0, V, (rows,), device=gpu, generator=g, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(eager)
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)
        at = 0
        for b, p in enumerate(trees):
            s = slice(at, at + len(p))
            path, nxt = ref.accept(eager[2][s].cpu().numpy(), tok[s].tolist(), p, u[s].cpu().numpy(), 0.9,
                                   draft[s].cpu().numpy())
            assert eager[3][b].tolist() == path + [-1] * (20 - len(path)) and eager[5][b].item() == nxt
            at += len(p)
    paths = [p[:a + 1] for p, a in zip(held[3].tolist(), held[4].tolist())]
    c.KeepPath(seqs, n, paths)
    assert [c.TotalLen(0, s) for s in seqs] == [a + len(p) for a, p in zip(T, paths)]
    at = 0
    for b in range(B):
        k, _ = c.View(0, b)
        assert torch.equal(k[0, :, T[b]:].transpose(0, 1), kn[at:at + n[b]][paths[b]])
        at += n[b]


def test_two_streams(gpu):
    """Handles on two streams at once: each one's calls are its own."""
    from relux_amd import KVCache
    g = torch.Generator(device=gpu).manual_seed(9)
    H, KVH, D, T, n = 32, 8, 128, 3000, 30
    par = torch.arange(-1, n - 1, dtype=torch.int32, device=gpu)
    work = []
    for _ in range(2):
        s = torch.cuda.Stream()
        K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
        q = torch.randn(n, H, D, device=gpu, generator=g).bfloat16()
        c = KVCache(num_layers=1, max_len=T + n, num_kv_heads=KVH, head_dim=D, device=gpu.index)
        c.Append(0, K, V, n_tok=[T + n], layout="SHD")
        work.append((s, c, q, c.AttendTree(0, q, H, par)))
    torch.cuda.synchronize()
    for s, c, q, _ in work:
        c.use_stream(s)
    outs = [[torch.empty_like(w[3]) for _ in range(8)] for w in work]
    torch.cuda.synchronize()
    for i in range(8):
        for k, (s, c, q, _) in enumerate(work):
            c.AttendTree(0, q, H, par, out=outs[k][i])
    torch.cuda.synchronize()
    for k, w in enumerate(work):
        for o in outs[k]:
            assert torch.equal(o, w[3])


def test_what_a_graph_cannot_hold_is_refused(gpu):
    """Staged plans, table writes under way and kept paths do not go into a graph; nothing changes."""
    from relux_amd import KVCache, ReluxError, Sampler, tree_accept_async
    B, H, KVH, D = 70, 2, 1, 16
    c = KVCache(num_layers=1, max_len=64, num_kv_heads=KVH, head_dim=D, max_seqs=B, device=gpu.index)
    k = torch.randn(B * 20, KVH, D, device=gpu)
    c.Append(0, k, k, seq_ids=list(range(B)), n_tok=[20] * B, layout="SHD")
    q, par = torch.randn(B * 4, H, D, device=gpu), torch.full((B * 4,), -1, dtype=torch.int32, device=gpu)
    want = c.AttendTree(0, q, H, par, seq_ids=list(range(B)), n_nodes=[4] * B)
    few = c.AttendTree(0, q[:4], H, par[:4])
    t, u = torch.randn(300, 10, device=gpu), torch.rand(300, device=gpu)
    out, stream = torch.empty_like(want), torch.cuda.Stream()
    torch.cuda.synchronize()
    c.use_stream(stream)

    def refused(call, match):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            with pytest.raises(ReluxError, match=match):
                call()

    refused(lambda: c.AttendTree(0, q, H, par, seq_ids=list(range(B)), n_nodes=[4] * B, out=out), "64 sequences")
    refused(lambda: c.KeepPath(0, 4, [0, 2]), "captured")
    refused(lambda: tree_accept_async(c, t, torch.zeros(300, dtype=torch.int32, device=gpu), par[:300].new_zeros(300),
                                      [1] * 300, u, Sampler()), "256 sequences")
    c.Rollback(seq=1, n_tokens=8)  # its second page goes back: a table write under way
    refused(lambda: c.AttendTree(0, q[:4], H, par[:4], out=out[:4]), "table writes")
    with torch.cuda.stream(stream):
        assert torch.equal(c.AttendTree(0, q[:4], H, par[:4]), few)
        assert c.TotalLen(0, 0) == 20 and c.TotalLen(0, 1) == 12
    torch.cuda.synchronize()
    c.close()


def test_pages_past_32_bit_offsets(gpu):
    """A tree on pages whose byte offsets in the pools pass 2^32: attention, kept path, gather."""
    from relux_amd import KVCache
    g = torch.Generator(device=gpu).manual_seed(31)
    H, KVH, D, T, n, far = 16, 8, 128, 333, 40, 9 * 2 ** 18  # 9 * 2^18 tokens of 2 KB: 4.5 GiB a pool
    c = KVCache(num_layers=1, max_len=far, num_kv_heads=KVH, head_dim=D, max_seqs=2, pool_pages=far // 16 + 32,
                device=gpu.index)
    fill = torch.zeros(2 ** 18, KVH, D, device=gpu, dtype=torch.bfloat16)
    for _ in range(9):
        c.Append(0, fill, fill, n_tok=[2 ** 18], layout="SHD")
    K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c.Append(0, K, V, seq_ids=[1], n_tok=[T + n], layout="SHD")
    assert min(p for p in c.PageTable(0, 1) if p >= 0) * 16 * KVH * D * 2 > 2 ** 32
    rng = random.Random(4)
    tree = [-1] + [rng.randint(max(0, j - 5), j - 1) for j in range(1, n)]
    q = torch.randn(n, H, D, device=gpu, generator=g)
    got = c.AttendTree(0, q, H, torch.tensor(tree, dtype=torch.int32, device=gpu), seq_ids=[1], n_nodes=[n])
    want, size = ref.attend(q, K, V, tree)
    # weights and scores in parts of bf16 as exact as f32: 2^-16 covers both
    assert ((got.double() - want).abs() <= 4 * 2.0 ** -16 * size + 1e-7).all()
    path = ref.ancestors(tree, n - 1)[::-1]
    c.KeepPath(1, n, path)
    k, v = c.View(0, 1)
    keep = list(range(T)) + [T + j for j in path]
    assert torch.equal(k[0].transpose(0, 1), K[keep]) and torch.equal(v[0].transpose(0, 1), V[keep])
    c.close()
