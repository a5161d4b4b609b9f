"""Trees of drafts over the paged cache against 64-bit definitions: attention,
rotary positions, acceptance, kept paths, and the refusals of each."""
import math
import random

import numpy as np
import pytest
import torch

from oracle import tree as ref

pytestmark = pytest.mark.gpu


def _tree(shape, n, rng):
    if shape == "chain":
        return list(range(-1, n - 1))
    if shape == "star":
        return [-1] + [0] * (n - 1)
    if shape == "roots":  # several roots, and parents that name no earlier node
        return [rng.choice([-1, -7, j, j + 1, n, 1 << 30, max(0, j - 2)]) for j in range(n)]
    return [-1] + [rng.randint(max(0, j - 9), j - 1) for j in range(1, n)]


def _cache(gpu, KVH, D, P, lens, **kw):
    from relux_amd import KVCache
    return KVCache(num_layers=1, max_len=max(lens) + 8 * P, num_kv_heads=KVH, head_dim=D, page_tokens=P,
                   max_seqs=len(lens), device=gpu.index, **kw)


def _fill(c, K, V, P):
    """Append every sequence's tokens page by page in turn, so that pages interleave."""
    done = [0] * len(K)
    while True:
        seqs = [i for i in range(len(K)) if done[i] < K[i].shape[0]]
        if not seqs:
            return
        n = [min(P + 5, K[i].shape[0] - done[i]) for i in seqs]
        c.Append(0, torch.cat([K[i][done[i]:done[i] + m] for i, m in zip(seqs, n)]),
                 torch.cat([V[i][done[i]:done[i] + m] for i, m in zip(seqs, n)]), seq_ids=seqs, n_tok=n, layout="SHD")
        for i, m in zip(seqs, n):
            done[i] += m


def _bound(want, size, dtype):
    # bf16: each weight is off by half a step, 2^-8, in the sum and in its norm, and the output by half a
    # step.  f32: weights in bf16 parts, at least two, 2^-16 at the worst in both, scores within 2^-16 (128 products
    # summed in f32) in both.
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * want.abs() + 2 * 2.0 ** -8 * size + 1e-6
    return 4 * 2.0 ** -16 * size + 1e-7


def _check(out, wants, dtype):
    at = 0
    for want, size in wants:
        got = out[at:at + want.shape[0]].double()
        at += want.shape[0]
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        bad = ~same & ~((got - want).abs() <= _bound(want, size, dtype))
        assert not bad.any(), (int(bad.sum()), float((got - want).abs().nan_to_num().max()))


# heads, kv heads, head dim, page, context tokens and nodes of every sequence, queries, tree
CASES = [
    (32, 8, 128, 16, [0], [1], None, "chain"),                 # a single token, nothing before it
    (32, 8, 128, 16, [1, 15, 16, 17], [1, 1, 2, 3], None, "random"),
    (32, 8, 128, 16, [200], [7], None, "random"),
    (8, 2, 64, 48, [31, 64, 1000], [33, 32, 31], None, "random"),  # pages that are no power of two
    (16, 16, 80, 32, [700, 33, 1500], [31, 1, 13], [15, 1, 6], "random"),  # the last levels alone
    (64, 8, 128, 16, [4000, 900, 12], [64, 40, 64], None, "random"),
    (28, 4, 128, 16, [500, 37], [61, 5], None, "star"),        # 7 heads a kv head
    (16, 1, 64, 16, [130], [40], None, "random"),              # 16 heads on one
    (3, 1, 96, 16, [100, 5], [50, 11], None, "random"),
    (4, 2, 2, 16, [40], [9], None, "random"),                  # rows padded to 8, stored as 16
    (5, 1, 20, 32, [90], [30], None, "random"),
    (4, 4, 32, 16, [77], [70], None, "roots"),
    (8, 4, 256, 16, [3000, 20], [20, 40], None, "random"),
    (6, 2, 200, 64, [513], [33], None, "random"),
    (8, 2, 128, 16, [300, 20], [256, 256], [256, 3], "chain"),
    (8, 2, 128, 16, [0], [256], None, "random"),
    (4, 2, 64, 16, [90 + 7 * i for i in range(70)], [1 + i % 9 for i in range(70)], None, "random"),  # staged plan
    (8, 2, 128, 16, [20000], [5], None, "random"),             # cut along the keys
    (32, 8, 128, 64, [9000, 100, 5000], [20, 9, 64], None, "random"),
]


@pytest.mark.parametrize("H,KVH,D,P,T,n,m,shape", CASES)
@pytest.mark.parametrize("q_dtype,out_dtype,layout", [(torch.bfloat16, torch.bfloat16, "SHD"),
                                                     (torch.float32, torch.float32, "HSD"),
                                                     (torch.bfloat16, torch.float32, "SHD")])
def test_attend_tree(gpu, H, KVH, D, P, T, n, m, shape, q_dtype, out_dtype, layout):
    rng, g = random.Random(D + sum(T)), torch.Generator(device=gpu).manual_seed(D + sum(n))
    m = m or n
    K = [torch.randn(a + b, KVH, D, device=gpu, generator=g).bfloat16() for a, b in zip(T, n)]
    V = [torch.randn(a + b, KVH, D, device=gpu, generator=g).bfloat16() for a, b in zip(T, n)]
    q = [(torch.randn(k, H, D, device=gpu, generator=g) * 1.5).to(q_dtype) for k in m]
    trees = [_tree(shape, k, rng) for k in n]
    c = _cache(gpu, KVH, D, P, [a + b for a, b in zip(T, n)])
    _fill(c, K, V, P)
    order = list(range(len(T)))
    rng.shuffle(order)
    flat = torch.cat([(q[i].transpose(0, 1) if layout == "HSD" else q[i]).reshape(-1) for i in order])
    parents = torch.tensor(sum((trees[i] for i in order), []), dtype=torch.int32, device=gpu)
    guard = torch.full((flat.numel() + 64,), 7.0, dtype=out_dtype, device=gpu)  # behind the last row: left as it was
    c.AttendTree(0, flat, H, parents, seq_ids=order, n_nodes=[n[i] for i in order], n_q=[m[i] for i in order],
                 layout=layout, out=guard[:flat.numel()])
    assert (guard[flat.numel():] == 7.0).all()
    out, at = [], 0
    for i in order:
        part = guard[at:at + m[i] * H * D]
        out.append(part.view(H, m[i], D).transpose(0, 1) if layout == "HSD" else part.view(m[i], H, D))
        at += m[i] * H * D
    _check(torch.cat(out), [ref.attend(q[i], K[i], V[i], trees[i]) for i in order], out_dtype)
    c.close()


@pytest.mark.parametrize("H,KVH,D,T,n", [(8, 2, 128, 70, 40), (32, 8, 128, 8000, 33), (4, 4, 64, 10, 20),
                                         (8, 2, 256, 200, 9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("where", ["k", "v", "tail"])
def test_values_that_are_not_finite(gpu, H, KVH, D, T, n, dtype, where):
    """What a query does not attend does not reach it: infinities and NaN in other branches' keys and
    values, and in the slots behind the last token."""
    rng, g = random.Random(1), torch.Generator(device=gpu).manual_seed(2)
    K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    tree = _tree("random", n, rng)
    x = K if where == "k" else V
    c = _cache(gpu, KVH, D, 16, [T + n + 30])
    if where == "tail":
        bad = torch.full((30, KVH, D), math.nan, device=gpu).bfloat16()
        c.Append(0, torch.cat([K, bad]), torch.cat([V, bad]), n_tok=[T + n + 30], layout="SHD")
        c.Rollback(0, 30)
    else:
        for j, v in ((n - 1, math.nan), (n - 2, math.inf), (n // 2, -math.inf)):
            x[T + j, :, rng.randrange(D)] = v
        c.Append(0, K, V, n_tok=[T + n], layout="SHD")
    q = torch.randn(n, H, D, device=gpu, generator=g).to(dtype)
    out = c.AttendTree(0, q, H, torch.tensor(tree, dtype=torch.int32, device=gpu), out_dtype=dtype)
    want, size = ref.attend(q, K, V, tree)
    clean = torch.isfinite(want).all(dim=2)
    assert clean.any() and (where == "tail" or not clean.all())
    if where == "k":  # a query that attends such a key has no defined sum
        out, want, size = (torch.where(clean[..., None], t, torch.zeros_like(t)) for t in (out, want, size))
    _check(out, [(want, size)], dtype)
    c.close()


def test_scores_far_apart(gpu):
    """Weights between 2^-1000 and 1, the largest key late or early: the running maximum moves far."""
    g = torch.Generator(device=gpu).manual_seed(5)
    T, n, H, KVH, D = 3000, 17, 8, 2, 128
    K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    K[:, 0] *= torch.linspace(0.1, 30, T + n, device=gpu)[:, None].bfloat16()
    K[:, 1] *= torch.linspace(30, 0.1, T + n, device=gpu)[:, None].bfloat16()
    tree = _tree("random", n, random.Random(4))
    c = _cache(gpu, KVH, D, 16, [T + n])
    c.Append(0, K, V, n_tok=[T + n], layout="SHD")
    q = (torch.randn(n, H, D, device=gpu, generator=g) * 3).bfloat16()
    out = c.AttendTree(0, q, H, torch.tensor(tree, dtype=torch.int32, device=gpu), out_dtype=torch.bfloat16)
    _check(out, [ref.attend(q, K, V, tree)], torch.bfloat16)
    c.close()


def test_a_chain_is_causal_attention(gpu):
    """A tree without branches is what Attend computes, and an evicted sequence keeps its live tokens."""
    g = torch.Generator(device=gpu).manual_seed(6)
    H, KVH, D, T, n = 16, 4, 128, 400, 12
    K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c = _cache(gpu, KVH, D, 16, [T + n])
    c.Append(0, K, V, n_tok=[T + n], layout="SHD")
    c.Evict(0, 3)
    q = torch.randn(n, H, D, device=gpu, generator=g)
    parents = torch.arange(-1, n - 1, dtype=torch.int32, device=gpu)
    got, plain = c.AttendTree(0, q, H, parents), c.Attend(0, q, H, n_q=[n])
    assert (got - plain).abs().max() <= 2e-2  # Attend rounds queries and weights to bf16
    _check(got, [ref.attend(q, K[48:], V[48:], parents.tolist())], torch.float32)
    c.close()


def test_attend_tree_in_a_graph(gpu):
    """A captured call replayed on changed queries, trees and cache bytes."""
    g = torch.Generator(device=gpu).manual_seed(8)
    H, KVH, D, T, n = 32, 8, 128, 5000, 24
    K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c = _cache(gpu, KVH, D, 16, [T + n])
    c.Append(0, K, V, n_tok=[T + n], layout="SHD")
    q, rng = torch.zeros(n, H, D, device=gpu, dtype=torch.bfloat16), random.Random(3)
    parents, out = torch.zeros(n, dtype=torch.int32, device=gpu), torch.zeros_like(q)
    c.AttendTree(0, q, H, parents, out=out)  # the workspace is there
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    c.use_stream(stream)
    with torch.cuda.graph(graph, stream=stream):
        c.AttendTree(0, q, H, parents, out=out)
    for _ in range(3):
        tree = _tree("random", n, rng)
        q.copy_(torch.randn(n, H, D, device=gpu, generator=g))
        parents.copy_(torch.tensor(tree, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, [ref.attend(q, K, V, tree)], torch.bfloat16)
    c.close()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [6, 70])
def test_queries_and_outputs_off_alignment(gpu, dtype, n):
    g = torch.Generator(device=gpu).manual_seed(n)
    H, KVH, D, T = 8, 2, 64, 500
    K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c = _cache(gpu, KVH, D, 16, [T + n])
    c.Append(0, K, V, n_tok=[T + n], layout="SHD")
    par = torch.arange(-1, n - 1, dtype=torch.int32, device=gpu)
    buf = torch.randn(n * H * D + 1, device=gpu, generator=g).to(dtype)
    out = torch.full((n * H * D + 3,), 5.0, device=gpu, dtype=dtype)
    c.AttendTree(0, buf[1:], H, par, out=out[1:-2])
    assert torch.equal(out[1:-2], c.AttendTree(0, buf[1:].clone(), H, par, out_dtype=dtype))
    assert out[0] == 5.0 and (out[-2:] == 5.0).all()
    c.close()


def test_tree_after_evicted_pages(gpu):
    """A sequence whose first pages are gone: the tree attends what is left, the kept path stands behind it."""
    g, rng = torch.Generator(device=gpu).manual_seed(6), random.Random(6)
    H, KVH, D, T, n = 8, 4, 64, 200, 30
    K, V = (torch.randn(T + n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    c = _cache(gpu, KVH, D, 16, [T + n])
    c.Append(0, K[:T], V[:T], n_tok=[T], layout="SHD")
    c.Evict(0, 3)
    c.Append(0, K[T:], V[T:], n_tok=[n], layout="SHD")
    tree = _tree("random", n, rng)
    q = torch.randn(n, H, D, device=gpu, generator=g)
    got = c.AttendTree(0, q, H, torch.tensor(tree, dtype=torch.int32, device=gpu))
    _check(got, [ref.attend(q, K[48:], V[48:], tree)], torch.float32)
    path = ref.ancestors(tree, n - 1)[::-1]
    c.KeepPath(0, n, path)
    k, v = c.View(0)
    keep = list(range(48, T)) + [T + j for j in path]
    assert torch.equal(k[0].transpose(0, 1), K[keep]) and torch.equal(v[0].transpose(0, 1), V[keep])
    c.close()


# ---- rotary positions --------------------------------------------------------------------

@pytest.mark.parametrize("rows,heads,D,rd", [(1, 1, 2, 2), (3, 5, 8, 8), (16, 40, 128, 128), (7, 3, 80, 32),
                                             (33, 9, 96, 48), (129, 2, 20, 10), (5, 4, 7, 6), (4, 2, 16, 0),
                                             (1000, 33, 256, 256), (3001, 8, 64, 64)])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotate(gpu, rows, heads, D, rd, halves, dtype):
    from relux_amd import rope_frequencies
    g = torch.Generator(device=gpu).manual_seed(rows + D)
    inv, scale = rope_frequencies(rd, 10000.0, dict(type="yarn", factor=8.0, original=4096), gpu) if rd \
        else (torch.zeros(0, device=gpu), 1.0)
    pos = torch.randint(-1000, 1000000, (rows,), device=gpu, generator=g, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    pos[-1] = 0 if rows == 1 else -2 ** 31
    x = torch.randn(rows, heads, D, device=gpu, generator=g).to(dtype)
    c = _cache(gpu, 1, 64, 16, [16])
    layout = "halves" if halves else "pairs"
    want = ref.rotate(x, pos, inv, halves, scale)
    # the pair's products and sum in f32, the angle within 2^-22, the output by half a step
    size = x.double().abs().amax(dim=-1, keepdim=True) * scale * 2
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -21 * size
    got = c.Rotate(x, pos, inv, layout=layout, scale=scale)
    assert ((got.double() - want).abs() <= tol).all()
    if rd < D:
        assert torch.equal(got[..., rd:], x[..., rd:])
    # strided heads, an odd storage offset, other memory left as it was; in place
    for off, pad in ((0, 8), (1, 3)):
        buf = torch.full((rows * (heads * (D + pad) + pad) + off,), 3.0, dtype=dtype, device=gpu)
        view = buf[off:].view(rows, heads * (D + pad) + pad)[:, :heads * (D + pad)].unflatten(1, (heads, D + pad))
        view = view[..., :D]
        c.Rotate(x, pos, inv, layout=layout, scale=scale, out=view)
        assert torch.equal(view, got)
        view.fill_(3.0)
        assert (buf == 3.0).all()
        view.copy_(x)
        assert c.Rotate(view, pos, inv, layout=layout, scale=scale, out=view).data_ptr() == view.data_ptr()
        assert torch.equal(view, got)
    t = x.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    assert torch.equal(c.Rotate(t, pos, inv, layout=layout, scale=scale), got)
    c.close()


def test_rotation_gradient(gpu):
    """The rotation by negated positions is the gradient: the formula's, and differences in f64."""
    from relux_amd import rope_frequencies
    g = torch.Generator(device=gpu).manual_seed(9)
    inv, _ = rope_frequencies(16, 10000.0, None, gpu)
    pos = torch.randint(0, 5000, (6,), device=gpu, generator=g, dtype=torch.int32)
    c = _cache(gpu, 1, 64, 16, [16])
    for halves in (False, True):
        x, w = (torch.randn(6, 3, 24, device=gpu, generator=g) for _ in range(2))
        grad = c.Rotate(w, -pos, inv, layout="halves" if halves else "pairs", scale=1.5)
        leaf = x.double().requires_grad_()
        a = pos.double()[:, None] * inv.double()[None]
        cs, sn = torch.cos(a)[:, None] * 1.5, torch.sin(a)[:, None] * 1.5
        x0, x1 = (leaf[..., :8], leaf[..., 8:16]) if halves else (leaf[..., :16:2], leaf[..., 1:16:2])
        w0, w1 = (w[..., :8], w[..., 8:16]) if halves else (w[..., :16:2], w[..., 1:16:2])
        ((x0 * cs - x1 * sn) * w0 + (x0 * sn + x1 * cs) * w1).sum().add((leaf[..., 16:] * w[..., 16:]).sum()).backward()
        assert (grad.double() - leaf.grad).abs().max() <= 2.0 ** -20 * 4 * 1.5
        step = torch.zeros_like(x, dtype=torch.float64)
        step[2, 1, 5] = 1e-4
        f = [(ref.rotate(x.double() + k * step, pos, inv, halves, 1.5) * w.double()).sum() for k in (1, -1)]
        assert abs(float(f[0] - f[1]) / 2e-4 - float(grad[2, 1, 5])) <= 1e-4
    c.close()


def test_rotate_is_the_fused_step_s_rotation(gpu):
    """Where ProjectAppend's tables reach, Rotate gives the same rows up to the tables' f32 angles."""
    from relux_amd import rope_frequencies, rope_tables
    g = torch.Generator(device=gpu).manual_seed(10)
    x = torch.randn(50, 4, 64, device=gpu, generator=g)
    inv, _ = rope_frequencies(64, 10000.0, None, gpu)
    pos = torch.arange(50, dtype=torch.int32, device=gpu)
    cos, sin = rope_tables(64, 10000.0, 50, gpu)
    x0, x1 = x[..., 0::2], x[..., 1::2]
    want = torch.stack([x0 * cos[:, None] - x1 * sin[:, None], x0 * sin[:, None] + x1 * cos[:, None]], -1).flatten(-2)
    c = _cache(gpu, 1, 64, 16, [16])
    # angles up to 50 rounded to f32 twice, and frequencies by two roundings: 50 * 3 * 2^-24
    assert (c.Rotate(x, pos, inv) - want).abs().max() <= 50 * 4 * 2.0 ** -24 * 2 * float(x.abs().max())
    c.close()


# ---- acceptance ----------------------------------------------------------------------------

def _drafts(B, V, n, T, draft, seed, gpu, spread=3.0):
    rng, gen = random.Random(seed), np.random.default_rng(seed)
    sizes = [n if isinstance(n, int) else rng.randint(*n) for _ in range(B)]
    trees = [_tree("random", k, rng) for k in sizes]
    rows = sum(sizes)
    d = (gen.standard_normal((rows, V)) * spread).astype(np.float32)
    t = (d + gen.standard_normal((rows, V)) * 0.8).astype(np.float32)
    tok, at = np.zeros(rows, np.int32), 0
    for p in trees:
        for j in range(len(p)):
            kids = [c for c in range(len(p)) if p[c] == j]
            noisy = d[at + j] / T + gen.gumbel(size=V)
            tok[[at + c for c in kids]] = np.argsort(-noisy)[np.arange(len(kids)) % V]
        at += len(p)
    u = gen.random(rows, dtype=np.float32)
    return sizes, trees, t, d if draft else None, tok, u


def _accept(gpu, sizes, trees, t, d, tok, u, T, **kw):
    from relux_amd import Sampler, tree_accept
    c = _cache(gpu, 1, 64, 16, [16])
    to = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(gpu)
    got = tree_accept(c, to(t), to(tok), torch.tensor(sum(trees, []), dtype=torch.int32, device=gpu), sizes, to(u),
                      Sampler(temperature=T), draft_logits=to(d), **kw)
    c.close()
    return got


def _want(sizes, trees, t, d, tok, u, T):
    paths, nxt, at = [], [], 0
    for n, p in zip(sizes, trees):
        s = slice(at, at + n)
        path, x = ref.accept(t[s], tok[s], p, u[s], T, None if d is None else d[s])
        paths.append(path)
        nxt.append(x)
        at += n
    return paths, nxt


@pytest.mark.parametrize("B,V,n,T", [(1, 1, 1, 1.0), (3, 2, (1, 9), 1.0), (5, 7, (1, 40), 0.7), (4, 255, 20, 1.0),
                                     (9, 1000, (2, 64), 0.8), (3, 4097, 30, 1.0), (2, 32000, 33, 0.9),
                                     (2, 50257, 12, 1.0), (1, 128001, 9, 0.6), (1, 300, 256, 1.0),
                                     (300, 50, (1, 6), 1.0)])
@pytest.mark.parametrize("draft", [True, False])
def test_tree_accept(gpu, B, V, n, T, draft):
    case = _drafts(B, V, n, T, draft, V + B, gpu)
    assert _accept(gpu, *case, T) == _want(*case, T)


@pytest.mark.parametrize("draft", [True, False])
def test_tree_accept_emits_the_target_s_distribution(gpu, draft):
    """20000 trees of 6 nodes over 12 tokens: the first token after the root is distributed as the target
    alone would draw it, whichever way it came (chi-square of 11 degrees, 1 in 10^4: 37.4)."""
    gen, B, V, n = np.random.default_rng(11), 20000, 12, 6
    d1, t1 = gen.standard_normal(V) * 1.5, gen.standard_normal(V) * 1.5
    q = np.exp(d1) / np.exp(d1).sum()
    d, t = (np.broadcast_to(a.astype(np.float32), (B * n, V)) for a in (d1, t1))
    noisy = np.log(q) + gen.gumbel(size=(B, V))
    tok = np.zeros((B, n), np.int32)
    tok[:, 1:5] = np.argsort(-noisy, axis=1)[:, :4] if draft else np.argsort(-q)[:4]
    trees = [[-1, 0, 0, 0, 0, 1]] * B
    paths, nxt = _accept(gpu, [n] * B, trees, t, d if draft else None, tok.reshape(-1), gen.random(B * n, dtype=np.float32),
                         1.0)
    first = [tok[b, p[1]] if len(p) > 1 else x for b, (p, x) in enumerate(zip(paths, nxt))]
    want = np.exp(t1) / np.exp(t1).sum() * B
    chi = ((np.bincount(first, minlength=V) - want) ** 2 / want).sum()
    assert chi < 37.4, chi
    assert 0.2 * B < sum(len(p) > 1 for p in paths) < B


def test_tree_accept_edges(gpu):
    """Tokens of no vocabulary and repeated siblings are passed over, parents outside the tree make nodes
    unreachable, a sharp temperature is greedy, masked (-inf) entries are never drawn."""
    V, T = 40, 1.0
    gen = np.random.default_rng(12)
    t = (gen.standard_normal((8, V)) * 2).astype(np.float32)
    d = (t + gen.standard_normal((8, V))).astype(np.float32)
    t[:, 30:] = -np.inf
    for trial in range(40):
        tok = gen.integers(0, 30, 8).astype(np.int32)
        tok[2] = [-1, V, 1 << 30][trial % 3]
        tok[4] = tok[3]
        trees = [[-1, 0, 0, 0, 0, [5, -3, 8, 1 << 30][trial % 4], 3, 6]]
        u = gen.random(8, dtype=np.float32)
        for dd in (d, None):
            case = ([8], trees, t, dd, tok, u)
            got = _accept(gpu, *case, T)
            assert got == _want(*case, T)
            assert got[1][0] < 30
    best = t[:, :30].argmax(1)
    tok = np.array([0, (best[0] + 1) % 30, best[0], 1, best[2], 2, 3, best[4]], np.int32)
    trees = [[-1, 0, 0, 1, 2, 2, 4, 4]]
    for T in (0.0, 1e-3):
        paths, nxt = _accept(gpu, [8], trees, t, None, tok, np.full(8, 0.5, np.float32), T)
        assert paths == [[0, 2, 4, 7]] and nxt == [best[7]]
    # rows without probability: some token of the vocabulary
    for fill in (np.nan, -np.inf):
        paths, nxt = _accept(gpu, [8], trees, np.full_like(t, fill), d, tok, u, 1.0)
        assert 0 <= nxt[0] < V


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("mask", [-np.inf, np.finfo(np.float32).min])
def test_tree_accept_few_tokens_far_below_zero(gpu, mask, draft):
    """Rows of masked entries but for a few, whose logits lie hundreds below zero."""
    V, gen = 20000, np.random.default_rng(21)
    live = np.array([3, 4, 5, 4940, 4941, 9999, 19990, 19999])
    for trial in range(20):
        t, d = (np.full((9, V), mask, np.float32) for _ in range(2))
        t[:, live] = gen.standard_normal((9, 8)) - 700
        d[:, live] = t[:, live] + 0.5 * gen.standard_normal((9, 8))
        tok = gen.choice(live, 9).astype(np.int32)
        case = ([9], [[-1, 0, 0, 0, 1, 1, 2, 4, 4]], t, d if draft else None, tok, gen.random(9, dtype=np.float32))
        assert _accept(gpu, *case, 1.0) == _want(*case, 1.0)


def test_tree_accept_strided_rows_and_guards(gpu):
    from relux_amd import Sampler, tree_accept_async
    sizes, trees, t, d, tok, u = _drafts(5, 333, (3, 20), 1.0, True, 77, gpu)
    c = _cache(gpu, 1, 64, 16, [16])
    rows, to = sum(sizes), lambda a: torch.from_numpy(a).to(gpu)
    wide = torch.randn(2, rows, 400, device=gpu)
    wide[0, :, 5:338], wide[1, :, 5:338] = to(t), to(d)
    path, acc, nxt = (torch.full((s,), 99, dtype=torch.int32, device=gpu) for s in (6 * 30, 6, 6))
    tree_accept_async(c, wide[0, :, 5:338], to(tok), torch.tensor(sum(trees, []), dtype=torch.int32, device=gpu),
                      sizes, to(u), Sampler(), draft_logits=wide[1, :, 5:338], path=path[:150].view(5, 30),
                      n_acc=acc[:5], next_tok=nxt[:5])
    c.Sync()
    paths, want = _want(sizes, trees, t, d, tok, u, 1.0)
    assert path[:150].view(5, 30).tolist() == [p + [-1] * (30 - len(p)) for p in paths]
    assert acc.tolist() == [len(p) - 1 for p in paths] + [99] and nxt.tolist() == want + [99]
    assert (path[150:] == 99).all()
    c.close()


# ---- kept paths ------------------------------------------------------------------------------

def _state(c, layers, seqs):
    return [(c.SeqState(l, s), c.PageTable(l, s)) for l in range(layers) for s in seqs] + \
        [c.FreeList(l) for l in range(layers)]


@pytest.mark.parametrize("KVH,D,P,T,n", [(8, 128, 16, [200], [8]), (2, 64, 16, [0, 15, 31], [1, 33, 64]),
                                         (1, 16, 16, [3], [40]), (4, 80, 48, [47, 100], [50, 7]),
                                         (2, 256, 32, [33], [256]), (4, 20, 16, [10, 0], [20, 3]),
                                         (8, 128, 16, [30 + i for i in range(12)], [20] * 12)])
@pytest.mark.parametrize("levels", [1, 2])
def test_keep_path(gpu, KVH, D, P, T, n, levels):
    """The cache after a kept path is the cache that was given the kept tokens alone: bytes, tables, free
    lists, append history."""
    from relux_amd import KVCache
    layers, g, rng = 3, torch.Generator(device=gpu).manual_seed(D), random.Random(D + P)
    B = len(T)
    make = lambda: KVCache(num_layers=layers, max_len=max(a + b for a, b in zip(T, n)) + P, num_kv_heads=KVH,
                           head_dim=D, page_tokens=P, max_seqs=B, device=gpu.index)
    a, b = make(), make()
    seqs = list(range(B))
    paths = []
    for k in n:
        p = ref.ancestors(_tree("random", k, rng), rng.randrange(k))[::-1]
        paths.append(rng.choice([p, p, p[:1], [], list(range(k)), sorted(rng.sample(range(k), rng.randint(0, k)))]))
    paths[0] = sorted(rng.sample(range(n[0]), max(1, n[0] // 2)))
    for layer in range(layers):
        K, V = (torch.randn(sum(T) + sum(n), KVH, D, device=gpu, generator=g) for _ in range(2))
        ctx = [i for i in seqs if T[i]]
        at = np.cumsum([0] + T + n).tolist()
        take = lambda x, i: x[at[i]:at[i + 1]]
        for c in (a, b):
            if ctx:
                c.Append(layer, torch.cat([take(K, i) for i in ctx]), torch.cat([take(V, i) for i in ctx]),
                         seq_ids=ctx, n_tok=[T[i] for i in ctx], layout="SHD")
        cut = [k // 2 if levels == 2 else 0 for k in n]
        for lo, hi in ((0, 1), (1, 2)):
            ends = [[0, x, k] for x, k in zip(cut, n)]
            m = [e[hi] - e[lo] for e in ends]
            if sum(m):
                a.Append(layer, torch.cat([take(K, B + i)[ends[i][lo]:ends[i][hi]] for i in seqs]),
                         torch.cat([take(V, B + i)[ends[i][lo]:ends[i][hi]] for i in seqs]), seq_ids=seqs, n_tok=m,
                         layout="SHD")
        kept = [i for i in seqs if paths[i]]
        b.Append(layer, torch.cat([take(K, B + i)[paths[i]] for i in kept]),
                 torch.cat([take(V, B + i)[paths[i]] for i in kept]), seq_ids=kept, n_tok=[len(paths[i]) for i in kept],
                 layout="SHD")
    if B == 1:
        a.KeepPath(0, n[0], paths[0])
    else:
        a.KeepPath(seqs, n, paths)
    for layer in range(layers):
        for i in seqs:
            for x, y in zip(a.View(layer, i), b.View(layer, i)):
                assert (x is None and y is None) or torch.equal(x.view(torch.int16), y.view(torch.int16))
    for i in seqs:  # (pages of a batch are handed out in another order)
        for layer in range(layers):
            x, y = a.SeqState(layer, i), b.SeqState(layer, i)
            assert x == y
            assert sum(p >= 0 for p in a.PageTable(layer, i)) == y["pages"]
            assert len(a.FreeList(layer)) == len(b.FreeList(layer))
    if B == 1:
        assert _state(a, layers, seqs) == _state(b, layers, seqs)
    if D % 8 == 0 and all(paths[i] != list(range(n[i])) or levels == 1 for i in seqs):
        live = [i for i in seqs if T[i] + len(paths[i])]
        q = torch.randn(len(live), KVH, D, device=gpu, generator=g)
        assert torch.equal(a.AttendRefImage(0, q, KVH, seq_ids=live), b.AttendRefImage(0, q, KVH, seq_ids=live))
    a.close()
    b.close()


def test_keep_path_one_layer_and_the_step_after(gpu):
    """A single layer's path; then the next tree's attention over what was kept."""
    g = torch.Generator(device=gpu).manual_seed(14)
    H, KVH, D, T, n = 8, 2, 128, 50, 30
    K, V = (torch.randn(T + 2 * n, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
    from relux_amd import KVCache
    c = KVCache(num_layers=2, max_len=200, num_kv_heads=KVH, head_dim=D, max_seqs=1, device=gpu.index)
    for layer in (0, 1):
        c.Append(layer, K[:T + n], V[:T + n], n_tok=[T + n], layout="SHD")
    path = [0, 2, 5, 11, 29]
    c.KeepPath(0, n, path, layer=1)
    assert [c.TotalLen(layer) for layer in (0, 1)] == [T + n, T + len(path)]
    c.Append(1, K[T + n:], V[T + n:], n_tok=[n], layout="SHD")
    tree = _tree("random", n, random.Random(2))
    rows = list(range(T)) + [T + j for j in path] + list(range(T + n, T + 2 * n))
    q = torch.randn(n, H, D, device=gpu, generator=g).bfloat16()
    out = c.AttendTree(1, q, H, torch.tensor(tree, dtype=torch.int32, device=gpu), out_dtype=torch.bfloat16)
    _check(out, [ref.attend(q, K[rows], V[rows], tree)], torch.bfloat16)
    c.close()


@pytest.mark.parametrize("T", [1, 3, 8, 9])
def test_gather_of_a_few_tokens(gpu, T):
    g = torch.Generator(device=gpu).manual_seed(T)
    for KVH, D in ((1, 16), (1, 8), (3, 64)):
        K, V = (torch.randn(T, KVH, D, device=gpu, generator=g).bfloat16() for _ in range(2))
        c = _cache(gpu, KVH, D, 16, [T])
        c.Append(0, K, V, n_tok=[T], layout="SHD")
        k, v = c.View(0)
        assert torch.equal(k[0].transpose(0, 1), K) and torch.equal(v[0].transpose(0, 1), V)
        c.close()


# ---- refusals ----------------------------------------------------------------------------------

def test_refusals(gpu):
    from relux_amd import KVCache, MLACache, ReluxError, ReluxPanic, Sampler, tree_accept_async
    c = KVCache(num_layers=2, max_len=400, num_kv_heads=2, head_dim=64, max_seqs=2, device=gpu.index)
    k = torch.randn(300, 2, 64, device=gpu)
    for layer in (0, 1):
        c.Append(layer, k, k, n_tok=[300], layout="SHD")
    q, par = torch.randn(4, 4, 64, device=gpu), torch.full((4,), -1, dtype=torch.int32, device=gpu)
    before = _state(c, 2, [0, 1])
    with pytest.raises(ReluxPanic):
        c.AttendTree(2, q, 4, par)
    with pytest.raises(ReluxError, match="holding 0"):
        c.AttendTree(0, q, 4, par, seq_ids=[1])
    with pytest.raises(ReluxError, match="listed twice"):
        c.AttendTree(0, q, 4, par, seq_ids=[0, 0], n_nodes=[2, 2])
    with pytest.raises(ReluxError, match="divisible"):
        c.AttendTree(0, q.view(4 * 4 // 1, 1, 64)[:9].contiguous(), 3, par[:3])
    with pytest.raises(ReluxError, match="overlap"):
        c.AttendTree(0, q, 4, par, out=q)
    for kw in (dict(n_nodes=[0]), dict(n_nodes=[257]), dict(n_q=[5]), dict(n_q=[0])):
        with pytest.raises(ValueError):
            c.AttendTree(0, q, 4, par, **kw)
    with pytest.raises(TypeError):
        c.AttendTree(0, q, 4, par.long())
    with pytest.raises(TypeError):
        c.AttendTree(0, q, 4, par.cpu())
    with pytest.raises(TypeError):
        c.AttendTree(0, q.half(), 4, par)
    for n, path in ((301, [0]), (4, [0, 4]), (4, [0, 0]), (4, [2, 1]), (4, [-1]), (4, [0, 1, 2, 3, 4]), (-1, [])):
        with pytest.raises(ReluxError):
            c.KeepPath(0, n, path)
    with pytest.raises(ReluxError):
        c.KeepPath([0, 0], [4, 4], [[0], [0]])
    with pytest.raises(ReluxPanic):
        c.KeepPath(0, 4, [0], layer=2)
    m = MLACache(num_layers=1, max_len=64, device=gpu.index)
    with pytest.raises(ReluxError, match="MLA"):
        KVCache.KeepPath(m, 0, 0, [])
    assert _state(c, 2, [0, 1]) == before
    x, pos = torch.randn(6, 2, 8, device=gpu), torch.zeros(6, dtype=torch.int32, device=gpu)
    inv = torch.ones(4, device=gpu)
    with pytest.raises(ReluxError, match="overlap"):
        c.Rotate(x[:5], pos[:5], inv, out=x[1:])
    with pytest.raises(ReluxError, match="strides"):
        c.Rotate(x, pos, inv, out=torch.empty(6, 1, 8, device=gpu).expand(6, 2, 8))
    with pytest.raises(ValueError):
        c.Rotate(x, pos, torch.ones(5, device=gpu))
    with pytest.raises(ValueError):
        c.Rotate(x, pos, inv, layout="both")
    with pytest.raises(ValueError):
        c.Rotate(x.transpose(1, 2), pos, inv)
    with pytest.raises(TypeError):
        c.Rotate(x, pos.long(), inv)
    with pytest.raises(TypeError):
        c.Rotate(x, pos, inv.double())
    t, tok, u = torch.randn(4, 10, device=gpu), par.clone(), torch.rand(4, device=gpu)
    for s in (Sampler(top_k=3), Sampler(top_p=0.5), Sampler(min_p=0.1), Sampler(repeat_penalty=1.2)):
        with pytest.raises(ReluxError, match="temperature"):
            tree_accept_async(c, t, tok, par, [4], u, s)
    for args in ((t.double(), tok, par, [4], u), (t, tok.long(), par, [4], u), (t, tok, par[:3], [4], u),
                 (t, tok, par, [4], u.double())):
        with pytest.raises(TypeError):
            tree_accept_async(c, *args, Sampler())
    for n in ([3], [0, 4], [257]):
        with pytest.raises((ValueError, TypeError)):
            tree_accept_async(c, t, tok, par, n, u, Sampler())
    c.close()
    m.close()
