"""Trees of drafts without a GPU: frequencies, refusals before the library, the
decoder's bookkeeping over a model of plain tables, and the plans of the tree
attention (relux_amd/csrc/rlx_tree_plan.h)."""
import math
import os
import subprocess

import numpy as np
import pytest
import torch

from oracle import tree as ref
from relux_amd import Draws, KVCache, Sampler, TreeSpeculativeDecoder, rope_frequencies, sampling, tree_accept_async

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "relux_amd", "csrc")


def test_rope_frequencies():
    inv, scale = rope_frequencies(128, 10000.0)
    want = np.float64(10000.0) ** (-2.0 * np.arange(64) / 128)
    assert scale == 1.0 and inv.dtype == torch.float32
    np.testing.assert_array_equal(inv.numpy(), want.astype(np.float32))
    lin, s = rope_frequencies(128, 10000.0, dict(type="linear", factor=4.0))
    np.testing.assert_allclose(lin.numpy(), want / 4, rtol=2.0 ** -23)
    assert s == 1.0
    ntk, s = rope_frequencies(128, 10000.0, dict(type="ntk", factor=4.0))
    np.testing.assert_allclose(ntk.numpy()[[0, 63]], [1.0, want[63] / 4], rtol=1e-6)  # fastest as it was, slowest / 4
    yarn, s = rope_frequencies(128, 10000.0, dict(type="yarn", factor=4.0, original=4096))
    turns = 4096 * want / (2 * math.pi)
    kept, cut = turns > 40, turns < 0.8
    np.testing.assert_allclose(yarn.numpy()[kept], want[kept], rtol=2.0 ** -23)
    np.testing.assert_allclose(yarn.numpy()[cut], want[cut] / 4, rtol=2.0 ** -23)
    mid = yarn.numpy()[~kept & ~cut] / want[~kept & ~cut]
    assert (np.diff(mid) <= 0).all() and mid.min() >= 0.25 and mid.max() <= 1.0
    assert s == pytest.approx(0.1 * math.log(4.0) + 1.0)


@pytest.mark.parametrize("args", [(0,), (7,), (8, 1.0), (8, 10000.0, dict(type="linear", factor=0.5)),
                                  (8, 10000.0, dict(type="other", factor=2.0))])
def test_rope_frequencies_refusals(args):
    with pytest.raises(ValueError):
        rope_frequencies(*args)


def _no_gpu_cache(**kw):
    """A cache object without a handle: what it refuses, it refuses before the library."""
    c = KVCache.__new__(KVCache)
    c._h, c._lib, c.device, c.num_kv_heads, c.head_dim = None, None, torch.device("cpu"), 2, 8
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_refusals_before_the_library():
    c = _no_gpu_cache()
    x, pos, inv = torch.zeros(3, 2, 8), torch.zeros(3, dtype=torch.int32), torch.ones(4)
    for args, kw, err in (((x[0], pos, inv), {}, ValueError), ((x, pos, inv), dict(layout="neox"), ValueError),
                          ((x, pos, torch.ones(5)), {}, ValueError), ((x, pos, inv.double()), {}, TypeError),
                          ((x, pos.long(), inv), {}, TypeError), ((x, pos[:2], inv), {}, TypeError),
                          ((x, pos, inv), dict(out=x[:2]), ValueError), ((x.transpose(1, 2), pos, inv), {}, ValueError),
                          ((x.half(), pos, inv), {}, TypeError)):
        with pytest.raises(err):
            c.Rotate(*args, **kw)
    q, par = torch.zeros(4, 4, 8), torch.full((4,), -1, dtype=torch.int32)
    for kw in (dict(n_nodes=[0]), dict(n_nodes=[257]), dict(n_q=[5]), dict(n_q=[0]), dict(seq_ids=[0, 1]),
               dict(seq_ids=[0, 1], n_nodes=[4]), dict(out=torch.zeros(3)), dict(n_nodes=[5])):
        with pytest.raises((ValueError, TypeError)):
            c.AttendTree(0, q, 4, par, **kw)
    with pytest.raises(ValueError):
        c.KeepPath([0, 1], [4], [[0]])
    t, tok, u = torch.zeros(4, 10), par, torch.zeros(4)
    for args, kw in (((t, tok, par, [3], u), {}), ((t, tok, par, [0, 4], u), {}), ((t, tok, par, [257], u), {}),
                     ((t.double(), tok, par, [4], u), {}), ((t, tok, par, [4], u), dict(draft_logits=t[:, :9])),
                     ((t, tok, par, [4], u), dict(path=torch.zeros(1, 3, dtype=torch.int32))),
                     ((t, tok.long(), par, [4], u), {}), ((t.t(), tok, par, [4], u), {})):
        with pytest.raises((ValueError, TypeError)):
            tree_accept_async(c, *args, Sampler(), **kw)
    for kw in (dict(widths=()), dict(widths=(0,)), dict(branch=0), dict(widths=(200, 56))):
        with pytest.raises(ValueError):
            TreeSpeculativeDecoder(None, None, **kw)


class _Table:
    """A model whose next-token logits depend on the last two tokens."""

    def __init__(self, V, seed, near=None):
        g = np.random.default_rng(seed)
        self.w = g.standard_normal((V, V, V)) * 2
        if near is not None:
            self.w = near.w + self.w * 0.4
        self.seq, self.tree, self.cache = [], 0, None

    def reset(self):
        self.seq, self.tree = [], 0

    def _row(self, ctx):
        a, b = ([0, 0] + ctx)[-2:]
        return torch.from_numpy(self.w[a, b].astype(np.float32))

    def forward(self, ids):
        out = []
        for x in ids:
            self.seq.append(x)
            out.append(self._row(self.seq))
        return torch.stack(out)

    def forward_tree(self, ids, parents, depths, n_new):
        assert self.tree == len(ids) - n_new  # the earlier nodes are here already
        self.tree = len(ids)
        out = []
        for j in range(len(ids) - n_new, len(ids)):
            up = ref.ancestors(parents, j)[::-1]
            assert depths[j] == len(up) - 1
            out.append(self._row(self.seq + [ids[a] for a in up]))
        self.ids = list(ids)
        return torch.stack(out)

    def keep_path(self, n_nodes, path):
        assert n_nodes == self.tree and path[0] == 0 and all(a < b for a, b in zip(path, path[1:]))
        self.seq += [self.ids[j] for j in path]
        self.tree = 0


def _plain_accept(cache, t, tok, parents, n_nodes, u, sampler, draft_logits=None):
    path, nxt = ref.accept(t.numpy(), tok.numpy(), parents.tolist(), u.numpy(), max(sampler.Temperature, 1e-5),
                           draft_logits.numpy())
    return [path], [nxt]


@pytest.mark.parametrize("widths,branch", [((4, 4, 4, 2), 2), ((1, 1, 1), 1), ((3,), 3), ((2, 5), 4), ((30, 30), 8)])
def test_decoder_greedy_is_the_target_s(monkeypatch, widths, branch):
    monkeypatch.setattr(sampling, "tree_accept", _plain_accept)
    t = _Table(11, 1)
    d = _Table(11, 2, near=t)
    dec = TreeSpeculativeDecoder(d, t, widths=widths, branch=branch,
                                 sampling=Sampler(temperature=1e-3, rand=Draws(seed=3)))
    got, rate = dec.Generate([3, 1, 4], 40)
    plain = _Table(11, 1)
    plain.forward([3, 1])
    want, x = [], 4
    for _ in range(40):
        x = int(plain.forward([x])[-1].argmax())
        want.append(x)
    assert got == want and 0.0 < rate <= 1.0
    n = min(len(t.seq), 43)
    assert n > 3 and t.seq[:n] == ([3, 1, 4] + want)[:n]
    assert d.seq == t.seq  # both caches hold the committed tokens but the newest


def test_decoder_samples_the_target_s_distribution(monkeypatch):
    """First tokens of 3000 generations at temperature 1: chi-square of 6 degrees, 1 in 10^4: 27.9."""
    monkeypatch.setattr(sampling, "tree_accept", _plain_accept)
    t = _Table(7, 5)
    t.w *= 0.5
    d = _Table(7, 6, near=t)
    dec = TreeSpeculativeDecoder(d, t, widths=(3, 2), branch=2, sampling=Sampler(rand=Draws(seed=8)))
    n = 3000
    first = [dec.Generate([2, 5], 1)[0][0] for _ in range(n)]
    p = np.exp(t.w[2, 5].astype(np.float32).astype(np.float64))
    want = p / p.sum() * n
    assert ((np.bincount(first, minlength=7) - want) ** 2 / want).sum() < 27.9


def test_plans(tmp_path):
    """Every plan has a kernel and cuts no sequence into more parts than it has steps."""
    src = tmp_path / "plan.cpp"
    src.write_text("""
#include "rlx_tree_plan.h"
#include <cstdio>
#include <cstdlib>
int main() {
    srand(1);
    const int hds[] = {16, 32, 64, 96, 128, 256};
    for (int i = 0; i < 20000; i++) {
        std::vector<rlx::TreeLoad> load(1 + rand() % 70);
        const int span = 1 << rand() % 18, rows = 1 << rand() % 13;
        for (auto &l : load) l = {1 + rand() % span, 1 + rand() % rows};
        const int hd = hds[rand() % 6], kvh = 1 << rand() % 7;
        const bool fine = rand() % 2;
        const auto p = rlx::tree_plan(load, kvh, 256, hd, fine);
        if (!rlx::tree_has_tile(p.tile, hd, fine) || p.cuts.size() != load.size()) return printf("tile %d\\n", p.tile), 1;
        for (size_t k = 0; k < load.size(); k++)
            if (p.cuts[k] < 1 || p.cuts[k] > (load[k].len + 127) / 128) return printf("cuts %d\\n", p.cuts[k]), 1;
    }
    return 0;
}
""")
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", exe], check=True)
    r = subprocess.run([exe], stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stdout
