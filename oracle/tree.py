"""Trees of drafts in 64 bits, from the definitions: rotary positions, tree
attention, the acceptance walk."""
import math

import numpy as np
import torch


def ancestors(parents, j):
    """Node j and the nodes above it; a parent outside [0, j) ends the chain."""
    out = [j]
    while 0 <= parents[j] < j:
        j = parents[j]
        out.append(j)
    return out


def rotate(x, positions, inv_freq, halves, scale=1.0):
    """x [rows, heads, D] (any type) -> f64; inv_freq as f32 values."""
    x = x.double().clone()
    rd = 2 * inv_freq.numel()
    a = positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = (torch.cos(a) * scale)[:, None], (torch.sin(a) * scale)[:, None]
    if halves:
        i0, i1 = slice(0, rd // 2), slice(rd // 2, rd)
    else:
        i0, i1 = slice(0, rd, 2), slice(1, rd, 2)
    x0, x1 = x[..., i0].clone(), x[..., i1].clone()
    x[..., i0], x[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    return x


def attend(q, K, V, parents, scale=None):
    """q [m, H, D]: the last m nodes; K, V [T, KVH, D], the last len(parents) of T
    tokens the nodes.  Returns (out, sum of w |v|), f64 [m, H, D]: a masked key has
    no part in either, whatever it holds."""
    m, H, D = q.shape
    T, KVH, _ = K.shape
    n, G = len(parents), H // KVH
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(m, H, D, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    see = torch.zeros(m, T, dtype=torch.bool)
    see[:, :T - n] = True
    for i in range(m):
        see[i, [T - n + a for a in ancestors(parents, n - m + i)]] = True
    see = see.to(q.device)
    for h in range(KVH):
        k, v = K[:, h].double(), V[:, h].double()
        qh = q[:, h * G:(h + 1) * G].double().reshape(m * G, D)
        s = (torch.matmul(qh, k.t().contiguous()) * scale).view(m, G, T)
        s = torch.where(see[:, None, :], s, torch.full_like(s, -math.inf))
        w = torch.softmax(s, dim=-1)
        plain = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
        o = torch.matmul(w.view(m * G, T), plain).view(m, G, D)
        size[:, h * G:(h + 1) * G] = torch.matmul(w.view(m * G, T), plain.abs()).view(m, G, D)
        for t in torch.nonzero(~torch.isfinite(v).all(dim=1)).flatten().tolist():
            add = torch.where(torch.isfinite(v[t]), torch.zeros_like(v[t]), v[t])
            o = torch.where(see[:, t, None, None], o + add, o)
        out[:, h * G:(h + 1) * G] = o
    return out, size


def accept(t_logits, tokens, parents, uniforms, temperature, d_logits=None):
    """One tree (numpy arrays): (path, next token), the residual distributions
    written out and rescaled after every rejection."""
    temp = np.float64(np.float32(temperature))

    def probs(row):
        x = np.asarray(row, np.float64) / temp
        x = np.exp(x - x.max())
        return x / x.sum()

    n, V = t_logits.shape
    node, path = 0, [0]
    while True:
        p = probs(t_logits[node])
        q = probs(d_logits[node]) if d_logits is not None else None
        went, gone = None, set()
        for c in range(node + 1, n):
            x = int(tokens[c])
            if parents[c] != node or not 0 <= x < V or x in gone:
                continue
            u = np.float64(uniforms[c])
            if u * (q[x] if q is not None else 1.0) < p[x]:
                went = c
                break
            gone.add(x)
            if q is None:
                p[x] = 0.0
            else:
                p = np.maximum(p - q, 0.0)
                q[x] = 0.0
                if q.sum() > 0:
                    q = q / q.sum()
            p = p / p.sum()
        if went is None:
            break
        node = went
        path.append(node)
    cum = np.cumsum(p)
    nxt = min(int(np.searchsorted(cum, np.float64(uniforms[0]) * cum[-1], side="right")), V - 1)
    return path, nxt
