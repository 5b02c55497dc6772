"""A plain model of speculative decoding over trees, one sequence and one row
after the other, in 64 bits: what the kernels of include/ecf8_draft.h are
compared with."""

from __future__ import annotations

import math

import torch

D = 128


def random_tree(rng, n, kids, chain=False):
    """Parents of n rows: row 0 has none, the others an earlier row, at most
    ``kids`` the same."""
    parents, count = [-1] * min(n, 1), [0] * n
    for i in range(1, n):
        p = i - 1 if chain else rng.randrange(i)
        if count[p] >= kids:
            p = i - 1
        count[p] += 1
        parents.append(p)
    return parents


def masks(parents):
    """Each row's ancestors and itself, as bits."""
    out = []
    for i, p in enumerate(parents):
        out.append(1 << i | (out[p] if p >= 0 else 0))
    return out


def signed(bits):
    """64 bits as an int64 holds them."""
    return bits - 2 ** 64 if bits >= 2 ** 63 else bits


def verify(parents, tokens, target, accept, sample, draft=None):
    """(path, emitted) of one sequence; target, draft float64 [n, V]."""
    here, path, emitted = 0, [0], []
    while True:
        w, mass = target[here].clone(), 1.0
        for c in (i for i, p in enumerate(parents) if p == here):
            t = tokens[c]
            if draft is None:
                ok = accept[c] * mass < w[t]
            else:
                ok = accept[c] * draft[here, t] * mass < w[t]
            if ok:
                here = c
                path.append(c)
                emitted.append(t)
                break
            if draft is None:
                mass -= float(w[t])
                w[t] = 0.0
            else:
                w = (w / mass - draft[here]).clamp(min=0)
                mass = float(w.sum())
        else:
            if not float(w.sum()) > 0:
                w = target[here]
            upto = torch.cumsum(w, 0)
            emitted.append(int((upto > sample * float(w.sum())).nonzero()[0]))
            return path, emitted


def attention(q, k, v, seen):
    """q [n, Hq, D], k and v [L, Hkv, D] float64, seen [n, L]: the outputs and the
    sums of |p v| that their error is in proportion to, [n, Hq, D]; zeros where
    nothing is seen."""
    G = q.shape[1] // k.shape[1]
    k, v = (t.repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))
    e = q.transpose(0, 1) @ k.transpose(1, 2).contiguous() / math.sqrt(D)
    e = e.masked_fill(~seen, -math.inf)
    p = torch.softmax(e, -1).masked_fill(~seen.any(-1)[:, None], 0.0)
    return (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
