"""GPU numerics of the ragged-batch kernels (include/ecf8_paged.h) against a
plain model of the page bookkeeping and float64 restatements in torch.

Tolerance of the attention, per output o: probabilities are rounded to bf16
by factors 1 + d, |d| <= 2^-8 (half a step), in both sums, so that the quotient
is off by sum p d (v - o): at most 2^-8 of A = sum p |v| and of |o|.  The output
is rounded to bf16 (2^-8 of it).  The rest is fp32: a score's 128
products sum to within 128 * 2^-24 of sum |q k| / sqrt(128), below 64 here:
2^-11 in the exponent; sums of at most 2^12 terms are within 2^-12, the
exponential within 2^-20.  Together below 2^-10 of A."""

from __future__ import annotations

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _rand(*shape, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale).to(torch.bfloat16)


# ------------------------------------------------------------------ the plan


class Model:
    """The page bookkeeping, one sequence and one page after the other."""

    def __init__(self, seqs, pages, page, width):
        self.S, self.page, self.width = seqs, page, width
        self.stack = list(range(pages - 1, -1, -1))
        self.pages = [[] for _ in range(seqs)]

    def step(self, cached, new, release, rows):
        stack, held = list(self.stack), [list(p) for p in self.pages]
        for s in range(self.S):
            if release[s]:
                stack += held[s]
                held[s] = []
        slots, positions, starts = [], [], [0]
        ok = sum(new) <= rows
        for s in range(self.S):
            c, n = cached[s], new[s]
            if c < 0 or n < 0 or c + n > self.width * self.page:
                ok = False
                break
            while ok and len(held[s]) * self.page < c + n:
                if not stack:
                    ok = False
                    break
                held[s].append(stack.pop())
            if not ok:
                break
            for p in range(c, c + n):
                slots.append(held[s][p // self.page] * self.page + p % self.page)
                positions.append(p)
            starts.append(len(slots))
        if not ok:
            return dict(ok=False, starts=[0] * (self.S + 1), lengths=[0] * self.S,
                        slots=[-1] * rows, positions=[-1] * rows)
        self.stack, self.pages = stack, held
        pad = [-1] * (rows - len(slots))
        return dict(ok=True, starts=starts, lengths=[c + n for c, n in zip(cached, new)],
                    slots=slots + pad, positions=positions + pad)

    def table(self):
        return [p + [-1] * (self.width - len(p)) for p in self.pages]


@pytest.mark.parametrize("S,page,max_len,rows", [
    (1, 1, 40, 64), (1, 1024, 5000, 4096), (3, 16, 100, 200), (64, 16, 300, 4096),
    (65, 8, 130, 4097), (257, 64, 1000, 9000), (1025, 32, 200, 5000), (4096, 16, 64, 20000)])
def test_plan_matches_the_model(cuda_device, S, page, max_len, rows):
    """Steps of idle, running, finished, replaced and shortened sequences;
    steps that do not fit in between; each planned twice."""
    from ecf8_amd._lib import ECF8Error
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    rng = random.Random(S * 1000 + page)
    width = -(-max_len // page)
    pages = max(2, int(S * width * 0.7))
    b = PagedBatch(S, rows, pages, page, max_len, 8, 2, cuda_device)
    m = Model(S, pages, page, width)
    length = [0] * S
    refused = 0
    for k in range(12):
        room, cached, new, release = rows, [], [], []
        for s in range(S):
            out = rng.random() < 0.2
            c = 0 if out else length[s]
            if not out and rng.random() < 0.1:
                c = rng.randint(0, c)  # tokens taken back: the pages stay
            n = rng.choice([0, 1, 1, rng.randint(0, max_len)])
            n = min(n, width * page - c, room)
            room -= n
            cached.append(c), new.append(n), release.append(int(out))
        if k == 5:
            new[rng.randrange(S)] = -1
        if k == 7:
            cached[rng.randrange(S)] = width * page + 1
        want = m.step(cached, new, release, rows)
        refused += not want["ok"]
        for again in range(2):
            rel = _ints(release if not again else [0] * S, cuda_device)
            paged_plan(b, _ints(cached, cuda_device), _ints(new, cuda_device),
                       rel if any(release) else None)
            torch.cuda.synchronize()
            if want["ok"]:
                b.raise_refused()
            else:
                with pytest.raises(ECF8Error):
                    b.raise_refused()
            for name in ("starts", "lengths", "slots", "positions"):
                assert getattr(b, name).tolist() == want[name], (k, again, name)
            assert b.table.tolist() == m.table(), (k, again)
            assert b.owned.tolist() == [len(p) for p in m.pages]
            left = int(b.n_free)
            assert b.free[:left].tolist() == m.stack, (k, again)
        if want["ok"]:
            length = want["lengths"]
    assert 2 <= refused < 12
    held = sorted(p for q in m.pages for p in q) + sorted(m.stack)
    assert sorted(held) == list(range(pages))  # no page lost or held twice


def test_plan_refuses_a_full_step_and_takes_it_later(cuda_device):
    """Exactly enough rows and pages; one too many; then after a release."""
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    b = PagedBatch(2, 40, 4, 8, 40, 1, 1, cuda_device)

    def plan(cached, new, release=None):
        paged_plan(b, _ints(cached, cuda_device), _ints(new, cuda_device),
                   None if release is None else _ints(release, cuda_device))
        torch.cuda.synchronize()
        bad, b.refused[0] = int(b.refused[0]), 0
        return bad

    assert plan([0, 0], [24, 8]) == 0 and int(b.n_free) == 0
    table = b.table.clone()
    assert plan([24, 8], [1, 0]) == 1 and torch.equal(b.table, table)
    assert int(b.n_free) == 0 and b.owned.tolist() == [3, 1] and b.lengths.tolist() == [0, 0]
    assert plan([0, 0], [41, 0], [1, 1]) == 1 and torch.equal(b.table, table)  # too many rows
    assert plan([24, 0], [1, 0], [0, 1]) == 0 and b.owned.tolist() == [4, 0]
    assert b.table[0, 3].item() == table[1, 0].item()


# --------------------------------------------------------------- cache write


def _batch(dev, cached, new, page, Hq, Hkv, seed, rows=None):
    """A planned batch over pages in shuffled order."""
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    S = len(new)
    pages = sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 3
    b = PagedBatch(S, rows or max(1, sum(new)), pages, page, max(max(c + n for c, n in zip(cached, new)), 1),
                   Hq, Hkv, dev)
    gen = torch.Generator().manual_seed(seed)
    b.free.copy_(torch.randperm(pages, generator=gen, dtype=torch.int32))
    paged_plan(b, _ints(cached, dev), _ints(new, dev))
    torch.cuda.synchronize()
    b.raise_refused()
    return b


def _turned(x, w, cos, sin):
    x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    a, b = x[..., :64], x[..., 64:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


@pytest.mark.parametrize("cached,new,page,Hq,Hkv,fp8,extra", [
    ([0], [1], 1, 1, 1, False, 0), ([5, 0, 31], [1, 0, 1], 16, 8, 2, False, 3),
    ([0, 7, 100], [33, 1, 65], 32, 32, 8, False, 2), ([0, 7, 100], [33, 1, 65], 32, 32, 4, True, 2),
    ([3], [700], 64, 5, 5, True, 0), ([0, 0], [200, 900], 128, 7, 1, False, 1),
    ([9, 0], [700, 400], 16, 30, 6, False, 1), ([9, 0], [700, 400], 16, 50, 10, True, 1)])
def test_write_matches_fp64(cuda_device, cached, new, page, Hq, Hkv, fp8, extra):
    """q rounded to bf16 (2^-8 of it), pools to bf16 or e4m3 (2^-4 of it, or
    half the smallest step 2^-10 of a scale); before that fp32, within 2^-19
    of the row's largest value.  The values are below 448 scales.  Rows past
    the last and every other slot keep what they held."""
    from ecf8_amd.paged_kernels import paged_qk_norm_rope

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(Hq * 100 + page)
    N = sum(new)
    b = _batch(dev, cached, new, page, Hq, Hkv, page, rows=N + extra)
    qkv = _rand(N + extra, (Hq + 2 * Hkv) * D, gen=gen, scale=3.0)
    qn, kn = 1 + _rand(D, gen=gen, scale=0.3), 1 + _rand(D, gen=gen, scale=0.3)
    ang = torch.rand(b.max_len, 64, generator=gen, device=dev) * 6.28
    cos, sin = torch.cos(ang), torch.sin(ang)
    q_out = torch.full((N + extra, Hq, D), 7.0, dtype=torch.bfloat16, device=dev)
    pools = [_rand(b.pages, Hkv, page, D, gen=gen) for _ in range(2)]
    scales = [None, None]
    if fp8:
        pools = [p.to(torch.float8_e4m3fn) for p in pools]
        scales = [0.1 + 0.2 * torch.rand(Hkv, generator=gen, device=dev) for _ in range(2)]
    before = [p.clone() for p in pools]
    paged_qk_norm_rope(qkv, b, qn, kn, 1e-6, cos, sin, q_out, *pools, *scales)
    torch.cuda.synchronize()
    b.raise_refused()
    x = qkv[:N].double().view(N, -1, D)
    pos, slots = b.positions[:N].long(), b.slots[:N].long()
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    want = [_turned(x[:, :Hq], qn, c, s), _turned(x[:, Hq: Hq + Hkv], kn, c, s), x[:, Hq + Hkv:]]

    def near(got, want, step, least=0.0):
        top = want.abs().amax(-1, keepdim=True)
        return bool(((got - want).abs() <= want.abs() * step + least + top * 2.0 ** -19).all())

    assert near(q_out[:N].double(), want[0], 2.0 ** -8)
    assert bool((q_out[N:] == 7.0).all())
    for pool, old, y, scale in zip(pools, before, want[1:], scales):
        rows, was = (p.float().permute(0, 2, 1, 3).reshape(-1, Hkv, D) for p in (pool, old))
        got = rows[slots].double()
        if fp8:
            y = y / scale.double()[:, None]
            assert float(y.abs().max()) < 448
            assert near(got, y, 2.0 ** -4, 2.0 ** -10)
        else:
            assert near(got, y, 2.0 ** -8)
        keep = torch.ones(rows.shape[0], dtype=torch.bool, device=dev)
        keep[slots] = False
        assert torch.equal(rows[keep], was[keep])


def test_write_clamps_and_keeps_nan(cuda_device):
    """Values past 448 scales become +-448, infinite ones too, NaN stays."""
    from ecf8_amd.paged_kernels import paged_qk_norm_rope

    dev = cuda_device
    b = _batch(dev, [0], [1], 1, 1, 1, 0)
    qkv = torch.zeros(1, 3 * D, dtype=torch.bfloat16, device=dev)
    qkv[0, 2 * D: 2 * D + 6] = torch.tensor([1e4, -1e4, math.inf, -math.inf, math.nan, 448.0])
    one = torch.ones(D, dtype=torch.bfloat16, device=dev)
    tab = torch.ones(b.max_len, 64, device=dev)
    pools = [torch.zeros(b.pages, 1, 1, D, device=dev).to(torch.float8_e4m3fn) for _ in range(2)]
    q_out = torch.empty(1, 1, D, dtype=torch.bfloat16, device=dev)
    sc = torch.ones(1, device=dev)
    paged_qk_norm_rope(qkv, b, one, one, 1e-6, tab, tab, q_out, *pools, sc, sc)
    got = pools[1].float()[int(b.slots[0]), 0, 0, :6].tolist()
    assert got[:4] == [448.0, -448.0, 448.0, -448.0] and math.isnan(got[4]) and got[5] == 448.0


# ----------------------------------------------------------------- attention


def _attention64(q, k, v, first):
    """q [n, Hq, D] at positions first.., k / v [L, Hkv, D]: (output, A)."""
    n, Hq, _ = q.shape
    G = Hq // k.shape[1]
    k, v = (t.double().repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))
    e = q.double().transpose(0, 1) @ k.transpose(1, 2).contiguous() / math.sqrt(D)
    at = torch.arange(k.shape[1], device=q.device)
    e.masked_fill_(at[None] > first + torch.arange(n, device=q.device)[:, None], -math.inf)
    p = torch.softmax(e, -1)
    return (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)


def _close(got, want, A):
    bound = (2 * want.abs() + A) * 2.0 ** -8 + A * 2.0 ** -10
    return bool(((got.double() - want).abs() <= bound).all())


PAGED = [
    # cached, new, page, Hq, Hkv, max_new
    ([0], [1], 16, 4, 1, 1), ([640], [1], 64, 32, 8, 1), ([0, 31, 32, 127, 128, 129], [1] * 6, 16, 8, 2, 1),
    ([1000, 0, 3, 500], [1, 0, 1, 0], 1, 16, 2, 1), ([2047, 63, 4095], [1, 1, 1], 256, 4, 4, 1),
    ([300, 17], [1, 1], 8, 32, 1, 1),                       # 32 rows of one token
    ([100, 5], [1, 1], 32, 40, 1, 1),                       # more heads than rows of a tile
    ([700, 64, 1], [5, 3, 8], 16, 8, 2, 8), ([40, 2000], [33, 1], 16, 12, 4, None),
    ([0, 0, 0], [1, 129, 70], 64, 6, 3, None), ([513, 0, 9], [257, 1, 0], 32, 8, 1, None),
    ([3000, 1], [70, 300], 128, 32, 8, None), ([0], [1000], 512, 4, 2, None),
    ([5], [600], 4, 3, 3, 600), ([4000] * 9, [2] * 9, 16, 16, 2, 2),
    ([60000, 0, 33000], [1, 1, 1], 128, 8, 1, 1),           # many parts
    ([9000, 200], [200, 2], 16, 12, 2, None),               # tiles in many parts
    ([0, 100, 0, 31], [48, 47, 49, 96], 64, 4, 1, None),    # tiles of 191 to 193 rows
    ([3] * 300, [1, 2, 0] * 100, 2, 4, 4, 2),
    ([10, 300], [2, 1], 16, 1024, 1, None), ([1024, 1023, 2048], [1, 2, 40], 1024, 6, 2, None),
    ([700, 40], [1, 60], 16, 300, 300, None), ([5] * 4096, [1] * 4096, 8, 2, 1, 1)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("cached,new,page,Hq,Hkv,max_new", PAGED)
def test_paged_attention_matches_fp64(cuda_device, cached, new, page, Hq, Hkv, max_new, fp8):
    """Lengths at the edges of pages, key steps, row tiles and splits; idle
    sequences; pages and positions that no token holds are NaN."""
    from ecf8_amd.paged_kernels import paged_attention

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(sum(cached) + page + Hq)
    N, extra = sum(new), 2
    b = _batch(dev, cached, new, page, Hq, Hkv, 7, rows=N + extra)
    q = _rand(N + extra, Hq + 3, D, gen=gen, scale=1.5)[:, 1: 1 + Hq]  # rows with a stride
    pools = [torch.full((b.pages, Hkv, page, D), math.nan, dtype=torch.bfloat16, device=dev)
             for _ in range(2)]
    scales = [None, None]
    if fp8:
        pools = [p.to(torch.float8_e4m3fn) for p in pools]
        scales = [0.05 + 0.1 * torch.rand(Hkv, generator=gen, device=dev) for _ in range(2)]
    dense = []
    for s, (c, n) in enumerate(zip(cached, new)):
        L = c + n if n else c
        p = torch.arange(L, device=dev)
        page_of, off = b.table[s, p // page].long(), p % page
        kv = []
        for pool, scale in zip(pools, scales):
            x = _rand(L, Hkv, D, gen=gen)
            if fp8:
                x = (x * 12).to(torch.float8_e4m3fn)
                pool.view(torch.uint8)[page_of, :, off] = x.view(torch.uint8)
                x = x.double() * scale.double()[:, None]
            else:
                pool[page_of, :, off] = x
            kv.append(x)
        dense.append(kv)
    out = torch.full((N + extra, Hq * D + 8), 3.0, dtype=torch.bfloat16, device=dev)
    got = paged_attention(q, *pools, b, out[:, : Hq * D], max_new=max_new, k_scale=scales[0],
                          v_scale=scales[1])
    torch.cuda.synchronize()
    b.raise_refused()
    at = 0
    for (k, v), c, n in zip(dense, cached, new):
        if n:
            want, A = _attention64(q[at: at + n], k, v, c)
            assert _close(got[at: at + n].unflatten(1, (Hq, D)), want, A), (c, n)
            at += n
    assert bool((out[N:] == 3.0).all()) and bool((out[:, Hq * D:] == 3.0).all())


RAGGED = [
    ([1], 4, 1), ([1, 1, 1], 8, 8), ([31, 32, 33], 8, 2), ([0, 5, 0, 64, 0], 4, 4),
    ([127, 1, 128, 129], 16, 4), ([257, 63], 6, 1), ([300, 0, 511], 32, 8), ([1100], 4, 1),
    ([7] * 70, 12, 4), ([2, 900, 40], 40, 1), ([513], 5, 5),
    # in tiles: 49152 rows and heads on
    ([1600], 32, 8), ([700, 0, 1100, 3], 32, 8), ([47, 48, 49, 1000], 48, 12), ([130, 33], 320, 2),
    ([200], 250, 250), ([20] * 140 + [300], 32, 4), ([1] * 600 + [950], 32, 32),
    ([3, 60], 1024, 1), ([70], 1024, 1024)]


@pytest.mark.parametrize("lens,Hq,Hkv", RAGGED)
def test_ragged_attention_matches_fp64(cuda_device, lens, Hq, Hkv):
    """Slices of one projection output; rows before the first and after the
    last sequence, which hold NaN, are neither read nor written."""
    from ecf8_amd.paged_kernels import ragged_attention

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(sum(lens) + Hq)
    before, after = 2, 3
    N = sum(lens) + before + after
    qkv = _rand(N, Hq + 2 * Hkv, D, gen=gen, scale=1.2)
    qkv[:before], qkv[N - after:] = math.nan, math.nan
    q, k, v = qkv[:, :Hq], qkv[:, Hq: Hq + Hkv], qkv[:, Hq + Hkv:]
    starts = [before]
    for n in lens:
        starts.append(starts[-1] + n)
    out = torch.full((N, Hq * D), 3.0, dtype=torch.bfloat16, device=dev)
    ragged_attention(q, k, v, _ints(starts, dev), out)
    for a, n in zip(starts, lens):
        if n:
            want, A = _attention64(q[a: a + n], k[a: a + n], v[a: a + n], 0)
            assert _close(out[a: a + n].unflatten(1, (Hq, D)), want, A), (a, n)
    assert bool((out[:before] == 3.0).all()) and bool((out[N - after:] == 3.0).all())


@pytest.mark.parametrize("paged,T,Hq", [(False, 150, 4), (True, 150, 4), (False, 150, 384),
                                        (True, 7, 4)])
def test_attention_of_infinite_and_nan_values(cuda_device, paged, T, Hq):
    """A value of infinity or NaN reaches the queries at and after its
    position, in its own dimension, and no query before it; a key of NaN
    reaches its later queries, in every dimension."""
    from ecf8_amd.paged_kernels import paged_attention, ragged_attention

    dev, Hkv = cuda_device, 2
    gen = torch.Generator(device=dev).manual_seed(3)
    q, k, v = (_rand(T, h, D, gen=gen) for h in (Hq, Hkv, Hkv))
    clean, A = _attention64(q, k, v, 0)
    marks = [(5, 3, math.inf), (66, 40, -math.inf), (9, 77, math.nan), (7, 100, math.inf),
             (68, 100, -math.inf)] if T > 100 else [(1, 3, math.inf), (2, 5, math.nan)]
    for t, d, x in marks:
        v[t, :, d] = x
    last = T - 10 if T > 100 else T - 2
    k[last, :, 0] = math.nan
    out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=dev)
    if paged:
        b = _batch(dev, [0], [T], 16, Hq, Hkv, 1)
        pools = [torch.full((b.pages, Hkv, 16, D), math.nan, dtype=torch.bfloat16, device=dev)
                 for _ in range(2)]
        for pool, x in zip(pools, (k, v)):
            pool[(b.slots // 16).long(), :, (b.slots % 16).long()] = x
        paged_attention(q, *pools, b, out)
    else:
        ragged_attention(q, k, v, _ints([0, T], dev), out)
    want = clean.clone()
    for t, d, x in marks:
        # the earlier mark of a dimension, added to: inf - inf is NaN
        want[t:, :, d] = want[t:, :, d].where(want[t:, :, d].isinf(), torch.zeros((), dtype=torch.float64, device=dev)) + x
    want[last:] = math.nan
    assert torch.equal(out.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(out[inf].double(), want[inf])
    # where the marked values do not reach: the clean result
    fine = want.isfinite()
    bound = (2 * clean.abs() + A) * 2.0 ** -8 + A * 2.0 ** -10
    assert bool(((out.double() - clean).abs() <= bound)[fine].all())
    assert int(fine.sum()) > T * Hq * D // 2


@pytest.mark.parametrize("T,Hq", [(70, 4), (150, 384)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_very_large_scores(cuda_device, T, Hq, sign):
    """Equal scores of +-1.6e7 (in powers of two): the mean of the values."""
    from ecf8_amd.paged_kernels import ragged_attention

    dev, Hkv = cuda_device, 2
    gen = torch.Generator(device=dev).manual_seed(6)
    q = torch.full((T, Hq, D), 1000.0, dtype=torch.bfloat16, device=dev)
    k = torch.full((T, Hkv, D), sign * 1000.0, dtype=torch.bfloat16, device=dev)
    v = _rand(T, Hkv, D, gen=gen)
    out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=dev)
    ragged_attention(q, k, v, _ints([0, T], dev), out)
    counts = torch.arange(1, T + 1, device=dev, dtype=torch.float64)[:, None, None]
    mean, A = ((x.double().cumsum(0) / counts).repeat_interleave(Hq // Hkv, 1) for x in (v, v.abs()))
    assert _close(out, mean, A)
