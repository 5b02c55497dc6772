"""What the attention of few rows keeps: probabilities in two parts of bf16, to
2^-15 of each, and infinities and NaN where keys are split over workgroups.

Tolerance per output o, with A = sum p |v|: the output's rounding to bf16, 2^-8
of |o|.  Probabilities are off by 2^-15 at most, in both sums: 2^-15 of A and of
|o| <= A.  The rest is fp32: a score's 128 products sum to within 128 * 2^-24 of
sum |q k| / sqrt(128), below 64 here: 2^-11 in the exponent; sums of at most 2^12
terms in a row are within 2^-12, the exponential within 2^-20.  Together below
2^-10 of A."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _rand(*shape, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale).to(torch.bfloat16)


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


def _batch(dev, cached, new, page, Hq, Hkv):
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    pages = sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 3
    b = PagedBatch(len(new), sum(new), pages, page, max(c + n for c, n in zip(cached, new)), Hq,
                   Hkv, dev)
    paged_plan(b, _ints(cached, dev), _ints(new, dev))
    torch.cuda.synchronize()
    b.raise_refused()
    return b


def _filled(b, cached, new, fp8, gen):
    """Pools with random keys and values; NaN where no token is.  Returns the pools, the
    scales and each sequence's float64 keys and values [L, Hkv, D]."""
    dev, page = b.device, b.page_size
    pools = [torch.full((b.pages, b.Hkv, page, D), math.nan, dtype=torch.bfloat16, device=dev)
             for _ in range(2)]
    scales = [None, None]
    if fp8:
        pools = [p.to(torch.float8_e4m3fn) for p in pools]
        scales = [0.05 + 0.1 * torch.rand(b.Hkv, generator=gen, device=dev) for _ in range(2)]
    dense = []
    for s, (c, n) in enumerate(zip(cached, new)):
        p = torch.arange(c + n, device=dev)
        page_of, off = b.table[s, p // page].long(), p % page
        kv = []
        for pool, scale in zip(pools, scales):
            x = _rand(c + n, b.Hkv, D, gen=gen)
            if fp8:
                x = (x * 12).to(torch.float8_e4m3fn)
                pool.view(torch.uint8)[page_of, :, off] = x.view(torch.uint8)
                x = x.double() * scale.double()[:, None]
            else:
                pool[page_of, :, off] = x
            kv.append(x.double())
        dense.append(kv)
    return pools, scales, dense


def _fine(got, want, A):
    """Within the tolerance, and the root mean square of the errors at most 1.1
    times that of the rounded output (one part of bf16: 1.4 times)."""
    error = (got.double() - want).abs()
    rounded = (want.bfloat16().double() - want).square().mean().sqrt()
    return (bool((error <= want.abs() * 2.0 ** -8 + A * 2.0 ** -10).all())
            and float(error.square().mean().sqrt()) <= 1.1 * float(rounded))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("cached,new,page,Hq,Hkv", [
    ([640, 31, 2047], [1, 1, 1], 16, 32, 8), ([500, 90], [1, 1], 64, 32, 1),
    ([700, 64, 300], [5, 3, 8], 16, 8, 2), ([20_000, 100], [1, 1], 128, 8, 1),
    ([33, 9000], [30, 32], 4, 4, 4)])
def test_paged_attention_of_few_rows_keeps_its_probabilities(cuda_device, cached, new, page, Hq,
                                                             Hkv, fp8):
    from ecf8_amd.paged_kernels import paged_attention

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(sum(cached) + Hq)
    b = _batch(dev, cached, new, page, Hq, Hkv)
    pools, scales, dense = _filled(b, cached, new, fp8, gen)
    q = _rand(sum(new), Hq, D, gen=gen, scale=1.2)
    out = torch.empty(sum(new), Hq, D, dtype=torch.bfloat16, device=dev)
    paged_attention(q, *pools, b, out, max_new=max(new), k_scale=scales[0], v_scale=scales[1])
    at = 0
    want, A = zip(*(_attention64(q[a: a + n], k, v, c) for (k, v), c, n, a in zip(
        dense, cached, new, [sum(new[:i]) for i in range(len(new))])))
    for c, n, w, a in zip(cached, new, want, A):
        assert _fine(out[at: at + n], w, a), (c, n)
        at += n


@pytest.mark.parametrize("lens,Hq,Hkv", [([300, 40, 200], 8, 2), ([500], 5, 5), ([129, 64], 40, 1)])
def test_small_packed_prompts_keep_their_probabilities(cuda_device, lens, Hq, Hkv):
    from ecf8_amd.paged_kernels import ragged_attention

    dev, N = cuda_device, sum(lens)
    assert N * Hq < 256 * 192  # in 32 rows a workgroup
    gen = torch.Generator(device=dev).manual_seed(N)
    q, k, v = (_rand(N, h, D, gen=gen, scale=1.2) for h in (Hq, Hkv, Hkv))
    out = torch.empty(N, Hq, D, dtype=torch.bfloat16, device=dev)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    ragged_attention(q, k, v, _ints(starts, dev), out)
    want, A = zip(*(_attention64(q[a: a + n], k[a: a + n], v[a: a + n], 0)
                    for a, n in zip(starts, lens)))
    assert _fine(out, torch.cat(want), torch.cat(A))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("cached,new", [([9000], [1]), ([9000], [100])])
def test_infinite_and_nan_values_in_split_parts(cuda_device, cached, new, fp8):
    """Values of infinity (bf16) and NaN (either) in the first, a middle and the
    last part of a split sequence reach every query that reads them, in their own
    dimensions; a NaN key reaches its later queries in all."""
    from ecf8_amd.paged_kernels import paged_attention

    dev, Hq, Hkv, page = cuda_device, 8, 2, 16
    gen = torch.Generator(device=dev).manual_seed(12)
    c, n = cached[0], new[0]
    b = _batch(dev, cached, new, page, Hq, Hkv)
    joins = b.work[8:16].view(torch.int32).tolist()
    assert joins[n > 1] > 0  # it is split
    pools, scales, ((k, v),) = _filled(b, cached, new, fp8, gen)
    q = _rand(n, Hq, D, gen=gen)
    clean, A = _attention64(q, k, v, c)

    def put(pool, pos, dims, x):
        page_of, off = int(b.table[0, pos // page]), pos % page
        if fp8:
            pool.view(torch.uint8)[page_of, :, off, dims] = 0x7f
        else:
            pool[page_of, :, off, dims] = x

    marks = [(3, 5, math.nan), (4500, 70, math.nan), (c + n // 2, 90, math.nan)]
    if not fp8:
        marks += [(2, 11, math.inf), (4600, 100, -math.inf), (c, 101, math.inf),
                  (7, 120, math.inf), (8000, 120, -math.inf)]
    want = clean.clone()
    row = torch.arange(n, device=dev)
    for pos, d, x in marks:
        put(pools[1], pos, d, x)
        reads = row + c >= pos
        old = want[reads, :, d]
        want[reads, :, d] = torch.where(old.isfinite(), torch.zeros_like(old), old) + x
    if n > 1:
        put(pools[0], c + n - 5, 0, math.nan)
        want[n - 5:] = math.nan
    out = torch.empty(n, Hq, D, dtype=torch.bfloat16, device=dev)
    paged_attention(q, *pools, b, out, k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[want.isinf()].double(), want[want.isinf()])
    fine = want.isfinite()
    bound = (2 * clean.abs() + A) * 2.0 ** -8 + A * 2.0 ** -10  # (tiles: one part of bf16)
    assert bool(((out.double() - clean).abs() <= bound)[fine].all()) and bool(fine.any())


def test_attention_of_more_than_1024_tiles(cuda_device):
    """Tiles past the plan's first 1024, some of them in many parts.  Bound as for
    probabilities in one part of bf16: 2^-8 of A and of |o| more."""
    from ecf8_amd.paged_kernels import paged_attention

    dev, page, Hq, Hkv = cuda_device, 64, 32, 1
    cached, new = [0] * 14 + [20_000], [420] * 14 + [300]
    assert sum(-(-n * Hq // 192) for n in new) > 1024
    gen = torch.Generator(device=dev).manual_seed(2)
    b = _batch(dev, cached, new, page, Hq, Hkv)
    pools, scales, dense = _filled(b, cached, new, False, gen)
    q = _rand(sum(new), Hq, D, gen=gen, scale=1.2)
    out = torch.empty(sum(new), Hq, D, dtype=torch.bfloat16, device=dev)
    paged_attention(q, *pools, b, out)
    at = 0
    for (k, v), c, n in zip(dense, cached, new):
        want, A = _attention64(q[at: at + n], k, v, c)
        bound = (2 * want.abs() + A) * 2.0 ** -8 + A * 2.0 ** -10
        assert bool(((out[at: at + n].double() - want).abs() <= bound).all()), (c, n)
        at += n
