"""The cache write at head counts on both sides of its forms, one and three heads
a lane: the same values whatever the number of rows of the call, and float64's.

Tolerance: q and bf16 pools are rounded to bf16 (2^-8 of a value), e4m3 codes by
2^-4 of theirs or half the smallest step, 2^-10; before that fp32, within 2^-19
of a row's largest value."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

D, EPS = 128, 1e-6


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv", [
    (8, 4), (9, 1), (16, 2), (24, 4), (32, 8), (39, 3), (26, 13), (20, 20), (59, 1), (32, 16), (64, 4)])
def test_write_of_many_rows_is_that_of_few(cuda_device, Hq, Hkv, fp8):
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan, paged_qk_norm_rope

    dev, H, page, L = cuda_device, Hq + 2 * Hkv, 16, 2100
    gen = torch.Generator(device=dev).manual_seed(H)
    qkv = (torch.randn(L, H * D, generator=gen, device=dev) * 3).bfloat16()
    norms = [(1 + 0.3 * torch.randn(D, generator=gen, device=dev)).bfloat16() for _ in range(2)]
    ang = torch.rand(2112, 64, generator=gen, device=dev) * 6.28
    cos, sin = torch.cos(ang), torch.sin(ang)
    kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
    scales = ([0.1 + 0.2 * torch.rand(Hkv, generator=gen, device=dev) for _ in range(2)] if fp8
              else [None, None])

    def written(step):
        """q, k and v rows of the sequence, ``step`` rows a call."""
        b = PagedBatch(1, step, -(-L // page), page, 2112, Hq, Hkv, dev)
        pools = [torch.zeros(b.pages, Hkv, page, D, device=dev).to(kind) for _ in range(2)]
        q = torch.empty(L, Hq, D, dtype=torch.bfloat16, device=dev)
        for at in range(0, L, step):
            n = min(step, L - at)
            paged_plan(b, _ints([at], dev), _ints([n], dev))
            paged_qk_norm_rope(qkv[at: at + n], b, *norms, EPS, cos, sin, q[at: at + n], *pools,
                               *scales)
        torch.cuda.synchronize()
        b.raise_refused()
        p = torch.arange(L, device=dev)
        where = b.table[0, p // page].long(), p % page
        rows = [x.view(torch.uint8 if fp8 else torch.int16)[where[0], :, where[1]].view(kind)
                for x in pools]
        return [q, *rows]

    many, few = written(L), written(100)
    for x, y in zip(many, few):
        as_int = torch.uint8 if x.element_size() == 1 else torch.int16
        assert torch.equal(x.view(as_int), y.view(as_int))
    x = qkv.double().view(L, H, D)
    c, s = cos.double()[:L, None], sin.double()[:L, None]

    def turned(x, w):
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        return torch.cat([x[..., :64] * c - x[..., 64:] * s, x[..., 64:] * c + x[..., :64] * s], -1)

    want = [turned(x[:, :Hq], norms[0]), turned(x[:, Hq: Hq + Hkv], norms[1]), x[:, Hq + Hkv:]]
    for i, (got, w) in enumerate(zip(many, want)):
        step, least = 2.0 ** -8, 0.0
        if fp8 and i:
            w = w / scales[i - 1].double()[:, None]
            step, least = 2.0 ** -4, 2.0 ** -10
            assert float(w.abs().max()) < 448
        top = w.abs().amax(-1, keepdim=True)
        assert bool(((got.double() - w).abs() <= w.abs() * step + least + top * 2.0 ** -19).all())
