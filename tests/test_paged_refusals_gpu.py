"""Steps that the ragged-batch attention refuses on the device, and calls that
it must not refuse."""

from __future__ import annotations

import pytest
import torch

from ecf8_amd._lib import ECF8Error

pytestmark = pytest.mark.gpu

D = 128


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _planned(dev, cached, new, Hq=4, Hkv=1):
    """A planned batch, q of zeros, pools whose values are all 2, and out of 3."""
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    b = PagedBatch(len(new), sum(new), 64, 16, 512, Hq, Hkv, dev)
    paged_plan(b, _ints(cached, dev), _ints(new, dev))
    q = torch.zeros(sum(new), Hq, D, dtype=torch.bfloat16, device=dev)
    pools = [torch.full((64, Hkv, 16, D), 2.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    out = torch.full((sum(new), Hq * D), 3.0, dtype=torch.bfloat16, device=dev)
    torch.cuda.synchronize()
    b.raise_refused()
    return b, q, pools, out


@pytest.mark.parametrize("bound", [3, 2 ** 31, 2 ** 60, 2 ** 61, 2 ** 62, 2 ** 63 - 1, 2 ** 80])
@pytest.mark.parametrize("new", [[3, 1], [1, 60]])
def test_any_large_max_new_is_no_bound(cuda_device, new, bound):
    """Also where its product with the heads of a group (4) passes 64 bits."""
    from ecf8_amd._lib import lib
    from ecf8_amd.paged_kernels import paged_attention

    b, q, pools, out = _planned(cuda_device, [300, 7], new)
    bound = max(bound, max(new))
    paged_attention(q, *pools, b, out, max_new=bound)
    torch.cuda.synchronize()
    b.raise_refused()
    assert bool((out == 2.0).all())
    if bound < 2 ** 63:
        out.fill_(3.0)
        assert lib().ecf8_paged_attention(
            q.data_ptr(), 4 * D, sum(new), b._ref, *(p.data_ptr() for p in pools), 0, None, None,
            bound, out.data_ptr(), 4 * D, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        b.raise_refused()
        assert bool((out == 2.0).all())


@pytest.mark.parametrize("new,max_new", [
    ([4], 1), ([2, 1], 1), ([8], 5), ([8, 1], 7), ([1, 40], 9), ([1, 40], 39), ([300, 2], 250)])
def test_more_new_tokens_than_max_new_are_refused(cuda_device, new, max_new):
    """Also where the kernels launched for max_new could do the step."""
    from ecf8_amd.paged_kernels import paged_attention

    b, q, pools, out = _planned(cuda_device, [0] * len(new), new)
    paged_attention(q, *pools, b, out, max_new=max_new)
    torch.cuda.synchronize()
    with pytest.raises(ECF8Error):
        b.raise_refused()
    paged_attention(q, *pools, b, out, max_new=max(new))
    torch.cuda.synchronize()
    b.raise_refused()
    assert bool((out == 2.0).all())


@pytest.mark.parametrize("new", [[1, 1], [60, 3]])
def test_a_schedule_of_other_sizes_is_not_read(cuda_device, new):
    """A work buffer that was never planned, or planned for a batch of other
    sizes: no row is written, and the step is refused; one of zeros is an
    empty step."""
    from ecf8_amd.paged_kernels import PagedBatch, paged_attention, paged_plan

    dev, Hq, Hkv = cuda_device, 8, 2
    b, q, pools, out = _planned(dev, [300, 5], new, Hq, Hkv)

    def refused():
        out.fill_(3.0)
        paged_attention(q, *pools, b, out)
        torch.cuda.synchronize()
        bad, b.refused[0] = int(b.refused[0]), 0
        return bad

    assert refused() == 0 and bool((out == 2.0).all())
    planned = b.work.clone()
    for fill in (0x01, 0x5a, 0x7f, 0x80, 0xff):
        b.work.fill_(fill)
        assert refused() == 1 and bool((out == 3.0).all()), fill
    b.work[:256].zero_()
    assert refused() == 0 and bool((out == 3.0).all())
    # a smaller batch's schedule, in the larger one's buffer, and the other way round
    small = PagedBatch(2, sum(new), 32, 16, 512, Hq, Hkv, dev)
    paged_plan(small, _ints([300, 5], dev), _ints(new, dev))
    b.work[: small.work.numel()].copy_(small.work)
    assert refused() == 1 and bool((out == 3.0).all())
    for field, other in (("seqs", 1), ("rows", sum(new) - 1), ("width", b._c.width - 1)):
        b.work.copy_(planned)
        was = getattr(b._c, field)
        setattr(b._c, field, other)
        rows = min(sum(new), b._c.rows)
        out.fill_(3.0)
        paged_attention(q[:rows], *pools, b, out)
        torch.cuda.synchronize()
        bad, b.refused[0] = int(b.refused[0]), 0
        setattr(b._c, field, was)
        assert bad == 1 and bool((out == 3.0).all()), field
    b.work.copy_(planned)
    assert refused() == 0 and bool((out == 2.0).all())


@pytest.mark.parametrize("Hq", [4, 400])  # 32 rows a workgroup, and tiles
@pytest.mark.parametrize("starts", [
    [100, -2 ** 31], [200, -2 ** 31 + 5, 200], [3] * 150 + [-2 ** 31], [-2 ** 31, 2 ** 31 - 1]])
def test_packed_starts_at_the_ends_of_int32_stay_in_range(cuda_device, starts, Hq):
    """No difference of starts overflows: no row but those of [0, N) is touched."""
    from ecf8_amd.paged_kernels import ragged_attention

    dev, N = cuda_device, 200
    x = torch.zeros(N, Hq + 2, D, dtype=torch.bfloat16, device=dev)
    x[:, Hq + 1:] = 2.0
    whole = torch.full((N + 20, Hq * D), 3.0, dtype=torch.bfloat16, device=dev)
    out = whole[10: N + 10]
    ragged_attention(x[:, :Hq], x[:, Hq: Hq + 1], x[:, Hq + 1:], _ints(starts, dev), out)
    torch.cuda.synchronize()
    assert bool((whole[:10] == 3.0).all()) and bool((whole[N + 10:] == 3.0).all())
    assert bool(((out == 2.0) | (out == 3.0)).all())
    if starts[0] < 0:  # one sequence, cut to the rows that there are
        assert bool((out == 2.0).all())


@pytest.mark.parametrize("Hq", [4, 400])  # 32 rows a workgroup, and tiles
@pytest.mark.parametrize("starts,bad", [
    ([0, 200], 0), ([7, 9, 9, 150], 0), ([0, 0, 0], 0), ([-1, 200], 1), ([0, 201], 1), ([150, 0], 1),
    ([0, 90, 89, 200], 1), ([0, 500, 200], 1), ([-9, -5], 1), ([201, 201], 1), ([0, 2 ** 31 - 1], 1),
    ([-2 ** 31, 10], 1), ([200, -2 ** 31], 1),
    (list(range(201)), 0), (list(range(150)) + [100] + list(range(150, 200)), 1),
    ([i // 5 for i in range(1001)], 0), ([i // 5 for i in range(1001)] + [0], 1),
    ([5] + [i // 5 for i in range(1001)], 1)])
def test_packed_starts_out_of_order_are_refused(cuda_device, starts, bad, Hq):
    """Equal values, so a row is their mean or as it was; no row but those of
    [0, N) is touched."""
    from ecf8_amd.head_kernels import refusal_flag
    from ecf8_amd.paged_kernels import ragged_attention

    dev, N = cuda_device, 200
    x = torch.zeros(N, Hq + 2, D, dtype=torch.bfloat16, device=dev)
    x[:, Hq + 1:] = 2.0
    whole = torch.full((N + 20, Hq * D), 3.0, dtype=torch.bfloat16, device=dev)
    out = whole[10: N + 10]
    flag = refusal_flag()
    parts = x[:, :Hq], x[:, Hq: Hq + 1], x[:, Hq + 1:]
    ragged_attention(*parts, _ints(starts, dev), out, flag)
    torch.cuda.synchronize()
    assert int(flag) == bad
    assert bool((whole[:10] == 3.0).all()) and bool((whole[N + 10:] == 3.0).all())
    assert bool(((out == 2.0) | (out == 3.0)).all())
    if not bad:
        assert bool((out[starts[0]: starts[-1]] == 2.0).all())
        ragged_attention(*parts, _ints(starts, dev), out)  # without a flag
        torch.cuda.synchronize()
        assert int(flag) == 0


def test_flags_of_other_devices_and_empty_ones_are_refused(cuda_device):
    from ecf8_amd.head_kernels import _flag_ptr, refusal_flag

    flag = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    assert _flag_ptr(flag, flag.device) == flag.data_ptr()
    assert _flag_ptr(refusal_flag(), flag.device)
    for bad, dev in ((flag, torch.device("cuda", 1)), (flag[:0], flag.device),
                     (refusal_flag()[:0], flag.device), (flag.cpu(), flag.device)):
        with pytest.raises(ECF8Error):
            _flag_ptr(bad, dev)
