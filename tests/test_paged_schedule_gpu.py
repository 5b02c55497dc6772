"""The attention's schedule that ``paged_plan`` leaves in a batch's work buffer:
every row's keys covered once, parts and joins within their places, and no
item much longer than an equal share of the work."""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

# of csrc/ecf8_paged_layout.h
FEW_ROWS, FEW_KEYS, TILE_ROWS, TILE_KEYS, MIN_UNITS, TILE_START, SLOTS = 32, 128, 192, 64, 4, 4, 512


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def _lists(b):
    """(items of few rows, tiles, joins of each) of the planned step, as lists
    of the structures' eight ints, and the targets the keys are cut for."""
    S, rows, G = b.max_seqs, b.max_rows, b.Hq // b.Hkv
    target = max(1, SLOTS // b.Hkv)
    counts = b.work[:16].view(torch.int32).tolist()
    at, lists = 256, []
    room = [target + S, rows * G // TILE_ROWS + S + 2 * target, target, target]
    for n, most in zip(counts, room):
        assert 0 <= n <= most, (counts, room)
        lists.append(b.work[at: at + 32 * n].view(torch.int32).view(n, 8).tolist())
        at += -(-32 * most // 256) * 256
    return lists, target


def _check(b, cached, new):
    """Asserts what the attention relies on; (longest item, share) of each class,
    in units of keys."""
    (few, tiles, few_joins, tile_joins), target = _lists(b)
    G = b.Hq // b.Hkv
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    want = [{}, {}]  # (seq, row0) -> positions that its rows read together
    for s, (c, n) in enumerate(zip(cached, new)):
        if 0 < n * G <= FEW_ROWS:
            want[0][s, 0] = c + n
        else:
            for r in range(0, n * G, TILE_ROWS):
                want[1][s, r] = c + min(n, (r + TILE_ROWS - 1) // G + 1)
    out = []
    for items, joins, ends, unit, start in ((few, few_joins, want[0], FEW_KEYS, 0),
                                            (tiles, tile_joins, want[1], TILE_KEYS, TILE_START)):
        pieces = {}
        for seq, row0, k0, k1, part, start_row, n, c in items:
            assert (start_row, n, c) == (starts[seq], new[seq], cached[seq])
            assert k0 % unit == 0 and k0 < k1
            pieces.setdefault((seq, row0), []).append((k0, k1, part))
        assert pieces.keys() == ends.keys()
        used, joined = set(), {}
        for row0, part, n, start_row, tokens, *_ in joins:
            places = set(range(part, part + n))
            assert n > 1 and part >= 0 and part + n <= 2 * target and not places & used
            used |= places
            joined[start_row, row0, part] = n, tokens
        for (seq, row0), p in pieces.items():
            p.sort()
            assert p[0][0] == 0 and p[-1][1] == ends[seq, row0]
            assert all(x[1] == y[0] for x, y in zip(p, p[1:]))
            if len(p) == 1:
                assert p[0][2] == -1
            else:
                first = p[0][2]
                assert [x[2] for x in p] == list(range(first, first + len(p)))
                assert joined.pop((starts[seq], row0, first)) == (len(p), new[seq])
        assert not joined
        units = [-(-e // unit) for e in ends.values()]
        share = -(-sum(u + start for u in units) // target)
        longest = max([-(-(k1 - k0) // unit) for _, _, k0, k1, *_ in items], default=0)
        out.append((longest, max(1, share)))
    return out


def _plan(dev, cached, new, page, Hq, Hkv):
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    S = len(new)
    pages = sum(-(-(c + n) // page) for c, n in zip(cached, new))
    b = PagedBatch(S, max(1, sum(new)), pages, page, max(c + n for c, n in zip(cached, new)), Hq,
                   Hkv, dev)
    paged_plan(b, _ints(cached, dev), _ints(new, dev))
    torch.cuda.synchronize()
    b.raise_refused()
    return b


# a long context's chunk beside prompts: 1024 tiles, just more, many more, and
# the long one's tiles past the first 1024
SCHEDULES = [
    ([100_000] + [0] * 46, [64] + [1024] * 46, 64, 32, 8), ([100_000] + [0] * 47, [64] + [1024] * 47, 64, 32, 8),
    ([0] * 47 + [100_000], [1024] * 47 + [64], 64, 32, 8), ([100_000] + [0] * 30, [64] + [407] * 30, 64, 32, 2),
    ([0] * 14 + [20_000], [420] * 14 + [300], 64, 32, 1), ([0, 200_000, 5], [9000, 700, 2], 128, 32, 4),
    ([0] * 300 + [50_000], [60] * 300 + [128], 16, 64, 4), ([50_000] * 40, [128] * 40, 256, 32, 1),
    ([700, 0, 30_000, 12], [1, 0, 1, 3], 16, 8, 2), ([9000] * 600, [1] * 600, 128, 32, 8)]


@pytest.mark.parametrize("cached,new,page,Hq,Hkv", SCHEDULES)
def test_schedule_is_whole_and_even(cuda_device, cached, new, page, Hq, Hkv):
    b = _plan(cuda_device, cached, new, page, Hq, Hkv)
    (few, few_share), (tile, tile_share) = _check(b, cached, new)
    assert few <= few_share
    # a cut leaves MIN_UNITS on both sides, so a piece has at most as many more at
    # each end; a share has two such ends at least
    assert tile <= max(tile_share, 2 * MIN_UNITS) + 2 * MIN_UNITS


@pytest.mark.parametrize("seed", range(6))
def test_schedule_of_drawn_steps(cuda_device, seed):
    rng = random.Random(seed)
    Hkv = rng.choice([1, 2, 8, 32])
    Hq = Hkv * rng.choice([1, 4, 7, 16])
    S = rng.choice([3, 60, 900])
    cached = [rng.choice([0, 0, rng.randint(0, 60_000)]) for _ in range(S)]
    new = [rng.choice([0, 1, 1, rng.randint(1, 40), rng.randint(1, 200_000 // S)]) for _ in range(S)]
    new[rng.randrange(S)] = 33
    b = _plan(cuda_device, cached, new, 64, Hq, Hkv)
    (few, few_share), (tile, tile_share) = _check(b, cached, new)
    assert few <= few_share
    assert tile <= max(tile_share, 2 * MIN_UNITS) + 2 * MIN_UNITS
