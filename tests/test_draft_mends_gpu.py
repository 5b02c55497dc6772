"""GPU tests of drafted trees at the places where a kernel was once wrong or less exact
than it says (include/ecf8_draft.h), beside those of test_draft_gpu.py."""

from __future__ import annotations

import math
import random

import draft_model as M
import numpy as np
import pytest
import torch
from test_draft_gpu import D, _check, _filled, _rand, _refused, _seen, _step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,nodes,idle", [(32, 8, 17, 0), (32, 8, 32, 40), (16, 2, 16, 0),
                                               (128, 1, 1, 0), (16, 1, 5, 300)])
def test_probabilities_of_up_to_128_rows_enter_in_two_parts(cuda_device, Hq, Hkv, nodes, idle, fp8):
    """Few keys, whose probabilities are far above the rounding: bf16 once would be off by
    up to 2^-8 of A, where the bound is 2^-10 of A and the output's rounding."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, rng = cuda_device, random.Random(nodes)
    gen = torch.Generator(device=dev).manual_seed(nodes)
    cached = [1, 2, 3, 5, 0] + [0] * idle
    trees = [M.random_tree(rng, nodes, 2) for _ in range(5)] + [[]] * idle
    b, t, _ = _step(dev, cached, trees, 16, Hq, Hkv, max_nodes=nodes)
    pools, scales, dense = _filled(b, [c + len(x) for c, x in zip(cached, trees)], fp8, gen)
    q = _rand(5 * nodes, Hq, D, gen=gen, scale=0.3)
    out = torch.empty(5 * nodes, Hq * D, dtype=torch.bfloat16, device=dev)
    draft_attention(q, *pools, t, out, *scales)
    assert not _refused(b)
    for i in range(5):
        at = slice(i * nodes, (i + 1) * nodes)
        want, A = M.attention(q[at].double(), *dense[i],
                              _seen(M.masks(trees[i]), cached[i], nodes, dev))
        _check(out[at].view(nodes, Hq, D), want, A, True)


# rows of a sequence and KV head: the kernels of 16, 32, 64, 128 and 256
@pytest.mark.parametrize("Hq", [4, 8, 16, 32, 64])
@pytest.mark.parametrize("cached", [20, 3000])
def test_attention_over_a_plan_of_another_step_writes_nothing(cuda_device, cached, Hq):
    """Where none of the sequences that the plan knew has changed: all were idle, or the
    last one was; where one was too long for a tree; and where the step is planned again."""
    from ecf8_amd.draft_kernels import DraftTrees, draft_attention, draft_plan
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    dev, n = cuda_device, 4
    b = PagedBatch(3, 3 * n, 1000, 16, 4000, Hq, 1, dev)
    t = DraftTrees(b, n, 2)
    pools = [torch.full((b.pages, 1, 16, D), 2.0, dtype=torch.bfloat16, device=dev)
             for _ in range(2)]
    parents = torch.tensor([-1, 0, 0, 1] * 3, dtype=torch.int32).to(dev)
    q = torch.zeros(3 * n, Hq, D, dtype=torch.bfloat16, device=dev)
    out = torch.empty(3 * n, Hq * D, dtype=torch.bfloat16, device=dev)

    def plan(*new):
        lengths = [[cached if k else 0 for k in new], new]
        paged_plan(b, *(torch.tensor(x, dtype=torch.int32).to(dev) for x in lengths))

    def attend():
        out.fill_(3.0)
        draft_attention(q, *pools, t, out)
        return _refused(b)

    for before, now in (((0, 0, 0), (n, n, n)), ((0, 0, 0), (0, 0, 1)), ((n, n, 0), (n, n, n)),
                        ((n, 0, 0), (n, 0, 1)), ((n, 0, n), (n, 0, n)), ((n, 2 * n, 0), (n, n, n))):
        plan(*before)
        draft_plan(t, parents)
        assert _refused(b) == (max(before) > n)
        attend()
        plan(*now)
        assert attend() == 1, (before, now)
        assert bool((out == 3.0).all()), (before, now)
        draft_plan(t, parents)
        assert attend() == 0
        rows = sum(now)
        assert bool((out[:rows] == 2.0).all()) and bool((out[rows:] == 3.0).all())


@pytest.mark.parametrize("drawn", [False, True])
def test_verification_over_a_plan_of_another_step_is_refused(cuda_device, drawn):
    """Never planned, planned before the step changed, and planned again: no sequence has a
    result of another step's parents."""
    from ecf8_amd.draft_kernels import DraftTrees, draft_plan, draft_verify
    from ecf8_amd.paged_kernels import paged_plan

    dev, V = cuda_device, 40
    b, t, _ = _step(dev, [5, 9, 0], [[-1, 0, 1], [-1, 0], []], max_nodes=4, kids=2, rows=12)
    p = torch.full((6, V), 1.0 / V, device=dev)
    tokens = torch.arange(6, device=dev)
    accept, sample = torch.zeros(6, device=dev), torch.zeros(3, device=dev)

    def verify(t):
        for x in (t.kept, t.path, t.emitted, t.next_token):
            x.fill_(77)
        draft_verify(t, tokens, p, accept, sample, draft=p if drawn else None)
        return _refused(b)

    def idle(t):
        return (bool((t.kept == 0).all()) and
                all(bool((x == -1).all()) for x in (t.path, t.emitted, t.next_token)))

    assert verify(t) == 0 and t.kept.tolist() == [3, 2, 0]
    assert verify(DraftTrees(b, 4, 2)) == 1
    fresh = DraftTrees(b, 4, 2)
    assert verify(fresh) == 1 and idle(fresh)
    for cached, new in (([8, 11, 0], [3, 2, 0]), ([5, 9, 0], [3, 2, 1]), ([5, 9, 0], [3, 2, 1])):
        paged_plan(b, *(torch.tensor(x, dtype=torch.int32).to(dev) for x in (cached, new)))
        assert verify(t) == 1 and idle(t)
        draft_plan(t, torch.tensor([-1, 0, 0, -1, 0, -1], dtype=torch.int32).to(dev))
        assert verify(t) == 0 and t.kept.tolist() == [2, 2, new[2]]


def test_a_move_of_another_step_is_refused(cuda_device):
    """The next step's lengths would send the kept rows to other places: after its plan
    nothing moves.  Paths of a caller's own do, of trees that were never planned."""
    from ecf8_amd.draft_kernels import DraftTrees, KeepPlan, draft_keep, draft_plan
    from ecf8_amd.paged_kernels import paged_plan

    dev = cuda_device
    b, t, parents = _step(dev, [5, 0], [[-1, 0, 1, 0], []], max_nodes=4, kids=2, rows=8)
    pools = [torch.zeros(b.pages, 1, 16, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    page = int(b.table[0, 0])

    def keep(t):
        for p in pools:
            p[page, 0] = torch.arange(16, device=dev)[:, None].bfloat16()
        t.kept.copy_(torch.tensor([2, 0]))
        t.path.copy_(torch.tensor([[0, 3, -1, -1], [-1] * 4]))
        draft_keep(KeepPlan(t, [tuple(pools)]))
        bad = _refused(b)
        assert torch.equal(*pools)
        return bad, [int(x) for x in pools[0][page, 0, :, 0]]

    rows = list(range(16))
    moved = rows[:6] + [8] + rows[7:]
    assert keep(t) == (0, moved)
    for cached, new in (([7, 0], [4, 0]), ([5, 0], [4, 3]), ([5, 0], [4, 0])):
        paged_plan(b, *(torch.tensor(x, dtype=torch.int32).to(dev) for x in (cached, new)))
        assert keep(t) == (1, rows), (cached, new)
    draft_plan(t, parents)
    assert keep(t) == (0, moved)
    assert keep(DraftTrees(b, 4, 2)) == (0, moved)


def _wave_scan(v):
    """The inclusive sums of 64 values in the order in which a wave adds them."""
    for o in (1, 2, 4, 8):
        v = [x + v[i - o] if i % 16 >= o else x for i, x in enumerate(v)]
    v = [x + v[i // 16 * 16 - 1] if i // 16 in (1, 3) else x for i, x in enumerate(v)]
    return [x + v[31] if i >= 32 else x for i, x in enumerate(v)]


def _sums_that_differ(seed):
    """(values, i): half of the sum of 64 fp32 values lies between the wave's sums up to i - 1
    and up to i, although value i is zero: the two were added in different orders."""
    rng = random.Random(seed)
    while True:
        v = [float(np.float32(rng.random() * 2.0 ** -rng.randrange(60))) if rng.random() < 0.5 else 0.0
             for _ in range(64)]
        upto = _wave_scan(v)
        for i in range(1, 60):
            if v[i] == 0.0 and upto[i] > upto[i - 1]:
                # values after i that double the sum before it
                rest, parts = 2 * upto[i - 1] - upto[i], []
                for _ in range(3):
                    parts.append(float(np.float32(rest - sum(parts))))
                if min(parts) < 0 or sum(parts) != rest:
                    continue
                w = v[: i + 1] + [0.0] * (63 - i)
                for at, x in zip(rng.sample(range(i + 1, 64), 3), parts):
                    w[at] = x
                upto = _wave_scan(w)
                if w[next(k for k in range(64) if upto[k] > 0.5 * upto[63])] == 0.0:
                    return w, i


@pytest.mark.parametrize("drawn", [False, True])
def test_the_next_token_is_never_of_a_run_of_nothing(cuda_device, drawn):
    """Probabilities whose partial sums, one a run of the vocabulary, rise by a rounding where
    nothing is, and a sample that falls between the two: the token before or after is meant."""
    from ecf8_amd.draft_kernels import draft_verify

    dev, S, V = cuda_device, 24, 256  # 64 runs of four
    cases = [_sums_that_differ(seed) for seed in range(S)]
    b, t, _ = _step(dev, [1] * S, [[-1]] * S, max_nodes=1, kids=1)
    p = torch.zeros(S, V)
    for s, (w, _) in enumerate(cases):
        p[s, s % 4:: 4] = torch.tensor(w)
    p = p.to(dev)
    half = torch.full((S,), 0.5, device=dev)
    draft_verify(t, torch.zeros(S, dtype=torch.int64, device=dev), p, half, half,
                 draft=p.clone() if drawn else None)
    assert not _refused(b)
    for s, (w, i) in enumerate(cases):
        has = [k for k in range(64) if w[k]]
        near = [max(k for k in has if k < i), min(k for k in has if k > i)]
        assert int(t.next_token[s]) in [4 * k + s % 4 for k in near], s


LOG2E = 1.4426950408889634


def _scale_error(t):
    """What rounding log2(e) / t to fp32 changes, relative to it."""
    return float(np.float32(LOG2E / t)) * t / LOG2E - 1


def test_sums_of_probabilities_have_all_of_the_temperature(cuda_device):
    """One logit of 0 and n of -D, at temperatures of which D log2(e) / T is 12 to within
    2^-22: as a product with both parts it rounds to 12, the terms are 2^-12 and sums of them
    exact in fp32, so the first probability is off by 2^-22 ln 2 of the exponent and 2^-23 of
    the quotient.  With log2(e) / T rounded to fp32 the product is the next value, 2^-20 away,
    and the sum off by 2^-20 ln 2, four times that."""
    from ecf8_amd.draft_kernels import token_probabilities

    dev, V = cuda_device, 151_936
    cases = []
    for D in np.arange(4.0, 16.0, 0.0625):  # (exact in bf16)
        t = float(np.float32(D * LOG2E / 12))
        if (abs(D * LOG2E / t - 12) < 2.0 ** -22
                and abs(float(np.float32(D) * np.float32(LOG2E / t)) - 12) >= 2.0 ** -21):
            cases.append((float(D), t))
    assert len(cases) > 3
    x = torch.zeros(len(cases), V, device=dev)
    x[:, :-1] = -torch.tensor([d for d, _ in cases], device=dev)[:, None]
    for first in (V - 1, 0, 70_001):
        row = x.roll(first + 1, 1).bfloat16()
        out = torch.empty(row.shape, device=dev)
        token_probabilities(row, torch.tensor([t for _, t in cases], device=dev), out)
        for i, (d, t) in enumerate(cases):
            want = torch.softmax(row[i].double() / t, -1)
            error = ((out[i].double() - want).abs() / want).amax()
            # (and the others' of the same exponent once more, and of a product)
            assert abs(float(out[i, first]) / float(want[first]) - 1) <= 0.7 * 2 ** -22 + 2 ** -23, (d, t)
            assert float(error) <= 1.4 * 2 ** -22 + 2 ** -22, (d, t)
            assert abs(float(out[i].double().sum()) - 1) <= 2 ** -22, (d, t)


def test_small_probabilities_have_all_of_the_temperature(cuda_device):
    """One logit of 0 and others so far below that the sum is 1: a probability e^-|e| has the
    exponent's one rounding, |e| 2^-24 (the logits' differences are exact), and the
    exponential's, 2^-22.  Temperatures whose log2(e) / T is off by nearly 2^-24 in fp32."""
    from ecf8_amd.draft_kernels import token_probabilities

    dev, V, rng = cuda_device, 4096, random.Random(1)
    temps = []
    while len(temps) < 8:
        t = float(np.float32(2.0 ** rng.randrange(-4, 3) * LOG2E * (1 - 0.01 * rng.random())))
        if abs(_scale_error(t)) > 0.8 * 2 ** -24:
            temps.append(t)
    for t in temps:
        step = 2.0 ** math.floor(math.log2(t / 2))
        k = torch.arange(V, device=dev) % 256
        x = (-step * k).bfloat16()
        keep = (-x.double() / t > 40) & (-x.double() / t < 85)
        x = torch.where(keep, x, -math.inf)
        x[17] = 0.0
        assert int(keep.sum()) > V // 16
        out = torch.empty(1, V, device=dev)
        token_probabilities(x[None], t, out)
        e = x.double() / t
        bound = e.abs() * 2.0 ** -24 + 2.0 ** -22
        error = out[0].double() / e.exp() - 1
        assert bool((error[keep].abs() <= bound[keep]).all()), t
        assert float(out[0, 17]) == 1.0


@pytest.mark.parametrize("N,V", [(1, 1), (3, 9), (5, 4099), (5, 151_936), (70, 50_257), (300, 2048),
                                 (2, 300_001)])
@pytest.mark.parametrize("scale", [0.1, 3.0, 60.0])
def test_probabilities_to_the_last_bits(cuda_device, N, V, scale):
    """A difference of logits and its product round once each, 2^-24 of the exponent e; the
    exponential by 2^-23.  Sums are taken in up to 36 additions in a row, 2^-24 each, and
    rescaled up to 11 times, 2^-22 each, which split an exponent without adding to it; the
    quotient's two roundings are 2^-23.  In all (|e| + sum p |e| + 45) 2^-23 of p, and of the
    row's sum twice the weighted part."""
    from ecf8_amd.draft_kernels import token_probabilities

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(V)
    x = _rand(N, V, gen=gen, scale=scale)
    temps = torch.tensor([[0.7, 1.0, 2.5, 0.05, 0.013][i % 5] for i in range(N)], device=dev)
    out = torch.empty(N, V, device=dev)
    token_probabilities(x, temps, out)
    for i in range(N):
        e = x[i].double()
        e = (e - e.max()) / float(temps[i])
        want = torch.softmax(e, -1)
        mean = float((want * e.abs()).sum())
        error = (out[i].double() - want).abs()
        assert bool((error <= want * (e.abs() + mean + 45) * 2.0 ** -23 + 2.0 ** -126).all()), i
        assert abs(float(out[i].double().sum()) - 1) <= (2 * mean + 45) * 2.0 ** -23 + V * 2.0 ** -126, i
