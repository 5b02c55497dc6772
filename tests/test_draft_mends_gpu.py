"""GPU tests of drafted trees at the places where a kernel was once wrong or less exact
than it says (include/ecf8_draft.h), beside those of test_draft_gpu.py."""

from __future__ import annotations

import random

import draft_model as M
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
