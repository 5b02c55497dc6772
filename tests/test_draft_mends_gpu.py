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
