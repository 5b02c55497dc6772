"""GPU tests of the speculative-decoding kernels (include/ecf8_draft.h) against
the plain model of draft_model.py.

Tolerance of the attention, per output o with A = sum p |v|: the output's rounding
to bf16, 2^-8 of |o|.  Probabilities are rounded in two parts, 2^-15 of A and |o|,
or (more than 64 rows of a sequence and KV head) once, 2^-8 of A and of |o| in
both sums.  The rest is fp32: a score's 128 products sum to within 128 * 2^-24 of
sum |q k| / sqrt(128), below 64 here: 2^-11 in the exponent; sums of at most 2^12
terms in a row are within 2^-12, the exponential within 2^-20.  Together below 2^-10
of A.

Tolerance of a probability p = e / S: x - max is off by 2^-24 of it (bf16 values of
different exponents), and so is the product with log2(e) / T after its correction,
so the exponent t = (x - max) / T by 2^-23 |t| in all, e by that and 2^-22 (the
exponential and one more rounding); S is a sum of positive terms, each off by no
more than that weighted by itself, in runs of at most 2^10 additions: 2^-14 + its
terms' errors.  |t| is taken at the element for e, and at most 32 for what carries
S.  Below 2^-126 zero may stand for p."""

from __future__ import annotations

import math
import random

import draft_model as M
import pytest
import torch

from ecf8_amd._lib import ECF8Error

pytestmark = pytest.mark.gpu

D = 128


def _ints(v, dev, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).to(dev)


def _rand(*shape, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale).to(torch.bfloat16)


def _refused(b):
    torch.cuda.synchronize()
    bad, b.refused[0] = int(b.refused[0]), 0
    return bad


def _step(dev, cached, trees, page=16, Hq=4, Hkv=1, max_nodes=64, kids=64, rows=None):
    """A batch and trees, planned: (batch, trees, parents)."""
    from ecf8_amd.draft_kernels import DraftTrees, draft_plan
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    new = [len(t) for t in trees]
    pages = sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 3
    b = PagedBatch(len(new), rows or max(1, sum(new)), pages, page,
                   max(c + n for c, n in zip(cached, new)) or 1, Hq, Hkv, dev)
    # pages in no order
    b.free.copy_(torch.randperm(pages, generator=torch.Generator().manual_seed(pages)).int())
    t = DraftTrees(b, max_nodes, kids)
    paged_plan(b, _ints(cached, dev), _ints(new, dev))
    parents = _ints([p for tree in trees for p in tree] or [-1], dev)
    draft_plan(t, parents)
    return b, t, parents


# ------------------------------------------------------------------ the plan


@pytest.mark.parametrize("S,nodes,page", [(1, 1, 16), (1, 64, 1), (5, 64, 8), (16, 5, 16),
                                          (17, 33, 64), (300, 12, 16), (4096, 4, 16)])
def test_plan_matches_the_model(cuda_device, S, nodes, page):
    rng = random.Random(S + nodes)
    for chain in (False, True):
        trees = [M.random_tree(rng, rng.choice([0, 1, nodes, rng.randint(1, nodes)]),
                               rng.choice([1, 3, 64]), chain) for _ in range(S)]
        trees[0] = M.random_tree(rng, nodes, 64, chain)
        cached = [rng.choice([0, 1, 31, rng.randint(0, 200)]) for _ in range(S)]
        b, t, parents = _step(cuda_device, cached, trees, page)
        assert not _refused(b)
        bits = [m for tree in trees for m in M.masks(tree)]
        n = len(bits)
        assert t.masks[:n].tolist() == [M.signed(m) for m in bits]
        assert t.parents[:n].tolist() == parents[:n].tolist()
        want = [c + bin(m).count("1") - 1 for c, tree in zip(cached, trees) for m in M.masks(tree)]
        assert b.positions[:n].tolist() == want


BAD_TREES = [[0, 0], [-1, 1], [-1, 0, 2], [-1, -1], [-1, 0, -5], [-1, 0, 0, 0, 0], [1, 0],
             [-1, 2 ** 31 - 1], [-1, -2 ** 31], [5]]


@pytest.mark.parametrize("bad", BAD_TREES)
def test_a_tree_that_is_none_is_refused_alone(cuda_device, bad):
    """Its rows are on their own; the sequences around it are planned."""
    trees = [[-1, 0, 1], bad, [-1, 0, 0]]
    b, t, parents = _step(cuda_device, [7, 20, 40], trees, kids=3)
    assert _refused(b)
    n = len(bad)
    assert t.masks[: 6 + n].tolist() == [1, 3, 7] + [1 << i for i in range(n)] + [1, 3, 5]
    assert t.parents[3: 3 + n].tolist() == [-1] * n
    assert b.positions[: 6 + n].tolist() == [7, 8, 9] + [20] * n + [40, 41, 41]


def test_too_many_rows_are_refused(cuda_device):
    """More than max_nodes, or than parents holds: nothing of them is attended."""
    from ecf8_amd.draft_kernels import draft_attention, draft_plan

    dev = cuda_device
    b, t, parents = _step(dev, [20, 20], [M.random_tree(random.Random(1), 6, 8), [-1, 0]],
                          max_nodes=5)
    assert _refused(b)
    assert t.masks.tolist() == [0] * 6 + [1, 3] and t.parents.tolist() == [-1] * 7 + [0]
    pools = [torch.full((b.pages, 1, 16, D), 2.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    q = torch.zeros(8, 4, D, dtype=torch.bfloat16, device=dev)
    out = torch.full((8, 4 * D), 3.0, dtype=torch.bfloat16, device=dev)
    draft_attention(q, *pools, t, out)
    assert not _refused(b)
    assert bool((out[:6] == 3.0).all()) and bool((out[6:] == 2.0).all())
    b, t, parents = _step(dev, [20, 20], [[-1, 0], [-1, 0]])
    assert not _refused(b)
    draft_plan(t, parents[:3].contiguous())
    assert _refused(b)
    pools = [torch.full((b.pages, 1, 16, D), 2.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    out.fill_(3.0)
    draft_attention(q[:4], *pools, t, out)
    assert not _refused(b)
    assert bool((out[2:] == 3.0).all()) and bool((out[:2] == 2.0).all())


# ------------------------------------------------------------ the attention


def _filled(b, lengths, fp8, gen, spread=1.0):
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
    for s, L in enumerate(lengths):
        p = torch.arange(L, device=dev)
        page_of, off = b.table[s, p // page].long(), p % page
        kv = []
        for pool, scale in zip(pools, scales):
            x = _rand(L, b.Hkv, D, gen=gen, scale=spread)
            if fp8:
                x = (x * 12).to(torch.float8_e4m3fn)
                pool.view(torch.uint8)[page_of, :, off] = x.view(torch.uint8)
                x = x.double() * scale.double()[:, None]
            else:
                pool[page_of, :, off] = x
            kv.append(x.double())
        dense.append(kv)
    return pools, scales, dense


def _seen(bits, cached, n, dev):
    """[n, cached + n]: what rows of these masks read."""
    tail = torch.tensor([[m >> j & 1 for j in range(n)] for m in bits], dtype=torch.bool)
    return torch.cat([torch.ones(n, cached, dtype=torch.bool), tail], 1).to(dev)


def _check(got, want, A, fine):
    bound = (want.abs() * 2.0 ** -8 + A * 2.0 ** -10 if fine else
             (2 * want.abs() + A) * 2.0 ** -8 + A * 2.0 ** -10)
    error = (got.double() - want).abs()
    assert bool((error <= bound).all()), float((error / bound.clamp(min=1e-30)).max())


# heads of a group times rows: workgroups of 16, 32, 64, 128, 256 rows, and several of 256
SHAPES = [(4, 1, 4), (32, 8, 8), (8, 8, 32), (32, 8, 13), (32, 4, 16), (32, 8, 27), (16, 16, 64),
          (32, 8, 64), (32, 4, 64), (40, 2, 64), (1, 1, 1), (3, 1, 7), (128, 1, 9)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [1, 16, 256])
@pytest.mark.parametrize("Hq,Hkv,nodes", SHAPES)
def test_attention(cuda_device, Hq, Hkv, nodes, page, fp8):
    """Trees after no, few and many cached tokens, idle sequences among them, single
    rows beside full trees; rows past the last one are left alone."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, rng = cuda_device, random.Random(Hq * nodes + page)
    gen = torch.Generator(device=dev).manual_seed(nodes)
    cached = [0, 700, 33, 5, 1500, 128, 0]
    new = [nodes, nodes, 0, 1, max(1, nodes // 2), nodes, 1]
    trees = [M.random_tree(rng, n, rng.choice([1, 2, 64])) for n in new]
    b, t, _ = _step(dev, cached, trees, page, Hq, Hkv, max_nodes=nodes)
    pools, scales, dense = _filled(b, [c + n for c, n in zip(cached, new)], fp8, gen)
    N = sum(new)
    wide = torch.randn(N, Hq * D + 64, generator=gen, device=dev).bfloat16()
    q = wide[:, : Hq * D]
    out = torch.full((N + 2, Hq * D), 7.0, dtype=torch.bfloat16, device=dev)
    assert draft_attention(q, *pools, t, out, *scales) is out
    assert not _refused(b)
    assert bool((out[N:] == 7.0).all())
    a = 0
    for c, tree, (k, v) in zip(cached, trees, dense):
        n = len(tree)
        if n:
            want, A = M.attention(q[a: a + n].double().view(n, Hq, D), k, v,
                                  _seen(M.masks(tree), c, n, dev))
            _check(out[a: a + n].view(n, Hq, D), want, A, nodes * (Hq // Hkv) <= 64)
        a += n


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,nodes,cached", [
    (8, 2, 3, [9000, 10]), (8, 2, 16, [20_000, 127, 4000]), (16, 2, 16, [6000, 6000, 1]),
    (32, 4, 30, [30_000]), (16, 2, 64, [5000, 77])])
def test_attention_of_split_keys(cuda_device, Hq, Hkv, nodes, cached, fp8):
    """Long contexts of few sequences, whose keys are split over workgroups."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, rng = cuda_device, random.Random(nodes)
    gen = torch.Generator(device=dev).manual_seed(nodes)
    trees = [M.random_tree(rng, nodes, 3) for _ in cached]
    b, t, _ = _step(dev, cached, trees, 64, Hq, Hkv, max_nodes=nodes)
    pools, scales, dense = _filled(b, [c + nodes for c in cached], fp8, gen)
    q = _rand(nodes * len(cached), Hq, D, gen=gen, scale=1.5)
    out = torch.empty(nodes * len(cached), Hq * D, dtype=torch.bfloat16, device=dev)
    draft_attention(q, *pools, t, out, *scales)
    assert not _refused(b)
    for i, (c, tree, (k, v)) in enumerate(zip(cached, trees, dense)):
        at = slice(i * nodes, (i + 1) * nodes)
        want, A = M.attention(q[at].double(), k, v, _seen(M.masks(tree), c, nodes, dev))
        _check(out[at].view(nodes, Hq, D), want, A, nodes * (Hq // Hkv) <= 64)


@pytest.mark.parametrize("Hq,Hkv,nodes", [(4, 1, 3), (8, 1, 8), (16, 1, 9)])
def test_attention_of_thousands_of_sequences(cuda_device, Hq, Hkv, nodes):
    """More tiles than the plan has threads, in a batch with room for more rows than
    its trees can have: equal values of a sequence, so each output is its value."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, S, rng = cuda_device, 2500, random.Random(nodes)
    new = [rng.choice([0, 1, nodes]) for _ in range(S)]
    cached = [rng.choice([0, 3, 40]) for _ in range(S)]
    cached[7], new[7] = 9000, nodes
    trees = [M.random_tree(rng, n, 3) for n in new]
    b, t, _ = _step(dev, cached, trees, 16, Hq, Hkv, max_nodes=nodes, rows=S * nodes + 1000)
    owner = torch.zeros(b.pages, dtype=torch.float32, device=dev)
    for s in range(S):
        owner[b.table[s, : int(b.owned[s])].long()] = s % 256 - 100
    pool = owner[:, None, None, None].expand(-1, Hkv, 16, D).bfloat16().contiguous()
    q = torch.randn(sum(new), Hq, D, generator=torch.Generator(device=dev).manual_seed(1),
                    device=dev).bfloat16()
    out = torch.full((sum(new), Hq * D), 7.0, dtype=torch.bfloat16, device=dev)
    draft_attention(q, torch.zeros_like(pool), pool, t, out)
    assert not _refused(b)
    want = _ints([s % 256 - 100 for s in range(S) for _ in range(new[s])], dev).float()
    assert bool((out.float() == want[:, None]).all())


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (16, 2), (32, 2), (32, 1)])
@pytest.mark.parametrize("cached", [0, 5, 31, 32, 300, 3000])
def test_masks_of_the_callers_own(cuda_device, cached, Hq, Hkv):
    """Any masks after the plan: all ones, later rows alone, none at all (zeros where
    nothing is cached), bits past the sequence's rows."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, n = cuda_device, 13
    gen = torch.Generator(device=dev).manual_seed(cached)
    rng = random.Random(cached)
    b, t, _ = _step(dev, [cached], [M.random_tree(rng, n, 3)], 16, Hq, Hkv, max_nodes=n)
    pools, _, [(k, v)] = _filled(b, [cached + n], False, gen)
    q = _rand(n, Hq, D, gen=gen)
    out = torch.full((n, Hq * D), 7.0, dtype=torch.bfloat16, device=dev)
    bits = [rng.choice([0, 2 ** 64 - 1, 1 << (n - 1), 1 << rng.randrange(64), rng.getrandbits(64),
                        0xfff << n]) for _ in range(n)]
    bits[3], bits[4] = 0, 0xffff << n
    t.masks.copy_(_ints([M.signed(m) for m in bits], dev, torch.int64))
    draft_attention(q, *pools, t, out)
    assert not _refused(b)
    want, A = M.attention(q.double(), k, v, _seen(bits, cached, n, dev))
    _check(out.view(n, Hq, D), want, A, n * (Hq // Hkv) <= 64)
    if cached == 0:
        assert bool((out[3:5] == 0).all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (16, 2), (32, 2), (32, 1)])
@pytest.mark.parametrize("cached", [0, 40, 2000])
def test_what_a_row_does_not_read_does_not_reach_it(cuda_device, cached, Hq, Hkv, fp8):
    """Infinite and NaN keys and values of other branches; those of its own do."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, n = cuda_device, 11
    gen = torch.Generator(device=dev).manual_seed(cached)
    # two branches: odd rows, even rows
    tree = [-1, 0, 0] + [i - 2 for i in range(3, n)]
    b, t, _ = _step(dev, [cached], [tree], 16, Hq, Hkv, max_nodes=n)
    pools, scales, [(k, v)] = _filled(b, [cached + n], fp8, gen)
    q = _rand(n, Hq, D, gen=gen)
    clean, out = (torch.empty(n, Hq * D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    draft_attention(q, *pools, t, clean, *scales)
    for pool, bad in zip(pools, (math.nan, math.nan if fp8 else math.inf)):
        pos = cached + 5  # an odd row
        flat = pool.view(torch.uint8) if fp8 else pool
        code = torch.tensor(bad).to(pool.dtype).to(dev)
        flat[b.table[0, pos // 16].long(), :, pos % 16] = code.view(torch.uint8) if fp8 else code
    draft_attention(q, *pools, t, out, *scales)
    assert not _refused(b)
    reads = torch.tensor([m >> 5 & 1 for m in M.masks(tree)], dtype=torch.bool)
    assert torch.equal(out[~reads.to(dev)], clean[~reads.to(dev)])
    assert reads.sum() == 3 and bool((~out[reads.to(dev)].float().isfinite()).all())


def test_infinite_values_arrive_as_infinite(cuda_device):
    """A value of +inf at a position that is read gives +inf, not NaN."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, n = cuda_device, 9
    for Hq in (1, 4, 8, 16, 32):
        gen = torch.Generator(device=dev).manual_seed(Hq)
        b, t, _ = _step(dev, [70], [[-1] + [0] * (n - 1)], 16, Hq, 1, max_nodes=n)
        pools, _, _ = _filled(b, [70 + n], False, gen)
        pools[1][b.table[0, 4].long(), :, 73 - 64] = math.inf  # row 3's
        pools[1][b.table[0, 1].long(), :, 4, 7] = -math.inf    # position 20's, dim 7
        q = _rand(n, Hq, D, gen=gen)
        out = torch.empty(n, Hq, D, dtype=torch.bfloat16, device=dev)
        draft_attention(q, *pools, t, out)
        torch.cuda.synchronize()
        dims = torch.arange(D, device=dev) != 7
        assert bool((out[3][:, dims] == math.inf).all()) and bool(out[3][:, 7].isnan().all())
        others = torch.arange(n, device=dev) != 3
        assert bool(out[others][:, :, dims].isfinite().all())
        assert bool((out[others][:, :, 7] == -math.inf).all())


def test_scores_of_any_size(cuda_device):
    """Keys whose scores are -inf, or thousands apart."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, n, c = cuda_device, 8, 50
    for Hq in (1, 4, 8, 16, 32):
        gen = torch.Generator(device=dev).manual_seed(Hq)
        b, t, _ = _step(dev, [c], [list(range(-1, n - 1))], 16, Hq, 1, max_nodes=n)
        pools, _, [(k, v)] = _filled(b, [c + n], False, gen)
        pos = torch.arange(c + n, device=dev)
        where = b.table[0, pos // 16].long(), slice(None), pos % 16
        k[:] = 0
        k[:, :, 0] = torch.linspace(-20_000, 100, c + n, device=dev)[:, None]
        pools[0][where] = k.bfloat16()
        k = pools[0][where].double()
        q = torch.ones(n, Hq, D, dtype=torch.bfloat16, device=dev)
        out = torch.empty(n, Hq, D, dtype=torch.bfloat16, device=dev)
        draft_attention(q, *pools, t, out)
        want, A = M.attention(q.double(), k, v, _seen(M.masks(list(range(-1, n - 1))), c, n, dev))
        _check(out, want, A, n * Hq <= 64)
        # all scores -inf but those of row 6's key
        pools[0][where] = torch.where(pos[:, None, None] == c + 6, 1.0, -math.inf).bfloat16().expand_as(k)
        draft_attention(q, *pools, t, out)
        torch.cuda.synchronize()
        assert bool((out[6:].double() == v[c + 6]).all())


# One workgroup a sequence and head where all of them can have a CU of their own, its
# keys in two halves; two a CU, of half the waves, in larger batches (idle sequences
# here).  32 KV heads: pieces of many steps.
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("idle", [0, 9])
@pytest.mark.parametrize("nodes", [10, 16, 29, 32])
def test_attention_of_long_pieces(cuda_device, nodes, idle, fp8):
    """Lengths at the border of one and two halves, and far from it; callers' masks."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, rng, Hq, Hkv = cuda_device, random.Random(nodes + idle), 128, 32
    gen = torch.Generator(device=dev).manual_seed(nodes)
    lengths = [480, 4100, 481, 513, 1030, 512] + [0] * idle
    cached = [max(0, L - nodes) for L in lengths]
    trees = [M.random_tree(rng, nodes if L else 0, 3) for L in lengths]
    b, t, _ = _step(dev, cached, trees, 16, Hq, Hkv, max_nodes=nodes)
    pools, scales, dense = _filled(b, lengths, fp8, gen)
    bits = [[rng.choice([m, 0, rng.getrandbits(64)]) for m in M.masks(tree)] for tree in trees]
    t.masks.copy_(_ints([M.signed(m) for x in bits for m in x], dev, torch.int64))
    q = _rand(6 * nodes, Hq, D, gen=gen, scale=1.5)
    out = torch.empty(6 * nodes, Hq * D, dtype=torch.bfloat16, device=dev)
    draft_attention(q, *pools, t, out, *scales)
    assert not _refused(b)
    for i, (c, (k, v)) in enumerate(zip(cached[:6], dense)):
        at = slice(i * nodes, (i + 1) * nodes)
        want, A = M.attention(q[at].double(), k, v, _seen(bits[i], c, nodes, dev))
        _check(out[at].view(nodes, Hq, D), want, A, nodes * (Hq // Hkv) <= 64)


@pytest.mark.parametrize("idle", [0, 9])
@pytest.mark.parametrize("nodes", [12, 30])
def test_infinities_in_long_pieces(cuda_device, nodes, idle):
    """Infinities and NaN of both halves and of the tree; scores of -inf in either half,
    and thousands apart."""
    from ecf8_amd.draft_kernels import draft_attention

    dev, rng, Hq, Hkv, S, c = cuda_device, random.Random(nodes), 128, 32, 4, 2500
    gen = torch.Generator(device=dev).manual_seed(nodes)
    cached, L = [c] * S + [0] * idle, c + nodes
    tree = M.random_tree(rng, nodes, 3)
    b, t, _ = _step(dev, cached, [tree] * S + [[]] * idle, 16, Hq, Hkv, max_nodes=nodes)
    pools, _, dense = _filled(b, [L] * S + [0] * idle, False, gen)
    q = _rand(S * nodes, Hq, D, gen=gen)
    out = torch.empty(S * nodes, Hq, D, dtype=torch.bfloat16, device=dev)
    draft_attention(q, *pools, t, out)
    clean = out.clone()
    seen = _seen(M.masks(tree), c, nodes, dev)
    marks = [(3, 5, math.inf), (1100, 9, -math.inf), (2400, 11, math.nan), (1300, 13, math.inf),
             (7, 13, -math.inf), (c + 2, 20, math.inf), (c + nodes - 1, 21, math.nan)]
    want = clean.clone()
    saved = pools[1].clone()
    for pos, d, x in marks:
        pools[1][b.table[:S, pos // 16].long(), :, pos % 16, d] = x
        reads = seen[:, pos].repeat(S)
        old = want[reads, :, d]
        want[reads, :, d] = torch.where(old.isfinite(), torch.zeros_like(old), old) + x
    draft_attention(q, *pools, t, out)
    assert not _refused(b)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out[~want.isnan()], want[~want.isnan()])
    pools[1].copy_(saved)
    pos = torch.arange(L, device=dev)
    q.fill_(1.0)
    for only in (40, 2450):  # in the first and in the last half
        for s in range(S):
            where = b.table[s, pos // 16].long(), slice(None), pos % 16
            k = torch.where(pos[:, None, None] == only, 1.0, -math.inf).bfloat16()
            pools[0][where] = k.expand(L, Hkv, D)
        draft_attention(q, *pools, t, out)
        torch.cuda.synchronize()
        for s in range(S):
            v = dense[s][1][only].repeat_interleave(Hq // Hkv, 0)
            assert bool((out[s * nodes: (s + 1) * nodes].double() == v).all()), (only, s)
    for slope in (1, -1):
        key = torch.linspace(-20_000 * slope, 100 * slope, L, device=dev)
        k = torch.zeros(L, Hkv, D, device=dev)
        k[:, :, 0] = key[:, None]
        for s in range(S):
            pools[0][b.table[s, pos // 16].long(), :, pos % 16] = k.bfloat16()
        draft_attention(q, *pools, t, out)
        for s in range(S):
            at = slice(s * nodes, (s + 1) * nodes)
            x, A = M.attention(q[at].double(), k.bfloat16().double(), dense[s][1], seen)
            _check(out[at], x, A, nodes * (Hq // Hkv) <= 64)


def test_a_plan_of_another_step_is_refused(cuda_device):
    """Trees never planned, planned for the step before, or for other sizes."""
    from ecf8_amd.draft_kernels import DraftTrees, draft_attention, draft_plan
    from ecf8_amd.paged_kernels import paged_plan

    dev = cuda_device
    for Hq, long in ((4, 60), (4, 4000), (32, 4000)):
        trees = [[-1, 0, 1, 1], [-1, 0]]
        b, t, parents = _step(dev, [long, 7], trees, 16, Hq, 1, rows=20)
        pools = [torch.full((b.pages, 1, 16, D), 2.0, dtype=torch.bfloat16, device=dev)
                 for _ in range(2)]
        q = torch.zeros(6, Hq, D, dtype=torch.bfloat16, device=dev)
        out = torch.full((6, Hq * D), 3.0, dtype=torch.bfloat16, device=dev)

        def attend(trees, q=q):
            out.fill_(3.0)
            draft_attention(q, *pools, trees, out)
            return _refused(b)

        assert attend(t) == 0 and bool((out == 2.0).all())
        assert attend(DraftTrees(b, 64, 64)) == 1 and bool((out == 3.0).all())
        assert attend(t, q[:5]) == 1 and bool((out[5:] == 3.0).all())  # fewer rows than the step's
        paged_plan(b, _ints([long - 3, 7], dev), _ints([4, 2], dev))
        assert attend(t) == 1
        assert bool((out[:4] == 3.0).all())
        draft_plan(t, parents)
        assert attend(t) == 0 and bool((out == 2.0).all())
        other = DraftTrees(b, 32, 64)
        other.work[:256].copy_(t.work[:256])
        assert attend(other) == 1 and bool((out == 3.0).all())
        paged_plan(b, _ints([0, 0], dev), _ints([0, 0], dev))
        draft_plan(t, parents)
        assert attend(t) == 0 and bool((out == 3.0).all())


# -------------------------------------------------------- probabilities


def _probability_bound(x, t):
    """want and its tolerance, of float64 logits x [V] at temperature t."""
    e = (x - x.max()) / t
    want = torch.exp(e)
    want = want / want.sum()
    relative = e.abs() * 2.0 ** -23 + 32 * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -14
    return want, want * relative + 2.0 ** -126


@pytest.mark.parametrize("N,V", [(1, 1), (1, 7), (3, 8), (2, 257), (5, 4099), (1, 151_936),
                                 (70, 50_257), (300, 2048), (2, 300_001)])
@pytest.mark.parametrize("scale", [0.1, 3.0, 60.0])
def test_probabilities(cuda_device, N, V, scale):
    """One temperature for all, and one of each row, zero among them."""
    from ecf8_amd.draft_kernels import token_probabilities

    dev = cuda_device
    gen = torch.Generator(device=dev).manual_seed(V)
    x = _rand(N, V, gen=gen, scale=scale)
    out = torch.full((N + 1, V), 7.0, device=dev)
    temps = torch.tensor([[0.7, 0.0, 1.0, 2.5, 0.05, -1.0][i % 6] for i in range(N)], device=dev)
    for t in (0.9, temps):
        assert token_probabilities(x, t, out) is out
        assert bool((out[N:] == 7.0).all())
        for i in range(N):
            ti = t if isinstance(t, float) else float(t[i])
            if ti > 0:
                want, bound = _probability_bound(x[i].double(), ti)
                assert bool(((out[i].double() - want).abs() <= bound).all()), (i, ti)
            else:
                want = torch.zeros(V, device=dev)
                want[(x[i] == x[i].max()).nonzero()[0]] = 1.0
                assert torch.equal(out[i], want), i


def test_probabilities_of_strided_and_unaligned_rows(cuda_device):
    from ecf8_amd.draft_kernels import token_probabilities

    dev, N, V = cuda_device, 5, 3001
    gen = torch.Generator(device=dev).manual_seed(3)
    x = _rand(N, V + 20, gen=gen)
    whole = torch.full((N, V + 9), 7.0, device=dev)
    for a, c in ((0, 0), (1, 1), (3, 2), (8, 5)):
        part, out = x[:, a: a + V], whole.fill_(7.0)[:, c: c + V]
        token_probabilities(part, 1.0, out)
        for i in range(N):
            want, bound = _probability_bound(part[i].double(), 1.0)
            assert bool(((out[i].double() - want).abs() <= bound).all())
        assert bool((whole[:, :c] == 7.0).all()) and bool((whole[:, c + V:] == 7.0).all())


def test_probabilities_of_strange_logits(cuda_device):
    """-inf is zero; NaN, +inf and rows of -inf alone are NaN; a greedy row's NaN is its
    largest, ties go to the lowest index; temperatures near zero and infinite."""
    from ecf8_amd.draft_kernels import token_probabilities

    dev, V = cuda_device, 40_000
    gen = torch.Generator(device=dev).manual_seed(3)
    x = _rand(1, V, gen=gen).repeat(8, 1)
    x[0, : V - 3] = -math.inf          # whole runs of it
    x[1, 7] = math.nan
    x[2, 20_000] = math.inf
    x[3] = -math.inf
    out = torch.empty(8, V, device=dev)
    token_probabilities(x, 1.0, out)
    want, bound = _probability_bound(x[0].double(), 1.0)
    assert bool(((out[0].double() - want).nan_to_num(nan=1.0).abs() <= bound.nan_to_num()).all())
    assert bool((out[0, : V - 3] == 0).all()) and abs(float(out[0].sum()) - 1) < 1e-5
    assert bool(out[1:4].isnan().all()) and bool(out[4:].isfinite().all())
    token_probabilities(x, 0.0, out)
    top = out.argmax(-1).tolist()
    assert bool((out.sum(-1) == 1).all()) and top[1] == 7 and top[2] == 20_000 and top[3] == 0
    x[4, 100], x[4, 39_999], x[4, 50] = 50.0, 50.0, 50.0
    x[5] = 0.0
    x[5, 1::2] = -0.0
    token_probabilities(x, torch.zeros(8, device=dev), out)
    assert out.argmax(-1).tolist()[4:6] == [50, 0] and bool((out.sum(-1) == 1).all())
    for t, even in ((1e-30, False), (1e-45, False), (3e38, True), (math.inf, True)):
        token_probabilities(x[4:7], torch.full((3,), t, device=dev), out[:3])
        got = out[:3].double()
        if even:
            assert bool(((got * V - 1).abs() < 1e-3).all())
        else:
            ties = x[4:7] == x[4:7].amax(-1, keepdim=True)
            want = ties / ties.sum(-1, keepdim=True)
            assert bool(((got - want).abs() <= want * 2.0 ** -20).all())
    token_probabilities(x[4:7], math.nan, out[:3])
    assert bool(out[:3].isnan().all())


# --------------------------------------------------------- verification


def _distributions(N, V, gen, sharp, near):
    a = torch.randn(N, V, generator=gen, device=gen.device) * sharp
    b = a + near * torch.randn(N, V, generator=gen, device=gen.device)
    return torch.softmax(a, -1), torch.softmax(b, -1)


def _drafted(trees, draft, gen, drawn):
    """Tokens of the packed rows: of a row's children, its most probable ones, or
    drawn from its probabilities."""
    tokens, a = [], 0
    for tree in trees:
        kids = [sum(p == i for p in tree) for i in range(len(tree))]
        given = [0] * len(tree)
        for i, p in enumerate(tree):
            if p < 0:
                tokens.append(3 % draft.shape[1])
                continue
            row = draft[a + p]
            if drawn:
                tokens.append(int(torch.multinomial(row, 1, generator=gen)))
            else:
                tokens.append(int(torch.topk(row, kids[p]).indices[given[p]]))
            given[p] += 1
        a += len(tree)
    return tokens


@pytest.mark.parametrize("rows", [None, 1000])
@pytest.mark.parametrize("V", [1, 2, 255, 257])
def test_verify_of_small_vocabularies_in_large_batches(cuda_device, V, rows):
    """A batch with room for more rows than its trees can have; one token."""
    from ecf8_amd.draft_kernels import draft_verify

    dev, S, n, rng = cuda_device, 7, 9, random.Random(V)
    gen = torch.Generator(device=dev).manual_seed(V)
    trees = [M.random_tree(rng, rng.choice([n, 4, 0]), 3) for _ in range(S)]
    b, t, _ = _step(dev, [5] * S, trees, 16, max_nodes=n, kids=3, rows=rows)
    N = sum(len(x) for x in trees)
    target, draft = _distributions(N, V, gen, 1.0, 0.7)
    tokens = _drafted(trees, draft, gen, True)
    accept, sample = (torch.rand(k, generator=gen, device=dev) for k in (N, S))
    draft_verify(t, _ints(tokens, dev, torch.int64), target, accept, sample, draft=draft)
    assert not _refused(b)
    a = 0
    for s, tree in enumerate(trees):
        k = len(tree)
        if k:
            assert _verified(t, s) == M.verify(
                tree, tokens[a: a + k], target[a: a + k].double().cpu(), accept[a: a + k].tolist(),
                float(sample[s]), draft[a: a + k].double().cpu())
        a += k


def _verified(t, s):
    n = int(t.kept[s])
    path, emitted = t.path[s].tolist(), t.emitted[s].tolist()
    assert path[n:] == [-1] * (t.max_nodes - n) and emitted[n:] == [-1] * (t.max_nodes - n)
    if n:
        assert emitted[n - 1] == int(t.next_token[s])
    return path[:n], emitted[:n]


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("S,nodes,kids,V,sharp,near", [
    (1, 1, 1, 5, 1.0, 1.0), (1, 64, 1, 300, 1.0, 0.1), (5, 64, 63, 70, 1.0, 1.0),
    (40, 12, 3, 1000, 2.0, 0.5), (40, 12, 3, 63, 0.5, 3.0), (16, 26, 4, 50_257, 3.0, 0.5),
    (9, 33, 2, 151_936, 3.0, 0.3), (200, 6, 2, 997, 2.0, 1.0), (3, 20, 19, 64, 0.1, 0.1),
    (30, 26, 4, 5003, 12.0, 1.0), (64, 64, 8, 997, 8.0, 2.0)])
def test_verify_matches_the_model(cuda_device, S, nodes, kids, V, sharp, near, drawn):
    from ecf8_amd.draft_kernels import draft_verify

    dev, rng = cuda_device, random.Random(S * nodes + V)
    gen = torch.Generator(device=dev).manual_seed(S + V)
    new = [rng.choice([nodes, nodes, rng.randint(1, nodes), 0]) for _ in range(S)]
    new[0] = nodes
    trees = [M.random_tree(rng, n, min(kids, V)) for n in new]
    b, t, _ = _step(dev, [5] * S, trees, 16, max_nodes=nodes, kids=kids)
    N = sum(new)
    target, draft = _distributions(N, V, gen, sharp, near)
    tokens = _drafted(trees, draft, gen, drawn)
    accept, sample = (torch.rand(k, generator=gen, device=dev) for k in (N, S))
    draft_verify(t, _ints(tokens, dev, torch.int64), target, accept, sample,
                 draft=draft if drawn else None)
    assert not _refused(b)
    a, lengths = 0, []
    p64, q64, u, v = target.double().cpu(), draft.double().cpu(), accept.tolist(), sample.tolist()
    for s, tree in enumerate(trees):
        n = len(tree)
        got = _verified(t, s)
        if not n:
            assert got == ([], []) and int(t.next_token[s]) == -1
            continue
        want = M.verify(tree, tokens[a: a + n], p64[a: a + n], u[a: a + n], v[s],
                        q64[a: a + n] if drawn else None)
        assert got == want, (s, n)
        lengths.append(len(want[0]))
        a += n
    if sharp > 5:  # few tokens have most of the probability, so drafts are accepted
        assert max(lengths) > 3


@pytest.mark.parametrize("drawn", [False, True])
def test_emitted_tokens_are_distributed_as_the_targets(cuda_device, drawn):
    """4096 sequences of the same probabilities, three drafts of the first token: of N
    draws a token of probability p is drawn N p times within 5.5 standard
    deviations (one in 10^7, for each of 24 tokens and four runs)."""
    from ecf8_amd.draft_kernels import draft_verify

    dev, S, V = cuda_device, 4096, 24
    gen = torch.Generator(device=dev).manual_seed(11)
    p, q = (x[0] for x in _distributions(1, V, gen, 1.5, 1.5))
    b, t, _ = _step(dev, [1] * S, [[-1, 0, 0, 0]] * S, 16, max_nodes=4, kids=3)
    count = torch.zeros(V, dtype=torch.float64, device=dev)
    top = torch.topk(q, 3).indices
    for _ in range(4):
        tokens = torch.zeros(S, 4, dtype=torch.int64, device=dev)
        tokens[:, 1:] = torch.multinomial(q, 3 * S, replacement=True, generator=gen).view(S, 3) \
            if drawn else top
        accept, sample = (torch.rand(k, generator=gen, device=dev) for k in (4 * S, S))
        rows = p.expand(4 * S, V).contiguous()
        draft_verify(t, tokens.view(-1), rows, accept, sample,
                     draft=q.expand(4 * S, V).contiguous() if drawn else None)
        assert not _refused(b)
        count += torch.bincount(t.emitted[:, 0], minlength=V)
        # the second token, where there is one, is drawn from p too: no more to be accepted
        assert bool(((t.kept == 1) | (t.kept == 2)).all())
    n = 4 * S
    want = p.double() * n
    assert bool(((count - want).abs() <= 5.5 * (want * (1 - p.double())).sqrt() + 1).all())
    assert 0.05 < float((t.kept == 2).double().mean()) < 0.95


def test_verify_at_the_borders(cuda_device):
    """Probabilities of one and zero, equal ones, random numbers of 0 and next to 1,
    the same draft twice, a residual of nothing, drafts outside the vocabulary."""
    from ecf8_amd.draft_kernels import draft_verify

    dev, V = cuda_device, 130
    almost = 1 - 2.0 ** -24

    def run(tree, tokens, target, accept, sample, draft=None):
        b, t, _ = _step(dev, [3], [tree], 16, max_nodes=8, kids=7)
        args = [torch.tensor(x, dtype=torch.float32).to(dev) for x in (target, accept, [sample])]
        draft_verify(t, _ints(tokens, dev, torch.int64), *args,
                     draft=None if draft is None else torch.tensor(draft).float().to(dev))
        return _refused(b), *_verified(t, 0)

    def one(*at):
        return [1.0 / len(at) if v in at else 0.0 for v in range(V)]

    # greedy rows: the draft that is the largest is taken whatever the numbers
    for u in (0.0, almost):
        assert run([-1, 0, 0, 2], [9, 5, 7, 100], [one(7), one(0), one(100), one(129)], [u] * 4,
                   u) == (0, [0, 2, 3], [7, 100, 129])
        # none is: the target's own
        assert run([-1, 0, 0], [9, 5, 7], [one(8), one(0), one(0)], [u] * 3, u) == (0, [0], [8])
    # of equal ones the sample says which
    four = one(3, 4, 5, 129)
    for u, want in ((0.0, 3), (0.2499, 3), (0.25, 4), (0.5, 5), (0.75, 129), (almost, 129)):
        assert run([-1], [0], [four], [0.5], u) == (0, [0], [want])
    # a sample of one or more, or below zero, or NaN: the last, or the first
    for u, want in ((1.0, 129), (7.0, 129), (-1.0, 3), (math.nan, 3)):
        assert run([-1], [0], [four], [0.5], u) == (0, [0], [want])
    # the same draft twice: not left after it was rejected
    assert run([-1, 0, 0, 0], [0, 3, 3, 4], [four] * 4, [0, 0.9, 0.0, 0.9], 0.0) == (0, [0], [5])
    assert run([-1, 0, 0, 0], [0, 3, 3, 4], [four] * 4, [0, 0.9, 0.0, 0.3], 0.0) == (0, [0, 3], [4, 3])
    # drawn, p = q: always accepted; nothing left by q > p: the target's own
    assert run([-1, 0], [0, 4], [four] * 2, [0, almost], 0.3, [four] * 2) == (0, [0, 1], [4, 4])
    more = [2 * x for x in four]
    assert run([-1, 0], [0, 4], [four] * 2, [0, 0.6], 0.3, [more] * 2) == (0, [0], [4])
    # a draft that q holds impossible: taken if the target has it
    assert run([-1, 0], [0, 3], [four] * 2, [0, 0.9], 0.0, [one(9)] * 2) == (0, [0, 1], [3, 3])
    assert run([-1, 0], [0, 9], [four] * 2, [0, 0.0], 0.0, [one(9)] * 2) == (0, [0], [3])
    # drafts outside the vocabulary: never taken, and refused
    for bad in (V, -1, 2 ** 40, -2 ** 63):
        for draft in (None, [one(9)] * 2):
            assert run([-1, 0], [0, bad], [four] * 2, [0, 0.0], 0.0, draft)[0] == 1
            assert run([-1, 0], [0, bad], [four] * 2, [0, 0.0], 0.0, draft)[1] == [0]
    # (row 0's token has no part in it)
    assert run([-1, 0], [-1, 3], [four] * 2, [0, 0.0], 0.0) == (0, [0, 1], [3, 3])
    # no probabilities
    for row in ([0.0] * V, [math.nan] * V, [math.inf] * V):
        assert run([-1], [0], [row], [0.5], 0.5) == (1, [0], [-1])


def test_verify_of_strided_rows_and_refused_steps(cuda_device):
    from ecf8_amd.draft_kernels import draft_verify

    dev, S, V, n = cuda_device, 6, 1001, 7
    gen = torch.Generator(device=dev).manual_seed(5)
    trees = [M.random_tree(random.Random(s), n, 2) for s in range(S)]
    b, t, _ = _step(dev, [5] * S, trees, 16, max_nodes=n, kids=2)
    target, draft = _distributions(S * n, V, gen, 2.0, 0.5)
    tokens = _ints(_drafted(trees, draft, gen, True), dev, torch.int64)
    accept, sample = (torch.rand(k, generator=gen, device=dev) for k in (S * n, S))
    draft_verify(t, tokens, target, accept, sample, draft=draft)
    want = t.kept.clone(), t.path.clone(), t.emitted.clone(), t.next_token.clone()
    wide = [torch.full((S * n, V + 13), 9.0, device=dev) for _ in range(2)]
    p, q = wide[0][:, 3: 3 + V], wide[1][:, 8: 8 + V]
    p.copy_(target), q.copy_(draft)
    t.kept.zero_(), t.path.zero_(), t.emitted.zero_(), t.next_token.zero_()
    draft_verify(t, tokens, p, accept, sample, draft=q)
    assert not _refused(b)
    assert all(torch.equal(x, y) for x, y in zip(want, (t.kept, t.path, t.emitted, t.next_token)))
    # fewer rows than the step's: the last sequence is not verified
    m = S * n - 1
    draft_verify(t, tokens[:m], p[:m], accept[:m], sample, draft=q[:m])
    assert _refused(b)
    assert torch.equal(t.emitted[: S - 1], want[2][: S - 1])
    assert int(t.kept[S - 1]) == 0 and int(t.next_token[S - 1]) == -1
    for bad in (dict(tokens=tokens[:m]), dict(accept=accept[:m]), dict(sample=sample[:1]),
                dict(draft=draft[:m]), dict(target=target.double()), dict(tokens=tokens.int()),
                dict(target=target.t()), dict(draft=draft.cpu())):
        kw = {**dict(tokens=tokens, target=target, accept=accept, sample=sample, draft=draft), **bad}
        with pytest.raises(ECF8Error):
            draft_verify(t, **kw)


# ------------------------------------------------------------- the move


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("S,nodes,page,Hkv,layers", [
    (1, 1, 16, 2, 1), (1, 64, 1, 1, 3), (5, 64, 4, 3, 2), (7, 26, 16, 8, 36), (40, 9, 64, 2, 5),
    (3, 33, 1024, 1, 70)])
def test_keep_matches_the_model(cuda_device, S, nodes, page, Hkv, layers, fp8):
    """Every byte of every pool; chains, paths at random, whole paths of every other
    row, idle sequences."""
    from ecf8_amd.draft_kernels import KeepPlan, draft_keep

    dev, rng = cuda_device, random.Random(S + nodes)
    gen = torch.Generator(device=dev).manual_seed(S)
    new = [rng.choice([0, 1, nodes, rng.randint(1, nodes)]) for _ in range(S)]
    new[0] = nodes
    cached = [rng.choice([0, 1, 15, rng.randint(0, 100)]) for _ in range(S)]
    b, t, _ = _step(dev, cached, [M.random_tree(rng, n, 8) for n in new], page, Hkv, Hkv,
                    max_nodes=nodes)
    pools = [torch.randint(256, (b.pages, Hkv, page, D * (1 if fp8 else 2)), generator=gen,
                           device=dev, dtype=torch.uint8) for _ in range(2 * layers)]
    kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
    typed = [p.view(kind) for p in pools]
    plan = KeepPlan(t, list(zip(typed[::2], typed[1::2])))
    for how in ("some", "all", "odd", "one"):
        paths = []
        for n in new:
            rows = list(range(n))
            path = {"some": [r for r in rows if r == 0 or rng.random() < 0.4], "all": rows,
                    "odd": rows[:1] + rows[1:: 2][1:], "one": rows[:1]}[how]
            paths.append(path)
        t.kept.copy_(_ints([len(p) for p in paths], dev))
        t.path.copy_(_ints([p + [-1] * (nodes - len(p)) for p in paths], dev))
        want = [p.clone() for p in pools]
        for s, path in enumerate(paths):
            if path:
                pos = cached[s] + torch.tensor(path, device=dev)
                to = cached[s] + torch.arange(len(path), device=dev)
                for w, p in zip(want, pools):
                    w[b.table[s, to // page].long(), :, to % page] = \
                        p[b.table[s, pos // page].long(), :, pos % page]
        draft_keep(plan)
        assert not _refused(b)
        for i, (w, p) in enumerate(zip(want, pools)):
            assert torch.equal(w, p), (how, i)


def test_keep_refuses_paths_that_are_none(cuda_device):
    """It is cut before the first row that is no later one, or not the sequence's."""
    from ecf8_amd.draft_kernels import KeepPlan, draft_keep

    dev = cuda_device
    b, t, _ = _step(dev, [10], [list(range(-1, 7))], 16, 1, 1, max_nodes=12)
    pool = [torch.zeros(b.pages, 1, 16, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    plan = KeepPlan(t, [tuple(pool)])
    for kept, path, moved in ((4, [0, 2, 2, 5], [0, 2]), (3, [0, 3, 8], [0, 3]), (3, [1, 2, 3], []),
                              (3, [0, -1, 4], [0]), (13, [0, 2, 3], [0, 2, 3]), (2 ** 31 - 1, [0], [0])):
        for p in pool:
            p.zero_()
            p[int(b.table[0, 0]), 0, :] = torch.arange(16, device=dev)[:, None].bfloat16()
            p[int(b.table[0, 1]), 0, :] = torch.arange(16, 32, device=dev)[:, None].bfloat16()
        t.kept.fill_(kept)
        t.path.copy_(_ints([path + [-1] * (12 - len(path))], dev))
        draft_keep(plan)
        assert _refused(b)
        want = list(range(32))
        for i, r in enumerate(moved):
            want[10 + i] = 10 + r
        for p in pool:
            got = torch.cat([p[int(b.table[0, 0]), 0, :, 0], p[int(b.table[0, 1]), 0, :, 0]])
            assert got.tolist() == want, (kept, path)
    t.kept.fill_(-5)
    draft_keep(plan)
    assert not _refused(b)  # idle
    with pytest.raises(ECF8Error):
        KeepPlan(t, [(pool[0], pool[0])])
    with pytest.raises(ECF8Error):
        KeepPlan(t, [(pool[0], pool[1].to(torch.float8_e4m3fn))])
    with pytest.raises(ECF8Error):
        KeepPlan(t, [(pool[0], pool[1][:1])])
