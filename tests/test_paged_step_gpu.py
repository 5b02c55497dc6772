"""The ragged-batch kernels together, as a server runs them: plan, write and
attention of one step after the other, eager, captured and on other streams."""

from __future__ import annotations

import math
import random

import pytest
import torch

from ecf8_amd._lib import ECF8Error

pytestmark = pytest.mark.gpu

D, HQ, HKV, EPS = 128, 8, 2, 1e-6


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


class _Server:
    """A batch, one layer's pools and weights, and what each sequence holds."""

    def __init__(self, dev, S, rows, pages, page, max_len, fp8=False, seed=0):
        from ecf8_amd.paged_kernels import PagedBatch

        gen = torch.Generator(device=dev).manual_seed(seed)
        self.dev, self.S, self.rows, self.fp8, self.gen = dev, S, rows, fp8, gen
        self.batch = PagedBatch(S, rows, pages, page, max_len, HQ, HKV, dev)
        kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
        self.pools = [torch.full((pages, HKV, page, D), math.nan, device=dev).to(kind)
                      for _ in range(2)]
        self.scales = ([torch.full((HKV,), x, device=dev) for x in (0.03, 0.02)] if fp8
                       else [None, None])
        self.norms = [(1 + 0.2 * torch.randn(D, generator=gen, device=dev)).bfloat16()
                      for _ in range(2)]
        ang = torch.rand(self.batch.max_len, 64, generator=gen, device=dev) * 6.28
        self.tables = torch.cos(ang), torch.sin(ang)
        self.qkv = torch.zeros(rows, (HQ + 2 * HKV) * D, dtype=torch.bfloat16, device=dev)
        self.q = torch.zeros(rows, HQ, D, dtype=torch.bfloat16, device=dev)
        self.out = torch.zeros(rows, HQ * D, dtype=torch.bfloat16, device=dev)
        self.cached, self.new, self.release = (torch.zeros(S, dtype=torch.int32, device=dev)
                                               for _ in range(3))
        self.held = [[] for _ in range(S)]  # the qkv rows of each sequence so far

    def step(self):
        from ecf8_amd.paged_kernels import paged_attention, paged_plan, paged_qk_norm_rope

        paged_plan(self.batch, self.cached, self.new, self.release)
        paged_qk_norm_rope(self.qkv, self.batch, *self.norms, EPS, *self.tables, self.q,
                           *self.pools, *self.scales)
        paged_attention(self.q, *self.pools, self.batch, self.out, k_scale=self.scales[0],
                        v_scale=self.scales[1])

    def feed(self, new, release):
        """The next step's inputs: new tokens and released sequences."""
        for s in range(self.S):
            if release[s]:
                self.held[s] = []
        self.cached.copy_(_ints([len(h) for h in self.held], self.dev))
        self.new.copy_(_ints(new, self.dev))
        self.release.copy_(_ints(release, self.dev))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=self.gen, device=self.dev) * 2)
        at = 0
        for s, n in enumerate(new):
            self.held[s] += list(self.qkv[at: at + n].clone())
            at += n
        return at

    def check(self, new):
        """q and the pages against float64: rounded to bf16 (2^-8 of it) or e4m3
        (2^-4, or half the smallest step 2^-10; past 448 scales 448), fp32 before
        that (2^-19 of a row's largest).  The attention against float64 of that q and these
        pages: 2^-8 of A = sum p |v|, twice 2^-8 of the output, 2^-10 of A (see
        test_paged_gpu)."""
        b, page = self.batch, self.batch.page_size
        at = 0

        def near(got, want, step, least=0.0):
            top = want.abs().amax(-1, keepdim=True)
            return bool(((got - want).abs() <= want.abs() * step + least + top * 2.0 ** -19).all())

        for s, n in enumerate(new):
            L = len(self.held[s])
            if not L:
                continue
            x = torch.stack(self.held[s]).double().view(L, -1, D)
            c, sn = (t.double()[:L, None] for t in self.tables)

            def turned(x, w):
                x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
                a, b = x[..., :64], x[..., 64:]
                return torch.cat([a * c - b * sn, b * c + a * sn], -1)

            p = torch.arange(L, device=self.dev)
            where = b.table[s, p // page].long(), p % page
            kv = []
            for pool, scale, want in zip(self.pools, self.scales, (
                    turned(x[:, HQ: HQ + HKV], self.norms[1]), x[:, HQ + HKV:])):
                if self.fp8:
                    got = pool.view(torch.uint8)[where[0], :, where[1]].view(pool.dtype).double()
                    codes = (want / scale.double()[:, None]).clamp(-448, 448)
                    assert near(got, codes, 2.0 ** -4, 2.0 ** -10)
                    got = got * scale.double()[:, None]
                else:
                    got = pool[where[0], :, where[1]].double()
                    assert near(got, want, 2.0 ** -8)
                kv.append(got.repeat_interleave(HQ // HKV, 1).transpose(0, 1).contiguous())
            if not n:
                continue
            q = self.q[at: at + n].double()
            assert near(q, turned(x[:, :HQ], self.norms[0])[-n:], 2.0 ** -8)
            e = q.transpose(0, 1) @ kv[0].transpose(1, 2).contiguous() / math.sqrt(D)
            e.masked_fill_(p[None] > L - n + torch.arange(n, device=self.dev)[:, None], -math.inf)
            w = torch.softmax(e, -1)
            want, A = (w @ kv[1]).transpose(0, 1), (w @ kv[1].abs()).transpose(0, 1)
            got = self.out[at: at + n].view(n, HQ, D).double()
            bound = (2 * want.abs() + A) * 2.0 ** -8 + A * 2.0 ** -10
            assert bool(((got - want).abs() <= bound).all()), (s, n)
            at += n


def _traffic(rng, server, steps, cap):
    """New tokens and releases of some steps of a server: prompts, single
    tokens, chunks, idle and finished sequences."""
    out = []
    length = [0] * server.S
    for _ in range(steps):
        release = [int(length[s] > 0 and rng.random() < 0.2) for s in range(server.S)]
        new, left = [], server.rows
        for s in range(server.S):
            if release[s]:
                length[s] = 0
            n = rng.choice([0, 1, 1, 1, 5, 70]) if length[s] else rng.choice([0, 1, 33, 150])
            n = min(n, left, cap - length[s])
            new.append(n)
            left -= n
            length[s] += n
        out.append((new, release))
    return out


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [4, 16, 128])
def test_served_steps(cuda_device, page, fp8):
    server = _Server(cuda_device, 6, 400, 6 * (-(-600 // page)), page, 600, fp8, seed=page)
    for new, release in _traffic(random.Random(page), server, 8, 600):
        n = server.feed(new, release)
        server.out.fill_(5.0)
        server.step()
        torch.cuda.synchronize()
        server.batch.raise_refused()
        server.check(new)
        assert bool((server.out[n:] == 5.0).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_captured_steps_replay_with_other_lengths(cuda_device, fp8):
    """One captured step, replayed for every step of the traffic, against the
    same steps launched one by one on a batch of their own."""
    a, b = (_Server(cuda_device, 5, 300, 200, 16, 500, fp8, seed=9) for _ in range(2))
    for pool, other in zip(a.pools, b.pools):
        other.copy_(pool)
    a.step()  # an empty step: everything is loaded and warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for new, release in _traffic(random.Random(5), a, 10, 500):
        n = a.feed(new, release)
        b.feed(new, release)
        assert torch.equal(a.qkv, b.qkv)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        a.batch.raise_refused()
        assert torch.equal(a.out[:n], b.out[:n])
        for x, y in ((a.batch.table, b.batch.table), (a.batch.lengths, b.batch.lengths),
                     (a.batch.slots, b.batch.slots), (a.batch.n_free, b.batch.n_free)):
            assert torch.equal(x, y)
        a.check(new)


def test_two_batches_on_two_streams(cuda_device):
    """Steps of two batches in flight at once, against the same steps alone."""
    together = [_Server(cuda_device, 4, 300, 150, 16, 500, seed=s) for s in (1, 2)]
    alone = [_Server(cuda_device, 4, 300, 150, 16, 500, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, y in zip(_traffic(random.Random(1), together[0], 5, 500),
                    _traffic(random.Random(2), together[1], 5, 500)):
        rows = [t.feed(*z) for t, z in zip(together, (x, y))]
        for t, z in zip(alone, (x, y)):
            t.feed(*z)
        torch.cuda.synchronize()
        for t, stream in zip(together, streams):
            with torch.cuda.stream(stream):
                t.step()
        torch.cuda.synchronize()
        for t, u, n in zip(together, alone, rows):
            u.step()
            torch.cuda.synchronize()
            assert torch.equal(t.out[:n], u.out[:n])


def test_packed_prompts_captured(cuda_device):
    """ragged_attention in a graph whose prompts' lengths change between the
    replays, against eager calls."""
    from ecf8_amd.paged_kernels import ragged_attention

    dev, N = cuda_device, 700
    gen = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(N, HQ + 2 * HKV, D, generator=gen, device=dev).bfloat16()
    parts = x[:, :HQ], x[:, HQ: HQ + HKV], x[:, HQ + HKV:]
    starts = _ints([0, 0, 0, 0, N], dev)
    out, eager = (torch.zeros(N, HQ * D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    ragged_attention(*parts, starts, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ragged_attention(*parts, starts, out)
    for cuts in ([0, 1, 2, 3, 700], [0, 350, 350, 351, 600], [5, 100, 300, 699, 700], [0, 0, 0, 0, 0]):
        starts.copy_(_ints(cuts, dev))
        x.copy_(torch.randn(x.shape, generator=gen, device=dev))
        out.fill_(2.0)
        eager.fill_(2.0)
        graph.replay()
        ragged_attention(*parts, starts, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert bool((out[cuts[-1]:] == 2.0).all()) and bool((out[: cuts[0]] == 2.0).all())


def test_pools_past_four_gigabytes(cuda_device):
    """Pages at the far end of pools of 3 * 2^30 elements: 64-bit offsets."""
    from ecf8_amd.paged_kernels import PagedBatch, paged_attention, paged_plan, paged_qk_norm_rope

    dev, page, pages, Hkv, T = cuda_device, 1024, 1024, 24, 200
    b = PagedBatch(2, T, pages, page, 2048, Hkv, Hkv, dev)
    b.free.copy_(torch.arange(pages, dtype=torch.int32))  # the last page on top
    pools = [torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    assert pools[0].numel() > 2 ** 31
    gen = torch.Generator(device=dev).manual_seed(8)
    qkv = torch.randn(T, 3 * Hkv * D, generator=gen, device=dev).bfloat16()
    one = torch.ones(D, dtype=torch.bfloat16, device=dev)
    cos, sin = torch.ones(b.max_len, 64, device=dev), torch.zeros(b.max_len, 64, device=dev)
    q = torch.empty(T, Hkv, D, dtype=torch.bfloat16, device=dev)
    out = torch.empty(T, Hkv * D, dtype=torch.bfloat16, device=dev)
    paged_plan(b, _ints([0, 0], dev), _ints([T - 1, 1], dev))
    paged_qk_norm_rope(qkv, b, one, one, EPS, cos, sin, q, *pools)
    paged_attention(q, *pools, b, out)
    torch.cuda.synchronize()
    b.raise_refused()
    assert b.table[:, 0].tolist() == [pages - 1, pages - 2]
    x = qkv.view(T, 3, Hkv, D)
    assert torch.equal(pools[1][pages - 1, :, : T - 1], x[: T - 1, 2].transpose(0, 1))
    assert torch.equal(pools[1][pages - 2, :, 0], x[T - 1, 2])
    assert torch.equal(out[0].view(Hkv, D), x[0, 2])          # a first token reads its own value
    assert torch.equal(out[T - 1].view(Hkv, D), x[T - 1, 2])
    k = pools[0][pages - 1, :, : T - 1].double()
    p = torch.softmax((q[T - 2].double()[:, None] * k).sum(-1) / math.sqrt(D), -1)
    v = x[: T - 1, 2].double().transpose(0, 1)
    want, A = (p[..., None] * v).sum(1), (p[..., None] * v.abs()).sum(1)
    assert bool(((out[T - 2].view(Hkv, D).double() - want).abs()
                 <= (2 * want.abs() + A) * 2.0 ** -8 + A * 2.0 ** -10).all())


@pytest.mark.parametrize("new,rows,max_new", [
    ([50, 1], 51, 1), ([50, 1], 51, 8), ([3, 20], 23, 8), ([8, 1], 9, 4), ([3, 20], 20, None)])
def test_attention_refuses_more_than_it_was_launched_for(cuda_device, new, rows, max_new):
    """max_new or the rows below those of the step: the flag is set."""
    from ecf8_amd.paged_kernels import PagedBatch, paged_attention, paged_plan

    dev = cuda_device
    b = PagedBatch(2, sum(new), 16, 16, 64, 4, 1, dev)
    paged_plan(b, _ints([0, 0], dev), _ints(new, dev))
    q = torch.zeros(sum(new), 4, D, dtype=torch.bfloat16, device=dev)
    out = torch.full((sum(new) + 1, 4 * D), 3.0, dtype=torch.bfloat16, device=dev)
    pools = [torch.zeros(16, 1, 16, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    torch.cuda.synchronize()
    b.raise_refused()
    paged_attention(q[:rows], *pools, b, out, max_new=max_new)
    torch.cuda.synchronize()
    with pytest.raises(ECF8Error):
        b.raise_refused()
    assert bool((out[rows:] == 3.0).all())
    b.raise_refused()  # once


def test_inputs_of_autograd_are_refused(cuda_device):
    from ecf8_amd.paged_kernels import PagedBatch, paged_attention, paged_qk_norm_rope, ragged_attention

    dev = cuda_device
    x = torch.zeros(4, 3, D, dtype=torch.bfloat16, device=dev, requires_grad=True)
    out = torch.zeros(4, D, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ECF8Error, match="autograd"):
        ragged_attention(x[:, :1], x[:, 1:2], x[:, 2:], _ints([0, 4], dev), out)
    b = PagedBatch(1, 4, 4, 4, 16, 1, 1, dev)
    pools = [torch.zeros(4, 1, 4, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    with pytest.raises(ECF8Error, match="autograd"):
        paged_attention(x[:, :1], *pools, b, out)
    one = torch.ones(D, dtype=torch.bfloat16, device=dev)
    tab = torch.ones(b.max_len, 64, device=dev)
    with pytest.raises(ECF8Error, match="autograd"):
        paged_qk_norm_rope(x.view(4, 3 * D), b, one, one, EPS, tab, tab, out, *pools)
    with torch.no_grad():
        ragged_attention(x[:, :1], x[:, 1:2], x[:, 2:], _ints([0, 4], dev), out)
