"""Speculative steps as a server runs them, all operators of include/ecf8_draft.h
one after the other beside the paged cache's: eager, captured, on other streams,
with sequences that finish and are replaced."""

from __future__ import annotations

import math
import random

import draft_model as M
import pytest
import torch

pytestmark = pytest.mark.gpu

D, HQ, HKV, EPS, V, KIDS = 128, 8, 2, 1e-6, 500, 3


def _ints(v, dev, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).to(dev)


class _Server:
    """A batch and its trees, two layers' pools, what each sequence holds, and a
    drafter whose probabilities lie next to the model's."""

    def __init__(self, dev, S, nodes, fp8=False, seed=0, page=16, max_len=300):
        from ecf8_amd.draft_kernels import DraftTrees, KeepPlan
        from ecf8_amd.paged_kernels import PagedBatch

        self.dev, self.S, self.nodes, self.rows, self.max_len = dev, S, nodes, S * nodes, max_len
        self.gen = torch.Generator(device=dev).manual_seed(seed)
        self.rng = random.Random(seed)
        pages = S * -(-max_len // page)
        self.batch = PagedBatch(S, self.rows, pages, page, max_len, HQ, HKV, dev)
        self.trees = DraftTrees(self.batch, nodes, KIDS)
        kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
        self.layers = [[torch.full((pages, HKV, page, D), math.nan, device=dev).to(kind)
                        for _ in range(2)] for _ in range(2)]
        self.scales = ([torch.full((HKV,), x, device=dev) for x in (0.03, 0.02)] if fp8
                       else [None, None])
        self.keep = KeepPlan(self.trees, self.layers)
        self.norms = [(1 + 0.2 * torch.randn(D, generator=self.gen, device=dev)).bfloat16()
                      for _ in range(2)]
        ang = torch.rand(self.batch.max_len, 64, generator=self.gen, device=dev) * 6.28
        self.tables = torch.cos(ang), torch.sin(ang)
        N = self.rows
        bf = dict(dtype=torch.bfloat16, device=dev)
        self.qkv = [torch.zeros(N, (HQ + 2 * HKV) * D, **bf) for _ in range(2)]
        self.q = [torch.zeros(N, HQ, D, **bf) for _ in range(2)]
        self.out = [torch.zeros(N, HQ * D, **bf) for _ in range(2)]
        self.logits = torch.zeros(N, V, **bf)
        self.draft, self.target = (torch.zeros(N, V, device=dev) for _ in range(2))
        self.cached, self.new, self.release = (torch.zeros(S, dtype=torch.int32, device=dev)
                                               for _ in range(3))
        self.parents = torch.full((N,), -1, dtype=torch.int32, device=dev)
        self.tokens = torch.zeros(N, dtype=torch.int64, device=dev)
        self.temperature, self.accept = (torch.zeros(N, device=dev) for _ in range(2))
        self.sample = torch.zeros(S, device=dev)
        self.held = [0] * S
        self.drawn = True

    def step(self):
        from ecf8_amd import draft_kernels as K
        from ecf8_amd.paged_kernels import paged_plan, paged_qk_norm_rope

        paged_plan(self.batch, self.cached, self.new, self.release)
        K.draft_plan(self.trees, self.parents)
        for qkv, q, out, pools in zip(self.qkv, self.q, self.out, self.layers):
            paged_qk_norm_rope(qkv, self.batch, *self.norms, EPS, *self.tables, q, *pools,
                               *self.scales)
            K.draft_attention(q, *pools, self.trees, out, *self.scales)
        K.token_probabilities(self.logits, self.temperature, self.target)
        K.draft_verify(self.trees, self.tokens, self.target, self.accept, self.sample,
                       draft=self.draft if self.drawn else None)

    def move(self):
        from ecf8_amd.draft_kernels import draft_keep

        draft_keep(self.keep)

    def feed(self):
        """The next step's inputs: trees, drafts and random numbers; some sequences
        finish, are idle or start with their only token."""
        g, dev = self.gen, self.dev
        release = [int(h + self.nodes > self.max_len or self.rng.random() < 0.1) for h in self.held]
        self.held = [0 if r else h for h, r in zip(self.held, release)]
        n = [self.rng.choice([0, 1, self.nodes, self.nodes, self.rng.randint(1, self.nodes)])
             for _ in range(self.S)]
        self.tree = [M.random_tree(self.rng, k, KIDS) for k in n]
        self.cached.copy_(_ints(self.held, dev))
        self.new.copy_(_ints(n, dev))
        self.release.copy_(_ints(release, dev))
        for x in self.qkv:
            x.copy_(torch.randn(x.shape, generator=g, device=dev) * 2)
        self.logits.copy_(torch.randn(self.logits.shape, generator=g, device=dev) * 3)
        guess = self.logits.float() + 0.4 * torch.randn(self.logits.shape, generator=g, device=dev)
        self.draft.copy_(torch.softmax(guess, -1))
        N = sum(n)
        flat = [p for t in self.tree for p in t]
        self.parents.fill_(-1)
        self.parents[:N] = _ints(flat, dev)
        first = [i - k for t, a in zip(self.tree, _ends(n)) for i, k in [(a, len(t))]]
        above = [f + max(p, 0) for t, f in zip(self.tree, first) for p in t]
        rank = [sum(x == p for x in t[:i]) for t in self.tree for i, p in enumerate(t)]
        if N:
            picks = (torch.multinomial(self.draft, KIDS, replacement=True, generator=g)
                     if self.drawn else torch.topk(self.draft, KIDS, -1).indices)
            self.tokens[:N] = picks[_ints(above, dev, torch.int64), _ints(rank, dev, torch.int64)]
        t = torch.rand(self.S, generator=g, device=dev) + 0.3
        t[::3] = 0.0
        self.temperature.fill_(1.0)
        if N:
            self.temperature[:N] = t.repeat_interleave(_ints(n, dev, torch.int64))
        self.accept.copy_(torch.rand(self.rows, generator=g, device=dev))
        self.sample.copy_(torch.rand(self.S, generator=g, device=dev))
        return N

    def pages(self, pool, s, length):
        p = torch.arange(length, device=self.dev)
        page = self.batch.page_size
        x = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool.view(torch.int16)
        return x[self.batch.table[s, p // page].long(), :, p % page]

    def check(self):
        """The step before the move; returns what the pages have to hold after it."""
        a, after = 0, []
        for s, tree in enumerate(self.tree):
            n, c = len(tree), self.held[s]
            if not n:
                after.append([self.pages(p, s, c).clone() for l in self.layers for p in l])
                continue
            bits = M.masks(tree)
            depth = [bin(m).count("1") - 1 for m in bits]
            seen = torch.cat([torch.ones(n, c, dtype=torch.bool), torch.tensor(
                [[bool(m >> j & 1) for j in range(n)] for m in bits])], 1).to(self.dev)
            for qkv, q, out, pools in zip(self.qkv, self.q, self.out, self.layers):
                # keys turned at the rows' depths
                x = qkv[a: a + n].double().view(n, -1, D)[:, HQ: HQ + HKV]
                x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * self.norms[1].double()
                cs, sn = (t.double()[c + torch.tensor(depth, device=self.dev)][:, None]
                          for t in self.tables)
                u, v = x[..., :64], x[..., 64:]
                x = torch.cat([u * cs - v * sn, v * cs + u * sn], -1)
                kv = []
                for pool, scale in zip(pools, self.scales):
                    y = self.pages(pool, s, c + n).view(pool.dtype)
                    y = y.double() if scale is None else y.double() * scale.double()[:, None]
                    kv.append(y)
                step = 2.0 ** -8 if self.scales[0] is None else 2.0 ** -4
                top = x.abs().amax(-1, keepdim=True)
                floor = 0.0 if self.scales[0] is None else 2.0 ** -10 * 0.03
                assert bool(((kv[0][c:] - x).abs() <= x.abs() * step + floor + top * 2.0 ** -19).all())
                want, A = M.attention(q[a: a + n].double(), *kv, seen)
                got = out[a: a + n].view(n, HQ, D).double()
                # the output's rounding, 2^-8 of it, and fp32's, 2^-10 of A; over 64 rows of a
                # KV head probabilities p are rounded to bf16 by 1 + d, |d| <= 2^-8, in both
                # sums: sum p d (v - o), at most 2^-8 of A and of |o|
                bound = want.abs() * 2.0 ** -8 + A * 2.0 ** -10
                if self.nodes * HQ // HKV > 64:
                    bound += (want.abs() + A) * 2.0 ** -8
                assert bool(((got - want).abs() <= bound).all()), (s, n)
            path, emitted = M.verify(
                tree, self.tokens[a: a + n].tolist(), self.target[a: a + n].double().cpu(),
                self.accept[a: a + n].tolist(), float(self.sample[s]),
                self.draft[a: a + n].double().cpu() if self.drawn else None)
            k = len(path)
            assert int(self.trees.kept[s]) == k
            assert self.trees.path[s, :k].tolist() == path
            assert self.trees.emitted[s, :k].tolist() == emitted
            rows = list(range(c)) + [c + r for r in path]
            after.append([self.pages(p, s, c + n)[rows].clone() for l in self.layers for p in l])
            self.held[s] = c + k
            a += n
        return after

    def moved(self, after):
        for s, want in enumerate(after):
            got = [self.pages(p, s, want[0].shape[0]) for l in self.layers for p in l]
            assert all(torch.equal(x, y) for x, y in zip(got, want)), s


def _ends(n):
    out, a = [], 0
    for k in n:
        a += k
        out.append(a)
    return out


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("nodes,fp8,page", [(4, False, 16), (8, True, 1), (16, False, 64),
                                            (30, True, 16), (1, False, 16)])
def test_served_steps(cuda_device, nodes, fp8, page, drawn):
    server = _Server(cuda_device, 5, nodes, fp8, seed=nodes, page=page)
    server.drawn = drawn
    accepted = 0
    for _ in range(12):
        N = server.feed()
        for out in server.out:
            out.fill_(5.0)
        server.step()
        torch.cuda.synchronize()
        server.batch.raise_refused()
        after = server.check()
        assert all(bool((out[N:] == 5.0).all()) for out in server.out)
        server.move()
        torch.cuda.synchronize()
        server.batch.raise_refused()
        server.moved(after)
        accepted += int((server.trees.kept > 1).sum())
    assert accepted or nodes == 1


@pytest.mark.parametrize("drawn", [False, True])
def test_captured_steps_replay_with_other_trees(cuda_device, drawn):
    """One captured step with its move, replayed for every step, against the same
    steps launched one by one on buffers of their own."""
    a, b = (_Server(cuda_device, 4, 10, seed=3) for _ in range(2))
    a.drawn = b.drawn = drawn
    a.step(), a.move()  # an empty step: everything is loaded and warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(), a.move()
    for _ in range(8):
        N = a.feed()
        assert b.feed() == N
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        b.batch.raise_refused()
        after = b.check()
        b.move()
        torch.cuda.synchronize()
        a.batch.raise_refused()
        a.held = list(b.held)
        for x, y in ((a.trees.kept, b.trees.kept), (a.trees.path, b.trees.path),
                     (a.trees.emitted, b.trees.emitted), (a.target, b.target),
                     (a.batch.positions[:N], b.batch.positions[:N])):
            assert torch.equal(x, y)
        for x, y in zip(a.out, b.out):
            assert torch.equal(x[:N], y[:N])
        a.moved(after), b.moved(after)


def test_two_servers_on_two_streams(cuda_device):
    """Steps of two batches in flight at once, against the same steps alone."""
    together = [_Server(cuda_device, 3, 9, seed=s) for s in (1, 2)]
    alone = [_Server(cuda_device, 3, 9, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(6):
        for t in together + alone:
            t.feed()
        torch.cuda.synchronize()
        for t, stream in zip(together, streams):
            with torch.cuda.stream(stream):
                t.step(), t.move()
        torch.cuda.synchronize()
        for t, u in zip(together, alone):
            u.step()
            torch.cuda.synchronize()
            after = u.check()
            u.move()
            torch.cuda.synchronize()
            t.held = list(u.held)
            t.moved(after), u.moved(after)
            assert torch.equal(t.trees.emitted, u.trees.emitted)


def test_pools_past_four_gigabytes(cuda_device):
    """Trees on pages at the far end of pools of 3 * 2^30 elements."""
    from ecf8_amd.draft_kernels import DraftTrees, KeepPlan, draft_attention, draft_keep, draft_plan
    from ecf8_amd.paged_kernels import PagedBatch, paged_plan

    dev, page, pages, Hkv, c, n = cuda_device, 1024, 1024, 24, 100, 9
    for group in (1, 4, 8):
        b = PagedBatch(1, n, pages, page, 2048, Hkv * group, Hkv, dev)
        b.free.copy_(torch.arange(pages, dtype=torch.int32))  # the last page on top
        t = DraftTrees(b, n)
        gen = torch.Generator(device=dev).manual_seed(group)
        pools = [torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
        assert pools[0].numel() > 2 ** 31
        for p in pools:
            p[-1, :, : c + n] = torch.randn(Hkv, c + n, D, generator=gen, device=dev)
        tree = M.random_tree(random.Random(group), n, 2)
        paged_plan(b, _ints([c], dev), _ints([n], dev))
        draft_plan(t, _ints(tree, dev))
        q = torch.randn(n, Hkv * group, D, generator=gen, device=dev).bfloat16()
        out = torch.empty(n, Hkv * group, D, dtype=torch.bfloat16, device=dev)
        draft_attention(q, *pools, t, out)
        torch.cuda.synchronize()
        b.raise_refused()
        assert int(b.table[0, 0]) == pages - 1
        k, v = (p[-1, :, : c + n].transpose(0, 1).double() for p in pools)
        seen = torch.tensor([[True] * c + [bool(m >> j & 1) for j in range(n)]
                             for m in M.masks(tree)], device=dev)
        want, A = M.attention(q.double(), k, v, seen)
        bound = want.abs() * 2.0 ** -8 + A * 2.0 ** -10  # as in _Server.check
        if n * group > 64:
            bound += (want.abs() + A) * 2.0 ** -8
        assert bool(((out.double() - want).abs() <= bound).all())
        t.kept.fill_(2)
        t.path.copy_(_ints([[0, 7] + [-1] * (n - 2)], dev))
        draft_keep(KeepPlan(t, [tuple(pools)]))
        torch.cuda.synchronize()
        b.raise_refused()
        for p, x in zip(pools, (k, v)):
            assert torch.equal(p[-1, :, c + 1].double(), x[c + 7])
        del pools
