"""The operators of speculative decoding over a paged KV cache, as cases that
can be measured.  A drafter proposes a tree of tokens for each sequence, one
step runs the model on all of them, and the target's probabilities decide which
stay: the trees' masks and positions (``draft_plan``), the attention of their
rows over the pages (``draft_attention``), the target's probabilities
(``token_probabilities``), their verification from given random numbers
(``draft_verify``), and the cache's rows of what was accepted moved together
(``draft_keep``).

``run`` computes a case in elementary torch operations, or, where ``own`` is
set, through ``ecf8_amd.draft_kernels``.  ``exact`` restates the operators
whose outputs are computed numbers in 64 bits, row by row.

Heads, layers and the vocabulary are those of the configurations in
``ecf8_amd.llm`` (32 query / 8 KV heads of 128, 36 layers, 151936 tokens) and
``ecf8_amd.moe`` (32 / 4).
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
HQ, D = 32, 128


def listed() -> list[dict]:
    return [
        # The bookkeeping of a step of 16 sequences, four drafted tokens in a row each.
        {"name": "plan_chains", "kind": "plan", "seqs": 16, "nodes": 5, "kids": 1, "ragged": False,
         "cached": 2048, "page": 16},
        # The same of a full server: trees of up to 32 tokens, some sequences idle.
        {"name": "plan_trees", "kind": "plan", "seqs": 512, "nodes": 32, "kids": 8, "ragged": True,
         "cached": 1024, "page": 64},
        # One user, a small tree: latency.
        {"name": "attend_one", "kind": "attend", "seqs": 1, "nodes": 8, "kids": 3, "ragged": False,
         "cached": 640, "page": 64, "kv_heads": 8, "fp8": False},
        # A served batch, four drafted tokens in a row each.
        {"name": "attend_chains", "kind": "attend", "seqs": 64, "nodes": 5, "kids": 1,
         "ragged": False, "cached": 8192, "page": 16, "kv_heads": 8, "fp8": False},
        # Trees of up to 26 tokens, some sequences idle.
        {"name": "attend_trees", "kind": "attend", "seqs": 24, "nodes": 26, "kids": 4,
         "ragged": True, "cached": 6000, "page": 16, "kv_heads": 8, "fp8": False},
        # Full trees after long contexts in an FP8 cache.
        {"name": "attend_long_fp8", "kind": "attend", "seqs": 8, "nodes": 64, "kids": 8,
         "ragged": False, "cached": 32_768, "page": 128, "kv_heads": 4, "fp8": True},
        # One user's step: five rows at one temperature.
        {"name": "probabilities_few", "kind": "probabilities", "rows": 5, "vocab": 151_936,
         "greedy": False},
        # A served batch's step: rows of different temperatures, greedy ones among them.
        {"name": "probabilities_many", "kind": "probabilities", "rows": 416, "vocab": 151_936,
         "greedy": True},
        # Drafts that a drafter took as its most probable tokens: trees of 26.
        {"name": "verify_top", "kind": "verify", "seqs": 16, "nodes": 26, "kids": 4,
         "ragged": False, "vocab": 151_936, "drawn": False},
        # Drafts drawn from the drafter's probabilities, up to two a token.
        {"name": "verify_drawn", "kind": "verify", "seqs": 64, "nodes": 8, "kids": 2,
         "ragged": False, "vocab": 151_936, "drawn": True},
        # One user's accepted path, in the caches of all layers.
        {"name": "keep_one", "kind": "keep", "seqs": 1, "nodes": 8, "kids": 3, "ragged": False,
         "cached": 500, "page": 64, "kv_heads": 8, "fp8": False, "layers": 36},
        # A served batch's.
        {"name": "keep_batch", "kind": "keep", "seqs": 64, "nodes": 26, "kids": 4, "ragged": False,
         "cached": 120, "page": 16, "kv_heads": 8, "fp8": False, "layers": 36},
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["plan", "attend", "attend", "attend", "probabilities", "verify", "verify",
                       "keep"])
    if kind == "probabilities":
        return {"kind": kind, "rows": _log(rng, 1, 400), "vocab": _log(rng, 1000, 152_064),
                "greedy": rng.random() < 0.5}
    case = {"kind": kind, "seqs": _log(rng, 1, 512 if kind == "plan" else 64),
            "nodes": _log(rng, 1, 32 if kind == "plan" else 64), "kids": rng.choice([1, 2, 3, 4, 8]),
            "ragged": rng.random() < 0.4}
    S, T = case["seqs"], case["nodes"]
    page = rng.choice([1, 8, 16, 16, 32, 64, 128, 256])
    if kind == "plan":
        return {**case, "cached": _log(rng, 1, 4096), "page": max(page, 8)}
    if kind == "verify":
        drawn = rng.random() < 0.5
        if drawn:
            case["kids"] = min(case["kids"], 3)
            T = case["nodes"] = min(T, 24)
        S = case["seqs"] = max(1, min(S, 400 // T))
        return {**case, "vocab": _log(rng, 1000, 152_064), "drawn": drawn}
    heads = {"page": page, "kv_heads": rng.choice([1, 2, 4, 8, 8, 16, 32]),
             "fp8": rng.random() < 0.4}
    if kind == "keep":
        S = case["seqs"] = min(S, max(1, 1600 // T))
        layers = max(1, min(_log(rng, 1, 48), 72_000 // (S * (T + 100) * heads["kv_heads"] // 8 + 1)))
        return {**case, "cached": _log(rng, 1, 100), "layers": layers, **heads}
    most = min(131_072, 200_000 // S, 16_000_000 // (S * T))
    return {**case, "cached": _log(rng, 1, max(1, most)), **heads}


# ------------------------------------------------------------------ inputs


def _sizes(case, seed):
    """(tokens in the cache, rows of the tree) of each sequence, which a scheduler
    knows on the host: the case's, in the seed's order."""
    S, most, nodes = case["seqs"], case.get("cached", 0), case["nodes"]
    rng = random.Random(1000 * S + nodes)
    cached = [int(rng.random() * most) for _ in range(S)]
    cached[0] = most
    new = [nodes] * S
    if case["ragged"]:
        new = [rng.randint(1, nodes) for _ in range(S)]
        if case["kind"] != "keep":
            new = [0 if i % 5 == 2 else n for i, n in enumerate(new)]
        new[0] = nodes
    order = list(range(S))
    random.Random(int(seed)).shuffle(order)
    return [cached[i] for i in order], [new[i] for i in order]


def _trees(case, seed, new):
    """Each sequence's parents: row 0 is the last accepted token, the others are
    drafted after an earlier row, at most ``kids`` after one."""
    rng = random.Random(int(seed) * 7919 + 1)
    trees = []
    for n in new:
        parents, count = [-1] * min(n, 1), [0] * n
        for i in range(1, n):
            p = rng.randrange(i)
            if count[p] >= case["kids"]:
                p = i - 1
            count[p] += 1
            parents.append(p)
        trees.append(parents)
    return trees


def _flat(lists):
    return [x for one in lists for x in one]


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).to(DEV)


def _normal(*shape, gen, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _step(case, seed, gen):
    """A step's sequences, their trees, and block tables over shuffled pages."""
    cached, new = _sizes(case, seed)
    trees = _trees(case, seed, new)
    S, page, kv = case["seqs"], case.get("page", 64), case.get("kv_heads", 8)
    held = [-(-(c + n) // page) for c, n in zip(cached, new)]
    width, total = max(1, max(held)), sum(held)
    pages = total + total // 8 + 1
    perm = torch.randperm(pages, generator=gen, device=DEV).int()
    n = _ints(held)
    at = torch.arange(width, device=DEV)[None] + (torch.cumsum(n, 0) - n)[:, None]
    table = torch.where(torch.arange(width, device=DEV)[None] < n[:, None],
                        perm[at.clamp(max=pages - 1)], -1).int().contiguous()
    s = SimpleNamespace(kind=case["kind"], cached_h=cached, new_h=new, trees_h=trees, seqs=S,
                        nodes=case["nodes"], rows=sum(new), page=page, pages=pages, width=width,
                        cached=_ints(cached), new=_ints(new), table=table,
                        starts=_ints([0] + torch.tensor(new).cumsum(0).tolist()),
                        parents=_ints(_flat(trees)),
                        seq=_ints(_flat([i] * k for i, k in enumerate(new)), torch.int64))
    if own:  # the handles of the step's bookkeeping
        from ecf8_amd.draft_kernels import DraftTrees, draft_plan
        from ecf8_amd.paged_kernels import PagedBatch, paged_plan

        s.batch = PagedBatch(S, s.rows, pages, page, width * page, HQ, kv, DEV)
        s.batch.table.copy_(table)
        s.batch.owned.copy_(n)
        s.batch.free[: pages - total].copy_(perm[total:])
        s.batch.n_free.fill_(pages - total)
        paged_plan(s.batch, s.cached, s.new)
        s.trees = DraftTrees(s.batch, case["nodes"], max_children=case["kids"])
        if case["kind"] != "plan":
            draft_plan(s.trees, s.parents)
    return s


def prepare(case: dict, seed: int):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    kind = case["kind"]
    if kind == "probabilities":
        N, V = case["rows"], case["vocab"]
        # runs of rows (a sequence's) share a temperature; a greedy one's is zero
        t = 0.4 + 0.9 * torch.rand(N // 8 + 1, generator=gen, device=DEV)
        if case["greedy"]:
            t[::3] = 0.0
        t = t.repeat_interleave(8)[:N] if case["greedy"] else t[:1].expand(N)
        return SimpleNamespace(kind=kind, logits=_normal(N, V, gen=gen, scale=3.0),
                               temperature=t.contiguous(),
                               out=torch.empty(N, V, device=DEV))
    s = _step(case, seed, gen)
    if kind == "plan":
        return s
    if kind == "verify":
        N, V = s.rows, case["vocab"]
        # few tokens have most of the probability, and the drafter's are near them
        logits = _normal(N, V, gen=gen, scale=6.0, dtype=torch.float32)
        guess = 0.95 * logits + _normal(N, V, gen=gen, scale=0.8, dtype=torch.float32)
        s.target = torch.softmax(logits, -1)
        s.draft = torch.softmax(guess, -1)
        del logits
        kids, rank = case["kids"], []
        for parents in s.trees_h:
            rank += [parents[:i].count(p) for i, p in enumerate(parents)]
        first = s.starts[s.seq]
        above = (first + s.parents.clamp(min=0)).long()
        if case["drawn"]:
            picks = torch.multinomial(s.draft, kids, replacement=True, generator=gen)
        else:
            picks = torch.topk(guess, kids, -1).indices
            s.draft = None
        root = torch.randint(V, (N,), generator=gen, device=DEV)
        s.tokens = torch.where(s.parents < 0, root, picks[above, _ints(rank, torch.int64)])
        s.accept = torch.rand(N, generator=gen, device=DEV)
        s.sample = torch.rand(s.seqs, generator=gen, device=DEV)
        return s
    Hkv = case["kv_heads"]

    def pools(n):
        x = torch.randn(n, s.pages, Hkv, s.page, D, generator=gen, device=DEV, dtype=torch.bfloat16)
        return (x * 16).to(torch.float8_e4m3fn) if case["fp8"] else x

    if kind == "keep":
        s.pools = pools(2 * case["layers"])
        s.layers = list(zip(s.pools[::2], s.pools[1::2]))
        paths = []
        rng = random.Random(int(seed) + 17)
        for parents in s.trees_h:
            at, path = rng.randrange(len(parents)), []
            while at >= 0:
                path.append(at)
                at = parents[at]
            paths.append(path[::-1])
        s.kept = _ints([len(p) for p in paths])
        s.path = _ints([p + [-1] * (s.nodes - len(p)) for p in paths])
        if own:  # as draft_verify leaves them
            from ecf8_amd.draft_kernels import KeepPlan

            s.trees.kept.copy_(s.kept)
            s.trees.path.copy_(s.path)
            s.keep = KeepPlan(s.trees, s.layers)
        return s
    s.kp, s.vp = pools(2)
    s.ks = s.vs = None
    if case["fp8"]:
        s.ks, s.vs = (0.05 + 0.03 * torch.rand(Hkv, generator=gen, device=DEV) for _ in range(2))
    s.q = _normal(s.rows, HQ, D, gen=gen, scale=1.5)
    s.out = torch.empty(s.rows, HQ * D, dtype=torch.bfloat16, device=DEV)
    return s


# ------------------------------------------------------------- plain forms


def _padded(x, s):
    """Packed rows [N, ...] -> [S, T, ...], and which of them are rows."""
    t = torch.arange(s.nodes, device=DEV)
    at = s.starts[:-1, None] + t
    return x[at.clamp(max=x.shape[0] - 1).long()], t[None] < s.new[:, None]


def _ancestors(s):
    """[S, T] int64: bit j of row i is set where i is j or after it."""
    up, live = _padded(s.parents, s)
    up = torch.where(live, up, -1).long()
    bits = (torch.ones_like(up) << torch.arange(s.nodes, device=DEV)).expand(up.shape)
    for _ in range(6):  # 64 rows
        over = up.clamp(min=0)
        bits = torch.where(up >= 0, bits | bits.gather(1, over), bits)
        up = torch.where(up >= 0, up.gather(1, over), -1)
    return bits


def _packed(x, s):
    return x[s.seq, torch.arange(s.rows, device=DEV) - s.starts[s.seq]]


def _plain_plan(s):
    bits = _packed(_ancestors(s), s)
    depth = ((bits[:, None] >> torch.arange(64, device=DEV)) & 1).sum(1) - 1
    return {"masks": bits, "positions": (s.cached[s.seq] + depth).int()}


def _plain_attend(s):
    S, T, L, Hkv = s.seqs, s.nodes, s.width * s.page, s.kp.shape[1]
    G = HQ // Hkv
    at = s.table.clamp(min=0).long()

    def read(pool, scale):
        x = pool.view(torch.uint8)[at].view(pool.dtype) if scale is not None else pool[at]
        x = x.float().permute(0, 2, 1, 3, 4).reshape(S, Hkv, L, D)
        if scale is not None:
            x = x * scale[:, None, None]
        # positions past a sequence's end hold other tokens' values
        return x.masked_fill(torch.arange(L, device=DEV)[:, None]
                             >= (s.cached + s.new)[:, None, None, None], 0.0)

    q, _ = _padded(s.q.float(), s)
    q = q.view(S, T, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * T, D)
    score = torch.matmul(q, read(s.kp, s.ks).transpose(-1, -2)).view(S, Hkv, G, T, L)
    score *= 1 / math.sqrt(D)
    pos = torch.arange(L, device=DEV)
    off = (pos[None] - s.cached[:, None]).clamp(max=64)  # of the tree's rows
    seen = (_ancestors(s)[:, :, None] >> off.clamp(0, 63)[:, None]) & 1
    seen = (off < 0)[:, None] | ((off < 64)[:, None] & (seen == 1))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    o = torch.matmul(p.view(S, Hkv, G * T, L), read(s.vp, s.vs))
    o = o / p.sum(-1).view(S, Hkv, G * T, 1)
    o = o.view(S, Hkv, G, T, D).permute(0, 3, 1, 2, 4).reshape(S, T, HQ * D)
    s.out.copy_(_packed(o, s))
    return s.out


def _plain_probabilities(s):
    x = s.logits.float()
    top = x.amax(-1, keepdim=True)
    t = s.temperature[:, None]
    e = ((x - top) / torch.where(t > 0, t, 1.0)).exp()
    at = torch.arange(x.shape[1], device=DEV)
    first = torch.where(x == top, at, x.shape[1]).amin(-1, keepdim=True)
    s.out.copy_(torch.where(t > 0, e / e.sum(-1, keepdim=True), (at == first).float()))
    return s.out


def _plain_verify(s):
    """Row by row, all sequences at once; 64 bits, since a draft next to its border
    must fall on the same side."""
    S, T = s.seqs, s.nodes
    every = torch.arange(S, device=DEV)
    up, live = _padded(s.parents, s)
    token, _ = _padded(s.tokens, s)
    u, _ = _padded(s.accept, s)
    first = s.starts[:-1].long().clamp(max=s.rows - 1)
    here = torch.zeros(S, dtype=torch.int64, device=DEV)  # the last accepted row
    w = s.target[first].double()  # what the next token's probability is in proportion to
    mass = torch.ones(S, dtype=torch.float64, device=DEV)
    path = torch.full((S, T), -1, dtype=torch.int64, device=DEV)
    emitted = torch.full((S, T), -1, dtype=torch.int64, device=DEV)
    any_row = s.new > 0
    path[:, 0] = torch.where(any_row, 0, -1)
    kept = any_row.long()
    for j in range(1, T):
        tried = live[:, j] & (up[:, j] == here)
        c = token[:, j]
        wc = w[every, c]
        limit = u[:, j].double() * mass
        if s.draft is not None:
            q = s.draft[first + here].double()
            limit = limit * q[every, c]
        yes = tried & (limit < wc)
        no = tried & ~yes
        if s.draft is not None:
            less = (w / mass[:, None] - q).clamp(min=0)
            w = torch.where(no[:, None], less, w)
            mass = torch.where(no, less.sum(-1), mass)
        else:
            w[every, c] = torch.where(no, 0.0, wc)
            mass = torch.where(no, mass - wc, mass)
        slot = kept.clamp(max=T - 1)
        path[every, slot] = torch.where(yes, j, path[every, slot])
        emitted[every, slot - 1] = torch.where(yes, c, emitted[every, slot - 1])
        kept += yes
        here = torch.where(yes, j, here)
        w = torch.where(yes[:, None], s.target[(first + here).clamp(max=s.rows - 1)].double(), w)
        mass = torch.where(yes, 1.0, mass)
    # nothing left: the target's own probabilities
    whole = s.target[(first + here).clamp(max=s.rows - 1)].double()
    w = torch.where((w.sum(-1) > 0)[:, None], w, whole)
    upto = torch.cumsum(w, -1)
    over = upto > s.sample.double()[:, None] * w.sum(-1)[:, None]
    at = torch.arange(w.shape[1], device=DEV)
    token = torch.where(over, at, w.shape[1]).amin(-1)
    token = torch.where(any_row, token, -1)
    last = (kept - 1).clamp(min=0)
    emitted[every, last] = torch.where(any_row, token, emitted[every, last])
    return {"kept": kept.int(), "path": path.int(), "emitted": emitted, "next": token}


def _plain_keep(s):
    t = torch.arange(s.nodes, device=DEV)
    live = t[None] < s.kept[:, None]

    def place(row):
        pos = s.cached[:, None] + torch.where(live, row, 0)
        return s.table.gather(1, (pos // s.page).long()).long(), (pos % s.page).long()

    (a, b), (c, d) = place(s.path), place(t[None])
    for layer in s.layers:
        for pool in layer:
            x = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
            x[c, :, d] = x[a, :, b]
    return s.pools


def run(state):
    s = state
    if not own:
        return {"plan": _plain_plan, "attend": _plain_attend, "verify": _plain_verify,
                "probabilities": _plain_probabilities, "keep": _plain_keep}[s.kind](s)
    from ecf8_amd import draft_kernels as K

    if s.kind == "plan":
        K.draft_plan(s.trees, s.parents)
        return {"masks": s.trees.masks, "positions": s.batch.positions}
    if s.kind == "attend":
        return K.draft_attention(s.q, s.kp, s.vp, s.trees, s.out, k_scale=s.ks, v_scale=s.vs)
    if s.kind == "probabilities":
        return K.token_probabilities(s.logits, s.temperature, s.out)
    if s.kind == "verify":
        t = s.trees
        K.draft_verify(t, s.tokens, s.target, s.accept, s.sample, draft=s.draft)
        return {"kept": t.kept, "path": t.path, "emitted": t.emitted, "next": t.next_token}
    K.draft_keep(s.keep)
    return s.pools


# ------------------------------------------------------------ work, 64 bits


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "probabilities":
        n = case["rows"] * case["vocab"]
        return {"bytes": 6 * n, "flops": 5 * n}
    cached, new = _sizes(case, 1)
    S, N = case["seqs"], sum(new)
    if kind == "plan":
        return {"bytes": 8 * S + N * (4 + 8 + 4), "flops": 0}  # lengths, parents; masks, positions
    if kind == "verify":
        # the last row's probabilities, and the drafter's for it; a few of the others
        each = 2 if case["drawn"] else 1
        live = sum(n > 0 for n in new)
        return {"bytes": live * 4 * case["vocab"] * each + N * (8 + 4 + 4 + 4 * each),
                "flops": 3 * live * case["vocab"] * each}
    size = 1 if case["fp8"] else 2
    if kind == "keep":
        # half of a path's rows move, at a guess: they are read and written
        moved = sum(max(0.0, math.log2(n)) / 2 for n in new if n)
        return {"bytes": int(moved * case["layers"] * 2 * 2 * case["kv_heads"] * D * size),
                "flops": 0}
    pairs = 0
    for c, parents in zip(cached, _trees(case, 1, new)):
        depth = []
        for p in parents:
            depth.append(1 if p < 0 else depth[p] + 1)
        pairs += c * len(parents) + sum(depth)
    keys = sum(c + n for c, n in zip(cached, new) if n)
    return {"bytes": 2 * size * keys * case["kv_heads"] * D + 2 * 2 * N * HQ * D,
            "flops": 4 * D * HQ * pairs}


def exact(case: dict, seed: int):
    if case["kind"] not in ("attend", "probabilities"):
        return None  # whole numbers, and values moved
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "probabilities":
        out = torch.zeros(s.out.shape, dtype=torch.float64, device=DEV)
        for i, t in enumerate(s.temperature.tolist()):
            x = s.logits[i].double()
            if t > 0:
                e = torch.exp((x - x.max()) / t)
                out[i] = e / e.sum()
            else:
                out[i, int((x == x.max()).nonzero()[0])] = 1.0
        return out
    out = torch.empty(s.rows, HQ, D, dtype=torch.float64, device=DEV)
    a, G = 0, HQ // case["kv_heads"]
    for i, (c, n) in enumerate(zip(s.cached_h, s.new_h)):
        if not n:
            continue
        p = torch.arange(c + n, device=DEV)
        page, off = s.table[i, p // s.page].long(), p % s.page
        seen = torch.zeros(n, c + n, dtype=torch.bool)
        seen[:, :c] = True
        for t, up in enumerate(s.trees_h[i]):
            if up >= 0:
                seen[t] = seen[up]
            seen[t, c + t] = True
        hidden = ~seen.to(DEV)
        for h in range(case["kv_heads"]):
            if s.ks is not None:
                k, v = (x.float()[page, h, off].double() * sc[h].double()
                        for x, sc in ((s.kp, s.ks), (s.vp, s.vs)))
            else:
                k, v = (x[page, h, off].double() for x in (s.kp, s.vp))
            for g in range(h * G, (h + 1) * G):
                e = s.q[a: a + n, g].double() @ k.T / math.sqrt(D)
                e[hidden] = -math.inf
                out[a: a + n, g] = torch.softmax(e, -1) @ v
        a += n
    return out.flatten(1)
