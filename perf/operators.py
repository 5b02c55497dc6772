"""The operators of a ragged batch over a paged KV cache, as cases that can
be measured: a step's block tables and slot maps (``paged_plan``), the head
norms, rotary embedding and cache write of its rows (``paged_qk_norm_rope``),
their attention over the pages (``paged_attention``), and the causal
attention of whole packed prompts without a cache (``ragged_attention``).

``run`` computes a case in elementary torch operations in fp32, or, where
``own`` is set, through ``ecf8_amd.paged_kernels``.  ``exact`` restates the
operators in 64 bits, one sequence after the other.

Heads are those of the configurations in ``ecf8_amd.llm`` (32 query / 8 KV
heads of 128) and ``ecf8_amd.moe`` (32 / 4).
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
D = 128
EPS = 1e-6
THETA = 1_000_000.0
FP8_MAX = 448.0


def listed() -> list[dict]:
    return [
        # The bookkeeping of every decode step of a server: 64 running
        # sequences get one token each.
        {"name": "plan_step", "kind": "plan", "seqs": 64, "rows": 64, "cached": 8192, "page": 16,
         "admit": False},
        # A full batch replaced: 512 finished sequences give their pages back,
        # 512 prompts take their places.
        {"name": "plan_admit", "kind": "plan", "seqs": 512, "rows": 32768, "cached": 0, "page": 64,
         "admit": True},
        # The cache write of a decode step of 16 sequences.
        {"name": "write_step", "kind": "write", "seqs": 16, "rows": 16, "cached": 2048, "page": 16,
         "kv_heads": 8, "fp8": False},
        # The cache write of one prefill chunk of many prompts.
        {"name": "write_prompt", "kind": "write", "seqs": 24, "rows": 8192, "cached": 0,
         "page": 64, "kv_heads": 8, "fp8": False},
        # The same into an FP8 cache, an odd number of rows at odd positions.
        {"name": "write_prompt_fp8", "kind": "write", "seqs": 7, "rows": 4099, "cached": 777,
         "page": 128, "kv_heads": 4, "fp8": True},
        # One user's next token: latency.
        {"name": "attend_one", "kind": "attend", "seqs": 1, "new": 1, "cached": 640, "page": 64,
         "kv_heads": 8, "fp8": False, "mixed": False, "idle": False},
        # A decode step of a served batch: 64 contexts of up to 8192 tokens.
        {"name": "attend_batch", "kind": "attend", "seqs": 64, "new": 1, "cached": 8192,
         "page": 16, "kv_heads": 8, "fp8": False, "mixed": False, "idle": False},
        # A decode step over few, very long contexts in an FP8 cache.
        {"name": "attend_long_fp8", "kind": "attend", "seqs": 6, "new": 1, "cached": 100_003,
         "page": 128, "kv_heads": 4, "fp8": True, "mixed": False, "idle": False},
        # Chunked prefill: a 1024-token chunk of one long prompt beside the
        # decode steps of 8 other sequences.
        {"name": "attend_chunk", "kind": "attend", "seqs": 9, "new": 1024, "cached": 8192,
         "page": 16, "kv_heads": 8, "fp8": False, "mixed": True, "idle": False},
        # A few short prompts: latency.
        {"name": "prompt_short", "kind": "prompt", "seqs": 5, "rows": 301, "kv_heads": 8},
        # A prefill batch of prompts of different lengths.
        {"name": "prompt_packed", "kind": "prompt", "seqs": 24, "rows": 8192, "kv_heads": 8},
        # One long prompt.
        {"name": "prompt_long", "kind": "prompt", "seqs": 1, "rows": 8192, "kv_heads": 8},
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["plan", "write", "write", "attend", "attend", "attend", "prompt", "prompt"])
    page = rng.choice([1, 8, 16, 16, 32, 64, 128, 256])
    heads = {"kv_heads": rng.choice([1, 2, 4, 8, 8, 16, 32])}
    if kind == "plan":
        seqs = _log(rng, 1, 1024)
        if rng.random() < 0.5:
            return {"kind": kind, "seqs": seqs, "rows": seqs, "cached": _log(rng, 16, 8192),
                    "page": max(page, 8), "admit": False}
        return {"kind": kind, "seqs": seqs, "rows": _log(rng, seqs, 32768), "cached": 0,
                "page": max(page, 8), "admit": True}
    if kind == "write":
        seqs = _log(rng, 1, 64)
        return {"kind": kind, "seqs": seqs, "rows": _log(rng, seqs, 8192),
                "cached": _log(rng, 1, 8192), "page": page, **heads, "fp8": rng.random() < 0.5}
    if kind == "prompt":
        rows = _log(rng, 1, 8192)
        return {"kind": kind, "seqs": min(rows, _log(rng, 1, 64)), "rows": rows, **heads}
    seqs = _log(rng, 1, 128)
    new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 1024)])
    cached = _log(rng, 1, min(131072, 300_000 // seqs))
    new = max(1, min(new, 64_000_000 // (seqs * (cached + 1024))))
    return {"kind": kind, "seqs": seqs, "new": new, "cached": cached, "page": page, **heads,
            "fp8": rng.random() < 0.4, "mixed": rng.random() < 0.3, "idle": rng.random() < 0.3}


# ------------------------------------------------------------------ inputs


def _split(total: int, parts: int, gen) -> list[int]:
    """``total`` tokens over ``parts`` sequences of different lengths."""
    w = -torch.log(torch.rand(parts, generator=gen, dtype=torch.float64).clamp_min(1e-9)) + 0.05
    cut = (torch.cumsum(w, 0) / w.sum() * total).round().long()
    cut[-1] = total
    return torch.diff(cut, prepend=cut.new_zeros(1)).tolist()


def _lengths(case, seed):
    """(tokens in the cache, new tokens) of each sequence, which a scheduler
    knows on the host: the case's, in the seed's order."""
    g = torch.Generator().manual_seed(case["seqs"])
    S, most = case["seqs"], case.get("cached", 0)
    cached = (torch.rand(S, generator=g) * most).long().tolist()
    cached[0] = most
    if case["kind"] == "attend":
        new = [case["new"]] + [1 if case["mixed"] else case["new"]] * (S - 1)
        if case["idle"]:
            new = [n if i % 3 != 1 else 0 for i, n in enumerate(new)]
    elif case["kind"] == "plan" and not case["admit"]:
        new = [1] * S
    else:
        new = _split(case["rows"], S, g)
    order = torch.randperm(S, generator=torch.Generator().manual_seed(int(seed))).tolist()
    return [cached[i] for i in order], [new[i] for i in order]


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).to(DEV)


def _normal(*shape, gen, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _pool(pages, kv_heads, page, fp8, gen):
    x = torch.randn(pages, kv_heads, page, D, generator=gen, device=DEV, dtype=torch.bfloat16)
    return (x * 16).to(torch.float8_e4m3fn) if fp8 else x


def _paged(case, seed, gen):
    """Block tables over shuffled pages, and the step's row maps."""
    cached, new = _lengths(case, seed)
    S, page = case["seqs"], case["page"]
    held = [-(-(c + n) // page) for c, n in zip(cached, new)]
    width, total = max(held), sum(held)
    pages = total + total // 8 + 1
    perm = torch.randperm(pages, generator=gen, device=DEV).int()
    n = _ints(held)
    at = torch.arange(width, device=DEV)[None] + (torch.cumsum(n, 0) - n)[:, None]
    table = torch.where(torch.arange(width, device=DEV)[None] < n[:, None],
                        perm[at.clamp(max=pages - 1)], -1).int().contiguous()
    s = SimpleNamespace(cached_h=cached, new_h=new, cached=_ints(cached), new=_ints(new),
                        table=table, owned=n, pages=pages, page=page, width=width, seqs=S,
                        rows=sum(new), lengths=_ints([c + k for c, k in zip(cached, new)]),
                        starts=_ints([0] + torch.tensor(new).cumsum(0).tolist()))
    seq = [i for i, k in enumerate(new) for _ in range(k)]
    s.seq = _ints(seq, torch.int64)
    s.positions = s.cached[s.seq] + (torch.arange(s.rows, device=DEV) - s.starts[s.seq])
    s.slots = s.table[s.seq, s.positions // page].long() * page + s.positions % page
    if own:  # the handle of the step's bookkeeping, planned as for every layer's call
        from ecf8_amd.paged_kernels import PagedBatch, paged_plan

        s.batch = PagedBatch(S, max(1, s.rows), pages, page, width * page, 32, case["kv_heads"],
                             DEV)
        s.batch.table.copy_(table)
        s.batch.owned.copy_(n)
        s.batch.free[: pages - total].copy_(perm[total:])
        s.batch.n_free.fill_(pages - total)
        paged_plan(s.batch, s.cached, s.new)
    return s


def _rotary(length, device=DEV):
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=device) / D)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case: dict, seed: int):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    kind, Hkv = case["kind"], case.get("kv_heads", 8)
    if kind == "plan":
        cached, new = _lengths(case, seed)
        S, page = case["seqs"], case["page"]
        held = [-(-c // page) if not case["admit"] else (7 * i) % 40 for i, c in enumerate(cached)]
        width = max(max(-(-(c + n) // page) for c, n in zip(cached, new)), max(held))
        pages = sum(held) + sum(-(-(c + n) // page) for c, n in zip(cached, new)) + 5
        perm = torch.randperm(pages, generator=gen, device=DEV).int()
        table = torch.full((S, width), -1, dtype=torch.int32)
        at, host = 0, perm.cpu()
        for i, h in enumerate(held):
            table[i, :h] = host[at: at + h]
            at += h
        s = SimpleNamespace(cached=_ints(cached), new=_ints(new),
                            release=_ints([1] * S) if case["admit"] else None)
        state = dict(table=table.to(DEV), owned=_ints(held), free=torch.roll(perm, -at).contiguous(),
                     n_free=_ints([pages - at]))
        if own:
            from ecf8_amd.paged_kernels import PagedBatch

            s.batch = PagedBatch(S, sum(new), pages, page, width * page, 32, 8, DEV)
            for k, v in state.items():
                getattr(s.batch, k).copy_(v)
        else:
            s.batch = SimpleNamespace(page=page, max_rows=sum(new), **state)
        return s
    if kind == "prompt":
        _, new = _lengths(case, seed)
        N = sum(new)
        s = SimpleNamespace(rows=N, seqs=len(new), new_h=new, longest=max(new),
                            starts=_ints([0] + torch.tensor(new).cumsum(0).tolist()),
                            seq=_ints([i for i, k in enumerate(new) for _ in range(k)],
                                      torch.int64))
        # views of a fused projection's output
        qkv = _normal(N, 32 + 2 * Hkv, D, gen=gen)
        s.q, s.k, s.v = qkv[:, :32], qkv[:, 32: 32 + Hkv], qkv[:, 32 + Hkv:]
        s.out = torch.empty(N, 32 * D, dtype=torch.bfloat16, device=DEV)
        return s
    s = _paged(case, seed, gen)
    s.kp, s.vp = (_pool(s.pages, Hkv, s.page, case["fp8"], gen) for _ in range(2))
    s.ks = s.vs = None
    if case["fp8"]:
        s.ks, s.vs = (0.05 + 0.03 * torch.rand(Hkv, generator=gen, device=DEV) for _ in range(2))
    if kind == "write":
        s.qkv = _normal(s.rows, (32 + 2 * Hkv) * D, gen=gen, scale=2.0)
        s.qn, s.kn = (1 + _normal(D, gen=gen, scale=0.2) for _ in range(2))
        s.cos, s.sin = _rotary(s.width * s.page)
        s.q_out = torch.zeros(s.rows, 32, D, dtype=torch.bfloat16, device=DEV)
    else:
        s.q = _normal(s.rows, 32, D, gen=gen, scale=1.5)
        s.out = torch.empty(s.rows, 32 * D, dtype=torch.bfloat16, device=DEV)
        s.most_new = max(s.new_h)
    return s


# ------------------------------------------------------------- plain forms


def _plain_plan(s):
    b = s.batch
    S, W = b.table.shape
    page, pages = b.page, b.free.numel()
    col = torch.arange(W, device=DEV)[None]
    kv = s.cached + s.new
    back = torch.zeros_like(col.expand(S, W), dtype=torch.bool)
    owned = b.owned
    if s.release is not None:
        back = (s.release != 0)[:, None] & (col < owned[:, None])
        owned = torch.where(s.release != 0, 0, owned)
    extra = ((kv + page - 1) // page - owned).clamp(min=0)
    take = torch.cumsum(extra, 0)
    n_back = back.sum()
    ok = ((s.cached >= 0).all() & (s.new >= 0).all() & (kv <= W * page).all()
          & (s.new.sum() <= b.max_rows) & (take[-1] <= b.n_free[0] + n_back))
    # returned pages go on the stack in the table's order, new ones come off it
    spot = torch.where(back, b.n_free + torch.cumsum(back.flatten(), 0).view(S, W) - 1, pages)
    free = torch.cat([b.free, b.free.new_zeros(1)]).scatter(0, spot.flatten(), b.table.flatten())
    table = torch.where(back, -1, b.table)
    top = b.n_free + n_back
    fresh = (col >= owned[:, None]) & (col < (owned + extra)[:, None])
    nth = (take - extra)[:, None] + col - owned[:, None]
    page_of = free[(top - 1 - nth).clamp(0, pages)]
    table = torch.where(fresh, page_of, table).int()
    ends = torch.cumsum(s.new, 0)
    starts = torch.cat([ends.new_zeros(1), ends])
    row = torch.arange(b.max_rows, device=DEV)
    seq = torch.searchsorted(ends, row, right=True).clamp(max=S - 1)
    live = (row < ends[-1]) & ok
    pos = s.cached[seq] + row - starts[seq]
    slot = table[seq, (pos // page).clamp(0, W - 1)].long() * page + pos % page
    b.table.copy_(torch.where(ok, table, b.table))
    b.free.copy_(torch.where(ok, free[:pages], b.free))
    b.n_free.copy_(torch.where(ok, top - take[-1], b.n_free))
    b.owned.copy_(torch.where(ok, owned + extra, b.owned))
    return {"table": b.table, "owned": b.owned, "free": b.free, "n_free": b.n_free,
            "starts": torch.where(ok, starts, 0).int(), "lengths": torch.where(ok, kv, 0).int(),
            "slots": torch.where(live, slot, -1).int(),
            "positions": torch.where(live, pos, -1).int()}


def _norm_rope(x, w, cos, sin):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    a, b = x[..., : D // 2], x[..., D // 2:]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_write(s):
    Hkv = s.kp.shape[1]
    x = s.qkv.float().view(s.rows, 32 + 2 * Hkv, D)
    cos, sin = s.cos[s.positions], s.sin[s.positions]
    q = _norm_rope(x[:, :32], s.qn, cos, sin)
    k = _norm_rope(x[:, 32: 32 + Hkv], s.kn, cos, sin)
    v = x[:, 32 + Hkv:]
    s.q_out.copy_(q)
    page, off = s.slots // s.page, s.slots % s.page
    for pool, y, scale in ((s.kp, k, s.ks), (s.vp, v, s.vs)):
        if scale is None:
            pool[page, :, off] = y.to(pool.dtype)
        else:
            code = (y / scale[:, None]).clamp(-FP8_MAX, FP8_MAX).to(pool.dtype)
            pool.view(torch.uint8)[page, :, off] = code.view(torch.uint8)
    return {"q": s.q_out, "k": s.kp, "v": s.vp}


def _plain_attention(q, k, v, limit):
    """q [S, T, Hq, D], k / v [S, Hkv, L, D], limit [S, T]: query t of
    sequence s reads keys below limit; fp32 [S, T, Hq, D]."""
    S, T, Hq, _ = q.shape
    Hkv, L = k.shape[1:3]
    G = Hq // Hkv
    q = q.float().view(S, T, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * T, D)
    score = torch.matmul(q, k.float().transpose(-1, -2)).view(S, Hkv, G, T, L)
    score *= 1 / math.sqrt(D)
    hidden = torch.arange(L, device=DEV) >= limit[..., None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    o = torch.matmul(p.view(S, Hkv, G * T, L), v.float()) / p.sum(-1).view(S, Hkv, G * T, 1)
    return o.view(S, Hkv, G, T, D).permute(0, 3, 1, 2, 4).reshape(S, T, Hq, D)


def _padded(x, starts, T):
    """Packed rows [N, ...] -> [S, T, ...], sequences from their first row."""
    at = starts[:-1, None] + torch.arange(T, device=DEV)
    return x[at.clamp(max=x.shape[0] - 1)]


def _plain_attend(s):
    Hkv, T, L = s.kp.shape[1], s.most_new, s.width * s.page
    at = s.table.clamp(min=0).long()

    def read(pool, scale):
        x = pool.view(torch.uint8)[at].view(pool.dtype) if scale is not None else pool[at]
        x = x.float().permute(0, 2, 1, 3, 4).reshape(s.seqs, Hkv, L, D)
        if scale is not None:
            x = x * scale[:, None, None]
        # positions past a sequence's end hold other tokens' values
        return x.masked_fill(torch.arange(L, device=DEV)[:, None] >= s.lengths[:, None, None, None],
                             0.0)

    limit = s.cached[:, None] + torch.arange(1, T + 1, device=DEV)
    o = _plain_attention(_padded(s.q, s.starts, T), read(s.kp, s.ks), read(s.vp, s.vs), limit)
    s.out.copy_(o[s.seq, torch.arange(s.rows, device=DEV) - s.starts[s.seq]].reshape(s.rows, -1))
    return s.out


def _plain_prompt(s):
    T = s.longest
    k, v = (_padded(x, s.starts, T).transpose(1, 2) for x in (s.k, s.v))
    limit = torch.arange(1, T + 1, device=DEV).expand(s.seqs, T)
    o = _plain_attention(_padded(s.q, s.starts, T), k, v, limit)
    s.out.copy_(o[s.seq, torch.arange(s.rows, device=DEV) - s.starts[s.seq]].reshape(s.rows, -1))
    return s.out


def run(state):
    s = state
    if hasattr(s, "q_out"):
        if own:
            from ecf8_amd.paged_kernels import paged_qk_norm_rope

            paged_qk_norm_rope(s.qkv, s.batch, s.qn, s.kn, EPS, s.cos, s.sin, s.q_out, s.kp, s.vp,
                               k_scale=s.ks, v_scale=s.vs)
            return {"q": s.q_out, "k": s.kp, "v": s.vp}
        return _plain_write(s)
    if hasattr(s, "longest"):
        if own:
            from ecf8_amd.paged_kernels import ragged_attention

            return ragged_attention(s.q, s.k, s.v, s.starts, s.out)
        return _plain_prompt(s)
    if hasattr(s, "most_new"):
        if own:
            from ecf8_amd.paged_kernels import paged_attention

            return paged_attention(s.q, s.kp, s.vp, s.batch, s.out, max_new=s.most_new,
                                   k_scale=s.ks, v_scale=s.vs)
        return _plain_attend(s)
    if own:
        from ecf8_amd.paged_kernels import paged_plan

        b = s.batch
        paged_plan(b, s.cached, s.new, s.release)
        return {"table": b.table, "owned": b.owned, "free": b.free, "n_free": b.n_free,
                "starts": b.starts, "lengths": b.lengths, "slots": b.slots,
                "positions": b.positions}
    return _plain_plan(s)


# ------------------------------------------------------------ work, 64 bits


def work(case: dict) -> dict:
    cached, new = _lengths(case, 1)
    kind, Hkv, S, N = case["kind"], case.get("kv_heads", 8), case["seqs"], sum(new)
    if kind == "plan":
        page = case["page"]
        # lengths in and out, two ints a row, the pages that change hands or are looked up
        touched = sum(-(-(c + n) // page) - c // page for c, n in zip(cached, new))
        return {"bytes": 4 * (6 * S + 2 * N + (3 if case["admit"] else 1) * touched), "flops": 0}
    size = 1 if case.get("fp8") else 2
    if kind == "write":
        rows = {c + i for c, n in zip(cached, new) for i in range(n)}
        return {"bytes": N * D * (2 * (32 + 2 * Hkv) + 2 * 32 + 2 * size * Hkv) + 512 * len(rows),
                "flops": 10 * N * D * (32 + Hkv)}
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
    keys = sum(c + n for c, n in zip(cached, new) if n)
    return {"bytes": 2 * size * keys * Hkv * D + 2 * 2 * N * 32 * D, "flops": 4 * D * 32 * pairs}


def _exact_heads(q, k, v, first):
    """One sequence in float64: q [n, Hq, D] at positions first.., k and v [L,
    Hkv, D]."""
    n, Hq, _ = q.shape
    L, Hkv, _ = k.shape
    out = torch.empty(n, Hq, D, dtype=torch.float64, device=DEV)
    over = torch.arange(L, device=DEV)[None] > first + torch.arange(n, device=DEV)[:, None]
    for h in range(Hq):
        kh = h * Hkv // Hq
        e = q[:, h].double() @ k[:, kh].double().T / math.sqrt(D)
        e[over] = -math.inf
        out[:, h] = torch.softmax(e, -1) @ v[:, kh].double()
    return out


def exact(case: dict, seed: int):
    if case["kind"] == "plan":
        return None  # whole numbers only
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "prompt":
        out = torch.empty(s.rows, 32 * D, dtype=torch.float64, device=DEV)
        a = 0
        for n in s.new_h:
            out[a: a + n] = _exact_heads(s.q[a: a + n], s.k[a: a + n], s.v[a: a + n], 0).flatten(1)
            a += n
        return out
    if case["kind"] == "write":
        Hkv, pages = case["kv_heads"], s.pages
        x = s.qkv.double().view(s.rows, -1, D)
        pools = [p.double().permute(0, 2, 1, 3).reshape(pages * s.page, Hkv, D).clone()
                 for p in (s.kp, s.vp)]
        cos, sin = (t.double()[s.positions] for t in (s.cos, s.sin))

        def turned(h, w):
            y = x[:, h]
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            c, n = torch.cat([cos, cos], -1), torch.cat([-sin, sin], -1)
            return y * c + torch.roll(y, D // 2, -1) * n

        q = torch.stack([turned(h, s.qn) for h in range(32)], 1)
        for h in range(Hkv):
            for pool, y, scale in ((pools[0], turned(32 + h, s.kn), s.ks),
                                   (pools[1], x[:, 32 + Hkv + h], s.vs)):
                pool[s.slots, h] = y if scale is None else \
                    (y / scale[h].double()).clamp(-FP8_MAX, FP8_MAX)
        k, v = (p.view(pages, s.page, Hkv, D).permute(0, 2, 1, 3) for p in pools)
        return {"q": q, "k": k, "v": v}
    out = torch.empty(s.rows, 32 * D, dtype=torch.float64, device=DEV)
    a = 0
    for i, (c, n) in enumerate(zip(s.cached_h, s.new_h)):
        if not n:
            continue
        p = torch.arange(c + n, device=DEV)
        page, off = s.table[i, p // s.page].long(), p % s.page
        k, v = (x.float()[page, :, off].double() if x.dtype == torch.float8_e4m3fn
                else x[page, :, off].double() for x in (s.kp, s.vp))
        if s.ks is not None:
            k, v = k * s.ks.double()[:, None], v * s.vs.double()[:, None]
        out[a: a + n] = _exact_heads(s.q[a: a + n], k, v, c).flatten(1)
        a += n
    return out
