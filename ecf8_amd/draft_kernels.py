"""Python wrappers of the speculative-decoding kernels (include/ecf8_draft.h):
trees of drafted tokens over the paged cache of ``paged_kernels``.

A step in which every sequence runs its last token and a tree of drafted ones is

    paged_plan(batch, cached, new)               # new: rows of each tree
    draft_plan(trees, parents)                   # masks, rotary positions, schedule
    for each layer:
        paged_qk_norm_rope(qkv, batch, ...)      # at the rows' depths
        draft_attention(q, k_pool, v_pool, trees, out)
    token_probabilities(logits, temperature, target)
    draft_verify(trees, tokens, target, accept, sample, draft)
    draft_keep(keep)                             # what was accepted, in all layers
    cached += trees.kept

and emits ``trees.emitted[s, :kept[s]]`` of each sequence, whose last token is row
0 of its next tree.  All calls launch on torch's current stream and read lengths,
trees and results on the device, so a step can be captured as a HIP graph.  Trees
hold one step at a time, like their batch, and one work buffer: calls with the same
trees have to be ordered, on one stream or by events."""

from __future__ import annotations

import ctypes

import torch

from ._lib import ECF8Error, lib
from .paged_kernels import (HEAD_DIM, PagedBatch, _heads, _launch, _pools, _unfollowed, _want)

MAX_NODES = 64


class _Trees(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in (
        "masks", "parents", "kept", "path", "emitted", "next_token", "work")] +
        [("work_bytes", ctypes.c_int64)] +
        [(n, ctypes.c_int) for n in ("max_nodes", "max_children")])


class DraftTrees:
    """Device buffers of the trees of ``batch``'s steps: up to ``max_nodes`` (at
    most 64) rows of a sequence, row 0 its last token, and up to ``max_children``
    rows drafted after one row:

    * ``masks`` int64 [max_rows]: bit j of a row is set where it reads row j of
      its sequence; ``parents`` int32 [max_rows];
    * ``kept`` int32 [max_seqs], ``path`` int32 [max_seqs, max_nodes]: how many
      and which rows stay after the verification, -1 past them;
    * ``emitted`` int64 [max_seqs, max_nodes]: as many tokens, the accepted ones
      and the next, -1 past them; ``next_token`` int64 [max_seqs].

    Kernels and launches go by ``max_nodes`` and ``max_children``, not by what a step's
    trees hold, so give a chain's (``max_children=1``) where drafts are chains: 64 drawn
    chains of 5 are verified in 24 us, and in 49 with room for 8 children.

    What the device refuses is the batch's to raise (``batch.raise_refused``)."""

    def __init__(self, batch: PagedBatch, max_nodes: int = MAX_NODES, max_children: int = 8):
        n = lib().ecf8_draft_work_bytes(batch.max_seqs, batch.max_rows, batch.Hq, batch.Hkv,
                                        max_nodes, max_children)
        if n < 0:
            raise ECF8Error(f"trees have 1..{MAX_NODES} rows and 1..{MAX_NODES} children of a row")
        dev, S = batch.device, batch.max_seqs
        self.batch, self.max_nodes, self.max_children = batch, max_nodes, max_children
        self.masks = torch.zeros(batch.max_rows, dtype=torch.int64, device=dev)
        self.parents = torch.full((batch.max_rows,), -1, dtype=torch.int32, device=dev)
        self.kept = torch.zeros(S, dtype=torch.int32, device=dev)
        self.path = torch.full((S, max_nodes), -1, dtype=torch.int32, device=dev)
        self.emitted = torch.full((S, max_nodes), -1, dtype=torch.int64, device=dev)
        self.next_token = torch.full((S,), -1, dtype=torch.int64, device=dev)
        self.work = torch.empty(n, dtype=torch.uint8, device=dev)
        self.work[:256].zero_()  # no step planned yet
        self._c = _Trees(*(t.data_ptr() for t in (
            self.masks, self.parents, self.kept, self.path, self.emitted, self.next_token,
            self.work)), n, max_nodes, max_children)
        self._ref = ctypes.addressof(self._c)


def draft_plan(trees: DraftTrees, parents):
    """The trees of the step that ``paged_plan`` planned: ``parents`` int32
    [rows], of each packed row the row of its sequence that it follows, -1 for
    row 0.  Fills ``masks`` and ``parents``, sets the batch's positions to cached +
    depth, and plans ``draft_attention``.  A tree that is none, has more than
    ``max_nodes`` rows or ``max_children`` children sets the batch's ``refused``.
    Once for every ``paged_plan``, also where that plans a step a second time."""
    batch = trees.batch
    _want(parents, torch.int32, "parents", batch.device)
    if parents.numel() > batch.max_rows or parents.numel() < 1:
        raise ECF8Error(f"parents must hold 1..{batch.max_rows} values")
    _launch("ecf8_draft_plan", batch.device, batch._ref, trees._ref, parents.data_ptr(),
            parents.numel())


def draft_attention(q, k_pool, v_pool, trees: DraftTrees, out, k_scale=None, v_scale=None):
    """paged_attention of a step's trees: row t of sequence s reads the cached
    positions and those of the rows in its mask (``trees.masks``, which a caller
    may rewrite after the plan).  A row that reads nothing is zeros; rows past the
    last sequence of ``out`` are left as they were, and all of them, with the batch's
    ``refused`` set, where the trees were not planned for the batch's step.  Probabilities are kept to
    2^-15 where max_nodes * Hq / Hkv is up to 128, and rounded to bf16 once above.
    Returns ``out``."""
    batch = trees.batch
    dev, rows = batch.device, q.shape[0]
    _unfollowed("q out k_pool v_pool k_scale v_scale", q, out, k_pool, v_pool, k_scale, v_scale)
    qs, os = _heads(q, batch.Hq, "q", dev), _heads(out, batch.Hq, "out", dev)
    if not 1 <= rows <= batch.max_rows or out.shape[0] < rows:
        raise ECF8Error(f"q must have 1..{batch.max_rows} rows, and out as many")
    fp8, ks, vs = _pools(batch, k_pool, v_pool, k_scale, v_scale)
    _launch("ecf8_draft_attention", dev, q.data_ptr(), qs, rows, batch._ref, trees._ref,
            k_pool.data_ptr(), v_pool.data_ptr(), fp8, ks, vs, out.data_ptr(), os)
    return out


def _matrix(t, dtype, name, dev):
    """Row stride of a matrix whose rows are contiguous."""
    if not t.is_cuda or t.device != dev or t.dtype != dtype:
        raise ECF8Error(f"{name} must be {dtype} on {dev}")
    if t.dim() != 2 or t.shape[0] < 1 or t.shape[1] < 1 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ECF8Error(f"{name} must be a matrix, its rows contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def token_probabilities(logits, temperature, out):
    """out fp32 [N, V] = softmax(logits / temperature) of bf16 logits [N, V] (rows
    of any stride).  ``temperature``: a number or fp32 [N] on the device; zero or
    less: one at the largest logit (the lowest index of them), zero elsewhere.
    Returns ``out``."""
    dev = logits.device
    per_row = torch.is_tensor(temperature)
    _unfollowed("logits out temperature", logits, out, temperature if per_row else None)
    ld = _matrix(logits, torch.bfloat16, "logits", dev)
    ldo = _matrix(out, torch.float32, "out", dev)
    N, V = logits.shape
    if out.shape[0] < N or out.shape[1] != V or N > 65535:
        raise ECF8Error(f"out must be [>= {N}, {V}], and rows at most 65535")
    if per_row:
        _want(temperature, torch.float32, "temperature", dev)
        if temperature.numel() != N:
            raise ECF8Error(f"temperature must hold {N} values")
    work = torch.empty(N * 64, dtype=torch.int64, device=dev)
    _launch("ecf8_token_probabilities", dev, logits.data_ptr(), ld, N, V,
            temperature.data_ptr() if per_row else None, 0.0 if per_row else float(temperature),
            out.data_ptr(), ldo, work.data_ptr(), work.numel() * 8)
    return out


def draft_verify(trees: DraftTrees, tokens, target, accept, sample, draft=None):
    """Verify the step's drafts: ``tokens`` int64 [N] of the packed rows,
    ``target`` fp32 [N, V] the model's probabilities after each of them, ``accept``
    fp32 [N] and ``sample`` fp32 [max_seqs] random numbers in [0, 1).  Children of
    a row are tried in order.  Without ``draft`` they are different tokens, chosen
    in any way that does not look at the random numbers (a drafter's most probable
    ones); with ``draft`` fp32 [N, V] they were drawn, independently, from that
    row's probabilities.  Either way the emitted tokens are distributed as the
    target's own.  Fills ``kept``, ``path``, ``emitted`` and ``next_token``; trees that
    were not planned for the batch's step are refused, all sequences idle."""
    batch = trees.batch
    dev = batch.device
    _unfollowed("target accept sample draft", target, accept, sample, draft)
    ld = _matrix(target, torch.float32, "target", dev)
    N, V = target.shape
    if N > batch.max_rows:
        raise ECF8Error(f"target must have 1..{batch.max_rows} rows")
    _want(tokens, torch.int64, "tokens", dev)
    _want(accept, torch.float32, "accept", dev)
    _want(sample, torch.float32, "sample", dev)
    if tokens.numel() != N or accept.numel() != N or sample.numel() != batch.max_seqs:
        raise ECF8Error(f"tokens and accept must hold {N} values, sample {batch.max_seqs}")
    ldd = 0
    if draft is not None:
        ldd = _matrix(draft, torch.float32, "draft", dev)
        if draft.shape != target.shape:
            raise ECF8Error(f"draft must be [{N}, {V}]")
    _launch("ecf8_draft_verify", dev, batch._ref, trees._ref, tokens.data_ptr(), N,
            target.data_ptr(), ld, None if draft is None else draft.data_ptr(), ldd, V,
            accept.data_ptr(), sample.data_ptr())


class KeepPlan:
    """The pools of all layers, checked once: ``layers`` is a list of (k_pool,
    v_pool), bf16 or e4m3 alike, which have to stay in place while it is used."""

    def __init__(self, trees: DraftTrees, layers):
        batch = trees.batch
        self.trees = trees
        self.pools = [p for pair in layers for p in pair]
        if not self.pools:
            raise ECF8Error("there must be a layer")
        self.fp8 = int(self.pools[0].dtype == torch.float8_e4m3fn)
        shape = (batch.pages, batch.Hkv, batch.page_size, HEAD_DIM)
        for p in self.pools:
            _want(p, torch.float8_e4m3fn if self.fp8 else torch.bfloat16, "pool", batch.device)
            if p.shape != shape:
                raise ECF8Error(f"pools must be {list(shape)}")
        if len({p.data_ptr() for p in self.pools}) != len(self.pools):
            raise ECF8Error("a pool may be there once")
        _unfollowed("pool " * len(self.pools), *self.pools)
        self._c = (ctypes.c_void_p * len(self.pools))(*(p.data_ptr() for p in self.pools))
        self._ref = ctypes.addressof(self._c)


def draft_keep(plan: KeepPlan):
    """Move the keys and values of the accepted rows together: in all pools the row
    at position cached[s] + path[s, i] goes to cached[s] + i, i < kept[s].  The next
    step has ``kept`` more tokens in the cache.  Before ``paged_plan`` plans the next
    one: the trees are of another step then, which is refused.  Once a step and list of
    pools: a second call would move what is in its place."""
    trees, batch = plan.trees, plan.trees.batch
    _launch("ecf8_draft_keep", batch.device, batch._ref, trees._ref, plan._ref, len(plan.pools),
            plan.fp8)
