"""Python wrappers of the ragged-batch kernels (include/ecf8_paged.h):
sequences of different lengths over a paged KV cache, and packed prompts.

A step of a served batch is

    paged_plan(batch, cached, new, release)      # once: pages, slots, schedule
    for each layer:
        paged_qk_norm_rope(qkv, batch, ...)      # q, and k / v into the pages
        paged_attention(q, k_pool, v_pool, batch, out)

with one ``PagedBatch`` for all layers and one pair of pools a layer.  Every
call launches on torch's current stream of the tensors' device and reads the
lengths on the device, so a step can be captured as a HIP graph and replayed
with other lengths.  A batch holds one step at a time: steps that may overlap
(two streams, two graphs in flight) need a batch each."""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from ._lib import ECF8Error, check, lib
from .head_kernels import _flag_ptr, refusal_flag
from .llm_kernels import _need

HEAD_DIM = 128


class _Batch(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in (
        "table", "owned", "free_pages", "n_free", "starts", "lengths", "slots", "positions",
        "refused", "work")] + [("work_bytes", ctypes.c_int64)] +
        [(n, ctypes.c_int) for n in ("seqs", "rows", "pages", "page_size", "width", "Hq", "Hkv")])


class PagedBatch:
    """Device buffers of a batch of up to ``max_seqs`` sequences of up to
    ``max_len`` tokens over pools of ``pages`` pages of ``page_size`` (a power
    of two up to 1024) positions, for steps of up to ``max_rows`` new tokens
    and layers of ``Hq`` query and ``Hkv`` KV heads:

    * ``table`` int32 [max_seqs, width], ``owned`` [max_seqs]: each sequence's
      pages in order (-1 past them);
    * ``free`` int32 [pages], ``n_free`` [1]: stack of the free pages, all of
      them at first;
    * ``starts`` [max_seqs + 1], ``lengths`` [max_seqs], ``slots`` and
      ``positions`` [max_rows]: the planned step's rows;
    * ``refused``: a flag in host memory, nonzero once a kernel refused a
      step's values (``raise_refused``)."""

    def __init__(self, max_seqs: int, max_rows: int, pages: int, page_size: int, max_len: int,
                 Hq: int, Hkv: int, device):
        n = lib().ecf8_paged_work_bytes(max_seqs, max_rows, Hq, Hkv) if Hkv > 0 else -1
        if n < 0:
            raise ECF8Error("a batch has 1..4096 sequences, 1..262144 rows and Hq a multiple of "
                            "Hkv up to 1024")
        if not 1 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ECF8Error("page_size must be a power of two up to 1024")
        if not 1 <= max_len <= 2**24 - page_size or pages < 1:
            raise ECF8Error("max_len must be 1..2**24 - page_size, and there must be a page")
        width = -(-max_len // page_size)
        if max_seqs * width >= 2**31 or pages * page_size * Hkv >= 2**31:
            raise ECF8Error("tables and pools hold less than 2**31 entries and rows")
        i32 = dict(dtype=torch.int32, device=device)
        self.max_seqs, self.max_rows, self.pages = max_seqs, max_rows, pages
        self.page_size, self.max_len, self.Hq, self.Hkv = page_size, width * page_size, Hq, Hkv
        self.table = torch.full((max_seqs, width), -1, **i32)
        self.owned = torch.zeros(max_seqs, **i32)
        self.free = torch.arange(pages - 1, -1, -1, **i32)  # page 0 on top
        self.n_free = torch.full((1,), pages, **i32)
        self.starts = torch.zeros(max_seqs + 1, **i32)
        self.lengths = torch.zeros(max_seqs, **i32)
        self.slots = torch.full((max_rows,), -1, **i32)
        self.positions = torch.full((max_rows,), -1, **i32)
        self.work = torch.empty(n, dtype=torch.uint8, device=device)
        self.work[:256].zero_()  # no step planned yet
        self.device = self.work.device
        self.refused = refusal_flag()
        self._refused_host = self.refused.numpy()
        self._c = _Batch(*(t.data_ptr() for t in (
            self.table, self.owned, self.free, self.n_free, self.starts, self.lengths, self.slots,
            self.positions, self.refused, self.work)), n, max_seqs, max_rows, pages, page_size,
            width, Hq, Hkv)
        self._ref = ctypes.addressof(self._c)

    def raise_refused(self):
        """Raise if a kernel refused a step since the last call (synchronize
        first to cover every launched step)."""
        if self._refused_host[0]:
            self.refused.zero_()
            raise ECF8Error("a step did not fit: lengths out of range, too few free pages, or more "
                            "rows or new tokens than the call allowed for")


def _launch(name, dev, *args):
    fn = getattr(lib(), name)
    # (the stream's handle: torch.cuda.current_stream takes 1.8 us of a call's 10)
    if dev.index == torch.cuda.current_device():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(dev.index)), name)
    else:
        with torch.cuda.device(dev):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(dev.index)), name)


def _unfollowed(names, *tensors):
    """Refuses tensors that autograd follows, backward or forward."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ECF8Error(f"{_name(names, tensors, t)} is followed by autograd: these "
                                "kernels have no backward")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ECF8Error(f"{_name(names, tensors, t)} is followed by autograd: these "
                                "kernels have no tangent")


def _name(names, tensors, t):
    return next(n for n, u in zip(names.split(), tensors) if u is t)


def _want(t, dtype, name, dev):
    """_need, at half of its price where all is well."""
    if t.dtype is not dtype or not t.is_cuda or t.device != dev or not t.is_contiguous():
        _need(t, dtype, name, dev)


def _ints(t, n, name, dev):
    _want(t, torch.int32, name, dev)
    if t.numel() != n:
        raise ECF8Error(f"{name} must hold {n} values")


def _heads(t, heads, name, dev):
    """Row stride of ``t``: bf16 [N, heads, 128] or [N, heads * 128], a row's
    heads contiguous."""
    if not t.is_cuda or t.device != dev or t.dtype != torch.bfloat16:
        raise ECF8Error(f"{name} must be bfloat16 on {dev}")
    shape, stride = t.shape, t.stride()
    if not ((len(shape) == 2 and shape[1] == heads * HEAD_DIM and stride[1] == 1)
            or (len(shape) == 3 and shape[1:] == (heads, HEAD_DIM) and stride[2] == 1
                and (stride[1] == HEAD_DIM or heads == 1))):
        raise ECF8Error(f"{name} {tuple(shape)} must be [rows, {heads}, {HEAD_DIM}], heads of a "
                        "row contiguous")
    return stride[0] if shape[0] > 1 else heads * HEAD_DIM


def _pools(batch, k_pool, v_pool, k_scale, v_scale):
    """Checks a layer's pools; (1 if they hold e4m3 codes, scale addresses)."""
    dev, fp8 = batch.device, k_pool.dtype == torch.float8_e4m3fn
    shape = (batch.pages, batch.Hkv, batch.page_size, HEAD_DIM)
    for t, n in ((k_pool, "k_pool"), (v_pool, "v_pool")):
        _want(t, torch.float8_e4m3fn if fp8 else torch.bfloat16, n, dev)
        if t.shape != shape:
            raise ECF8Error(f"{n} must be {list(shape)}")
    if not fp8:
        if k_scale is not None or v_scale is not None:
            raise ECF8Error("scales belong to e4m3 pools")
        return 0, None, None
    if k_scale is None or v_scale is None:
        raise ECF8Error("e4m3 pools need k_scale and v_scale")
    for t, n in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        _want(t, torch.float32, n, dev)
        if t.numel() != batch.Hkv:
            raise ECF8Error(f"{n} must hold one scale per KV head")
    return 1, k_scale.data_ptr(), v_scale.data_ptr()


def paged_plan(batch: PagedBatch, cached, new, release=None):
    """Plan one step: sequence s has ``cached[s]`` tokens in the cache and
    brings ``new[s]`` more (0: idle); ``release[s]`` != 0 first gives back the
    pages it owns (int32 [max_seqs] each).  Allocates pages, and fills
    ``starts``, ``lengths`` (cached + new), ``slots`` and ``positions``.  A
    step that does not fit sets ``refused``, changes no page and is planned
    empty.  The inputs are read by the launch alone.  To plan a step a second
    time, leave ``release`` out: it would give the new pages back as well."""
    dev = batch.device
    _ints(cached, batch.max_seqs, "cached", dev)
    _ints(new, batch.max_seqs, "new", dev)
    if release is not None:
        _ints(release, batch.max_seqs, "release", dev)
    _launch("ecf8_paged_plan", dev, batch._ref, cached.data_ptr(), new.data_ptr(),
            None if release is None else release.data_ptr())


def paged_qk_norm_rope(qkv, batch: PagedBatch, q_norm, k_norm, eps, cos_t, sin_t, q_out, k_pool,
                       v_pool, k_scale=None, v_scale=None):
    """qk_norm_rope for the planned step's packed rows: qkv bf16 [rows, (Hq +
    2 * Hkv) * 128] -> q_out bf16 [rows, Hq, 128] and, at each row's slot,
    the pools [pages, Hkv, page_size, 128], bf16 or e4m3fn (codes of x / scale,
    fp32 scales [Hkv]).  cos_t / sin_t fp32 [>= max_len, 64]."""
    dev, Hq, Hkv = batch.device, batch.Hq, batch.Hkv
    _unfollowed("qkv q_norm k_norm cos sin q_out k_pool v_pool k_scale v_scale", qkv, q_norm,
                k_norm, cos_t, sin_t, q_out, k_pool, v_pool, k_scale, v_scale)
    for t, n in ((qkv, "qkv"), (q_norm, "q_norm"), (k_norm, "k_norm"), (q_out, "q_out")):
        _want(t, torch.bfloat16, n, dev)
    _want(cos_t, torch.float32, "cos", dev)
    _want(sin_t, torch.float32, "sin", dev)
    rows = qkv.shape[0]
    if qkv.dim() != 2 or qkv.shape[1] != (Hq + 2 * Hkv) * HEAD_DIM or not 1 <= rows <= batch.max_rows:
        raise ECF8Error(f"qkv must be [1..{batch.max_rows}, {(Hq + 2 * Hkv) * HEAD_DIM}]")
    if q_out.numel() < rows * Hq * HEAD_DIM:
        raise ECF8Error("q_out too small")
    if q_norm.numel() != HEAD_DIM or k_norm.numel() != HEAD_DIM:
        raise ECF8Error("q_norm / k_norm must be [128]")
    if (cos_t.dim() != 2 or cos_t.shape != sin_t.shape or cos_t.shape[1] != HEAD_DIM // 2
            or cos_t.shape[0] < batch.max_len):
        raise ECF8Error(f"rotary tables must be [>= {batch.max_len}, 64]")
    fp8, ks, vs = _pools(batch, k_pool, v_pool, k_scale, v_scale)
    _launch("ecf8_paged_qk_norm_rope", dev, qkv.data_ptr(), rows, batch._ref, q_norm.data_ptr(),
            k_norm.data_ptr(), float(eps), cos_t.data_ptr(), sin_t.data_ptr(), cos_t.shape[0],
            q_out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), fp8, ks, vs)


def paged_attention(q, k_pool, v_pool, batch: PagedBatch, out, max_new=None, k_scale=None,
                    v_scale=None):
    """Attention of the planned step's rows over the pages: token t of
    sequence s reads positions [0, cached[s] + t].  q, out bf16 [rows, Hq,
    128] or [rows, Hq * 128], rows of any 16-byte aligned stride; rows past
    the last sequence of ``out`` are left as they were.  ``max_new``: at least
    the new tokens of any sequence (default: any number); one token each runs
    one kernel less.  Returns ``out``."""
    dev, rows = batch.device, q.shape[0]
    _unfollowed("q out k_pool v_pool k_scale v_scale", q, out, k_pool, v_pool, k_scale, v_scale)
    qs, os = _heads(q, batch.Hq, "q", dev), _heads(out, batch.Hq, "out", dev)
    if not 1 <= rows <= batch.max_rows or out.shape[0] < rows:
        raise ECF8Error(f"q must have 1..{batch.max_rows} rows, and out as many")
    most = rows if max_new is None else min(int(max_new), rows)
    if most < 1:
        raise ECF8Error("max_new must be positive")
    fp8, ks, vs = _pools(batch, k_pool, v_pool, k_scale, v_scale)
    _launch("ecf8_paged_attention", dev, q.data_ptr(), qs, rows, batch._ref, k_pool.data_ptr(),
            v_pool.data_ptr(), fp8, ks, vs, most, out.data_ptr(), os)
    return out


def ragged_attention(q, k, v, starts, out, refused=None):
    """Causal attention of packed prompts of different lengths, without a
    cache: sequence s has rows [starts[s], starts[s + 1]) (int32, on the
    device, ascending) of q [N, Hq, 128] and k, v [N, Hkv, 128] (bf16, e.g.
    slices of a fused projection's output), Hq a multiple of Hkv; row t reads
    rows 0..t of its sequence.  Probabilities are rounded to bf16 once from
    49152 (N * Hq) on, and kept to 2^-15 below.  out: bf16 [N, Hq * 128] or [N, Hq, 128], rows
    outside every sequence left as they were.  ``refused`` (a refusal_flag()):
    set by starts that are not ascending or outside [0, N], whose rows are
    incomplete.  Returns ``out``."""
    dev = q.device
    _unfollowed("q k v out", q, k, v, out)
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] < 1:
        raise ECF8Error("q, k, v must be [rows, heads, 128]")
    N, Hq, Hkv = q.shape[0], q.shape[1], k.shape[1]
    strides = [_heads(q, Hq, "q", dev), _heads(k, Hkv, "k", dev), _heads(v, Hkv, "v", dev)]
    os = _heads(out, Hq, "out", dev)
    if k.shape[0] != N or v.shape[0] != N or out.shape[0] < N:
        raise ECF8Error("q, k and v must have the same rows, and out as many")
    _want(starts, torch.int32, "starts", dev)
    if starts.numel() < 2:
        raise ECF8Error("starts must hold the sequences' first rows and the end")
    _launch("ecf8_ragged_attention_checked", dev, q.data_ptr(), strides[0], k.data_ptr(), strides[1],
            v.data_ptr(), strides[2], N, starts.data_ptr(), starts.numel() - 1, Hq, Hkv,
            out.data_ptr(), os, _flag_ptr(refused, dev))
    return out
