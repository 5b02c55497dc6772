"""What the ragged-batch entry points (include/ecf8_paged.h) refuse before
any HIP call, and what their Python wrappers refuse before that.  CPU only."""

from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 1 << 20  # never dereferenced: every call below is rejected first


def _batch(**kw):
    from ecf8_amd._lib import lib
    from ecf8_amd.paged_kernels import _Batch

    f = dict(table=FAKE, owned=FAKE, free_pages=FAKE, n_free=FAKE, starts=FAKE, lengths=FAKE,
             slots=FAKE, positions=FAKE, refused=None, work=FAKE, seqs=4, rows=16, pages=64,
             page_size=16, width=8, Hq=8, Hkv=2)
    f.update(kw)
    if "work_bytes" not in f:
        f["work_bytes"] = max(0, lib().ecf8_paged_work_bytes(4, 16, 8, 2))
        if f["seqs"] > 0 and f["rows"] > 0 and f["Hkv"] > 0:
            f["work_bytes"] = lib().ecf8_paged_work_bytes(f["seqs"], f["rows"], f["Hq"], f["Hkv"])
    return _Batch(**f)


BAD_BATCH = [
    (dict(table=None), 1), (dict(positions=None), 1), (dict(work=None), 1), (dict(seqs=0), 1),
    (dict(rows=0), 1), (dict(pages=0), 1), (dict(page_size=0), 1), (dict(Hkv=0), 1),
    (dict(seqs=4097), 2), (dict(rows=(1 << 18) + 1), 2), (dict(page_size=24), 2),
    (dict(page_size=2048), 2), (dict(Hq=9), 2), (dict(Hq=1), 2), (dict(Hq=1026), 2),
    (dict(width=1 << 21), 2), (dict(pages=1 << 27), 2), (dict(pages=1 << 26), 2),
    (dict(starts=FAKE + 2), 3), (dict(work=FAKE + 8), 3), (dict(refused=FAKE + 1), 3),
    (dict(work_bytes=1024), 6)]


@pytest.mark.parametrize("kw,status", BAD_BATCH)
def test_a_bad_batch_is_refused_by_every_entry_point(kw, status):
    from ecf8_amd._lib import lib

    L, b = lib(), _batch(**kw)
    at = ctypes.addressof(b)
    assert L.ecf8_paged_plan(at, FAKE, FAKE, None, None) == status
    assert L.ecf8_paged_qk_norm_rope(FAKE, 1, at, FAKE, FAKE, 1e-6, FAKE, FAKE, 128, FAKE, FAKE,
                                     FAKE, 0, None, None, None) == status
    assert L.ecf8_paged_attention(FAKE, 1024, 1, at, FAKE, FAKE, 0, None, None, 1, FAKE, 1024,
                                  None) == status


def test_work_bytes():
    from ecf8_amd._lib import lib

    f = lib().ecf8_paged_work_bytes
    assert f(1, 1, 1, 1) > 0 and f(4096, 1 << 18, 1024, 1) > 0
    for bad in ((0, 1, 1, 1), (4097, 1, 1, 1), (1, 0, 1, 1), (1, (1 << 18) + 1, 1, 1),
                (1, 1, 3, 2), (1, 1, 0, 1), (1, 1, 1, 0), (1, 1, -2, -1), (1, 1, 2048, 1)):
        assert f(*bad) == -1, bad


def test_plan_rejects_before_launch():
    from ecf8_amd._lib import lib

    b = _batch()
    at = ctypes.addressof(b)
    for args, status in (((None, FAKE, FAKE, None), 1), ((at, None, FAKE, None), 1),
                         ((at, FAKE, None, None), 1), ((at, FAKE + 1, FAKE, None), 3),
                         ((at, FAKE, FAKE + 2, None), 3), ((at, FAKE, FAKE, FAKE + 3), 3)):
        assert lib().ecf8_paged_plan(*args, None) == status, args


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=None), 1), (dict(q_out=None), 1), (dict(vp=None), 1), (dict(n=0), 1), (dict(n=17), 6),
    (dict(table=0), 1), (dict(table=(1 << 24) + 1), 2), (dict(fp8=1), 1),
    (dict(fp8=1, ks=FAKE, vs=FAKE + 2), 3), (dict(qkv=FAKE + 8), 3), (dict(cos=FAKE + 4), 3),
    (dict(kp=FAKE + 8), 3), (dict(qn=FAKE + 2), 3)])
def test_write_rejects_before_launch(kw, status):
    from ecf8_amd._lib import lib

    a = dict(qkv=FAKE, n=16, qn=FAKE, kn=FAKE, cos=FAKE, sin=FAKE, table=128, q_out=FAKE, kp=FAKE,
             vp=FAKE, fp8=0, ks=None, vs=None)
    a.update(kw)
    b = _batch()
    assert lib().ecf8_paged_qk_norm_rope(
        a["qkv"], a["n"], ctypes.addressof(b), a["qn"], a["kn"], 1e-6, a["cos"], a["sin"],
        a["table"], a["q_out"], a["kp"], a["vp"], a["fp8"], a["ks"], a["vs"], None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(out=None), 1), (dict(kp=None), 1), (dict(n=0), 1), (dict(n=17), 6),
    (dict(most=0), 1), (dict(fp8=1, ks=FAKE), 1), (dict(qs=1020), 2), (dict(qs=512), 2),
    (dict(os=1022), 2), (dict(os=512), 2), (dict(q=FAKE + 8), 3), (dict(out=FAKE + 4), 3),
    (dict(vp=FAKE + 8), 3), (dict(fp8=1, ks=FAKE, vs=FAKE + 1), 3)])
def test_attention_rejects_before_launch(kw, status):
    from ecf8_amd._lib import lib

    a = dict(q=FAKE, qs=1024, n=16, kp=FAKE, vp=FAKE, fp8=0, ks=None, vs=None, most=1, out=FAKE,
             os=1024)
    a.update(kw)
    b = _batch()
    assert lib().ecf8_paged_attention(a["q"], a["qs"], a["n"], ctypes.addressof(b), a["kp"],
                                      a["vp"], a["fp8"], a["ks"], a["vs"], a["most"], a["out"],
                                      a["os"], None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(starts=None), 1), (dict(n=0), 1), (dict(s=0), 1), (dict(hkv=0), 1),
    (dict(hq=-8), 1), (dict(hq=9), 2), (dict(s=4097), 2), (dict(n=(1 << 18) + 1), 2),
    (dict(qs=1028), 2), (dict(ks=128), 2), (dict(vs=260), 2), (dict(os=1020), 2),
    (dict(k=FAKE + 8), 3), (dict(out=FAKE + 4), 3), (dict(starts=FAKE + 2), 3)])
def test_ragged_rejects_before_launch(kw, status):
    from ecf8_amd._lib import lib

    a = dict(q=FAKE, qs=1024, k=FAKE, ks=256, v=FAKE, vs=256, n=16, starts=FAKE, s=2, hq=8, hkv=2,
             out=FAKE, os=1024)
    a.update(kw)
    assert lib().ecf8_ragged_attention(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["n"],
                                       a["starts"], a["s"], a["hq"], a["hkv"], a["out"], a["os"],
                                       None) == status


def test_the_struct_is_the_headers():
    import os
    import re

    from ecf8_amd.paged_kernels import _Batch

    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "ecf8_paged.h")).read()
    body = text[text.index("typedef struct ecf8_paged_batch"):text.index("} ecf8_paged_batch;")]
    assert re.findall(r"\b(\w+);", body) == [n for n, _ in _Batch._fields_]


@pytest.mark.parametrize("args", [
    (0, 1, 8, 16, 64, 8, 2), (1, 0, 8, 16, 64, 8, 2), (1, 1, 0, 16, 64, 8, 2),
    (1, 1, 8, 24, 64, 8, 2), (1, 1, 8, 2048, 64, 8, 2), (1, 1, 8, 16, 0, 8, 2),
    (1, 1, 8, 16, 1 << 24, 8, 2), (1, 1, 8, 16, 64, 9, 2), (1, 1, 8, 16, 64, 8, 0),
    (4096, 1, 8, 1, 1 << 20, 8, 2), (1, 1, 1 << 27, 16, 64, 8, 2)])
def test_a_batch_refuses_its_sizes(args):
    from ecf8_amd._lib import ECF8Error
    from ecf8_amd.paged_kernels import PagedBatch

    with pytest.raises(ECF8Error):
        PagedBatch(*args, "cpu")


def test_wrappers_refuse_host_tensors_and_shapes():
    """Tensors that are not on the GPU never reach a launch."""
    from ecf8_amd import paged_kernels as P
    from ecf8_amd._lib import ECF8Error

    b = P.PagedBatch(2, 4, 8, 16, 64, 4, 2, "cpu")
    assert b.max_len == 64 and b.table.shape == (2, 4) and b.free.tolist() == list(range(7, -1, -1))
    two = torch.zeros(2, dtype=torch.int32)
    bf = dict(dtype=torch.bfloat16)
    q, kv = torch.zeros(4, 4, 128, **bf), torch.zeros(4, 2, 128, **bf)
    pool = torch.zeros(8, 2, 16, 128, **bf)
    tab, w = torch.zeros(64, 64), torch.zeros(128, **bf)
    with pytest.raises(ECF8Error):
        P.paged_plan(b, two, two)
    with pytest.raises(ECF8Error):
        P.paged_qk_norm_rope(torch.zeros(4, 8 * 128, **bf), b, w, w, 1e-6, tab, tab, q, pool, pool)
    with pytest.raises(ECF8Error):
        P.paged_attention(q, pool, pool, b, torch.zeros(4, 512, **bf))
    with pytest.raises(ECF8Error):
        P.ragged_attention(q, kv, kv, torch.zeros(3, dtype=torch.int32), torch.zeros(4, 512, **bf))
    b.refused[0] = 1
    with pytest.raises(ECF8Error):
        b.raise_refused()
    b.raise_refused()
