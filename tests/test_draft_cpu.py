"""What the speculative-decoding entry points (include/ecf8_draft.h) refuse
before any HIP call, and what their Python wrappers refuse before that.  CPU
only."""

from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch

FAKE = 1 << 20  # never dereferenced: every call below is rejected first


def _batch(**kw):
    from ecf8_amd._lib import lib
    from ecf8_amd.paged_kernels import _Batch

    f = dict(table=FAKE, owned=FAKE, free_pages=FAKE, n_free=FAKE, starts=FAKE, lengths=FAKE,
             slots=FAKE, positions=FAKE, refused=None, work=FAKE, seqs=4, rows=16, pages=64,
             page_size=16, width=8, Hq=8, Hkv=2)
    f["work_bytes"] = lib().ecf8_paged_work_bytes(4, 16, 8, 2)
    f.update(kw)
    return _Batch(**f)


def _trees(**kw):
    from ecf8_amd._lib import lib
    from ecf8_amd.draft_kernels import _Trees

    f = dict(masks=FAKE, parents=FAKE, kept=FAKE, path=FAKE, emitted=FAKE, next_token=FAKE,
             work=FAKE, max_nodes=8, max_children=3)
    f["work_bytes"] = lib().ecf8_draft_work_bytes(4, 16, 8, 2, 8, 3)
    f.update(kw)
    return _Trees(**f)


def _calls(b, t):
    """Every entry point of a batch and its trees, with arguments that it takes."""
    from ecf8_amd._lib import lib

    L, pools, held = lib(), (ctypes.c_void_p * 2)(FAKE, FAKE), (b, t)
    b = None if b is None else ctypes.addressof(b)
    t = None if t is None else ctypes.addressof(t)
    return {
        "held": lambda: held, "plan": lambda p=FAKE, n=16: L.ecf8_draft_plan(b, t, p, n, None),
        "attend": lambda q=FAKE, qs=1024, n=16, k=FAKE, v=FAKE, fp8=0, ks=None, vs=None, out=FAKE,
        os=1024: L.ecf8_draft_attention(q, qs, n, b, t, k, v, fp8, ks, vs, out, os, None),
        "verify": lambda tok=FAKE, n=16, p=FAKE, lp=1000, q=None, lq=0, V=1000, u=FAKE, s=FAKE:
        L.ecf8_draft_verify(b, t, tok, n, p, lp, q, lq, V, u, s, None),
        "keep": lambda p=pools, n=2, fp8=0: L.ecf8_draft_keep(b, t, p, n, fp8, None)}


BAD = [("b", dict(table=None), 1), ("b", dict(seqs=0), 1), ("b", dict(page_size=24), 2),
       ("b", dict(Hq=9), 2), ("b", dict(work=FAKE + 8), 3), ("b", dict(work_bytes=10), 6),
       ("t", dict(masks=None), 1), ("t", dict(parents=None), 1), ("t", dict(kept=None), 1),
       ("t", dict(path=None), 1), ("t", dict(emitted=None), 1), ("t", dict(next_token=None), 1),
       ("t", dict(work=None), 1), ("t", dict(max_nodes=0), 1), ("t", dict(max_children=-1), 1),
       ("t", dict(max_nodes=65), 2), ("t", dict(max_children=65), 2), ("t", dict(masks=FAKE + 4), 3),
       ("t", dict(emitted=FAKE + 4), 3), ("t", dict(next_token=FAKE + 1), 3),
       ("t", dict(path=FAKE + 2), 3), ("t", dict(work=FAKE + 8), 3), ("t", dict(work_bytes=10), 6)]


@pytest.mark.parametrize("which,kw,status", BAD)
def test_a_bad_batch_or_trees_are_refused_by_every_entry_point(which, kw, status):
    b, t = (_batch(**kw), _trees()) if which == "b" else (_batch(), _trees(**kw))
    for name in ("plan", "attend", "verify", "keep"):
        for calls, want in ((_calls(b, t), status), (_calls(_batch(), None), 1),
                            (_calls(None, _trees()), 1)):
            assert calls[name]() == want, name


@pytest.mark.parametrize("name,kw,status", [
    ("plan", dict(p=None), 1), ("plan", dict(p=FAKE + 2), 3), ("plan", dict(n=0), 1),
    ("plan", dict(n=17), 6),
    ("attend", dict(q=None), 1), ("attend", dict(out=None), 1), ("attend", dict(v=None), 1),
    ("attend", dict(n=0), 1), ("attend", dict(n=17), 6), ("attend", dict(fp8=1, ks=FAKE), 1),
    ("attend", dict(qs=1020), 2), ("attend", dict(qs=512), 2), ("attend", dict(os=1022), 2),
    ("attend", dict(os=512), 2), ("attend", dict(q=FAKE + 8), 3), ("attend", dict(k=FAKE + 8), 3),
    ("attend", dict(out=FAKE + 4), 3), ("attend", dict(fp8=1, ks=FAKE + 2, vs=FAKE), 3),
    ("verify", dict(tok=None), 1), ("verify", dict(p=None), 1), ("verify", dict(u=None), 1),
    ("verify", dict(s=None), 1), ("verify", dict(n=0), 1), ("verify", dict(V=0), 1),
    ("verify", dict(n=17), 6), ("verify", dict(lp=999), 2), ("verify", dict(q=FAKE, lq=999), 2),
    ("verify", dict(V=(1 << 30) + 1, lp=1 << 31), 2), ("verify", dict(tok=FAKE + 4), 3),
    ("verify", dict(p=FAKE + 2), 3), ("verify", dict(q=FAKE + 1, lq=1000), 3),
    ("verify", dict(u=FAKE + 2), 3), ("verify", dict(s=FAKE + 2), 3),
    ("keep", dict(p=None), 1), ("keep", dict(n=0), 1),
    ("keep", dict(p=(ctypes.c_void_p * 2)(FAKE, None)), 1),
    ("keep", dict(p=(ctypes.c_void_p * 2)(FAKE, FAKE + 8)), 3)])
def test_calls_reject_before_launch(name, kw, status):
    calls = _calls(_batch(), _trees())  # (holds both)
    assert calls[name](**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), 1), (dict(out=None), 1), (dict(work=None), 1), (dict(n=0), 1), (dict(V=0), 1),
    (dict(n=65536), 2), (dict(V=(1 << 30) + 1), 2), (dict(ld=999), 2), (dict(ldo=999), 6),
    (dict(bytes=10), 6), (dict(x=FAKE + 1), 3), (dict(out=FAKE + 2), 3), (dict(t=FAKE + 2), 3),
    (dict(work=FAKE + 4), 3)])
def test_probabilities_reject_before_launch(kw, status):
    from ecf8_amd._lib import lib

    a = dict(x=FAKE, ld=1000, n=4, V=1000, t=None, out=FAKE, ldo=1000, work=FAKE, bytes=1 << 20)
    a.update(kw)
    assert lib().ecf8_token_probabilities(a["x"], a["ld"], a["n"], a["V"], a["t"], 1.0, a["out"],
                                          a["ldo"], a["work"], a["bytes"], None) == status


def test_work_bytes():
    from ecf8_amd._lib import lib

    f, g = lib().ecf8_draft_work_bytes, lib().ecf8_probability_work_bytes
    assert f(1, 1, 1, 1, 1, 1) > 0 and f(4096, 1 << 18, 1024, 1, 64, 64) > 0
    for bad in ((0, 1, 1, 1, 1, 1), (1, 0, 1, 1, 1, 1), (1, 1, 3, 2, 1, 1), (1, 1, 1, 1, 0, 1),
                (1, 1, 1, 1, 65, 1), (1, 1, 1, 1, 1, 0), (1, 1, 1, 1, 1, 65), (4097, 1, 1, 1, 1, 1)):
        assert f(*bad) == -1, bad
    assert g(3) == 3 * 64 * 8 and g(0) == -1 and g(65536) == -1


def test_the_struct_is_the_headers():
    from ecf8_amd.draft_kernels import _Trees

    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "ecf8_draft.h")).read()
    body = text[text.index("typedef struct ecf8_draft_trees"):text.index("} ecf8_draft_trees;")]
    assert re.findall(r"\b(\w+);", body) == [n for n, _ in _Trees._fields_]


def _on_host():
    from ecf8_amd.draft_kernels import DraftTrees
    from ecf8_amd.paged_kernels import PagedBatch

    return DraftTrees(PagedBatch(2, 6, 8, 16, 64, 4, 2, "cpu"), 4, 3)


@pytest.mark.parametrize("args", [(0, 1), (65, 1), (4, 0), (4, 65), (-1, 2)])
def test_trees_refuse_their_sizes(args):
    from ecf8_amd._lib import ECF8Error
    from ecf8_amd.draft_kernels import DraftTrees

    with pytest.raises(ECF8Error):
        DraftTrees(_on_host().batch, *args)


def test_wrappers_refuse_host_tensors():
    """Tensors that are not on the GPU never reach a launch."""
    from ecf8_amd import draft_kernels as K
    from ecf8_amd._lib import ECF8Error

    t = _on_host()
    assert t.masks.shape == (6,) and t.path.shape == t.emitted.shape == (2, 4)
    pool, q = torch.zeros(8, 2, 16, 128).bfloat16(), torch.zeros(6, 4, 128).bfloat16()
    p, u = torch.rand(6, 9), torch.rand(6)
    for call in (lambda: K.draft_plan(t, torch.zeros(6, dtype=torch.int32)),
                 lambda: K.draft_attention(q, pool, pool, t, q.clone()),
                 lambda: K.token_probabilities(p.bfloat16(), 1.0, p),
                 lambda: K.draft_verify(t, torch.zeros(6, dtype=torch.int64), p, u, u[:2]),
                 lambda: K.KeepPlan(t, [(pool, pool.clone())]), lambda: K.KeepPlan(t, [])):
        with pytest.raises(ECF8Error):
            call()


@pytest.mark.parametrize("name", "q out k_pool v_pool k_scale v_scale logits probabilities "
                         "temperature target accept sample draft".split())
def test_tensors_of_autograd_are_refused_by_name(name):
    """There is no backward, so no call may silently cut a graph."""
    from ecf8_amd import draft_kernels as K
    from ecf8_amd._lib import ECF8Error

    t = _on_host()
    bf = dict(dtype=torch.bfloat16)
    attend = dict(q=torch.zeros(6, 4, 128, **bf), out=torch.zeros(6, 512, **bf),
                  k_pool=torch.zeros(8, 2, 16, 128, **bf), v_pool=torch.zeros(8, 2, 16, 128, **bf),
                  k_scale=torch.ones(2), v_scale=torch.ones(2))
    verify = dict(target=torch.rand(6, 9), accept=torch.rand(6), sample=torch.rand(2),
                  draft=torch.rand(6, 9))
    probs = dict(logits=torch.zeros(6, 9, **bf), temperature=torch.ones(6), out=torch.zeros(6, 9))
    kw, call = ((attend, lambda **k: K.draft_attention(trees=t, **k)) if name in attend else
                (verify, lambda **k: K.draft_verify(t, torch.zeros(6, dtype=torch.int64), **k))
                if name in verify else (probs, lambda **k: K.token_probabilities(**k)))
    key = "out" if name == "probabilities" else name
    kw[key].requires_grad_()
    with pytest.raises(ECF8Error, match=f"{key} is followed by autograd"):
        call(**kw)
