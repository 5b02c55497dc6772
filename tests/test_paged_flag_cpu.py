"""Refusals of ecf8_ragged_attention_checked before any HIP call.  CPU only."""

from __future__ import annotations

import pytest
import torch

FAKE = 1 << 20  # never dereferenced: every call below is rejected first


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(starts=None), 1), (dict(n=0), 1), (dict(s=0), 1), (dict(hkv=0), 1),
    (dict(hq=9), 2), (dict(s=4097), 2), (dict(n=(1 << 18) + 1), 2), (dict(qs=1028), 2),
    (dict(os=1020), 2), (dict(k=FAKE + 8), 3), (dict(starts=FAKE + 2), 3), (dict(flag=FAKE + 2), 3)])
def test_checked_call_rejects_before_launch(kw, status):
    from ecf8_amd._lib import lib

    a = dict(q=FAKE, qs=1024, k=FAKE, ks=256, v=FAKE, vs=256, n=16, starts=FAKE, s=2, hq=8, hkv=2,
             out=FAKE, os=1024, flag=FAKE)
    a.update(kw)
    assert lib().ecf8_ragged_attention_checked(
        a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["n"], a["starts"], a["s"], a["hq"],
        a["hkv"], a["out"], a["os"], a["flag"], None) == status


def test_flags_of_other_kinds_are_refused():
    from ecf8_amd._lib import ECF8Error
    from ecf8_amd.head_kernels import _flag_ptr

    dev = torch.device("cuda", 0)
    assert _flag_ptr(None, dev) is None
    for flag in (torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(ECF8Error):
            _flag_ptr(flag, dev)
