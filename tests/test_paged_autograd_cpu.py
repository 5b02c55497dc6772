"""The ragged-batch calls have no backward: every floating-point input that
autograd follows is refused, by name, before anything else.  CPU only."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

D = 128


def _calls():
    """(call of keyword arguments, its tensors) of each entry point."""
    from ecf8_amd import paged_kernels as P

    b = P.PagedBatch(2, 4, 8, 16, 64, 4, 2, "cpu")
    bf = dict(dtype=torch.bfloat16)
    q, out, pool = torch.zeros(4, 4, D, **bf), torch.zeros(4, 4 * D, **bf), torch.zeros(8, 2, 16, D, **bf)
    scales = dict(k_scale=torch.ones(2), v_scale=torch.ones(2))
    return {
        "write": (lambda **t: P.paged_qk_norm_rope(batch=b, eps=1e-6, cos_t=t.pop("cos"), sin_t=t.pop("sin"), **t),
                  dict(qkv=torch.zeros(4, 8 * D, **bf), q_norm=torch.ones(D, **bf),
                       k_norm=torch.ones(D, **bf), cos=torch.zeros(64, 64), sin=torch.zeros(64, 64),
                       q_out=q.clone(), k_pool=pool.clone(), v_pool=pool.clone(), **scales)),
        "attend": (lambda **t: P.paged_attention(batch=b, **t),
                   dict(q=q.clone(), out=out.clone(), k_pool=pool.clone(), v_pool=pool.clone(), **scales)),
        "prompt": (lambda **t: P.ragged_attention(starts=torch.zeros(3, dtype=torch.int32), **t),
                   dict(q=q.clone(), k=q[:, :2].clone(), v=q[:, :2].clone(), out=out.clone())),
    }


NAMES = [(c, n) for c, names in (
    ("write", "qkv q_norm k_norm cos sin q_out k_pool v_pool k_scale v_scale"),
    ("attend", "q out k_pool v_pool k_scale v_scale"), ("prompt", "q k v out")) for n in names.split()]


@pytest.mark.parametrize("call,name", NAMES)
def test_what_backward_follows_is_refused(call, name):
    from ecf8_amd._lib import ECF8Error

    run, tensors = _calls()[call]
    tensors[name].requires_grad_()
    with pytest.raises(ECF8Error, match=f"^{name} is followed by autograd"):
        run(**tensors)
    with torch.no_grad(), pytest.raises(ECF8Error) as e:  # (not on the GPU)
        run(**tensors)
    assert "autograd" not in str(e.value)


@pytest.mark.parametrize("call,name", NAMES)
def test_what_forward_mode_follows_is_refused(call, name):
    from ecf8_amd._lib import ECF8Error

    run, tensors = _calls()[call]
    with forward_ad.dual_level():
        with pytest.raises(ECF8Error) as e:
            run(**tensors)
        assert "autograd" not in str(e.value)
        tensors[name] = forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))
        with pytest.raises(ECF8Error, match=f"^{name} is followed by autograd"):
            run(**tensors)
