"""CPU-side checks of what the training operators refuse at the edges of fp32 and of their calls."""
import ctypes as C

import pytest

pytest.importorskip("torch")

from forward_b200 import capi, training as T  # noqa: E402


def _step(**kw):
    """Status of a step over no tensors: what its numbers are checked for."""
    c = T.AdamWConfig(1e-3, 0.9, 0.999, 1e-8, 1.0, 1, None, None, None, None)
    for k, v in kw.items():
        setattr(c, k, v)
    return T._lib().fwd_eb_adamw_step(None, 0, C.byref(c), None)


@pytest.mark.parametrize("kw", [
    dict(eps=1e-40), dict(eps=1e-60), dict(eps=2.0 ** -127), dict(eps=1e38), dict(eps=1e39),   # its reciprocal is not normal
    dict(lr=1e39), dict(grad_scale=-1e39),
])
def test_adamw_numbers_that_fp32_cannot_hold(kw):
    assert _step(**kw) == capi.EINVAL


@pytest.mark.parametrize("kw", [dict(eps=0.0), dict(eps=2.0 ** -126), dict(eps=2.0 ** 126), dict(lr=0.0), dict(lr=3e38),
                                dict(grad_scale=-3e38), dict(grad_scale=1e-40)])
def test_adamw_numbers_that_fp32_holds(kw):
    assert _step(**kw) == 0
