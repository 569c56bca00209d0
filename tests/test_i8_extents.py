"""Refusals of the 8-bit and mixture-of-experts entry points at the ends of their 32-bit sizes, on the host (the pointers are
never followed)."""
from __future__ import annotations

import pytest

from test_i8_args import A, combine, grouped, plan, product, quantize, route
from webllm_b200 import jsep
from webllm_b200.build_ext import build


@pytest.fixture(scope="module", autouse=True)
def lib():
    build()
    return jsep.load_library()


HUGE = [
    (quantize, dict(K=2**31 - 1, x_stride=2**31, q_stride=2**31, q_ptr=A << 32, scale_ptr=A << 33), "K=2147483647"),
    (quantize, dict(K=2**31 - 1023, x_stride=2**31, q_stride=2**31, q_ptr=A << 32, scale_ptr=A << 33), "K=2147482625"),
    (quantize, dict(N=2**31 - 7, q_ptr=A << 32, scale_ptr=A << 33), "N=2147483641"),
    (product, dict(M=2**31 - 200, y_stride=2**31, w_scale_ptr=A << 16, y_ptr=A << 32), "M=2147483448"),
    (product, dict(N=2**31 - 1, q_scale_ptr=A << 16, y_ptr=A << 32), "N=2147483647"),
    (grouped, dict(M=2**31 - 200, y_stride=2**31, w_expert_bytes=1 << 38, w_scale_ptr=A << 16, y_ptr=A << 32), "M=2147483448"),
    (grouped, dict(n_tokens=2**31 - 1, n_used=1, y_ptr=A << 32), "2\\^31"),
    (route, dict(n_tokens=2**31 - 1, n_used=1, ids_ptr=A << 32, weights_ptr=A << 33), "2\\^31"),
    (plan, dict(n_tokens=2**30 - 1, n_used=2, offsets_ptr=A << 32, order_ptr=A << 33), "2\\^31"),
    (combine, dict(M=2**31 - 1, z_stride=2**31, y_stride=2**31, y_ptr=A << 32), "M=2147483647"),
]


@pytest.mark.parametrize("call,kw,why", HUGE, ids=[f"{c.__name__}-{i}" for i, (c, _, _) in enumerate(HUGE)])
def test_extents_next_to_2_31_are_refused(call, kw, why):
    """Where an index that goes past the last one would leave 32 bits."""
    with pytest.raises(jsep.WllmError, match=why):
        call(**kw)
