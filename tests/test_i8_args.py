"""Refusals of the 8-bit and mixture-of-experts entry points, on the host: every
argument is checked before the library's state is, so nothing here needs a GPU
(the pointers are never followed)."""
from __future__ import annotations

import ctypes

import pytest

from webllm_b200 import jsep
from webllm_b200.build_ext import build

F32, F16, BF16 = jsep.GGML_TYPE_F32, jsep.GGML_TYPE_F16, jsep.GGML_TYPE_BF16
# addresses far apart, 256-byte aligned, never followed
A, B, C, D, E_, F = (0x10000000 * i for i in range(1, 7))


@pytest.fixture(scope="module", autouse=True)
def lib():
    build()
    return jsep.load_library()


def quantize(**kw):
    a = dict(x_type=F32, x_ptr=A, x_stride=64, N=4, K=64, q_ptr=B, q_stride=64, scale_ptr=C)
    return jsep.quantize_i8(**(a | kw))


def product(**kw):
    a = dict(w_ptr=A, w_row_bytes=64, w_scale_ptr=B, q_ptr=C, q_stride=64, q_scale_ptr=D, y_type=F32, y_ptr=E_,
             y_stride=32, M=32, K=64, N=4)
    return jsep.mul_mat_i8(**(a | kw))


def route(**kw):
    a = dict(logits_ptr=A, logits_stride=8, n_tokens=4, n_expert=8, n_used=2, score=jsep.MOE_SOFTMAX, normalize=True,
             scale=1.0, ids_ptr=B, weights_ptr=C)
    return jsep.moe_route(**(a | kw))


def plan(**kw):
    a = dict(ids_ptr=A, n_tokens=4, n_used=2, n_expert=8, offsets_ptr=B, order_ptr=C)
    return jsep.moe_plan(**(a | kw))


def grouped(**kw):
    a = dict(w_ptr=A, w_row_bytes=64, w_expert_bytes=64 * 32, w_scale_ptr=B, q_ptr=C, q_stride=64, q_scale_ptr=D,
             q_per_slot=False, offsets_ptr=E_, order_ptr=E_ + 4096, y_type=F32, y_ptr=F, y_stride=32, M=32, K=64,
             n_expert=8, n_tokens=4, n_used=2)
    return jsep.mul_mat_id_i8(**(a | kw))


def combine(**kw):
    a = dict(z_type=F32, z_ptr=A, z_stride=32, weights_ptr=B, y_type=F32, y_ptr=C, y_stride=32, n_tokens=4, n_used=2, M=32)
    return jsep.moe_combine(**(a | kw))


CASES = [
    (quantize, dict(x_type=jsep.GGML_TYPE_Q8_0), "x_type"),
    (quantize, dict(K=0), "K=0"),
    (quantize, dict(N=-1), "N=-1"),
    (quantize, dict(glu=3, up_ptr=D, up_stride=64), "glu kind"),
    (quantize, dict(glu=jsep.GLU_SWIGLU), "null"),
    (quantize, dict(glu=jsep.GLU_SWIGLU, up_ptr=D, up_stride=64, rms_norm=True), "glu and rms_norm"),
    (quantize, dict(rms_norm=True, eps=-1.0), "eps"),
    (quantize, dict(rms_norm=True, eps=float("nan")), "eps"),
    (quantize, dict(rms_norm=True, gain_ptr=D + 2), "aligned"),
    (quantize, dict(x_ptr=0), "null"),
    (quantize, dict(scale_ptr=0), "null"),
    (quantize, dict(x_ptr=A + 2), "aligned"),
    (quantize, dict(x_type=F16, x_ptr=A + 1), "aligned"),
    (quantize, dict(scale_ptr=C + 1), "aligned"),
    (quantize, dict(x_stride=-64), "x_stride"),
    (quantize, dict(q_stride=63), "q_stride"),
    (quantize, dict(q_ptr=A), "overlaps an input"),
    (quantize, dict(scale_ptr=A + 4 * 255), "overlaps an input"),
    (quantize, dict(scale_ptr=B + 252), "q overlaps scale"),
    (quantize, dict(rms_norm=True, gain_ptr=B), "overlaps an input"),
    (product, dict(y_type=jsep.GGML_TYPE_Q4_0), "y_type"),
    (product, dict(M=0), "M=0"),
    (product, dict(K=131072, w_row_bytes=131072, q_stride=131072), "int32 sum"),
    (product, dict(w_ptr=0), "null"),
    (product, dict(q_scale_ptr=0), "null"),
    (product, dict(w_scale_ptr=B + 1), "aligned"),
    (product, dict(y_ptr=E_ + 2), "aligned"),
    (product, dict(w_row_bytes=63), "w_row_bytes"),
    (product, dict(q_stride=63), "q_stride"),
    (product, dict(y_stride=31), "y_stride"),
    (product, dict(w_row_bytes=1 << 40), "w_row_bytes"),
    (product, dict(y_ptr=A + 64 * 31), "overlaps"),
    (product, dict(y_ptr=D), "overlaps"),
    (route, dict(logits_type=jsep.GGML_TYPE_Q8_0), "logits_type"),
    (route, dict(n_used=0), "n_used=0"),
    (route, dict(n_used=33, n_expert=64), "n_used=33"),
    (route, dict(n_used=9), "n_used=9 of"),
    (route, dict(n_expert=1025), "n_expert=1025"),
    (route, dict(n_tokens=-1), "n_tokens=-1"),
    (route, dict(n_tokens=1 << 30, n_used=2), "2^31"),
    (route, dict(score=2), "score"),
    (route, dict(ids_ptr=0), "null"),
    (route, dict(logits_ptr=A + 1), "aligned"),
    (route, dict(logits_stride=-8), "stride"),
    (route, dict(weights_ptr=B + 4), "overlap"),
    (route, dict(ids_ptr=A + 124), "overlap"),
    (plan, dict(n_expert=0), "n_expert=0"),
    (plan, dict(offsets_ptr=0), "null"),
    (plan, dict(order_ptr=0), "null"),
    (plan, dict(order_ptr=C + 2), "aligned"),
    (plan, dict(offsets_ptr=A + 28), "overlap"),
    (plan, dict(order_ptr=B + 32), "overlap"),
    (grouped, dict(y_type=99), "y_type"),
    (grouped, dict(K=0), "K=0"),
    (grouped, dict(K=131072, w_row_bytes=1 << 17, w_expert_bytes=1 << 22, q_stride=1 << 17), "int32 sum"),
    (grouped, dict(n_used=40), "n_used=40"),
    (grouped, dict(offsets_ptr=0), "null"),
    (grouped, dict(order_ptr=E_ + 4098), "aligned"),
    (grouped, dict(w_expert_bytes=64 * 31 + 63), "w_expert_bytes"),
    (grouped, dict(q_stride=63), "q_stride"),
    (grouped, dict(y_stride=31), "y_stride"),
    (grouped, dict(y_ptr=E_), "overlaps"),
    (grouped, dict(y_ptr=C), "overlaps"),
    (combine, dict(z_type=12), "types"),
    (combine, dict(y_type=12), "types"),
    (combine, dict(M=0), "M=0"),
    (combine, dict(n_used=33), "n_used=33"),
    (combine, dict(z_ptr=0), "null"),
    (combine, dict(y_ptr=C + 2), "aligned"),
    (combine, dict(y_stride=31), "y_stride"),
    (combine, dict(z_stride=-1), "z_stride"),
    (combine, dict(y_ptr=A + 4 * 32 * 7), "overlaps"),
]


@pytest.mark.parametrize("call,kw,why", CASES, ids=[f"{c.__name__}-{i}" for i, (c, _, _) in enumerate(CASES)])
def test_refused(call, kw, why):
    with pytest.raises(jsep.WllmError, match=why.replace("^", r"\^").replace("*", r"\*")):
        call(**kw)


def test_null_and_reserved_args(lib):
    for fn in (lib.wllm_quantize_i8, lib.wllm_mul_mat_i8, lib.wllm_mul_mat_id_i8):
        assert fn(None, None) == jsep.STATUS_FAILED
        assert "null args" in jsep.last_error()
    a = jsep.MulMatIdI8Args(32, 64, 8, 4, 2, 0, F32, 1, A, 64, 64 * 32, B, C, 64, D, E_, E_ + 4096, F, 32)
    assert lib.wllm_mul_mat_id_i8(ctypes.byref(a), None) == jsep.STATUS_FAILED
    assert "reserved" in jsep.last_error()


@pytest.mark.parametrize("call", [quantize, product, route, plan, grouped, combine])
def test_good_arguments_need_a_bound_library(call):
    """What is left to refuse a good call is the missing wllm_init (other tests of the session may have bound a GPU,
    where these addresses must not be followed: only an unbound library is asked)."""
    c = ctypes.c_void_p(0)
    if jsep.load_library().wllm_get_stream(ctypes.byref(c)) == jsep.STATUS_OK:
        pytest.skip("the library is bound to a GPU in this process")
    with pytest.raises(jsep.WllmError, match="wllm_init"):
        call()


def test_struct_sizes_match_the_header():
    """The ctypes structures and the header's are laid out alike (natural alignment, no packing)."""
    assert ctypes.sizeof(jsep.QuantizeI8Args) == 88
    assert ctypes.sizeof(jsep.MulMatI8Args) == 80
    assert ctypes.sizeof(jsep.MulMatIdI8Args) == 120
