"""GPU tests of the 8-bit products and the mixture-of-experts operators against
plain implementations in 64 bits.

Tolerances, with u = eps / 2 of a type (half a step, relative to the value):
 - quantize: none. The scale is one f32 division and q the nearest integer to an
   exact quotient; a float64 quotient of two f32 numbers cannot round across a
   half (v - h s is 0 or at least 2^-33 of v, where a float64 is off by 2^-53).
 - products: the sum is exact; acc -> f32, two f32 products and the rounding to
   y's type: 3 u(f32) + u(y), plus half a subnormal step of an f16 y.
 - router weights: expf (2 ulp = 4 u), its argument's subtraction (u times the
   argument, at most |l - max|), sums of at most 1024 of them, a division and a
   product: see `weight_tol`.
 - combine: k products and sums in f32 of given rows: (k + 1) u(f32) of
   sum |w z|, plus u(y).
"""
from __future__ import annotations

import os
import subprocess
import sys
import zlib

import numpy as np
import pytest

from oracle import oracle as O
from webllm_b200 import jsep, synth

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


@pytest.fixture(scope="module")
def rt(runtime):
    return runtime


def types(torch):
    return {"f32": (torch.float32, jsep.GGML_TYPE_F32), "f16": (torch.float16, jsep.GGML_TYPE_F16),
            "bf16": (torch.bfloat16, jsep.GGML_TYPE_BF16)}


def here(torch):
    return torch.cuda.current_stream().cuda_stream or jsep.STREAM_LEGACY


def up16(n):
    return (n + 15) // 16 * 16


def gen_of(torch, *key):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def ref_quantize(torch, v):
    """(q, s) of float64 rows whose values are f32 numbers."""
    a = v.abs().amax(1)
    s = (a / 127).to(torch.float32)
    sd = s.double()[:, None]
    q = torch.where(sd > 0, v / sd, torch.zeros_like(v)).round().clamp(-127, 127)
    bad = ~torch.isfinite(v).all(1)
    s[bad] = float("nan")
    q[bad] = 0
    return q.to(torch.int8), s


def quantize(torch, x, **kw):
    """q (rows padded to 16 bytes with a mark behind K) and scales of x through the library."""
    N, K = x.shape
    q = torch.full((N, up16(K)), 77, dtype=torch.int8, device="cuda")
    s = torch.full((N,), -1.0, device="cuda")
    t = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[x.dtype]
    jsep.quantize_i8(t, x.data_ptr(), x.stride(0), N, K, q.data_ptr(), q.stride(0), s.data_ptr(), stream=here(torch), **kw)
    torch.cuda.synchronize()
    assert (q[:, K:] == 77).all(), "bytes behind a row were written"
    return q, s


def weights8(torch, g, rows, K, pitch=None):
    w = torch.randint(-127, 128, (rows, pitch or up16(K)), dtype=torch.int8, device="cuda", generator=g)
    return w, torch.rand(rows, device="cuda", generator=g) * 0.01 + 1e-3


def close(torch, y, ref, extra=0.0):
    """y against a float64 reference within the products' tolerance; `extra`: an absolute part."""
    u = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[y.dtype]
    sub = 2.0 ** -25 if y.dtype == torch.float16 else 0.0
    tol = (3.01 * U32 + 1.001 * u) * ref.abs() + sub + extra
    off = (y.double() - ref).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((off - tol).max()):.3g}, first {bad.nonzero()[0].tolist()}"


# ---------------------------------------------------------------- quantiser


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,K", [(1, 1), (1, 7), (3, 64), (2, 255), (5, 1000), (1, 4096), (700, 333), (600, 4096), (2, 16384),
                                 (1, 16385), (3, 40001), (530, 20000), (700, 5), (1501, 1024), (3000, 2047), (513, 2064)])
def test_quantize(rt, torch, t, N, K):
    g = gen_of(torch, "quantize", t, N, K)
    x = (torch.randn(N, K, device="cuda", generator=g) * torch.rand(N, 1, device="cuda", generator=g) * 5).to(types(torch)[t][0])
    q, s = quantize(torch, x)
    rq, rs = ref_quantize(torch, x.double())
    assert torch.equal(s, rs)
    assert torch.equal(q[:, :K], rq)


def test_quantize_borders(rt, torch):
    """Quotients at and next to every half: multiples of s / 2 and their f32 neighbours."""
    for top in (127.0, 127.0 * 0.7853, 3.3e38, 1e-30):
        s = np.float32(np.float64(np.float32(top)) / 127)
        h = (np.arange(-254, 255, dtype=np.float64) * 0.5 * np.float64(s)).astype(np.float32)
        h = h[np.abs(h) <= np.float32(top)]
        row = np.concatenate([h, np.nextafter(h, np.float32(np.inf)), np.nextafter(h, np.float32(-np.inf)), [np.float32(top)]])
        row = row[np.abs(row) <= np.float32(top)].astype(np.float32)
        x = torch.from_numpy(row).cuda()[None]
        q, qs = quantize(torch, x)
        rq, rs = ref_quantize(torch, x.double())
        assert torch.equal(qs, rs)
        assert torch.equal(q[:, : len(row)], rq), top


def test_quantize_extremes(rt, torch):
    """Zero rows, the smallest and largest numbers, NaN and infinities: each row by its own rule."""
    K = 48
    rows = [torch.zeros(K), torch.full((K,), -0.0), torch.full((K,), 1e-45), torch.linspace(-1, 1, K) * 1e-40,
            torch.linspace(-1, 1, K) * 2.0 ** -126, torch.linspace(-1, 1, K) * 2.0 ** -100, torch.linspace(-1, 1, K) * 3.4028234e38]
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.linspace(-2, 3, K)
        r[17] = bad
        rows += [r, torch.full((K,), bad)]
    x = torch.stack(rows).cuda()
    q, s = quantize(torch, x)
    rq, rs = ref_quantize(torch, x.double())
    assert torch.equal(torch.nan_to_num(s, nan=-7.0), torch.nan_to_num(rs, nan=-7.0))
    assert torch.equal(q[:, :K], rq)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("off,extra", [(0, 0), (1, 0), (0, 3), (8, 8)])
def test_quantize_strides_and_alignment(rt, torch, t, off, extra):
    """Rows at odd offsets and strides, a zero stride (one row for all), q rows back to back; a CTA a row and a warp a row."""
    for N, K in ((9, 203), (601, 203)):
        quantize_strided(torch, t, off, extra, N, K)


def quantize_strided(torch, t, off, extra, N, K):
    g = gen_of(torch, "strides", t, off, extra, N)
    dt, tt = types(torch)[t]
    flat = torch.randn(off + N * (K + extra), device="cuda", generator=g).to(dt)
    x = flat[off:].view(N, K + extra)[:, :K]
    q = torch.zeros(N * K + 5, dtype=torch.int8, device="cuda")
    s = torch.zeros(N, device="cuda")
    for stride in (K + extra, 0):
        jsep.quantize_i8(tt, x.data_ptr(), stride, N, K, q.data_ptr(), K, s.data_ptr(), stream=here(torch))
        torch.cuda.synchronize()
        rq, rs = ref_quantize(torch, (x if stride else x[:1].expand(N, K)).double())
        assert torch.equal(q[: N * K].view(N, K), rq) and torch.equal(s, rs)
        assert (q[N * K :] == 0).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,K", [(1, 96), (3, 1000), (600, 333), (600, 2048), (2, 20000)])
def test_quantize_rms_norm(rt, torch, t, N, K):
    """|q - v / s| <= 1/2 and s = max|v| / 127, v off by eps: the sum of squares (at most 40 terms a thread at these
    sizes, then a tree of 10), a mean, a root, a reciprocal and two products: 64 u(f32)."""
    g = gen_of(torch, "rms", t, N, K)
    x = torch.randn(N, K, device="cuda", generator=g).to(types(torch)[t][0])
    for gain in (None, torch.rand(K, device="cuda", generator=g) + 0.5):
        q, s = quantize(torch, x, rms_norm=True, gain_ptr=0 if gain is None else gain.data_ptr(), eps=1e-5)
        xd = x.double()
        v = xd / (xd.square().mean(1, keepdim=True) + 1e-5).sqrt() * (1.0 if gain is None else gain.double())
        eps = 64 * U32
        assert ((s.double() * 127 / v.abs().amax(1) - 1).abs() <= eps + 2 * U32).all()
        assert ((q[:, :K].double() - v / s.double()[:, None]).abs() <= 0.5 + 127 * (eps + 2 * U32)).all()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", [jsep.GLU_SWIGLU, jsep.GLU_GELU])
@pytest.mark.parametrize("N,K", [(1, 72), (5, 1001), (600, 512), (600, 333), (520, 1500)])
def test_quantize_glu(rt, torch, t, kind, N, K):
    """act(g) u within eps |v| + tiny: __expf is off by 2 + 1.16 |g| ulp, |g| <= 20, the division by 2 ulp and the rest
    by 2: 30 ulp = 60 u(f32). GELU is an f16 number: at most one step (2^-10, or 2^-24 below the normals) beside."""
    g = gen_of(torch, "glu", t, kind, N, K)
    dt = types(torch)[t][0]
    both = (torch.randn(N, 2 * K, device="cuda", generator=g) * 3).clamp(-20, 20).to(dt)
    both[:, : K // 8] *= 2  # past +-10 too
    both[:, : K // 8].clamp_(-20, 20)
    gate, up = both[:, :K], both[:, K:]
    q, s = quantize(torch, gate, glu=kind, up_ptr=up.data_ptr(), up_stride=2 * K)
    a, u = gate.double(), up.double()
    eps = 60 * U32
    if kind == jsep.GLU_SWIGLU:
        v = a / (1 + (-a).exp()) * u
        tol = eps * v.abs()
    else:
        f = gate.float().half().double()
        v = 0.5 * f * (1 + torch.tanh(0.7978845608028654 * f * (1 + 0.044715 * f * f)))
        v = torch.where(a <= -10, torch.zeros_like(v), torch.where(a >= 10, a, v.half().double())) * u
        eps = eps + 2.0 ** -10
        tol = eps * v.abs() + 2.0 ** -24 * u.abs()
    top = (v.abs().amax(1), tol.amax(1))
    assert ((s.double() * 127 - top[0]).abs() <= top[1] + 2 * U32 * top[0]).all()
    sd = s.double()[:, None]
    assert ((q[:, :K].double() * sd - v).abs() <= 0.5 * sd + tol + 127 * sd * 2 * U32).all()


# ---------------------------------------------------------------- dense product


def run_product(torch, w, ws, q, qs, M, K, N, t="f32", y=None):
    dt, tt = types(torch)[t]
    if y is None:
        y = torch.full((N, M), float("nan"), dtype=dt, device="cuda")
    jsep.mul_mat_i8(w.data_ptr(), w.stride(0), ws.data_ptr(), q.data_ptr(), q.stride(0), qs.data_ptr(), tt, y.data_ptr(),
                    y.stride(0), M, K, N, stream=here(torch))
    torch.cuda.synchronize()
    return y


def ref_product(torch, w, ws, q, qs, K):
    return (q[:, :K].double() @ w[:, :K].double().t()) * qs.double()[:, None] * ws.double()[None]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,N", [
    (128, 128, 16),                                    # one tile, one chunk
    (1, 1, 1), (5, 17, 3), (128, 16, 1), (130, 144, 1),  # less than a tile and a chunk
    (256, 4096, 1), (300, 2000, 2), (64, 14336, 5),    # K split over a cluster
    (1000, 1000, 17), (257, 1152, 48), (129, 640, 64), (127, 640, 65),
    (512, 512, 250), (384, 777, 256), (200, 900, 257), (640, 1300, 700),  # several token tiles
    (20000, 256, 40), (2304, 9216, 33),                # more items than SMs
])
def test_product(rt, torch, t, M, K, N):
    g = gen_of(torch, "product", M, K, N)
    w, ws = weights8(torch, g, M, K)
    q, qs = weights8(torch, g, N, K)
    close(torch, run_product(torch, w, ws, q, qs, M, K, N, t), ref_product(torch, w, ws, q, qs, K))


def test_product_many_shapes(rt, torch):
    """Sizes drawn over the whole range, so that every mode, token tile and split of the kernel's plan comes up, with
    whole and ragged tiles, even and odd output strides."""
    rng = np.random.default_rng(5)
    for i in range(60):
        M, K, N = (int(np.exp(rng.uniform(np.log(lo), np.log(hi)))) for lo, hi in ((1, 3000), (1, 6000), (1, 1500)))
        g = gen_of(torch, "many", i)
        w, ws = weights8(torch, g, M, K)
        q, qs = weights8(torch, g, N, K)
        t = ("f32", "f16", "bf16")[i % 3]
        wide = torch.full((N, M + i % 4), 5.0, dtype=types(torch)[t][0], device="cuda")
        run_product(torch, w, ws, q, qs, M, K, N, t, y=wide[:, :M])
        close(torch, wide[:, :M], ref_product(torch, w, ws, q, qs, K))
        assert (wide[:, M:] == 5).all(), (M, K, N)


@pytest.mark.parametrize("M,K,N", [(200, 131071, 3), (130, 131071, 70)])
def test_product_largest_sums(rt, torch, M, K, N):
    """Every product at its largest: 131071 * 128 * 128 is the largest sum below 2^31."""
    w = torch.full((M, up16(K)), -128, dtype=torch.int8, device="cuda")
    q = torch.full((N, up16(K)), -128, dtype=torch.int8, device="cuda")
    q[N // 2] = 127
    ones = torch.ones(max(M, N), device="cuda")
    close(torch, run_product(torch, w, ones, q, ones, M, K, N), ref_product(torch, w, ones[:M], q, ones[:N], K))


@pytest.mark.parametrize("wp,qp,off", [(0, 0, 0), (3, 0, 0), (0, 5, 0), (13, 13, 1), (16, 32, 0)])
def test_product_strides_and_alignment(rt, torch, wp, qp, off):
    """Rows that are no multiples of 16 bytes apart, bases off by one, wider outputs that keep what is beside the rows."""
    M, K, N = 77, 211, 19
    g = gen_of(torch, "alignment", wp, qp, off)
    w = torch.randint(-127, 128, (off + M * (K + wp),), dtype=torch.int8, device="cuda", generator=g)[off:].view(M, -1)
    q = torch.randint(-127, 128, (off + N * (K + qp),), dtype=torch.int8, device="cuda", generator=g)[off:].view(N, -1)
    ws, qs = torch.rand(M, device="cuda", generator=g), torch.rand(N, device="cuda", generator=g)
    for t in ("f32", "bf16"):
        wide = torch.full((N, M + 3), 5.0, dtype=types(torch)[t][0], device="cuda")
        run_product(torch, w, ws, q, qs, M, K, N, t, y=wide[:, 1:])
        close(torch, wide[:, 1 : M + 1], ref_product(torch, w, ws, q, qs, K))
        assert (wide[:, 0] == 5).all() and (wide[:, M + 1 :] == 5).all()


def test_product_non_finite_scales(rt, torch):
    """A token row without a scale (NaN) is NaN in every channel; the others are untouched by it."""
    M, K, N = 200, 256, 20
    g = gen_of(torch, "nan")
    w, ws = weights8(torch, g, M, K)
    x = torch.randn(N, K, device="cuda", generator=g)
    x[3, 5], x[11, 0] = float("nan"), float("inf")
    x[7] = 0
    q, qs = quantize(torch, x)
    y = run_product(torch, w, ws, q, qs, M, K, N)
    assert torch.isnan(y[[3, 11]]).all() and (y[7] == 0).all()
    keep = [n for n in range(N) if n not in (3, 11)]
    close(torch, y[keep], ref_product(torch, w, ws, q[keep], qs[keep], K))


def test_product_far_offsets(rt, torch):
    """Weights past 2^32 bytes: the last channels come from far behind the base."""
    M, K, N = 300_000, 16384, 2
    g = gen_of(torch, "far")
    w = torch.randint(-127, 128, (M, K), dtype=torch.int8, device="cuda", generator=g)
    ws = torch.rand(M, device="cuda", generator=g)
    q, qs = weights8(torch, g, N, K)
    y = run_product(torch, w, ws, q, qs, M, K, N)
    for m in (0, M // 2, M - 257):
        close(torch, y[:, m : m + 257], ref_product(torch, w[m : m + 257], ws[m : m + 257], q, qs, K))


def test_no_rows(rt, torch):
    y = torch.ones(4, device="cuda")
    jsep.quantize_i8(0, 0, 64, 0, 64, 0, 64, 0, stream=here(torch))
    jsep.mul_mat_i8(0, 64, 0, 0, 64, 0, 0, y.data_ptr(), 32, 32, 64, 0, stream=here(torch))
    jsep.moe_route(0, 8, 0, 8, 2, jsep.MOE_SOFTMAX, True, 1.0, 0, 0, stream=here(torch))
    jsep.moe_combine(0, 0, 32, 0, 0, y.data_ptr(), 32, 0, 2, 32, stream=here(torch))
    offsets = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    jsep.moe_plan(0, 0, 2, 8, offsets.data_ptr(), 0, stream=here(torch))
    torch.cuda.synchronize()
    assert (y == 1).all() and (offsets == 0).all()


# ---------------------------------------------------------------- router and plan


def ref_route(torch, l, k, softmax, normalize, scale):
    """ids and weights of float64 logits, row by row on the host."""
    l = l.double().cpu()
    T, E = l.shape
    ids, w = torch.full((T, k), -1, dtype=torch.int32), torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        live = [e for e in range(E) if l[t, e] > -float("inf")]
        best = sorted(live, key=lambda e: (-float(l[t, e]), e))[:k]
        if not best:
            continue
        if softmax:
            top = float(l[t, best[0]])
            p = {e: 1.0 if float(l[t, e]) == top else float(np.exp(float(l[t, e]) - top)) for e in live}
            total = sum(p[e] for e in (best if normalize else live))
        else:
            p = {e: float(1 / (1 + np.exp(-min(max(float(l[t, e]), -700.0), 700.0)))) for e in live}
            total = sum(p[e] for e in best) if normalize else 1.0
        for j, e in enumerate(best):
            ids[t, j] = e
            w[t, j] = p[e] / total * scale
    return ids, w


def route(torch, l, k, score, normalize, scale=1.0):
    T, E = l.shape
    ids = torch.full((T, k), -9, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), -9.0, device="cuda")
    t = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[l.dtype]
    jsep.moe_route(l.data_ptr(), l.stride(0), T, E, k, score, normalize, scale, ids.data_ptr(), w.data_ptr(), logits_type=t,
                   stream=here(torch))
    torch.cuda.synchronize()
    return ids, w


def weight_tol(l, E):
    """Relative: two expf (4 u each) whose arguments are off by u |l - max| or u |l| (|l| <= 50 here: 100 u), a sum of
    E / 32 terms a lane and a tree of 5, a division, a product."""
    return (2 * 4 + 100 + E / 32 + 5 + 3) * U32


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", [jsep.MOE_SOFTMAX, jsep.MOE_SIGMOID])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (7, 60, 4), (33, 128, 8), (5, 200, 6), (3, 256, 1), (9, 1024, 32), (2, 32, 32)])
def test_route(rt, torch, t, score, normalize, T, E, k):
    g = gen_of(torch, "route", T, E, k)
    l = (torch.randn(T, E, device="cuda", generator=g) * 3).to(types(torch)[t][0])  # f16 and bf16 logits tie now and then
    ids, w = route(torch, l, k, score, normalize, 2.5)
    ri, rw = ref_route(torch, l, k, score == jsep.MOE_SOFTMAX, normalize, 2.5)
    assert torch.equal(ids.cpu(), ri)
    assert ((w.double().cpu() - rw).abs() <= weight_tol(l, E) * rw + 1e-37).all()


@pytest.mark.parametrize("score", [jsep.MOE_SOFTMAX, jsep.MOE_SIGMOID])
@pytest.mark.parametrize("normalize", [False, True])
def test_route_masks_and_ties(rt, torch, score, normalize):
    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 8, [-0.0, 0.0] * 4, [-inf] * 8, [nan] * 8, [nan, 1, -inf, 2, nan, 3, -inf, 0], [-inf, 5] + [-inf] * 6,
            [inf, 1, inf, 2, 3, inf, 0, 0], [inf] + [-inf] * 7, [-3.4028234e38] * 8, [3.4028234e38, -3.4028234e38, 1, 1, 2, 2, 3, 3],
            [-200.0] * 8, [1, 2, 3, 4, 4, 3, 2, 1], [nan, inf, -inf, 0, 0, 0, 0, 0]]
    l = torch.tensor(rows, device="cuda")
    ids, w = route(torch, l, 3, score, normalize)
    ri, rw = ref_route(torch, torch.where(torch.isnan(l), -inf, l), 3, score == jsep.MOE_SOFTMAX, normalize, 1.0)
    if score == jsep.MOE_SIGMOID and normalize:
        for r in (8, 10):  # every sigmoid is below the smallest f32: their sum is 0, and so are the weights
            rw[r] = 0
    assert torch.equal(ids.cpu(), ri)
    assert ((w.double().cpu() - rw).abs() <= weight_tol(l, 8) * rw + 1e-37).all()


def test_route_row_stride(rt, torch):
    l = torch.randn(6, 40, device="cuda", generator=gen_of(torch, "stride"))
    ids, w = route(torch, l[:, 3:23], 5, jsep.MOE_SOFTMAX, True)
    ri, _ = ref_route(torch, l[:, 3:23], 5, True, True, 1.0)
    assert torch.equal(ids.cpu(), ri)


def plan_of(torch, ids, E):
    T, k = ids.shape
    offsets = torch.full((E + 1,), -9, dtype=torch.int32, device="cuda")
    order = torch.full((T * k,), -9, dtype=torch.int32, device="cuda")
    jsep.moe_plan(ids.data_ptr(), T, k, E, offsets.data_ptr(), order.data_ptr(), stream=here(torch))
    torch.cuda.synchronize()
    return offsets, order


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 64), (3, 2, 5), (513, 3, 7), (511, 8, 128), (4096, 4, 60), (8192, 8, 128),
                                   (2049, 2, 1024), (40000, 2, 3), (8192, 8, 1024), (200000, 8, 300)])
def test_plan(rt, torch, T, k, E):
    g = gen_of(torch, "plan", T, k, E)
    ids = torch.randint(-2, E + 2, (T, k), dtype=torch.int32, device="cuda", generator=g)  # some outside 0..E-1
    offsets, order = plan_of(torch, ids, E)
    flat = ids.flatten().cpu().numpy().astype(np.int64)
    key = np.where((flat < 0) | (flat >= E), E, flat)
    assert np.array_equal(order.cpu().numpy(), np.argsort(key, kind="stable"))
    assert np.array_equal(offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]))


def test_plan_unaligned_ids(rt, torch):
    buf = torch.randint(0, 9, (1 + 777 * 2,), dtype=torch.int32, device="cuda", generator=gen_of(torch, "unaligned"))
    offsets, order = plan_of(torch, buf[1:].view(777, 2), 9)
    assert np.array_equal(order.cpu().numpy(), np.argsort(buf[1:].cpu().numpy(), kind="stable"))


# ---------------------------------------------------------------- grouped product and combine


def run_grouped(torch, w, ws, q, qs, per_slot, offsets, order, M, K, E, T, k, t="f32", y=None):
    dt, tt = types(torch)[t]
    if y is None:
        y = torch.full((T * k, M), float("nan"), dtype=dt, device="cuda")
    jsep.mul_mat_id_i8(w.data_ptr(), w.stride(1), w.stride(0), ws.data_ptr(), q.data_ptr(), q.stride(0), qs.data_ptr(), per_slot,
                       offsets.data_ptr(), order.data_ptr(), tt, y.data_ptr(), y.stride(0), M, K, E, T, k, stream=here(torch))
    torch.cuda.synchronize()
    return y


def ref_grouped(torch, w, ws, q, qs, per_slot, ids, K):
    T, k = ids.shape
    E, M = ws.shape
    y = torch.zeros(T * k, M, dtype=torch.float64, device="cuda")
    flat = ids.flatten()
    for e in range(E):
        at = (flat == e).nonzero().flatten()
        row = at if per_slot else at // k
        y[at] = ref_product(torch, w[e], ws[e], q[row], qs[row], K)
    return y


def spread(torch, g, T, k, E, how):
    """Expert ids: even, on few experts, on one, with slots that have none, or with the same expert twice in a token."""
    if how == "even":
        return torch.rand(T, E, device="cuda", generator=g).argsort(1)[:, :k].to(torch.int32).contiguous()
    if how == "few":
        return torch.randint(0, min(3, E), (T, k), dtype=torch.int32, device="cuda", generator=g)
    if how == "one":
        return torch.full((T, k), E - 1, dtype=torch.int32, device="cuda")
    if how == "none":
        return torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    return torch.randint(-2, E + 1, (T, k), dtype=torch.int32, device="cuda", generator=g)


@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("how", ["even", "few", "one", "none", "holes"])
@pytest.mark.parametrize("T,k,E,M,K", [(1, 1, 1, 5, 33), (1, 8, 64, 256, 1024), (2, 4, 8, 130, 700), (37, 4, 60, 300, 1152),
                                       (100, 2, 4, 257, 256), (700, 2, 8, 128, 384), (300, 8, 16, 384, 129)])
def test_grouped(rt, torch, per_slot, how, T, k, E, M, K):
    g = gen_of(torch, "grouped", how, T, k, E, M, K)
    w, ws = weights8(torch, g, E * M, K)
    w, ws = w.view(E, M, -1), ws.view(E, M)
    q, qs = weights8(torch, g, T * k if per_slot else T, K)
    ids = spread(torch, g, T, k, E, how)
    offsets, order = plan_of(torch, ids, E)
    ref = ref_grouped(torch, w, ws, q, qs, per_slot, ids, K)
    for t in ("f32", "bf16"):
        close(torch, run_grouped(torch, w, ws, q, qs, per_slot, offsets, order, M, K, E, T, k, t), ref)


def test_grouped_many_shapes(rt, torch):
    """Sizes and routings drawn over the whole range, skewed ones among them."""
    rng = np.random.default_rng(6)
    for i in range(40):
        T, M, K = (int(np.exp(rng.uniform(np.log(lo), np.log(hi)))) for lo, hi in ((1, 2000), (1, 1200), (1, 2000)))
        E = int(rng.integers(1, 40))
        k = int(rng.integers(1, min(E, 8) + 1))
        g = gen_of(torch, "grouped many", i)
        w, ws = weights8(torch, g, E * M, K)
        w, ws = w.view(E, M, -1), ws.view(E, M)
        per_slot = bool(i & 1)
        q, qs = weights8(torch, g, T * k if per_slot else T, K)
        like = torch.randn(E, device="cuda", generator=g) * (i % 5)  # how much some experts are liked
        ids = (torch.randn(T, E, device="cuda", generator=g) + like).topk(k, 1).indices.to(torch.int32)
        ids[torch.rand(T, k, device="cuda", generator=g) < 0.1 * (i % 3)] = -1
        offsets, order = plan_of(torch, ids, E)
        t = ("f32", "f16", "bf16")[i % 3]
        y = run_grouped(torch, w, ws, q, qs, per_slot, offsets, order, M, K, E, T, k, t)
        close(torch, y, ref_grouped(torch, w, ws, q, qs, per_slot, ids, K))


@pytest.mark.parametrize("pitch,gap", [(0, 0), (5, 0), (16, 64), (16, 8)])
def test_grouped_strides_and_alignment(rt, torch, pitch, gap):
    """Rows and experts apart, odd strides (CUDA cores), wider outputs that keep what is beside the rows."""
    T, k, E, M, K = 11, 3, 5, 70, 96
    g = gen_of(torch, "grouped strides", pitch, gap)
    flat = torch.randint(-127, 128, (E * (M * (K + pitch) + gap),), dtype=torch.int8, device="cuda", generator=g)
    w = flat.as_strided((E, M, K), (M * (K + pitch) + gap, K + pitch, 1))
    ws = torch.rand(E, M, device="cuda", generator=g)
    q, qs = weights8(torch, g, T, K)
    ids = spread(torch, g, T, k, E, "holes")
    offsets, order = plan_of(torch, ids, E)
    wide = torch.full((T * k, M + 5), 5.0, device="cuda")
    run_grouped(torch, w, ws, q, qs, False, offsets, order, M, K, E, T, k, y=wide[:, 2:])
    close(torch, wide[:, 2 : M + 2], ref_grouped(torch, w, ws, q, qs, False, ids, K))
    assert (wide[:, :2] == 5).all() and (wide[:, M + 2 :] == 5).all()


@pytest.mark.parametrize("zt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("yt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,k,M,off", [(1, 1, 1, 0), (1, 8, 4096, 0), (33, 3, 1001, 0), (5, 32, 64, 1), (70000, 1, 8, 0)])
def test_combine(rt, torch, zt, yt, T, k, M, off):
    g = gen_of(torch, "combine", zt, yt, T, k, M)
    (zd, zn), (yd, yn) = types(torch)[zt], types(torch)[yt]
    z = torch.randn(T * k, M + off, device="cuda", generator=g).to(zd)[:, off:]
    w = torch.rand(T, k, device="cuda", generator=g)
    y = torch.full((T, M), float("nan"), dtype=yd, device="cuda")
    jsep.moe_combine(zn, z.data_ptr(), M + off, w.data_ptr(), yn, y.data_ptr(), M, T, k, M, stream=here(torch))
    torch.cuda.synchronize()
    parts = z.double().reshape(T, k, M) * w.double()[:, :, None]
    close(torch, y, parts.sum(1), extra=(k + 1) * U32 * parts.abs().sum(1))


# ---------------------------------------------------------------- together


def moe_layer(torch, x, wr, up, up_s, down, down_s, k, bufs):
    """One mixture-of-experts block through the entry points, into `bufs` (one dict, so that it can be captured)."""
    T, K = x.shape
    E, M2 = up_s.shape
    F = M2 // 2
    st, P = here(torch), lambda n: bufs[n].data_ptr()
    torch.mm(x, wr, out=bufs["logits"])
    jsep.moe_route(P("logits"), E, T, E, k, jsep.MOE_SOFTMAX, True, 1.0, P("ids"), P("weights"), stream=st)
    jsep.moe_plan(P("ids"), T, k, E, P("offsets"), P("order"), stream=st)
    jsep.quantize_i8(0, x.data_ptr(), K, T, K, P("q"), K, P("s"), stream=st)
    jsep.mul_mat_id_i8(up.data_ptr(), K, M2 * K, up_s.data_ptr(), P("q"), K, P("s"), False, P("offsets"), P("order"), 0, P("h"), M2, M2, K,
                       E, T, k, stream=st)
    jsep.quantize_i8(0, P("h"), M2, T * k, F, P("hq"), F, P("hs"), glu=jsep.GLU_SWIGLU, up_ptr=P("h") + 4 * F, up_stride=M2, stream=st)
    jsep.mul_mat_id_i8(down.data_ptr(), F, K * F, down_s.data_ptr(), P("hq"), F, P("hs"), True, P("offsets"), P("order"), 0, P("z"), K, K, F,
                       E, T, k, stream=st)
    jsep.moe_combine(0, P("z"), K, P("weights"), 0, P("y"), K, T, k, K, stream=st)


def layer_bufs(torch, T, K, F, E, k):
    n = lambda *s, t=torch.float32: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    i8, i32 = torch.int8, torch.int32
    return {"logits": n(T, E), "ids": n(T, k, t=i32), "weights": n(T, k), "offsets": n(E + 1, t=i32), "order": n(T * k, t=i32),
            "q": n(T, K, t=i8), "s": n(T), "h": n(T * k, 2 * F), "hq": n(T * k, F, t=i8), "hs": n(T * k), "z": n(T * k, K), "y": n(T, K)}


@pytest.mark.parametrize("T", [1, 5, 300])
def test_moe_layer(rt, torch, T):
    """Router, plan, gate|up, SwiGLU, down and sum, each step against 64 bits on what the step before it gave."""
    K, F, E, k = 256, 192, 12, 3
    g = gen_of(torch, "layer", T)
    wr = torch.randn(K, E, device="cuda", generator=g) * 0.1
    up, ups = weights8(torch, g, E * 2 * F, K)
    dn, dns = weights8(torch, g, E * K, F)
    up, ups, dn, dns = up.view(E, 2 * F, K), ups.view(E, 2 * F), dn.view(E, K, F), dns.view(E, K)
    x = torch.randn(T, K, device="cuda", generator=g)
    b = layer_bufs(torch, T, K, F, E, k)
    moe_layer(torch, x, wr, up, ups, dn, dns, k, b)
    torch.cuda.synchronize()
    ri, rw = ref_route(torch, b["logits"], k, True, True, 1.0)
    assert torch.equal(b["ids"].cpu(), ri)
    rq, rs = ref_quantize(torch, x.double())
    assert torch.equal(b["q"], rq) and torch.equal(b["s"], rs)
    close(torch, b["h"], ref_grouped(torch, up, ups, b["q"], b["s"], False, b["ids"], K))
    gate, u = b["h"].double().chunk(2, 1)
    v = gate / (1 + (-gate).exp()) * u
    eps = (2 + 1.16 * gate.abs().amax() + 6) * 2 * U32
    assert ((b["hq"].double() * b["hs"].double()[:, None] - v).abs() <= 0.5 * b["hs"].double()[:, None] + eps * v.abs().amax(1, keepdim=True)).all()
    close(torch, b["z"], ref_grouped(torch, dn, dns, b["hq"], b["hs"], True, b["ids"], F))
    parts = b["z"].double().view(T, k, K) * b["weights"].double()[:, :, None]
    close(torch, b["y"], parts.sum(1), extra=(k + 1) * U32 * parts.abs().sum(1))


def test_captured_layers_share_nothing(rt, torch):
    """Two captured layers, replayed in turn and at once on two streams, after new inputs: what a fresh call gives."""
    K, F, E, k, T = 256, 128, 8, 2, 40
    g = gen_of(torch, "capture")
    runs = []
    for _ in range(2):
        up, ups = weights8(torch, g, E * 2 * F, K)
        dn, dns = weights8(torch, g, E * K, F)
        a = (torch.randn(T, K, device="cuda", generator=g), torch.randn(K, E, device="cuda", generator=g), up.view(E, 2 * F, K),
             ups.view(E, 2 * F), dn.view(E, K, F), dns.view(E, K), k)
        b = layer_bufs(torch, T, K, F, E, k)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            moe_layer(torch, *a, b)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            moe_layer(torch, *a, b)
        runs.append((a, b, graph, torch.cuda.Stream()))
    for _ in range(3):
        for a, b, _, _ in runs:
            a[0].copy_(torch.randn(T, K, device="cuda", generator=g))
            b["y"].fill_(float("nan"))
        torch.cuda.synchronize()
        for _, _, graph, side in runs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for a, b, _, _ in runs:
            fresh = layer_bufs(torch, T, K, F, E, k)
            moe_layer(torch, *a, fresh)
            torch.cuda.synchronize()
            assert torch.equal(fresh["y"], b["y"])


CAPTURED_FIRST = """
import torch
from webllm_b200 import jsep
jsep.install_jsep_callbacks(0)
T, K, E, k, M = 70, 256, 8, 2, 384
x = torch.randn(T, K, device="cuda")
w, t = torch.randint(-127, 128, (E, M, K), dtype=torch.int8, device="cuda"), torch.rand(E, M, device="cuda")
n = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")
ids, wt, of, od = n(T, k, t=torch.int32), n(T, k), n(E + 1, t=torch.int32), n(T * k, t=torch.int32)
q, s, y, z, d = n(T, K, t=torch.int8), n(T), n(T * k, M), n(T, M), n(T, M)
l = torch.randn(T, E, device="cuda")
def calls():
    st = torch.cuda.current_stream().cuda_stream or jsep.STREAM_LEGACY
    jsep.moe_route(l.data_ptr(), E, T, E, k, jsep.MOE_SOFTMAX, True, 1.0, ids.data_ptr(), wt.data_ptr(), stream=st)
    jsep.moe_plan(ids.data_ptr(), T, k, E, of.data_ptr(), od.data_ptr(), stream=st)
    jsep.quantize_i8(0, x.data_ptr(), K, T, K, q.data_ptr(), K, s.data_ptr(), stream=st)
    jsep.mul_mat_id_i8(w.data_ptr(), K, M * K, t.data_ptr(), q.data_ptr(), K, s.data_ptr(), False, of.data_ptr(), od.data_ptr(), 0,
                       y.data_ptr(), M, M, K, E, T, k, stream=st)
    jsep.moe_combine(0, y.data_ptr(), M, wt.data_ptr(), 0, z.data_ptr(), M, T, k, M, stream=st)
    jsep.mul_mat_i8(w.data_ptr(), K, t.data_ptr(), q.data_ptr(), K, s.data_ptr(), 0, d.data_ptr(), M, M, K, T, stream=st)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
z1, d1 = z.clone(), d.clone()
z.zero_(), d.zero_()
calls()
torch.cuda.synchronize()
assert z1.abs().sum() > 0 and torch.equal(z, z1) and torch.equal(d, d1)
print("captured first")
"""


def test_first_calls_may_be_captured():
    """In a new process the first calls of all are made while a stream is being captured."""
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout[-1500:] + r.stderr[-1500:]


def test_many_streams_at_once(rt, torch):
    """Different products at the same time on four streams, pairs and splits among them: each what it is alone."""
    shapes = [(512, 1024, 300), (3000, 512, 1), (256, 4096, 40), (1024, 2048, 130)]
    work = []
    for M, K, N in shapes:
        g = gen_of(torch, "streams", M)
        w, ws = weights8(torch, g, M, K)
        q, qs = weights8(torch, g, N, K)
        work.append((M, K, N, w, ws, q, qs, run_product(torch, w, ws, q, qs, M, K, N), torch.zeros(N, M, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(25):
        for M, K, N, w, ws, q, qs, _, y, st in work:
            jsep.mul_mat_i8(w.data_ptr(), w.stride(0), ws.data_ptr(), q.data_ptr(), q.stride(0), qs.data_ptr(), 0, y.data_ptr(), M, M, K, N,
                            stream=st.cuda_stream)
    torch.cuda.synchronize()
    for *_, alone, y, _ in work:
        assert torch.equal(alone, y)


def test_library_stream_and_its_graphs(rt, torch):
    """Stream 0 is the library's own, and its graph recorder takes the calls too."""
    M, K, N = 256, 1024, 3
    g = gen_of(torch, "own stream")
    w, ws = weights8(torch, g, M, K)
    x = torch.randn(N, K, device="cuda", generator=g)
    q, s = torch.empty(N, K, dtype=torch.int8, device="cuda"), torch.empty(N, device="cuda")
    y = torch.zeros(N, M, device="cuda")

    def calls():
        jsep.quantize_i8(0, x.data_ptr(), K, N, K, q.data_ptr(), K, s.data_ptr())
        jsep.mul_mat_i8(w.data_ptr(), K, ws.data_ptr(), q.data_ptr(), K, s.data_ptr(), 0, y.data_ptr(), M, M, K, N)

    torch.cuda.synchronize()
    k0 = rt.counters()["kernels_launched"]
    calls()
    rt.jsep_sync()
    assert rt.counters()["kernels_launched"] - k0 == 2
    first = y.clone()
    jsep.Graph.begin()
    calls()
    graph = jsep.Graph.end()
    y.zero_()
    torch.cuda.synchronize()
    k0 = rt.counters()["kernels_launched"]
    graph.launch()
    rt.jsep_sync()
    assert rt.counters()["kernels_launched"] - k0 == 2
    assert torch.equal(y, first)
    graph.destroy()
    close(torch, y, ref_product(torch, w, ws, q, s, K))


def test_gguf_weight_to_int8(rt, torch):
    """A GGUF weight becomes an int8 one with the same entry points: dequantize, then quantise its rows; the product is
    then within the two roundings to int8 of MUL_MAT over the blocks."""
    M, K, N = 192, 1024, 9
    g = gen_of(torch, "gguf")
    w = synth.weights_torch(g, O.TYPE_Q6_K, M, K, torch.device("cuda", 0))
    wf = torch.empty(M, K, device="cuda")
    jsep.dequantize_device(O.TYPE_Q6_K, w.data_ptr(), wf.data_ptr(), M * K, here(torch))
    torch.cuda.synchronize()
    wq, ws = quantize(torch, wf)
    x = torch.randn(N, K, device="cuda", generator=g)
    q, qs = quantize(torch, x)
    y = run_product(torch, wq, ws, q, qs, M, K, N)
    close(torch, y, ref_product(torch, wq, ws, q, qs, K))
    # |x' - x| <= s/2 and |w' - w| <= t/2, so a product is off by at most (s |w'| + t |x|) / 2
    bound = (qs.double()[:, None] * (wq.double() * ws.double()[:, None]).abs().sum(1)[None] + ws.double()[None] * x.double().abs().sum(1)[:, None]) / 2
    assert ((y.double() - x.double() @ wf.double().t()).abs() <= bound * 1.0001).all()
