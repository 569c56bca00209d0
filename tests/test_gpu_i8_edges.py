"""GPU tests of the 8-bit and mixture-of-experts operators at the ends of what they accept, against plain implementations
in 64 bits."""
from __future__ import annotations

import os
import subprocess
import sys
import zlib

import pytest

from test_i8_plan import GROUPS, LONG, PRODUCTS
from webllm_b200 import jsep

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half a step of an f32, relative
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


@pytest.fixture(scope="module")
def rt(runtime):
    return runtime


def here(torch):
    return torch.cuda.current_stream().cuda_stream or jsep.STREAM_LEGACY


def up16(n):
    return (n + 15) // 16 * 16


def gen_of(torch, *key):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def quantize(torch, x, **kw):
    """q and scales of the rows of x through the library."""
    N, K = x.shape
    q = torch.full((N, up16(K)), 77, dtype=torch.int8, device="cuda")
    s = torch.full((N,), -1.0, device="cuda")
    t = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[x.dtype]
    jsep.quantize_i8(t, x.data_ptr(), x.stride(0), N, K, q.data_ptr(), q.stride(0), s.data_ptr(), stream=here(torch), **kw)
    torch.cuda.synchronize()
    assert (q[:, K:] == 77).all(), "bytes behind a row were written"
    return q[:, :K], s


def run_fresh(code, *args):
    """`code` in a new process, where no call has set a kernel's attributes yet."""
    r = subprocess.run([sys.executable, "-c", code, *map(str, args)], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as expected" in r.stdout, r.stdout[-1500:] + r.stderr[-1500:]


FIRST_PLAN = """
import sys
import numpy as np
import torch
from webllm_b200 import jsep
jsep.install_jsep_callbacks(0)
slots, E = map(int, sys.argv[1:])
ids = np.random.default_rng(slots).integers(-1, E + 1, (slots, 1), dtype=np.int32)
dev, offsets, order = torch.from_numpy(ids).cuda(), torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty(slots, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
jsep.moe_plan(dev.data_ptr(), slots, 1, E, offsets.data_ptr(), order.data_ptr(), stream=jsep.STREAM_LEGACY)
torch.cuda.synchronize()
key = np.where((ids < 0) | (ids >= E), E, ids).flatten().astype(np.int64)
assert np.array_equal(order.cpu().numpy(), np.argsort(key, kind="stable"))
assert np.array_equal(offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]))
print("as expected")
"""


@pytest.mark.parametrize("slots,E", [(2048, 360), (1408, 511), (1900, 383), (16384, 360)])
def test_first_plan_of_a_process(slots, E):
    """Sizes whose shared memory is within 48 KB only without what the kernel holds statically: as the first plan of a
    process (a larger one before it raises the kernel's limit for the rest)."""
    run_fresh(FIRST_PLAN, slots, E)


FIRST_PLAN_CAPTURED = FIRST_PLAN.replace("jsep.moe_plan(", """graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    jsep.moe_plan(""").replace("stream=jsep.STREAM_LEGACY)", "stream=torch.cuda.current_stream().cuda_stream)\ngraph.replay()")


@pytest.mark.parametrize("slots,E", [(65536, 128), (40000, 1024)])
def test_first_plan_of_a_process_is_captured(slots, E):
    """A plan of many CTAs, whose cluster size is looked up in the same call, while a stream is being captured."""
    run_fresh(FIRST_PLAN_CAPTURED, slots, E)


# ---------------------------------------------------------------- quantiser


@pytest.mark.parametrize("t", ["float32", "bfloat16"])
@pytest.mark.parametrize("N,K", [(1, 5), (3, 1001), (2, 20000), (600, 333), (700, 64)])
def test_rms_norm_of_any_finite_row(rt, torch, t, N, K):
    """Rows whose squares overflow an f32 or fall below its normals, among ordinary ones: x / sqrt(mean(x^2) + eps) is of
    order 1 for all of them. |q - v / s| <= 1/2 and s = max|v| / 127 with v off by eps: what test_quantize_rms_norm allows
    for f32 sums (64 u); the sums of these rows are doubles."""
    g = gen_of(torch, "far", t, N, K)
    eps = 64 * U32
    for e in (1e-5, 0.0):
        # by rows: ordinary, squares past the largest f32, and near the largest value; with eps = 0 tiny ones too
        sizes = [1.0, 1e20, 3e37, 1e30] + ([1e-21, 1e-25, 1e-37] if e == 0 else [])
        size = torch.tensor(sizes, device="cuda", dtype=torch.float64)[torch.arange(N, device="cuda") % len(sizes)]
        x = (torch.randn(N, K, device="cuda", generator=g).clamp(-4, 4).double() * size[:, None]).to(getattr(torch, t))
        for gain in (None, torch.rand(K, device="cuda", generator=g) + 0.5):
            q, s = quantize(torch, x, rms_norm=True, gain_ptr=0 if gain is None else gain.data_ptr(), eps=e)
            xd = x.double()
            v = xd / (xd.square().mean(1, keepdim=True) + e).sqrt() * (1.0 if gain is None else gain.double())
            assert ((s.double() * 127 / v.abs().amax(1) - 1).abs() <= eps + 2 * U32).all()
            assert ((q.double() - v / s.double()[:, None]).abs() <= 0.5 + 127 * (eps + 2 * U32)).all()


@pytest.mark.parametrize("size", [1.0, 1e25])
@pytest.mark.parametrize("N", [4, 604])
def test_rms_norm_of_rows_with_nan_or_infinity(rt, torch, N, size):
    """Such a row has scale NaN and q = 0; the rows beside it have theirs."""
    x = torch.randn(N, 300, device="cuda", generator=gen_of(torch, "bad", N)) * size
    alone = quantize(torch, x, rms_norm=True, eps=1e-6)
    x[1, 7], x[2, 299] = float("nan"), -float("inf")
    q, s = quantize(torch, x, rms_norm=True, eps=1e-6)
    assert torch.isnan(s[1:3]).all() and (q[1:3] == 0).all()
    keep = [n for n in range(N) if n not in (1, 2)]
    assert torch.equal(q[keep], alone[0][keep]) and torch.equal(s[keep], alone[1][keep]) and torch.isfinite(s[keep]).all()


@pytest.mark.parametrize("t", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("N,K", [(1, 8), (3, 1001), (2, 20000), (600, 333), (700, 64)])
def test_swiglu_of_gates_far_below_zero(rt, torch, t, off, N, K):
    """silu(g) u of rows whose gates all lie between -70 and -130: s = max|v| / 127 and |q - v / s| <= 1/2 with v off by eps.
    e^g by the SFU: its argument g log2(e) is off by u |g| log2(e), which is u |g| of the result, and each of at most four
    factors by 2 ulp = 4 u; five products and 1 + e^-g by u each: u (130 + 16 + 6), and what is below f32's normals by
    half a step of theirs (2^-150). s too may be below them: then it is off from a / 127 by up to 2^-150, and the value at
    q = 127, the largest, by 127 times that."""
    g = gen_of(torch, "deep", t, off, N, K)
    dt = getattr(torch, t)
    low = 60.0 * torch.rand(N, 1, device="cuda", generator=g)  # a row's gates within 8 of each other
    gate = (-70 - low - 8 * torch.rand(N, K + off, device="cuda", generator=g)).clamp(min=-130).to(dt)[:, off:]
    up = (torch.randn(N, K, device="cuda", generator=g) * (1e4 if t == "float16" else 1e30)).clamp(-6e4 if t == "float16" else -3e38, 6e4 if t == "float16" else 3e38).to(dt)
    x = gate.contiguous() if off == 0 else gate
    tt = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[dt]
    q, s = torch.zeros(N, K, dtype=torch.int8, device="cuda"), torch.zeros(N, device="cuda")
    jsep.quantize_i8(tt, x.data_ptr(), x.stride(0), N, K, q.data_ptr(), K, s.data_ptr(), glu=jsep.GLU_SWIGLU, up_ptr=up.data_ptr(), up_stride=K,
                     stream=here(torch))
    torch.cuda.synchronize()
    gd = gate.double()
    v = gd / (1 + (-gd).exp()) * up.double()
    eps, sub = (130 + 16 + 6) * U32, 2.0 ** -150
    top, sd = v.abs().amax(1), s.double()
    assert ((sd * 127 - top).abs() <= (eps + 2 * U32) * top + 4 * sub + 127 * sub).all()
    live = sd > 0
    assert (q[~live] == 0).all() and (top[~live] <= 127 * sub * 2).all()
    assert ((q.double() * sd[:, None] - v).abs() <= 0.5 * sd[:, None] + eps * v.abs() + 127 * sd[:, None] * 2 * U32 + (127 + 6) * sub).all()


# ---------------------------------------------------------------- router


@pytest.mark.parametrize("E,k", [(8, 3), (60, 8), (1024, 32)])
@pytest.mark.parametrize("normalize", [False, True])
def test_sigmoid_of_logits_far_below_zero(rt, torch, E, k, normalize):
    """Rows of logits about -60, -70, .. -103, where a sigmoid is e^l and, from -87 on, below f32's normals: the weights by the
    64-bit formula. e^l and e^(l - top) by expf (2 ulp = 4 u, their arguments off by at most u 104), a sum of at most 32 terms
    (5 steps), a quotient and a product, and half a subnormal step (2^-150) where the weight itself is so small; a
    normalised one's terms are e^(l - top), whose rounding is relative to 1."""
    g = gen_of(torch, "sigmoid", E, k)
    base = torch.tensor([-60.0, -63.9, -64.1, -70, -85, -87, -88, -89, -90, -95, -100, -101], device="cuda")[:, None]
    l = base - 2 * torch.rand(len(base), E, device="cuda", generator=g)
    ids, w = torch.empty(len(base), k, dtype=torch.int32, device="cuda"), torch.empty(len(base), k, device="cuda")
    jsep.moe_route(l.data_ptr(), E, len(base), E, k, jsep.MOE_SIGMOID, normalize, 1.0, ids.data_ptr(), w.data_ptr(), stream=here(torch))
    torch.cuda.synchronize()
    best = l.sort(dim=1, descending=True, stable=True)
    assert torch.equal(ids.long(), best.indices[:, :k])
    p = 1 / (1 + (-best.values[:, :k].double()).exp())
    ref = p / p.sum(1, keepdim=True) if normalize else p
    tol = (4 + 104 + 5 + 4 + 2) * U32 * ref * (2 if normalize else 1) + 2.0 ** -150
    assert ((w.double() - ref).abs() <= tol).all()


# ---------------------------------------------------------------- grouped product


def grouped(torch, w, ws, q, qs, per_slot, ids, M, K, t="float32"):
    """The grouped product of ids [T][k] through the library's plan, and that plan."""
    (T, k), E = ids.shape, ws.shape[0]
    offsets, order = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty(T * k, dtype=torch.int32, device="cuda")
    y = torch.full((T * k, M), float("nan"), dtype=getattr(torch, t), device="cuda")
    st = here(torch)
    jsep.moe_plan(ids.data_ptr(), T, k, E, offsets.data_ptr(), order.data_ptr(), stream=st)
    jsep.mul_mat_id_i8(w.data_ptr(), w.stride(1), w.stride(0), ws.data_ptr(), q.data_ptr(), q.stride(0), qs.data_ptr(), per_slot, offsets.data_ptr(),
                       order.data_ptr(), {"float32": 0, "float16": 1, "bfloat16": 30}[t], y.data_ptr(), M, M, K, E, T, k, stream=st)
    torch.cuda.synchronize()
    return y


def ref_grouped(torch, w, ws, q, qs, per_slot, ids, K):
    (T, k), flat = ids.shape, ids.flatten()
    y = torch.zeros(T * k, ws.shape[1], dtype=torch.float64, device="cuda")
    for e in flat.unique().tolist():
        if 0 <= e < ws.shape[0]:
            at = (flat == e).nonzero().flatten()
            row = at if per_slot else at // k
            y[at] = (q[row, :K].double() @ w[e, :, :K].double().t()) * qs[row].double()[:, None] * ws[e].double()
    return y


def close(torch, y, ref):
    """The sum is exact: acc -> f32, two f32 products and the rounding to y's type."""
    u = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[y.dtype]
    sub = 2.0 ** -25 if y.dtype == torch.float16 else 0.0
    bad = ~((y.double() - ref).abs() <= (3.01 * U32 + 1.001 * u) * ref.abs() + sub)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("per_slot", [False, True])
@pytest.mark.parametrize("K", [1, 15, 17, 127, 129, 130, 255, 257, 1000, 1535])
def test_grouped_rows_that_end_inside_a_piece(rt, torch, per_slot, K):
    """Every row's last 16 bytes partly behind K, the last row at the end of its buffer, with marks behind each row."""
    T, k, E, M = 61, 3, 7, 140
    g = gen_of(torch, "pieces", K, per_slot)
    pitch = up16(K)
    rows = T * k if per_slot else T
    w = torch.randint(-127, 128, (E, M, pitch), dtype=torch.int8, device="cuda", generator=g)
    ws, qs = torch.rand(E, M, device="cuda", generator=g), torch.rand(rows, device="cuda", generator=g)
    flat = torch.full(((rows - 1) * pitch + K,), 99, dtype=torch.int8, device="cuda")  # nothing behind the last row's K values
    q = flat.as_strided((rows, K), (pitch, 1))
    q.copy_(torch.randint(-127, 128, (rows, K), dtype=torch.int8, device="cuda", generator=g))
    ids = torch.randint(-1, E, (T, k), dtype=torch.int32, device="cuda", generator=g)
    close(torch, grouped(torch, w, ws, q, qs, per_slot, ids, M, K), ref_grouped(torch, w, ws, q, qs, per_slot, ids, K))


# ---------------------------------------------------------------- errors


def test_a_refused_launch_is_reported_once(rt, torch):
    """A launch that CUDA refuses (here: into a capture that something else has invalidated) fails its own call; the next
    wllm_sync does not fail for it too."""
    from cuda.bindings import runtime as cudart

    logits = torch.randn(2, 8, device="cuda")
    ids, w = torch.full((2, 2), -9, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, device="cuda")
    torch.cuda.synchronize()
    err, st = cudart.cudaStreamCreateWithFlags(cudart.cudaStreamNonBlocking)
    assert err == cudart.cudaError_t.cudaSuccess
    (err,) = cudart.cudaStreamBeginCapture(st, cudart.cudaStreamCaptureMode.cudaStreamCaptureModeThreadLocal)
    assert err == cudart.cudaError_t.cudaSuccess
    (err,) = cudart.cudaStreamSynchronize(st)  # not allowed in a capture: it is invalid from here on
    assert err != cudart.cudaError_t.cudaSuccess
    with pytest.raises(jsep.WllmError, match="wllm_moe_route"):
        jsep.moe_route(logits.data_ptr(), 8, 2, 8, 2, jsep.MOE_SOFTMAX, True, 1.0, ids.data_ptr(), w.data_ptr(), stream=int(st))
    cudart.cudaStreamEndCapture(st)
    cudart.cudaStreamDestroy(st)
    cudart.cudaGetLastError()
    rt.jsep_sync()
    jsep.moe_route(logits.data_ptr(), 8, 2, 8, 2, jsep.MOE_SOFTMAX, True, 1.0, ids.data_ptr(), w.data_ptr(), stream=here(torch))
    torch.cuda.synchronize()
    assert torch.equal(ids.long(), logits.topk(2, 1).indices)


# ---------------------------------------------------------------- every form of the products' kernel


def product(torch, w, ws, q, qs, M, K, N, t="float32"):
    y = torch.full((N, M), float("nan"), dtype=getattr(torch, t), device="cuda")
    jsep.mul_mat_i8(w.data_ptr(), w.stride(0), ws.data_ptr(), q.data_ptr(), q.stride(0), qs.data_ptr(), {"float32": 0, "float16": 1, "bfloat16": 30}[t],
                    y.data_ptr(), M, M, K, N, stream=here(torch))
    torch.cuda.synchronize()
    return y


def rows8(torch, g, *shape):
    """int8 rows of the last of `shape` values, padded to 16 bytes with values of their own, and scales."""
    q = torch.randint(-127, 128, (*shape[:-1], up16(shape[-1])), dtype=torch.int8, device="cuda", generator=g)
    return q, torch.rand(shape[:-1], device="cuda", generator=g) * 0.01 + 1e-3


@pytest.mark.parametrize("i", range(len(PRODUCTS)))
def test_product_of_every_mode(rt, torch, i):
    M, K, N = PRODUCTS[i][3:]
    g = gen_of(torch, "mode", i)
    (w, ws), (q, qs) = rows8(torch, g, M, K), rows8(torch, g, N, K)
    ref = (q[:, :K].double() @ w[:, :K].double().t()) * qs.double()[:, None] * ws.double()
    for t in ("float32", "float16", "bfloat16"):
        close(torch, product(torch, w, ws, q, qs, M, K, N, t), ref)


@pytest.mark.parametrize("how", ["even", "skewed", "holes"])
@pytest.mark.parametrize("i", range(len(GROUPS)))
def test_grouped_of_every_mode(rt, torch, i, how):
    """Routings that the plan, which counts on an even one, does not expect among them: most slots on one expert, and slots
    and experts without one another."""
    M, K, E, T, k = GROUPS[i][3:]
    g = gen_of(torch, "grouped mode", i, how)
    per_slot = bool(i & 1)
    (w, ws), (q, qs) = rows8(torch, g, E, M, K), rows8(torch, g, T * k if per_slot else T, K)
    if how == "even":
        ids = torch.rand(T, E, device="cuda", generator=g).argsort(1)[:, :k].to(torch.int32).contiguous()
    elif how == "skewed":
        ids = torch.where(torch.rand(T, k, device="cuda", generator=g) < 0.9, E - 1, 0).to(torch.int32)
    else:
        ids = torch.randint(-3, E + 2, (T, k), dtype=torch.int32, device="cuda", generator=g)
        ids[ids == E // 2] = -1
    ref = ref_grouped(torch, w, ws, q, qs, per_slot, ids, K)
    for t in ("float32", "bfloat16"):
        close(torch, grouped(torch, w, ws, q, qs, per_slot, ids, M, K, t), ref)


@pytest.mark.parametrize("how", ["even", "skewed", "holes", "none"])
@pytest.mark.parametrize("E", [575, 576, 577, 1000, 1024])
def test_grouped_of_many_experts(rt, torch, E, how):
    """More experts than the kernel has threads: its running sum over their tiles takes a second step."""
    M, K, T, k = 140, 200, 300, 5
    g = gen_of(torch, "many experts", E, how)
    (w, ws), (q, qs) = rows8(torch, g, E, M, K), rows8(torch, g, T, K)
    if how == "even":
        ids = torch.rand(T, E, device="cuda", generator=g).argsort(1)[:, :k].to(torch.int32).contiguous()
    elif how == "skewed":  # the last experts
        ids = (E - 1 - torch.randint(0, 4, (T, k), device="cuda", generator=g) ** 2).to(torch.int32)
    elif how == "holes":
        ids = torch.randint(-E, E, (T, k), dtype=torch.int32, device="cuda", generator=g)
    else:
        ids = torch.full((T, k), E, dtype=torch.int32, device="cuda")
    close(torch, grouped(torch, w, ws, q, qs, False, ids, M, K), ref_grouped(torch, w, ws, q, qs, False, ids, K))


# ---------------------------------------------------------------- far offsets


def test_grouped_weights_past_32_bits(rt, torch):
    """Experts whose weights begin past 2^32 bytes."""
    E, M, K, T, k = 140, 4096, 8192, 9, 3
    g = gen_of(torch, "far experts")
    (w, ws), (q, qs) = rows8(torch, g, E, M, K), rows8(torch, g, T, K)
    ids = torch.tensor([E - 1, E - 2, 0], dtype=torch.int32, device="cuda").repeat(T, 1)
    close(torch, grouped(torch, w, ws, q, qs, False, ids, M, K), ref_grouped(torch, w, ws, q, qs, False, ids, K))


def test_rows_past_2_31_elements(rt, torch):
    """Outputs of a dense and a grouped product, inputs of the quantiser and of the weighted sum whose last rows lie past
    2^31 elements (f16, so past 2^32 bytes too)."""
    N, M, K = 66000, 33000, 32
    g = gen_of(torch, "far rows")
    (w, ws), (q, qs) = rows8(torch, g, 2, M, K), rows8(torch, g, N, K)
    some = torch.cat([torch.arange(0, 3), torch.arange(N // 2, N // 2 + 3), torch.arange(N - 40, N)]).cuda()

    def ref(e):
        return (q[some, :K].double() @ w[e, :, :K].double().t()) * qs[some].double()[:, None] * ws[e].double()

    y = product(torch, w[0], ws[0], q, qs, M, K, N, "float16")
    close(torch, y[some], ref(0))
    ids = torch.ones(N, 1, dtype=torch.int32, device="cuda")
    del y
    y = grouped(torch, w, ws, q, qs, False, ids, M, K, "float16")
    close(torch, y[some], ref(1))
    # rows of y in pairs, weighted
    T, weights = N // 2, torch.rand(N // 2, 2, device="cuda", generator=g)
    z = torch.full((T, M), float("nan"), device="cuda")
    jsep.moe_combine(jsep.GGML_TYPE_F16, y.data_ptr(), M, weights.data_ptr(), 0, z.data_ptr(), M, T, 2, M, stream=here(torch))
    torch.cuda.synchronize()
    parts = y.view(T, 2, M)[-40:].double() * weights[-40:, :, None].double()
    off = (z[-40:].double() - parts.sum(1)).abs()
    assert (off <= 3 * U32 * parts.abs().sum(1)).all()  # two products and a sum
    del z, parts, off
    q8, s = quantize(torch, y)
    v = y[some].double()
    rs = (v.abs().amax(1) / 127).float()
    assert torch.equal(s[some], rs)
    assert torch.equal(q8[some], (v / rs.double()[:, None]).round().clamp(-127, 127).to(torch.int8))


# ---------------------------------------------------------------- rows that are not ordinary, in every form of the quantiser


@pytest.mark.parametrize("t", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("kind", [0, jsep.GLU_SWIGLU, jsep.GLU_GELU])
@pytest.mark.parametrize("N,K", [(13, 100), (13, 20003), (613, 100), (613, 1999)])
def test_quantize_rows_that_are_not_ordinary(rt, torch, t, kind, N, K):
    """NaN, infinities, zero, the smallest and the largest numbers in rows of their own among ordinary rows: a CTA and a warp
    a row, in whole vectors and behind them. The others come out as they do without."""
    g = gen_of(torch, "not ordinary", t, kind, N, K)
    dt = getattr(torch, t)
    top, low = torch.finfo(dt).max, torch.finfo(dt).tiny
    x = torch.randn(N, K, device="cuda", generator=g).to(dt)
    up = torch.randn(N, K, device="cuda", generator=g).to(dt)
    kw = dict(glu=kind, up_ptr=up.data_ptr(), up_stride=K) if kind else {}
    alone = quantize(torch, x, **kw)
    bad = {1: (0, float("nan")), 2: (K - 1, float("nan")), 3: (K // 2, float("inf")), 4: (K - 1, float("inf"))}
    for r, (k, v) in bad.items():
        x[r, k] = v
    x[5] = 0
    x[6] = -0.0
    x[7] = top
    x[8], up[8] = low, 1
    x[9], up[9] = 1, low
    if kind:
        up[10, K - 2] = float("nan")
        bad[10] = None
    q, s = quantize(torch, x, **kw)
    for r in bad:
        assert torch.isnan(s[r]) and (q[r] == 0).all(), r
    assert (s[5:7] == 0).all() and (q[5:7] == 0).all()
    rest = [n for n in range(N) if n not in (1, 2, 3, 4, 5, 6, 7, 8, 9, 10)]
    assert torch.equal(q[rest], alone[0][rest]) and torch.equal(s[rest], alone[1][rest])
    if not kind:
        for r in (7, 8, 9, 10):
            v = x[r].double()
            rs = (v.abs().amax() / 127).float()
            assert torch.equal(s[r], rs)
            assert torch.equal(q[r], (v / rs.double()).round().clamp(-127, 127).to(torch.int8))


# ---------------------------------------------------------------- waits that give up


@pytest.mark.parametrize("i", range(len(LONG)))
def test_a_wait_that_gives_up_is_reported(rt, torch, i):
    """With a limit of one poll (4 us) the epilogue of a long K, whose MMAs take 10 us and more, gives up, in every mode: the
    launch ends, the next wllm_sync says so, nothing is stored, and with the limit restored the same call gives what it gave
    before. Nothing stalls here: what the epilogue would not wait for is on its way, and the kernel ends after it."""
    M, K, E, N = LONG[i][2:]  # E = 0: dense
    g = gen_of(torch, "waits", i)
    (w, ws), (q, qs) = rows8(torch, g, max(E, 1), M, K), rows8(torch, g, N, K)
    offsets = (torch.arange(E + 1, device="cuda") * (N // max(E, 1))).to(torch.int32)
    order = torch.arange(N, dtype=torch.int32, device="cuda")
    y = torch.full((N, M), float("nan"), device="cuda")
    torch.cuda.synchronize()

    def call():  # on the library's stream, which wllm_sync waits for
        if E:
            jsep.mul_mat_id_i8(w.data_ptr(), w.stride(1), w.stride(0), ws.data_ptr(), q.data_ptr(), q.stride(0), qs.data_ptr(), False, offsets.data_ptr(),
                               order.data_ptr(), 0, y.data_ptr(), M, M, K, E, N, 1)
        else:
            jsep.mul_mat_i8(w.data_ptr(), w.stride(1), ws.data_ptr(), q.data_ptr(), q.stride(0), qs.data_ptr(), 0, y.data_ptr(), M, M, K, N)
        return jsep.load_library().wllm_sync()

    assert call() == jsep.STATUS_OK
    before = y.clone()
    assert not torch.isnan(before).any()
    y.fill_(float("nan"))
    torch.cuda.synchronize()
    try:
        jsep.set_wait_limit(1)
        rc = call()
    finally:
        jsep.set_wait_limit(0)
    msg = jsep.last_error()
    assert rc == jsep.STATUS_FAILED and "gave up waiting" in msg and "8-bit" in msg, msg
    assert int(msg.split("code 0x")[1].split(":")[0], 16) >> 24 & 2, msg  # an accumulator
    assert torch.isnan(y).all()
    assert call() == jsep.STATUS_OK
    assert torch.equal(y, before)
