// The mixture-of-experts operators around the grouped product: the router
// (wllm_moe_route), the slots sorted by expert (wllm_moe_plan) and the
// weighted sum over a token's slots (wllm_moe_combine).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "wllm_internal.h"

namespace wllm {
namespace {

__device__ __forceinline__ void pdl_begin() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}

// ---------------------------------------------------------------- router
//
// One warp per token, E / 32 logits a lane in registers. A logit's key is its
// bits in an unsigned order (0 for NaN and -inf, which are never chosen); each
// of the k steps is one warp-wide maximum of the keys and one minimum of the
// expert numbers that hold it, so ties go to the lowest expert. Bound: launch
// latency for few tokens, the k dependent reductions for many (the logits are
// read once: 4 E bytes a token).
constexpr int kRouteWarps = 4;

template <typename T, int LANE>  // LANE: logits a lane holds, E <= 32 LANE
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const MoeRoute P) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
    if (t >= P.T) return;
    const T* row = static_cast<const T*>(P.logits) + t * P.stride;
    float l[LANE];
    uint32_t key[LANE];
#pragma unroll
    for (int i = 0; i < LANE; ++i) {
        const int e = lane + 32 * i;
        l[i] = e < P.E ? to_f32(row[e]) : __uint_as_float(0xff800000u);
    }
    float top = __uint_as_float(0xff800000u);
#pragma unroll
    for (int i = 0; i < LANE; ++i) {
        const uint32_t b = __float_as_uint(l[i] + 0.f);  // -0 and +0 are one value
        const bool masked = !(l[i] > __uint_as_float(0xff800000u));
        key[i] = masked ? 0u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
        if (!masked) top = fmaxf(top, l[i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // exp(l - top); a logit of +inf counts as 1 and every finite one as 0 then
    auto weight = [&](float v) {
        if (P.score == kMoeSigmoid) return 1.f / (1.f + expf(-v));
        return v == top ? 1.f : expf(v - top);
    };
    float all = 0.f;
    if (P.score == kMoeSoftmax && !P.normalize) {
#pragma unroll
        for (int i = 0; i < LANE; ++i)
            if (key[i]) all += weight(l[i]);
#pragma unroll
        for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    // lane j keeps the j-th choice
    int mine = -1;
    float w = 0.f;
    for (int j = 0; j < P.k; ++j) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < LANE; ++i)
            if (key[i] > best) best = key[i], at = i;
        const uint32_t most = __reduce_max_sync(0xffffffffu, best);
        if (most == 0) break;
        const int e = __reduce_min_sync(0xffffffffu, best == most ? lane + 32 * at : 0x7fffffff);
        if ((e & 31) == lane) {
#pragma unroll
            for (int i = 0; i < LANE; ++i)
                if (i == (e >> 5)) key[i] = 0;
        }
        if (lane == j) {
            mine = e;
            const uint32_t b = (most & 0x80000000u) ? (most & 0x7fffffffu) : ~most;
            w = weight(__uint_as_float(b));
        }
    }
    float sum = all;
    if (P.normalize) {
        sum = w;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane < P.k) {
        if (P.normalize || P.score == kMoeSoftmax) w = sum > 0.f ? w / sum : 0.f;
        P.ids[t * P.k + lane] = mine;
        P.weights[t * P.k + lane] = w * P.scale;
    }
}

// ---------------------------------------------------------------- plan
//
// Slots in a stable order of their expert, without atomics: CTA e counts the
// ids below e (its base) and places the slots of expert e behind it, in rising
// order; CTA E does so for the slots without an expert (an id outside 0..E-1).
// Every CTA reads all ids twice (from L2): 8 T k bytes, some microseconds up
// to 65,536 slots, and no step waits on another CTA.
constexpr int kPlanThreads = 512;
constexpr int kPlanIds = 8;  // consecutive ids of a thread and step

template <bool VEC>
__device__ __forceinline__ void load_ids(const int32_t* ids, int64_t i, int64_t n, int E, int (&v)[kPlanIds]) {
    if (VEC && i + kPlanIds <= n) {
        const int4 a = *reinterpret_cast<const int4*>(ids + i), b = *reinterpret_cast<const int4*>(ids + i + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < kPlanIds; ++j) v[j] = i + j < n ? ids[i + j] : 0x7fffffff;
    }
#pragma unroll
    for (int j = 0; j < kPlanIds; ++j) {
        if (i + j >= n) v[j] = E + 1;  // no slot
        else if (v[j] < 0 || v[j] >= E) v[j] = E;
    }
}

template <bool VEC>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const int32_t* ids, int64_t n, int E, int32_t* offsets,
                                                            int32_t* order) {
    __shared__ int part[2][kPlanThreads / 32];
    pdl_begin();
    const int e = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int warps = blockDim.x >> 5;
    const int64_t step = static_cast<int64_t>(blockDim.x) * kPlanIds;
    int below = 0;
    for (int64_t i = static_cast<int64_t>(threadIdx.x) * kPlanIds; i < n; i += step) {
        int v[kPlanIds];
        load_ids<VEC>(ids, i, n, E, v);
#pragma unroll
        for (int j = 0; j < kPlanIds; ++j) below += v[j] < e;
    }
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) part[0][warp] = below;
    __syncthreads();
    int base = __reduce_add_sync(0xffffffffu, lane < warps ? part[0][lane] : 0);
    if (threadIdx.x == 0) offsets[e] = base;
    int flip = 1;
    for (int64_t at = 0; at < n; at += step, flip ^= 1) {
        const int64_t i = at + static_cast<int64_t>(threadIdx.x) * kPlanIds;
        int v[kPlanIds];
        load_ids<VEC>(ids, i, n, E, v);
        int own = 0;
#pragma unroll
        for (int j = 0; j < kPlanIds; ++j) own += v[j] == e;
        int before = own;  // inclusive sum over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += u;
        }
        if (lane == 31) part[flip][warp] = before;
        __syncthreads();
        const int w = lane < warps ? part[flip][lane] : 0;
        int pos = base + before - own + __reduce_add_sync(0xffffffffu, lane < warp ? w : 0);
        base += __reduce_add_sync(0xffffffffu, w);
#pragma unroll
        for (int j = 0; j < kPlanIds; ++j)
            if (v[j] == e) order[pos++] = static_cast<int32_t>(i + j);
    }
}

// ---------------------------------------------------------------- combine
//
// y[t][m] = sum_j weight[t][j] z[t k + j][m], in f32 and in the order of j (no
// atomics, so the sum does not depend on timing). Bound: HBM or L2, one read of
// the slots' rows; a thread takes 16 bytes of each.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = to_f32(p[0]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

template <int N>
__device__ __forceinline__ void store_n(int type, void* base, int64_t at, const float (&v)[N]) {
    if (type == kTypeF32) {
        float* p = static_cast<float*>(base) + at;
        if constexpr (N == 1) p[0] = v[0];
        else
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        return;
    }
    uint16_t h[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        h[i] = type == kTypeF16 ? __half_as_ushort(__float2half_rn(v[i])) : __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
    uint16_t* p = static_cast<uint16_t*>(base) + at;
    if constexpr (N == 1) p[0] = h[0];
    else
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<uint2*>(p + i) = make_uint2(h[i] | (static_cast<uint32_t>(h[i + 1]) << 16),
                                                          h[i + 2] | (static_cast<uint32_t>(h[i + 3]) << 16));
}

template <typename T, int N>
__global__ void __launch_bounds__(256) combine_kernel(const MoeCombine P) {
    pdl_begin();
    const int64_t m = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * N;
    if (m >= P.M) return;
    for (int64_t t = blockIdx.y; t < P.T; t += gridDim.y) {
        const T* z = static_cast<const T*>(P.z) + t * P.k * P.z_stride + m;
        const float* w = P.weights + t * P.k;
        float sum[N];
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = 0.f;
#pragma unroll 8
        for (int j = 0; j < P.k; ++j) {
            float v[N];
            load_n<T, N>(z + j * P.z_stride, v);
            const float f = w[j];
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] = fmaf(f, v[i], sum[i]);
        }
        store_n<N>(P.y_type, P.y, t * P.y_stride + m, sum);
    }
}

template <typename... A>
int launch(void (*kernel)(A...), dim3 grid, int threads, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess ? 1 : -static_cast<int>(e);
}

template <typename T>
int route(const MoeRoute& o, cudaStream_t stream) {
    const dim3 grid((o.T + kRouteWarps - 1) / kRouteWarps);
    const int threads = o.T == 1 ? 32 : 32 * kRouteWarps;
    if (o.E <= 64) return launch(route_kernel<T, 2>, grid, threads, stream, o);
    if (o.E <= 128) return launch(route_kernel<T, 4>, grid, threads, stream, o);
    if (o.E <= 256) return launch(route_kernel<T, 8>, grid, threads, stream, o);
    return launch(route_kernel<T, 32>, grid, threads, stream, o);
}

template <typename T>
int combine(const MoeCombine& o, cudaStream_t stream) {
    constexpr int N = 16 / sizeof(T);
    const int ysize = o.y_type == kTypeF32 ? 4 : 2;
    const uintptr_t zb = reinterpret_cast<uintptr_t>(o.z) | static_cast<uintptr_t>(o.z_stride * sizeof(T));
    const uintptr_t yb = reinterpret_cast<uintptr_t>(o.y) | static_cast<uintptr_t>(o.y_stride * ysize);
    const bool vec = o.M % N == 0 && ((zb | yb) & 15) == 0;
    const int64_t lanes = vec ? o.M / N : o.M;
    const int threads = static_cast<int>(std::min<int64_t>(256, (lanes + 31) / 32 * 32));
    const dim3 grid(static_cast<unsigned>((lanes + threads - 1) / threads), std::min(o.T, 65535));
    return vec ? launch(combine_kernel<T, N>, grid, threads, stream, o) : launch(combine_kernel<T, 1>, grid, threads, stream, o);
}

}  // namespace

int launch_moe_route(const MoeRoute& o, cudaStream_t stream) {
    return o.type == kTypeF32 ? route<float>(o, stream) : (o.type == kTypeF16 ? route<__half>(o, stream) : route<__nv_bfloat16>(o, stream));
}

int launch_moe_plan(const int32_t* ids, int64_t slots, int E, int32_t* offsets, int32_t* order, cudaStream_t stream) {
    const bool vec = (reinterpret_cast<uintptr_t>(ids) & 15) == 0;
    const int threads = static_cast<int>(std::min<int64_t>(kPlanThreads, (std::max<int64_t>(slots, 1) + kPlanIds * 32 - 1) / (kPlanIds * 32) * 32));
    return launch(vec ? plan_kernel<true> : plan_kernel<false>, dim3(E + 1), threads, stream, ids, slots, E, offsets, order);
}

int launch_moe_combine(const MoeCombine& o, cudaStream_t stream) {
    return o.z_type == kTypeF32 ? combine<float>(o, stream) : (o.z_type == kTypeF16 ? combine<__half>(o, stream) : combine<__nv_bfloat16>(o, stream));
}

}  // namespace wllm
