// The mixture-of-experts operators around the grouped product: the router
// (wllm_moe_route), the slots sorted by expert (wllm_moe_plan) and the
// weighted sum over a token's slots (wllm_moe_combine).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "i8_plan.h"
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
// expert numbers that hold it, so ties go to the lowest expert. The weights
// are computed once, lane j the j-th's. Bound: launch latency for few tokens, the
// integer pipe for many (busy for 75 % of the time with the k walks over the keys;
// the logits are read once: 4 E bytes a token): 8192 tokens, 8 of 128 experts, 7.9
// us.
constexpr int kRouteWarps = 4;

template <typename T, int LANE>  // LANE: logits a lane holds, E <= 32 LANE
__global__ void __launch_bounds__(32 * kRouteWarps) route_kernel(const MoeRoute P) {
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + (threadIdx.x >> 5);
    if (t >= P.T) return;
    const T* row = static_cast<const T*>(P.logits) + t * P.stride;
    const float none = __uint_as_float(0xff800000u);
    float l[LANE];
    uint32_t key[LANE];
#pragma unroll
    for (int i = 0; i < LANE; ++i) {
        const int e = lane + 32 * i;
        l[i] = e < P.E ? to_f32(row[e]) : none;
    }
#pragma unroll
    for (int i = 0; i < LANE; ++i) {
        const uint32_t b = __float_as_uint(l[i] + 0.f);  // -0 and +0 are one value
        key[i] = !(l[i] > none) ? 0u : ((b & 0x80000000u) ? ~b : (b | 0x80000000u));
    }
    // lane j keeps the j-th choice
    int mine = -1;
    uint32_t mine_key = 0, first = 0;
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
        if (lane == j) mine = e, mine_key = most;
        if (j == 0) first = most;
    }
    auto value = [](uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); };
    const float top = value(first);
    // exp(l - top); a logit of +inf counts as 1 and every finite one as 0 then. A
    // sigmoid that is shared out among those of the chosen is exp(l - top) too where
    // all are so small that 1 + exp(l) is 1: exp(l) itself keeps few bits below -87.
    const bool shares = P.score == kMoeSoftmax || (P.normalize && top < -64.f);
    auto weight = [&](float v) {
        if (shares) return v == top ? 1.f : expf(v - top);
        const float e = expf(-fabsf(v));
        return (v < 0.f ? e : 1.f) / (1.f + e);
    };
    float w = mine >= 0 ? weight(value(mine_key)) : 0.f;
    if (P.normalize || P.score == kMoeSoftmax) {
        float sum = w;
        if (!P.normalize) {
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < LANE; ++i)
                if (l[i] > none) sum += weight(l[i]);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        // (0 where the chosen sigmoids are, and so their sum)
        w = sum > 0.f && (P.score == kMoeSoftmax || expf(top) > 0.f) ? w / sum : 0.f;
    }
    if (lane < P.k) {
        P.ids[t * P.k + lane] = mine;
        P.weights[t * P.k + lane] = w * P.scale;
    }
}

// ---------------------------------------------------------------- plan
//
// Slots in a stable order of their key, the expert (E for an id outside
// 0..E-1), without global atomics and without workspace: one cluster of up to 16
// CTAs, each warp with a run of consecutive slots. Every warp counts its run's
// keys in shared memory; the counts of the warps before it, of the CTAs before
// its own (distributed shared memory) and of the smaller keys give each key's
// first place, and a second walk over the run places the slots, lanes with equal
// keys in their order (they find each other with a ballot for each bit). Bound:
// latency (8 T k bytes are moved): 10 us for 65,536 slots and 128 experts, 4 for
// 8 slots; a CTA per expert that read all ids took 26, 8 CTAs 17.
constexpr int kPlanBatch = 8;   // ids a lane fetches at once

__device__ __forceinline__ int plan_key(const int32_t* ids, int64_t i, int64_t end, int E) {
    if (i >= end) return E + 1;  // no slot
    const int id = ids[i];
    return id < 0 || id >= E ? E : id;
}
// The lanes that hold the same key (of `bits` bits).
__device__ __forceinline__ uint32_t same_key(int key, int bits) {
    uint32_t same = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool set = (key >> b) & 1;
        const uint32_t lanes = __ballot_sync(0xffffffffu, set);
        same &= set ? lanes : ~lanes;
    }
    return same;
}

__global__ void __launch_bounds__(32 * kPlanWarps) plan_kernel(const int32_t* ids, int64_t n, int E, int32_t* offsets,
                                                               int32_t* order) {
    extern __shared__ int32_t plan_smem[];
    const int keys = E + 1, warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ctas = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
    int32_t* count = plan_smem;               // [warps][keys], then each warp's next place among the CTA's
    int32_t* total = count + warps * keys;    // [keys] of this CTA
    int32_t* first = total + keys;            // [keys] where this CTA's slots of a key begin
    __shared__ int32_t part[kPlanWarps];
    for (int i = threadIdx.x; i < warps * keys; i += blockDim.x) count[i] = 0;
    pdl_begin();
    const int bits = 32 - __clz(keys);  // of E + 1, the largest key
    const int64_t all_warps = static_cast<int64_t>(ctas) * warps;
    const int64_t run = (n + 32 * all_warps - 1) / (32 * all_warps) * 32;
    const int64_t begin = (static_cast<int64_t>(cta) * warps + warp) * run, end = min(begin + run, n);
    __syncthreads();
    int32_t* own = count + warp * keys;
    // every batch's ids are fetched together; a run of one batch keeps them for the second walk
    int key[kPlanBatch];
    auto fetch = [&](int64_t at) {
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) key[j] = plan_key(ids, at + 32 * j + lane, end, E);
    };
    for (int64_t at = begin; at < end; at += 32 * kPlanBatch) {
        fetch(at);
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) {
            if (at + 32 * j >= end) break;
            if (key[j] <= E) atomicAdd(&own[key[j]], 1);  // a count does not depend on the order
        }
    }
    __syncthreads();
    // counts of a key: exclusive over the warps (a lane each), and the CTA's total
    if (warps <= 4) {
        // few warps: a thread for each key
        for (int e = threadIdx.x; e < keys; e += blockDim.x) {
            int c[4], sum = 0;
#pragma unroll
            for (int w = 0; w < 4; ++w) c[w] = count[w * keys + e];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                count[w * keys + e] = sum;
                sum += c[w];
            }
            total[e] = sum;
        }
    } else {
        for (int e = warp; e < keys; e += warps) {
            const int c = lane < warps ? count[lane * keys + e] : 0;
            int sum = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            if (lane < warps) count[lane * keys + e] = sum - c;
            if (lane == 31) total[e] = sum;
        }
    }
    __syncthreads();
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    // a key's first place: smaller keys everywhere, then the CTAs before this one
    int carry = 0;
    for (int base = 0; base < keys; base += blockDim.x) {
        const int e = base + threadIdx.x;
        int everywhere = 0, before = 0;
        if (e < keys) {
            if (ctas == 1) {
                everywhere = total[e];
            } else {
                const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(total + e));
                int c[kPlanCtas];
#pragma unroll
                for (int r = 0; r < kPlanCtas; ++r) {
                    uint32_t remote;
                    c[r] = 0;
                    if (r >= ctas) continue;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(r));
                    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c[r]) : "r"(remote) : "memory");
                }
#pragma unroll
                for (int r = 0; r < kPlanCtas; ++r) {
                    everywhere += c[r];
                    if (r < cta) before += c[r];
                }
            }
        }
        int sum = everywhere;  // inclusive over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        if (base) __syncthreads();  // part of the step before has been read
        if (lane == 31) part[warp] = sum;
        __syncthreads();
        const int p = lane < warps ? part[lane] : 0;
        const int smaller = carry + sum - everywhere + __reduce_add_sync(0xffffffffu, lane < warp ? p : 0);
        carry += __reduce_add_sync(0xffffffffu, p);
        if (e < keys) {
            if (cta == 0) offsets[e] = smaller;
            first[e] = smaller + before;
        }
    }
    // no CTA ends while another reads its totals; what was read needs no order
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    __syncthreads();
    for (int64_t at = begin; at < end; at += 32 * kPlanBatch) {
        if (run > 32 * kPlanBatch) fetch(at);
#pragma unroll
        for (int j = 0; j < kPlanBatch; ++j) {
            if (at + 32 * j >= end) break;
            const uint32_t same = same_key(key[j], bits);
            const int place = key[j] <= E ? first[key[j]] + own[key[j]] + __popc(same & ((1u << lane) - 1)) : 0;
            __syncwarp();
            if (key[j] <= E) {
                order[place] = static_cast<int32_t>(at + 32 * j + lane);
                if (lane == __ffs(same) - 1) own[key[j]] += __popc(same);
            }
            __syncwarp();
        }
    }
    if (ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// ---------------------------------------------------------------- combine
//
// y[t][m] = sum_j weight[t][j] z[t k + j][m], in f32 and in the order of j (no
// atomics, so the sum does not depend on timing). Bound: HBM or L2, one read of
// the slots' rows; a thread takes 16 bytes of each: 4096 tokens, 8 f16 rows of
// 4096, 44 us, 6.9 TB/s (above what HBM copies at: part of it is still in L2).
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
    const int threads = static_cast<int>(std::min<int64_t>(vec ? 256 : 128, (lanes + 31) / 32 * 32));
    const dim3 grid(static_cast<unsigned>((lanes + threads - 1) / threads), std::min(o.T, 65535));
    return vec ? launch(combine_kernel<T, N>, grid, threads, stream, o) : launch(combine_kernel<T, 1>, grid, threads, stream, o);
}

}  // namespace

int launch_moe_route(const MoeRoute& o, cudaStream_t stream) {
    return o.type == kTypeF32 ? route<float>(o, stream) : (o.type == kTypeF16 ? route<__half>(o, stream) : route<__nv_bfloat16>(o, stream));
}

int launch_moe_plan(const int32_t* ids, int64_t slots, int E, int32_t* offsets, int32_t* order, cudaStream_t stream) {
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return -static_cast<int>(e);
    if (dev < 0 || dev >= kMaxDevices) return -static_cast<int>(cudaErrorInvalidDevice);
    // The kernel's attributes are per device, and set ahead of its first launch
    // whatever that one needs: static shared memory counts against the 48 KB that a
    // launch has without them, so the dynamic size alone does not tell.
    static int most_ctas[kMaxDevices] = {};
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    if (most_ctas[dev] == 0) {
        const int smem = plan_smem(kPlanWarps, kMaxExperts);
        cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return -static_cast<int>(e);
        // a partition of a GPU may have no 16 SMs that can form a cluster
        int clusters = 0;
        cfg.gridDim = dim3(kPlanCtas);
        cfg.blockDim = dim3(32 * kPlanWarps);
        cfg.dynamicSmemBytes = smem;
        attr[0].val.clusterDim.x = kPlanCtas;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&clusters, plan_kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            clusters = 0;
        }
        most_ctas[dev] = clusters > 0 ? kPlanCtas : kPortableCtas;
    }
    const PlanShape p = plan_shape(slots, E, most_ctas[dev]);
    cfg.gridDim = dim3(p.ctas);
    cfg.blockDim = dim3(32 * p.warps);
    cfg.dynamicSmemBytes = p.smem;
    attr[0].val.clusterDim.x = static_cast<unsigned>(p.ctas);
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, plan_kernel, ids, slots, E, offsets, order);
    return e == cudaSuccess ? 1 : -static_cast<int>(e);
}

int launch_moe_combine(const MoeCombine& o, cudaStream_t stream) {
    return o.z_type == kTypeF32 ? combine<float>(o, stream) : (o.z_type == kTypeF16 ? combine<__half>(o, stream) : combine<__nv_bfloat16>(o, stream));
}

}  // namespace wllm
