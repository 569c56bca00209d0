// Row quantiser of the 8-bit products (wllm_quantize_i8): N rows of K values
// become int8 with one scale each.
//
//   a = max_k |v_k|     s = fl(a / 127)     q_k = nearest integer to v_k / s
//
// v is the row itself, RMS_NORM(x) * gain, or act(gate) * up. Ties go to the
// even integer and the quotient is the exact one, so q does not depend on how
// a division is rounded: t = v * (1/s) is within 127 * 2^-22 of the quotient,
// so only a t within 1/10000 of a half can round to the wrong integer, and
// there the remainder r = v - q s decides (one FMA; where 2|r| is near s it
// has at most 24 bits, so it is exact, and FMA's rounding is monotone
// elsewhere). A row whose a is below 2^-100, where 1/s could overflow, or
// s be rounded to a few bits, takes double quotients, clamped to +-127.
// A row that holds a NaN or an infinity has no scale: s = NaN and q = 0, so
// every product of it is NaN.
//
// Bound: HBM (one read of the row, K + 4 bytes written). One CTA per row; the
// row's values stay in registers (32 a thread) between the maximum and the
// rounding, so rows up to 32 * 512 values are read once; longer rows are read
// again (from L2) in the second pass.
// Threads: rows that are few take one 8-value vector a thread (latency), many
// rows four (fewer barriers a byte).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "wllm_internal.h"

namespace wllm {
namespace {

constexpr int kVec = 8;    // values of a thread's vector
constexpr int kKeep = 4;   // vectors a thread keeps in registers
constexpr int kMaxThreads = 512;
constexpr int kFewRows = 512;  // at most this many rows: one vector a thread

// A thread's vector of 8 values as it lies in memory.
template <typename T>
struct Raw {
    static constexpr int kWords = kVec * sizeof(T) / 4;
    uint32_t w[kWords];
};

template <typename T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float (&v)[kVec]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = __uint_as_float(r.w[j]);
    } else {
#pragma unroll
        for (int i = 0; i < kVec / 2; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(r.w[i] << 16), v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
            }
        }
    }
}

// Values [8 i, 8 i + 8) of a row, zeros behind its end. VEC: the row starts on
// a 16-byte boundary.
template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> load_part(const T* row, int i, int K) {
    Raw<T> r;
    if (VEC && (i + 1) * kVec <= K) {
        const uint4* p = reinterpret_cast<const uint4*>(row + static_cast<int64_t>(i) * kVec);
#pragma unroll
        for (int h = 0; h < Raw<T>::kWords / 4; ++h) {
            const uint4 a = p[h];
            r.w[4 * h] = a.x, r.w[4 * h + 1] = a.y, r.w[4 * h + 2] = a.z, r.w[4 * h + 3] = a.w;
        }
    } else {
        using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
        const U* p = reinterpret_cast<const U*>(row);
#pragma unroll
        for (int h = 0; h < Raw<T>::kWords; ++h) {
            r.w[h] = 0;
#pragma unroll
            for (int j = 0; j < 4 / static_cast<int>(sizeof(T)); ++j) {
                const int k = i * kVec + h * (4 / static_cast<int>(sizeof(T))) + j;
                if (k < K) r.w[h] |= static_cast<uint32_t>(p[k]) << (16 * j);
            }
        }
    }
    return r;
}

// The largest |value| of vectors so far. The bits of |v| order like its value,
// with NaN above infinity; 16-bit types are compared two at a time.
template <typename T>
__device__ __forceinline__ uint32_t max_raw(uint32_t top, const Raw<T>& r) {
#pragma unroll
    for (int h = 0; h < Raw<T>::kWords; ++h) {
        if constexpr (sizeof(T) == 4) top = max(top, r.w[h] & 0x7fffffffu);
        else top = __vmaxu2(top, r.w[h] & 0x7fff7fffu);
    }
    return top;
}
// Its bits as an f32's.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t top) {
    if constexpr (sizeof(T) == 4) return top;
    const uint32_t h = max(top & 0xffffu, top >> 16);
    if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(h))));
    return h << 16;
}

// silu(g) * u and gelu(g) * u, as wllm_mul_mat_glu_batch computes them
__device__ __forceinline__ float x_sigmoid(float x, float z) { return __fdividef(x, 1.f + __expf(-z)); }
__device__ __forceinline__ float glu(int kind, float g, float u) {
    if (kind == kProSwiglu) return __fmul_rn(x_sigmoid(g, g), u);
    float y;
    if (g <= -10.f) {
        y = 0.f;
    } else if (g >= 10.f) {
        y = g;
    } else {
        const float f = __half2float(__float2half_rn(g));
        const float s = (0.7978845608028654f * f) * (1.f + (0.044715f * f) * f);
        y = __half2float(__float2half_rn(x_sigmoid(f, 2.f * s)));
    }
    return __fmul_rn(y, u);
}

// Block-wide maximum (of bits) and sum; `part` holds one word per warp.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* part) {
    v = __reduce_max_sync(0xffffffffu, v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0u);
}
__device__ __forceinline__ float block_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The nearest integer to v / s where t = v * (1/s) is too near a half to tell.
__device__ __forceinline__ float settle(float v, float s, float q) {
    const float r = 2.f * fmaf(-q, s, v);
    const bool odd = static_cast<int>(q) & 1;
    if (r > s || (r == s && odd)) return q + 1.f;
    if (r < -s || (r == -s && odd)) return q - 1.f;
    return q;
}
// The same in a row of tiny values.
__device__ __noinline__ float settle_tiny(float v, float s) {
    return s > 0.f ? static_cast<float>(fmin(fmax(rint(static_cast<double>(v) / s), -127.0), 127.0)) : 0.f;
}

// Eight int8 of a vector.
__device__ __forceinline__ uint2 quantize8(const float (&v)[kVec], float s, float inv, bool tiny) {
    constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: adding it rounds to the nearest integer (ties to even)
    float m[kVec];
    float worst = 0.f;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        const float t = v[j] * inv;
        m[j] = __fadd_rn(t, kMagic);
        worst = fmaxf(worst, fabsf(t - (m[j] - kMagic)));
    }
    if (worst > 0.4999f) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) m[j] = settle(v[j], s, m[j] - kMagic) + kMagic;
    }
    if (tiny) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) m[j] = settle_tiny(v[j], s) + kMagic;
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t a = __byte_perm(__float_as_uint(m[4 * h]), __float_as_uint(m[4 * h + 1]), 0x0040);
        const uint32_t b = __byte_perm(__float_as_uint(m[4 * h + 2]), __float_as_uint(m[4 * h + 3]), 0x0040);
        w[h] = __byte_perm(a, b, 0x5410);
    }
    return make_uint2(w[0], w[1]);
}

// PRO: kProNone, kProNorm, or kProSwiglu for both GLU kinds (P.kind tells).
// Without a prologue the kept vectors stay as they were loaded (16 registers
// of a 16-bit type), so three CTAs of 512 threads fit an SM (two of f32 or with
// a prologue): at one CTA the loads of the next row do not overlap the rounding
// of this one (8192 x 14336 bf16: 223 us against 62).
template <typename T, bool VEC, int PRO>
__global__ void __launch_bounds__(kMaxThreads, PRO == kProNone && sizeof(T) == 2 ? 3 : 2) quantize_i8_kernel(const QuantizeI8 P) {
    __shared__ uint32_t part_max[kMaxThreads / 32];
    __shared__ float part_sum[kMaxThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t r = blockIdx.x;
    const T* x = static_cast<const T*>(P.x) + r * P.x_stride;
    const int K = P.K, parts = (K + kVec - 1) / kVec;
    const int step = blockDim.x;
    float rms = 1.f;
    uint32_t top = 0;

    // s, 1/s and the stores are the same for every prologue
    float s = 0.f, inv = 0.f;
    bool bad = false, tiny = false;
    auto set_scale = [&]() {
        top = block_max(top, part_max);
        bad = top >= 0x7f800000u;
        const float a = __uint_as_float(top);
        s = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a, 127.f);
        tiny = a < 0x1p-100f;
        inv = bad || tiny ? 0.f : __fdiv_rn(1.f, s);
        if (threadIdx.x == 0) P.scale[r] = s;
    };
    int8_t* q = P.q + r * P.q_stride;
    const bool wide = ((reinterpret_cast<uintptr_t>(P.q) | static_cast<uintptr_t>(P.q_stride)) & 7) == 0;
    auto store = [&](int i, float (&v)[kVec]) {
        uint2 w = quantize8(v, s, inv, tiny);
        if (bad) w = make_uint2(0, 0);
        if (wide && (i + 1) * kVec <= K) {
            *reinterpret_cast<uint2*>(q + static_cast<int64_t>(i) * kVec) = w;
        } else {
            const uint64_t b = (static_cast<uint64_t>(w.y) << 32) | w.x;
            for (int j = 0; j < kVec && i * kVec + j < K; ++j) q[i * kVec + j] = static_cast<int8_t>(b >> (8 * j));
        }
    };

    if constexpr (PRO == kProNone) {
        Raw<T> keep[kKeep];
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            const int i = threadIdx.x + c * step;
            if (i < parts) keep[c] = load_part<T, VEC>(x, i, K);
            else
#pragma unroll
                for (int h = 0; h < Raw<T>::kWords; ++h) keep[c].w[h] = 0;
        }
#pragma unroll
        for (int c = 0; c < kKeep; ++c) top = max_raw<T>(top, keep[c]);
        for (int i = threadIdx.x + kKeep * step; i < parts; i += step) top = max_raw<T>(top, load_part<T, VEC>(x, i, K));
        top = top_bits<T>(top);
        set_scale();
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            const int i = threadIdx.x + c * step;
            if (i < parts) {
                float v[kVec];
                unpack<T>(keep[c], v);
                store(i, v);
            }
        }
        for (int i = threadIdx.x + kKeep * step; i < parts; i += step) {
            float v[kVec];
            unpack<T>(load_part<T, VEC>(x, i, K), v);
            store(i, v);
        }
    } else {
        const T* up = PRO == kProSwiglu ? static_cast<const T*>(P.up) + r * P.up_stride : nullptr;
        float keep[kKeep][kVec];
        auto value = [&](const Raw<T>& a, const Raw<T>& b, float (&v)[kVec]) {
            unpack<T>(a, v);
            if constexpr (PRO == kProSwiglu) {
                float u[kVec];
                unpack<T>(b, u);
#pragma unroll
                for (int j = 0; j < kVec; ++j) v[j] = glu(P.kind, v[j], u[j]);
            }
        };
        auto value_at = [&](int i, float (&v)[kVec]) {
            const Raw<T> a = load_part<T, VEC>(x, i, K);
            value(a, PRO == kProSwiglu ? load_part<T, VEC>(up, i, K) : a, v);
        };
        auto scaled = [&](int i, float (&v)[kVec]) {
            if constexpr (PRO == kProNorm) {
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    v[j] = __fmul_rn(v[j], rms);
                    if (P.gain) v[j] = i * kVec + j < K ? __fmul_rn(v[j], P.gain[i * kVec + j]) : 0.f;
                }
            }
        };
        auto max_of = [&](const float (&v)[kVec]) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        };
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            const int i = threadIdx.x + c * step;
            if (i < parts) value_at(i, keep[c]);
            else
#pragma unroll
                for (int j = 0; j < kVec; ++j) keep[c][j] = 0.f;
        }
        if constexpr (PRO == kProNorm) {
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < kKeep; ++c)
#pragma unroll
                for (int j = 0; j < kVec; ++j) sum = fmaf(keep[c][j], keep[c][j], sum);
            for (int i = threadIdx.x + kKeep * step; i < parts; i += step) {
                float v[kVec];
                value_at(i, v);
#pragma unroll
                for (int j = 0; j < kVec; ++j) sum = fmaf(v[j], v[j], sum);
            }
            rms = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fdiv_rn(block_sum(sum, part_sum), static_cast<float>(K)), P.eps)));
#pragma unroll
            for (int c = 0; c < kKeep; ++c) {
                const int i = threadIdx.x + c * step;
                if (i < parts) scaled(i, keep[c]);
            }
        }
#pragma unroll
        for (int c = 0; c < kKeep; ++c) max_of(keep[c]);
        for (int i = threadIdx.x + kKeep * step; i < parts; i += step) {
            float v[kVec];
            value_at(i, v);
            scaled(i, v);
            max_of(v);
        }
        set_scale();
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            const int i = threadIdx.x + c * step;
            if (i < parts) store(i, keep[c]);
        }
        for (int i = threadIdx.x + kKeep * step; i < parts; i += step) {
            float v[kVec];
            value_at(i, v);
            scaled(i, v);
            store(i, v);
        }
    }
}

template <typename T, bool VEC>
void (*pick(int kind))(QuantizeI8) {
    return kind == kProNone ? quantize_i8_kernel<T, VEC, kProNone>
                            : (kind == kProNorm ? quantize_i8_kernel<T, VEC, kProNorm> : quantize_i8_kernel<T, VEC, kProSwiglu>);
}

}  // namespace

int launch_quantize_i8(const QuantizeI8& o, cudaStream_t stream) {
    const int size = o.x_type == kTypeF32 ? 4 : 2;
    uintptr_t bits = reinterpret_cast<uintptr_t>(o.x) | static_cast<uintptr_t>(o.x_stride * size);
    if (o.up) bits |= reinterpret_cast<uintptr_t>(o.up) | static_cast<uintptr_t>(o.up_stride * size);
    const bool vec = (bits & 15) == 0;
    void (*kernel)(QuantizeI8) = nullptr;
    if (o.x_type == kTypeF32) kernel = vec ? pick<float, true>(o.kind) : pick<float, false>(o.kind);
    else if (o.x_type == kTypeF16) kernel = vec ? pick<__half, true>(o.kind) : pick<__half, false>(o.kind);
    else kernel = vec ? pick<__nv_bfloat16, true>(o.kind) : pick<__nv_bfloat16, false>(o.kind);
    const int parts = (o.K + kVec - 1) / kVec;
    const int want = o.N <= kFewRows ? parts : (parts + kKeep - 1) / kKeep;
    const int threads = std::min(kMaxThreads, (want + 31) / 32 * 32);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(o.N);
    cfg.blockDim = dim3(threads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, o);
    return e == cudaSuccess ? 1 : -static_cast<int>(e);
}

}  // namespace wllm
