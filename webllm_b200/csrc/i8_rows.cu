// Row quantiser of the 8-bit products (wllm_quantize_i8): N rows of K values
// become int8 with one scale each.
//
//   a = max_k |v_k|     s = fl(a / 127)     q_k = nearest integer to v_k / s
//
// v is the row itself, RMS_NORM(x) * gain, or act(gate) * up. Ties go to the
// even integer and the quotient is the exact one, so q does not depend on how
// a division is rounded: v is multiplied by 1/s once a little too small and
// once a little too large, each product and its rounding to an integer one FMA
// (two values an instruction), and only where the two integers differ the
// remainder r = v - q s decides (one FMA; where 2|r| is near s it has at most
// 24 bits, so it is exact, and FMA's rounding is monotone elsewhere). Of f32
// values that is 3 in 100,000; of bf16 ones, whose quotients 127 v / a are ratios
// of small numbers, one in some hundred is an exact tie. A row whose a is below
// 2^-100, where 1/s could overflow or s be rounded to a few bits, takes double
// quotients, clamped to +-127.
// A row that holds a NaN or an infinity has no scale: s = NaN and q = 0, so
// every product of it is NaN.
//
// Bound: HBM (one read of the row, K + 4 bytes written): 8192 x 14336 bf16 in 54
// us, 6.5 TB/s; 4096 x 14336 f32 in 43.5 us, 6.8 TB/s (above what HBM copies at:
// part of it is still in L2). Behind a prologue not: silu(gate) * up of 32768 x
// 1536 bf16 takes 57 us, 4.4 TB/s, with the SFU busy for 44 % of the time, an
// instruction issued in 54 % and most waits for loads, of which 64 registers a
// thread leave 32 warps an SM to have in flight; gelu(gate) * up of 8192 x 8192 bf16
// 103 us, 3.3 TB/s (issue 69 %); RMS_NORM(x) * gain of 8192 x 4096 bf16 43 us, 2.3
// TB/s (issue 42 %, waits for loads and for the gain, read value by value). One
// CTA per row; the row's values stay in registers between the maximum and the rounding, so rows
// up to 32 values a thread are read once; longer rows are read again (from L2)
// in the second pass.
// Threads: rows that are few take one 8-value vector a thread (latency), many
// rows as many as its registers keep (fewer barriers a byte), and many short rows
// a warp each, eight a CTA (25,960 x 256, silu(gate) * up: 11 us against 29
// with a CTA a row).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "wllm_internal.h"

namespace wllm {
namespace {

constexpr int kVec = 8;    // values of a thread's vector
// Vectors a thread keeps in registers: 32 of them, as loaded or (with a
// prologue) as f32.
__host__ __device__ constexpr int keep_vecs(int size, int pro) { return size == 2 && pro == kProNone ? 8 : 4; }
constexpr int kMaxThreads = 512;
constexpr int kWarpRows = 8;   // rows of a CTA whose warps take one each
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

// Values [8 i, 8 i + 8) of a row. VEC: the row starts on a 16-byte boundary;
// otherwise they are shifted out of the 16-byte words that they lie in (each of
// which holds at least one of them, so no word that is read is wholly outside
// the row). Every vector of a row is shifted alike.
template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> load_vec(const T* row, int i) {
    constexpr int kPieces = Raw<T>::kWords / 4;
    Raw<T> r;
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + static_cast<int64_t>(i) * kVec);
    const uint4* p = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15));
    const uint32_t off = VEC ? 0 : static_cast<uint32_t>(at & 15);
    uint32_t w[4 * kPieces + 4];
#pragma unroll
    for (int h = 0; h < kPieces + (VEC ? 0 : 1); ++h) {
        const uint4 a = h < kPieces || off ? p[h] : make_uint4(0, 0, 0, 0);
        w[4 * h] = a.x, w[4 * h + 1] = a.y, w[4 * h + 2] = a.z, w[4 * h + 3] = a.w;
    }
    if constexpr (VEC) {
#pragma unroll
        for (int h = 0; h < Raw<T>::kWords; ++h) r.w[h] = w[h];
    } else {
        // by words, then by bytes
        const uint32_t words = off >> 2, bits = (off & 3) * 8;
        if (words & 2) {
#pragma unroll
            for (int h = 0; h + 2 < 4 * kPieces + 4; ++h) w[h] = w[h + 2];
        }
        if (words & 1) {
#pragma unroll
            for (int h = 0; h + 1 < 4 * kPieces + 4; ++h) w[h] = w[h + 1];
        }
#pragma unroll
        for (int h = 0; h < Raw<T>::kWords; ++h) r.w[h] = __funnelshift_r(w[h], w[h + 1], bits);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
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

// Two f32 in a register pair, and their packed arithmetic.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    return static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float low(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// silu(g) * u and gelu(g) * u, as wllm_mul_mat_glu_batch computes them: x / (1 +
// e^-z) with the SFU's exponential and reciprocal. Both flush results below the
// normals to zero: an e^-z below 2^-126 is lost in the sum anyway, but a
// reciprocal of more than 2^126 (a gate below some -87) is not, since u, or a row
// whose gates are all so small, brings it back. A row with a gate below kDeep is
// computed value by value, such gates' with silu_deep.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float x_sigmoid(float x, float z) { return x * rcp(1.f + ex2(z * -kLog2e)); }
constexpr float kDeep = -87.f;
// There 1 + e^-g is e^-g to the last bit: g e^g u, e^g in four factors that stay
// normal wherever the product can.
__device__ __forceinline__ float silu_deep(float g, float u) {
    const float h = ex2(g * (0.25f * kLog2e));
    return g * h * h * u * h * h;
}
// The bits of a vector's lowest gate, where it is negative (there the bits order by
// size, above all positive ones), and whether they are below kDeep.
template <typename T>
__device__ __forceinline__ uint32_t lowest(uint32_t most, const Raw<T>& r) {
#pragma unroll
    for (int h = 0; h < Raw<T>::kWords; ++h) {
        if constexpr (sizeof(T) == 4) most = max(most, r.w[h]);
        else most = __vmaxu2(most, r.w[h]);
    }
    return most;
}
template <typename T>
__device__ __forceinline__ bool is_deep(uint32_t most) {
    if constexpr (sizeof(T) == 4) return most > 0xC2AE0000u;
    return max(most & 0xffffu, most >> 16) > (std::is_same<T, __half>::value ? 0xD570u : 0xC2AEu);
}
__device__ __forceinline__ float glu(int kind, float g, float u) {
    if (kind == kProSwiglu) return g < kDeep ? silu_deep(g, u) : __fmul_rn(x_sigmoid(g, g), u);
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

// The same of a vector, silu two values an instruction.
__device__ __forceinline__ void glu8(int kind, float (&v)[kVec], const float (&u)[kVec]) {
    if (kind == kProSwiglu) {
#pragma unroll
        for (int j = 0; j < kVec; j += 2) {
            const uint64_t g = pack2(v[j], v[j + 1]), z = mul2(g, pack2(-kLog2e, -kLog2e));
            const uint64_t d = add2(pack2(ex2(low(z)), ex2(high(z))), pack2(1.f, 1.f));
            const uint64_t y = mul2(mul2(g, pack2(rcp(low(d)), rcp(high(d)))), pack2(u[j], u[j + 1]));
            v[j] = low(y), v[j + 1] = high(y);
        }
    } else {
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = glu(kind, v[j], u[j]);
    }
}

// Maximum (of bits) and sum over a row's threads: a warp (WARP) or the block;
// `part` holds one word per warp.
template <bool WARP>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* part) {
    v = __reduce_max_sync(0xffffffffu, v);
    if constexpr (WARP) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0u);
}
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (WARP) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = v;
    __syncthreads();
    v = lane < warps ? part[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: a sum with it is rounded to the nearest integer (ties to even)

// A row's scale and what its values are multiplied by: 1/s a little too small
// and a little too large (by 2^-21, where 1/s is off by 2^-24).
struct Scale {
    float s, lo, hi;
};

// Of the integers (as sums with kMagic) that v * lo and v * hi round to, the
// nearest to v / s; where they differ the remainder of the smaller decides.
__device__ __forceinline__ uint32_t nearest(float v, float s, uint32_t lo, uint32_t hi) {
    const float r = fabsf(2.f * fmaf(-(__uint_as_float(lo) - kMagic), s, v));
    return r > s || (r == s && (lo & 1)) ? hi : lo;
}
__device__ __forceinline__ int8_t quantize1(float v, const Scale& c) {
    return static_cast<int8_t>(nearest(v, c.s, __float_as_uint(fmaf(v, c.lo, kMagic)), __float_as_uint(fmaf(v, c.hi, kMagic))));
}
// In a row of tiny values, where 1/s could overflow, or one that is computed value
// by value.
__device__ __forceinline__ int8_t quantize_exact(float v, float s) {
    return s > 0.f ? static_cast<int8_t>(fmin(fmax(rint(static_cast<double>(v) / s), -127.0), 127.0)) : 0;
}

// Eight int8 of a vector.
__device__ __forceinline__ uint2 quantize8(const float (&v)[kVec], const Scale& c) {
    const uint64_t magic = pack2(kMagic, kMagic), lo = pack2(c.lo, c.lo), hi = pack2(c.hi, c.hi);
    uint32_t m[kVec], n[kVec], apart = 0;
#pragma unroll
    for (int j = 0; j < kVec; j += 2) {
        const uint64_t p = pack2(v[j], v[j + 1]);
        const uint64_t a = fma2(p, lo, magic), b = fma2(p, hi, magic);
        m[j] = static_cast<uint32_t>(a), m[j + 1] = static_cast<uint32_t>(a >> 32);
        n[j] = static_cast<uint32_t>(b), n[j + 1] = static_cast<uint32_t>(b >> 32);
        apart |= (m[j] ^ n[j]) | (m[j + 1] ^ n[j + 1]);
    }
    if (apart) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) m[j] = nearest(v[j], c.s, m[j], n[j]);
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        w[h] = __byte_perm(__byte_perm(m[4 * h], m[4 * h + 1], 0x0040), __byte_perm(m[4 * h + 2], m[4 * h + 3], 0x0040), 0x5410);
    return make_uint2(w[0], w[1]);
}

// PRO: kProNone, kProNorm, or kProSwiglu for both GLU kinds (P.kind tells).
// VEC: rows of x and up start on 16-byte boundaries, rows of q on 8-byte ones.
// At 64 registers and some 114 KB of a full SM's loads in flight, the loads of
// other rows run while one is rounded.
template <typename T, bool VEC, int PRO, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : kMaxThreads, WARP ? 4 : 2) quantize_i8_kernel(const QuantizeI8 P) {
    constexpr int kKeep = keep_vecs(sizeof(T), PRO);
    __shared__ uint32_t part_max[kMaxThreads / 32];
    __shared__ float part_sum[kMaxThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t r = WARP ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && r >= P.N) return;
    const T* x = static_cast<const T*>(P.x) + r * P.x_stride;
    const T* up = PRO == kProSwiglu ? static_cast<const T*>(P.up) + r * P.up_stride : nullptr;
    int8_t* q = P.q + r * P.q_stride;
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int K = P.K, vecs = K / kVec, step = WARP ? 32 : blockDim.x;  // whole vectors; up to 7 values behind them
    float rms = 1.f, pre = 1.f;  // behind RMS_NORM: 1 / rms, and what x is multiplied by ahead of it

    // the prologue on a vector's or a single value
    auto value = [&](const Raw<T>& a, const Raw<T>& b, float (&v)[kVec]) {
        unpack<T>(a, v);
        if constexpr (PRO == kProSwiglu) {
            float u[kVec];
            unpack<T>(b, u);
            glu8(P.kind, v, u);
        }
        if constexpr (PRO == kProNorm) {
#pragma unroll
            for (int j = 0; j < kVec; ++j) v[j] *= pre;
        }
    };
    uint32_t low_gate = 0;  // lowest() of this thread's gates
    auto value_at = [&](int i, float (&v)[kVec]) {
        const Raw<T> a = load_vec<T, VEC>(x, i);
        if constexpr (PRO == kProSwiglu) low_gate = lowest(low_gate, a);
        value(a, PRO == kProSwiglu ? load_vec<T, VEC>(up, i) : a, v);
    };
    auto scaled = [&](int k, float v) {
        if constexpr (PRO == kProNorm) {
            v = __fmul_rn(v, rms);
            if (P.gain) v = __fmul_rn(v, P.gain[k]);
        }
        return v;
    };
    auto scaled_vec = [&](int i, float (&v)[kVec]) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) v[j] = scaled(i * kVec + j, v[j]);
    };
    auto single = [&](int k) {
        const float v = to_f32(x[k]);
        if constexpr (PRO == kProNorm) return v * pre;
        return PRO == kProSwiglu ? glu(P.kind, v, to_f32(up[k])) : v;
    };
    auto bits = [](float v) { return __float_as_uint(v) & 0x7fffffffu; };
    // a NaN stays in `most`, as one whose bits are above infinity's
    auto max_vec = [&](float most, const float (&v)[kVec]) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(v[j])));
        return most;
    };
    const bool wide = VEC || ((reinterpret_cast<uintptr_t>(P.q) | static_cast<uintptr_t>(P.q_stride)) & 7) == 0;
    auto store = [&](int i, const float (&v)[kVec], const Scale& c) {
        const uint2 w = quantize8(v, c);
        if (wide) {
            *reinterpret_cast<uint2*>(q + static_cast<int64_t>(i) * kVec) = w;
        } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                q[static_cast<int64_t>(i) * kVec + j] = static_cast<int8_t>((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
        }
    };

    // ---- into registers (all loads of the kept vectors in flight together), and the maximum
    uint32_t top = 0;
    Raw<T> raw[PRO == kProNone ? kKeep : 1];
    float keep[PRO == kProNone ? 1 : kKeep][kVec];
    if constexpr (PRO == kProNone) {
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            const int i = tid + c * step;
            if (i < vecs) raw[c] = load_vec<T, VEC>(x, i);
            else
#pragma unroll
                for (int h = 0; h < Raw<T>::kWords; ++h) raw[c].w[h] = 0;
        }
#pragma unroll
        for (int c = 0; c < kKeep; ++c) top = max_raw<T>(top, raw[c]);
        for (int i = tid + kKeep * step; i < vecs; i += step) top = max_raw<T>(top, load_vec<T, VEC>(x, i));
        top = top_bits<T>(top);
    } else {
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            const int i = tid + c * step;
            if (i < vecs) value_at(i, keep[c]);
            else
#pragma unroll
                for (int j = 0; j < kVec; ++j) keep[c][j] = 0.f;
        }
        if constexpr (PRO == kProNorm) {
            auto square_sum = [&] {
                float sum = 0.f;
                auto add_vec = [&](const float (&v)[kVec]) {
#pragma unroll
                    for (int j = 0; j < kVec; ++j) sum = fmaf(v[j], v[j], sum);
                };
#pragma unroll
                for (int c = 0; c < kKeep; ++c) add_vec(keep[c]);
                for (int i = tid + kKeep * step; i < vecs; i += step) {
                    float v[kVec];
                    value_at(i, v);
                    add_vec(v);
                }
                for (int k = vecs * kVec + tid; k < K; k += step) sum = fmaf(single(k), single(k), sum);
                return row_sum<WARP>(sum, part_sum);
            };
            const float mean = __fadd_rn(__fdiv_rn(square_sum(), static_cast<float>(K)), P.eps);
            if (mean >= 0x1p-100f && mean <= 3.402823466e38f) {
                rms = __fdiv_rn(1.f, __fsqrt_rn(mean));
            } else {
                // Squares past the largest f32, or (with an eps of next to nothing) so small
                // that what was lost below the normals counts: x * 2^-96 or x * 2^96
                // instead, exact but for values that are nothing beside the row's others.
                pre = mean < 1.f ? 0x1p96f : 0x1p-96f;
#pragma unroll
                for (int c = 0; c < kKeep; ++c)
#pragma unroll
                    for (int j = 0; j < kVec; ++j) keep[c][j] *= pre;
                if constexpr (!WARP) __syncthreads();  // the first sum's parts have been read
                rms = static_cast<float>(1.0 / sqrt(static_cast<double>(square_sum()) / K + static_cast<double>(P.eps) * pre * pre));
            }
#pragma unroll
            for (int c = 0; c < kKeep; ++c)
                if (tid + c * step < vecs) scaled_vec(tid + c * step, keep[c]);
        }
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < kKeep; ++c) most = max_vec(most, keep[c]);
        for (int i = tid + kKeep * step; i < vecs; i += step) {
            float v[kVec];
            value_at(i, v);
            scaled_vec(i, v);
            most = max_vec(most, v);
        }
        top = bits(most);
    }
    for (int k = vecs * kVec + tid; k < K; k += step) top = max(top, bits(scaled(k, single(k))));
    // the sign bit, above all maxima: this row has a gate that glu8 does not hold for
    if (PRO == kProSwiglu && P.kind == kProSwiglu && is_deep<T>(low_gate)) top |= 0x80000000u;
    top = row_max<WARP>(top, part_max);
    const bool deep = PRO == kProSwiglu && (top >> 31);
    if (deep) {
        top = 0;
        for (int k = tid; k < K; k += step) top = max(top, bits(single(k)));
        if constexpr (!WARP) __syncthreads();  // part_max has been read
        top = row_max<WARP>(top, part_max);
    }

    // ---- the scale
    const float a = __uint_as_float(top);
    const bool bad = top >= 0x7f800000u;  // NaN or infinity
    Scale c;
    c.s = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a, 127.f);
    if (tid == 0) P.scale[r] = c.s;
    if (bad || a < 0x1p-100f || deep) {
        for (int k = tid; k < K; k += step) q[k] = bad ? 0 : quantize_exact(scaled(k, single(k)), c.s);
        return;
    }
    const float inv = __fdiv_rn(1.f, c.s);
    c.lo = inv * (1.f - 0x1p-21f), c.hi = inv * (1.f + 0x1p-21f);

    // ---- rounding
#pragma unroll
    for (int n = 0; n < kKeep; ++n) {
        const int i = tid + n * step;
        if (i < vecs) {
            if constexpr (PRO == kProNone) {
                float v[kVec];
                unpack<T>(raw[n], v);
                store(i, v, c);
            } else {
                store(i, keep[n], c);
            }
        }
    }
    for (int i = tid + kKeep * step; i < vecs; i += step) {
        float v[kVec];
        value_at(i, v);
        scaled_vec(i, v);
        store(i, v, c);
    }
    for (int k = vecs * kVec + tid; k < K; k += step) q[k] = quantize1(scaled(k, single(k)), c);
}

template <typename T, bool VEC, bool WARP>
void (*pick(int kind))(QuantizeI8) {
    return kind == kProNone ? quantize_i8_kernel<T, VEC, kProNone, WARP>
                            : (kind == kProNorm ? quantize_i8_kernel<T, VEC, kProNorm, WARP> : quantize_i8_kernel<T, VEC, kProSwiglu, WARP>);
}
template <typename T>
void (*pick(bool vec, bool warp, int kind))(QuantizeI8) {
    if (warp) return vec ? pick<T, true, true>(kind) : pick<T, false, true>(kind);
    return vec ? pick<T, true, false>(kind) : pick<T, false, false>(kind);
}

}  // namespace

int launch_quantize_i8(const QuantizeI8& o, cudaStream_t stream) {
    const int size = o.x_type == kTypeF32 ? 4 : 2;
    uintptr_t bits = reinterpret_cast<uintptr_t>(o.x) | static_cast<uintptr_t>(o.x_stride * size);
    if (o.up) bits |= reinterpret_cast<uintptr_t>(o.up) | static_cast<uintptr_t>(o.up_stride * size);
    const bool vec = (bits & 15) == 0 && ((reinterpret_cast<uintptr_t>(o.q) | static_cast<uintptr_t>(o.q_stride)) & 7) == 0;
    // many rows that a warp's registers hold: a warp each
    const int vecs = std::max(1, o.K / kVec), keep = keep_vecs(size, o.kind);
    const bool warp = o.N > kFewRows && vecs <= 32 * keep;
    void (*const kernel)(QuantizeI8) = o.x_type == kTypeF32   ? pick<float>(vec, warp, o.kind)
                                       : o.x_type == kTypeF16 ? pick<__half>(vec, warp, o.kind)
                                                              : pick<__nv_bfloat16>(vec, warp, o.kind);
    const int want = o.N <= kFewRows ? vecs : (vecs + keep - 1) / keep;
    const int threads = warp ? 32 * kWarpRows : std::min(kMaxThreads, (want + 31) / 32 * 32);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(warp ? (o.N + kWarpRows - 1) / kWarpRows : o.N);
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
