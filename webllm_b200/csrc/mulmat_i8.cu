// Products of 8-bit integers with a scale per token and per channel, dense
// (wllm_mul_mat_i8) and grouped by expert (wllm_mul_mat_id_i8), on tcgen05:
//
//   y[n][m] = (sum_k q[n][k] w[m][k]) * s[n] * t[m]
//
// The sum is exact: int8 x int8 -> int32 MMAs (kind::i8), and K <= 131071
// keeps it below 2^31. So however K is split, the result is the same.
//
// The weights are the MMA's A operand (128 channels, the TMEM lanes) and the
// tokens its B operand (N = 16..256, the TMEM columns): one kernel then serves
// a single token and a prompt, a lane's column values are one channel's, and a
// warp's store covers 32 consecutive channels of a token's row.
//
//  - warp 0 (TMA): per 128-byte chunk of K one box of 128 weight rows, and of
//    dense tokens one box of the tile's rows, into a ring of stages (K-major,
//    128-byte swizzle).
//  - warps 10..17 (grouped only): an expert's tokens are gathered through the
//    sorted slots with 16-byte cp.async, straight into the swizzled layout, so
//    no sorted copy of the activations is ever written. (TMA's gather of four
//    rows a copy is slower: 648 us against 399 for the step of 4096 tokens in 8
//    of 128 experts, 1536 -> 4096, at the time that both were tried, and 80
//    against 58 for 512 tokens in 8 of 64, 2048 -> 2048.)
//  - warp 1 (MMA): one thread issues the 4 K=32 MMAs of a chunk.
//  - warps 2..9 (epilogue): TMEM -> scales -> y, while the next tile's MMAs
//    fill the other accumulator. An item's rows and scales are fetched ahead of
//    the wait for its accumulator.
//
// CTAs are persistent over the items (expert, channel tile, token tile), in one
// of these modes (plan() chooses by a model of their cost):
//  - single: an item is 128 channels;
//  - pair: two CTAs of a cluster share an item of 256 channels (cta_group::2):
//    each loads its own 128 weight rows and half of the tokens, which both read,
//    so a chunk of a 256-token tile takes 32 KB of an SM's L2 bandwidth instead
//    of 48 (8192^3: 2960 TOP/s; a single CTA per item, 2430);
//  - split: where the items are fewer than the SMs (single tokens, small
//    batches), S = 2, 4 or 8 CTAs of a cluster share an item's K: each leaves
//    its int32 tile in its own shared memory, and after a cluster barrier CTA r
//    adds the S tiles of its share of the columns through distributed shared
//    memory.
//
// Bounds: HBM (the weights, once) up to a few hundred tokens (1 x 4096 -> 14336:
// 13 us, of which some 4 are set-up, first bytes and the last tile), the tensor
// pipe above (4096 x 14336 -> 4096: 160 us, 3.0 POP/s; in a long run the power
// limit, 2.5 to 2.8).
//
// Every mbarrier wait is bounded (wllm_set_wait_limit): on time-out the CTA records
// an error code (read by wllm_sync), stops issuing, waits for its copies and MMAs
// in flight and frees its TMEM.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "i8_plan.h"
#include "wllm_internal.h"

namespace wllm {

__device__ unsigned int g_i8_error = 0;

namespace {

constexpr int kEpiWarps = 8;        // two for each quarter of the TMEM lanes
constexpr int kThreads = 64 + 32 * kEpiWarps;  // copies, MMAs, epilogue
constexpr int kLoaders = 128;       // threads that gather a stage's tokens; there are two such groups
constexpr int kMaxStages = 12;
constexpr int kSmemBytes = 208 * 1024;  // dynamic, beside up to 17 KB of tables and barriers
constexpr uint32_t kSpinLimit = 1u << 20;  // polls of a barrier, each of which the hardware ends after 4 us: some 4 s

struct I8Args {
    CUtensorMap wmap;  // weights: [E][M][K] bytes, box 128 x 128 x 1
    CUtensorMap xmap;  // dense tokens: [rows][K] bytes, box 128 x the tile's rows of one CTA
    MulMatI8 o;
    int32_t tile_n;    // tokens of a full tile, a multiple of 16 (pair: of 32)
    int32_t tiles_m, tiles_n, chunks, stages, splits;  // tiles_n: dense; chunks: of a stage's bytes of K
    int32_t tmem_cols;
    uint32_t spin_limit;  // polls before a wait gives up
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Bounded wait; a time-out poisons the CTA (every later wait returns at once).
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, unsigned code, volatile int* poisoned, uint32_t limit) {
    for (uint32_t i = 0; i < limit; ++i) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 255u) == 255u && *poisoned) return false;
    }
    *poisoned = 1;
    atomicOr(&g_i8_error, code);
    return false;
}
// Bounded wait whatever the poison flag says, for what is in flight at exit.
__device__ __forceinline__ bool mbar_drain(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kSpinLimit; ++i)
        if (mbar_try(bar, parity)) return true;
    atomicOr(&g_i8_error, 8u);
    return false;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* tm, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(tm), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// Weights are read once a launch, or by token tiles that run side by side: first
// out of L2, so that they do not drive out what the kernels hand to each other
// (37 tokens in 4 of 60 experts, 1152 -> 2304, the block's last product: 32.2 ->
// 28.6 us).
__device__ __forceinline__ uint64_t evict_first() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], "
        "%6;" ::"r"(dst),
        "l"(tm), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}
// The address, for all CTAs of the cluster, of what lies at p's place in CTA `rank`.
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// The same copies into this CTA's memory, signalled on the barrier of the pair's
// first CTA (bar: an address of in_cta).
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(tm), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_3d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, uint32_t bar,
                                            uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, "
        "%4}], [%5], %6;" ::"r"(dst),
        "l"(tm), "r"(x), "r"(y), "r"(z), "r"(bar), "l"(policy)
        : "memory");
}
// 16 bytes to shared memory: `bytes` of src, then zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrives on the barrier at bar's place in CTA `rank` of the cluster. What it
// orders is not memory that the other CTA's threads read, but the tensor pipe's
// operands (fenced for its proxy by the caller) and accumulators. (Released at
// cluster scope the arrive waits for the thread's global stores: 1500 clocks a
// chunk, 144 us against 64 for 512 tokens in 8 of 64 experts, 2048 -> 2048.)
__device__ __forceinline__ void mbar_arrive_at(uint64_t* bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(in_cta(bar, rank)) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// UMMA shared-memory descriptor: K-major, 128-byte swizzle, 8-row groups 1024
// bytes apart, version 1.
__device__ __forceinline__ uint64_t umma_desc(uint32_t saddr) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor, kind::i8: signed A and B (K-major), s32 accumulator.
__device__ __forceinline__ uint32_t i8_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        :
        : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives on bar in both CTAs of the pair when the MMAs so far are done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 16 consecutive columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// True in one lane of a converged warp. (Under `lane == 0` instead, the compiler
// cannot tell that one thread issues a copy or an MMA, whose operands are
// uniform registers, and wraps each in a loop over the active lanes: 700 clocks
// a chunk where the MMAs take 512.)
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}
// A place in the ring of stages and the parity of its round.
struct Ring {
    int stages, s = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next() {
        if (++s == stages) s = 0, parity ^= 1;
    }
};
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same without ordering memory (global stores before it are not waited for).
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster(const int* p, uint32_t rank, int v) {
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(in_cta(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ int4 ld_cluster4(uint32_t local, uint32_t rank) {
    uint32_t remote;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(remote)
                 : "memory");
    return v;
}

// Two f32 in a register pair, and their packed arithmetic.
__device__ __forceinline__ uint64_t pack2(uint32_t a, uint32_t b) { return static_cast<uint64_t>(b) << 32 | a; }
__device__ __forceinline__ uint64_t pack2(float a, float b) { return pack2(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ float low(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// y in its type: the sum in f32, times the two scales in f32, then one rounding.
__device__ __forceinline__ float scaled(int32_t acc, float s, float t) { return __fmul_rn(__fmul_rn(__int2float_rn(acc), s), t); }
// The same of two sums, without the conversion pipe (8 clocks a warp and sum,
// more than an item's MMAs leave at K = 1536): the halves hi, lo of a sum are
// exact as floats (as_float(2^23's bits + lo) - 2^23), and hi * 65536 + lo is one
// FMA, so the conversion is rounded once, as __int2float_rn's.
__device__ __forceinline__ uint64_t scaled2(int32_t a, int32_t b, uint64_t s, uint64_t t) {
    const uint64_t hi = add2(pack2(static_cast<uint32_t>(0x4B400000 + (a >> 16)), static_cast<uint32_t>(0x4B400000 + (b >> 16))),
                             pack2(-12582912.f, -12582912.f));
    const uint64_t lo = add2(pack2(0x4B000000u | (a & 0xffff), 0x4B000000u | (b & 0xffff)), pack2(-8388608.f, -8388608.f));
    return mul2(mul2(fma2(hi, pack2(65536.f, 65536.f), lo), s), t);
}
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ uint32_t half_pair(const __half*, uint64_t v) {
    const __half2 h = __floats2half2_rn(low(v), high(v));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t half_pair(const __nv_bfloat16*, uint64_t v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(low(v), high(v));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_y(const MulMatI8& o, int64_t at, float v) {
    if (o.y_type == kTypeF32) put(static_cast<float*>(o.y) + at, v);
    else if (o.y_type == kTypeF16) put(static_cast<__half*>(o.y) + at, v);
    else put(static_cast<__nv_bfloat16*>(o.y) + at, v);
}

// An item: `rows` token rows from position `first` on, of expert e, against
// the channels from m0 on. A group's token tiles are of one size (the least
// multiple of 16, or 32 of a pair, that covers it in as many tiles), its channel
// tiles come one after the other with the token tiles of one channel tile next
// to each other (they read the same weights).
struct Item {
    int e, m0, first, rows;
};

// Walks the items i of a CTA in rising order. cum[e]: token tiles of the experts
// before e, begin[e]: their slots (grouped; E + 1 entries each).
template <bool GROUPED, int MODE>
struct Walk {
    const I8Args& P;
    const int32_t* cum;
    const int32_t* begin;
    int e = 0;

    __device__ __forceinline__ Item at(int i) {
        constexpr int kM = is_pair(MODE) ? 2 * kTileM : kTileM;
        constexpr int kStep = is_pair(MODE) ? 32 : 16;
        Item it;
        if constexpr (!GROUPED) {
            const int c = P.tiles_n == 1 ? i : i / P.tiles_n;  // (no division for few tokens: an item may be 1000 clocks)
            it.e = 0;
            it.m0 = c * kM;
            it.first = (i - c * P.tiles_n) * P.tile_n;
            it.rows = min(P.tile_n, P.o.N - it.first);
        } else {
            while (cum[e + 1] * P.tiles_m <= i) ++e;
            const int tiles = cum[e + 1] - cum[e], j = i - cum[e] * P.tiles_m;
            const int n = begin[e + 1] - begin[e];
            it.e = e;
            if (tiles == 1) {
                it.m0 = j * kM;
                it.first = begin[e];
                it.rows = n;
            } else {
                const int c = j / tiles, size = ((n - 1) / tiles + kStep) / kStep * kStep;  // (n + tiles may pass 2^31)
                it.m0 = c * kM;
                it.first = begin[e] + (j - c * tiles) * size;
                it.rows = min(size, begin[e + 1] - it.first);
            }
        }
        return it;
    }
};

// Every other 16 columns of an accumulator, of the 32 lanes (channels) that this
// warp holds, into y: column n of the tile is the row at[n] (elements from y's
// start) with scale s[n].
template <typename T>
__device__ __forceinline__ void store_tile(const MulMatI8& o, uint32_t taddr, int first, int rows, int m, float tm, const int64_t* at,
                                           const float* s) {
    T* y = static_cast<T*>(o.y) + m;
    const int lane = threadIdx.x & 31;
    const bool live = m < o.M, whole = __all_sync(0xffffffffu, live);
    // 16-bit values of two neighbouring channels go out as one word: the lanes of
    // a pair exchange one of their two columns
    const bool words = sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(o.y) & 3) == 0 && (o.y_stride & 1) == 0;
    const uint64_t t2 = pack2(tm, tm);
    for (int n = first; n < rows; n += 32) {
        int32_t acc[16];
        tmem_ld16(taddr + n, acc);
        if (whole && n + 16 <= rows && (sizeof(T) == 4 || words)) {  // no branch between the stores
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const uint64_t v = scaled2(acc[j], acc[j + 1], *reinterpret_cast<const uint64_t*>(s + n + j), t2);
                if constexpr (sizeof(T) == 4) {
                    put(y + at[n + j], low(v));
                    put(y + at[n + j + 1], high(v));
                } else {
                    const uint32_t own = half_pair(y, v), other = __shfl_xor_sync(0xffffffffu, own, 1);
                    // even lanes: column j of channels m, m + 1; odd: column j + 1 of m - 1, m
                    const uint32_t w = __byte_perm(own, other, lane & 1 ? 0x3276 : 0x5410);
                    *reinterpret_cast<uint32_t*>(y - (lane & 1) + at[n + j + (lane & 1)]) = w;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const uint64_t v = scaled2(acc[j], acc[j + 1], *reinterpret_cast<const uint64_t*>(s + n + j), t2);
                if (n + j < rows && live) put(y + at[n + j], low(v));
                if (n + j + 1 < rows && live) put(y + at[n + j + 1], high(v));
            }
        }
    }
}

template <bool GROUPED, int MODE>
__global__ void __launch_bounds__(GROUPED ? kThreads + 2 * kLoaders : kThreads, 1) i8_kernel(const __grid_constant__ I8Args P) {
    constexpr bool SPLIT = MODE == kSplit, PAIR = is_pair(MODE);
    constexpr int kTokens = MODE == kPair ? kMaxTileN : (PAIR ? kMaxShortN : kMaxSingleN);
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_free[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int poison;
    __shared__ int32_t cum[GROUPED ? kMaxExperts + 1 : 1], begin[GROUPED ? kMaxExperts + 1 : 1];
    __shared__ int32_t warp_sum[(kThreads + 2 * kLoaders) / 32];
    __shared__ int64_t out_at[2][kTokens];  // where a tile's rows begin in y
    __shared__ __align__(8) float out_scale[2][kTokens];
    static_assert(kTokens <= 32 * kEpiWarps, "a thread of the epilogue for each row of a tile");
    // 1024-byte alignment for the swizzled tiles
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    volatile int* poisoned = &poison;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kSub = chunks_of_stage(MODE);
    const int stages = P.stages, b_bytes = (PAIR ? P.tile_n / 2 : P.tile_n) * kChunk;
    const int stage_bytes = kSub * (kABytes + b_bytes);  // kSub weight chunks, then as many of the tokens
    uint32_t rank = 0;  // in the cluster
    if constexpr (MODE != kSingle) asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
    const int c0 = SPLIT ? static_cast<int>(static_cast<int64_t>(P.chunks) * rank / P.splits) : 0;
    const int c1 = SPLIT ? static_cast<int>(static_cast<int64_t>(P.chunks) * (rank + 1) / P.splits) : P.chunks;
    const int group = SPLIT ? P.splits : (PAIR ? 2 : 1);  // CTAs that share an item
    const int item0 = blockIdx.x / group, item_step = gridDim.x / group;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1 + (GROUPED ? (PAIR ? 2 : 1) * kLoaders / 32 : 0));
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_free[b], (PAIR ? 2 : 1) * kEpiWarps);
        }
        poison = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&P.wmap) : "memory");
        if constexpr (!GROUPED) asm volatile("prefetch.tensormap [%0];" ::"l"(&P.xmap) : "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                         "r"(P.tmem_cols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                         "r"(P.tmem_cols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    tc_fence_before();
    if constexpr (PAIR) cluster_sync();  // the other CTA's barriers are set up too
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // Nothing of the inputs is touched ahead of this: the kernel before may be the
    // one that quantises the weights. (Bringing the first weights into L2 from
    // here gained nothing: 14.1 us without, 14.1 to 14.6 with, 1 x 4096 -> 14336.)
    asm volatile("griddepcontrol.wait;" ::: "memory");

    int items;
    if constexpr (GROUPED) {
        // token tiles of each expert, then their running sum
        int carry = 0;
        for (int base = 0; base < P.o.E; base += blockDim.x) {
            const int e = base + threadIdx.x;
            int tiles = 0;
            if (e < P.o.E) {
                const int at = P.o.offsets[e];
                begin[e] = at;
                tiles = (P.o.offsets[e + 1] - at + P.tile_n - 1) / P.tile_n;
            }
            int sum = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            __syncthreads();  // warp_sum of the step before has been read
            if (lane == 31) warp_sum[warp] = sum;
            __syncthreads();
            int before = carry;
            for (int w = 0; w < (kThreads + 2 * kLoaders) / 32; ++w) {
                if (w < warp) before += warp_sum[w];
                carry += warp_sum[w];
            }
            if (e < P.o.E) cum[e + 1] = before + sum;
        }
        if (threadIdx.x == 0) {
            cum[0] = 0;
            begin[P.o.E] = P.o.offsets[P.o.E];
        }
        __syncthreads();
        items = carry * P.tiles_m;
    } else {
        items = P.tiles_n * P.tiles_m;
    }
    Walk<GROUPED, MODE> walk{P, cum, begin};

    if (warp == 0) {
        if (elect_one()) {
            // ---------------- copies ----------------
            Ring ring{stages};
            int filled = 0;  // stages filled so far, up to the ring's size
            const uint64_t policy = evict_first();
            const uint32_t full0 = PAIR ? in_cta(full, 0) : 0;  // the pair's first CTA's
            bool ok = true;
            for (int i = item0; i < items && ok; i += item_step) {
                const Item it = walk.at(i);
                const int m0 = it.m0 + (PAIR ? kTileM * rank : 0);
                const int cols = (it.rows + 31) & ~31, n0 = it.first + (PAIR ? rank * (cols / 2) : 0);
                for (int c = c0; c < c1; ++c) {
                    const int s = ring.s;
                    ok = filled < stages || mbar_wait(&empty[s], ring.parity ^ 1, 1u, poisoned, P.spin_limit);
                    if (!ok) break;
                    const uint32_t a = smem_u32(smem + s * stage_bytes);
                    const uint32_t b = a + kSub * kABytes;
                    if constexpr (PAIR) {
                        if (rank == 0) mbar_expect_tx(&full[s], 2 * (GROUPED ? kSub * kABytes : stage_bytes));
                    } else {
                        mbar_expect_tx(&full[s], GROUPED ? kSub * kABytes : stage_bytes);
                    }
#pragma unroll
                    for (int h = 0; h < kSub; ++h) {
                        const int k = (c * kSub + h) * kChunk;
                        if constexpr (PAIR) {
                            tma_3d_pair(a + h * kABytes, &P.wmap, k, m0, it.e, full0 + 8 * s, policy);
                            if constexpr (!GROUPED) tma_2d_pair(b + h * b_bytes, &P.xmap, k, n0, full0 + 8 * s);
                        } else {
                            tma_3d(a + h * kABytes, &P.wmap, k, m0, it.e, &full[s], policy);
                            if constexpr (!GROUPED) tma_2d(b + h * b_bytes, &P.xmap, k, n0, &full[s]);
                        }
                    }
                    if (filled < stages) ++filled;
                    ring.next();
                }
            }
            // The copies in flight land before the CTA ends. (Nothing else is left to do
            // here; where all went well the MMAs wait for the same.) Those of a pair's
            // second CTA are signalled to the first, but their stages are freed here.
            for (int p = 0; p < filled; ++p) {
                ring.s = ring.s ? ring.s - 1 : (ring.parity ^= 1, stages - 1);
                if (!mbar_drain(PAIR && rank ? &empty[ring.s] : &full[ring.s], ring.parity)) break;
            }
        }
    } else if (warp == 1) {
        Ring ring{stages};
        bool ok = true;
        if ((!PAIR || rank == 0) && elect_one()) {
            // ---------------- MMAs ----------------
            uint32_t t = 0;
            uint64_t* last = nullptr;  // the barrier of the last commit, and its parity
            uint32_t last_parity = 0;
            for (int i = item0; i < items && ok; i += item_step, ++t) {
                const Item it = walk.at(i);
                const uint32_t idesc = PAIR ? i8_idesc(2 * kTileM, (it.rows + 31) & ~31) : i8_idesc(kTileM, (it.rows + 15) & ~15);
                const uint32_t buf = t & 1, d = tmem + buf * P.tile_n;
                ok = t < 2 || mbar_wait(&acc_free[buf], ((t >> 1) - 1) & 1, 2u, poisoned, P.spin_limit);
                if (!ok) break;
                tc_fence_after();
                for (int c = c0; c < c1; ++c) {
                    const int s = ring.s;
                    ok = mbar_wait(&full[s], ring.parity, 4u, poisoned, P.spin_limit);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + s * stage_bytes);
#pragma unroll
                    for (int h = 0; h < kSub; ++h) {
                        const uint64_t ad = umma_desc(a + h * kABytes), bd = umma_desc(a + kSub * kABytes + h * b_bytes);
#pragma unroll
                        for (int j = 0; j < kChunk / 32; ++j) {
                            const uint32_t more = c > c0 || h > 0 || j > 0;
                            if constexpr (PAIR) umma_i8_pair(d, ad + 2 * j, bd + 2 * j, idesc, more);
                            else umma_i8(d, ad + 2 * j, bd + 2 * j, idesc, more);
                        }
                    }
                    if constexpr (PAIR) umma_commit_pair(&empty[s]);
                    else umma_commit(&empty[s]);
                    last = &empty[s], last_parity = ring.parity;
                    ring.next();
                }
                if (!ok) break;  // an accumulator that is not whole is not handed over
                if constexpr (PAIR) umma_commit_pair(&acc_full[buf]);
                else umma_commit(&acc_full[buf]);
            }
            // MMAs in flight end before the TMEM is freed
            if (last) mbar_drain(last, last_parity);
        }
    } else if (warp < 2 + kEpiWarps) {
        // ---------------- epilogue ----------------
        const int quad = warp & 3;                // the TMEM lanes this warp may read
        const int n0 = (warp - 2) / 4 % 2 * 16;   // it takes every other 16 columns, from here on
        // An item's channel scale and, of the row that this thread looks after, the
        // place in y and the scale are fetched while the item before it is stored.
        const int mine = threadIdx.x - 64;
        auto channel = [&](const Item& it) { return it.m0 + (PAIR ? kTileM * rank : 0) + 32 * quad + lane; };
        auto fetch_channel = [&](const Item& it) {
            const int m = channel(it);
            return m < P.o.M ? P.o.w_scale[static_cast<int64_t>(it.e) * P.o.M + m] : 0.f;
        };
        auto fetch_row = [&](const Item& it) {
            if (mine >= it.rows) return -1;
            return GROUPED ? P.o.order[it.first + mine] : it.first + mine;
        };
        auto fetch_scale = [&](int row) { return row < 0 ? 0.f : P.o.q_scale[!GROUPED || P.o.per_slot ? row : row / P.o.k]; };
        Item next{};
        float next_tm = 0.f, next_scale = 0.f;
        int next_row = -1;
        if (item0 < items) {
            next = walk.at(item0);
            next_tm = fetch_channel(next);
            next_row = fetch_row(next);
            next_scale = fetch_scale(next_row);
        }
        uint32_t t = 0;
        bool ok = true;
        for (int i = item0; i < items; i += item_step, ++t) {
            const Item it = next;
            const uint32_t buf = t & 1;
            const int m = channel(it);
            const float tm = next_tm;
            if (mine < it.rows) {
                out_at[buf][mine] = next_row * P.o.y_stride;
                out_scale[buf][mine] = next_scale;
            }
            const bool more = i + item_step < items;
            if (more) {
                next = walk.at(i + item_step);
                next_tm = fetch_channel(next);
                next_row = fetch_row(next);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");  // the epilogue warps
            // after a time-out the items are still walked (the epilogue's warps meet at
            // the barrier above), without their stores and without handing accumulators
            // back; a warp's lanes, which read the TMEM together, give up together
            ok = __all_sync(0xffffffffu, ok && mbar_wait(&acc_full[buf], (t >> 1) & 1, 2u, poisoned, P.spin_limit));
            tc_fence_after();
            if (more) next_scale = fetch_scale(next_row);
            const uint32_t d = tmem + buf * P.tile_n + (static_cast<uint32_t>(32 * quad) << 16);
            if (!ok) {
            } else if constexpr (SPLIT) {
                // the stages are free by now: all copies have landed and all MMAs have read them
                int32_t* part = reinterpret_cast<int32_t*>(smem) + 32 * quad + lane;
                for (int n = n0; n < it.rows; n += 32) {
                    int32_t acc[16];
                    tmem_ld16(d + n, acc);
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(n + j) * kTileM] = acc[j];
                }
            } else if (P.o.y_type == kTypeF32) {
                store_tile<float>(P.o, d, n0, it.rows, m, tm, out_at[buf], out_scale[buf]);
            } else if (P.o.y_type == kTypeF16) {
                store_tile<__half>(P.o, d, n0, it.rows, m, tm, out_at[buf], out_scale[buf]);
            } else {
                store_tile<__nv_bfloat16>(P.o, d, n0, it.rows, m, tm, out_at[buf], out_scale[buf]);
            }
            tc_fence_before();
            __syncwarp();
            if (ok && lane == 0) {
                if constexpr (PAIR) mbar_arrive_at(&acc_free[buf], 0);
                else mbar_arrive(&acc_free[buf]);
            }
        }
    } else if constexpr (GROUPED) {
        // ---------------- gathered tokens ----------------
        // Two groups of threads take the stages in turn, so that one's address
        // and barrier work overlaps the other's. Of a stage, thread x of a group
        // takes 16-byte piece x % 8 of rows x / 8, x / 8 + 16, ..
        const int x = (threadIdx.x - kThreads) % kLoaders, piece = x & 7, r0 = x >> 3;
        const int mine = (threadIdx.x - kThreads) / kLoaders;
        constexpr int kRows = (PAIR ? kTokens / 2 : kTokens) / 16;
        auto cols_of = [&](const Item& it) { return PAIR ? ((it.rows + 31) & ~31) / 2 : (it.rows + 15) & ~15; };  // of this CTA
        int slot[kRows];
        auto fetch = [&](const Item& it) {
            const int cols = cols_of(it), skip = PAIR ? static_cast<int>(rank) * cols : 0;
#pragma unroll
            for (int r = 0; r < kRows; ++r)  // what is behind the last row reads that row again
                if (r * 16 < cols) slot[r] = P.o.order[it.first + min(skip + r0 + 16 * r, it.rows - 1)];
        };
        Item it{};
        if (item0 < items) fetch(it = walk.at(item0));
        // A stage is told to the MMA thread (of the pair's first CTA) when the
        // group's next one has been issued and this one has landed: one arrival a
        // warp, and the fence for the tensor pipe's proxy by the threads that
        // wrote. (An arrival of every thread, triggered by its copies, took 128
        // arrivals a stage on one barrier, and a pair's second CTA a warp that
        // passed them on: 900 clocks a chunk, whatever the copies.)
        auto tell = [&](int s) {
            fence_async();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_at(&full[s], 0);
                else mbar_arrive(&full[s]);
            }
        };
        Ring ring{stages};
        int q = 0, untold = -1;  // stages so far; the group's stage that has not been told
        bool ok = true;
        for (int i = item0; i < items && ok; i += item_step) {
            const int cols = cols_of(it);
            const int8_t* row[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                row[r] = P.o.q + (r * 16 < cols ? static_cast<int64_t>(P.o.per_slot ? slot[r] : slot[r] / P.o.k) * P.o.q_stride : 0);
            if (i + item_step < items) fetch(it = walk.at(i + item_step));  // the next item's, while this one's are copied
            for (int c = c0; c < c1; ++c, ++q, ring.next()) {
                if ((q & 1) != mine) continue;
                const int s = ring.s;
                ok = q < stages || mbar_wait(&empty[s], ring.parity ^ 1, 1u, poisoned, P.spin_limit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                // piece p of row r lies at r * 128 + (p ^ (r % 8)) * 16; of the last piece only
                // the row's own bytes are read, and zeros stand behind them
#pragma unroll
                for (int h = 0; h < kSub; ++h) {
                    const int k = (c * kSub + h) * kChunk + piece * 16;
                    const uint32_t bytes = piece_bytes(P.o.K, k);
                    const int at = k < P.o.K ? k : 0;
                    const uint32_t dst = smem_u32(smem + s * stage_bytes) + kSub * kABytes + h * b_bytes + r0 * kChunk + ((piece ^ (r0 & 7)) << 4);
#pragma unroll
                    for (int r = 0; r < kRows; ++r)
                        if (r * 16 < cols) cp_async16(dst + r * 16 * kChunk, row[r] + at, bytes);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                if (untold >= 0) {
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    tell(untold);
                }
                untold = s;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (untold >= 0) tell(untold);
    }
    if constexpr (SPLIT) {
        // one item per cluster, so that the sum over the splits comes after all roles;
        // a tile that one CTA gave up on is summed by none
        if (*poisoned)
            for (int r = 0; r < P.splits; ++r) st_cluster(&poison, r, 1);
        __syncwarp();
        cluster_sync();
        if (item0 < items && !*poisoned) {
            const Item it = walk.at(item0);
            // a warp sums a column's 128 channels, four a lane, over the splits at once
            const uint32_t part = smem_u32(smem) + 16 * lane;
            const int per = (it.rows + P.splits - 1) / P.splits, n0 = rank * per, n1 = min(n0 + per, it.rows);
            const int m = it.m0 + 4 * lane;
            for (int n = n0 + warp; n < n1; n += blockDim.x / 32) {
                int4 v[8];
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < P.splits) v[r] = ld_cluster4(part + 4 * kTileM * n, r);
                int acc[4] = {0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (r < P.splits) acc[0] += v[r].x, acc[1] += v[r].y, acc[2] += v[r].z, acc[3] += v[r].w;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (m + j < P.o.M)
                        store_y(P.o, out_at[0][n] + m + j,
                                scaled(acc[j], out_scale[0][n], P.o.w_scale[static_cast<int64_t>(it.e) * P.o.M + m + j]));
            }
        }
    }
    if constexpr (GROUPED) {
        // slots without an expert come last in the order: their rows are zero
        for (int64_t p = P.o.offsets[P.o.E] + blockIdx.x; p < P.o.slots; p += gridDim.x) {
            const int64_t row = P.o.order[p];
            for (int m = threadIdx.x; m < P.o.M; m += blockDim.x) store_y(P.o, row * P.o.y_stride + m, 0.f);
        }
    }
    __syncwarp();
    tc_fence_before();
    // no CTA ends while another reads its tile or signals its barriers
    if constexpr (MODE != kSingle) cluster_meet();
    else __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P.tmem_cols));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P.tmem_cols));
    }
}

// Rows whose addresses are not multiples of 16 bytes, which the tensor maps
// cannot take: one warp per output, lanes along K. Not tuned.
template <bool GROUPED>
__global__ void __launch_bounds__(256) i8_general_kernel(const MulMatI8 o) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
    const int64_t rows = GROUPED ? o.slots : o.N;
    for (int64_t x = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); x < rows * o.M; x += warps) {
        const int64_t p = x / o.M;
        const int m = static_cast<int>(x % o.M);
        int e = 0;
        int64_t row = p, from = p;
        if constexpr (GROUPED) {
            row = o.order[p];
            from = o.per_slot ? row : row / o.k;
            if (p >= o.offsets[o.E]) {
                if (lane == 0) store_y(o, row * o.y_stride + m, 0.f);
                continue;
            }
            int hi = o.E - 1;  // the last expert whose first slot is at or before p
            while (e < hi) {
                const int mid = (e + hi + 1) >> 1;
                if (o.offsets[mid] <= p) e = mid;
                else hi = mid - 1;
            }
        }
        const int8_t* w = o.w + e * o.w_expert_bytes + m * o.w_row_bytes;
        const int8_t* q = o.q + from * o.q_stride;
        int acc = 0;
        for (int k = lane; k < o.K; k += 32) acc += static_cast<int>(w[k]) * q[k];
        acc = __reduce_add_sync(0xffffffffu, acc);
        if (lane == 0) store_y(o, row * o.y_stride + m, scaled(acc, o.q_scale[from], o.w_scale[static_cast<int64_t>(e) * o.M + m]));
    }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn i8_encoder() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        cudaGetLastError();
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

bool encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, cuuint32_t rows) {
    const cuuint32_t box[3] = {kChunk, rows, 1}, es[3] = {1, 1, 1};
    return i8_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GROUPED>
int launch_general(const MulMatI8& o, cudaStream_t stream, int num_sms) {
    const int64_t outs = (GROUPED ? o.slots : o.N) * static_cast<int64_t>(o.M);
    const int blocks = static_cast<int>(std::min<int64_t>((outs + 7) / 8, 8 * num_sms));
    i8_general_kernel<GROUPED><<<blocks, 256, 0, stream>>>(o);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 1 : -static_cast<int>(e);
}

std::atomic<uint32_t> g_i8_wait_limit{kSpinLimit};

template <bool GROUPED>
int launch(const MulMatI8& o, cudaStream_t stream, int num_sms) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(o.w) | reinterpret_cast<uintptr_t>(o.q) |
                           static_cast<uintptr_t>(o.w_row_bytes) | static_cast<uintptr_t>(o.q_stride) |
                           static_cast<uintptr_t>(o.E > 1 ? o.w_expert_bytes : 0);
    if ((bits & 15) || !i8_encoder()) return launch_general<GROUPED>(o, stream, num_sms);
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return -static_cast<int>(e);
    if (dev < 0 || dev >= kMaxDevices) return -static_cast<int>(cudaErrorInvalidDevice);

    const Plan plan = wllm::plan<GROUPED>({o.M, o.K, o.N, o.E, o.slots}, num_sms);
    if (plan.items > 0x7fffffff) return -static_cast<int>(cudaErrorInvalidValue);
    I8Args P{};
    P.o = o;
    P.tile_n = plan.tile_n;
    P.splits = plan.splits;
    P.spin_limit = g_i8_wait_limit.load();
    const bool pair = is_pair(plan.mode);
    const int tile_m = pair ? 2 * kTileM : kTileM, sub = chunks_of_stage(plan.mode);
    P.tiles_m = (o.M + tile_m - 1) / tile_m;
    P.tiles_n = GROUPED ? 0 : (o.N - 1) / P.tile_n + 1;
    P.chunks = (o.K + sub * kChunk - 1) / (sub * kChunk);
    const int tokens = pair ? P.tile_n / 2 : P.tile_n;  // of a CTA's stage
    const int stage_bytes = sub * (kABytes + tokens * kChunk);
    P.stages = std::min(kMaxStages, (kSmemBytes - 1024) / stage_bytes);
    P.tmem_cols = 32;
    while (P.tmem_cols < 2 * P.tile_n) P.tmem_cols *= 2;
    {
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.K), static_cast<cuuint64_t>(o.M), static_cast<cuuint64_t>(o.E)};
        const cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.w_row_bytes),
                                       static_cast<cuuint64_t>(o.E > 1 ? o.w_expert_bytes : o.w_row_bytes * o.M)};
        if (!encode(&P.wmap, o.w, 3, dims, strides, kTileM)) return -static_cast<int>(cudaErrorInvalidValue);
    }
    if (!GROUPED) {
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(o.K), static_cast<cuuint64_t>(o.N)};
        const cuuint64_t strides[1] = {static_cast<cuuint64_t>(o.q_stride)};
        if (!encode(&P.xmap, o.q, 2, dims, strides, tokens)) return -static_cast<int>(cudaErrorInvalidValue);
    }
    void (*const kernels[4])(I8Args) = {i8_kernel<GROUPED, kSingle>, i8_kernel<GROUPED, kSplit>, i8_kernel<GROUPED, kPair>,
                                        i8_kernel<GROUPED, kPairShort>};
    static bool configured[kMaxDevices][4] = {};  // the attribute is per device
    if (!configured[dev][plan.mode]) {
        const cudaError_t e = cudaFuncSetAttribute(kernels[plan.mode], cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
        if (e != cudaSuccess) return -static_cast<int>(e);
        configured[dev][plan.mode] = true;
    }
    const int group = pair ? 2 : P.splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(
        plan.mode == kSplit ? plan.items * group : std::min<int64_t>(plan.items, num_sms / group) * group));
    cfg.blockDim = dim3(GROUPED ? kThreads + 2 * kLoaders : kThreads);
    cfg.dynamicSmemBytes = 1024 + P.stages * stage_bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(group);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = group > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernels[plan.mode], P);
    return e == cudaSuccess ? 1 : -static_cast<int>(e);
}

}  // namespace

// Whether there has been a launch whose waits could have given up: hosts that
// use none of this pay nothing for it in wllm_sync.
static bool g_i8_launched = false;

int launch_mul_mat_i8(const MulMatI8& o, cudaStream_t stream, int num_sms) {
    g_i8_launched = true;
    return launch<false>(o, stream, num_sms);
}
int launch_mul_mat_id_i8(const MulMatI8& o, cudaStream_t stream, int num_sms) {
    g_i8_launched = true;
    return launch<true>(o, stream, num_sms);
}

void set_i8_wait_limit(uint32_t polls) { g_i8_wait_limit.store(polls ? polls : kSpinLimit); }

unsigned read_and_clear_i8_error() {
    if (!g_i8_launched) return 0;
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_i8_error, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
    if (v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(g_i8_error, &z, sizeof(z));
    }
    return v;
}

}  // namespace wllm
