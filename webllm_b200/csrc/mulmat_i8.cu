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
//  - warp 0 (TMA): per 128-byte chunk of K one box of 128 weight rows and the
//    tile's token rows into a ring of stages (K-major, 128-byte swizzle). Dense
//    tokens come as one box; an expert's tokens are gathered, four rows a copy
//    (tile::gather4), through the sorted slots, so no sorted copy of the
//    activations is ever written.
//  - warp 1 (MMA): one thread issues the 4 K=32 MMAs of a chunk.
//  - warps 2..5 (epilogue): TMEM -> scales -> y, while the next tile's MMAs
//    fill the other accumulator.
//
// CTAs are persistent over the items (expert, channel tile, token tile). Where
// the items are fewer than the SMs (single tokens, small batches), S = 2, 4 or
// 8 CTAs of a cluster share an item's K: each leaves its int32 tile in its own
// shared memory, and after a cluster barrier CTA r adds the S tiles of its
// share of the columns through distributed shared memory.
//
// Bounds: HBM (the weights, once) up to a few hundred tokens, the tensor pipe
// above.
//
// Every mbarrier wait is bounded: on time-out the CTA records an error code
// (read by wllm_sync), stops issuing, waits for its copies and MMAs in flight
// and frees its TMEM.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>

#include "wllm_internal.h"

namespace wllm {

__device__ unsigned int g_i8_error = 0;

namespace {

constexpr int kTileM = 128;    // channels of a tile
constexpr int kMaxTileN = 256; // tokens of a tile
constexpr int kChunk = 128;    // bytes of K of a stage
constexpr int kABytes = kTileM * kChunk;
constexpr int kThreads = 192;
constexpr int kMaxStages = 12;
constexpr int kSmemBytes = 220 * 1024;  // dynamic, beside about 5 KB of tables and barriers
constexpr uint32_t kSpinLimit = 1u << 26;

struct I8Args {
    CUtensorMap wmap;  // weights: [E][M][K] bytes, box 128 x 128 x 1
    CUtensorMap xmap;  // tokens: [rows][K] bytes, box 128 x tile_n (dense) or 128 x 1 (gathered)
    MulMatI8 o;
    int32_t tile_n;    // tokens of a full tile, a multiple of 16
    int32_t tiles_m, chunks, stages, splits;
    int32_t tmem_cols;
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
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, unsigned code, volatile int* poisoned) {
    for (uint32_t i = 0; i < kSpinLimit; ++i) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 255u) == 255u && *poisoned) return false;
    }
    *poisoned = 1;
    atomicOr(&g_i8_error, code);
    return false;
}
// Bounded wait whatever the poison flag says, for what is in flight at exit.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < kSpinLimit; ++i)
        if (mbar_try(bar, parity)) return;
    atomicOr(&g_i8_error, 8u);
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
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(tm), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}
// Four rows of 128 bytes from byte x on.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* tm, int x, int4 rows, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(tm), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* tm, int x, int y, int z) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(tm), "r"(x), "r"(y), "r"(z) : "memory");
}

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
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int32_t ld_cluster(uint32_t local, uint32_t rank) {
    uint32_t remote;
    int32_t v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
    return v;
}

// y[row][m] in y's type: the two scales in f32, then one rounding.
__device__ __forceinline__ void store_y(const MulMatI8& o, int64_t row, int m, int32_t acc, float s, float t) {
    const float v = __fmul_rn(__fmul_rn(__int2float_rn(acc), s), t);
    const int64_t at = row * o.y_stride + m;
    if (o.y_type == kTypeF32) static_cast<float*>(o.y)[at] = v;
    else if (o.y_type == kTypeF16) static_cast<__half*>(o.y)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(o.y)[at] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ void zero_y(const MulMatI8& o, int64_t row, int m) {
    const int64_t at = row * o.y_stride + m;
    if (o.y_type == kTypeF32) static_cast<float*>(o.y)[at] = 0.f;
    else static_cast<uint16_t*>(o.y)[at] = 0;
}

// An item: `rows` token rows from position `first` on, of expert e, against
// channels m0.. . A group's token tiles are of one size (the least multiple of
// 16 that covers it in as many tiles), its channel tiles come one after the
// other with the token tiles of one channel tile next to each other (they read
// the same weights).
struct Item {
    int e, m0, first, rows;
};

// Rows of each of the `tiles` tiles of a group of n.
__device__ __forceinline__ int tile_rows(int n, int tiles) { return ((n + tiles - 1) / tiles + 15) & ~15; }

// cum[e]: token tiles of the experts before e (GROUPED); E + 1 entries.
template <bool GROUPED>
__device__ __forceinline__ Item item_of(const I8Args& P, const int32_t* cum, int64_t i) {
    Item it;
    if constexpr (!GROUPED) {
        const int tiles = (P.o.N + P.tile_n - 1) / P.tile_n;
        it.e = 0;
        it.m0 = static_cast<int>(i / tiles) * kTileM;
        it.first = static_cast<int>(i % tiles) * P.tile_n;
        it.rows = min(P.tile_n, P.o.N - it.first);
    } else {
        const int64_t u = i / P.tiles_m;  // the token tile that holds the item if groups had one channel tile
        int lo = 0, hi = P.o.E - 1;       // the last expert whose first tile is at or before u
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cum[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        const int tiles = cum[lo + 1] - cum[lo];
        const int j = static_cast<int>(i - static_cast<int64_t>(cum[lo]) * P.tiles_m);
        const int begin = P.o.offsets[lo], n = P.o.offsets[lo + 1] - begin;
        const int size = tile_rows(n, tiles);
        it.e = lo;
        it.m0 = (j / tiles) * kTileM;
        it.first = begin + (j % tiles) * size;
        it.rows = min(size, begin + n - it.first);
    }
    return it;
}

// GROUPED: tokens by expert. SPLIT: a cluster of P.splits CTAs shares an item's
// K (one item per cluster).
template <bool GROUPED, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) i8_kernel(const __grid_constant__ I8Args P) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_free[2];
    __shared__ uint32_t tmem_slot;
    __shared__ int poison;
    __shared__ int32_t cum[GROUPED ? kMaxExperts + 1 : 1];
    __shared__ int32_t warp_sum[GROUPED ? kThreads / 32 : 1];
    // 1024-byte alignment for the swizzled tiles
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    volatile int* poisoned = &poison;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int stages = P.stages, stage_bytes = kABytes + P.tile_n * kChunk;
    const uint32_t rank = SPLIT ? blockIdx.x % P.splits : 0;
    const int c0 = SPLIT ? static_cast<int>(static_cast<int64_t>(P.chunks) * rank / P.splits) : 0;
    const int c1 = SPLIT ? static_cast<int>(static_cast<int64_t>(P.chunks) * (rank + 1) / P.splits) : P.chunks;
    const int64_t item0 = SPLIT ? blockIdx.x / P.splits : blockIdx.x;
    const int64_t item_step = SPLIT ? gridDim.x / P.splits : gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_free[b], 4);
        }
        poison = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&P.wmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&P.xmap) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(P.tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");

    int64_t items;
    if constexpr (GROUPED) {
        // token tiles of each expert, then their running sum
        int carry = 0;
        for (int base = 0; base < P.o.E; base += kThreads) {
            const int e = base + threadIdx.x;
            int tiles = 0;
            if (e < P.o.E) tiles = (P.o.offsets[e + 1] - P.o.offsets[e] + P.tile_n - 1) / P.tile_n;
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
            for (int w = 0; w < kThreads / 32; ++w) {
                if (w < warp) before += warp_sum[w];
                carry += warp_sum[w];
            }
            if (e < P.o.E) cum[e + 1] = before + sum;
        }
        if (threadIdx.x == 0) cum[0] = 0;
        items = static_cast<int64_t>(carry) * P.tiles_m;
    } else {
        items = static_cast<int64_t>((P.o.N + P.tile_n - 1) / P.tile_n) * P.tiles_m;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        // ---------------- copies ----------------
        uint32_t q = 0;  // stages filled so far
        bool ok = true;
        for (int64_t i = item0; i < items && ok; i += item_step) {
            const Item it = item_of<GROUPED>(P, cum, i);
            const int cols = (it.rows + 15) & ~15;
            int4 rows[2];
            if constexpr (GROUPED) {
                // copies lane and lane + 32 of the item: four token rows each; what
                // is behind the last row reads that row again
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    int r[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int slot = P.o.order[it.first + min((lane + 32 * g) * 4 + j, it.rows - 1)];
                        r[j] = P.o.per_slot ? slot : slot / P.o.k;
                    }
                    rows[g] = make_int4(r[0], r[1], r[2], r[3]);
                }
            }
            for (int c = c0; c < c1; ++c, ++q) {
                const int s = q % stages;
                if (q >= static_cast<uint32_t>(stages) && !mbar_wait(&empty[s], ((q / stages) - 1) & 1, 1u, poisoned)) {
                    ok = false;
                    break;
                }
                const uint32_t a = smem_u32(smem + s * stage_bytes), b = a + kABytes;
                if constexpr (GROUPED) {
                    if (lane == 0) {
                        mbar_expect_tx(&full[s], kABytes + cols * kChunk);
                        tma_3d(a, &P.wmap, c * kChunk, it.m0, it.e, &full[s]);
                    }
                    __syncwarp();
                    for (int g = 0; g < 2; ++g)
                        if ((lane + 32 * g) * 4 < cols)
                            tma_gather4(b + (lane + 32 * g) * 4 * kChunk, &P.xmap, c * kChunk, g ? rows[1] : rows[0], &full[s]);
                } else if (lane == 0) {
                    mbar_expect_tx(&full[s], kABytes + P.tile_n * kChunk);
                    tma_3d(a, &P.wmap, c * kChunk, it.m0, 0, &full[s]);
                    tma_2d(b, &P.xmap, c * kChunk, it.first, &full[s]);
                }
                __syncwarp();
            }
            ok = __all_sync(0xffffffffu, ok);
        }
        if (!ok || *poisoned) {  // the copies in flight land before the CTA ends
            for (uint32_t p = q > static_cast<uint32_t>(stages) ? q - stages : 0; p < q; ++p)
                mbar_drain(&full[p % stages], (p / stages) & 1);
        }
    } else if (warp == 1) {
        // ---------------- MMAs ----------------
        if (lane == 0) {
            uint32_t q = 0, t = 0;
            bool ok = true;
            for (int64_t i = item0; i < items && ok; i += item_step, ++t) {
                const Item it = item_of<GROUPED>(P, cum, i);
                const uint32_t idesc = i8_idesc(kTileM, (it.rows + 15) & ~15);
                const uint32_t buf = t & 1, d = tmem + buf * P.tile_n;
                if (t >= 2 && !mbar_wait(&acc_free[buf], ((t >> 1) - 1) & 1, 2u, poisoned)) break;
                tc_fence_after();
                for (int c = c0; c < c1; ++c, ++q) {
                    const int s = q % stages;
                    if (!mbar_wait(&full[s], (q / stages) & 1, 4u, poisoned)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem + s * stage_bytes);
                    const uint64_t ad = umma_desc(a), bd = umma_desc(a + kABytes);
#pragma unroll
                    for (int j = 0; j < kChunk / 32; ++j) umma_i8(d, ad + 2 * j, bd + 2 * j, idesc, c > c0 || j > 0);
                    umma_commit(&empty[s]);
                }
                umma_commit(&acc_full[buf]);
            }
            // MMAs still in flight (only after a time-out) end before the TMEM is freed
            if (*poisoned && q > 0) mbar_drain(&empty[(q - 1) % stages], ((q - 1) / stages) & 1);
        }
    } else {
        // ---------------- epilogue ----------------
        const int quad = warp & 3;  // the TMEM lanes this warp may read
        uint32_t t = 0;
        for (int64_t i = item0; i < items; i += item_step, ++t) {
            const Item it = item_of<GROUPED>(P, cum, i);
            const uint32_t buf = t & 1;
            const int m = it.m0 + 32 * quad + lane;
            const float tm = m < P.o.M ? P.o.w_scale[static_cast<int64_t>(it.e) * P.o.M + m] : 0.f;
            if (!mbar_wait(&acc_full[buf], (t >> 1) & 1, 2u, poisoned)) break;
            tc_fence_after();
            for (int n = 0; n < it.rows; n += 16) {
                int32_t acc[16];
                tmem_ld16(tmem + buf * P.tile_n + n + (static_cast<uint32_t>(32 * quad) << 16), acc);
                if constexpr (SPLIT) {
                    // the stages are free by now: all copies have landed and all MMAs have read them
                    int32_t* part = reinterpret_cast<int32_t*>(smem);
#pragma unroll
                    for (int j = 0; j < 16; ++j) part[(n + j) * kTileM + 32 * quad + lane] = acc[j];
                } else {
                    // lane j < 16 fetches column j's output row and scale
                    int row = 0;
                    float s = 0.f;
                    if (n + (lane & 15) < it.rows) {
                        row = it.first + n + (lane & 15);
                        if constexpr (GROUPED) row = P.o.order[row];
                        s = P.o.q_scale[!GROUPED || P.o.per_slot ? row : row / P.o.k];
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int rj = __shfl_sync(0xffffffffu, row, j);
                        const float sj = __shfl_sync(0xffffffffu, s, j);
                        if (n + j < it.rows && m < P.o.M) store_y(P.o, rj, m, acc[j], sj, tm);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_free[buf]);
        }
    }
    if constexpr (SPLIT) {
        // one item per cluster, so that the sum over the splits comes after all roles
        __syncwarp();
        cluster_sync();
        if (item0 < items && !*poisoned) {
            const Item it = item_of<GROUPED>(P, cum, item0);
            const uint32_t part = smem_u32(smem);
            const int per = (it.rows + P.splits - 1) / P.splits, n0 = rank * per, n1 = min(n0 + per, it.rows);
            for (int x = n0 * kTileM + threadIdx.x; x < n1 * kTileM; x += kThreads) {
                const int n = x / kTileM, m = it.m0 + x % kTileM;
                if (m >= P.o.M) continue;
                int32_t acc = 0;
                for (int r = 0; r < P.splits; ++r) acc += ld_cluster(part + 4 * x, r);
                int row = it.first + n;
                if constexpr (GROUPED) row = P.o.order[row];
                const float s = P.o.q_scale[!GROUPED || P.o.per_slot ? row : row / P.o.k];
                store_y(P.o, row, m, acc, s, P.o.w_scale[static_cast<int64_t>(it.e) * P.o.M + m]);
            }
        }
        cluster_sync();  // no CTA ends while another reads its tile
    }
    if constexpr (GROUPED) {
        // slots without an expert come last in the order: their rows are zero
        for (int64_t p = P.o.offsets[P.o.E] + blockIdx.x; p < P.o.slots; p += gridDim.x) {
            const int64_t row = P.o.order[p];
            for (int m = threadIdx.x; m < P.o.M; m += kThreads) zero_y(P.o, row, m);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P.tmem_cols));
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
                if (lane == 0) zero_y(o, row, m);
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
        if (lane == 0) store_y(o, row, m, acc, o.q_scale[from], o.w_scale[static_cast<int64_t>(e) * o.M + m]);
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

template <bool GROUPED, bool SPLIT>
cudaError_t configure(int dev) {
    static bool done[kMaxDevices] = {};  // the attribute is per device
    if (done[dev]) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(i8_kernel<GROUPED, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    done[dev] = e == cudaSuccess;
    return e;
}

template <bool GROUPED>
int launch(const MulMatI8& o, cudaStream_t stream, int num_sms) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(o.w) | reinterpret_cast<uintptr_t>(o.q) |
                           static_cast<uintptr_t>(o.w_row_bytes) | static_cast<uintptr_t>(o.q_stride) |
                           static_cast<uintptr_t>(o.E > 1 ? o.w_expert_bytes : 0);
    if ((bits & 15) || !i8_encoder()) return launch_general<GROUPED>(o, stream, num_sms);
    int dev = 0;
    if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return -static_cast<int>(e);
    if (dev < 0 || dev >= kMaxDevices) return -static_cast<int>(cudaErrorInvalidDevice);

    I8Args P{};
    P.o = o;
    P.tiles_m = (o.M + kTileM - 1) / kTileM;
    P.chunks = (o.K + kChunk - 1) / kChunk;
    // tokens of a tile, and how many items there are at most
    int64_t items;
    if (GROUPED) {
        // an expert's mean share, doubled (groups are ragged), in tiles of at most 256
        const int64_t mean = (2 * o.slots + o.E - 1) / o.E;
        P.tile_n = static_cast<int>(std::min<int64_t>(kMaxTileN, std::min<int64_t>((mean + 15) / 16 * 16, (o.slots + 15) / 16 * 16)));
        items = std::min<int64_t>(o.slots, o.slots / P.tile_n + o.E) * P.tiles_m;
    } else {
        const int tiles = (o.N + kMaxTileN - 1) / kMaxTileN;
        P.tile_n = ((o.N + tiles - 1) / tiles + 15) / 16 * 16;
        items = static_cast<int64_t>((o.N + P.tile_n - 1) / P.tile_n) * P.tiles_m;
    }
    P.splits = 1;
    if (P.tile_n <= 64)
        while (P.splits < 8 && items * P.splits * 2 <= num_sms && P.chunks >= P.splits * 4) P.splits *= 2;
    const int stage_bytes = kABytes + P.tile_n * kChunk;
    P.stages = std::min(kMaxStages, (kSmemBytes - 1024) / stage_bytes);
    P.tmem_cols = 32;
    while (P.tmem_cols < 2 * P.tile_n) P.tmem_cols *= 2;
    {
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(o.K), static_cast<cuuint64_t>(o.M), static_cast<cuuint64_t>(o.E)};
        const cuuint64_t strides[2] = {static_cast<cuuint64_t>(o.w_row_bytes),
                                       static_cast<cuuint64_t>(o.E > 1 ? o.w_expert_bytes : o.w_row_bytes * o.M)};
        if (!encode(&P.wmap, o.w, 3, dims, strides, kTileM)) return -static_cast<int>(cudaErrorInvalidValue);
    }
    {
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(o.K), static_cast<cuuint64_t>(o.N)};
        const cuuint64_t strides[1] = {static_cast<cuuint64_t>(o.q_stride)};
        if (!encode(&P.xmap, o.q, 2, dims, strides, GROUPED ? 1 : P.tile_n)) return -static_cast<int>(cudaErrorInvalidValue);
    }
    const bool split = P.splits > 1;
    if (const cudaError_t e = split ? configure<GROUPED, true>(dev) : configure<GROUPED, false>(dev); e != cudaSuccess)
        return -static_cast<int>(e);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(split ? items * P.splits : std::min<int64_t>(items, num_sms)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = 1024 + P.stages * stage_bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(P.splits);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, split ? i8_kernel<GROUPED, true> : i8_kernel<GROUPED, false>, P);
    return e == cudaSuccess ? 1 : -static_cast<int>(e);
}

}  // namespace

int launch_mul_mat_i8(const MulMatI8& o, cudaStream_t stream, int num_sms) { return launch<false>(o, stream, num_sms); }
int launch_mul_mat_id_i8(const MulMatI8& o, cudaStream_t stream, int num_sms) { return launch<true>(o, stream, num_sms); }

unsigned read_and_clear_i8_error() {
    unsigned v = 0;
    if (cudaMemcpyFromSymbol(&v, g_i8_error, sizeof(v)) != cudaSuccess) return 0xFFFFFFFFu;
    if (v) {
        const unsigned z = 0;
        cudaMemcpyToSymbol(g_i8_error, &z, sizeof(z));
    }
    return v;
}

}  // namespace wllm
