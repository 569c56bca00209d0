// What the 8-bit and mixture-of-experts launches and kernels decide from sizes
// alone: plain arithmetic, without CUDA, so that it can be checked on the host
// over every size.
#pragma once
#include <stdint.h>

#include <algorithm>
#include <cmath>

#ifdef __CUDACC__
#define WLLM_HD __host__ __device__
#else
#define WLLM_HD
#endif

namespace wllm {

// How many bytes of a row of K the 16-byte piece at byte k holds: what a copy of
// it reads, so that nothing behind the row is.
WLLM_HD constexpr int piece_bytes(int K, int k) { return k >= K ? 0 : (K - k < 16 ? K - k : 16); }

constexpr int kTileM = 128;    // channels of a tile
constexpr int kMaxTileN = 256; // tokens of a pair's tile
constexpr int kMaxShortN = 128; // of a pair's with two chunks a stage
constexpr int kMaxSingleN = 64; // of a single CTA's or a split one
constexpr int kChunk = 128;    // bytes of K of a swizzled row
constexpr int kABytes = kTileM * kChunk;

enum Mode : int { kSingle = 0, kSplit = 1, kPair = 2, kPairShort = 3 };
// Chunks of a stage. A stage costs its copy and MMA warps some 350 clocks of
// waits and issue whatever its size; the MMAs of a pair's chunk with 256 tokens
// take 512, those of fewer tokens less, so there (kPairShort: at most 128
// tokens) two chunks share a stage.
WLLM_HD constexpr int chunks_of_stage(int mode) { return mode == kPair ? 1 : 2; }
WLLM_HD constexpr bool is_pair(int mode) { return mode >= kPair; }

// A product's sizes: N dense tokens, or `slots` in E experts.
struct I8Shape {
    int M, K, N, E;
    int64_t slots;
};
// The mode, the token tile, the split of K and how many items there are at most.
struct Plan {
    Mode mode;
    int tile_n, splits;
    int64_t items;
};

// Clocks that a launch is expected to take, from what its parts were measured
// to: a stage costs its MMAs, its bytes from L2 (57 a clock and SM, 45 over all
// SMs), or the 380 clocks of its waits and issue; an item some 600 more, where K
// is split 4000 and 50 a token (the cluster's start and barrier, the sum of the
// tiles). Clusters of 2, 4 and 8 leave SMs of a GPC unused. What HBM adds is the
// same for all plans. Grouped, the items are the expected ones of an even
// routing. (Against the best of all plans, forced one by one, over 20 shapes
// from 1 x 4096 x 4096 to 2000 tokens in 4 of 256 experts: within 15% but for one
// at 19%.)
template <bool GROUPED>
double clocks(const I8Shape& o, const Plan& p, int num_sms, double used) {
    const bool pair = is_pair(p.mode);
    const int sub = chunks_of_stage(p.mode), step = pair ? 32 : 16, tile_m = pair ? 2 * kTileM : kTileM;
    const double tiles_m = (o.M + tile_m - 1) / tile_m;
    double items, cols = p.tile_n;
    if (GROUPED) {
        const double mean = o.slots / used;
        const double tiles = mean <= p.tile_n / 2 ? 1.0 : mean / p.tile_n + 0.5;  // of an expert, ragged groups among them
        items = used * tiles * tiles_m;
        cols = std::min<double>(p.tile_n, std::ceil(mean / tiles / step) * step);
    } else {
        items = static_cast<double>((o.N - 1) / p.tile_n + 1) * tiles_m;
    }
    const int lost = p.splits == 8 ? 4 : (p.splits == 4 ? 3 : (p.splits == 2 ? 2 : 0));
    const double units = std::max(1, num_sms / (pair ? 2 : p.splits) - lost);
    const double waves = GROUPED ? std::max(1.0, items / units + 0.5) : std::ceil(items / units);
    const int chunks = (o.K + sub * kChunk - 1) / (sub * kChunk);
    const double mma = 4.0 * sub * std::max(36.0, cols / 2), bytes = sub * (kABytes + (pair ? cols / 2 : cols) * kChunk);
    const double stage = std::max(380.0, std::max(mma, bytes / 57));
    const double own = waves * ((chunks + p.splits - 1) / p.splits * stage + (p.splits > 1 ? 4000.0 + 50 * cols : 600.0));
    return std::max(own, items * chunks * bytes * (pair ? 2 : 1) / (45.0 * num_sms));
}

template <bool GROUPED>
Plan plan(const I8Shape& o, int num_sms) {
    Plan best{};
    double best_clocks = 0;
    // experts that an even routing reaches
    const double used = GROUPED ? std::max(1.0, o.E * (1.0 - std::exp(-static_cast<double>(o.slots) / o.E))) : 1.0;
    auto consider = [&](Mode mode, int tile_n, int splits) {
        const Plan p{mode, tile_n, splits, 0};
        const double c = clocks<GROUPED>(o, p, num_sms, used);
        if (best.tile_n == 0 || c < best_clocks) best = p, best_clocks = c;
    };
    // token tiles worth a look: of a dense product those that cover N in equal
    // parts, as few as the mode allows or up to seven more; of groups all sizes
    // up to the slots
    auto sizes = [&](int most, int step, auto&& use) {
        if (GROUPED) {
            for (int n = step; n <= most; n += n < 64 ? step : 64) {
                use(n);
                if (n >= o.slots) break;
            }
        } else {
            const int least = (o.N - 1) / most + 1;
            for (int tiles = least; tiles < least + 8; ++tiles) {
                const int n = ((o.N - 1) / tiles + step) / step * step;  // (N + tiles may pass 2^31)
                use(n);
                if (n == step) break;
            }
        }
    };
    const int chunks = (o.K + 2 * kChunk - 1) / (2 * kChunk);
    sizes(kMaxSingleN, 16, [&](int n) {
        for (int s = 1; s <= 8 && s <= chunks; s *= 2) consider(s > 1 ? kSplit : kSingle, n, s);
    });
    if (o.M > kTileM) sizes(kMaxTileN, 32, [&](int n) { consider(n <= kMaxShortN ? kPairShort : kPair, n, 1); });
    const int tile_m = is_pair(best.mode) ? 2 * kTileM : kTileM;
    const int64_t tiles_m = (o.M + tile_m - 1) / tile_m;
    // of groups at most one started tile more than the whole ones of each expert
    best.items = tiles_m * (GROUPED ? std::min<int64_t>(o.slots, o.slots / best.tile_n + o.E) : (o.N - 1) / best.tile_n + 1);
    return best;
}

// The launch of wllm_moe_plan: 64 slots a warp before there is another warp (four
// at least, for the walks over the keys), all warps of a CTA before another CTA.
// Up to `most` CTAs, one cluster: 16 where the device can place one (65,536 slots,
// 128 experts: 10 us), otherwise the 8 that every device can (17 us).
constexpr int kPlanWarps = 32;
constexpr int kPlanCtas = 16;
constexpr int kPortableCtas = 8;
struct PlanShape {
    int warps, ctas, smem;
};
WLLM_HD constexpr int plan_smem(int warps, int E) { return (warps + 2) * (E + 1) * 4; }
inline PlanShape plan_shape(int64_t slots, int E, int most) {
    const int64_t want = std::max<int64_t>(4, (slots + 63) / 64);
    const int warps = static_cast<int>(std::min<int64_t>(kPlanWarps, want));
    return {warps, static_cast<int>(std::min<int64_t>(most, (want + kPlanWarps - 1) / kPlanWarps)), plan_smem(warps, E)};
}

}  // namespace wllm
