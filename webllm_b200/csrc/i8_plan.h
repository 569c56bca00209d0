// What the 8-bit and mixture-of-experts launches and kernels decide from sizes
// alone: plain arithmetic, without CUDA, so that it can be checked on the host
// over every size.
#pragma once
#include <stdint.h>

#include <algorithm>

#ifdef __CUDACC__
#define WLLM_HD __host__ __device__
#else
#define WLLM_HD
#endif

namespace wllm {

// How many bytes of a row of K the 16-byte piece at byte k holds: what a copy of
// it reads, so that nothing behind the row is.
WLLM_HD constexpr int piece_bytes(int K, int k) { return k >= K ? 0 : (K - k < 16 ? K - k : 16); }

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
