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

}  // namespace wllm
