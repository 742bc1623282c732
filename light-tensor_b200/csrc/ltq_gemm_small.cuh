// Host-visible interface of the product kernel for calls with few output tiles (ltq_gemm_small.cu).
#pragma once
#include "ltq_common.cuh"
#include "ltq_gemm_tc.cuh"

namespace ltq {

// Tile width (a multiple of 16, at most 128), the number of CTAs that share a tile's K, 128-byte lines of K per copy, and how often
// that fills the device.
struct SmallPlan {
    uint32_t bn, split, lines, rounds;
};
SmallPlan small_plan(uint64_t M, uint64_t N, uint64_t K, int sms);
// Encodes the activation map and, unless *map_b fits already, the weight map.  0 on success.
int small_maps(const SmallPlan &p, const uint8_t *A, uint64_t M, uint64_t K, TcOperandMap *map_a, const uint8_t *B, uint64_t N, TcOperandMap *map_b);
// Token output modes only.  `early_weights`: see launch_gemv.
cudaError_t launch_gemm_small(const TcOperandMap &map_a, const TcOperandMap &map_b, const SmallPlan &p, uint64_t M, uint64_t N, uint64_t K,
                              const Epilogue &epi, void *out, uint32_t *status, cudaStream_t stream, bool early_weights);

}  // namespace ltq
