// Noise of the draws without given numbers (decode.cu, draw.cu): the token drawn is the first with the largest of logit / T - log(-log(x)), x
// uniform in (0, 1) by a hash of (seed, step, row, token).  One form for all kernels, so that a seed gives the same tokens by each of them.
#pragma once
#include "common.cuh"

namespace apb {

__device__ __forceinline__ uint32_t hash_u32(uint32_t x) {
  x ^= x >> 16;
  x *= 0x7feb352dU;
  x ^= x >> 15;
  x *= 0x846ca68bU;
  x ^= x >> 16;
  return x;
}
// The part of (seed, step, row), mixed once; a token's hash is one more round over it and a Weyl step.
__device__ __forceinline__ uint32_t noise_base(uint32_t seed, uint32_t step, int row) {
  return hash_u32(seed ^ (step * 0x9E3779B9u)) ^ hash_u32(static_cast<uint32_t>(row) * 0x85ebca6bU + 1u);
}
// x is the middle of one of 2^24 steps.  The middle of the last one, 1 - 2^-25, rounds to 1 in fp32, whose logarithm is 0 and would make the
// noise infinite, so that a token with that hash (one of 2^24) would win whatever its logit is: its -log(x) is 2^-25.  Every other x has a larger
// one, by the approximate logarithm too (0.68e-7 at least, over all of them), and keeps it.
__device__ __forceinline__ float draw_noise(uint32_t base, int token) {
  const uint32_t h = hash_u32(base + static_cast<uint32_t>(token) * 0x9E3779B9u);
  const float x = (static_cast<float>(h >> 8) + 0.5f) * (1.f / 16777216.f);
  return -__logf(fmaxf(-__logf(x), 0x1p-25f));
}

}  // namespace apb
