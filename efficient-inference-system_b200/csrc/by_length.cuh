// by_length.cuh -- the order in which CTAs take a batch's sequences.
//
// CTAs start in the order of their numbers.  Where they are more than fit the
// GPU at once and sequences differ in length, a long one that starts late is
// what the GPU waits for at the end: number z therefore takes the z-th longest.
// Each CTA ranks for itself, about 1 us before its first key, so it pays where
// shares are long and waves few.  As they come -> longest first, lengths from an
// eighth of the longest up, us: 4-bit decode (bf16, B x H sequences and heads)
//   head_dim 64, 64 x 8: longest 256 9.1 -> 10.4, 1,024 17.1 -> 16.0, 2,048
//   27.2 -> 22.9; 100 x 16: 512 29.4 -> 35.3, 2,048 61.2 -> 64.9;
//   head_dim 128, 64 x 32: 8,192 301 -> 280;
//   head_dim 256, 64 x 8: 1,024 43.1 -> 34.5; 100 x 16: 512 60.5 -> 65.8, 2,048
//   172.8 -> 169.5;
// key weights of one query, 32 x 32: 4-bit keys of 128 channels 512 16.0 -> 16.9,
//   1,024 26.1 -> 25.1, 8,192 136 -> 119; bf16 of 128 8,192 257 -> 228, of 64 4,096
//   71.3 -> 70.7, 8,192 134 -> 127 (64 x 32: 239 -> 246), of 256 1,024 59.2 -> 66.8,
//   4,096 204 -> 207 (never faster); fp32 of 64 512 37.7 -> 33.2, 4,096 218 -> 172.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace b2pa {

constexpr int kOrdered = 128;  // sequences at most: a thread ranks one against all

// The index of the z-th longest of B sequences (ties: the lower index first),
// for a whole CTA of at least kOrdered threads; two __syncthreads and a few
// hundred instructions.
__device__ __forceinline__ int nth_longest(const int32_t* seq_lens, int B, int z) {
  __shared__ __align__(16) int32_t lens[kOrdered];
  __shared__ int found;
  const int i = threadIdx.x;
  int mine = 0;
  if (i < kOrdered) lens[i] = mine = i < B ? seq_lens[i] : INT32_MIN;
  __syncthreads();
  if (i < B) {
    int above = 0;
    for (int j = 0; j < B; j += 4) {
      const int4 x = *reinterpret_cast<const int4*>(lens + j);
      above += (x.x > mine || (x.x == mine && j < i)) + (x.y > mine || (x.y == mine && j + 1 < i)) +
               (x.z > mine || (x.z == mine && j + 2 < i)) + (x.w > mine || (x.w == mine && j + 3 < i));
    }
    if (above == z) found = i;
  }
  __syncthreads();
  return found;
}

// Worth it?  Every wave of CTAs (`per_sm` on an SM) pays the ranking, and the end
// comes earlier by a part of the longest CTA's time, which has `keys`: at least
// `least`, and more than `per_wave` for every wave behind the first.
inline int orders_by_length(int B, int64_t ctas, int per_sm, int64_t keys, int least, int64_t per_wave) {
  const int64_t wave = (int64_t)per_sm * device_sm_count();
  return B > 1 && B <= kOrdered && keys >= least && ctas > wave && keys * wave > per_wave * (ctas - wave);
}

}  // namespace b2pa
