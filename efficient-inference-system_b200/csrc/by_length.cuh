// by_length.cuh -- the order in which CTAs take a batch's sequences.
//
// CTAs start in the order of their numbers.  Where they are more than fit the
// GPU at once and sequences differ in length, a long one that starts late is
// what the GPU waits for at the end: number z therefore takes the z-th longest.
// As they come -> longest first (lengths U[1,024, 8,192], in us): 4-bit decode of
// 64 sequences and 32 heads of 128 292 -> 274, of 8 and 16 heads of 256 74 ->
// 61; key weights of one query on 32 sequences and 32 heads of 128, 4-bit keys,
// 132 -> 116; where all fit at once it would cost about 1 us.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace b2pa {

constexpr int kOrdered = 128;  // sequences at most: a thread ranks one against all

// The index of the z-th longest of B sequences (ties: the lower index first),
// for a whole CTA of at least kOrdered threads; one __syncthreads and a few
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

// Worth it: more CTAs than the GPU holds at once, `per_sm` on an SM.
inline int orders_by_length(int B, int64_t ctas, int per_sm) {
  return B > 1 && B <= kOrdered && ctas > (int64_t)per_sm * device_sm_count();
}

}  // namespace b2pa
