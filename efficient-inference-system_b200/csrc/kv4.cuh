// kv4.cuh -- the 4-bit page format of the KV cache.
//
// A row of D channels (one token, one head, K or V) is cut into groups of
// 16.  A group stores a scale s and 16 codes c in -7..7; it stands for the
// values c * s.
//
//   s: an unsigned 8-bit float with 5 exponent and 3 mantissa bits.  The byte
//      shifted left by 7 is the fp16 number (range 2^-17 .. 9216 here), so a
//      group keeps its relative precision over the whole range of activations
//      without a second, per-tensor factor.  s = max|x| / 7 rounded to
//      nearest even; the cap keeps 7 * s finite in fp16 (64,512).  The byte
//      255 (an fp16 NaN) marks a group that held a NaN or an infinity.
//   c: round-to-nearest-even(x / s), clamped to -7..7, stored as c + 8.
//      c * s has at most 7 significant bits: exact in bf16, fp16 and fp32.
//
// Both quotients are single correctly rounded fp32 divisions.  That decides
// as exact arithmetic would: a border t of either rounding times its divisor
// d (7, or a scale of 4 significant bits) is representable, and the fp32
// neighbours of t * d lie more than half an ulp of t away from t after the
// division (ulp(t * d) / d > ulp(t) / 2 as d's significand is below 2), so
// no x off the border is rounded onto it.
//
// 4.5 bits a value.  Uniform levels rather than a 4-bit float: with one scale
// per 16 values the group maximum sits at the last level, and uniform steps
// of s give a mean squared error of s^2 / 12 over the whole range, where
// e2m1 (steps of s/2, s and 2s of its own scale max/6) gives 1.4 times that
// for normally distributed rows.
//
// A head page of block_size rows is 9/16 * block_size * D bytes:
//   codes  [block_size][D / 2], channel 2i in the low nibble of byte i;
//   scales [block_size][D / 16] in the K pool, [D / 16][block_size] in the V
//   pool: the decode kernel wants, per thread, neighbouring groups of one key
//   for K and neighbouring keys of one group for V.
// Pools are uint8 [num_blocks, H, block_size, D * 9 / 16], contiguous.
#pragma once

#include "common.cuh"

namespace b2pa {

__host__ __device__ constexpr int kv4_page_bytes(int block_size, int D) { return block_size * (D / 16) * 9; }

constexpr uint32_t kKv4NanScale = 255;
constexpr uint32_t kKv4MaxScale = 225;  // 9216

__device__ __forceinline__ float kv4_scale(uint32_t code) {
  return __half2float(__ushort_as_half((unsigned short)(code << 7)));
}

// Scale code of a group from the bits of its largest magnitude (a NaN's or
// infinity's bits compare above every finite one's).
__device__ __forceinline__ uint32_t kv4_scale_code(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return kKv4NanScale;
  const float y = __fdiv_rn(__uint_as_float(max_bits), 7.0f);
  if (y < 0x1p-14f) return (uint32_t)__float2int_rn(y * 0x1p17f);
  uint32_t u = __float_as_uint(y);
  u += 0x7ffffu + ((u >> 20) & 1u);
  const uint32_t code = (((u >> 23) - 112u) << 3) | ((u >> 20) & 7u);
  return code < kKv4MaxScale ? code : kKv4MaxScale;
}

// Eight codes of one group, packed; s is the value of its scale code.
__device__ __forceinline__ uint32_t kv4_pack8(const float* x, float s) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int c = 0;
    if (s > 0.f) {  // false for a zero scale and for a NaN
      c = __float2int_rn(__fdiv_rn(x[i], s));
      c = c < -7 ? -7 : (c > 7 ? 7 : c);
    }
    w |= (uint32_t)(c + 8) << (4 * i);
  }
  return w;
}

__device__ __forceinline__ void kv4_unpack8(uint32_t w, float s, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)((int)((w >> (4 * i)) & 15u) - 8) * s;
}

}  // namespace b2pa
