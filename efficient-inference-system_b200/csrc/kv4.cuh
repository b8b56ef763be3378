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
// infinity's bits compare above every finite one's).  16-bit values T have at
// most 11 bits, so top / 7 lies on a border of two scales or at least 2^-11 of
// itself away from it: a product with 1 / 7 rounded, itself rounded to 13 bits
// (2^-17 in the subnormal range: a border is an odd multiple of 2^-18), is on
// the border with it, and a division can be spared.
template <typename T>
__device__ __forceinline__ uint32_t kv4_scale_code(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return kKv4NanScale;
  const float top = __uint_as_float(max_bits);
  float y;
  if constexpr (std::is_same<T, float>::value)
    y = __fdiv_rn(top, 7.0f);
  else
    y = __uint_as_float((__float_as_uint(top * (1.f / 7.f)) + 0x400u) & ~0x7ffu);
  if (y < 0x1p-14f) return (uint32_t)__float2int_rn(y * 0x1p17f);
  uint32_t u = __float_as_uint(y);
  u += 0x7ffffu + ((u >> 20) & 1u);
  const uint32_t code = (((u >> 23) - 112u) << 3) | ((u >> 20) & 7u);
  return code < kKv4MaxScale ? code : kKv4MaxScale;
}

// Eight codes of one group, packed; s is the value of its scale code.
template <typename T>
__device__ __forceinline__ uint32_t kv4_pack8(const float* x, uint32_t code, float s) {
  if (!(s > 0.f)) return 0x88888888u;  // a zero scale, or a NaN: zeros
  uint32_t w = 0;
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      int c = __float2int_rn(__fdiv_rn(x[i], s));
      c = c < -7 ? -7 : (c > 7 ? 7 : c);
      w |= (uint32_t)(c + 8) << (4 * i);
    }
  } else {
    // 16-bit x, without a division: x times 1 / s (off by less than 2^-18)
    // goes to a multiple of 2^-13 in the addition to 1536, then to an integer,
    // ties to even.  x has at most 11 bits, so x / s lies on a border k + 1/2
    // or at least 0.49 / 2047 > 2^-12.1 away from it: the first rounding puts
    // the former on the border and leaves the latter on its side.  Pairs of
    // values, codes collected by multiplications: the other pipe unpacks x.
    const float r = __fdividef(1.f, s);
    auto both = [](float y) { return make_float2(y, y); };
    // |x| / s is at most 7 (1 + 1/16) unless the scale is subnormal or capped
    const bool clamp = code < 8u || code >= kKv4MaxScale;
    float2 c[4];  // codes i and i + 4
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = fma2(make_float2(x[i], x[i + 4]), both(r), both(1536.f));
      if (clamp) {
        c[i].x = fminf(fmaxf(c[i].x, 1529.f), 1543.f);
        c[i].y = fminf(fmaxf(c[i].y, 1529.f), 1543.f);
      }
      c[i] = add2(add2(c[i], both(12582912.f - 1536.f)), both(-12582912.f));
    }
    float2 v = fma2(c[3], both(16.f), c[2]);
    v = fma2(v, both(16.f), c[1]);
    v = fma2(v, both(16.f), c[0]);
    v = add2(v, both(8388608.f + 0x8888));
    w = __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x5410);
  }
  return w;
}

// Eight values of one group, exact.
// fp32: a nibble in the mantissa of 2^23, one subtraction, one multiplication
// (packed pairs).
__device__ __forceinline__ void kv4_unpack8(uint32_t w, float s, float* x) {
  const float2 m = make_float2(-8388616.f, -8388616.f), z = make_float2(0.f, 0.f), ss = make_float2(s, s);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float2 v = make_float2(__uint_as_float((w >> (4 * i) & 15u) | 0x4b000000u),
                           __uint_as_float((w >> (4 * i + 4) & 15u) | 0x4b000000u));
    v = fma2(add2(v, m), ss, z);
    x[i] = v.x;
    x[i + 1] = v.y;
  }
}
// 16-bit types: the same two steps on the pairs that a mask leaves (channels
// i and i + 4), then the pairs in order.
__device__ __forceinline__ uint4 kv4_in_order(uint32_t c04, uint32_t c15, uint32_t c26, uint32_t c37) {
  return make_uint4(__byte_perm(c04, c15, 0x5410), __byte_perm(c26, c37, 0x5410), __byte_perm(c04, c15, 0x7632),
                    __byte_perm(c26, c37, 0x7632));
}
__device__ __forceinline__ uint4 kv4_unpack8(uint32_t w, uint32_t code, __half) {
  const __half2 s = __half2half2(__ushort_as_half((unsigned short)(code << 7)));
  const __half2 k1032 = __half2half2(__ushort_as_half(0x6408)), k72 = __half2half2(__ushort_as_half(0xd480)),
                k16th = __half2half2(__ushort_as_half(0x2c00));
  auto lo = [&](uint32_t x) {  // 1024 + c
    const uint32_t y = (x & 0x000f000fu) | 0x64006400u;
    const __half2 v = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&y), k1032), s);
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  auto hi = [&](uint32_t x) {  // 16 (64 + c)
    const uint32_t y = (x & 0x00f000f0u) | 0x64006400u;
    const __half2 v = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&y), k16th, k72), s);
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  return kv4_in_order(lo(w), hi(w), lo(w >> 8), hi(w >> 8));
}
__device__ __forceinline__ uint4 kv4_unpack8(uint32_t w, uint32_t code, __nv_bfloat16) {
  const __nv_bfloat162 s = __float2bfloat162_rn(kv4_scale(code)), k136 = __float2bfloat162_rn(136.f);
  auto pick = [&](uint32_t x) {
    const uint32_t y = (x & 0x000f000fu) | 0x43004300u;  // 128 + c
    const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&y), k136), s);
    return *reinterpret_cast<const uint32_t*>(&v);
  };
  return kv4_in_order(pick(w), pick(w >> 4), pick(w >> 8), pick(w >> 12));
}

// Eight values of one group, to 16-byte aligned memory.
template <typename T>
__device__ __forceinline__ void kv4_store8(T* dst, uint32_t w, uint32_t code) {
  if constexpr (std::is_same<T, float>::value) {
    float x[8];
    kv4_unpack8(w, kv4_scale(code), x);
    reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(dst) = kv4_unpack8(w, code, T{});
  }
}

}  // namespace b2pa
