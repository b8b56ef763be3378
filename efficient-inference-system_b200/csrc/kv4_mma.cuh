// kv4_mma.cuh -- one query against packed 4-bit keys on the tensor core
// (mma.sync m16n8k16), shared by the decode attention and the accumulation of
// key weights.  How codes become operands is told in kv4_decode.cu.
#pragma once

#include "common.cuh"
#include "kv4.cuh"

namespace b2pa {

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float warp_redux_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// x as hi + lo fp16 halves, for a pair.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = half2_bits(h);
  lo = half2_bits(__floats2half2_rn(x - f.x, y - f.y));
}


// Eight fp32 values, scaled, as fp16 halves hi + lo.
__device__ __forceinline__ void split8(const float* x, float f, uint4& hi, uint4& lo) {
  uint32_t* h = &hi.x;
  uint32_t* l = &lo.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float u = x[2 * i] * f, v = x[2 * i + 1] * f;
    const __half2 p = __floats2half2_rn(u, v);
    const float2 w = __half22float2(p);
    h[i] = half2_bits(p);
    l[i] = half2_bits(__floats2half2_rn(u - w.x, v - w.y));
  }
}

// One 4-bit word (8 channels of scale s) as 4 operand registers, exact, in
// the order 0 4 1 5 2 6 3 7: a masked nibble pair in the mantissa is 1024 + c,
// or 16 (64 + c) for the upper nibbles.
__device__ __forceinline__ uint4 unpack_word(uint32_t w, __half2 s) {
  const __half2 k1032 = __half2half2(__ushort_as_half(0x6408)), k72 = __half2half2(__ushort_as_half(0xd480)),
                k16th = __half2half2(__ushort_as_half(0x2c00));
  auto lo = [&](uint32_t x) {
    const uint32_t y = (x & 0x000f000fu) | 0x64006400u;
    return half2_bits(__hmul2(__hsub2(*reinterpret_cast<const __half2*>(&y), k1032), s));
  };
  auto hi = [&](uint32_t x) {
    const uint32_t y = (x & 0x00f000f0u) | 0x64006400u;
    return half2_bits(__hmul2(__hfma2(*reinterpret_cast<const __half2*>(&y), k16th, k72), s));
  };
  return make_uint4(lo(w), hi(w), lo(w >> 8), hi(w >> 8));
}
// Two scale codes, in the low bytes, as pairs.
__device__ __forceinline__ __half2 scale_pair(uint32_t codes, uint32_t select) {
  const uint32_t x = __byte_perm(codes, 0, select) << 7;
  return *reinterpret_cast<const __half2*>(&x);
}

// A pair of codes in nibble J & 1 of the low bytes of x as fp16 numbers (16
// times them for an upper nibble): the nibble alone, a subnormal, (c + 8) *
// 2^-24, or, SIGNED, c itself, taken exactly from 1024 + (c + 8).
template <bool SIGNED, int J>
__device__ __forceinline__ uint32_t code_pair(uint32_t x) {
  constexpr uint32_t mask = (J & 1) ? 0x00f000f0u : 0x000f000fu;
  if constexpr (!SIGNED) return x & mask;
  const uint32_t y = (x & mask) | 0x64006400u, off = (J & 1) ? 0x64806480u : 0x64086408u;  // 1152, 1032
  return half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&y), *reinterpret_cast<const __half2*>(&off)));
}
// Channels r and r + 4 of a word, r = 0 .. 3.
template <bool SIGNED>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t (&f)[4]) {
  f[0] = code_pair<SIGNED, 0>(w);
  f[1] = code_pair<SIGNED, 1>(w);
  f[2] = code_pair<SIGNED, 0>(w >> 8);
  f[3] = code_pair<SIGNED, 1>(w >> 8);
}

// How a lane (g = lane / 4, t = lane % 4) holds the K row of one key.
template <int D>
struct KeyWords {
  static constexpr int NG = D / 16;              // groups per row
  static constexpr int SETS = D == 256 ? 2 : 1;  // column sets of 8 groups
  static constexpr int KW = D / 32;              // words per lane and row (rows g and g + 8)
  static constexpr int KB = KW * 4 < 16 ? KW * 4 : 16;  // bytes per piece: bytes t * KB + c * 4 * KB of the row
  static constexpr int KC = KW * 4 / KB;         // pieces per row
  // first channel of word w of lane t; its 8 channels lie in one group
  __device__ static constexpr int channel(int w, int t) {
    return D == 64 ? 16 * t + 8 * w : (w >> 2) * 128 + 32 * t + 8 * (w & 3);
  }
};

// One key row as operand registers with its scales applied: block w (word w
// of lane t) of a product over D channels.
template <int D>
__device__ __forceinline__ void unpack_key_row(const uint8_t* page, int row, int bs, uint4 (&f)[D / 32]) {
  const int t = threadIdx.x & 3;
  const uint8_t* scales = page + bs * (D / 2) + row * (D / 16);
  if constexpr (D == 64) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(page + row * 32 + 8 * t));
    const __half2 sc = scale_pair(__ldg(scales + t), 0x4040);
    f[0] = unpack_word(w.x, sc);
    f[1] = unpack_word(w.y, sc);
  } else {
#pragma unroll
    for (int c = 0; c < D / 128; ++c) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(page + row * (D / 2) + 64 * c + 16 * t));
      const uint32_t sc = __ldg(reinterpret_cast<const uint16_t*>(scales + 8 * c + 2 * t));
      const __half2 s0 = scale_pair(sc, 0x4040), s1 = scale_pair(sc, 0x4141);
      f[4 * c + 0] = unpack_word(w.x, s0);
      f[4 * c + 1] = unpack_word(w.y, s0);
      f[4 * c + 2] = unpack_word(w.z, s1);
      f[4 * c + 3] = unpack_word(w.w, s1);
    }
  }
}

// Where 8 consecutive channels (number c8) of a query row go, in bytes, so
// that its blocks match unpack_key_row's.
template <int D>
__device__ constexpr int query_place(int c8) {
  return D == 64 ? (c8 & 1) * 64 + (c8 >> 1) * 16 : ((c8 >> 4) * 4 + (c8 & 3)) * 64 + ((c8 >> 2) & 3) * 16;
}

// ROWS query rows (zeros from `count` on) into shared memory as fp16 operands:
// rows of fp32 (PARTS = 2: hi, then lo ROWS * PITCH bytes on) and of bf16 are
// scaled into fp16's range, unit[r] undoing it; KV4: in query_place's blocks
// and unpack_word's order, else as they lie.
template <typename T, bool KV4, int D, int ROWS, int PITCH, int PARTS, int THREADS>
__device__ __forceinline__ void convert_queries(const T* q, int64_t stride, int count, uint8_t* dst, float* unit) {
  constexpr bool SCALED = !std::is_same<T, __half>::value;
  constexpr int C8 = (D < 32 ? 32 : D) / 8;  // 8-channel pieces per row (whole blocks)
  constexpr int LPR = C8 < 32 ? C8 : 32;     // lanes per row
  constexpr int V = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31, c = lane % LPR;
#pragma unroll 4
  for (int r = (threadIdx.x >> 5) * (32 / LPR) + lane / LPR; r < ROWS; r += THREADS / LPR) {
    float x[8] = {};
    if (r < count && 8 * c < D) {
      const T* row = q + r * stride + 8 * c;
#pragma unroll
      for (int i = 0; i < 8; i += V) {
        Vec<T, V> v;
        v.w = ld_global_nc<uint4>(row + i);
        v.to_float(x + i);
      }
    }
    float f = 1.f, back = 1.f;
    if constexpr (SCALED) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
      for (int o = LPR / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
      f = range_factor(top, back);
    }
    int at = 16 * c;
    if constexpr (KV4) {
      const float y[8] = {x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = y[i];
      at = query_place<D>(c);
    }
    uint4 hi, lo;
    split8(x, f, hi, lo);
    *reinterpret_cast<uint4*>(dst + r * PITCH + at) = hi;
    if constexpr (PARTS == 2) *reinterpret_cast<uint4*>(dst + (ROWS + r) * PITCH + at) = lo;
    if (c == 0) unit[r] = back;
  }
}

// The query as the product's column operand: column n holds its channels of
// group n (D = 64: the low halves of group n - 4 from column 4 on; D = 256: a
// second set for groups 8..15), scaled by 2^e into fp16's range (its largest
// magnitude near 2^13): exact for 16-bit q, hi + lo for fp32.
template <typename T, int D>
struct KeyQuery {
  using C = KeyWords<D>;
  static constexpr bool QLO = std::is_same<T, float>::value && D != 64;  // low halves as a second product
  // Codes enter as subnormals c + 8, with the 8 taken out of the sums, or as
  // numbers c.  The former costs a few 2^-20 of a logit: the sums are larger
  // than the result, and the product aligns subnormal operands by an exponent
  // up to 10 too large.  (Key weights of a 16-bit q, in fp32: 5e-7 off with the
  // former and 3e-7 with the latter, which took 152 us where it took 132.)
  static constexpr bool SIGNED = std::is_same<T, float>::value;
  uint4 raw[C::KW][sizeof(T) / 2];  // the channels of this lane's column, 8 per word
  uint32_t qh[C::KW][4], ql[QLO ? C::KW : 1][4];
  float init[C::SETS][2];  // -8 sum(q) of columns 2t, 2t+1, in the product's units
  float unit, down_q;      // logit (log2) = product * unit * 2^-e (two factors: neither overflows)

  // 1: word w's group is this lane's column, 2: the column takes its low halves
  __device__ __forceinline__ static int column_of(int w) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = C::channel(w, t) / 16;
    return (D == 64 ? g == group : g == (group & 7)) ? 1 : D == 64 && g == group + 4 ? 2 : 0;
  }
  __device__ __forceinline__ void load(const T* q) {
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int w = 0; w < C::KW; ++w)
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        raw[w][i] = make_uint4(0, 0, 0, 0);
        if (column_of(w)) raw[w][i] = ld_global_nc<uint4>(q + C::channel(w, t) + i * (16 / (int)sizeof(T)));
      }
  }
  __device__ __forceinline__ void prepare(float qscale) {
    const int t = threadIdx.x & 3;
    float x[C::KW][8], top = 0.f;
#pragma unroll
    for (int w = 0; w < C::KW; ++w) {
      constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < 8 / N; ++i) {
        Vec<T, N> v;
        v.w = raw[w][i];
        v.to_float(&x[w][i * N]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[w][i]));
    }
    top = warp_redux_max(top);
    // 2^e by exponent arithmetic; 0, tiny, infinite and NaN maxima keep a finite factor
    int e = 140 - (int)(__float_as_uint(top) >> 23);  // top's exponent field + e = 13 + 127
    e = e > 100 ? 100 : e;
    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
    unit = SIGNED ? qscale : qscale * 0x1p24f;
    down_q = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int w = 0; w < C::KW; ++w) {
      const int col = column_of(w);
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // operand register r: channels r and r + 4 of the word
        const float f = (r & 1) ? up * 0.0625f : up;
        uint32_t hi, lo;
        split2(x[w][r] * f, x[w][r + 4] * f, hi, lo);
        qh[w][r] = col == 1 ? hi : col == 2 ? lo : 0u;
        if constexpr (QLO) ql[w][r] = col == 1 ? lo : 0u;
      }
    }
    // 8 sum(q) of a column: every lane sums its operand registers (undoing the
    // 1/16), lanes of one column (same g) add up, then columns 2t and 2t+1.
#pragma unroll
    for (int s = 0; s < C::SETS; ++s) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < C::KW; ++w) {
        if (C::SETS == 2 && (w >> 2) != s) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&qh[w][r]));
          float z = y.x + y.y;
          if constexpr (QLO) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&ql[w][r]));
            z += v.x + v.y;
          }
          sum += (r & 1) ? z * 16.f : z;
        }
      }
      sum += __shfl_xor_sync(kFullMask, sum, 1);
      sum += __shfl_xor_sync(kFullMask, sum, 2);
      sum *= SIGNED ? 0.f : -8.f * 0x1p-24f;
      init[s][0] = __shfl_sync(kFullMask, sum, 8 * t);
      init[s][1] = __shfl_sync(kFullMask, sum, 8 * t + 4);
    }
  }

  // This lane's part of the products of keys g and g + 8 (words ka, kb; w0 and
  // w1: the scale codes of groups 2t, 2t+1 of each set, in the low bytes).
  // The four lanes of a key have to be added up and scaled: finish().
  __device__ __forceinline__ void logits(const uint32_t (&ka)[C::KW], const uint32_t (&kb)[C::KW],
                                         const uint32_t (&w0)[C::SETS], const uint32_t (&w1)[C::SETS], float& z0,
                                         float& z1) const {
    float s[2][4];  // two chains of products
    if constexpr (C::SETS == 2) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[x][0] = s[x][2] = init[x][0];
        s[x][1] = s[x][3] = init[x][1];
      }
    } else {
      s[0][0] = s[0][2] = init[0][0];
      s[0][1] = s[0][3] = init[0][1];
      s[1][0] = s[1][1] = s[1][2] = s[1][3] = 0.f;
    }
#pragma unroll
    for (int w = 0; w < C::KW; ++w) {
      float(&c)[4] = s[C::SETS == 2 ? w >> 2 : w & 1];
      uint32_t u[4], v[4];
      code_pairs<SIGNED>(ka[w], u);
      code_pairs<SIGNED>(kb[w], v);
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        mma_f16(c, u[r], v[r], u[r + 1], v[r + 1], qh[w][r], qh[w][r + 1]);
        if constexpr (QLO) mma_f16(c, u[r], v[r], u[r + 1], v[r + 1], ql[w][r], ql[w][r + 1]);
      }
    }
    if constexpr (C::SETS == 1) {
#pragma unroll
      for (int k = 0; k < 4; ++k) s[0][k] += s[1][k];
    }
    z0 = z1 = 0.f;
#pragma unroll
    for (int x = 0; x < C::SETS; ++x) {
      const uint32_t h0 = __byte_perm(w0[x], 0, 0x4140) << 7, h1 = __byte_perm(w1[x], 0, 0x4140) << 7;
      const float2 s0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
      const float2 s1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
      z0 = fmaf(s[x][0], s0.x, fmaf(s[x][1], s0.y, z0));
      z1 = fmaf(s[x][2], s1.x, fmaf(s[x][3], s1.y, z1));
    }
  }
  __device__ __forceinline__ float finish(float z) const {
    z += __shfl_xor_sync(kFullMask, z, 1);
    z += __shfl_xor_sync(kFullMask, z, 2);
    return z * unit * down_q;
  }
  // Where a lane's two scale codes of set x lie in the row's codes.
  __device__ __forceinline__ static int scale_at(int x) {
    const int t = threadIdx.x & 3;
    return D == 64 ? 2 * (t & 1) : 8 * x + 2 * t;
  }
};

}  // namespace b2pa
