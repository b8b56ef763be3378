// key_weights.cu -- accumulated attention weight of every cached key.
//
// For each head and cached key j of sequence b:
//     w[j] += sum over counted queries t of softmax_j(q_t . K^T scale),
// query t (position seq_len - cur_len + t) seeing keys 0 .. min(seq_len,
// pos + 1) - 1, and counting when cur_len - window <= t < cur_len (all of
// them without a window).
//
// Several queries (key_weights_tile_kernel): two launches of one matrix
// product Q.K^T, on the tensor cores.  The first has queries as rows and
// keeps each row's running maximum and sum (keys may be split between CTAs);
// the second has keys as rows and adds exp(logit - lse) along its columns, so
// every key's sum stays in one thread and needs no atomics: results do not
// depend on the order of anything.  The product is computed twice because the
// alternative, keeping T x L logits, costs more bytes than the product costs
// time.  Operands: 16-bit types as they are; fp32 in two tf32 halves (three
// products, 22 bits); 4-bit keys as fp16 (exact), with q scaled by a power of
// two into fp16's range, in two halves if it is fp32.
//
// One query (key_weights_step_kernel, plain pools): bound by reading K once.
// A cluster of CTAs shares a sequence, each keeps its logits in shared
// memory, and after one exchange of (maximum, sum) writes its own weights:
// one launch.  4-bit pools take the decode kernel's K half (kv4_decode.cu).
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace cg = cooperative_groups;

namespace b2pa {

namespace {

struct Span {
  int64_t L, past;
  int first, count;  // counted queries first .. first + count - 1
};

__device__ __forceinline__ Span span_of(const KeyWeightArgs& a, int b) {
  Span s;
  const int64_t len = a.seq_lens[b], cap = (int64_t)a.max_pages * a.block_size;
  int64_t cur = a.cur_lens[b];
  s.past = len - cur;
  s.L = len < cap ? len : cap;
  cur = cur < a.T ? cur : a.T;
  s.first = a.window > 0 && cur > a.window ? (int)(cur - a.window) : 0;
  s.count = cur > s.first ? (int)(cur - s.first) : 0;
  return s;
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// ------------------------------------------------------------ several queries
template <typename T, bool KV4>
struct Op {
  static constexpr bool TF32 = std::is_same<T, float>::value && !KV4;
  static constexpr int PARTS = std::is_same<T, float>::value && KV4 ? 2 : 1;  // halves of q held in shared memory
  static constexpr int BYTES = TF32 ? 4 : 2;
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value && !KV4;
  static constexpr bool SCALED = KV4 && !std::is_same<T, __half>::value;  // q scaled per row into fp16's range
};

// Rows of the product's two operands in shared memory.  A warp reads 16-byte
// pieces of 8 rows (4 lanes along a row): with a row pitch of 64 modulo 128
// bytes no two lanes of a quarter warp meet in a bank.
template <typename T, bool KV4, int D, int PASS>
struct Shape {
  using O = Op<T, KV4>;
  static constexpr int RB = D * O::BYTES < 64 ? 64 : D * O::BYTES;  // bytes per row, whole 64-byte blocks
  static constexpr int PITCH = RB % 128 == 0 ? RB + 64 : RB;
  static constexpr int MT = RB <= 256 && PASS == 2 ? 2 : 1;  // 16-row tiles per warp
  static constexpr int ROWS = 64 * MT;
  static constexpr int COLS = RB <= 512 ? 64 : 32;
  static constexpr int NT = COLS / 8;
  static constexpr int ROW_PARTS = PASS == 1 ? O::PARTS : 1;
  static constexpr int COL_PARTS = PASS == 1 ? 1 : O::PARTS;
  static constexpr int ROW_BYTES = ROWS * PITCH, COL_BYTES = COLS * PITCH;
  static constexpr int SMEM = ROW_PARTS * ROW_BYTES + 2 * COL_PARTS * COL_BYTES;
};

template <typename O>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (O::BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// x = hi + lo with hi of 11 significant bits (tf32); lo keeps the next 11.
__device__ __forceinline__ void split_tf32(const uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = x & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
// In place: x becomes hi.
__device__ __forceinline__ void split_tf32(uint4& x, uint4& lo) {
  split_tf32(x.x, x.x, lo.x);
  split_tf32(x.y, x.y, lo.y);
  split_tf32(x.z, x.z, lo.z);
  split_tf32(x.w, x.w, lo.w);
}

// One 4-bit word as 8 fp16 values in the order 0 4 1 5 2 6 3 7 (each masked
// pair of nibbles gives one register: 1024 + c, then 16 (64 + c) for the
// upper nibbles).
__device__ __forceinline__ uint4 word_to_half(uint32_t w, __half2 s) {
  const __half2 k1032 = __half2half2(__ushort_as_half(0x6408)), k72 = __half2half2(__ushort_as_half(0xd480)),
                k16th = __half2half2(__ushort_as_half(0x2c00));
  auto lo = [&](uint32_t x) {
    const uint32_t y = (x & 0x000f000fu) | 0x64006400u;
    return __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&y), k1032), s);
  };
  auto hi = [&](uint32_t x) {
    const uint32_t y = (x & 0x00f000f0u) | 0x64006400u;
    return __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&y), k16th, k72), s);
  };
  uint4 r;
  __half2 h[4] = {lo(w), hi(w), lo(w >> 8), hi(w >> 8)};
  r.x = *reinterpret_cast<uint32_t*>(&h[0]);
  r.y = *reinterpret_cast<uint32_t*>(&h[1]);
  r.z = *reinterpret_cast<uint32_t*>(&h[2]);
  r.w = *reinterpret_cast<uint32_t*>(&h[3]);
  return r;
}

constexpr int kTileThreads = 128;

// Loads key rows (plain: asynchronously; 4-bit: through registers, so that
// the loads of the next tile are in flight during the product of this one).
template <typename T, bool KV4, int D, int N, int RB, int PITCH>
struct KeyLoader {
  static constexpr int UNITS = KV4 ? N * (D / 32) : N * (RB / 16);
  static constexpr int PER = (UNITS + kTileThreads - 1) / kTileThreads;
  uint4 raw[KV4 ? PER : 1];
  uint32_t scales[KV4 ? PER : 1];

  __device__ __forceinline__ static int32_t block_of(const KeyWeightArgs& a, const int32_t* table, int64_t j, int64_t L) {
    if (j >= L) return -1;
    const int32_t blk = table[j >> a.bs_log2];
    return blk < a.num_blocks ? blk : -1;
  }

  __device__ __forceinline__ void fetch(const KeyWeightArgs& a, const int32_t* table, int h, int64_t j0, int64_t L,
                                        uint32_t dst) {
    const int bs = a.block_size;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * kTileThreads;
      if (UNITS % kTileThreads != 0 && u >= UNITS) break;
      if constexpr (KV4) {
        const int r = u / (D / 32), c = u % (D / 32);
        const int64_t j = j0 + r;
        const int32_t blk = block_of(a, table, j, L);
        raw[i] = make_uint4(0, 0, 0, 0);
        scales[i] = 0;
        if (blk >= 0) {
          const uint8_t* page = static_cast<const uint8_t*>(a.k_pool) + ((int64_t)blk * a.H + h) * kv4_page_bytes(bs, D);
          const int row = (int)(j & (bs - 1));
          raw[i] = *reinterpret_cast<const uint4*>(page + row * (D / 2) + 16 * c);
          scales[i] = *reinterpret_cast<const uint16_t*>(page + bs * (D / 2) + row * (D / 16) + 2 * c);
        }
      } else {
        const int r = u / (RB / 16), c = u % (RB / 16);
        const int64_t j = j0 + r;
        const int32_t blk = block_of(a, table, j, L);
        const bool ok = blk >= 0 && 16 * c < D * (int)sizeof(T);
        const char* src = static_cast<const char*>(a.k_pool);
        if (ok) src += ((((int64_t)blk * a.H + h) * bs + (j & (bs - 1))) * D) * (int64_t)sizeof(T) + 16 * c;
        copy16(dst + r * PITCH + 16 * c, src, ok);
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* dst) {
    if constexpr (KV4) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int u = threadIdx.x + i * kTileThreads;
        if (UNITS % kTileThreads != 0 && u >= UNITS) break;
        const int r = u / (D / 32), c = u % (D / 32);
        const uint32_t* w = &raw[i].x;
        const __half2 s0 = __half2half2(__ushort_as_half((unsigned short)((scales[i] & 255u) << 7)));
        const __half2 s1 = __half2half2(__ushort_as_half((unsigned short)((scales[i] >> 8) << 7)));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<uint4*>(dst + r * PITCH + 64 * c + 16 * k) = word_to_half(w[k], k < 2 ? s0 : s1);
      }
    }
  }
};

// Loads counted queries i0 .. i0 + N - 1; zeros past the count.  4-bit pools:
// converted to fp16 (one warp per row), unit[r] = the factor that turns the
// product back into a logit.
template <typename T, bool KV4, int D, int N, int RB, int PITCH>
__device__ __forceinline__ void load_queries(const KeyWeightArgs& a, const Span& s, int h, int b, int i0, uint8_t* dst,
                                             float* unit, float qscale) {
  using O = Op<T, KV4>;
  const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1];
  if constexpr (!KV4) {
    constexpr int CH = RB / 16;
    for (int u = threadIdx.x; u < N * CH; u += kTileThreads) {
      const int r = u / CH, c = u % CH;
      const bool ok = i0 + r < s.count && 16 * c < D * (int)sizeof(T);
      const char* src = reinterpret_cast<const char*>(q);
      if (ok) src += (int64_t)(s.first + i0 + r) * a.sq[2] * (int)sizeof(T) + 16 * c;
      copy16(smem_u32(dst) + r * PITCH + 16 * c, src, ok);
    }
  } else {
    constexpr int LPR = D / 8;  // lanes per row, 8 channels each
    const int lane = threadIdx.x & 31, sub = lane % LPR;
    for (int r = (threadIdx.x >> 5) * (32 / LPR) + lane / LPR; r < N; r += kTileThreads / LPR) {
      float x[8] = {};
      const bool ok = i0 + r < s.count;
      if (ok) {
        const T* row = q + (int64_t)(s.first + i0 + r) * a.sq[2] + 8 * sub;
        constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += V) {
          Vec<T, V> v;
          v.w = ld_global_nc<uint4>(row + i);
          v.to_float(x + i);
        }
      }
      float f = 1.f, back = 1.f;
      if constexpr (O::SCALED) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
        for (int o = LPR / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
        int e = 137 - (int)(__float_as_uint(top) >> 23);  // largest magnitude near 2^10
        e = e > 100 ? 100 : e;
        f = __uint_as_float((uint32_t)(127 + e) << 23);
        back = __uint_as_float((uint32_t)(127 - e) << 23);
      }
      uint32_t hi[4], lo[4];
      constexpr int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = x[order[2 * i]] * f, v = x[order[2 * i + 1]] * f;
        const __half2 hh = __floats2half2_rn(u, v);
        hi[i] = *reinterpret_cast<const uint32_t*>(&hh);
        if constexpr (O::PARTS == 2) {
          const float2 w = __half22float2(hh);
          const __half2 ll = __floats2half2_rn(u - w.x, v - w.y);
          lo[i] = *reinterpret_cast<const uint32_t*>(&ll);
        }
      }
      *reinterpret_cast<uint4*>(dst + r * PITCH + 16 * sub) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      if constexpr (O::PARTS == 2)
        *reinterpret_cast<uint4*>(dst + N * PITCH + r * PITCH + 16 * sub) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      if (sub == 0) unit[r] = back;
    }
  }
}

// acc = rows . cols^T for this warp's MT * 16 rows and all NT * 8 columns.
template <typename S>
__device__ __forceinline__ void product(const uint8_t* rows, const uint8_t* cols, float (&acc)[S::MT][S::NT][4]) {
  using O = typename S::O;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int m = 0; m < S::MT; ++m)
#pragma unroll
    for (int n = 0; n < S::NT; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[m][n][k] = 0.f;
  const uint8_t* ra = rows + (warp * S::MT * 16 + g) * S::PITCH + 16 * t;
  const uint8_t* cb = cols + g * S::PITCH + 16 * t;
#pragma unroll 2
  for (int kb = 0; kb < S::RB; kb += 64) {
    uint4 x[S::MT][2], xl[S::MT][2];
#pragma unroll
    for (int m = 0; m < S::MT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[m][i] = *reinterpret_cast<const uint4*>(ra + (m * 16 + 8 * i) * S::PITCH + kb);
        if constexpr (O::TF32) split_tf32(x[m][i], xl[m][i]);
        if constexpr (S::ROW_PARTS == 2)
          xl[m][i] = *reinterpret_cast<const uint4*>(ra + S::ROW_BYTES + (m * 16 + 8 * i) * S::PITCH + kb);
      }
#pragma unroll
    for (int n = 0; n < S::NT; ++n) {
      uint4 y = *reinterpret_cast<const uint4*>(cb + n * 8 * S::PITCH + kb), yl;
      if constexpr (O::TF32) split_tf32(y, yl);
      if constexpr (S::COL_PARTS == 2) yl = *reinterpret_cast<const uint4*>(cb + S::COL_BYTES + n * 8 * S::PITCH + kb);
#pragma unroll
      for (int m = 0; m < S::MT; ++m) {
        float(&c)[4] = acc[m][n];
        const uint4 &u = x[m][0], &v = x[m][1], &ul = xl[m][0], &vl = xl[m][1];
        if constexpr (O::TF32) {
          mma_tf32(c, ul.x, vl.x, ul.y, vl.y, y.x, y.y);
          mma_tf32(c, u.x, v.x, u.y, v.y, yl.x, yl.y);
          mma_tf32(c, u.x, v.x, u.y, v.y, y.x, y.y);
          mma_tf32(c, ul.z, vl.z, ul.w, vl.w, y.z, y.w);
          mma_tf32(c, u.z, v.z, u.w, v.w, yl.z, yl.w);
          mma_tf32(c, u.z, v.z, u.w, v.w, y.z, y.w);
        } else {
          if constexpr (S::ROW_PARTS == 2) {
            mma16<O>(c, ul.x, vl.x, ul.y, vl.y, y.x, y.y);
            mma16<O>(c, ul.z, vl.z, ul.w, vl.w, y.z, y.w);
          }
          if constexpr (S::COL_PARTS == 2) {
            mma16<O>(c, u.x, v.x, u.y, v.y, yl.x, yl.y);
            mma16<O>(c, u.z, v.z, u.w, v.w, yl.z, yl.w);
          }
          mma16<O>(c, u.x, v.x, u.y, v.y, y.x, y.y);
          mma16<O>(c, u.z, v.z, u.w, v.w, y.z, y.w);
        }
      }
    }
  }
}

// PASS 1: rows are queries, (maximum, sum) of each over one of nsplit ranges
// of keys goes to part[query][split].  PASS 2: rows are keys, columns queries.
template <typename T, bool KV4, int D, int PASS>
__global__ void __launch_bounds__(kTileThreads) key_weights_tile_kernel(KeyWeightArgs a, float qscale, int nsplit,
                                                                        float2* part) {
  using S = Shape<T, KV4, D, PASS>;
  using O = Op<T, KV4>;
  extern __shared__ __align__(16) uint8_t tile_smem[];
  __shared__ float row_unit[S::ROWS], col_unit[2][S::COLS], col_lse[2][S::COLS];
  __shared__ uint8_t col_ok[2][S::COLS];
  uint8_t* rows = tile_smem;
  uint8_t* cols[2] = {tile_smem + S::ROW_PARTS * S::ROW_BYTES,
                      tile_smem + S::ROW_PARTS * S::ROW_BYTES + S::COL_PARTS * S::COL_BYTES};
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const Span s = span_of(a, b);
  const int32_t* table = a.page_table + (int64_t)b * a.pt_stride;
  const int64_t head = (int64_t)b * a.H + h;
  float acc[S::MT][S::NT][4];

  if constexpr (PASS == 1) {
    const int tile = blockIdx.x / nsplit, split = blockIdx.x % nsplit;
    const int i0 = tile * S::ROWS;
    if (blockIdx.x == 0 && h == 0 && tid == 0 && (int64_t)a.seq_lens[b] > s.L)
      set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    if (i0 >= s.count) return;
    const int last = i0 + S::ROWS < s.count ? i0 + S::ROWS : s.count;
    int64_t kend = s.past + s.first + last;
    kend = kend < s.L ? kend : s.L;
    const int64_t tiles = kend > 0 ? (kend + S::COLS - 1) / S::COLS : 0, per = (tiles + nsplit - 1) / nsplit;
    const int64_t c0 = split * per < tiles ? split * per : tiles, c1 = c0 + per < tiles ? c0 + per : tiles;
    load_queries<T, KV4, D, S::ROWS, S::RB, S::PITCH>(a, s, h, b, i0, rows, row_unit, qscale);
    KeyLoader<T, KV4, D, S::COLS, S::RB, S::PITCH> keys;
    auto mark = [&](int64_t c, int buf) {
      for (int r = tid; r < S::COLS; r += kTileThreads) {
        const int64_t j = c * S::COLS + r;
        int ok = 0;
        if (j < kend) {
          const int32_t blk = table[j >> a.bs_log2];
          ok = blk >= 0 && blk < a.num_blocks;
          if (blk >= a.num_blocks) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
        }
        col_ok[buf][r] = (uint8_t)ok;
      }
    };
    float m[S::MT][2], l[S::MT][2], unit[S::MT][2];
#pragma unroll
    for (int x = 0; x < S::MT; ++x) m[x][0] = m[x][1] = -INFINITY, l[x][0] = l[x][1] = 0.f;
    if (c0 < c1) {
      keys.fetch(a, table, h, c0 * S::COLS, kend, smem_u32(cols[0]));
      keys.store(cols[0]);
      mark(c0, 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int64_t c = c0; c < c1; ++c) {
      const int buf = (int)(c - c0) & 1;
      if (c + 1 < c1) keys.fetch(a, table, h, (c + 1) * S::COLS, kend, smem_u32(cols[buf ^ 1]));
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      if (c == c0) {
#pragma unroll
        for (int x = 0; x < S::MT; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            unit[x][i] = O::SCALED ? qscale * row_unit[warp * S::MT * 16 + x * 16 + g + 8 * i] : qscale;
      }
      product<S>(rows, cols[buf], acc);
#pragma unroll
      for (int x = 0; x < S::MT; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = i0 + warp * S::MT * 16 + x * 16 + g + 8 * i;
          const int64_t seen = s.past + s.first + r + 1 - c * S::COLS;  // columns below it are visible
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < S::NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int col = n * 8 + 2 * t + e;
              float& z = acc[x][n][2 * i + e];
              z = col < seen && col_ok[buf][col] ? z * unit[x][i] : -INFINITY;
              top = fmaxf(top, z);
            }
          top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
          top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
          const float mn = fmaxf(m[x][i], top), ref = mn == -INFINITY ? 0.f : mn;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < S::NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) sum += fast_exp2(acc[x][n][2 * i + e] - ref);
          l[x][i] = l[x][i] * fast_exp2(m[x][i] - ref) + sum;
          m[x][i] = mn;
        }
      __syncthreads();
      if (c + 1 < c1) {
        keys.store(cols[buf ^ 1]);
        mark(c + 1, buf ^ 1);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int x = 0; x < S::MT; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[x][i] += __shfl_xor_sync(kFullMask, l[x][i], 1);
        l[x][i] += __shfl_xor_sync(kFullMask, l[x][i], 2);
        const int r = i0 + warp * S::MT * 16 + x * 16 + g + 8 * i;
        if (t == 0 && r < s.count) part[(head * a.T + r) * nsplit + split] = make_float2(m[x][i], l[x][i]);
      }
  } else {
    const int64_t j0 = (int64_t)blockIdx.x * S::ROWS;
    if (j0 >= s.L) return;
    // the first counted query that sees key j0 or a later one
    int64_t from = j0 - s.past - s.first;
    from = from > 0 ? from : 0;
    const int c0 = from < s.count ? (int)(from / S::COLS) : 0;
    const int c1 = from < s.count ? (s.count + S::COLS - 1) / S::COLS : 0;
    float sum[S::MT][2];
#pragma unroll
    for (int x = 0; x < S::MT; ++x) sum[x][0] = sum[x][1] = 0.f;
    // columns' log-sum-exps, +inf where a query does not count or sees nothing
    auto load_lse = [&](int c, int buf) {
      for (int r = tid; r < S::COLS; r += kTileThreads) {
        const int i = c * S::COLS + r;
        float lse = INFINITY;
        if (i < s.count) {
          const float2* p = part + (head * a.T + i) * nsplit;
          float M = -INFINITY, l = 0.f;
          for (int k = 0; k < nsplit; ++k) M = fmaxf(M, p[k].x);
          const float ref = M == -INFINITY ? 0.f : M;
          for (int k = 0; k < nsplit; ++k) l += p[k].y * fast_exp2(p[k].x - ref);
          if (l != 0.f) lse = ref + log2f(l);
        }
        col_lse[buf][r] = lse;
      }
    };
    KeyLoader<T, KV4, D, S::ROWS, S::RB, S::PITCH> keys;
    if (c0 < c1) {
      keys.fetch(a, table, h, j0, s.L, smem_u32(rows));
      load_queries<T, KV4, D, S::COLS, S::RB, S::PITCH>(a, s, h, b, c0 * S::COLS, cols[0], col_unit[0], qscale);
      load_lse(c0, 0);
      keys.store(rows);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int c = c0; c < c1; ++c) {
      const int buf = (c - c0) & 1;
      if (c + 1 < c1) {
        load_queries<T, KV4, D, S::COLS, S::RB, S::PITCH>(a, s, h, b, (c + 1) * S::COLS, cols[buf ^ 1],
                                                          col_unit[buf ^ 1], qscale);
        load_lse(c + 1, buf ^ 1);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      product<S>(rows, cols[buf], acc);
      // key j is seen by columns at or above j - past - first - c * COLS
      const int64_t base = j0 - s.past - s.first - (int64_t)c * S::COLS;
      const bool whole = base + S::ROWS - 1 <= 0;
#pragma unroll
      for (int n = 0; n < S::NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = n * 8 + 2 * t + e;
          const float lse = col_lse[buf][col], unit = O::SCALED ? qscale * col_unit[buf][col] : qscale;
#pragma unroll
          for (int x = 0; x < S::MT; ++x)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int r = warp * S::MT * 16 + x * 16 + g + 8 * i;
              const float p = fast_exp2(fmaf(acc[x][n][2 * i + e], unit, -lse));
              if (whole || base + r <= col) sum[x][i] += p;
            }
        }
      __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < S::MT; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sum[x][i] += __shfl_xor_sync(kFullMask, sum[x][i], 1);
        sum[x][i] += __shfl_xor_sync(kFullMask, sum[x][i], 2);
        const int64_t j = j0 + warp * S::MT * 16 + x * 16 + g + 8 * i;
        if (t == 0 && j < s.L) {
          const int32_t blk = table[j >> a.bs_log2];
          if (blk >= 0 && blk < a.num_blocks) {
            const int64_t at = ((int64_t)blk * a.H + h) * a.block_size + (j & (a.block_size - 1));
            a.w_out[at] = a.w_in[at] + sum[x][i];
          }
        }
      }
  }
}

// ------------------------------------------------------------------ one query
constexpr int kStepThreads = 256;

// How a warp takes its rows.  16-bit rows are tensor-core operands as they
// lie: a lane loads its fragment (16 bytes of row g and of row g + 8 per 64
// bytes of row), and the one query stands in all 8 columns, so every lane gets
// its rows' logits without a conversion or a shuffle.  fp32 rows are summed by
// the lanes that share a row.
template <typename T, int D>
struct StepRows {
  static constexpr int RB = D * (int)sizeof(T);
  static constexpr bool MMA = sizeof(T) == 2;
  // MMA: 64-byte blocks per row, 16-row tiles per turn (8 loads in flight)
  static constexpr int NB = RB < 64 ? 1 : RB / 64, TILES = NB < 4 ? 4 / NB : 1;
  // else: lanes per row, 16-byte pieces per lane, rows per load, rows per lane
  static constexpr int LPR = RB / 16 < 32 ? RB / 16 : 32, CPL = RB / 16 / LPR, RP = 32 / LPR, R = 8 / CPL;
  static constexpr int RW = MMA ? 16 * TILES : RP * R;  // rows per warp and turn
};

template <typename T, int D>
__global__ void __launch_bounds__(kStepThreads) key_weights_step_kernel(KeyWeightArgs a, float qscale, float* far,
                                                                        int64_t far_stride) {
  using S = StepRows<T, D>;
  using O = Op<T, false>;
  constexpr int RB = S::RB, RW = S::RW, E = 16 / (int)sizeof(T);
  extern __shared__ float near[];
  __shared__ float red[2][kStepThreads / 32];
  __shared__ float cta_m, cta_l;
  pdl_wait();
  pdl_launch_dependents();
  const int ns = gridDim.x, rank = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Span s = span_of(a, b);
  if (rank == 0 && h == 0 && tid == 0 && (int64_t)a.seq_lens[b] > s.L) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  const uint32_t blocks = a.num_blocks < INT32_MAX ? (uint32_t)a.num_blocks : (uint32_t)INT32_MAX;
  const int L = s.L > 0 ? (int)s.L : 0;  // positions fit 31 bits
  int vis = s.past + 1 < L ? (int)(s.past + 1) : L;
  if (s.count == 0 || vis < 0 || blocks == 0) vis = 0;
  const int turns = (L + RW - 1) / RW, per = (turns + ns - 1) / ns * RW;  // keys per CTA
  const int64_t lo64 = (int64_t)rank * per;
  const int lo = lo64 < L ? (int)lo64 : L, hi = lo + (int64_t)per < L ? lo + per : L;
  const int bs = a.block_size, sh = a.bs_log2;
  const int32_t* table = a.page_table + (int64_t)b * a.pt_stride;
  // logits of this CTA's keys
  float* z = far ? far + ((int64_t)b * a.H + h) * far_stride + lo : near;
  const int seen = vis < hi ? vis : hi;  // keys [lo, seen) have a logit
  const char* const pages = static_cast<const char*>(a.k_pool) + (int64_t)h * bs * RB;
  const uint64_t block_bytes = (uint64_t)a.H * bs * RB;
  const T* const q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1];

  float top = -INFINITY;
  constexpr int kWarps = kStepThreads / 32;
  auto ids_of = [&](int64_t j0) {  // lane l: the l-th page from key j0's
    const int64_t pg = (j0 >> sh) + lane;
    return j0 < seen && pg << sh < seen ? table[pg] : -1;
  };
  int64_t j0 = lo + warp * RW;
  int ids = ids_of(j0);
  bool past_pool = false;
  // Row j of the turn at j0: where it is (block 0 for one that is not seen).
  auto locate = [&](int64_t j, bool& ok) -> const char* {
    const uint32_t blk = (uint32_t)__shfl_sync(kFullMask, ids, (int)((j >> sh) - (j0 >> sh)));
    ok = j < seen && blk < blocks;
    past_pool |= j < seen && (int)blk >= (int)blocks;
    return pages + (ok ? blk : 0u) * block_bytes + (int)(j & (bs - 1)) * RB;
  };
  if constexpr (S::MMA) {
    const int g = lane >> 2, t = lane & 3;
    uint4 qf[S::NB];
#pragma unroll
    for (int c = 0; c < S::NB; ++c) {
      qf[c] = make_uint4(0, 0, 0, 0);
      if (c * 32 + 8 * t < D) qf[c] = ld_global_nc<uint4>(q + c * 32 + 8 * t);
    }
    for (; j0 < seen; j0 += kWarps * RW) {
      const int next = ids_of(j0 + kWarps * RW);
      uint4 raw[S::TILES][2][S::NB];
      bool ok[S::TILES][2];
#pragma unroll
      for (int x = 0; x < S::TILES; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const char* src = locate(j0 + x * 16 + g + 8 * i, ok[x][i]);
#pragma unroll
          for (int c = 0; c < S::NB; ++c) {
            raw[x][i][c] = make_uint4(0, 0, 0, 0);
            if (RB >= 64 || 16 * t < RB) raw[x][i][c] = ld_global_nc<uint4>(src + c * 64 + 16 * t);
          }
        }
#pragma unroll
      for (int x = 0; x < S::TILES; ++x) {
        float c0[4] = {}, c1[4] = {};
#pragma unroll
        for (int c = 0; c < S::NB; ++c) {
          const uint4 &u = raw[x][0][c], &v = raw[x][1][c], &y = qf[c];
          mma16<O>(c0, u.x, v.x, u.y, v.y, y.x, y.y);
          mma16<O>(c1, u.z, v.z, u.w, v.w, y.z, y.w);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float dot = ok[x][i] ? (c0[2 * i] + c1[2 * i]) * qscale : -INFINITY;
          top = fmaxf(top, dot);
          const int64_t j = j0 + x * 16 + g + 8 * i;
          if (t == 0 && j < seen) z[j - lo] = dot;
        }
      }
      ids = next;
    }
  } else {
    const int sub = lane % S::LPR;
    float qf[S::CPL][E];
#pragma unroll
    for (int c = 0; c < S::CPL; ++c) {
      Vec<T, E> v;
      v.w = ld_global_nc<uint4>(q + (c * S::LPR + sub) * E);
      v.to_float(qf[c]);
#pragma unroll
      for (int i = 0; i < E; ++i) qf[c][i] *= qscale;
    }
    for (; j0 < seen; j0 += kWarps * RW) {
      const int next = ids_of(j0 + kWarps * RW);
      uint4 raw[S::R][S::CPL];
      bool ok[S::R];
#pragma unroll
      for (int r = 0; r < S::R; ++r) {
        const char* src = locate(j0 + r * S::RP + lane / S::LPR, ok[r]);
#pragma unroll
        for (int c = 0; c < S::CPL; ++c) raw[r][c] = ld_global_nc<uint4>(src + (c * S::LPR + sub) * 16);
      }
#pragma unroll
      for (int r = 0; r < S::R; ++r) {
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < S::CPL; ++c) {
          Vec<T, E> v;
          v.w = raw[r][c];
          float k[E];
          v.to_float(k);
#pragma unroll
          for (int i = 0; i < E; ++i) dot = fmaf(qf[c][i], k[i], dot);
        }
#pragma unroll
        for (int o = S::LPR / 2; o >= 1; o >>= 1) dot += __shfl_xor_sync(kFullMask, dot, o);
        if (!ok[r]) dot = -INFINITY;
        top = fmaxf(top, dot);
        const int64_t j = j0 + r * S::RP + lane / S::LPR;
        if (sub == r % S::LPR && j < seen) z[j - lo] = dot;
      }
      ids = next;
    }
  }
  if (past_pool) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  // this CTA's maximum and sum
  top = warp_max(top);
  if (lane == 0) red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, red[0][w]);
  float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  const int mine = hi - lo, logits = seen > lo ? seen - lo : 0;
  for (int i = tid; i < logits; i += kStepThreads) sum += fast_exp2(z[i] - ref);
  sum = warp_sum(sum);
  if (lane == 0) red[1][warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum += red[1][w];
  // the sequence's
  if (ns > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) {
      cta_m = top;
      cta_l = sum;
    }
    cluster.sync();
    top = -INFINITY;
    for (int r = 0; r < ns; ++r) top = fmaxf(top, *cluster.map_shared_rank(&cta_m, r));
    ref = top == -INFINITY ? 0.f : top;
    sum = 0.f;
    for (int r = 0; r < ns; ++r)
      sum += *cluster.map_shared_rank(&cta_l, r) * fast_exp2(*cluster.map_shared_rank(&cta_m, r) - ref);
    cluster.sync();
  }
  const float lse = sum != 0.f ? ref + log2f(sum) : INFINITY;
  float* const w_out = a.w_out + (int64_t)h * bs;
  const float* const w_in = a.w_in + (int64_t)h * bs;
  for (int i = tid; i < mine; i += kStepThreads) {
    const int j = lo + i;
    const uint32_t blk = (uint32_t)__ldg(table + (j >> sh));
    if (blk < blocks) {
      const uint64_t at = (uint64_t)blk * (uint32_t)(a.H * bs) + (j & (bs - 1));
      w_out[at] = w_in[at] + (i < logits ? fast_exp2(z[i] - lse) : 0.f);
    }
  }
}

// ------------------------------------------------------------------- launches
// Key ranges of the first pass: enough CTAs for two waves of four per SM.
int split_of(int B, int H, int count, int64_t keys, int rows, int cols) {
  const int64_t tiles = (int64_t)B * H * ((count + rows - 1) / rows);
  int ns = 1;
  while (ns < 16 && tiles * ns < 4 * device_sm_count() && keys >= (int64_t)cols * 4 * ns * 2) ns *= 2;
  return ns;
}

int counted_most(int T, int window) { return window > 0 && window < T ? window : T; }

template <typename T, bool KV4, int D>
int tile_launch(const KeyWeightArgs& a, cudaStream_t st) {
  using S1 = Shape<T, KV4, D, 1>;
  using S2 = Shape<T, KV4, D, 2>;
  const float qscale = a.scale * kLog2e;
  const int64_t keys = (int64_t)a.max_pages * a.block_size;
  const int count = counted_most(a.T, a.window);
  const int ns = split_of(a.B, a.H, count, keys, S1::ROWS, S1::COLS);
  float2* part = static_cast<float2*>(a.workspace);
  auto k1 = key_weights_tile_kernel<T, KV4, D, 1>;
  auto k2 = key_weights_tile_kernel<T, KV4, D, 2>;
  int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(k1), S1::SMEM);
  if (rc == B2PA_OK) rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(k2), S2::SMEM);
  if (rc != B2PA_OK || keys == 0) return rc;
  cudaError_t e = launch_pdl(k1, dim3((unsigned)((count + S1::ROWS - 1) / S1::ROWS * ns), (unsigned)a.H, (unsigned)a.B),
                             dim3(kTileThreads), S1::SMEM, st, a, qscale, ns, part);
  if (e == cudaSuccess)
    e = launch_pdl(k2, dim3((unsigned)((keys + S2::ROWS - 1) / S2::ROWS), (unsigned)a.H, (unsigned)a.B),
                   dim3(kTileThreads), S2::SMEM, st, a, qscale, ns, part);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "key_weights launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

// Logits of one CTA that shared memory holds beside a second CTA.
constexpr int64_t kNearKeys = 24 * 1024;

int step_split(int64_t pairs, int64_t keys) {
  int ns = 1;
  while (ns < 8 && (pairs * ns < 4 * device_sm_count() || keys > kNearKeys * ns) && keys >= 512 * ns) ns *= 2;
  return ns;
}

template <typename T, int D>
int step_launch(const KeyWeightArgs& a, cudaStream_t st) {
  const int64_t keys = (int64_t)a.max_pages * a.block_size;
  if (keys == 0) return B2PA_OK;
  const int ns = step_split((int64_t)a.B * a.H, keys);
  const int64_t per = (keys + ns - 1) / ns + 128;  // a CTA's keys, rounded up to whole turns
  const bool far = per > kNearKeys + 128;
  const int smem = far ? 0 : (int)(per * 4);
  auto kern = key_weights_step_kernel<T, D>;
  const int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(kern), smem);
  if (rc != B2PA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ns, (unsigned)a.H, (unsigned)a.B);
  cfg.blockDim = dim3(kStepThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ns;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, a.scale * kLog2e,
                                           far ? static_cast<float*>(a.workspace) : static_cast<float*>(nullptr), keys);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "key_weights launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

template <typename T>
int weights_as(const KeyWeightArgs& a, cudaStream_t s) {
  if (a.pool_dtype == B2PA_DTYPE_KV4) {
    switch (a.D) {
      case 64: return tile_launch<T, true, 64>(a, s);
      case 128: return tile_launch<T, true, 128>(a, s);
      default: return tile_launch<T, true, 256>(a, s);
    }
  }
#define B2PA_WEIGHTS_CASE(DD) \
  case DD: return a.T == 1 ? step_launch<T, DD>(a, s) : tile_launch<T, false, DD>(a, s);
  switch (a.D) {
    B2PA_WEIGHTS_CASE(16)
    B2PA_WEIGHTS_CASE(32)
    B2PA_WEIGHTS_CASE(64)
    B2PA_WEIGHTS_CASE(128)
    default: return a.T == 1 ? step_launch<T, 256>(a, s) : tile_launch<T, false, 256>(a, s);
  }
#undef B2PA_WEIGHTS_CASE
}

}  // namespace

size_t key_weights_workspace(int B, int H, int T, int D, int max_pages, int block_size, int dtype, int pool_dtype) {
  (void)D, (void)dtype;
  const int64_t keys = (int64_t)max_pages * block_size;
  if (T == 1 && pool_dtype != B2PA_DTYPE_KV4) {
    const int ns = step_split((int64_t)B * H, keys);
    return (keys + ns - 1) / ns > kNearKeys ? (size_t)B * H * keys * sizeof(float) : 0;
  }
  return (size_t)B * H * T * 16 * sizeof(float2);
}

int launch_key_weights(const KeyWeightArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return weights_as<float>(a, s);
    case B2PA_DTYPE_BF16: return weights_as<__nv_bfloat16>(a, s);
    default: return weights_as<__half>(a, s);
  }
}

}  // namespace b2pa
