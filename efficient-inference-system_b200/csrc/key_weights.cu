// key_weights.cu -- accumulated attention weight of every cached key.
//
// For each head and cached key j of sequence b:
//     w[j] += sum over counted queries t of softmax_j(q_t . K^T scale),
// query t (position seq_len - cur_len + t) seeing keys 0 .. min(seq_len,
// pos + 1) - 1, and counting when cur_len - window <= t < cur_len (all of
// them without a window).
//
// Several queries: two launches over one matrix product K.Q^T on the tensor
// cores.  The first finds each query's maximum and sum (keys may be split
// between CTAs); the second, with keys as rows, adds exp(logit - lse) along the
// queries, so every key's sum stays in one thread and needs no atomics: results
// do not depend on the order of anything.  The product is computed twice
// because the alternative, keeping T x L logits, costs more bytes than the
// product costs time.  Both passes round a logit before they subtract from it: a
// fused product would leave the rounded reference by up to half a unit of its
// last place, a factor of every weight (2 % at logits of 500,000).
// Operands: 16-bit types as they are; 4-bit keys unpacked (exactly) to fp16;
// fp32 as two fp16 halves each (22 bits, three products), rows scaled by powers
// of two into fp16's range.
//   head_dim 64 and 128: key_weights_tc.cu (tcgen05).
//   head_dim 16, 32 and 256: key_weights_tile_kernel here (mma.sync), whose key
//   rows go from global memory to registers -- each is used by one warp only --
//   with 64 queries in shared memory as columns; the first launch keeps, per
//   lane and column, a maximum and a sum over the rows that the lane sees.
//   Bound by instruction issue, about five instructions a logit.
//
// One query (key_weights_step_kernel): bound by reading K once.
// A cluster of CTAs shares a sequence, each keeps its logits in shared
// memory, and after one exchange of (maximum, sum) writes its own weights:
// one launch.  4-bit keys take the product of the decode kernel (kv4_mma.cuh).
#include <cooperative_groups.h>

#include "by_length.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "kv4_mma.cuh"

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
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value && !KV4;  // operand type (else fp16)
  static constexpr bool F32 = std::is_same<T, float>::value;                   // in two fp16 halves
  static constexpr bool SCALED = F32 || (KV4 && std::is_same<T, __nv_bfloat16>::value);  // q rows, into fp16's range
  static constexpr bool PREP = F32 || KV4;  // q rows are converted or reordered: once, by the first pass
};

template <typename O>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (O::BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kTileThreads = 128;
constexpr int kCols = 64;  // queries per tile

template <typename T, bool KV4, int D>
struct Shape {
  using O = Op<T, KV4>;
  static constexpr int NB = D < 32 ? 1 : D / 32;          // blocks of 32 channels: two products of 16
  static constexpr int KPARTS = O::F32 && !KV4 ? 2 : 1;   // halves of a key / of a query
  static constexpr int QPARTS = O::F32 ? 2 : 1;
  // 16-row tiles per warp: two share every load of the queries, one leaves
  // room for more warps, which pays for fp32 (three products a load; 256
  // queries, head_dim 64: 57 us with two, 51 with one) and for wide rows
  static constexpr int MT = KPARTS == 1 && NB <= 4 ? 2 : 1;
  static constexpr int WROWS = 16 * MT, ROWS = 4 * WROWS;  // keys per warp and CTA
  static constexpr int PITCH = NB * 64 % 128 == 0 ? NB * 64 + 64 : NB * 64;  // a quarter warp's two rows in other banks
  static constexpr int Q_BYTES = QPARTS * kCols * PITCH;  // a tile of queries
  static constexpr int Q_SAVED = O::PREP ? Q_BYTES + kCols * 4 : 0;  // ... with its factors, in the workspace
};

// Counted queries i0 .. i0 + 63 into shared memory (zeros past the count):
// copies of the rows, or what the first pass converts them to, with unit[r]
// the factor that undoes a row's scaling.
template <typename T, bool KV4, int D>
__device__ __forceinline__ void load_queries(const KeyWeightArgs& a, const Span& s, int h, int b, int i0, uint8_t* dst,
                                             float* unit) {
  using S = Shape<T, KV4, D>;
  using O = typename S::O;
  constexpr int C8 = S::NB * 4;  // 8-channel pieces per row (whole blocks)
  const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1];
  if constexpr (!O::PREP) {
    for (int u = threadIdx.x; u < kCols * C8; u += kTileThreads) {
      const int r = u / C8, c = u % C8;
      const bool ok = i0 + r < s.count && 8 * c < D;
      copy16(smem_u32(dst) + r * S::PITCH + 16 * c, ok ? q + (int64_t)(s.first + i0 + r) * a.sq[2] + 8 * c : q, ok);
    }
  } else {
    convert_queries<T, KV4, D, kCols, S::PITCH, S::QPARTS, kTileThreads>(q + (int64_t)(s.first + i0) * a.sq[2], a.sq[2],
                                                                        s.count - i0, dst, unit);
  }
}

// A converted tile to and from the workspace.
template <typename S>
__device__ __forceinline__ void save_queries(uint8_t* to, const uint8_t* tile, const float* unit) {
  for (int i = threadIdx.x * 16; i < S::Q_BYTES; i += kTileThreads * 16)
    *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(tile + i);
  if (threadIdx.x < kCols) reinterpret_cast<float*>(to + S::Q_BYTES)[threadIdx.x] = unit[threadIdx.x];
}
template <typename S>
__device__ __forceinline__ void fetch_saved(uint8_t* tile, float* unit, const uint8_t* from) {
  for (int i = threadIdx.x * 16; i < S::Q_BYTES; i += kTileThreads * 16) copy16(smem_u32(tile) + i, from + i, true);
  if (threadIdx.x < kCols / 4) copy16(smem_u32(unit) + 16 * threadIdx.x, from + S::Q_BYTES + 16 * threadIdx.x, true);
}

// A warp's key rows as operand fragments: rows g and g + 8 of each 16-row tile.
template <typename T, bool KV4, int D>
struct Keys {
  using S = Shape<T, KV4, D>;
  uint4 x[S::MT][2][S::NB];
  uint4 lo[S::KPARTS == 2 ? S::MT : 1][2][S::KPARTS == 2 ? S::NB : 1];
  float back[S::MT][2];  // undoes the scaling of fp32 rows
  bool ok[S::MT][2];     // the row is a key (its page exists)

  __device__ __forceinline__ static uint32_t block_of(const KeyWeightArgs& a, const int32_t* table, int64_t j,
                                                      int64_t end, uint32_t blocks, bool& ok, bool& past_pool) {
    const uint32_t blk = j < end ? (uint32_t)__ldg(table + (j >> a.bs_log2)) : 0xffffffffu;
    ok = blk < blocks;
    past_pool |= (int)blk >= (int)blocks;
    return ok ? blk : 0u;
  }

  // Rows j0 + 16 m + g (+ 8), those below `end`.
  __device__ __forceinline__ void load(const KeyWeightArgs& a, const int32_t* table, int h, int64_t j0, int64_t end,
                                       uint32_t blocks, bool& past_pool) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int bs = a.block_size;
#pragma unroll
    for (int m = 0; m < S::MT; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4(&f)[S::NB] = x[m][i];
        const int64_t j = j0 + 16 * m + 8 * i + g;
        const uint32_t blk = block_of(a, table, j, end, blocks, ok[m][i], past_pool);
        const int row = (int)(j & (bs - 1));
        if constexpr (KV4) {
          const uint8_t* page = static_cast<const uint8_t*>(a.k_pool) +
                                (uint64_t)(blk * (uint64_t)a.H + h) * (uint32_t)kv4_page_bytes(bs, D);
          unpack_key_row<D>(page, row, bs, f);
        } else {
          const T* src = static_cast<const T*>(a.k_pool) + ((blk * (uint64_t)a.H + h) * bs + row) * D + 8 * t;
          if constexpr (!S::O::F32) {
#pragma unroll
            for (int c = 0; c < S::NB; ++c) {
              f[c] = make_uint4(0, 0, 0, 0);
              if (D >= 32 || 8 * t < D) f[c] = __ldg(reinterpret_cast<const uint4*>(src + 32 * c));
            }
          } else {
            float v[S::NB][8], top = 0.f;
#pragma unroll
            for (int c = 0; c < S::NB; ++c)
#pragma unroll
              for (int k = 0; k < 8; k += 4) {
                float4 y = make_float4(0, 0, 0, 0);
                if (D >= 32 || 8 * t < D) y = __ldg(reinterpret_cast<const float4*>(src + 32 * c + k));
                *reinterpret_cast<float4*>(&v[c][k]) = y;
                top = fmaxf(top, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
              }
            top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
            top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
            const float up = range_factor(top, back[m][i]);
#pragma unroll
            for (int c = 0; c < S::NB; ++c) split8(v[c], up, f[c], lo[m][i][c]);
          }
        }
      }
  }

  // acc = rows . columns 8n .. 8n+7
  __device__ __forceinline__ void product(const uint8_t* q, int n, float (&acc)[S::MT][4]) const {
    using O = typename S::O;
    const int lane = threadIdx.x & 31;
    const uint8_t* at = q + (n * 8 + (lane >> 2)) * S::PITCH + 16 * (lane & 3);
#pragma unroll
    for (int m = 0; m < S::MT; ++m)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[m][k] = 0.f;
#pragma unroll
    for (int c = 0; c < S::NB; ++c) {
      const uint4 y = *reinterpret_cast<const uint4*>(at + 64 * c);
      uint4 yl;
      if constexpr (S::QPARTS == 2) yl = *reinterpret_cast<const uint4*>(at + kCols * S::PITCH + 64 * c);
#pragma unroll
      for (int m = 0; m < S::MT; ++m) {
        const uint4 &u = x[m][0][c], &v = x[m][1][c];
        if constexpr (S::KPARTS == 2) {
          const uint4 &ul = lo[m][0][c], &vl = lo[m][1][c];
          mma16<O>(acc[m], ul.x, vl.x, ul.y, vl.y, y.x, y.y);
          mma16<O>(acc[m], ul.z, vl.z, ul.w, vl.w, y.z, y.w);
        }
        if constexpr (S::QPARTS == 2) {
          mma16<O>(acc[m], u.x, v.x, u.y, v.y, yl.x, yl.y);
          mma16<O>(acc[m], u.z, v.z, u.w, v.w, yl.z, yl.w);
        }
        mma16<O>(acc[m], u.x, v.x, u.y, v.y, y.x, y.y);
        mma16<O>(acc[m], u.z, v.z, u.w, v.w, y.z, y.w);
      }
    }
  }
};

// PASS 1: grid (query tile x key range, head, sequence); (maximum, sum) of
// each query over one of nsplit ranges of keys goes to part[query][split].
// PASS 2: grid (key tiles, taken in turn; head; sequence).
template <typename T, bool KV4, int D, int PASS>
__global__ void __launch_bounds__(kTileThreads, Shape<T, KV4, D>::KPARTS == 2 && D <= 128 ? 4 : 0) key_weights_tile_kernel(KeyWeightArgs a, float qscale, int nsplit,
                                                                        float2* part, uint8_t* saved, int chunks_most) {
  using S = Shape<T, KV4, D>;
  using O = typename S::O;
  extern __shared__ __align__(16) uint8_t queries[];  // PASS 2: two tiles
  __shared__ __align__(16) float col_unit[2][kCols], col_lse[2][kCols];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const Span s = span_of(a, b);
  const int32_t* table = a.page_table + (int64_t)b * a.pt_stride;
  const int64_t head = (int64_t)b * a.H + h;
  const uint32_t blocks = a.num_blocks < INT32_MAX ? (uint32_t)a.num_blocks : (uint32_t)INT32_MAX;
  if (blocks == 0) return;
  bool past_pool = false;
  Keys<T, KV4, D> keys;
  float acc[S::MT][4];
  constexpr int NT = kCols / 8;

  if constexpr (PASS == 1) {
    const int tile = blockIdx.x / nsplit, split = blockIdx.x % nsplit;
    const int i0 = tile * kCols;
    if (blockIdx.x == 0 && h == 0 && tid == 0 && (int64_t)a.seq_lens[b] > s.L)
      set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    if (i0 >= s.count) return;
    load_queries<T, KV4, D>(a, s, h, b, i0, queries, col_unit[0]);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (O::PREP && split == 0) save_queries<S>(saved + (head * chunks_most + tile) * S::Q_SAVED, queries, col_unit[0]);
    const int last = i0 + kCols < s.count ? i0 + kCols : s.count;
    int64_t kend = s.past + s.first + last;  // keys that the last of the queries sees
    kend = kend < s.L ? kend : s.L;
    const int64_t whole = s.past + s.first + i0 + 1;  // keys below it are seen by every query
    // Per column (8n + 2t + e): reference and sum of exp2(logit - reference)
    // over the rows of this lane.  The reference need not be the maximum: it
    // moves when a logit passes it by 2^8.
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
    bool set = false;  // every column of this warp has a reference
    const int64_t turn = (int64_t)nsplit * 4 * S::WROWS;
    const int64_t start = ((int64_t)split * 4 + warp) * S::WROWS;
    for (int64_t j0 = start; j0 < kend; j0 += turn) {
      keys.load(a, table, h, j0, kend, blocks, past_pool);
      bool plain = j0 + S::WROWS <= whole;
#pragma unroll
      for (int x = 0; x < S::MT; ++x) plain = plain && keys.ok[x][0] && keys.ok[x][1];
      plain = __all_sync(kFullMask, plain);
      auto unit_of = [&](int col, int x, int i) {
        float u = O::SCALED ? qscale * col_unit[0][col] : qscale;
        if constexpr (S::KPARTS == 2) u *= keys.back[x][i];
        return u;
      };
      auto highest = [&](const float (&z)[S::MT][2]) {
        float up = fmaxf(z[0][0], z[0][1]);
        if constexpr (S::MT == 2) up = fmaxf(up, fmaxf(z[1][0], z[1][1]));
        return up;
      };
      if (plain && set) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          keys.product(queries, n, acc);
          float z[2][S::MT][2], top[2];  // logit - reference
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 0; x < S::MT; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) z[e][x][i] = __fsub_rn(acc[x][2 * i + e] * unit_of(n * 8 + 2 * t + e, x, i), m[n][e]);
            top[e] = highest(z[e]);
          }
          if (__any_sync(kFullMask, fmaxf(top[0], top[1]) > 8.f)) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (top[e] > 8.f) {
                const int col = n * 8 + 2 * t + e;
                float up = -INFINITY;  // (the logit itself: a reference plus a difference would be rounded)
#pragma unroll
                for (int x = 0; x < S::MT; ++x)
                  up = fmaxf(up, fmaxf(acc[x][e] * unit_of(col, x, 0), acc[x][2 + e] * unit_of(col, x, 1)));
                l[n][e] *= fast_exp2(m[n][e] - up);
                m[n][e] = up;
#pragma unroll
                for (int x = 0; x < S::MT; ++x)
#pragma unroll
                  for (int i = 0; i < 2; ++i) z[e][x][i] = __fsub_rn(acc[x][2 * i + e] * unit_of(col, x, i), up);
              }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < S::MT; ++x) l[n][e] += fast_exp2(z[e][x][0]) + fast_exp2(z[e][x][1]);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          keys.product(queries, n, acc);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = n * 8 + 2 * t + e;
            float z[S::MT][2];  // logit
#pragma unroll
            for (int x = 0; x < S::MT; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                z[x][i] = acc[x][2 * i + e] * unit_of(col, x, i);
                if (!(keys.ok[x][i] && j0 + 16 * x + 8 * i + g < whole + col)) z[x][i] = -INFINITY;
              }
            const float up = fmaxf(m[n][e], highest(z)), ref = up == -INFINITY ? 0.f : up;
            l[n][e] = m[n][e] == -INFINITY ? l[n][e] : l[n][e] * fast_exp2(m[n][e] - ref);
            m[n][e] = up;
#pragma unroll
            for (int x = 0; x < S::MT; ++x) l[n][e] += fast_exp2(z[x][0] - ref) + fast_exp2(z[x][1] - ref);
          }
        }
        // (a column whose logits are all -inf or NaN keeps the careful path)
        bool all_set = true;
#pragma unroll
        for (int n = 0; n < NT; ++n) all_set = all_set && m[n][0] > -INFINITY && m[n][1] > -INFINITY;
        set = __all_sync(kFullMask, all_set);
      }
    }
    if (past_pool) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    // join: the 8 lanes of a column, then the warps
    __shared__ float2 joined[4][kCols];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float M = m[n][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(kFullMask, M, o));
        float sum = l[n][e] * fast_exp2(m[n][e] - (M == -INFINITY ? 0.f : M));
        if (m[n][e] == -INFINITY) sum = l[n][e];  // nothing seen (0), or NaN
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(kFullMask, sum, o);
        if (g == 0) joined[warp][n * 8 + 2 * t + e] = make_float2(M, sum);
      }
    __syncthreads();
    if (tid < kCols && i0 + tid < s.count) {
      float M = -INFINITY, sum = 0.f;
      for (int w = 0; w < 4; ++w) M = fmaxf(M, joined[w][tid].x);
      for (int w = 0; w < 4; ++w) sum += joined[w][tid].y * fast_exp2(joined[w][tid].x - (M == -INFINITY ? 0.f : M));
      part[(head * a.T + i0 + tid) * nsplit + split] = make_float2(M, sum);
    }
  } else {
    // columns' log-sum-exps, +inf where a query does not count or sees nothing
    auto load_lse = [&](int c, int buf) {
      for (int r = tid; r < kCols; r += kTileThreads) {
        const int i = c * kCols + r;
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
    const int chunks = (s.count + kCols - 1) / kCols;
    int held = -1;  // the only query tile, once loaded
    const int64_t turn = (int64_t)gridDim.x * S::ROWS, mine = warp * S::WROWS;
    for (int64_t j0 = (int64_t)blockIdx.x * S::ROWS; j0 < s.L; j0 += turn) {
      const int64_t w0 = j0 + mine;
      keys.load(a, table, h, w0, s.L, blocks, past_pool);
      float sum[S::MT][2];
#pragma unroll
      for (int x = 0; x < S::MT; ++x) sum[x][0] = sum[x][1] = 0.f;
      // the first counted query that sees key j0 or a later one
      int64_t from = j0 - s.past - s.first;
      from = from > 0 ? from : 0;
      const int c0 = from < s.count ? (int)(from / kCols) : chunks;
      auto fetch = [&](int c) {
        if (c < chunks && !(chunks == 1 && held == 0)) {
          uint8_t* to = queries + (c & 1) * S::Q_BYTES;
          if constexpr (O::PREP)
            fetch_saved<S>(to, col_unit[c & 1], saved + (head * chunks_most + c) * S::Q_SAVED);
          else
            load_queries<T, KV4, D>(a, s, h, b, c * kCols, to, col_unit[c & 1]);
          load_lse(c, c & 1);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      fetch(c0);
      for (int c = c0; c < chunks; ++c) {
        const int buf = c & 1;
        fetch(c + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        // key j is seen by columns at or above j - past - first - 64 c
        const int64_t base = w0 - s.past - s.first - (int64_t)c * kCols;
        const int left = s.count - c * kCols;  // columns that are queries
        const bool plain = base + S::WROWS - 1 <= 0 && left >= kCols;
        auto add = [&](auto masked) {
#pragma unroll 2
          for (int n = 0; n < NT; ++n) {
            keys.product(queries + buf * S::Q_BYTES, n, acc);
            const int col = n * 8 + 2 * t;
            const float2 lse = *reinterpret_cast<const float2*>(&col_lse[buf][col]);
            float2 unit = make_float2(qscale, qscale);
            if constexpr (O::SCALED) {
              const float2 back = *reinterpret_cast<const float2*>(&col_unit[buf][col]);
              unit.x *= back.x;
              unit.y *= back.y;
            }
#pragma unroll
            for (int x = 0; x < S::MT; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float u0 = unit.x, u1 = unit.y;
                if constexpr (S::KPARTS == 2) u0 *= keys.back[x][i], u1 *= keys.back[x][i];
                float p0 = fast_exp2(__fsub_rn(acc[x][2 * i] * u0, lse.x));
                float p1 = fast_exp2(__fsub_rn(acc[x][2 * i + 1] * u1, lse.y));
                if constexpr (decltype(masked)::value) {
                  const int64_t r = base + 16 * x + 8 * i + g;
                  if (r > col || col >= left) p0 = 0.f;
                  if (r > col + 1 || col + 1 >= left) p1 = 0.f;
                }
                sum[x][i] += p0 + p1;
              }
          }
        };
        if (plain)
          add(std::false_type{});
        else
          add(std::true_type{});
        __syncthreads();
      }
      if (chunks == 1 && c0 == 0) held = 0;
#pragma unroll
      for (int x = 0; x < S::MT; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sum[x][i] += __shfl_xor_sync(kFullMask, sum[x][i], 1);
          sum[x][i] += __shfl_xor_sync(kFullMask, sum[x][i], 2);
          const int64_t j = w0 + 16 * x + 8 * i + g;
          if (t == 0 && keys.ok[x][i]) {
            const uint32_t blk = (uint32_t)__ldg(table + (j >> a.bs_log2));
            const uint64_t at = (blk * (uint64_t)a.H + h) * a.block_size + (j & (a.block_size - 1));
            a.w_out[at] = a.w_in[at] + sum[x][i];
          }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (past_pool) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  }
}

// ------------------------------------------------------------------ one query
constexpr int kStepThreads = 256;

// How a warp takes its rows.  16-bit rows are tensor-core operands as they
// lie: a lane loads its fragment (16 bytes of row g and of row g + 8 per 64
// bytes of row), and the one query stands in all 8 columns, so every lane gets
// its rows' logits without a conversion or a shuffle.  fp32 rows are summed by
// the lanes that share a row.  4-bit rows: packed words and scale codes, as
// KeyQuery wants them.
template <typename T, bool KV4, int D>
struct StepRows {
  static constexpr int RB = KV4 ? D / 2 : D * (int)sizeof(T);
  static constexpr bool MMA = sizeof(T) == 2;
  // MMA: 64-byte blocks per row, 16-row tiles per turn (8 loads in flight)
  static constexpr int NB = RB < 64 ? 1 : RB / 64, TILES = NB < 4 ? 4 / NB : 1;
  // else: lanes per row, 16-byte pieces per lane, rows per load, rows per lane
  static constexpr int LPR = RB / 16 < 32 ? RB / 16 : 32, CPL = RB / 16 / LPR, RP = 32 / LPR, R = 8 / CPL;
  static constexpr int PACKED = D == 256 ? 1 : 2;  // 16-row tiles of 4-bit rows per turn
  static constexpr int RW = KV4 ? 16 * PACKED : MMA ? 16 * TILES : RP * R;  // rows per warp and turn
  static constexpr bool ORDERS = KV4 || !MMA || D != 256;  // by length, where that pays (by_length.cuh)
};

template <typename T, bool KV4, int D>
__global__ void __launch_bounds__(kStepThreads, KV4 ? 3 : 0) key_weights_step_kernel(KeyWeightArgs a, float qscale, float* far,
                                                                        int64_t far_stride, int by_length) {
  using S = StepRows<T, KV4, D>;
  using O = Op<T, false>;
  constexpr int RB = S::RB, RW = S::RW, E = 16 / (int)sizeof(T);
  extern __shared__ float near[];
  __shared__ float red[2][kStepThreads / 32];
  __shared__ float cta_m, cta_l;
  pdl_wait();
  pdl_launch_dependents();
  const int ns = gridDim.x, rank = blockIdx.x, h = blockIdx.y;
  const int b = S::ORDERS && by_length ? nth_longest(a.seq_lens, gridDim.z, blockIdx.z) : (int)blockIdx.z;
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
  const uint32_t seen = vis < hi ? vis : hi;  // keys [lo, seen) have a logit
  const uint32_t page_bytes = KV4 ? kv4_page_bytes(bs, D) : bs * RB;
  const char* const pages = static_cast<const char*>(a.k_pool) + (int64_t)h * page_bytes;
  const uint64_t block_bytes = (uint64_t)a.H * page_bytes;
  const T* const q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1];

  float top = -INFINITY;
  constexpr int kWarps = kStepThreads / 32;
  auto ids_of = [&](uint32_t j0) {  // lane l: the l-th page from key j0's
    const uint32_t pg = (j0 >> sh) + lane;
    return j0 < seen && pg << sh < seen ? table[pg] : -1;
  };
  uint32_t j0 = lo + warp * RW;  // (a turn past the last position fits 32 bits unsigned)
  int ids = ids_of(j0);
  bool past_pool = false;
  // Row j of the turn at j0: its page (block 0's for one that is not seen).
  auto page_of = [&](uint32_t j, bool& ok) -> const char* {
    const uint32_t blk = (uint32_t)__shfl_sync(kFullMask, ids, (int)((j >> sh) - (j0 >> sh)));
    ok = j < seen && blk < blocks;
    past_pool |= j < seen && (int)blk >= (int)blocks;
    return pages + (ok ? blk : 0u) * block_bytes;
  };
  auto locate = [&](uint32_t j, bool& ok) -> const char* { return page_of(j, ok) + (int)(j & (bs - 1)) * RB; };
  if constexpr (KV4) {
    using W = KeyWords<D>;
    using Q = KeyQuery<T, D>;
    const int g = lane >> 2, t = lane & 3;
    Q query;
    query.load(q);
    query.prepare(qscale);
    for (; j0 < seen; j0 += kWarps * RW) {
      const int next = ids_of(j0 + kWarps * RW);
      uint32_t words[S::PACKED][2][W::KW], codes[S::PACKED][2][W::SETS];
      bool ok[S::PACKED][2];
#pragma unroll
      for (int x = 0; x < S::PACKED; ++x) {
        const char* above = pages;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t j = j0 + x * 16 + g + 8 * i;
          const char* page;
          if (i == 1 && bs >= 16) {  // on the page of the row 8 above
            page = above;
            ok[x][1] = ok[x][0] && j < seen;
          } else {
            page = page_of(j, ok[x][i]);
          }
          above = page;
          const int row = (int)(j & (bs - 1));
          const char* src = page + row * RB + t * W::KB;
#pragma unroll
          for (int c = 0; c < W::KC; ++c) {
            if constexpr (W::KB == 16)
              *reinterpret_cast<uint4*>(&words[x][i][4 * c]) = ld_global_nc<uint4>(src + 64 * c);
            else
              *reinterpret_cast<uint2*>(&words[x][i][0]) = ld_global_nc<uint2>(src);
          }
          const char* sc = page + bs * RB + row * (D / 16);
#pragma unroll
          for (int k = 0; k < W::SETS; ++k)
            codes[x][i][k] = __ldg(reinterpret_cast<const uint16_t*>(sc + Q::scale_at(k)));
        }
      }
#pragma unroll
      for (int x = 0; x < S::PACKED; ++x) {
        float z2[2];
        query.logits(words[x][0], words[x][1], codes[x][0], codes[x][1], z2[0], z2[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float all = query.finish(z2[i]);
          const float dot = ok[x][i] ? all : -INFINITY;
          top = fmaxf(top, dot);
          const uint32_t j = j0 + x * 16 + g + 8 * i;
          if (t == 0 && j < seen) z[j - lo] = dot;
        }
      }
      ids = next;
    }
  } else if constexpr (S::MMA) {
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
          const uint32_t j = j0 + x * 16 + g + 8 * i;
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
        const uint32_t j = j0 + r * S::RP + lane / S::LPR;
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
  const int mine = hi - lo, logits = (int)seen > lo ? (int)seen - lo : 0;
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
size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Key ranges of the first pass: one wave of per_sm CTAs per SM, with
// two tiles of 32 keys a warp.  A CTA costs 4 us beside its keys (lengths,
// then queries, then a table entry, then keys), so more and smaller ones are
// slower.
int split_of(int B, int H, int count, int64_t keys, int per_sm) {
  const int64_t tiles = (int64_t)B * H * ((count + kCols - 1) / kCols);
  int64_t ns = per_sm * device_sm_count() / tiles;
  const int64_t most = keys / (4 * 32 * 2);
  ns = ns < most ? ns : most;
  return ns < 1 ? 1 : ns > 16 ? 16 : (int)ns;
}

bool takes_tcgen05(int D) { return D == 64 || D == 128; }  // key_weights_tc.cu

int counted_most(int T, int window) { return window > 0 && window < T ? window : T; }

template <typename T, bool KV4, int D>
int tile_launch(const KeyWeightArgs& a, cudaStream_t st) {
  using S = Shape<T, KV4, D>;
  const float qscale = a.scale * kLog2e;
  const int64_t keys = (int64_t)a.max_pages * a.block_size;
  if (keys == 0) return B2PA_OK;
  const int count = counted_most(a.T, a.window);
  const int ns = split_of(a.B, a.H, count, keys, S::KPARTS == 2 ? 4 : 3);
  float2* part = static_cast<float2*>(a.workspace);
  const int chunks = (count + kCols - 1) / kCols;
  uint8_t* saved = static_cast<uint8_t*>(a.workspace) + up256((size_t)a.B * a.H * a.T * 16 * sizeof(float2));
  auto k1 = key_weights_tile_kernel<T, KV4, D, 1>;
  auto k2 = key_weights_tile_kernel<T, KV4, D, 2>;
  int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(k1), S::Q_BYTES);
  if (rc == B2PA_OK) rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(k2), 2 * S::Q_BYTES);
  if (rc != B2PA_OK) return rc;
  cudaError_t e = launch_pdl(k1, dim3((unsigned)((count + kCols - 1) / kCols * ns), (unsigned)a.H, (unsigned)a.B),
                             dim3(kTileThreads), S::Q_BYTES, st, a, qscale, ns, part, saved, chunks);
  // One tile of queries stays in shared memory while a CTA takes several key
  // tiles; more than one passes by for every key tile.
  int64_t tiles = (keys + S::ROWS - 1) / S::ROWS;
  if (count <= kCols) {
    const int64_t most = (int64_t)8 * device_sm_count() / ((int64_t)a.B * a.H) + 1;
    tiles = tiles < most ? tiles : most;
  }
  if (e == cudaSuccess)
    e = launch_pdl(k2, dim3((unsigned)tiles, (unsigned)a.H, (unsigned)a.B), dim3(kTileThreads), 2 * S::Q_BYTES, st, a,
                   qscale, ns, part, saved, chunks);
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

template <typename T, bool KV4, int D>
int step_launch(const KeyWeightArgs& a, cudaStream_t st) {
  const int64_t keys = (int64_t)a.max_pages * a.block_size;
  if (keys == 0) return B2PA_OK;
  const int ns = step_split((int64_t)a.B * a.H, keys);
  const int64_t per = (keys + ns - 1) / ns + 128;  // a CTA's keys, rounded up to whole turns
  const bool far = per > kNearKeys + 128;
  const int smem = far ? 0 : (int)(per * 4);
  auto kern = key_weights_step_kernel<T, KV4, D>;
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
  // CTAs on an SM: by registers (64 a thread, else 80)
  using S = StepRows<T, KV4, D>;
  constexpr bool ROWS32 = !KV4 && sizeof(T) == 4, ROWS16 = !KV4 && !ROWS32;
  const int by_length = S::ORDERS && orders_by_length(a.B, (int64_t)ns * a.H * a.B, ROWS32 && D != 128 ? 4 : 3, keys / ns,
                                                      ROWS32 ? 256 : 512,
                                                      ROWS32                ? 150
                                                      : !ROWS16 || D == 128 ? 800
                                                      : D == 64             ? 2600
                                                                            : 1200);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, a.scale * kLog2e,
                                           far ? static_cast<float*>(a.workspace) : static_cast<float*>(nullptr), keys,
                                           by_length);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "key_weights launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

template <typename T>
int weights_as(const KeyWeightArgs& a, cudaStream_t s) {
  if (a.pool_dtype == B2PA_DTYPE_KV4) {
    switch (a.D) {
      case 64: return step_launch<T, true, 64>(a, s);
      case 128: return step_launch<T, true, 128>(a, s);
      default: return a.T == 1 ? step_launch<T, true, 256>(a, s) : tile_launch<T, true, 256>(a, s);
    }
  }
  switch (a.D) {
    case 16: return a.T == 1 ? step_launch<T, false, 16>(a, s) : tile_launch<T, false, 16>(a, s);
    case 32: return a.T == 1 ? step_launch<T, false, 32>(a, s) : tile_launch<T, false, 32>(a, s);
    case 64: return step_launch<T, false, 64>(a, s);
    case 128: return step_launch<T, false, 128>(a, s);
    default: return a.T == 1 ? step_launch<T, false, 256>(a, s) : tile_launch<T, false, 256>(a, s);
  }
}

}  // namespace

size_t key_weights_workspace(int B, int H, int T, int D, int max_pages, int block_size, int dtype, int pool_dtype) {
  const int64_t keys = (int64_t)max_pages * block_size;
  if (T == 1) {
    const int ns = step_split((int64_t)B * H, keys);
    return (keys + ns - 1) / ns > kNearKeys ? (size_t)B * H * keys * sizeof(float) : 0;
  }
  // the first pass's partials, then its converted queries: at most two fp16
  // halves a channel, rows padded by a block, and a factor each
  size_t saved = 0;
  if (!takes_tcgen05(D) && (pool_dtype == B2PA_DTYPE_KV4 || dtype == B2PA_DTYPE_F32)) {
    const size_t blocks = D < 32 ? 1 : D / 32, parts = dtype == B2PA_DTYPE_F32 ? 2 : 1;
    saved = (size_t)B * H * ((T + kCols - 1) / kCols) * (parts * kCols * (blocks + 1) * 64 + kCols * 4);
  }
  return up256((size_t)B * H * T * 16 * sizeof(float2)) + saved;
}

int launch_key_weights(const KeyWeightArgs& a, cudaStream_t s) {
  if (a.T > 1 && takes_tcgen05(a.D)) return launch_key_weights_tc(a, counted_most(a.T, a.window), s);
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return weights_as<float>(a, s);
    case B2PA_DTYPE_BF16: return weights_as<__nv_bfloat16>(a, s);
    default: return weights_as<__half>(a, s);
  }
}

}  // namespace b2pa
