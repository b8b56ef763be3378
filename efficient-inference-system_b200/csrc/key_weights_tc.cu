// key_weights_tc.cu -- accumulated attention weight of every cached key from
// several queries, for head_dim 64 and 128 (what is computed: key_weights.cu).
//
// Two launches over one product, as in key_weights.cu, but on the 5th
// generation tensor cores: tiles of 128 keys x up to 128 queries, fp32
// accumulators in TMEM, so that the warps are left with the softmax -- about
// six instructions a logit -- and with putting key rows in place.
//   PASS 1: queries are the product's rows.  A thread owns one query, reads its
//     logits from TMEM and keeps the running maximum and sum in two registers.
//   PASS 2: keys are the rows.  A thread owns one key and adds
//     exp(logit - lse) along the queries: no atomics, no shuffles.
// Per CTA: 4 warps for that, two times 4 that load key rows (4-bit rows are
// unpacked, fp32 rows split in two fp16 halves and scaled, on the way to shared
// memory; each group has every other tile and a stage of its own, so that two
// tiles' loads are under way), one that issues the products; two accumulators,
// every hand-over through an mbarrier.  Operands lie in K-major tiles with the
// 128-byte swizzle.  Two CTAs per SM.
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "kv4_mma.cuh"
#include "tcgen05.cuh"

namespace b2pa {

namespace {

constexpr int kRows = 128;       // keys, and queries, per tile
constexpr int kRoleThreads = 128;
constexpr int kTcThreads = 3 * kRoleThreads + 32;  // softmax, even tiles' and odd tiles' loads; products
constexpr int kLate = 4;         // tiles whose masks are kept: loading runs at most 3 ahead of reading

template <typename T, bool KV4, int D>
struct Tc {
  static constexpr bool F32 = std::is_same<T, float>::value;
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value && !KV4;             // operand type
  static constexpr bool QSCALED = F32 || (KV4 && std::is_same<T, __nv_bfloat16>::value);  // into fp16's range
  static constexpr bool KSCALED = F32 && !KV4;
  static constexpr int QP = F32 ? 2 : 1, KP = KSCALED ? 2 : 1;  // fp16 halves
  static constexpr int TILE = kRows * D * 2;
  static constexpr int SMEM = QP * TILE + 2 * KP * TILE + 1024;
};

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

// Byte offset of 8-channel piece c of row r in a tile.
__device__ __forceinline__ uint32_t place(int r, int c) {
  return (uint32_t)(c >> 3) * (kRows * 128) + tc::sw128_offset(r, c & 7);
}

// Rows 32 warp .. 32 warp + 31 of a tile from fp32 or 16-bit values, as fp16 (or
// bf16) operands; src_of(r): row r's values, null for zeros (read from `any`
// then: no load hangs on a branch); done(r, back): the factor that undoes its
// scaling.  D / 8 lanes read along a row, four rows' loads are under way at once.
template <typename T, int D, bool SCALED, bool PERM, int PARTS, typename Src, typename Done>
__device__ __forceinline__ void put_rows(int warp, uint8_t* tile, const void* any, Src src_of, Done done) {
  constexpr int LPR = D / 8, RPI = 32 / LPR, N = 16 / (int)sizeof(T), W = 8 / N;
  const int lane = threadIdx.x & 31, c = lane % LPR;
#pragma unroll 1
  for (int it0 = 0; it0 < LPR; it0 += 4) {
    uint4 raw[4][W];
    uint32_t there = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const T* src = src_of(warp * 32 + (it0 + u) * RPI + lane / LPR);
      there |= (src != nullptr ? 1u : 0u) << u;
      src = src != nullptr ? src : static_cast<const T*>(any);
#pragma unroll
      for (int i = 0; i < W; ++i) raw[u][i] = ld_global_nc<uint4>(src + 8 * c + i * N);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = warp * 32 + (it0 + u) * RPI + lane / LPR;
      if (!(there >> u & 1u)) {
#pragma unroll
        for (int i = 0; i < W; ++i) raw[u][i] = make_uint4(0, 0, 0, 0);
      }
      uint4 hi = raw[u][0], lo = make_uint4(0, 0, 0, 0);
      float back = 1.f;
      if constexpr (SCALED) {
        float x[8], top = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          Vec<T, N> v;
          v.w = raw[u][i];
          v.to_float(x + i * N);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
        for (int o = LPR / 2; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
        const float f = range_factor(top, back);
        if constexpr (PERM) {
          const float y[8] = {x[0], x[4], x[1], x[5], x[2], x[6], x[3], x[7]};
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = y[i];
        }
        split8(x, f, hi, lo);
      } else if constexpr (PERM) {
        hi = make_uint4(__byte_perm(hi.x, hi.z, 0x5410), __byte_perm(hi.x, hi.z, 0x7632),
                        __byte_perm(hi.y, hi.w, 0x5410), __byte_perm(hi.y, hi.w, 0x7632));
      }
      *reinterpret_cast<uint4*>(tile + place(r, c)) = hi;
      if constexpr (PARTS == 2) *reinterpret_cast<uint4*>(tile + kRows * D * 2 + place(r, c)) = lo;
      if (c == 0) done(r, back);
    }
  }
}

__device__ __forceinline__ void role_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kRoleThreads) : "memory"); }

// Waits for a phase; gives up after the library's limit, or when another role
// did.  The timer is read every 256 tries only: reading it takes about a
// microsecond, in which a phase that completes goes unseen.
__device__ __forceinline__ bool wait_or_stop(uint64_t* bar, uint32_t parity, int32_t* status, volatile int* stop) {
  uint64_t t0 = 0;
  for (uint32_t n = 1;; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if (n % 256 != 0) continue;
    if (*stop) return false;
    const uint64_t now = global_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      set_status(status, B2PA_ERR_DEVICE_TIMEOUT);
      *stop = 1;
      return false;
    }
  }
}

// Rows 32 warp .. 32 warp + 31 of a tile as they lie (16-bit values): copied
// asynchronously, complete when it returns.
template <typename T, int D, typename Src>
__device__ __forceinline__ void copy_rows(int warp, uint8_t* tile, const void* any, Src src_of) {
  constexpr int LPR = D / 8, RPI = 32 / LPR;
  const int lane = threadIdx.x & 31, c = lane % LPR;
#pragma unroll
  for (int it = 0; it < LPR; ++it) {
    const int r = warp * 32 + it * RPI + lane / LPR;
    const T* src = src_of(r);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(tile) + place(r, c)),
                 "l"(src != nullptr ? static_cast<const void*>(src + 8 * c) : any), "r"(src != nullptr ? 16 : 0)
                 : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, bool KV4, int D, int PASS>
__global__ void __launch_bounds__(kTcThreads, 2) key_weights_tc_kernel(KeyWeightArgs a, float qscale, int nsplit, float2* part) {
  using S = Tc<T, KV4, D>;
  extern __shared__ uint8_t tc_smem[];
  __shared__ uint64_t full[2], empty[2], acc_full[2], acc_empty[2], q_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int stop_flag;
  __shared__ uint32_t key_mask[kLate][4];  // which keys of a tile are there
  __shared__ __align__(16) float key_back[S::KSCALED ? kLate : 1][kRows];
  __shared__ __align__(16) float q_unit[kRows], q_lse[kRows];  // (a query's unit * scale; -lse)
  volatile int* stop = &stop_flag;
  uint8_t* const base = tc_smem + (1024 - (smem_u32(tc_smem) & 1023u)) % 1024;
  uint8_t* const qt = base;
  uint8_t* const kt = base + S::QP * S::TILE;

  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], kRoleThreads);
      mbar_init(&empty[i], 1);
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kRoleThreads);
    }
    mbar_init(&q_full, kRoleThreads);
    stop_flag = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tc::tmem_alloc(&tmem_slot, 256);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;

  // PASS 2 needs nothing of PASS 1 but its partial sums, and PASS 1 let it start
  // after waiting for what was before: it waits where it reads them.
  if (PASS == 1) {
    pdl_wait();
    pdl_launch_dependents();
  }
  const Span s = span_of(a, b);
  const int32_t* table = a.page_table + (int64_t)b * a.pt_stride;
  const int64_t head = (int64_t)b * a.H + h;
  const uint32_t blocks = a.num_blocks < INT32_MAX ? (uint32_t)a.num_blocks : (uint32_t)INT32_MAX;
  const int bs = a.block_size, sh = a.bs_log2;
  const int64_t q0 = s.past + s.first;  // position of counted query 0

  // The work of this CTA, the same for every role: chunks of queries, and for
  // each the key tiles tile0, tile0 + step, .. below tiles_of(chunk).
  const int split = PASS == 1 ? blockIdx.x % nsplit : 0;
  const int tile0 = PASS == 1 ? split : (int)blockIdx.x, step = PASS == 1 ? nsplit : (int)gridDim.x;
  const int chunk0 = PASS == 1 ? (int)blockIdx.x / nsplit : 0;
  const int chunks = PASS == 1 ? chunk0 + 1 : (s.count + kRows - 1) / kRows > 1 ? (s.count + kRows - 1) / kRows : 1;
  auto tiles_of = [&](int c) -> int {  // PASS 2: the first chunk also copies the weights of keys that nobody sees
    const int last = (c + 1) * kRows < s.count ? (c + 1) * kRows : s.count;
    int64_t end = PASS == 2 && c == 0 ? s.L : q0 + last;
    end = end < s.L ? end : s.L;
    return end > 0 && blocks > 0 ? (int)((end + kRows - 1) / kRows) : 0;
  };
  const bool idle = PASS == 1 && chunk0 * kRows >= s.count;

  if (!idle && warp < 4) {
    // ------------------------------------------------------------- softmax
    bool ok = true;
    int i = 0;  // tiles so far
    for (int c = chunk0; c < chunks; ++c) {
      const int n = s.count - c * kRows;  // queries of the chunk (and zeros behind them)
      const int tiles = tiles_of(c);
      // PASS 1, up to 64 queries: heads take turns with the upper and the lower
      // rows, so that all four parts of the SM get exponentials to compute
      const int shift = PASS == 1 && n <= kRows / 2 && (h & 1) ? kRows / 2 : 0;
      const int mine = tid - shift;  // this thread's query
      float m = -INFINITY, l = 0.f;
      if (tile0 < tiles) {
      // (every warp passes the barriers of every chunk, whatever became of its waits)
      role_sync();  // nobody reads the chunk before any more
      {
        const T* const q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1] +
                           (int64_t)(s.first + c * kRows) * a.sq[2];
        const auto src = [&](int r) { return r >= shift && r - shift < n ? q + (r - shift) * a.sq[2] : nullptr; };
        if constexpr (!S::QSCALED && !KV4) {
          copy_rows<T, D>(warp, qt, a.q, src);
          q_unit[tid] = qscale;
        } else {
          put_rows<T, D, S::QSCALED, KV4, S::QP>(warp, qt, a.q, src, [&](int r, float back) { q_unit[r] = qscale * back; });
        }
      }
      tc::fence_proxy_async_smem();
      mbar_arrive(&q_full);
      if constexpr (PASS == 2) {
        pdl_wait();
        pdl_launch_dependents();
        float lse = INFINITY;
        if (tid < n) {
          const float2* p = part + (head * a.T + c * kRows + tid) * nsplit;
          float M = -INFINITY, l = 0.f;
          for (int k = 0; k < nsplit; ++k) M = fmaxf(M, p[k].x);
          const float ref = M == -INFINITY ? 0.f : M;
          for (int k = 0; k < nsplit; ++k) l += p[k].y * fast_exp2(p[k].x - ref);
          if (l != 0.f) lse = ref + log2f(l);
        }
        q_lse[tid] = -lse;
      }
      role_sync();
      const float unit = q_unit[tid];
      for (int tile = tile0; ok && tile < tiles; tile += step, ++i) {
        const int buf = i & 1;
        ok = __all_sync(kFullMask, wait_or_stop(&acc_full[buf], (uint32_t)(i >> 1) & 1u, a.status, stop));
        if (!ok) break;
        tc::fence_after_sync();
        const uint32_t acc = tmem + buf * kRows + ((uint32_t)warp << 21);  // this warp's 32 lanes
        const int64_t j0 = (int64_t)tile * kRows;
        if constexpr (PASS == 1) {
          if (warp * 32 - shift < n && warp * 32 >= shift) {  // (a warp of padding has nothing to do)
            const int64_t seen = q0 + c * kRows + mine + 1 - j0;  // keys of the tile that this query sees
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
              const int64_t left = seen - 32 * k;
              uint32_t mask = left >= 32 ? kFullMask : left <= 0 ? 0u : (1u << left) - 1u;
              mask &= key_mask[i % kLate][k];
              float v[32];
              tc::tmem_ld32(acc + 32 * k, v);
              if constexpr (S::KSCALED) {
                const float4* kb = reinterpret_cast<const float4*>(&key_back[i % kLate][32 * k]);
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                  const float4 y = kb[x];
                  v[4 * x] *= y.x;
                  v[4 * x + 1] *= y.y;
                  v[4 * x + 2] *= y.z;
                  v[4 * x + 3] *= y.w;
                }
              }
              if (!(unit > 0.f)) {  // (a scale that is not positive: the largest product shall be the largest logit)
                const float sign = unit < 0.f ? -1.f : 0.f;
#pragma unroll
                for (int x = 0; x < 32; ++x) v[x] *= sign;
              }
              if (__any_sync(kFullMask, mask != kFullMask)) {
#pragma unroll
                for (int x = 0; x < 32; ++x) v[x] = mask >> x & 1u ? v[x] : -INFINITY;
              }
              float top = fmax3(v[0], v[1], v[2]), top2 = fmax3(v[3], v[4], v[5]);
#pragma unroll
              for (int x = 6; x < 30; x += 4) {
                top = fmax3(v[x], v[x + 1], top);
                top2 = fmax3(v[x + 2], v[x + 3], top2);
              }
              top = fmax3(v[30], v[31], fmaxf(top, top2));
              const float size = unit != 0.f ? fabsf(unit) : 1.f;  // (hidden ones, at -inf, stay so)
              top = fmaxf(m, top * size);  // m, in logits
              const float ref = top == -INFINITY ? 0.f : top;
              const float2 u2 = make_float2(size, size), r2 = make_float2(-ref, -ref);
              const float2 zero = make_float2(0.f, 0.f);
              float2 sum0 = zero, sum1 = zero;
#pragma unroll
              for (int x = 0; x < 32; x += 4) {
                const float2 y = add2(fma2(make_float2(v[x], v[x + 1]), u2, zero), r2),
                             z = add2(fma2(make_float2(v[x + 2], v[x + 3]), u2, zero), r2);
                sum0 = add2(sum0, make_float2(fast_exp2(y.x), fast_exp2(y.y)));
                sum1 = add2(sum1, make_float2(fast_exp2(z.x), fast_exp2(z.y)));
              }
              l = (m == -INFINITY ? l : l * fast_exp2(m - ref)) + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
              m = top;
            }
          }
          tc::fence_before_sync();
          mbar_arrive(&acc_empty[buf]);
        } else {
          const bool there = key_mask[i % kLate][warp] >> lane & 1u;
          const int64_t first = j0 + tid - q0 - (int64_t)c * kRows;  // the first query of the chunk that sees this key
          const float back2 = S::KSCALED ? key_back[i % kLate][tid] : 1.f;
          const int lanes = (n < kRows ? n : kRows);
          float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
#pragma unroll 1
          for (int k = 0; 32 * k < lanes; ++k) {
            const int64_t before = first - 32 * k;  // queries of these 32 that do not see the key
            uint32_t mask = before <= 0 ? kFullMask : before >= 32 ? 0u : kFullMask << before;
            if (lanes - 32 * k < 32) mask &= (1u << (lanes - 32 * k)) - 1u;
            const bool all = __all_sync(kFullMask, mask == kFullMask);
            float v[32];
            tc::tmem_ld32(acc + 32 * k, v);
            const float4* ls = reinterpret_cast<const float4*>(&q_lse[32 * k]);
            const float4* un = reinterpret_cast<const float4*>(&q_unit[32 * k]);
            if constexpr (S::KSCALED) {
#pragma unroll
              for (int x = 0; x < 32; ++x) v[x] *= back2;
            }
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const float4 z = ls[x];
              float4 u = make_float4(qscale, qscale, qscale, qscale);
              if constexpr (S::QSCALED) u = un[x];
              const float2 zero = make_float2(0.f, 0.f);
              float2 p = add2(fma2(make_float2(v[4 * x], v[4 * x + 1]), make_float2(u.x, u.y), zero), make_float2(z.x, z.y));
              float2 r = add2(fma2(make_float2(v[4 * x + 2], v[4 * x + 3]), make_float2(u.z, u.w), zero), make_float2(z.z, z.w));
              p = make_float2(fast_exp2(p.x), fast_exp2(p.y));
              r = make_float2(fast_exp2(r.x), fast_exp2(r.y));
              if (!all) {
                p.x = mask >> (4 * x) & 1u ? p.x : 0.f;
                p.y = mask >> (4 * x + 1) & 1u ? p.y : 0.f;
                r.x = mask >> (4 * x + 2) & 1u ? r.x : 0.f;
                r.y = mask >> (4 * x + 3) & 1u ? r.y : 0.f;
              }
              sum0 = add2(sum0, p);
              sum1 = add2(sum1, r);
            }
          }
          tc::fence_before_sync();
          mbar_arrive(&acc_empty[buf]);
          if (there) {
            const int64_t j = j0 + tid;
            const uint32_t blk = (uint32_t)__ldg(table + (j >> sh));
            const uint64_t at = (blk * (uint64_t)a.H + h) * bs + (j & (bs - 1));
            a.w_out[at] = (c == 0 ? a.w_in[at] : a.w_out[at]) + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
          }
        }
      }
      }
      if (PASS == 1 && ok && mine >= 0 && mine < n)
        part[(head * a.T + c * kRows + mine) * nsplit + split] = make_float2(m, l);
    }
  } else if (!idle && warp < 12) {
    // ------------------------------------------------------------ key rows
    const int group = (warp - 4) >> 2, w = warp & 3;  // tiles of this group's parity; rows 32 w .. 32 w + 31
    const uint32_t page_bytes = KV4 ? kv4_page_bytes(bs, D) : bs * D * (int)sizeof(T);
    const char* const pool = static_cast<const char*>(a.k_pool) + (uint64_t)h * page_bytes;
    const uint64_t block_bytes = (uint64_t)a.H * page_bytes;
    uint8_t* const to = kt + group * (S::KP * S::TILE);
    bool ok = true, past_pool = false;
    // Pages of a tile, one per lane (a tile starts a page): ids past the pool
    // and pages behind the sequence as -1.
    auto ids_of = [&](int tile) -> int {
      const int64_t page = ((int64_t)tile * kRows >> sh) + lane;
      const int id = lane < kRows >> sh && page << sh < s.L ? __ldg(table + page) : -1;
      past_pool |= id >= (int)blocks;
      return id < (int)blocks ? id : -1;
    };
    constexpr int LPR = D / 32, IT = LPR;  // 4-bit rows: lanes (16 bytes each) per row, rows per lane
    uint4 raw[KV4 ? IT : 1];
    uint32_t sc[KV4 ? IT : 1];
    int ids = -1;
    auto fetch = [&](int tile) {  // a tile's pages, and its 4-bit rows
      ids = ids_of(tile);
      if constexpr (KV4) {
#pragma unroll
        for (int x = 0; x < IT; ++x) {
          const int r = w * 32 + x * (32 / LPR) + lane / LPR;
          const int blk = __shfl_sync(kFullMask, ids, r >> sh);
          const char* page = pool + (uint32_t)(blk >= 0 ? blk : 0) * block_bytes;
          const int row = r & (bs - 1);
          raw[x] = ld_global_nc<uint4>(page + row * (D / 2) + 16 * (lane % LPR));
          sc[x] = __ldg(reinterpret_cast<const uint16_t*>(page + bs * (D / 2) + row * (D / 16) + 2 * (lane % LPR)));
        }
      }
    };
    int i = 0;  // tiles so far, of both groups
    for (int c = chunk0; c < chunks && ok; ++c) {
      const int tiles = tiles_of(c);
      int mine = tile0 + ((i & 1) == group ? 0 : step);  // this group's first tile of the chunk
      if (mine < tiles) fetch(mine);
      for (int tile = tile0; tile < tiles; tile += step, ++i) {
        if ((i & 1) != group) continue;
        if (i >= 2) ok = __all_sync(kFullMask, wait_or_stop(&empty[group], (uint32_t)((i >> 1) - 1) & 1u, a.status, stop));
        if (!ok) break;
        const int64_t j0 = (int64_t)tile * kRows;
        const int my_blk = __shfl_sync(kFullMask, ids, (w * 32 + lane) >> sh);
        const uint32_t mask = __ballot_sync(kFullMask, my_blk >= 0 && j0 + w * 32 + lane < s.L);
        if (lane == 0) key_mask[i % kLate][w] = mask;
        if constexpr (KV4) {
#pragma unroll
          for (int x = 0; x < IT; ++x) {
            const int q = x * (32 / LPR) + lane / LPR, r = w * 32 + q, p0 = 4 * (lane % LPR);
            const bool there = mask >> q & 1u;
            const __half2 s0 = scale_pair(sc[x], 0x4040), s1 = scale_pair(sc[x], 0x4141);
            const uint32_t* word = &raw[x].x;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<uint4*>(to + place(r, p0 + k)) =
                  there ? unpack_word(word[k], k < 2 ? s0 : s1) : make_uint4(0, 0, 0, 0);
          }
        } else {
          const auto src = [&](int r) -> const T* {
            const int blk = __shfl_sync(kFullMask, ids, r >> sh);
            if (!(mask >> (r & 31) & 1u)) return nullptr;
            return reinterpret_cast<const T*>(pool + (uint32_t)blk * block_bytes) + (r & (bs - 1)) * D;
          };
          if constexpr (S::KSCALED)
            put_rows<T, D, true, false, S::KP>(w, to, a.k_pool, src, [&](int r, float back) { key_back[i % kLate][r] = back; });
          else
            copy_rows<T, D>(w, to, a.k_pool, src);
        }
        tc::fence_proxy_async_smem();
        mbar_arrive(&full[group]);
        if (tile + 2 * step < tiles) fetch(tile + 2 * step);
      }
    }
    if (past_pool) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  } else if (!idle && lane == 0) {
    // ------------------------------------------------------------ products
    bool ok = true;
    int i = 0;
    const uint64_t dq = tc::smem_desc(smem_u32(qt), 16, 1024), dk = tc::smem_desc(smem_u32(kt), 16, 1024);
    int loads = 0;  // of queries so far: only chunks with tiles load them
    for (int c = chunk0; c < chunks && ok; ++c) {
      const int tiles = tiles_of(c);
      if (tile0 >= tiles) continue;
      ok = wait_or_stop(&q_full, (uint32_t)loads & 1u, a.status, stop);
      ++loads;
      int n = s.count - c * kRows;
      n = n < 1 ? 32 : n < kRows ? (n + 31) / 32 * 32 : kRows;
      const uint32_t idesc = tc::idesc_f16(128, PASS == 1 ? kRows : n, S::BF16 ? 1 : 0, 0, 0);
      for (int tile = tile0; tile < tiles && ok; tile += step, ++i) {
        const int st = i & 1;
        ok = wait_or_stop(&full[st], (uint32_t)(i >> 1) & 1u, a.status, stop) &&
             (i < 2 || wait_or_stop(&acc_empty[st], (uint32_t)((i >> 1) - 1) & 1u, a.status, stop));
        if (!ok) break;
        tc::fence_after_sync();
        const uint64_t dks = dk + (uint64_t)((st * S::KP * S::TILE) >> 4);
        const uint32_t acc = tmem + st * kRows;
#pragma unroll
        for (int x = 0; x < D / 16; ++x) {
          const uint64_t off = (uint64_t)(((x >> 2) * (kRows * 128) + (x & 3) * 32) >> 4);
          const uint64_t q = dq + off, k = dks + off;
          auto mma = [&](uint64_t u, uint64_t v, bool more) {
            tc::mma_f16_ss(acc, PASS == 1 ? u : v, PASS == 1 ? v : u, idesc, more);
          };
          mma(q, k, x > 0);
          if constexpr (S::QP == 2) mma(q + (S::TILE >> 4), k, true);
          if constexpr (S::KP == 2) mma(q, k + (S::TILE >> 4), true);
        }
        tc::commit(&empty[st]);
        tc::commit(&acc_full[st]);
      }
    }
  }
  if (PASS == 1 && blockIdx.x == 0 && h == 0 && tid == 0 && (int64_t)a.seq_lens[b] > s.L)
    set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  __syncwarp();
  if (PASS == 2) {  // (and where a CTA had no keys)
    pdl_wait();
    pdl_launch_dependents();
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 256);
  }
}

template <typename T, bool KV4, int D>
int tc_launch(const KeyWeightArgs& a, int count, cudaStream_t st) {
  using S = Tc<T, KV4, D>;
  const float qscale = a.scale * kLog2e;
  const int64_t keys = (int64_t)a.max_pages * a.block_size, tiles = (keys + kRows - 1) / kRows;
  if (keys == 0) return B2PA_OK;
  float2* part = static_cast<float2*>(a.workspace);
  // Shares of 16 key tiles of the longest sequence: a CTA starts up in about 3
  // us and takes a tile in about 1.5, and with one wave of larger shares the
  // longest sequence sets the time (4 sequences of 1,500 to 7,700 keys, 64
  // queries, 4-bit keys: one wave 113 us, shares of 16 tiles 89, of 8 100, of 4
  // 126); fewer tiles while they leave less than one wave of two CTAs per SM.
  const int64_t chunks = (count + kRows - 1) / kRows, pairs = (int64_t)a.B * a.H, wave = 2 * (int64_t)device_sm_count();
  auto shares = [&](int64_t have) {
    int64_t n = (tiles + 16 - 1) / 16;
    const int64_t fill = wave / have;
    n = n > fill ? n : fill;
    const int64_t most = (tiles + 1) / 2;
    n = n < most ? n : most;
    return n > 1 ? n : 1;
  };
  int64_t ns = shares(pairs * chunks);
  ns = ns > 16 ? 16 : ns;
  const int64_t gx = shares(pairs);
  auto k1 = key_weights_tc_kernel<T, KV4, D, 1>;
  auto k2 = key_weights_tc_kernel<T, KV4, D, 2>;
  int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(k1), S::SMEM);
  if (rc == B2PA_OK) rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(k2), S::SMEM);
  if (rc != B2PA_OK) return rc;
  cudaError_t e = launch_pdl(k1, dim3((unsigned)(chunks * ns), (unsigned)a.H, (unsigned)a.B), dim3(kTcThreads), S::SMEM, st,
                             a, qscale, (int)ns, part);
  if (e == cudaSuccess)
    e = launch_pdl(k2, dim3((unsigned)gx, (unsigned)a.H, (unsigned)a.B), dim3(kTcThreads), S::SMEM, st, a, qscale, (int)ns,
                   part);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "key_weights launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

template <typename T>
int tc_as(const KeyWeightArgs& a, int count, cudaStream_t st) {
  if (a.pool_dtype == B2PA_DTYPE_KV4)
    return a.D == 64 ? tc_launch<T, true, 64>(a, count, st) : tc_launch<T, true, 128>(a, count, st);
  return a.D == 64 ? tc_launch<T, false, 64>(a, count, st) : tc_launch<T, false, 128>(a, count, st);
}

}  // namespace

int launch_key_weights_tc(const KeyWeightArgs& a, int count, cudaStream_t s) {
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return tc_as<float>(a, count, s);
    case B2PA_DTYPE_BF16: return tc_as<__nv_bfloat16>(a, count, s);
    default: return tc_as<__half>(a, count, s);
  }
}

}  // namespace b2pa
