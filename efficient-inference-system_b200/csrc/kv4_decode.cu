// kv4_decode.cu -- single-query paged attention over a 4-bit cache (format:
// kv4.cuh).
//
// For sequence b the query sits at position seq_len - cur_len and sees keys
// 0 .. min(seq_len, seq_len - cur_len + 1) - 1; out = softmax(q.K^T scale).V
// with K and V the values the pages stand for, in fp32, stored in the type of
// q; zeros when no key is visible.
//
// A cached value is half a byte, so at HBM speed an SM has to take in over 40
// values a cycle: unpacking, not multiplying, is what could bound this
// kernel.  It is built to spend few instructions per packed word of 8:
//
//   * codes go to the tensor core (mma.sync m16n8k16) as they are.  A masked
//     nibble in the low bits of a half is the fp16 number c * 2^-24 (a
//     subnormal; 16 c * 2^-24 for the upper nibble, whose factor the other
//     operand carries), so a word of 8 codes becomes 4 operand registers with
//     one shift and four ANDs.  Stored codes are c + 8: the 8 is taken out
//     through the accumulator (K: it starts at -8 sum(q); V: one more product
//     against a constant operand sums the weights).  That leaves the rounding
//     of sums that are larger than the result, by 8 sum(p s) / |sum(p s c)|,
//     a hundred times for 1,000 keys of like weight: 1e-5 of the output, far
//     below a 16-bit one's own rounding; for fp32 one subtraction per register
//     takes it out first (5.1e-5 -> below 1e-6 of the output).
//   * scales stay out of the unpacking.  The 8 columns of the product that a
//     single query leaves idle are the groups: column n holds the query's
//     channels of group n and zeros (K), or the weights times group n's scale
//     (V).  So S[key] = sum_n s[key, n] C[key, n], one multiply per 16
//     values, and out[channel] is C[channel, its own group].
//   * both products keep fp32's accuracy: q and the weights enter as two fp16
//     halves (hi + lo, 22 bits; a 16-bit q needs one), scaled by powers of two
//     into fp16's range -- q by its own maximum, the weights by the largest V
//     scale so far, which is tracked like the softmax maximum.
//   * a lane fetches exactly the bytes that it consumes (its fragment of the
//     tile) with asynchronous copies into its own slots of a ring of two
//     stages, so the ring needs no block-wide barrier; only a tile's 16 K
//     scales rows and its visibility mask are read across the warp.
//
// One warp works on steps of two tiles of 16 keys (head_dim 256: one); the 8 (4)
// warps of a CTA take turns over a sequence's steps, and a cluster of 1 to 8
// CTAs splits a long sequence.  The
// partial softmaxes meet in shared memory, across the cluster through
// distributed shared memory: one launch, no scratch.
#include <cooperative_groups.h>

#include "by_length.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "kv4_mma.cuh"

namespace cg = cooperative_groups;

namespace b2pa {

namespace {

constexpr int kStages = 2;

// Asynchronous copy of N bytes (4, 8 or 16) to shared memory, both addresses
// with a constant offset.
template <int N, int DST, int SRC>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0+%2], [%1+%3], %4;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC), "n"(N)
                 : "memory");
}

template <int D, int W = 8>
struct Tile : KeyWords<D> {
  using KeyWords<D>::NG;
  using KeyWords<D>::SETS;
  using KeyWords<D>::KB;
  using KeyWords<D>::KC;
  static constexpr int VW = D / 64;          // V words per lane and key (keys 4t .. 4t+3)
  static constexpr int VB = VW * 4;          // bytes per V copy
  static constexpr int OFF_V = 2 * KC * KB * 32;
  static constexpr int OFF_KS = OFF_V + 4 * VB * 32;
  static constexpr int OFF_VS = OFF_KS + 16 * NG;
  static constexpr int OFF_MASK = OFF_VS + 128 * SETS;  // after the last tile
  static constexpr int TILE = OFF_MASK;      // bytes of one tile
  static constexpr int TP = D == 256 ? 1 : 2;  // tiles per step: independent work to hide the products' latency
  static constexpr int BYTES = TP * TILE + 16;
  static constexpr int WARPS = W;
};

constexpr int kMaxCluster = 8;

template <int D, int W>
struct Smem {
  float acc[W][D];
  float m[W], l[W];
  // rank 0: every CTA's sums
  float cta_acc[kMaxCluster][D];
  float cta_m[kMaxCluster], cta_l[kMaxCluster];
};

struct DecodeKv4Params {
  const void* q;
  int64_t sq_b, sq_h;
  const uint8_t* k_pool;
  const uint8_t* v_pool;
  int64_t num_blocks;
  const int32_t* page_table;
  int64_t pt_stride;
  int max_pages;
  const int32_t* seq_lens;
  const int32_t* cur_lens;
  void* out;
  int64_t so_b, so_h;
  int H;
  float qscale;  // scale * log2(e)
  int32_t* status;
  int by_length;  // CTAs take the sequences longest first
};

}  // namespace

template <typename T, int D, int BS, int W>
__global__ void __launch_bounds__(W * 32, D == 256 ? 8 / W : 16 / W) kv4_decode_kernel(DecodeKv4Params p) {
  using C = Tile<D, W>;
  using Q = KeyQuery<T, D>;
  // The weights' low halves.  bf16 outputs do without: a weight rounded to 11
  // bits is off by 2^-12 at most, an eighth of the output's own rounding, and
  // the roundings of different keys are independent.  (D = 64 has them in
  // columns 4..7, at no cost.)
  constexpr bool PLO = !std::is_same<T, __nv_bfloat16>::value && D != 64;
  constexpr bool SIGNED = Q::SIGNED;
  constexpr int PAGE = kv4_page_bytes(BS, D), CODES = BS * (D / 2);
  extern __shared__ __align__(16) uint8_t ring_all[];
  __shared__ Smem<D, W> sm;
  const int ns = gridDim.x, rank = blockIdx.x, h = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = ring_all + warp * (kStages * C::BYTES);
  const uint32_t ring_at = smem_u32(ring);

  // The cluster's other CTAs have to be running before their shared memory is
  // written (at the end): arrive here, wait there.
  if (ns > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();
  const int b = p.by_length ? nth_longest(p.seq_lens, gridDim.z, blockIdx.z) : (int)blockIdx.z;
  // Three loads that do not wait for one another: the lengths, q, and the
  // first block ids.  Steps go round the cluster's warps, so a warp's first
  // step does not depend on the length.
  const int64_t len = p.seq_lens[b], cur = p.cur_lens[b], cap = (int64_t)p.max_pages * BS;
  Q query;
  query.load(static_cast<const T*>(p.q) + (int64_t)b * p.sq_b + (int64_t)h * p.sq_h);
  constexpr int KEYS = 16 * C::TP;  // per step
  const int step0 = rank * C::WARPS + warp, turn = ns * C::WARPS;  // this warp's steps: step0 + i * turn
  const int32_t* table = p.page_table + (int64_t)b * p.pt_stride;
  // block ids of this warp's next steps, one per lane: a step has PAGES pages
  constexpr int PAGES = BS >= KEYS ? 1 : KEYS / BS, AHEAD = 32 / PAGES;
  auto load_ids = [&](int i0) -> int {
    const int64_t page = (step0 + (int64_t)turn * (i0 + lane / PAGES)) * KEYS / BS + lane % PAGES;
    return page < p.max_pages ? table[page] : -1;
  };
  int ids = load_ids(0);

  int64_t vis = len - cur + 1;
  vis = vis < len ? vis : len;
  vis = vis < cap ? vis : cap;
  vis = vis > 0 ? vis : 0;
  if (len > cap && rank == 0 && h == 0 && tid == 0) set_status(p.status, B2PA_ERR_BAD_BLOCK_ID);
  const int nvis = (int)vis;
  const int steps = (nvis + KEYS - 1) / KEYS;
  const int mine = steps > step0 ? (steps - step0 + turn - 1) / turn : 0;
  // Where this lane's pieces lie in block 0 (a warp's steps start at the same
  // row of their pages: WARPS is even) and in stage 0; every other address is
  // one multiply-add away.
  const int row0 = BS == 32 && C::TP == 1 ? 16 * (step0 & 1) : 0;
  const int64_t block_bytes = (int64_t)p.H * PAGE;
  const int vrow = BS == 8 ? 4 * (t & 1) : row0 + 4 * t;
  const int kpiece = 4 * lane % (16 * C::NG);  // K scales: 16 rows, linear
  const int krow = kpiece / C::NG;
  const uint8_t* const k_at = p.k_pool + (int64_t)h * PAGE + (row0 + g) * (D / 2) + t * C::KB;
  const uint8_t* const v_at = p.v_pool + (int64_t)h * PAGE + vrow * (D / 2) + g * C::VB;
  const uint8_t* const ks_at =
      p.k_pool + (int64_t)h * PAGE + CODES + (BS == 8 ? krow & 7 : row0 + krow) * C::NG + kpiece % C::NG;
  const uint8_t* const vs_at =
      p.v_pool + (int64_t)h * PAGE + CODES + (C::SETS == 2 ? 2 * g : D == 64 ? (g & 3) : g) * BS + vrow;
  const uint32_t k_to = ring_at + lane * C::KB, v_to = ring_at + C::OFF_V + lane * C::VB,
                 s_to = ring_at + C::OFF_KS + lane * 4;
  // Starts the copies of this warp's i-th step.  A page that is not there is
  // not copied: the mask hides whatever its stage holds.
  auto fetch = [&](int i) {
    if (i < mine) {
      if (i % AHEAD == 0 && i > 0) ids = load_ids(i);
      const uint32_t st = (i % kStages) * C::BYTES;
      const int left = nvis - (step0 + turn * i) * KEYS;
      uint32_t mask = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
#pragma unroll
      for (int x = 0; x < C::TP; ++x) {
        constexpr int ROWS = BS == 32 ? 16 : 0;  // rows from one tile to the next within a page
        // ids past the pool are reported where keys would be seen in them
        int b0 = __shfl_sync(kFullMask, ids, i % AHEAD * PAGES + (BS == 32 ? 0 : x * (16 / BS)));
        int b1 = BS == 8 ? __shfl_sync(kFullMask, ids, i % AHEAD * PAGES + 2 * x + 1) : b0;
        if (left <= 16 * x) b0 = -1;
        if (left <= 16 * x + (BS == 8 ? 8 : 0)) b1 = -1;
        if (b0 >= p.num_blocks || b1 >= p.num_blocks) {
          set_status(p.status, B2PA_ERR_BAD_BLOCK_ID);
          if (b0 >= p.num_blocks) b0 = -1;
          if (b1 >= p.num_blocks) b1 = -1;
        }
        if (b0 < 0) mask &= ~((BS == 8 ? 0xffu : 0xffffu) << (16 * x));
        if (BS == 8 && b1 < 0) mask &= ~(0xff00u << (16 * x));
        const int bv = BS == 8 && t >= 2 ? b1 : b0;
        const int bk = BS == 8 && krow >= 8 ? b1 : b0;  // (D = 256: pieces 32.. are of the second page)
        const uint32_t kd = k_to + st + x * C::TILE, vd = v_to + st + x * C::TILE, sd = s_to + st + x * C::TILE;
        if (b0 >= 0) {
          const uint8_t* k = k_at + b0 * block_bytes + x * ROWS * (D / 2);
          copy_async<C::KB, 0, 0>(kd, k);
          if constexpr (C::KC == 2) copy_async<C::KB, 64 * C::KB, 4 * C::KB>(kd, k);
          if constexpr (BS != 8) {
            copy_async<C::KB, 32 * C::KB, 8 * (D / 2)>(kd, k);
            if constexpr (C::KC == 2) copy_async<C::KB, 96 * C::KB, 8 * (D / 2) + 4 * C::KB>(kd, k);
          }
        }
        if (BS == 8 && b1 >= 0) {
          const uint8_t* k = k_at + b1 * block_bytes;
          copy_async<C::KB, 32 * C::KB, 0>(kd, k);
          if constexpr (C::KC == 2) copy_async<C::KB, 96 * C::KB, 4 * C::KB>(kd, k);
        }
        if (bv >= 0) {
          const uint8_t* v = v_at + bv * block_bytes + x * ROWS * (D / 2);
          copy_async<C::VB, 0, 0>(vd, v);
          copy_async<C::VB, 32 * C::VB, D / 2>(vd, v);
          copy_async<C::VB, 64 * C::VB, 2 * (D / 2)>(vd, v);
          copy_async<C::VB, 96 * C::VB, 3 * (D / 2)>(vd, v);
          const uint8_t* vs = vs_at + bv * block_bytes + x * ROWS;
          copy_async<4, C::OFF_VS - C::OFF_KS, 0>(sd, vs);
          if constexpr (C::SETS == 2) copy_async<4, C::OFF_VS - C::OFF_KS + 128, BS>(sd, vs);
        }
        if constexpr (D == 256) {  // two pieces per lane, 8 rows apart
          if (b0 >= 0) copy_async<4, 0, 0>(sd, ks_at + b0 * block_bytes);
          if (b1 >= 0) copy_async<4, 128, BS == 8 ? 0 : 8 * C::NG>(sd, ks_at + b1 * block_bytes);
        } else if (bk >= 0 && (D == 128 || lane < 16)) {
          copy_async<4, 0, 0>(sd, ks_at + bk * block_bytes + x * ROWS * C::NG);
        }
      }
      if (C::TP == 1) mask &= 0xffffu;
      if (lane == 0) *reinterpret_cast<uint32_t*>(ring + st + C::TP * C::TILE) = mask;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);

  query.prepare(p.qscale);

  float acc[C::VW][4][4];              // [word][nibble][fragment]: channels 8 * word + nibble (+ 4)
  float eights[C::SETS][4];            // 8 * sum of the weight operand, per column
#pragma unroll
  for (int u = 0; u < C::VW; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[u][j][k] = 0.f;
#pragma unroll
  for (int s = 0; s < C::SETS; ++s)
#pragma unroll
    for (int k = 0; k < 4; ++k) eights[s][k] = 0.f;
  float m = -INFINITY, l = 0.f;
  uint32_t top_e = 0;  // largest V scale exponent so far; weights are scaled by 2^(29 - top_e)

  auto rescale = [&](float f) {
#pragma unroll
    for (int u = 0; u < C::VW; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[u][j][k] *= f;
#pragma unroll
    for (int s = 0; s < C::SETS; ++s)
#pragma unroll
      for (int k = 0; k < 4; ++k) eights[s][k] *= f;
  };

  for (int i = 0; i < mine; ++i) {
    fetch(i + kStages - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint8_t* stage = ring + (i % kStages) * C::BYTES;
    const uint32_t mask = *reinterpret_cast<const uint32_t*>(stage + C::TP * C::TILE);
    if (mask == 0) {
      __syncwarp();
      continue;
    }
    float z0[C::TP], z1[C::TP];  // logits of keys g, g + 8 of each tile
    uint32_t vs[C::TP][C::SETS];
#pragma unroll
    for (int y = 0; y < C::TP; ++y) {
      const uint8_t* st = stage + y * C::TILE;
      // ---- logits
      uint32_t ka[C::KW], kb[C::KW];  // rows g and g + 8
#pragma unroll
      for (int c = 0; c < C::KC; ++c) {
        if constexpr (C::KB == 16) {
          *reinterpret_cast<uint4*>(&ka[4 * c]) = *reinterpret_cast<const uint4*>(st + ((2 * c) * 32 + lane) * 16);
          *reinterpret_cast<uint4*>(&kb[4 * c]) = *reinterpret_cast<const uint4*>(st + ((2 * c + 1) * 32 + lane) * 16);
        } else {
          *reinterpret_cast<uint2*>(&ka[0]) = *reinterpret_cast<const uint2*>(st + lane * 8);
          *reinterpret_cast<uint2*>(&kb[0]) = *reinterpret_cast<const uint2*>(st + (32 + lane) * 8);
        }
      }
      uint32_t w0[C::SETS], w1[C::SETS];
#pragma unroll
      for (int x = 0; x < C::SETS; ++x) {
        w0[x] = *reinterpret_cast<const uint16_t*>(st + C::OFF_KS + g * C::NG + Q::scale_at(x));
        w1[x] = *reinterpret_cast<const uint16_t*>(st + C::OFF_KS + (g + 8) * C::NG + Q::scale_at(x));
        vs[y][x] = *reinterpret_cast<const uint32_t*>(st + C::OFF_VS + (x * 32 + lane) * 4);
      }
      query.logits(ka, kb, w0, w1, z0[y], z1[y]);
    }
#pragma unroll
    for (int y = 0; y < C::TP; ++y) {
      z0[y] = query.finish(z0[y]);
      z1[y] = query.finish(z1[y]);
    }
    if (mask != (C::TP == 1 ? 0xffffu : 0xffffffffu)) {
#pragma unroll
      for (int y = 0; y < C::TP; ++y) {
        const uint32_t mk = mask >> (16 * y);
        if (!(mk >> g & 1u)) z0[y] = -INFINITY;
        if (!(mk >> (g + 8) & 1u)) z1[y] = -INFINITY;
        // an unseen key's scale may be anything, NaN included: zero
        const uint32_t four = mk >> (4 * t) & 15u;
        const uint32_t keep = (four & 1u) * 0xffu | (four >> 1 & 1u) * 0xff00u | (four >> 2 & 1u) * 0xff0000u |
                              (four >> 3 & 1u) * 0xff000000u;
#pragma unroll
        for (int x = 0; x < C::SETS; ++x) vs[y][x] &= keep;
      }
    }
    // ---- running maximum, weights
    float top = fmaxf(z0[0], z1[0]);
    if constexpr (C::TP == 2) top = fmaxf(top, fmaxf(z0[1], z1[1]));
    top = warp_redux_max(top);
    if (top > m) {
      const float f = fast_exp2(m - top);  // 0 for the first step
      m = top;
      l *= f;
      rescale(f);
    }
    const float ref = m == -INFINITY ? 0.f : m;
    // ---- a V scale above the largest exponent so far?
    uint32_t big = 0;  // larger of two bytes, in halves
#pragma unroll
    for (int y = 0; y < C::TP; ++y)
#pragma unroll
      for (int x = 0; x < C::SETS; ++x)
        big = __vmaxu2(big, __vmaxu2(vs[y][x] & 0x00ff00ffu, vs[y][x] >> 8 & 0x00ff00ffu));
    // a byte of at least 8 (top_e + 1) carries into bit 8
    if (__any_sync(kFullMask, (big + (0x100u - 8u * (top_e + 1u)) * 0x10001u) & 0x01000100u)) {
      uint32_t most = 0;
#pragma unroll
      for (int y = 0; y < C::TP; ++y)
#pragma unroll
        for (int x = 0; x < C::SETS; ++x)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t c = vs[y][x] >> (8 * k) & 255u;
            // not a NaN group's: its column is lost, the others keep their range
            most = c <= kKv4MaxScale && c > most ? c : most;
          }
      most = __reduce_max_sync(kFullMask, most) >> 3;
      if (most > top_e) {
        rescale(__uint_as_float((127u - (most - top_e)) << 23));
        top_e = most;
      }
    }
    const float up = __uint_as_float((127u + 29u - top_e) << 23);
#pragma unroll
    for (int y = 0; y < C::TP; ++y) {
      const uint8_t* st = stage + y * C::TILE;
      const float p0 = fast_exp2(z0[y] - ref), p1 = fast_exp2(z1[y] - ref);
      l += p0 + p1;
      // ---- weights of keys 4t .. 4t+3 (lane 4 * (key & 7) holds key and key + 8)
      const float both = (t < 2 ? p0 : p1) * up;
      float pk[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) pk[k] = __shfl_sync(kFullMask, both, 4 * ((4 * t + k) & 7) + (t < 2 ? 0 : 2));
      uint32_t bh[C::SETS][2], bl[C::SETS][2];
#pragma unroll
      for (int x = 0; x < C::SETS; ++x) {
        const uint32_t h01 = __byte_perm(vs[y][x], 0, 0x4140) << 7, h23 = __byte_perm(vs[y][x], 0, 0x4342) << 7;
        const float2 s01 = __half22float2(*reinterpret_cast<const __half2*>(&h01));
        const float2 s23 = __half22float2(*reinterpret_cast<const __half2*>(&h23));
        split2(pk[0] * s01.x, pk[1] * s01.y, bh[x][0], bl[x][0]);
        split2(pk[2] * s23.x, pk[3] * s23.y, bh[x][1], bl[x][1]);
        if (D == 64 && g >= 4) {  // columns 4..7: the low halves of groups 0..3
          bh[x][0] = bl[x][0];
          bh[x][1] = bl[x][1];
        }
        constexpr uint32_t EIGHT = 0x00080008u;
        if constexpr (!SIGNED) mma_f16(eights[x], EIGHT, EIGHT, EIGHT, EIGHT, bh[x][0], bh[x][1]);
        if constexpr (!SIGNED && PLO) mma_f16(eights[x], EIGHT, EIGHT, EIGHT, EIGHT, bl[x][0], bl[x][1]);
      }
      // ---- out += V^T . weights
      uint32_t v[4][C::VW];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint8_t* at = st + C::OFF_V + (k * 32 + lane) * C::VB;
        if constexpr (C::VW == 1) v[k][0] = *reinterpret_cast<const uint32_t*>(at);
        if constexpr (C::VW == 2) *reinterpret_cast<uint2*>(&v[k][0]) = *reinterpret_cast<const uint2*>(at);
        if constexpr (C::VW == 4) *reinterpret_cast<uint4*>(&v[k][0]) = *reinterpret_cast<const uint4*>(at);
      }
#pragma unroll
      for (int u = 0; u < C::VW; ++u) {
        const int x = C::SETS == 2 ? u >> 1 : 0;
        uint32_t c01 = __byte_perm(v[0][u], v[1][u], 0x5410), d01 = __byte_perm(v[0][u], v[1][u], 0x7632);
        uint32_t c23 = __byte_perm(v[2][u], v[3][u], 0x5410), d23 = __byte_perm(v[2][u], v[3][u], 0x7632);
        auto add = [&](auto j_) {
          constexpr int j = decltype(j_)::value;
          const uint32_t a0 = code_pair<SIGNED, j>(c01), a1 = code_pair<SIGNED, j>(d01),
                         a2 = code_pair<SIGNED, j>(c23), a3 = code_pair<SIGNED, j>(d23);
          mma_f16(acc[u][j], a0, a1, a2, a3, bh[x][0], bh[x][1]);
          if constexpr (PLO) mma_f16(acc[u][j], a0, a1, a2, a3, bl[x][0], bl[x][1]);
        };
        add(std::integral_constant<int, 0>{});
        add(std::integral_constant<int, 1>{});
        c01 >>= 8, d01 >>= 8, c23 >>= 8, d23 >>= 8;
        add(std::integral_constant<int, 2>{});
        add(std::integral_constant<int, 3>{});
      }
    }
    __syncwarp();  // every lane is done with the stage before it is refilled
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- this warp's sums: channel c sits in the column of its group
  l += __shfl_xor_sync(kFullMask, l, 4);
  l += __shfl_xor_sync(kFullMask, l, 8);
  l += __shfl_xor_sync(kFullMask, l, 16);
  if (lane == 0) {
    sm.m[warp] = m;
    sm.l[warp] = l;
  }
  {
    const float down = __uint_as_float((127u + top_e - 29u + (SIGNED ? 0u : 24u)) << 23);
    const int col = D == 64 ? g >> 1 : g;  // this lane's rows' group, as a column
#pragma unroll
    for (int u = 0; u < C::VW; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = C::SETS == 2 ? u >> 1 : 0;
        float lo = (col & 1) ? acc[u][j][1] : acc[u][j][0], hi = (col & 1) ? acc[u][j][3] : acc[u][j][2];
        const float e = (col & 1) ? eights[x][1] : eights[x][0];
        if (j & 1) lo *= 0.0625f, hi *= 0.0625f;
        lo = (lo - e) * down;
        hi = (hi - e) * down;
        if (D == 64) {  // the low halves' columns are two lanes further
          lo += __shfl_xor_sync(kFullMask, lo, 2);
          hi += __shfl_xor_sync(kFullMask, hi, 2);
        }
        if (t == (col >> 1)) {
          const int ch = g * (D / 8) + 8 * u + j;
          sm.acc[warp][ch] = lo;
          sm.acc[warp][ch + 4] = hi;
        }
      }
  }
  __syncthreads();
  // ---- the CTA's, then the cluster's
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < C::WARPS; ++w) M = fmaxf(M, sm.m[w]);
  float ref = M == -INFINITY ? 0.f : M;
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < C::WARPS; ++w) total += sm.l[w] * fast_exp2(sm.m[w] - ref);
  constexpr int PER = (D + C::WARPS * 32 - 1) / (C::WARPS * 32);
  float o[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = tid + i * C::WARPS * 32;
    o[i] = 0.f;
    if (d < D) {
#pragma unroll
      for (int w = 0; w < C::WARPS; ++w)
        if (sm.m[w] != -INFINITY || sm.l[w] != 0.f) o[i] += sm.acc[w][d] * fast_exp2(sm.m[w] - ref);
    }
  }
  if (ns > 1) {
    // every CTA writes its sums into rank 0's shared memory and leaves
    cg::cluster_group cluster = cg::this_cluster();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    Smem<D, W>* dst = cluster.map_shared_rank(&sm, 0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int d = tid + i * C::WARPS * 32;
      if (d < D) dst->cta_acc[rank][d] = o[i];
    }
    if (tid == 0) {
      dst->cta_m[rank] = M;
      dst->cta_l[rank] = total;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    M = -INFINITY;
    for (int r = 0; r < ns; ++r) M = fmaxf(M, sm.cta_m[r]);
    ref = M == -INFINITY ? 0.f : M;
    total = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = 0.f;
    for (int r = 0; r < ns; ++r) {
      const float f = fast_exp2(sm.cta_m[r] - ref);
      total += sm.cta_l[r] * f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int d = tid + i * C::WARPS * 32;
        if (d < D) o[i] += sm.cta_acc[r][d] * f;
      }
    }
  }
  T* out = static_cast<T*>(p.out) + (int64_t)b * p.so_b + (int64_t)h * p.so_h;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = tid + i * C::WARPS * 32;
    if (d < D) out[d] = from_f32<T>(total != 0.f ? o[i] / total : 0.f);
  }
}

template <typename T, int D, int BS, int W>
static int decode_launch(const AttnArgs& a, int ns, cudaStream_t s) {
  using C = Tile<D, W>;
  DecodeKv4Params p;
  p.q = a.q;
  p.sq_b = a.sq[0];
  p.sq_h = a.sq[1];
  p.k_pool = static_cast<const uint8_t*>(a.k_pool);
  p.v_pool = static_cast<const uint8_t*>(a.v_pool);
  p.num_blocks = a.num_blocks;
  p.page_table = a.page_table;
  p.pt_stride = a.pt_stride;
  p.max_pages = a.max_pages;
  p.seq_lens = a.seq_lens;
  p.cur_lens = a.cur_lens;
  p.out = a.out;
  p.so_b = a.so[0];
  p.so_h = a.so[1];
  p.H = a.H;
  p.qscale = a.scale * kLog2e;
  p.status = a.status;
  p.by_length = orders_by_length(a.B, (int64_t)ns * a.H * a.B, 2, (int64_t)a.max_pages * BS / ns, 512,
                                 D == 64 ? 900 : D == 128 ? 650 : 350);
  constexpr int smem = C::WARPS * kStages * C::BYTES;
  auto kern = kv4_decode_kernel<T, D, BS, W>;
  const int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(kern), smem);
  if (rc != B2PA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ns, (unsigned)a.H, (unsigned)a.B);
  cfg.blockDim = dim3(C::WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ns;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "paged_decode_kv4 launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

template <typename T, int D>
static int decode_blocks(const AttnArgs& a, cudaStream_t s) {
  // CTAs per sequence and head: one wave of the two CTAs an SM holds, while
  // every warp keeps a step of the longest sequence that the table has room for
  // (the host does not know the lengths).  A CTA costs about 4 us
  // beside its keys (loads that depend on one another, the merge), so more
  // waves of smaller shares are slower: 64 sequences of 128-1,024 tokens and 8
  // heads of 64 (fp32) take 16.8 us with 1 CTA each, 24.8 with 2; 64 of
  // 1,024-8,192 and 32 heads of 128 (bf16) 273 and 312; one sequence of 8,001
  // tokens and 32 heads of 128 46.0 us with 1, 25.9 with 2, 18.7 with 4, 14.3
  // with 8.  head_dim 256 takes half as many warps a CTA (registers).
  constexpr int W = D == 256 ? 4 : 8;
  const int64_t pairs = (int64_t)a.B * a.H;
  const int64_t steps = ((int64_t)a.max_pages * a.block_size + 31) / 32;
  int ns = 1;
  while (ns < kMaxCluster && pairs * ns < 2 * device_sm_count() && steps > W * ns) ns *= 2;
  switch (a.block_size) {
    case 8: return decode_launch<T, D, 8, W>(a, ns, s);
    case 16: return decode_launch<T, D, 16, W>(a, ns, s);
    default: return decode_launch<T, D, 32, W>(a, ns, s);
  }
}

template <typename T>
static int decode_as(const AttnArgs& a, cudaStream_t s) {
  switch (a.D) {
    case 64: return decode_blocks<T, 64>(a, s);
    case 128: return decode_blocks<T, 128>(a, s);
    default: return decode_blocks<T, 256>(a, s);
  }
}

int launch_kv4_decode(const AttnArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return decode_as<float>(a, s);
    case B2PA_DTYPE_BF16: return decode_as<__nv_bfloat16>(a, s);
    default: return decode_as<__half>(a, s);
  }
}

}  // namespace b2pa
