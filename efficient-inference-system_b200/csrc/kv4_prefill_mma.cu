// kv4_prefill_mma.cu -- chunked prefill straight from 4-bit pages, for shapes
// that have no tcgen05 kernel to run on unpacked pages (head_dim 256) and for
// inputs that it does not take: see kv4_prefill.cu for which call takes which.
//
// One CTA takes 64 queries of a (head, sequence); each of its 4 warps 16 of
// them with all channels.  Tiles of keys are unpacked to fp16 (exact) into
// shared memory once per CTA, in the order in which the products' operands are
// read: a lane's registers of one key row, or of a pair of keys and a channel,
// lie together, so both sides move 16 bytes a lane without bank conflicts.
// One pass with the running maximum and sum of the softmax in fp32; q enters
// as one fp16 half, or two (fp32), rows scaled by powers of two; the weights
// as one half (a rounding of 2^-12, below that of 16-bit outputs) or two.
// A cluster of up to 8 CTAs shares the keys of few queries and joins the
// partial results through distributed shared memory.
// A NaN group of V at a key that only some of the tile's queries see must not
// meet the others' zero weights: it is put in shared memory as zeros, and the
// queries that see the first of a group's get their NaN at the end.
// What bounds it: mma.sync, about 520 TFLOP/s on this device, and the shared
// memory reads that feed it (half a 16-byte read per product).
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "kv4_mma.cuh"

namespace cg = cooperative_groups;

namespace b2pa {

namespace {

constexpr int kRows = 64, kThreads = 128;

template <typename T, int D>
struct Pf {
  static constexpr bool F32 = std::is_same<T, float>::value;
  static constexpr int PARTS = F32 ? 2 : 1;
  static constexpr int KT = F32 && D == 256 ? 32 : 64;  // keys per tile: two CTAs per SM
  static constexpr int NB = D / 32;                      // 32-channel blocks
  static constexpr int PITCH = D * 2 + 64;               // bytes per query row
  static constexpr int Q_BYTES = PARTS * kRows * PITCH;
  static constexpr int T_BYTES = KT * D * 2;             // unpacked K, or V
  static constexpr int O_BYTES = kRows * D * 4;          // the cluster's exchange, over all of it
  static constexpr int SMEM = Q_BYTES + 2 * T_BYTES > O_BYTES ? Q_BYTES + 2 * T_BYTES : O_BYTES;
  static constexpr int VW = D / 64;                      // V words per lane and key
  static constexpr int VL = KT == 64 ? VW : VW / 2;      // ... per unpacking item (4 items, one per warp)
};

// The words of V of one key for lane group g, `VL` of them.
template <int VL>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[VL]) {
  if constexpr (VL == 4)
    *reinterpret_cast<uint4*>(w) = __ldg(reinterpret_cast<const uint4*>(p));
  else if constexpr (VL == 2)
    *reinterpret_cast<uint2*>(w) = __ldg(reinterpret_cast<const uint2*>(p));
  else
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
}

// What the weights of a row are taken relative to: 15 below its maximum, so that
// they go up to 2^15 (the division by their sum takes that out again) and one of
// 2^-29 of the largest is still a normal fp16 number.  A far maximum, whose own
// rounding would carry the largest past fp16's range, is taken as it is.
__device__ __forceinline__ float reference(float m) { return fabsf(m) < 0x1p20f ? m - 15.f : m; }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    kv4_prefill_kernel(AttnArgs a, float qscale, const uint32_t* flag, uint32_t epoch) {
  using P = Pf<T, D>;
  constexpr int KT = P::KT, NK = KT / 8, NC = D / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float unit[kRows];
  __shared__ uint8_t key_ok[KT];
  __shared__ float2 row_ml[kRows];
  __shared__ int any_nan;
  __shared__ int nan_at[D / 16];  // first key, of those that not every query of the tile sees, with a NaN group
  uint8_t* const qs = smem;
  uint4* const kf = reinterpret_cast<uint4*>(smem + P::Q_BYTES);               // [key / 8][block][lane]
  uint4* const vf = reinterpret_cast<uint4*>(smem + P::Q_BYTES + P::T_BYTES);  // [key / 16][channel pair][lane]
  pdl_wait();
  pdl_launch_dependents();
  if (flag != nullptr && *reinterpret_cast<const volatile uint32_t*>(flag) != epoch) return;  // nothing to redo
  cg::cluster_group cluster = cg::this_cluster();
  const int ns = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int i0 = blockIdx.x / ns * kRows;
  const int bs = a.block_size, sh = __ffs(bs) - 1, page_bytes = kv4_page_bytes(bs, D);
  const int64_t len = a.seq_lens[b], cap = (int64_t)a.max_pages * bs, past = len - a.cur_lens[b];
  const int64_t L = len < cap ? len : cap;
  if (len > cap && blockIdx.x == 0 && h == 0 && tid == 0) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  const uint32_t blocks = a.num_blocks < INT32_MAX ? (uint32_t)a.num_blocks : (uint32_t)INT32_MAX;
  const int32_t* table = a.page_table + (int64_t)b * a.pt_stride;

  const int last = i0 + kRows < a.T ? i0 + kRows : a.T;
  int64_t kend = past + last;  // keys that the last query sees
  kend = kend < L ? kend : L;
  if (blocks == 0) kend = 0;
  convert_queries<T, true, D, kRows, P::PITCH, P::PARTS, kThreads>(
      static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1] + (int64_t)i0 * a.sq[2], a.sq[2], a.T - i0,
      qs, unit);

  if (tid < D / 16) nan_at[tid] = INT32_MAX;
  if (tid == 0) any_nan = 0;
  float o[NC][4];  // rows g, g + 8; channels 2t * NC + n and (2t + 1) * NC + n
#pragma unroll
  for (int n = 0; n < NC; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, scale[2];
  const int64_t first_seen = past + i0 + 1;  // keys below it are seen by every query of the tile

  // Page of key j of this head (block 0's for one that is not there).
  auto page_of = [&](int64_t j, bool& ok) {
    const uint32_t blk = j < kend ? (uint32_t)__ldg(table + (j >> sh)) : 0xffffffffu;
    ok = blk < blocks;
    if ((int)blk >= (int)blocks) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    return ((ok ? blk : 0u) * (uint64_t)a.H + h) * (uint32_t)page_bytes;
  };

  for (int64_t j0 = (int64_t)rank * KT; j0 < kend; j0 += (int64_t)ns * KT) {
    __syncthreads();  // the tile before is used up (and, at first, q is in place)
    // ---- K: 8 keys a turn; lane (g, t) takes its words of key g
#pragma unroll
    for (int n = warp; n < NK; n += 4) {
      const int64_t j = j0 + n * 8 + g;
      bool ok;
      const uint8_t* page = static_cast<const uint8_t*>(a.k_pool) + page_of(j, ok);
      uint4 f[P::NB];
      unpack_key_row<D>(page, (int)(j & (bs - 1)), bs, f);
#pragma unroll
      for (int w = 0; w < P::NB; ++w) kf[(n * P::NB + w) * 32 + lane] = ok ? f[w] : make_uint4(0, 0, 0, 0);
      if (t == 0) key_ok[n * 8 + g] = ok ? 1 : 0;
    }
    // ---- V: 16 keys a turn; lane (g, t) takes channels g D/8 .. of keys
    // 2t, 2t+1, 8+2t, 9+2t and pairs the keys
    {
      constexpr int HALVES = P::VW / P::VL;
      const int ks = warp / HALVES, u0 = warp % HALVES * P::VL;
      uint32_t v[4][P::VL];
      uint32_t sc[4][2];  // scale codes of this lane's one or two groups
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t j = j0 + ks * 16 + (k & 1) + 2 * t + (k >> 1) * 8;
        bool ok;
        const uint8_t* page = static_cast<const uint8_t*>(a.v_pool) + page_of(j, ok);
        const int row = (int)(j & (bs - 1));
        load_words<P::VL>(page + row * (D / 2) + g * (D / 16) + 4 * u0, v[k]);
        const uint8_t* codes = page + bs * (D / 2) + row;
        if constexpr (D == 256) {
          sc[k][0] = __ldg(codes + (2 * g + (u0 >> 1)) * bs);
          sc[k][1] = P::VL == 4 ? __ldg(codes + (2 * g + 1) * bs) : sc[k][0];
        } else {
          sc[k][0] = sc[k][1] = __ldg(codes + (D == 64 ? g >> 1 : g) * bs);
        }
        if (!ok) {
          sc[k][0] = sc[k][1] = 0;
#pragma unroll
          for (int u = 0; u < P::VL; ++u) v[k][u] = 0x88888888u;
        }
      }
      if (j0 + KT > first_seen) {  // (all loads are under way by now)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int64_t j = j0 + ks * 16 + (k & 1) + 2 * t + (k >> 1) * 8;
            if (sc[k][x] == kKv4NanScale && j >= first_seen) {
              const int group = D == 256 ? 2 * g + (P::VL == 4 ? x : u0 >> 1) : D == 64 ? g >> 1 : g;
              atomicMin(&nan_at[group], (int)j);
              any_nan = 1;
              sc[k][x] = 0;
            }
          }
      }
      const __half2 k1032 = __half2half2(__ushort_as_half(0x6408)), k72 = __half2half2(__ushort_as_half(0xd480)),
                    k16th = __half2half2(__ushort_as_half(0x2c00));
#pragma unroll
      for (int u = 0; u < P::VL; ++u) {
        const int x = D == 256 && P::VL == 4 ? u >> 1 : 0;
        const __half2 s01 = scale_pair(sc[0][x] | sc[1][x] << 8, 0x4140), s23 = scale_pair(sc[2][x] | sc[3][x] << 8, 0x4140);
        // [low or high half of the word][keys 0, 1 or 2, 3]
        uint32_t c[2][2] = {{__byte_perm(v[0][u], v[1][u], 0x5410), __byte_perm(v[2][u], v[3][u], 0x5410)},
                            {__byte_perm(v[0][u], v[1][u], 0x7632), __byte_perm(v[2][u], v[3][u], 0x7632)}};
        uint4* dst = vf + (ks * (NC / 2) + (u0 + u) * 4) * 32 + lane;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int j = 0; j < 2; ++j) {  // channels 2j, 2j + 1 of the half word
            uint32_t r[4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t y = c[half][k] >> (8 * j);
              const uint32_t lo = (y & 0x000f000fu) | 0x64006400u, hi = (y & 0x00f000f0u) | 0x64006400u;
              const __half2 s = k ? s23 : s01;
              r[k] = half2_bits(__hmul2(__hsub2(*reinterpret_cast<const __half2*>(&lo), k1032), s));
              r[2 + k] = half2_bits(__hmul2(__hfma2(*reinterpret_cast<const __half2*>(&hi), k16th, k72), s));
            }
            dst[(half * 2 + j) * 32] = make_uint4(r[0], r[1], r[2], r[3]);
          }
      }
    }
    __syncthreads();
    scale[0] = qscale * unit[warp * 16 + g];
    scale[1] = qscale * unit[warp * 16 + g + 8];
    // ---- S = Q . K^T
    float s[NK][4];
#pragma unroll
    for (int n = 0; n < NK; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    const uint8_t* qa = qs + (warp * 16 + g) * P::PITCH + 16 * t;
#pragma unroll
    for (int w = 0; w < P::NB; ++w) {
      const uint4 u = *reinterpret_cast<const uint4*>(qa + 64 * w), v = *reinterpret_cast<const uint4*>(qa + 8 * P::PITCH + 64 * w);
      uint4 ul, vl;
      if constexpr (P::F32) {
        ul = *reinterpret_cast<const uint4*>(qa + kRows * P::PITCH + 64 * w);
        vl = *reinterpret_cast<const uint4*>(qa + (kRows + 8) * P::PITCH + 64 * w);
      }
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const uint4 y = kf[(n * P::NB + w) * 32 + lane];
        if constexpr (P::F32) {
          mma_f16(s[n], ul.x, vl.x, ul.y, vl.y, y.x, y.y);
          mma_f16(s[n], ul.z, vl.z, ul.w, vl.w, y.z, y.w);
        }
        mma_f16(s[n], u.x, v.x, u.y, v.y, y.x, y.y);
        mma_f16(s[n], u.z, v.z, u.w, v.w, y.z, y.w);
      }
    }
    // ---- logits, masks, running maximum
    bool plain = j0 + KT <= first_seen && j0 + KT <= kend;
#pragma unroll
    for (int i = 0; i < KT; i += 32) plain = plain && key_ok[i + lane];
    plain = __all_sync(kFullMask, plain);
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = k >> 1, col = n * 8 + 2 * t + (k & 1);
        s[n][k] *= scale[r];
        if (!plain && !(key_ok[col] && j0 + col < first_seen + warp * 16 + g + 8 * r && j0 + col < kend))
          s[n][k] = -INFINITY;
        top[r] = fmaxf(top[r], s[n][k]);
      }
    float f[2];
    bool move = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(kFullMask, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(kFullMask, top[r], 2));
      const float up = fmaxf(m[r], top[r]);
      f[r] = m[r] == up ? 1.f : fast_exp2(reference(m[r]) - reference(up));
      move = move || m[r] != up;
      m[r] = up;
      l[r] *= f[r];
    }
    if (__any_sync(kFullMask, move)) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        o[n][0] *= f[0];
        o[n][1] *= f[0];
        o[n][2] *= f[1];
        o[n][3] *= f[1];
      }
    }
    const float ref[2] = {m[0] == -INFINITY ? 0.f : reference(m[0]), m[1] == -INFINITY ? 0.f : reference(m[1])};
    // ---- O += P . V, 16 keys at a time
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks) {
      uint32_t ph[4], plo[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // rows g, g + 8 of keys 2t, 2t+1; then of keys 8+2t, 9+2t
        const int r = k & 1, n = 2 * ks + (k >> 1);
        const float x = fast_exp2(s[n][2 * r] - ref[r]), y = fast_exp2(s[n][2 * r + 1] - ref[r]);
        l[r] += x + y;
        split2(x, y, ph[k], plo[k]);
      }
#pragma unroll
      for (int c = 0; c < NC / 2; ++c) {
        const uint4 y = vf[(ks * (NC / 2) + c) * 32 + lane];
        if constexpr (P::F32) {
          mma_f16(o[2 * c], plo[0], plo[1], plo[2], plo[3], y.x, y.y);
          mma_f16(o[2 * c + 1], plo[0], plo[1], plo[2], plo[3], y.z, y.w);
        }
        mma_f16(o[2 * c], ph[0], ph[1], ph[2], ph[3], y.x, y.y);
        mma_f16(o[2 * c + 1], ph[0], ph[1], ph[2], ph[3], y.z, y.w);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(kFullMask, l[r], 1);
    l[r] += __shfl_xor_sync(kFullMask, l[r], 2);
  }
  __syncthreads();
  if (any_nan) {
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (nan_at[((2 * t + (k & 1)) * NC + n) / 16] < first_seen + warp * 16 + g + 8 * (k >> 1))
          o[n][k] = __uint_as_float(0x7fffffffu);
  }
  T* const out = static_cast<T*>(a.out) + (int64_t)b * a.so[0] + (int64_t)h * a.so[1] + (int64_t)i0 * a.so[2];
  constexpr int V = 16 / (int)sizeof(T);
  if (ns == 1) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = warp * 16 + g + 8 * r;
      const float inv = l[r] != 0.f ? 1.f / l[r] : 0.f;
      if (i0 + row < a.T) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int n = 0; n < NC; n += V) {
            float x[V];
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = o[n + k][2 * r + e] * inv;
            Vec<T, V> y;
            y.from_float(x);
            *reinterpret_cast<uint4*>(out + row * a.so[2] + (2 * t + e) * NC + n) = y.w;
          }
      }
    }
    return;
  }
  // ---- the cluster's: every CTA lays its sums down, each joins some rows
  __syncthreads();
  float* const mine = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = warp * 16 + g + 8 * r;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int n = 0; n < NC; n += 4)
        *reinterpret_cast<float4*>(mine + row * D + (2 * t + e) * NC + n) =
            make_float4(o[n][2 * r + e], o[n + 1][2 * r + e], o[n + 2][2 * r + e], o[n + 3][2 * r + e]);
    if (t == 0) row_ml[row] = make_float2(reference(m[r]), l[r]);
  }
  cluster.sync();
  const int share = kRows / ns;
  for (int i = tid; i < share * (D / 4); i += kThreads) {
    const int row = rank * share + i / (D / 4), d = i % (D / 4) * 4;
    if (i0 + row >= a.T) continue;
    float M = -INFINITY, sum = 0.f;
    for (int k = 0; k < ns; ++k) M = fmaxf(M, cluster.map_shared_rank(&row_ml[0], k)[row].x);
    const float zero = M == -INFINITY ? 0.f : M;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < ns; ++k) {
      const float2 ml = cluster.map_shared_rank(&row_ml[0], k)[row];
      const float w = fast_exp2(ml.x - zero);
      const float4 y = *reinterpret_cast<const float4*>(cluster.map_shared_rank(mine, k) + row * D + d);
      sum += ml.y * w;
      x.x += y.x * w;
      x.y += y.y * w;
      x.z += y.z * w;
      x.w += y.w * w;
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    const float z[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
    Vec<T, 4> y;
    y.from_float(z);
    *reinterpret_cast<decltype(y.w)*>(out + row * a.so[2] + d) = y.w;
  }
  cluster.sync();  // no CTA leaves while its sums are being read
}

template <typename T, int D>
int prefill_as(const AttnArgs& a, const uint32_t* flag, uint32_t epoch, cudaStream_t s) {
  using P = Pf<T, D>;
  const int64_t tiles = (int64_t)a.B * a.H * ((a.T + kRows - 1) / kRows);
  const int64_t keys = (int64_t)a.max_pages * a.block_size;
  int ns = 1;
  while (ns < 8 && tiles * ns < 2 * device_sm_count() && keys >= (int64_t)2 * P::KT * ns) ns *= 2;
  auto kern = kv4_prefill_kernel<T, D>;
  const int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(kern), P::SMEM);
  if (rc != B2PA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.T + kRows - 1) / kRows * ns), (unsigned)a.H, (unsigned)a.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = P::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ns;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, a.scale * kLog2e, flag, epoch);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "paged_prefill_kv4 launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

template <typename T>
int prefill_dims(const AttnArgs& a, const uint32_t* flag, uint32_t epoch, cudaStream_t s) {
  switch (a.D) {
    case 64: return prefill_as<T, 64>(a, flag, epoch, s);
    case 128: return prefill_as<T, 128>(a, flag, epoch, s);
    default: return prefill_as<T, 256>(a, flag, epoch, s);
  }
}

}  // namespace

int launch_kv4_prefill_mma(const AttnArgs& a, const uint32_t* flag, uint32_t epoch, cudaStream_t s) {
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return prefill_dims<float>(a, flag, epoch, s);
    case B2PA_DTYPE_BF16: return prefill_dims<__nv_bfloat16>(a, flag, epoch, s);
    default: return prefill_dims<__half>(a, flag, epoch, s);
  }
}

}  // namespace b2pa
