// evict.cu -- eviction from a paged cache by accumulated attention weight.
//
// Of a sequence of n tokens, every head keeps k = min(keep, n): its last
// min(recent, k), and of the others those with the largest weight (ties: the
// lower position; a NaN weight counts as the largest).  Heads choose for
// themselves -- a page holds one row per head and slot, and all heads keep
// equally many, so one block table still serves them.  The kept rows of K, V
// and the weights move, in order, to positions 0 .. k-1: in the same pages, or
// in the pages of a second table.
//
//   evict_both_kernel    the two below in one CTA per (head, sequence), for
//       short sequences;
//   evict_select_kernel  one CTA per (head, sequence): radix selection of the
//       smallest kept weight (digits of 11, 11 and 10 bits of order-preserving
//       keys, which shared memory holds when they fit; it ends early once a
//       digit's count is exactly what is still wanted), then the kept
//       positions in ascending order, each warp counting and then writing a
//       range of its own;
//   evict_move_kernel    one CTA per (row slice, head, sequence), bound by the
//       bytes of the kept rows, read and written once.  In place, row r moves
//       to r' <= r and the rows of one slice move in ascending order: a chunk
//       is read whole into registers before any of it is written, and a later
//       chunk's sources lie behind everything that an earlier one writes.
//       Four CTAs per SM, 8 words in flight per thread, keep enough reads
//       under way while some of them store.
//       Slices of a row (K, V, their scales, the weights; K and V in parts of
//       64 bytes or more when there are few sequences) do not meet and run in
//       parallel.
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace b2pa {

namespace {

constexpr int kMoveThreads = 256;
constexpr int kMoveWords = 8;  // words in flight per thread and chunk

// Larger weight, larger key; any NaN is largest; both zeros alike.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

struct Kept {
  int n, k;
};
__device__ __forceinline__ Kept kept_of(const EvictArgs& a, int b) {
  int64_t n = a.seq_lens[b];
  const int64_t cap = (int64_t)a.max_pages * a.block_size;
  n = n < cap ? n : cap;
  n = n > 0 ? n : 0;
  return {(int)n, (int)(n < a.keep ? n : a.keep)};
}

constexpr int kBins = 2048;

// The kept positions of head h of sequence b, by the whole CTA.
template <int THREADS>
__device__ __forceinline__ void select_kept(const EvictArgs& a, int cached, uint32_t* keys, int h, int b, const Kept& s) {
  constexpr int WARPS = THREADS / 32;
  __shared__ uint32_t hist[2][kBins];
  __shared__ uint32_t found[3];
  __shared__ uint32_t totals[8];
  __shared__ int2 warp_count[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (h == 0 && tid == 0 && a.seq_lens[b] > s.n) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  int32_t* out = a.kept + ((int64_t)b * a.H + h) * a.keep;
  for (int i = s.k + tid; i < a.keep; i += THREADS) out[i] = -1;
  if (s.n == s.k) {
    for (int i = tid; i < s.k; i += THREADS) out[i] = i;
    return;
  }
  const int sure = a.recent < s.k ? a.recent : s.k;
  const int cand = s.n - sure, need = s.k - sure;
  for (int i = tid; i < sure; i += THREADS) out[need + i] = cand + i;
  if (need == 0) return;

  const int32_t* row = a.page_table + (int64_t)b * a.pt_stride;
  auto key_of = [&](int j) -> uint32_t {
    const int32_t blk = __ldg(row + (j >> a.bs_log2));
    if (blk < 0 || blk >= a.num_blocks) return 0;  // reported by the move
    return weight_key(a.weights[((int64_t)blk * a.H + h) * a.block_size + (j & (a.block_size - 1))]);
  };
  for (int i = tid; i < 2 * kBins; i += THREADS) (&hist[0][0])[i] = 0;
  if (cached) {  // four keys at a time: they share a page
#pragma unroll 2
    for (int j = 4 * tid; j < cand; j += 4 * THREADS) {
      const int32_t blk = __ldg(row + (j >> a.bs_log2));
      uint4 k = make_uint4(0, 0, 0, 0);
      if (blk >= 0 && blk < a.num_blocks) {
        const float4 w = *reinterpret_cast<const float4*>(
            a.weights + ((int64_t)blk * a.H + h) * a.block_size + (j & (a.block_size - 1)));
        k = make_uint4(weight_key(w.x), weight_key(w.y), weight_key(w.z), weight_key(w.w));
      }
      *reinterpret_cast<uint4*>(keys + j) = k;
    }
  }
  __syncthreads();
  uint32_t prefix = 0, mask = 0, left = (uint32_t)need;
  bool all = false;  // every key that matches the prefix is taken
  for (int pass = 0; pass < 3 && !all; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 1023u : 2047u;
    uint32_t* hs = hist[pass & 1];
    auto count = [&](uint32_t key) {
      if ((key & mask) == prefix) atomicAdd(&hs[(key >> shift) & digit], 1u);
    };
    if (cached) {
      const int whole = cand & ~3;
      for (int j = 4 * tid; j < whole; j += 4 * THREADS) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + j);
        count(k.x);
        count(k.y);
        count(k.z);
        count(k.w);
      }
      if (tid < cand - whole) count(keys[whole + tid]);
    } else {
#pragma unroll 4
      for (int j = tid; j < cand; j += THREADS) count(key_of(j));
    }
    __syncthreads();
    // thread t < 256 holds digits kBins-1-8t .. kBins-8-8t: counts from the top
    uint32_t c[8], sum = 0, inc = 0;
    if (tid < 256) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = hs[kBins - 1 - 8 * tid - i];
      inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(kFullMask, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) totals[warp] = inc;
    }
    __syncthreads();
    if (tid < 256) {
      uint32_t above = inc - sum;
      for (int w = 0; w < warp; ++w) above += totals[w];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (above < left && above + c[i] >= left) {
          found[0] = kBins - 1 - 8 * tid - i;
          found[1] = left - above;
          found[2] = c[i];
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= digit << shift;
    left = found[1];
    all = left == found[2];
    if (pass == 0) {  // pass 2 counts in this buffer again
      for (int i = tid; i < kBins; i += THREADS) hs[i] = 0;
    }
  }
  // The kept are the keys above the prefix's range and the first `left` within
  // it.  Each warp takes a range of keys: counts, then writes.
  const int span = (cand + WARPS * 32 - 1) / (WARPS * 32) * 32;
  const int lo = warp * span < cand ? warp * span : cand, hi = lo + span < cand ? lo + span : cand;
  int gt = 0, eq = 0;
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int j = j0 + lane;
    const uint32_t key = j < hi ? ((cached ? keys[j] : key_of(j)) & mask) : 0u;
    gt += __popc(__ballot_sync(kFullMask, j < hi && key > prefix));
    eq += __popc(__ballot_sync(kFullMask, j < hi && key == prefix));
  }
  if (lane == 0) warp_count[warp] = make_int2(gt, eq);
  __syncthreads();
  {
    const int2 c = lane < warp ? warp_count[lane] : make_int2(0, 0);  // WARPS <= 32
    gt = __reduce_add_sync(kFullMask, c.x);
    eq = __reduce_add_sync(kFullMask, c.y);
  }
  const uint32_t below = (1u << lane) - 1u;
  const int want = (int)left;
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int j = j0 + lane;
    const uint32_t key = j < hi ? ((cached ? keys[j] : key_of(j)) & mask) : 0u;
    const bool is_gt = j < hi && key > prefix, is_eq = j < hi && key == prefix;
    const uint32_t bg = __ballot_sync(kFullMask, is_gt), be = __ballot_sync(kFullMask, is_eq);
    const int e = eq + __popc(be & below);
    if (is_gt || (is_eq && e < want)) out[gt + __popc(bg & below) + (e < want ? e : want)] = j;
    gt += __popc(bg);
    eq += __popc(be);
  }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(EvictArgs a, int cached) {
  extern __shared__ __align__(16) uint32_t keys[];
  pdl_wait();
  pdl_launch_dependents();
  select_kept<THREADS>(a, cached, keys, blockIdx.x, blockIdx.y, kept_of(a, blockIdx.y));
}

// One slice of the rows: 1 << words_log2 words of VB bytes per row, at
// page + offset + slot * row_stride + word * word_stride.
struct Slice {
  char* pool;
  uint32_t page_bytes;
  int offset, row_stride, word_stride, words_log2;
};

template <int VB> struct MoveWord { using type = typename VecWord<VB>::type; };
template <> struct MoveWord<1> { using type = uint8_t; };

template <int VB>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const Slice& sl, int h, int b, const Kept& s) {
  using W = typename MoveWord<VB>::type;
  const int32_t* kept = a.kept + ((int64_t)b * a.H + h) * a.keep;
  const int32_t* src_row = a.page_table + (int64_t)b * a.pt_stride;
  const int32_t* dst_row = a.out_table ? a.out_table + (int64_t)b * a.out_stride : src_row;
  const int sh = a.bs_log2, low = a.block_size - 1;
  // this thread's word of a row, and its first row of a chunk
  const int word = threadIdx.x & ((1 << sl.words_log2) - 1), row0 = threadIdx.x >> sl.words_log2;
  const int step = kMoveThreads >> sl.words_log2, chunk = step * kMoveWords;
  char* const base = sl.pool + (int64_t)h * sl.page_bytes + sl.offset + (int64_t)word * sl.word_stride;
  const uint64_t block_bytes = (uint64_t)a.H * sl.page_bytes;
  const uint32_t blocks = a.num_blocks < INT32_MAX ? (uint32_t)a.num_blocks : (uint32_t)INT32_MAX;
  auto at = [&](uint32_t blk, int slot) -> W* {
    return reinterpret_cast<W*>(base + blk * block_bytes + slot * sl.row_stride);
  };
  if (blocks == 0) {
    if (s.k > 0) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    return;
  }
  bool bad = false;
  // Rows past the last are read again as the last, rows of a bad page as
  // block 0's: no load hangs on a branch, and neither is stored.
  int src[kMoveWords];  // positions of a chunk's rows
  auto positions = [&](int r0) {
#pragma unroll
    for (int u = 0; u < kMoveWords; ++u) {
      const int r = r0 + row0 + u * step;
      src[u] = kept[r < s.k ? r : s.k - 1];  // (maybe this CTA's own writes)
    }
  };
  if (s.k > 0) positions(0);
  for (int r0 = 0; r0 < s.k; r0 += chunk) {
    W v[kMoveWords];
    uint32_t blk[kMoveWords], ok = 0;
#pragma unroll
    for (int u = 0; u < kMoveWords; ++u) blk[u] = (uint32_t)__ldg(src_row + (src[u] >> sh));
#pragma unroll
    for (int u = 0; u < kMoveWords; ++u) {
      const bool in = blk[u] < blocks;
      ok |= (in ? 1u : 0u) << u;
      v[u] = *at(in ? blk[u] : 0u, src[u] & low);
    }
    positions(r0 + chunk);  // in flight with the rows
#pragma unroll
    for (int u = 0; u < kMoveWords; ++u) {
      const int r = r0 + row0 + u * step;
      blk[u] = (uint32_t)__ldg(dst_row + ((r < s.k ? r : s.k - 1) >> sh));
    }
    __syncthreads();  // the whole chunk has been read
#pragma unroll
    for (int u = 0; u < kMoveWords; ++u) {
      const int r = r0 + row0 + u * step;
      const bool fine = (ok >> u & 1u) && blk[u] < blocks;
      bad |= !fine;
      if (fine && r < s.k) *at(blk[u], r & low) = v[u];
    }
  }
  // the slots behind the kept rows in their last page
  const int end = (s.k + low) & ~low;
  for (int r = s.k + row0; r < end; r += step) {
    const uint32_t to = (uint32_t)__ldg(dst_row + (r >> sh));
    bad |= to >= blocks;
    if (to < blocks) *at(to, r & low) = W{};
  }
  if (bad) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
}

// Slice number `part` of the rows: K and V in 1 << slices_log2 parts each, the
// weights, and the scales of 4-bit K and V.
__device__ __forceinline__ void move_part(const EvictArgs& a, int part, int slices_log2, int h, int b, const Kept& s) {
  const bool kv4 = a.dtype == B2PA_DTYPE_KV4;
  const int row_bytes = kv4 ? a.D / 2 : a.D * a.elem;
  const uint32_t page_bytes = kv4 ? kv4_page_bytes(a.block_size, a.D) : a.block_size * row_bytes;
  if (part < 2 << slices_log2) {
    const int width = row_bytes >> slices_log2;
    Slice sl{static_cast<char*>(part & 1 ? a.v_pool : a.k_pool), page_bytes, part / 2 * width, row_bytes, 16,
             31 - __clz(width / 16)};
    move_rows<16>(a, sl, h, b, s);
    return;
  }
  part -= 2 << slices_log2;
  if (part == 0) {
    Slice sl{reinterpret_cast<char*>(a.weights), 4u * a.block_size, 0, 4, 4, 0};
    move_rows<4>(a, sl, h, b, s);
  } else if (part == 1) {
    Slice sl{static_cast<char*>(a.k_pool), page_bytes, a.block_size * row_bytes, a.D / 16, 4, 31 - __clz(a.D / 64)};
    move_rows<4>(a, sl, h, b, s);
  } else {
    Slice sl{static_cast<char*>(a.v_pool), page_bytes, a.block_size * row_bytes, 1, a.block_size,
             31 - __clz(a.D / 16)};
    move_rows<1>(a, sl, h, b, s);
  }
}

__global__ void __launch_bounds__(kMoveThreads, 4) evict_move_kernel(EvictArgs a, int slices_log2) {
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.y, b = blockIdx.z;
  const Kept s = kept_of(a, b);
  if (!a.out_table && s.n == s.k) return;  // nothing leaves
  move_part(a, blockIdx.x, slices_log2, h, b, s);
}

// Both at once: a CTA selects and then moves the rows of its head and sequence.
__global__ void __launch_bounds__(kMoveThreads, 4) evict_both_kernel(EvictArgs a, int cached) {
  extern __shared__ __align__(16) uint32_t keys[];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y;
  const Kept s = kept_of(a, b);
  select_kept<kMoveThreads>(a, cached, keys, h, b, s);
  if (!a.out_table && s.n == s.k) return;
  __syncthreads();  // the positions are written; the weights have been read
  const int parts = a.dtype == B2PA_DTYPE_KV4 ? 5 : 3;
  for (int part = 0; part < parts; ++part) move_part(a, part, 0, h, b, s);
}

// `kern` with shared memory for the keys where they fit.
int launch_with_keys(const EvictArgs& a, void (*kern)(EvictArgs, int), int threads, cudaStream_t st) {
  const int64_t longest = (int64_t)a.max_pages * a.block_size;
  constexpr int64_t kFixed = 2 * kBins * 4 + 1024;  // static shared memory
  const int cached = longest * 4 + kFixed <= device_max_smem_optin();
  const size_t smem = cached ? (size_t)longest * 4 : 0;
  const int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(kern), (int)smem);
  if (rc != B2PA_OK) return rc;
  const cudaError_t e = launch_pdl(kern, dim3((unsigned)a.H, (unsigned)a.B), dim3(threads), smem, st, a, cached);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "evict launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

}  // namespace

int launch_evict(const EvictArgs& a, cudaStream_t st) {
  if (a.keep <= 0) return B2PA_OK;
  const bool kv4 = a.dtype == B2PA_DTYPE_KV4;
  const int64_t pairs = (int64_t)a.B * a.H;
  // few keys a thread: a small CTA, so that an SM runs several sequences at once
  const bool few = (int64_t)a.max_pages * a.block_size <= 2048;
  // One launch while a CTA's rows are few and most SMs have one: heads that are
  // done selecting move while others select.  Two launches -> one, us: 64
  // sequences of 128-1,024 to 200, 8 heads of 64, fp32 33 -> 29; of 1,024 to
  // 300, heads of 128, bf16: 128 heads in all 21 -> 18, 256 30 -> 26, but 64 15
  // -> 16 and 8 8 -> 13; of 2,000 to 1,500: 128 heads 55 -> 63, 512 158 -> 164.
  if (few && a.keep <= 1024 && 4 * pairs >= 3 * device_sm_count())
    return launch_with_keys(a, evict_both_kernel, kMoveThreads, st);
  const int rc = few ? launch_with_keys(a, evict_select_kernel<256>, 256, st)
                     : launch_with_keys(a, evict_select_kernel<1024>, 1024, st);
  if (rc != B2PA_OK) return rc;
  // rows in parts of 64 bytes or more while the parts are fewer than four CTAs per SM
  const int row_bytes = kv4 ? a.D / 2 : a.D * a.elem;
  int slices_log2 = 0;
  while ((row_bytes >> slices_log2) > 64 && (pairs * 2 << slices_log2) < 4 * device_sm_count()) ++slices_log2;
  const cudaError_t e =
      launch_pdl(evict_move_kernel, dim3((unsigned)((2 << slices_log2) + (kv4 ? 3 : 1)), (unsigned)a.H, (unsigned)a.B),
                 dim3(kMoveThreads), 0, st, a, slices_log2);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "evict launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

}  // namespace b2pa
