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
//   evict_select_kernel  one CTA per (head, sequence): radix selection of the
//       k-th largest weight (four passes of 8 bits over order-preserving
//       keys, held in shared memory when they fit), then the kept positions
//       in ascending order;
//   evict_move_kernel    one CTA per (row slice, head, sequence).  In place,
//       row r moves to r' <= r and the rows of one slice are moved in
//       ascending order: a chunk is read whole into registers before any of
//       it is written, and a later chunk's sources lie behind everything that
//       an earlier one writes.  Slices of a row (64 bytes of K or V, the
//       scales, the weights) do not meet, so they run in parallel.
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace b2pa {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kMoveVecs = 8;  // words in flight per thread

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

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(EvictArgs a, int cached) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[256];
  __shared__ uint32_t found[2];
  __shared__ uint32_t totals[2][32];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Kept s = kept_of(a, b);
  if (h == 0 && tid == 0 && a.seq_lens[b] > s.n) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  int32_t* out = a.kept + ((int64_t)b * a.H + h) * a.keep;
  for (int i = s.k + tid; i < a.keep; i += kSelectThreads) out[i] = -1;
  if (s.n == s.k) {
    for (int i = tid; i < s.k; i += kSelectThreads) out[i] = i;
    return;
  }
  const int sure = a.recent < s.k ? a.recent : s.k;
  const int cand = s.n - sure, need = s.k - sure;
  for (int i = tid; i < sure; i += kSelectThreads) out[need + i] = cand + i;
  if (need == 0) return;

  const int32_t* row = a.page_table + (int64_t)b * a.pt_stride;
  auto key_of = [&](int j) -> uint32_t {
    const int32_t blk = row[j >> a.bs_log2];
    if (blk < 0 || blk >= a.num_blocks) return 0;  // reported by the move
    return weight_key(a.weights[((int64_t)blk * a.H + h) * a.block_size + (j & (a.block_size - 1))]);
  };
  if (cached) {
    for (int j = tid; j < cand; j += kSelectThreads) keys[j] = key_of(j);
    __syncthreads();
  }
  uint32_t prefix = 0, mask = 0, left = (uint32_t)need;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j < cand; j += kSelectThreads) {
      const uint32_t key = cached ? keys[j] : key_of(j);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // lane l holds digits 255-8l .. 248-8l: counts from the top
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - 8 * lane - i];
      uint32_t above = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(kFullMask, above, o);
        if (lane >= o) above += y;
      }
      above -= sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (above < left && above + c[i] >= left) {
          found[0] = 255 - 8 * lane - i;
          found[1] = left - above;
        }
        above += c[i];
      }
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= 255u << shift;
    left = found[1];
    __syncthreads();
  }
  // every key above the threshold, and the first `left` that equal it
  uint32_t gt_before = 0, eq_before = 0;
  int turn = 0;
  for (int j0 = 0; j0 < cand; j0 += kSelectThreads, turn ^= 1) {
    const int j = j0 + tid;
    uint32_t key = 0;
    if (j < cand) key = cached ? keys[j] : key_of(j);
    const bool gt = j < cand && key > prefix, eq = j < cand && key == prefix;
    const uint32_t bg = __ballot_sync(kFullMask, gt), be = __ballot_sync(kFullMask, eq);
    if (lane == 0) totals[turn][warp] = __popc(bg) | (__popc(be) << 16);
    __syncthreads();
    const uint32_t mine = totals[turn][lane];
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(kFullMask, inc, o);
      if (lane >= o) inc += y;
    }
    const uint32_t here = __shfl_sync(kFullMask, inc - mine, warp), all = __shfl_sync(kFullMask, inc, 31);
    const uint32_t below = (1u << lane) - 1u;
    const uint32_t g = gt_before + (here & 0xffffu) + __popc(bg & below);
    const uint32_t e = eq_before + (here >> 16) + __popc(be & below);
    if (gt || (eq && e < left)) out[g + (e < left ? e : left)] = j;
    gt_before += all & 0xffffu;
    eq_before += all >> 16;
  }
}

// One slice of the rows: words of VB bytes, `words` per row, at
// page + offset + slot * row_stride + word * word_stride.
struct Slice {
  char* pool;
  int64_t page_bytes;
  int offset, row_stride, word_stride, words;
};

template <int VB> struct MoveWord { using type = typename VecWord<VB>::type; };
template <> struct MoveWord<1> { using type = uint8_t; };

template <int VB>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const Slice& sl, int h, int b, const Kept& s) {
  using W = typename MoveWord<VB>::type;
  const int32_t* kept = a.kept + ((int64_t)b * a.H + h) * a.keep;
  const int32_t* src_row = a.page_table + (int64_t)b * a.pt_stride;
  const int32_t* dst_row = a.out_table ? a.out_table + (int64_t)b * a.out_stride : src_row;
  auto at = [&](int32_t blk, int slot, int c) -> W* {
    return reinterpret_cast<W*>(sl.pool + ((int64_t)blk * a.H + h) * sl.page_bytes + sl.offset + slot * sl.row_stride +
                                c * sl.word_stride);
  };
  const int bs = a.block_size, sh = a.bs_log2;
  const int64_t total = (int64_t)s.k * sl.words;
  for (int64_t base = 0; base < total; base += kMoveThreads * kMoveVecs) {
    W v[kMoveVecs];
    bool ok[kMoveVecs];
#pragma unroll
    for (int u = 0; u < kMoveVecs; ++u) {
      const int64_t e = base + u * kMoveThreads + threadIdx.x;
      ok[u] = false;
      if (e < total) {
        const int r = (int)(e / sl.words), c = (int)(e - (int64_t)r * sl.words);
        const int j = kept[r];
        const int32_t blk = src_row[j >> sh];
        ok[u] = blk >= 0 && blk < a.num_blocks;
        if (ok[u])
          v[u] = *at(blk, j & (bs - 1), c);
        else
          set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveVecs; ++u) {
      const int64_t e = base + u * kMoveThreads + threadIdx.x;
      if (ok[u]) {
        const int r = (int)(e / sl.words), c = (int)(e - (int64_t)r * sl.words);
        const int32_t blk = dst_row[r >> sh];
        if (blk >= 0 && blk < a.num_blocks)
          *at(blk, r & (bs - 1), c) = v[u];
        else
          set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
      }
    }
  }
  // the slots behind the kept rows in their last page
  const int behind = (s.k + bs - 1) / bs * bs - s.k;
  for (int e = threadIdx.x; e < behind * sl.words; e += kMoveThreads) {
    const int r = s.k + e / sl.words, c = e % sl.words;
    const int32_t blk = dst_row[r >> sh];
    if (blk >= 0 && blk < a.num_blocks) *at(blk, r & (bs - 1), c) = W{};
  }
}

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(EvictArgs a, int row_slices) {
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.y, b = blockIdx.z;
  const Kept s = kept_of(a, b);
  if (!a.out_table && s.n == s.k) return;  // nothing leaves
  int part = blockIdx.x;
  const bool kv4 = a.dtype == B2PA_DTYPE_KV4;
  const int row_bytes = kv4 ? a.D / 2 : a.D * a.elem;
  const int64_t page_bytes = kv4 ? kv4_page_bytes(a.block_size, a.D) : (int64_t)a.block_size * row_bytes;
  if (part < 2 * row_slices) {
    const int width = row_bytes / row_slices;
    Slice sl{static_cast<char*>(part & 1 ? a.v_pool : a.k_pool), page_bytes, part / 2 * width, row_bytes, 16, width / 16};
    move_rows<16>(a, sl, h, b, s);
    return;
  }
  part -= 2 * row_slices;
  if (part == 0) {
    Slice sl{reinterpret_cast<char*>(a.weights), 4ll * a.block_size, 0, 4, 4, 1};
    move_rows<4>(a, sl, h, b, s);
  } else if (part == 1) {
    Slice sl{static_cast<char*>(a.k_pool), page_bytes, a.block_size * row_bytes, a.D / 16, 4, a.D / 64};
    move_rows<4>(a, sl, h, b, s);
  } else {
    Slice sl{static_cast<char*>(a.v_pool), page_bytes, a.block_size * row_bytes, 1, a.block_size, a.D / 16};
    move_rows<1>(a, sl, h, b, s);
  }
}

}  // namespace

int launch_evict(const EvictArgs& a, cudaStream_t st) {
  if (a.keep <= 0) return B2PA_OK;
  const bool kv4 = a.dtype == B2PA_DTYPE_KV4;
  const int64_t longest = (int64_t)a.max_pages * a.block_size;
  const int64_t room = (device_max_smem_optin() - 4096) / 4;
  const int cached = longest <= room;
  const size_t smem = cached ? (size_t)longest * 4 : 0;
  int rc = set_max_dynamic_smem_cached(reinterpret_cast<const void*>(evict_select_kernel), (int)smem);
  if (rc != B2PA_OK) return rc;
  cudaError_t e = launch_pdl(evict_select_kernel, dim3((unsigned)a.H, (unsigned)a.B), dim3(kSelectThreads), smem, st, a,
                             cached);
  if (e == cudaSuccess) {
    const int row_bytes = kv4 ? a.D / 2 : a.D * a.elem;
    const int slices = row_bytes >= 64 ? row_bytes / 64 : 1;
    e = launch_pdl(evict_move_kernel, dim3((unsigned)(2 * slices + (kv4 ? 3 : 1)), (unsigned)a.H, (unsigned)a.B),
                   dim3(kMoveThreads), 0, st, a, slices);
  }
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "evict launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

}  // namespace b2pa
