// kv4_prefill.cu -- chunked prefill over a 4-bit cache (format: kv4.cuh).
//
// A prompt chunk of T queries makes 4 T L D operations of every L keys, so
// its time is the tensor cores' and not the cache's.  Where the tcgen05 kernel
// of the plain pools can do the rest (head_dim 64 and 128; else
// kv4_prefill_mma.cu does it all), the pages that the call reads are written out
// in the workspace, in q's type or, for fp32, in fp16 (exact either way: a stored
// value has 7 significant bits, so fp32 q needs two products where fp32 pages
// need three), as a pool of B * max_pages blocks with a table of their own, and
// that kernel runs on it; rows past a sequence's length are written as zeros.
// The workspace is thus a 16-bit copy of the call's pages, by the width of the
// table: 3.6 times the 4-bit pages' bytes, for one layer at a time.
// Two kinds of inputs are not for that kernel: NaN groups of V at keys that only
// some of the chunk's queries see (a zero weight times NaN), and scores whose own
// rounding shows (past 2^24, for fp32 2^18).  They leave the call's number in a flag, and the kernel of
// kv4_prefill_mma.cu, launched behind it, redoes the call if it finds it there.
// The number is part of a captured graph: once a replay has set it, later ones
// redo the call too.
#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace b2pa {

// One CTA per (page, sequence): dequantises every head's K and V page.
template <typename T>
__global__ void __launch_bounds__(256) kv4_unpack_kernel(AttnArgs a, T* k_out, T* v_out, int32_t* table,
                                                         uint32_t* flag, uint32_t epoch) {
  pdl_wait();
  pdl_launch_dependents();
  const int p = blockIdx.x, b = blockIdx.y;
  const int64_t slot = (int64_t)b * a.max_pages + p;
  const int BS = a.block_size, D = a.D;
  const int64_t first = (int64_t)p * BS;
  const int64_t L = a.seq_lens[b];
  const bool used = first < L;
  int32_t blk = used ? a.page_table[(int64_t)b * a.pt_stride + p] : -1;
  if (used && (blk < 0 || blk >= a.num_blocks)) {
    if (threadIdx.x == 0 && blk >= a.num_blocks) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    blk = -1;
  }
  if (threadIdx.x == 0) table[slot] = blk >= 0 ? (int32_t)slot : -1;
  if (blk < 0) return;
  const int page_bytes = kv4_page_bytes(BS, D), codes = BS * (D / 2);
  const int wpr_log2 = 31 - __clz(D / 8), head_log2 = wpr_log2 + (31 - __clz(BS));  // words per row, per head page
  const uint8_t* kp = static_cast<const uint8_t*>(a.k_pool) + (uint64_t)blk * a.H * page_bytes;
  const uint8_t* vp = static_cast<const uint8_t*>(a.v_pool) + (uint64_t)blk * a.H * page_bytes;
  T* ko = k_out + ((slot * a.H) << head_log2) * 8;
  T* vo = v_out + ((slot * a.H) << head_log2) * 8;
  const int rows = L - first < BS ? (int)(L - first) : BS;  // the others are zeros
  const int64_t all_see = L - a.cur_lens[b] + 1 - first;      // rows below it are seen by every query
  bool nan = false;
#pragma unroll 2
  for (int i = threadIdx.x; i < a.H << head_log2; i += blockDim.x) {
    const int h = i >> head_log2, r = i & ((1 << head_log2) - 1);  // word r of the head's page
    const int row = r >> wpr_log2, g = (r & ((1 << wpr_log2) - 1)) >> 1;
    const uint8_t* kh = kp + h * page_bytes;
    const uint8_t* vh = vp + h * page_bytes;
    uint32_t wk = *reinterpret_cast<const uint32_t*>(kh + 4 * r), wv = *reinterpret_cast<const uint32_t*>(vh + 4 * r);
    uint32_t ck = kh[codes + row * (D / 16) + g], cv = vh[codes + g * BS + row];
    if (row >= rows) wk = wv = 0x88888888u, ck = cv = 0;
    nan |= cv == kKv4NanScale && row >= all_see;
    kv4_store8(ko + (int64_t)i * 8, wk, ck);
    kv4_store8(vo + (int64_t)i * 8, wv, cv);
  }
  if (nan) *flag = epoch;
}

static size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Whether the tcgen05 kernel takes the shape.  Unpacking and that kernel -> straight
// from the pages (us; 2 sequences, 32 heads, 1,021 queries behind prefixes of 1,024
// and 7,168): fp32 head_dim 64 265 -> 974, 128 409 -> 1,344; bf16 64 196 -> 791, 128
// 293 -> 1,088; head_dim 256 only straight, 2,390 and 1,676.
static bool takes_unpacked(int B, int H, int D, int max_pages, int block_size, int type) {
  return max_pages > 0 && prefill_uses_tensor_cores(D, block_size, type, (int64_t)B * max_pages * H * block_size);
}

Kv4PrefillPlan make_kv4_prefill_plan(int B, int H, int T, int D, int max_pages, int block_size, int dtype) {
  Kv4PrefillPlan pl = {};
  const int type = dtype == B2PA_DTYPE_F32 ? (int)B2PA_DTYPE_F16 : dtype;  // of the unpacked pages
  if (!takes_unpacked(B, H, D, max_pages, block_size, type)) return pl;
  pl.unpack = 1;
  pl.inner_bytes = dtype == B2PA_DTYPE_F32 ? make_prefill_plan(B, H, T, D, max_pages, block_size, type, kHalvesKtCap).bytes
                                           : make_prefill_plan(B, H, T, D, max_pages, block_size, type).bytes;
  const size_t pool = up256((size_t)B * max_pages * H * block_size * D * 2);
  pl.off_v = pool;
  pl.off_table = 2 * pool;
  pl.off_flag = up256(2 * pool + 4 * (size_t)B * max_pages);
  pl.off_inner = pl.off_flag + 256;
  pl.bytes = pl.off_inner + pl.inner_bytes;
  return pl;
}

template <typename T>
static cudaError_t unpack_as(const AttnArgs& a, char* ws, const Kv4PrefillPlan& pl, uint32_t epoch, cudaStream_t s) {
  return launch_pdl(kv4_unpack_kernel<T>, dim3((unsigned)a.max_pages, (unsigned)a.B), dim3(256), 0, s, a,
                    reinterpret_cast<T*>(ws + pl.off_k), reinterpret_cast<T*>(ws + pl.off_v),
                    reinterpret_cast<int32_t*>(ws + pl.off_table), reinterpret_cast<uint32_t*>(ws + pl.off_flag), epoch);
}

int launch_kv4_prefill(const AttnArgs& a, const Kv4PrefillPlan& pl, cudaStream_t s) {
  if (!pl.unpack) return launch_kv4_prefill_mma(a, nullptr, 0, s);
  static std::atomic<uint32_t> calls{0};
  const uint32_t epoch = calls.fetch_add(1, std::memory_order_relaxed) * 2654435761u + 0x9e3779b9u;
  char* ws = static_cast<char*>(a.workspace);
  uint32_t* flag = reinterpret_cast<uint32_t*>(ws + pl.off_flag);
  AttnArgs in = a;
  const cudaError_t e = a.dtype == B2PA_DTYPE_BF16 ? unpack_as<__nv_bfloat16>(a, ws, pl, epoch, s)
                                                   : unpack_as<__half>(a, ws, pl, epoch, s);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "paged_prefill_kv4 launch: %s", cudaGetErrorString(e));
  in.k_pool = ws + pl.off_k;
  in.v_pool = ws + pl.off_v;
  in.num_blocks = (int64_t)a.B * a.max_pages;
  in.page_table = reinterpret_cast<const int32_t*>(ws + pl.off_table);
  in.pt_stride = a.max_pages;
  in.workspace = ws + pl.off_inner;
  in.workspace_bytes = pl.inner_bytes;
  int rc;
  switch (a.dtype) {
    case B2PA_DTYPE_F32: rc = launch_paged_prefill_f32_on_halves(in, flag, epoch, s); break;
    case B2PA_DTYPE_BF16: rc = launch_paged_prefill_bf16(in, s, flag, epoch); break;
    default: rc = launch_paged_prefill_f16(in, s, flag, epoch); break;
  }
  if (rc != B2PA_OK) return rc;
  return launch_kv4_prefill_mma(a, flag, epoch, s);
}

}  // namespace b2pa
