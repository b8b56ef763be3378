// abi_compress.cu -- extern "C" entry points of the cache-compression
// operators: the 4-bit KV cache and eviction by accumulated attention weight
// (declared in b2pa.h).  Same conventions as abi.cu: arguments are checked on
// the host, nothing allocates or synchronises, errors are status codes.
#include <cuda_runtime.h>

#include "b2pa.h"
#include "kernels.h"

using namespace b2pa;

namespace {

constexpr int kMaxGrid = 65535;

bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Sizes common to every entry point.
int check_sizes(const char* fn, int B, int H, int T, int D, int block_size, int max_pages, int64_t num_blocks) {
  if (B < 0 || H <= 0 || T < 0 || D <= 0 || block_size <= 0 || max_pages < 0 || num_blocks < 0)
    return set_error(B2PA_ERR_INVALID_ARGUMENT,
                     "%s: bad sizes B=%d H=%d T=%d D=%d block_size=%d max_pages=%d num_blocks=%lld", fn, B, H, T, D,
                     block_size, max_pages, (long long)num_blocks);
  if (!block_size_supported(block_size))
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: block_size %d not built", fn, block_size);
  if (B > kMaxGrid || H > kMaxGrid)
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: B=%d or H=%d above %d", fn, B, H, kMaxGrid);
  if ((int64_t)max_pages * block_size > INT32_MAX)
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: max_pages %d of %d rows exceed 2^31 positions", fn, max_pages, block_size);
  return B2PA_OK;
}

int check_table(const char* fn, const int32_t* table, int64_t stride, int max_pages) {
  if (max_pages > 0 && !table) return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: null page_table", fn);
  if (max_pages > 0 && stride < max_pages)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: page-table row stride %lld < max_pages %d", fn, (long long)stride,
                     max_pages);
  return B2PA_OK;
}

int check_kv4(const char* fn, int D, const void* k_pool, const void* v_pool) {
  if (!kv4_head_dim_supported(D))
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: head_dim %d not built for 4-bit pages (64, 128, 256)", fn, D);
  if (!aligned_to(k_pool, 16) || !aligned_to(v_pool, 16))
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: pool base pointers must be 16-byte aligned", fn);
  return B2PA_OK;
}

// q and out (may be null): unit D stride, rows 16-byte aligned.
int check_rows(const char* fn, const void* q, const int64_t* qs, const void* out, const int64_t* os, int es) {
  for (int n = 0; n < 2; ++n) {
    const void* p = n ? out : q;
    const int64_t* s = n ? os : qs;
    if (!p) continue;
    if (s[3] != 1) return set_error(B2PA_ERR_UNSUPPORTED, "%s: q/out need a unit D stride", fn);
    bool ok = aligned_to(p, 16);
    for (int i = 0; i < 3; ++i) ok = ok && (s[i] * es) % 16 == 0;
    if (!ok) return set_error(B2PA_ERR_UNSUPPORTED, "%s: q/out rows must be 16-byte aligned", fn);
  }
  return B2PA_OK;
}

int check_workspace(const char* fn, const void* ws, size_t have, size_t need) {
  if (need == 0) return B2PA_OK;
  if (!ws || have < need)
    return set_error(B2PA_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", fn, have, need);
  if (!aligned_to(ws, 256)) return set_error(B2PA_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", fn);
  return B2PA_OK;
}

#define B2PA_TRY(expr)               \
  do {                               \
    const int rc_ = (expr);          \
    if (rc_ != B2PA_OK) return rc_;  \
  } while (0)

int attention_args(const char* fn, AttnArgs& a, const void* q, const int64_t* qs, const void* k_pool,
                   const void* v_pool, int64_t num_blocks, const int32_t* page_table, int64_t pt_stride, int max_pages,
                   const int32_t* seq_lens, const int32_t* cur_lens, void* out, const int64_t* os, int B, int H, int T,
                   int D, int block_size, float scale, int dtype, void* workspace, size_t workspace_bytes,
                   int32_t* status) {
  B2PA_TRY(check_sizes(fn, B, H, T, D, block_size, max_pages, num_blocks));
  if (dtype_size(dtype) == 0) return set_error(B2PA_ERR_UNSUPPORTED, "%s: unknown dtype %d", fn, dtype);
  B2PA_TRY(check_kv4(fn, D, k_pool, v_pool));
  if (B == 0 || T == 0) return B2PA_OK;
  if (!q || !qs || !k_pool || !v_pool || !seq_lens || !cur_lens || !out || !os)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  B2PA_TRY(check_table(fn, page_table, pt_stride, max_pages));
  B2PA_TRY(check_rows(fn, q, qs, out, os, dtype_size(dtype)));
  a = AttnArgs{};
  a.q = q;
  a.out = out;
  for (int i = 0; i < 4; ++i) {
    a.sq[i] = qs[i];
    a.so[i] = os[i];
  }
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.num_blocks = num_blocks;
  a.page_table = page_table;
  a.pt_stride = pt_stride;
  a.max_pages = max_pages;
  a.seq_lens = seq_lens;
  a.cur_lens = cur_lens;
  a.B = B;
  a.H = H;
  a.T = T;
  a.D = D;
  a.block_size = block_size;
  a.dtype = dtype;
  a.scale = scale;
  a.workspace = workspace;
  a.workspace_bytes = workspace_bytes;
  a.status = status;
  return B2PA_OK;
}

}  // namespace

extern "C" {

int b2pa_kv4_append(const void* k_new, const int64_t new_k_strides[4], const void* v_new,
                    const int64_t new_v_strides[4], void* k_pool, void* v_pool, int64_t num_blocks,
                    const int32_t* page_table, int64_t pt_stride, int max_pages, const int32_t* start_pos,
                    const int32_t* lengths, int64_t* seq_lens_out, int B, int H, int T, int D, int block_size,
                    int dtype, int32_t* status, void* stream) {
  const char* fn = "kv4_append";
  B2PA_TRY(check_sizes(fn, B, H, T, D, block_size, max_pages, num_blocks));
  if (dtype_size(dtype) == 0) return set_error(B2PA_ERR_UNSUPPORTED, "%s: unknown dtype %d", fn, dtype);
  B2PA_TRY(check_kv4(fn, D, k_pool, v_pool));
  if (B == 0 || (T == 0 && !seq_lens_out)) return B2PA_OK;
  if ((T > 0 && (!k_new || !v_new)) || !k_pool || !v_pool || !new_k_strides || !new_v_strides || !start_pos || !lengths)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  B2PA_TRY(check_table(fn, page_table, pt_stride, max_pages));
  AppendArgs a{};
  a.k_new = k_new;
  a.v_new = v_new;
  for (int i = 0; i < 4; ++i) {
    a.sk[i] = new_k_strides[i];
    a.sv[i] = new_v_strides[i];
  }
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.num_blocks = num_blocks;
  a.page_table = page_table;
  a.pt_stride = pt_stride;
  a.max_pages = max_pages;
  a.start_pos = start_pos;
  a.lengths = lengths;
  a.B = B;
  a.H = H;
  a.T = T;
  a.D = D;
  a.block_size = block_size;
  a.dtype = dtype;
  a.bs_log2 = block_size_log2(block_size);
  a.status = status;
  return launch_kv4_append(a, seq_lens_out, static_cast<cudaStream_t>(stream));
}

int b2pa_kv4_read(const void* k_pool, const void* v_pool, int64_t num_blocks, const int32_t* page_table,
                  int64_t pt_stride, int max_pages, const int32_t* start_pos, const int32_t* lengths, void* k_out,
                  const int64_t k_strides[4], void* v_out, const int64_t v_strides[4], int B, int H, int T, int D,
                  int block_size, int dtype, int32_t* status, void* stream) {
  const char* fn = "kv4_read";
  B2PA_TRY(check_sizes(fn, B, H, T, D, block_size, max_pages, num_blocks));
  if (dtype_size(dtype) == 0) return set_error(B2PA_ERR_UNSUPPORTED, "%s: unknown dtype %d", fn, dtype);
  B2PA_TRY(check_kv4(fn, D, k_pool, v_pool));
  if (B == 0 || T == 0) return B2PA_OK;
  if (!k_out || !v_out || !k_pool || !v_pool || !k_strides || !v_strides || !start_pos || !lengths)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (k_strides[3] != 1 || v_strides[3] != 1)
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: k_out/v_out need a unit D stride", fn);
  B2PA_TRY(check_table(fn, page_table, pt_stride, max_pages));
  Kv4ReadArgs a{};
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.num_blocks = num_blocks;
  a.page_table = page_table;
  a.pt_stride = pt_stride;
  a.max_pages = max_pages;
  a.start_pos = start_pos;
  a.lengths = lengths;
  a.k_out = k_out;
  a.v_out = v_out;
  for (int i = 0; i < 4; ++i) {
    a.sk[i] = k_strides[i];
    a.sv[i] = v_strides[i];
  }
  a.B = B;
  a.H = H;
  a.T = T;
  a.D = D;
  a.block_size = block_size;
  a.dtype = dtype;
  a.bs_log2 = block_size_log2(block_size);
  a.status = status;
  return launch_kv4_read(a, static_cast<cudaStream_t>(stream));
}

int b2pa_paged_decode_kv4(const void* q, const int64_t q_strides[4], const void* k_pool, const void* v_pool,
                          int64_t num_blocks, const int32_t* page_table, int64_t pt_stride, int max_pages,
                          const int32_t* seq_lens, const int32_t* cur_lens, void* out, const int64_t out_strides[4],
                          int B, int H, int D, int block_size, float scale, int dtype, int32_t* status,
                          void* stream) {
  const char* fn = "paged_decode_kv4";
  AttnArgs a{};
  B2PA_TRY(attention_args(fn, a, q, q_strides, k_pool, v_pool, num_blocks, page_table, pt_stride, max_pages, seq_lens,
                          cur_lens, out, out_strides, B, H, 1, D, block_size, scale, dtype, nullptr, 0, status));
  if (B == 0) return B2PA_OK;
  return launch_kv4_decode(a, static_cast<cudaStream_t>(stream));
}

size_t b2pa_paged_prefill_kv4_workspace_size(int B, int H, int T, int D, int max_pages, int block_size, int dtype) {
  if (B <= 0 || H <= 0 || T <= 0 || D <= 0 || max_pages < 0 || block_size <= 0 || dtype_size(dtype) == 0) return 0;
  return make_kv4_prefill_plan(B, H, T, D, max_pages, block_size, dtype).bytes;
}

int b2pa_paged_prefill_kv4(const void* q, const int64_t q_strides[4], const void* k_pool, const void* v_pool,
                           int64_t num_blocks, const int32_t* page_table, int64_t pt_stride, int max_pages,
                           const int32_t* seq_lens, const int32_t* cur_lens, void* out, const int64_t out_strides[4],
                           int B, int H, int T, int D, int block_size, float scale, int dtype, void* workspace,
                           size_t workspace_bytes, int32_t* status, void* stream) {
  const char* fn = "paged_prefill_kv4";
  AttnArgs a{};
  B2PA_TRY(attention_args(fn, a, q, q_strides, k_pool, v_pool, num_blocks, page_table, pt_stride, max_pages, seq_lens,
                          cur_lens, out, out_strides, B, H, T, D, block_size, scale, dtype, workspace, workspace_bytes,
                          status));
  if (B == 0 || T == 0) return B2PA_OK;
  if (T > 65535 * 32) return set_error(B2PA_ERR_UNSUPPORTED, "%s: T=%d too large", fn, T);
  if ((int64_t)B * max_pages > INT32_MAX)
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: B * max_pages = %lld slots exceed the int32 table", fn,
                     (long long)B * max_pages);
  const Kv4PrefillPlan plan = make_kv4_prefill_plan(B, H, T, D, max_pages, block_size, dtype);
  B2PA_TRY(check_workspace(fn, workspace, workspace_bytes, plan.bytes));
  return launch_kv4_prefill(a, plan, static_cast<cudaStream_t>(stream));
}

size_t b2pa_key_weights_workspace_size(int B, int H, int T, int D, int max_pages, int block_size, int dtype,
                                       int pool_dtype) {
  if (B <= 0 || H <= 0 || T <= 0 || D <= 0 || max_pages < 0 || block_size <= 0 || dtype_size(dtype) == 0) return 0;
  return key_weights_workspace(B, H, T, D, max_pages, block_size, dtype, pool_dtype);
}

int b2pa_key_weights(const void* q, const int64_t q_strides[4], const void* k_pool, int pool_dtype, int64_t num_blocks,
                     const int32_t* page_table, int64_t pt_stride, int max_pages, const int32_t* seq_lens,
                     const int32_t* cur_lens, int window, const float* weights_in, float* weights_out, int B, int H,
                     int T, int D, int block_size, float scale, int dtype, void* workspace, size_t workspace_bytes,
                     int32_t* status, void* stream) {
  const char* fn = "key_weights";
  B2PA_TRY(check_sizes(fn, B, H, T, D, block_size, max_pages, num_blocks));
  if (dtype_size(dtype) == 0) return set_error(B2PA_ERR_UNSUPPORTED, "%s: unknown dtype %d", fn, dtype);
  if (pool_dtype != dtype && pool_dtype != B2PA_DTYPE_KV4)
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: a pool of type %d needs a q of the same type, not %d", fn, pool_dtype,
                     dtype);
  if (pool_dtype == B2PA_DTYPE_KV4) {
    B2PA_TRY(check_kv4(fn, D, k_pool, k_pool));
  } else if (!head_dim_supported(D)) {
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: head_dim %d not built", fn, D);
  }
  if (window < 0) return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: window %d < 0", fn, window);
  if (B == 0 || T == 0) return B2PA_OK;
  if (!q || !q_strides || !k_pool || !seq_lens || !cur_lens || !weights_in || !weights_out)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  B2PA_TRY(check_table(fn, page_table, pt_stride, max_pages));
  B2PA_TRY(check_rows(fn, q, q_strides, nullptr, nullptr, dtype_size(dtype)));
  if (!aligned_to(k_pool, 16))
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: pool base pointers must be 16-byte aligned", fn);
  B2PA_TRY(check_workspace(fn, workspace, workspace_bytes,
                           key_weights_workspace(B, H, T, D, max_pages, block_size, dtype, pool_dtype)));
  KeyWeightArgs a{};
  a.q = q;
  for (int i = 0; i < 4; ++i) a.sq[i] = q_strides[i];
  a.k_pool = k_pool;
  a.num_blocks = num_blocks;
  a.page_table = page_table;
  a.pt_stride = pt_stride;
  a.max_pages = max_pages;
  a.seq_lens = seq_lens;
  a.cur_lens = cur_lens;
  a.w_in = weights_in;
  a.w_out = weights_out;
  a.window = window;
  a.B = B;
  a.H = H;
  a.T = T;
  a.D = D;
  a.block_size = block_size;
  a.dtype = dtype;
  a.pool_dtype = pool_dtype;
  a.bs_log2 = block_size_log2(block_size);
  a.scale = scale;
  a.workspace = workspace;
  a.status = status;
  return launch_key_weights(a, static_cast<cudaStream_t>(stream));
}

int b2pa_evict(void* k_pool, void* v_pool, int pool_dtype, float* weights, int64_t num_blocks,
               const int32_t* page_table, int64_t pt_stride, int max_pages, const int32_t* out_table,
               int64_t out_stride, const int32_t* seq_lens, int keep, int recent, int32_t* kept, int B, int H, int D,
               int block_size, int32_t* status, void* stream) {
  const char* fn = "evict";
  B2PA_TRY(check_sizes(fn, B, H, 1, D, block_size, max_pages, num_blocks));
  if (pool_dtype == B2PA_DTYPE_KV4) {
    B2PA_TRY(check_kv4(fn, D, k_pool, v_pool));
  } else {
    if (dtype_size(pool_dtype) == 0) return set_error(B2PA_ERR_UNSUPPORTED, "%s: unknown dtype %d", fn, pool_dtype);
    if (!head_dim_supported(D)) return set_error(B2PA_ERR_UNSUPPORTED, "%s: head_dim %d not built", fn, D);
    if (!aligned_to(k_pool, 16) || !aligned_to(v_pool, 16))
      return set_error(B2PA_ERR_UNSUPPORTED, "%s: pool base pointers must be 16-byte aligned", fn);
  }
  if (keep < 0 || recent < 0)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: keep %d and recent %d must not be negative", fn, keep, recent);
  if (B == 0 || keep == 0) return B2PA_OK;
  if (!k_pool || !v_pool || !weights || !seq_lens || !kept)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: null pointer argument", fn);
  if (!aligned_to(weights, 16))
    return set_error(B2PA_ERR_UNSUPPORTED, "%s: weights must be 16-byte aligned", fn);
  B2PA_TRY(check_table(fn, page_table, pt_stride, max_pages));
  if (out_table && out_stride * (int64_t)block_size < keep)
    return set_error(B2PA_ERR_INVALID_ARGUMENT, "%s: out_table rows of %lld pages do not hold %d rows", fn,
                     (long long)out_stride, keep);
  EvictArgs a{};
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.weights = weights;
  a.num_blocks = num_blocks;
  a.page_table = page_table;
  a.pt_stride = pt_stride;
  a.max_pages = max_pages;
  a.out_table = out_table;
  a.out_stride = out_stride;
  a.seq_lens = seq_lens;
  a.keep = keep;
  a.recent = recent;
  a.kept = kept;
  a.B = B;
  a.H = H;
  a.D = D;
  a.block_size = block_size;
  a.dtype = pool_dtype;
  a.bs_log2 = block_size_log2(block_size);
  a.elem = dtype_size(pool_dtype);
  a.status = status;
  return launch_evict(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
