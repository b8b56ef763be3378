// key_weights.cu -- accumulated attention weight of every cached key.
//
// For each head and cached key j of sequence b:
//     w[j] += sum over counted queries t of softmax_j(q_t . K^T scale),
// query t (position seq_len - cur_len + t) seeing keys 0 .. min(seq_len,
// pos + 1) - 1, and counting when cur_len - window <= t < cur_len (all of
// them without a window).  Two passes: the log-sum-exp of every counted
// query, then each key's sum of exp(logit - lse).
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace b2pa {

namespace {

// One channel of a key row.
template <typename T, bool KV4>
__device__ __forceinline__ float key_channel(const void* pool, int64_t page, int row, int d, int BS, int D) {
  if constexpr (KV4) {
    const uint8_t* p = static_cast<const uint8_t*>(pool) + page * kv4_page_bytes(BS, D);
    const int c = (int)(p[row * (D / 2) + d / 2] >> (4 * (d & 1)) & 15) - 8;
    return (float)c * kv4_scale(p[BS * (D / 2) + row * (D / 16) + d / 16]);
  } else {
    return to_f32(static_cast<const T*>(pool)[(page * BS + row) * D + d]);
  }
}

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

template <typename T, bool KV4>
__global__ void __launch_bounds__(128) key_lse_kernel(KeyWeightArgs a, float qscale) {
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const Span s = span_of(a, b);
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && (int64_t)a.seq_lens[b] > s.L)
    set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i >= s.count) return;
  const int t = s.first + i;
  const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1] + (int64_t)t * a.sq[2];
  int64_t vis = s.past + t + 1;
  vis = vis < s.L ? vis : s.L;
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < vis; ++j) {
    const int32_t blk = a.page_table[(int64_t)b * a.pt_stride + j / a.block_size];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0 && blk >= a.num_blocks) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
      continue;
    }
    const int64_t page = (int64_t)blk * a.H + h;
    float dot = 0.f;
    for (int d = lane; d < a.D; d += 32)
      dot += to_f32(q[d]) * key_channel<T, KV4>(a.k_pool, page, (int)(j % a.block_size), d, a.block_size, a.D);
    dot = warp_sum(dot) * qscale;
    const float mn = fmaxf(m, dot);
    const float ref = mn == -INFINITY ? 0.f : mn;
    l = l * fast_exp2(m - ref) + fast_exp2(dot - ref);
    m = mn;
  }
  if (lane == 0) a.lse[((int64_t)b * a.H + h) * a.T + i] = m == -INFINITY ? -INFINITY : m + log2f(l);
}

template <typename T, bool KV4>
__global__ void __launch_bounds__(128) key_sum_kernel(KeyWeightArgs a, float qscale) {
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const Span s = span_of(a, b);
  const int64_t j = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (j >= s.L) return;
  const int32_t blk = a.page_table[(int64_t)b * a.pt_stride + j / a.block_size];
  if (blk < 0 || blk >= a.num_blocks) return;
  const int64_t page = (int64_t)blk * a.H + h;
  const int row = (int)(j % a.block_size);
  float sum = 0.f;
  for (int i = 0; i < s.count; ++i) {
    const int t = s.first + i;
    if (j > s.past + t) continue;
    const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1] + (int64_t)t * a.sq[2];
    float dot = 0.f;
    for (int d = lane; d < a.D; d += 32)
      dot += to_f32(q[d]) * key_channel<T, KV4>(a.k_pool, page, row, d, a.block_size, a.D);
    dot = warp_sum(dot) * qscale;
    const float lse = a.lse[((int64_t)b * a.H + h) * a.T + i];
    if (lse != -INFINITY) sum += fast_exp2(dot - lse);
  }
  if (lane == 0) a.w_out[page * a.block_size + row] = a.w_in[page * a.block_size + row] + sum;
}

template <typename T, bool KV4>
int weights_as(const KeyWeightArgs& a, cudaStream_t s) {
  const float qscale = a.scale * kLog2e;
  const int64_t keys = (int64_t)a.max_pages * a.block_size;
  cudaError_t e = launch_pdl(key_lse_kernel<T, KV4>, dim3((unsigned)((a.T + 3) / 4), (unsigned)a.H, (unsigned)a.B),
                             dim3(128), 0, s, a, qscale);
  if (e == cudaSuccess && keys > 0)
    e = launch_pdl(key_sum_kernel<T, KV4>, dim3((unsigned)((keys + 3) / 4), (unsigned)a.H, (unsigned)a.B), dim3(128), 0,
                   s, a, qscale);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "key_weights launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

}  // namespace

size_t key_weights_workspace(int B, int H, int T, int D, int max_pages, int block_size, int dtype, int pool_dtype) {
  (void)D, (void)max_pages, (void)block_size, (void)dtype, (void)pool_dtype;
  return (size_t)B * H * T * sizeof(float);
}

int launch_key_weights(const KeyWeightArgs& a0, cudaStream_t s) {
  KeyWeightArgs a = a0;
  a.lse = static_cast<float*>(a.workspace);
  const bool kv4 = a.pool_dtype == B2PA_DTYPE_KV4;
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return kv4 ? weights_as<float, true>(a, s) : weights_as<float, false>(a, s);
    case B2PA_DTYPE_BF16: return kv4 ? weights_as<__nv_bfloat16, true>(a, s) : weights_as<__nv_bfloat16, false>(a, s);
    default: return kv4 ? weights_as<__half, true>(a, s) : weights_as<__half, false>(a, s);
  }
}

}  // namespace b2pa
