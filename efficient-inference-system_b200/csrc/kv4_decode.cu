// kv4_decode.cu -- single-query paged attention over a 4-bit cache (format:
// kv4.cuh).
//
// For sequence b the query sits at position seq_len - cur_len and sees keys
// 0 .. min(seq_len, seq_len - cur_len + 1) - 1; out = softmax(q.K^T scale).V
// with K and V the values the pages stand for, in fp32, stored in the type of
// q; zeros when no key is visible.
//
// One CTA per (head, sequence); each warp takes every fourth key with its own
// online softmax (running maximum, sum and output), joined in shared memory.
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace b2pa {

template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_decode_kernel(AttnArgs a, float qscale) {
  constexpr int E = D / 32;  // channels per lane
  __shared__ float sm_m[4], sm_l[4], sm_acc[4][D];
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int BS = a.block_size;
  int64_t L = a.seq_lens[b];
  const int64_t cap = (int64_t)a.max_pages * BS;
  if (L > cap) {
    if (threadIdx.x == 0) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    L = cap;
  }
  int64_t vis = (int64_t)a.seq_lens[b] - a.cur_lens[b] + 1;
  vis = vis < L ? vis : L;
  const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.sq[0] + (int64_t)h * a.sq[1] + lane * E;
  float x[E], acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    x[i] = to_f32(q[i]) * qscale;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int page_bytes = kv4_page_bytes(BS, D);
  for (int64_t j = warp; j < vis; j += 4) {
    const int32_t blk = a.page_table[(int64_t)b * a.pt_stride + j / BS];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0 && blk >= a.num_blocks) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
      continue;
    }
    const int row = (int)(j % BS);
    const uint8_t* kp = static_cast<const uint8_t*>(a.k_pool) + ((int64_t)blk * a.H + h) * page_bytes;
    const uint8_t* vp = static_cast<const uint8_t*>(a.v_pool) + ((int64_t)blk * a.H + h) * page_bytes;
    const int codes = BS * (D / 2), g = lane * E / 16;
    const float ks = kv4_scale(kp[codes + row * (D / 16) + g]);
    const float vs = kv4_scale(vp[codes + g * BS + row]);
    float dot = 0.f, v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = lane * E + i, sh = 4 * (c & 1);
      dot += x[i] * (float)((int)(kp[row * (D / 2) + c / 2] >> sh & 15) - 8) * ks;
      v[i] = (float)((int)(vp[row * (D / 2) + c / 2] >> sh & 15) - 8) * vs;
    }
    dot = warp_sum(dot);
    const float mn = fmaxf(m, dot);
    // a logit of -inf (an infinite query) leaves nothing to subtract
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float corr = fast_exp2(m - ref), p = fast_exp2(dot - ref);
    m = mn;
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = acc[i] * corr + p * v[i];
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) sm_acc[warp][lane * E + i] = acc[i];
  __syncthreads();
  float M = -INFINITY;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w]);
  if (M == -INFINITY) M = 0.f;
  float total = 0.f;
  for (int w = 0; w < 4; ++w) total += sm_l[w] * fast_exp2(sm_m[w] - M);
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.so[0] + (int64_t)h * a.so[1];
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float o = 0.f;
    for (int w = 0; w < 4; ++w) o += sm_acc[w][d] * fast_exp2(sm_m[w] - M);
    out[d] = from_f32<T>(total != 0.f ? o / total : 0.f);
  }
}

template <typename T>
static int decode_as(const AttnArgs& a, cudaStream_t s) {
  const dim3 grid((unsigned)a.H, (unsigned)a.B);
  const float qscale = a.scale * kLog2e;
  cudaError_t e;
  switch (a.D) {
    case 64: e = launch_pdl(kv4_decode_kernel<T, 64>, grid, dim3(128), 0, s, a, qscale); break;
    case 128: e = launch_pdl(kv4_decode_kernel<T, 128>, grid, dim3(128), 0, s, a, qscale); break;
    default: e = launch_pdl(kv4_decode_kernel<T, 256>, grid, dim3(128), 0, s, a, qscale); break;
  }
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "paged_decode_kv4 launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

size_t kv4_decode_workspace(int, int, int, int, int) { return 0; }

int launch_kv4_decode(const AttnArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return decode_as<float>(a, s);
    case B2PA_DTYPE_BF16: return decode_as<__nv_bfloat16>(a, s);
    default: return decode_as<__half>(a, s);
  }
}

}  // namespace b2pa
