// kv4_rows.cu -- rows into and out of the 4-bit paged pools (format: kv4.cuh).
//
//   kv4_append_kernel  quantises the new tokens' K and V rows into their
//                      pages, one CTA per (token, sequence);
//   kv4_read_kernel    reads rows back as the values they stand for.
//
// Both are bound by the bytes they move (D * element size in and 9/16 D out a
// row, or the reverse).  A thread takes half a group (8 channels) of K and of
// V: one 16-byte load each for 16-bit rows, two for fp32, so the four loads
// are in flight together; a group's maximum takes one shuffle between the
// two threads that share it, and the maximum is taken on the bits of |x|, so
// a NaN or infinity wins it.
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace b2pa {

// Eight channels of a row as fp32: 16-byte loads when VEC, else one by one
// with any channel stride.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int64_t sd, float* x) {
  if constexpr (VEC) {
    constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      Vec<T, N> v;
      v.w = ld_global_nc<uint4>(p + i * N);
      v.to_float(x + i * N);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i * sd]);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (VEC) {
    constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      Vec<T, N> v;
      v.from_float(x + i * N);
      *reinterpret_cast<uint4*>(p + i * N) = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(x[i]);
  }
}

__device__ __forceinline__ uint32_t max_abs_bits(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
    m = m > u ? m : u;
  }
  return m;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(128) kv4_append_kernel(AppendArgs a, int64_t* seq_out) {
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, b = blockIdx.y;
  int len = a.lengths[b];
  len = len < a.T ? len : a.T;
  if (seq_out != nullptr && t == 0 && threadIdx.x == 0) seq_out[b] = (int64_t)a.start_pos[b] + (len > 0 ? len : 0);
  if (t >= len) return;
  const int64_t pos = (int64_t)a.start_pos[b] + t;
  const int64_t page = pos / a.block_size;
  int32_t blk = -1;
  if (pos >= 0 && page < a.max_pages) blk = a.page_table[(int64_t)b * a.pt_stride + page];
  if (blk < 0 || blk >= a.num_blocks) {
    if (threadIdx.x == 0) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
    return;
  }
  const int row = (int)(pos - page * a.block_size);
  const int wpr = a.D / 8;  // words (8 codes) per row: even, so a group's two threads sit in one warp
  const int page_bytes = kv4_page_bytes(a.block_size, a.D);
  const int groups = a.D / 16;
  const T* kn = static_cast<const T*>(a.k_new) + (int64_t)b * a.sk[0] + (int64_t)t * a.sk[2];
  const T* vn = static_cast<const T*>(a.v_new) + (int64_t)b * a.sv[0] + (int64_t)t * a.sv[2];
  char* kp = static_cast<char*>(a.k_pool) + (int64_t)blk * a.H * page_bytes;
  char* vp = static_cast<char*>(a.v_pool) + (int64_t)blk * a.H * page_bytes;
  const int total = a.H * wpr;
  for (int i0 = 0; i0 < total; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    const bool live = i < total;
    const int h = live ? i / wpr : 0;
    const int w = live ? i - h * wpr : 0;
    float xk[8], xv[8];
    load8<T, VEC>(kn + (int64_t)h * a.sk[1] + (int64_t)(8 * w) * a.sk[3], a.sk[3], xk);
    load8<T, VEC>(vn + (int64_t)h * a.sv[1] + (int64_t)(8 * w) * a.sv[3], a.sv[3], xv);
    uint32_t mk = max_abs_bits(xk), mv = max_abs_bits(xv);
    const uint32_t ok = __shfl_xor_sync(kFullMask, mk, 1), ov = __shfl_xor_sync(kFullMask, mv, 1);
    mk = mk > ok ? mk : ok;
    mv = mv > ov ? mv : ov;
    if (!live) continue;
    const uint32_t ck = kv4_scale_code(mk), cv = kv4_scale_code(mv);
    char* kh = kp + (int64_t)h * page_bytes;
    char* vh = vp + (int64_t)h * page_bytes;
    const int codes = a.block_size * (a.D / 2);
    *reinterpret_cast<uint32_t*>(kh + row * (a.D / 2) + 4 * w) = kv4_pack8(xk, kv4_scale(ck));
    *reinterpret_cast<uint32_t*>(vh + row * (a.D / 2) + 4 * w) = kv4_pack8(xv, kv4_scale(cv));
    if ((w & 1) == 0) {
      kh[codes + row * groups + w / 2] = (char)ck;
      vh[codes + (w / 2) * a.block_size + row] = (char)cv;
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(128) kv4_read_kernel(Kv4ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, b = blockIdx.y;
  const int64_t pos = (int64_t)a.start_pos[b] + t;
  const int64_t page = pos / a.block_size;
  bool live = t < a.lengths[b];
  int32_t blk = -1;
  if (live) {
    if (pos >= 0 && page < a.max_pages) blk = a.page_table[(int64_t)b * a.pt_stride + page];
    if (blk < 0 || blk >= a.num_blocks) {
      if (threadIdx.x == 0) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
      live = false;
    }
  }
  const int row = (int)(pos - page * a.block_size);
  const int wpr = a.D / 8;
  const int page_bytes = kv4_page_bytes(a.block_size, a.D);
  const int codes = a.block_size * (a.D / 2);
  const int groups = a.D / 16;
  T* ko = static_cast<T*>(a.k_out) + (int64_t)b * a.sk[0] + (int64_t)t * a.sk[2];
  T* vo = static_cast<T*>(a.v_out) + (int64_t)b * a.sv[0] + (int64_t)t * a.sv[2];
  for (int i = threadIdx.x; i < a.H * wpr; i += blockDim.x) {
    const int h = i / wpr;
    const int w = i - h * wpr;
    float xk[8] = {}, xv[8] = {};
    if (live) {
      const char* kh = static_cast<const char*>(a.k_pool) + ((int64_t)blk * a.H + h) * page_bytes;
      const char* vh = static_cast<const char*>(a.v_pool) + ((int64_t)blk * a.H + h) * page_bytes;
      const uint32_t wk = *reinterpret_cast<const uint32_t*>(kh + row * (a.D / 2) + 4 * w);
      const uint32_t wv = *reinterpret_cast<const uint32_t*>(vh + row * (a.D / 2) + 4 * w);
      const uint32_t ck = (uint8_t)kh[codes + row * groups + w / 2];
      const uint32_t cv = (uint8_t)vh[codes + (w / 2) * a.block_size + row];
      kv4_unpack8(wk, kv4_scale(ck), xk);
      kv4_unpack8(wv, kv4_scale(cv), xv);
    }
    store8<T, VEC>(ko + (int64_t)h * a.sk[1] + 8 * w, xk);
    store8<T, VEC>(vo + (int64_t)h * a.sv[1] + 8 * w, xv);
  }
}

static bool rows16(const void* p, const int64_t* s, int es) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[3] == 1;
  for (int i = 0; i < 3; ++i) ok = ok && (s[i] * es) % 16 == 0;
  return ok;
}

template <typename T>
static int append_as(const AppendArgs& a, int64_t* seq_out, cudaStream_t s) {
  const bool vec = rows16(a.k_new, a.sk, sizeof(T)) && rows16(a.v_new, a.sv, sizeof(T));
  const dim3 grid((unsigned)a.T, (unsigned)a.B);
  const cudaError_t e = vec ? launch_pdl(kv4_append_kernel<T, true>, grid, dim3(128), 0, s, a, seq_out)
                            : launch_pdl(kv4_append_kernel<T, false>, grid, dim3(128), 0, s, a, seq_out);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "kv4_append launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

int launch_kv4_append(const AppendArgs& a, int64_t* seq_out, cudaStream_t s) {
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return append_as<float>(a, seq_out, s);
    case B2PA_DTYPE_BF16: return append_as<__nv_bfloat16>(a, seq_out, s);
    default: return append_as<__half>(a, seq_out, s);
  }
}

template <typename T>
static int read_as(const Kv4ReadArgs& a, cudaStream_t s) {
  const bool vec = rows16(a.k_out, a.sk, sizeof(T)) && rows16(a.v_out, a.sv, sizeof(T));
  const dim3 grid((unsigned)a.T, (unsigned)a.B);
  const cudaError_t e = vec ? launch_pdl(kv4_read_kernel<T, true>, grid, dim3(128), 0, s, a)
                            : launch_pdl(kv4_read_kernel<T, false>, grid, dim3(128), 0, s, a);
  if (e != cudaSuccess) return set_error(B2PA_ERR_CUDA, "kv4_read launch: %s", cudaGetErrorString(e));
  return B2PA_OK;
}

int launch_kv4_read(const Kv4ReadArgs& a, cudaStream_t s) {
  switch (a.dtype) {
    case B2PA_DTYPE_F32: return read_as<float>(a, s);
    case B2PA_DTYPE_BF16: return read_as<__nv_bfloat16>(a, s);
    default: return read_as<__half>(a, s);
  }
}

}  // namespace b2pa
