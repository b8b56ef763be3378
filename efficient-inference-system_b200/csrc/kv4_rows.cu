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

__device__ __forceinline__ uint32_t max_abs_bits(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;
    m = m > u ? m : u;
  }
  return m;
}

// A CTA takes the rows of one token and all heads, or -- vectorised, for
// prompts -- of several neighbouring tokens of a sequence: the table entry and
// the addresses of a (head, word) are worked out once for all of them.
template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(128) kv4_append_kernel(AppendArgs a, int64_t* seq_out) {
  pdl_wait();
  pdl_launch_dependents();
  const int t0 = blockIdx.x * TOKENS, b = blockIdx.y;
  int len = a.lengths[b];
  len = len < a.T ? len : a.T;
  if (seq_out != nullptr && t0 == 0 && threadIdx.x == 0) seq_out[b] = (int64_t)a.start_pos[b] + (len > 0 ? len : 0);
  if (t0 >= len) return;
  const int64_t start = a.start_pos[b];
  // a token's block (or -1) and row
  int32_t blk[TOKENS];
  int row[TOKENS];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const int64_t pos = start + t0 + i, page = pos >> a.bs_log2;
    blk[i] = -1;
    row[i] = (int)(pos & (a.block_size - 1));
    if (t0 + i < len) {
      if (pos >= 0 && page < a.max_pages) blk[i] = a.page_table[(int64_t)b * a.pt_stride + page];
      if (blk[i] < 0 || blk[i] >= a.num_blocks) {
        blk[i] = -1;
        bad = true;
      }
    }
  }
  if (bad && threadIdx.x == 0) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  const int wpr = a.D / 8;  // words (8 codes) per row: a power of two, so a group's two threads sit in one warp
  const int wpr_log2 = 31 - __clz(wpr);
  const int page_bytes = kv4_page_bytes(a.block_size, a.D);
  const int codes = a.block_size * (a.D / 2), groups = a.D / 16;
  const uint64_t block_bytes = (uint64_t)a.H * page_bytes;
  const T* kn = static_cast<const T*>(a.k_new) + (int64_t)b * a.sk[0] + (int64_t)t0 * a.sk[2];
  const T* vn = static_cast<const T*>(a.v_new) + (int64_t)b * a.sv[0] + (int64_t)t0 * a.sv[2];
  const int total = a.H << wpr_log2;
  for (int i0 = 0; i0 < total; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x;
    const bool in = i < total;
    const int h = in ? i >> wpr_log2 : 0, w = i & (wpr - 1);
    const T* ksrc = kn + (int64_t)h * a.sk[1] + (int64_t)(8 * w) * a.sk[3];
    const T* vsrc = vn + (int64_t)h * a.sv[1] + (int64_t)(8 * w) * a.sv[3];
    float xk[TOKENS][8], xv[TOKENS][8];
#pragma unroll
    for (int n = 0; n < TOKENS; ++n)
      if (blk[n] >= 0) {
        load8<T, VEC>(ksrc + n * a.sk[2], a.sk[3], xk[n]);
        load8<T, VEC>(vsrc + n * a.sv[2], a.sv[3], xv[n]);
      }
    char* kdst = static_cast<char*>(a.k_pool) + (int64_t)h * page_bytes;
    char* vdst = static_cast<char*>(a.v_pool) + (int64_t)h * page_bytes;
#pragma unroll
    for (int n = 0; n < TOKENS; ++n)
      if (blk[n] >= 0) {  // the same for the whole CTA
        uint32_t mk = max_abs_bits(xk[n]), mv = max_abs_bits(xv[n]);
        const uint32_t ok = __shfl_xor_sync(kFullMask, mk, 1), ov = __shfl_xor_sync(kFullMask, mv, 1);
        mk = mk > ok ? mk : ok;
        mv = mv > ov ? mv : ov;
        const uint32_t ck = kv4_scale_code(mk), cv = kv4_scale_code(mv);
        const uint32_t pk = kv4_pack8<T>(xk[n], kv4_scale(ck)), pv = kv4_pack8<T>(xv[n], kv4_scale(cv));
        if (in) {
          char* kh = kdst + blk[n] * block_bytes;
          char* vh = vdst + blk[n] * block_bytes;
          *reinterpret_cast<uint32_t*>(kh + row[n] * (a.D / 2) + 4 * w) = pk;
          *reinterpret_cast<uint32_t*>(vh + row[n] * (a.D / 2) + 4 * w) = pv;
          // lane pairs split the two scale bytes
          if ((w & 1) == 0)
            kh[codes + row[n] * groups + (w >> 1)] = (char)ck;
          else
            vh[codes + (w >> 1) * a.block_size + row[n]] = (char)cv;
        }
      }
  }
}

template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(128) kv4_read_kernel(Kv4ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int t0 = blockIdx.x * TOKENS, b = blockIdx.y;
  const int64_t start = a.start_pos[b];
  const int len = a.lengths[b];
  int32_t blk[TOKENS];
  int row[TOKENS];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    const int64_t pos = start + t0 + i, page = pos >> a.bs_log2;
    blk[i] = -1;
    row[i] = (int)(pos & (a.block_size - 1));
    if (t0 + i < len) {
      if (pos >= 0 && page < a.max_pages) blk[i] = a.page_table[(int64_t)b * a.pt_stride + page];
      if (blk[i] < 0 || blk[i] >= a.num_blocks) {
        blk[i] = -1;
        bad = true;
      }
    }
  }
  if (bad && threadIdx.x == 0) set_status(a.status, B2PA_ERR_BAD_BLOCK_ID);
  const int wpr = a.D / 8, wpr_log2 = 31 - __clz(wpr);
  const int page_bytes = kv4_page_bytes(a.block_size, a.D);
  const int codes = a.block_size * (a.D / 2), groups = a.D / 16;
  const uint64_t block_bytes = (uint64_t)a.H * page_bytes;
  T* ko = static_cast<T*>(a.k_out) + (int64_t)b * a.sk[0] + (int64_t)t0 * a.sk[2];
  T* vo = static_cast<T*>(a.v_out) + (int64_t)b * a.sv[0] + (int64_t)t0 * a.sv[2];
  for (int i = threadIdx.x; i < a.H << wpr_log2; i += blockDim.x) {
    const int h = i >> wpr_log2, w = i & (wpr - 1);
    const char* ksrc = static_cast<const char*>(a.k_pool) + (int64_t)h * page_bytes;
    const char* vsrc = static_cast<const char*>(a.v_pool) + (int64_t)h * page_bytes;
    uint32_t wk[TOKENS], wv[TOKENS], ck[TOKENS], cv[TOKENS];
#pragma unroll
    for (int n = 0; n < TOKENS; ++n) {
      wk[n] = wv[n] = 0x88888888u;  // zeros
      ck[n] = cv[n] = 0;
      if (blk[n] >= 0) {
        const char* kh = ksrc + blk[n] * block_bytes;
        const char* vh = vsrc + blk[n] * block_bytes;
        wk[n] = *reinterpret_cast<const uint32_t*>(kh + row[n] * (a.D / 2) + 4 * w);
        wv[n] = *reinterpret_cast<const uint32_t*>(vh + row[n] * (a.D / 2) + 4 * w);
        ck[n] = (uint8_t)kh[codes + row[n] * groups + (w >> 1)];
        cv[n] = (uint8_t)vh[codes + (w >> 1) * a.block_size + row[n]];
      }
    }
#pragma unroll
    for (int n = 0; n < TOKENS; ++n)
      if (t0 + n < a.T) {
        T* kd = ko + (int64_t)h * a.sk[1] + n * a.sk[2] + 8 * w;
        T* vd = vo + (int64_t)h * a.sv[1] + n * a.sv[2] + 8 * w;
        if constexpr (VEC) {
          kv4_store8(kd, wk[n], ck[n]);
          kv4_store8(vd, wv[n], cv[n]);
        } else {
          float x[8];
          kv4_unpack8(wk[n], kv4_scale(ck[n]), x);
          for (int c = 0; c < 8; ++c) kd[c] = from_f32<T>(x[c]);
          kv4_unpack8(wv[n], kv4_scale(cv[n]), x);
          for (int c = 0; c < 8; ++c) vd[c] = from_f32<T>(x[c]);
        }
      }
  }
}

static bool rows16(const void* p, const int64_t* s, int es) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[3] == 1;
  for (int i = 0; i < 3; ++i) ok = ok && (s[i] * es) % 16 == 0;
  return ok;
}

// Tokens per CTA: 4 once that still leaves several CTAs per SM.
static bool many_tokens(int B, int T) { return (int64_t)B * ((T + 3) / 4) >= 4 * (int64_t)device_sm_count(); }

template <typename T>
static int append_as(const AppendArgs& a, int64_t* seq_out, cudaStream_t s) {
  const bool vec = rows16(a.k_new, a.sk, sizeof(T)) && rows16(a.v_new, a.sv, sizeof(T));
  const dim3 one((unsigned)a.T, (unsigned)a.B), four((unsigned)((a.T + 3) / 4), (unsigned)a.B);
  cudaError_t e;
  if (!vec)
    e = launch_pdl(kv4_append_kernel<T, false, 1>, one, dim3(128), 0, s, a, seq_out);
  else if (!many_tokens(a.B, a.T))
    e = launch_pdl(kv4_append_kernel<T, true, 1>, one, dim3(128), 0, s, a, seq_out);
  else
    e = launch_pdl(kv4_append_kernel<T, true, 4>, four, dim3(128), 0, s, a, seq_out);
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
  const dim3 one((unsigned)a.T, (unsigned)a.B), four((unsigned)((a.T + 3) / 4), (unsigned)a.B);
  cudaError_t e;
  if (!vec)
    e = launch_pdl(kv4_read_kernel<T, false, 1>, one, dim3(128), 0, s, a);
  else if (!many_tokens(a.B, a.T))
    e = launch_pdl(kv4_read_kernel<T, true, 1>, one, dim3(128), 0, s, a);
  else
    e = launch_pdl(kv4_read_kernel<T, true, 4>, four, dim3(128), 0, s, a);
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
