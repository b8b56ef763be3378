// kv4_rows.cu -- rows into and out of the 4-bit paged pools (format: kv4.cuh).
//
//   kv4_append_kernel  quantises the new tokens' K and V rows into their
//                      pages, one CTA per (token, sequence);
//   kv4_read_kernel    reads rows back as the values they stand for.
//
// The bytes they move (D * element size in and 9/16 D out a row, or the
// reverse) bound them from below: for 6,260 rows of 32 heads of 128 in bf16, in
// 8 x 1,531 slots whose others are read back as zeros, 20 and 36 us at copy
// bandwidth; they take 26 and 42 (fp32 append: 60 for 36, with 17 divisions a
// group).  The append spends instructions, some 65 a word of 8 codes.  There a
// thread takes whole groups (16 channels) of K and of V, so a group's scale and
// reciprocal are worked out once; the group's maximum is taken on the bits of
// |x| (pairs of 16-bit values at a time), so a NaN or an infinity wins it.
// Prompts: a CTA takes two neighbouring tokens, all of whose loads are under way
// at once.
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace b2pa {

// One group of a row: 16-byte loads when VEC, else channel by channel with
// any stride.
template <typename T, bool VEC>
struct Group {
  uint4 raw[sizeof(T)];  // 16 channels as they lie in memory

  __device__ __forceinline__ void load(const T* p, int64_t sd) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) raw[i] = ld_global_nc<uint4>(p + i * (16 / (int)sizeof(T)));
    } else {
      T* x = reinterpret_cast<T*>(raw);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = p[i * sd];
    }
  }
  // Bits of the largest magnitude as fp32.
  __device__ __forceinline__ uint32_t max_bits() const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t u = w[i] & 0x7fffffffu;
        m = m > u ? m : u;
      }
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
      m = (m >> 16) > (m & 0xffffu) ? m >> 16 : m & 0xffffu;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return m << 16;
      return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));  // NaN and infinity stay so
    }
  }
  // Channels 8 * half .. 8 * half + 7.
  __device__ __forceinline__ void to_float(int half, float* x) const {
    constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      Vec<T, N> v;
      v.w = raw[half * (8 / N) + i];
      v.to_float(x + i * N);
    }
  }
};

// Block ids (-1: not there) and rows of the tokens t0 .. t0 + TOKENS - 1.
template <int TOKENS>
struct Places {
  int32_t blk[TOKENS];
  int row[TOKENS];
  __device__ __forceinline__ Places(const int32_t* table, int64_t start, int t0, int len, int bs_log2, int max_pages,
                                    int64_t num_blocks, int32_t* status) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
      const int64_t pos = start + t0 + i, page = pos >> bs_log2;
      blk[i] = -1;
      row[i] = (int)(pos & ((1 << bs_log2) - 1));
      if (t0 + i < len) {
        if (pos >= 0 && page < max_pages) blk[i] = table[page];
        if (blk[i] < 0 || blk[i] >= num_blocks) {
          blk[i] = -1;
          bad = true;
        }
      }
    }
    if (bad && threadIdx.x == 0) set_status(status, B2PA_ERR_BAD_BLOCK_ID);
  }
};

template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(128) kv4_append_kernel(AppendArgs a, int64_t* seq_out) {
  pdl_wait();
  pdl_launch_dependents();
  const int t0 = blockIdx.x * TOKENS, b = blockIdx.y;
  int len = a.lengths[b];
  len = len < a.T ? len : a.T;
  const int64_t start = a.start_pos[b];
  if (seq_out != nullptr && t0 == 0 && threadIdx.x == 0) seq_out[b] = start + (len > 0 ? len : 0);
  if (t0 >= len) return;
  const Places<TOKENS> at(a.page_table + (int64_t)b * a.pt_stride, start, t0, len, a.bs_log2, a.max_pages, a.num_blocks,
                          a.status);
  const int gpr_log2 = 31 - __clz(a.D / 16);  // groups per row: a power of two
  const int page_bytes = kv4_page_bytes(a.block_size, a.D);
  const int codes = a.block_size * (a.D / 2);
  const uint64_t block_bytes = (uint64_t)a.H * page_bytes;
  const T* kn = static_cast<const T*>(a.k_new) + (int64_t)b * a.sk[0] + (int64_t)t0 * a.sk[2];
  const T* vn = static_cast<const T*>(a.v_new) + (int64_t)b * a.sv[0] + (int64_t)t0 * a.sv[2];
  for (int i = threadIdx.x; i < a.H << gpr_log2; i += blockDim.x) {
    const int h = i >> gpr_log2, g = i & ((1 << gpr_log2) - 1);
    const T* ksrc = kn + (int64_t)h * a.sk[1] + (int64_t)(16 * g) * a.sk[3];
    const T* vsrc = vn + (int64_t)h * a.sv[1] + (int64_t)(16 * g) * a.sv[3];
    Group<T, VEC> k[TOKENS], v[TOKENS];
#pragma unroll
    for (int n = 0; n < TOKENS; ++n)
      if (at.blk[n] >= 0) {
        k[n].load(ksrc + n * a.sk[2], a.sk[3]);
        v[n].load(vsrc + n * a.sv[2], a.sv[3]);
      }
    char* kdst = static_cast<char*>(a.k_pool) + (int64_t)h * page_bytes;
    char* vdst = static_cast<char*>(a.v_pool) + (int64_t)h * page_bytes;
    auto quantise = [&](const Group<T, VEC>& x, uint32_t& code) {
      code = kv4_scale_code<T>(x.max_bits());
      const float s = kv4_scale(code);
      float f[8];
      uint2 w;
      x.to_float(0, f);
      w.x = kv4_pack8<T>(f, code, s);
      x.to_float(1, f);
      w.y = kv4_pack8<T>(f, code, s);
      return w;
    };
#pragma unroll
    for (int n = 0; n < TOKENS; ++n)
      if (at.blk[n] >= 0) {
        char* kh = kdst + at.blk[n] * block_bytes;
        char* vh = vdst + at.blk[n] * block_bytes;
        uint32_t code;
        *reinterpret_cast<uint2*>(kh + at.row[n] * (a.D / 2) + 8 * g) = quantise(k[n], code);
        kh[codes + at.row[n] * (a.D / 16) + g] = (char)code;
        *reinterpret_cast<uint2*>(vh + at.row[n] * (a.D / 2) + 8 * g) = quantise(v[n], code);
        vh[codes + g * a.block_size + at.row[n]] = (char)code;
      }
  }
}

template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(128) kv4_read_kernel(Kv4ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int t0 = blockIdx.x * TOKENS, b = blockIdx.y;
  int len = a.lengths[b];
  len = len < a.T ? len : a.T;
  const Places<TOKENS> at(a.page_table + (int64_t)b * a.pt_stride, a.start_pos[b], t0, len, a.bs_log2, a.max_pages,
                          a.num_blocks, a.status);
  // a thread reads one word of K and of V per token, so that a warp's stores
  // are contiguous (whole groups per thread: 61 us where this took 40)
  const int wpr_log2 = 31 - __clz(a.D / 8);
  const int page_bytes = kv4_page_bytes(a.block_size, a.D);
  const int codes = a.block_size * (a.D / 2);
  const uint64_t block_bytes = (uint64_t)a.H * page_bytes;
  T* ko = static_cast<T*>(a.k_out) + (int64_t)b * a.sk[0] + (int64_t)t0 * a.sk[2];
  T* vo = static_cast<T*>(a.v_out) + (int64_t)b * a.sv[0] + (int64_t)t0 * a.sv[2];
  for (int i = threadIdx.x; i < a.H << wpr_log2; i += blockDim.x) {
    const int h = i >> wpr_log2, w = i & ((1 << wpr_log2) - 1);
    const char* ksrc = static_cast<const char*>(a.k_pool) + (int64_t)h * page_bytes;
    const char* vsrc = static_cast<const char*>(a.v_pool) + (int64_t)h * page_bytes;
    uint32_t wk[TOKENS], wv[TOKENS], ck[TOKENS], cv[TOKENS];
#pragma unroll
    for (int n = 0; n < TOKENS; ++n) {
      wk[n] = wv[n] = 0x88888888u;  // zeros
      ck[n] = cv[n] = 0;
      if (at.blk[n] >= 0) {
        const char* kh = ksrc + at.blk[n] * block_bytes;
        const char* vh = vsrc + at.blk[n] * block_bytes;
        wk[n] = *reinterpret_cast<const uint32_t*>(kh + at.row[n] * (a.D / 2) + 4 * w);
        wv[n] = *reinterpret_cast<const uint32_t*>(vh + at.row[n] * (a.D / 2) + 4 * w);
        ck[n] = (uint8_t)kh[codes + at.row[n] * (a.D / 16) + (w >> 1)];
        cv[n] = (uint8_t)vh[codes + (w >> 1) * a.block_size + at.row[n]];
      }
    }
    auto put = [&](T* dst, uint32_t word, uint32_t code) {
      if constexpr (VEC) {
        kv4_store8(dst, word, code);
      } else {
        float x[8];
        kv4_unpack8(word, kv4_scale(code), x);
        for (int c = 0; c < 8; ++c) dst[c] = from_f32<T>(x[c]);
      }
    };
#pragma unroll
    for (int n = 0; n < TOKENS; ++n)
      if (t0 + n < a.T) {
        put(ko + (int64_t)h * a.sk[1] + n * a.sk[2] + 8 * w, wk[n], ck[n]);
        put(vo + (int64_t)h * a.sv[1] + n * a.sv[2] + 8 * w, wv[n], cv[n]);
      }
  }
}

static bool rows16(const void* p, const int64_t* s, int es) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[3] == 1;
  for (int i = 0; i < 3; ++i) ok = ok && (s[i] * es) % 16 == 0;
  return ok;
}

// Several tokens per CTA once that still leaves several CTAs per SM.
static bool many_tokens(int B, int T) { return (int64_t)B * ((T + 1) / 2) >= 4 * (int64_t)device_sm_count(); }

template <typename T>
static int append_as(const AppendArgs& a, int64_t* seq_out, cudaStream_t s) {
  const bool vec = rows16(a.k_new, a.sk, sizeof(T)) && rows16(a.v_new, a.sv, sizeof(T));
  // (no tokens: the lengths are still written)
  const dim3 one((unsigned)(a.T > 0 ? a.T : 1), (unsigned)a.B), two((unsigned)((a.T + 1) / 2), (unsigned)a.B);
  cudaError_t e;
  if (!vec)
    e = launch_pdl(kv4_append_kernel<T, false, 1>, one, dim3(128), 0, s, a, seq_out);
  else if (!many_tokens(a.B, a.T))
    e = launch_pdl(kv4_append_kernel<T, true, 1>, one, dim3(128), 0, s, a, seq_out);
  else
    e = launch_pdl(kv4_append_kernel<T, true, 2>, two, dim3(128), 0, s, a, seq_out);
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
  const dim3 one((unsigned)a.T, (unsigned)a.B), two((unsigned)((a.T + 1) / 2), (unsigned)a.B);
  cudaError_t e;
  if (!vec)
    e = launch_pdl(kv4_read_kernel<T, false, 1>, one, dim3(128), 0, s, a);
  else if (!many_tokens(a.B, a.T))
    e = launch_pdl(kv4_read_kernel<T, true, 1>, one, dim3(128), 0, s, a);
  else
    e = launch_pdl(kv4_read_kernel<T, true, 2>, two, dim3(128), 0, s, a);
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
