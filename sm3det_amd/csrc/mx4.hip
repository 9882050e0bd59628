// mx4.hip -- microscaled 4-bit rows (MXFP4): quantisation and its inverse.
//
// Block of 32 elements x_i of a row: E = max(floor(log2 max|x_i|) - 2, -127), code_i = rne_e2m1(x_i / 2^E), saturating at 6.
// floor(log2) is the exponent field of the largest magnitude (subnormal maxima have field 0 and land on the clamp), the
// rounding is v_cvt_scalef32_pk_fp4_* (nearest even, saturating; exact for every power-of-two scale down to the subnormal
// 2^-127).  One thread takes 8 consecutive elements: a 16-byte load (two for fp32), the block's maximum over 4 lanes by two
// cross-lane steps, a 4-byte store.  Bound by HBM: 131072 x 384 fp16 in 26 us (4.9 TB/s read and written; a copy reaches 5.1) and back
// in 18 us (the codes come from the last-level cache).
#include "common.h"

namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float scale_of(int byte) {  // 2^(byte - 127)
  return __uint_as_float(byte > 0 ? (unsigned)byte << 23 : 0x00400000u);
}

template <int TYPE> struct Elem;
template <> struct Elem<SM3_DT_F32> { typedef float T; };
template <> struct Elem<SM3_DT_F16> { typedef _Float16 T; };
template <> struct Elem<SM3_DT_BF16> { typedef __bf16 T; };

// VEC: rows start at 16-byte addresses and k % 8 == 0
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) quantize_kernel(const void* __restrict__ x_, long rows, int k, long ld,
                                                       unsigned* __restrict__ codes, unsigned char* __restrict__ scales,
                                                       unsigned octets, long total) {
  typedef typename Elem<TYPE>::T T;
  const T* x = (const T*)x_;
  // the loop's trip count is uniform over groups of 4 lanes (octets % 16 == 0): their cross-lane steps see each other
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long row = total < (1L << 31) ? (long)((unsigned)i / octets) : i / octets;
    const int o = (int)(i - row * octets), c = o * 8;
    T v[8];
    const T* at = x + row * ld + c;
    if (VEC) {
      if (c < k) {
        constexpr int W = sizeof(T) * 8 / 16;
#pragma unroll
        for (int w = 0; w < W; w++) ((v4u*)v)[w] = __builtin_nontemporal_load((const v4u*)at + w);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (T)0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = c + j < k ? at[j] : (T)0.f;
    }
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const unsigned b = __float_as_uint((float)v[j]) & 0x7fffffffu;  // monotone in |x|; infinities and NaNs on top
      m = b > m ? b : m;
    }
    unsigned t = __shfl_xor(m, 1);
    m = t > m ? t : m;
    t = __shfl_xor(m, 2);
    m = t > m ? t : m;
    const bool bad = m >= 0x7f800000u;
    int byte = (int)(m >> 23) - 2;
    byte = byte < 0 ? 0 : byte;
    const float s = scale_of(byte);
    unsigned u = 0;
    if constexpr (TYPE == SM3_DT_F32) {
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[0], v[1], s, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2], v[3], s, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4], v[5], s, 2);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6], v[7], s, 3);
    } else if constexpr (TYPE == SM3_DT_F16) {
      const v2h* p = (const v2h*)v;
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[0], s, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[1], s, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[2], s, 2);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[3], s, 3);
    } else {
      const v2b* p = (const v2b*)v;
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[0], s, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[1], s, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[2], s, 2);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[3], s, 3);
    }
    codes[i] = bad ? 0u : u;
    if ((o & 3) == 0) scales[i >> 2] = (unsigned char)(bad ? 255 : byte);
  }
}

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const unsigned* __restrict__ codes,
                                                         const unsigned char* __restrict__ scales, int k,
                                                         void* __restrict__ y_, unsigned octets, long total) {
  typedef typename Elem<TYPE>::T T;
  T* y = (T*)y_;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long row = total < (1L << 31) ? (long)((unsigned)i / octets) : i / octets;
    const int c = (int)(i - row * octets) * 8;
    if (c >= k) continue;
    const unsigned u = codes[i];
    const int byte = scales[i >> 2];
    const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : scale_of(byte);
    T v[8];
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 1);
    const v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(u, 1.0f, 3);
    const float f[8] = {a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (T)(f[j] * s);
    T* at = y + row * k + c;
    if (VEC) {
      constexpr int W = sizeof(T) * 8 / 16;
#pragma unroll
      for (int w = 0; w < W; w++) __builtin_nontemporal_store(((const v4u*)v)[w], (v4u*)at + w);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) { if (c + j < k) at[j] = v[j]; }
    }
  }
}

constexpr int kMaxRow = 0x7fffff80;  // (padded, its elements are counted in 31 bits)

inline unsigned blocks_for(long total) {
  const long b = (total + 255) / 256;
  return (unsigned)(b > 16384 ? 16384 : b);
}

}  // namespace

extern "C" {

int sm3_mx4_quantize(const void* x, int type, long rows, int k, long ld, uint8_t* codes, uint8_t* scales,
                     sm3_stream_t stream) {
  if (rows < 0 || k < 1 || ld < k || type < 0 || type > SM3_DT_BF16) return SM3_ERR_INVALID_ARG;
  if (k > kMaxRow) return SM3_ERR_UNSUPPORTED;
  if (rows == 0) return SM3_OK;
  if (!x || !codes || !scales || ((uintptr_t)codes & 3)) return SM3_ERR_INVALID_ARG;
  const unsigned octets = (unsigned)((k + 127) / 128 * 16);
  const long total = rows * octets;
  const int es = type == SM3_DT_F32 ? 4 : 2;
  const bool vec = k % 8 == 0 && ld * es % 16 == 0 && (uintptr_t)x % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
#define SM3_Q(T) \
  (vec ? quantize_kernel<T, true><<<blocks_for(total), 256, 0, st>>>(x, rows, k, ld, (unsigned*)codes, scales, octets, total) \
       : quantize_kernel<T, false><<<blocks_for(total), 256, 0, st>>>(x, rows, k, ld, (unsigned*)codes, scales, octets, total))
  if (type == SM3_DT_F32) SM3_Q(SM3_DT_F32);
  else if (type == SM3_DT_F16) SM3_Q(SM3_DT_F16);
  else SM3_Q(SM3_DT_BF16);
#undef SM3_Q
  return launch_status();
}

int sm3_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, long rows, int k, void* y, int type,
                       sm3_stream_t stream) {
  if (rows < 0 || k < 1 || type < 0 || type > SM3_DT_BF16) return SM3_ERR_INVALID_ARG;
  if (k > kMaxRow) return SM3_ERR_UNSUPPORTED;
  if (rows == 0) return SM3_OK;
  if (!y || !codes || !scales || ((uintptr_t)codes & 3)) return SM3_ERR_INVALID_ARG;
  const unsigned octets = (unsigned)((k + 127) / 128 * 16);
  const long total = rows * octets;
  const bool vec = k % 8 == 0 && (uintptr_t)y % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
#define SM3_D(T) \
  (vec ? dequantize_kernel<T, true><<<blocks_for(total), 256, 0, st>>>((const unsigned*)codes, scales, k, y, octets, total) \
       : dequantize_kernel<T, false><<<blocks_for(total), 256, 0, st>>>((const unsigned*)codes, scales, k, y, octets, total))
  if (type == SM3_DT_F32) SM3_D(SM3_DT_F32);
  else if (type == SM3_DT_F16) SM3_D(SM3_DT_F16);
  else SM3_D(SM3_DT_BF16);
#undef SM3_D
  return launch_status();
}

}  // extern "C"
