// mx4_few.hip -- 4-bit products for a handful of rows per expert (serving single tokens), one launch.
//
// Every weight is read once and multiplied with at most 16 rows, so the product is bound by the weights' bytes or, at the sizes
// of a detector's FFN, by latency: no LDS staging, no separate quantisation pass.  A workgroup owns 16 output columns x 16 rows;
// its four waves take every fourth step of 128 elements.  A lane loads 16 bytes of a weight row straight into the register
// operand of the matrix instruction, loads the 32 elements of x that meet them and quantises them in place: the 32 elements of
// a lane ARE one block, so its maximum needs no other lane.  The waves' fp32 sums are added in LDS in a fixed order.
// Measured (one token, 4096 x 1024, bf16, GELU): 4.3 us against 1.9 us quantise + 7.6 us tile kernel.  With more tiles its time is the
// rows' quantisation, once per 16 columns (which sizes come here: mx4_gemm.hip).
#include "expert_plan.h"
#include "mx4_few.h"

namespace {
using namespace sm3x;

template <int TYPE> struct Elem;
template <> struct Elem<DT_F32> { typedef float T; };
template <> struct Elem<DT_F16> { typedef _Float16 T; };
template <> struct Elem<DT_BF16> { typedef __bf16 T; };

// rows [row0, row0 + rows) of expert g that row tile `tile` of 16 covers (g = -1: rows of no expert, -2: nothing); the experts'
// ranges are clamped to [0, S] and made monotone
__device__ __forceinline__ void find_rows(const int* offsets, int G, int S, int tile, int& g, int& row0, int& rows) {
  constexpr int BM = 16;
  g = -2;
  row0 = rows = 0;
  int last = S;
  if (offsets == nullptr) {
    g = 0;
    row0 = tile * BM;
  } else {
    const int lane = threadIdx.x & 63;
    int first = offsets[0];
    first = first < 0 ? 0 : first > S ? S : first;
    int carry = first, before = 0;
    last = 0;
    for (int base = 0; base < G; base += 64) {
      const int e = base + lane;
      int end = e < G ? offsets[e + 1] : 0;
      end = end < 0 ? 0 : end > S ? S : end;
      end = end < carry ? carry : end;
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(end, d);
        if (lane >= d && o > end) end = o;
      }
      int start = __shfl_up(end, 1);
      if (lane == 0) start = carry;
      const int n = e < G ? (end - start + BM - 1) / BM : 0;
      int incl = n;
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
      }
      const unsigned long long hit = __ballot(tile - before < incl);
      if (hit) {
        const int l = __ffsll(hit) - 1;
        g = base + l;
        row0 = __shfl(start, l) + (tile - before - __shfl(incl - n, l)) * BM;
        last = __shfl(end, l);
        break;
      }
      before += __shfl(incl, 63);
      carry = __shfl(end, 63);
    }
    if (g == -2) {  // behind the last expert, then before the first
      const int i = tile - before, behind = (S - carry + BM - 1) / BM;
      if (i < behind) {
        g = -1;
        row0 = carry + i * BM;
        last = S;
      } else if ((i - behind) * BM < first) {
        g = -1;
        row0 = (i - behind) * BM;
        last = first;
      }
    }
  }
  rows = last - row0 < BM ? last - row0 : BM;
  if (rows <= 0) g = -2;
  g = __builtin_amdgcn_readfirstlane(g);
  row0 = __builtin_amdgcn_readfirstlane(row0);
  rows = __builtin_amdgcn_readfirstlane(rows);
}

// 32 elements -> their codes and scale byte (the rules of sm3_mx4_quantize)
template <int TYPE>
__device__ __forceinline__ v4i quantize_block(const typename Elem<TYPE>::T (&x)[32], int& byte) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 32; j++) {
    const unsigned b = __float_as_uint((float)x[j]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  const bool bad = m >= 0x7f800000u;
  byte = (int)(m >> 23) - 2;
  byte = byte < 0 ? 0 : byte;
  const float s = __uint_as_float(byte > 0 ? (unsigned)byte << 23 : 0x00400000u);
  v4i codes;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    unsigned u = 0;
    if constexpr (TYPE == DT_F32) {
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[8 * w], x[8 * w + 1], s, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[8 * w + 2], x[8 * w + 3], s, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[8 * w + 4], x[8 * w + 5], s, 2);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[8 * w + 6], x[8 * w + 7], s, 3);
    } else if constexpr (TYPE == DT_F16) {
      const v2h* p = (const v2h*)(x + 8 * w);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[0], s, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[1], s, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[2], s, 2);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(u, p[3], s, 3);
    } else {
      const v2b* p = (const v2b*)(x + 8 * w);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[0], s, 0);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[1], s, 1);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[2], s, 2);
      u = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(u, p[3], s, 3);
    }
    codes[w] = bad ? 0 : (int)u;
  }
  if (bad) byte = 255;
  return codes;
}

template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) few_kernel(const sm3x::Few P) {
  typedef typename Elem<TYPE>::T T;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, g4 = lane >> 4;
  const int col0 = blockIdx.x * 16;
  int g, row0, rows;
  find_rows(P.offsets, P.G, P.S, blockIdx.y, g, row0, rows);
  if (g == -2) return;
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  if (g >= 0) {
    const int steps = P.kp / 128, col = col0 + r16;
    const bool real = r16 < rows, wreal = col < P.cols;
    // (lanes without a column or a row read what the last one reads; their products are stored by nobody)
    const long wrow = (long)g * P.cols + (wreal ? col : P.cols - 1);
    const unsigned char* w = P.codes + wrow * (P.kp / 2) + g4 * 16;
    const unsigned char* ws = P.scales + wrow * (P.kp / 32) + g4;
    const T* x = (const T*)P.x + (long)(row0 + (real ? r16 : rows - 1)) * P.ldx;
    for (int s0 = wave; s0 < steps; s0 += 8) {  // two of this wave's steps at once: their loads are in flight together
      v4i q[2];
      int qs[2];
      T v[2][32];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int s = s0 + 4 * h < steps ? s0 + 4 * h : s0;
        q[h] = *(const v4i*)(w + (long)s * 64);
        qs[h] = ws[s * 4];
        const int c = s * 128 + g4 * 32;
        if (VEC) {
          constexpr int W = 16 / sizeof(T);
#pragma unroll
          for (int j = 0; j < 32; j += W) {
            if (c + j < P.k) *(v4i*)(v[h] + j) = *(const v4i*)(x + c + j);
            else *(v4i*)(v[h] + j) = v4i{0, 0, 0, 0};
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j++) v[h][j] = c + j < P.k ? x[c + j] : (T)0.f;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; h++) {
        if (s0 + 4 * h < steps) {
          int byte;
          const v4i p = quantize_block<TYPE>(v[h], byte);
          acc = mma<K_MX4>(q[h], p, acc, qs[h], byte, 0);
        }
      }
    }
  }
  __shared__ v4f part[4][64];
  part[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int z = 1; z < 4; z++) acc += part[z][lane];
  const int n = col0 + 4 * g4, have = P.cols - n;
  if (r16 >= rows || have <= 0) return;
  float v[8] = {acc[0], acc[1], acc[2], acc[3], 0.f, 0.f, 0.f, 0.f};
  if (g >= 0) {
    if (P.bias) {
      float b[8];
      bias8(b, P.bias, P.bias_type, (long)g * P.cols + n, (long)g * P.cols + P.cols - 1);
#pragma unroll
      for (int r = 0; r < 4; r++) v[r] += b[r];
    }
    if (P.act) gelu8(v);
  }
  store8(P.out, P.out_type, (long)(row0 + r16) * P.cols + n, v, have < 4 ? have : 4, false);
}

}  // namespace

namespace sm3x {

int launch_few(const Few& P, int type, long row_tiles, hipStream_t st) {
  const int es = type == DT_F32 ? 4 : 2;
  const bool vec = (uintptr_t)P.x % 16 == 0 && P.ldx * es % 16 == 0 && P.k * es % 16 == 0;
  const dim3 grid((unsigned)((P.cols + 15) / 16), (unsigned)row_tiles);
#define SM3_FEW(T) (vec ? few_kernel<T, true><<<grid, 256, 0, st>>>(P) : few_kernel<T, false><<<grid, 256, 0, st>>>(P))
  if (type == DT_F32) SM3_FEW(DT_F32);
  else if (type == DT_F16) SM3_FEW(DT_F16);
  else SM3_FEW(DT_BF16);
#undef SM3_FEW
  return launch_status();
}

}  // namespace sm3x
