// expert_tile.h -- the tile engine of the products grouped by expert: C = P . Q^T per expert, 16-bit or microscaled 4-bit
// operands, fp32 accumulation on the matrix cores.
//
// One step of a tile consumes 128 BYTES of the reduction of every operand row: 64 16-bit elements or 256 4-bit ones.  Both
// are two rounds of the 16x16 matrix instruction with 16 bytes per lane and operand (v_mfma_f32_16x16x32_{f16,bf16},
// v_mfma_scale_f32_16x16x128_f8f6f4), so one loader, one LDS layout and one loop serve all types.
//   * Global memory -> LDS directly (buffer_load_dwordx4 ... lds: no VGPRs, asynchronous); the buffer descriptor's range check
//     returns zeros for rows behind the expert's last and for the reduction's tail.
//   * LDS holds 16-byte granules.  The DMA writes lane-linearly, so the bank swizzle is applied to the SOURCE address.
//       row operands      [row][8 granules], granule g at position g ^ (row & 7)
//       column operands   [64 reduction rows][cols / 8 granules], granule g at g ^ swz(row); fragments come out of
//                         ds_read_b64_tr_b16 (lane i of 16 receives column i of a 4 x 16 block)
//   * The order of the reduction inside an instruction is free as long as both operands agree.
// Q rides in the instruction's first operand: a lane then owns four CONSECUTIVE output columns of one output row.
#pragma once
#include "common.h"

namespace sm3x {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

enum { DT_F32 = SM3_DT_F32, DT_F16 = SM3_DT_F16, DT_BF16 = SM3_DT_BF16 };
enum { K_F16 = 0, K_BF16 = 1, K_MX4 = 2 };   // operand kinds
enum { M_NT = 0, M_NN = 1, M_TN = 2 };       // P, Q: row|row, row|column, column|column operands

constexpr int kStepBytes = 128;   // reduction bytes of a row operand per step
constexpr int kStepRed = 64;      // reduction rows of a column operand per step (16-bit types)
constexpr unsigned kOutOfRange = 0x80000000u;  // a byte offset no descriptor covers: the load returns zeros

struct Params {
  const char* p;                  // NT / NN: (S, red) activation rows.  TN: (S, rows_out) -- the gradient
  const char* q;                  // NT: (G, cols, red) weights.  NN: (G, red, cols).  TN: (S, cols) -- the activations
  long ldp, ldq, strideq;         // bytes between rows; bytes between experts' weights
  const unsigned char* ps;        // MX4: scale bytes of p and q, pitches in bytes
  const unsigned char* qs;
  long ldps, ldqs, strideqs;
  long red;                       // NT / NN: reduction length in BYTES of a p row (whole 16-byte granules)
  long qred;                      // NN: rows of one expert's weights (the reduction length itself)
  void* out;                      // NT / NN: (S, cols).  TN: (G, rows_out, cols)
  int rows_out, cols;             // TN: output rows of one expert; output columns
  int out_type, bias_type, act, vec;
  const void* bias;               // (G, cols) or null
  float* bsum;                    // TN: per work unit column sums of p (units, rows_out) fp32, or null
  const int* offsets;             // (G + 1) device, or null: one group of all S rows
  int G;
  long S;
  int ntiles;                     // column tiles
  long mtiles;                    // row tiles the grid provides for (an upper bound where the groups are ragged)
  int splits;                     // NT / NN: slices of the reduction; > 1: fp32 partials (splits, S, cols) in `part`
  long unit_rows;                 // TN: reduction rows per work unit
  float* part;                    // fp32 partials, or null: the result goes straight to `out`
};

// ---- which rows a tile covers -------------------------------------------------------------------------------------
// The experts' row ranges are read from the device offsets: clamped to [0, S] and made monotone (running maximum), so that no
// content of the array can lead an access out of range.  Tiles are numbered expert by expert; behind them come the rows that
// belong to no expert (before the first, behind the last), whose outputs are zero.
struct RowTile {
  int g;           // expert, -1: rows of no expert, -2: nothing to do
  long row0;
  int rows;
  int part_of_g;   // index of this tile within its expert
};

template <bool KEEP_EMPTY>  // KEEP_EMPTY: an expert without rows still gets one unit (its gradient is zero)
__device__ __forceinline__ RowTile find_rows(const Params& P, long tile, int bm) {
  RowTile t{-2, 0, 0, 0};
  if (P.offsets == nullptr) {
    const long r0 = tile * bm;
    if (r0 < P.S || (KEEP_EMPTY && tile == 0)) {
      t.g = 0;
      t.row0 = r0;
      t.rows = (int)((P.S - r0 < bm) ? P.S - r0 : bm);
      t.part_of_g = (int)tile;
    }
    return t;
  }
  const int lane = threadIdx.x & 63;
  const int S = (int)P.S;
  int first = P.offsets[0];
  first = first < 0 ? 0 : first > S ? S : first;
  int carry_end = first;
  long carry_tiles = 0;
  for (int base = 0; base < P.G; base += 64) {
    const int g = base + lane;
    int end = g < P.G ? P.offsets[g + 1] : 0;
    end = end < 0 ? 0 : end > S ? S : end;
    end = end < carry_end ? carry_end : end;
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(end, d);
      if (lane >= d && o > end) end = o;
    }
    int start = __shfl_up(end, 1);
    if (lane == 0) start = carry_end;
    const int len = end - start;
    int n = g < P.G ? (len + bm - 1) / bm : 0;
    if (KEEP_EMPTY && g < P.G && n == 0) n = 1;
    int incl = n;
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(incl, d);
      if (lane >= d) incl += o;
    }
    const unsigned long long hit = __ballot(tile - carry_tiles < incl);
    if (hit) {
      const int l = __ffsll(hit) - 1;
      const int before = __shfl(incl - n, l);
      const int s0 = __shfl(start, l), e0 = __shfl(end, l);
      const int idx = (int)(tile - carry_tiles) - before;
      t.g = base + l;
      t.part_of_g = idx;
      t.row0 = (long)s0 + (long)idx * bm;
      const long left = e0 - t.row0;
      t.rows = (int)(left < bm ? (left < 0 ? 0 : left) : bm);
      break;
    }
    carry_tiles += __shfl(incl, 63);
    carry_end = __shfl(end, 63);
  }
  if (t.g == -2 && !KEEP_EMPTY) {  // rows of no expert
    long i = tile - carry_tiles;
    const long behind = ((long)S - carry_end + bm - 1) / bm;
    long r0 = -1, r1 = 0;
    if (i < behind) {
      r0 = carry_end + i * bm;
      r1 = S;
    } else if ((i - behind) * bm < first) {
      r0 = (i - behind) * bm;
      r1 = first;
    }
    if (r0 >= 0) {
      t.g = -1;
      t.row0 = r0;
      t.rows = (int)(r1 - r0 < bm ? r1 - r0 : bm);
    }
  }
  t.g = __builtin_amdgcn_readfirstlane(t.g);
  t.row0 = (long)__builtin_amdgcn_readfirstlane((int)t.row0);
  t.rows = __builtin_amdgcn_readfirstlane(t.rows);
  t.part_of_g = __builtin_amdgcn_readfirstlane(t.part_of_g);
  return t;
}

// ---- global -> LDS ------------------------------------------------------------------------------------------------
__device__ __forceinline__ v4i descriptor(const void* base, long bytes) {
  const unsigned long long a = (unsigned long long)base;
  v4i r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : bytes));
  r[3] = 0x00027000;
  return r;
}

// 64 lanes x 16 (4) bytes from base + voff to LDS byte address `lds` + lane * 16 (4).  No result register; the caller waits
// with wait_and_sync() before anything reads the LDS bytes.
__device__ __forceinline__ void dma16(unsigned lds, unsigned voff, v4i desc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(voff), "s"(desc) : "memory", "m0");
}
__device__ __forceinline__ void dma4(unsigned lds, unsigned voff, v4i desc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(voff), "s"(desc) : "memory", "m0");
}
// this wave's direct loads have landed; after the barrier everybody's have
__device__ __forceinline__ void wait_and_sync() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// swizzle of a column operand's row: spreads the 4 rows x 32 bytes that 16 lanes of a transposing read touch over the banks
__device__ __forceinline__ int col_swz(int row, int granules) {
  return (2 * ((row & 3) | ((row >> 1) & 4))) & (granules - 1);
}

// One operand tile of BX rows (row operand) or BX columns (column operand): 128 * BX bytes of LDS per step, loaded by
// `waves` waves with BX / 8 / waves instructions each.
template <int BX, bool COL, int WAVES>
struct Loader {
  static constexpr int N = BX / 8 / WAVES;
  static_assert(BX / 8 % WAVES == 0 && N >= 1, "every wave loads the same number of 1 KB pieces");
  unsigned voff[N];
  int gran;  // row operand: this lane's granule of the step (loop tail)

  __device__ __forceinline__ void init(int wave, int lane, long ld) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int piece = wave * N + i;
      if constexpr (!COL) {
        const int row = piece * 8 + (lane >> 3);
        gran = (lane & 7) ^ (lane >> 3);
        voff[i] = (unsigned)(row * ld) + gran * 16;
      } else {
        constexpr int GR = BX / 8, RP = 64 / GR;  // granules per row, rows per piece
        const int row = piece * RP + lane / GR;
        voff[i] = (unsigned)(row * ld) + (((lane % GR) ^ col_swz(row, GR)) * 16);
      }
    }
  }
  // left: bytes (row operand) of the reduction that remain from this step on
  __device__ __forceinline__ void load(unsigned lds, int wave, const char* base, long bytes, long left) const {
    const v4i d = descriptor(base, bytes);
    const unsigned cut = (!COL && gran * 16 >= left) ? kOutOfRange : 0u;
#pragma unroll
    for (int i = 0; i < N; i++) dma16(lds + (wave * N + i) * 1024, voff[i] | cut, d);
  }
};

// ---- fragments ----------------------------------------------------------------------------------------------------
// row operand, 16 rows from `row16`, round s (0, 1) of a step
template <int KIND>
__device__ __forceinline__ v4i frag_row(const char* tile, int row16, int s, int lane) {
  const int r = row16 + (lane & 15), g = KIND == K_MX4 ? 2 * (lane >> 4) + s : 4 * s + (lane >> 4);
  return *(const v4i*)(tile + r * 128 + ((g ^ (r & 7)) * 16));
}
// column operand, 16 columns from `col16` of a tile BX columns wide, round s: 8 of the 32 reduction rows per lane
template <int BX>
__device__ __forceinline__ v4i frag_col(const char* tile, int col16, int s, int lane) {
  constexpr int GR = BX / 8;
  const int j = lane & 15, r0 = 32 * s + 8 * (lane >> 4) + (j >> 2);
  const int g = col16 / 8 + ((j & 3) >> 1);
  typedef __attribute__((address_space(3))) v4s lv4s;
  union { v4s h[2]; v4i w; } u;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = r0 + 4 * h;
    const char* a = tile + r * (BX * 2) + ((g ^ col_swz(r, GR)) * 16) + (j & 1) * 8;
    u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s*)a);
  }
  return u.w;
}

template <int KIND>
__device__ __forceinline__ v4f mma(v4i q, v4i p, v4f c, int qscale, int pscale, int s) {
  if constexpr (KIND == K_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, q), __builtin_bit_cast(v8h, p), c, 0, 0, 0);
  else if constexpr (KIND == K_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, q), __builtin_bit_cast(v8b, p), c, 0, 0, 0);
  else {
    v8i a = __builtin_shufflevector(q, q, 0, 1, 2, 3, -1, -1, -1, -1);
    v8i b = __builtin_shufflevector(p, p, 0, 1, 2, 3, -1, -1, -1, -1);
    // the scale operands hold this lane's two blocks of the step in bytes 0 and 1: `s` picks one
    return s == 0 ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 0, qscale, 0, pscale)
                  : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, 1, qscale, 1, pscale);
  }
}

// ---- epilogue -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ float gelu(float h) {  // h * Phi(h), erfc by Abramowitz & Stegun 7.1.26 (|error| <= 1.5e-7)
  const float e = __expf(-0.5f * h * h);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752440f, fabsf(h), 1.0f));
  float q = fmaf(1.061405429f, t, -1.453152027f);
  q = fmaf(q, t, 1.421413741f);
  q = fmaf(q, t, -0.284496736f);
  q = fmaf(q, t, 0.254829592f);
  const float tail = 0.5f * q * t * e;  // Phi(-|h|)
  return h * (h >= 0.f ? 1.0f - tail : tail);
}

__device__ __forceinline__ float load_bias(const void* b, int type, long i) {
  if (type == DT_F32) return ((const float*)b)[i];
  if (type == DT_F16) return (float)((const _Float16*)b)[i];
  return (float)((const __bf16*)b)[i];
}

// four consecutive columns of one row; n: how many of them exist
__device__ __forceinline__ void store4(void* out, int type, long at, v4f v, int n, bool vec) {
  if (type == DT_F32) {
    float* o = (float*)out + at;
    if (vec && n == 4) *(v4f*)o = v;
    else
      for (int r = 0; r < 4; r++) { if (r < n) o[r] = v[r]; }
  } else if (type == DT_F16) {
    typedef _Float16 v4h __attribute__((ext_vector_type(4)));
    _Float16* o = (_Float16*)out + at;
    const v4h h = __builtin_convertvector(v, v4h);
    if (vec && n == 4) *(v4h*)o = h;
    else
      for (int r = 0; r < 4; r++) { if (r < n) o[r] = h[r]; }
  } else {
    typedef __bf16 v4b __attribute__((ext_vector_type(4)));
    __bf16* o = (__bf16*)out + at;
    const v4b h = __builtin_convertvector(v, v4b);
    if (vec && n == 4) *(v4b*)o = h;
    else
      for (int r = 0; r < 4; r++) { if (r < n) o[r] = h[r]; }
  }
}

// ---- the kernel ---------------------------------------------------------------------------------------------------
// BM output rows (P) x BN output columns (Q); WM x WN waves.
template <int KIND, int MODE, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * 64) tile_kernel(const Params P) {
  constexpr int WAVES = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr bool PCOL = MODE == M_TN, QCOL = MODE != M_NT;
  static_assert(KIND != K_MX4 || MODE == M_NT, "4-bit operands: rows only");
  constexpr int kTile = (BM + BN) * kStepBytes;
  constexpr int kScales = KIND == K_MX4 ? (BM + BN) * 8 : 0;
  __shared__ __attribute__((aligned(1024))) char lds[2][kTile + kScales];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;

  // tile of this workgroup: consecutive tiles on one XCD (they share weights in its L2), bands of 4 row tiles
  const long total = P.mtiles * P.ntiles;
  const long per = (total + kNumXCD - 1) / kNumXCD;
  const long lin = (long)(blockIdx.x % kNumXCD) * per + blockIdx.x / kNumXCD;
  if (lin >= total || (long)(blockIdx.x / kNumXCD) >= per) return;
  const long band = lin / (4L * P.ntiles), in = lin % (4L * P.ntiles);
  const long left = P.mtiles - band * 4;
  const int deep = left < 4 ? (int)left : 4;
  const int nt = (int)(in / deep);
  const long mt = band * 4 + in % deep;

  long red_steps, row0 = 0, prow0 = 0;
  int rows, g, mtile = 0;
  RowTile t;
  if constexpr (MODE == M_TN) {
    const int mt_per_unit = (P.rows_out + BM - 1) / BM;
    t = find_rows<true>(P, mt / mt_per_unit, (int)P.unit_rows);
    if (t.g < 0) return;
    g = t.g;
    mtile = (int)(mt % mt_per_unit);
    prow0 = (long)mtile * BM;
    rows = t.rows;                      // reduction rows
    red_steps = (rows + kStepRed - 1) / kStepRed;
  } else {
    t = find_rows<false>(P, mt, BM);
    if (t.g == -2) return;
    g = t.g;
    row0 = t.row0;
    rows = t.rows;
    red_steps = g < 0 ? 0 : (P.red + kStepBytes - 1) / kStepBytes;
  }
  const long col0 = (long)nt * BN;

  // this slice of the reduction
  long step0 = 0, step1 = red_steps;
  if (MODE != M_TN && P.splits > 1) {
    const long each = (red_steps + P.splits - 1) / P.splits;
    step0 = blockIdx.y * each;
    step1 = step0 + each < red_steps ? step0 + each : red_steps;
    if (step0 > step1) step0 = step1;
  }

  Loader<BM, PCOL, WAVES> lp;
  Loader<BN, QCOL, WAVES> lq;
  lp.init(wave, lane, P.ldp);
  lq.init(wave, lane, P.ldq);
  const unsigned base = __builtin_amdgcn_readfirstlane((int)lds_address(&lds[0][0]));

  const int qrows = (int)(P.cols - col0 < BN ? P.cols - col0 : BN);
  auto load_step = [&](long it, int buf) {
    const unsigned at = base + buf * (kTile + kScales);
    if constexpr (!PCOL) {
      const long k = it * kStepBytes;
      lp.load(at, wave, P.p + row0 * P.ldp + k, (long)(rows - 1) * P.ldp + P.red - k, P.red - k);
    } else {
      const long r = it * kStepRed, n = rows - r < kStepRed ? rows - r : kStepRed;
      const long wide = ((long)P.rows_out * 2 + 15) & ~15L;
      lp.load(at, wave, P.p + (t.row0 + r) * P.ldp + prow0 * 2, (n - 1) * P.ldp + wide - prow0 * 2, 0);
    }
    const unsigned qa = at + BM * kStepBytes;
    if constexpr (MODE == M_NT) {
      const long k = it * kStepBytes;
      lq.load(qa, wave, P.q + g * P.strideq + col0 * P.ldq + k, (long)(qrows - 1) * P.ldq + P.red - k, P.red - k);
    } else {
      const long wide = ((long)P.cols * 2 + 15) & ~15L;
      const long r = it * kStepRed;
      long n, first;
      const char* q;
      if constexpr (MODE == M_NN) {
        n = P.qred - r;
        q = P.q + g * P.strideq;
        first = r;
      } else {
        n = rows - r;
        q = P.q;
        first = t.row0 + r;
      }
      if (n > kStepRed) n = kStepRed;
      lq.load(qa, wave, q + first * P.ldq + col0 * 2, (n - 1) * P.ldq + wide - col0 * 2, 0);
    }
    if constexpr (KIND == K_MX4) {  // 8 scale bytes per row and step: 32 rows per instruction
      const unsigned sa = at + kTile;
      const long kb = it * 8, most = P.red / 16;  // scale bytes of a row
#pragma unroll
      for (int c = 0; c < ((BM + BN) / 32 + WAVES - 1) / WAVES; c++) {
        const int i = c * WAVES + wave;
        if (i >= (BM + BN) / 32) break;
        const bool isp = i < BM / 32;
        const int row = (isp ? i : i - BM / 32) * 32 + (lane >> 1);
        const long ld = isp ? P.ldps : P.ldqs;
        const char* b = (const char*)(isp ? P.ps + row0 * P.ldps : P.qs + g * P.strideqs + col0 * P.ldqs) + kb;
        const int n = isp ? rows : qrows;
        const unsigned cut = kb + 4 * (lane & 1) >= most ? kOutOfRange : 0u;
        dma4(sa + i * 256, ((unsigned)(row * ld) + 4 * (lane & 1)) | cut, descriptor(b, (long)(n - 1) * ld + most - kb));
      }
    }
  };

  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int j = 0; j < FN; j++) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  v4f bacc[FM];  // TN: column sums of p, by a product with ones (workgroups of the first column tile)
#pragma unroll
  for (int i = 0; i < FM; i++) bacc[i] = v4f{0.f, 0.f, 0.f, 0.f};
  const bool sums = MODE == M_TN && P.bsum != nullptr && nt == 0 && wn == 0;

  if (step0 < step1) load_step(step0, 0);
  for (long it = step0; it < step1; it++) {
    const int buf = (int)(it - step0) & 1;
    wait_and_sync();
    if (it + 1 < step1) load_step(it + 1, buf ^ 1);
    const char* tp = lds[buf];
    const char* tq = lds[buf] + BM * kStepBytes;
    int ps[FM] = {}, qs[FN] = {};
    if constexpr (KIND == K_MX4) {
      const char* ts = lds[buf] + kTile;
#pragma unroll
      for (int i = 0; i < FM; i++)
        ps[i] = *(const unsigned short*)(ts + (wm * (BM / WM) + i * 16 + (lane & 15)) * 8 + 2 * (lane >> 4));
#pragma unroll
      for (int j = 0; j < FN; j++)
        qs[j] = *(const unsigned short*)(ts + (BM + wn * (BN / WN) + j * 16 + (lane & 15)) * 8 + 2 * (lane >> 4));
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
      v4i fq[FN], fp[FM];
#pragma unroll
      for (int j = 0; j < FN; j++) {
        if constexpr (QCOL) fq[j] = frag_col<BN>(tq, wn * (BN / WN) + j * 16, s, lane);
        else fq[j] = frag_row<KIND>(tq, wn * (BN / WN) + j * 16, s, lane);
      }
#pragma unroll
      for (int i = 0; i < FM; i++) {
        if constexpr (PCOL) fp[i] = frag_col<BM>(tp, wm * (BM / WM) + i * 16, s, lane);
        else fp[i] = frag_row<KIND>(tp, wm * (BM / WM) + i * 16, s, lane);
      }
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mma<KIND>(fq[j], fp[i], acc[i][j], qs[j], ps[i], s);
      if constexpr (MODE == M_TN) {
        if (sums) {
          const int one = KIND == K_F16 ? 0x3c003c00 : 0x3f803f80;
          const v4i ones = {one, one, one, one};
#pragma unroll
          for (int i = 0; i < FM; i++) bacc[i] = mma<KIND>(ones, fp[i], bacc[i], 0, 0, s);
        }
      }
    }
  }

  // a lane holds columns 4 (lane / 16) .. + 3 of output row lane % 16 of every 16 x 16 block
  const long unit = MODE == M_TN ? mt / ((P.rows_out + BM - 1) / BM) : 0;
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const int m = wm * (BM / WM) + i * 16 + (lane & 15);
    if constexpr (MODE == M_TN) {
      const long orow = prow0 + m;
      if (orow >= P.rows_out) continue;
      if (sums && lane < 16) P.bsum[unit * P.rows_out + orow] = bacc[i][0];
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const long n = col0 + wn * (BN / WN) + j * 16 + 4 * (lane >> 4);
        const int have = (int)(P.cols - n < 4 ? P.cols - n : 4);
        if (have <= 0) continue;
        if (P.part) store4(P.part, DT_F32, (unit * P.rows_out + orow) * P.cols + n, acc[i][j], have, P.cols % 4 == 0);
        else store4(P.out, P.out_type, ((long)g * P.rows_out + orow) * P.cols + n, acc[i][j], have, P.vec);
      }
    } else {
      if (m >= rows) continue;
      const long orow = row0 + m;
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const long n = col0 + wn * (BN / WN) + j * 16 + 4 * (lane >> 4);
        const int have = (int)(P.cols - n < 4 ? P.cols - n : 4);
        if (have <= 0) continue;
        v4f v = acc[i][j];
        if (P.part) {
          store4(P.part, DT_F32, ((long)blockIdx.y * P.S + orow) * P.cols + n, v, have, P.cols % 4 == 0);
          continue;
        }
        if (g >= 0) {
#pragma unroll
          for (int r = 0; r < 4; r++) {
            if (P.bias && r < have) v[r] += load_bias(P.bias, P.bias_type, (long)g * P.cols + n + r);
            if (P.act) v[r] = gelu(v[r]);
          }
        }
        store4(P.out, P.out_type, orow * P.cols + n, v, have, P.vec);
      }
    }
  }
}

}  // namespace sm3x
