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
#include <type_traits>
#include <utility>

#include "common.h"

namespace sm3x {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

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
  int out_type, bias_type, act;
  int wide;                       // result rows allow 16-byte stores
  int bias_lds;                   // bias rows may be loaded as 4-byte words and their bytes are counted in 32 bits
  const void* bias;               // (G, cols) or null
  void* db;                       // TN: column sums of p per expert (G, rows_out) of bias_type, or null;
  float* bsum;                    // where units are parts of experts: per unit (units, rows_out) fp32
  const int* offsets;             // (G + 1) device, or null: one group of all S rows
  int G;
  long S;
  int ntiles;                     // column tiles
  int phase;                      // NT / NN: 0 all tiles; 1 the whole rounds of coarse tiles, 2 what they leave (see Jobs)
  int splits;                     // NT / NN: slices of the reduction; > 1: fp32 partials (splits, S, cols) in `part`
  long unit_rows;                 // TN: reduction rows per work unit
  float* part;                    // fp32 partials, or null: the result goes straight to `out`
};

// ---- the jobs of a workgroup ----------------------------------------------------------------------------------------
// A job is one output tile (of one slice of the reduction).  Row tiles are numbered expert by expert; behind them come the
// tiles of rows that belong to no expert (behind the last, before the first), whose outputs are zero.  Jobs run in bands of 4 row
// tiles; consecutive jobs run on one XCD (they share operands in its L2).
// The experts' row ranges are read from the device offsets: clamped to [0, S] and made monotone (running maximum), so that no
// content of the array can lead an access out of range.
struct Job {
  int g, row0, rows;  // expert (-1: rows of no expert); NT / NN: output rows.  TN: reduction rows
  int col0, prow0;    // first output column; TN: first output row
  int unit;           // slice (NT / NN) or work unit (TN) the result belongs to
  int s0, s1;         // steps
};
struct Sources {
  const char *p, *q, *ps, *qs;  // operands, 4-bit operands' scales
  int pn, qn, psn, qsn;         // bytes behind them
};
constexpr int kMaxJobs = 64;  // of one workgroup: lane l of every wave holds job l

struct Jobs {
  int g, row0, rows, col0, prow0, unit;  // of this lane's job
  int count;

  // BM, BN: output tile; row tiles are BM rows (NT / NN) or a work unit of unit_rows reduction rows (TN) with `mper` tiles each
  template <bool TN, int BM, int BN>
  __device__ __forceinline__ void init(const Params& P) {
    constexpr int kCoarse = 256;  // tile of the rounds that a second launch finishes (phases 1 and 2, NT / NN)
    const bool rest = !TN && P.phase == 2;
    const int bm = TN ? (int)P.unit_rows : rest ? kCoarse : BM;
    const unsigned mper = TN ? (unsigned)(P.rows_out + BM - 1) / BM : 1u;  // TN: row tiles of a unit
    const int lane = threadIdx.x & 63, S = (int)P.S;
    const auto clamp = [&](int v) { return v < 0 ? 0 : v > S ? S : v; };
    const auto tiles_of = [&](int len) { return (int)((unsigned)(len + (unsigned)bm - 1u) / (unsigned)bm); };
    const auto ends_from = [&](int e) { return P.offsets[1 + (e + lane < P.G ? e + lane : 0)]; };
    // owned: row tiles of the experts; last: where the last expert ends.  An expert without rows has one (empty) unit in TN.
    int first = 0, last = S, owned = tiles_of(S);
    if (TN && owned == 0) owned = 1;
    // up to 64 experts: lane e holds expert e's range and its share of the running count (TN: in the order of work)
    const bool lanes = P.offsets != nullptr && P.G <= 64;
    int from = 0, len = 0, n = 0, incl = 0, expert = lane, unit0 = 0;
    const auto count_up = [&](int v) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        v += lane >= d ? o : 0;
      }
      return v;
    };
    if (P.offsets != nullptr) {
      const int ends = ends_from(0), raw = P.offsets[0];
      first = clamp(__builtin_amdgcn_readfirstlane(raw));
      if (lanes) {
        int to = lane < P.G ? clamp(ends) : 0;
        to = to < first ? first : to;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int o = __shfl_up(to, d);
          to = lane >= d && o > to ? o : to;
        }
        from = __shfl_up(to, 1);
        if (lane == 0) from = first;
        len = lane < P.G ? to - from : 0;
        n = tiles_of(len);
        if (TN && lane < P.G && n == 0) n = 1;
        incl = count_up(n);
        last = __builtin_amdgcn_readlane(to, 63);
        owned = __builtin_amdgcn_readlane(incl, 63);
        if (TN && P.part == nullptr) {  // longest expert first (ties: the lower index)
          int rank = 0;
          for (int e = 0; e < P.G; e++) {
            const int l = __builtin_amdgcn_readlane(len, e);
            rank += l > len || (l == len && e < lane) ? 1 : 0;
          }
          const int to_lane = 4 * (lane < P.G ? rank : lane);
          unit0 = __builtin_amdgcn_ds_permute(to_lane, incl - n);
          expert = __builtin_amdgcn_ds_permute(to_lane, lane);
          from = __builtin_amdgcn_ds_permute(to_lane, from);
          len = __builtin_amdgcn_ds_permute(to_lane, len);
          n = __builtin_amdgcn_ds_permute(to_lane, n);
          incl = count_up(n);
        }
      } else {
        last = first;
        owned = 0;
        int held = ends;
        for (int e = 0; e < P.G; e++) {
          if (e && (e & 63) == 0) held = ends_from(e);
          const int end = clamp(__builtin_amdgcn_readlane(held, e & 63));
          const int to = end > last ? end : last, m = tiles_of(to - last);
          owned += TN && m == 0 ? 1 : m;
          last = to;
        }
      }
    }
    const int behind = TN ? 0 : tiles_of(S - last), before = TN ? 0 : tiles_of(first);
    const unsigned ntiles = (unsigned)P.ntiles, mtiles = (unsigned)(owned + behind + before);
    const unsigned stride = gridDim.x / kNumXCD, xcd = blockIdx.x % kNumXCD, slot = blockIdx.x / kNumXCD;
    unsigned t;
    int quarter = 0;
    if constexpr (!TN) {
      const unsigned tiles = mtiles * ntiles;
      // phase 1 runs whole rounds of one coarse tile per CU (and a last one that is at least a quarter full), phase 2 cuts the
      // tiles that are left into four, one quarter per CU
      const unsigned over = tiles % kNumCU, coarse = over > kNumCU / 4 ? tiles : tiles - over;
      const unsigned jobs = P.phase == 0 ? tiles * (unsigned)P.splits : rest ? (tiles - coarse) * 4u : coarse;
      const unsigned per = (jobs + kNumXCD - 1) / kNumXCD;
      const unsigned begin = xcd * per, limit = begin + per < jobs ? begin + per : jobs;
      const unsigned mine = begin + slot, job = mine + lane * stride;
      count = mine < limit ? (int)((limit - mine + stride - 1) / stride) : 0;  // (<= kMaxJobs: the grid is made for it)
      const unsigned tile = rest ? coarse + job / 4u : job;
      const unsigned z = tiles ? tile / tiles : 0u, lin = tile - z * tiles;  // (lanes behind the last job: nobody reads theirs)
      const unsigned band = lin / (4u * ntiles), in = lin - band * 4u * ntiles;
      const unsigned left = mtiles - band * 4u, deep = left < 4u ? (left ? left : 1u) : 4u;
      const unsigned nt = in / deep;
      t = band * 4u + (in - nt * deep);
      quarter = rest ? (int)(job & 3u) : 0;
      col0 = (int)(nt * (rest ? kCoarse : BN)) + (quarter >> 1) * BN;
      prow0 = 0;
      unit = (int)z;
    } else {
      // Where units are whole experts they differ in length: every XCD gets an eighth of EACH unit's tiles, units follow each
      // other from the longest to the shortest (up to 64 experts), and every other round of workgroups runs backwards
      // (16384 rows, 8 experts, 4096 x 1024: 228 -> 156 us).  Units cut to one length stay whole on an XCD, which then reads
      // their rows once (65536 rows, 1024 x 256: 85 -> 69 us).
      const unsigned tiles = mper * ntiles;
      unsigned u, tile;
      if (P.part == nullptr) {
        const unsigned per = (tiles + kNumXCD - 1) / kNumXCD, jobs = per * (unsigned)owned;
        const unsigned job = lane * stride + ((lane & 1) ? stride - 1 - slot : slot);
        count = (int)((jobs + stride - 1) / stride);
        u = job / per;
        tile = xcd * per + (job - u * per);
        t = job < jobs && tile < tiles ? u : ~0u;  // (position of the unit in the order of work; none)
      } else {
        const unsigned jobs = tiles * (unsigned)owned, per = (jobs + kNumXCD - 1) / kNumXCD;
        const unsigned begin = xcd * per, limit = begin + per < jobs ? begin + per : jobs;
        const unsigned mine = begin + slot, job = mine + lane * stride;
        count = mine < limit ? (int)((limit - mine + stride - 1) / stride) : 0;
        u = job / tiles;
        tile = job - u * tiles;
        t = job < limit ? u : ~0u;
      }
      const unsigned pt = tile / ntiles;
      prow0 = (int)(pt * BM);
      col0 = (int)((tile - pt * ntiles) * BN);
    }
    g = -1;
    row0 = 0;
    int end_row = 0;
    if constexpr (!TN) {  // rows of no expert, unless one is found below
      const int i = (int)t - owned;
      row0 = i < behind ? last + i * bm : (i - behind) * bm;
      end_row = i < behind ? S : first;
    }
    if (P.offsets == nullptr) {
      if (t < (unsigned)owned) {
        g = 0;
        row0 = (int)t * bm;
        end_row = S;
        if (TN) unit = (int)t;
      }
    } else if (lanes) {
      int e = 0;  // the lane whose running count first exceeds t
#pragma unroll
      for (int step = 32; step; step >>= 1) e += (unsigned)__shfl(incl, e + step - 1) <= t ? step : 0;
      e = e < 63 ? e : 63;
      const int at = (int)t - __shfl(incl - n, e), f = __shfl(from, e), l = __shfl(len, e), x = __shfl(expert, e);
      const int u = __shfl(unit0, e);
      if (t < (unsigned)owned) {
        g = x;
        row0 = f + at * bm;
        end_row = f + l;
        if (TN) unit = P.part == nullptr ? u + at : (int)t;
      }
    } else {
      int at = 0, prev = first, held = ends_from(0);
      for (int e = 0; e < P.G; e++) {
        if (e && (e & 63) == 0) held = ends_from(e);
        const int end = clamp(__builtin_amdgcn_readlane(held, e & 63));
        const int to = end > prev ? end : prev;
        int m = tiles_of(to - prev);
        if (TN && m == 0) m = 1;
        if (t != ~0u && (int)t >= at && (int)t < at + m) {
          g = e;
          row0 = prev + ((int)t - at) * bm;
          end_row = to;
          if (TN) unit = (int)t;
        }
        at += m;
        prev = to;
      }
    }
    rows = end_row - row0;
    rows = rows < 0 ? 0 : rows > bm ? bm : rows;
    if (rest) {  // this quarter of the coarse tile, if it has one
      row0 += (quarter & 1) * BM;
      rows -= (quarter & 1) * BM;
      rows = rows < 0 ? 0 : rows > BM ? BM : rows;
      if (rows == 0 || col0 >= P.cols) {
        g = -1;
        rows = 0;
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // (nothing of this is in flight when the loader starts to count its own loads)
  }
};

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

__device__ __forceinline__ void move(v4i& desc, long by) {
  const unsigned long long a = ((unsigned long long)(unsigned)desc[1] << 32 | (unsigned)desc[0]) + by;
  desc[0] = (int)(unsigned)a;
  desc[1] = (int)(unsigned)(a >> 32);
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
// this wave's direct loads have landed and its LDS reads are done; after the barrier everybody's.  (The builtin, not asm: the
// compiler then knows that its own loads and stores are complete too and inserts no waits for them into the loop.)
// All but the LATER loads issued last (the steps behind).
template <int LATER>
__device__ __forceinline__ void wait_and_sync() {
  static_assert(LATER < 64, "six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (LATER & 15) | (LATER >> 4) << 14);  // vmcnt(LATER) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <class T>
__device__ __forceinline__ T* uniform(T* p) {
  const unsigned long long a = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)a), hi = __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32));
  return (T*)((unsigned long long)hi << 32 | lo);
}

// The same where AFTER stores may stand behind those loads (`stored`: they do).  Loads and stores of a wave complete in the order
// of issue as far as the counter goes, so the loads are waited for without the stores.  The branch is inside the asm: one that
// the compiler sees would split the rounds' blocks.
template <int LATER, int AFTER>
__device__ __forceinline__ void wait_and_sync(int stored) {
  static_assert(LATER + AFTER < 64, "six bits");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  asm volatile("s_cmp_lg_u32 %0, 0\n\ts_waitcnt vmcnt(%1)\n\ts_cbranch_scc1 .Lloaded%=\n\ts_waitcnt vmcnt(%2)\n.Lloaded%=:"
               :: "s"(__builtin_amdgcn_readfirstlane(stored)), "n"(LATER + AFTER), "n"(LATER) : "memory", "scc");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// swizzle of a column operand's row: spreads the 4 rows x 32 bytes that 16 lanes of a transposing read touch over the banks
__device__ __forceinline__ int col_swz(int row, int granules) {
  return (2 * ((row & 3) | ((row >> 1) & 4))) & (granules - 1);
}

// One operand tile of BX rows (row operand) or BX columns (column operand): 128 * BX bytes of LDS per step, loaded by
// `waves` waves with N = BX / 8 / waves instructions ("pieces") each.
template <int BX, bool COL, int WAVES>
struct Loader {
  static constexpr int N = BX / 8 / WAVES;
  static_assert(BX / 8 % WAVES == 0 && N >= 1, "every wave loads the same number of 1 KB pieces");
  unsigned voff[N];
  int gran;   // row operand: this lane's granule of a step
  v4i desc;   // of the step being loaded: advanced from step to step, so that a step costs a handful of scalar instructions
  bool tail;  // row operand: the step is the reduction's last and part-filled, voff of the lanes behind its end is out of range

  __device__ __forceinline__ void init(int wave, int lane, long ld) {
    tail = false;
    gran = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int piece = wave * N + i;
      if constexpr (!COL) {
        voff[i] = (unsigned)((piece * 8 + (lane >> 3)) * ld) + gran * 16;
      } else {
        constexpr int GR = BX / 8, RP = 64 / GR;  // granules per row, rows per piece
        const int row = piece * RP + lane / GR;
        voff[i] = (unsigned)(row * ld) + (((lane % GR) ^ col_swz(row, GR)) * 16);
      }
    }
  }
  // bytes <= 0: nothing is read, zeros arrive
  __device__ __forceinline__ void start(const char* base, long bytes) {
    desc = descriptor(base, bytes);
    if (!COL && tail) {
#pragma unroll
      for (int i = 0; i < N; i++) voff[i] &= ~kOutOfRange;
      tail = false;
    }
  }
  __device__ __forceinline__ void cut(int left) {  // row operand: fewer than kStepBytes remain
    tail = true;
#pragma unroll
    for (int i = 0; i < N; i++) voff[i] |= gran * 16 >= left ? kOutOfRange : 0u;
  }
  __device__ __forceinline__ void piece(unsigned lds, int wave, int i) const { dma16(lds + (wave * N + i) * 1024, voff[i], desc); }
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
// GELU(h) = h Phi(h) = max(h, 0) - |h| Phi(-|h|), with Phi(-a) = 2^p(a): log2 Phi(-a) is so smooth that a polynomial of degree 7
// (fitted here by linear programming on [0, 6], minimax in the error relative to |h|, then rounded to fp32) leaves 4.5e-8 |h|,
// 1.2e-7 |h| with the fp32 rounding of its evaluation; behind 6 |h| Phi(-|h|) is below 6e-9.  One transcendental instruction and 11 others: with the
// erfc form of Abramowitz & Stegun 7.1.26 (two and 12, error 1e-7) the epilogue of a 4-bit product was bound by GELU.
// (h / 2 + |h| / 2 is max(h, 0) that lets a NaN through.)
// Eight at once, step by step, so that no instruction waits for the one before it.
__device__ __forceinline__ void gelu8(float (&h)[8]) {
  constexpr float c[8] = {-0.9999998807907104f,   -1.1511108875274658f, -0.4591531455516815f,    -0.05269111320376396f,
                          0.007389274425804615f, -0.0004212373751215637f, -5.390329170040786e-05f, 8.470114153169561e-06f};
  float a[8], p[8];
#pragma unroll
  for (int r = 0; r < 8; r++) a[r] = fminf(fabsf(h[r]), 6.0f);
#pragma unroll
  for (int r = 0; r < 8; r++) p[r] = fmaf(c[7], a[r], c[6]);
#pragma unroll
  for (int k = 5; k >= 0; k--) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 8; r++) p[r] = fmaf(p[r], a[r], c[k]);
  }
#pragma unroll
  for (int r = 0; r < 8; r++) p[r] = __builtin_amdgcn_exp2f(p[r]);
#pragma unroll
  for (int r = 0; r < 8; r++) h[r] = fmaf(-a[r], p[r], fmaf(0.5f, fabsf(h[r]), 0.5f * h[r]));
}

// the eight values b[at .. at + 7], indexes clamped to `most` (what lies behind is not stored)
__device__ __forceinline__ void bias8(float (&v)[8], const void* b, int type, long at, long most) {
  if (type == DT_F32) {
#pragma unroll
    for (int r = 0; r < 8; r++) v[r] = ((const float*)b)[at + r < most ? at + r : most];
  } else {
    unsigned short h[8];
#pragma unroll
    for (int r = 0; r < 8; r++) h[r] = ((const unsigned short*)b)[at + r < most ? at + r : most];
#pragma unroll
    for (int r = 0; r < 8; r++)
      v[r] = type == DT_F16 ? (float)__builtin_bit_cast(_Float16, h[r]) : __uint_as_float((unsigned)h[r] << 16);
  }
}

// four consecutive ones (a multiple of 4 from the row's start: the row may be read in words), their place clamped to `most`
__device__ __forceinline__ v4f bias4(const void* b, int type, long at, long most) {
  at = at < most ? at : most;
  if (type == DT_F32) {
    const float* f = (const float*)b + at;
    return v4f{f[0], f[1], f[2], f[3]};
  }
  const unsigned short* u = (const unsigned short*)b + at;
  unsigned short h[4];
#pragma unroll
  for (int r = 0; r < 4; r++) h[r] = u[r];
  v4f v;
#pragma unroll
  for (int r = 0; r < 4; r++) v[r] = type == DT_F16 ? (float)__builtin_bit_cast(_Float16, h[r]) : __uint_as_float((unsigned)h[r] << 16);
  return v;
}

__device__ __forceinline__ unsigned pack2(float a, float b, int type) {  // rounded to nearest even
  if (type == DT_F16) return __builtin_bit_cast(unsigned, v2h{(_Float16)a, (_Float16)b});
  return __builtin_bit_cast(unsigned, v2b{(__bf16)a, (__bf16)b});
}

// eight consecutive values of one row, `n` of them exist; wide: 16-byte stores are allowed (and n is a multiple of what one holds)
__device__ __forceinline__ void store8(void* out, int type, long at, const float (&v)[8], int n, bool wide) {
  if (type == DT_F32) {
    float* o = (float*)out + at;
    if (wide) {
      if (n >= 4) *(v4f*)o = v4f{v[0], v[1], v[2], v[3]};
      if (n >= 8) *(v4f*)(o + 4) = v4f{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int r = 0; r < 8; r++) { if (r < n) o[r] = v[r]; }
    }
    return;
  }
  v8s h;
  if (type == DT_F16) {
#pragma unroll
    for (int r = 0; r < 8; r++) h[r] = __builtin_bit_cast(short, (_Float16)v[r]);
  } else {
#pragma unroll
    for (int r = 0; r < 8; r++) h[r] = __builtin_bit_cast(short, (__bf16)v[r]);
  }
  short* o = (short*)out + at;
  if (wide) *(v8s*)o = h;
  else {
#pragma unroll
    for (int r = 0; r < 8; r++) { if (r < n) o[r] = h[r]; }
  }
}

template <int... I, class F>
__device__ __forceinline__ void for_each_of(std::integer_sequence<int, I...>, F f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void for_each(F f) { for_each_of(std::make_integer_sequence<int, N>{}, f); }

// ---- the kernel ---------------------------------------------------------------------------------------------------
// BM output rows (P) x BN output columns (Q); WM x WN waves, MINW waves per SIMD.
//
// A workgroup runs through a list of tiles (jobs) as ONE sequence of steps: the loader is NB steps ahead of the matrix unit (two;
// four in the lone quarters of phase 2) and walks into the next tile while the current one is finished and stored, so a tile costs
// neither a ramp nor a drain.
// NB LDS buffers, one barrier per step.  A step is two rounds; while the matrix unit works on one round's fragments, the
// next round's are read from LDS, piece by piece between the instructions (round 1 reads round 0 of the NEXT step, so the
// barrier stands between the rounds: by then this step's buffer has been read out and the next one has landed):
//     round 0: multiply f0 | read f1 from buffer i
//     wait for the loads of step i + 1 (issued NB - 1 steps ago), barrier
//     round 1: multiply f1 | read f0 from buffer i + 1 | start loading step i + NB into buffer i
//
// Bounds (8 uneven experts, bf16).  16384 x 4096 x 1024: with the same operands call after call 127 us forward, 142 input gradient, 138
// weight gradient (1080, 970, 1000 TF/s); with other operands each call 149, 156, 166; in a training step, kernel by kernel,
// 146 + 21 (quarters), 136 + 53, 177.  The matrix unit is 40-60 % busy at the 1.6 GHz the part falls to; 128 x 128 tiles there want
// 20 TB/s from L2, 256 x 256 ones half of it.  65536 x 1024 x 256: 54, 45, 64 us with the same operands, 78, 59, 85 with others, 80, 61,
// 61 + 11 (join) in a training step; 4 steps per tile, bound by the steps' latency (a lone step takes 0.7-0.9 us whatever its
// arithmetic).  Storing nothing saved 4 us there; non-temporal stores save 2 us of a lone 4-bit product and cost the feed-forward
// 3 %, whose second product then finds less of the first one's result in the caches.  MINW: two workgroups of 128 x 128 per CU
// cover each other's waits; three of 32 x 128 where rows are few.
template <int KIND, int MODE, int BM, int BN, int WM, int WN, int MINW, int NB = 2>
__global__ void __launch_bounds__(WM * WN * 64, MINW) tile_kernel(const Params P) {
  constexpr int WAVES = WM * WN, TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr bool PCOL = MODE == M_TN, QCOL = MODE != M_NT;
  static_assert(FN % 2 == 0, "the epilogue takes blocks in pairs");
  static_assert(KIND != K_MX4 || MODE == M_NT, "4-bit operands: rows only");
  constexpr bool ACT = KIND == K_MX4;  // (the 16-bit products have no activation: their gradients would need its derivative)
  constexpr int kTile = (BM + BN) * kStepBytes;
  constexpr int NS = KIND == K_MX4 ? ((BM + BN) / 32 + WAVES - 1) / WAVES : 0;  // scale pieces of a wave: 32 rows x 8 bytes each
  constexpr int kScales = NS * WAVES * 256;
  constexpr int kBuf = kTile + kScales;
  constexpr int SR = NB == 2 ? 8 : 4;                // epilogue for rows without 16-byte stores: SR rows of a wave's columns
  constexpr int kStage = SR * (TN * 4 + 16);
  constexpr int kBias = MODE == M_TN ? 0 : 4 * BN * 4 + 256;  // bias rows of four jobs (the loader is at most two ahead)
  __shared__ __attribute__((aligned(1024))) char lds[NB * kBuf + WAVES * kStage + kBias];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;

  Jobs jobs;
  jobs.init<MODE == M_TN, BM, BN>(P);
  const int red_steps = MODE == M_TN ? 0 : (int)((P.red + kStepBytes - 1) / kStepBytes);
  const int slice = MODE == M_TN ? 0 : (red_steps + P.splits - 1) / P.splits;
  auto steps_of = [&](Job& w) {
    if constexpr (MODE == M_TN) {
      w.s0 = 0;
      w.s1 = (w.rows + kStepRed - 1) / kStepRed;
    } else {
      const int steps = w.g < 0 ? 0 : red_steps, a = w.unit * slice;
      w.s0 = a < steps ? a : steps;
      w.s1 = w.s0 + slice < steps ? w.s0 + slice : steps;
    }
  };
  auto job_of = [&](int j) {
    Job w;
    w.g = __builtin_amdgcn_readlane(jobs.g, j);
    w.row0 = __builtin_amdgcn_readlane(jobs.row0, j);
    w.rows = __builtin_amdgcn_readlane(jobs.rows, j);
    w.col0 = __builtin_amdgcn_readlane(jobs.col0, j);
    w.prow0 = __builtin_amdgcn_readlane(jobs.prow0, j);
    w.unit = __builtin_amdgcn_readlane(jobs.unit, j);
    steps_of(w);
    return w;
  };

  // ---- the loader
  Loader<BM, PCOL, WAVES> lp;
  Loader<BN, QCOL, WAVES> lq;
  lp.init(wave, lane, P.ldp);
  lq.init(wave, lane, P.ldq);
  constexpr int ND = lp.N + lq.N + NS;
  const unsigned base = __builtin_amdgcn_readfirstlane((int)lds_address(lds));
  char* const bias_lds = lds + NB * kBuf + WAVES * kStage;

  // Where a job's first step begins in memory, and the bytes from there to the operand's end.  Computed for all jobs at once, lane
  // j's for job j, and read from there when the loader enters the job: computed anew they are 300 scalar instructions per tile
  // (4-bit 16384 x 2048 x 512: 47.8 -> 45.5 us; feed-forward of 65536 x 192: 100 -> 94.5).  Not held by 256 x 256 tiles, which
  // have neither registers for it nor too few steps to hide it, nor by TN's long units (no gain).
  constexpr bool kHeld = BM < 256 && MODE != M_TN;
  auto sources_of = [&](const Job& w) {
    const long k = (long)w.s0 * kStepBytes, r = (long)w.s0 * kStepRed;
    const int qrows = P.cols - w.col0 < BN ? P.cols - w.col0 : BN;
    const auto to_int = [](long n) { return n < 0 ? 0 : (int)n; };
    Sources b{};
    if constexpr (MODE == M_TN) {
      b.p = P.p + w.row0 * P.ldp + (long)w.prow0 * 2;
      b.q = P.q + w.row0 * P.ldq + (long)w.col0 * 2;
    } else {
      b.p = P.p + (long)w.row0 * P.ldp + k;
      b.pn = to_int((long)(w.rows - 1) * P.ldp + (P.red - k));
      if constexpr (MODE == M_NN) b.q = P.q + w.g * P.strideq + r * P.ldq + (long)w.col0 * 2;
      else {
        b.q = P.q + w.g * P.strideq + (long)w.col0 * P.ldq + k;
        b.qn = to_int((long)(qrows - 1) * P.ldq + (P.red - k));
      }
    }
    if constexpr (KIND == K_MX4) {
      b.ps = (const char*)P.ps + (long)w.row0 * P.ldps + w.s0 * 8;
      b.qs = (const char*)P.qs + w.g * P.strideqs + (long)w.col0 * P.ldqs + w.s0 * 8;
      b.psn = to_int((w.rows - 1) * P.ldps + (P.red - k) / 16);
      b.qsn = to_int((qrows - 1) * P.ldqs + (P.red - k) / 16);
    }
    return b;
  };
  Sources held{};
  if constexpr (kHeld) {
    Job w{};
    w.g = jobs.g;
    w.row0 = jobs.row0;
    w.rows = jobs.rows;
    w.col0 = jobs.col0;
    w.prow0 = jobs.prow0;
    w.unit = jobs.unit;
    steps_of(w);
    held = sources_of(w);
  }
  int lj = 0, lit = 0, lnum = -1;  // job being loaded, its step, its ordinal among the jobs that load anything
  auto from_lane = [&](const char* p) {
    const unsigned long long a = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)a, lj), hi = __builtin_amdgcn_readlane((int)(unsigned)(a >> 32), lj);
    return (const char*)((unsigned long long)hi << 32 | lo);
  };
  Job lw{};
  bool more = true;
  int kleft = 0, rleft = 0;  // row operand: bytes, column operand: rows of the reduction that remain
  const int pw = (P.rows_out * 2 + 15) & ~15, qw = (P.cols * 2 + 15) & ~15;  // bytes of a column operand's rows
  // MX4: scale pieces
  unsigned svoff[NS ? NS : 1], scut = 0;
  v4i sdesc[NS ? NS : 1];
  if constexpr (KIND == K_MX4) {
#pragma unroll
    for (int c = 0; c < NS; c++) {
      const int i = c * WAVES + wave, row = (i < BM / 32 ? i : i - BM / 32) * 32 + (lane >> 1);
      svoff[c] = (unsigned)(row * (int)(i < BM / 32 ? P.ldps : P.ldqs)) + 4 * (lane & 1);
    }
  }
  // the bias row of a job travels with its first step as one more piece (slot: the job's ordinal modulo 4; other steps load
  // nothing into a fifth)
  const int bes = P.bias_type == DT_F32 ? 4 : 2;
  const unsigned bias_none = base + (unsigned)(bias_lds - lds) + 4 * (BN * 4);
  unsigned bias_to = bias_none;
  v4i bdesc = descriptor(P.bias, 0);

  auto last_rows = [&]() {  // column operands: the rows of the step that exist
    const int n = rleft < kStepRed ? rleft : kStepRed;
    if constexpr (PCOL) lp.desc[2] = (n - 1) * (int)P.ldp + pw - lw.prow0 * 2;
    if constexpr (QCOL) lq.desc[2] = (n - 1) * (int)P.ldq + qw - lw.col0 * 2;
  };
  auto last_bytes = [&]() {  // row operands: fewer than a step's bytes remain
    if constexpr (!PCOL) lp.cut(kleft);
    if constexpr (!QCOL) lq.cut(kleft);
    if constexpr (KIND == K_MX4) scut = 4 * (lane & 1) >= kleft / 16 ? kOutOfRange : 0u;
  };
  auto enter = [&]() {  // the first job from lj on that has steps: descriptors of its first one
    for (;; lj++) {
      if (lj >= jobs.count) {  // nothing is left: empty descriptors (zeros arrive)
        more = false;
        lp.desc[2] = 0;
        lq.desc[2] = 0;
        bdesc[2] = 0;
        bias_to = bias_none;
        if constexpr (KIND == K_MX4) {
#pragma unroll
          for (int c = 0; c < NS; c++) sdesc[c][2] = 0;
        }
        return;
      }
      lw = job_of(lj);
      if (lw.s0 < lw.s1) break;
    }
    lit = lw.s0;
    lnum++;
    kleft = (int)(P.red - (long)lit * kStepBytes);
    rleft = MODE == M_TN ? lw.rows - lit * kStepRed : (int)(P.qred - (long)lit * kStepRed);
    Sources b;
    if constexpr (kHeld) {
      b = {from_lane(held.p), from_lane(held.q), from_lane(held.ps), from_lane(held.qs)};
      b.pn = __builtin_amdgcn_readlane(held.pn, lj);
      b.qn = __builtin_amdgcn_readlane(held.qn, lj);
      b.psn = __builtin_amdgcn_readlane(held.psn, lj);
      b.qsn = __builtin_amdgcn_readlane(held.qsn, lj);
    } else {
      b = sources_of(lw);
    }
    lp.start(b.p, b.pn);
    lq.start(b.q, b.qn);
    if constexpr (KIND == K_MX4) {
      scut = 0;
#pragma unroll
      for (int c = 0; c < NS; c++) {
        const int i = c * WAVES + wave;  // (pieces behind the last read nothing; their zeros go to padding)
        sdesc[c] = descriptor(i < BM / 32 ? b.ps : b.qs, i < BM / 32 ? b.psn : i < (BM + BN) / 32 ? b.qsn : 0);
      }
    }
    if constexpr (PCOL || QCOL) last_rows();
    if constexpr (!PCOL) { if (kleft < kStepBytes) last_bytes(); }
    if constexpr (MODE != M_TN) {
      if (P.bias_lds && wave * 256 < BN * bes) {
        bdesc = descriptor((const char*)P.bias + ((long)lw.g * P.cols + lw.col0) * bes, (long)(P.cols - lw.col0) * bes);
        bias_to = base + (unsigned)(bias_lds - lds) + (lnum & 3) * (BN * 4) + wave * 256;
      }
    }
  };
  auto advance = [&]() {  // to the next step (of the next job where this one ends)
    if (!more) return;
    if (++lit >= lw.s1) {
      lj++;
      enter();
      return;
    }
    move(lp.desc, PCOL ? kStepRed * P.ldp : kStepBytes);
    move(lq.desc, QCOL ? kStepRed * P.ldq : kStepBytes);
    if constexpr (!PCOL) lp.desc[2] -= kStepBytes;
    if constexpr (!QCOL) lq.desc[2] -= kStepBytes;
    kleft -= kStepBytes;
    rleft -= kStepRed;
    if constexpr (KIND == K_MX4) {
#pragma unroll
      for (int c = 0; c < NS; c++) {
        move(sdesc[c], 8);
        sdesc[c][2] = sdesc[c][2] > 8 ? sdesc[c][2] - 8 : 0;
      }
    }
    if constexpr (PCOL || QCOL) { if (rleft < kStepRed) last_rows(); }
    if constexpr (!PCOL) { if (kleft < kStepBytes) last_bytes(); }
    bdesc[2] = 0;
    bias_to = bias_none;
  };
  auto dma = [&](unsigned at, int d) {  // piece d of the step, into the buffer at LDS address `at`
    if (d < lp.N) lp.piece(at, wave, d);
    else if (d < lp.N + lq.N) lq.piece(at + BM * kStepBytes, wave, d - lp.N);
    else if constexpr (KIND == K_MX4) {  // 8 scale bytes per row and step: 32 rows per instruction
      const int c = d - lp.N - lq.N;
      dma4(at + kTile + (c * WAVES + wave) * 256, svoff[c] | scut, sdesc[c]);
    }
  };
  auto dma_bias = [&]() {
    if constexpr (MODE != M_TN) dma4(bias_to, wave * 256 + lane * 4, bdesc);
  };
  static_assert(MODE == M_TN || WAVES * 256 >= BN * 4, "one bias piece per wave");

  // ---- fragments (and scale pairs) of the two rounds
  v4i fp[2][FM], fq[2][FN];
  int ps[2][FM] = {}, qs[2][FN] = {};  // [1]: of the next step, read with its round 0
  constexpr int NR = FM + FN;
  auto read = [&](const char* buf, int s, int r) {  // fragment r of round s
    if (r < FN) {
      if constexpr (QCOL) fq[s][r] = frag_col<BN>(buf + BM * kStepBytes, wn * TN + r * 16, s, lane);
      else fq[s][r] = frag_row<KIND>(buf + BM * kStepBytes, wn * TN + r * 16, s, lane);
    } else {
      const int i = r - FN;
      if constexpr (PCOL) fp[s][i] = frag_col<BM>(buf, wm * TM + i * 16, s, lane);
      else fp[s][i] = frag_row<KIND>(buf, wm * TM + i * 16, s, lane);
    }
  };
  auto read_scale = [&](const char* buf, int set, int r) {
    const char* ts = buf + kTile + 2 * (lane >> 4) + (lane & 15) * 8;
    if (r < FN) qs[set][r] = *(const unsigned short*)(ts + (BM + wn * TN + r * 16) * 8);
    else ps[set][r - FN] = *(const unsigned short*)(ts + (wm * TM + (r - FN) * 16) * 8);
  };

  v4f acc[FM][FN];
  float bacc[FM];  // TN: column sums of p (tiles of the first columns), this lane's share of the reduction
  bool sums = false;
  // round s: multiply; at even distances issue the NR reads of the other round and (round 1) the ND pieces
  auto round = [&](auto S, const char* next, unsigned into) {
    constexpr int s = decltype(S)::value;
    constexpr int T = FM * FN;
#pragma unroll
    for (int q = 0; q < T; q++) {
      const int i = q / FN, j = q % FN;
#pragma unroll
      for (int r = q * NR / T; r < (q + 1) * NR / T; r++) {
        read(next, s ^ 1, r);
        if constexpr (KIND == K_MX4 && s == 1) read_scale(next, 1, r);
      }
      if constexpr (s == 1) {
#pragma unroll
        for (int d = q * ND / T; d < (q + 1) * ND / T; d++) dma(into, d);
        if (q == T / 2) dma_bias();
      }
      acc[i][j] = mma<KIND>(fq[s][j], fp[s][i], acc[i][j], qs[0][j], ps[0][i], s);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MODE == M_TN) {
      if (sums) {
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
          for (int h = 0; h < 4; h++) {
            const int two = fp[s][i][h];  // (a value of its own: a bit cast of the vector's element itself reads element 0)
            if constexpr (KIND == K_F16)
              bacc[i] = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, two), __builtin_bit_cast(v2h, 0x3c003c00), bacc[i], false);
            else
              bacc[i] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, two), __builtin_bit_cast(v2b, 0x3f803f80), bacc[i],
                                                        false);
          }
      }
    }
  };

  constexpr int NL = ND + (MODE == M_TN ? 0 : 1);  // loads of a wave and step
  enter();
  if (more) {
#pragma unroll
    for (int n = 0; n < NB; n++) {
      if (n) advance();
#pragma unroll
      for (int d = 0; d < ND; d++) dma(base + n * kBuf, d);
      dma_bias();
    }
    wait_and_sync<(NB - 1) * NL>();
#pragma unroll
    for (int r = 0; r < NR; r++) {
      read(lds, 0, r);
      if constexpr (KIND == K_MX4) read_scale(lds, 0, r);
    }
  }

  unsigned off = 0;
  int num = -1;
  constexpr int kStores = FM * FN / 2;  // at least so many stores end a tile ...
  int stored = 0;                       // ... and one has ended since the last step (rows with 16-byte stores only)
  for (int cj = 0; cj < jobs.count; cj++) {
    const Job w = job_of(cj);
    if (MODE == M_TN && w.g < 0) continue;  // (the XCDs' shares of a unit's tiles are rounded up)
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    if constexpr (MODE == M_TN) {
      sums = P.db != nullptr && w.col0 == 0 && wn == 0;
#pragma unroll
      for (int i = 0; i < FM; i++) bacc[i] = 0.f;
    }
    if (w.s0 < w.s1) num++;
    for (int it = w.s0; it < w.s1; it++) {
      // (everything with branches stands before the rounds: the multiplications are free of side effects, and the compiler
      // would move those of a round behind a branch that follows it, away from the loads they are to cover)
      advance();
      __builtin_amdgcn_sched_barrier(0);
      round(std::integral_constant<int, 0>{}, lds + off, 0);
      wait_and_sync<(NB - 2) * NL, kStores>(stored);
      stored = 0;
      __builtin_amdgcn_sched_barrier(0);
      const unsigned next = off == (NB - 1) * kBuf ? 0u : off + kBuf;
      round(std::integral_constant<int, 1>{}, lds + next, base + off);
      if constexpr (KIND == K_MX4) {
#pragma unroll
        for (int j = 0; j < FN; j++) qs[0][j] = qs[1][j];
#pragma unroll
        for (int i = 0; i < FM; i++) ps[0][i] = ps[1][i];
      }
      off = next;
    }

    int lane = threadIdx.x & 63;  // (opaque: what follows is computed here and not kept in registers through the loop)
    asm volatile("" : "+v"(lane));
    // ---- the tile is complete: a lane holds columns 4 (lane / 16) .. + 3 of output row lane % 16 of every 16 x 16 block
    if (MODE == M_TN && sums) {
#pragma unroll
      for (int i = 0; i < FM; i++) {
        float v = bacc[i];  // the four lane groups hold different reduction rows of the same column
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        const int orow = w.prow0 + wm * TM + i * 16 + lane;
        if (lane < 16 && orow < P.rows_out) {
          if (P.bsum) P.bsum[(long)w.unit * P.rows_out + orow] = v;
          else if (P.bias_type == DT_F32) ((float*)P.db)[(long)w.g * P.rows_out + orow] = v;
          else ((unsigned short*)P.db)[(long)w.g * P.rows_out + orow] = (unsigned short)pack2(v, 0.f, P.bias_type);
        }
      }
    }
    void* const out = P.part ? (void*)P.part : P.out;
    const int type = P.part ? DT_F32 : P.out_type;
    const long first = P.part ? (MODE == M_TN ? (long)w.unit * P.rows_out : (long)w.unit * P.S)
                              : (MODE == M_TN ? (long)w.g * P.rows_out : 0L);
    const int orow0 = (MODE == M_TN ? w.prow0 : w.row0) + wm * TM;       // first output row of the wave ...
    const int olim = MODE == M_TN ? P.rows_out : w.row0 + w.rows;        // ... and the end of the rows the tile may write
    const bool finish = MODE != M_TN && P.part == nullptr && w.g >= 0;
    if (P.wide) {
      // Straight from the accumulators.  fp32: a lane's four columns are one 16-byte store.  16 bits: two neighbouring blocks
      // (j, j + 1) are exchanged between the 16-lane rows (v_permlane16_swap: odd rows of the one with even rows of the
      // other), which leaves every lane eight consecutive columns; a store instruction covers 64 contiguous bytes of 16 rows.
      v4f bias[FN];
      const int bcol = wn * TN + 4 * (lane >> 4);
#pragma unroll
      for (int j = 0; j < FN; j++) bias[j] = v4f{0.f, 0.f, 0.f, 0.f};
      if (MODE != M_TN && finish && P.bias) {
        if (P.bias_lds) {
#pragma unroll
          for (int j = 0; j < FN; j++) bias[j] = bias4(bias_lds + (num & 3) * (BN * 4), P.bias_type, bcol + j * 16, BN - 4);
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        } else {
          const long at = (long)w.g * P.cols;
#pragma unroll
          for (int j = 0; j < FN; j++) bias[j] = bias4(P.bias, P.bias_type, at + w.col0 + bcol + j * 16, at + P.cols - 4);
          __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        }
        // waited for here, on this path: left to the first use, the compiler puts a wait for EVERY load into the next tile's loop
      }
      // One straight run of instructions per result type, with the activation or without: the descriptor's range check drops the
      // rows behind olim, an address out of range the columns behind the last (65536 x 1024 x 256, bf16: a tile's end took
      // 6200 cycles with branches, 2600 without; 4-bit 16384 x 2048 x 512 with GELU 53 -> 43 us).
      const auto emit = [&](auto type_of, auto act_of) {
        constexpr int type = decltype(type_of)::value, es = type == DT_F32 ? 4 : 2;
        const int g16 = lane >> 4, ncol = w.col0 + wn * TN, pitch = P.cols * es;
        const int have = P.cols - ncol, rows = olim - orow0 < TM ? olim - orow0 : TM;
        const auto to = __builtin_amdgcn_make_buffer_rsrc(
            uniform((char*)out + (first + orow0) * pitch + (long)ncol * es), (short)0,
            __builtin_amdgcn_readfirstlane(rows > 0 && have > 0 ? (rows - 1) * pitch + have * es : 0), 0x00020000);
#pragma unroll
        for (int j = 0; j < FN; j++)  // (opaque: the sums would else be moved in front of the choice of the type, all at once)
          asm volatile("; results of type %1" : "+v"(bias[j]) : "n"(type + 8 * decltype(act_of)::value));
        unsigned at[FN];  // of the columns of block j (16 bits: of blocks j and j + 1)
#pragma unroll
        for (int j = 0; j < FN; j++) {
          const int n = j * 16 + (type == DT_F32 ? 4 * g16 : (g16 & 1) * 16 + (g16 >> 1) * 8);
          at[j] = (unsigned)((lane & 15) * pitch + n * es) | (n < have ? 0u : kOutOfRange);
        }
        for_each<FM>([&](auto I) {  // (the accumulators are registers: their indexes have to be constants)
          constexpr int i = decltype(I)::value;
          const unsigned down = (unsigned)(i * 16 * pitch);
#pragma unroll
          for (int j = 0; j < FN; j += 2) {
            float v[8];
#pragma unroll
            for (int r = 0; r < 4; r++) {
              v[r] = acc[i][j][r] + bias[j][r];
              v[r + 4] = acc[i][j + 1][r] + bias[j + 1][r];
            }
            if constexpr (decltype(act_of)::value) gelu8(v);
            if constexpr (type == DT_F32) {
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v4f{v[0], v[1], v[2], v[3]}), to, at[j] + down, 0, 0);
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, v4f{v[4], v[5], v[6], v[7]}), to, at[j + 1] + down, 0, 0);
            } else {
              unsigned h[4];
#pragma unroll
              for (int r = 0; r < 4; r++) h[r] = pack2(v[2 * r], v[2 * r + 1], type);
              const auto lo = __builtin_amdgcn_permlane16_swap(h[0], h[2], false, false);
              const auto hi = __builtin_amdgcn_permlane16_swap(h[1], h[3], false, false);
              __builtin_amdgcn_raw_buffer_store_b128(v4u{lo[0], hi[0], lo[1], hi[1]}, to, at[j] + down, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);  // (all pairs at once would want more registers than there are)
          }
        });
      };
      using F32 = std::integral_constant<int, DT_F32>;
      using F16 = std::integral_constant<int, DT_F16>;
      using BF16 = std::integral_constant<int, DT_BF16>;
      stored = 1;
      if constexpr (!ACT) {  // 16-bit operands: results of their type, or partial sums
        if (P.part) emit(F32{}, std::false_type{});
        else if constexpr (KIND == K_F16) emit(F16{}, std::false_type{});
        else emit(BF16{}, std::false_type{});
      } else if (P.act && !P.part) {  // (rows of no expert: GELU keeps the zero)
        if (type == DT_F32) emit(F32{}, std::true_type{});
        else if (type == DT_F16) emit(F16{}, std::true_type{});
        else emit(BF16{}, std::true_type{});
      } else {
        if (type == DT_F32) emit(F32{}, std::false_type{});
        else if (type == DT_F16) emit(F16{}, std::false_type{});
        else emit(BF16{}, std::false_type{});
      }
      continue;
    }
    // Rows that allow no 16-byte stores: SR rows at a time go through this wave's own strip of LDS; a lane then holds eight
    // consecutive columns of a row.  (The loop is not unrolled: code for all of it would not stay in the instruction cache.)
    constexpr int LR = TN / 8, PASS = 64 / LR > SR ? 1 : SR * LR / 64;  // lanes per row; passes over SR rows
    constexpr int pitch = TN * 4 + 16;                               // (16 bytes between the rows move their banks apart)
    const int crow = lane / LR, ccol = lane % LR * 8, n = w.col0 + wn * TN + ccol;
    float bias[8] = {};
    if (finish && P.bias) {
      if (P.bias_lds) {
        bias8(bias, bias_lds + (num & 3) * (BN * 4), P.bias_type, wn * TN + ccol, BN - 1);
      } else {
        bias8(bias, P.bias, P.bias_type, (long)w.g * P.cols + n, (long)w.g * P.cols + P.cols - 1);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      }
    }
    char* const stage = lds + NB * kBuf + wave * kStage;
    const int have = P.cols - n;
    for (int strip = 0; strip < 16 / SR * FM; strip++) {
      const int orow = orow0 + strip * SR;
      if (orow >= olim) break;
      for_each<FM>([&](auto I) {
        constexpr int i = decltype(I)::value;
        if (strip / (16 / SR) == i && (lane & 15) / SR == strip % (16 / SR)) {
#pragma unroll
          for (int j = 0; j < FN; j++) *(v4f*)(stage + lane % SR * pitch + (j * 16 + 4 * (lane >> 4)) * 4) = acc[i][j];
          asm volatile("; rows %0" ::"n"(i * 16));  // (keeps the branches' ends apart: merged, they would index acc at run time)
        }
      });
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int c = 0; c < PASS; c++) {
        const int row = crow + c * (64 / LR);
        if (row < SR && orow + row < olim && have > 0) {
          const v4f lo = *(const v4f*)(stage + row * pitch + ccol * 4), hi = *(const v4f*)(stage + row * pitch + ccol * 4 + 16);
          float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
          for (int r = 0; r < 8; r++) v[r] += bias[r];
          if (ACT && finish && P.act) gelu8(v);
          store8(out, type, (first + orow + row) * P.cols + n, v, have, P.wide);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
  // the loads behind the last step have written their zeros before the LDS is given back
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

}  // namespace sm3x
