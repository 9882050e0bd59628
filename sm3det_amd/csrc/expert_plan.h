// expert_plan.h -- host side of the grouped products: checks, launch shapes, workspaces, the joins of split reductions.
#pragma once
#include "expert_tile.h"

namespace sm3x {

// rows a grid has to provide for: every expert may end in a part-filled tile, and so may the rows before the first and behind
// the last expert
inline long row_tiles(long S, int G, bool grouped, long bm) {
  if (!grouped) return (S + bm - 1) / bm;
  return S / bm + (S < G ? S : G) + 2;
}

struct Plan {
  int bm, bn;          // tile
  long mtiles, per_xcd;  // row tiles; jobs of one XCD
  int ntiles, splits;  // NT / NN: slices of the reduction
  bool coarse;         // NT / NN: 256 x 256 tiles, the last partial round in quarters
  long unit_rows, units;  // TN: reduction rows per work unit
  size_t part_bytes, bsum_bytes;
  // copies of the operands made first: padded rows (16-bit), packed rows (4-bit; codes, then scales)
  size_t p_bytes, p_scale_bytes, q_bytes;
  size_t total() const { return part_bytes + bsum_bytes + p_bytes + p_scale_bytes + q_bytes; }
};

// elements of an operand's row (16 bits), and between rows: byte offsets inside a tile of up to 256 rows have 31 bits
constexpr long kMostElements = 1L << 22;

// A grid's first dimension holds fewer than 2^32 threads; a launch of more ends without an error and without its work.
inline bool launchable(long blocks, long threads) { return blocks * threads < 1L << 32; }

// workgroups per XCD: as many as are resident at once, each with its share of the jobs -- at most kMaxJobs of them
inline long workgroups(const Plan& pl, int per_cu) {
  const long most = (long)kNumCU / kNumXCD * per_cu, least = (pl.per_xcd + kMaxJobs - 1) / kMaxJobs;
  return pl.per_xcd < most ? pl.per_xcd : most > least ? most : least;
}

// jobs are counted in 31 bits
inline bool fits(const Plan& p) {
  return (double)p.per_xcd * kNumXCD < 2.0e9 && (double)p.units < 2.0e9 && launchable(workgroups(p, 3) * kNumXCD, p.coarse ? 512 : 256);
}

inline int check_desc(const sm3_expert_desc* d, bool mx4) {
  if (!d || d->num_groups < 1 || d->rows < 0 || d->rows > 0x7fffff00L || d->red < 1 || d->cols < 1) return SM3_ERR_INVALID_ARG;
  if (d->mode < SM3_GEMM_NT || d->mode > SM3_GEMM_TN || (mx4 && d->mode != SM3_GEMM_NT)) return SM3_ERR_INVALID_ARG;
  if (!d->offsets && d->num_groups != 1) return SM3_ERR_INVALID_ARG;
  if (d->num_groups > 65535) return SM3_ERR_UNSUPPORTED;  // (a dimension of a grid)
  if (d->act < 0 || d->act > 1 || d->bias_type < 0 || d->bias_type > SM3_DT_BF16) return SM3_ERR_INVALID_ARG;
  if (d->out_type < 0 || d->out_type > SM3_DT_BF16) return SM3_ERR_INVALID_ARG;
  if (d->mode == SM3_GEMM_TN ? d->rows_out < 1 || d->bias || d->act : d->bias_grad != nullptr) return SM3_ERR_INVALID_ARG;
  const bool reads = d->rows > 0;  // (a weight gradient over no rows writes zeros)
  if (!d->out || (reads && (!d->p || !d->q))) return SM3_ERR_INVALID_ARG;
  const long prow = d->mode == SM3_GEMM_TN ? d->rows_out : d->red, qrow = d->mode == SM3_GEMM_NT ? d->red : d->cols;
  if (prow > kMostElements || qrow > kMostElements || d->cols > 1 << 30) return SM3_ERR_UNSUPPORTED;
  if (mx4) {
    if (!d->q_scales || (uintptr_t)d->q % 16 || (uintptr_t)d->q_scales % 4) return SM3_ERR_INVALID_ARG;
    if (d->p_scales) {
      if ((uintptr_t)d->p % 16 || (uintptr_t)d->p_scales % 4) return SM3_ERR_INVALID_ARG;
    } else if (d->type < 0 || d->type > SM3_DT_BF16 || d->ldp < d->red) {
      return SM3_ERR_INVALID_ARG;
    }
  } else {
    if (d->type != SM3_DT_F16 && d->type != SM3_DT_BF16) return SM3_ERR_INVALID_ARG;
    if (d->out_type != d->type || d->act) return SM3_ERR_INVALID_ARG;
    if (d->ldp < prow || d->ldq < qrow) return SM3_ERR_INVALID_ARG;
  }
  return SM3_OK;
}

// rows the tile kernel can read as they are
inline bool readable(const void* p, long ld, long row) {
  return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && row % 8 == 0 && ld <= kMostElements;
}

inline Plan plan_tiles(const sm3_expert_desc* d, bool mx4) {
  Plan p{};
  const bool grouped = d->offsets != nullptr;
  if (d->mode == SM3_GEMM_TN) {
    p.bm = p.bn = 128;
    p.ntiles = (d->cols + p.bn - 1) / p.bn;
    const long mt = (d->rows_out + p.bm - 1) / p.bm, tiles = mt * p.ntiles;
    // too few tiles to fill the chip: the reduction is cut into units whose fp32 partials a second launch adds in order
    p.unit_rows = d->rows > 0 ? d->rows : 1;
    p.units = d->num_groups;
    if (tiles * d->num_groups < 2 * kNumCU) {
      long want = (3L * kNumCU + tiles - 1) / tiles;
      long r = (d->rows + want - 1) / want;
      r = (r + kStepRed - 1) / kStepRed * kStepRed;
      if (r < 4 * kStepRed) r = 4 * kStepRed;
      if (r < d->rows) {
        p.unit_rows = r;
        p.units = d->rows / r + d->num_groups;
        p.part_bytes = align_up((size_t)p.units * d->rows_out * d->cols * 4, 256);
        if (d->bias_grad) p.bsum_bytes = align_up((size_t)p.units * d->rows_out * 4, 256);
      }
    }
    p.mtiles = p.units * mt;
    p.splits = 1;
    p.per_xcd = p.units * ((tiles + kNumXCD - 1) / kNumXCD);
    return p;
  }
  const long per_expert = d->rows / (d->num_groups < d->rows ? d->num_groups : d->rows > 0 ? d->rows : 1);
  p.bm = per_expert <= 48 ? 32 : 128;
  p.bn = 128;
  // Much work per CU: 256 x 256 tiles move half the bytes per product through L2, but a partial last round costs a whole one, so
  // that one runs in quarters in a second launch.  Measured over 4096 to 65536 rows of 8 uneven experts, 256 to 4096 columns and
  // reductions of 512 to 4096, bf16, the same operands call after call: where the rule takes them they need 0.77 to 1.02 of the time of
  // 128 x 128 tiles (16384 rows, 4096 x 1024: 153 -> 136 us, 4096 x 4096: 564 -> 485; 65536 rows, 1024 x 4096: 628 -> 485).  Where it
  // does not: 1.0 to 1.25 with one to two rounds of 8 or 16 steps (16384 rows, 2048 x 512: 46 -> 51), up to 3.3 with less than
  // one; a handful of sizes next to its border would have gained up to 14 % (32768 rows, 256 x 4096: 119 -> 103).  (The rounds are
  // whole ones: a quotient without its rest.)
  const long red_steps = ((mx4 ? (d->red + 127) / 128 * 64 : d->red * 2L) + kStepBytes - 1) / kStepBytes;
  const long some = d->offsets ? (d->num_groups < d->rows ? d->num_groups : d->rows) / 2 : 0;  // half a tile is lost per expert
  const long expected = ((d->rows + 255) / 256 + some) * ((d->cols + 255L) / 256);
  // (256 rows of the longest reduction would be 2^31 bytes, one more than a tile's range counts: 128 x 128 tiles)
  const bool countable = d->red <= kMostElements - 8;
  if (!mx4 && countable && expected / kNumCU * red_steps >= 48 && red_steps >= 8 && d->cols % 256 == 0) {
    p.coarse = true;
    p.bm = p.bn = 256;
  }
  p.ntiles = (d->cols + p.bn - 1) / p.bn;
  p.mtiles = row_tiles(d->rows, d->num_groups, grouped, p.bm);
  p.splits = 1;
  const long steps = ((mx4 ? (d->red + 127) / 128 * 64 : d->red * 2L) + kStepBytes - 1) / kStepBytes;
  const long tiles = p.mtiles * p.ntiles;
  if (tiles < kNumCU && steps >= 8) {
    long s = (2L * kNumCU + tiles - 1) / tiles;
    if (s > steps / 4) s = steps / 4;
    if (s > 16) s = 16;
    if (s > 1) {
      p.splits = (int)s;
      p.part_bytes = align_up((size_t)s * d->rows * d->cols * 4, 256);
    }
  }
  p.per_xcd = (tiles * p.splits + kNumXCD - 1) / kNumXCD;
  return p;
}

inline Plan make_plan(const sm3_expert_desc* d, bool mx4) {
  Plan p = plan_tiles(d, mx4);
  if (mx4) {
    if (!d->p_scales) {
      const size_t kp = ((size_t)d->red + 127) / 128 * 128;
      p.p_bytes = align_up(d->rows * kp / 2, 256);
      p.p_scale_bytes = align_up(d->rows * kp / 32, 256);
    }
  } else {
    const long prow = d->mode == SM3_GEMM_TN ? d->rows_out : d->red, qrow = d->mode == SM3_GEMM_NT ? d->red : d->cols;
    const long qrows = d->mode == SM3_GEMM_TN ? d->rows : (long)d->num_groups * (d->mode == SM3_GEMM_NT ? d->cols : d->red);
    if (!readable(d->p, d->ldp, prow)) p.p_bytes = align_up((size_t)d->rows * ((prow + 7) / 8 * 8) * 2, 256);
    if (!readable(d->q, d->ldq, qrow)) p.q_bytes = align_up((size_t)qrows * ((qrow + 7) / 8 * 8) * 2, 256);
  }
  return p;
}

// ---- joins --------------------------------------------------------------------------------------------------------
// out[s][n] = act(sum over slices + bias of the row's expert); eight columns of a row per thread.  Bound by latency: the rows are
// few where the reduction is sliced.
static __global__ void __launch_bounds__(256) join_rows_kernel(const Params P) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 8, lane = threadIdx.x & 63;
  for (long s = blockIdx.y; s < P.S; s += gridDim.y) {
    int g = P.offsets ? -1 : 0;
    if (P.offsets) {  // first expert whose end lies behind the row
      for (int b = 0; b < P.G && g < 0; b += 64) {
        const unsigned long long hit = __ballot(b + lane < P.G && P.offsets[b + lane + 1] > s);
        if (hit) g = b + __ffsll(hit) - 1;
      }
      if (s < P.offsets[0]) g = -1;
    }
    if (n >= P.cols) continue;
    const int have = P.cols - n;
    float v[8] = {};
    for (int z = 0; z < P.splits; z++) {
      const float* at = P.part + ((long)z * P.S + s) * P.cols + n;
#pragma unroll
      for (int r = 0; r < 8; r++) v[r] += r < have ? at[r] : 0.f;
    }
    if (g >= 0) {
      if (P.bias) {
        float b[8];
        bias8(b, P.bias, P.bias_type, (long)g * P.cols + n, (long)g * P.cols + P.cols - 1);
#pragma unroll
        for (int r = 0; r < 8; r++) v[r] += b[r];
      }
      if (P.act) gelu8(v);
    }
    store8(P.out, P.out_type, s * P.cols + n, v, have, P.cols % (P.out_type == DT_F32 ? 4 : 8) == 0 && (uintptr_t)P.out % 16 == 0);
  }
}

// out[g][i] = sum over the work units of expert g, in their order; `n` values per unit.  Blocks [0, split) of a row of the grid
// join the weight gradient's partials, the others the bias gradient's.  Bound by reading the partials (65536 rows cut into about 55
// units of 1 MB: 11 us).
struct Join {
  const float* part;
  void* out;
  int type;
  long n;
};
static __global__ void __launch_bounds__(256) join_units_kernel(const Params P, const Join a, const Join b, unsigned split) {
  const Join J = blockIdx.x < split ? a : b;
  const float* const part = J.part;
  const long n = J.n;
  const int g = blockIdx.y, lane = threadIdx.x & 63;
  long first = 0;
  int count = 0;
  const int S = (int)P.S;
  if (P.offsets == nullptr) {
    count = S > 0 ? (int)((S + P.unit_rows - 1) / P.unit_rows) : 1;
  } else {
    int carry = P.offsets[0];
    carry = carry < 0 ? 0 : carry > S ? S : carry;
    for (int b = 0; b <= g; b += 64) {
      int end = b + lane < P.G ? P.offsets[b + lane + 1] : 0;
      end = end < 0 ? 0 : end > S ? S : end;
      end = end < carry ? carry : end;
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(end, d);
        if (lane >= d && o > end) end = o;
      }
      int start = __shfl_up(end, 1);
      if (lane == 0) start = carry;
      int u = b + lane < P.G ? (int)((end - start + P.unit_rows - 1) / P.unit_rows) : 0;
      if (b + lane < P.G && u == 0) u = 1;
      int incl = u;
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
      }
      if (g < b + 64) {
        count = __shfl(u, g - b);
        first += __shfl(incl, g - b) - count;
      } else {
        first += __shfl(incl, 63);
        carry = __shfl(end, 63);
      }
    }
  }
  const long i = ((long)(blockIdx.x < split ? blockIdx.x : blockIdx.x - split) * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  const int have = (int)(n - i < 8 ? n - i : 8);
  float v[8] = {};
  const bool whole = n % 8 == 0;
  for (int u = 0; u < count; u++) {
    const float* at = part + (first + u) * n + i;
    if (whole) {
      const v4f lo = *(const v4f*)at, hi = *(const v4f*)(at + 4);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        v[r] += lo[r];
        v[r + 4] += hi[r];
      }
    } else {
#pragma unroll
      for (int r = 0; r < 8; r++) v[r] += r < have ? at[r] : 0.f;
    }
  }
  store8(J.out, J.type, (long)g * n + i, v, have, whole && (uintptr_t)J.out % 16 == 0);
}

// parts of the workspace
struct Spaces {
  char *p, *p_scales, *q;
  float *part, *bsum;
  Spaces(const Plan& pl, void* ws) {
    char* at = (char*)ws;
    p = at;
    p_scales = (at += pl.p_bytes);
    q = (at += pl.p_scale_bytes);
    part = pl.part_bytes ? (float*)(at + pl.q_bytes) : nullptr;
    bsum = pl.bsum_bytes ? (float*)(at + pl.q_bytes + pl.part_bytes) : nullptr;
  }
};

inline Params params_of(const sm3_expert_desc* d, const Plan& pl, bool mx4, const Spaces& ws) {
  Params P{};
  P.p = pl.p_bytes ? ws.p : (const char*)d->p;
  P.q = pl.q_bytes ? ws.q : (const char*)d->q;
  P.S = d->rows;
  P.G = d->num_groups;
  P.offsets = d->offsets;
  P.out = d->out;
  P.out_type = d->out_type;
  P.bias = d->bias;
  P.bias_type = d->bias_type;
  P.act = d->act;
  P.cols = d->cols;
  P.rows_out = d->rows_out;
  if (mx4) {
    const long kp = (d->red + 127) / 128 * 128;
    P.ldp = P.ldq = P.red = kp / 2;
    P.ldps = P.ldqs = kp / 32;
    P.strideq = d->cols * P.ldq;
    P.strideqs = d->cols * P.ldqs;
    P.ps = pl.p_scale_bytes ? (const unsigned char*)ws.p_scales : d->p_scales;
    P.qs = d->q_scales;
  } else {
    const long prow = d->mode == SM3_GEMM_TN ? d->rows_out : d->red, qrow = d->mode == SM3_GEMM_NT ? d->red : d->cols;
    P.ldp = pl.p_bytes ? (prow + 7) / 8 * 16 : d->ldp * 2;
    P.ldq = pl.q_bytes ? (qrow + 7) / 8 * 16 : d->ldq * 2;
    P.red = d->red * 2L;
    P.qred = d->red;
    P.strideq = (d->mode == SM3_GEMM_NT ? (long)d->cols : (long)d->red) * P.ldq;
    // (rows whose length is no multiple of 8 are padded copies: the granule at the end of the reduction holds zeros)
    if (d->mode != SM3_GEMM_TN) P.red = (P.red + 15) & ~15L;
  }
  P.ntiles = pl.ntiles;
  P.splits = pl.splits;
  P.unit_rows = pl.unit_rows;
  P.part = ws.part;
  const long bes = d->bias_type == SM3_DT_F32 ? 4 : 2;
  P.bias_lds = d->bias && (uintptr_t)d->bias % 4 == 0 && d->cols * bes % 4 == 0 && d->cols * bes < 1L << 32;
  P.wide = P.part ? d->cols % 4 == 0 : d->cols % (d->out_type == SM3_DT_F32 ? 4 : 8) == 0 && (uintptr_t)d->out % 16 == 0;
  if (d->cols > 1 << 20) P.wide = 0;  // (those stores address a tile's 128 rows with 31 bits)
  P.bsum = ws.bsum;
  P.db = d->bias_grad;
  return P;
}

inline dim3 grid_of(const Plan& pl, int per_cu) { return dim3((unsigned)(workgroups(pl, per_cu) * kNumXCD)); }

inline int finish(const Params& P, const Plan& pl, const sm3_expert_desc* d, hipStream_t st) {
  if (d->mode == SM3_GEMM_TN) {
    if (!P.part) return SM3_OK;
    const long n = (long)P.rows_out * P.cols;
    const Join w = {P.part, P.out, P.out_type, n}, b = {P.bsum, d->bias_grad, d->bias_type, P.rows_out};
    const unsigned nw = (unsigned)((n + 2047) / 2048), nb = P.bsum ? (unsigned)((P.rows_out + 2047) / 2048) : 0;
    join_units_kernel<<<dim3(nw + nb, P.G), 256, 0, st>>>(P, w, b, nw);
  } else if (P.part) {
    join_rows_kernel<<<dim3((unsigned)((P.cols + 2047) / 2048), (unsigned)(P.S < 32768 ? P.S : 32768)), 256, 0, st>>>(P);
  }
  return launch_status();
}

}  // namespace sm3x
