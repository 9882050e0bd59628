// expert_gemm.hip -- 16-bit products grouped by expert: forward (NT), input gradient (NN), weight and bias gradient (TN) of one
// linear layer per expert over expert-major rows of ragged counts.  Engine: expert_tile.h; launch plan: expert_plan.h.
#include "expert_plan.h"

using namespace sm3x;

namespace {

template <int KIND, int MODE>
void launch_mode(const Params& P, const Plan& pl, hipStream_t st) {
  if constexpr (MODE != M_TN) {
    if (pl.coarse) {
      Params Q = P;
      Q.phase = 1;
      tile_kernel<KIND, MODE, 256, 256, 2, 4, 2><<<grid_of(pl, 1), 512, 0, st>>>(Q);
      Q.phase = 2;
      tile_kernel<KIND, MODE, 128, 128, 2, 2, 1, 4><<<kNumCU, 256, 0, st>>>(Q);
      return;
    }
    if (pl.bm == 32) {
      tile_kernel<KIND, MODE, 32, 128, 1, 4, 2><<<grid_of(pl, 3), 256, 0, st>>>(P);
      return;
    }
  }
  tile_kernel<KIND, MODE, 128, 128, 2, 2, 2><<<grid_of(pl, 2), 256, 0, st>>>(P);
}

template <int KIND>
int launch(const Params& P, const Plan& pl, int mode, hipStream_t st) {
  if (mode == SM3_GEMM_NT) launch_mode<KIND, M_NT>(P, pl, st);
  else if (mode == SM3_GEMM_NN) launch_mode<KIND, M_NN>(P, pl, st);
  else launch_mode<KIND, M_TN>(P, pl, st);
  return launch_status();
}

// Rows that the tile kernel cannot read as they are, copied to 16-byte aligned ones with zeros up to the next multiple of 8:
// blocks [0, split) take the first matrix, the others the second.  A copy, bound by launch latency at the sizes it serves (1999 x 203 and
// 585 x 203: 3.4 us).
struct PadRows {
  const uint16_t* src;
  uint16_t* dst;
  long rows, ld;
  int k;
};
__global__ void __launch_bounds__(256) pad_rows_kernel(const PadRows a, const PadRows b, unsigned split) {
  const bool second = blockIdx.x >= split;
  const PadRows m = second ? b : a;
  const unsigned block = second ? blockIdx.x - split : blockIdx.x, blocks = second ? gridDim.x - split : split;
  const int octets = (m.k + 7) / 8;
  const long total = m.rows * octets;
  for (long i = (long)block * 256 + threadIdx.x; i < total; i += (long)blocks * 256) {
    const long row = total < (1L << 31) ? (long)((unsigned)i / (unsigned)octets) : i / octets;
    const int c = (int)(i - row * octets) * 8;
    const uint16_t* at = m.src + row * m.ld + c;
    v8s v;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = c + j < m.k ? (short)at[j] : (short)0;
    *(v8s*)(m.dst + i * 8) = v;
  }
}

unsigned pad_blocks(const PadRows& m) {
  const long b = (m.rows * ((m.k + 7) / 8) + 255) / 256;
  return (unsigned)(b > 8192 ? 8192 : b);
}

}  // namespace

extern "C" {

size_t sm3_expert_gemm_h16_workspace_bytes(const sm3_expert_desc* d) {
  return check_desc(d, false) == SM3_OK ? make_plan(d, false).total() : 0;
}

int sm3_expert_gemm_h16(const sm3_expert_desc* d, void* workspace, size_t workspace_bytes, sm3_stream_t stream) {
  const int err = check_desc(d, false);
  if (err != SM3_OK) return err;
  if (d->mode != SM3_GEMM_TN && d->rows == 0) return SM3_OK;
  const Plan pl = make_plan(d, false);
  const size_t need = pl.total();
  if (!fits(pl)) return SM3_ERR_UNSUPPORTED;
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return SM3_ERR_WORKSPACE;
  const Spaces ws(pl, workspace);
  const Params P = params_of(d, pl, false, ws);
  hipStream_t st = (hipStream_t)stream;
  if (pl.p_bytes || pl.q_bytes) {
    const int prow = d->mode == SM3_GEMM_TN ? d->rows_out : d->red, qrow = d->mode == SM3_GEMM_NT ? d->red : d->cols;
    const long qrows = d->mode == SM3_GEMM_TN ? d->rows : (long)d->num_groups * (d->mode == SM3_GEMM_NT ? d->cols : d->red);
    const PadRows a = {(const uint16_t*)d->p, (uint16_t*)ws.p, pl.p_bytes ? (long)d->rows : 0L, (long)d->ldp, prow};
    const PadRows b = {(const uint16_t*)d->q, (uint16_t*)ws.q, pl.q_bytes ? qrows : 0L, (long)d->ldq, qrow};
    const unsigned na = pad_blocks(a), nb = pad_blocks(b);
    if (na + nb) pad_rows_kernel<<<na + nb, 256, 0, st>>>(a, b, na);
  }
  const int rc = d->type == SM3_DT_F16 ? launch<K_F16>(P, pl, d->mode, st) : launch<K_BF16>(P, pl, d->mode, st);
  return rc != SM3_OK ? rc : finish(P, pl, d, st);
}

}  // extern "C"
