// expert_gemm.hip -- 16-bit products grouped by expert: forward (NT), input gradient (NN), weight and bias gradient (TN) of one
// linear layer per expert over expert-major rows of ragged counts.  Engine: expert_tile.h; launch plan: expert_plan.h.
#include "expert_plan.h"

using namespace sm3x;

namespace {

template <int KIND, int MODE>
void launch_mode(const Params& P, const Plan& pl, hipStream_t st) {
  if (MODE != M_TN && pl.bm == 32) tile_kernel<KIND, MODE == M_TN ? M_NT : MODE, 32, 128, 1, 4, 2><<<grid_of(pl, 3), 256, 0, st>>>(P);
  else tile_kernel<KIND, MODE, 128, 128, 2, 2, 2><<<grid_of(pl, 2), 256, 0, st>>>(P);
}

template <int KIND>
int launch(const Params& P, const Plan& pl, int mode, hipStream_t st) {
  if (mode == SM3_GEMM_NT) launch_mode<KIND, M_NT>(P, pl, st);
  else if (mode == SM3_GEMM_NN) launch_mode<KIND, M_NN>(P, pl, st);
  else launch_mode<KIND, M_TN>(P, pl, st);
  return launch_status();
}

__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* __restrict__ src, long rows, int k, long ld,
                                                       uint16_t* __restrict__ dst, int octets) {
  const long total = rows * octets;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
    const long row = i / octets;
    const int c = (int)(i - row * octets) * 8;
    const uint16_t* at = src + row * ld + c;
    v8s v;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = c + j < k ? (short)at[j] : (short)0;
    *(v8s*)(dst + i * 8) = v;
  }
}

}  // namespace

extern "C" {

size_t sm3_expert_gemm_h16_workspace_bytes(const sm3_expert_desc* d) {
  if (check_desc(d, false) != SM3_OK) return 0;
  const Plan pl = make_plan(d, false);
  return pl.part_bytes + pl.bsum_bytes;
}

int sm3_expert_gemm_h16(const sm3_expert_desc* d, void* workspace, size_t workspace_bytes, sm3_stream_t stream) {
  const int err = check_desc(d, false);
  if (err != SM3_OK) return err;
  if (d->mode != SM3_GEMM_TN && d->rows == 0) return SM3_OK;
  const Plan pl = make_plan(d, false);
  const size_t need = pl.part_bytes + pl.bsum_bytes;
  if (!fits(pl)) return SM3_ERR_UNSUPPORTED;
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return SM3_ERR_WORKSPACE;
  const Params P = params_of(d, pl, false, workspace);
  hipStream_t st = (hipStream_t)stream;
  const int rc = d->type == SM3_DT_F16 ? launch<K_F16>(P, pl, d->mode, st) : launch<K_BF16>(P, pl, d->mode, st);
  return rc != SM3_OK ? rc : finish(P, pl, d, st);
}

int sm3_pad_rows_h16(const void* src, long rows, int k, long ld, void* dst, int kp, sm3_stream_t stream) {
  if (rows < 0 || k < 1 || ld < k || kp < k || kp % 8) return SM3_ERR_INVALID_ARG;
  if (rows == 0) return SM3_OK;
  if (!src || !dst || (uintptr_t)dst % 16) return SM3_ERR_INVALID_ARG;
  const long blocks = (rows * (kp / 8) + 255) / 256;
  pad_rows_kernel<<<(unsigned)(blocks > 16384 ? 16384 : blocks), 256, 0, (hipStream_t)stream>>>(
      (const uint16_t*)src, rows, k, ld, (uint16_t*)dst, kp / 8);
  return launch_status();
}

}  // extern "C"
