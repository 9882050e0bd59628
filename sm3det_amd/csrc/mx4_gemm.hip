// mx4_gemm.hip -- products of microscaled 4-bit rows, dense and grouped by expert: v_mfma_scale_f32_16x16x128_f8f6f4 with both
// operands e2m1 and the blocks' scale bytes as its scale operands (no dequantised copy exists anywhere).
#include "expert_plan.h"

using namespace sm3x;

extern "C" {

size_t sm3_mx4_gemm_workspace_bytes(const sm3_expert_desc* d) {
  return check_desc(d, true) == SM3_OK ? make_plan(d, true).total() : 0;
}

int sm3_mx4_gemm(const sm3_expert_desc* d, void* workspace, size_t workspace_bytes, sm3_stream_t stream) {
  const int err = check_desc(d, true);
  if (err != SM3_OK) return err;
  if (d->rows == 0) return SM3_OK;
  const Plan pl = make_plan(d, true);
  if (!fits(pl)) return SM3_ERR_UNSUPPORTED;
  const size_t need = pl.total();
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return SM3_ERR_WORKSPACE;
  const Spaces ws(pl, workspace);
  const Params P = params_of(d, pl, true, ws);
  hipStream_t st = (hipStream_t)stream;
  if (pl.p_bytes) {
    const int rc = sm3_mx4_quantize(d->p, d->type, d->rows, d->red, d->ldp, (uint8_t*)ws.p, (uint8_t*)ws.p_scales, stream);
    if (rc != SM3_OK) return rc;
  }
  if (pl.bm == 32) tile_kernel<K_MX4, M_NT, 32, 128, 1, 4, 2><<<grid_of(pl, 3), 256, 0, st>>>(P);
  else tile_kernel<K_MX4, M_NT, 128, 128, 2, 2, 2><<<grid_of(pl, 2), 256, 0, st>>>(P);
  const int rc = launch_status();
  return rc != SM3_OK ? rc : finish(P, pl, d, st);
}

}  // extern "C"
