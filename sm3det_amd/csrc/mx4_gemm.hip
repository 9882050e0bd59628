// mx4_gemm.hip -- products of microscaled 4-bit rows, dense and grouped by expert: v_mfma_scale_f32_16x16x128_f8f6f4 with both
// operands e2m1 and the blocks' scale bytes as its scale operands (no dequantised copy exists anywhere).
#include "expert_plan.h"
#include "mx4_few.h"

using namespace sm3x;

namespace {

// A handful of rows, not yet quantised: one launch without a workspace (mx4_few.hip).  Up to 16 rows an expert's rows are one tile
// there.  Every 16 columns of every tile quantise their rows again, so its time grows with tiles x columns x reduction (the tiles as
// the host can bound them: the rows' spread over the experts is known to the device alone), while quantisation, tile kernel and their
// host side cost about 13 us from the start.  Measured on 2 to 64 experts, 64 x 64 to 4096 x 1024, bf16 / fp32 rows, us per call
// back to back, here against there: up to 1 M of that product 9 against 13.5; 8 experts, 64 rows, 4096 x 1024 (3.1 M) 12.6 / 17.3
// against 13.8 / 15.2; 16 experts, 256 rows, 2048 x 512 (2.1 M) 14.4 / 23.8 against 13.5 / 15.7; 64 experts, 1000 rows, 4096 x
// 1024 (33 M) 102 / 188 against 30 / 31.
bool few(const sm3_expert_desc* d) {
  const long experts = d->num_groups < d->rows ? d->num_groups : d->rows;
  if (d->p_scales || d->rows > 16 * experts) return false;
  if (row_tiles(d->rows, d->num_groups, d->offsets != nullptr, 16) >= 65536 || !launchable((d->cols + 15) / 16, 256)) return false;
  const double work = (double)(d->rows / 16 + experts) * ((d->cols + 15) / 16) * ((d->red + 127) / 128 * 128);
  return d->rows <= 16 || work <= (d->type == SM3_DT_F32 ? 2.5e6 : 3.4e6);
}

}  // namespace

extern "C" {

size_t sm3_mx4_gemm_workspace_bytes(const sm3_expert_desc* d) {
  return check_desc(d, true) == SM3_OK && !few(d) ? make_plan(d, true).total() : 0;
}

int sm3_mx4_gemm(const sm3_expert_desc* d, void* workspace, size_t workspace_bytes, sm3_stream_t stream) {
  const int err = check_desc(d, true);
  if (err != SM3_OK) return err;
  if (d->rows == 0) return SM3_OK;
  if (few(d)) {
    const Few f = {d->p, d->ldp, (const unsigned char*)d->q, d->q_scales, d->red, (d->red + 127) / 128 * 128, d->cols,
                   d->num_groups, (int)d->rows, d->offsets, d->bias, d->bias_type, d->act, d->out_type, d->out};
    return launch_few(f, d->type, row_tiles(d->rows, d->num_groups, d->offsets != nullptr, 16), (hipStream_t)stream);
  }
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
