// GEMM of e4m3 operands with one f32 scale per block of 128 (see gemm_tiles.h for the kernels):
//   C[m, n] = sum over blocks kb of sa[kb][m] * sb(kb, n) * (sum over the block's k of A[m, k] * B[n, k])
// A's scales are per row, B's per 128 x 128 tile (a weight: forward and input gradient) or per row (weight gradient).
#include "gemm_tiles.h"

namespace gmd {
namespace tiles {

int launch_fp8(const Args& p, int b_blocks, int out_dtype, hipStream_t st) {
  if (b_blocks == GMD_BLOCK_TILES)
    return out_dtype == GMD_DT_BF16 ? launch_forward<kFp8Tiles, __bf16>(p, st) : launch_forward<kFp8Tiles, float>(p, st);
  return out_dtype == GMD_DT_BF16 ? launch_forward<kFp8Rows, __bf16>(p, st) : launch_forward<kFp8Rows, float>(p, st);
}

}  // namespace tiles
}  // namespace gmd

extern "C" {

int gmd_gemm_block_launch(const gmd_gemm_block_t* g, void* hip_stream) {
  using namespace gmd::tiles;
  if (!g || g->m < 0 || g->n < 0 || g->k < 0 || std::max({g->m, g->n, g->k}) > kMaxSize) {
    gmd::set_error("block GEMM: negative sizes, or sizes over 2^31 - 1024");
    return GMD_ERR_BADPARAM;
  }
  if (g->n % 8 || g->k % 16) {
    gmd::set_error("block GEMM shape: N in multiples of 8, K in multiples of 16 (gmd_block_quantize pads rows to 16 with zeros)");
    return GMD_ERR_BADPARAM;
  }
  if ((g->b_blocks != GMD_BLOCK_ROWS && g->b_blocks != GMD_BLOCK_TILES) || (g->out_dtype != GMD_DT_BF16 && g->out_dtype != GMD_DT_F32)) {
    gmd::set_error("block GEMM: B's blocks are rows or tiles, the result is bf16 or f32");
    return GMD_ERR_BADPARAM;
  }
  if (g->m == 0 || g->n == 0) return GMD_OK;
  const int64_t kb = ((int64_t)g->k + 127) / 128;
  Args p;
  memset(&p, 0, sizeof p);
  p.m = g->m, p.n = g->n, p.k = g->k, p.groups = 1;
  p.lda = g->lda ? g->lda : g->k, p.ldb = g->ldb ? g->ldb : g->k, p.ldc = g->ldc ? g->ldc : g->n;
  p.ld_sa = g->ld_scale_a ? g->ld_scale_a : g->m;
  p.ld_sb = g->ld_scale_b ? g->ld_scale_b : g->b_blocks == GMD_BLOCK_TILES ? kb : g->n;
  p.a = (const char*)g->a, p.b = (const char*)g->b, p.c = g->c, p.sa = g->scale_a, p.sb = g->scale_b;
  const char* bad = bad_operand(g->c, p.ldc, g->n, g->out_dtype == GMD_DT_BF16 ? 2 : 4);
  if (!bad && g->k > 0) {
    bad = bad_operand(g->a, p.lda, g->k, 1);
    if (!bad) bad = bad_operand(g->b, p.ldb, g->k, 1);
    if (!bad && (!p.sa || !p.sb || (((uintptr_t)p.sa | (uintptr_t)p.sb) & 3))) bad = "null or misaligned scales";
    if (!bad && (p.ld_sa < g->m || p.ld_sb > 1 << 28 || p.ld_sb < (g->b_blocks == GMD_BLOCK_TILES ? kb : g->n))) bad = "a stride of scales shorter than what it spans, or over 2^28";
  }
  if (!bad) bad = gmd::elsewhere((hipStream_t)hip_stream, {g->a, g->b, g->c, p.sa, p.sb});
  if (bad) {
    gmd::set_error("block GEMM: %s", bad);
    return GMD_ERR_BADPARAM;
  }
  return launch_fp8(p, g->b_blocks, g->out_dtype, (hipStream_t)hip_stream);
}

}  // extern "C"
