// GEMMs grouped by expert: rows sorted by expert, expert e owning rows offsets[e] .. offsets[e + 1] - 1 (device memory).
//   forward  c[t, n]    = sum over k of a[t, k] * b[e][n, k]          a = x,  b = W
//   dgrad    c[t, k]    = sum over n of a[t, n] * b[e][n, k]          a = dy, b = W
//   wgrad    c[e][n, k] = sum over e's rows t of a[t, n] * b[t, k]    a = dy, b = x
// One launch for all experts; nothing is read back to the host and no workspace is needed, so a launch can be captured.
#include "gemm_tiles.h"

namespace gmd {
namespace tiles {
namespace {

template <typename OUT>
int launch_bf16(int op, const Args& p, hipStream_t st) {
  if (op == GMD_GROUPED_FORWARD) return launch_forward<kBf16, OUT>(p, st);
  if (op == GMD_GROUPED_DGRAD) {
    // As in the forward, but always 64 columns a workgroup: a row of W is read in pieces of that many.  Six waves leave room for two
    // workgroups a CU (64 experts of 4096 x 2048 for 300 rows: 167 us, eight waves 176, four 191); with two blocks of rows and a
    // K of up to 32 steps four are better, three workgroups of which fit (117 experts of 384 x 784 for 2398 rows 21 us, six 38;
    // 64 experts of 2048 x 2048 for 1500 rows 116 and 125; but 8 experts of 4096 x 4096 for 200 rows 59 and 53).
    const int rows = (int)(((int64_t)p.m + p.groups - 1) / p.groups);
    if (rows <= 16) return launch_few<kBf16, false, true, 1, 4, 6, 1, OUT>(p, st);
    if (rows <= 32)
      return p.k <= 32 * 64 ? launch_few<kBf16, false, true, 2, 4, 4, 1, OUT>(p, st) : launch_few<kBf16, false, true, 2, 4, 6, 1, OUT>(p, st);
    if (grid_of(p, 64, 64) <= 2 * kCUs) return launch_few<kBf16, false, true, 4, 4, 4, 1, OUT>(p, st);
    return large_tiles(p, 64) ? launch_tile<kBf16, false, true, 256, 256, 2, 4, OUT>(p, st) : launch_tile<kBf16, false, true, 128, 128, 4, 2, OUT>(p, st);
  }
  if (grid_for(p, true, 64, 64) <= 2 * kCUs) return launch_few<kBf16, true, true, 4, 4, 4, 1, OUT>(p, st);
  Args one = p;  // an expert's share of the rows is its contraction
  one.offsets = nullptr, one.k = (int)(((int64_t)p.k + p.groups - 1) / p.groups);
  const double steps = std::ceil(one.k / 64.0);
  // The last tile may be one of an expert with several times the average's rows (three are assumed): in one or two rounds that
  // decides (32 experts of 976 x 496, 31k rows: small 92 us, large 114; 64 of 512 x 512, 3000 rows: 15 and 22).
  const double large = p.groups * tiles_of(one, 256, 256), most = p.groups > 1 ? 3 * steps : steps;
  if (std::max(TileCost::large(large, steps), TileCost::large(1, most)) >=
      std::max(TileCost::small(p.groups * tiles_of(one, 128, 128), steps), TileCost::small(512, most)))
    return launch_tile<kBf16, true, true, 128, 128, 4, 2, OUT>(p, st);
  // Tiles cost what their experts have of rows.  Walked in fixed turns they save the start of a workgroup each (16 experts of 4096 x
  // 4096, 16k rows: 447 us, 516 one by one; 32 of 2048 x 2048, 16k rows: 169 and 181), but are uneven unless an expert fills
  // whole rounds, the rows are few, or the rounds many (16 experts of 4096 x 2048, 16k rows: 267 and 262; 8 of them, 8k rows: 140
  // and 129; 32 of 1024 x 1024, 8k rows: 41 and 36).
  const bool walk = large >= 256.0 * p.groups || steps <= 2 || (steps <= 8 && large >= 8 * 256);
  return walk ? launch_tile<kBf16, true, true, 256, 256, 2, 4, OUT, true>(p, st) : launch_tile<kBf16, true, true, 256, 256, 2, 4, OUT, false>(p, st);
}

}  // namespace
}  // namespace tiles
}  // namespace gmd

extern "C" {

int gmd_grouped_gemm_launch(const gmd_grouped_gemm_t* g, void* hip_stream) {
  using namespace gmd::tiles;
  auto refuse = [](const char* why) {
    gmd::set_error("grouped GEMM: %s", why);
    return GMD_ERR_BADPARAM;
  };
  if (!g || std::min({g->rows, g->n, g->k, g->groups}) < 0 || std::max({g->rows, g->n, g->k}) > kMaxSize || g->groups > 1 << 20)
    return refuse("negative sizes, sizes over 2^31 - 1024, or more than 2^20 experts");
  if (g->op != GMD_GROUPED_FORWARD && g->op != GMD_GROUPED_DGRAD && g->op != GMD_GROUPED_WGRAD) return refuse("op is forward, dgrad or wgrad");
  if (g->dtype != GMD_DT_BF16 && g->dtype != GMD_DT_FP8) return refuse("operands are bf16 or fp8");
  if (g->out_dtype != GMD_DT_BF16 && g->out_dtype != GMD_DT_F32) return refuse("the result is bf16 or f32");
  const bool fp8 = g->dtype == GMD_DT_FP8, wgrad = g->op == GMD_GROUPED_WGRAD, dgrad = g->op == GMD_GROUPED_DGRAD;
  if (fp8 && g->op != GMD_GROUPED_FORWARD)
    return refuse("fp8 runs forward only: the input gradient is a forward with transposed weights, the weight gradient is taken in bf16");
  if (g->n % 8 || g->k % (fp8 ? 16 : 8)) return refuse("N in multiples of 8, K in multiples of 8 (bf16) or 16 (fp8)");
  const int elem = fp8 ? 1 : 2, out = g->out_dtype == GMD_DT_BF16 ? 2 : 4;
  const int64_t kb = ((int64_t)g->k + 127) / 128, nb = ((int64_t)g->n + 127) / 128;
  const int64_t a_cols = g->op == GMD_GROUPED_FORWARD ? g->k : g->n;
  const int64_t c_cols = g->op == GMD_GROUPED_FORWARD ? g->n : g->k;
  if (c_cols == 0 || g->groups == 0 || (wgrad ? g->n : g->rows) == 0) return GMD_OK;  // an empty result
  if (!g->offsets || ((uintptr_t)g->offsets & 3)) return refuse("null or misaligned offsets");
  const int64_t lda = g->lda ? g->lda : a_cols, ldb = g->ldb ? g->ldb : g->k, ldc = g->ldc ? g->ldc : c_cols;
  const int64_t stride_w = g->stride_w ? g->stride_w : (int64_t)g->n * (wgrad ? ldc : ldb);
  const char* bad = bad_operand(g->c, ldc, c_cols, out);
  if (!bad && a_cols > 0 && g->rows > 0) bad = bad_operand(g->a, lda, a_cols, elem);
  if (!bad && (wgrad ? g->rows > 0 : g->n > 0 && g->k > 0)) bad = bad_operand(g->b, ldb, g->k, elem);
  if (!bad && (stride_w * (wgrad ? out : elem) % 16 || stride_w < (int64_t)(g->n - 1) * (wgrad ? ldc : ldb) + g->k))
    bad = "an expert stride that is not a multiple of 16 bytes or shorter than an expert";
  Args p;
  memset(&p, 0, sizeof p);
  p.a = (const char*)g->a, p.b = (const char*)g->b, p.c = g->c, p.offsets = g->offsets, p.groups = g->groups;
  p.lda = lda * elem, p.ldb = ldb * elem, p.ldc = ldc;
  if (wgrad) {
    p.m = g->n, p.n = g->k, p.k = g->rows, p.stride_c = stride_w;
  } else {
    p.m = g->rows, p.n = dgrad ? g->k : g->n, p.k = dgrad ? g->n : g->k, p.stride_b = stride_w * elem;
  }
  if (fp8 && !bad && g->k > 0) {
    p.sa = g->scale_a, p.sb = g->scale_b;
    p.ld_sa = g->ld_scale_a ? g->ld_scale_a : g->rows;
    p.ld_sb = g->ld_scale_b ? g->ld_scale_b : kb;
    p.stride_sb = g->stride_scale ? g->stride_scale : nb * p.ld_sb;
    if (!p.sa || !p.sb || (((uintptr_t)p.sa | (uintptr_t)p.sb) & 3)) bad = "null or misaligned scales";
    else if (p.ld_sa < g->rows || p.ld_sb > 1 << 28 || p.ld_sb < kb || p.stride_sb < (nb - 1) * p.ld_sb + kb) bad = "a stride of scales shorter than what it spans, or over 2^28";
  }
  if (!bad) bad = gmd::elsewhere((hipStream_t)hip_stream, {g->a, g->b, g->c, g->offsets, p.sa, p.sb});
  if (bad) return refuse(bad);
  if (fp8) return launch_fp8(p, GMD_BLOCK_TILES, g->out_dtype, (hipStream_t)hip_stream);
  return g->out_dtype == GMD_DT_BF16 ? launch_bf16<__bf16>(g->op, p, (hipStream_t)hip_stream)
                                     : launch_bf16<float>(g->op, p, (hipStream_t)hip_stream);
}

}  // extern "C"
