// Quantisation to e4m3 with one f32 scale per block of 128 (the operands of block_gemm.hip and grouped_gemm.hip).
//   amax = max |x| over the block, at least 2^-96;  scale = f32(amax / 448);  q = e4m3(f32(x * f32(448 / amax)))
// 448 is e4m3's largest value, so the block's largest element maps onto it; rounding is to nearest, ties to even.
// The floor of 2^-96 keeps 448 / amax finite; a block of zeros gets the scale 2^-96 / 448 and zeros.  amax is taken on the
// bit patterns, where NaN > infinity > every number: a block that holds an infinity or a NaN gets an infinite or NaN scale,
// and every product that reads it becomes NaN.
#include "diag_common.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr unsigned kAmaxMin = (127u - 96u) << 23;  // 2^-96

__device__ __forceinline__ void scale_of(unsigned amax_bits, float* scale, float* inv) {
  const float amax = __builtin_bit_cast(float, max(amax_bits, kAmaxMin));
  *scale = amax / 448.f;
  *inv = 448.f / amax;
}

__device__ __forceinline__ unsigned magnitude(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

struct QuantArgs {
  const char* src;
  uint8_t* dst;
  float* scales;
  int64_t ld_src, ld_dst, ld_scales;  // elements
  int rows, cols;                     // of src
  int vec;                            // src rows can be read in 16-byte pieces
};

// A workgroup takes one 128 x 128 region of src into registers: thread t holds eight consecutive columns 8 (t % 16) of rows
// t / 16 + 16 i.  That fits all four forms: a row's block lies in 16 neighbouring lanes, a column's in the 16 row groups of
// four waves, a tile in the workgroup.
template <typename SRC, bool TILES, bool TRANS>
__global__ __launch_bounds__(256) void quantize_kernel(QuantArgs p) {
  constexpr int kRows = 8;
  const int t = threadIdx.x, c16 = t & 15, rg = t >> 4;
  const int regions_c = (p.cols + 127) / 128;
  const int br = blockIdx.x / regions_c, bc = blockIdx.x % regions_c;
  const int col = bc * 128 + c16 * 8;
  __shared__ unsigned red[16][132];
  __shared__ __attribute__((aligned(16))) uint8_t turned[TRANS ? 128 * 144 : 16];

  float x[kRows][8];
#pragma unroll
  for (int i = 0; i < kRows; i++) {
    const int row = br * 128 + rg + 16 * i;
    const SRC* s = (const SRC*)p.src + (int64_t)row * p.ld_src + col;
    if (row < p.rows && p.vec && col + 8 <= p.cols) {
      if constexpr (sizeof(SRC) == 2) {
        const u32x4 v = *(const u32x4*)s;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          x[i][2 * j] = __builtin_bit_cast(float, v[j] << 16);
          x[i][2 * j + 1] = __builtin_bit_cast(float, v[j] & 0xffff0000u);
        }
      } else {
        const f32x4 v = *(const f32x4*)s, w = *(const f32x4*)(s + 4);
#pragma unroll
        for (int j = 0; j < 4; j++) x[i][j] = v[j], x[i][4 + j] = w[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) x[i][j] = row < p.rows && col + j < p.cols ? (float)s[j] : 0.f;
    }
  }

  // the block's scale, for each element this thread holds
  float inv[TILES ? 1 : TRANS ? 8 : kRows];
  if constexpr (!TILES && !TRANS) {
#pragma unroll
    for (int i = 0; i < kRows; i++) {
      unsigned m = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) m = max(m, magnitude(x[i][j]));
#pragma unroll
      for (int off = 8; off; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, 16));
      float scale;
      scale_of(m, &scale, &inv[i]);
      const int row = br * 128 + rg + 16 * i;
      if (c16 == 0 && row < p.rows) p.scales[bc * p.ld_scales + row] = scale;
    }
  } else if constexpr (!TILES) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < kRows; i++) m = max(m, magnitude(x[i][j]));
      red[rg][c16 * 8 + j] = m;
    }
    __syncthreads();
    if (t < 128) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < 16; i++) m = max(m, red[i][t]);
      float scale, v;
      scale_of(m, &scale, &v);
      if (bc * 128 + t < p.cols) p.scales[br * p.ld_scales + bc * 128 + t] = scale;
      red[0][t] = __builtin_bit_cast(unsigned, v);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++) inv[j] = __builtin_bit_cast(float, red[0][c16 * 8 + j]);
  } else {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < kRows; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) m = max(m, magnitude(x[i][j]));
#pragma unroll
    for (int off = 32; off; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, 64));
    if ((t & 63) == 0) red[0][t >> 6] = m;
    __syncthreads();
    m = max(max(red[0][0], red[0][1]), max(red[0][2], red[0][3]));
    float scale;
    scale_of(m, &scale, &inv[0]);
    if (t == 0) p.scales[TRANS ? (int64_t)bc * p.ld_scales + br : (int64_t)br * p.ld_scales + bc] = scale;
  }

#pragma unroll
  for (int i = 0; i < kRows; i++) {
    unsigned w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; j++) y[j] = x[i][4 * h + j] * inv[TILES ? 0 : TRANS ? 4 * h + j : i];
      unsigned v = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], v, true);
    }
    if constexpr (!TRANS) {
      // elements up to the next multiple of 16 columns are written, as zeros behind the last one
      const int row = br * 128 + rg + 16 * i;
      if (row < p.rows && col < ((p.cols + 15) & ~15)) *(u32x2*)(p.dst + (int64_t)row * p.ld_dst + col) = u32x2{w[0], w[1]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) turned[(c16 * 8 + j) * 144 + rg + 16 * i] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
  }
  if constexpr (TRANS) {
    __syncthreads();
    const int rows16 = (p.rows + 15) & ~15;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int c = (t >> 3) + 32 * i, r = br * 128 + (t & 7) * 16;
      if (bc * 128 + c < p.cols && r < rows16)
        *(u32x4*)(p.dst + (int64_t)(bc * 128 + c) * p.ld_dst + r) = *(const u32x4*)(turned + c * 144 + (t & 7) * 16);
    }
  }
}

template <typename SRC>
void launch_quantize(const QuantArgs& p, bool tiles, bool trans, unsigned grid, hipStream_t st) {
  if (tiles) {
    if (trans) quantize_kernel<SRC, true, true><<<grid, 256, 0, st>>>(p);
    else quantize_kernel<SRC, true, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (trans) quantize_kernel<SRC, false, true><<<grid, 256, 0, st>>>(p);
    else quantize_kernel<SRC, false, false><<<grid, 256, 0, st>>>(p);
  }
}

}  // namespace

extern "C" {

int gmd_block_quantize_launch(const gmd_block_quantize_t* q, void* hip_stream) {
  auto refuse = [](const char* why) {
    gmd::set_error("block quantise: %s", why);
    return GMD_ERR_BADPARAM;
  };
  if (!q || q->rows < 0 || q->cols < 0) return refuse("negative sizes");
  if (q->src_dtype != GMD_DT_BF16 && q->src_dtype != GMD_DT_F32) return refuse("the source is bf16 or f32");
  if (q->blocks != GMD_BLOCK_ROWS && q->blocks != GMD_BLOCK_TILES) return refuse("blocks are rows or tiles");
  if (q->rows == 0 || q->cols == 0) return GMD_OK;
  const int64_t r = q->transpose ? q->cols : q->rows, c = q->transpose ? q->rows : q->cols;  // of what is laid out
  const int64_t kb = (c + 127) / 128, c16 = (c + 15) & ~(int64_t)15, elem = q->src_dtype == GMD_DT_BF16 ? 2 : 4;
  QuantArgs p;
  p.src = (const char*)q->src, p.dst = (uint8_t*)q->dst, p.scales = q->scales;
  p.rows = q->rows, p.cols = q->cols;
  p.ld_src = q->ld_src ? q->ld_src : q->cols;
  p.ld_dst = q->ld_dst ? q->ld_dst : c16;
  p.ld_scales = q->ld_scales ? q->ld_scales : q->blocks == GMD_BLOCK_ROWS ? r : kb;
  if (!p.src || !p.dst || !p.scales) return refuse("a null pointer");
  if (((uintptr_t)p.src & (elem - 1)) || ((uintptr_t)p.dst & 15) || ((uintptr_t)p.scales & 3)) return refuse("a misaligned pointer (16 bytes for the e4m3 result)");
  if (p.ld_src < q->cols) return refuse("a source row stride shorter than a row");
  if (p.ld_dst < c16 || p.ld_dst % 16) return refuse("a result row stride that is not a multiple of 16 or shorter than a row rounded up to 16");
  if (p.ld_scales < (q->blocks == GMD_BLOCK_ROWS ? r : kb)) return refuse("a stride of scales shorter than what it spans");
  p.vec = (((uintptr_t)p.src | (uintptr_t)(p.ld_src * elem)) & 15) == 0;
  const int64_t grid = (((int64_t)q->rows + 127) / 128) * (((int64_t)q->cols + 127) / 128);
  if (grid > 0x7fffffff) return refuse("too many blocks for one launch");
  if (q->src_dtype == GMD_DT_BF16) launch_quantize<__bf16>(p, q->blocks == GMD_BLOCK_TILES, q->transpose != 0, (unsigned)grid, (hipStream_t)hip_stream);
  else launch_quantize<float>(p, q->blocks == GMD_BLOCK_TILES, q->transpose != 0, (unsigned)grid, (hipStream_t)hip_stream);
  GMD_HIP(hipGetLastError());
  return GMD_OK;
}

}  // extern "C"
