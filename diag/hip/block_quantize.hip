// Quantisation to e4m3 with one f32 scale per block of 128 (the operands of block_gemm.hip and grouped_gemm.hip).
//   amax = max |x| over the block, at least 2^-96;  scale = f32(amax / 448);  q = e4m3(f32(x * f32(448 / amax)))
// 448 is e4m3's largest value, so the block's largest element maps onto it; rounding is to nearest, ties to even.
// The floor of 2^-96 keeps 448 / amax finite; a block of zeros gets the scale 2^-96 / 448 and zeros.  amax is taken on the
// bit patterns, where NaN > infinity > every number: a block that holds an infinity or a NaN gets an infinite or NaN scale,
// and every product that reads it becomes NaN.
#include "diag_common.h"

#include <type_traits>

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
  int stream;                         // the result is stored past the caches
  int near;                           // regions that share lines of the result run on one XCD
};

// Sixteen bytes at any element's address: rows of an odd length are read in the same pieces as others.  8192 x 4100 bf16,
// rows: 23.2 us, with single elements for rows that do not begin at 16 bytes 48.5.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef f32x4 __attribute__((aligned(4))) f32x4_any;

// Eight consecutive elements of a row, held as they are read (four registers of bf16) and widened where they are used; zeros
// outside the matrix.
template <typename SRC>
struct Eight {
  typename std::conditional<sizeof(SRC) == 2, u32x4, f32x4[2]>::type v;
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (sizeof(SRC) == 2) return __builtin_bit_cast(float, j & 1 ? v[j / 2] & 0xffff0000u : v[j / 2] << 16);
    else return v[j / 4][j % 4];
  }
};
template <typename SRC>
__device__ __forceinline__ Eight<SRC> load8(const QuantArgs& p, int row, int col) {
  const SRC* s = (const SRC*)p.src + (int64_t)row * p.ld_src + col;
  Eight<SRC> x;
  if (row < p.rows && col + 8 <= p.cols) {
    if constexpr (sizeof(SRC) == 2) x.v = *(const u32x4_any*)s;
    else x.v[0] = *(const f32x4_any*)s, x.v[1] = *(const f32x4_any*)(s + 4);
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const SRC e = row < p.rows && col + j < p.cols ? s[j] : (SRC)0.f;
      if constexpr (sizeof(SRC) == 2) x.v[j / 2] = j & 1 ? x.v[j / 2] | (unsigned)__builtin_bit_cast(uint16_t, e) << 16 : __builtin_bit_cast(uint16_t, e);
      else x.v[j / 4][j % 4] = e;
    }
  }
  return x;
}
template <typename T>
__device__ __forceinline__ void store(const QuantArgs& p, uint8_t* to, const T& v) {
  if (p.stream) __builtin_nontemporal_store(v, (T*)to);
  else *(T*)to = v;
}
template <typename SRC>
__device__ __forceinline__ unsigned magnitude8(const Eight<SRC>& x) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) m = max(m, magnitude(x[j]));
  return m;
}
__device__ __forceinline__ unsigned e4m3x4(float a, float b, float c, float d) {
  const unsigned v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

// Blocks of a row, not transposed: a wave takes 512 columns (four blocks, sixteen lanes each) of two rows, all loads in
// flight before the first is used.  Memory-bound: reads of 1 KiB (bf16) and writes of 512 bytes per wave and row.
// 16384 x 7168 bf16 from memory in 63.7 us, 5.5 TB/s (one row per wave 67.9 us, four 68.9, eight 73.4).
constexpr int kRowsWave = 2, kRowsGroup = 8, kColsGroup = 512;
template <typename SRC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int groups_c = (p.cols + kColsGroup - 1) / kColsGroup;
  const int row0 = (int)blockIdx.x / groups_c * kRowsGroup + wave * kRowsWave;
  const int col = (int)blockIdx.x % groups_c * kColsGroup + lane * 8;
  if (row0 >= p.rows) return;
  Eight<SRC> x[kRowsWave];
#pragma unroll
  for (int i = 0; i < kRowsWave; i++) x[i] = load8<SRC>(p, row0 + i, col);
  const int last16 = (p.cols + 15) & ~15;
  float scale[kRowsWave];
#pragma unroll
  for (int i = 0; i < kRowsWave; i++) {
    unsigned m = magnitude8(x[i]);
#pragma unroll
    for (int off = 8; off; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, 16));
    float inv;
    scale_of(m, &scale[i], &inv);
    // elements up to the next multiple of 16 columns are written, as zeros behind the last one
    if (row0 + i < p.rows && col < last16)
      store(p, p.dst + (int64_t)(row0 + i) * p.ld_dst + col,
            u32x2{e4m3x4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv), e4m3x4(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv)});
  }
  if ((lane & 15) == 0 && col < p.cols) {
    float* const to = p.scales + (int64_t)(col / 128) * p.ld_scales + row0;
    if (row0 + kRowsWave <= p.rows) {
      __builtin_memcpy(to, scale, sizeof scale);
    } else {
#pragma unroll
      for (int i = 0; i < kRowsWave; i++)
        if (row0 + i < p.rows) to[i] = scale[i];
    }
  }
}

// The other three forms: a workgroup takes one 128 x 128 region of src into registers, thread t the eight consecutive columns
// 8 (t % 16) of rows 4 (t / 16) + r + 64 h (r < 4, h < 2), so that a column's block lies in the sixteen row groups and a tile in the
// workgroup, and four rows of a column pack into one dword of the transposed image.  In that image (128 bytes per column)
// the 16-byte chunks of a column are permuted by chunk ^ (column / 8), which leaves the dword writes at two per bank and the
// 16-byte reads at one.
// Memory-bound: what counts is how many regions a CU has in flight.  bf16 is held as it is read, which with 16 KiB of LDS lets
// eight workgroups share a CU: 16384 x 4096 bf16 39.4 us by tiles, 45.8 transposed (5.1 and 4.4 TB/s; widened at once, with six
// workgroups, 50.1 and 55.4); f32 64.0 and 70.2 us (5.2 and 4.8 TB/s).
template <typename SRC, bool TILES, bool TRANS>
__global__ __launch_bounds__(256) void quantize_region_kernel(QuantArgs p) {
  static_assert(TILES || TRANS, "rows are quantize_rows_kernel's");
  const int t = threadIdx.x, c16 = t & 15, rg = t >> 4;
  const int regions_c = (p.cols + 127) / 128;
  int br = blockIdx.x / regions_c, bc = blockIdx.x % regions_c;
  if (p.near) {  // workgroups are dealt to the eight XCDs in turn: each takes a run of regions, along a row of the result
    const int n = gridDim.x, xcd = blockIdx.x & 7, at = xcd * (n >> 3) + min(xcd, n & 7) + (blockIdx.x >> 3);
    const int regions_r = n / regions_c;
    br = TRANS ? at % regions_r : at / regions_c, bc = TRANS ? at / regions_r : at % regions_c;
  }
  const int col = bc * 128 + c16 * 8;
  // the maxima, and in their place the transposed image when they have been read
  __shared__ __attribute__((aligned(16))) unsigned turned[TRANS ? 128 * 32 : 4];
  unsigned(*const red)[128] = (unsigned(*)[128])turned;

  Eight<SRC> x[2][4];
#pragma unroll
  for (int h = 0; h < 2; h++)
#pragma unroll
    for (int r = 0; r < 4; r++) x[h][r] = load8<SRC>(p, br * 128 + rg * 4 + r + 64 * h, col);

  float inv[TILES ? 1 : 8];
  if constexpr (!TILES) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      unsigned m = 0;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) m = max(m, magnitude(x[h][r][j]));
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
    __syncthreads();
  } else {
    unsigned m = 0;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) m = max(m, magnitude8(x[h][r]));
#pragma unroll
    for (int off = 32; off; off >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, off, 64));
    if ((t & 63) == 0) turned[t >> 6] = m;
    __syncthreads();
    m = max(max(turned[0], turned[1]), max(turned[2], turned[3]));
    if constexpr (TRANS) __syncthreads();
    float scale;
    scale_of(m, &scale, &inv[0]);
    if (t == 0) p.scales[TRANS ? (int64_t)bc * p.ld_scales + br : (int64_t)br * p.ld_scales + bc] = scale;
  }

  if constexpr (sizeof(SRC) == 2) {
    // widened once more below: kept as f32 from here on they would be 64 registers in place of 32
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) asm volatile("" : "+v"(x[h][r].v));
  }
  if constexpr (!TRANS) {
    const int last16 = (p.cols + 15) & ~15;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int row = br * 128 + rg * 4 + r + 64 * h;
        const Eight<SRC>& v = x[h][r];
        if (row < p.rows && col < last16)
          store(p, p.dst + (int64_t)row * p.ld_dst + col, u32x2{e4m3x4(v[0] * inv[0], v[1] * inv[0], v[2] * inv[0], v[3] * inv[0]),
                                                                e4m3x4(v[4] * inv[0], v[5] * inv[0], v[6] * inv[0], v[7] * inv[0])});
      }
  } else {
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float f = inv[TILES ? 0 : j];
        const int chunk = (rg >> 2) + 4 * h;
        turned[(c16 * 8 + j) * 32 + (chunk ^ (c16 & 7)) * 4 + (rg & 3)] = e4m3x4(x[h][0][j] * f, x[h][1][j] * f, x[h][2][j] * f, x[h][3][j] * f);
      }
    __syncthreads();
    const int rows16 = (p.rows + 15) & ~15;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int c = (t >> 3) + 32 * i, chunk = t & 7, r = br * 128 + chunk * 16;
      if (bc * 128 + c < p.cols && r < rows16)
        store(p, p.dst + (int64_t)(bc * 128 + c) * p.ld_dst + r, *(const u32x4*)(turned + c * 32 + (chunk ^ ((c >> 3) & 7)) * 4));
    }
  }
}

// In bands of src's rows where one launch would have 2^32 threads or more; a row of regions always fits (2^24 - 8 at most).
template <typename SRC>
int launch_quantize(const QuantArgs& p, bool tiles, bool trans, hipStream_t st) {
  const bool rows = !tiles && !trans;
  const int group_r = rows ? kRowsGroup : 128, group_c = rows ? kColsGroup : 128;
  const int64_t across = (p.cols + (int64_t)group_c - 1) / group_c, down = (p.rows + (int64_t)group_r - 1) / group_r;
  const int64_t most = (((int64_t)1 << 32) / 256 - 1) / across;
  for (int64_t at = 0; at < down; at += most) {
    const int64_t n = std::min(most, down - at), first = at * group_r;
    QuantArgs b = p;
    b.rows = (int)std::min<int64_t>(p.rows - first, n * group_r);
    b.src += first * p.ld_src * (int64_t)sizeof(SRC);
    b.dst += trans ? first : first * p.ld_dst;
    b.scales += rows ? first : trans && tiles ? first / 128 : first / 128 * p.ld_scales;
    const unsigned grid = (unsigned)(n * across);
    if (rows) quantize_rows_kernel<SRC><<<grid, 256, 0, st>>>(b);
    else if (!trans) quantize_region_kernel<SRC, true, false><<<grid, 256, 0, st>>>(b);
    else if (tiles) quantize_region_kernel<SRC, true, true><<<grid, 256, 0, st>>>(b);
    else quantize_region_kernel<SRC, false, true><<<grid, 256, 0, st>>>(b);
    GMD_HIP(hipGetLastError());
  }
  return GMD_OK;
}

}  // namespace

extern "C" {

int gmd_block_quantize_launch(const gmd_block_quantize_t* q, void* hip_stream) {
  auto refuse = [](const char* why) {
    gmd::set_error("block quantise: %s", why);
    return GMD_ERR_BADPARAM;
  };
  constexpr int kMaxSize = 0x7fffffff - 1023;  // rounded up to a region it still fits 31 bits
  if (!q || q->rows < 0 || q->cols < 0 || q->rows > kMaxSize || q->cols > kMaxSize) return refuse("negative sizes, or sizes over 2^31 - 1024");
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
  if (const char* bad = gmd::elsewhere((hipStream_t)hip_stream, {p.src, p.dst, p.scales})) return refuse(bad);
  // A result that the caches would keep for the product that reads it is stored through them; a larger one is not (16384 x 7168:
  // 56.3 against 68.2 us).  32 MiB: the L2s of the eight XCDs together.
  p.stream = r * c16 > (32 << 20);
  // Where rows of the result do not begin at lines of 128 bytes, neighbours on a row of it share lines, which one L2 joins
  // (8200 x 4100 transposed, f32: 39.1 us against 44.1, bf16 26.2 against 32.0; by tiles bf16 25.9 against 32.8); where they do,
  // the plain order spreads the memory's channels better (16384 x 4096 bf16 by tiles 39.4 against 44.0).
  p.near = (((uintptr_t)p.dst | (uintptr_t)p.ld_dst) & 127) != 0;
  const bool tiles = q->blocks == GMD_BLOCK_TILES, trans = q->transpose != 0;
  return q->src_dtype == GMD_DT_BF16 ? launch_quantize<__bf16>(p, tiles, trans, (hipStream_t)hip_stream)
                                     : launch_quantize<float>(p, tiles, trans, (hipStream_t)hip_stream);
}

}  // extern "C"
