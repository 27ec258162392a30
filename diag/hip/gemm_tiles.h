// Device code shared by the block-scaled fp8 and the expert-grouped GEMM kernels (gfx950).
//
// One product:  C[m, n] = sum over k of A[m, k] * B[n, k], with
//   * elements bf16, or e4m3 with one f32 scale per block of 128 k (Kind);
//   * either operand with its k contiguous, or "transposed": k as the row, m or n contiguous (bf16 only);
//   * rows of A, and with them B, dealt to experts (Args::offsets), or the k range dealt to experts (weight gradient).
// A K-step is 128 bytes of k: 64 bf16 or one block of 128 e4m3.
#pragma once

#include "diag_common.h"

namespace gmd {
namespace tiles {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// What the operands hold: bf16; e4m3 with A's scales per row and B's per 128 x 128 tile; e4m3 with both per row.
enum Kind { kBf16 = 0, kFp8Tiles = 1, kFp8Rows = 2 };

constexpr int kStepBytes = 128;

struct Args {
  const char* a;
  const char* b;
  void* c;
  const float* sa;      // [k blocks][rows of A], ld_sa apart
  const float* sb;      // kFp8Tiles: [n blocks][k blocks], ld_sb apart; kFp8Rows: [k blocks][n], ld_sb apart
  const int* offsets;   // device, groups + 1 row numbers; null = one product
  int64_t lda, ldb;     // bytes between rows
  int64_t ldc;          // elements between rows
  int64_t ld_sa, ld_sb;
  int64_t stride_b, stride_sb, stride_c;  // from one expert to the next: bytes, floats, elements
  int m, n, k;          // rows of C, columns of C, contraction; with a weight gradient k is the total number of rows
  int groups;
};

// Sixteen zero bytes: where a lane whose chunk of k lies beyond the contraction fetches from.
static __device__ const uint4 g_zero16 = {0, 0, 0, 0};

// ------------------------------------------------------------------------------------------------ tile of a block --
// Workgroup ids are dealt to the eight XCDs in turn; the remapped ids of one XCD are contiguous, so that its L2 holds the
// operand panels that neighbouring tiles share.  A bijection of 0 .. n-1 for any n.
__device__ __forceinline__ int xcd_contiguous(int id, int n) {
  const int x = id & 7, q = n >> 3, r = n & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}

// Tiles in panels of eight rows of tiles, rows first inside a panel: neighbours share the B panel, and eight A panels
// are walked again for the next column.
__device__ __forceinline__ void tile_walk(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int panel = id / (8 * tiles_n), first = panel * 8, rows = min(8, tiles_m - first), in = id - panel * 8 * tiles_n;
  *tm = first + in % rows;
  *tn = in / rows;
}

struct Tile {
  int group;
  int m0, m_end;  // first row of C, and where the rows that this product may touch end
  int n0;
};

// Rows of expert g.  The offsets are the caller's data: whatever they hold, the rows stay inside [0, rows).
__device__ __forceinline__ void group_rows(const int* __restrict__ offsets, int g, int rows, int* lo, int* hi) {
  *lo = min(max(offsets[g], 0), rows);
  *hi = min(max(offsets[g + 1], *lo), rows);
}

// The tile that workgroup `id` of a launch over all experts' rows computes.  The host does not know the offsets, so the
// grid is an upper bound (rows / bm + groups rows of tiles); ids beyond the real number return false.  Every wave scans
// the tile counts, 64 experts at a time.
__device__ __forceinline__ bool find_tile(const Args& p, int bm, int bn, int id, Tile* t) {
  const int tiles_n = (p.n + bn - 1) / bn;
  if (!p.offsets) {
    const int tiles_m = (p.m + bm - 1) / bm;
    int tm, tn;
    tile_walk(xcd_contiguous(id, tiles_m * tiles_n), tiles_m, tiles_n, &tm, &tn);
    t->group = 0, t->m0 = tm * bm, t->m_end = p.m, t->n0 = tn * bn;
    return true;
  }
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 64) {
    int lo = 0, hi = 0;
    if (g0 + lane < p.groups) group_rows(p.offsets, g0 + lane, p.m, &lo, &hi);
    int tiles = (hi - lo + bm - 1) / bm;
#pragma unroll
    for (int off = 32; off; off >>= 1) tiles += __shfl_xor(tiles, off, 64);
    total += tiles;
  }
  total = __builtin_amdgcn_readfirstlane(total);
  if (id >= total * tiles_n) return false;
  const int work = xcd_contiguous(id, total * tiles_n);
  int before = 0;  // tiles of the experts in front
  for (int g0 = 0; g0 < p.groups; g0 += 64) {
    int lo = 0, hi = 0;
    if (g0 + lane < p.groups) group_rows(p.offsets, g0 + lane, p.m, &lo, &hi);
    const int mine = (hi - lo + bm - 1) / bm * tiles_n;
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    const int in = work - before;
    const unsigned long long has = __ballot(in < upto);
    if (has) {
      const int l = __builtin_ctzll(has);  // the first expert whose tiles reach past this one
      const int glo = __builtin_amdgcn_readfirstlane(__shfl(lo, l, 64)), ghi = __builtin_amdgcn_readfirstlane(__shfl(hi, l, 64));
      const int first = __builtin_amdgcn_readfirstlane(__shfl(upto - mine, l, 64));
      int tm, tn;
      tile_walk(in - first, (ghi - glo + bm - 1) / bm, tiles_n, &tm, &tn);
      t->group = g0 + l, t->m0 = glo + tm * bm, t->m_end = ghi, t->n0 = tn * bn;
      return true;
    }
    before += __builtin_amdgcn_readfirstlane(__shfl(upto, 63, 64));
  }
  return false;
}

// ------------------------------------------------------------------------------------------------------ LDS image --
// k contiguous: 8 rows x 128 bytes per KiB, which is what one wave-wide LDS-DMA instruction of 16 bytes a lane writes,
// the 16-byte chunks of row r permuted by chunk ^ swizzle(r).  A fragment read (ds_read_b128, lane (fr, fq): row fr, chunk
// fq or 4 + fq) is served in groups of 16 lanes that touch 16 rows; the permutation gives each group sixteen slots of its
// own.  It lives in the source address and in the read address, never in the DMA's destination.
__device__ __forceinline__ int chunk_swizzle(int row) { return ((row >> 1) & 3) << 1; }

// Transposed: 64 rows of k, the m or n side contiguous.  Fragments come through ds_read_b64_tr_b16: within each group of 16
// lanes lane i supplies the address of 4 elements of row i / 4, columns 4 (i % 4) .., and receives column i of the four rows.
// A read's 16 rows are a multiple of the row size apart, so 32-byte units of a row are permuted by unit ^ f(row) with f
// running over all eight values within the rows that half a wave touches.
__device__ __forceinline__ int unit_swizzle(int row) { return ((row >> 3) & 1) * 4 + (row & 3); }

__device__ __forceinline__ void load_lds16(const char* src, char* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// One operand's way into LDS.  ROWS: rows of the tile (its m or n extent); WAVES share the 1-KiB pieces.  DEAL: LDS row
// 16 b + f of a wave's WT rows holds tile row f * (WT / 16) + b, so that a fragment lane's rows are consecutive.
template <bool TRANS, int ROWS, int WAVES, int DEAL>
struct Stage {
  static constexpr int kPieces = ROWS / 8 / WAVES;
  static_assert(kPieces * 8 * WAVES == ROWS, "whole pieces per wave");
  static constexpr int kChunks = ROWS / 8;  // transposed: 16-byte chunks per row of k
  const char* base;        // first row of the tile, first k
  uint32_t off[kPieces];   // a lane's place in it
  int chunk[kPieces];      // its chunk of the 128 bytes (k contiguous) or its row of the 64 (transposed)
  int64_t ld;

  // first: first row (column) of the tile, rows_left >= 1: how many of them exist; the rest repeat the last one.
  __device__ __forceinline__ void init(const char* p, int64_t ld_, int64_t first, int rows_left, int wave, int lane) {
    ld = ld_;
    base = TRANS ? p + first * 2 : p + first * ld;
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
      const int piece = wave * kPieces + i;
      if constexpr (TRANS) {
        const int pos = piece * 64 + lane, r = pos / kChunks;
        const int c = (pos % kChunks) ^ ((2 * unit_swizzle(r)) & (kChunks - 1));
        const int col = min(c * 8, rows_left - 8);  // the extent is a multiple of 8
        off[i] = (uint32_t)(r * ld) + (uint32_t)col * 2;
        chunk[i] = r;
      } else {
        const int l = piece * 8 + (lane >> 3);
        int row = l;
        if constexpr (DEAL != 0) row = l / DEAL * DEAL + (l & 15) * (DEAL / 16) + (l % DEAL >> 4);
        const int c = (lane & 7) ^ chunk_swizzle(l);
        off[i] = (uint32_t)(min(row, rows_left - 1) * ld) + (uint32_t)c * 16;
        chunk[i] = c;
      }
    }
  }
  // K-step kt into `tile`; `left` = k (elements if transposed, bytes if not) from this step on: what lies beyond is zero.
  __device__ __forceinline__ void fetch(int kt, int64_t left, char* tile, int wave) const {
    const char* src = base + (TRANS ? (int64_t)kt * 64 * ld : (int64_t)kt * kStepBytes);
    asm volatile("" : "+s"(src));  // one scalar base per step; otherwise the compiler keeps a 64-bit address per piece and lane
    char* const dst = tile + wave * kPieces * 1024;
    if (left >= (TRANS ? 64 : kStepBytes)) {
#pragma unroll
      for (int i = 0; i < kPieces; i++) load_lds16(src + off[i], dst + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; i++) {
        const bool in = TRANS ? chunk[i] < left : chunk[i] * 16 < left;
        load_lds16(in ? src + off[i] : (const char*)&g_zero16, dst + i * 1024);
      }
    }
  }
};

// A wave's fragments of one operand: blocks of 16 rows, two halves of the K-step each (bf16: two substeps of 32 k; fp8:
// registers 0-3 and 4-7 of the one K = 128 operand).
template <bool TRANS, int ROWS, int NB>
struct Frags {
  int off[TRANS ? NB : 2];
  __device__ __forceinline__ void init(int first, int lane) {
    const int fr = lane & 15, fq = lane >> 4;
    if constexpr (TRANS) {
      const int r = 8 * fq + (fr >> 2);
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const int unit = (first / 16 + b) ^ (unit_swizzle(r) & (ROWS / 16 - 1));
        off[b] = r * (ROWS * 2) + unit * 32 + (fr & 3) * 8;
      }
    } else {
      const int l = first + fr;
#pragma unroll
      for (int h = 0; h < 2; h++) off[h] = (l >> 3) * 1024 + (l & 7) * 128 + (((4 * h + fq) ^ chunk_swizzle(l)) << 4);
    }
  }
  __device__ __forceinline__ i32x4 read(const char* tile, int b, int h) const {
    if constexpr (TRANS) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
      typedef int i32x2 __attribute__((ext_vector_type(2)));
      const char* q = tile + off[b] + h * 32 * (ROWS * 2);
      const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)q));
      const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(q + 4 * (ROWS * 2))));
      return i32x4{lo.x, lo.y, hi.x, hi.y};
    } else {
      return *(const i32x4*)(tile + off[h] + b * 2048);
    }
  }
};

__device__ __forceinline__ f32x4 mfma_bf16(const i32x4& b, const i32x4& a, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
// Unscaled K = 128 product of e4m3 (scale operands of zero select the unscaled instruction).
__device__ __forceinline__ f32x4 mfma_fp8(const i32x8& b, const i32x8& a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
// Sixteen e4m3 as bf16 (exact): two fragments of eight.
__device__ __forceinline__ void widen(const i32x4& v, i32x4* lo, i32x4* hi) {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int x = __builtin_bit_cast(int, (v2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, false));
    const int y = __builtin_bit_cast(int, (v2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, true));
    i32x4* const to = i < 2 ? lo : hi;
    (*to)[2 * (i & 1)] = x;
    (*to)[2 * (i & 1) + 1] = y;
  }
}
// One K-step's fragment of an operand, by what it is multiplied as.  0: bf16.  1: e4m3 on the K = 128 fp8 instruction.  That instruction aligns the
// products of each group of eight k to the largest of them and drops what lies below 2^-13 of its binade (measured with one large and one small product
// per group; the K = 32 and K = 64 fp8 forms do the same), at most 2^-10 of the sum of
// magnitudes and about 5e-6 of the result on normal data.  A bf16 result rounds coarser than that; an f32 result does not,
// so for it (2) the elements are widened to bf16 and multiplied on the bf16 instruction, which keeps f32 sums, at half the rate.
template <int FORM>
struct Operand;
template <>
struct Operand<0> {
  i32x4 v[2];
  __device__ __forceinline__ void set(const i32x4& lo, const i32x4& hi) { v[0] = lo, v[1] = hi; }
  static __device__ __forceinline__ void accumulate(const Operand& b, const Operand& a, f32x4& c) {
    c = mfma_bf16(b.v[0], a.v[0], c);
    c = mfma_bf16(b.v[1], a.v[1], c);
  }
};
template <>
struct Operand<1> {
  i32x8 v;
  __device__ __forceinline__ void set(const i32x4& lo, const i32x4& hi) { v = i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}; }
  static __device__ __forceinline__ f32x4 product(const Operand& b, const Operand& a) { return mfma_fp8(b.v, a.v); }
};
template <>
struct Operand<2> {
  i32x4 v[4];
  __device__ __forceinline__ void set(const i32x4& lo, const i32x4& hi) {
    widen(lo, &v[0], &v[1]);
    widen(hi, &v[2], &v[3]);
  }
  static __device__ __forceinline__ f32x4 product(const Operand& b, const Operand& a) {
    f32x4 c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++) c = mfma_bf16(b.v[i], a.v[i], c);
    return c;
  }
};

// Eight f32 of a row -> C: one 16-byte store of bf16 or two of f32.  C is not read again by this kernel.
template <typename OUT>
__device__ __forceinline__ void store8(OUT* dst, const f32x4& x, const f32x4& y) {
  if constexpr (sizeof(OUT) == 2) {
    u32x4 o;
    o[0] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{x[0], x[1]}, bf16x2));
    o[1] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{x[2], x[3]}, bf16x2));
    o[2] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{y[0], y[1]}, bf16x2));
    o[3] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{y[2], y[3]}, bf16x2));
    *(u32x4*)dst = o;
  } else {
    *(f32x4*)dst = x;
    *(f32x4*)(dst + 4) = y;
  }
}

// ------------------------------------------------------------------------------------------------------ tile kernel --
// BM x BN of C per workgroup, WM x WN waves, K-steps double buffered in LDS: the next step's DMA is issued before this one
// is computed on, one barrier per step.  The MFMA takes B's fragment first, so lane (fr, fq) of a 16 x 16 block holds row fr
// and columns 4 fq .. 4 fq + 3.
//
// Block-scaled fp8: the matrix instruction sums one block of 128 k from zero and its result is added with one FMA per
// element, acc += (sa * sb) * block.  With rows dealt to lanes (Stage's DEAL) a lane's scales of A are MB consecutive floats
// per K-step, and B's tile scale is one scalar per wave.
template <int KIND, bool TA, bool TB, bool WGRAD, int BM, int BN, int WM, int WN, typename OUT>
__global__ __launch_bounds__(WM * WN * 64) void tile_kernel(Args p) {
  constexpr int kWaves = WM * WN, WTM = BM / WM, WTN = BN / WN, MB = WTM / 16, NB = WTN / 16;
  constexpr bool kFp8 = KIND != kBf16, kNarrow = sizeof(OUT) == 2;
  constexpr int kElem = kFp8 ? 1 : 2, kStepK = kStepBytes / kElem;
  static_assert(!kFp8 || (!TA && !TB && WTN <= 128), "block-scaled fp8: k contiguous, a wave's columns inside one tile of scales");
  constexpr int kABytes = BM * kStepBytes, kBufBytes = (BM + BN) * kStepBytes;
  constexpr int kStrip = WTN * 4 + 16;  // epilogue: one row of a wave's strip of 16 rows
  static_assert(kWaves * 16 * kStrip <= 2 * kBufBytes, "the epilogue's strips fit into the operand buffers");
  constexpr int kScaleWaves = kFp8 ? BM / 64 + (KIND == kFp8Rows ? BN / 64 : 1) : 0, kScaleBytes = kScaleWaves * 256;
  static_assert(kScaleWaves <= kWaves && BN <= 64 * 128, "one DMA of scales per wave and step");
  __shared__ __attribute__((aligned(16))) char smem[2 * kBufBytes + 2 * kScaleBytes];
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  Tile t;
  int64_t k_first = 0;
  int K = p.k;
  if constexpr (WGRAD) {
    const int tiles_m = (p.m + BM - 1) / BM, tiles_n = (p.n + BN - 1) / BN;
    const int work = xcd_contiguous(blockIdx.x, gridDim.x);
    int tm, tn, lo, hi;
    t.group = work / (tiles_m * tiles_n);
    tile_walk(work - t.group * tiles_m * tiles_n, tiles_m, tiles_n, &tm, &tn);
    t.m0 = tm * BM, t.m_end = p.m, t.n0 = tn * BN;
    group_rows(p.offsets, t.group, p.k, &lo, &hi);
    k_first = lo, K = hi - lo;
  } else {
    if (!find_tile(p, BM, BN, blockIdx.x, &t)) return;  // the whole workgroup, before any barrier
  }
  const char* const B = p.b + (WGRAD ? 0 : t.group * p.stride_b);
  Stage<TA, BM, kWaves, kFp8 ? WTM : 0> ga;
  Stage<TB, BN, kWaves, 0> gb;
  ga.init(p.a + (TA ? k_first * p.lda : 0), p.lda, t.m0, t.m_end - t.m0, wave, lane);
  gb.init(B + (TB ? k_first * p.ldb : 0), p.ldb, t.n0, p.n - t.n0, wave, lane);
  Frags<TA, BM, MB> fa;
  Frags<TB, BN, NB> fb;
  fa.init(wm * WTM, lane);
  fb.init(wn * WTN, lane);

  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; i++)
#pragma unroll
    for (int j = 0; j < NB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Scales of one K-step travel with its operands: A's of the tile's rows and B's of its columns (or of its 128-column
  // tiles) in a slot of their own behind the operand buffers, one DMA of 4 bytes a lane for 64 of them.  Loaded by each wave for
  // itself into registers they cost more than the matrix work: nine loads of their own per lane, wave and step.
  const float* const SB = kFp8 ? p.sb + t.group * p.stride_sb : nullptr;
  const float* scale_src = nullptr;  // this lane's, at step 0
  int64_t scale_ld = 0;
  if constexpr (kFp8) {
    if (wave < BM / 64) {
      scale_src = p.sa + min(t.m0 + wave * 64 + lane, t.m_end - 1), scale_ld = p.ld_sa;
    } else if (KIND == kFp8Rows) {
      scale_src = SB + min(t.n0 + (wave - BM / 64) * 64 + lane, p.n - 1), scale_ld = p.ld_sb;
    } else {
      scale_src = SB + (int64_t)(min(t.n0 + lane * 128, p.n - 1) / 128) * p.ld_sb, scale_ld = 1;
    }
  }
  auto fetch_scales = [&](int kt) {
    if (wave < kScaleWaves)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(scale_src + kt * scale_ld),
                                       (__attribute__((address_space(3))) void*)(smem + 2 * kBufBytes + (kt & 1) * kScaleBytes + wave * 256), 4, 0, 0);
  };
  constexpr int kSb = KIND == kFp8Rows ? NB : 1;
  float sl[MB];   // sa * sb (tiles) or sa (rows) of the running step
  f32x4 sb[kSb];  // rows: sb of this lane's columns
  auto read_scales = [&](int kt) {
    const float* const q = (const float*)(smem + 2 * kBufBytes + (kt & 1) * kScaleBytes);
#pragma unroll
    for (int i = 0; i < MB; i += 4) {
      const f32x4 v = *(const f32x4*)(q + wm * WTM + fr * MB + i);
#pragma unroll
      for (int r = 0; r < 4; r++) sl[i + r] = v[r];
    }
    if constexpr (KIND == kFp8Tiles) {
      const float b = q[BM + wn * WTN / 128];
#pragma unroll
      for (int i = 0; i < MB; i++) sl[i] *= b;
    } else {
#pragma unroll
      for (int j = 0; j < NB; j++) sb[j] = *(const f32x4*)(q + BM + wn * WTN + j * 16 + fq * 4);
    }
  };

  const int steps = (int)(((int64_t)K + kStepK - 1) / kStepK);
  auto fetch = [&](int kt) {
    char* const buf = smem + (kt & 1) * kBufBytes;
    const int64_t left = (int64_t)K - (int64_t)kt * kStepK;
    ga.fetch(kt, TA ? left : left * kElem, buf, wave);
    gb.fetch(kt, TB ? left : left * kElem, buf + kABytes, wave);
    if constexpr (kFp8) fetch_scales(kt);
  };

  // One step: row blocks i = 0 .. MB-1 of the wave's tile against its NB column blocks.  A's fragment of the next row block
  // is read while this one is multiplied.  The last row block holds the step's one synchronisation: every fragment of this
  // buffer has been read and the next buffer has landed; behind it go the DMA of step kt + 2 into this buffer and the reads of
  // the next step's first fragments, each of B's as soon as its registers have been consumed, so that the matrix pipe does not
  // drain at a step's edge.
  typedef Operand<kFp8 ? (kNarrow ? 1 : 2) : 0> Op;
  Op bf[NB], af[2];
  f32x4 part[4];       // block sums on their way to the accumulators
  auto add = [&](int i, int j, int slot, float s) {
#pragma unroll
    for (int r = 0; r < 4; r++)
      acc[i][j][r] = __builtin_fmaf(KIND == kFp8Tiles ? s : s * sb[KIND == kFp8Tiles ? 0 : j][r], part[slot][r], acc[i][j][r]);
    asm volatile("" : "+v"(acc[i][j]));  // here, between the MFMAs: left to itself the compiler sinks all of them behind the last
  };
  auto sync = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0), as the builtin, so that the compiler's own count agrees
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (steps > 0) {
    fetch(0);
    if (steps > 1) fetch(1);
    sync();
    if constexpr (kFp8) read_scales(0);
#pragma unroll
    for (int j = 0; j < NB; j++) bf[j].set(fb.read(smem + kABytes, j, 0), fb.read(smem + kABytes, j, 1));
    af[0].set(fa.read(smem, 0, 0), fa.read(smem, 0, 1));
  }
  for (int kt = 0; kt < steps; kt++) {
    const char* const la = smem + (kt & 1) * kBufBytes;
    const char* const na = smem + ((kt + 1) & 1) * kBufBytes;
    const char* const nb = na + kABytes;
#pragma unroll
    for (int i = 0; i < MB; i++) {
      if (i + 1 < MB) {
        af[(i + 1) & 1].set(fa.read(la, i + 1, 0), fa.read(la, i + 1, 1));
      } else {
        sync();
        if (kt + 2 < steps) fetch(kt + 2);
        af[0].set(fa.read(na, 0, 0), fa.read(na, 0, 1));  // (behind the last step: landed data that nothing uses)
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NB; j++) {
        const int at = i * NB + j;
        if constexpr (kFp8) {
          part[at & 3] = Op::product(bf[j], af[i & 1]);
          __builtin_amdgcn_sched_barrier(0);
          if (at >= 2) add((at - 2) / NB, (at - 2) % NB, (at - 2) & 3, sl[(at - 2) / NB]);
        } else {
          Op::accumulate(bf[j], af[i & 1], acc[i][j]);
        }
        if (i + 1 == MB) bf[j].set(fb.read(nb, j, 0), fb.read(nb, j, 1));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (kFp8) {
      add(MB - 1, NB - 2, (MB * NB - 2) & 3, sl[MB - 1]);
      add(MB - 1, NB - 1, (MB * NB - 1) & 3, sl[MB - 1]);
      read_scales(kt + 1);
    }
  }
  __syncthreads();  // every wave is done with the operand buffers

  // Epilogue: 16 rows of the wave's tile at a time through a strip of LDS of its own, so that neighbouring lanes store
  // neighbouring columns of one row.
  char* const strip = smem + wave * 16 * kStrip;
  OUT* const C = (OUT*)p.c + (WGRAD ? t.group * p.stride_c : 0);
  constexpr int kLanesPerRow = WTN / 8, kRowsPerPass = 64 / kLanesPerRow;
#pragma unroll
  for (int i = 0; i < MB; i++) {
#pragma unroll
    for (int j = 0; j < NB; j++) *(f32x4*)(strip + fr * kStrip + (j * 16 + fq * 4) * 4) = acc[i][j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kRowsPerPass) {
      const int f = r0 + lane / kLanesPerRow, c8 = lane % kLanesPerRow * 8;
      const f32x4 x = *(const f32x4*)(strip + f * kStrip + c8 * 4), y = *(const f32x4*)(strip + f * kStrip + c8 * 4 + 16);
      const int row = t.m0 + wm * WTM + (kFp8 ? f * MB + i : i * 16 + f), col = t.n0 + wn * WTN + c8;
      if (row < t.m_end && col < p.n) store8<OUT>(C + row * p.ldc + col, x, y);  // N is a multiple of 8
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------------------------------------------- few-row kernel --
// Up to 16 MB rows x 16 columns per workgroup: what bounds such a product is reading B once, so B goes straight from memory
// to the registers that the MFMA takes (lane (fr, fq): row fr, chunks fq and 4 + fq of the 128 bytes) and the eight waves
// share the K-steps in turn, four at a time in flight each.  Their sums are joined in LDS in the order of the waves.
constexpr int kFewWaves = 8;
template <int KIND, int MB, typename OUT>
__global__ __launch_bounds__(kFewWaves * 64) void few_rows_kernel(Args p) {
  constexpr bool kFp8 = KIND != kBf16, kNarrow = sizeof(OUT) == 2;
  constexpr int kElem = kFp8 ? 1 : 2;
  constexpr int U = MB <= 2 ? 4 : 2;
  __shared__ f32x4 sums[kFewWaves][MB][64];
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Tile t;
  if (!find_tile(p, MB * 16, 16, blockIdx.x, &t)) return;
  const int kbytes = p.k * kElem;
  const int steps = (kbytes + kStepBytes - 1) / kStepBytes;
  const char* const zero = (const char*)&g_zero16;
  const char* const b_row = p.b + t.group * p.stride_b + (int64_t)min(t.n0 + fr, p.n - 1) * p.ldb + fq * 16;
  const char* a_row[MB];
  int row[MB];
#pragma unroll
  for (int i = 0; i < MB; i++) {
    row[i] = min(t.m0 + i * 16 + fr, t.m_end - 1);
    a_row[i] = p.a + (int64_t)row[i] * p.lda + fq * 16;
  }
  const float* const SB = kFp8 ? p.sb + t.group * p.stride_sb : nullptr;
  const int col4 = min(t.n0 + fq * 4, p.n - 4);
  f32x4 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto load2 = [&](const char* q, int kt, i32x4* lo, i32x4* hi) {
    const int at = kt * kStepBytes + fq * 16;  // byte of k of the first chunk; the second is 64 further on
    const char* r = q + (int64_t)kt * kStepBytes;
    *lo = *(const i32x4*)(at < kbytes ? r : zero);
    *hi = *(const i32x4*)(at + 64 < kbytes ? r + 64 : zero);
  };
  for (int k0 = wave; k0 < steps; k0 += kFewWaves * U) {
    i32x4 bl[U], bh[U], al[U][MB], ah[U][MB];
    float sa[U][MB];
    f32x4 sb[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int kt = k0 + u * kFewWaves;
      if (kt < steps) {
        load2(b_row, kt, &bl[u], &bh[u]);
#pragma unroll
        for (int i = 0; i < MB; i++) load2(a_row[i], kt, &al[u][i], &ah[u][i]);
        if constexpr (kFp8) {
#pragma unroll
          for (int i = 0; i < MB; i++) sa[u][i] = p.sa[kt * p.ld_sa + row[i]];
          if constexpr (KIND == kFp8Tiles) {
            sb[u][0] = SB[(int64_t)(t.n0 / 128) * p.ld_sb + kt];
          } else {
            const float* r = SB + kt * p.ld_sb + col4;
            sb[u] = f32x4{r[0], r[1], r[2], r[3]};
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (k0 + u * kFewWaves >= steps) break;
      Operand<kNarrow ? 1 : 2> bf;
      if constexpr (kFp8) bf.set(bl[u], bh[u]);
#pragma unroll
      for (int i = 0; i < MB; i++) {
        if constexpr (kFp8) {
          Operand<kNarrow ? 1 : 2> af;
          af.set(al[u][i], ah[u][i]);
          const f32x4 part = Operand<kNarrow ? 1 : 2>::product(bf, af);
#pragma unroll
          for (int r = 0; r < 4; r++) acc[i][r] = __builtin_fmaf(sa[u][i] * (KIND == kFp8Tiles ? sb[u][0] : sb[u][r]), part[r], acc[i][r]);
        } else {
          acc[i] = mfma_bf16(bl[u], al[u][i], acc[i]);
          acc[i] = mfma_bf16(bh[u], ah[u][i], acc[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MB; i++) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave < MB) {  // wave i joins block i: lane (fr, fq) holds row fr, columns 4 fq ..
    f32x4 v = sums[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; w++) v += sums[w][wave][lane];
    const int r = t.m0 + wave * 16 + fr, col = t.n0 + fq * 4;
    if (r < t.m_end && col < p.n) {
      OUT* dst = (OUT*)p.c + r * p.ldc + col;
      if constexpr (sizeof(OUT) == 2) *(bf16x4*)dst = __builtin_convertvector(v, bf16x4);
      else *(f32x4*)dst = v;
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ host --
// Workgroups of a launch in tiles of bm x bn: with experts an upper bound, since the host does not know their rows.
inline int64_t grid_of(const Args& p, int bm, int bn) {
  const int64_t tiles_n = ((int64_t)p.n + bn - 1) / bn;
  const int64_t tiles_m = p.offsets ? (int64_t)p.m / bm + std::min(p.groups, p.m) : ((int64_t)p.m + bm - 1) / bm;
  return tiles_m * tiles_n;
}
inline int launched(const char* what, int64_t grid) {
  if (grid <= 0 || grid > 0x7fffffff) {
    set_error("%s: %lld workgroups do not fit into one launch", what, (long long)grid);
    return GMD_ERR_BADPARAM;
  }
  return GMD_OK;
}

// Block-scaled fp8, one product or one per expert (block_gemm.hip).
int launch_fp8(const Args& p, int b_blocks, int out_dtype, hipStream_t st);
// Shared refusals: null when the pointer, the row stride and the extent fit the kernels, else what is wrong.
// row_bytes: what a row holds; the lane offsets inside a 256-row tile are 32 bits, hence the limit on ld_bytes.
inline const char* bad_operand(const void* p, int64_t ld_bytes, int64_t row_bytes) {
  if (!p) return "a null pointer";
  if ((uintptr_t)p & 15) return "a pointer that is not 16-byte aligned";
  if (ld_bytes & 15) return "a row stride that is not a multiple of 16 bytes";
  if (ld_bytes < row_bytes) return "a row stride shorter than a row";
  if (ld_bytes > (8 << 20)) return "a row stride over 8 MiB";
  return nullptr;
}

}  // namespace tiles
}  // namespace gmd
