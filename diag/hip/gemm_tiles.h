// Device code shared by the block-scaled fp8 and the expert-grouped GEMM kernels (gfx950).
//
// One product:  C[m, n] = sum over k of A[m, k] * B[n, k], with
//   * elements bf16, or e4m3 with one f32 scale per block of 128 k (Kind);
//   * either operand with its k contiguous, or "transposed": k as the row, m or n contiguous (bf16 only);
//   * rows of A, and with them B, dealt to experts (Args::offsets), or the k range dealt to experts (weight gradient).
// A K-step is 128 bytes of k: 64 bf16 or one block of 128 e4m3.
#pragma once

#include <cmath>
#include <type_traits>

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

// Tiles in panels of four rows of tiles, rows first inside a panel: neighbours share the B panel, and four A panels
// are walked again for the next column.
__device__ __forceinline__ void tile_walk(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
  const int panel = id / (4 * tiles_n), first = panel * 4, rows = min(4, tiles_m - first), in = id - panel * 4 * tiles_n;
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

// The tiles of a launch over all experts' rows, in the order of the ids.  The host does not know the offsets, so its grid is an
// upper bound (rows / bm + groups rows of tiles); ids beyond the real number have no tile.  Every wave scans the tile counts, 64
// experts at a time, and keeps those of the last 64.
struct RowTiles {
  int bm, bn, tiles_n, total;
  int lo, hi, upto;  // of expert g0 + lane; tiles up to and with it, among these 64

  __device__ __forceinline__ void scan(const Args& p, int g0) {
    const int lane = threadIdx.x & 63;
    lo = hi = 0;
    if (g0 + lane < p.groups) group_rows(p.offsets, g0 + lane, p.m, &lo, &hi);
    upto = (hi - lo + bm - 1) / bm * tiles_n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off, 64);
      if (lane >= off) upto = __builtin_elementwise_add_sat(upto, v);  // (offsets that descend can sum to more than 31 bits)
    }
  }
  __device__ __forceinline__ void init(const Args& p, int bm_, int bn_) {
    bm = bm_, bn = bn_, tiles_n = (p.n + bn - 1) / bn;
    if (!p.offsets) {
      total = (p.m + bm - 1) / bm * tiles_n;
      return;
    }
    total = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
      scan(p, g0);
      total = __builtin_elementwise_add_sat(total, __builtin_amdgcn_readlane(upto, 63));
    }
    total = min(total, (p.m / bm + min(p.groups, p.m)) * tiles_n);  // as the host's grid; offsets that ascend stay under it
  }
  __device__ __forceinline__ bool find(const Args& p, int id, Tile* t) {
    if (id >= total) return false;
    const int work = xcd_contiguous(id, total);
    int tm, tn;
    if (!p.offsets) {
      tile_walk(work, (p.m + bm - 1) / bm, tiles_n, &tm, &tn);
      t->group = 0, t->m0 = tm * bm, t->m_end = p.m, t->n0 = tn * bn;
      return true;
    }
    int before = 0;  // tiles of the experts in front
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
      if (p.groups > 64) scan(p, g0);  // up to 64 are still there
      const int in = work - before;
      const unsigned long long has = __ballot(in < upto);
      if (has) {
        const int l = __builtin_ctzll(has);  // the first expert whose tiles reach past this one
        const int glo = __builtin_amdgcn_readlane(lo, l), ghi = __builtin_amdgcn_readlane(hi, l);
        const int tiles_m = (ghi - glo + bm - 1) / bm, first = l ? __builtin_amdgcn_readlane(upto, l - 1) : 0;
        tile_walk(in - first, tiles_m, tiles_n, &tm, &tn);
        t->group = g0 + l, t->m0 = glo + tm * bm, t->m_end = ghi, t->n0 = tn * bn;
        return true;
      }
      before = __builtin_elementwise_add_sat(before, __builtin_amdgcn_readlane(upto, 63));
    }
    return false;
  }
};

// The weight gradient's tiles, an expert's rows as the contraction of each.  Every XCD takes an eighth of every expert's tiles,
// neighbours of the walk: the experts' numbers of rows differ, and with them what a tile costs (16k rows over 16 experts of 4096
// x 2048: 305 us, with whole experts dealt to the XCDs 470).
struct WgradTiles {
  int bm, bn, tiles_m, tiles_n, eighth, ids;
  int lo, hi;  // of expert `lane`

  __device__ __forceinline__ void init(const Args& p, int bm_, int bn_) {
    const int lane = threadIdx.x & 63;
    bm = bm_, bn = bn_, tiles_m = (p.m + bm - 1) / bm, tiles_n = (p.n + bn - 1) / bn, eighth = (tiles_m * tiles_n + 7) / 8;
    ids = p.groups * eighth * 8;
    lo = hi = 0;
    if (lane < p.groups) group_rows(p.offsets, lane, p.k, &lo, &hi);
  }
  __device__ __forceinline__ bool find(const Args& p, int id, Tile* t, int64_t* k_first, int* K) const {
    const int slot = id >> 3, work = (id & 7) * eighth + slot % eighth, g = slot / eighth;
    if (work >= tiles_m * tiles_n) return false;
    int tm, tn, first, end;
    tile_walk(work, tiles_m, tiles_n, &tm, &tn);
    t->group = g, t->m0 = tm * bm, t->m_end = p.m, t->n0 = tn * bn;
    if (g < 64) first = __builtin_amdgcn_readlane(lo, g), end = __builtin_amdgcn_readlane(hi, g);
    else group_rows(p.offsets, g, p.k, &first, &end);
    *k_first = first, *K = end - first;
    return true;
  }
};

// ------------------------------------------------------------------------------------------------------ LDS image --
// k contiguous: 8 rows x 128 bytes per KiB, which is what one wave-wide LDS-DMA instruction of 16 bytes a lane writes,
// the 16-byte chunks of row r permuted by chunk ^ swizzle(r).  A fragment read (ds_read_b128, lane (fr, fq): row fr, chunk
// fq or 4 + fq) is served in groups of 16 lanes that touch 16 rows; the permutation gives each group sixteen slots of its
// own.  It lives in the source address and in the read address, never in the DMA's destination.
__device__ __forceinline__ int chunk_swizzle(int row) { return ((row >> 1) & 3) << 1; }

// Transposed: 64 rows of k, the m or n side contiguous.  Fragments come through ds_read_b64_tr_b16: within each group of 16
// lanes lane i supplies the address of 4 elements of row i / 4, columns 4 (i % 4) .., and receives column i of the four rows.
// Half a wave touches rows 0-3 and 8-11 (and the like), 32 bytes each; the 32-byte units of a row are permuted by
// unit ^ unit_swizzle(row) so that these eight units lie in different banks (64 banks of 4 bytes).  COLS: columns of the image.
template <int COLS>
__device__ __forceinline__ int unit_swizzle(int row) {
  if constexpr (COLS >= 128) return ((row >> 3) & 1) * 4 + (row & 3);
  if constexpr (COLS == 64) return ((row >> 3) & 1) * 2 + ((row >> 1) & 1);
  if constexpr (COLS == 32) return (row >> 3) & 1;
  return 0;  // one unit a row
}

// One LDS-DMA instruction: SGPR base + 32-bit VGPR offset -> M0 + lane * BYTES.  Through the builtin every one costs a 64-bit
// vector add as well, and the compiler keeps the addresses of a whole step in registers.
template <int BYTES>
__device__ __forceinline__ void dma(const void* src, uint32_t off, char* dst) {
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst;
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(src), "s"(lds) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(src), "s"(lds) : "memory", "m0");
}

// One operand's way into LDS.  ROWS: rows of the tile (its m or n extent); WAVES share the 1-KiB pieces.
// HALVES = the rows WT of a wave's tile: the first half of a wave's pieces fill the first half of every wave's rows, so that
// the two halves can be fetched and waited for apart (transposed: an image of its own for each wave row and half); 0: no halves.
// DEAL (k contiguous, halves): LDS row 16 b + f of a wave's rows holds row f * (WT / 16) + b, so that a fragment lane's rows are
// consecutive.
template <bool TRANS, int ROWS, int WAVES, int HALVES, bool DEAL>
struct Stage {
  static constexpr int kPieces = ROWS / 8 / WAVES;
  static_assert(kPieces * 8 * WAVES == ROWS && (!HALVES || kPieces % 2 == 0), "whole pieces per wave and half");
  static constexpr int kCols = HALVES ? HALVES / 2 : ROWS;  // transposed: columns of an image
  static constexpr int kChunks = kCols / 8;                 // ... and 16-byte chunks of its rows, which is also its size in KiB
  const char* base;        // first row of the tile, first k
  uint32_t off[kPieces];   // a lane's place in it
  int64_t ld;

  // Which KiB of the tile's image piece i of a wave is.
  static __device__ __forceinline__ int place(int wave, int i) {
    if constexpr (HALVES == 0) {
      return wave * kPieces + i;
    } else {
      constexpr int per = kPieces / 2, block = HALVES / 16;  // pieces per wave and half; KiB of one wave row's half
      const int q = wave * per + i % per;                    // among the pieces of this half
      return q / block * 2 * block + i / per * block + q % block;
    }
  }
  // first: first row (column) of the tile, rows_left >= 1: how many of them exist; the rest repeat the last one.
  __device__ __forceinline__ void init(const char* p, int64_t ld_, int64_t first, int rows_left, int wave, int lane) {
    ld = ld_;
    base = TRANS ? p + first * 2 : p + first * ld;
#pragma unroll
    for (int i = 0; i < kPieces; i++) {
      const int piece = place(wave, i);
      if constexpr (TRANS) {
        const int image = piece / kChunks, pos = piece % kChunks * 64 + lane, r = pos / kChunks;
        const int c = (pos % kChunks) ^ (2 * unit_swizzle<kCols>(r));
        const int col = min(image * kCols + c * 8, rows_left - 8);  // the extent is a multiple of 8
        off[i] = (uint32_t)(r * ld) + (uint32_t)col * 2;
      } else {
        const int l = piece * 8 + (lane >> 3);
        int row = l;
        if constexpr (DEAL) row = l / HALVES * HALVES + (l & 15) * (HALVES / 16) + (l % HALVES >> 4);
        const int c = (lane & 7) ^ chunk_swizzle(l);
        off[i] = (uint32_t)(min(row, rows_left - 1) * ld) + (uint32_t)c * 16;
      }
    }
  }
  __device__ __forceinline__ const char* step_base(int kt) const {
    return base + (TRANS ? (int64_t)kt * 64 * ld : (int64_t)kt * kStepBytes);
  }
  // Piece i of a K-step that lies inside k as a whole.
  __device__ __forceinline__ void fetch(const char* src, char* tile, int wave, int i) const {
    dma<16>(src, off[i], tile + place(wave, i) * 1024);
  }
  // Piece i of any K-step; `left` = k (elements if transposed, bytes if not) from this step on: what lies beyond is zero.
  __device__ __forceinline__ void fetch_edge(const char* src, int64_t left, char* tile, int wave, int i) const {
    const int lane = threadIdx.x & 63;
    const int at = TRANS ? (place(wave, i) % kChunks * 64 + lane) / kChunks : ((lane & 7) ^ chunk_swizzle(lane >> 3)) * 16;  // its row or byte of k
    const bool in = at < left;
    const char* const from = in ? src + off[i] : (const char*)&g_zero16;
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)(tile + place(wave, i) * 1024), 16, 0, 0);
  }
};

// A wave's fragments of one operand: blocks of 16 rows, two halves of the K-step each (bf16: two substeps of 32 k; fp8:
// registers 0-3 and 4-7 of the one K = 128 operand).
template <bool TRANS, int ROWS, int NB, int HALVES>
struct Frags {
  static constexpr int kCols = HALVES ? HALVES / 2 : ROWS;
  int off[TRANS ? NB : 2];
  __device__ __forceinline__ void init(int first, int lane) {
    const int fr = lane & 15, fq = lane >> 4;
    if constexpr (TRANS) {
      const int r = 8 * fq + (fr >> 2);  // (rows 4, 32 and 36 further on have the same permutation)
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const int col = first + 16 * b;
        off[b] = col / kCols * (kCols * 128) + r * (kCols * 2) + ((col % kCols / 16) ^ unit_swizzle<kCols>(r)) * 32 + (fr & 3) * 8;
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
      const char* q = tile + off[b] + h * 32 * (kCols * 2);
      const i32x2 lo = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)q));
      const i32x2 hi = __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(q + 4 * (kCols * 2))));
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
// One K-step's fragment of an operand, by what it is multiplied as.  0: bf16.  1: e4m3 on the K = 128 fp8 instruction.  That
// instruction aligns the products of each group of eight k to the largest of them and drops what lies below 2^-13 of its binade
// (measured with one large and one small product per group; the K = 32 and K = 64 fp8 forms do the same), at most 2^-10 of the
// sum of magnitudes; on average 1.1e-5 of the results' rms on normal data and 2.2 to 2.9e-5 where one channel in a hundred is
// twenty times as large (K of 2048 to 8192).  A bf16 result takes it where the matrix pipe is what bounds it: one element in a hundred or
// fifty becomes a neighbour of the nearest bf16, and the error against 64 bits, 1.66e-3 rms, grows by at most 4e-7.  Where large
// products cancel, what is dropped can exceed the rounding of the small result.  An f32 result does not take it, nor a bf16 one of
// few rows, for which it would gain nothing: for them (2) the elements are widened to bf16 and multiplied on the bf16 instruction,
// which keeps f32 sums (1e-7), at half the rate.
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

// ------------------------------------------------------------------------------------------------------ tile kernel --
// BM x BN of C per workgroup, WM x WN waves, two buffers of a K-step each in LDS, refilled in halves while the other is computed
// on.  The MFMA takes B's fragment first, so lane (fr, fq) of a 16 x 16 block holds row fr and columns 4 fq .. 4 fq + 3.
// Compute-bound: 8192^3 takes 440 us of e4m3 (2.50 PFLOP/s; the multiply-adds of the scales, 64 registers a wave and step, run
// beside the matrix pipe) and 705 us of bf16 (1.56 PFLOP/s; with four waves of 128 x 128, which read a third less LDS, the same).
// What a short K pays on top is the epilogue, 4 to 5 us of a tile, and the first step's latency: 32k rows of 32 experts, 4096 x
// 2048 bf16, 485 us (1.13 PFLOP/s).
//
// Block-scaled fp8: the matrix instruction sums one block of 128 k from zero and its result is added with one FMA per
// element, acc += (sa * sb) * block.  With rows dealt to lanes (Stage's DEAL) a lane's scales of A are MB consecutive floats
// per K-step, and B's tile scale is one scalar per wave.
template <int KIND, int BM, int BN, int WM, int WN, bool MANY, typename OUT>
struct TileLds {  // two buffers of operands and scales; MANY: behind them the epilogue's strips, which else take their place
  static constexpr bool kNarrow = sizeof(OUT) == 2;
  static constexpr int kOperands = (BM + BN) * kStepBytes, kScales = KIND != kBf16 ? WM * WN * 256 : 0;
  static constexpr int kStripRows = kNarrow ? 16 : 8, kStrip = BN / WN * (int)sizeof(OUT) + 16, kStrips = WM * WN * kStripRows * kStrip;
  static_assert(kStrips <= 2 * kOperands, "the epilogue's strips fit into the operand buffers");
  static constexpr int kBytes = 2 * (kOperands + kScales) + (MANY ? kStrips : 0);
};
// Computes the tiles that next(&tile, &k_first, &K) names until it returns false; without MANY one.
template <int KIND, bool TA, bool TB, bool WGRAD, int BM, int BN, int WM, int WN, bool MANY, typename OUT, typename NEXT>
__device__ __forceinline__ void compute_tiles(const Args& p, char* const smem, NEXT next_tile) {
  constexpr int kWaves = WM * WN, WTM = BM / WM, WTN = BN / WN, MB = WTM / 16, NB = WTN / 16;
  constexpr bool kFp8 = KIND != kBf16, kNarrow = sizeof(OUT) == 2;
  constexpr int kElem = kFp8 ? 1 : 2, kStepK = kStepBytes / kElem;
  static_assert(!kFp8 || (!TA && !TB && WTN <= 128), "block-scaled fp8: k contiguous, a wave's columns inside one tile of scales");
  typedef TileLds<KIND, BM, BN, WM, WN, MANY, OUT> Lds;
  constexpr int kABytes = BM * kStepBytes, kBufBytes = Lds::kOperands, kScaleBytes = Lds::kScales;
  constexpr int kStripRows = Lds::kStripRows, kStrip = Lds::kStrip, kStripBytes = kStripRows * kStrip;
  static_assert(!kFp8 || BM / 64 + (KIND == kFp8Rows ? BN / 64 : 1) <= kWaves, "one DMA of scales per wave and step");
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;

  Tile t{0, 0, 0, 0};  // the tile at hand
  int64_t k_first = 0;
  int K = p.k;
  auto locate = [&]() {
    const bool found = next_tile(&t, &k_first, &K);
    // (uniform as they are; said so, the compiler keeps them, and the DMA's base addresses, in scalar registers across the loop)
    t.group = __builtin_amdgcn_readfirstlane(t.group), t.m0 = __builtin_amdgcn_readfirstlane(t.m0);
    t.m_end = __builtin_amdgcn_readfirstlane(t.m_end), t.n0 = __builtin_amdgcn_readfirstlane(t.n0);
    k_first = __builtin_amdgcn_readfirstlane((int)k_first), K = __builtin_amdgcn_readfirstlane(K);
    return (bool)__builtin_amdgcn_readfirstlane(found);
  };
  if (!locate()) return;  // the whole workgroup, before any barrier
  typedef Stage<TA, BM, kWaves, WTM, kFp8> StageA;
  typedef Stage<TB, BN, kWaves, 0, false> StageB;
  StageA ga;
  StageB gb;
  Frags<TA, BM, MB, WTM> fa;
  Frags<TB, BN, NB, 0> fb;
  fa.init(wm * WTM, lane);
  fb.init(wn * WTN, lane);

  f32x4 acc[MB][NB];

  // Scales of one K-step travel with its operands: A's of the tile's rows and B's of its columns (or of its 128-column
  // tiles) in a slot of their own behind the operand buffers, one DMA of 4 bytes a lane for 64 of them.  Loaded by each wave for
  // itself into registers they cost more than the matrix work: nine loads of their own per lane, wave and step.
  const float* scale_src = nullptr;  // at step 0, this wave's part
  uint32_t scale_off = 0;            // this lane's place in it
  int64_t scale_ld = 0;
  auto scales_of_tile = [&](int lane) {
    const float* const SB = p.sb + t.group * p.stride_sb;
    if (wave < BM / 64) {
      const int row = t.m0 + wave * 64;
      scale_src = p.sa + min(row, t.m_end - 1), scale_ld = p.ld_sa;
      scale_off = (uint32_t)max(min(lane, t.m_end - 1 - row), 0) * 4;
    } else if (KIND == kFp8Rows) {
      const int col = t.n0 + (wave - BM / 64) * 64;
      scale_src = SB + min(col, p.n - 1), scale_ld = p.ld_sb;
      scale_off = (uint32_t)max(min(lane, p.n - 1 - col), 0) * 4;
    } else {  // (all waves that are left, so that every wave has as many DMAs in flight)
      scale_src = SB + (int64_t)(t.n0 / 128) * p.ld_sb, scale_ld = 1;
      scale_off = (uint32_t)(min(min(lane, BN / 128 - 1), (p.n - 1) / 128 - t.n0 / 128) * p.ld_sb * 4);
    }
  };
  auto fetch_scales = [&](int kt) {
    dma<4>(scale_src + kt * scale_ld, scale_off, smem + 2 * kBufBytes + (kt & 1) * kScaleBytes + wave * 256);
  };
  constexpr int kSb = KIND == kFp8Rows ? NB : 1;
  float sl[MB];   // sa * sb (tiles) or sa (rows) of the running step
  f32x4 sb[kSb];  // rows: sb of this lane's columns
  auto read_scales = [&](int kt) {
    const float* const q = (const float*)(smem + 2 * kBufBytes + (kt & 1) * kScaleBytes);
#pragma unroll
    for (int i = 0; i < MB; i += 2) {
      const f32x2 v = *(const f32x2*)(q + wm * WTM + fr * MB + i);
      sl[i] = v[0], sl[i + 1] = v[1];
    }
    if constexpr (KIND == kFp8Tiles) {
      sb[0][0] = q[BM + wn * WTN / 128];
    } else {
#pragma unroll
      for (int j = 0; j < NB; j++) sb[j] = *(const f32x4*)(q + BM + wn * WTN + j * 16 + fq * 4);
    }
  };
  auto join_scales = [&]() {  // tiles; apart from the reads, which it has to wait for
#pragma unroll
    for (int i = 0; i < MB; i++) sl[i] *= sb[0][0];
  };

  int steps = 0, whole = 0;  // K-steps; those that lie inside k
  auto prepare = [&]() {
    int own = lane;
    asm volatile("" : "+v"(own));  // as in store_tile
    ga.init(p.a + (TA ? k_first * p.lda : 0), p.lda, t.m0, t.m_end - t.m0, wave, own);
    gb.init(p.b + (WGRAD ? 0 : t.group * p.stride_b) + (TB ? k_first * p.ldb : 0), p.ldb, t.n0, p.n - t.n0, wave, own);
    if constexpr (kFp8) scales_of_tile(own);
    steps = (int)(((int64_t)K + kStepK - 1) / kStepK), whole = K / kStepK;
  };
  // The DMAs of one step and wave in the order they are issued: B, the first half of A, the scales (the first kFirst), and
  // the second half of A (kSecond).
  constexpr int kHalfA = StageA::kPieces / 2, kFirst = StageB::kPieces + kHalfA + (kFp8 ? 1 : 0), kSecond = kHalfA;
  auto fetch = [&](int kt, const char* src_a, const char* src_b, int piece) {
    char* const buf = smem + (kt & 1) * kBufBytes;
    if (piece < StageB::kPieces) gb.fetch(src_b, buf + kABytes, wave, piece);
    else if (piece < StageB::kPieces + kHalfA) ga.fetch(src_a, buf, wave, piece - StageB::kPieces);
    else if (kFp8 && piece == kFirst - 1) fetch_scales(kt);
    else ga.fetch(src_a, buf, wave, piece - kFirst + kHalfA);
  };
  auto fetch_edge = [&](int kt, int from, int to) {
    char* const buf = smem + (kt & 1) * kBufBytes;
    const int64_t left = (int64_t)K - (int64_t)kt * kStepK;
#pragma unroll
    for (int piece = from; piece < to; piece++) {
      if (piece < StageB::kPieces) gb.fetch_edge(gb.step_base(kt), TB ? left : left * kElem, buf + kABytes, wave, piece);
      else if (piece < StageB::kPieces + kHalfA) ga.fetch_edge(ga.step_base(kt), TA ? left : left * kElem, buf, wave, piece - StageB::kPieces);
      else if (kFp8 && piece == kFirst - 1) fetch_scales(kt);
      else ga.fetch_edge(ga.step_base(kt), TA ? left : left * kElem, buf, wave, piece - kFirst + kHalfA);
    }
  };

  // One step multiplies the wave's MB row blocks by its NB column blocks, row by row, A's fragment of the next row block being
  // read meanwhile; B's stay in registers for the step.  The last two row blocks go in halves, (MB-2, first half) | (MB-1, first
  // half) (MB-2, second half) (MB-1, second half), and behind the bar each of B's fragments of the next step is read as soon as
  // its registers have been consumed, so that the matrix pipe does not drain at a step's edge.
  // Two buffers, refilled in halves so that the DMA never drains either: two synchronisations per step,
  //   kMid (the first half of A and all of B have been read): the second half of A must have landed; B, the first half of A and
  //        the scales of step kt + 2 go out;
  //   kBar (all of A has been read): B, the first half of A and the scales of step kt + 1 must have landed; the second half of A
  //        of step kt + 2 goes out.
  // Each has one and a half steps to arrive, with the other group in flight behind it (the counted waits).  With the whole
  // buffer refilled at kBar and waited for a step later, a step could not be shorter than a memory latency plus its 64 KiB:
  // 8192^3 block-scaled 505 us, in halves 454.
  constexpr int kProducts = MB * NB, kTail = (MB - 2) * NB, kHalf = NB / 2, kBar = kTail + kHalf, kMid = (MB / 2 - 1) * NB;
  constexpr int kPer = (kFirst + kBar - kMid - 1) / (kBar - kMid);  // DMAs behind one product, all of the first group before kBar
  static_assert(MB % 2 == 0 && NB == 4 && kSecond <= kProducts - kBar, "the pieces fit behind the products");
  auto row_of = [](int at) { return at < kTail ? at / NB : MB - 2 + (at - kTail) / kHalf % 2; };
  auto col_of = [](int at) { return at < kTail ? at % NB : (at - kTail) % kHalf + (at - kTail >= NB ? kHalf : 0); };
  typedef Operand<kFp8 ? (kNarrow ? 1 : 2) : 0> Op;
  Op bf[NB], af[2];
  f32x4 part[4];       // block sums on their way to the accumulators, two MFMAs behind
  float s_tail[2];     // the scales of the last two row blocks, while the next step's arrive
  auto add = [&](int at) {
    const int i = row_of(at), j = col_of(at);
    const float s = KIND == kFp8Rows || i < MB - 2 ? sl[i] : s_tail[i - (MB - 2)];
#pragma unroll
    for (int r = 0; r < 4; r++)
      acc[i][j][r] = __builtin_fmaf(KIND == kFp8Tiles ? s : s * sb[KIND == kFp8Tiles ? 0 : j][r], part[at & 3][r], acc[i][j][r]);
    asm volatile("" : "+v"(acc[i][j]));  // here, between the MFMAs: left to itself the compiler sinks all of them behind the last
  };
  // vmcnt(behind) lgkmcnt(0) and a barrier; `behind`: DMAs that may stay in flight, and with `stored` the stores of the tile before.
  constexpr int kStores = MB * 16 * (int)sizeof(OUT) / 16 * (WTN / 4) / 16;
  bool after_stores = false;  // exactly kStores of them were issued behind the DMAs of steps 0 and 1
  auto sync = [&](auto behind, bool stored = false) {
    constexpr int n = decltype(behind)::value, m = n + kStores;
    static_assert(!MANY || m < 64, "vmcnt counts to 63");
    if (MANY && stored) __builtin_amdgcn_s_waitcnt((m & 15) | 0x70 | (m >> 4) << 14);
    else __builtin_amdgcn_s_waitcnt((n & 15) | 0x70 | (n >> 4) << 14);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  const std::integral_constant<int, 0> none;
  const std::integral_constant<int, kFirst + kSecond> step_behind;
  auto begin = [&]() {
    if (steps > 0) fetch_edge(0, 0, kFirst + kSecond);
    if (steps > 1) fetch_edge(1, 0, kFirst + kSecond);
  };
  auto first_fragments = [&]() {
    if (steps > 1) sync(std::integral_constant<int, kFirst + 2 * kSecond>(), after_stores);
    else sync(none);
#pragma unroll
    for (int j = 0; j < NB; j++) {
      bf[j].set(fb.read(smem + kABytes, j, 0), fb.read(smem + kABytes, j, 1));
      if (j == kHalf - 1) af[0].set(fa.read(smem, 0, 0), fa.read(smem, 0, 1));
    }
    if constexpr (kFp8) {
      read_scales(0);
      if constexpr (KIND == kFp8Tiles) join_scales();
#pragma unroll
      for (int i = 0; i < 4; i++) part[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      s_tail[0] = s_tail[1] = 0.f;
    }
  };
  // FULL: step kt + 2 exists and lies inside k.
  auto step = [&](int kt, auto FULL) {
    constexpr bool kFull = decltype(FULL)::value;
    const char* const la = smem + (kt & 1) * kBufBytes;
    const char* const na = smem + ((kt + 1) & 1) * kBufBytes;
    const char* const nb = na + kABytes;
    const bool more = kFull || kt + 1 < steps, more2 = kFull || kt + 2 < steps;  // (in flight behind kMid's and kBar's)
    const char* const src_a = ga.step_base(kt + 2);
    const char* const src_b = gb.step_base(kt + 2);
#pragma unroll
    for (int at = 0; at < kProducts; at++) {
      const int i = row_of(at), j = col_of(at);
      if (at == kMid) {
        if (more) sync(step_behind, after_stores && kt <= 1);
        else sync(none);
        if (!kFull && more2) fetch_edge(kt + 2, 0, kFirst);
      }
      if (at % NB == 0 && at <= kTail) af[(i + 1) & 1].set(fa.read(la, i + 1, 0), fa.read(la, i + 1, 1));
      if (at == kBar) {
        if (more2) sync(step_behind, after_stores && kt == 0);
        else sync(none);
        if (!kFull && more2) fetch_edge(kt + 2, kFirst, kFirst + kSecond);
        if constexpr (KIND == kFp8Tiles) {
          s_tail[0] = sl[MB - 2], s_tail[1] = sl[MB - 1];
          read_scales(kt + 1);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kFp8) {
        part[at & 3] = Op::product(bf[j], af[i & 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (KIND == kFp8Tiles || at >= 2) add((at + kProducts - 2) % kProducts);  // (at first the last two of the step before, or zeros)
      } else {
        Op::accumulate(bf[j], af[i & 1], acc[i][j]);
      }
      if (i == MB - 1) bf[j].set(fb.read(nb, j, 0), fb.read(nb, j, 1));  // (behind the last step: landed data that nothing uses)
      if (at == kTail + NB + kHalf - 1) af[0].set(fa.read(na, 0, 0), fa.read(na, 0, 1));
      if constexpr (kFull) {
        if (at >= kMid && at < kBar) {
#pragma unroll
          for (int q = (at - kMid) * kPer; q < (at - kMid + 1) * kPer && q < kFirst; q++) fetch(kt + 2, src_a, src_b, q);
        } else if (at >= kBar && at - kBar < kSecond) {
          fetch(kt + 2, src_a, src_b, kFirst + at - kBar);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (KIND == kFp8Tiles) {
      join_scales();
    } else if constexpr (kFp8) {  // no registers for a second set of B's scales: the last two sums are added first
      add(kProducts - 2);
      add(kProducts - 1);
      read_scales(kt + 1);
    }
  };
  // A wave whose part of the tile has no rows or columns of C keeps its share of the DMAs and the synchronisations and leaves the
  // matrix pipe to the wave beside it.
  auto idle_steps = [&]() {
    if (steps > 1) sync(std::integral_constant<int, kFirst + 2 * kSecond>(), after_stores);
    else sync(none);
    for (int kt = 0; kt < steps; kt++) {
      const bool more = kt + 1 < steps, more2 = kt + 2 < steps;
      if (more) sync(step_behind, after_stores && kt <= 1);
      else sync(none);
      if (more2) fetch_edge(kt + 2, 0, kFirst);
      if (more2) sync(step_behind, after_stores && kt == 0);
      else sync(none);
      if (more2) fetch_edge(kt + 2, kFirst, kFirst + kSecond);
    }
  };
  // Epilogue: kStripRows rows of a wave's tile at a time through a strip of LDS of its own, so that neighbouring lanes store
  // neighbouring columns of one row.
  constexpr int kCols16 = 16 / (int)sizeof(OUT);  // columns of a 16-byte store
  constexpr int kLanesPerRow = WTN / kCols16, kRowsPerPass = 64 / kLanesPerRow;
  char* const strip = smem + (MANY ? 2 * (kBufBytes + kScaleBytes) : 0) + wave * kStripBytes;
  auto store_tile = [&](const Tile& o, auto FULL) {
    int own = lane;
    asm volatile("" : "+v"(own));  // what follows from the lane is worked out here and not kept in registers across the K loop
    const int strip_row = own / kLanesPerRow, strip_col = own % kLanesPerRow * kCols16, fr = own & 15, fq = own >> 4;
    constexpr int kApart = kFp8 ? MB : 1;  // rows of C between rows of the strip
    const uint32_t off = (uint32_t)((strip_row * kApart * p.ldc + strip_col) * (int)sizeof(OUT));
    OUT* const base = (OUT*)p.c + (WGRAD ? o.group * p.stride_c : 0) + (int64_t)(o.m0 + wm * WTM) * p.ldc + o.n0 + wn * WTN;
    const bool col_in = o.n0 + wn * WTN + strip_col < p.n;  // N is a multiple of 8
#pragma unroll
    for (int i = 0; i < MB; i++) {
#pragma unroll
      for (int h = 0; h < 16 / kStripRows; h++) {
        if (kNarrow || fr / kStripRows == h) {
#pragma unroll
          for (int j = 0; j < NB; j++) {
            OUT* const to = (OUT*)(strip + fr % kStripRows * kStrip) + j * 16 + fq * 4;
            if constexpr (kNarrow) *(bf16x4*)to = __builtin_convertvector(acc[i][j], bf16x4);
            else *(f32x4*)to = acc[i][j];
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r0 = 0; r0 < kStripRows; r0 += kRowsPerPass) {
          const int row = kFp8 ? (h * kStripRows + r0) * MB + i : i * 16 + h * kStripRows + r0;  // of the pass's first strip row
          char* const to = (char*)(base + row * p.ldc);
          const u32x4 v = *(const u32x4*)(strip + (r0 + strip_row) * kStrip + strip_col * (int)sizeof(OUT));
          // As asm, so that there are exactly kStores of them for the counted waits (and the wait state that a wide store's data
          // needs).
          if constexpr (decltype(FULL)::value == 2) {
            asm volatile("global_store_dwordx4 %0, %1, %2 nt\n\ts_nop 1" ::"v"(off), "v"(v), "s"(to) : "memory");
          } else if constexpr (decltype(FULL)::value == 1) {
            asm volatile("global_store_dwordx4 %0, %1, %2\n\ts_nop 1" ::"v"(off), "v"(v), "s"(to) : "memory");
          } else if (o.m0 + wm * WTM + row + strip_row * kApart < o.m_end && col_in) {
            *(u32x4*)(to + off) = v;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  };

  const bool lines = MANY && (((uintptr_t)p.c | (uintptr_t)(p.ldc * (int)sizeof(OUT))) & 127) == 0;
  prepare();
  begin();
  for (;;) {
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
      for (int j = 0; j < NB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (t.m0 + wm * WTM >= t.m_end || t.n0 + wn * WTN >= p.n) {
      if (steps > 0) idle_steps();
    } else if (steps > 0) {
      first_fragments();
      int kt = 0;
      for (; kt + 2 < whole; kt++) step(kt, std::true_type());
      for (; kt < steps; kt++) step(kt, std::false_type());
      if constexpr (KIND == kFp8Tiles) {
        add(kProducts - 2);
        add(kProducts - 1);
      }
    }
    // Since the last kBar nothing but registers is needed of this tile's operands, so the next tile's first steps are on
    // their way while this one is stored (and its stores while the next one is computed on).
    const Tile o = t;
    bool next = false;
    if constexpr (MANY) {
      next = locate();
      if (next) {
        prepare();
        begin();
      }
    } else {
      __syncthreads();  // the strips lie in the operand buffers: every wave is done with them
    }
    const bool full = MANY && o.m0 + BM <= o.m_end && o.n0 + BN <= p.n;
    // Whole lines go past the caches, which would not keep a result of that many tiles (8192^3 bf16 dgrad 728 us, through them
    // 764); rows that do not begin at a line share theirs with the next tile (5120 x 8184 x 352: 47.5 us through the caches, 58.0).
    if (!full) store_tile(o, std::integral_constant<int, 0>());
    else if (lines) store_tile(o, std::integral_constant<int, MANY ? 2 : 0>());
    else store_tile(o, std::integral_constant<int, MANY ? 1 : 0>());
    if (!next) break;
    after_stores = full;
  }
}

// MANY: kCUs workgroups walk the tiles, one of 256 x 256 a CU, ids blockIdx.x, blockIdx.x + kCUs, ...  What is left for a last
// round of up to half the CUs is computed in quarters of those tiles, by twice or four times as many CUs.
template <int KIND, bool TA, bool TB, bool WGRAD, int BM, int BN, int WM, int WN, bool MANY, typename OUT>
__global__ __launch_bounds__(WM * WN * 64) void tile_kernel(Args p) {
  typedef TileLds<KIND, BM, BN, WM, WN, MANY, OUT> Lds;
  __shared__ __attribute__((aligned(16))) char smem[Lds::kBytes];
  // MANY: a round of ids on, and 17 of 32 places along this XCD's part of it: what comes at a fixed distance and costs more or less
  // than the rest (rows of tiles that an expert's end leaves part empty, experts) would fall to the same workgroups (32 experts of
  // 640 rows, 4096 x 7168 e4m3: 556 us; one place 580, none 645).
  int id = blockIdx.x;
  auto next_id = [&]() { return (id & ~(kCUs - 1)) + kCUs + ((id + 17 * 8) & (kCUs - 1)); };
  if constexpr (WGRAD) {
    WgradTiles tiles;
    tiles.init(p, BM, BN);
    compute_tiles<KIND, TA, TB, WGRAD, BM, BN, WM, WN, MANY, OUT>(p, smem, [&](Tile* t, int64_t* k_first, int* K) {
      bool found = false;
      while (!found && id < tiles.ids) {
        found = tiles.find(p, id, t, k_first, K);
        id = MANY ? next_id() : tiles.ids;
      }
      return found;
    });
  } else if constexpr (!MANY) {
    compute_tiles<KIND, TA, TB, WGRAD, BM, BN, WM, WN, false, OUT>(p, smem, [&](Tile* t, int64_t*, int*) {
      RowTiles tiles;
      tiles.init(p, BM, BN);
      return tiles.find(p, blockIdx.x, t);
    });
  } else {
    RowTiles tiles;
    tiles.init(p, BM, BN);
    const int rest = tiles.total % kCUs, quartered = rest <= kCUs / 2 ? rest : 0, whole = tiles.total - quartered;
    compute_tiles<KIND, TA, TB, WGRAD, BM, BN, WM, WN, true, OUT>(p, smem, [&](Tile* t, int64_t*, int*) {
      if (id >= whole) return false;
      const bool found = tiles.find(p, id, t);
      id = next_id();
      return found;
    });
    typedef TileLds<KIND, BM / 2, BN / 2, 4, 2, false, OUT> Quarter;
    static_assert(WM * WN == 8 && Quarter::kBytes <= Lds::kBytes, "the same waves and LDS");
    for (int q = blockIdx.x; q < (quartered + 7) / 8 * 32; q += kCUs) {  // eight tiles at a time, so that an XCD has a tile's quarters
      const int of = whole + q / 32 * 8 + q % 8, part = q / 8 % 4;
      __syncthreads();  // the LDS of what came before
      compute_tiles<KIND, TA, TB, WGRAD, BM / 2, BN / 2, 4, 2, false, OUT>(p, smem, [&](Tile* t, int64_t*, int*) {
        if (!tiles.find(p, of, t)) return false;
        t->m0 += part / 2 * (BM / 2), t->n0 += part % 2 * (BN / 2);
        return t->m0 < t->m_end && t->n0 < p.n;
      });
    }
  }
}

// ---------------------------------------------------------------------------------------------------- few-row kernel --
// 16 MB rows by 16 NB columns per workgroup, whose W waves share the K-steps in turn.  What bounds a product of few rows is the
// rate at which operands come in, and the tile above leaves most of the chip idle: here K is spread over the waves, every wave
// walks its own steps through a ring of U slots of LDS that no other wave touches (no barrier until the end), and the W sums
// are joined in LDS in the order of the waves.
// Through LDS and not straight into registers because of the address path: it takes a quad of lanes that asks for 64
// contiguous bytes in one cycle, but lanes of an MFMA operand are neighbours in different rows, one lane a cycle (64 rows of
// 512 x 8192 e4m3: 21.7 us loaded directly, 9.3 this way).  64 experts of 4096 x 7168 e4m3, of which 69 rows reach 38, 183 us, 6.1 TB/s; one token
// through 4096 x 7168 5.4 us from the caches, three of which are the launch and the first step's latency.
// WIDE: e4m3 elements are widened and multiplied as bf16, with f32 sums, for a bf16 result as well.
template <int KIND, bool TA, bool TB, int MB, int NB, int W, int U, bool WIDE, typename OUT>
__global__ __launch_bounds__(W * 64) void few_rows_kernel(Args p) {
  constexpr bool kFp8 = KIND != kBf16, kWgrad = TA;
  constexpr int kElem = kFp8 ? 1 : 2, kStepK = kStepBytes / kElem;
  constexpr int kPieces = 2 * (MB + NB), kScaleDmas = !kFp8 ? 0 : KIND == kFp8Rows ? 2 : 1, kDmas = kPieces + kScaleDmas;
  constexpr int kSlot = kPieces * 1024 + kScaleDmas * 256;
  static_assert(MB <= 4 && NB <= 4 && 128 % (NB * 16) == 0, "a step's scales in one DMA each, the columns inside one tile of scales");
  static_assert((U - 1) * kDmas < 64 && W * MB * NB * 1024 <= W * U * kSlot, "vmcnt counts to 63; the sums fit into the ring");
  static_assert(!kFp8 || (!TA && !TB), "block-scaled fp8: k contiguous");
  __shared__ __attribute__((aligned(16))) char smem[W * U * kSlot];
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Tile t;
  int64_t k_first = 0;
  int K = p.k;
  if constexpr (kWgrad) {
    WgradTiles tiles;
    tiles.init(p, MB * 16, NB * 16);
    if (!tiles.find(p, blockIdx.x, &t, &k_first, &K)) return;
  } else {
    RowTiles tiles;
    tiles.init(p, MB * 16, NB * 16);
    if (!tiles.find(p, blockIdx.x, &t)) return;
  }
  const int steps = (int)(((int64_t)K + kStepK - 1) / kStepK), whole = K / kStepK;
  const int mine = steps > wave ? (steps - wave + W - 1) / W : 0;  // this wave's: wave, wave + W, ...
  char* const ring = smem + wave * U * kSlot;

  Stage<TA, MB * 16, 1, 0, false> ga;
  Stage<TB, NB * 16, 1, 0, false> gb;
  ga.init(p.a + (TA ? k_first * p.lda : 0), p.lda, t.m0, t.m_end - t.m0, 0, lane);
  gb.init(p.b + (kWgrad ? 0 : t.group * p.stride_b) + (TB ? k_first * p.ldb : 0), p.ldb, t.n0, p.n - t.n0, 0, lane);
  Frags<TA, MB * 16, MB, 0> fa;
  Frags<TB, NB * 16, NB, 0> fb;
  fa.init(0, lane);
  fb.init(0, lane);
  const float* const sa_base = kFp8 ? p.sa + t.m0 : nullptr;
  const uint32_t sa_off = (uint32_t)min(lane, t.m_end - 1 - t.m0) * 4;
  const float* const SB = !kFp8 ? nullptr : p.sb + t.group * p.stride_sb + (KIND == kFp8Rows ? (int64_t)t.n0 : (int64_t)(t.n0 / 128) * p.ld_sb);
  const uint32_t sb_off = (uint32_t)min(lane, p.n - 1 - t.n0) * 4;
  auto issue = [&](int s) {
    const int kt = wave + s * W;
    char* const slot = ring + s % U * kSlot;
    if (kt < whole) {
      const char* const at_a = ga.step_base(kt);
      const char* const at_b = gb.step_base(kt);
#pragma unroll
      for (int i = 0; i < 2 * MB; i++) ga.fetch(at_a, slot, 0, i);
#pragma unroll
      for (int i = 0; i < 2 * NB; i++) gb.fetch(at_b, slot + MB * 2048, 0, i);
    } else {  // K ends inside this step: zeros behind it
      const int64_t left = (int64_t)K - (int64_t)kt * kStepK;
#pragma unroll
      for (int i = 0; i < 2 * MB; i++) ga.fetch_edge(ga.step_base(kt), TA ? left : left * kElem, slot, 0, i);
#pragma unroll
      for (int i = 0; i < 2 * NB; i++) gb.fetch_edge(gb.step_base(kt), TB ? left : left * kElem, slot + MB * 2048, 0, i);
    }
    if constexpr (kFp8) dma<4>(sa_base + kt * p.ld_sa, sa_off, slot + kPieces * 1024);
    if constexpr (KIND == kFp8Rows) dma<4>(SB + kt * p.ld_sb, sb_off, slot + kPieces * 1024 + 256);
  };
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; i++)
#pragma unroll
    for (int j = 0; j < NB; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < U; u++)
    if (u < mine) issue(u);
  for (int s = 0; s < mine; s++) {
    // the oldest slot has landed: the U - 1 behind it may be in flight
    if (s + U <= mine) __builtin_amdgcn_s_waitcnt(((U - 1) * kDmas & 15) | 0xf70 | ((U - 1) * kDmas >> 4) << 14);
    else __builtin_amdgcn_s_waitcnt(0xf70);
    asm volatile("" ::: "memory");
    const char* const slot = ring + s % U * kSlot;
    typedef Operand<kFp8 ? (WIDE ? 2 : 1) : 0> Op;
    Op af[MB], bf[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) bf[j].set(fb.read(slot + MB * 2048, j, 0), fb.read(slot + MB * 2048, j, 1));
#pragma unroll
    for (int i = 0; i < MB; i++) af[i].set(fa.read(slot, i, 0), fa.read(slot, i, 1));
    float sa[MB];
    f32x4 sb[KIND == kFp8Rows ? NB : 1];
    if constexpr (kFp8) {
      const float* const q = (const float*)(slot + kPieces * 1024);
#pragma unroll
      for (int i = 0; i < MB; i++) sa[i] = q[i * 16 + fr];
      if constexpr (KIND == kFp8Tiles) {
        sb[0][0] = ((const __attribute__((address_space(4))) float*)SB)[wave + s * W];  // one scalar load
      } else {
#pragma unroll
        for (int j = 0; j < NB; j++) sb[j] = *(const f32x4*)(q + 64 + j * 16 + fq * 4);
      }
    }
    if (s + U < mine) {
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot has been read and can be refilled
      asm volatile("" ::: "memory");
      issue(s + U);
    }
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
      for (int j = 0; j < NB; j++) {
        if constexpr (kFp8) {
          const f32x4 part = Op::product(bf[j], af[i]);
#pragma unroll
          for (int r = 0; r < 4; r++)
            acc[i][j][r] = __builtin_fmaf(sa[i] * (KIND == kFp8Tiles ? sb[0][0] : sb[KIND == kFp8Tiles ? 0 : j][r]), part[r], acc[i][j][r]);
        } else {
          Op::accumulate(bf[j], af[i], acc[i][j]);
        }
      }
  }
  __syncthreads();
  f32x4* const sums = (f32x4*)smem;  // [wave][block][lane]
#pragma unroll
  for (int i = 0; i < MB; i++)
#pragma unroll
    for (int j = 0; j < NB; j++) sums[(wave * MB * NB + i * NB + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int q = wave; q < MB * NB; q += W) {
    f32x4 v = sums[q * 64 + lane];
#pragma unroll
    for (int w = 1; w < W; w++) v += sums[(w * MB * NB + q) * 64 + lane];
    const int r = t.m0 + q / NB * 16 + fr, col = t.n0 + q % NB * 16 + fq * 4;
    if (r < t.m_end && col < p.n) {
      OUT* dst = (OUT*)p.c + (kWgrad ? t.group * p.stride_c : 0) + r * p.ldc + col;
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
inline int64_t grid_for(const Args& p, bool wgrad, int bm, int bn) {
  if (!wgrad) return grid_of(p, bm, bn);
  const int64_t tiles = (((int64_t)p.m + bm - 1) / bm) * (((int64_t)p.n + bn - 1) / bn);
  return p.groups * ((tiles + 7) / 8 * 8);  // WgradTiles
}
// Sizes and grids up to here: rounded up to a tile, or a round of workgroups further, they still fit 31 bits.
constexpr int kMaxSize = 0x7fffffff - 1023;
// A launch holds fewer than 2^32 threads.
inline int launched(const char* what, int64_t grid, int threads) {
  if (grid <= 0 || grid > kMaxSize || grid * threads >= (int64_t)1 << 32) {
    set_error("%s: %lld workgroups of %d threads do not fit into one launch", what, (long long)grid, threads);
    return GMD_ERR_BADPARAM;
  }
  return GMD_OK;
}

// The K-contiguous product (forward, and every block-scaled one): which kernel.
// `rows` is what one product has: all of them, or an expert's share on average (the host does not see the offsets).
// * The few-row kernel gives a workgroup 16 MB x 16 NB of C with K spread over its waves.  MB is 1 up to 16 rows, 2 up to 32 and 4
//   beyond; NB is the smallest of 1, 2 and 4 whose grid still fits the chip at one workgroup a CU: every doubling of NB
//   halves the times A is read, but a CU without a workgroup is lost (32 x 4096 x 7168 e4m3: NB 1 9.9 us, NB 2 12.0; 32 x 7168 x
//   2048: 8.2 and 6.0).  Past that, NB 4: up to 32 rows always, since what is read then is B, once; with more rows up to two
//   workgroups a CU (128 x 7168 x 2048: 9.8 us, tiles 14.6; 512 x 3840 x 2048: 13.6 and 13.7).  Over 32 rows two of these shapes
//   are traded for one of 32 rows: 64 x 16 for 32 x 32, and 64 x 64 that are between one and two a CU for 32 x 64 where those are
//   at most two a CU as well (203 x 4120 x 2064: 10.0 us, in 64 x 64 13.5, in tiles 17.3).
// * Experts with up to 32 rows on average take it as well, in workgroups of four waves so that several fit on a CU and hide each
//   other's start: 64 experts of 2048 x 2048 bf16 for 64 rows 43.4 us (tiles 58.5), for 2048 rows 62 (65.6).
// * Tiles of 128 x 128 with eight waves, two workgroups a CU, or of 256 x 256, one a CU: by a model of their rounds over the
//   chip, fitted on 2048 x 4096 x 4096 (small 42, large 54 us), 2048 x 7168 x 512 (18 and 15) and 8192^3 (646 and 430).
struct TileCost {
  static double small(double tiles, double steps) {  // rounds of 512; half a round or less runs alone on its CUs
    const double full = std::floor(tiles / 512), rest = tiles - 512 * full;
    return full * (1.2 * steps + 4) + (rest > 256 ? 1.2 * steps + 4 : rest > 0 ? 0.6 * steps + 4 : 0);
  }
  static double large(double tiles, double steps) { return std::ceil(tiles / 256) * (1.55 * steps + 8); }
  static double walked(double tiles, double steps) {  // ... with a short last round in quarters (tile_kernel)
    const double rest = tiles - 256 * std::floor(tiles / 256);
    return large(tiles, steps) - (rest > 0 && rest <= 64 ? 0.95 * steps + 4 : rest > 0 && rest <= 128 ? 0.35 * steps : 0);
  }
};
// Tiles that a launch really has: with experts about half a row of tiles each is cut off.
inline double tiles_of(const Args& p, int bm, int bn) {
  const double rows = p.offsets ? p.m / (double)bm + 0.5 * std::min(p.groups, p.m) : std::ceil(p.m / (double)bm);
  return rows * std::ceil(p.n / (double)bn);
}
inline bool large_tiles(const Args& p, int step_k) {
  const double steps = std::ceil(p.k / (double)step_k);
  return TileCost::walked(tiles_of(p, 256, 256), steps) < TileCost::small(tiles_of(p, 128, 128), steps);
}

template <int KIND, bool TA, bool TB, int BM, int BN, int WM, int WN, typename OUT, bool MANY = (BM * BN >= 256 * 256)>
int launch_tile(const Args& p, hipStream_t st) {
  int64_t grid = grid_for(p, TA, BM, BN);
  if (int rc = launched("GEMM", grid, MANY ? 1 : WM * WN * 64)) return rc;
  // One large tile fits a CU: that many workgroups walk the tiles (8192^3 e4m3 440 us, launched one by one 455).
  if (MANY) grid = kCUs;
  tile_kernel<KIND, TA, TB, TA, BM, BN, WM, WN, MANY, OUT><<<(unsigned)grid, WM * WN * 64, 0, st>>>(p);
  GMD_HIP(hipGetLastError());
  return GMD_OK;
}
template <int KIND, bool TA, bool TB, int MB, int NB, int W, int U, typename OUT, bool WIDE = KIND != kBf16 && sizeof(OUT) == 4>
int launch_few(const Args& p, hipStream_t st) {
  const int64_t grid = grid_for(p, TA, MB * 16, NB * 16);
  if (int rc = launched("GEMM", grid, W * 64)) return rc;
  few_rows_kernel<KIND, TA, TB, MB, NB, W, U, WIDE, OUT><<<(unsigned)grid, W * 64, 0, st>>>(p);
  GMD_HIP(hipGetLastError());
  return GMD_OK;
}
// Both operands by rows are one product, bf16 operands always one for each expert.
template <int KIND, typename OUT>
int launch_forward(const Args& p, hipStream_t st) {
  constexpr bool kSingle = KIND != kBf16, kExperts = KIND != kFp8Rows;
  // Up to 32 rows the operands' way in from memory is what bounds a product, and f32 sums cost nothing to 3 %: 64 experts of 4096 x 7168
  // for 69 rows 183.0 us (on the fp8 instruction 182.7), for 1497 rows 349 (347), 1 x 4096 x 7168 7.44 (7.27), 32 x 4096 x 7168
  // 9.46 (9.17); with B in the caches up to 19 % (1 x 4096 x 7168 5.4 and 4.5).  With more rows they cost 6 to 20 % of what the
  // few-row kernel takes (128 x 7168 x 2048 9.8 and 8.9, 256 x 7168 x 2048 14.4 and 11.6) and as much again of the tiles
  // (8192^3 986 and 437), so bf16 results there take the instruction.
  constexpr bool kWide = KIND != kBf16;
  const int rows = p.offsets ? (int)(((int64_t)p.m + p.groups - 1) / p.groups) : p.m;
  const int mb = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  const int nb = grid_of(p, 16 * mb, 16) <= kCUs ? 1 : grid_of(p, 16 * mb, 32) <= kCUs ? 2 : grid_of(p, 16 * mb, 64) <= kCUs ? 4 : 0;
  if (mb == 1) {
    if (nb == 1) return launch_few<KIND, false, false, 1, 1, 8, 2, OUT, kWide>(p, st);
    // (e4m3 experts: a slot less in flight leaves room for twice the workgroups, 128 experts of 2048 x 1024 for 128 rows 42 -> 34 us)
    if constexpr (kExperts)
      if (!kSingle || p.offsets) return launch_few<KIND, false, false, 1, 2, 4, KIND == kBf16 ? 2 : 1, OUT, kWide>(p, st);
    if constexpr (kSingle) return nb == 2 ? launch_few<KIND, false, false, 1, 2, 4, 2, OUT, kWide>(p, st) : launch_few<KIND, false, false, 1, 4, 4, 2, OUT, kWide>(p, st);
  }
  if (mb == 2) {
    if (nb == 1) return launch_few<KIND, false, false, 2, 1, 8, 2, OUT, kWide>(p, st);
    if constexpr (kExperts)
      if (!kSingle || p.offsets) return launch_few<KIND, false, false, 2, 4, 4, 1, OUT, kWide>(p, st);
    if constexpr (kSingle) return nb == 2 ? launch_few<KIND, false, false, 2, 2, 4, 2, OUT, kWide>(p, st) : launch_few<KIND, false, false, 2, 4, 4, 2, OUT, kWide>(p, st);
  }
  // (as many workgroups as 64 x 16, which reads a quarter more: 64 x 4096 x 7168 9.0 us, 10.4; 128 x 2048 x 8192 9.6 and 10.7)
  if (nb == 1) return launch_few<KIND, false, false, 2, 2, 8, 1, OUT>(p, st);
  if (nb == 2) return launch_few<KIND, false, false, 4, 2, 8, 1, OUT>(p, st);
  if (nb == 4) return launch_few<KIND, false, false, 4, 4, 4, 2, OUT>(p, st);
  // (a few more than one workgroup a CU: half as large they are two on every CU, and not two on some, 203 x 4120 x 4096 12.3 against
  // 15.0 us; with four of the half ones a CU the large ones read less, 256 x 7168 x 2048 11.9 against 14.0)
  if constexpr (kSingle)
    if (!p.offsets && grid_of(p, 32, 64) <= 2 * kCUs) return launch_few<KIND, false, false, 2, 4, 4, 1, OUT>(p, st);
  // (one slot each leaves room for two workgroups a CU)
  if (grid_of(p, 64, 64) <= 2 * kCUs) return launch_few<KIND, false, false, 4, 4, 4, 1, OUT>(p, st);
  // (f32 results of e4m3 operands are computed on widened fragments, which do not fit the large tile's registers)
  if constexpr (KIND == kBf16 || sizeof(OUT) == 2)
    if (large_tiles(p, KIND == kBf16 ? 64 : 128)) return launch_tile<KIND, false, false, 256, 256, 2, 4, OUT>(p, st);
  // (widening costs a wave per fragment, not per product: four waves of 64 x 64 have fewer of them per product than eight of 32 x 64,
  // 2048 x 7168 x 8192 276 against 326 us.  With one workgroup or none on most CUs four waves are too few to hide their latencies, and
  // either eight are better, 3584 x 1024 x 7168 by rows 75 against 96 us, or, where it has B's scales as scalars, the few-row kernel,
  // by tiles 65 against 89; 5590 x 808 x 7248 94 and 125; 4096 x 1792 x 2048 43 and 41)
  if constexpr (KIND != kBf16 && sizeof(OUT) == 4) {
    if (grid_of(p, 128, 128) > (KIND == kFp8Tiles ? kCUs * 3 / 2 : kCUs)) return launch_tile<KIND, false, false, 128, 128, 2, 2, OUT>(p, st);
    if constexpr (KIND == kFp8Tiles) return launch_few<KIND, false, false, 4, 4, 4, 1, OUT>(p, st);
    else return launch_tile<KIND, false, false, 128, 128, 4, 2, OUT>(p, st);
  } else {
    return launch_tile<KIND, false, false, 128, 128, 4, 2, OUT>(p, st);
  }
}

// Block-scaled fp8, one product or one per expert (block_gemm.hip).
int launch_fp8(const Args& p, int b_blocks, int out_dtype, hipStream_t st);
// Shared refusals: null when the pointer, the row stride and the extent fit the kernels, else what is wrong.
// ld and row in elements of `elem` bytes; the lane offsets inside a 256-row tile are 32 bits, hence the limit on the stride.
inline const char* bad_operand(const void* p, int64_t ld, int64_t row, int elem) {
  if (!p) return "a null pointer";
  if ((uintptr_t)p & 15) return "a pointer that is not 16-byte aligned";
  if (ld < row) return "a row stride shorter than a row";
  if (ld > (8 << 20) / elem) return "a row stride over 8 MiB";
  if (ld * elem & 15) return "a row stride that is not a multiple of 16 bytes";
  return nullptr;
}

}  // namespace tiles
}  // namespace gmd
