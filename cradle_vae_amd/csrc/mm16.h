// Tile products on the 16-bit matrix cores (v_mfma_f32_32x32x16_{bf16,f16}, fp32 accumulation), shared by the gated
// feed-forward block (gated_mlp.hip) and the orthogonalised update (orthogonalize.hip).
//
// An operand is one to three planes of 16-bit numbers whose sum is the operand:
//   1  the 16-bit number itself (bf16 / fp16 tensors): one product per element pair;
//   2  hi + lo: in fp16 22 significant bits, for operands whose range is known (hi hi + hi lo + lo hi), or an intermediate
//      result of 16-bit tensors held in twice their bits (times a one-plane operand: two products);
//   3  p0 + p1 + p2 in bf16 (24 significant bits, any range): the six products of order <= 2.
// The dropped products of 2 x 2 and 3 x 3 planes are below 2^-22 of |a||b|, near fp32's own rounding of a product, so they give
// fp32 results at 3 or 6 products of a rate 16 times that of v_mfma_f32_32x32x2_f32: the split is what makes fp32 fast here.
//
// Orientation per operand: K-major ([row][k], k contiguous) or MN-major ([k][row], rows contiguous); the second is
// transposed on its way from LDS to registers by ds_read_tr16_b64, so no transposed copy is ever made in memory.
//
// Staging: buffer loads straight into LDS, 16 bytes per lane, double-buffered; an element outside the operand is zero (its
// offset lies outside the buffer descriptor).  The LDS side of such a load is linear in the lane, so the layout that keeps
// the fragment reads free of bank conflicts is made by permuting which 16-byte piece of a row a lane fetches:
//   K-major : piece c of row r lies at c ^ swz(r), so that 8 (and 16) consecutive rows' pieces c fall into distinct banks;
//   MN-major: piece c of k-row k at c ^ 2 f(k & 3), f = {0,2,5,7} ({0,1,2,3} for 64 rows), so that the 4 x 32 bytes a 16-lane group transposes (and
//             the two groups of a half wave) fall into distinct banks.
//
// Operands are handed over with: 16-byte aligned base, leading dimension % 8 == 0, and contiguous extents that are readable
// up to the next multiple of 8 elements -- zero there if the contiguous axis is the inner one (checked / packed by callers).
#pragma once
#include "common.h"

namespace cradle {
namespace mm16 {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16;

enum Elem { BF16 = 0, F16 = 1 };

__device__ __forceinline__ u16 bits_bf16(float v) { return __builtin_bit_cast(u16, (__bf16)v); }
__device__ __forceinline__ u16 bits_f16(float v) { return __builtin_bit_cast(u16, (_Float16)v); }
__device__ __forceinline__ float from_bf16(u16 b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
__device__ __forceinline__ float from_f16(u16 b) { return (float)__builtin_bit_cast(_Float16, b); }

// v as NPL planes of ELEM numbers (round to nearest each).  A value that is not finite, or rounds to an infinity in the first
// plane, keeps zeros in the others: the product is then an infinity or NaN in the rows and columns it belongs to.
template <int ELEM, int NPL>
__device__ __forceinline__ void split(float v, u16 (&p)[NPL]) {
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    p[i] = ELEM == BF16 ? bits_bf16(v) : bits_f16(v);
    const float r = ELEM == BF16 ? from_bf16(p[i]) : from_f16(p[i]);
    v = fabsf(r) <= 3.4028235e38f ? v - r : 0.f;
  }
}

struct Operand {
  const u16* p;
  int64_t ld;     // elements between rows (K-major) or between k-rows (MN-major)
  int64_t plane;  // elements between planes
  int64_t batch;  // elements between the matrices of a batch (blockIdx.y)
};

struct Args {
  Operand A, B;
  int M, N, K;           // N: columns of the output (for a paired product: of each half)
  int tiles_m, tiles_n;
  int up_row;            // paired product: rows of B from here on are the second half
  int k_tiles_per_split; // blockIdx.z-th share of the K tiles
  int symmetric;         // 1: only the tiles on and below the diagonal are computed (square tiles, tiles_m == tiles_n)
};

// Tile (BM x BN) of WAVES_M x WAVES_N waves, K step BK; operands of NPA and NPB planes of ELEM numbers.
template <int ELEM_, int NPA_, int NPB_, int BM_, int BN_, int BK_, int WAVES_M_, int WAVES_N_, bool AK_, bool BKM_>
struct Tile {
  static constexpr int ELEM = ELEM_, NPA = NPA_, NPB = NPB_, BM = BM_, BN = BN_, BK = BK_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
  static constexpr bool A_KMAJOR = AK_, B_KMAJOR = BKM_;
  static constexpr int NW = WAVES_M * WAVES_N, NT = 64 * NW;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 32, TN = WN / 32;
  static constexpr int CA = BM * BK / 8, CB = BN * BK / 8;  // 16-byte pieces per plane
  static constexpr int STAGE = NPA * CA + NPB * CB;
  static constexpr int LDS_BYTES = 2 * STAGE * 16;
  static_assert(BK == 32 || BK == 64, "K step");
  static_assert(CA % NT == 0 && CB % NT == 0, "tile too small for the workgroup");
};

template <int BK>
__device__ __forceinline__ int swz(int row) {
  return BK == 64 ? (row ^ (row >> 3)) & 7 : ((row >> 1) ^ (row >> 3)) & 3;
}
template <int ROWS>
__device__ __forceinline__ int swz_k(int k) {
  static_assert(ROWS == 64 || ROWS % 128 == 0, "");  // (64: eight pieces per k-row, so the permutation has to stay below eight)
  return ROWS == 64 ? 2 * (k & 3) : 2 * (2 * (k & 3) + ((k >> 1) & 1));
}

template <int ELEM>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (ELEM == BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// One operand's share of a stage: ROWS tile rows (of M or N) x BK, all planes.
template <class T, bool KMAJOR, int ROWS, int NPL>
struct Stager {
  static constexpr int CH = ROWS * T::BK / 8, NI = CH / T::NT, BK = T::BK;
  static constexpr int CPR = KMAJOR ? BK / 8 : ROWS / 8;  // pieces per LDS row
  static constexpr uint32_t OUT = 0x80000000u;            // beyond every descriptor
  uint32_t off[NI];  // byte offset of this lane's piece at K tile 0 (OUT: its row lies outside)
  int lim[NI];       // the piece is inside while k0 < lim (K-major) / k-row k0 + row < K (MN-major: lim = K - row)
  uint32_t bytes;
  const u16* base;

  // row0: first tile row; rows: rows of the operand; map: tile row -> operand row or -1 (paired products)
  template <class Map>
  __device__ __forceinline__ void init(const Operand& o, int row0, int rows, int K, const Map& map) {
    base = o.p + (int64_t)blockIdx.y * o.batch;
    if constexpr (KMAJOR) {
      // offsets from the tile's lowest row; 32 bits hold them: the host limits the rows a tile can span
      const int first = map.first(row0);
      base += (int64_t)first * o.ld;
      const int64_t left = ((int64_t)(map.total(rows) - 1 - first) * o.ld + ((K + 7) & ~7)) * 2;
      bytes = left < 0x7fffff00 ? (uint32_t)left : 0x7fffff00u;
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        const int l = it * T::NT + threadIdx.x, r = l / CPR, c = (l % CPR) ^ swz<BK>(r);
        const int g = map(row0, r, rows);
        off[it] = g < 0 ? OUT : (uint32_t)((int64_t)(g - first) * o.ld * 2 + c * 16);
        lim[it] = g < 0 ? -1 : K - c * 8;
      }
    } else {
      base += row0;
      // (bytes depends on the K tile: see rsrc)
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        const int l = it * T::NT + threadIdx.x, r = l / CPR, c = (l % CPR) ^ swz_k<ROWS>(r);
        off[it] = (uint32_t)((int64_t)r * o.ld * 2 + c * 16);
        lim[it] = row0 + c * 8 < rows ? K - r : -1;
      }
      bytes = (uint32_t)(((int64_t)(BK - 1) * o.ld + ROWS) * 2);
    }
  }

  // issues the loads of K tile k0 (a multiple of BK) into dst (this stage's pieces, plane after plane)
  __device__ __forceinline__ void issue(const Operand& o, u32x4* dst, int k0) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int p = 0; p < NPL; ++p) {
      const u16* b = base + p * o.plane + (KMAJOR ? 0 : (int64_t)k0 * o.ld);
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<u16*>(b), 0, bytes, 0x00020000);
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        const uint32_t a = KMAJOR ? off[it] + (uint32_t)k0 * 2 : off[it];
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(dst + p * CH + it * T::NT + wave * 64), 16,
                                                 k0 < lim[it] ? a : OUT, 0, 0, 0);
      }
    }
  }

  // 32 tile rows from `row`, 16 k from kk*16, as an MFMA operand: lane (li, lh) holds row + li, k = 8 lh .. 8 lh + 7
  __device__ __forceinline__ static u32x4 frag(const u32x4* src, int row, int kk, int lane) {
    const int li = lane & 31, lh = lane >> 5;
    if constexpr (KMAJOR) {
      const int r = row + li;
      return src[r * CPR + ((kk * 2 + lh) ^ swz<BK>(r))];
    } else {
      // a 16-lane group transposes 4 k-rows x 16 columns: its lane i reads columns 4 (i & 3).. of k-row i >> 2
      const int i = lane & 15, kq = i >> 2, col = row + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
      const int k = kk * 16 + lh * 8 + kq;
      const char* s = reinterpret_cast<const char*>(src) + (k * CPR + ((col >> 3) ^ swz_k<ROWS>(kq))) * 16 + (col & 4) * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)s);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(s + 4 * CPR * 16));
      const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
      return u32x4{a.x, a.y, b.x, b.y};
    }
  }
};

// tile rows are operand rows
struct PlainMap {
  __device__ __forceinline__ int first(int row0) const { return row0; }
  __device__ __forceinline__ int total(int rows) const { return rows; }
  __device__ __forceinline__ int operator()(int row0, int r, int rows) const { return row0 + r < rows ? row0 + r : -1; }
};
// paired product: of each wave's WN tile rows the first half are columns f of the first matrix, the second half the same
// columns of the second (operand rows f and up + f), so that a lane's accumulators hold both numbers of a column
template <int WN>
struct PairMap {
  int up;
  __device__ __forceinline__ int first(int row0) const { return row0; }
  __device__ __forceinline__ int total(int rows) const { return up + rows; }
  __device__ __forceinline__ int operator()(int row0, int r, int rows) const {
    const int f = row0 + (r / WN) * (WN / 2) + r % (WN / 2);
    return f < rows ? f + (r % WN >= WN / 2 ? up : 0) : -1;
  }
};

// Order of the tiles: workgroups go round-robin over the eight XCDs, so the tiles of one XCD (its own L2) are a contiguous
// run of a raster of 8 tile rows at a time.
__device__ __forceinline__ void tile_of(const Args& a, int& tm, int& tn) {
  const int nwg = gridDim.x;
  int wg = blockIdx.x;
  const int q = nwg / 8, r = nwg % 8, xcd = wg % 8, pos = wg / 8;
  wg = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + pos;
  if (a.symmetric) {  // tile rows' lengths are 1, 2, 3 ...
    int t = (int)((sqrtf(8.0f * wg + 1.0f) - 1.0f) * 0.5f);
    while ((t + 1) * (t + 2) / 2 <= wg) ++t;
    while (t * (t + 1) / 2 > wg) --t;
    tm = t;
    tn = wg - t * (t + 1) / 2;
    return;
  }
  constexpr int G = 8;
  const int per = G * a.tiles_n, g = wg / per, in = wg % per, rows = min(G, a.tiles_m - g * G);
  tm = g * G + in % rows;
  tn = in / rows;
}

// C tile = A B^T over this workgroup's K share, handed to the epilogue in registers: the second operand's rows are the MFMA's
// first operand, so that four accumulator elements of a lane are four consecutive columns of one row (each_piece).
// Epi::PAIR: a column's two halves are accumulators j and j + TN / 2 of the same lane.
template <class T, class Epi>
__global__ __launch_bounds__(T::NT, 1) void product_kernel(const Args a, const Epi epi) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass only needs the launch stub; with the body it leaves some of them out)
  static_assert(!Epi::PAIR || T::TN % 2 == 0, "a wave holds both halves of a column");
  using SA = Stager<T, T::A_KMAJOR, T::BM, T::NPA>;
  using SB = Stager<T, T::B_KMAJOR, T::BN, T::NPB>;
  __shared__ u32x4 st0[T::STAGE];
  __shared__ u32x4 st1[T::STAGE];
  int tm, tn;
  tile_of(a, tm, tn);
  const int row0 = tm * T::BM, col0 = tn * (Epi::PAIR ? T::BN / 2 : T::BN);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WAVES_N, wn = wave % T::WAVES_N;
  SA sa;
  SB sb;
  sa.init(a.A, row0, a.M, a.K, PlainMap{});
  if constexpr (Epi::PAIR) sb.init(a.B, col0, a.N, a.K, PairMap<T::WN>{a.up_row});
  else sb.init(a.B, col0, a.N, a.K, PlainMap{});

  const int k_tiles = (a.K + T::BK - 1) / T::BK;
  const int kt0 = blockIdx.z * a.k_tiles_per_split, kt1 = min(k_tiles, kt0 + a.k_tiles_per_split);

  f32x16 acc[T::TM][T::TN];
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  auto issue = [&](u32x4* st, int kt) {
    sa.issue(a.A, st, kt * T::BK);
    sb.issue(a.B, st + T::NPA * T::CA, kt * T::BK);
  };
  auto wait_all = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  // products of one stage; the next stage's loads are issued once this stage's first fragments are on their way
  auto step = [&](const u32x4* cur, u32x4* nxt, int kt_next) {
    const u32x4* ca = cur;
    const u32x4* cb = cur + T::NPA * T::CA;
    if (kt_next < kt1) issue(nxt, kt_next);
#pragma unroll
    for (int kk = 0; kk < T::BK / 16; ++kk) {
      u32x4 fa[T::NPA][T::TM], fb[T::NPB][T::TN];
#pragma unroll
      for (int p = 0; p < T::NPA; ++p)
#pragma unroll
        for (int i = 0; i < T::TM; ++i) fa[p][i] = SA::frag(ca + p * T::CA, wm * T::WM + i * 32, kk, lane);
#pragma unroll
      for (int p = 0; p < T::NPB; ++p)
#pragma unroll
        for (int j = 0; j < T::TN; ++j) fb[p][j] = SB::frag(cb + p * T::CB, wn * T::WN + j * 32, kk, lane);
      // planes pa + pb < max(NPA, NPB), the smallest products first
#pragma unroll
      for (int s = (T::NPA > T::NPB ? T::NPA : T::NPB) - 1; s >= 0; --s)
#pragma unroll
        for (int pa = T::NPA - 1; pa >= 0; --pa) {
          const int pb = s - pa;
          if (pb < 0 || pb >= T::NPB) continue;
#pragma unroll
          for (int i = 0; i < T::TM; ++i)
#pragma unroll
            for (int j = 0; j < T::TN; ++j) acc[i][j] = mfma<T::ELEM>(fb[pb][j], fa[pa][i], acc[i][j]);
        }
    }
    wait_all();
  };

  if (kt0 < kt1) {
    issue(st0, kt0);
    wait_all();
    for (int kt = kt0; kt < kt1; kt += 2) {
      step(st0, st1, kt + 1);
      if (kt + 1 < kt1) step(st1, st0, kt + 2);
    }
  }

  epi.template store<T>(a, acc, row0 + wm * T::WM, col0 + wn * (Epi::PAIR ? T::WN / 2 : T::WN), lane, tm, tn, wm);
#endif
}

// Walks a wave's accumulators in pieces of four consecutive columns: fn(i, m, j, q, n).  m, n: first row / column of the wave.
template <class T, int TN, class Fn>
__device__ __forceinline__ void each_piece(int m0, int n0, int lane, const Fn& fn) {
  const int li = lane & 31, lh = lane >> 5;
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) fn(i, m0 + i * 32 + li, j, q, n0 + j * 32 + q * 8 + lh * 4);
}
template <int Q>
__device__ __forceinline__ f32x4 quarter(const f32x16& c) {
  return f32x4{c[4 * Q], c[4 * Q + 1], c[4 * Q + 2], c[4 * Q + 3]};
}
__device__ __forceinline__ f32x4 quarter(const f32x16& c, int q) {
  return q == 0 ? quarter<0>(c) : q == 1 ? quarter<1>(c) : q == 2 ? quarter<2>(c) : quarter<3>(c);
}

// four numbers as NPL planes at p (8-byte aligned; the planes lie `plane` elements apart)
template <int ELEM, int NPL>
__device__ __forceinline__ void store_planes(u16* p, int64_t plane, f32x4 v) {
  u16 s[4][NPL];
#pragma unroll
  for (int e = 0; e < 4; ++e) split<ELEM, NPL>(v[e], s[e]);
#pragma unroll
  for (int k = 0; k < NPL; ++k)
    *reinterpret_cast<u32x2*>(p + k * plane) = u32x2{s[0][k] | (uint32_t)s[1][k] << 16, s[2][k] | (uint32_t)s[3][k] << 16};
}

}  // namespace mm16
}  // namespace cradle
