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
// Staging: buffer loads straight into LDS, 16 bytes per lane, two to four stages; an element outside the operand is zero (its
// offset lies outside the buffer descriptor).  The LDS side of such a load is linear in the lane, so the layout that keeps
// the fragment reads free of bank conflicts is made by permuting which 16-byte piece of a row a lane fetches:
//   K-major : piece c of row r lies at c ^ swz(r), so that the rows a 16-byte read serves at once -- 16 consecutive ones, or four
//             groups of four at 0, 12, 20, 24 (measured: the counter of bank conflicts) -- fall into distinct banks;
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

// one number of a tensor of type CRADLE_F32 / BF16 / F16
__device__ __forceinline__ float load_as(const void* p, int64_t i, int dtype) {
  if (dtype == CRADLE_F32) return static_cast<const float*>(p)[i];
  const u16 b = static_cast<const u16*>(p)[i];
  return dtype == CRADLE_BF16 ? from_bf16(b) : from_f16(b);
}
__device__ __forceinline__ void store_as(void* p, int64_t i, int dtype, float v) {
  if (dtype == CRADLE_F32) static_cast<float*>(p)[i] = v;
  else static_cast<u16*>(p)[i] = dtype == CRADLE_BF16 ? bits_bf16(v) : bits_f16(v);
}
__device__ __forceinline__ void store4(void* p, int64_t i, int dtype, f32x4 v, int n, bool vec) {
  if (vec && n >= 4) {
    if (dtype == CRADLE_F32) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
    } else {
      u16 s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = dtype == CRADLE_BF16 ? bits_bf16(v[e]) : bits_f16(v[e]);
      *reinterpret_cast<u32x2*>(static_cast<u16*>(p) + i) = u32x2{s[0] | (uint32_t)s[1] << 16, s[2] | (uint32_t)s[3] << 16};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) store_as(p, i + e, dtype, v[e]);
}

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
  int k_tiles_per_split; // K tiles of a share
  int split;             // this workgroup's share (set in the kernel)
  int symmetric;         // 1: only the tiles on and below the diagonal are computed (square tiles, tiles_m == tiles_n)
};

// Tile (BM x BN) of WAVES_M x WAVES_N waves, K step BK, STAGES buffers in LDS; operands of NPA and NPB planes of ELEM numbers.
template <int ELEM_, int NPA_, int NPB_, int BM_, int BN_, int BK_, int STAGES_, int WAVES_M_, int WAVES_N_, bool AK_, bool BKM_>
struct Tile {
  static constexpr int STAGES = STAGES_;
  static constexpr int ELEM = ELEM_, NPA = NPA_, NPB = NPB_, BM = BM_, BN = BN_, BK = BK_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
  static constexpr bool A_KMAJOR = AK_, B_KMAJOR = BKM_;
  static constexpr int NW = WAVES_M * WAVES_N, NT = 64 * NW;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, TM = WM / 32, TN = WN / 32;
  static constexpr int CA = BM * BK / 8, CB = BN * BK / 8;  // 16-byte pieces per plane
  static constexpr int STAGE = NPA * CA + NPB * CB;
  static constexpr int LDS_BYTES = STAGES * STAGE * 16;
  static constexpr int LOADS = (NPA * CA + NPB * CB) / NT;    // per thread and stage
  static constexpr int ROW = WN + 4;                          // floats of an epilogue row in LDS (the padding spreads the banks)
  static constexpr int ROWS_BYTES = 32 * ROW * 4, ROWS_PER_STAGE = STAGE * 16 / ROWS_BYTES;
  static constexpr bool TURNS = NW == 8 && STAGES == 2;                // two waves per SIMD, taking turns (product_kernel)
  static constexpr int TURN_K = NPA == 1 && NPB == 1 ? 2 : 1;          // MFMA steps of a turn
  static_assert(BK == 32 || BK == 64, "K step");
  static_assert(STAGES >= 2 && STAGES <= 4 && (STAGES - 1) * LOADS < 64, "loads in flight");
  static_assert(LDS_BYTES <= 160 * 1024, "LDS");
  static_assert(ROWS_PER_STAGE * STAGES >= NW, "the waves' epilogue rows fit into the stages");
  static_assert(CA % NT == 0 && CB % NT == 0, "tile too small for the workgroup");
};

template <int BK>
__device__ __forceinline__ int swz(int row) {
  return BK == 64 ? (row ^ (row >> 3)) & 7 : ((row >> 2) ^ (row & 16 ? 3 : 0)) & 3;
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
__device__ __forceinline__ void tile_of(const Args& a, int wg, int nwg, int& tm, int& tn) {
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

// orders the LDS accesses of one wave's lanes (they execute in order; the compiler must keep them so)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The W columns from c0 on of 32 epilogue rows in pieces of four, consecutive lanes consecutive pieces: fn(row, column, piece)
template <class T, int W, class Fn>
__device__ __forceinline__ void each_piece(float* buf, int lane, const Fn& fn) {
  constexpr int P = W / 4;
#pragma unroll
  for (int it = 0; it < 32 * P / 64; ++it) {
    const int idx = it * 64 + lane, r = idx / P, c = idx % P * 4;
    fn(r, c, reinterpret_cast<f32x4*>(buf + r * T::ROW + c));
  }
}

// The same with what memory holds for each piece: all of load(row, column) first, so that the loads are in flight together (a
// store between them would make each wait for the one before), then fn(row, column, piece, loaded).
template <class T, int W, class Load, class Fn>
__device__ __forceinline__ void each_piece(float* buf, int lane, const Load& load, const Fn& fn) {
  constexpr int P = W / 4, IT = 32 * P / 64;
  decltype(load(0, 0)) v[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) v[it] = load((it * 64 + lane) / P, (it * 64 + lane) % P * 4);
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int r = (it * 64 + lane) / P, c = (it * 64 + lane) % P * 4;
    fn(r, c, reinterpret_cast<f32x4*>(buf + r * T::ROW + c), v[it]);
  }
}

// The same, turned: four rows of one column, consecutive lanes consecutive rows: fn(first row, column, numbers)
template <class T, int W, class Fn>
__device__ __forceinline__ void each_turned_piece(const float* buf, int lane, const Fn& fn) {
#pragma unroll
  for (int it = 0; it < W / 8; ++it) {
    const int r = lane % 8 * 4, c = it * 8 + lane / 8;
    fn(r, c, f32x4{buf[r * T::ROW + c], buf[(r + 1) * T::ROW + c], buf[(r + 2) * T::ROW + c], buf[(r + 3) * T::ROW + c]});
  }
}

// C tile = A B^T over this workgroup's K share.  Loads run STAGES K tiles ahead of the products and fragments one MFMA step (16
// of K) ahead: before its last MFMA step a K tile waits for the next stage's loads (s_waitcnt vmcnt of the later stages' count), then
// for the other waves -- whose fragments of this stage are in registers by then --, refills this stage and fetches the next
// one's first fragments, all of it under the products still to come.  The stages are separate arrays and the loop is unrolled
// over them, so that the compiler can tell the buffer being filled from the one being read and adds no wait of its own.
// The second operand's rows are the MFMA's first operand: four accumulator elements of a lane are four consecutive columns of
// one row.  The epilogue gets the tile 32 rows of a wave at a time, turned through LDS so that consecutive lanes hold
// consecutive pieces of a row: its loads and stores then cover whole cache lines.
// Epi: begin(n0, lane) once -> state (a lane's column does not change), emit(a, buf, m0, n0, lane, state, tm, tn) for every 32 rows,
// finish(...) once; Epi::PAIR: columns [0, WN / 2) of buf are the
// first half's, [WN / 2, WN) the second's.
// wg of nwg: this workgroup among those of its share; st0.. : the stages (of at least T::STAGE pieces, as many as T has).
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass only needs the launch stubs; with the body it leaves some of them out)
template <class T, class Epi>
__device__ __forceinline__ void product_body(const Args& a, const Epi& epi, int wg, int nwg, u32x4* st0, u32x4* st1, u32x4* st2, u32x4* st3) {
  static_assert(!Epi::PAIR || T::TN % 2 == 0, "a wave holds both halves of a column");
  using SA = Stager<T, T::A_KMAJOR, T::BM, T::NPA>;
  using SB = Stager<T, T::B_KMAJOR, T::BN, T::NPB>;
  constexpr int S = T::STAGES;
  int tm, tn;
  tile_of(a, wg, nwg, tm, tn);
  const int row0 = tm * T::BM, col0 = tn * (Epi::PAIR ? T::BN / 2 : T::BN);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / T::WAVES_N, wn = wave % T::WAVES_N;
  SA sa;
  SB sb;
  sa.init(a.A, row0, a.M, a.K, PlainMap{});
  if constexpr (Epi::PAIR) sb.init(a.B, col0, a.N, a.K, PairMap<T::WN>{a.up_row});
  else sb.init(a.B, col0, a.N, a.K, PlainMap{});

  const int k_tiles = (a.K + T::BK - 1) / T::BK;
  const int kt0 = a.split * a.k_tiles_per_split, kt1 = min(k_tiles, kt0 + a.k_tiles_per_split);

  // Where the registers allow, the products of lower planes are summed apart: in one accumulator each of them would be rounded
  // at the size of the whole sum (six roundings per 16 of K instead of one).
  constexpr bool APART = (T::NPA > 1 || T::NPB > 1) && T::TM * T::TN <= 4;
  f32x16 acc[T::TM][T::TN], low[APART ? T::TM : 1][APART ? T::TN : 1];
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[i][j][e] = 0.f;
        if constexpr (APART) low[i][j][e] = 0.f;
      }

  // (beyond the share's last tile every piece lies outside: the count of loads in flight stays the same)
  auto issue = [&](u32x4* st, int kt) {
    const int k0 = kt < kt1 ? kt * T::BK : 0x40000000;
    sa.issue(a.A, st, k0);
    sb.issue(a.B, st + T::NPA * T::CA, k0);
  };
  auto barrier = [&]() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  u32x4 fa[2][T::NPA][T::TM], fb[2][T::NPB][T::TN];
  auto fetch = [&](const u32x4* st, int kk, int f) {
    const u32x4* ca = st;
    const u32x4* cb = st + T::NPA * T::CA;
#pragma unroll
    for (int p = 0; p < T::NPA; ++p)
#pragma unroll
      for (int i = 0; i < T::TM; ++i) fa[f][p][i] = SA::frag(ca + p * T::CA, wm * T::WM + i * 32, kk, lane);
#pragma unroll
    for (int p = 0; p < T::NPB; ++p)
#pragma unroll
      for (int j = 0; j < T::TN; ++j) fb[f][p][j] = SB::frag(cb + p * T::CB, wn * T::WN + j * 32, kk, lane);
  };
  // planes pa + pb < max(NPA, NPB), the smallest products first
  auto multiply = [&](int f) {
#pragma unroll
    for (int s = (T::NPA > T::NPB ? T::NPA : T::NPB) - 1; s >= 0; --s)
#pragma unroll
      for (int pa = T::NPA - 1; pa >= 0; --pa) {
        const int pb = s - pa;
        if (pb < 0 || pb >= T::NPB) continue;
#pragma unroll
        for (int i = 0; i < T::TM; ++i)
#pragma unroll
          for (int j = 0; j < T::TN; ++j) {
            f32x16& c = APART && s > 0 ? low[APART ? i : 0][APART ? j : 0] : acc[i][j];
            c = mfma<T::ELEM>(fb[f][pb][j], fa[f][pa][i], c);
          }
      }
  };
  if constexpr (T::TURNS) {
    // Two waves per SIMD take turns (8192 x 10240 x 4096 in bf16: 532 -> 516 us, 4096^3 in three planes 573 -> 558): while one multiplies, the other fetches its next fragments.  Waves 4..7 run one turn (a
    // barrier) behind waves 0..3.  Turn pair t of a K tile: fetch KT MFMA steps of fragments | barrier | multiply them | barrier.
    // The stage read last is refilled in the first turn of the next tile (both halves have left it by then); a wave's own loads
    // of the next stage have landed before the barrier behind its last fetch of this one, one turn before anybody reads it.
    constexpr int KT = T::TURN_K, NT = T::BK / 16 / KT;
    const bool second = wave >= T::NW / 2;
    issue(st0, kt0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    barrier();
    if (second) barrier();
    auto step = [&](const u32x4* cur, u32x4* nxt, int kt) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (t == 0) issue(nxt, kt + 1);
#pragma unroll
        for (int k = 0; k < KT; ++k) fetch(cur, t * KT + k, k);
        if (t == NT - 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        barrier();
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int k = 0; k < KT; ++k) multiply(k);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        barrier();
      }
    };
    for (int kt = kt0; kt < kt1; kt += 2) {
      step(st0, st1, kt);
      if (kt + 1 < kt1) step(st1, st0, kt + 1);
    }
    if (!second) barrier();
  } else {
    auto step = [&](u32x4* cur, const u32x4* nxt, int kt) {
#pragma unroll
      for (int kk = 0; kk < T::BK / 16; ++kk) {
        if (kk + 1 < T::BK / 16) {
          fetch(cur, kk + 1, (kk + 1) & 1);
        } else {
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 2) * T::LOADS) : "memory");
          barrier();
          issue(cur, kt + S);
          fetch(nxt, 0, 0);
        }
        multiply(kk & 1);
      }
    };

    issue(st0, kt0);
    issue(st1, kt0 + 1);
    if constexpr (S > 2) issue(st2, kt0 + 2);
    if constexpr (S > 3) issue(st3, kt0 + 3);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * T::LOADS) : "memory");
    barrier();
    fetch(st0, 0, 0);
    for (int kt = kt0; kt < kt1; kt += S) {
      step(st0, st1, kt);
      if constexpr (S == 2) {
        if (kt + 1 < kt1) step(st1, st0, kt + 1);
      } else {
        if (kt + 1 < kt1) step(st1, st2, kt + 1);
        if constexpr (S == 3) {
          if (kt + 2 < kt1) step(st2, st0, kt + 2);
        } else {
          if (kt + 2 < kt1) step(st2, st3, kt + 2);
          if (kt + 3 < kt1) step(st3, st0, kt + 3);
        }
      }
    }
  }
  if constexpr (APART) {
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int j = 0; j < T::TN; ++j) acc[i][j] += low[i][j];
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  barrier();

  // this wave's 32 epilogue rows lie in one of the stages, which nobody reads any more
  const int slot = wave / T::ROWS_PER_STAGE, in = wave % T::ROWS_PER_STAGE;
  u32x4* st = slot == 0 ? st0 : st1;
  if constexpr (S > 2) st = slot == 2 ? st2 : st;
  if constexpr (S > 3) st = slot == 3 ? st3 : st;
  float* buf = reinterpret_cast<float*>(st) + in * 32 * T::ROW;
  const int li = lane & 31, lh = lane >> 5;
  const int m0 = row0 + wm * T::WM, n0 = col0 + wn * (Epi::PAIR ? T::WN / 2 : T::WN);
  typename Epi::State state = epi.template begin<T>(n0, lane);
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(buf + li * T::ROW + j * 32 + q * 8 + lh * 4) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    wave_sync();
    epi.template emit<T>(a, buf, m0 + i * 32, n0, lane, state, tm, tn);
    wave_sync();
  }
  epi.template finish<T>(a, n0, lane, state, tm, wm);
}
#endif

// one product: blockIdx.x the tile, y the matrix of a batch, z the share of K
template <class T, class Epi>
__global__ __launch_bounds__(T::NT, 1) void product_kernel(const Args args, const Epi epi) {
#ifdef __HIP_DEVICE_COMPILE__
  __shared__ u32x4 st0[T::STAGE];
  __shared__ u32x4 st1[T::STAGE];
  __shared__ u32x4 st2[T::STAGES > 2 ? T::STAGE : 1];
  __shared__ u32x4 st3[T::STAGES > 3 ? T::STAGE : 1];
  Args a = args;
  a.split = blockIdx.z;
  product_body<T, Epi>(a, epi, blockIdx.x, gridDim.x, st0, st1, st2, st3);
#endif
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
