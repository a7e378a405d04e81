// Orthogonalised update: the odd polynomial iteration that sends every singular value of a matrix towards one,
//   X_0 = G / (|G|_F + eps),   S = X X^T,   X <- a X + (b S + c S S) X      (on the smaller side of the matrix)
// as three tile products per step (mm16.h), the polynomial in their epilogues.
//
// Numbers: X, S and B = b S + c S S are kept as two fp16 planes (hi + lo, 22 bits), three products per element pair with fp32
// accumulation.  The iteration is normalised, |X_ij| <= |X|_2 <= max |p(s)|, so fp16's range is no obstacle: everything is held
// times 2^12, which puts the lo plane of an entry of size 2^-6 (a 4096-wide matrix) well above fp16's subnormals and keeps
// |X|, |S| = |X|^2 and |B| below 15.9 (checked for the coefficients by the caller) below its largest number.  fp32 results at three products of a rate
// 16 times the fp32 matrix instruction's.  fp16 tensors take the same path: one plane's error would show in their last bits.
// bf16 tensors multiply with the hi plane alone in the first two steps of five (one_plane; X itself, and a X, keep both): of many
// singular values all are small then, and so is everything (b S + c S S) X adds.  In an emulation over full-rank, orthogonal,
// spiked, decaying and low-rank matrices (tests/test_operator_precision_cpu.py) the error after the final rounding is 1.00 to 1.06
// times that of the rounding alone; with a third step of one plane it is up to 1.9, with few singular values up to 3.9 and
// over 12 steps, all but two of them so, 28.
// S and B are symmetric: only the tiles on and below the diagonal are computed, the epilogue stores them twice.
// The norm is accumulated in fp64 (squares of fp32 gradients leave fp32's range).
// Measured, five steps: 4096 x 8192 in bf16 5.14 and 5.28 ms on two cards (two-plane steps at 1060 TFLOP/s, one-plane steps at 830:
// the epilogue that reads and writes both planes of X is not hidden); 5000 x 400 in fp32 209 us, 2 x 513 x 1001 in fp16 192 us: chains
// of 22 and 17 launches of 4 to 15 us.
#include "mm16.h"

namespace cradle {
namespace {

using namespace mm16;

constexpr float kScale = 4096.f;  // X, S, B are held times this
constexpr int kCUs = 256;

struct Tensor {
  const void* p;
  int64_t ld, batch;
  int dtype, rows, cols;
};

// v -> v kScale / (|G|_F + eps), from the sum of squares.  The norm and its reciprocal can lie beyond fp32, so the divisor's power
// of two goes first (exactly) and what is left of it, near one, second.
struct Scale {
  float two, rest;
  __device__ __forceinline__ Scale(double sumsq, float eps) {
    const double d = sqrt(sumsq) + (double)eps;
    int e = (int)(__double2hiint(d) >> 20 & 0x7ff) - 1023;
    e = e < -126 ? -126 : e > 149 ? 149 : e;
    two = ldexpf(1.f, -e);
    rest = kScale / (float)ldexp(d, -e);
  }
  __device__ __forceinline__ float operator()(float v) const { return v * two * rest; }
};

// partial sums of squares, (batch, gridDim.x) doubles: a wave takes every 4 gridDim.x-th row, 16 bytes per lane where rows allow
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void sumsq_kernel(const Tensor g, double* __restrict__ part) {
  __shared__ double red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int V = !VEC ? 1 : DT == CRADLE_F32 ? 4 : 8, ES = DT == CRADLE_F32 ? 4 : 2;
  // (a row in parts of 4096 elements, so that a few long rows are shared out too)
  const int parts = (g.cols + 4095) / 4096;
  const int64_t items = (int64_t)g.rows * parts;
  double s = 0;
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < items; t += (int64_t)gridDim.x * 4) {
    const int64_t row = (int64_t)blockIdx.y * g.batch + (t / parts) * g.ld;
    const int c0 = (int)(t % parts) * 4096, c1 = min(g.cols, c0 + 4096);
    float f = 0.f;
    double d = 0;
#pragma unroll 4
    for (int c = c0 + lane * V; c < c1; c += 64 * V) {
      if constexpr (VEC) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const char*>(g.p) + (row + c) * ES);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint32_t bits = w[DT == CRADLE_F32 ? e : 0];  // (a copy: bit_cast of a vector's element takes the first one)
          const float v = DT == CRADLE_F32 ? __builtin_bit_cast(float, bits)
                          : DT == CRADLE_BF16 ? from_bf16((u16)(w[e / 2] >> (e % 2 * 16))) : from_f16((u16)(w[e / 2] >> (e % 2 * 16)));
          if constexpr (DT == CRADLE_F16) f = fmaf(v, v, f);  // (64 squares below 2^32 each: no overflow)
          else d += (double)v * v;
        }
      } else {
        const float v = load_as(g.p, row + c, DT);
        if constexpr (DT == CRADLE_F16) f = fmaf(v, v, f);
        else d += (double)v * v;
      }
    }
    s += d + f;
  }
  for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X (times kScale) as two planes of rows x ldx, rows <= columns: G or its transpose.  64 x 64 tiles through LDS.
__global__ __launch_bounds__(256) void pack_kernel(const Tensor g, const double* __restrict__ part, int parts, float eps, int flip,
                                                   u16* __restrict__ x, int64_t plane, int64_t batch, int m, int n, int ldx) {
  __shared__ float tile[64][65];
  __shared__ double red[4];
  const int64_t base = (int64_t)blockIdx.z * g.batch;
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;  // of X
  const int g0 = flip ? n0 : m0, g1 = flip ? m0 : n0;    // of G
  const int c = threadIdx.x % 64;
  float v[16];
  const auto load = [&](int dtype) {
#pragma unroll
    for (int k = 0; k < 16; ++k)  // (unconditional loads from clamped places, all in flight at once, under the norm's sum)
      v[k] = load_as(g.p, base + (int64_t)min(g0 + k * 4 + (int)threadIdx.x / 64, g.rows - 1) * g.ld + min(g1 + c, g.cols - 1), dtype);
  };
  double s = 0;
  for (int t = threadIdx.x; t < parts; t += 256) s += part[(int64_t)blockIdx.z * parts + t];
  if (g.dtype == CRADLE_F32) load(CRADLE_F32);
  else if (g.dtype == CRADLE_BF16) load(CRADLE_BF16);
  else load(CRADLE_F16);
  for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = (red[0] + red[1]) + (red[2] + red[3]);
  const Scale scale(s, eps);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = k * 4 + threadIdx.x / 64;
    tile[r][c] = g0 + r < g.rows && g1 + c < g.cols ? scale(v[k]) : 0.f;
  }
  __syncthreads();
  u16* out = x + (int64_t)blockIdx.z * batch;
  for (int i = threadIdx.x; i < 64 * 16; i += 256) {
    const int r = i / 16, n = i % 16 * 4;
    if (m0 + r >= m || n0 + n >= ldx) continue;
    f32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = flip ? tile[n + e][r] : tile[r][n + e];
    store_planes<F16, 2>(out + (int64_t)(m0 + r) * ldx + n0 + n, plane, w);
  }
}

struct NoState {};
// four consecutive numbers of a two-plane matrix (NPL = 1: of its hi plane)
struct Raw {
  u32x2 h, l;
};
template <int NPL>
__device__ __forceinline__ Raw load_raw(const u16* p, int64_t plane) {
  return Raw{*reinterpret_cast<const u32x2*>(p), NPL == 2 ? *reinterpret_cast<const u32x2*>(p + plane) : u32x2{0, 0}};
}
template <int NPL>
__device__ __forceinline__ f32x4 value_of(const Raw& r) {
  f32x4 v = {from_f16((u16)r.h.x), from_f16((u16)(r.h.x >> 16)), from_f16((u16)r.h.y), from_f16((u16)(r.h.y >> 16))};
  if constexpr (NPL == 2) v += f32x4{from_f16((u16)r.l.x), from_f16((u16)(r.l.x >> 16)), from_f16((u16)r.l.y), from_f16((u16)(r.l.y >> 16))};
  return v;
}

__device__ __forceinline__ f32x4 load_planes(const u16* p, int64_t plane) { return value_of<2>(load_raw<2>(p, plane)); }

// out = alpha acc + beta add, a symmetric matrix of `size` rows, ld = size rounded up to 64 (padding columns zero).  Tiles below the
// diagonal are stored a second time, turned, above it.
template <int NPL>
struct SymEpi {
  [[maybe_unused]] static constexpr bool PAIR = false;
  using State = NoState;
  template <class T>
  __device__ __forceinline__ NoState begin(int, int) const { return {}; }
  float alpha, beta;
  const u16* add;  // or NULL
  u16* out;
  int64_t plane, batch;
  int size, ld;
  // what is added at (m, n) (places beyond the matrix: its last, not used)
  __device__ __forceinline__ Raw addend(int m, int n) const {
    if (!add) return Raw{};
    return load_raw<NPL>(add + (int64_t)blockIdx.y * batch + (int64_t)min(m, size - 1) * ld + min(n, ld - 4), plane);
  }
  __device__ __forceinline__ f32x4 value(int m, int n, f32x4 v, const Raw& r) const {
    v *= alpha;
    if (m < size && n < ld && add) v += beta * value_of<NPL>(r);
    return v;
  }
  __device__ __forceinline__ void put(int row, int col, f32x4 v) const {
    if (row < size && col < ld) store_planes<F16, NPL>(out + (int64_t)blockIdx.y * batch + (int64_t)row * ld + col, plane, v);
  }
  template <class T>
  __device__ __forceinline__ void emit(const Args&, float* buf, int m0, int n0, int lane, NoState&, int tm, int tn) const {
    const auto load = [&](int r, int c) { return addend(m0 + r, n0 + c); };
    each_piece<T, T::WN>(buf, lane, load, [&](int r, int c, f32x4* p, const Raw& old) {
      const f32x4 v = value(m0 + r, n0 + c, *p, old);
      put(m0 + r, n0 + c, v);
      *p = v;
    });
    if (tm == tn) return;
    wave_sync();
    each_turned_piece<T, T::WN>(buf, lane, [&](int r, int c, f32x4 v) { put(n0 + c, m0 + r, v); });
  }
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int, int, NoState&, int, int) const {}
};

// fp32 partial sums of a symmetric product split along K: (split, batch, size, ld)
struct SymPartialEpi {
  [[maybe_unused]] static constexpr bool PAIR = false;
  using State = NoState;
  template <class T>
  __device__ __forceinline__ NoState begin(int, int) const { return {}; }
  float* partial;
  int size, ld;
  template <class T>
  __device__ __forceinline__ void emit(const Args&, float* buf, int m0, int n0, int lane, NoState&, int, int) const {
    float* base = partial + ((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * size * ld;
    each_piece<T, T::WN>(buf, lane, [&](int r, int c, const f32x4* p) {
      const int m = m0 + r, n = n0 + c;
      if (m < size && n < ld) *reinterpret_cast<f32x4*>(base + (int64_t)m * ld + n) = *p;
    });
  }
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int, int, NoState&, int, int) const {}
};
// joins the splits of the tiles on and below the diagonal, one workgroup per 32 x 32 block of the result
template <int NPL>
__global__ __launch_bounds__(256) void sym_join_kernel(const float* __restrict__ partial, int splits, int tile, const SymEpi<NPL> epi) {
  __shared__ float turned[32][33];
  const int r = threadIdx.x / 8, c = threadIdx.x % 8 * 4;
  const int m0 = blockIdx.z * 32, n0 = blockIdx.x * 32, m = m0 + r, n = n0 + c;
  if (n0 / tile > m0 / tile) return;  // (tiles are multiples of 32: the whole workgroup)
  const int64_t per = (int64_t)gridDim.y * epi.size * epi.ld;
  f32x4 v = {0, 0, 0, 0};
  if (m < epi.size && n < epi.ld) {
    const float* p = partial + ((int64_t)blockIdx.y * epi.size + m) * epi.ld + n;
#pragma unroll 4
    for (int z = 0; z < splits; ++z) v += *reinterpret_cast<const f32x4*>(p + z * per);
  }
  v = epi.value(m, n, v, epi.addend(m, n));
  epi.put(m, n, v);
  if (n0 / tile == m0 / tile) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) turned[c + e][r] = v[e];
  __syncthreads();
  epi.put(n0 + r, m0 + c, f32x4{turned[r][c], turned[r][c + 1], turned[r][c + 2], turned[r][c + 3]});
}

// X' = a X + B X as planes, or (last step) the result itself, turned back where G was
struct StepEpi {
  [[maybe_unused]] static constexpr bool PAIR = false;
  using State = NoState;
  template <class T>
  __device__ __forceinline__ NoState begin(int, int) const { return {}; }
  float a, alpha;
  const u16* x;
  u16* out;
  int64_t plane, batch;
  int ld;
  void* result;  // or NULL
  int64_t ld_result, batch_result;
  int dtype, flip, vec;
  template <class T>
  __device__ __forceinline__ void emit(const Args& ar, float* buf, int m0, int n0, int lane, NoState&, int, int) const {
    const int64_t b = (int64_t)blockIdx.y * batch, br = (int64_t)blockIdx.y * batch_result;
    const auto load = [&](int r, int c) { return load_raw<2>(x + b + (int64_t)min(m0 + r, ar.M - 1) * ld + min(n0 + c, ld - 4), plane); };
    each_piece<T, T::WN>(buf, lane, load, [&](int r, int c, f32x4* p, const Raw& old) {
      const int m = m0 + r, n = n0 + c;
      if (m >= ar.M || n >= ld) return;
      const f32x4 v = alpha * *p + a * value_of<2>(old);
      if (!result) store_planes<F16, 2>(out + b + (int64_t)m * ld + n, plane, v);
      else if (flip) *p = v * (1.f / kScale);
      else store4(result, br + (int64_t)m * ld_result + n, dtype, v * (1.f / kScale), ar.N - n, vec);
    });
    if (!result || !flip) return;
    wave_sync();
    each_turned_piece<T, T::WN>(buf, lane, [&](int r, int c, f32x4 v) {
      if (n0 + c < ar.N && m0 + r < ar.M) store4(result, br + (int64_t)(n0 + c) * ld_result + m0 + r, dtype, v, ar.M - m0 - r, vec);
    });
  }
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int, int, NoState&, int, int) const {}
};

// ---------------------------------------------------------------------------------------------------------------
// small matrices: the whole iteration in one workgroup's LDS
// ---------------------------------------------------------------------------------------------------------------
// X (MP x NP) and S (MP x MP) as two planes each, zero beyond the matrix; B replaces S and X' replaces X once every wave has its
// tiles of them in registers.  One launch instead of 3 steps + 2, whose cost at these sizes is the launches and the loads' latency:
// eight 128 x 128 fp32 matrices, five steps: 111 us in 17 launches, 59 us in this one (8.6 us a step, of which the matrix
// instructions take 4; the rest is LDS latency and the barriers between the three products).
// A piece of 16 bytes at c of row r lies at c ^ turn(r): rows of 16 pieces and more serve both the K-major reads (16 rows, one
// piece) and the transposing ones (4 rows, 4 pieces) without bank conflicts; 8-piece rows (S of 64) are read K-major only.
template <int COLS>
__device__ __forceinline__ int small_turn(int r) {
  return COLS == 64 ? (r ^ (r >> 3)) & 7 : ((r & 3) << 2) | ((r >> 2) & 3);
}
template <int COLS>
__device__ __forceinline__ u32x4 small_rows(const u32x4* m, int row, int kk, int lane) {  // 32 rows, k = 16 kk ..: K-major
  const int r = row + (lane & 31), c = kk * 2 + (lane >> 5);
  return m[r * (COLS / 8) + (c ^ small_turn<COLS>(r))];
}
template <int COLS>
__device__ __forceinline__ u32x4 small_cols(const u32x4* m, int col, int kk, int lane) {  // 32 columns, k = rows 16 kk ..
  const int i = lane & 15, kq = i >> 2, n = col + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
  const int k = kk * 16 + (lane >> 5) * 8 + kq;
  const char* a = reinterpret_cast<const char*>(m + k * (COLS / 8) + ((n >> 3) ^ small_turn<COLS>(k))) + (n & 4) * 2;
  const char* b = reinterpret_cast<const char*>(m + (k + 4) * (COLS / 8) + ((n >> 3) ^ small_turn<COLS>(k + 4))) + (n & 4) * 2;
  const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a));
  const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)b));
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}
// four consecutive numbers of a row
template <int COLS>
__device__ __forceinline__ u16* small_at(u32x4* m, int r, int c) {
  return reinterpret_cast<u16*>(m + r * (COLS / 8) + ((c >> 3) ^ small_turn<COLS>(r))) + (c & 4);
}

// TR x TC tiles of 32 x 32 on NW waves.  A wave's PER tiles share the second operand (TC < NW: every NW / TC-th tile row of one tile
// column) or are whole tile columns (TC >= NW).
template <int TR, int TC, int NW>
struct SmallTiles {
  static constexpr int PER = TC >= NW ? TR * (TC / NW) : (TR + NW / TC - 1) / (NW / TC);  // tiles of a wave
  __device__ __forceinline__ static int row(int wave, int i) { return TC >= NW ? i % TR : wave / TC + i * (NW / TC); }
  __device__ __forceinline__ static int col(int wave, int i) { return TC >= NW ? wave + i / TR * NW : wave % TC; }
  // acc = A B over kt 16s (an even number): rows(plane, first row, 16) of A, other(plane, first row or column, 16) of B
  template <class Rows, class Other>
  __device__ __forceinline__ static void multiply(f32x16 (&acc)[PER], int wave, int kt, const Rows& rows, const Other& other) {
    constexpr bool APART = PER <= 2;  // lower planes summed apart where the registers allow
    constexpr int NP_ = TC >= NW ? TR : PER, NQ = TC >= NW ? PER / TR : 1;  // different first / second operands of a wave
    f32x16 low[APART ? PER : 1];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[i][e] = 0.f;
        if constexpr (APART) low[i][e] = 0.f;
      }
    if (row(wave, PER - 1) >= TR && (PER > 1 || row(wave, 0) >= TR)) return;  // (more waves than tiles)
    u32x4 p[2][NP_][2], q[2][NQ][2];
    auto fetch = [&](int f, int kk) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int i = 0; i < NP_; ++i) p[f][i][w] = rows(w, row(wave, i) * 32, kk);
#pragma unroll
        for (int i = 0; i < NQ; ++i) q[f][i][w] = other(w, col(wave, i * TR) * 32, kk);
      }
    };
    auto product = [&](int f) {
#pragma unroll
      for (int s = 0; s < 3; ++s)  // lo hi, hi lo, hi hi
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          f32x16& c = APART && s < 2 ? low[APART ? i : 0] : acc[i];
          c = mfma<F16>(q[f][TC >= NW ? i / TR : 0][s == 0], p[f][TC >= NW ? i % TR : i][s == 1], c);
        }
    };
    fetch(0, 0);
#pragma unroll 1
    for (int kk = 0; kk < kt; kk += 2) {  // fragments one step ahead of the products
      fetch(1, kk + 1);
      product(0);
      fetch(0, min(kk + 2, kt - 1));
      product(1);
    }
    if constexpr (APART)
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] += low[i];
  }
  // fn(tile's accumulators' four numbers, row, first column) for every piece this wave holds
  template <class Fn>
  __device__ __forceinline__ static void each(f32x16 (&acc)[PER], int wave, int lane, const Fn& fn) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (row(wave, i) >= TR) continue;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        f32x4 w = {acc[i][4 * v], acc[i][4 * v + 1], acc[i][4 * v + 2], acc[i][4 * v + 3]};
        fn(w, row(wave, i) * 32 + (lane & 31), col(wave, i) * 32 + v * 8 + (lane >> 5) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][4 * v + e] = w[e];
      }
    }
  }
};

template <int MP, int NP, int kSmallThreads>
__global__ __launch_bounds__(kSmallThreads, 1) void small_kernel(const Tensor g, float eps, int flip, int m, int n, int steps, float a,
                                                                 float b, float c, void* __restrict__ out, int64_t ld_out,
                                                                 int64_t batch_out) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int XP = MP * NP / 8, SP = MP * MP / 8;  // pieces per plane
  constexpr int NW = kSmallThreads / 64, PT = MP * NP / 4 / kSmallThreads;  // waves; pieces of four per thread
  using TS = SmallTiles<MP / 32, MP / 32, NW>;
  using TX = SmallTiles<MP / 32, NP / 32, NW>;
  static_assert(TS::PER == 1 || (MP / 32) % TS::PER == 0, "whole tiles per wave");
  __shared__ u32x4 X[2 * XP];
  __shared__ u32x4 S[2 * SP];
  __shared__ double red[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t base = (int64_t)blockIdx.x * g.batch;

  // X_0: read once into registers (flip: consecutive threads take consecutive rows of X, that is consecutive numbers of a row of G)
  f32x4 x[PT];
  double s = 0;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int t = i * kSmallThreads + threadIdx.x;
    const int r = flip ? t % MP : t / (NP / 4), c0 = (flip ? t / MP : t % (NP / 4)) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int rr = min(r, m - 1), cc = min(c0 + e, n - 1);  // (clamped loads: see the mask below)
      x[i][e] = load_as(g.p, base + (flip ? (int64_t)cc * g.ld + rr : (int64_t)rr * g.ld + cc), g.dtype);
    }
  }
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int t = i * kSmallThreads + threadIdx.x;
    const int r = flip ? t % MP : t / (NP / 4), c0 = (flip ? t / MP : t % (NP / 4)) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[i][e] = r < m && c0 + e < n ? x[i][e] : 0.f;
      s += (double)x[i][e] * x[i][e];
    }
  }
  for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) s += red[w];
  const Scale scale(s, eps);
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    const int t = i * kSmallThreads + threadIdx.x;
    const int r = flip ? t % MP : t / (NP / 4), c0 = (flip ? t / MP : t % (NP / 4)) * 4;
    f32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = scale(x[i][e]);
    store_planes<F16, 2>(small_at<NP>(X, r, c0), (int64_t)XP * 8, w);
  }
  __syncthreads();

  auto x_rows = [&](int w, int r, int kk) { return small_rows<NP>(X + w * XP, r, kk, lane); };
  auto x_cols = [&](int w, int col, int kk) { return small_cols<NP>(X + w * XP, col, kk, lane); };
  auto s_rows = [&](int w, int r, int kk) { return small_rows<MP>(S + w * SP, r, kk, lane); };
  auto s_put = [&](const f32x4& v, int r, int c0) { store_planes<F16, 2>(small_at<MP>(S, r, c0), (int64_t)SP * 8, v); };
  const int kn = (n + 31) / 32 * 2, km = (m + 31) / 32 * 2;  // (16s of the two inner axes; zeros behind the matrix)
  for (int k = 0; k < steps; ++k) {
    f32x16 acc[TS::PER];
    TS::multiply(acc, wave, kn, x_rows, x_rows);  // S = X X^T
    TS::each(acc, wave, lane, [&](f32x4& v, int r, int c0) {
      v *= 1.f / kScale;
      s_put(v, r, c0);
    });
    __syncthreads();
    TS::multiply(acc, wave, km, s_rows, s_rows);  // B = b S + c S S, its own S read before anybody overwrites it
    TS::each(acc, wave, lane, [&](f32x4& v, int r, int c0) { v = v * (c / kScale) + b * load_planes(small_at<MP>(S, r, c0), (int64_t)SP * 8); });
    __syncthreads();
    TS::each(acc, wave, lane, [&](f32x4& v, int r, int c0) { s_put(v, r, c0); });
    __syncthreads();
    f32x16 next[TX::PER];
    TX::multiply(next, wave, km, s_rows, x_cols);  // X' = a X + B X
    TX::each(next, wave, lane, [&](f32x4& v, int r, int c0) { v = v * (1.f / kScale) + a * load_planes(small_at<NP>(X, r, c0), (int64_t)XP * 8); });
    __syncthreads();
    if (k + 1 < steps) {
      TX::each(next, wave, lane, [&](f32x4& v, int r, int c0) { store_planes<F16, 2>(small_at<NP>(X, r, c0), (int64_t)XP * 8, v); });
      __syncthreads();
    } else {
      const int64_t o = (int64_t)blockIdx.x * batch_out;
      TX::each(next, wave, lane, [&](f32x4& v, int r, int c0) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r < m && c0 + e < n)
            store_as(out, o + (flip ? (int64_t)(c0 + e) * ld_out + r : (int64_t)r * ld_out + c0 + e), g.dtype, v[e] * (1.f / kScale));
      });
    }
  }
#endif
}

// whether LDS and the registers hold it (64 x 512 spills and gains nothing: 96 us against 98 us as separate launches)
bool small_fits(int m, int n) { return (m <= 128 && n <= 128) || (m <= 64 && n <= 256); }

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------
// rows on whole cache lines, which a K tile's pieces then cover (rows of 8 elements' multiples: 2 x 513 x 1001 225 -> 199 us,
// 5000 x 400 264 -> 246 us)
inline int64_t up64(int64_t v) { return (v + 63) & ~(int64_t)63; }

// Square tiles of 256, 192, 128 and 64 (the 192-wide ones only for the symmetric products: their 192 rows do not fit the
// MN-major staging).  One workgroup per CU, two of the smallest.  The 128-wide tile has eight waves and four stages: short sums are
// bound by the loads' latency (2048 x 2048 x 512 on two planes: 15.7 us, with four waves and two longer stages 17.8).
template <bool BK, int NPL>
struct Tiles {
  static constexpr int K = NPL == 1 ? 64 : 32;
  using T256 = Tile<F16, NPL, NPL, 256, 256, K, 2, 2, 4, true, BK>;
  using T192 = Tile<F16, NPL, NPL, 192, 192, K, 3, 2, 2, true, true>;
  using T128 = Tile<F16, NPL, NPL, 128, 128, K, 4, 2, 4, true, BK>;
  using T64 = Tile<F16, NPL, NPL, 64, 64, 64, 2, 2, 2, true, BK>;
  using T64Deep = Tile<F16, NPL, NPL, 64, 64, 64, 4, 2, 2, true, BK>;
};

inline int64_t tile_count(int64_t M, int64_t N, int t, bool sym) {
  const int64_t a = (M + t - 1) / t, b = (N + t - 1) / t;
  return sym ? a * (a + 1) / 2 : a * b;
}
// Time of a product in us, from the rounds its tiles need and what a full round took here (K = 8192, one tile per CU: 256 616 us, 192
// 384, 128 181, 64 77 and two per CU 101), a start-up of 2 us per round, and for a product split along K the pass that joins
// the fp32 partial sums.  A triangle of large tiles often fills its last round badly: 4096 x 4096 has 136 tiles of 256 (616 us
// at K = 8192), 528 of 128 (543) and 253 of 192 (384).
inline double product_us(int64_t M, int64_t N, int64_t K, int64_t batch, bool sym, int tile, int splits) {
  const int64_t n = tile_count(M, N, tile, sym) * batch * splits;
  const double share = (double)((K + splits - 1) / splits) / 8192.0;
  double t, rounds;
  if (tile == 64) {
    const int64_t full = n / (2 * kCUs), rest = n % (2 * kCUs);
    rounds = (double)full + (rest ? 1 : 0);
    t = share * (101.0 * (double)full + (rest > kCUs ? 101.0 : rest ? 77.0 : 0.0));
  } else {
    rounds = (double)((n + kCUs - 1) / kCUs);
    t = share * rounds * (tile == 256 ? 616.0 : tile == 192 ? 384.0 : 181.0);
  }
  if (splits > 1) t += 4.5 + (double)batch * splits * (double)M * N * (sym ? 0.5 : 1.0) * 8.0 / 4.0e6;
  return t + 2.0 * rounds + 2.0;
}
struct Choice {
  int tile, splits;
};
inline Choice choose(int64_t M, int64_t N, int64_t K, int64_t batch, bool sym) {
  Choice best{64, 1};
  double t = 1e30;
  for (const int tile : {256, 192, 128, 64}) {
    if (tile == 192 && !sym) continue;
    for (int splits = 1; splits == 1 || (sym && splits <= 32 && K / splits >= 256); ++splits) {
      const double u = product_us(M, N, K, batch, sym, tile, splits);
      if (u < t) t = u, best = {tile, splits};
    }
  }
  return best;
}

template <class T, class Epi>
void launch(Args a, const Epi& epi, int cols, int batch, int splits, bool sym, hipStream_t s) {
  a.tiles_m = (a.M + T::BM - 1) / T::BM;
  a.tiles_n = (cols + T::BN - 1) / T::BN;
  const int k_tiles = (a.K + T::BK - 1) / T::BK;
  a.k_tiles_per_split = (k_tiles + splits - 1) / splits;
  a.symmetric = sym;
  const int64_t n = sym ? (int64_t)a.tiles_m * (a.tiles_m + 1) / 2 : (int64_t)a.tiles_m * a.tiles_n;
  hipLaunchKernelGGL((product_kernel<T, Epi>), dim3((unsigned)n, (unsigned)batch, (unsigned)splits), dim3(T::NT), 0, s, a, epi);
}
template <bool BK, int NPL, class Epi>
void product(const Args& a, const Epi& epi, int cols, int batch, const Choice& ch, bool sym, hipStream_t s) {
  using TT = Tiles<BK, NPL>;
  if (ch.tile == 256) launch<typename TT::T256>(a, epi, cols, batch, ch.splits, sym, s);
  else if (ch.tile == 128) launch<typename TT::T128>(a, epi, cols, batch, ch.splits, sym, s);
  else if (ch.tile == 64 && a.K / ch.splits >= 384 && tile_count(a.M, cols, 64, sym) * batch * ch.splits <= kCUs)
    launch<typename TT::T64Deep>(a, epi, cols, batch, ch.splits, sym, s);  // (one per CU: the LDS is better spent on loads in flight)
  else if (ch.tile == 64) launch<typename TT::T64>(a, epi, cols, batch, ch.splits, sym, s);
  else if constexpr (BK) launch<typename TT::T192>(a, epi, cols, batch, ch.splits, sym, s);
}
// a symmetric product, split along K or not
template <int NPL>
void symmetric_product(const Args& a, const SymEpi<NPL>& epi, int batch, const Choice& ch, float* partial, hipStream_t s) {
  if (ch.splits == 1) return product<true, NPL>(a, epi, a.M, batch, ch, true, s);
  product<true, NPL>(a, SymPartialEpi{partial, epi.size, epi.ld}, a.M, batch, ch, true, s);
  const int blocks = (epi.ld + 31) / 32;
  hipLaunchKernelGGL(sym_join_kernel<NPL>, dim3(blocks, batch, blocks), dim3(256), 0, s, partial, ch.splits, ch.tile, epi);
}
// one step: S and B with NPL planes, X' = out (always two planes) or the result
struct Step {
  Operand x, s, b;
  u16 *sm, *bm;
  int64_t s_plane, s_batch;
  int M, N, lds, batch;
  float b_coeff, c_coeff;
  float* partial;
  Choice cs, cb, cx;
};
template <int NPL>
void step(const Step& t, const StepEpi& out, hipStream_t s) {
  Args ar{};
  ar.A = t.x, ar.B = t.x, ar.M = t.M, ar.N = t.M, ar.K = t.N;
  symmetric_product(ar, SymEpi<NPL>{1.f / kScale, 0.f, nullptr, t.sm, t.s_plane, t.s_batch, t.M, t.lds}, t.batch, t.cs, t.partial, s);
  ar.A = t.s, ar.B = t.s, ar.K = t.M;
  symmetric_product(ar, SymEpi<NPL>{t.c_coeff / kScale, t.b_coeff, t.sm, t.bm, t.s_plane, t.s_batch, t.M, t.lds}, t.batch, t.cb, t.partial, s);
  ar.A = t.b, ar.B = t.x, ar.N = t.N;
  product<false, NPL>(ar, out, t.N, t.batch, t.cx, false, s);
}

struct Layout {
  int64_t x_plane, s_plane, x_batch, s_batch;  // elements
  int64_t norm, x0, x1, sm, bm, partial, total;  // byte offsets
  int ldx, lds, parts;
  Choice cs, cb, cx;  // S, B, X'
};
inline int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }
Layout layout_of(int64_t batch, int64_t m, int64_t n) {  // m <= n
  Layout l;
  l.ldx = (int)up64(n), l.lds = (int)up64(m);
  l.x_plane = m * l.ldx, l.s_plane = m * l.lds;
  l.x_batch = 2 * l.x_plane, l.s_batch = 2 * l.s_plane;
  if (small_fits((int)m, (int)n)) {
    l.total = 0;
    return l;
  }
  l.cs = choose(m, m, n, batch, true);
  l.cb = choose(m, m, m, batch, true);
  l.cx = choose(m, n, m, batch, false);
  int64_t o = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = o;
    o += align256(bytes);
    return r;
  };
  // workgroups of the norm: at least 4 K elements each, at most 1024 per matrix (4096 x 8192 in bf16: 256 40 us, 1024 19 us)
  l.parts = (int)((m * n + 4095) / 4096 < 1024 ? (m * n + 4095) / 4096 : 1024);
  l.norm = take(batch * l.parts * 8);
  l.x0 = take(batch * l.x_batch * 2);
  l.x1 = take(batch * l.x_batch * 2);
  l.sm = take(batch * l.s_batch * 2);
  l.bm = take(batch * l.s_batch * 2);
  const int most = l.cs.splits > l.cb.splits ? l.cs.splits : l.cb.splits;
  l.partial = take(most > 1 ? (int64_t)most * batch * m * l.lds * 4 : 0);
  l.total = o;
  return l;
}

// Steps of a bf16 update whose products take X, S and B as one plane: early ones, three or more before the end (what a step gets
// wrong is taken on by the next ones with slopes of up to 3.9, so not in long iterations either), of matrices with many singular
// values (m: the smaller side).  4096 x 8192, five steps: two planes throughout 6.61 ms, this rule 5.13, one plane in a
// third step 4.38; 2 x 513 x 1001: 193, 174 and 165 us.
bool one_plane(int k, int m, int steps) { return k < 2 && k + 3 < steps && steps <= 8 && m >= 128; }

int check_sizes(const char* what, int batch, int m, int n) {
  CRADLE_CHECK_ARG(batch >= 1 && batch <= 65535 && m >= 1 && n >= 1 && m <= (1 << 17) && n <= (1 << 17),
                   "%s: batch=%d m=%d n=%d (1 <= batch <= 65535, sides <= 2^17)", what, batch, m, n);
  return CRADLE_OK;
}

}  // namespace
}  // namespace cradle

using namespace cradle;

extern "C" {

int64_t cradle_orthogonalize_workspace_bytes(int batch, int m, int n) {
  if (check_sizes("orthogonalize_workspace_bytes", batch, m, n) != CRADLE_OK) return -1;
  return layout_of(batch, m < n ? m : n, m < n ? n : m).total;
}

int cradle_orthogonalize(const void* g, int64_t ld_g, int64_t batch_stride_g, void* out, int64_t ld_out, int64_t batch_stride_out,
                         int dtype, int batch, int m, int n, int steps, float a, float b, float c, float eps, void* workspace,
                         int64_t workspace_bytes, cradle_stream_t s) {
  const int rc = check_sizes("orthogonalize", batch, m, n);
  if (rc != CRADLE_OK) return rc;
  CRADLE_CHECK_ARG(dtype == CRADLE_F32 || dtype == CRADLE_BF16 || dtype == CRADLE_F16, "orthogonalize: dtype %d", dtype);
  CRADLE_CHECK_ARG(g && out && ld_g >= n && ld_out >= n, "orthogonalize: null pointer or leading dimension below the row length");
  CRADLE_CHECK_ARG(steps >= 1 && steps <= 64, "orthogonalize: steps=%d (1..64)", steps);
  const bool flip = m > n;
  const int M = flip ? n : m, N = flip ? m : n;
  const Layout l = layout_of(batch, M, N);
  CRADLE_CHECK_ARG(l.total == 0 || (workspace && workspace_bytes >= l.total && ((uintptr_t)workspace & 15) == 0),
                   "orthogonalize: workspace of %lld bytes (16-byte aligned) needed", (long long)l.total);
  char* w = static_cast<char*>(workspace);
  double* norm = reinterpret_cast<double*>(w + l.norm);
  u16 *x = reinterpret_cast<u16*>(w + l.x0), *x_next = reinterpret_cast<u16*>(w + l.x1);
  u16 *sm = reinterpret_cast<u16*>(w + l.sm), *bm = reinterpret_cast<u16*>(w + l.bm);
  float* partial = reinterpret_cast<float*>(w + l.partial);
  const Tensor gt{g, ld_g, batch_stride_g, dtype, m, n};
  if (small_fits(M, N)) {
#define CRADLE_NS_SMALL(MP, NP, THREADS)                                                                                              \
  hipLaunchKernelGGL((small_kernel<MP, NP, THREADS>), dim3(batch), dim3(THREADS), 0, s, gt, eps, (int)flip, M, N, steps, a, b, c, out, \
                     ld_out, batch_stride_out)
    if (M > 64) CRADLE_NS_SMALL(128, 128, 1024);
    else if (N <= 128) CRADLE_NS_SMALL(64, 128, 512);
    else CRADLE_NS_SMALL(64, 256, 1024);
#undef CRADLE_NS_SMALL
    CRADLE_CHECK_LAUNCH("orthogonalize");
    return CRADLE_OK;
  }
  const int V = dtype == CRADLE_F32 ? 4 : 8;
  const bool vec = n % V == 0 && ld_g % V == 0 && batch_stride_g % V == 0 && ((uintptr_t)g & 15) == 0;
  auto sumsq = dtype == CRADLE_F32    ? (vec ? sumsq_kernel<CRADLE_F32, true> : sumsq_kernel<CRADLE_F32, false>)
               : dtype == CRADLE_BF16 ? (vec ? sumsq_kernel<CRADLE_BF16, true> : sumsq_kernel<CRADLE_BF16, false>)
                                      : (vec ? sumsq_kernel<CRADLE_F16, true> : sumsq_kernel<CRADLE_F16, false>);
  hipLaunchKernelGGL(sumsq, dim3(l.parts, batch), dim3(256), 0, s, gt, norm);
  hipLaunchKernelGGL(pack_kernel, dim3((N + 63) / 64, (M + 63) / 64, batch), dim3(256), 0, s, gt, norm, l.parts, eps, (int)flip, x, l.x_plane,
                     l.x_batch, M, N, l.ldx);
  const int vec_out = ld_out % 4 == 0 && batch_stride_out % 4 == 0 && ((uintptr_t)out & (dtype == CRADLE_F32 ? 15 : 7)) == 0;
  for (int k = 0; k < steps; ++k) {
    const Step t{{x, l.ldx, l.x_plane, l.x_batch}, {sm, l.lds, l.s_plane, l.s_batch}, {bm, l.lds, l.s_plane, l.s_batch},
                 sm, bm, l.s_plane, l.s_batch, M, N, l.lds, batch, b, c, partial, l.cs, l.cb, l.cx};
    const StepEpi epi{a, 1.f / kScale, x, x_next, l.x_plane, l.x_batch, l.ldx, k + 1 == steps ? out : nullptr, ld_out, batch_stride_out,
                      dtype, (int)flip, vec_out};
    if (dtype == CRADLE_BF16 && one_plane(k, M, steps)) step<1>(t, epi, s);
    else step<2>(t, epi, s);
    u16* next = x_next;
    x_next = x;
    x = next;
  }
  CRADLE_CHECK_LAUNCH("orthogonalize");
  return CRADLE_OK;
}

}  // extern "C"
