// Orthogonalised update: the odd polynomial iteration that sends every singular value of a matrix towards one,
//   X_0 = G / (|G|_F + eps),   S = X X^T,   X <- a X + (b S + c S S) X      (on the smaller side of the matrix)
// as three tile products per step (mm16.h), the polynomial in their epilogues.
//
// Numbers: X, S and B = b S + c S S are kept as two fp16 planes (hi + lo, 22 bits), three products per element pair with fp32
// accumulation.  The iteration is normalised, |X_ij| <= |X|_2 <= max |p(s)|, so fp16's range is no obstacle: everything is held
// times 2^12, which puts the lo plane of an entry of size 2^-6 (a 4096-wide matrix) well above fp16's subnormals and keeps
// |X| < 16 (checked for the coefficients by the caller) below its largest number.  fp32 results at three products of a rate
// 16 times the fp32 matrix instruction's; 16-bit tensors take the same path, because the iteration multiplies the error in
// a small singular value by up to a per step (3.4^5 = 480) and one fp16 or bf16 plane would show.
// S and B are symmetric: only the tiles on and below the diagonal are computed, the epilogue stores them twice.
// The norm is accumulated in fp64 (squares of fp32 gradients leave fp32's range).
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
  double s = (int)threadIdx.x < parts ? part[(int64_t)blockIdx.z * parts + threadIdx.x] : 0.0;  // (parts <= 256)
  for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = (red[0] + red[1]) + (red[2] + red[3]);
  const float scale = kScale / ((float)sqrt(s) + eps);
  const int64_t base = (int64_t)blockIdx.z * g.batch;
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;  // of X
  const int g0 = flip ? n0 : m0, g1 = flip ? m0 : n0;    // of G
  for (int i = threadIdx.x; i < 64 * 64; i += 256) {
    const int r = i / 64, c = i % 64;
    tile[r][c] = g0 + r < g.rows && g1 + c < g.cols ? load_as(g.p, base + (int64_t)(g0 + r) * g.ld + g1 + c, g.dtype) * scale : 0.f;
  }
  __syncthreads();
  u16* out = x + (int64_t)blockIdx.z * batch;
  for (int i = threadIdx.x; i < 64 * 16; i += 256) {
    const int r = i / 16, c = i % 16 * 4;
    if (m0 + r >= m || n0 + c >= ldx) continue;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = flip ? tile[c + e][r] : tile[r][c + e];
    store_planes<F16, 2>(out + (int64_t)(m0 + r) * ldx + n0 + c, plane, v);
  }
}

// four consecutive numbers of a two-plane matrix
__device__ __forceinline__ f32x4 load_planes(const u16* p, int64_t plane) {
  const u32x2 h = *reinterpret_cast<const u32x2*>(p), l = *reinterpret_cast<const u32x2*>(p + plane);
  return f32x4{from_f16((u16)h.x) + from_f16((u16)l.x), from_f16((u16)(h.x >> 16)) + from_f16((u16)(l.x >> 16)),
               from_f16((u16)h.y) + from_f16((u16)l.y), from_f16((u16)(h.y >> 16)) + from_f16((u16)(l.y >> 16))};
}

struct NoState {};

// out = alpha acc + beta add, a symmetric matrix of `size` rows, ld = size rounded up to 8 (padding columns zero).  Tiles below the
// diagonal are stored a second time, turned, above it.
struct SymEpi {
  [[maybe_unused]] static constexpr bool PAIR = false;
  using State = NoState;
  float alpha, beta;
  const u16* add;  // or NULL
  u16* out;
  int64_t plane, batch;
  int size, ld;
  __device__ __forceinline__ f32x4 value(int m, int n, f32x4 v) const {
    v *= alpha;
    if (m < size && n < ld && add) v += beta * load_planes(add + (int64_t)blockIdx.y * batch + (int64_t)m * ld + n, plane);
    return v;
  }
  __device__ __forceinline__ void put(int row, int col, f32x4 v) const {
    if (row < size && col < ld) store_planes<F16, 2>(out + (int64_t)blockIdx.y * batch + (int64_t)row * ld + col, plane, v);
  }
  template <class T>
  __device__ __forceinline__ void emit(const Args&, float* buf, int m0, int n0, int lane, NoState&, int tm, int tn) const {
    each_piece<T, T::WN>(buf, lane, [&](int r, int c, f32x4* p) {
      const f32x4 v = value(m0 + r, n0 + c, *p);
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
__global__ __launch_bounds__(256) void sym_join_kernel(const float* __restrict__ partial, int splits, int tile, const SymEpi epi) {
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
  v = epi.value(m, n, v);
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
    each_piece<T, T::WN>(buf, lane, [&](int r, int c, f32x4* p) {
      const int m = m0 + r, n = n0 + c;
      if (m >= ar.M || n >= ld) return;
      const f32x4 v = alpha * *p + a * load_planes(x + b + (int64_t)m * ld + n, plane);
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
// host side
// ---------------------------------------------------------------------------------------------------------------
inline int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }

// three tile sizes: the largest whose tiles still occupy the chip
template <bool BK>
struct Tiles {
  using Large = Tile<F16, 2, 2, 256, 256, 32, 2, 2, 4, true, BK>;
  using Medium = Tile<F16, 2, 2, 128, 128, 32, 2, 2, 2, true, BK>;
  using Small = Tile<F16, 2, 2, 64, 64, 64, 2, 2, 2, true, BK>;
};

inline int64_t tile_count(int64_t M, int64_t N, int t, bool sym) {
  const int64_t a = (M + t - 1) / t, b = (N + t - 1) / t;
  return sym ? a * (a + 1) / 2 : a * b;
}
inline int pick_tile(int64_t M, int64_t N, int64_t batch, bool sym) {
  if (tile_count(M, N, 256, sym) * batch >= kCUs) return 256;
  if (tile_count(M, N, 128, sym) * batch >= kCUs) return 128;
  return 64;
}
// shares of the K axis of a symmetric product whose tiles leave CUs idle, each at least 512 long
inline int pick_splits(int64_t m, int64_t K, int64_t batch, int tile) {
  const int64_t t = tile_count(m, m, tile, true) * batch;
  if (t >= kCUs) return 1;
  const int64_t want = (kCUs + t - 1) / t, most = K / 512;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s);
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
template <bool BK, class Epi>
void product(const Args& a, const Epi& epi, int cols, int batch, int tile, int splits, bool sym, hipStream_t s) {
  if (tile == 256) launch<typename Tiles<BK>::Large>(a, epi, cols, batch, splits, sym, s);
  else if (tile == 128) launch<typename Tiles<BK>::Medium>(a, epi, cols, batch, splits, sym, s);
  else launch<typename Tiles<BK>::Small>(a, epi, cols, batch, splits, sym, s);
}

struct Layout {
  int64_t x_plane, s_plane, x_batch, s_batch;  // elements
  int64_t norm, x0, x1, sm, bm, partial, total;  // byte offsets
  int ldx, lds, tile_s, splits, parts;
};
inline int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }
Layout layout_of(int64_t batch, int64_t m, int64_t n) {  // m <= n
  Layout l;
  l.ldx = (int)up8(n), l.lds = (int)up8(m);
  l.x_plane = m * l.ldx, l.s_plane = m * l.lds;
  l.x_batch = 2 * l.x_plane, l.s_batch = 2 * l.s_plane;
  l.tile_s = pick_tile(m, m, batch, true);
  l.splits = pick_splits(m, n, batch, l.tile_s);
  int64_t o = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = o;
    o += align256(bytes);
    return r;
  };
  // workgroups of the norm: 16 K elements each, at most 256 per matrix
  l.parts = (int)((m * n + 16383) / 16384 < 256 ? (m * n + 16383) / 16384 : 256);
  l.norm = take(batch * l.parts * 8);
  l.x0 = take(batch * l.x_batch * 2);
  l.x1 = take(batch * l.x_batch * 2);
  l.sm = take(batch * l.s_batch * 2);
  l.bm = take(batch * l.s_batch * 2);
  l.partial = take(l.splits > 1 ? (int64_t)l.splits * batch * m * l.lds * 4 : 0);
  l.total = o;
  return l;
}

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
  CRADLE_CHECK_ARG(workspace && workspace_bytes >= l.total && ((uintptr_t)workspace & 15) == 0,
                   "orthogonalize: workspace of %lld bytes (16-byte aligned) needed", (long long)l.total);
  char* w = static_cast<char*>(workspace);
  double* norm = reinterpret_cast<double*>(w + l.norm);
  u16 *x = reinterpret_cast<u16*>(w + l.x0), *x_next = reinterpret_cast<u16*>(w + l.x1);
  u16 *sm = reinterpret_cast<u16*>(w + l.sm), *bm = reinterpret_cast<u16*>(w + l.bm);
  float* partial = reinterpret_cast<float*>(w + l.partial);
  const Tensor gt{g, ld_g, batch_stride_g, dtype, m, n};
  const int V = dtype == CRADLE_F32 ? 4 : 8;
  const bool vec = n % V == 0 && ld_g % V == 0 && batch_stride_g % V == 0 && ((uintptr_t)g & 15) == 0;
  auto sumsq = dtype == CRADLE_F32    ? (vec ? sumsq_kernel<CRADLE_F32, true> : sumsq_kernel<CRADLE_F32, false>)
               : dtype == CRADLE_BF16 ? (vec ? sumsq_kernel<CRADLE_BF16, true> : sumsq_kernel<CRADLE_BF16, false>)
                                      : (vec ? sumsq_kernel<CRADLE_F16, true> : sumsq_kernel<CRADLE_F16, false>);
  hipLaunchKernelGGL(sumsq, dim3(l.parts, batch), dim3(256), 0, s, gt, norm);
  hipLaunchKernelGGL(pack_kernel, dim3((N + 63) / 64, (M + 63) / 64, batch), dim3(256), 0, s, gt, norm, l.parts, eps, (int)flip, x, l.x_plane,
                     l.x_batch, M, N, l.ldx);
  const int vec_out = ld_out % 4 == 0 && batch_stride_out % 4 == 0 && ((uintptr_t)out & (dtype == CRADLE_F32 ? 15 : 7)) == 0;
  const int tile_x = pick_tile(M, N, batch, false);
  for (int k = 0; k < steps; ++k) {
    const Operand xo{x, l.ldx, l.x_plane, l.x_batch}, so{sm, l.lds, l.s_plane, l.s_batch}, bo{bm, l.lds, l.s_plane, l.s_batch};
    Args ar{};
    ar.A = xo, ar.B = xo, ar.M = M, ar.N = M, ar.K = N;
    const SymEpi es{1.f / kScale, 0.f, nullptr, sm, l.s_plane, l.s_batch, M, l.lds};
    if (l.splits > 1) {
      product<true>(ar, SymPartialEpi{partial, M, l.lds}, M, batch, l.tile_s, l.splits, true, s);
      const int blocks = (M + 31) / 32, cols = (l.lds + 31) / 32, rows = cols > blocks ? cols : blocks;
      hipLaunchKernelGGL(sym_join_kernel, dim3(cols, batch, rows), dim3(256), 0, s, partial, l.splits, l.tile_s, es);
    } else {
      product<true>(ar, es, M, batch, l.tile_s, 1, true, s);
    }
    ar.A = so, ar.B = so, ar.K = M;
    product<true>(ar, SymEpi{c / kScale, b, sm, bm, l.s_plane, l.s_batch, M, l.lds}, M, batch, l.tile_s, 1, true, s);
    ar.A = bo, ar.B = xo, ar.N = N;
    const bool last = k + 1 == steps;
    product<false>(ar, StepEpi{a, 1.f / kScale, x, x_next, l.x_plane, l.x_batch, l.ldx, last ? out : nullptr, ld_out, batch_stride_out, dtype,
                               (int)flip, vec_out},
                   N, batch, tile_x, 1, false, s);
    u16* t = x;
    x = x_next;
    x_next = t;
  }
  CRADLE_CHECK_LAUNCH("orthogonalize");
  return CRADLE_OK;
}

}  // extern "C"
