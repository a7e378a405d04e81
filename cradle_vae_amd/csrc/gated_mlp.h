// The gated feed-forward block and its backward pass:
//   [g | u] = x W_in^T + b_in,   h = act(g) * u,   y = h W_out^T + b_out (+ residual)
//   dh = dy W_out,  dg = dh u act'(g),  du = dh act(g)
//   dx = [dg | du] W_in,  dW_in = [dg | du]^T x,  dW_out = dy^T h,  db_in / db_out: column sums of [dg | du] / dy
// Two products forward (x W_in^T with both projections, the activation and the gating in its epilogue), four backward (the
// first with the whole elementwise backward in its epilogue, the others in one launch); mm16.h has the tile product and what bounds it.
//
// Numbers: bf16 / fp16 tensors multiply as they are; fp32 tensors as three bf16 planes (six products, fp32's accuracy at
// 2.6x the rate of the fp32 matrix instruction).  Sums, pre-activations and biases are fp32.  h and [dg | du] are inputs of a
// matrix product and so are rounded once to the operand's type, an error of the size of the result's own last rounding; small
// blocks, whose few numbers would not average it out and which are bound by latency, keep them in two planes instead.
// In fp16 they have its range as well, with either number of planes: an h beyond 65504 is infinite, a [dg | du] below 2^-24 zero.
// (bf16 planes beside fp16 tensors would keep fp32's range, at three products instead of one for four of the six.)
// The saved pre-activations stay fp32 (rounded to bf16 they would put two more roundings into every gradient).
// A handful of rows (inference of single cells) take kernels that read the weights once, coalesced, with fp32 arithmetic.
//
// Measured on two cards, forward and backward: 8192 rows, 4096 x 10240 in bf16 5.2 and 5.3 ms, 1160 to 1190 TFLOP/s (library products
// of these sizes: 1290 to 1560), bound by the matrix cores and the epilogues that a 256 x 256 tile, alone on its CU, does not
// hide; 1537 rows, 1000 x 2731 in fp16 195 and 199 us and 2560 rows, 400 x 800 in fp32 161 and 168 us, bound by the loads' latency
// over sums of 13 to 30 K tiles.
#pragma once
#include <type_traits>

#include "mm16.h"

namespace cradle {
namespace gated {

using namespace mm16;

enum Act { SILU = 0, GELU = 1 };

// act(g) and act'(g), in a handful of instructions: an epilogue has one or two waves per SIMD and nothing to hide long sequences
// behind (with the library's expf, erfcf and divisions the first backward product of 1537 x 1000 x 2731 takes 45 us).
// silu: g s, s = 1 / (1 + exp(-g)) on the hardware's exp2 and reciprocal: relative to s off by (1 - s) (1.5 |g| + 3) + 2 times
// 2^-24, the exponent's argument being rounded (|g| s (1 - s) is at most 0.23, so that is no more than act's own rounding).
// gelu: g Phi(g).  FINE (fp32 tensors): Phi(g) = erfc(-g / sqrt(2)) / 2 by the library's erfcf, accurate relative to Phi down its
// tail.  Otherwise (16-bit tensors, whose half step is 2^-12 and more) Phi(-|g|) = (a1 t + ... + a5 t^5) exp(-g^2 / 2) / 2, t =
// 1 / (1 + 0.3275911 |g| / sqrt(2)): the rational approximation 7.1.26 of Abramowitz and Stegun's Handbook of Mathematical
// Functions, off by at most 0.75e-7, and 2.3e-7 (2^-22) as evaluated in fp32.
// Limits: a gate of 0 with its argument infinite is 0.
__device__ __forceinline__ float sigmoid(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g));
}
__device__ __forceinline__ float gauss(float g) { return __builtin_amdgcn_exp2f(-0.72134752044448170f * g * g); }  // exp(-g^2 / 2)
// Phi(g); e = gauss(g)
template <bool FINE>
__device__ __forceinline__ float normal_cdf(float g, float e) {
  if constexpr (FINE) return 0.5f * erfcf(-0.70710678118654752f * g);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.23164188f, fabsf(g), 1.f));
  const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5307027145f, -0.7265760135f), 0.7107068705f), -0.142248368f), 0.127414796f) * e;
  return g < 0.f ? q : 1.f - q;
}
template <bool FINE>
__device__ __forceinline__ void act_both(int act, float g, float& a, float& da) {
  if (act == SILU) {
    const float s = sigmoid(g);
    a = s == 0.f ? 0.f : g * s;
    da = s == 0.f ? 0.f : s * fmaf(g, 1.f - s, 1.f);
    if (g == INFINITY) da = 1.f;
  } else {
    const float e = gauss(g);
    const float cdf = normal_cdf<FINE>(g, e);
    a = cdf == 0.f ? 0.f : g * cdf;
    da = e == 0.f ? cdf : fmaf(g * 0.39894228040143268f, e, cdf);
  }
}
template <bool FINE>
__device__ __forceinline__ float act_only(int act, float g) {
  const float s = act == SILU ? sigmoid(g) : normal_cdf<FINE>(g, gauss(g));
  return s == 0.f ? 0.f : g * s;
}

// ---------------------------------------------------------------------------------------------------------------
// packing: a tensor as operand planes with padded, zero-filled rows
// ---------------------------------------------------------------------------------------------------------------
struct PackJob {
  const void* src;
  u16* dst;
  int64_t ld_src, plane;
  int rows, cols, rows_dst, ld_dst;
  int gap_at, gap;  // destination rows [gap_at, gap_at + gap) are zero, and so are those behind the source's last
  int vec;          // the source's rows start on 16 bytes
};
struct PackJobs {
  PackJob job[4];
};

// one thread per 8 destination elements; ELEM planes.  DT: the source's type; rows with a 16-byte aligned start are read in
// 16-byte pieces.
template <int ELEM, int NPL>
__global__ __launch_bounds__(256) void pack_kernel(const PackJobs js) {
  constexpr int DT = NPL == 3 ? CRADLE_F32 : ELEM == BF16 ? CRADLE_BF16 : CRADLE_F16;
  const PackJob j = js.job[blockIdx.y];
  const int per = j.ld_dst / 8;
  const int64_t total = (int64_t)j.rows_dst * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int r = (int)(t / per), c0 = (int)(t % per) * 8;
    const int src = r < j.gap_at ? r : r - j.gap;
    const bool zero = (r >= j.gap_at && r < j.gap_at + j.gap) || src >= j.rows;
    const int64_t s = (int64_t)(zero ? 0 : src) * j.ld_src;
    u16 p[8][NPL];
    if constexpr (DT == CRADLE_F32) {
      const float* q = static_cast<const float*>(j.src) + s;
      float v[8];
      if (j.vec && c0 + 8 <= j.cols) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(q + c0), b = *reinterpret_cast<const f32x4*>(q + c0 + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = q[min(c0 + e, j.cols - 1)];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) split<ELEM, NPL>(!zero && c0 + e < j.cols ? v[e] : 0.f, p[e]);
    } else {  // the numbers as they are
      const u16* q = static_cast<const u16*>(j.src) + s;
      u16 v[8];
      if (j.vec && c0 + 8 <= j.cols) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(q + c0);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (u16)(a[e / 2] >> 16 * (e % 2));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = q[min(c0 + e, j.cols - 1)];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e][0] = !zero && c0 + e < j.cols ? v[e] : (u16)0;
    }
#pragma unroll
    for (int k = 0; k < NPL; ++k) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = p[2 * e][k] | (uint32_t)p[2 * e + 1][k] << 16;
      *reinterpret_cast<u32x4*>(j.dst + k * j.plane + (int64_t)r * j.ld_dst + c0) = w;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// epilogues
// ---------------------------------------------------------------------------------------------------------------
struct NoState {};
// a vector's four numbers at n (zero beyond its end, or without it)
struct Four {
  f32x4 v, w;
};
__device__ __forceinline__ f32x4 load4(const void* p, int64_t i, int n, int dtype) {
  f32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < n) v[e] = load_as(p, i + e, dtype);
  return v;
}

// h = act(g) u as operand planes (columns [hidden, ld) zero), g and u saved
template <int ELEM, int NPH>
struct GateEpi {
  static constexpr bool PAIR = true;
  using State = Four;  // the bias of this lane's columns
  int act, hidden, hidden_p;  // hidden_p: row length of h, the padding zero
  int dtype;
  const void* bias;  // (2 hidden) or NULL
  u16* h;
  int64_t h_plane;
  float* gu;  // (rows, 2 hidden_p) or NULL
  template <class T>
  __device__ __forceinline__ Four begin(int n0, int lane) const {
    static_assert(64 % (T::WN / 8) == 0, "a lane keeps its columns");
    const int n = n0 + lane % (T::WN / 8) * 4;
    if (!bias || n >= hidden) return Four{};
    return Four{load4(bias, n, hidden - n, dtype), load4(bias, (int64_t)hidden + n, hidden - n, dtype)};
  }
  template <class T>
  __device__ __forceinline__ void emit(const Args& a, float* buf, int m0, int n0, int lane, const Four& b, int, int) const {
    each_piece<T, T::WN / 2>(buf, lane, [&](int r, int c, const f32x4* p) {
      const int m = m0 + r, n = n0 + c;
      if (m >= a.M || n >= hidden_p) return;
      const f32x4 g = *p + b.v, u = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + T::WN / 2) + b.w;
      f32x4 h4;
#pragma unroll
      for (int e = 0; e < 4; ++e) h4[e] = n + e < hidden ? act_only<NPH == 3>(act, g[e]) * u[e] : 0.f;
      store_planes<ELEM, NPH>(h + (int64_t)m * hidden_p + n, h_plane, h4);
      if (gu) {
        float* o = gu + (int64_t)m * 2 * hidden_p + n;
        *reinterpret_cast<f32x4*>(o) = g;
        *reinterpret_cast<f32x4*>(o + hidden_p) = u;
      }
    });
  }
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int, int, const Four&, int, int) const {}
};

// acc = dh: dg = dh u act'(g), du = dh act(g) as operand planes side by side (rows of 2 hidden_p, padding zero), and, for the
// bias gradient, their fp32 column sums over this wave's rows
struct ColumnSums {
  f32x4 g, u;
};
template <int ELEM, int NPD>
struct GateBwdEpi {
  static constexpr bool PAIR = false;
  using State = ColumnSums;
  int act, hidden, hidden_p;
  const float* gu;
  u16* d;  // (rows, 2 hidden_p)
  int64_t d_plane;
  float* partial;  // (tiles_m * WAVES_M, 2 hidden_p) or NULL
  template <class T>
  __device__ __forceinline__ ColumnSums begin(int, int) const { return ColumnSums{}; }
  template <class T>
  __device__ __forceinline__ void emit(const Args& a, float* buf, int m0, int n0, int lane, ColumnSums& s, int, int) const {
    each_piece<T, T::WN>(buf, lane, [&](int r, int c, const f32x4* p) {
      const int m = m0 + r, n = n0 + c;
      if (m >= a.M || n >= hidden_p) return;
      const float* o = gu + (int64_t)m * 2 * hidden_p + n;
      const f32x4 g = *reinterpret_cast<const f32x4*>(o), u = *reinterpret_cast<const f32x4*>(o + hidden_p), dh = *p;
      f32x4 dg, du;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float av, dav;
        act_both<NPD == 3>(act, g[e], av, dav);
        const bool in = n + e < hidden;
        dg[e] = in ? dh[e] * u[e] * dav : 0.f;
        du[e] = in ? dh[e] * av : 0.f;
      }
      u16* q = d + (int64_t)m * 2 * hidden_p + n;
      store_planes<ELEM, NPD>(q, d_plane, dg);
      store_planes<ELEM, NPD>(q + hidden_p, d_plane, du);
      s.g += dg;
      s.u += du;
    });
  }
  // a lane has seen the same four columns in every row it took: lanes a row's length apart hold the other rows
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int n0, int lane, ColumnSums& s, int tm, int wm) const {
    if (!partial) return;
    constexpr int P = T::WN / 4;
    static_assert(P < 64 && 64 % P == 0, "columns of a wave");
#pragma unroll
    for (int k = P; k < 64; k *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s.g[e] += __shfl_xor(s.g[e], k);
        s.u[e] += __shfl_xor(s.u[e], k);
      }
    const int n = n0 + lane * 4;
    if (lane < P && n < hidden_p) {
      float* o = partial + (int64_t)(tm * T::WAVES_M + wm) * 2 * hidden_p + n;
      *reinterpret_cast<f32x4*>(o) = s.g;
      *reinterpret_cast<f32x4*>(o + hidden_p) = s.u;
    }
  }
};

// C (+ bias + residual) in the tensors' type.  Rows from gap_at on belong gap rows further up (the padding behind each half of
// [dg | du]^T x); the padding rows are not stored.
struct OutEpi {
  static constexpr bool PAIR = false;
  using State = Four;  // the bias of this lane's columns
  void* out;
  int64_t ld;
  int dtype;
  const void* bias;
  const void* res;
  int64_t ld_res;
  int rows, gap_at, gap, cols;
  int vec;  // rows of out are aligned for four elements at a time
  __device__ __forceinline__ f32x4 bias_at(int n) const { return bias && n < cols ? load4(bias, n, cols - n, dtype) : f32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void put(int m, int n, f32x4 v, f32x4 b) const {
    if (m >= gap_at) {
      if (m < gap_at + gap) return;
      m -= gap;
    }
    if (m >= rows || n >= cols) return;
    const int left = cols - n;
    v += b;
    if (res) v += load4(res, (int64_t)m * ld_res + n, left, dtype);
    store4(out, (int64_t)m * ld + n, dtype, v, left, vec);
  }
  template <class T>
  __device__ __forceinline__ Four begin(int n0, int lane) const {
    static_assert(64 % (T::WN / 4) == 0, "a lane keeps its columns");
    return Four{bias_at(n0 + lane % (T::WN / 4) * 4), {}};
  }
  template <class T>
  __device__ __forceinline__ void emit(const Args&, float* buf, int m0, int n0, int lane, const Four& b, int, int) const {
    each_piece<T, T::WN>(buf, lane, [&](int r, int c, const f32x4* p) { put(m0 + r, n0 + c, *p, b.v); });
  }
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int, int, const Four&, int, int) const {}
};

// fp32 partial sums of a product split along K: (splits, M, Np), Np = N rounded up to 4
struct PartialEpi {
  static constexpr bool PAIR = false;
  using State = NoState;
  float* partial;
  int Np;
  template <class T>
  __device__ __forceinline__ NoState begin(int, int) const { return {}; }
  template <class T>
  __device__ __forceinline__ void emit(const Args& a, float* buf, int m0, int n0, int lane, NoState&, int, int) const {
    float* base = partial + (int64_t)a.split * a.M * Np;
    each_piece<T, T::WN>(buf, lane, [&](int r, int c, const f32x4* p) {
      const int m = m0 + r, n = n0 + c;
      if (m < a.M && n < a.N) *reinterpret_cast<f32x4*>(base + (int64_t)m * Np + n) = *p;
    });
  }
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int, int, NoState&, int, int) const {}
};

// column sums in two passes with a fixed order.  First: shares of rows_per rows of a (rows, cols) tensor, eight rows' loads in flight
// per thread.
struct ColumnShares {
  const void* src;
  int64_t ld;
  int rows, cols, rows_per, blocks_n;  // blocks_n: 64 columns each
  float* partial;
  int blocks = 0;
};
template <int DT>
__device__ __forceinline__ void column_share(const ColumnShares& j, int block, float (*red)[64]) {
  const int c = block % j.blocks_n * 64 + (threadIdx.x & 63), share = block / j.blocks_n, w = threadIdx.x >> 6;
  const int r1 = min(j.rows, (share + 1) * j.rows_per);
  float s = 0.f;
  if (c < j.cols)
    for (int r = share * j.rows_per + w; r < r1; r += 32) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = r + 4 * k < r1 ? load_as(j.src, (int64_t)(r + 4 * k) * j.ld + c, DT) : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  red[w][threadIdx.x & 63] = s;
  __syncthreads();
  if (w == 0 && c < j.cols)
    j.partial[(int64_t)share * j.cols + c] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}
template <int DT>
static __global__ __launch_bounds__(256) void column_shares_kernel(const ColumnShares j) {
  __shared__ float red[4][64];
  column_share<DT>(j, blockIdx.x, red);
}

// What is left to do once the products of a pass are done, in one launch: joining products split along K (partial sums in the
// order of the splits, then the output's epilogue) and the second passes of column sums (partial rows in a fixed order; columns from
// gap_at on are read gap further right).
struct FinishJob {
  const float* partial;
  int n, ld;         // splits / partial rows; floats of a row
  int M;             // rows of the output (0: a column sum)
  int cols, gap_at, gap;
  OutEpi out;        // its tensor is the column sums' output too
  int first, blocks; // workgroups
};
struct Finish {
  FinishJob job[5];
  int n = 0, blocks = 0;
  void add(const FinishJob& j, int64_t blocks_of_job) {
    job[n] = j;
    job[n].first = blocks;
    job[n].blocks = (int)blocks_of_job;
    blocks += job[n].blocks;
    ++n;
  }
};
static __global__ __launch_bounds__(256) void finish_kernel(const Finish f) {
  int k = 0;
  while (k + 1 < f.n && (int)blockIdx.x >= f.job[k + 1].first) ++k;
  const FinishJob& j = f.job[k];
  const int block = blockIdx.x - j.first;
  if (j.M) {
    const int64_t per = j.ld / 4, total = (int64_t)j.M * per, stride = (int64_t)j.M * j.ld;
    for (int64_t t = (int64_t)block * 256 + threadIdx.x; t < total; t += (int64_t)j.blocks * 256) {
      f32x4 s = {0, 0, 0, 0};
#pragma unroll 4
      for (int z = 0; z < j.n; ++z) s += *reinterpret_cast<const f32x4*>(j.partial + z * stride + t * 4);
      const int n = (int)(t % per) * 4;
      j.out.put((int)(t / per), n, s, j.out.bias_at(n));
    }
    return;
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = block * 64 + lane;
  __shared__ float red[4][64];
  float s = 0.f;
  if (c < j.cols) {
    const float* p = j.partial + c + (c >= j.gap_at ? j.gap : 0);
#pragma unroll 8
    for (int r = w; r < j.n; r += 4) s += p[(int64_t)r * j.ld];
  }
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && c < j.cols) store_as(j.out.out, c, j.out.dtype, (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
}
inline void run_finish(const Finish& f, hipStream_t s) {
  if (f.n) hipLaunchKernelGGL(finish_kernel, dim3(f.blocks), dim3(256), 0, s, f);
}
inline void add_column_sums(Finish& f, const float* partial, int n, int ld, int cols, int gap_at, int gap, void* out, int dtype) {
  FinishJob j{};
  j.partial = partial, j.n = n, j.ld = ld, j.cols = cols, j.gap_at = gap_at, j.gap = gap;
  j.out.out = out, j.out.dtype = dtype;
  f.add(j, (cols + 63) / 64);
}

// ---------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------
inline int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }
inline int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }
inline int esize(int dtype) { return dtype == CRADLE_F32 ? 4 : 2; }

constexpr int kFewRows = 8;   // (few_rows)
constexpr int kCUs = 256;

// Below this many products per projection (2^28: under 2 us of the matrix cores) a block's time is its launches, and the second
// plane of h and [dg | du] costs nothing that shows; above, it would cost a third of the forward and most of the backward pass again.
constexpr int64_t kSmallWork = 1LL << 28;

struct Plan {
  int M, K, F, O;
  int Fp;                // row length of h and of each half of [dg | du]
  int dtype, elem, npl;  // planes of the tensors' operands
  int nph;               // planes of h and [dg | du]: twice a 16-bit tensor's bits while that is free
};

// A K tile's share of a row, in elements: rows that start on a multiple of it are staged in whole cache lines (three planes: half
// lines).  1537 x 5462 x 1000 on one plane: 40.5 us with rows of 1000, 32.5 us with rows of 1024; 2560 x 1600 x 400 on three: 28.6
// and 25.8 us.
inline int line_of(int planes) { return planes == 3 ? 32 : 64; }
// Rows that a 16-bit operand with other rows meets in a product along its own ones, from which on it is packed into such rows: a
// fifth of 2 rows cols other / 600 TFLOP/s is then more than the packing's 4 rows cols bytes at 5 TB/s.
constexpr int kManyRows = 2048;

inline Plan plan_of(const cradle_gated_mlp_desc* d) {
  Plan p;
  p.M = d->rows;
  p.K = d->width;
  p.F = d->hidden;
  p.O = d->out_width;
  p.dtype = d->dtype;
  p.elem = d->dtype == CRADLE_F16 ? F16 : BF16;
  p.npl = d->dtype == CRADLE_F32 ? 3 : 1;
  const int run = line_of(p.npl);
  // (the padding is multiplied too: at most a 16th; a 16-bit W_in that a gap would have to be packed for stays as it is for few rows)
  const bool packs = p.npl == 3 || p.F % 8 != 0 || p.M >= kManyRows;
  p.Fp = packs && p.F >= 16 * run ? (p.F + run - 1) / run * run : (int)up8(p.F);
  p.nph = p.npl == 1 && (int64_t)p.M * p.F * (p.K + p.O) < kSmallWork ? 2 : p.npl;
  return p;
}

// a 16-bit tensor whose rows can be staged as they lie in memory
inline bool direct(const void* p, int64_t ld, int cols, int dtype) {
  return dtype != CRADLE_F32 && cols % 8 == 0 && ld % 8 == 0 && ((uintptr_t)p & 15) == 0;
}

struct Bump {
  char* base;
  int64_t off = 0;
  void* take(int64_t bytes) {
    void* r = base ? base + off : nullptr;
    off += align256(bytes);
    return r;
  }
};

// operand of tensor `src` (rows x cols): itself, or packed into the workspace (a job is queued)
// with rows_dst rows, gap of them between the two halves.  other: rows it meets in a product along its own rows (0: none such).
inline Operand operand(const Plan& p, const void* src, int64_t ld, int rows, int cols, int rows_dst, int gap_at, int gap, int other, Bump& ws,
                       PackJobs& js, int& n_jobs) {
  const int run = line_of(p.npl);
  if (direct(src, ld, cols, p.dtype) && gap == 0 && (ld % run == 0 || other < kManyRows)) return {static_cast<const u16*>(src), ld, 0, 0};
  const int64_t ldp = (cols + run - 1) / run * run, plane = (int64_t)rows_dst * ldp;
  u16* dst = static_cast<u16*>(ws.take(plane * p.npl * 2));
  js.job[n_jobs++] = {src, dst, ld, plane, rows, cols, rows_dst, (int)ldp, gap_at, gap,
                      ld % (p.npl == 3 ? 4 : 8) == 0 && ((uintptr_t)src & 15) == 0};
  return {dst, ldp, plane, 0};
}

template <int ELEM, int NPL>
void run_pack(const Plan& p, PackJobs& js, int n_jobs, hipStream_t s) {
  if (!n_jobs) return;
  int64_t most = 0;
  for (int i = 0; i < n_jobs; ++i) {
    const int64_t t = (int64_t)js.job[i].rows_dst * (js.job[i].ld_dst / 8);
    most = t > most ? t : most;
  }
  const int64_t blocks = (most + 255) / 256;
  const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096), (unsigned)n_jobs);
  hipLaunchKernelGGL((pack_kernel<ELEM, NPL>), grid, dim3(256), 0, s, js);
}

// Two tiles per operand format.  Large: 256 x 256 (more than one plane: 256 x 128, to fit the LDS), eight waves, one workgroup per
// CU.  Small: 128 x 128 (more than one plane: 128 x 64), four waves, two workgroups per CU.
template <int ELEM, int NPA, int NPB, bool AK, bool BK>
struct Tiles {
  static constexpr bool ONE = NPA == 1 && NPB == 1, THREE = NPA == 3;
  using Large = Tile<ELEM, NPA, NPB, 256, ONE ? 256 : 128, ONE ? 64 : 32, ONE || THREE ? 2 : 3, ONE ? 2 : 4, ONE ? 4 : 2, AK, BK>;
  using Small = Tile<ELEM, NPA, NPB, 128, ONE ? 128 : 64, THREE ? 32 : 64, 2, ONE ? 2 : 4, ONE ? 2 : 1, AK, BK>;
};

template <class T, class Epi>
void launch(Args a, const Epi& epi, int cols, int splits, hipStream_t s) {
  a.tiles_m = (a.M + T::BM - 1) / T::BM;
  const int bn = Epi::PAIR ? T::BN / 2 : T::BN;
  a.tiles_n = (cols + bn - 1) / bn;
  const int k_tiles = (a.K + T::BK - 1) / T::BK;
  a.k_tiles_per_split = (k_tiles + splits - 1) / splits;
  a.symmetric = 0;
  hipLaunchKernelGGL((product_kernel<T, Epi>), dim3((unsigned)(a.tiles_m * a.tiles_n), 1, (unsigned)splits), dim3(T::NT), 0, s, a, epi);
}

template <class T>
int64_t tiles(const Args& a, int cols, bool pair) {
  const int bn = pair ? T::BN / 2 : T::BN;
  return (int64_t)((a.M + T::BM - 1) / T::BM) * ((cols + bn - 1) / bn);
}

// Time of a product on tiles of one size: the CUs with the most tiles finish last, a large tile's rate is 1.2 times a small
// one's (measured on 8192 x 10240 x 4096 in bf16: 1290 and 1090 TFLOP/s).
template <class L, class S>
bool use_large(const Args& a, int cols, bool pair) {
  const int64_t l = (tiles<L>(a, cols, pair) + kCUs - 1) / kCUs * L::BM * L::BN, s = (tiles<S>(a, cols, pair) + kCUs - 1) / kCUs * S::BM * S::BN;
  return l * 5 <= s * 6;
}

template <int ELEM, int NPA, int NPB, bool AK, bool BK, class Epi>
void product(const Args& a, const Epi& epi, int cols, hipStream_t s) {
  using TT = Tiles<ELEM, NPA, NPB, AK, BK>;
  if (use_large<typename TT::Large, typename TT::Small>(a, cols, Epi::PAIR)) launch<typename TT::Large>(a, epi, cols, 1, s);
  else launch<typename TT::Small>(a, epi, cols, 1, s);
}

// A product whose output has too few small tiles for the chip (two per CU at a time) is split along K, into shares of at
// least four K tiles; its partial sums cost a pass over them.  Forward pass, whole and split: 512 rows, 512 x 1024 in fp32 54 and 40 us;
// 2560 rows, 400 x 800 in fp32 66 and 62; 1537 rows, 1000 x 2731 in fp16 87 and 76; 4096 rows, 512 x 1024 in bf16 38 and 40.
template <int ELEM, int NPA, int NPB, bool AK, bool BK>
int splits_of(const Args& a) {
  using TT = Tiles<ELEM, NPA, NPB, AK, BK>;
  const int64_t t = tiles<typename TT::Small>(a, a.N, false);
  const int k_tiles = (a.K + TT::Small::BK - 1) / TT::Small::BK;
  const int64_t want = 2 * kCUs / t, most = k_tiles / 4;
  if (t >= kCUs || want < 2 || most < 2) return 1;
  return (int)(want < most ? want : most);
}

// A product's result into its tensor, or, split along K, into partial sums (splits, M, Np) that `finish` joins.
struct EitherEpi {
  static constexpr bool PAIR = false;
  using State = Four;
  OutEpi out;
  PartialEpi partial;
  template <class T>
  __device__ __forceinline__ Four begin(int n0, int lane) const { return out.begin<T>(n0, lane); }
  template <class T>
  __device__ __forceinline__ void emit(const Args& a, float* buf, int m0, int n0, int lane, const Four& b, int tm, int tn) const {
    NoState none;
    if (partial.partial) partial.emit<T>(a, buf, m0, n0, lane, none, tm, tn);
    else out.emit<T>(a, buf, m0, n0, lane, b, tm, tn);
  }
  template <class T>
  __device__ __forceinline__ void finish(const Args&, int, int, const Four&, int, int) const {}
};

// Independent products of small tiles in one launch, of up to three types of tiles: the backward pass's last three.  Each alone
// fills the chip about once, with a start and an end at which much of it waits: 2560 rows, 400 x 800 in fp32 81 us in three
// launches, 67 in one; 1537 rows, 1000 x 2731 in fp16 82 and 67.
struct Products {
  Args a[3];
  EitherEpi e[3];
  int tiles[3] = {0, 0, 0}, first[3] = {0, 0, 0}, blocks = 0;
  ColumnShares sums{};  // ride along behind them
};
template <class T0, class T1, class T2>
__global__ __launch_bounds__(256, 2) void products_kernel(const Products p) {
#ifdef __HIP_DEVICE_COMPILE__
  static_assert(T0::NT == 256 && T1::NT == 256 && T2::NT == 256 && T0::STAGES == 2 && T1::STAGES == 2 && T2::STAGES == 2, "small tiles");
  constexpr int A = T0::STAGE > T1::STAGE ? T0::STAGE : T1::STAGE, STAGE = A > T2::STAGE ? A : T2::STAGE;
  __shared__ u32x4 st0[STAGE];
  __shared__ u32x4 st1[STAGE];
  if ((int)blockIdx.x >= p.blocks) {
    constexpr int DT = T0::NPB == 3 ? CRADLE_F32 : T0::ELEM == BF16 ? CRADLE_BF16 : CRADLE_F16;
    return column_share<DT>(p.sums, blockIdx.x - p.blocks, reinterpret_cast<float(*)[64]>(st0));
  }
  const int k = (int)blockIdx.x >= p.first[2] ? 2 : (int)blockIdx.x >= p.first[1] ? 1 : 0, block = blockIdx.x - p.first[k];
  Args a = p.a[k];
  a.split = block / p.tiles[k];
  const int wg = block % p.tiles[k];
  if (k == 0) {
    product_body<T0, EitherEpi>(a, p.e[0], wg, p.tiles[0], st0, st1, nullptr, nullptr);
  } else if constexpr (std::is_same_v<T1, T2>) {
    product_body<T1, EitherEpi>(a, p.e[k], wg, p.tiles[k], st0, st1, nullptr, nullptr);
  } else if (k == 1) {
    product_body<T1, EitherEpi>(a, p.e[1], wg, p.tiles[1], st0, st1, nullptr, nullptr);
  } else {
    product_body<T2, EitherEpi>(a, p.e[2], wg, p.tiles[2], st0, st1, nullptr, nullptr);
  }
#endif
}

// shares that a split along K comes to (every share has work), and the joining of their sums
template <class T>
int shares_of(Args& a, int splits) {
  const int k_tiles = (a.K + T::BK - 1) / T::BK;
  a.k_tiles_per_split = (k_tiles + splits - 1) / splits;
  return (k_tiles + a.k_tiles_per_split - 1) / a.k_tiles_per_split;
}
inline PartialEpi split_product(const Args& a, const OutEpi& epi, float* partial, int shares, Finish& finish) {
  FinishJob j{};
  j.partial = partial, j.n = shares, j.ld = (a.N + 3) & ~3, j.M = a.M, j.out = epi;
  const int64_t blocks = ((int64_t)a.M * (j.ld / 4) + 255) / 256;
  finish.add(j, blocks < 1024 ? blocks : 1024);
  return PartialEpi{partial, j.ld};
}

// A product into its tensor
template <int ELEM, int NPA, int NPB, bool AK, bool BK>
void product_out(Args a, const OutEpi& epi, float* partial, Finish& finish, hipStream_t s) {
  const int splits = splits_of<ELEM, NPA, NPB, AK, BK>(a);
  if (splits == 1) return product<ELEM, NPA, NPB, AK, BK>(a, epi, a.N, s);
  using Small = typename Tiles<ELEM, NPA, NPB, AK, BK>::Small;
  const int shares = shares_of<Small>(a, splits);
  launch<Small>(a, split_product(a, epi, partial, shares, finish), a.N, shares, s);
}
// the same, at once with large tiles (splits == 0), else as the k-th of `ps`
template <int ELEM, int NPA, int NPB, bool AK, bool BK>
void product_out(Args a, const OutEpi& epi, int splits, float* partial, Products& ps, int k, Finish& finish, hipStream_t s) {
  using TT = Tiles<ELEM, NPA, NPB, AK, BK>;
  using Small = typename TT::Small;
  if (!splits) return launch<typename TT::Large>(a, epi, a.N, 1, s);
  const int shares = shares_of<Small>(a, splits);
  a.tiles_m = (a.M + Small::BM - 1) / Small::BM;
  a.tiles_n = (a.N + Small::BN - 1) / Small::BN;
  a.symmetric = 0;
  ps.a[k] = a;
  ps.e[k] = EitherEpi{epi, splits > 1 ? split_product(a, epi, partial, shares, finish) : PartialEpi{}};
  ps.tiles[k] = a.tiles_m * a.tiles_n;
  ps.blocks += ps.tiles[k] * shares;
}
template <class T0, class T1, class T2>
void run_products(const Products& p, hipStream_t s) {
  if (p.blocks) hipLaunchKernelGGL((products_kernel<T0, T1, T2>), dim3((unsigned)(p.blocks + p.sums.blocks)), dim3(256), 0, s, p);
}

inline int64_t partial_floats(const Args& a, int splits) { return splits < 2 ? 0 : (int64_t)splits * a.M * ((a.N + 3) & ~3); }

// Splits along K of products that share a launch: shares of about equal length, 0.7 of what each of the 2 kCUs places gets in
// all -- shorter ones cost more partial sums, longer ones leave places idle at the end (both passes of 8192 rows, 512 x 1024 in fp32
// with 0.5 556 us, 0.7 536, 1.4 616; 4096 rows in bf16 126, 125, 118).  0: large tiles are faster.
struct Splits {
  double work = 0;  // K tiles of all small tiles
  template <int ELEM, int NPA, int NPB, bool AK, bool BK>
  int of(const Args& a) const {
    using TT = Tiles<ELEM, NPA, NPB, AK, BK>;
    if (use_large<typename TT::Large, typename TT::Small>(a, a.N, false)) return 0;
    const int k_tiles = (a.K + TT::Small::BK - 1) / TT::Small::BK, most = k_tiles / 4;
    const int n = (int)(k_tiles * (2 * kCUs / 0.7) / work + 0.5);
    return n < 1 || most < 1 ? 1 : n < most ? n : most;
  }
  template <int ELEM, int NPA, int NPB, bool AK, bool BK>
  void add(const Args& a) {
    using TT = Tiles<ELEM, NPA, NPB, AK, BK>;
    if (use_large<typename TT::Large, typename TT::Small>(a, a.N, false)) return;
    work += (double)tiles<typename TT::Small>(a, a.N, false) * ((a.K + TT::Small::BK - 1) / TT::Small::BK);
  }
};

inline int vec_ok(const void* p, int64_t ld, int dtype) { return ld % 4 == 0 && ((uintptr_t)p & (dtype == CRADLE_F32 ? 15 : 7)) == 0; }
constexpr int kNoGap = 0x7fffffff;

inline Args args_of(const Operand& A, const Operand& B, int M, int N, int K) {
  Args a{};
  a.A = A, a.B = B, a.M = M, a.N = N, a.K = K;
  return a;
}

// ---- forward: workspace = packed x, W_in, W_out | h when it is not saved | partial sums
template <int ELEM, int NPL, int NPH>
int64_t forward(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  Bump ws{static_cast<char*>(workspace)};
  PackJobs js{};
  int n = 0;
  const int gap = p.Fp - p.F;
  const Operand x = operand(p, d->x, d->ld_x, p.M, p.K, p.M, kNoGap, 0, 2 * p.F, ws, js, n);
  const Operand w_in = operand(p, d->w_in, d->ld_w_in, 2 * p.F, p.K, 2 * p.Fp, p.F, gap, p.M, ws, js, n);
  const Operand w_out = operand(p, d->w_out, d->ld_w_out, p.O, p.F, p.O, kNoGap, 0, p.M, ws, js, n);
  const int64_t h_plane = (int64_t)p.M * p.Fp;
  // (the inner extent is F: of h's padding and of a directly staged W_out's neighbours nothing is multiplied)
  const Args out_args = args_of({}, w_out, p.M, p.O, p.F);
  u16* h = static_cast<u16*>(d->saved_h ? d->saved_h : ws.take(h_plane * NPH * 2));
  float* partial = static_cast<float*>(ws.take(partial_floats(out_args, splits_of<ELEM, NPH, NPL, true, true>(out_args)) * 4));
  if (!run) return ws.off;
  run_pack<ELEM, NPL>(p, js, n, s);
  Args a = args_of(x, w_in, p.M, p.F, p.K);
  a.up_row = p.Fp;
  product<ELEM, NPL, NPL, true, true>(
      a, GateEpi<ELEM, NPH>{d->act, p.F, p.Fp, p.dtype, d->b_in, h, h_plane, static_cast<float*>(d->saved_gu)}, p.F, s);
  const Operand hop{h, p.Fp, h_plane, 0};
  Finish finish;
  product_out<ELEM, NPH, NPL, true, true>(
      args_of(hop, w_out, p.M, p.O, p.F),
      OutEpi{d->y, d->ld_y, p.dtype, d->b_out, d->residual, d->ld_residual, p.M, kNoGap, 0, p.O, vec_ok(d->y, d->ld_y, p.dtype)}, partial, finish, s);
  run_finish(finish, s);
  return ws.off;
}

constexpr int kColsumRows = 64;  // rows per first-pass share of a column sum, more when there are more than 512 shares
inline int colsum_rows(int rows) {
  const int most = (rows + 511) / 512;
  return most > kColsumRows ? most : kColsumRows;
}

// ---- backward: workspace = packed x, W_in, W_out, dy | [dg | du] | partial sums of dx, dW_in, dW_out | of the column sums
template <int ELEM, int NPL, int NPH>
int64_t backward(const cradle_gated_mlp_desc* d, const Plan& p, void* workspace, hipStream_t s, bool run) {
  Bump ws{static_cast<char*>(workspace)};
  PackJobs js{};
  int n = 0;
  const int gap = p.Fp - p.F;
  const Operand x = operand(p, d->x, d->ld_x, p.M, p.K, p.M, kNoGap, 0, 0, ws, js, n);
  const Operand w_in = operand(p, d->w_in, d->ld_w_in, 2 * p.F, p.K, 2 * p.Fp, p.F, gap, 0, ws, js, n);
  const Operand w_out = operand(p, d->w_out, d->ld_w_out, p.O, p.F, p.O, kNoGap, 0, 0, ws, js, n);
  const Operand dy = operand(p, d->dy, d->ld_dy, p.M, p.O, p.M, kNoGap, 0, p.F, ws, js, n);
  const int64_t h_plane = (int64_t)p.M * p.Fp, d_plane = 2 * h_plane;
  u16* dgu = static_cast<u16*>(ws.take(d_plane * NPH * 2));
  const Operand dop{dgu, 2 * (int64_t)p.Fp, d_plane, 0};
  const Operand hop{static_cast<const u16*>(d->saved_h), p.Fp, h_plane, 0};
  const Args dx = args_of(dop, w_in, p.M, p.K, 2 * p.Fp), dw_in = args_of(dop, x, 2 * p.Fp, p.K, p.M), dw_out = args_of(dy, hop, p.O, p.F, p.M);
  Splits sp;
  if (d->dx) sp.add<ELEM, NPH, NPL, true, false>(dx);
  if (d->dw_in) sp.add<ELEM, NPH, NPL, false, false>(dw_in);
  if (d->dw_out) sp.add<ELEM, NPL, NPH, false, false>(dw_out);
  const int n_dx = d->dx ? sp.of<ELEM, NPH, NPL, true, false>(dx) : 0, n_in = d->dw_in ? sp.of<ELEM, NPH, NPL, false, false>(dw_in) : 0,
            n_out = d->dw_out ? sp.of<ELEM, NPL, NPH, false, false>(dw_out) : 0;
  float* p_dx = static_cast<float*>(ws.take(partial_floats(dx, n_dx) * 4));
  float* p_in = static_cast<float*>(ws.take(partial_floats(dw_in, n_in) * 4));
  float* p_out = static_cast<float*>(ws.take(partial_floats(dw_out, n_out) * 4));
  const int sum_rows = (p.M + 127) / 128 * 4;  // of either tile size: 128 rows are at most four wave rows
  float* sums = static_cast<float*>(ws.take(d->db_in ? (int64_t)sum_rows * 2 * p.Fp * 4 : 0));
  const int per = colsum_rows(p.M), shares = (p.M + per - 1) / per;
  float* sums_out = static_cast<float*>(ws.take(d->db_out ? (int64_t)shares * p.O * 4 : 0));
  if (!run) return ws.off;
  run_pack<ELEM, NPL>(p, js, n, s);

  Args a = args_of(dy, w_out, p.M, p.F, p.O);
  using TT = Tiles<ELEM, NPL, NPL, true, false>;
  const bool large = use_large<typename TT::Large, typename TT::Small>(a, p.F, false);
  product<ELEM, NPL, NPL, true, false>(
      a, GateBwdEpi<ELEM, NPH>{d->act, p.F, p.Fp, static_cast<const float*>(d->saved_gu), dgu, d_plane, d->db_in ? sums : nullptr}, p.F, s);
  Finish finish;
  if (d->db_in) {
    const int used = large ? (p.M + 255) / 256 * TT::Large::WAVES_M : (p.M + 127) / 128 * TT::Small::WAVES_M;
    add_column_sums(finish, sums, used, 2 * p.Fp, 2 * p.F, p.F, gap, d->db_in, p.dtype);
  }
  ColumnShares db_out{d->dy, d->ld_dy, p.M, p.O, per, (p.O + 63) / 64, sums_out};
  if (d->db_out) {
    db_out.blocks = db_out.blocks_n * shares;
    add_column_sums(finish, sums_out, shares, p.O, p.O, kNoGap, 0, d->db_out, p.dtype);
  }
  auto out = [&](void* q, int64_t ld, int rows, int gap_at, int g, int cols) {
    return OutEpi{q, ld, p.dtype, nullptr, nullptr, 0, rows, gap_at, g, cols, vec_ok(q, ld, p.dtype)};
  };
  Products ps;
  if (d->dx) product_out<ELEM, NPH, NPL, true, false>(dx, out(d->dx, d->ld_dx, p.M, kNoGap, 0, p.K), n_dx, p_dx, ps, 0, finish, s);
  ps.first[1] = ps.blocks;
  if (d->dw_in) product_out<ELEM, NPH, NPL, false, false>(dw_in, out(d->dw_in, p.K, 2 * p.F, p.F, gap, p.K), n_in, p_in, ps, 1, finish, s);
  ps.first[2] = ps.blocks;
  if (d->dw_out) product_out<ELEM, NPL, NPH, false, false>(dw_out, out(d->dw_out, p.F, p.O, kNoGap, 0, p.F), n_out, p_out, ps, 2, finish, s);
  ps.sums = db_out;
  if (!ps.blocks && db_out.blocks) {
    constexpr int DT = NPL == 3 ? CRADLE_F32 : ELEM == BF16 ? CRADLE_BF16 : CRADLE_F16;
    hipLaunchKernelGGL(column_shares_kernel<DT>, dim3((unsigned)db_out.blocks), dim3(256), 0, s, db_out);
  }
  run_products<typename Tiles<ELEM, NPH, NPL, true, false>::Small, typename Tiles<ELEM, NPH, NPL, false, false>::Small,
               typename Tiles<ELEM, NPL, NPH, false, false>::Small>(ps, s);
  run_finish(finish, s);
  return ws.off;
}

// Both passes per type, each in a source of its own (gated_mlp_{f32,bf16,f16}.hip).  run = false: only the workspace is sized.
int64_t forward_f32(const cradle_gated_mlp_desc*, const Plan&, void* workspace, hipStream_t, bool run);
int64_t forward_bf16(const cradle_gated_mlp_desc*, const Plan&, void* workspace, hipStream_t, bool run);
int64_t forward_f16(const cradle_gated_mlp_desc*, const Plan&, void* workspace, hipStream_t, bool run);
int64_t backward_f32(const cradle_gated_mlp_desc*, const Plan&, void* workspace, hipStream_t, bool run);
int64_t backward_bf16(const cradle_gated_mlp_desc*, const Plan&, void* workspace, hipStream_t, bool run);
int64_t backward_f16(const cradle_gated_mlp_desc*, const Plan&, void* workspace, hipStream_t, bool run);

}  // namespace gated
}  // namespace cradle
