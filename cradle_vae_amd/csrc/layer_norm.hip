// Layer norm over the last axis and its backward pass.
//   y  = xh w + b,  xh = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy w;   dw = sum over rows of dy xh,  db = sum over rows of dy
// Memory bound: x once in and y once out; x and dy in and dx out.  So a row lives in the registers of the threads that share
// it (one wave up to 1024 elements, a workgroup above), the mean and then the centred square sum are taken from there -- the
// second moment about the mean, not E[x^2] - mean^2, which cancels for rows far from zero -- and every element is moved once, in
// 16-byte pieces where the rows allow.  w and b stay in registers over all rows of a workgroup.
// dw and db: a thread owns the same columns in every row it sees, so they accumulate in its registers (fp32); the workgroups'
// partial rows are joined by a second launch in a fixed order.  Measured in bf16 on 32768 x 4096: 266 us for forward and
// backward together, 5.0 TB/s (a large copy reaches 5.25); alone, forward 102 us, backward 169 + 7 us.
#include "common.h"

namespace cradle {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ float widen(uint16_t b) {
  return DT == CRADLE_BF16 ? __builtin_bit_cast(float, (uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
}
template <int DT>
__device__ __forceinline__ uint16_t narrow(float v) {
  return DT == CRADLE_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (DT == CRADLE_F32) return static_cast<const float*>(p)[i];
  else return widen<DT>(static_cast<const uint16_t*>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (DT == CRADLE_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = narrow<DT>(v);
}

// The columns of one thread: NCH chunks of eight.  VEC: chunk c holds columns 8 (c TPR + t) ..+7 (16-byte pieces); otherwise
// element e of chunk c is column (8 c + e) TPR + t, so that a wave's loads are still consecutive.
template <int TPR, int NCH, bool VEC>
struct Cols {
  int t, width;
  __device__ __forceinline__ int col(int c, int e) const { return VEC ? 8 * (c * TPR + t) + e : (8 * c + e) * TPR + t; }
  __device__ __forceinline__ bool in(int c, int e) const { return col(c, e) < width; }
  template <int DT>
  __device__ __forceinline__ void load(const void* p, int64_t row0, float (&v)[NCH][8], float other) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if constexpr (VEC) {
        const int k = col(c, 0);
        if (k < width) {  // (width % 8 == 0: a chunk is in or out)
          if constexpr (DT == CRADLE_F32) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + row0 + k);
            const f32x4 b = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + row0 + k + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][e] = a[e], v[c][4 + e] = b[e];
          } else {
            const u32x4 a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + row0 + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[c][2 * e] = widen<DT>((uint16_t)a[e]), v[c][2 * e + 1] = widen<DT>((uint16_t)(a[e] >> 16));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[c][e] = other;
        }
      } else {
        // (unconditional loads from a clamped column: behind a branch each of them would be waited for on its own)
        float t[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = load1<DT>(p, row0 + min(col(c, e), width - 1));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = in(c, e) ? t[e] : other;
      }
    }
  }
  template <int DT>
  __device__ __forceinline__ void store(void* p, int64_t row0, const float (&v)[NCH][8]) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if constexpr (VEC) {
        const int k = col(c, 0);
        if (k < width) {
          if constexpr (DT == CRADLE_F32) {
            float* q = static_cast<float*>(p) + row0 + k;
            *reinterpret_cast<f32x4*>(q) = f32x4{v[c][0], v[c][1], v[c][2], v[c][3]};
            *reinterpret_cast<f32x4*>(q + 4) = f32x4{v[c][4], v[c][5], v[c][6], v[c][7]};
          } else {
            u32x4 a;
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] = narrow<DT>(v[c][2 * e]) | (uint32_t)narrow<DT>(v[c][2 * e + 1]) << 16;
            *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + row0 + k) = a;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (in(c, e)) store1<DT>(p, row0 + col(c, e), v[c][e]);
      }
    }
  }
  // a parameter vector of the tensors' type or fp32
  template <int DT>
  __device__ __forceinline__ void load_param(const void* p, bool fp32, float (&v)[NCH][8], float none) const {
    if (!p) {
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = none;
    } else if (fp32) {
      load<CRADLE_F32>(p, 0, v, 0.f);
    } else {
      load<DT>(p, 0, v, 0.f);
    }
  }
};

// sums of two numbers over the TPR threads of a row; `turn` alternates between two LDS slots, so one barrier per sum is enough
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2 (*slots)[TPR / 64], int& turn) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (TPR == 64) {
    return make_float2(a, b);
  } else {
    float2* slot = slots[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    float2 t = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) t.x += slot[w].x, t.y += slot[w].y;
    return t;
  }
}

template <int TPR>
constexpr int threads() { return TPR == 64 ? 256 : TPR; }  // four rows per workgroup where a row is one wave

template <int DT, int TPR, int NCH, bool VEC>
__global__ __launch_bounds__(threads<TPR>()) void fwd_kernel(const void* __restrict__ x, int64_t ld_x, const void* __restrict__ w,
                                                             const void* __restrict__ b, int w_fp32, float eps,
                                                             void* __restrict__ y, int64_t ld_y, float* __restrict__ mean,
                                                             float* __restrict__ rstd, int64_t rows, int width) {
  constexpr int RPB = threads<TPR>() / TPR;
  __shared__ float2 slots[2][TPR / 64];
  int turn = 0;
  const Cols<TPR, NCH, VEC> cols{(int)(threadIdx.x % TPR), width};
  float wv[NCH][8], bv[NCH][8];
  cols.template load_param<DT>(w, w_fp32, wv, 1.f);
  cols.template load_param<DT>(b, w_fp32, bv, 0.f);
  const float inv = 1.f / (float)width;
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; r < rows; r += (int64_t)gridDim.x * RPB) {
    float v[NCH][8];
    cols.template load<DT>(x, r * ld_x, v, 0.f);
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[c][e];
    const float mu = row_sum2<TPR>(s, 0.f, slots, turn).x * inv;
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] -= mu;
        q += cols.in(c, e) ? v[c][e] * v[c][e] : 0.f;
      }
    const float rs = 1.f / sqrtf(row_sum2<TPR>(q, 0.f, slots, turn).x * inv + eps);
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = v[c][e] * rs * wv[c][e] + bv[c][e];
    cols.template store<DT>(y, r * ld_y, v);
    if (threadIdx.x % TPR == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

// partial: (gridDim.x, 2, width) sums of dy xh and dy over the rows of each workgroup, or NULL
template <int DT, int TPR, int NCH, bool VEC, bool PARAMS>
__global__ __launch_bounds__(threads<TPR>()) void bwd_kernel(const void* __restrict__ dy, int64_t ld_dy, const void* __restrict__ x,
                                                             int64_t ld_x, const void* __restrict__ w, int w_fp32,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             void* __restrict__ dx, int64_t ld_dx, float* __restrict__ partial,
                                                             int64_t rows, int width) {
  constexpr int RPB = threads<TPR>() / TPR;
  __shared__ float2 slots[2][TPR / 64];
  int turn = 0;
  const Cols<TPR, NCH, VEC> cols{(int)(threadIdx.x % TPR), width};
  float wv[NCH][8], sw[NCH][8], sb[NCH][8];
  cols.template load_param<DT>(w, w_fp32, wv, 1.f);
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[c][e] = sb[c][e] = 0.f;
  const float inv = 1.f / (float)width;
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; r < rows; r += (int64_t)gridDim.x * RPB) {
    float g[NCH][8], v[NCH][8];
    const float mu = mean[r], rs = rstd[r];
    cols.template load<DT>(x, r * ld_x, v, mu);  // (columns beyond the width: xh = 0)
    cols.template load<DT>(dy, r * ld_dy, g, 0.f);
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[c][e] = (v[c][e] - mu) * rs;
        if constexpr (PARAMS) {
          sw[c][e] += g[c][e] * v[c][e];
          sb[c][e] += g[c][e];
        }
        g[c][e] *= wv[c][e];
        s0 += g[c][e];
        s1 += g[c][e] * v[c][e];
      }
    if (dx) {
      const float2 s = row_sum2<TPR>(s0, s1, slots, turn);
      const float m0 = s.x * inv, m1 = s.y * inv;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) g[c][e] = (g[c][e] - m0 - v[c][e] * m1) * rs;
      cols.template store<DT>(dx, r * ld_dx, g);
    }
  }
  if (!PARAMS || !partial) return;
  float* out = partial + (int64_t)blockIdx.x * 2 * width;
  if constexpr (RPB == 1) {
    cols.template store<CRADLE_F32>(out, 0, sw);
    cols.template store<CRADLE_F32>(out, width, sb);
  } else {  // four waves share the columns: joined through LDS, the sums of one array at a time
    __shared__ float red[RPB][8 * NCH * TPR];
    const int wave = threadIdx.x / TPR;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k) __syncthreads();
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) red[wave][(8 * c + e) * TPR + cols.t] = k ? sb[c][e] : sw[c][e];
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * NCH * TPR; i += threads<TPR>()) {
        const int ce = i / TPR, t = i % TPR, c = ce / 8, e = ce % 8;
        const int col = VEC ? 8 * (c * TPR + t) + e : ce * TPR + t;
        if (col < width) out[k * width + col] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
      }
    }
  }
}

// The parameters' gradients alone, for rows too wide for one pass's registers: a thread owns eight columns (of 2048 per
// workgroup) over a share of the rows.  partial: (gridDim.y, 2, width)
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void params_kernel(const void* __restrict__ dy, int64_t ld_dy, const void* __restrict__ x, int64_t ld_x,
                                                     const float* __restrict__ mean, const float* __restrict__ rstd,
                                                     float* __restrict__ partial, int64_t rows, int width) {
  const int first = blockIdx.x * 2048;
  const Cols<256, 1, VEC> cols{(int)threadIdx.x, min(width - first, 2048)};
  float sw[1][8] = {}, sb[1][8] = {};
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    float g[1][8], v[1][8];
    const float mu = mean[r], rs = rstd[r];
    cols.template load<DT>(x, r * ld_x + first, v, mu);
    cols.template load<DT>(dy, r * ld_dy + first, g, 0.f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sw[0][e] += g[0][e] * ((v[0][e] - mu) * rs);
      sb[0][e] += g[0][e];
    }
  }
  cols.template store<CRADLE_F32>(partial, (int64_t)blockIdx.y * 2 * width + first, sw);
  cols.template store<CRADLE_F32>(partial, ((int64_t)blockIdx.y * 2 + 1) * width + first, sb);
}

// sums n partial rows of 2 * width floats: sixteen waves take every sixteenth row of 64 columns, joined in wave order
__global__ __launch_bounds__(1024) void join_kernel(const float* __restrict__ partial, int n, int width, void* __restrict__ dw,
                                                    void* __restrict__ db, int dtype) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < 2 * width) {
#pragma unroll 8
    for (int r = wave; r < n; r += 16) s += partial[(int64_t)r * 2 * width + c];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= 2 * width) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += red[k][lane];
  void* out = c < width ? dw : db;
  const int i = c < width ? c : c - width;
  if (!out) return;
  if (dtype == CRADLE_F32) store1<CRADLE_F32>(out, i, s);
  else if (dtype == CRADLE_BF16) store1<CRADLE_BF16>(out, i, s);
  else store1<CRADLE_F16>(out, i, s);
}

constexpr int kMaxWidth = 32768;
constexpr int kOnePassWidth = 16384;  // above, dx and the parameters' gradients are two passes (one would spill)
constexpr int kCUs = 256;

// rows per workgroup and workgroups of a pass: enough of them to fill the chip, few enough that w, b (and the partial sums of
// the backward pass) are a small part of what is moved
int rows_per_block(int width) { return width <= 1024 ? 4 : 1; }
int64_t fwd_blocks(int64_t rows, int width) {
  const int64_t b = (rows + rows_per_block(width) - 1) / rows_per_block(width);
  const int64_t most = width <= 1024 ? 8 * kCUs : width <= 8192 ? 8 * kCUs : 2 * kCUs;
  return b < most ? b : most;
}
int64_t bwd_blocks(int64_t rows, int width) {
  const int64_t b = (rows + rows_per_block(width) - 1) / rows_per_block(width);
  const int64_t most = width <= 4096 ? 4 * kCUs : width <= 8192 ? 2 * kCUs : kCUs;
  return b < most ? b : most;  // (also the row shares of params_kernel: 16 column blocks x 256)
}

// Threads per row and chunks per thread by width, measured in bf16.  Forward, 32768 x 4096: 256 threads with two chunks 124 us,
// 512 with one 102 us.  The backward pass holds five numbers per column and has to stay below 128 registers (four waves per
// SIMD): 32768 x 4096: 256 with two 168 us, 512 with one 192 us; 16384 x 8192: 512 with two (130 registers) 275 us, 1024 with one
// 179 us.
#define CRADLE_LN_FWD_WIDTHS(CASE) \
  if (width <= 512) CASE(64, 1)             \
  else if (width <= 1024) CASE(64, 2)       \
  else if (width <= 2048) CASE(256, 1)      \
  else if (width <= 4096) CASE(512, 1)      \
  else if (width <= 8192) CASE(512, 2)      \
  else if (width <= 16384) CASE(1024, 2)    \
  else CASE(1024, 4)
#define CRADLE_LN_BWD_WIDTHS(CASE) \
  if (width <= 512) CASE(64, 1)             \
  else if (width <= 1024) CASE(64, 2)       \
  else if (width <= 2048) CASE(256, 1)      \
  else if (width <= 4096) CASE(256, 2)      \
  else if (width <= 8192) CASE(1024, 1)     \
  else if (width <= 16384) CASE(1024, 2)    \
  else CASE(1024, 4)

// 16-byte pieces: base and row starts aligned (parameter vectors: ld = 0)
bool vec_ok(const void* p, int64_t ld, int dtype) { return !p || (((uintptr_t)p & 15) == 0 && ld % (dtype == CRADLE_F32 ? 4 : 8) == 0); }

int check_common(const char* what, int dtype, int w_dtype, int64_t rows, int width) {
  CRADLE_CHECK_ARG(dtype == CRADLE_F32 || dtype == CRADLE_BF16 || dtype == CRADLE_F16, "%s: dtype %d", what, dtype);
  CRADLE_CHECK_ARG(w_dtype == dtype || w_dtype == CRADLE_F32, "%s: weights must be of the tensors' type or fp32", what);
  CRADLE_CHECK_ARG(rows >= 0 && width >= 1 && width <= kMaxWidth, "%s: rows=%lld width=%d (1 <= width <= %d)", what, (long long)rows,
                   width, kMaxWidth);
  return CRADLE_OK;
}

}  // namespace
}  // namespace cradle

using namespace cradle;

extern "C" {

int cradle_layer_norm_fwd(const void* x, int64_t ld_x, const void* weight, const void* bias, int dtype, int w_dtype, float eps,
                          void* y, int64_t ld_y, float* mean, float* rstd, int64_t rows, int width, cradle_stream_t s) {
  const int rc = check_common("layer_norm_fwd", dtype, w_dtype, rows, width);
  if (rc != CRADLE_OK) return rc;
  if (rows == 0) return CRADLE_OK;
  CRADLE_CHECK_ARG(x && y && ld_x >= width && ld_y >= width, "layer_norm_fwd: null pointer or leading dimension below the width");
  const bool vec = width % 8 == 0 && vec_ok(x, ld_x, dtype) && vec_ok(y, ld_y, dtype) && vec_ok(weight, 0, dtype) && vec_ok(bias, 0, dtype);
  const int w_fp32 = w_dtype == CRADLE_F32;
  const dim3 grid((unsigned)fwd_blocks(rows, width));
#define CRADLE_LN_FWD(DT, TPR, NCH, VEC)                                                                                        \
  hipLaunchKernelGGL((fwd_kernel<DT, TPR, NCH, VEC>), grid, dim3(threads<TPR>()), 0, s, x, ld_x, weight, bias, w_fp32, eps, y, \
                     ld_y, mean, rstd, rows, width)
#define CRADLE_LN_CASE(TPR, NCH)                                                   \
  {                                                                                \
    if (dtype == CRADLE_F32) {                                                     \
      if (vec) CRADLE_LN_FWD(CRADLE_F32, TPR, NCH, true);                          \
      else CRADLE_LN_FWD(CRADLE_F32, TPR, NCH, false);                             \
    } else if (dtype == CRADLE_BF16) {                                             \
      if (vec) CRADLE_LN_FWD(CRADLE_BF16, TPR, NCH, true);                         \
      else CRADLE_LN_FWD(CRADLE_BF16, TPR, NCH, false);                            \
    } else {                                                                       \
      if (vec) CRADLE_LN_FWD(CRADLE_F16, TPR, NCH, true);                          \
      else CRADLE_LN_FWD(CRADLE_F16, TPR, NCH, false);                             \
    }                                                                              \
  }
  CRADLE_LN_FWD_WIDTHS(CRADLE_LN_CASE)
#undef CRADLE_LN_CASE
  CRADLE_CHECK_LAUNCH("layer_norm_fwd");
  return CRADLE_OK;
}

int64_t cradle_layer_norm_workspace_floats(int64_t rows, int width) {
  if (rows <= 0 || width < 1 || width > kMaxWidth) return 0;
  return bwd_blocks(rows, width) * 2 * width;
}

int cradle_layer_norm_bwd(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const void* weight, const float* mean,
                          const float* rstd, int dtype, int w_dtype, void* dx, int64_t ld_dx, void* dweight, void* dbias,
                          float* workspace, int64_t workspace_floats, int64_t rows, int width, cradle_stream_t s) {
  const int rc = check_common("layer_norm_bwd", dtype, w_dtype, rows, width);
  if (rc != CRADLE_OK) return rc;
  CRADLE_CHECK_ARG(rows >= 1, "layer_norm_bwd: no rows (without rows the parameters' gradients are zero: the caller clears them)");
  CRADLE_CHECK_ARG(dy && x && mean && rstd && ld_dy >= width && ld_x >= width && (!dx || ld_dx >= width),
                   "layer_norm_bwd: null pointer or leading dimension below the width");
  const bool params = dweight || dbias;
  CRADLE_CHECK_ARG(!params || (workspace && workspace_floats >= cradle_layer_norm_workspace_floats(rows, width) &&
                               ((uintptr_t)workspace & 15) == 0),
                   "layer_norm_bwd: workspace of %lld floats (16-byte aligned) needed",
                   (long long)cradle_layer_norm_workspace_floats(rows, width));
  const bool vec = width % 8 == 0 && vec_ok(dy, ld_dy, dtype) && vec_ok(x, ld_x, dtype) && vec_ok(dx, ld_dx, dtype) && vec_ok(weight, 0, dtype);
  const int w_fp32 = w_dtype == CRADLE_F32;
  const int blocks = (int)bwd_blocks(rows, width);
  float* partial = params ? workspace : nullptr;
  const bool one_pass = width <= kOnePassWidth;
#define CRADLE_LN_BWD(DT, TPR, NCH, VEC)                                                                                               \
  {                                                                                                                                    \
    if (one_pass || dx)                                                                                                                \
      hipLaunchKernelGGL((bwd_kernel<DT, TPR, NCH, VEC, (NCH <= 2)>), dim3(blocks), dim3(threads<TPR>()), 0, s, dy, ld_dy, x, ld_x,     \
                         weight, w_fp32, mean, rstd, dx, ld_dx, partial, rows, width);                                                 \
    if (!one_pass && params)                                                                                                           \
      hipLaunchKernelGGL((params_kernel<DT, VEC>), dim3((width + 2047) / 2048, blocks), dim3(256), 0, s, dy, ld_dy, x, ld_x, mean, rstd, \
                         partial, rows, width);                                                                                        \
  }
#define CRADLE_LN_CASE(TPR, NCH)                                                   \
  {                                                                                \
    if (dtype == CRADLE_F32) {                                                     \
      if (vec) CRADLE_LN_BWD(CRADLE_F32, TPR, NCH, true)                           \
      else CRADLE_LN_BWD(CRADLE_F32, TPR, NCH, false)                              \
    } else if (dtype == CRADLE_BF16) {                                             \
      if (vec) CRADLE_LN_BWD(CRADLE_BF16, TPR, NCH, true)                          \
      else CRADLE_LN_BWD(CRADLE_BF16, TPR, NCH, false)                             \
    } else {                                                                       \
      if (vec) CRADLE_LN_BWD(CRADLE_F16, TPR, NCH, true)                           \
      else CRADLE_LN_BWD(CRADLE_F16, TPR, NCH, false)                              \
    }                                                                              \
  }
  CRADLE_LN_BWD_WIDTHS(CRADLE_LN_CASE)
#undef CRADLE_LN_CASE
  if (params)
    hipLaunchKernelGGL(join_kernel, dim3((2 * width + 63) / 64), dim3(1024), 0, s, workspace, blocks, width, dweight, dbias, w_dtype);
  CRADLE_CHECK_LAUNCH("layer_norm_bwd");
  return CRADLE_OK;
}

}  // extern "C"
