// Entry points of the gated feed-forward block (gated_mlp.h has the mathematics and the tile products) and its form for a
// few rows.
#include "gated_mlp.h"

namespace cradle {
namespace gated {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// a few rows: dot products along the weights' rows, fp32 arithmetic
// ---------------------------------------------------------------------------------------------------------------
// One wave per weight row (a pair of rows, gate and up, for GATE), R rows of x at once; VEC elements per lane and load.
template <int R, bool GATE>
__global__ __launch_bounds__(256) void few_rows_kernel(const void* __restrict__ x, int64_t ldx, int x_dtype,
                                                       const void* __restrict__ W, int64_t ldw, int dtype, int rows, int K, int N,
                                                       const void* __restrict__ bias, int act, float* __restrict__ h,
                                                       const void* __restrict__ res, int64_t ld_res, void* __restrict__ y,
                                                       int64_t ldy, int vec) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  constexpr int NW = GATE ? 2 : 1;
  float acc[NW][R];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[w][r] = 0.f;
  if (vec) {  // 16-byte pieces of W: 8 16-bit or 4 fp32 numbers
    const int V = dtype == CRADLE_F32 ? 4 : 8;
#pragma unroll 2
    for (int k = lane * V; k < K; k += 64 * V) {
      float wv[NW][8];
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const int64_t row = (int64_t)(w ? N + n : n) * ldw;
        if (dtype == CRADLE_F32) {
          const f32x4 t = *reinterpret_cast<const f32x4*>(static_cast<const float*>(W) + row + k);
#pragma unroll
          for (int e = 0; e < 4; ++e) wv[w][e] = t[e];
        } else {
          const u32x4 t = *reinterpret_cast<const u32x4*>(static_cast<const u16*>(W) + row + k);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const u16 a = (u16)t[e], b = (u16)(t[e] >> 16);
            wv[w][2 * e] = dtype == CRADLE_BF16 ? from_bf16(a) : from_f16(a);
            wv[w][2 * e + 1] = dtype == CRADLE_BF16 ? from_bf16(b) : from_f16(b);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= rows) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e >= V) break;
          const float xv = load_as(x, (int64_t)r * ldx + k + e, x_dtype);
#pragma unroll
          for (int w = 0; w < NW; ++w) acc[w][r] = fmaf(wv[w][e], xv, acc[w][r]);
        }
      }
    }
  } else {
    for (int k = lane; k < K; k += 64) {
      float wv[NW];
#pragma unroll
      for (int w = 0; w < NW; ++w) wv[w] = load_as(W, (int64_t)(w ? N + n : n) * ldw + k, dtype);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= rows) break;
        const float xv = load_as(x, (int64_t)r * ldx + k, x_dtype);
#pragma unroll
        for (int w = 0; w < NW; ++w) acc[w][r] = fmaf(wv[w], xv, acc[w][r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) break;
    float s0 = wave_sum(acc[0][r]);
    if constexpr (GATE) {
      float s1 = wave_sum(acc[1][r]);
      if (bias) {
        s0 += load_as(bias, n, dtype);
        s1 += load_as(bias, (int64_t)N + n, dtype);
      }
      if (lane == 0) h[(int64_t)r * N + n] = act_only(act, s0) * s1;
    } else if (lane == 0) {
      if (bias) s0 += load_as(bias, n, dtype);
      if (res) s0 += load_as(res, (int64_t)r * ld_res + n, dtype);
      store_as(y, (int64_t)r * ldy + n, dtype, s0);
    }
  }
}

int64_t forward_of(const cradle_gated_mlp_desc* d, const Plan& p, hipStream_t s, bool run) {
  return (p.dtype == CRADLE_F16 ? forward_f16 : p.dtype == CRADLE_BF16 ? forward_bf16 : forward_f32)(d, p, run ? d->workspace : nullptr, s, run);
}
int64_t backward_of(const cradle_gated_mlp_desc* d, const Plan& p, hipStream_t s, bool run) {
  return (p.dtype == CRADLE_F16 ? backward_f16 : p.dtype == CRADLE_BF16 ? backward_bf16 : backward_f32)(d, p, run ? d->workspace : nullptr, s, run);
}

bool few_rows(const cradle_gated_mlp_desc* d) { return d->rows <= kFewRows && !d->saved_gu; }

int check_desc(const cradle_gated_mlp_desc* d, const char* what) {
  CRADLE_CHECK_ARG(d, "%s: null descriptor", what);
  CRADLE_CHECK_ARG(d->rows >= 0 && d->width >= 1 && d->hidden >= 1 && d->out_width >= 1, "%s: rows=%d width=%d hidden=%d out_width=%d",
                   what, d->rows, d->width, d->hidden, d->out_width);
  CRADLE_CHECK_ARG(d->dtype == CRADLE_F32 || d->dtype == CRADLE_BF16 || d->dtype == CRADLE_F16, "%s: dtype %d", what, d->dtype);
  CRADLE_CHECK_ARG(d->act == SILU || d->act == GELU, "%s: activation %d", what, d->act);
  // 32-bit byte offsets inside a tile (mm16.h) and int element counts of the tile grids
  CRADLE_CHECK_ARG(d->width <= (1 << 20) && d->hidden <= (1 << 20) && d->out_width <= (1 << 20) && d->rows <= (1 << 24),
                   "%s: rows <= 2^24, widths <= 2^20 (got %d, %d, %d, %d)", what, d->rows, d->width, d->hidden, d->out_width);
  CRADLE_CHECK_ARG(((int64_t)d->hidden + 264) * (d->ld_w_in > d->width ? up8(d->ld_w_in) : up8(d->width)) < (1LL << 30),
                   "%s: hidden x ld(w_in) must stay below 2^30 elements", what);
  CRADLE_CHECK_ARG(d->ld_x >= d->width && d->ld_w_in >= d->width && d->ld_w_out >= d->hidden, "%s: leading dimension below the row length", what);
  CRADLE_CHECK_ARG(d->ld_x < (1 << 22) && d->ld_w_in < (1 << 22) && d->ld_w_out < (1 << 22) && d->ld_dy < (1 << 22),
                   "%s: leading dimensions must stay below 2^22", what);
  CRADLE_CHECK_ARG((!d->saved_gu) == (!d->saved_h), "%s: saved_gu and saved_h go together", what);
  return CRADLE_OK;
}

}  // namespace
}  // namespace gated
}  // namespace cradle

using namespace cradle;
using namespace cradle::gated;

extern "C" {

int64_t cradle_gated_mlp_saved_bytes(int rows, int hidden, int dtype, int64_t* h_bytes) {
  const int64_t n = (int64_t)rows * up8(hidden);
  if (h_bytes) *h_bytes = n * 2 * (dtype == CRADLE_F32 ? 3 : 1);
  return n * 2 * 4;
}

int64_t cradle_gated_mlp_workspace_bytes(const cradle_gated_mlp_desc* d, int backward_pass) {
  if (check_desc(d, "gated_mlp_workspace_bytes") != CRADLE_OK) return -1;
  const Plan p = plan_of(d);
  if (!backward_pass && few_rows(d)) return (int64_t)p.M * p.F * 4;
  return backward_pass ? backward_of(d, p, nullptr, false) : forward_of(d, p, nullptr, false);
}

int cradle_gated_mlp_fwd(const cradle_gated_mlp_desc* d, cradle_stream_t s) {
  const int rc = check_desc(d, "gated_mlp_fwd");
  if (rc != CRADLE_OK) return rc;
  if (d->rows == 0) return CRADLE_OK;
  CRADLE_CHECK_ARG(d->x && d->w_in && d->w_out && d->y, "gated_mlp_fwd: null pointer");
  CRADLE_CHECK_ARG(d->ld_y >= d->out_width && (!d->residual || d->ld_residual >= d->out_width), "gated_mlp_fwd: leading dimension below the row length");
  const int64_t need = cradle_gated_mlp_workspace_bytes(d, 0);
  CRADLE_CHECK_ARG(need == 0 || (d->workspace && d->workspace_bytes >= need && ((uintptr_t)d->workspace & 15) == 0),
                   "gated_mlp_fwd: workspace of %lld bytes (16-byte aligned) needed", (long long)need);
  const Plan p = plan_of(d);
  if (few_rows(d)) {
    float* h = static_cast<float*>(d->workspace);
    const int V = p.dtype == CRADLE_F32 ? 4 : 8;
    const int v1 = p.K % V == 0 && d->ld_w_in % V == 0 && ((uintptr_t)d->w_in & 15) == 0;
    const int v2 = p.F % V == 0 && d->ld_w_out % V == 0 && ((uintptr_t)d->w_out & 15) == 0;
    const dim3 g1((p.F + 3) / 4), g2((p.O + 3) / 4);
#define CRADLE_FEW(R)                                                                                                             \
  {                                                                                                                               \
    hipLaunchKernelGGL((few_rows_kernel<R, true>), g1, dim3(256), 0, s, d->x, d->ld_x, p.dtype, d->w_in, d->ld_w_in, p.dtype, p.M, \
                       p.K, p.F, d->b_in, d->act, h, nullptr, 0, nullptr, 0, v1);                                                 \
    hipLaunchKernelGGL((few_rows_kernel<R, false>), g2, dim3(256), 0, s, h, (int64_t)p.F, CRADLE_F32, d->w_out, d->ld_w_out,       \
                       p.dtype, p.M, p.F, p.O, d->b_out, 0, nullptr, d->residual, d->ld_residual, d->y, d->ld_y, v2);              \
  }
    if (p.M == 1) CRADLE_FEW(1) else CRADLE_FEW(kFewRows)
#undef CRADLE_FEW
  } else {
    forward_of(d, p, s, true);
  }
  CRADLE_CHECK_LAUNCH("gated_mlp_fwd");
  return CRADLE_OK;
}

int cradle_gated_mlp_bwd(const cradle_gated_mlp_desc* d, cradle_stream_t s) {
  const int rc = check_desc(d, "gated_mlp_bwd");
  if (rc != CRADLE_OK) return rc;
  CRADLE_CHECK_ARG(d->rows >= 1, "gated_mlp_bwd: rows=%d (without rows the gradients are zero: the caller clears them)", d->rows);
  CRADLE_CHECK_ARG(d->x && d->w_in && d->w_out && d->dy && d->saved_gu && d->saved_h, "gated_mlp_bwd: null pointer");
  CRADLE_CHECK_ARG(((uintptr_t)d->saved_gu & 15) == 0 && ((uintptr_t)d->saved_h & 15) == 0, "gated_mlp_bwd: saved buffers must be 16-byte aligned");
  CRADLE_CHECK_ARG(d->ld_dy >= d->out_width && (!d->dx || d->ld_dx >= d->width), "gated_mlp_bwd: leading dimension below the row length");
  const int64_t need = cradle_gated_mlp_workspace_bytes(d, 1);
  CRADLE_CHECK_ARG(d->workspace && d->workspace_bytes >= need && ((uintptr_t)d->workspace & 15) == 0,
                   "gated_mlp_bwd: workspace of %lld bytes (16-byte aligned) needed", (long long)need);
  const Plan p = plan_of(d);
  backward_of(d, p, s, true);
  CRADLE_CHECK_LAUNCH("gated_mlp_bwd");
  return CRADLE_OK;
}

}  // extern "C"
