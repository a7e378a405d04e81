// Entry points of the gated feed-forward block (gated_mlp.h has the mathematics and the tile products) and its form for a
// few rows.
#include "gated_mlp.h"

namespace cradle {
namespace gated {

namespace {

// ---------------------------------------------------------------------------------------------------------------
// a few rows: dot products along the weights' rows, fp32 arithmetic
// ---------------------------------------------------------------------------------------------------------------
// V consecutive numbers (16 bytes of a 16-bit or fp32 tensor)
template <int DT>
struct Piece {
  static constexpr int V = DT == CRADLE_F32 ? 4 : 8;
  u32x4 raw;
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (DT == CRADLE_F32) {
      const uint32_t w = raw[e];  // (a copy: bit_cast of a vector's element takes the first one)
      return __builtin_bit_cast(float, w);
    }
    const u16 b = (u16)(raw[e / 2] >> (e % 2 * 16));
    return DT == CRADLE_BF16 ? from_bf16(b) : from_f16(b);
  }
};

// One wave per weight row (GATE: per pair of rows, gate and up), R rows of x (type XT) at once.  VEC: the weight is read in 16-byte
// pieces, four in flight per lane and row; x comes from the caches, every wave reads all of it.
template <int DT, int XT, int R, bool GATE, bool VEC>
__global__ __launch_bounds__(256) void few_rows_kernel(const void* __restrict__ x, int64_t ldx, const void* __restrict__ W, int64_t ldw,
                                                       int rows, int K, int N, const void* __restrict__ bias, int act,
                                                       float* __restrict__ h, const void* __restrict__ res, int64_t ld_res,
                                                       void* __restrict__ y, int64_t ldy) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  constexpr int NW = GATE ? 2 : 1, V = VEC ? Piece<DT>::V : 1, U = 4;
  constexpr int ES = DT == CRADLE_F32 ? 4 : 2;
  const char* w0 = static_cast<const char*>(W) + (int64_t)n * ldw * ES;
  const char* w1 = static_cast<const char*>(W) + (int64_t)(N + n) * ldw * ES;
  float acc[NW][R];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[w][r] = 0.f;
  for (int k0 = lane * V; k0 < K; k0 += 64 * V * U) {
    Piece<DT> p[U][NW];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 64 * V;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        p[u][w].raw = u32x4{0, 0, 0, 0};
        if constexpr (VEC) {
          if (k < K) p[u][w].raw = *reinterpret_cast<const u32x4*>((w ? w1 : w0) + (int64_t)k * ES);
        } else if (k < K) {
          if constexpr (DT == CRADLE_F32) p[u][w].raw[0] = *reinterpret_cast<const uint32_t*>((w ? w1 : w0) + (int64_t)k * ES);
          else p[u][w].raw[0] = *reinterpret_cast<const u16*>((w ? w1 : w0) + (int64_t)k * ES);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * 64 * V;
      if (k >= K) break;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= rows) break;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xv = load_as(x, (int64_t)r * ldx + k + e, XT);
#pragma unroll
          for (int w = 0; w < NW; ++w) acc[w][r] = fmaf(p[u][w][e], xv, acc[w][r]);
        }
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
        s0 += load_as(bias, n, DT);
        s1 += load_as(bias, (int64_t)N + n, DT);
      }
      if (lane == 0) h[(int64_t)r * N + n] = act_only<DT == CRADLE_F32>(act, s0) * s1;
    } else if (lane == 0) {
      if (bias) s0 += load_as(bias, n, DT);
      if (res) s0 += load_as(res, (int64_t)r * ld_res + n, DT);
      store_as(y, (int64_t)r * ldy + n, DT, s0);
    }
  }
}

template <int DT, int R>
void few_rows_run(const cradle_gated_mlp_desc* d, const Plan& p, hipStream_t s) {
  float* h = static_cast<float*>(d->workspace);
  constexpr int V = Piece<DT>::V;
  const bool v1 = p.K % V == 0 && d->ld_w_in % V == 0 && ((uintptr_t)d->w_in & 15) == 0;
  const bool v2 = p.F % V == 0 && d->ld_w_out % V == 0 && ((uintptr_t)d->w_out & 15) == 0;
  auto up = v1 ? few_rows_kernel<DT, DT, R, true, true> : few_rows_kernel<DT, DT, R, true, false>;
  auto down = v2 ? few_rows_kernel<DT, CRADLE_F32, R, false, true> : few_rows_kernel<DT, CRADLE_F32, R, false, false>;
  hipLaunchKernelGGL(up, dim3((p.F + 3) / 4), dim3(256), 0, s, d->x, d->ld_x, d->w_in, d->ld_w_in, p.M, p.K, p.F, d->b_in, d->act, h,
                     nullptr, (int64_t)0, nullptr, (int64_t)0);
  hipLaunchKernelGGL(down, dim3((p.O + 3) / 4), dim3(256), 0, s, h, (int64_t)p.F, d->w_out, d->ld_w_out, p.M, p.F, p.O, d->b_out, 0,
                     nullptr, d->residual, d->ld_residual, d->y, d->ld_y);
}
template <int R>
void few_rows_by_type(const cradle_gated_mlp_desc* d, const Plan& p, hipStream_t s) {
  if (p.dtype == CRADLE_F32) few_rows_run<CRADLE_F32, R>(d, p, s);
  else if (p.dtype == CRADLE_BF16) few_rows_run<CRADLE_BF16, R>(d, p, s);
  else few_rows_run<CRADLE_F16, R>(d, p, s);
}

int64_t forward_of(const cradle_gated_mlp_desc* d, const Plan& p, hipStream_t s, bool run) {
  return (p.dtype == CRADLE_F16 ? forward_f16 : p.dtype == CRADLE_BF16 ? forward_bf16 : forward_f32)(d, p, run ? d->workspace : nullptr, s, run);
}
int64_t backward_of(const cradle_gated_mlp_desc* d, const Plan& p, hipStream_t s, bool run) {
  return (p.dtype == CRADLE_F16 ? backward_f16 : p.dtype == CRADLE_BF16 ? backward_bf16 : backward_f32)(d, p, run ? d->workspace : nullptr, s, run);
}

// The rows for which dot products beat the tile products, whose time hardly depends on so few rows.  Dot products | tiles in us,
// width x hidden: 4096 x 10240 in bf16, 1 row 41 | 70, 4 rows 66 | 63, 8 rows 96 | 72 (one row reads 252 MB of weights at 6.2 TB/s,
// partly from the last-level cache; each further one adds 8 us of arithmetic); 1024 x 2560 in bf16, 1 row 6 | 19, 8 rows 20 | 20;
// 512 x 1024 in fp32, 1 row 5 | 28, 8 rows 15 | 28.
bool few_rows(const cradle_gated_mlp_desc* d) {
  const int64_t weights = (int64_t)d->hidden * (2 * d->width + (int64_t)d->out_width);
  return !d->saved_gu && d->rows <= (weights < (1 << 24) ? kFewRows : kFewRows / 2);
}

int check_desc(const cradle_gated_mlp_desc* d, const char* what) {
  CRADLE_CHECK_ARG(d, "%s: null descriptor", what);
  CRADLE_CHECK_ARG(d->rows >= 0 && d->width >= 1 && d->hidden >= 1 && d->out_width >= 1, "%s: rows=%d width=%d hidden=%d out_width=%d",
                   what, d->rows, d->width, d->hidden, d->out_width);
  CRADLE_CHECK_ARG(d->dtype == CRADLE_F32 || d->dtype == CRADLE_BF16 || d->dtype == CRADLE_F16, "%s: dtype %d", what, d->dtype);
  CRADLE_CHECK_ARG(d->act == SILU || d->act == GELU, "%s: activation %d", what, d->act);
  // 32-bit byte offsets inside a tile (mm16.h) and int element counts of the tile grids
  CRADLE_CHECK_ARG(d->width <= (1 << 20) && d->hidden <= (1 << 20) && d->out_width <= (1 << 20) && d->rows <= (1 << 24),
                   "%s: rows <= 2^24, widths <= 2^20 (got %d, %d, %d, %d)", what, d->rows, d->width, d->hidden, d->out_width);
  const int64_t w_row = ((d->ld_w_in > d->width ? d->ld_w_in : d->width) + 63) / 64 * 64;  // (the longer row if it is packed)
  CRADLE_CHECK_ARG(((int64_t)d->hidden + 64 + 256) * w_row < (1LL << 30),
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

int64_t cradle_gated_mlp_saved_bytes(int rows, int width, int hidden, int out_width, int dtype, int64_t* h_bytes) {
  cradle_gated_mlp_desc d{};
  d.rows = rows, d.width = width, d.hidden = hidden, d.out_width = out_width, d.dtype = dtype;
  const Plan p = plan_of(&d);
  const int64_t n = (int64_t)rows * p.Fp;
  if (h_bytes) *h_bytes = n * 2 * p.nph;
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
  CRADLE_CHECK_ARG(((uintptr_t)d->saved_gu & 15) == 0 && ((uintptr_t)d->saved_h & 15) == 0, "gated_mlp_fwd: saved buffers must be 16-byte aligned");
  CRADLE_CHECK_ARG(d->ld_y >= d->out_width && (!d->residual || d->ld_residual >= d->out_width), "gated_mlp_fwd: leading dimension below the row length");
  const int64_t need = cradle_gated_mlp_workspace_bytes(d, 0);
  CRADLE_CHECK_ARG(need == 0 || (d->workspace && d->workspace_bytes >= need && ((uintptr_t)d->workspace & 15) == 0),
                   "gated_mlp_fwd: workspace of %lld bytes (16-byte aligned) needed", (long long)need);
  const Plan p = plan_of(d);
  if (few_rows(d)) {
    if (p.M == 1) few_rows_by_type<1>(d, p, s);
    else if (d->rows <= kFewRows / 2) few_rows_by_type<kFewRows / 2>(d, p, s);
    else few_rows_by_type<kFewRows>(d, p, s);
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
