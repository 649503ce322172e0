// RMS norm of rows with the residual's addition (gfx950):
//   t = x + residual,  rstd = 1 / sqrt(sum t^2 / C + eps),  y = t rstd w;
// backward, with dy and dt the gradients of y and t and hat = t rstd,
//   d = (dy w - hat sum(dy w hat) / C) rstd + dt,  dx = dresidual = d,
//   dw = sum over the rows of dy hat.
//
// A row belongs to 8 to 64 lanes, 8 channels of each vector of it, and stays in
// their registers from the first reading on.  Rows need no alignment beyond
// their elements': the vectors are loaded as they lie.  The norm is that of the
// sum before t is rounded to the residual's type; hat in the backward pass is
// formed from t as it is stored, half a step of that type away.
//
// The weight's gradient: every workgroup goes over its share of the rows with
// sums by channel in registers, and a second kernel adds the workgroups' sums, in
// a fixed order.
//
// Bound by memory: x, the residual, y and t once each, dy, dt, t and dx once each.
// 262144 rows of 512 channels, bf16 beside an fp32 residual: 267 us forward (6.0
// TB/s), 412 us backward (4.6 TB/s: three streams read, two written); 17920 rows of
// 128 in fp32, 9.2 and 9.3 + 4.3 us.
#include <type_traits>

#include "chain.h"

namespace {

constexpr int kRmsThreads = 256;
constexpr int kRmsMaxWidth = 8192;
constexpr int kRmsGroups = 1024;  // workgroups of the backward pass, at most

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MLCG_WAVE);
  return v;
}

// T: x, weight and y; R: the residual and t
template <typename T, typename R, int NV>
__global__ __launch_bounds__(kRmsThreads) void rms_forward(
    const T* __restrict__ x, int64_t x_ld, const R* __restrict__ residual, int64_t r_ld,
    const T* __restrict__ weight, int64_t rows, int width, int lanes, float eps,
    T* __restrict__ y, R* __restrict__ t, float* __restrict__ rstd) {
  const int per = kRmsThreads / lanes;
  const int64_t row = chain_group() * per + threadIdx.x / lanes;
  const int l = threadIdx.x % lanes;
  const bool in = row < rows;
  f32x8 v[NV];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int el = 8 * (l + i * lanes);
    v[i] = f32x8{};
    if (!in || el >= width) continue;
    v[i] = load_row8<T>(x + row * x_ld, el, width);
    if (residual) {
      v[i] += load_row8<R>(residual + row * r_ld, el, width);
      store_row8<R>(t + row * width, el, width, v[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(v[i][j], v[i][j], s);
  }
  s = lanes_sum(s, lanes);
  const float r = 1.0f / sqrtf(s / (float)width + eps);
  if (!in) return;
  if (l == 0) rstd[row] = r;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int el = 8 * (l + i * lanes);
    if (el >= width) continue;
    store_row8<T>(y + row * width, el, width, v[i] * r * load_row8<T>(weight, el, width));
  }
}

template <typename T, typename R, int NV>
__global__ __launch_bounds__(kRmsThreads) void rms_backward(
    const T* __restrict__ grad, const R* __restrict__ grad_t, const R* __restrict__ t,
    int64_t t_ld, const T* __restrict__ weight, const float* __restrict__ rstd, int64_t rows,
    int width, int lanes, T* __restrict__ dx, R* __restrict__ dr, float* __restrict__ part) {
  const int per = kRmsThreads / lanes, l = threadIdx.x % lanes;
  f32x8 dw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) dw[i] = f32x8{};
  const float inv = 1.0f / (float)width;
  for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < rows; r0 += (int64_t)gridDim.x * per) {
    const int64_t row = r0 + threadIdx.x / lanes;
    const bool in = row < rows;
    f32x8 hat[NV], d[NV];
    const float r = in ? rstd[row] : 0.0f;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int el = 8 * (l + i * lanes);
      hat[i] = d[i] = f32x8{};
      if (!in || el >= width) continue;
      hat[i] = load_row8<R>(t + row * t_ld, el, width) * r;
      const f32x8 g = load_row8<T>(grad + row * width, el, width);
      const f32x8 gh = g * hat[i];
      dw[i] += gh;
      const f32x8 w = load_row8<T>(weight, el, width);
      d[i] = g * w;
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fmaf(gh[j], w[j], s);
    }
    s = lanes_sum(s, lanes) * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int el = 8 * (l + i * lanes);
      if (!in || el >= width) continue;
      f32x8 o = (d[i] - hat[i] * s) * r;
      if (grad_t) o += load_row8<R>(grad_t + row * width, el, width);
      if (dx) store_row8<T>(dx + row * width, el, width, o);
      if (dr) store_row8<R>(dr + row * width, el, width, o);
    }
  }
  // the sums by channel of the rows that a workgroup has in flight, in order
  __shared__ float sum[kRmsThreads * 8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[threadIdx.x * 8 + j] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < 8 * lanes; c += kRmsThreads) {
      const int el = 8 * i * lanes + c;
      if (el >= width) continue;
      float a = 0.0f;
      for (int p = 0; p < per; ++p) a += sum[p * 8 * lanes + c];
      part[(int64_t)blockIdx.x * width + el] = a;
    }
  }
}

// dw[c] = sum over the n workgroups' sums: 16 channels a workgroup, 16 parts of n
template <typename T>
__global__ __launch_bounds__(kRmsThreads) void rms_weight_sum(const float* __restrict__ part,
                                                              int n, int width,
                                                              T* __restrict__ dw) {
  __shared__ float sum[16][17];
  const int c = threadIdx.x % 16, p = threadIdx.x / 16, el = 16 * blockIdx.x + c;
  float s = 0.0f;
  if (el < width) {
    int i = p;
    for (; i + 7 * 16 < n; i += 8 * 16) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = part[(int64_t)(i + 16 * j) * width + el];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; i < n; i += 16) s += part[(int64_t)i * width + el];
  }
  sum[p][c] = s;
  __syncthreads();
  if (p == 0 && el < width) {
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s += sum[j][c];
    dw[el] = (T)s;
  }
}

// lanes of a row, a power of two, and its vectors a lane
struct RmsShape {
  int lanes, vectors;
  explicit RmsShape(int width) {
    lanes = 8;
    while (lanes < MLCG_WAVE && 8 * lanes < width) lanes *= 2;
    vectors = (width + 8 * lanes - 1) / (8 * lanes);
  }
};

unsigned rms_groups(int64_t rows, int width) {
  const RmsShape sh(width);
  const int64_t steps = (rows + kRmsThreads / sh.lanes - 1) / (kRmsThreads / sh.lanes);
  return (unsigned)(steps < kRmsGroups ? (steps < 1 ? 1 : steps) : kRmsGroups);
}

struct RmsCall {
  const void *x, *residual, *weight, *grad, *grad_t;
  int64_t x_ld, r_ld, rows;
  int width;
  float eps;
  void *y, *t, *dx, *dr, *dw;
  float *rstd, *ws;
};

template <typename T, typename R, int NV>
int rms_launch(const RmsCall& a, bool backward, hipStream_t s) {
  const RmsShape sh(a.width);
  const dim3 block(kRmsThreads);
  if (!backward) {
    const dim3 grid = chain_grid(mlcg_div_up(a.rows, kRmsThreads / sh.lanes));
    hipLaunchKernelGGL((rms_forward<T, R, NV>), grid, block, 0, s, (const T*)a.x, a.x_ld,
                       (const R*)a.residual, a.r_ld, (const T*)a.weight, a.rows, a.width, sh.lanes,
                       a.eps, (T*)a.y, (R*)a.t, a.rstd);
    return mlcg_launch_status();
  }
  const unsigned n = rms_groups(a.rows, a.width);
  hipLaunchKernelGGL((rms_backward<T, R, NV>), dim3(n), block, 0, s, (const T*)a.grad,
                     (const R*)a.grad_t, (const R*)a.x, a.x_ld, (const T*)a.weight, a.rstd, a.rows,
                     a.width, sh.lanes, (T*)a.dx, (R*)a.dr, a.ws);
  hipLaunchKernelGGL((rms_weight_sum<T>), dim3(mlcg_div_up(a.width, 16)), block, 0, s, a.ws, (int)n,
                     a.width, (T*)a.dw);
  return mlcg_launch_status();
}

template <typename T, typename R>
int rms_vectors(const RmsCall& a, bool backward, hipStream_t s) {
  const int nv = RmsShape(a.width).vectors;
  if (nv <= 1) return rms_launch<T, R, 1>(a, backward, s);
  if (nv <= 2) return rms_launch<T, R, 2>(a, backward, s);
  if (nv <= 4) return rms_launch<T, R, 4>(a, backward, s);
  return rms_launch<T, R, 16>(a, backward, s);
}

int rms_types(const RmsCall& a, int dtype, int res_dtype, bool backward, hipStream_t s) {
  const bool wide = res_dtype == MLCG_DTYPE_F32;
  if (!wide && res_dtype != dtype) return MLCG_ERR_ARGUMENT;
  switch (dtype) {
    case MLCG_DTYPE_F32: return rms_vectors<float, float>(a, backward, s);
    case MLCG_DTYPE_F16:
      return wide ? rms_vectors<_Float16, float>(a, backward, s)
                  : rms_vectors<_Float16, _Float16>(a, backward, s);
    case MLCG_DTYPE_BF16:
      return wide ? rms_vectors<__bf16, float>(a, backward, s)
                  : rms_vectors<__bf16, __bf16>(a, backward, s);
    default: return MLCG_ERR_ARGUMENT;
  }
}

bool rms_ok(int64_t rows, int width, int64_t ld) {
  return rows >= 0 && rows < (int64_t(1) << 31) && width >= 1 && width <= kRmsMaxWidth &&
         (rows <= 1 || ld >= 0);
}

}  // namespace

extern "C" int mlcg_rms_norm_add(const void* x, int64_t x_ld, const void* residual, int64_t r_ld,
                                 const void* weight, int64_t rows, int width, int dtype,
                                 int residual_dtype, float eps, void* y, void* t, float* rstd,
                                 void* stream) {
  MLCG_REQUIRE(rms_ok(rows, width, x_ld) && rms_ok(rows, width, r_ld));
  if (rows == 0) return MLCG_OK;
  MLCG_REQUIRE(x && weight && y && rstd && (!residual || t));
  RmsCall a{};
  a.x = x, a.x_ld = x_ld, a.residual = residual, a.r_ld = r_ld, a.weight = weight, a.rows = rows;
  a.width = width, a.eps = eps, a.y = y, a.t = t, a.rstd = rstd;
  return rms_types(a, dtype, residual ? residual_dtype : dtype, false, mlcg_stream(stream));
}

extern "C" int64_t mlcg_rms_norm_add_workspace_floats(int64_t rows, int width) {
  if (rows < 0 || width < 1 || width > kRmsMaxWidth) return -1;
  return (int64_t)rms_groups(rows, width) * width;
}

extern "C" int mlcg_rms_norm_add_backward(const void* grad_y, const void* grad_t, const void* t,
                                          int64_t t_ld, const void* weight, const float* rstd,
                                          int64_t rows, int width, int dtype, int residual_dtype,
                                          void* grad_x, void* grad_residual, void* grad_weight,
                                          float* workspace, int64_t workspace_floats,
                                          void* stream) {
  MLCG_REQUIRE(rms_ok(rows, width, t_ld) && rows >= 1 && grad_y && t && weight && rstd &&
               grad_weight && workspace &&
               workspace_floats >= mlcg_rms_norm_add_workspace_floats(rows, width));
  RmsCall a{};
  a.grad = grad_y, a.grad_t = grad_t, a.x = t, a.x_ld = t_ld, a.weight = weight, a.rows = rows;
  a.width = width, a.dx = grad_x, a.dr = grad_residual, a.dw = grad_weight;
  a.rstd = const_cast<float*>(rstd), a.ws = workspace;
  return rms_types(a, dtype, residual_dtype, true, mlcg_stream(stream));
}
