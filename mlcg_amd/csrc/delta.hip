// Entry points of the gated delta rule (delta.h), and its step by one bead.
//
// The step: a workgroup has one head's state of one sequence in registers,
//   S <- e^g S,  u = beta (v - S^T k),  S <- S + k u^T,  o = scale S^T q,
// reads it once and writes it once; both sums over Dk go through LDS, in a fixed
// order.  Bound by memory: the states' bytes.  1024 sequences, 8 heads of 64 x 128,
// bf16: 109 us, 5.0 TB/s; 16 sequences, 4 heads of 32 x 32 in fp32: 6 us, a launch.
#include <type_traits>

#include "delta.h"

namespace {

constexpr int kStepThreads = 256;

struct StepArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  const float *decay, *beta, *state;
  int64_t batch;
  int heads, group, dk, dv;
  float scale;
  int normalize;
  float* next;
  void* out;
};

// A thread has W columns of every R-th row of the state, NR of them.
template <typename T, int W, int NR>
__global__ __launch_bounds__(kStepThreads) void delta_step_kernel(StepArgs a, int cols) {
  __shared__ float kq[2][128];
  __shared__ float part[kStepThreads * W];
  __shared__ float norm[2];
  const int R = kStepThreads / cols;  // rows in flight; threads past R cols have none
  const int h = blockIdx.y;
  const int64_t b = chain_group(), at = b * a.heads + h;
  if (b >= a.batch) return;
  const int r0 = threadIdx.x / cols, c0 = threadIdx.x % cols * W;
  const bool live = r0 < R;
  const float* const S = a.state + at * ((int64_t)a.dk * a.dv) + c0;
  float s[NR][W];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = r0 + i * R;
#pragma unroll
    for (int j = 0; j < W; ++j) s[i][j] = 0.0f;
    if (live && r < a.dk) {
      if constexpr (W == 4) {
        const float4 x = *reinterpret_cast<const float4*>(S + (int64_t)r * a.dv);
        s[i][0] = x.x, s[i][1] = x.y, s[i][2] = x.z, s[i][3] = x.w;
      } else {
        s[i][0] = S[(int64_t)r * a.dv];
      }
    }
  }
  {
    const int t = threadIdx.x & 127, which = threadIdx.x >> 7;
    const T* const src = which ? (const T*)a.q + b * a.q_row + h / a.group * a.q_head
                               : (const T*)a.k + b * a.k_row + h / a.group * a.k_head;
    kq[which][t] = t < a.dk ? (float)src[t] : 0.0f;
  }
  const float g = a.decay[at], beta = a.beta[at];
  __syncthreads();
  if (threadIdx.x < 128) {  // a wave each
    const int which = threadIdx.x / 64, l = threadIdx.x % 64;
    const float x = kq[which][l], y = kq[which][l + 64];
    const float n = mlcg_wave_sum(fmaf(x, x, y * y));
    if (l == 0) norm[which] = a.normalize ? 1.0f / sqrtf(n + 1e-6f) : 1.0f;
  }
  __syncthreads();
  const float decay = __builtin_amdgcn_exp2f(g * 1.4426950408889634f);
  const float rk = norm[0], rq = norm[1] * a.scale;
  float sum[W];
#pragma unroll
  for (int j = 0; j < W; ++j) sum[j] = 0.0f;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = r0 + i * R;
    const float kr = r < a.dk ? kq[0][r] * rk : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      s[i][j] *= decay;
      sum[j] = fmaf(kr, s[i][j], sum[j]);
    }
  }
  // part[r][c]: every thread then sums its own columns over the rows
  if (live)
#pragma unroll
    for (int j = 0; j < W; ++j) part[r0 * cols * W + c0 + j] = sum[j];
  __syncthreads();
  float u[W];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    float t = 0.0f;
    for (int r = 0; r < R; ++r) t += part[r * cols * W + c0 + j];
    const float v = c0 + j < a.dv
                        ? (float)((const T*)a.v)[b * a.v_row + h * a.v_head + c0 + j]
                        : 0.0f;
    u[j] = beta * (v - t);
    sum[j] = 0.0f;
  }
  float* const N = a.next + at * ((int64_t)a.dk * a.dv) + c0;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = r0 + i * R;
    if (!live || r >= a.dk) continue;
    const float kr = kq[0][r] * rk, qr = kq[1][r] * rq;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      s[i][j] = fmaf(kr, u[j], s[i][j]);
      sum[j] = fmaf(qr, s[i][j], sum[j]);
    }
    if constexpr (W == 4)
      *reinterpret_cast<float4*>(N + (int64_t)r * a.dv) =
          make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
    else
      N[(int64_t)r * a.dv] = s[i][0];
  }
  __syncthreads();
  if (live)
#pragma unroll
    for (int j = 0; j < W; ++j) part[r0 * cols * W + c0 + j] = sum[j];
  __syncthreads();
  for (int c = threadIdx.x; c < a.dv; c += kStepThreads) {
    float t = 0.0f;
    for (int r = 0; r < R; ++r) t += part[r * cols * W + c];
    ((T*)a.out)[at * a.dv + c] = (T)t;
  }
}

template <typename T, int W>
int launch_step(const StepArgs& a, hipStream_t s) {
  const int cols = a.dv / W, R = kStepThreads / cols;
  const dim3 grid = chain_grid(a.batch, a.heads), block(kStepThreads);
  const int rows = (a.dk + R - 1) / R;
  if (rows <= 4)
    hipLaunchKernelGGL((delta_step_kernel<T, W, 4>), grid, block, 0, s, a, cols);
  else if (W == 4 || rows <= 16)  // of 4 x 32 columns there are 16 at most
    hipLaunchKernelGGL((delta_step_kernel<T, W, 16>), grid, block, 0, s, a, cols);
  else
    hipLaunchKernelGGL((delta_step_kernel<T, 1, 64>), grid, block, 0, s, a, cols);
  return mlcg_launch_status();
}

template <typename T>
int step_of(const StepArgs& a, hipStream_t s) {
  const bool wide = a.dv % 4 == 0 && chain_aligned16(a.state) && chain_aligned16(a.next);
  return wide ? launch_step<T, 4>(a, s) : launch_step<T, 1>(a, s);
}

// workgroups of up to 512 threads along one axis; `kept` of so many takes 370 GB
constexpr int64_t kMostTiles = int64_t(1) << 23;

bool aligned32(const void* p) { return reinterpret_cast<uintptr_t>(p) % 32 == 0; }

// the parts of the buffers, in floats
struct Parts {
  int64_t fac, rows, mats, u, s0, seg_state, seg_map;
  int64_t chunks() const { return fac + 2 * rows + 2 * mats + seg_map; }
};
Parts parts(int64_t tiles, int64_t segs, int heads, int keys, int dk, int dv, int dtype) {
  const int64_t DK = delta_dk(dk), dvp = (dv + 31) / 32 * 32;
  const int64_t in = dtype == MLCG_DTYPE_F32 ? 3 : dtype == MLCG_DTYPE_F16 ? 2 : 1;
  const int64_t mid = 3;  // pieces of what is computed
  return Parts{tiles * heads * (kDeltaFactors * kDeltaRows),
               tiles * keys * in * (DK / 8) * 256,
               tiles * heads * mid * kDeltaLower * 256,
               tiles * heads * mid * (dvp / 8) * 256,
               tiles * heads * mid * (dvp / 16) * (DK / 32) * 256,
               segs * heads * DK * dvp,
               segs * heads * mid * (DK * DK / 2)};
}

bool delta_ok(const DeltaArgs& a, int dtype) {
  for (int64_t row : {a.q_row, a.k_row, a.v_row})  // 64 rows are within 32 bits
    if (row < 0 || row >= (int64_t(1) << 22)) return false;
  return a.beads >= 0 && a.beads < (int64_t(1) << 31) - 256 && a.heads >= 1 && a.heads <= 1024 &&
         a.keys >= 1 && a.heads % a.keys == 0 && a.dk >= 8 && a.dk <= 128 && a.dk % 8 == 0 &&
         a.dv >= 8 && a.dv <= 128 && a.dv % 8 == 0 && dtype >= MLCG_DTYPE_F32 && dtype <= MLCG_DTYPE_BF16;
}

}  // namespace

extern "C" int64_t mlcg_gated_delta_floats(int64_t n_tiles, int64_t n_split, int heads,
                                           int key_heads, int dk, int dv, int dtype, int which) {
  if (n_tiles < 0 || n_split < 0 || heads < 1 || key_heads < 1 || dk < 1 || dk > 128 || dv < 1 ||
      dv > 128 || dtype < MLCG_DTYPE_F32 || dtype > MLCG_DTYPE_BF16)
    return -1;
  const Parts p = parts(n_tiles, n_split, heads, key_heads, dk, dv, dtype);
  switch (which) {
    case 0: return p.chunks();
    case 1: return p.chunks() + p.u + p.s0;
    case 2: return 2 * p.seg_state;
    case 3: return 2 * p.seg_state + p.u + p.s0;
    default: return -1;
  }
}

namespace {

// the arrays in `kept`: factors, k, q, T, P, the segments' maps, and u and S0
void place(DeltaArgs& a, DeltaEnds& e, float* kept, const Parts& p, bool train, bool split) {
  a.fac = kept;
  float* at = kept + p.fac;
  a.K = reinterpret_cast<float4*>(at);
  a.Q = reinterpret_cast<float4*>(at + p.rows);
  at += 2 * p.rows;
  a.T = reinterpret_cast<float4*>(at);
  a.P = reinterpret_cast<float4*>(at + p.mats);
  at += 2 * p.mats;
  e.seg_map = split ? reinterpret_cast<float4*>(at) : nullptr;
  at += p.seg_map;
  a.U = train ? reinterpret_cast<float4*>(at) : nullptr;
  a.S0 = train ? reinterpret_cast<float4*>(at + p.u) : nullptr;
}

}  // namespace

extern "C" int mlcg_gated_delta(
    const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides, const float* decay, const float* beta, int64_t beads,
    int heads, int key_heads, int dk, int dv, int dtype, const int32_t* tiles, int64_t n_tiles,
    const int32_t* segments, int64_t n_segments, const int32_t* segment_first, int64_t n_whole,
    int split, const uint8_t* keep, const float* state, float scale, int normalize, int reverse,
    void* out, float* last_state, float* kept, int64_t kept_floats, int train, float* workspace,
    int64_t workspace_floats, void* stream) {
  MLCG_REQUIRE(q_strides && k_strides && v_strides && key_heads >= 1 && n_tiles >= 0 &&
               n_tiles < kMostTiles && n_segments >= 0 && n_segments < kMostTiles &&
               n_whole >= 0 && n_whole <= n_segments);
  DeltaArgs a{q, k, v, q_strides[0], q_strides[1], k_strides[0], k_strides[1], v_strides[0],
              v_strides[1], decay, beta, keep, beads, heads, key_heads, heads / key_heads, dk, dv,
              (dv + 31) / 32 * 32, scale, normalize, reverse,
              reinterpret_cast<const int4*>(tiles), (int)n_tiles,
              reinterpret_cast<const int4*>(segments), segment_first, (int)n_segments,
              (int)n_whole, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  MLCG_REQUIRE(delta_ok(a, dtype));
  if (beads == 0 || n_tiles == 0) return MLCG_OK;
  MLCG_REQUIRE(q && k && v && decay && beta && tiles && segments && segment_first && out && kept &&
               n_whole >= 1);
  const Parts p = parts(n_tiles, split ? n_segments : 0, heads, key_heads, dk, dv, dtype);
  MLCG_REQUIRE(kept_floats >= p.chunks() + (train ? p.u + p.s0 : 0) &&
               workspace_floats >= 2 * p.seg_state && (!split || workspace) && aligned32(kept) &&
               aligned32(workspace));
  DeltaEnds e{state, last_state, nullptr, nullptr, nullptr};
  place(a, e, kept, p, train, split);
  if (split) e.seg_last = workspace;
  float* const init = split ? workspace + p.seg_state : nullptr;
  hipStream_t s = mlcg_stream(stream);
  if (dtype == MLCG_DTYPE_F32) return delta_forward<float>(a, out, e, init, s);
  if (dtype == MLCG_DTYPE_F16) return delta_forward<_Float16>(a, out, e, init, s);
  return delta_forward<__bf16>(a, out, e, init, s);
}

extern "C" int mlcg_gated_delta_backward(
    const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides, const float* decay, const float* beta, int64_t beads,
    int heads, int key_heads, int dk, int dv, int dtype, const int32_t* tiles, int64_t n_tiles,
    const int32_t* segments, int64_t n_segments, const int32_t* segment_first, int64_t n_whole,
    int split, const uint8_t* keep, float scale, int normalize, int reverse, const float* kept,
    int64_t kept_floats, const void* grad_out, const float* grad_last_state, void* grad_q,
    void* grad_k, void* grad_v, float* grad_decay, float* grad_beta, float* grad_state,
    float* workspace, int64_t workspace_floats, void* stream) {
  MLCG_REQUIRE(q_strides && k_strides && v_strides && key_heads >= 1 && n_tiles >= 1 &&
               n_tiles < kMostTiles && n_segments >= 1 && n_segments < kMostTiles &&
               n_whole >= 1 && n_whole <= n_segments);
  DeltaArgs a{q, k, v, q_strides[0], q_strides[1], k_strides[0], k_strides[1], v_strides[0],
              v_strides[1], decay, beta, keep, beads, heads, key_heads, heads / key_heads, dk, dv,
              (dv + 31) / 32 * 32, scale, normalize, reverse,
              reinterpret_cast<const int4*>(tiles), (int)n_tiles,
              reinterpret_cast<const int4*>(segments), segment_first, (int)n_segments,
              (int)n_whole, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  MLCG_REQUIRE(delta_ok(a, dtype) && beads >= 1);
  MLCG_REQUIRE(q && k && v && decay && beta && tiles && segments && segment_first && kept &&
               grad_out && grad_q && grad_k && grad_v && grad_decay && grad_beta && workspace);
  const Parts p = parts(n_tiles, split ? n_segments : 0, heads, key_heads, dk, dv, dtype);
  MLCG_REQUIRE(kept_floats >= p.chunks() + p.u + p.s0 &&
               workspace_floats >= 2 * p.seg_state + p.u + p.s0 && aligned32(kept) &&
               aligned32(workspace));
  DeltaEnds e{grad_last_state, nullptr, nullptr, nullptr, nullptr};
  place(a, e, const_cast<float*>(kept), p, true, split);
  float* at = workspace;
  const DeltaBack b{grad_out, grad_q, grad_k, grad_v, grad_decay, grad_beta,
                    grad_state, reinterpret_cast<float4*>(at), reinterpret_cast<float4*>(at + p.s0)};
  at += p.s0 + p.u;
  if (split) e.seg_last = at;
  float* const init = split ? at + p.seg_state : nullptr;
  hipStream_t s = mlcg_stream(stream);
  if (dtype == MLCG_DTYPE_F32) return delta_backward<float>(a, b, e, init, s);
  if (dtype == MLCG_DTYPE_F16) return delta_backward<_Float16>(a, b, e, init, s);
  return delta_backward<__bf16>(a, b, e, init, s);
}

extern "C" int mlcg_gated_delta_step(const void* q, const int64_t* q_strides, const void* k,
                                     const int64_t* k_strides, const void* v,
                                     const int64_t* v_strides, const float* decay,
                                     const float* beta, int64_t batch, int heads, int key_heads,
                                     int dk, int dv, int dtype, const float* state, float scale,
                                     int normalize, void* out, float* next_state, void* stream) {
  MLCG_REQUIRE(q_strides && k_strides && v_strides && batch >= 0 && batch < (int64_t(1) << 31) &&
               heads >= 1 && heads <= 1024 && key_heads >= 1 && heads % key_heads == 0 &&
               dk >= 1 && dk <= 128 && dv >= 1 && dv <= 128);
  if (batch == 0) return MLCG_OK;
  MLCG_REQUIRE(q && k && v && decay && beta && state && out && next_state);
  const StepArgs a{q, k, v, q_strides[0], q_strides[1], k_strides[0], k_strides[1], v_strides[0],
                   v_strides[1], decay, beta, state, batch, heads, heads / key_heads, dk, dv, scale,
                   normalize, next_state, out};
  hipStream_t s = mlcg_stream(stream);
  switch (dtype) {
    case MLCG_DTYPE_F32: return step_of<float>(a, s);
    case MLCG_DTYPE_F16: return step_of<_Float16>(a, s);
    case MLCG_DTYPE_BF16: return step_of<__bf16>(a, s);
    default: return MLCG_ERR_ARGUMENT;
  }
}
