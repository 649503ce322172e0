// Group norm with an activation over chains of beads, channels last (gfx950).
//
// x is [S, C], the beads of all chains one after the other; the channels fall
// into G groups of P = C / G.  For every chain and group, over its n = len P
// values,  mean = sum x / n,  var = sum (x - mean)^2 / n,
//   hat = (x - mean) / sqrt(var + eps),  z = hat w_c + b_c,  y = act(z);
// backward, with dz = dy act'(z), A_c = sum dz and B_c = sum dz hat over the
// chain's beads (summed over the chains: the gradients of b_c and w_c),
//   dx = (dz w_c - sum_g w_c A_c / n - hat sum_g w_c B_c / n) / sqrt(var + eps).
//
// A workgroup's threads form TR rows x TC columns, a column one vector of W
// channels (16 bytes), and go down a chain or a slab of it NV rows of a thread
// at a time, with all loads of such a step in flight.
//
// Statistics: the mean of the first step's values, rounded, is the pivot p;
// s = sum (x - p) and q = sum (x - p)^2 give mean = p + s / n and var =
// (q - s^2 / n) / n.  As p is the mean of n1 of the n values, (p - mean)^2 <=
// var n / n1: the difference loses a factor of 1 + n / n1 at most (for a
// chain of one step nothing).  What the rounding of the mean leaves out is
// kept beside it, so that a deviation of a value far from zero is as exact as
// the value.  Every sum has a fixed order.
//
// Chains of up to kOneRows beads, or many chains: a workgroup takes a whole
// chain, twice over its rows, the second time from the cache; one launch
// forward, and backward one that writes dx and each workgroup's sums by
// channel over the chains it takes, and one that joins these.  Few long
// chains: slabs of them, joined in slab order, then a second reading.
//
// Measured: 2048 chains of up to 268 beads, 128 channels, bf16, silu: forward
// 47 us, backward 106 + 6; three and five passes over 79.5 MB, the second
// readings from the last cache: 5.0 and 3.75 TB/s against the 5.2 of a large
// copy.  The backward's vector instructions (the activation's derivative in
// both passes) take half of the SIMDs' cycles.  With the chain kept in
// registers (20 rows of a thread, two waves a SIMD) in place of the second
// reading: 57 and 244 us, as too few waves are left to hide the loads; 192
// chains of up to 80 in fp32 gained 2 us of 12 and of 15, less than such
// calls' launches cost.  One chain of 120001 beads of 256 channels, fp32, 123 MB
// a pass: statistics 22 us, application 38, backward 45 and 63, 5.4 to 6.5 TB/s
// over their one, two, two and three passes, whose number is what bounds it; as
// much with slabs of 128 and of 64 rows.
#include <algorithm>
#include <type_traits>

#include "chain.h"

namespace {

constexpr int kMaxWidth = 1024;
constexpr int kSlabRows = 256;

struct NormShape {
  const int4* tiles;  // (chain's first row, chain's length, slab's first row in it, chain)
  int n_tiles, size;  // slabs, and rows of a slab
  int C, G, TC, TR;
  int64_t chains;
};

__device__ __forceinline__ void act_z(int act, float z, float& y, float& d) {
  if (act == MLCG_ACT_NONE) {
    y = z;
    d = 1.0f;
  } else if (act == MLCG_ACT_SILU) {
    const float s = mlcg_sigmoid(z);
    y = z * s;
    d = fmaf(y, 1.0f - s, s);
  } else {
    float d2;
    mlcg_act(act, z, y, d, d2);
  }
}

__device__ __forceinline__ float act_value(int act, float z) {
  if (act == MLCG_ACT_NONE) return z;
  if (act == MLCG_ACT_SILU) return z * mlcg_sigmoid(z);
  return mlcg_act_value(act, z);
}

template <typename T, int W>
struct Vec {
  typedef T type __attribute__((ext_vector_type(W)));
};
template <typename T>
struct Vec<T, 1> {
  struct type {
    T x;
    __device__ T operator[](int) const { return x; }
    __device__ T& operator[](int) { return x; }
  };
};

// A thread's place among the rows and columns of a workgroup.
struct Place {
  int row, col;
  bool in;
  __device__ __forceinline__ Place(const NormShape& sh)
      : row(threadIdx.x / sh.TC), col(threadIdx.x % sh.TC), in(row < sh.TR) {}
};

// Rows of a thread's step: 16 channels of 16 bits, or 16 of 32 bits, in flight
// for each array; more would cost the waves that hide the latency.
template <int W>
constexpr int step_rows() {
  return W == 8 ? 2 : 4;
}

// the rows r0 + row + v TR, v < NV, of a column; those at or past `rows` are
// loaded as the last one
template <typename T, int W>
__device__ __forceinline__ void load_step(const NormShape& sh, const Place& at, const T* x,
                                          int64_t ld, int r0, int rows,
                                          typename Vec<T, W>::type (&out)[step_rows<W>()]) {
  constexpr int kNV = step_rows<W>();
#pragma unroll
  for (int v = 0; v < kNV; ++v) {
    const int r = min(r0 + at.row + v * sh.TR, rows - 1);
    out[v] = *reinterpret_cast<const typename Vec<T, W>::type*>(x + r * ld + at.col * W);
  }
}

__device__ __forceinline__ bool step_row(const NormShape& sh, const Place& at, int r0, int v,
                                         int rows) {
  return at.in && r0 + at.row + v * sh.TR < rows;
}

// Sums of K values a thread over the rows of its column: the rows that lie
// in one wave by a butterfly (TC divides 64), the rest through LDS.
// sums[col K + k], valid for every thread on return.
template <int K>
__device__ void column_sums(const NormShape& sh, const float (&v)[K], float* red, float* sums) {
  const int tid = threadIdx.x, nt = blockDim.x;
  const int col = tid % sh.TC, row = tid / sh.TC;
  const bool in_wave = sh.TC < 64 && 64 % sh.TC == 0;
  const int rows = in_wave ? nt / 64 : sh.TR;
  __syncthreads();  // red and sums may still be read
  if (in_wave) {
    float s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = v[k];
    for (int o = sh.TC; o < 64; o <<= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] += __shfl_xor(s[k], o, 64);
    if ((tid & 63) < sh.TC)
#pragma unroll
      for (int k = 0; k < K; ++k) red[((tid >> 6) * sh.TC + col) * K + k] = s[k];
  } else if (row < sh.TR) {
#pragma unroll
    for (int k = 0; k < K; ++k) red[(row * sh.TC + col) * K + k] = v[k];
  }
  __syncthreads();
  const int nc = sh.TC * K;
  for (int c = tid; c < nc; c += nt) {
    float t = 0.0f;
    for (int r = 0; r < rows; ++r) t += red[r * nc + c];
    sums[c] = t;
  }
  __syncthreads();
}

// a = the sum of the group's columns' first (of two, second) values, a wave a
// group: f(group, a, b) on its first lane.
template <typename F>
__device__ __forceinline__ void group_sums(const float* sums, int groups, int per, int values,
                                           F f) {
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < groups; g += blockDim.x >> 6) {
    float a = 0.0f, b = 0.0f;
    for (int c = lane; c < per; c += 64) {
      a += sums[values * (g * per + c)];
      if (values > 1) b += sums[values * (g * per + c) + 1];
    }
    a = mlcg_wave_sum(a);
    if (values > 1) b = mlcg_wave_sum(b);
    if (lane == 0) f(g, a, b);
  }
  __syncthreads();
}

// The statistics of `rows` rows from x on, by group, into LDS: the mean, its
// remainder and the sum of squared deviations.  K sums a vector, of W / K
// channels of one group each.
template <typename T, int W, int K>
__device__ __forceinline__ void row_stats(const NormShape& sh, const Place& at, const T* x,
                                          int64_t ld, int rows, float* lds, float* mean,
                                          float* rest, float* m2) {
  constexpr int kNV = step_rows<W>();
  float* red = lds;                         // blockDim 2 K
  float* sums = red + blockDim.x * 2 * K;   // TC 2 K
  const int P = sh.C / sh.G, per = P / (W / K);
  typename Vec<T, W>::type xv[kNV];
  load_step<T, W>(sh, at, x, ld, 0, rows, xv);
  float s[K] = {};
#pragma unroll
  for (int v = 0; v < kNV; ++v)
    if (step_row(sh, at, 0, v, rows))
#pragma unroll
      for (int j = 0; j < W; ++j) s[j / (W / K)] += (float)xv[v][j];
  column_sums<K>(sh, s, red, sums);
  const float first = 1.0f / ((float)min(rows, kNV * sh.TR) * (float)P);
  // the pivot comes back from LDS: rounded, as it is used
  group_sums(sums, sh.G, per, 1, [&](int g, float a, float) { mean[g] = a * first; });
  float p[W], d2[2 * K] = {};
#pragma unroll
  for (int j = 0; j < W; ++j) p[j] = mean[(at.col * W + j) / P];
  for (int r0 = 0;;) {
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      const bool ok = step_row(sh, at, r0, v, rows);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float d = ok ? (float)xv[v][j] - p[j] : 0.0f;
        const int k = j / (W / K);
        d2[2 * k] += d;
        d2[2 * k + 1] = fmaf(d, d, d2[2 * k + 1]);
      }
    }
    r0 += kNV * sh.TR;
    if (r0 >= rows) break;
    load_step<T, W>(sh, at, x, ld, r0, rows, xv);
  }
  column_sums<2 * K>(sh, d2, red, sums);
  const float inv = 1.0f / ((float)rows * (float)P);
  group_sums(sums, sh.G, per, 2, [&](int g, float a, float q) {
    const float pivot = mean[g], step = a * inv;
    float hi = pivot + step;
    asm("" : "+v"(hi));  // the rounded sum, as it is kept
    mean[g] = hi;
    rest[g] = (pivot - hi) + step;
    m2[g] = fmaxf(0.0f, q - step * a);
  });
}

// What the elementwise passes need of a thread's channels.
template <typename T, int W>
struct Channels {
  float mu[W], lo[W], rs[W], w[W], b[W];
  __device__ __forceinline__ Channels(int P, const Place& at, const float* mean,
                                      const float* rest, const float* rstd, const T* weight,
                                      const T* bias) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int c = at.col * W + j;
      mu[j] = mean[c / P];
      lo[j] = rest[c / P];
      rs[j] = rstd[c / P];
      w[j] = (float)weight[c];
      b[j] = (float)bias[c];
    }
  }
  // the remainder of the mean is below what 16 bits hold of a value
  __device__ __forceinline__ float hat(int j, float x) const {
    return sizeof(T) == 4 ? ((x - mu[j]) - lo[j]) * rs[j] : (x - mu[j]) * rs[j];
  }
};

template <typename T, int W>
__device__ __forceinline__ void apply_rows(const NormShape& sh, const Place& at,
                                           const Channels<T, W>& ch, const T* x, int64_t ld,
                                           int rows, int act, T* y) {
  constexpr int kNV = step_rows<W>();
  for (int r0 = 0; r0 < rows; r0 += kNV * sh.TR) {
    typename Vec<T, W>::type xv[kNV];
    load_step<T, W>(sh, at, x, ld, r0, rows, xv);
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      typename Vec<T, W>::type out;
#pragma unroll
      for (int j = 0; j < W; ++j)
        out[j] = (T)act_value(act, fmaf(ch.hat(j, (float)xv[v][j]), ch.w[j], ch.b[j]));
      if (step_row(sh, at, r0, v, rows))
        *reinterpret_cast<typename Vec<T, W>::type*>(
            y + (int64_t)(r0 + at.row + v * sh.TR) * sh.C + at.col * W) = out;
    }
  }
}

// One chain a workgroup.
template <typename T, int W, int K, int NT>
__global__ __launch_bounds__(NT) void norm_chain_kernel(NormShape sh, const T* __restrict__ x,
                                                          int64_t ld, const T* __restrict__ w,
                                                          const T* __restrict__ b, float eps,
                                                          int act, T* __restrict__ y,
                                                          float* __restrict__ stats) {
  extern __shared__ float lds[];
  float* mean = lds;  // G each
  float* rest = mean + sh.G;
  float* rstd = rest + sh.G;
  const int4 t = sh.tiles[blockIdx.x];
  const Place at(sh);
  const int P = sh.C / sh.G;
  const T* xt = x + (int64_t)t.x * ld;
  row_stats<T, W, K>(sh, at, xt, ld, t.y, rstd + sh.G, mean, rest, rstd);
  const float inv = 1.0f / ((float)t.y * (float)P);
  for (int g = threadIdx.x; g < sh.G; g += blockDim.x) {
    const float rs = 1.0f / sqrtf(rstd[g] * inv + eps);
    rstd[g] = rs;
    const int64_t k = (int64_t)t.w * sh.G + g, all = sh.chains * sh.G;
    stats[k] = mean[g];
    stats[all + k] = rest[g];
    stats[2 * all + k] = rs;
  }
  __syncthreads();
  const Channels<T, W> ch(P, at, mean, rest, rstd, w, b);
  apply_rows<T, W>(sh, at, ch, xt, ld, t.y, act, y + (int64_t)t.x * sh.C);
}

// (mean, its remainder, M2) of every group of a slab -> part[g][tile]
template <typename T, int W, int K, int NT>
__global__ __launch_bounds__(NT) void norm_part_kernel(NormShape sh, const T* __restrict__ x,
                                                         int64_t ld, float4* __restrict__ part) {
  extern __shared__ float lds[];
  float* mean = lds;  // G each
  float* rest = mean + sh.G;
  float* m2 = rest + sh.G;
  const int4 t = sh.tiles[blockIdx.x];
  const Place at(sh);
  row_stats<T, W, K>(sh, at, x + ((int64_t)t.x + t.z) * ld, ld, min(sh.size, t.y - t.z),
                           m2 + sh.G, mean, rest, m2);
  for (int g = threadIdx.x; g < sh.G; g += blockDim.x)
    part[(int64_t)g * sh.n_tiles + blockIdx.x] = make_float4(mean[g], rest[g], m2[g], 0.0f);
}

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = mlcg_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// A chain's statistics from its slabs', a workgroup a group: with n_t values of
// mean m_t and sum of squares M_t,  mean = sum n_t m_t / n  and  M = sum M_t +
// n_t (m_t - mean)^2.  stats: the mean, its remainder and 1 / sqrt(var + eps),
// [3][chains][G].
__global__ __launch_bounds__(256) void norm_join_kernel(NormShape sh,
                                                        const int32_t* __restrict__ first_tile,
                                                        const float4* __restrict__ part,
                                                        float eps, float* __restrict__ stats) {
  __shared__ float red[4];
  const int chain = blockIdx.x, g = blockIdx.y;
  const int t0 = first_tile[chain];
  if (t0 < 0) return;  // an empty chain has no slab and no statistics
  const int len = sh.tiles[t0].y;
  const int count = (len + sh.size - 1) / sh.size;
  const float4* p = part + (int64_t)g * sh.n_tiles + t0;
  const float n = (float)len;
  float s = 0.0f;
  for (int t = threadIdx.x; t < count; t += 256)
    s = fmaf((float)min(sh.size, len - t * sh.size), p[t].x, s);
  const float mu = block_sum(s, red) / n;
  float c = 0.0f;
  for (int t = threadIdx.x; t < count; t += 256)
    c = fmaf((float)min(sh.size, len - t * sh.size), (p[t].x - mu) + p[t].y, c);
  const float lo = block_sum(c, red) / n;
  const float P = (float)(sh.C / sh.G);
  float m2 = 0.0f;
  for (int t = threadIdx.x; t < count; t += 256) {
    const float d = (p[t].x - mu) + (p[t].y - lo);
    m2 += fmaf((float)min(sh.size, len - t * sh.size) * P * d, d, p[t].z);
  }
  m2 = block_sum(m2, red);
  if (threadIdx.x == 0) {
    const int64_t at = (int64_t)chain * sh.G + g, all = sh.chains * sh.G;
    stats[at] = mu;
    stats[all + at] = lo;
    stats[2 * all + at] = 1.0f / sqrtf(m2 / (n * P) + eps);
  }
}

template <typename T, int W, int NT>
__global__ __launch_bounds__(NT) void norm_apply_kernel(
    NormShape sh, const T* __restrict__ x, int64_t ld, const T* __restrict__ w,
    const T* __restrict__ b, const float* __restrict__ stats, int act, T* __restrict__ y) {
  const int4 t = sh.tiles[blockIdx.x];
  const Place at(sh);
  if (!at.in) return;
  const float* st = stats + (int64_t)t.w * sh.G;
  const int64_t all = sh.chains * sh.G;
  const Channels<T, W> ch(sh.C / sh.G, at, st, st + all, st + 2 * all, w, b);
  const int64_t first = (int64_t)t.x + t.z;
  apply_rows<T, W>(sh, at, ch, x + first * ld, ld, min(sh.size, t.y - t.z), act,
                   y + first * sh.C);
}

// ---------------------------------------------------------------------------
// Backward

// (A_c, B_c) of rows from x, dy on -> sums[2 c], sums[2 c + 1]
template <typename T, int W>
__device__ __forceinline__ void row_grads(const NormShape& sh, const Place& at,
                                          const Channels<T, W>& ch, const T* x, int64_t ld,
                                          const T* dy, int rows, int act, float* red,
                                          float* sums) {
  constexpr int kNV = step_rows<W>();
  float ab[2 * W] = {};
  for (int r0 = 0; r0 < rows; r0 += kNV * sh.TR) {
    typename Vec<T, W>::type xv[kNV], gv[kNV];
    load_step<T, W>(sh, at, x, ld, r0, rows, xv);
    load_step<T, W>(sh, at, dy, sh.C, r0, rows, gv);
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      const bool ok = step_row(sh, at, r0, v, rows);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float hat = ch.hat(j, (float)xv[v][j]);
        float yv, d;
        act_z(act, fmaf(hat, ch.w[j], ch.b[j]), yv, d);
        const float dz = ok ? (float)gv[v][j] * d : 0.0f;
        ab[2 * j] += dz;
        ab[2 * j + 1] = fmaf(dz, hat, ab[2 * j + 1]);
      }
    }
  }
  column_sums<2 * W>(sh, ab, red, sums);
}

// dx of rows from x, dy on, with the groups' sums of w A and w B
template <typename T, int W>
__device__ __forceinline__ void row_dx(const NormShape& sh, const Place& at,
                                       const Channels<T, W>& ch, const T* x, int64_t ld,
                                       const T* dy, int rows, int act, const float* s1,
                                       const float* s2, float inv, T* dx) {
  constexpr int kNV = step_rows<W>();
  const int P = sh.C / sh.G;
  float m1[W], m2[W];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    m1[j] = s1[(at.col * W + j) / P] * inv;
    m2[j] = s2[(at.col * W + j) / P] * inv;
  }
  for (int r0 = 0; r0 < rows; r0 += kNV * sh.TR) {
    typename Vec<T, W>::type xv[kNV], gv[kNV];
    load_step<T, W>(sh, at, x, ld, r0, rows, xv);
    load_step<T, W>(sh, at, dy, sh.C, r0, rows, gv);
#pragma unroll
    for (int v = 0; v < kNV; ++v) {
      typename Vec<T, W>::type out;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float hat = ch.hat(j, (float)xv[v][j]);
        float yv, d;
        act_z(act, fmaf(hat, ch.w[j], ch.b[j]), yv, d);
        // rounded as in the sums, not fused with the difference: the gradient
        // of a group of one value is then 0, not its rounding error times up
        // to 1 / sqrt(eps)
        float dh = (float)gv[v][j] * d * ch.w[j];
        asm("" : "+v"(dh));
        out[j] = (T)((dh - m1[j] - hat * m2[j]) * ch.rs[j]);
      }
      if (step_row(sh, at, r0, v, rows))
        *reinterpret_cast<typename Vec<T, W>::type*>(
            dx + (int64_t)(r0 + at.row + v * sh.TR) * sh.C + at.col * W) = out;
    }
  }
}

// dx of the chains blockIdx.x, blockIdx.x + gridDim.x, ... and the sums of A_c
// and B_c over them -> part[workgroup][2][C].  A chain needs the groups' sums
// alone (K of w A and of w B a vector); the channels' stay in the threads'
// registers until the last chain.
template <typename T, int W, int K, int NT>
__global__ __launch_bounds__(NT) void norm_chain_bwd_kernel(
    NormShape sh, const T* __restrict__ x, int64_t ld, const T* __restrict__ dy,
    const T* __restrict__ w, const T* __restrict__ b, const float* __restrict__ stats, int act,
    T* __restrict__ dx, float* __restrict__ part) {
  constexpr int kNV = step_rows<W>();
  extern __shared__ float lds[];
  float* red = lds;              // NT 2 W
  float* sums = red + NT * 2 * W;  // 2 C
  float* s1 = sums + 2 * sh.C;   // G each
  float* s2 = s1 + sh.G;
  const Place at(sh);
  const int P = sh.C / sh.G;
  const int64_t all = sh.chains * sh.G;
  float ab[2 * W] = {};
  for (int tile = blockIdx.x; tile < sh.n_tiles; tile += gridDim.x) {
    const int4 t = sh.tiles[tile];
    const float* st = stats + (int64_t)t.w * sh.G;
    const Channels<T, W> ch(P, at, st, st + all, st + 2 * all, w, b);
    const T* xt = x + (int64_t)t.x * ld;
    const T* dt = dy + (int64_t)t.x * sh.C;
    float wab[2 * K] = {};
    for (int r0 = 0; r0 < t.y; r0 += kNV * sh.TR) {
      typename Vec<T, W>::type xv[kNV], gv[kNV];
      load_step<T, W>(sh, at, xt, ld, r0, t.y, xv);
      load_step<T, W>(sh, at, dt, sh.C, r0, t.y, gv);
#pragma unroll
      for (int v = 0; v < kNV; ++v) {
        const bool ok = step_row(sh, at, r0, v, t.y);
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const float hat = ch.hat(j, (float)xv[v][j]);
          float yv, d;
          act_z(act, fmaf(hat, ch.w[j], ch.b[j]), yv, d);
          const float dz = ok ? (float)gv[v][j] * d : 0.0f;
          ab[2 * j] += dz;
          ab[2 * j + 1] = fmaf(dz, hat, ab[2 * j + 1]);
          float dh = dz * ch.w[j];
          asm("" : "+v"(dh));  // rounded, as in row_dx
          const int k = j / (W / K);
          wab[2 * k] += dh;
          wab[2 * k + 1] = fmaf(dh, hat, wab[2 * k + 1]);
        }
      }
    }
    column_sums<2 * K>(sh, wab, red, sums);
    group_sums(sums, sh.G, P / (W / K), 2, [&](int g, float a, float q) {
      s1[g] = a;
      s2[g] = q;
    });
    row_dx<T, W>(sh, at, ch, xt, ld, dt, t.y, act, s1, s2, 1.0f / ((float)t.y * (float)P),
                 dx + (int64_t)t.x * sh.C);
  }
  column_sums<2 * W>(sh, ab, red, sums);
  for (int c = threadIdx.x; c < sh.C; c += NT) {
    part[(int64_t)blockIdx.x * 2 * sh.C + c] = sums[2 * c];
    part[(int64_t)blockIdx.x * 2 * sh.C + sh.C + c] = sums[2 * c + 1];
  }
}

// (A_c, B_c) of a slab -> part[tile][2][C]
template <typename T, int W, int NT>
__global__ __launch_bounds__(NT) void norm_bwd_part_kernel(
    NormShape sh, const T* __restrict__ x, int64_t ld, const T* __restrict__ dy,
    const T* __restrict__ w, const T* __restrict__ b, const float* __restrict__ stats, int act,
    float* __restrict__ part) {
  extern __shared__ float lds[];
  float* red = lds;                        // blockDim 2 W
  float* sums = red + blockDim.x * 2 * W;  // 2 C
  const int4 t = sh.tiles[blockIdx.x];
  const Place at(sh);
  const int64_t all = sh.chains * sh.G, first = (int64_t)t.x + t.z;
  const float* st = stats + (int64_t)t.w * sh.G;
  const Channels<T, W> ch(sh.C / sh.G, at, st, st + all, st + 2 * all, w, b);
  row_grads<T, W>(sh, at, ch, x + first * ld, ld, dy + first * sh.C, min(sh.size, t.y - t.z), act,
                  red, sums);
  for (int c = threadIdx.x; c < sh.C; c += blockDim.x) {
    part[(int64_t)blockIdx.x * 2 * sh.C + c] = sums[2 * c];
    part[(int64_t)blockIdx.x * 2 * sh.C + sh.C + c] = sums[2 * c + 1];
  }
}

// out[seg][col] = sum over the segment's rows of in[row][col], `cols` columns:
// 8 columns x 128 slices of the rows a workgroup, the slices joined in order.
// Segments are the slabs of a chain (first_tile, tiles), or all `rows` rows.
template <typename O>
__global__ __launch_bounds__(1024) void norm_rows_kernel(const float* __restrict__ in, int cols,
                                                         const int32_t* __restrict__ first_tile,
                                                         const int4* __restrict__ tiles, int size,
                                                         int rows, O* __restrict__ out) {
  __shared__ float red[128][9];
  const int col = blockIdx.y * 8 + (threadIdx.x & 7), slice = threadIdx.x >> 3;
  int64_t r0 = 0;
  int n = rows;
  if (first_tile) {
    const int t0 = first_tile[blockIdx.x];
    r0 = t0 < 0 ? 0 : t0;
    n = t0 < 0 ? 0 : (tiles[t0].y + size - 1) / size;
  }
  float s = 0.0f;
  if (col < cols) {
#pragma unroll 8
    for (int r = slice; r < n; r += 128) s += in[(r0 + r) * cols + col];
  }
  red[slice][threadIdx.x & 7] = s;
  __syncthreads();
  if (threadIdx.x < 64) {  // 8 lanes a column: 16 slices each, then a butterfly
    const int c = threadIdx.x & 7;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[(threadIdx.x >> 3) * 16 + k][c];
    t += __shfl_xor(t, 8, 64);
    t += __shfl_xor(t, 16, 64);
    t += __shfl_xor(t, 32, 64);
    if (threadIdx.x < 8 && col < cols) out[(int64_t)blockIdx.x * cols + col] = (O)t;
  }
}

template <typename T, int W, int NT>
__global__ __launch_bounds__(NT) void norm_bwd_apply_kernel(
    NormShape sh, const T* __restrict__ x, int64_t ld, const T* __restrict__ dy,
    const T* __restrict__ w, const T* __restrict__ b, const float* __restrict__ stats,
    const float* __restrict__ chain_sums, int act, T* __restrict__ dx) {
  extern __shared__ float lds[];
  float* wa = lds;              // 2 C: (w A, w B) by channel
  float* s1 = wa + 2 * sh.C;    // G each
  float* s2 = s1 + sh.G;
  const int4 t = sh.tiles[blockIdx.x];
  const Place at(sh);
  const int P = sh.C / sh.G;
  const float* a = chain_sums + (int64_t)t.w * 2 * sh.C;
  for (int c = threadIdx.x; c < sh.C; c += blockDim.x) {
    wa[2 * c] = (float)w[c] * a[c];
    wa[2 * c + 1] = (float)w[c] * a[sh.C + c];
  }
  __syncthreads();
  group_sums(wa, sh.G, P, 2, [&](int g, float p, float q) {
    s1[g] = p;
    s2[g] = q;
  });
  const int64_t all = sh.chains * sh.G, first = (int64_t)t.x + t.z;
  const float* st = stats + (int64_t)t.w * sh.G;
  const Channels<T, W> ch(P, at, st, st + all, st + 2 * all, w, b);
  row_dx<T, W>(sh, at, ch, x + first * ld, ld, dy + first * sh.C, min(sh.size, t.y - t.z), act, s1,
               s2, 1.0f / ((float)t.y * (float)P), dx + first * sh.C);
}

// ---------------------------------------------------------------------------
// Launches

struct NormArgs {
  const void *x, *dy, *w, *b;
  int64_t ld, chains;
  const int4 *tiles, *whole;
  const int32_t* first_tile;
  int n_tiles, n_whole, max_len, C, G, act;
  float eps;
};

// A chain a workgroup where chains are short, or many of like lengths.  A longer
// one among many is one workgroup's work, about 50 us for each of its slabs
// forward and backward, so that it is slabs for all where it has more of them
// than a compute unit's share of the slabs or chains (a chain's joins cost 0.14
// us).  128 channels in fp32, forward and backward, a chain a workgroup / slabs:
// 600 chains of 100 and one of 3000 609 / 136 us, 512 of 100 and one of 50000
// 10060 / 139, 20000 of 30 and one of 50000 10857 / 2198; of like lengths, 512 of
// 5000 2032 / 2039, 600 of 1500 792 / 789.
constexpr int kOneRows = 1024, kOneChains = 512;

bool by_chain(int64_t max_len, int64_t n_whole, int64_t n_tiles, int64_t chains) {
  const int64_t longest = (max_len + kSlabRows - 1) / kSlabRows;
  return max_len <= kOneRows ||
         (n_whole >= kOneChains && longest <= std::max(n_tiles, chains) / 256);
}

// Threads of a workgroup: a column of every vector of a row, and at least 4
// rows of them where a row has no more than 256 vectors; twice as many where
// few chains leave compute units idle and one takes more than a step (192
// chains of up to 80 beads x 128 in fp32, both directions: 25 us against 31;
// 2048 of up to 268 in bf16: 257 against 199).
int norm_threads(const NormArgs& a, int W) {
  const int tc = a.C / W;
  if (tc > 64) return 1024;
  return by_chain(a.max_len, a.n_whole, a.n_tiles, a.chains) && a.n_whole <= 256 &&
                 a.max_len > 4 * (256 / tc)
             ? 512
             : 256;
}

// Sums a vector of W channels: one for each of its groups where they divide
// it, or one where it lies in one, or else one a channel.
int vector_sums(int W, int P) { return P % W == 0 ? 1 : W % P == 0 ? W / P : W; }

template <int W>
NormShape norm_shape(const NormArgs& a, bool one, int nt) {
  NormShape sh;
  sh.tiles = one ? a.whole : a.tiles;
  sh.n_tiles = one ? a.n_whole : a.n_tiles;
  sh.size = one ? a.max_len : kSlabRows;
  sh.C = a.C;
  sh.G = a.G;
  sh.TC = a.C / W;
  sh.TR = nt / sh.TC;
  sh.chains = a.chains;
  return sh;
}

// LDS above 64 KiB has to be asked for.
template <typename F>
int allow(F f, unsigned lds) {
  if (lds > 65536u &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(f),
                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
    return MLCG_ERR_LAUNCH;
  return MLCG_OK;
}

template <typename T, int W, int K, int NT>
int norm_fwd(const NormArgs& a, void* y, float* stats, float* ws, hipStream_t s) {
  const bool one = by_chain(a.max_len, a.n_whole, a.n_tiles, a.chains);
  const NormShape sh = norm_shape<W>(a, one, NT);
  constexpr int nt = NT;
  const unsigned lds = (unsigned)((3 * sh.G + (nt + sh.TC) * 2 * K) * sizeof(float));
  const T *x = (const T*)a.x, *w = (const T*)a.w, *b = (const T*)a.b;
  if (one) {
    auto f = norm_chain_kernel<T, W, K, NT>;
    if (int e = allow(f, lds)) return e;
    hipLaunchKernelGGL(f, dim3(sh.n_tiles), dim3(nt), lds, s, sh, x, a.ld, w, b, a.eps, a.act,
                       (T*)y, stats);
    return mlcg_launch_status();
  }
  float4* part = reinterpret_cast<float4*>(ws);
  auto f = norm_part_kernel<T, W, K, NT>;
  if (int e = allow(f, lds)) return e;
  hipLaunchKernelGGL(f, dim3(sh.n_tiles), dim3(nt), lds, s, sh, x, a.ld, part);
  hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)sh.chains, sh.G), dim3(256), 0, s, sh,
                     a.first_tile, part, a.eps, stats);
  hipLaunchKernelGGL((norm_apply_kernel<T, W, NT>), dim3(sh.n_tiles), dim3(nt), 0, s, sh, x, a.ld,
                     w, b, stats, a.act, (T*)y);
  return mlcg_launch_status();
}

template <typename T, int W, int K, int NT>
int norm_bwd(const NormArgs& a, const float* stats, void* dx, void* dbw, float* ws,
             hipStream_t s) {
  const bool one = by_chain(a.max_len, a.n_whole, a.n_tiles, a.chains);
  const NormShape sh = norm_shape<W>(a, one, NT);
  constexpr int nt = NT;
  const T *x = (const T*)a.x, *dy = (const T*)a.dy, *w = (const T*)a.w, *b = (const T*)a.b;
  const unsigned cols = mlcg_div_up(2 * sh.C, 8);
  if (one) {
    const unsigned lds = (unsigned)((nt * 2 * W + 2 * sh.C + 2 * sh.G) * sizeof(float));
    auto f = norm_chain_bwd_kernel<T, W, K, NT>;
    if (int e = allow(f, lds)) return e;
    const int groups = std::min(sh.n_tiles, 2048);
    hipLaunchKernelGGL(f, dim3(groups), dim3(nt), lds, s, sh, x, a.ld, dy, w, b, stats, a.act,
                       (T*)dx, ws);
    hipLaunchKernelGGL(norm_rows_kernel<T>, dim3(1, cols), dim3(1024), 0, s, ws, 2 * sh.C,
                       nullptr, nullptr, 1, groups, (T*)dbw);
    return mlcg_launch_status();
  }
  const unsigned lds = (unsigned)((nt * 2 * W + 2 * sh.C) * sizeof(float));
  auto f = norm_bwd_part_kernel<T, W, NT>;
  if (int e = allow(f, lds)) return e;
  float* part = ws;
  float* chain_sums = ws + (int64_t)sh.n_tiles * 2 * sh.C;
  hipLaunchKernelGGL(f, dim3(sh.n_tiles), dim3(nt), lds, s, sh, x, a.ld, dy, w, b, stats, a.act,
                     part);
  // chains on the grid's first axis: the second one ends at 65535
  hipLaunchKernelGGL(norm_rows_kernel<float>, dim3((unsigned)sh.chains, cols), dim3(1024), 0, s,
                     part, 2 * sh.C, a.first_tile, sh.tiles, sh.size, 0, chain_sums);
  hipLaunchKernelGGL((norm_bwd_apply_kernel<T, W, NT>), dim3(sh.n_tiles), dim3(nt),
                     (unsigned)((2 * sh.C + 2 * sh.G) * sizeof(float)), s, sh, x, a.ld, dy, w, b,
                     stats, chain_sums, a.act, (T*)dx);
  hipLaunchKernelGGL(norm_rows_kernel<T>, dim3(1, cols), dim3(1024), 0, s, chain_sums, 2 * sh.C,
                     nullptr, nullptr, 1, (int)sh.chains, (T*)dbw);
  return mlcg_launch_status();
}

// 16-byte vectors of channels, where every row begins at a multiple of them
template <typename T>
bool norm_vec(const NormArgs& a, const void* out) {
  constexpr int W = 16 / sizeof(T);
  return a.C % W == 0 && a.ld % W == 0 && chain_aligned16(a.x) && chain_aligned16(a.dy) &&
         chain_aligned16(out);
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == MLCG_DTYPE_F32) return f(float{});
  if (dtype == MLCG_DTYPE_F16) return f(_Float16{});
  return f(__bf16{});
}

template <int N>
using Int = std::integral_constant<int, N>;

template <int W, typename F>
int by_shape(const NormArgs& a, bool vec, F f) {
  auto threads = [&](auto w, auto k) {
    const int nt = norm_threads(a, decltype(w)::value);
    return nt == 256 ? f(w, k, Int<256>()) : nt == 512 ? f(w, k, Int<512>()) : f(w, k, Int<1024>());
  };
  if (!vec) return threads(Int<1>(), Int<1>());
  const int k = vector_sums(W, a.C / a.G);
  if (k == 1) return threads(Int<W>(), Int<1>());
  if (k == 2) return threads(Int<W>(), Int<2>());
  if (W == 8 && k == 4) return threads(Int<W>(), Int<4>());
  return threads(Int<W>(), Int<W>());
}

bool norm_args_ok(const NormArgs& a, int64_t rows, int64_t n_tiles, int64_t n_whole,
                  int64_t max_len, int dtype) {
  const int64_t most = int64_t(1) << 31;
  return rows >= 1 && rows < most && a.chains >= 1 && a.chains < most && n_tiles >= 1 &&
         n_tiles < most && n_whole >= 1 && n_whole <= n_tiles && max_len >= 1 && max_len <= rows &&
         a.C >= 1 && a.C <= kMaxWidth && a.G >= 1 && a.C % a.G == 0 && a.ld >= a.C &&
         a.act >= MLCG_ACT_TANH && a.act <= MLCG_ACT_NONE && dtype >= MLCG_DTYPE_F32 &&
         dtype <= MLCG_DTYPE_BF16 && a.x && a.w && a.b && a.tiles && a.whole && a.first_tile;
}

}  // namespace

extern "C" int64_t mlcg_group_norm_workspace_floats(int64_t n_tiles, int64_t chains,
                                                    int64_t n_whole, int64_t max_len, int width,
                                                    int groups, int backward) {
  if (n_tiles < 0 || chains < 0 || n_whole < 0 || max_len < 0 || width < 1 || groups < 1)
    return -1;
  if (by_chain(max_len, n_whole, n_tiles, chains))
    return backward ? 2 * std::min<int64_t>(n_whole, 2048) * width : 0;
  return backward ? 2 * (n_tiles + chains) * width : 4 * n_tiles * groups;
}

extern "C" int mlcg_group_norm_act(const void* x, int64_t ld, int64_t rows, int dtype,
                                   const void* weight, const void* bias, int width, int groups,
                                   const int32_t* tiles, const int32_t* first_tile,
                                   int64_t n_tiles, const int32_t* whole, int64_t n_whole,
                                   int64_t max_len, int64_t chains, float eps, int act, void* y,
                                   float* stats, float* workspace, int64_t workspace_floats,
                                   void* stream) {
  if (rows == 0) return MLCG_OK;
  const NormArgs a{x, nullptr, weight, bias, ld, chains, reinterpret_cast<const int4*>(tiles),
                   reinterpret_cast<const int4*>(whole), first_tile, (int)n_tiles, (int)n_whole,
                   (int)max_len, width, groups, act, eps};
  MLCG_REQUIRE(norm_args_ok(a, rows, n_tiles, n_whole, max_len, dtype) && y && stats);
  const int64_t need = mlcg_group_norm_workspace_floats(n_tiles, chains, n_whole, max_len, width,
                                                        groups, 0);
  MLCG_REQUIRE(workspace_floats >= need && (need == 0 || workspace));
  hipStream_t s = mlcg_stream(stream);
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    constexpr int W = 16 / (int)sizeof(T);
    const bool vec = norm_vec<T>(a, y);
    return by_shape<W>(a, vec, [&](auto w, auto k, auto nt) {
      return norm_fwd<T, decltype(w)::value, decltype(k)::value, decltype(nt)::value>(
          a, y, stats, workspace, s);
    });
  });
}

extern "C" int mlcg_group_norm_act_backward(
    const void* x, int64_t ld, const void* grad_y, int64_t rows, int dtype, const void* weight,
    const void* bias, int width, int groups, const int32_t* tiles, const int32_t* first_tile,
    int64_t n_tiles, const int32_t* whole, int64_t n_whole, int64_t max_len, int64_t chains,
    int act, const float* stats, void* grad_x, void* grad_bias_weight, float* workspace,
    int64_t workspace_floats, void* stream) {
  const NormArgs a{x, grad_y, weight, bias, ld, chains, reinterpret_cast<const int4*>(tiles),
                   reinterpret_cast<const int4*>(whole), first_tile, (int)n_tiles, (int)n_whole,
                   (int)max_len, width, groups, act, 0.0f};
  MLCG_REQUIRE(norm_args_ok(a, rows, n_tiles, n_whole, max_len, dtype) && grad_y && stats &&
               grad_x && grad_bias_weight && workspace);
  MLCG_REQUIRE(workspace_floats >= mlcg_group_norm_workspace_floats(
                                       n_tiles, chains, n_whole, max_len, width, groups, 1));
  hipStream_t s = mlcg_stream(stream);
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    constexpr int W = 16 / (int)sizeof(T);
    const bool vec = norm_vec<T>(a, grad_x);
    return by_shape<W>(a, vec, [&](auto w, auto k, auto nt) {
      return norm_bwd<T, decltype(w)::value, decltype(k)::value, decltype(nt)::value>(
          a, stats, grad_x, grad_bias_weight, workspace, s);
    });
  });
}
