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
// A workgroup holds a slab of a chain's rows in registers: its threads form
// TR rows x TC columns, a column one vector of W channels, and every thread
// has the rows tr, tr + TR, ... of its column.  The mean and the sum of
// squared deviations from it are two passes over the registers, so neither
// is formed from a difference of large sums; the second pass also gives what
// the rounding of the mean left out, which is kept beside it (a deviation of a
// value far from zero is then as exact as the value).  Slabs of one chain are
// joined from theirs in slab order; every sum has a fixed order.
#include "chain.h"

namespace {

constexpr int kMaxWidth = 1024;

struct NormShape {
  const int4* tiles;  // (chain's first row, chain's length, slab's first row in it, chain)
  int n_tiles, size;  // slabs, and rows of a slab
  int C, G, TC, TR, cols, per;  // cols columns of sums, per of them a group
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

// Sums of K values a thread over the rows of its column: the rows that lie
// in one wave by a butterfly (TC divides 64), the rest through LDS.  sums[c]
// for c < TC K, valid for every thread on return.
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

// out[g] = f times the sum of the group's `per` columns of in, a wave a group.
__device__ void group_sums(const float* in, int groups, int per, float* out, float f = 1.0f) {
  const int lane = threadIdx.x & 63;
  for (int g = threadIdx.x >> 6; g < groups; g += blockDim.x >> 6) {
    float t = 0.0f;
    for (int c = lane; c < per; c += 64) t += in[g * per + c];
    t = mlcg_wave_sum(t);
    if (lane == 0) out[g] = t * f;
  }
  __syncthreads();
}

template <typename T, int W, int NV>
__device__ __forceinline__ void load_slab(const NormShape& sh, const T* x, int64_t ld,
                                          int64_t first, int rows, int row, int col,
                                          typename Vec<T, W>::type (&out)[NV]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int r = row + v * sh.TR;
    if (row < sh.TR && r < rows)
      out[v] = *reinterpret_cast<const typename Vec<T, W>::type*>(x + (first + r) * ld + col * W);
    else
      out[v] = typename Vec<T, W>::type{};
  }
}

// (mean, its remainder, M2) of every group of a slab -> part[g][tile]
template <typename T, int W, int NV, bool GROUPED>
__global__ __launch_bounds__(1024) void norm_part_kernel(NormShape sh, const T* __restrict__ x,
                                                         int64_t ld, float4* __restrict__ part) {
  extern __shared__ float lds[];
  float* red = lds;                                  // blockDim * W
  float* sums = red + blockDim.x * W;                // C
  float* mean = sums + sh.C;                         // G
  float* rest = mean + sh.G;                         // G
  float* m2 = rest + sh.G;                           // G
  const int4 t = sh.tiles[blockIdx.x];
  const int rows = min(sh.size, t.y - t.z);
  const int col = threadIdx.x % sh.TC, row = threadIdx.x / sh.TC;
  typename Vec<T, W>::type xv[NV];
  load_slab<T, W, NV>(sh, x, ld, (int64_t)t.x + t.z, rows, row, col, xv);
  constexpr int K = GROUPED ? 1 : W;
  const float inv = 1.0f / ((float)rows * (float)(sh.C / sh.G));
  float s[K] = {};
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < W; ++j) s[GROUPED ? 0 : j] += (float)xv[v][j];
  column_sums<K>(sh, s, red, sums);
  // the mean comes back from LDS: rounded, as it is kept
  group_sums(sums, sh.G, sh.per, mean, inv);
  float mu[W];
#pragma unroll
  for (int j = 0; j < W; ++j) mu[j] = mean[(col * W + j) / (sh.C / sh.G)];
  float c[K] = {};
#pragma unroll
  for (int k = 0; k < K; ++k) s[k] = 0.0f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const bool ok = row < sh.TR && row + v * sh.TR < rows;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float d = ok ? (float)xv[v][j] - mu[j] : 0.0f;
      c[GROUPED ? 0 : j] += d;
      s[GROUPED ? 0 : j] = fmaf(d, d, s[GROUPED ? 0 : j]);
    }
  }
  column_sums<K>(sh, c, red, sums);
  group_sums(sums, sh.G, sh.per, rest);
  column_sums<K>(sh, s, red, sums);
  group_sums(sums, sh.G, sh.per, m2);
  for (int g = threadIdx.x; g < sh.G; g += blockDim.x) {
    const float lo = rest[g] * inv;
    part[(int64_t)g * sh.n_tiles + blockIdx.x] =
        make_float4(mean[g], lo, fmaxf(0.0f, m2[g] - lo * rest[g]), 0.0f);
  }
}

// A chain's statistics from its slabs': with n_t values of mean m_t and sum of
// squares M_t,  mean = sum n_t m_t / n  and  M = sum M_t + n_t (m_t - mean)^2.
// stats: the mean, its remainder and 1 / sqrt(var + eps), [3][chains][G].
__global__ __launch_bounds__(256) void norm_join_kernel(NormShape sh,
                                                        const int32_t* __restrict__ first_tile,
                                                        const float4* __restrict__ part,
                                                        float eps, float* __restrict__ stats) {
  const int chain = blockIdx.x, g = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int t0 = first_tile[chain];
  if (g >= sh.G || t0 < 0) return;  // an empty chain has no slab and no statistics
  const int len = sh.tiles[t0].y;
  const int count = (len + sh.size - 1) / sh.size;
  const float4* p = part + (int64_t)g * sh.n_tiles + t0;
  const float n = (float)len;
  float s = 0.0f;
  for (int t = lane; t < count; t += 64)
    s = fmaf((float)min(sh.size, len - t * sh.size), p[t].x, s);
  const float mu = mlcg_wave_sum(s) / n;
  float c = 0.0f;
  for (int t = lane; t < count; t += 64)
    c = fmaf((float)min(sh.size, len - t * sh.size), (p[t].x - mu) + p[t].y, c);
  const float lo = mlcg_wave_sum(c) / n;
  const float P = (float)(sh.C / sh.G);
  float m2 = 0.0f;
  for (int t = lane; t < count; t += 64) {
    const float d = (p[t].x - mu) + (p[t].y - lo);
    m2 += fmaf((float)min(sh.size, len - t * sh.size) * P * d, d, p[t].z);
  }
  m2 = mlcg_wave_sum(m2);
  if (lane == 0) {
    const int64_t at = (int64_t)chain * sh.G + g, all = (int64_t)gridDim.x * sh.G;
    stats[at] = mu;
    stats[all + at] = lo;
    stats[2 * all + at] = 1.0f / sqrtf(m2 / (n * P) + eps);
  }
}

// What the elementwise passes need of a thread's channels.
template <typename T, int W>
struct Channels {
  float mu[W], lo[W], rs[W], w[W], b[W];
  __device__ __forceinline__ Channels(const NormShape& sh, const float* stats, int64_t chain,
                                      int64_t chains, int col, const T* weight, const T* bias) {
    const int P = sh.C / sh.G;
    const int64_t all = chains * sh.G;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const int c = col * W + j;
      const int64_t at = chain * sh.G + c / P;
      mu[j] = stats[at];
      lo[j] = stats[all + at];
      rs[j] = stats[2 * all + at];
      w[j] = (float)weight[c];
      b[j] = (float)bias[c];
    }
  }
  __device__ __forceinline__ float hat(int j, float x) const {
    return ((x - mu[j]) - lo[j]) * rs[j];
  }
};

template <typename T, int W>
__global__ __launch_bounds__(1024) void norm_apply_kernel(
    NormShape sh, const T* __restrict__ x, int64_t ld, const T* __restrict__ w,
    const T* __restrict__ b, const float* __restrict__ stats, int64_t chains, int act,
    T* __restrict__ y) {
  const int4 t = sh.tiles[blockIdx.x];
  const int rows = min(sh.size, t.y - t.z);
  const int col = threadIdx.x % sh.TC, row = threadIdx.x / sh.TC;
  if (row >= sh.TR) return;
  const Channels<T, W> ch(sh, stats, t.w, chains, col, w, b);
  for (int r = row; r < rows; r += sh.TR) {
    const int64_t at = (int64_t)t.x + t.z + r;
    const auto xv = *reinterpret_cast<const typename Vec<T, W>::type*>(x + at * ld + col * W);
    typename Vec<T, W>::type out;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      float yv, d;
      act_z(act, fmaf(ch.hat(j, (float)xv[j]), ch.w[j], ch.b[j]), yv, d);
      out[j] = (T)yv;
    }
    *reinterpret_cast<typename Vec<T, W>::type*>(y + at * sh.C + col * W) = out;
  }
}

// (A_c, B_c) of a slab -> part[tile][2][C]
template <typename T, int W>
__global__ __launch_bounds__(1024) void norm_bwd_part_kernel(
    NormShape sh, const T* __restrict__ x, int64_t ld, const T* __restrict__ dy,
    const T* __restrict__ w, const T* __restrict__ b, const float* __restrict__ stats,
    int64_t chains, int act, float* __restrict__ part) {
  extern __shared__ float lds[];
  float* red = lds;                    // blockDim * W
  float* sums = red + blockDim.x * W;  // C
  const int4 t = sh.tiles[blockIdx.x];
  const int rows = min(sh.size, t.y - t.z);
  const int col = threadIdx.x % sh.TC, row = threadIdx.x / sh.TC;
  float A[W] = {}, B[W] = {};
  const Channels<T, W> ch(sh, stats, t.w, chains, col, w, b);
  if (row < sh.TR) {
    for (int r = row; r < rows; r += sh.TR) {
      const int64_t at = (int64_t)t.x + t.z + r;
      const auto xv = *reinterpret_cast<const typename Vec<T, W>::type*>(x + at * ld + col * W);
      const auto gv = *reinterpret_cast<const typename Vec<T, W>::type*>(dy + at * sh.C + col * W);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float hat = ch.hat(j, (float)xv[j]);
        float yv, d;
        act_z(act, fmaf(hat, ch.w[j], ch.b[j]), yv, d);
        const float dz = (float)gv[j] * d;
        A[j] += dz;
        B[j] = fmaf(dz, hat, B[j]);
      }
    }
  }
  column_sums<W>(sh, A, red, sums);
  for (int c = threadIdx.x; c < sh.C; c += blockDim.x)
    part[(int64_t)blockIdx.x * 2 * sh.C + c] = sums[c];
  column_sums<W>(sh, B, red, sums);
  for (int c = threadIdx.x; c < sh.C; c += blockDim.x)
    part[(int64_t)blockIdx.x * 2 * sh.C + sh.C + c] = sums[c];
}

// out[seg][col] = sum over the segment's rows of in[row][col], `cols` columns:
// 32 columns x 32 slices of the rows a workgroup, the slices joined in order.
// Segments are the slabs of a chain (first_tile, tiles), or all `rows` rows.
template <typename O>
__global__ __launch_bounds__(1024) void norm_rows_kernel(const float* __restrict__ in, int cols,
                                                         const int32_t* __restrict__ first_tile,
                                                         const int4* __restrict__ tiles, int size,
                                                         int rows, O* __restrict__ out) {
  __shared__ float red[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  int64_t r0 = 0;
  int n = rows;
  if (first_tile) {
    const int t0 = first_tile[blockIdx.y];
    r0 = t0 < 0 ? 0 : t0;
    n = t0 < 0 ? 0 : (tiles[t0].y + size - 1) / size;
  }
  float s = 0.0f;
  if (col < cols)
    for (int r = slice; r < n; r += 32) s += in[(r0 + r) * cols + col];
  red[slice][threadIdx.x & 31] = s;
  __syncthreads();
  if (slice == 0 && col < cols) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][threadIdx.x];
    out[(int64_t)blockIdx.y * cols + col] = (O)t;
  }
}

template <typename T, int W>
__global__ __launch_bounds__(1024) void norm_bwd_apply_kernel(
    NormShape sh, const T* __restrict__ x, int64_t ld, const T* __restrict__ dy,
    const T* __restrict__ w, const T* __restrict__ b, const float* __restrict__ stats,
    int64_t chains, const float* __restrict__ chain_sums, int act, T* __restrict__ dx) {
  extern __shared__ float lds[];
  float* wa = lds;          // C: w_c A_c, then w_c B_c
  float* s1 = wa + sh.C;    // G
  float* s2 = s1 + sh.G;    // G
  const int4 t = sh.tiles[blockIdx.x];
  const int rows = min(sh.size, t.y - t.z);
  const int col = threadIdx.x % sh.TC, row = threadIdx.x / sh.TC;
  const int P = sh.C / sh.G;
  for (int k = 0; k < 2; ++k) {
    const float* a = chain_sums + ((int64_t)t.w * 2 + k) * sh.C;
    for (int c = threadIdx.x; c < sh.C; c += blockDim.x) wa[c] = (float)w[c] * a[c];
    __syncthreads();
    group_sums(wa, sh.G, P, k == 0 ? s1 : s2);
  }
  if (row >= sh.TR) return;
  const float inv = 1.0f / ((float)t.y * (float)P);
  const Channels<T, W> ch(sh, stats, t.w, chains, col, w, b);
  float m1[W], m2[W];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    m1[j] = s1[(col * W + j) / P] * inv;
    m2[j] = s2[(col * W + j) / P] * inv;
  }
  for (int r = row; r < rows; r += sh.TR) {
    const int64_t at = (int64_t)t.x + t.z + r;
    const auto xv = *reinterpret_cast<const typename Vec<T, W>::type*>(x + at * ld + col * W);
    const auto gv = *reinterpret_cast<const typename Vec<T, W>::type*>(dy + at * sh.C + col * W);
    typename Vec<T, W>::type out;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float hat = ch.hat(j, (float)xv[j]);
      float yv, d;
      act_z(act, fmaf(hat, ch.w[j], ch.b[j]), yv, d);
      // rounded as in the sums, not fused with the difference: the gradient of a
      // group of one value is then 0, not its rounding error times up to 1 / sqrt(eps)
      float dh = (float)gv[j] * d * ch.w[j];
      asm("" : "+v"(dh));
      out[j] = (T)((dh - m1[j] - hat * m2[j]) * ch.rs[j]);
    }
    *reinterpret_cast<typename Vec<T, W>::type*>(dx + at * sh.C + col * W) = out;
  }
}

constexpr int kNV = 16, kNV1 = 32;  // rows of a thread: vectors, and single channels

// Threads of a workgroup: a column of every vector of a row, and at least 4
// rows of them where a row has no more than 256 vectors.
int norm_threads(int tc) { return tc <= 64 ? 256 : 1024; }

template <typename T, int W>
NormShape norm_shape(const int32_t* tiles, int n_tiles, int size, int C, int G) {
  NormShape sh;
  sh.tiles = reinterpret_cast<const int4*>(tiles);
  sh.n_tiles = n_tiles;
  sh.size = size;
  sh.C = C;
  sh.G = G;
  sh.TC = C / W;
  sh.TR = norm_threads(sh.TC) / sh.TC;
  sh.cols = 0;
  sh.per = 0;
  return sh;
}

template <typename T, int W>
int norm_fwd(NormShape sh, const T* x, int64_t ld, const T* w, const T* b,
             const int32_t* first_tile, int64_t chains, float eps, int act, T* y,
             float* stats, float* ws, hipStream_t s) {
  const int nt = norm_threads(sh.TC);
  constexpr int NV = W == 1 ? kNV1 : kNV;
  const int P = sh.C / sh.G;
  const unsigned lds = (unsigned)((nt * W + sh.C + 3 * sh.G) * sizeof(float));
  float4* part = reinterpret_cast<float4*>(ws);
  if (P % W == 0) {
    sh.per = P / W;
    hipLaunchKernelGGL((norm_part_kernel<T, W, NV, true>), dim3(sh.n_tiles), dim3(nt), lds, s, sh,
                       x, ld, part);
  } else {
    sh.per = P;
    hipLaunchKernelGGL((norm_part_kernel<T, W, NV, false>), dim3(sh.n_tiles), dim3(nt), lds, s,
                       sh, x, ld, part);
  }
  hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)chains, mlcg_div_up(sh.G, 4)), dim3(256), 0,
                     s, sh, first_tile, part, eps, stats);
  hipLaunchKernelGGL((norm_apply_kernel<T, W>), dim3(sh.n_tiles), dim3(nt), 0, s, sh, x, ld, w, b,
                     stats, chains, act, y);
  return mlcg_launch_status();
}

template <typename T, int W>
int norm_bwd(NormShape sh, const T* x, int64_t ld, const T* dy, const T* w, const T* b,
             const float* stats, const int32_t* first_tile, int64_t chains, int act, T* dx, T* dw_db, float* ws, hipStream_t s) {
  const int nt = norm_threads(sh.TC);
  const unsigned lds = (unsigned)((nt * W + sh.C) * sizeof(float));
  float* part = ws;
  float* chain_sums = ws + (int64_t)sh.n_tiles * 2 * sh.C;
  hipLaunchKernelGGL((norm_bwd_part_kernel<T, W>), dim3(sh.n_tiles), dim3(nt), lds, s, sh, x, ld,
                     dy, w, b, stats, chains, act, part);
  hipLaunchKernelGGL(norm_rows_kernel<float>, dim3(mlcg_div_up(2 * sh.C, 32), (unsigned)chains),
                     dim3(1024), 0, s, part, 2 * sh.C, first_tile, sh.tiles, sh.size, 0,
                     chain_sums);
  hipLaunchKernelGGL((norm_bwd_apply_kernel<T, W>), dim3(sh.n_tiles), dim3(nt),
                     (unsigned)((sh.C + 2 * sh.G) * sizeof(float)), s, sh, x, ld, dy, w, b, stats,
                     chains, chain_sums, act, dx);
  hipLaunchKernelGGL(norm_rows_kernel<T>, dim3(mlcg_div_up(2 * sh.C, 32), 1), dim3(1024), 0, s,
                     chain_sums, 2 * sh.C, nullptr, nullptr, 1, (int)chains, dw_db);
  return mlcg_launch_status();
}

template <typename T>
constexpr int vec_width() {
  return 16 / sizeof(T);
}

template <typename T>
bool norm_vec(const void* x, int64_t ld, const void* o1, const void* o2, int C) {
  constexpr int W = vec_width<T>();
  return C % W == 0 && ld % W == 0 && chain_aligned16(x) && chain_aligned16(o1) &&
         chain_aligned16(o2);
}

bool norm_args_ok(int64_t rows, int64_t chains, int64_t n_tiles, int size, int width, int groups,
                  int64_t ld, int act, int dtype) {
  return rows >= 0 && rows < (int64_t(1) << 31) && chains >= 0 && chains < (int64_t(1) << 31) &&
         n_tiles >= 0 && n_tiles < (int64_t(1) << 31) && size >= 1 && width >= 1 &&
         width <= kMaxWidth && groups >= 1 && width % groups == 0 && ld >= width &&
         act >= MLCG_ACT_TANH && act <= MLCG_ACT_NONE && dtype >= MLCG_DTYPE_F32 &&
         dtype <= MLCG_DTYPE_BF16;
}

}  // namespace

// Rows of a slab that fit the registers, a power of two of 32 to 256.
extern "C" int mlcg_group_norm_slab_rows(int width, int dtype) {
  if (width < 1 || width > kMaxWidth || dtype < MLCG_DTYPE_F32 || dtype > MLCG_DTYPE_BF16)
    return -1;
  const int W = dtype == MLCG_DTYPE_F32 ? 4 : 8;
  // the vector form's and the single-channel form's: the call decides which
  // runs, so a slab has to fit both
  int rows = 256;
  const int t1 = norm_threads(width), tv = norm_threads(width / W);
  while (rows > 32 && (rows > kNV1 * (t1 / width) ||
                       (width % W == 0 && rows > kNV * (tv / (width / W)))))
    rows >>= 1;
  return rows;
}

extern "C" int64_t mlcg_group_norm_workspace_floats(int64_t n_tiles, int64_t chains, int width,
                                                    int groups, int backward) {
  if (n_tiles < 0 || chains < 0 || width < 1 || groups < 1) return -1;
  return backward ? 2 * (n_tiles + chains) * width : 4 * n_tiles * groups;
}

extern "C" int mlcg_group_norm_act(const void* x, int64_t ld, int64_t rows, int dtype,
                                   const void* weight, const void* bias, int width, int groups,
                                   const int32_t* tiles, const int32_t* first_tile,
                                   int64_t n_tiles, int size, int64_t chains, float eps, int act,
                                   void* y, float* stats, float* workspace,
                                   int64_t workspace_floats, void* stream) {
  MLCG_REQUIRE(norm_args_ok(rows, chains, n_tiles, size, width, groups, ld, act, dtype));
  MLCG_REQUIRE(size <= mlcg_group_norm_slab_rows(width, dtype));
  if (rows == 0 || n_tiles == 0) return MLCG_OK;
  MLCG_REQUIRE(x && weight && bias && tiles && first_tile && y && stats && workspace);
  MLCG_REQUIRE(workspace_floats >=
               mlcg_group_norm_workspace_floats(n_tiles, chains, width, groups, 0));
  hipStream_t s = mlcg_stream(stream);
#define NORM_FWD(T)                                                                              \
  if (norm_vec<T>(x, ld, y, nullptr, width))                                                     \
    return norm_fwd<T, vec_width<T>()>(                                                          \
        norm_shape<T, vec_width<T>()>(tiles, (int)n_tiles, size, width, groups), (const T*)x,    \
        ld, (const T*)weight, (const T*)bias, first_tile, chains, eps, act, (T*)y, stats, workspace, s);                                                                           \
  return norm_fwd<T, 1>(norm_shape<T, 1>(tiles, (int)n_tiles, size, width, groups), (const T*)x, \
                        ld, (const T*)weight, (const T*)bias, first_tile, chains, eps, act,      \
                        (T*)y, stats, workspace, s);
  if (dtype == MLCG_DTYPE_F32) {
    NORM_FWD(float)
  } else if (dtype == MLCG_DTYPE_F16) {
    NORM_FWD(_Float16)
  }
  NORM_FWD(__bf16)
#undef NORM_FWD
}

extern "C" int mlcg_group_norm_act_backward(
    const void* x, int64_t ld, const void* grad_y, int64_t rows, int dtype, const void* weight,
    const void* bias, int width, int groups, const int32_t* tiles, const int32_t* first_tile,
    int64_t n_tiles, int size, int64_t chains, int act, const float* stats, void* grad_x, void* grad_weight_bias, float* workspace, int64_t workspace_floats,
    void* stream) {
  MLCG_REQUIRE(norm_args_ok(rows, chains, n_tiles, size, width, groups, ld, act, dtype));
  MLCG_REQUIRE(rows > 0 && n_tiles > 0 && size <= mlcg_group_norm_slab_rows(width, dtype));
  MLCG_REQUIRE(x && grad_y && weight && bias && tiles && first_tile && stats && grad_x &&
               grad_weight_bias && workspace);
  MLCG_REQUIRE(workspace_floats >=
               mlcg_group_norm_workspace_floats(n_tiles, chains, width, groups, 1));
  hipStream_t s = mlcg_stream(stream);
#define NORM_BWD(T)                                                                              \
  if (norm_vec<T>(x, ld, grad_y, grad_x, width))                                                 \
    return norm_bwd<T, vec_width<T>()>(                                                          \
        norm_shape<T, vec_width<T>()>(tiles, (int)n_tiles, size, width, groups), (const T*)x,    \
        ld, (const T*)grad_y, (const T*)weight, (const T*)bias, stats, first_tile, chains,  \
        act, (T*)grad_x, (T*)grad_weight_bias, workspace, s);                                    \
  return norm_bwd<T, 1>(norm_shape<T, 1>(tiles, (int)n_tiles, size, width, groups), (const T*)x, \
                        ld, (const T*)grad_y, (const T*)weight, (const T*)bias, stats,      \
                        first_tile, chains, act, (T*)grad_x, (T*)grad_weight_bias, workspace, s);
  if (dtype == MLCG_DTYPE_F32) {
    NORM_BWD(float)
  } else if (dtype == MLCG_DTYPE_F16) {
    NORM_BWD(_Float16)
  }
  NORM_BWD(__bf16)
#undef NORM_BWD
}
