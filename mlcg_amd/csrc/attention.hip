// Attention of the beads of a chain to each other with a learned bias by
// relative position (gfx950).
//
// For query bead i and key bead j of one chain, head h (R = reach):
//   l_ij = scale q_i.k_j + table[bucket_of[clip(p_j - p_i, -R, R) + R], h]
//   P_ij = exp(l_ij) / sum_j exp(l_ij)  over the present keys,   o_i = sum_j P_ij v_j
// (a row without any present key gives zeros), p the bead's index in its
// chain or a residue number; backward, with dP_ij = do_i . v_j,
//   delta_i = sum_j P_ij dP_ij = do_i . o_i,   dS_ij = P_ij (dP_ij - delta_i),
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,
//   dv_j = sum_i P_ij do_i,  dtable[b, h] = sum of dS_ij over the pairs in b.
// Neither the bias nor the probabilities are ever stored: the forward pass
// keeps the running maximum and sum of every row (base-2 exponents) and the
// log of the sum, from which the backward passes form P again.
//
// Tiles: a wave owns 32 queries (forward, dq) or 32 keys (dk, dv) as the
// columns of 32 x 32 MFMA tiles, so a lane is one query (key) and the softmax
// statistics are lane values; the other side comes in tiles of KT rows
// through LDS.  The 16 accumulators of a lane are rows 8 a + 4 g + c (g the
// lane's half): as the contraction over them is free to be permuted, they are
// used as the B operand of the next product as they are, and the A operand's
// tile is stored transposed with its rows in that order.  In 16 bits a step
// of 16 is one v_mfma_f32_32x32x16, in 32 bits eight v_mfma_f32_32x32x2.
//
// LDS rows hold 16-byte chunks, exchanged by row (xor), so that the 16-byte
// reads of 8 consecutive rows fall on all banks.
//
// The bias of an offset is one LDS value a head: an array over the offsets
// from -(R + M) to R + M, M beyond the largest span of a tile, so that a tile
// that touches the band |offset| < R needs no clipping; a tile outside of it
// has one value.  The table's gradient is summed by offset the same way (one
// array a wave, LDS adds in program order), then by bucket, then over the
// workgroups in a fixed order.
#include <type_traits>

#include "chain.h"

namespace {

constexpr int kQ = 32;                   // columns of a wave
constexpr int kSpan = 96;                // offsets beyond the reach that a tile can touch
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  const void *q, *k, *v, *table, *out_or_null, *grad;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int64_t beads;
  const int32_t* bucket_of;  // [2 reach + 1]
  const int4* tiles;         // (chain's first row, its length, tile's first row in it, chain)
  const uint8_t* keep;
  const int32_t* pos;
  float* lse;  // [heads][beads], base 2; +inf for a row without keys
  int n_tiles, heads, group, dim, reach, buckets, vec;
  float scale;
};

template <typename T>
constexpr int key_tile() {
  return sizeof(T) == 2 ? 64 : 32;
}

// element offset of (row, el) in an LDS tile of LEN elements a row
template <typename T, int LEN>
__device__ __forceinline__ int tile_at(int row, int el) {
  constexpr int EPC = 16 / sizeof(T), NCH = LEN / EPC;
  static_assert(NCH >= 4, "a row holds at least four chunks");
  const int sw = NCH >= 8 ? (row ^ (row >> 3)) & 7 : ((row >> 1) ^ (row >> 3)) & 3;
  return row * LEN + (((el / EPC) ^ sw) * EPC) + el % EPC;
}

// 8 consecutive elements of a row, from a multiple of 8
template <typename T, int LEN>
__device__ __forceinline__ v8<T> tile_frag(const T* tile, int row, int el) {
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const v8<T>*>(tile + tile_at<T, LEN>(row, el));
  } else {
    const v4<T> a = *reinterpret_cast<const v4<T>*>(tile + tile_at<T, LEN>(row, el));
    const v4<T> b = *reinterpret_cast<const v4<T>*>(tile + tile_at<T, LEN>(row, el + 4));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// where row 0..KT-1 of the contraction stands in a transposed tile's row
__device__ __forceinline__ int row_place(int r) {
  return (r & ~15) + ((r >> 2) & 1) * 8 + ((r >> 3) & 1) * 4 + (r & 3);
}

__device__ __forceinline__ void mma(f32x16& c, v8<__bf16> a, v8<__bf16> b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& c, v8<_Float16> a, v8<_Float16> b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& c, v8<float> a, v8<float> b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
}

// 4 elements from p, zero where !ok or past `left`
template <typename T>
__device__ __forceinline__ v4<T> load4(const T* p, bool ok, int left, int vec) {
  v4<T> r{};
  if (!ok || left <= 0) return r;
  if (vec) return *reinterpret_cast<const v4<T>*>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) r[j] = p[j];
  return r;
}

// 8 elements of a row at el: a B operand's fragment
template <typename T>
__device__ __forceinline__ v8<T> load8(const T* row, int el, bool ok, int dim, int vec) {
  const v4<T> a = load4<T>(row + el, ok, dim - el, vec);
  const v4<T> b = load4<T>(row + el + 4, ok, dim - el - 4, vec);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// KT rows from `src` (row stride `stride`, rows at or past `rows` and rows
// that keep0 marks absent as zeros) into a tile and / or its transpose.
template <typename T, int DP, int KT, int NT, bool ROWS, bool TRANS>
__device__ __forceinline__ void stage(const T* src, int64_t stride, int rows, const uint8_t* keep0,
                                      int dim, int vec, T* tile, T* trans) {
  constexpr int NJ = DP / 4, BLOCKS = KT / 4 * NJ;
  for (int i = threadIdx.x; i < BLOCKS; i += NT) {
    const int j = i % NJ, r0 = i / NJ * 4;
    v4<T> x[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool ok = r0 + r < rows && (!keep0 || keep0[r0 + r]);
      x[r] = load4<T>(src + (r0 + r) * stride + 4 * j, ok, dim - 4 * j, vec);
    }
    if (ROWS) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<v4<T>*>(tile + tile_at<T, DP>(r0 + r, 4 * j)) = x[r];
    }
    if (TRANS) {
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const v4<T> c = {x[0][d], x[1][d], x[2][d], x[3][d]};
        *reinterpret_cast<v4<T>*>(trans + tile_at<T, KT>(4 * j + d, row_place(r0))) = c;
      }
    }
  }
}

// ext[n] = log2(e) bias of the offset n - (reach + kSpan), clipped
template <typename T>
__device__ __forceinline__ void fill_bias(const AttnArgs& a, int head, float* ext) {
  const int n = 2 * (a.reach + kSpan) + 1;
  const T* table = (const T*)a.table;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int d = min(max(i - kSpan, 0), 2 * a.reach);
    ext[i] = kLog2e * (float)table[(int64_t)a.bucket_of[d] * a.heads + head];
  }
}

// clipped offset p_j - p_i as an index of ext, for any int32 positions
__device__ __forceinline__ int offset_cell(int pj, int pi, int reach) {
  return min(max(__builtin_elementwise_sub_sat(pj, pi), -reach), reach) + reach + kSpan;
}

template <typename T>
__device__ __forceinline__ v8<T> pack8(const float* p) {
  v8<T> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = (T)p[e];
  return r;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// the wave's 32 columns of  tile . B  for all KT rows of the tile
template <typename T, int DP, int KT>
__device__ __forceinline__ void tile_product(const T* tile, const v8<T> (&b)[DP / 16],
                                             f32x16 (&s)[KT / 32]) {
  const int col = threadIdx.x & 31, g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int n = 0; n < KT / 32; ++n) {
    s[n] = f32x16{};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
      mma(s[n], tile_frag<T, DP>(tile, 32 * n + col, 16 * k + 8 * g), b[k]);
  }
}

// acc += trans . P  with P the KT rows of a lane's column
template <typename T, int DP, int KT>
__device__ __forceinline__ void trans_product(const T* trans, const float (&p)[KT / 2],
                                              f32x16 (&acc)[DP / 32]) {
  const int col = threadIdx.x & 31, g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int u = 0; u < KT / 16; ++u) {
    const v8<T> b = pack8<T>(p + 8 * u);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
      mma(acc[n], tile_frag<T, KT>(trans, 32 * n + col, 16 * u + 8 * g), b);
  }
}

// a lane's column (32 DP / 32 rows of accumulators) as a row of dst
template <typename T, int DP>
__device__ __forceinline__ void store_column(T* dst, const f32x16 (&acc)[DP / 32], float f,
                                             int dim, int vec) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * n + 8 * a + 4 * g;
      v4<T> o;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = (T)(acc[n][4 * a + c] * f);
      if (vec) {
        if (d < dim) *reinterpret_cast<v4<T>*>(dst + d) = o;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (d + c < dim) dst[d + c] = o[c];
      }
    }
}

// The logits (base 2) of a tile whose lanes are queries and whose rows are
// keys: x[16 n + r] for key k0 + 32 n + 8 (r / 4) + 4 g + r % 4.
template <int KT>
__device__ __forceinline__ void query_logits(const AttnArgs& a, const f32x16 (&s)[KT / 32],
                                             const float* ext, const int* kpos, int k0, int qw,
                                             int qi, int qp, float (&x)[KT / 2]) {
  const int g = (threadIdx.x >> 5) & 1;
  const float c = a.scale * kLog2e;
  const int R = a.reach;
  if (a.pos) {
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) {
      const int key = 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * g + i % 4;
      x[i] = fmaf(s[i / 16][i % 16], c, ext[offset_cell(kpos[key], qp, R)]);
    }
  } else if (k0 - (qw + kQ - 1) >= R || k0 + KT - 1 - qw <= -R) {
    const float b = k0 > qw ? ext[2 * (R + kSpan)] : ext[0];
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) x[i] = fmaf(s[i / 16][i % 16], c, b);
  } else {
    const float* e = ext + (k0 - qi + 4 * g + R + kSpan);
#pragma unroll
    for (int i = 0; i < KT / 2; ++i)
      x[i] = fmaf(s[i / 16][i % 16], c, e[32 * (i / 16) + 8 * (i % 16 / 4) + i % 4]);
  }
}

// +inf for a present key of a tile, -inf for an absent one
__device__ __forceinline__ void stage_keys(const AttnArgs& a, const int4& t, int k0, int kt,
                                           float* cap, int* kpos) {
  const int i = threadIdx.x;
  if (i < kt) {
    const int64_t row = (int64_t)t.x + k0 + i;
    const bool in = k0 + i < t.y;
    cap[i] = in && (!a.keep || a.keep[row]) ? INFINITY : -INFINITY;
    kpos[i] = in && a.pos ? a.pos[row] : 0;
  }
}

template <int KT>
__device__ __forceinline__ void mask_logits(const float* cap, float (&x)[KT / 2]) {
  const int lane = threadIdx.x & 63, g = lane >> 5;
  if (__ballot(lane < KT && cap[lane < KT ? lane : 0] < 0.0f) == 0) return;
#pragma unroll
  for (int i = 0; i < KT / 2; ++i) {
    const int key = 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * g + i % 4;
    x[i] = cap[key] < 0.0f ? -INFINITY : x[i];
  }
}

template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void attn_fwd_kernel(AttnArgs a, T* __restrict__ out) {
  constexpr int KT = key_tile<T>();
  extern __shared__ __align__(16) unsigned char smem[];
  T* kt = reinterpret_cast<T*>(smem);
  T* vt = kt + KT * DP;
  float* cap = reinterpret_cast<float*>(vt + DP * KT);
  int* kpos = reinterpret_cast<int*>(cap + KT);
  float* ext = reinterpret_cast<float*>(kpos + KT);

  const int head = blockIdx.x % a.heads, kv = head / a.group;
  const int4 t = a.tiles[blockIdx.x / a.heads];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 5;
  const int qw = t.z + kQ * wave, qi = qw + (lane & 31);
  const bool q_ok = qi < t.y;
  const T* q = (const T*)a.q + ((int64_t)t.x + qi) * a.q_row + head * a.q_head;
  v8<T> qf[DP / 16];
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) qf[k] = load8<T>(q, 16 * k + 8 * g, q_ok, a.dim, a.vec);
  const int qp = a.pos && q_ok ? a.pos[(int64_t)t.x + qi] : 0;
  fill_bias<T>(a, head, ext);

  f32x16 acc[DP / 32] = {};
  float m = -INFINITY, l = 0.0f;
  for (int k0 = 0; k0 < t.y; k0 += KT) {
    const int64_t row0 = (int64_t)t.x + k0;
    const uint8_t* keep0 = a.keep ? a.keep + row0 : nullptr;
    __syncthreads();
    stage<T, DP, KT, 64 * NW, true, false>((const T*)a.k + row0 * a.k_row + kv * a.k_head, a.k_row,
                                           t.y - k0, keep0, a.dim, a.vec, kt, nullptr);
    stage<T, DP, KT, 64 * NW, false, true>((const T*)a.v + row0 * a.v_row + kv * a.v_head, a.v_row,
                                           t.y - k0, keep0, a.dim, a.vec, nullptr, vt);
    stage_keys(a, t, k0, KT, cap, kpos);
    __syncthreads();
    if (qw >= t.y) continue;
    f32x16 s[KT / 32];
    tile_product<T, DP, KT>(kt, qf, s);
    float x[KT / 2];
    query_logits<KT>(a, s, ext, kpos, k0, qw, qi, qp, x);
    mask_logits<KT>(cap, x);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < KT / 2; ++i) top = fmaxf(top, x[i]);
    top = fmaxf(top, other_half(top));
    const float m_new = fmaxf(m, top);
    const float base = m_new == -INFINITY ? 0.0f : m_new;  // no key so far: exp2(-inf) = 0
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    m = m_new;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i] - base);
      sum += x[i];
    }
    l = fmaf(l, alpha, sum);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][r] *= alpha;
    trans_product<T, DP, KT>(vt, x, acc);
  }
  if (!q_ok) return;
  l += other_half(l);
  const int64_t row = (int64_t)t.x + qi;
  store_column<T, DP>(out + (row * a.heads + head) * a.dim, acc, l == 0.0f ? 0.0f : 1.0f / l,
                      a.dim, a.vec);
  if (a.lse && g == 0)
    a.lse[head * a.beads + row] = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// The table's gradient of a workgroup: the waves' sums by offset (dd, one
// array of `cells` a wave, with the sums outside of the band in far[wave])
// to buckets.
template <int NW>
__device__ __forceinline__ void flush_offsets(const AttnArgs& a, float* dd, int cells,
                                              const int32_t* order, const int32_t* first,
                                              float* out) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < cells; i += 64 * NW) {
    float t = dd[i];
#pragma unroll
    for (int w = 1; w < NW; ++w) t += dd[w * cells + i];
    dd[i] = t;
  }
  __syncthreads();
  if (tid < 64) {  // the cells beyond the reach belong to its ends
    float lo = 0.0f, hi = 0.0f;
    for (int i = tid; i <= kSpan; i += 64) {
      lo += dd[i];
      hi += dd[cells - 1 - i];
    }
    lo = mlcg_wave_sum(lo);
    hi = mlcg_wave_sum(hi);
    if (tid == 0) {
      dd[kSpan] = lo;
      dd[cells - 1 - kSpan] = hi;
    }
  }
  __syncthreads();
  for (int b = tid; b < a.buckets; b += 64 * NW) {
    float t = 0.0f;
    for (int i = first[b]; i < first[b + 1]; ++i) t += dd[kSpan + order[i]];
    out[b] = t;
  }
}

// dq, delta and the workgroup's part of the table's gradient; lanes are
// queries as in the forward pass.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void attn_dq_kernel(AttnArgs a, const T* __restrict__ o,
                                                          T* __restrict__ dq,
                                                          float* __restrict__ delta_out,
                                                          const int32_t* __restrict__ order,
                                                          const int32_t* __restrict__ first,
                                                          float* __restrict__ dtable_part) {
  constexpr int KT = key_tile<T>();
  extern __shared__ __align__(16) unsigned char smem[];
  T* kt = reinterpret_cast<T*>(smem);
  T* ktr = kt + KT * DP;
  T* vt = ktr + KT * DP;
  float* cap = reinterpret_cast<float*>(vt + DP * KT);
  int* kpos = reinterpret_cast<int*>(cap + KT);
  float* ext = reinterpret_cast<float*>(kpos + KT);
  const int cells = 2 * (a.reach + kSpan) + 1, R = a.reach;
  float* dd = ext + cells;

  const int head = blockIdx.x % a.heads, kv = head / a.group, tile = blockIdx.x / a.heads;
  const int4 t = a.tiles[tile];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 5;
  const int qw = t.z + kQ * wave, qi = qw + (lane & 31);
  const bool q_ok = qi < t.y;
  const int64_t row = (int64_t)t.x + qi;
  const T* q = (const T*)a.q + row * a.q_row + head * a.q_head;
  const int64_t flat = (row * a.heads + head) * a.dim;
  v8<T> qf[DP / 16], gf[DP / 16];
  float delta = 0.0f;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    qf[k] = load8<T>(q, 16 * k + 8 * g, q_ok, a.dim, a.vec);
    gf[k] = load8<T>((const T*)a.grad + flat, 16 * k + 8 * g, q_ok, a.dim, a.vec);
    const v8<T> of = load8<T>(o + flat, 16 * k + 8 * g, q_ok, a.dim, a.vec);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[k][e], (float)of[e], delta);
  }
  delta += other_half(delta);
  const float lse = q_ok ? a.lse[head * a.beads + row] : INFINITY;
  const int qp = a.pos && q_ok ? a.pos[row] : 0;
  fill_bias<T>(a, head, ext);
  for (int i = threadIdx.x; i < NW * cells; i += 64 * NW) dd[i] = 0.0f;
  float* mine = dd + wave * cells;
  float far[2] = {0.0f, 0.0f};

  f32x16 acc[DP / 32] = {};
  for (int k0 = 0; k0 < t.y; k0 += KT) {
    const int64_t row0 = (int64_t)t.x + k0;
    const uint8_t* keep0 = a.keep ? a.keep + row0 : nullptr;
    __syncthreads();
    stage<T, DP, KT, 64 * NW, true, true>((const T*)a.k + row0 * a.k_row + kv * a.k_head, a.k_row,
                                          t.y - k0, keep0, a.dim, a.vec, kt, ktr);
    stage<T, DP, KT, 64 * NW, true, false>((const T*)a.v + row0 * a.v_row + kv * a.v_head, a.v_row,
                                           t.y - k0, keep0, a.dim, a.vec, vt, nullptr);
    stage_keys(a, t, k0, KT, cap, kpos);
    __syncthreads();
    if (qw >= t.y) continue;
    f32x16 s[KT / 32];
    tile_product<T, DP, KT>(kt, qf, s);
    float x[KT / 2];
    query_logits<KT>(a, s, ext, kpos, k0, qw, qi, qp, x);
    mask_logits<KT>(cap, x);
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] - lse);
    tile_product<T, DP, KT>(vt, gf, s);  // dP
    if (t.y <= KT) {
      // a chain of one tile: delta from P and dP themselves, so that a row
      // of one key has dS = 0 exactly
      delta = 0.0f;
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) delta = fmaf(x[i], s[i / 16][i % 16], delta);
      delta += other_half(delta);
    }
#pragma unroll
    for (int i = 0; i < KT / 2; ++i) x[i] *= s[i / 16][i % 16] - delta;
    if (a.pos) {
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) {
        const int key = 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * g + i % 4;
        atomicAdd(&mine[offset_cell(kpos[key], qp, R)], x[i]);
      }
    } else if (k0 - (qw + kQ - 1) >= R || k0 + KT - 1 - qw <= -R) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) sum += x[i];
      if (k0 > qw)
        far[1] += sum;
      else
        far[0] += sum;
    } else {
      float* e = mine + (k0 - qi + 4 * g + R + kSpan);
      if (q_ok) {
#pragma unroll
        for (int i = 0; i < KT / 2; ++i)
          atomicAdd(&e[32 * (i / 16) + 8 * (i % 16 / 4) + i % 4], x[i]);
      }
    }
    trans_product<T, DP, KT>(ktr, x, acc);
  }
  if (q_ok) {
    store_column<T, DP>(dq + flat, acc, a.scale, a.dim, a.vec);
    if (g == 0) delta_out[head * a.beads + row] = delta;
  }
  far[0] = mlcg_wave_sum(far[0]);
  far[1] = mlcg_wave_sum(far[1]);
  __syncthreads();
  if (lane == 0) {
    mine[0] += far[0];
    mine[cells - 1] += far[1];
  }
  flush_offsets<NW>(a, dd, cells, order, first,
                    dtable_part + ((int64_t)head * a.n_tiles + tile) * a.buckets);
}

// dk and dv; lanes are keys, the tiles hold queries.  The query heads that
// share a key/value head are taken one after the other.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void attn_dkv_kernel(AttnArgs a,
                                                           const float* __restrict__ delta,
                                                           T* __restrict__ dk,
                                                           T* __restrict__ dv) {
  constexpr int KT = key_tile<T>();
  extern __shared__ __align__(16) unsigned char smem[];
  T* qt = reinterpret_cast<T*>(smem);
  T* qtr = qt + KT * DP;
  T* gt = qtr + KT * DP;
  T* gtr = gt + KT * DP;
  float* lses = reinterpret_cast<float*>(gtr + DP * KT);
  float* dels = lses + KT;
  int* qpos = reinterpret_cast<int*>(dels + KT);
  float* ext = reinterpret_cast<float*>(qpos + KT);

  const int kv_heads = a.heads / a.group;
  const int kv = blockIdx.x % kv_heads;
  const int4 t = a.tiles[blockIdx.x / kv_heads];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 5;
  const int kw = t.z + kQ * wave, ki = kw + (lane & 31);
  const int64_t row = (int64_t)t.x + ki;
  const bool in = ki < t.y, k_ok = in && (!a.keep || a.keep[row]);
  const T* k = (const T*)a.k + row * a.k_row + kv * a.k_head;
  const T* v = (const T*)a.v + row * a.v_row + kv * a.v_head;
  v8<T> kf[DP / 16], vf[DP / 16];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    kf[i] = load8<T>(k, 16 * i + 8 * g, k_ok, a.dim, a.vec);
    vf[i] = load8<T>(v, 16 * i + 8 * g, k_ok, a.dim, a.vec);
  }
  const int kp = a.pos && in ? a.pos[row] : 0;
  const float c = a.scale * kLog2e;
  const int R = a.reach;

  f32x16 dka[DP / 32] = {}, dva[DP / 32] = {};
  for (int h = 0; h < a.group; ++h) {
    const int head = kv * a.group + h;
    __syncthreads();
    fill_bias<T>(a, head, ext);
    for (int q0 = 0; q0 < t.y; q0 += KT) {
      const int64_t row0 = (int64_t)t.x + q0;
      __syncthreads();
      stage<T, DP, KT, 64 * NW, true, true>((const T*)a.q + row0 * a.q_row + head * a.q_head,
                                            a.q_row, t.y - q0, nullptr, a.dim, a.vec, qt, qtr);
      stage<T, DP, KT, 64 * NW, true, true>(
          (const T*)a.grad + (row0 * a.heads + head) * a.dim, (int64_t)a.heads * a.dim, t.y - q0,
          nullptr, a.dim, a.vec, gt, gtr);
      if (threadIdx.x < KT) {
        const int i = threadIdx.x;
        const bool ok = q0 + i < t.y;
        lses[i] = ok ? a.lse[head * a.beads + row0 + i] : INFINITY;
        dels[i] = ok ? delta[head * a.beads + row0 + i] : 0.0f;
        qpos[i] = ok && a.pos ? a.pos[row0 + i] : 0;
      }
      __syncthreads();
      if (kw >= t.y) continue;
      f32x16 s[KT / 32];
      tile_product<T, DP, KT>(qt, kf, s);
      float x[KT / 2];
      const bool far_hi = kw - (q0 + KT - 1) >= R, far_lo = kw + kQ - 1 - q0 <= -R;
      if (a.pos) {
#pragma unroll
        for (int i = 0; i < KT / 2; ++i) {
          const int qr = 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * g + i % 4;
          x[i] = fmaf(s[i / 16][i % 16], c, ext[offset_cell(kp, qpos[qr], R)]);
        }
      } else if (far_hi || far_lo) {
        const float b = far_hi ? ext[2 * (R + kSpan)] : ext[0];
#pragma unroll
        for (int i = 0; i < KT / 2; ++i) x[i] = fmaf(s[i / 16][i % 16], c, b);
      } else {
        const float* e = ext + (ki - q0 - 4 * g + R + kSpan);
#pragma unroll
        for (int i = 0; i < KT / 2; ++i)
          x[i] = fmaf(s[i / 16][i % 16], c, e[-(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4)]);
      }
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) {
        const int qr = 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * g + i % 4;
        x[i] = __builtin_amdgcn_exp2f(x[i] - lses[qr]);
      }
      trans_product<T, DP, KT>(gtr, x, dva);
      tile_product<T, DP, KT>(gt, vf, s);  // dP
#pragma unroll
      for (int i = 0; i < KT / 2; ++i) {
        const int qr = 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * g + i % 4;
        x[i] *= s[i / 16][i % 16] - dels[qr];
      }
      trans_product<T, DP, KT>(qtr, x, dka);
    }
  }
  if (!in) return;
  const int64_t flat = (row * kv_heads + kv) * a.dim;
  if (!k_ok) {  // an absent key takes part in nothing
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) dka[n] = dva[n] = f32x16{};
  }
  store_column<T, DP>(dk + flat, dka, a.scale, a.dim, a.vec);
  store_column<T, DP>(dv + flat, dva, 1.0f, a.dim, a.vec);
}

// dtable[b][head] = sum of the workgroups' parts [head][tile][b]: 8 buckets x
// 32 slices of the tiles a workgroup, joined in order.
template <typename T>
__global__ __launch_bounds__(256) void attn_dtable_kernel(const float* __restrict__ part,
                                                          int n_tiles, int buckets, int heads,
                                                          T* __restrict__ dtable) {
  __shared__ float red[32][9];
  const int b = blockIdx.x * 8 + (threadIdx.x & 7), slice = threadIdx.x >> 3, head = blockIdx.y;
  float s = 0.0f;
  if (b < buckets)
    for (int i = slice; i < n_tiles; i += 32) s += part[((int64_t)head * n_tiles + i) * buckets + b];
  red[slice][threadIdx.x & 7] = s;
  __syncthreads();
  if (slice == 0 && b < buckets) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += red[i][threadIdx.x];
    dtable[(int64_t)b * heads + head] = (T)t;
  }
}

template <typename T, int DP>
constexpr int tile_bytes() {
  return key_tile<T>() * DP * (int)sizeof(T);
}

// LDS above 64 KiB has to be asked for, once a kernel.
int allow_lds(const void* f, unsigned bytes) {
  if (bytes <= 65536u) return MLCG_OK;
  return hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) ==
                 hipSuccess
             ? MLCG_OK
             : MLCG_ERR_LAUNCH;
}

template <typename T, int DP, int NW>
int launch_fwd(const AttnArgs& a, void* out, hipStream_t s) {
  const unsigned cells = 2 * (a.reach + kSpan) + 1;
  const unsigned lds = 2 * tile_bytes<T, DP>() + 4 * (2 * key_tile<T>() + cells);
  auto f = attn_fwd_kernel<T, DP, NW>;
  if (int e = allow_lds(reinterpret_cast<const void*>(f), lds)) return e;
  hipLaunchKernelGGL(f, dim3((unsigned)(a.n_tiles * a.heads)), dim3(64 * NW), lds, s, a, (T*)out);
  return mlcg_launch_status();
}

struct BwdOut {
  void *dq, *dk, *dv, *dtable;
  float* ws;
  const int32_t *order, *first;
};

template <typename T, int DP, int NW>
int launch_bwd(const AttnArgs& a, const BwdOut& o, hipStream_t s) {
  const unsigned cells = 2 * (a.reach + kSpan) + 1;
  const unsigned lds1 = 3 * tile_bytes<T, DP>() + 4 * (2 * key_tile<T>() + (NW + 1) * cells);
  const unsigned lds2 = 4 * tile_bytes<T, DP>() + 4 * (3 * key_tile<T>() + cells);
  auto f1 = attn_dq_kernel<T, DP, NW>;
  auto f2 = attn_dkv_kernel<T, DP, NW>;
  if (int e = allow_lds(reinterpret_cast<const void*>(f1), lds1)) return e;
  if (int e = allow_lds(reinterpret_cast<const void*>(f2), lds2)) return e;
  float* delta = o.ws;
  float* part = o.ws + a.heads * a.beads;
  hipLaunchKernelGGL(f1, dim3((unsigned)(a.n_tiles * a.heads)), dim3(64 * NW), lds1, s, a,
                     (const T*)a.out_or_null, (T*)o.dq, delta, o.order, o.first, part);
  hipLaunchKernelGGL(f2, dim3((unsigned)(a.n_tiles * (a.heads / a.group))), dim3(64 * NW), lds2, s,
                     a, delta, (T*)o.dk, (T*)o.dv);
  hipLaunchKernelGGL(attn_dtable_kernel<T>, dim3(mlcg_div_up(a.buckets, 8), a.heads), dim3(256), 0,
                     s, part, a.n_tiles, a.buckets, a.heads, (T*)o.dtable);
  return mlcg_launch_status();
}

template <typename F>
int by_dim(int dim, F f) {
  if (dim <= 32) return f(std::integral_constant<int, 32>());
  if (dim <= 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}

template <typename F>
int by_type(int dtype, F f) {
  switch (dtype) {
    case MLCG_DTYPE_F32: return f(float{});
    case MLCG_DTYPE_F16: return f(_Float16{});
    case MLCG_DTYPE_BF16: return f(__bf16{});
  }
  return MLCG_ERR_UNSUPPORTED;
}

// vector loads and stores of four elements: every row and head starts at a
// multiple of four
bool attn_vec(const AttnArgs& a, int size) {
  const void* p[] = {a.q, a.k, a.v, a.out_or_null, a.grad};
  for (const void* x : p)
    if (reinterpret_cast<uintptr_t>(x) % (4 * size)) return false;
  const int64_t st[] = {a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head, a.dim};
  for (int64_t x : st)
    if (x % 4) return false;
  return true;
}

bool attn_ok(const AttnArgs& a, int tile_rows, int dtype) {
  return a.beads >= 0 && a.beads < (int64_t(1) << 31) - 128 && a.n_tiles >= 0 && a.heads >= 1 &&
         a.heads <= 1024 && a.group >= 1 && a.heads % a.group == 0 && a.dim >= 1 && a.dim <= 128 &&
         a.reach >= 1 && a.reach <= 1024 && a.buckets >= 1 &&
         (int64_t)a.n_tiles * a.heads < (int64_t(1) << 31) &&
         (tile_rows == 32 || tile_rows == 128) && dtype >= MLCG_DTYPE_F32 &&
         dtype <= MLCG_DTYPE_BF16;
}

}  // namespace

extern "C" int64_t mlcg_chain_attention_workspace_floats(int64_t beads, int heads,
                                                         int64_t n_tiles, int buckets) {
  if (beads < 0 || heads < 1 || n_tiles < 0 || buckets < 1) return -1;
  return heads * (beads + n_tiles * buckets);
}

extern "C" int mlcg_chain_attention(const void* q, const int64_t* q_strides, const void* k,
                                    const int64_t* k_strides, const void* v,
                                    const int64_t* v_strides, int64_t beads, int heads,
                                    int kv_heads, int dim, int dtype, const void* table,
                                    int buckets, const int32_t* bucket_of, int reach, float scale,
                                    const int32_t* tiles, int64_t n_tiles, int tile_rows,
                                    const uint8_t* keep, const int32_t* positions, void* out,
                                    float* lse, void* stream) {
  MLCG_REQUIRE(q_strides && k_strides && v_strides && kv_heads >= 1 && heads >= 1 &&
               heads % kv_heads == 0 && n_tiles >= 0 && n_tiles < (int64_t(1) << 31));
  AttnArgs a{q, k, v, table, out, nullptr, q_strides[0], q_strides[1], k_strides[0],
             k_strides[1], v_strides[0], v_strides[1], beads, bucket_of,
             reinterpret_cast<const int4*>(tiles), keep, positions, lse, (int)n_tiles, heads,
             heads / kv_heads, dim, reach, buckets, 0, scale};
  MLCG_REQUIRE(attn_ok(a, tile_rows, dtype));
  if (beads == 0 || n_tiles == 0) return MLCG_OK;
  MLCG_REQUIRE(q && k && v && table && bucket_of && tiles && out);
  hipStream_t s = mlcg_stream(stream);
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    a.vec = attn_vec(a, sizeof(T));
    return by_dim(dim, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      return tile_rows == 32 ? launch_fwd<T, DP, 1>(a, out, s) : launch_fwd<T, DP, 4>(a, out, s);
    });
  });
}

extern "C" int mlcg_chain_attention_backward(
    const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides, int64_t beads, int heads, int kv_heads, int dim,
    int dtype, const void* table, int buckets, const int32_t* bucket_of,
    const int32_t* bucket_order, const int32_t* bucket_first, int reach, float scale,
    const int32_t* tiles, int64_t n_tiles, int tile_rows, const uint8_t* keep,
    const int32_t* positions, const void* out, const float* lse, const void* grad_out,
    void* grad_q, void* grad_k, void* grad_v, void* grad_table, float* workspace,
    int64_t workspace_floats, void* stream) {
  MLCG_REQUIRE(q_strides && k_strides && v_strides && kv_heads >= 1 && heads >= 1 &&
               heads % kv_heads == 0 && n_tiles >= 1 && n_tiles < (int64_t(1) << 31));
  AttnArgs a{q, k, v, table, out, grad_out, q_strides[0], q_strides[1], k_strides[0],
             k_strides[1], v_strides[0], v_strides[1], beads, bucket_of,
             reinterpret_cast<const int4*>(tiles), keep, positions, const_cast<float*>(lse),
             (int)n_tiles, heads, heads / kv_heads, dim, reach, buckets, 0, scale};
  MLCG_REQUIRE(attn_ok(a, tile_rows, dtype) && beads >= 1);
  MLCG_REQUIRE(q && k && v && table && bucket_of && bucket_order && bucket_first && tiles && out &&
               lse && grad_out && grad_q && grad_k && grad_v && grad_table && workspace);
  MLCG_REQUIRE(workspace_floats >=
               mlcg_chain_attention_workspace_floats(beads, heads, n_tiles, buckets));
  hipStream_t s = mlcg_stream(stream);
  const BwdOut o{grad_q, grad_k, grad_v, grad_table, workspace, bucket_order, bucket_first};
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    a.vec = attn_vec(a, sizeof(T));
    return by_dim(dim, [&](auto dp) {
      constexpr int DP = decltype(dp)::value;
      return tile_rows == 32 ? launch_bwd<T, DP, 1>(a, o, s) : launch_bwd<T, DP, 4>(a, o, s);
    });
  });
}
