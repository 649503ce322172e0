// The gated delta rule along chains of beads (gfx950).
//
// A head's state S (Dk x Dv, fp32) goes from bead to bead of a chain,
//   S <- e^g S,   S <- S + beta k (v - S^T k)^T,   o = scale S^T q,
// forwards or, `reverse`, from the last bead to the first; q and k may be
// brought to length one (r = 1 / sqrt(x.x + 1e-6)) before.  An absent bead
// (keep = 0) has no k, v, g and beta; its q still reads the state.
//
// Chunks of C = 64 beads.  With G the sum of g from the chunk's start up to and
// with a bead, E_ts = e^(G_t - G_s), S0 the state before the chunk and
//   A_ts = beta_t E_ts k_t.k_s (s < t),   P_ts = scale E_ts q_t.k_s (s <= t),
// what the beads add, u, and the outputs and the state after the chunk are
//   (1 + A) u = beta (v - e^G S0^T k),    T = (1 + A)^-1,
//   o = scale e^G S0^T q + P u,           S = e^G_C S0 + sum_s e^(G_C - G_s) k_s u_s^T.
// Backward, with D the gradient of the state after the chunk:
//   du = P^T do + e^(G_C - G_s) D^T k,    dr = T^T du,    dv = beta dr,
//   D0 = e^G_C D + sum scale e^G q do^T - sum beta e^G k dr^T,
// and with everything known at both ends of a chunk the other gradients:
//   dq_t  = scale (e^G_t S0 do_t + sum_s E_ts (do_t.u_s) k_s),
//   dkr_t = -(e^G_t S0 dr_t + sum_{s<t} E_ts (dr_t.u_s) k_s)        (k that reads)
//   dkw_s = e^(G_C-G_s) D u_s + sum_t scale E_ts (do_t.u_s) q_t
//           - sum_{t>s} beta_t E_ts (dr_t.u_s) k_t                   (k that writes)
//   dk = beta dkr + dkw,   dbeta_t = dr_t.v_t + k_t.dkr_t,
//   dG_t = q_t.dq_t + beta_t k_t.dkr_t - k_t.dkw_t, and <S, D> at the last one;
// dg is dG summed from the end of the chunk.
//
// Four kernels: delta_chunk forms T, P and the beads' factors of every chunk;
// delta_scan carries the state along the chunks (16 columns of it a wave) and
// gives u and o; delta_scan_back carries D; delta_grad gives the gradients of
// q, k, beta and g of every chunk.
//
// The state, and all sums, are fp32.  Products are on the bf16 matrix
// instructions with operands in pieces, x = x0 + x1 + ..., each the rounding
// of what the ones before leave: one for bf16 arrays and two for fp16 (exact),
// three for fp32 (2^-24); two for what is computed from 16-bit arrays (2^-17,
// and bf16's range, so that gradients of any size keep their digits), three
// from fp32.  Of the products of pieces those are taken that reach this far.
//
// A result of the 16 x 16 x 32 instruction has 4 rows of one column in a lane,
// which is half of what the next product wants of its right operand if its
// sum's index runs in the order 4 g + j, 16 + 4 g + j (g the lane's quarter): the
// chains K S -> T (..) -> K^T (..) stay in registers, and the left operands are
// read in that order, rows as they are or, by the transposing read, columns.
#pragma once

#include "chain.h"

constexpr int kDeltaRows = 64;       // beads of a chunk
constexpr int kDeltaThreads = 256;
constexpr int kDeltaFactors = 8;     // arrays of factors of a chunk and head
constexpr int kDeltaPlane = kDeltaRows * kDeltaRows;

// a chunk's factors, [kDeltaFactors][64] for each (chunk, head)
enum {
  kFacRead = 0,    // e^G r_k
  kFacWrite = 1,   // e^(G_C - G) r_k
  kFacBeta = 2,
  kFacOut = 3,     // scale e^G r_q
  kFacHi = 4,      // G / ln 2 in two parts: differences of them are exact where
  kFacLo = 5,      // large parts cancel
  kFacK = 6,       // r_k, 0 for an absent bead
  kFacQ = 7        // r_q
};

struct DeltaArgs {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  const float *decay, *beta;                            // [beads, heads]
  const uint8_t* keep;
  int64_t beads;
  int heads, keys, group, dk, dv, dvp;  // dvp: dv rounded up to 16
  float scale;
  int normalize, reverse, vec;  // vec: rows of q and k in 16-byte loads
  const int4* tiles;            // (chain's first row, its length, tile's first row in it, chain)
  int n_tiles;
  const int4* segs;             // (chain, first tile, tiles, 1 first of its chain | 2 last)
  const int* seg_first;         // [chains with beads + 1]
  int n_segs, n_whole;          // segments; chains with beads
  float* fac;
  __bf16 *T, *P;
  float *U, *S0;  // [heads, beads, dvp], [tile, heads, DK, dvp]
};

struct DeltaBack {
  const void* grad;       // [beads, heads, dv]
  const float* grad_state;
  void *dq, *dk, *dv;
  float *ddecay, *dbeta, *dstate;
  float *D, *dR;          // [tile, heads, DK, dvp], [heads, beads, dvp]
};

// where a scan begins and ends
struct DeltaEnds {
  const float* init;  // the caller's states [chain, heads, dk, dv], or of segments, or NULL
  float* last;        // the caller's
  const float* seg_init;  // [seg, heads, DK, dvp]
  float* seg_last;        // [seg, heads, DK, dvp]: the segments alone, from zero
  float* seg_map;         // [seg, heads, DK, DK]: what they make of a state
};

template <typename T>
int delta_forward(const DeltaArgs& a, void* out, const DeltaEnds& e, float* ws, hipStream_t s);
template <typename T>
int delta_backward(const DeltaArgs& a, const DeltaBack& b, const DeltaEnds& e, float* ws,
                   hipStream_t s);

static inline int delta_dk(int dk) { return dk <= 32 ? 32 : dk <= 64 ? 64 : 128; }

#ifdef MLCG_DELTA_TYPE

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// pieces of the arrays' elements and of what is computed from them
template <typename T> struct Pieces;
template <> struct Pieces<__bf16> { static constexpr int in = 1, mid = 2; };
template <> struct Pieces<_Float16> { static constexpr int in = 2, mid = 2; };
template <> struct Pieces<float> { static constexpr int in = 3, mid = 3; };

template <int N>
struct Frag {
  bf16x8 p[N];
};

template <int N>
__device__ __forceinline__ Frag<N> split8(f32x8 x) {
  Frag<N> f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    f.p[i] = __builtin_convertvector(x, bf16x8);
    if (i + 1 < N) x -= __builtin_convertvector(f.p[i], f32x8);
  }
  return f;
}
template <int N>
__device__ __forceinline__ Frag<N> split44(f32x4 lo, f32x4 hi) {
  return split8<N>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
template <int N, typename T>
__device__ __forceinline__ Frag<N> split_raw(v8<T> x) {
  if constexpr (sizeof(T) == 2 && N == 1) {
    Frag<N> f;
    f.p[0] = __builtin_bit_cast(bf16x8, x);
    return f;
  } else {
    return split8<N>(__builtin_convertvector(x, f32x8));
  }
}

// c += a b to the accuracy of the operand with more pieces
template <int NA, int NB>
__device__ __forceinline__ void mma(f32x4& c, const Frag<NA>& a, const Frag<NB>& b) {
  constexpr int most = NA > NB ? NA : NB;
#pragma unroll
  for (int o = most - 1; o >= 0; --o)  // the small products first
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = o - i;
      if (j >= 0 && j < NB)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], c, 0, 0, 0);
    }
}

__device__ __forceinline__ int wave_number() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

// A tile of 64 rows of LEN elements in LDS, in N planes.  A row's stride of 16
// more bytes moves it by four banks: the 16 rows x 16 bytes of half a wave of
// the reads below fall on all banks.
template <int N, int LEN>
struct Tile {
  static constexpr int stride = LEN + 8, plane = kDeltaRows * stride;
  __bf16 x[N * plane];

  // left operand: row `row`, its elements 32 kk + 4 g .. and 32 kk + 16 + 4 g ..
  __device__ __forceinline__ Frag<N> rows(int row, int kk) const {
    const int g = mlcg_lane() >> 4;
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const __bf16* p = x + i * plane + row * stride + 32 * kk + 4 * g;
      const bf16x4 lo = *reinterpret_cast<const bf16x4*>(p);
      const bf16x4 hi = *reinterpret_cast<const bf16x4*>(p + 16);
      f.p[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }
  // left operand: column 16 m + (lane & 15), its rows 32 kk + 4 g .. and 32 kk + 16 + 4 g ..
  __device__ __forceinline__ Frag<N> columns(int m, int kk) const {
    const int lane = mlcg_lane(), g = lane >> 4;
    // 16 lanes give the places of 4 rows x 16 columns, lane i those of row
    // i / 4, and get a column's 4 rows each
    const int row = 32 * kk + 4 * g + ((lane & 15) >> 2), el = 16 * m + 4 * (lane & 3);
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s16x4 r[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        r[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4*)(x + i * plane + (row + 16 * h) * stride + el));
      f.p[i] = __builtin_bit_cast(bf16x8,
                                  __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return f;
  }
};

// Where the beads of a chunk are.
struct Chunk {
  int64_t base;  // bead of row 0
  int n, step;   // rows, and +1 or -1
  __device__ __forceinline__ Chunk(const DeltaArgs& a, int tile) {
    const int4 t = a.tiles[tile];
    n = min(kDeltaRows, t.y - t.z);
    base = (int64_t)t.x + (a.reverse ? t.y - 1 - t.z : t.z);
    step = a.reverse ? -1 : 1;
  }
  __device__ __forceinline__ int64_t bead(int row) const { return base + (int64_t)row * step; }
};

// 8 elements of a row from el on, zeros past `len`
template <typename T>
__device__ __forceinline__ v8<T> load8(const T* row, int el, int len, bool vec) {
  v8<T> x{};
  if (vec) {
    if (el < len) x = *reinterpret_cast<const v8<T>*>(row + el);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (el + j < len) x[j] = row[el + j];
  }
  return x;
}

// A chunk's rows of q or k on their way to LDS.
template <typename T, int DK, int N>
struct StageRows {
  static constexpr int per_row = DK / 8, per = kDeltaRows * per_row / kDeltaThreads;
  v8<T> x[per];
  __device__ __forceinline__ void load(const DeltaArgs& a, const Chunk& c, const T* src,
                                       int64_t row_stride, bool masked) {
#pragma unroll
    for (int p = 0; p < per; ++p) {
      const int i = threadIdx.x + p * kDeltaThreads, row = i / per_row;
      x[p] = v8<T>{};
      if (row < c.n) {
        const int64_t bead = c.bead(row);
        if (!masked || !a.keep || a.keep[bead])
          x[p] = load8<T>(src + bead * row_stride, 8 * (i % per_row), a.dk, a.vec);
      }
    }
  }
  __device__ __forceinline__ void put(Tile<N, DK>& t) const {
#pragma unroll
    for (int p = 0; p < per; ++p) {
      const int i = threadIdx.x + p * kDeltaThreads;
      const Frag<N> f = split_raw<N, T>(x[p]);
#pragma unroll
      for (int j = 0; j < N; ++j)
        *reinterpret_cast<bf16x8*>(t.x + j * t.plane + i / per_row * t.stride +
                                   8 * (i % per_row)) = f.p[j];
    }
  }
};

// A chunk's T or P, planes of 64 x 64, on their way to LDS.
template <int N>
struct StageMatrix {
  static constexpr int per = N * kDeltaPlane / 8 / kDeltaThreads;
  bf16x8 x[per];
  __device__ __forceinline__ void load(const __bf16* src) {
#pragma unroll
    for (int p = 0; p < per; ++p)
      x[p] = *reinterpret_cast<const bf16x8*>(src + 8 * (threadIdx.x + p * kDeltaThreads));
  }
  __device__ __forceinline__ void put(Tile<N, kDeltaRows>& t) const {
#pragma unroll
    for (int p = 0; p < per; ++p) {
      const int i = threadIdx.x + p * kDeltaThreads, j = i / (kDeltaPlane / 8),
                r = i % (kDeltaPlane / 8);
      *reinterpret_cast<bf16x8*>(t.x + j * t.plane + r / 8 * t.stride + 8 * (r % 8)) = x[p];
    }
  }
};

__device__ __forceinline__ float exp2_of(float hi, float lo) {
  return __builtin_amdgcn_exp2f(hi + lo);
}

// sum over the four quarters of a wave
__device__ __forceinline__ float quarter_sum(float v) {
  v += __shfl_xor(v, 16, MLCG_WAVE);
  return v + __shfl_xor(v, 32, MLCG_WAVE);
}

// ---------------------------------------------------------------------------
// T, P and the factors of a chunk, for the heads of one key head.

template <typename T, int DK>
__global__ __launch_bounds__(kDeltaThreads) void delta_chunk(DeltaArgs a) {
  constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid, KS = DK / 32;
  constexpr int LD = kDeltaRows + 4;
  __shared__ __align__(16) float A[kDeltaRows][LD];
  __shared__ __align__(16) float diag[4][16][20];  // inverses of the diagonal blocks
  __shared__ float ghi[kDeltaRows], glo[kDeltaRows], rk[kDeltaRows], rq[kDeltaRows],
      be[kDeltaRows];
  const int tile = blockIdx.x, kh = blockIdx.y;
  const int w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const Chunk ch(a, tile);
  const T* const q = (const T*)a.q + kh * a.q_head;
  const T* const k = (const T*)a.k + kh * a.k_head;

  // products of this wave's 16 beads (columns) with those up to them (rows)
  Frag<NI> kb[KS], qb[KS];
  float nk = 0.0f, nq = 0.0f;
  const int row = 16 * w + c;
  bool there = false;
  {
    const bool in = row < ch.n;
    const int64_t bead = in ? ch.bead(row) : 0;
    there = in && (!a.keep || a.keep[bead]);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v8<T> x{}, y{};
      if (there) x = load8<T>(k + bead * a.k_row, 32 * s + 8 * g, a.dk, a.vec);
      if (in) y = load8<T>(q + bead * a.q_row, 32 * s + 8 * g, a.dk, a.vec);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        nk = fmaf((float)x[j], (float)x[j], nk);
        nq = fmaf((float)y[j], (float)y[j], nq);
      }
      kb[s] = split_raw<NI, T>(x);
      qb[s] = split_raw<NI, T>(y);
    }
  }
  nk = quarter_sum(nk);
  nq = quarter_sum(nq);
  if (g == 0) {
    rk[row] = !there ? 0.0f : a.normalize ? 1.0f / sqrtf(nk + 1e-6f) : 1.0f;
    rq[row] = a.normalize ? 1.0f / sqrtf(nq + 1e-6f) : 1.0f;
  }
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    kk[m] = f32x4{};
    qk[m] = f32x4{};
    if (m > w) continue;
    const int r = 16 * m + c;
    const bool in = r < ch.n;
    const int64_t bead = in ? ch.bead(r) : 0;
    const bool here = in && (!a.keep || a.keep[bead]);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v8<T> x{};
      if (here) x = load8<T>(k + bead * a.k_row, 32 * s + 8 * g, a.dk, a.vec);
      const Frag<NI> f = split_raw<NI, T>(x);
      mma(kk[m], f, kb[s]);
      mma(qk[m], f, qb[s]);
    }
  }

  for (int h = kh * a.group; h < (kh + 1) * a.group; ++h) {
    const int64_t at = (int64_t)tile * a.heads + h;
    __syncthreads();  // rk, rq; the last head's A has been read
    if (w == 0) {
      const bool in = lane < ch.n;
      const int64_t bead = in ? ch.bead(lane) : 0;
      const bool here = in && (!a.keep || a.keep[bead]);
      float d = here ? a.decay[bead * a.heads + h] : 0.0f;
      const float b = here ? a.beta[bead * a.heads + h] : 0.0f;
      if (d < -256.0f) d = -256.0f;  // e^g is 0 all the same, and -inf - -inf no number
      double G = (double)d * 1.4426950408889634;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(G, o, MLCG_WAVE);
        if (lane >= o) G += up;
      }
      const float hi = (float)G, lo = (float)(G - (double)hi);
      const float hc = __shfl(hi, 63, MLCG_WAVE), lc = __shfl(lo, 63, MLCG_WAVE);
      ghi[lane] = hi;
      glo[lane] = lo;
      be[lane] = b;
      const float e = exp2_of(hi, lo);
      float* const f = a.fac + at * (kDeltaFactors * kDeltaRows) + lane;
      f[kFacRead * kDeltaRows] = e * rk[lane];
      f[kFacWrite * kDeltaRows] = exp2_of(hc - hi, lc - lo) * rk[lane];
      f[kFacBeta * kDeltaRows] = b;
      f[kFacOut * kDeltaRows] = a.scale * e * rq[lane];
      f[kFacHi * kDeltaRows] = hi;
      f[kFacLo * kDeltaRows] = lo;
      f[kFacK * kDeltaRows] = rk[lane];
      f[kFacQ * kDeltaRows] = rq[lane];
    }
    __syncthreads();
    // rows s = 16 m + 4 g + i, column t = 16 w + c
    const float th = ghi[row], tl = glo[row], bt = be[row] * rk[row], qt = a.scale * rq[row];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f32x4 x, y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = 16 * m + 4 * g + i;
        const float e = s <= row ? exp2_of(th - ghi[s], tl - glo[s]) * rk[s] : 0.0f;
        x[i] = s < row ? bt * e * kk[m][i] : 0.0f;
        y[i] = s <= row ? qt * e * qk[m][i] : 0.0f;
      }
      *reinterpret_cast<f32x4*>(&A[row][16 * m + 4 * g]) = x;
      __bf16* p = a.P + at * (NM * kDeltaPlane) + row * kDeltaRows + 16 * m + 4 * g;
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        const bf16x4 z = __builtin_convertvector(y, bf16x4);
        *reinterpret_cast<bf16x4*>(p + i * kDeltaPlane) = z;
        y -= __builtin_convertvector(z, f32x4);
      }
    }
    __syncthreads();
    // (1 + A)^-1: column c of the inverse of this wave's diagonal block, by
    // substitution ...
    float z[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float s = r == c ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < r; ++j) s = fmaf(-A[16 * w + r][16 * w + j], z[j], s);
      z[r] = s;
    }
    if (g == 0)
#pragma unroll
      for (int r = 0; r < 16; ++r) diag[w][r][c] = z[r];
    __syncthreads();
    // ... and the blocks below it, T_i = -T_ii sum_j A_ij T_j, in fp32
    f32x4 t[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) t[m] = f32x4{};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < w) continue;
      if (i == w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[i][e] = diag[w][4 * g + e][c];
        continue;
      }
      f32x4 s{};
#pragma unroll
      for (int j = 0; j < i; ++j) {
        if (j < w) continue;
        const f32x4 l = *reinterpret_cast<const f32x4*>(&A[16 * i + c][16 * j + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s = __builtin_amdgcn_mfma_f32_16x16x4f32(l[e], t[j][e], s, 0, 0, 0);
      }
      const f32x4 l = *reinterpret_cast<const f32x4*>(&diag[i][c][4 * g]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        t[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-l[e], s[e], t[i], 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) A[16 * i + 4 * g + e][16 * w + c] = t[i][e];
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int i = threadIdx.x + p * kDeltaThreads, r = i / 8, s = 8 * (i % 8);
      const Frag<NM> f = split44<NM>(*reinterpret_cast<const f32x4*>(&A[r][s]),
                                     *reinterpret_cast<const f32x4*>(&A[r][s + 4]));
#pragma unroll
      for (int j = 0; j < NM; ++j)
        *reinterpret_cast<bf16x8*>(a.T + (at * NM + j) * kDeltaPlane + r * kDeltaRows + s) =
            f.p[j];
    }
  }
}

// ---------------------------------------------------------------------------
// The state along the chunks of a segment: 16 columns a wave, 64 a workgroup.

// a head's 16 x 4 rows of a column of v, do: rows 16 b + 4 g + i
template <typename T>
__device__ __forceinline__ void load_column(f32x4 (&x)[4], const Chunk& ch, const T* src,
                                            int64_t stride, bool in) {
  const int g = mlcg_lane() >> 4;
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * b + 4 * g + i;
      x[b][i] = in && r < ch.n ? (float)src[ch.bead(r) * stride] : 0.0f;
    }
}

template <typename T, int DK>
struct ScanTiles {
  static constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid;
  Tile<NI, DK> k, q;
  Tile<NM, kDeltaRows> t, p;
  float fac[4][kDeltaRows];  // the first four
  float decay;               // e^G_C
};

// a chunk's tiles on their way to LDS
template <typename T, int DK>
struct ScanStage {
  StageRows<T, DK, Pieces<T>::in> k, q;
  StageMatrix<Pieces<T>::mid> t, p;
  float fac, hi, lo;
  __device__ __forceinline__ void load(const DeltaArgs& a, int tile, int h) {
    const Chunk ch(a, tile);
    const int64_t at = (int64_t)tile * a.heads + h;
    k.load(a, ch, (const T*)a.k + h / a.group * a.k_head, a.k_row, true);
    q.load(a, ch, (const T*)a.q + h / a.group * a.q_head, a.q_row, false);
    t.load(a.T + at * (Pieces<T>::mid * kDeltaPlane));
    p.load(a.P + at * (Pieces<T>::mid * kDeltaPlane));
    const float* f = a.fac + at * (kDeltaFactors * kDeltaRows);
    fac = f[threadIdx.x];
    hi = f[kFacHi * kDeltaRows + 63];
    lo = f[kFacLo * kDeltaRows + 63];
  }
  __device__ __forceinline__ void put(ScanTiles<T, DK>& s) const {
    k.put(s.k);
    q.put(s.q);
    t.put(s.t);
    p.put(s.p);
    s.fac[threadIdx.x / kDeltaRows][threadIdx.x % kDeltaRows] = fac;
    if (threadIdx.x == 0) s.decay = exp2_of(hi, lo);
  }
};

// a state's 16 columns from `at` on: rows 16 b + 4 g + i, column c of them
template <int DK>
__device__ __forceinline__ void load_state(f32x4 (&s)[DK / 16], const float* at, int ld, int rows,
                                           bool in) {
  const int g = mlcg_lane() >> 4, c = mlcg_lane() & 15;
#pragma unroll
  for (int b = 0; b < DK / 16; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * b + 4 * g + i;
      s[b][i] = in && r < rows ? at[(int64_t)r * ld + c] : 0.0f;
    }
}
template <int DK>
__device__ __forceinline__ void store_state(const f32x4 (&s)[DK / 16], float* at, int ld, int rows,
                                            bool in) {
  const int g = mlcg_lane() >> 4, c = mlcg_lane() & 15;
#pragma unroll
  for (int b = 0; b < DK / 16; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * b + 4 * g + i;
      if (in && r < rows) at[(int64_t)r * ld + c] = s[b][i];
    }
}

// Alone: what a segment makes of the state zero (columns of v) and, in the
// workgroups past those, of every unit vector; no outputs.
template <typename T, int DK, bool ALONE>
__global__ __launch_bounds__(kDeltaThreads) void delta_scan(DeltaArgs a, DeltaEnds e, T* out) {
  constexpr int NM = Pieces<T>::mid, KS = DK / 32, B = DK / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  ScanTiles<T, DK>& sh = *reinterpret_cast<ScanTiles<T, DK>*>(smem);
  const int4 seg = a.segs[blockIdx.x];
  const int h = blockIdx.y, w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const int nz = (a.dv + 63) / 64;
  const bool unit = ALONE && (int)blockIdx.z >= nz;
  const int v0 = 64 * (unit ? blockIdx.z - nz : blockIdx.z) + 16 * w;
  const bool live = v0 < (unit ? DK : a.dvp);   // wave-uniform
  const bool in = !unit && v0 + c < a.dv;
  const T* const v = (const T*)a.v + h * a.v_head + (in ? v0 + c : 0);
  f32x4 S[B];
  if (ALONE) {
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[b][i] = unit && 16 * b + 4 * g + i == v0 + c ? 1.0f : 0.0f;
  } else if (e.seg_init) {
    load_state<DK>(S, e.seg_init + ((int64_t)blockIdx.x * a.heads + h) * (DK * a.dvp) + v0, a.dvp,
                   DK, live);
  } else {
    load_state<DK>(S, e.init + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                   a.dk, e.init && in);
  }
  ScanStage<T, DK> next;
  f32x4 vn[4];
  next.load(a, seg.y, h);
  load_column<T>(vn, Chunk(a, seg.y), v, a.v_row, in);
  for (int n = 0; n < seg.z; ++n) {
    const int tile = seg.y + n;
    next.put(sh);
    f32x4 X[4], O[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) X[b] = vn[b];
    __syncthreads();
    if (n + 1 < seg.z) {
      next.load(a, tile + 1, h);
      load_column<T>(vn, Chunk(a, tile + 1), v, a.v_row, in);
    }
    if (live) {
      const int64_t at = (int64_t)tile * a.heads + h;
      if (!ALONE && a.S0) store_state<DK>(S, a.S0 + at * (DK * a.dvp) + v0, a.dvp, DK, true);
      const Chunk ch(a, tile);
      Frag<NM> s[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) s[i] = split44<NM>(S[2 * i], S[2 * i + 1]);
      Frag<NM> x[2];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f32x4 y{};
        O[b] = f32x4{};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          mma(y, sh.k.rows(16 * b + c, i), s[i]);
          if (!ALONE) mma(O[b], sh.q.rows(16 * b + c, i), s[i]);
        }
        const f32x4 read = *reinterpret_cast<const f32x4*>(&sh.fac[kFacRead][16 * b + 4 * g]);
        const f32x4 beta = *reinterpret_cast<const f32x4*>(&sh.fac[kFacBeta][16 * b + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i)  // an absent bead's v may be no number
          X[b][i] = beta[i] == 0.0f ? 0.0f : beta[i] * fmaf(-read[i], y[i], X[b][i]);
      }
      x[0] = split44<NM>(X[0], X[1]);
      x[1] = split44<NM>(X[2], X[3]);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        X[b] = f32x4{};
#pragma unroll
        for (int i = 0; i <= b / 2; ++i) mma(X[b], sh.t.rows(16 * b + c, i), x[i]);
      }
      if (!ALONE) {
        x[0] = split44<NM>(X[0], X[1]);
        x[1] = split44<NM>(X[2], X[3]);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          O[b] *= *reinterpret_cast<const f32x4*>(&sh.fac[kFacOut][16 * b + 4 * g]);
#pragma unroll
          for (int i = 0; i <= b / 2; ++i) mma(O[b], sh.p.rows(16 * b + c, i), x[i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 16 * b + 4 * g + i;
            if (r >= ch.n) continue;
            const int64_t bead = ch.bead(r);
            if (a.U) a.U[(h * a.beads + bead) * a.dvp + v0 + c] = X[b][i];
            if (in) out[(bead * a.heads + h) * a.dv + v0 + c] = (T)O[b][i];
          }
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b)
        X[b] *= *reinterpret_cast<const f32x4*>(&sh.fac[kFacWrite][16 * b + 4 * g]);
      x[0] = split44<NM>(X[0], X[1]);
      x[1] = split44<NM>(X[2], X[3]);
      const float decay = sh.decay;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        S[b] *= decay;
#pragma unroll
        for (int i = 0; i < 2; ++i) mma(S[b], sh.k.columns(b, i), x[i]);
      }
    }
    __syncthreads();
  }
  if (!live) return;
  if (ALONE) {
    const int64_t at = (int64_t)blockIdx.x * a.heads + h;
    if (unit)
      store_state<DK>(S, e.seg_map + at * (DK * DK) + v0, DK, DK, true);
    else
      store_state<DK>(S, e.seg_last + at * (DK * a.dvp) + v0, a.dvp, DK, true);
  } else if (e.last && (seg.w & 2)) {
    store_state<DK>(S, e.last + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                    a.dk, in);
  }
}

// The states before the segments of a chain, one after the other: S <- M S + N.
// Backward: after them, the last one first, S <- M^T S + N.
template <int DK, bool BACK>
__global__ __launch_bounds__(kDeltaThreads) void delta_join(DeltaArgs a, DeltaEnds e,
                                                            float* seg_init) {
  constexpr int B = DK / 16;
  const int h = blockIdx.y, w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const int v0 = 64 * blockIdx.z + 16 * w;
  if (v0 >= a.dvp) return;
  const int first = a.seg_first[blockIdx.x], n = a.seg_first[blockIdx.x + 1] - first;
  const int chain = a.segs[first].x;
  f32x4 S[B];
  load_state<DK>(S, e.init + ((int64_t)chain * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                 a.dk, e.init && v0 + c < a.dv);
  for (int j = 0; j < n; ++j) {
    const int seg = first + (BACK ? n - 1 - j : j);
    const int64_t at = (int64_t)seg * a.heads + h;
    store_state<DK>(S, seg_init + at * (DK * a.dvp) + v0, a.dvp, DK, true);
    if (j + 1 == n) break;
    f32x4 next[B];
    load_state<DK>(next, e.seg_last + at * (DK * a.dvp) + v0, a.dvp, DK, true);
    const float* const M = e.seg_map + at * (DK * DK);
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < B; ++i) {
        f32x4 l;
        if (BACK) {
#pragma unroll
          for (int x = 0; x < 4; ++x) l[x] = M[(16 * i + 4 * g + x) * DK + 16 * b + c];
        } else {
          l = *reinterpret_cast<const f32x4*>(M + (16 * b + c) * DK + 16 * i + 4 * g);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
          next[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(l[x], S[i][x], next[b], 0, 0, 0);
      }
#pragma unroll
    for (int b = 0; b < B; ++b) S[b] = next[b];
  }
}

// The state's gradient along the chunks of a segment, the last one first.
template <typename T, int DK, bool ALONE>
__global__ __launch_bounds__(kDeltaThreads) void delta_scan_back(DeltaArgs a, DeltaBack o,
                                                                 DeltaEnds e) {
  constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid, KS = DK / 32, B = DK / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  ScanTiles<T, DK>& sh = *reinterpret_cast<ScanTiles<T, DK>*>(smem);
  const int4 seg = a.segs[blockIdx.x];
  const int h = blockIdx.y, w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const int v0 = 64 * blockIdx.z + 16 * w;
  const bool live = v0 < a.dvp, in = v0 + c < a.dv;
  const T* const grad = (const T*)o.grad + h * a.dv + (in ? v0 + c : 0);
  const int64_t grad_row = (int64_t)a.heads * a.dv;
  f32x4 D[B];
  if (ALONE) {
#pragma unroll
    for (int b = 0; b < B; ++b) D[b] = f32x4{};
  } else if (e.seg_init) {
    load_state<DK>(D, e.seg_init + ((int64_t)blockIdx.x * a.heads + h) * (DK * a.dvp) + v0, a.dvp,
                   DK, live);
  } else {
    load_state<DK>(D, e.init + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                   a.dk, e.init && in);
  }
  ScanStage<T, DK> next;
  f32x4 gn[4];
  next.load(a, seg.y + seg.z - 1, h);
  load_column<T>(gn, Chunk(a, seg.y + seg.z - 1), grad, grad_row, in);
  for (int n = seg.z - 1; n >= 0; --n) {
    const int tile = seg.y + n;
    next.put(sh);
    f32x4 G[4], X[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) G[b] = gn[b];
    __syncthreads();
    if (n > 0) {
      next.load(a, tile - 1, h);
      load_column<T>(gn, Chunk(a, tile - 1), grad, grad_row, in);
    }
    if (live) {
      const int64_t at = (int64_t)tile * a.heads + h;
      if (!ALONE) store_state<DK>(D, o.D + at * (DK * a.dvp) + v0, a.dvp, DK, true);
      const Chunk ch(a, tile);
      Frag<NM> d[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) d[i] = split44<NM>(D[2 * i], D[2 * i + 1]);
      const Frag<NI> go[2] = {split44<NI>(G[0], G[1]), split44<NI>(G[2], G[3])};
      Frag<NM> x[2];
      // du
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        X[b] = f32x4{};
#pragma unroll
        for (int i = 0; i < KS; ++i) mma(X[b], sh.k.rows(16 * b + c, i), d[i]);
        X[b] *= *reinterpret_cast<const f32x4*>(&sh.fac[kFacWrite][16 * b + 4 * g]);
#pragma unroll
        for (int i = b / 2; i < 2; ++i) mma(X[b], sh.p.columns(b, i), go[i]);
      }
      x[0] = split44<NM>(X[0], X[1]);
      x[1] = split44<NM>(X[2], X[3]);
      // dr
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        X[b] = f32x4{};
#pragma unroll
        for (int i = b / 2; i < 2; ++i) mma(X[b], sh.t.columns(b, i), x[i]);
        const f32x4 beta = *reinterpret_cast<const f32x4*>(&sh.fac[kFacBeta][16 * b + 4 * g]);
        const f32x4 read = *reinterpret_cast<const f32x4*>(&sh.fac[kFacRead][16 * b + 4 * g]);
        if (!ALONE) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 16 * b + 4 * g + i;
            if (r >= ch.n) continue;
            const int64_t bead = ch.bead(r);
            o.dR[(h * a.beads + bead) * a.dvp + v0 + c] = X[b][i];
            if (in) ((T*)o.dv)[(bead * a.heads + h) * a.dv + v0 + c] = (T)(beta[i] * X[b][i]);
          }
        }
        X[b] *= -(beta * read);
        G[b] *= *reinterpret_cast<const f32x4*>(&sh.fac[kFacOut][16 * b + 4 * g]);
      }
      x[0] = split44<NM>(X[0], X[1]);
      x[1] = split44<NM>(X[2], X[3]);
      const Frag<NM> gs[2] = {split44<NM>(G[0], G[1]), split44<NM>(G[2], G[3])};
      const float decay = sh.decay;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        D[b] *= decay;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          mma(D[b], sh.q.columns(b, i), gs[i]);
          mma(D[b], sh.k.columns(b, i), x[i]);
        }
      }
    }
    __syncthreads();
  }
  if (!live) return;
  if (ALONE) {
    store_state<DK>(D, e.seg_last + ((int64_t)blockIdx.x * a.heads + h) * (DK * a.dvp) + v0, a.dvp,
                    DK, true);
  } else if (o.dstate && (seg.w & 1)) {
    store_state<DK>(D, o.dstate + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0,
                    a.dv, a.dk, in);
  }
}

// ---------------------------------------------------------------------------
// The gradients of q, k, beta and g of a chunk's beads, for the heads of one
// key head; a wave has 16 beads, as columns.

template <typename T, int DK>
struct GradTiles {
  Tile<Pieces<T>::in, DK> k, q;
  float fac[kDeltaFactors][kDeltaRows];
  float dG[kDeltaRows];
  float ends[4];
};

// 8 floats of a padded row from el on, zeros past its end
__device__ __forceinline__ f32x8 load_f8(const float* row, int el, int len, bool in) {
  f32x8 x{};
  if (in && el < len) x = *reinterpret_cast<const f32x8*>(row + el);
  return x;
}

// 4 elements of a row from el on, as floats
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* row, int el, int len, bool vec) {
  f32x4 x{};
  if (vec) {
    if (el < len) x = __builtin_convertvector(*reinterpret_cast<const v4<T>*>(row + el), f32x4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (el + j < len) x[j] = (float)row[el + j];
  }
  return x;
}

template <typename T, int DK>
__global__ __launch_bounds__(kDeltaThreads) void delta_grad(DeltaArgs a, DeltaBack o, int gvec) {
  constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid, B = DK / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  GradTiles<T, DK>& sh = *reinterpret_cast<GradTiles<T, DK>*>(smem);
  const int tile = blockIdx.x, kh = blockIdx.y;
  const int w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const Chunk ch(a, tile);
  const T* const q = (const T*)a.q + kh * a.q_head;
  const T* const k = (const T*)a.k + kh * a.k_head;
  {
    StageRows<T, DK, NI> s;
    s.load(a, ch, k, a.k_row, true);
    s.put(sh.k);
    s.load(a, ch, q, a.q_row, false);
    s.put(sh.q);
  }
  const int row = 16 * w + c;
  const bool in = row < ch.n;
  const int64_t bead = in ? ch.bead(row) : 0;
  const bool there = in && (!a.keep || a.keep[bead]);
  f32x4 dq[B], dk[B];
#pragma unroll
  for (int b = 0; b < B; ++b) dq[b] = dk[b] = f32x4{};
  float rq = 0.0f, rk = 0.0f;

  for (int h = kh * a.group; h < (kh + 1) * a.group; ++h) {
    const int64_t at = (int64_t)tile * a.heads + h;
    __syncthreads();  // sh.dG of the last head has been read
    for (int i = threadIdx.x; i < kDeltaFactors * kDeltaRows; i += kDeltaThreads)
      sh.fac[i / kDeltaRows][i % kDeltaRows] = a.fac[at * (kDeltaFactors * kDeltaRows) + i];
    __syncthreads();
    const float* const U = a.U + h * a.beads * a.dvp;
    const float* const R = o.dR + h * a.beads * a.dvp;
    const T* const go = (const T*)o.grad + h * a.dv;
    const int64_t go_row = (int64_t)a.heads * a.dv;
    const float* const S0 = a.S0 + at * (DK * a.dvp);
    const float* const D = o.D + at * (DK * a.dvp);

    // [bead before][this wave's bead], and [bead after][this wave's bead]:
    // ou, ru = do_t.u_s and dr_t.u_s
    f32x4 ou0[4], ru0[4], ou1[4], ru1[4], hq[B], hr[B], hw[B];
#pragma unroll
    for (int m = 0; m < 4; ++m) ou0[m] = ru0[m] = ou1[m] = ru1[m] = f32x4{};
#pragma unroll
    for (int b = 0; b < B; ++b) hq[b] = hr[b] = hw[b] = f32x4{};
    float rv = 0.0f, sd = 0.0f;  // dr.v;  this wave's part of <S0, D>
    for (int v0 = 0; v0 < a.dvp; v0 += 32) {
      const int el = v0 + 8 * g;
      const f32x8 ur = load_f8(U + bead * a.dvp, el, a.dvp, in);
      const f32x8 rr = load_f8(R + bead * a.dvp, el, a.dvp, in);
      v8<T> gr{}, vr{};
      if (in) gr = load8<T>(go + bead * go_row, el, a.dv, gvec & 1);
      if (there) vr = load8<T>((const T*)a.v + bead * a.v_row + h * a.v_head, el, a.dv, gvec & 2);
#pragma unroll
      for (int j = 0; j < 8; ++j) rv = fmaf(rr[j], (float)vr[j], rv);
      const Frag<NM> ub = split8<NM>(ur), rb = split8<NM>(rr);
      const Frag<NI> gb = split_raw<NI, T>(gr);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int r = 16 * m + c;
        const bool rin = r < ch.n;
        const int64_t rb_ = rin ? ch.bead(r) : 0;
        if (m <= w) {
          const Frag<NM> f = split8<NM>(load_f8(U + rb_ * a.dvp, el, a.dvp, rin));
          mma(ou0[m], f, gb);
          mma(ru0[m], f, rb);
        }
        if (m >= w) {
          v8<T> x{};
          if (rin) x = load8<T>(go + rb_ * go_row, el, a.dv, gvec & 1);
          const Frag<NI> f = split_raw<NI, T>(x);
          mma(ou1[m], f, ub);
          const Frag<NM> f2 = split8<NM>(load_f8(R + rb_ * a.dvp, el, a.dvp, rin));
          mma(ru1[m], f2, ub);
        }
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const f32x8 s = load_f8(S0 + (16 * b + c) * a.dvp, el, a.dvp, true);
        const f32x8 d = load_f8(D + (16 * b + c) * a.dvp, el, a.dvp, true);
        if (b % 4 == w)
#pragma unroll
          for (int j = 0; j < 8; ++j) sd = fmaf(s[j], d[j], sd);
        const Frag<NM> f = split8<NM>(s);
        mma(hq[b], f, gb);
        mma(hr[b], f, rb);
        mma(hw[b], split8<NM>(d), ub);
      }
    }
    // factors of this wave's beads
    const float th = sh.fac[kFacHi][row], tl = sh.fac[kFacLo][row];
    const float ch_hi = sh.fac[kFacHi][63], ch_lo = sh.fac[kFacLo][63];
    const float first = exp2_of(th, tl), rest = exp2_of(ch_hi - th, ch_lo - tl);
    const float beta = sh.fac[kFacBeta][row];
    rk = sh.fac[kFacK][row];
    rq = sh.fac[kFacQ][row];
    float kd = 0.0f;  // k.(e^(G_C - G) D u)
#pragma unroll
    for (int b = 0; b < B; ++b) {
      hq[b] *= first;
      hr[b] *= -first;
      hw[b] *= rest;
      f32x4 x{};
      if (there) x = load4<T>(k + bead * a.k_row, 16 * b + 4 * g, a.dk, a.vec);
#pragma unroll
      for (int i = 0; i < 4; ++i) kd = fmaf(rk * x[i], hw[b][i], kd);
    }
    // inside the chunk
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * m + 4 * g + i;
        const float dh = th - sh.fac[kFacHi][r], dl = tl - sh.fac[kFacLo][r];
        const float xk = sh.fac[kFacK][r];
        const float e0 = r <= row ? exp2_of(dh, dl) * xk : 0.0f;
        ou0[m][i] = r <= row ? e0 * ou0[m][i] : 0.0f;
        ru0[m][i] = r < row ? -e0 * ru0[m][i] : 0.0f;
        const float e1 = r >= row ? exp2_of(-dh, -dl) : 0.0f;
        ou1[m][i] = r >= row ? e1 * sh.fac[kFacQ][r] * a.scale * ou1[m][i] : 0.0f;
        ru1[m][i] = r > row ? -e1 * xk * sh.fac[kFacBeta][r] * ru1[m][i] : 0.0f;
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const Frag<NM> o0 = split44<NM>(ou0[2 * i], ou0[2 * i + 1]);
      const Frag<NM> r0 = split44<NM>(ru0[2 * i], ru0[2 * i + 1]);
      const Frag<NM> o1 = split44<NM>(ou1[2 * i], ou1[2 * i + 1]);
      const Frag<NM> r1 = split44<NM>(ru1[2 * i], ru1[2 * i + 1]);
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const Frag<NI> kc = sh.k.columns(b, i), qc = sh.q.columns(b, i);
        mma(hq[b], kc, o0);
        mma(hr[b], kc, r0);
        mma(hw[b], qc, o1);
        mma(hw[b], kc, r1);
      }
    }
    float qd = 0.0f, kr = 0.0f, kw = 0.0f;
#pragma unroll
    for (int b = 0; b < B; ++b) {
      f32x4 x{}, y{};
      if (there) x = load4<T>(k + bead * a.k_row, 16 * b + 4 * g, a.dk, a.vec);
      if (in) y = load4<T>(q + bead * a.q_row, 16 * b + 4 * g, a.dk, a.vec);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qd = fmaf(rq * y[i], hq[b][i], qd);
        kr = fmaf(rk * x[i], hr[b][i], kr);
        kw = fmaf(rk * x[i], hw[b][i], kw);
      }
      dq[b] += hq[b];
      dk[b] += beta * hr[b] + hw[b];
    }
    qd = quarter_sum(qd);
    kr = quarter_sum(kr);
    kw = quarter_sum(kw);
    rv = quarter_sum(rv);
    if (g == 0) {
      sh.dG[row] = a.scale * qd + beta * kr - kw;
      if (in) o.dbeta[bead * a.heads + h] = there ? rv + kr : 0.0f;
    }
    // <S, D> = e^G_C <S0, D> + sum k.(e^(G_C - G) D u)
    const float end = mlcg_wave_sum(fmaf(exp2_of(ch_hi, ch_lo), sd, kd));
    if (lane == 0) sh.ends[w] = end;
    __syncthreads();
    if (w == 0) {
      double s = sh.dG[lane];
      if (lane == 63)
        s += ((double)sh.ends[0] + sh.ends[1]) + ((double)sh.ends[2] + sh.ends[3]);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double up = __shfl_down(s, d, MLCG_WAVE);
        if (lane + d < 64) s += up;
      }
      if (lane < ch.n) {
        const int64_t x = ch.bead(lane) * a.heads + h;
        const bool here = !a.keep || a.keep[ch.bead(lane)];
        // the derivative of e^g where that is 0
        o.ddecay[x] = !here || a.decay[x] < -104.0f ? 0.0f : (float)s;
      }
    }
  }
  // through the lengths of q and k
  float pq = 0.0f, pk = 0.0f;
  f32x4 kx[B], qx[B];
#pragma unroll
  for (int b = 0; b < B; ++b) {
    kx[b] = qx[b] = f32x4{};
    if (there) kx[b] = load4<T>(k + bead * a.k_row, 16 * b + 4 * g, a.dk, a.vec) * rk;
    if (in) qx[b] = load4<T>(q + bead * a.q_row, 16 * b + 4 * g, a.dk, a.vec) * rq;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pq = fmaf(qx[b][i], dq[b][i], pq);
      pk = fmaf(kx[b][i], dk[b][i], pk);
    }
  }
  pq = quarter_sum(pq);
  pk = quarter_sum(pk);
  if (!a.normalize) pq = pk = 0.0f;
  if (!in) return;
  T* const oq = (T*)o.dq + (bead * a.keys + kh) * a.dk;
  T* const ok = (T*)o.dk + (bead * a.keys + kh) * a.dk;
  const bool wide = a.dk % 4 == 0;
#pragma unroll
  for (int b = 0; b < B; ++b) {
    const int el = 16 * b + 4 * g;
    if (el >= a.dk) continue;
    const f32x4 x = (dq[b] - qx[b] * pq) * (a.scale * rq), y = (dk[b] - kx[b] * pk) * rk;
    if (wide) {
      *reinterpret_cast<v4<T>*>(oq + el) = __builtin_convertvector(x, v4<T>);
      *reinterpret_cast<v4<T>*>(ok + el) = __builtin_convertvector(y, v4<T>);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (el + i < a.dk) {
          oq[el + i] = (T)x[i];
          ok[el + i] = (T)y[i];
        }
    }
  }
}

// ---------------------------------------------------------------------------

inline bool lds_limit(const void* f, size_t bytes) {
  return hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) ==
         hipSuccess;
}

template <typename T, int DK>
int forward_dk(const DeltaArgs& a, T* out, DeltaEnds e, float* ws, hipStream_t s) {
  const size_t lds = sizeof(ScanTiles<T, DK>);
  const unsigned nz = mlcg_div_up(a.dv, 64);
  hipLaunchKernelGGL((delta_chunk<T, DK>), dim3(a.n_tiles, a.keys), dim3(kDeltaThreads), 0, s, a);
  if (e.seg_last) {
    const auto alone = delta_scan<T, DK, true>;
    if (!lds_limit(reinterpret_cast<const void*>(alone), lds)) return MLCG_ERR_LAUNCH;
    hipLaunchKernelGGL(alone, dim3(a.n_segs, a.heads, nz + mlcg_div_up(DK, 64)),
                       dim3(kDeltaThreads), lds, s, a, e, out);
    hipLaunchKernelGGL((delta_join<DK, false>), dim3(a.n_whole, a.heads, nz), dim3(kDeltaThreads),
                       0, s, a, e, ws);
    e.seg_init = ws;
  }
  const auto scan = delta_scan<T, DK, false>;
  if (!lds_limit(reinterpret_cast<const void*>(scan), lds)) return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(scan, dim3(a.n_segs, a.heads, nz), dim3(kDeltaThreads), lds, s, a, e, out);
  return mlcg_launch_status();
}

template <typename T, int DK>
int backward_dk(const DeltaArgs& a, const DeltaBack& o, DeltaEnds e, float* ws, hipStream_t s) {
  const size_t lds = sizeof(ScanTiles<T, DK>);
  const unsigned nz = mlcg_div_up(a.dv, 64);
  const dim3 grid(a.n_segs, a.heads, nz);
  if (e.seg_last) {
    const auto alone = delta_scan_back<T, DK, true>;
    if (!lds_limit(reinterpret_cast<const void*>(alone), lds)) return MLCG_ERR_LAUNCH;
    hipLaunchKernelGGL(alone, grid, dim3(kDeltaThreads), lds, s, a, o, e);
    hipLaunchKernelGGL((delta_join<DK, true>), dim3(a.n_whole, a.heads, nz), dim3(kDeltaThreads),
                       0, s, a, e, ws);
    e.seg_init = ws;
  }
  const auto scan = delta_scan_back<T, DK, false>;
  if (!lds_limit(reinterpret_cast<const void*>(scan), lds)) return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(scan, grid, dim3(kDeltaThreads), lds, s, a, o, e);
  const bool gv = a.dv % 8 == 0 && chain_aligned16(o.grad);
  const bool vv = a.dv % 8 == 0 && chain_aligned16(a.v) && a.v_row * sizeof(T) % 16 == 0 &&
                  a.v_head * sizeof(T) % 16 == 0;
  const auto grad = delta_grad<T, DK>;
  const size_t glds = sizeof(GradTiles<T, DK>);
  if (!lds_limit(reinterpret_cast<const void*>(grad), glds)) return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(grad, dim3(a.n_tiles, a.keys), dim3(kDeltaThreads), glds, s, a, o,
                     (gv ? 1 : 0) | (vv ? 2 : 0));
  return mlcg_launch_status();
}

template <typename T>
DeltaArgs with_vec(DeltaArgs a) {
  bool ok = a.dk % 8 == 0 && chain_aligned16(a.q) && chain_aligned16(a.k);
  for (int64_t x : {a.q_row, a.q_head, a.k_row, a.k_head}) ok = ok && x * sizeof(T) % 16 == 0;
  a.vec = ok;
  return a;
}

}  // namespace

template <>
int delta_forward<MLCG_DELTA_TYPE>(const DeltaArgs& args, void* out, const DeltaEnds& e, float* ws,
                                   hipStream_t s) {
  typedef MLCG_DELTA_TYPE T;
  const DeltaArgs a = with_vec<T>(args);
  switch (delta_dk(a.dk)) {
    case 32: return forward_dk<T, 32>(a, (T*)out, e, ws, s);
    case 64: return forward_dk<T, 64>(a, (T*)out, e, ws, s);
    default: return forward_dk<T, 128>(a, (T*)out, e, ws, s);
  }
}

template <>
int delta_backward<MLCG_DELTA_TYPE>(const DeltaArgs& args, const DeltaBack& b, const DeltaEnds& e,
                                    float* ws, hipStream_t s) {
  typedef MLCG_DELTA_TYPE T;
  const DeltaArgs a = with_vec<T>(args);
  switch (delta_dk(a.dk)) {
    case 32: return backward_dk<T, 32>(a, b, e, ws, s);
    case 64: return backward_dk<T, 64>(a, b, e, ws, s);
    default: return backward_dk<T, 128>(a, b, e, ws, s);
  }
}

#endif  // MLCG_DELTA_TYPE
