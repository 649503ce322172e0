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
// q, k, beta and g of every chunk.  Of few long chains the scans go over segments
// of chunks at the same time: once from the state zero and from all unit vectors,
// which gives the map of a segment, S -> M S + N; delta_join goes along these, and
// the scan proper begins each segment at the state that it gives.
//
// The state, and all sums, are fp32.  Products are on the bf16 matrix
// instructions with operands in pieces, x = x0 + x1 + ..., each the rounding
// of what the ones before leave: one for bf16 arrays and two for fp16 (exact),
// three for fp32 and for all that is computed (2^-24, and in bf16's range, so that
// gradients of any size keep their digits).  Of the products of pieces those are
// taken that reach this far.  Two pieces for what is computed from 16-bit arrays
// would take a fifth to a third less time, but leave the states and the gradients
// of decay and beta, which are fp32, 4e-6 to 1e-5 off.
//
// A result of the 16 x 16 x 32 instruction has 4 rows of one column in a lane,
// which is half of what the next product wants of its right operand if its
// sum's index runs in the order 4 g + j, 16 + 4 g + j (g the lane's quarter): the
// chains K S -> T (..) -> K^T (..) stay in registers.  k, q, T and P lie in memory
// and in LDS as the left operands that they are, in blocks of 16 rows x 32 columns:
// lane (g, c) has row c's elements 4 g .. and 16 + 4 g .. in the 16 bytes of slot
// 16 g + (c ^ 8 (g / 2)).  delta_chunk writes them so, absent beads and rows past
// the end as zeros, and every later copy is one of memory to LDS as it stands.
// The exchange of c spreads what the transposing read takes over more banks.
#pragma once

#include "chain.h"

constexpr int kDeltaRows = 64;       // beads of a chunk
constexpr int kDeltaThreads = 256;   // of delta_chunk and delta_grad
constexpr int kDeltaFactors = 8;     // arrays of factors of a chunk and head
constexpr int kDeltaLower = 6;       // blocks of a lower triangle, 16 x 32

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
  int heads, keys, group, dk, dv, dvp;  // dvp: dv rounded up to 32
  float scale;
  int normalize, reverse;
  const int4* tiles;            // (chain's first row, its length, tile's first row in it, chain)
  int n_tiles;
  const int4* segs;             // (chain, first tile, tiles, 1 first of its chain | 2 last)
  const int* seg_first;         // [chains with beads + 1]
  int n_segs, n_whole;          // segments; chains with beads
  float* fac;
  float4 *K, *Q;                // operands, [tile, keys, pieces, 4, DK / 32, 64 slots]
  float4 *T, *P;                // [tile, heads, pieces, 6, 64 slots]
  float4 *U, *S0;               // operands: u, and the states' transposes, or NULL
};

struct DeltaBack {
  const void* grad;       // [beads, heads, dv]
  void *dq, *dk, *dv;
  float *ddecay, *dbeta, *dstate;
  float4 *D, *dR;         // as S0 and U
};

// where a scan begins and ends
struct DeltaEnds {
  const float* init;      // the caller's states [chain, heads, dk, dv], or NULL
  float* last;            // the caller's
  const float* seg_init;  // [seg, heads, DK, dvp]
  float* seg_last;        // [seg, heads, DK, dvp]: the segments alone, from zero
  float4* seg_map;        // the transpose of what they make of a state, as operands
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
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;

// pieces of the arrays' elements and of what is computed from them
template <typename T> struct Pieces;
template <> struct Pieces<__bf16> { static constexpr int in = 1, mid = 3; };
template <> struct Pieces<_Float16> { static constexpr int in = 2, mid = 3; };
template <> struct Pieces<float> { static constexpr int in = 3, mid = 3; };

template <int N>
struct Frag {
  bf16x8 p[N];
};

// What a piece leaves is x - 1 x0 + 0 x0', one instruction on the pair that the
// rounding gave (exact: x0 is the rounding of x).
template <int N>
__device__ __forceinline__ Frag<N> split8(f32x8 x) {
  // (-1, 0) and (0, -1), from registers: as a constant in the instruction -1.0 is
  // taken by the hardware in another half than the compiler means
  uint32_t c0 = 0x0000BF80u, c1 = 0xBF800000u;
  asm("" : "+v"(c0), "+v"(c1));
  const bf16x2 first = __builtin_bit_cast(bf16x2, c0), second = __builtin_bit_cast(bf16x2, c1);
  Frag<N> f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    f.p[i] = __builtin_convertvector(x, bf16x8);
    if (i + 1 < N)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const bf16x2 h = {f.p[i][j], f.p[i][j + 1]};
        x[j] = __builtin_amdgcn_fdot2_f32_bf16(h, first, x[j], false);
        x[j + 1] = __builtin_amdgcn_fdot2_f32_bf16(h, second, x[j + 1], false);
      }
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
// the sum of the pieces
template <int N>
__device__ __forceinline__ f32x8 whole(const Frag<N>& f) {
  f32x8 x = __builtin_convertvector(f.p[N - 1], f32x8);
#pragma unroll
  for (int i = N - 2; i >= 0; --i) x += __builtin_convertvector(f.p[i], f32x8);
  return x;
}
template <int HALF>
__device__ __forceinline__ f32x4 half_of(f32x8 x) {
  return HALF ? __builtin_shufflevector(x, x, 4, 5, 6, 7)
              : __builtin_shufflevector(x, x, 0, 1, 2, 3);
}

// c += a b: products of pieces down to 2^-24 of the first (piece i is 2^-8i of its
// operand or less), those of two exact operands of two pieces with them
template <int NA, int NB>
__device__ __forceinline__ void mma(f32x4& c, const Frag<NA>& a, const Frag<NB>& b) {
  constexpr int last = NA + NB < 4 ? NA + NB - 2 : 2;
#pragma unroll
  for (int o = last; o >= 0; --o)  // the small products first
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = o - i;
      if (j >= 0 && j < NB)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], c, 0, 0, 0);
    }
}

// a value that all lanes have, as the one that it is
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int4 uniform(int4 x) {
  return make_int4(uniform(x.x), uniform(x.y), uniform(x.z), uniform(x.w));
}
__device__ __forceinline__ int wave_number() { return uniform(threadIdx.x >> 6); }

// A barrier for what the workgroup shares in LDS: loads and stores of memory stay
// on their way across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Operands in LDS: N planes of NB blocks.
template <int N, int NB>
struct Image {
  static constexpr int units = N * NB;  // of 1 KB
  float4 x[units * 64];

  __device__ static __forceinline__ int slot() {
    const int g = mlcg_lane() >> 4, c = mlcg_lane() & 15;
    return 16 * g + (c ^ (8 * (g >> 1)));
  }
  // a block as a left operand
  __device__ __forceinline__ Frag<N> rows(int block) const {
    Frag<N> f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      f.p[i] = __builtin_bit_cast(bf16x8, x[(i * NB + block) * 64 + slot()]);
    return f;
  }
  // The transposes of blocks b0 and b1 (32 rows), as left operands: columns 0 .. 15
  // and 16 .. 31 of them, and with c0 and c1 those of a second pair.  16 lanes give
  // the places of 4 rows x 16 columns, lane i those of row i / 4, and get a column's
  // 4 rows each.  The reads and their wait are one piece of assembly: before its own
  // form of this read (columns_now) the compiler waits for everything that is on its
  // way from memory, the next chunk, too; but that leaves it more freedom, and
  // delta_grad, whose registers are short, is faster with it (2 x 4099, 8 heads of 64
  // on 4 in bf16, 70 us against 76; 48 x 268, 8 heads of 16 in fp32, 37 against 41;
  // 512 x 100, 8 heads of 32 in bf16, 71 against 67).
  __device__ __forceinline__ lds_s16x4* column_place(int piece, int block) const {
    const int lane = mlcg_lane(), s = lane & 3, r = 4 * (lane >> 4) + ((lane & 15) >> 2);
    return (lds_s16x4*)&x[(piece * NB + block) * 64 + 16 * s + (r ^ (8 * (s >> 1)))];
  }
  __device__ __forceinline__ void columns_now(int b0, int b1, Frag<N> (&f)[2]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      lds_s16x4 *const p0 = column_place(i, b0), *const p1 = column_place(i, b1);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f[j].p[i] = joined(__builtin_amdgcn_ds_read_tr16_b64_v4i16(p0 + j),
                           __builtin_amdgcn_ds_read_tr16_b64_v4i16(p1 + j));
    }
  }
  __device__ static __forceinline__ bf16x8 joined(s16x4 lo, s16x4 hi) {
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  __device__ __forceinline__ void columns(int b0, int b1, Frag<N> (&f)[2]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s16x4 r0, r1, r2, r3;
      asm volatile(
          "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %5\n\t"
          "ds_read_b64_tr_b16 %2, %4 offset:8\n\tds_read_b64_tr_b16 %3, %5 offset:8\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
          : "v"(column_place(i, b0)), "v"(column_place(i, b1))
          : "memory");
      f[0].p[i] = joined(r0, r1);
      f[1].p[i] = joined(r2, r3);
    }
  }
  __device__ __forceinline__ void columns(int b0, int b1, int c0, int c1, Frag<N> (&f)[2],
                                          Frag<N> (&g)[2]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s16x4 r0, r1, r2, r3, q0, q1, q2, q3;
      asm volatile(
          "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %9\n\t"
          "ds_read_b64_tr_b16 %2, %8 offset:8\n\tds_read_b64_tr_b16 %3, %9 offset:8\n\t"
          "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %11\n\t"
          "ds_read_b64_tr_b16 %6, %10 offset:8\n\tds_read_b64_tr_b16 %7, %11 offset:8\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3), "=&v"(q0), "=&v"(q1), "=&v"(q2), "=&v"(q3)
          : "v"(column_place(i, b0)), "v"(column_place(i, b1)), "v"(column_place(i, c0)),
            "v"(column_place(i, c1))
          : "memory");
      f[0].p[i] = joined(r0, r1);
      f[1].p[i] = joined(r2, r3);
      g[0].p[i] = joined(q0, q1);
      g[1].p[i] = joined(q2, q3);
    }
  }
};

// UNITS x 1 KB from memory to LDS, on their way when this returns
template <int UNITS, int WAVES>
__device__ __forceinline__ void send_to_lds(float4* lds, const float4* src) {
  const int w = wave_number(), lane = mlcg_lane();
#pragma unroll
  for (int u = 0; u < (UNITS + WAVES - 1) / WAVES; ++u) {
    const int unit = u * WAVES + w;
    if ((u + 1) * WAVES <= UNITS || unit < UNITS)
      __builtin_amdgcn_global_load_lds((global_void*)(src + 64 * unit + lane),
                                       (lds_void*)(lds + 64 * unit), 16, 0, 0);
  }
}
// What this wave has sent for is there.  Memory is not touched across it in either
// direction: the wait by itself says nothing of memory to the compiler.
__device__ __forceinline__ void wait_for_memory() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);
  asm volatile("" ::: "memory");
}

// Where the beads of a chunk are.
struct Chunk {
  int64_t base;  // bead of row 0
  int n, step;   // rows, and +1 or -1
  Chunk() = default;
  __device__ __forceinline__ Chunk(const DeltaArgs& a, int tile) {
    const int4 t = uniform(a.tiles[tile]);
    n = min(kDeltaRows, t.y - t.z);
    base = (int64_t)t.x + (a.reverse ? t.y - 1 - t.z : t.z);
    step = a.reverse ? -1 : 1;
  }
  __device__ __forceinline__ int64_t bead(int row) const { return base + (int64_t)row * step; }
  // elements from row 0 to a row, rows past the end taken as the last one
  __device__ __forceinline__ int offset(int row, int stride) const {
    return min(row, n - 1) * step * stride;
  }
};

// The rows r + l of a whole chunk, r the same for all lanes and l of 0 .. most by
// lane, of an array of rows: an address that is the same for all lanes and an
// offset, not negative, that is the same for all r.
struct Lines {
  char* at;
  int stride;  // bytes
  uint32_t lane;
  __device__ __forceinline__ Lines(void* p, int64_t base, int step, int row_bytes, int l, int most,
                                   int column_bytes) {
    at = reinterpret_cast<char*>(p) + (step > 0 ? base : base - most) * row_bytes;
    stride = step * row_bytes;
    lane = (uint32_t)((step > 0 ? l : most - l) * row_bytes + column_bytes);
    // not known to be the same from chunk to chunk: its multiples would be kept
    asm volatile("" : "+s"(stride));
  }
  template <typename T>
  __device__ __forceinline__ T& row(int r) const {
    return *reinterpret_cast<T*>(at + r * stride + lane);
  }
};

// The chunks of a segment one after the other, without looking them up.
struct Walk {
  int first, len, at;  // the chain's first bead and length, the chunk's first row in it
  __device__ __forceinline__ Walk(const DeltaArgs& a, int tile) {
    const int4 t = uniform(a.tiles[tile]);
    first = t.x;
    len = t.y;
    at = t.z;
  }
  __device__ __forceinline__ Chunk chunk(const DeltaArgs& a, int rows_on) const {
    Chunk c;
    const int from = at + rows_on;
    c.n = min(kDeltaRows, len - from);
    c.base = (int64_t)first + (a.reverse ? len - 1 - from : from);
    c.step = a.reverse ? -1 : 1;
    return c;
  }
};

// elements that are aligned as one
template <typename T, int N>
struct loose {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// 4 elements of a row of len (a multiple of 8) from el on, zeros past its end: without
// a branch, so that loads are not waited for one by one
template <typename T>
__device__ __forceinline__ v4<T> load4(const T* row, int el, int len) {
  const v4<T> x = *reinterpret_cast<const typename loose<T, 4>::type*>(row + min(el, len - 4));
  return el < len ? x : v4<T>{};
}
// 4 values to a row of len (a multiple of 8) from el on
template <typename T>
__device__ __forceinline__ void store4(T* row, int el, int len, f32x4 x) {
  typedef typename loose<T, 4>::type vec;
  if (el < len) *reinterpret_cast<vec*>(row + el) = __builtin_convertvector(x, vec);
}

__device__ __forceinline__ float exp2_of(float hi, float lo) {
  return __builtin_amdgcn_exp2f(hi + lo);
}

// sum over the four quarters of a wave
__device__ __forceinline__ float quarter_sum(float v) {
  v += __shfl_xor(v, 16, MLCG_WAVE);
  return v + __shfl_xor(v, 32, MLCG_WAVE);
}

// ---------------------------------------------------------------------------
// T, P and the factors of a chunk, for the heads of one key head, and k and q as
// operands.  Where there are many chunks bound by what it writes: 1 x 120001 beads, 8
// heads of 64 in bf16, 221 us, 5.1 TB/s; 512 x 100, 4 heads of 32, 37 us, 4.6 TB/s.

template <typename T, int DK>
struct ChunkTiles {
  Image<Pieces<T>::in, DK / 8> k;
  float A[kDeltaRows][kDeltaRows + 4];
  float diag[4][16][20];  // inverses of the diagonal blocks
  float ghi[kDeltaRows], glo[kDeltaRows], rk[kDeltaRows], rq[kDeltaRows], be[kDeltaRows];
};

template <typename T, int DK>
__global__ __launch_bounds__(kDeltaThreads, (sizeof(T) == 4 && DK == 128 ? 2 : 4)) void delta_chunk(
    DeltaArgs a) {
  constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid, KS = DK / 32, NB = 4 * KS;
  extern __shared__ __align__(16) unsigned char smem[];
  ChunkTiles<T, DK>& sh = *reinterpret_cast<ChunkTiles<T, DK>*>(smem);
  auto& A = sh.A;
  const int tile = blockIdx.x, kh = blockIdx.y;
  const int w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const int slot = sh.k.slot();
  const Chunk ch(a, tile);
  const int row = 16 * w + c;
  const bool in = row < ch.n;
  const int64_t bead = ch.bead(min(row, ch.n - 1));
  const bool there = in && (!a.keep || a.keep[bead]);

  // the first wave makes a head's gates: what they are made of is sent for early
  const int64_t gate = ch.bead(min(lane, ch.n - 1));
  const bool gated = lane < ch.n && (!a.keep || a.keep[gate]);
  float dn = 0.0f, bn = 0.0f;
  const auto send_gates = [&](int h) {
    if (w == 0) {
      dn = a.decay[gate * a.heads + h];
      bn = a.beta[gate * a.heads + h];
    }
  };
  send_gates(kh * a.group);

  // this wave's 16 beads, as columns
  Frag<NI> kb[KS], qb[KS];
  float nk = 0.0f, nq = 0.0f;
  {
    const T* const q = (const T*)a.q + kh * a.q_head + bead * a.q_row;
    const T* const k = (const T*)a.k + kh * a.k_head + bead * a.k_row;
    v4<T> x[KS][2], y[KS][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[s][j] = load4<T>(k, 32 * s + 16 * j + 4 * g, a.dk);
        y[s][j] = load4<T>(q, 32 * s + 16 * j + 4 * g, a.dk);
      }
    const int64_t at = ((int64_t)tile * a.keys + kh) * (NI * NB * 64) + w * KS * 64 + slot;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      v8<T> u = __builtin_shufflevector(x[s][0], x[s][1], 0, 1, 2, 3, 4, 5, 6, 7);
      v8<T> v = __builtin_shufflevector(y[s][0], y[s][1], 0, 1, 2, 3, 4, 5, 6, 7);
      if (!there) u = v8<T>{};
      if (!in) v = v8<T>{};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        nk = fmaf((float)u[j], (float)u[j], nk);
        nq = fmaf((float)v[j], (float)v[j], nq);
      }
      kb[s] = split_raw<NI, T>(u);
      qb[s] = split_raw<NI, T>(v);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const float4 f = __builtin_bit_cast(float4, kb[s].p[i]);
        sh.k.x[(i * NB + w * KS + s) * 64 + slot] = f;
        a.K[at + (i * NB + s) * 64] = f;
        a.Q[at + (i * NB + s) * 64] = __builtin_bit_cast(float4, qb[s].p[i]);
      }
    }
  }
  nk = quarter_sum(nk);
  nq = quarter_sum(nq);
  if (g == 0) {
    sh.rk[row] = !there ? 0.0f : a.normalize ? 1.0f / sqrtf(nk + 1e-6f) : 1.0f;
    sh.rq[row] = a.normalize ? 1.0f / sqrtf(nq + 1e-6f) : 1.0f;
  }
  __syncthreads();
  // products with the beads up to them
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    kk[m] = f32x4{};
    qk[m] = f32x4{};
    if (m > w) continue;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const Frag<NI> f = sh.k.rows(m * KS + s);
      mma(kk[m], f, kb[s]);
      mma(qk[m], f, qb[s]);
    }
  }

  for (int h = kh * a.group; h < (kh + 1) * a.group; ++h) {
    const int64_t at = (int64_t)tile * a.heads + h;
    if (w == 0) {
      float d = gated ? dn : 0.0f;
      const float b = gated ? bn : 0.0f;
      if (h + 1 < (kh + 1) * a.group) send_gates(h + 1);
      if (d < -256.0f) d = -256.0f;  // e^g is 0 all the same, and -inf - -inf no number
      double G = (double)d * 1.4426950408889634;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(G, o, MLCG_WAVE);
        if (lane >= o) G += up;
      }
      const float hi = (float)G, lo = (float)(G - (double)hi);
      const float hc = __shfl(hi, 63, MLCG_WAVE), lc = __shfl(lo, 63, MLCG_WAVE);
      sh.ghi[lane] = hi;
      sh.glo[lane] = lo;
      sh.be[lane] = b;
      const float e = exp2_of(hi, lo), rk = sh.rk[lane], rq = sh.rq[lane];
      float* const f = a.fac + at * (kDeltaFactors * kDeltaRows) + lane;
      f[kFacRead * kDeltaRows] = e * rk;
      f[kFacWrite * kDeltaRows] = exp2_of(hc - hi, lc - lo) * rk;
      f[kFacBeta * kDeltaRows] = b;
      f[kFacOut * kDeltaRows] = a.scale * e * rq;
      f[kFacHi * kDeltaRows] = hi;
      f[kFacLo * kDeltaRows] = lo;
      f[kFacK * kDeltaRows] = rk;
      f[kFacQ * kDeltaRows] = rq;
    }
    __syncthreads();
    // rows s = 16 m + 4 g + i, column t = 16 w + c
    const float th = sh.ghi[row], tl = sh.glo[row];
    const float bt = sh.be[row] * sh.rk[row], qt = a.scale * sh.rq[row];
    f32x4 y[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = 16 * m + 4 * g + i;
        const float e = s <= row ? exp2_of(th - sh.ghi[s], tl - sh.glo[s]) * sh.rk[s] : 0.0f;
        x[i] = s < row ? bt * e * kk[m][i] : 0.0f;
        y[m][i] = s <= row ? qt * e * qk[m][i] : 0.0f;
      }
      if (m <= w) *reinterpret_cast<f32x4*>(&A[row][16 * m + 4 * g]) = x;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (j > w / 2) continue;
      const Frag<NM> f = split44<NM>(y[2 * j], y[2 * j + 1]);
#pragma unroll
      for (int i = 0; i < NM; ++i)
        a.P[((at * NM + i) * kDeltaLower + w + (w == 3) + j) * 64 + slot] =
            __builtin_bit_cast(float4, f.p[i]);
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
      for (int r = 0; r < 16; ++r) sh.diag[w][r][c] = z[r];
    __syncthreads();
    // ... and the blocks below it, T_i = -T_ii sum_j A_ij T_j, in fp32
    f32x4 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = f32x4{};
      if (i < w) continue;
      if (i == w) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[i][e] = sh.diag[w][4 * g + e][c];
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
      const f32x4 l = *reinterpret_cast<const f32x4*>(&sh.diag[i][c][4 * g]);
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
    for (int u = w; u < kDeltaLower; u += 4) {
      const int b = u < 2 ? u : 2 + (u - 2) / 2, j = u < 2 ? 0 : u % 2;
      const Frag<NM> f =
          split44<NM>(*reinterpret_cast<const f32x4*>(&A[16 * b + c][32 * j + 4 * g]),
                      *reinterpret_cast<const f32x4*>(&A[16 * b + c][32 * j + 16 + 4 * g]));
#pragma unroll
      for (int i = 0; i < NM; ++i)
        a.T[((at * NM + i) * kDeltaLower + u) * 64 + slot] = __builtin_bit_cast(float4, f.p[i]);
    }
    __syncthreads();  // A and the gates have been read
  }
}

// ---------------------------------------------------------------------------
// The state along the chunks of a segment: 16 columns a wave, all a workgroup.

// waves a SIMD of the scans: the registers are held to what so many leave
template <typename T, int DK>
constexpr int scan_waves() {
  return DK == 128 ? 1 : 2;
}

// what a chunk's step needs in LDS, the last two for outputs and backward
template <typename T, int DK>
struct ScanTiles {
  static constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid;
  Image<NI, DK / 8> k;
  Image<NM, kDeltaLower> t;
  float fac[4][kDeltaRows];  // the first four
  Image<NI, DK / 8> q;
  Image<NM, kDeltaLower> p;
  static constexpr size_t bytes(bool out) {
    return out ? sizeof(ScanTiles)
               : (NI * (DK / 8) + NM * kDeltaLower) * 1024 + 4 * kDeltaRows * sizeof(float);
  }
  template <int WAVES, bool OUT>
  __device__ __forceinline__ void send(const DeltaArgs& a, int tile, int h) {
    const int64_t at = (int64_t)tile * a.heads + h;
    const int64_t kat = ((int64_t)tile * a.keys + h / a.group) * (k.units * 64);
    send_to_lds<Image<NI, DK / 8>::units, WAVES>(k.x, a.K + kat);
    send_to_lds<Image<NM, kDeltaLower>::units, WAVES>(t.x, a.T + at * (t.units * 64));
    send_to_lds<1, WAVES>(reinterpret_cast<float4*>(fac),
                          reinterpret_cast<const float4*>(
                              a.fac + at * (kDeltaFactors * kDeltaRows)));
    if (OUT) {
      send_to_lds<Image<NI, DK / 8>::units, WAVES>(q.x, a.Q + kat);
      send_to_lds<Image<NM, kDeltaLower>::units, WAVES>(p.x, a.P + at * (p.units * 64));
    }
  }
};

// The parts of G_C of a chunk, on their way.
struct ChunkEnd {
  float hi, lo;
  __device__ __forceinline__ void load(const DeltaArgs& a, int tile, int h) {
    const float* const f =
        a.fac + ((int64_t)tile * a.heads + h) * (kDeltaFactors * kDeltaRows) + kDeltaRows - 1;
    hi = f[kFacHi * kDeltaRows];
    lo = f[kFacLo * kDeltaRows];
  }
};

// 16 x 4 rows of a lane's column of v or do on their way: rows 16 b + 4 g + i
template <typename T>
struct Columns {
  T x[16];
  // src: the first column; col: the lane's, one that is there
  __device__ __forceinline__ void load(const Chunk& ch, const T* src, int stride, int col) {
    const int g = mlcg_lane() >> 4;
    if (ch.n == kDeltaRows) {
      const Lines l(const_cast<T*>(src), ch.base, ch.step, stride * (int)sizeof(T), 4 * g, 12,
                    col * (int)sizeof(T));
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = l.row<const T>(16 * (r / 4) + r % 4);
    } else {
      const T* const p = src + ch.base * stride + col;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = p[ch.offset(16 * (r / 4) + 4 * g + r % 4, stride)];
    }
  }
  // the four rows of block b
  __device__ __forceinline__ f32x4 rows(int b) const {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)x[4 * b + i];
    return v;
  }
};

// A wave's right operands as they are to block row w of an image of `rows` of them:
// read as rows they are the transpose of what the wave has.
template <int N, int KS>
__device__ __forceinline__ void store_operand(float4* images, int64_t at, int rows, int w,
                                              const Frag<N> (&s)[KS]) {
  float4* const p = images + at * ((int64_t)N * rows * KS * 64) + Image<N, KS>::slot();
#pragma unroll
  for (int i = 0; i < KS; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j)
      p[((j * rows + w) * KS + i) * 64] = __builtin_bit_cast(float4, s[i].p[j]);
}
// The transpose of a chunk's rows, 4 of the wave's 16 columns of row 16 b + c in a
// lane, to an image of 64 rows and 32 kv columns: half of the blocks' elements.
template <int N>
__device__ __forceinline__ void store_half(float4* images, int64_t at, int kv, int w,
                                           f32x4 (&y)[4]) {
  bf16x4* const p = reinterpret_cast<bf16x4*>(images + at * ((int64_t)N * 4 * kv * 64) +
                                              Image<N, 4>::slot()) + (w & 1);
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const bf16x4 z = __builtin_convertvector(y[b], bf16x4);
      p[((j * 4 + b) * kv + w / 2) * 128] = z;
      if (j + 1 < N) y[b] -= __builtin_convertvector(z, f32x4);
    }
}

// a state's 16 columns from `at` on: rows 16 b + 4 g + i, column c of them
template <int B>
__device__ __forceinline__ void load_state(f32x4 (&s)[B], const float* at, int ld, int rows,
                                           bool in) {
  const int g = mlcg_lane() >> 4, c = mlcg_lane() & 15;
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * b + 4 * g + i;
      s[b][i] = in && r < rows ? at[r * ld + c] : 0.0f;
    }
}
template <int B>
__device__ __forceinline__ void store_state(const f32x4 (&s)[B], float* at, int ld, int rows,
                                            bool in) {
  const int g = mlcg_lane() >> 4, c = mlcg_lane() & 15;
  if (!in) return;
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (16 * b + 4 * g + i < rows) at[(16 * b + 4 * g + i) * ld + c] = s[b][i];
}
// ... all rows of a padded one
template <int B>
__device__ __forceinline__ void store_padded(const f32x4 (&s)[B], float* at, int ld) {
  const Lines l(at, 0, 1, 4 * ld, 4 * (mlcg_lane() >> 4), 12, 4 * (mlcg_lane() & 15));
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i) l.row<float>(16 * b + i) = s[b][i];
}

// The products of a chunk with a wave's columns: the left operands of several
// matrix instructions are sent for before the first of them.  y[b]: rows 16 b ..
// of the image times s, or, FLIP, the transpose of that.
template <bool FLIP, int N, int NB, int M, int KS>
__device__ __forceinline__ void rows_product(f32x4 (&y)[4], const Image<N, NB>& t,
                                             const Frag<M> (&s)[KS]) {
  constexpr int G = KS * N <= 4 ? 4 : KS * N <= 8 ? 2 : 1;
#pragma unroll
  for (int b = 0; b < 4; b += G) {
    Frag<N> f[G][KS];
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int i = 0; i < KS; ++i) f[j][i] = t.rows((b + j) * KS + i);
#pragma unroll
    for (int j = 0; j < G; ++j) y[b + j] = f32x4{};
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int j = 0; j < G; ++j) {
        if (FLIP)
          mma(y[b + j], s[i], f[j][i]);
        else
          mma(y[b + j], f[j][i], s[i]);
      }
  }
}
// s += (columns of the image) x, the image of 32 R rows
template <int B, int N, int NB, int M, int R>
__device__ __forceinline__ void columns_product(f32x4 (&s)[B], const Image<N, NB>& t,
                                                const Frag<M> (&x)[R]) {
  constexpr int KS = B / 2;
#pragma unroll
  for (int b = 0; b < B; b += 2) {
    Frag<N> f[R][2];
    const int b0 = b / 2;
    if constexpr (R == 1) {
      t.columns(b0, KS + b0, f[0]);
    } else {
#pragma unroll
      for (int i = 0; i < R; i += 2)
        t.columns(2 * i * KS + b0, (2 * i + 1) * KS + b0, (2 * i + 2) * KS + b0,
                  (2 * i + 3) * KS + b0, f[i], f[i + 1]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) mma(s[b + j], f[i][j], x[i]);
  }
}
// The blocks (b, i) of a lower triangle are 0 0, 1 0, 2 0, 2 1, 3 0, 3 1.
__device__ __forceinline__ constexpr int lower(int b, int i) { return b + (b == 3) + i; }
// y += (lower triangle) x, or, FLIP, the transpose of that
template <bool FLIP, int N, int M>
__device__ __forceinline__ void lower_product(f32x4 (&y)[4], const Image<N, kDeltaLower>& t,
                                              const Frag<M> (&x)[2]) {
  Frag<N> f[kDeltaLower];
#pragma unroll
  for (int u = 0; u < kDeltaLower; ++u) f[u] = t.rows(u);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int b = 2 * i; b < 4; ++b) {
      if (FLIP)
        mma(y[b], x[i], f[lower(b, i)]);
      else
        mma(y[b], f[lower(b, i)], x[i]);
    }
}
// y += (lower triangle)^T x, or, FLIP, the transpose of that
template <bool FLIP, int N, int M>
__device__ __forceinline__ void upper_product(f32x4 (&y)[4], const Image<N, kDeltaLower>& t,
                                              const Frag<M> (&x)[2]) {
  Frag<N> f[2][2], g[2];  // rows 0 .. 31's columns 0 .. 31; rows 32 .. 63's 0 .. 31, 32 .. 63
  t.columns(lower(0, 0), lower(1, 0), lower(2, 0), lower(3, 0), f[0], f[1]);
  t.columns(lower(2, 1), lower(3, 1), g);
  const auto product = [&](int b, const Frag<N>& l, const Frag<M>& r) {
    if (FLIP)
      mma(y[b], r, l);
    else
      mma(y[b], l, r);
  };
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    product(b, f[0][b], x[0]);
    product(b, f[1][b], x[1]);
    product(b + 2, g[b], x[1]);
  }
}
// the 16 B rows of a wave's columns as right operands
template <int N, int B>
__device__ __forceinline__ void split_rows(Frag<N> (&x)[B / 2], const f32x4 (&y)[B]) {
#pragma unroll
  for (int i = 0; i < B / 2; ++i) x[i] = split44<N>(y[2 * i], y[2 * i + 1]);
}
// a factor of the rows 16 b + 4 g ..
__device__ __forceinline__ f32x4 row_factor(const float* f, int b) {
  return *reinterpret_cast<const f32x4*>(f + 16 * b + 4 * (mlcg_lane() >> 4));
}

// Alone: what a segment makes of the state zero (columns of v) and, in the second
// workgroup, of every unit vector; no outputs.  Of two buffers the next chunk is
// sent to one while the other is worked on; with one the next workgroup on the
// compute unit works meanwhile.  512 x 100 beads, 4 heads of 32 in bf16: 49 us, 4.4
// TB/s, near a copy's rate; 1 x 120001, 8 heads of 64, segments of 64 chunks: 321 us, 3.3
// TB/s, and alone 261 us, 2.2 TB/s with the matrix instructions busy 31 % of the time.
template <typename T, int DK, int WAVES, bool ALONE>
__global__ __launch_bounds__(64 * WAVES, (scan_waves<T, DK>())) void delta_scan(
    DeltaArgs a, DeltaEnds e, T* out, int buffers) {
  constexpr int NM = Pieces<T>::mid, KS = DK / 32, B = DK / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  typedef ScanTiles<T, DK> Tiles;
  const int4 seg = uniform(a.segs[blockIdx.x]);
  const int h = blockIdx.y, w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const bool unit = ALONE && blockIdx.z == 1;
  const int v0 = 16 * w, col = min(v0 + c, a.dv - 1);
  const bool live = v0 < (unit ? DK : a.dvp);  // wave-uniform
  const T* const v = (const T*)a.v + h * a.v_head;
  f32x4 S[B];
  if (ALONE) {
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) S[b][i] = unit && 16 * b + 4 * g + i == v0 + c ? 1.0f : 0.0f;
  } else if (e.seg_init) {
    load_state<B>(S, e.seg_init + ((int64_t)blockIdx.x * a.heads + h) * (DK * a.dvp) + v0, a.dvp,
                  DK, live);
  } else {
    load_state<B>(S, e.init + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                  a.dk, e.init && v0 + c < a.dv);
  }
  const Walk walk(a, seg.y);
  Columns<T> vn;
  const auto tiles = [&](int n) {
    return reinterpret_cast<Tiles*>(smem + (n % buffers) * Tiles::bytes(!ALONE));
  };
  ChunkEnd end;
  end.load(a, seg.y, h);
  if (buffers == 2) tiles(0)->template send<WAVES, !ALONE>(a, seg.y, h);
  if (!unit) vn.load(walk.chunk(a, 0), v, (int)a.v_row, col);
  for (int n = 0; n < seg.z; ++n) {
    const int tile = seg.y + n;
    Tiles& sh = *tiles(n);
    if (buffers == 1) {
      if (n > 0) lds_barrier();
      sh.template send<WAVES, !ALONE>(a, tile, h);
    }
    wait_for_memory();
    lds_barrier();
    f32x4 X[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) X[b] = unit ? f32x4{} : vn.rows(b);
    const float decay = exp2_of(end.hi, end.lo);
    if (n + 1 < seg.z) {
      end.load(a, tile + 1, h);
      if (buffers == 2) tiles(n + 1)->template send<WAVES, !ALONE>(a, tile + 1, h);
      if (!unit) vn.load(walk.chunk(a, kDeltaRows * (n + 1)), v, (int)a.v_row, col);
    }
    if (!live) continue;
    const int64_t at = (int64_t)tile * a.heads + h;
    Frag<NM> s[KS], x[2];
    split_rows<NM>(s, S);
    if (!ALONE && a.S0) store_operand<NM, KS>(a.S0, at, a.dvp / 16, w, s);
    f32x4 Y[4];
    rows_product<false>(Y, sh.k, s);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const f32x4 read = row_factor(sh.fac[kFacRead], b), beta = row_factor(sh.fac[kFacBeta], b);
      X[b] = beta * (X[b] - read * Y[b]);
      if (a.keep)  // v of an absent bead may be no number
#pragma unroll
        for (int i = 0; i < 4; ++i) X[b][i] = beta[i] == 0.0f ? 0.0f : X[b][i];
    }
    if (a.dv != a.dvp && !unit && v0 + c >= a.dv)  // columns that are none stay zeros
#pragma unroll
      for (int b = 0; b < 4; ++b) X[b] = f32x4{};
    Frag<NM> xu[2];
    split_rows<NM>(xu, X);
#pragma unroll
    for (int b = 0; b < 4; ++b) X[b] = f32x4{};
    lower_product<false>(X, sh.t, xu);
    if (!ALONE) {
      split_rows<NM>(x, X);
      // o^T: four columns of one bead in a lane
      f32x4 O[4];
      rows_product<true>(O, sh.q, s);
#pragma unroll
      for (int b = 0; b < 4; ++b) O[b] *= sh.fac[kFacOut][16 * b + c];
      lower_product<true>(O, sh.p, x);
      const Chunk ch = walk.chunk(a, kDeltaRows * n);
      typedef typename loose<T, 4>::type vec;
      const int el = v0 + 4 * g;
      if (el < a.dv) {
        if (ch.n == kDeltaRows) {
          const Lines l(out, ch.base, ch.step, a.heads * a.dv * (int)sizeof(T), c, 15,
                        (h * a.dv + el) * (int)sizeof(T));
#pragma unroll
          for (int b = 0; b < 4; ++b) l.row<vec>(16 * b) = __builtin_convertvector(O[b], vec);
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (16 * b + c < ch.n)
              store4<T>(out + (ch.bead(16 * b + c) * a.heads + h) * a.dv, el, a.dv, O[b]);
        }
      }
      if (a.U) {
#pragma unroll
        for (int b = 0; b < 4; ++b) O[b] = f32x4{};
        lower_product<true>(O, sh.t, xu);
        store_half<NM>(a.U, at, a.dvp / 32, w, O);
      }
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) X[b] *= row_factor(sh.fac[kFacWrite], b);
    split_rows<NM>(x, X);
#pragma unroll
    for (int b = 0; b < B; ++b) S[b] *= decay;
    columns_product(S, sh.k, x);
  }
  if (!live) return;
  const int64_t at = (int64_t)blockIdx.x * a.heads + h;
  if (unit) {  // the map's transpose, as a left operand
    Frag<NM> s[KS];
    split_rows<NM>(s, S);
    typedef Image<NM, B * KS> Map;
    float4* const m = e.seg_map + at * (Map::units * 64);
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int j = 0; j < NM; ++j)
        m[(j * (B * KS) + w * KS + i) * 64 + Map::slot()] = __builtin_bit_cast(float4, s[i].p[j]);
  } else if (ALONE) {
    store_padded<B>(S, e.seg_last + at * (DK * a.dvp) + v0, a.dvp);
  } else if (e.last && (seg.w & 2)) {
    store_state<B>(S, e.last + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                   a.dk, v0 + c < a.dv);
  }
}

// The states before the segments of a chain, one after the other: S <- M S + N.
// Backward: after them, the last one first, S <- M^T S + N.  Bound by the latency of
// memory: while a segment's map is worked on, the next one's map and N are on their
// way, the map to the other of two buffers (with one, the maps of 128 channels, they
// are sent for when all are done with the last).  Before the barrier every wave waits
// for all that it sent, so that a map is whole and N there behind it.  8 heads of 64 in
// bf16: 18 us for the 11 segments of 2 x 4099 beads, 58 us for the 30 of 1 x 120001.
template <typename T, int DK, int WAVES, bool BACK>
__global__ __launch_bounds__(64 * WAVES) void delta_join(DeltaArgs a, DeltaEnds e,
                                                         float* seg_init, int buffers) {
  constexpr int NM = Pieces<T>::mid, KS = DK / 32, B = DK / 16;
  typedef Image<NM, B * KS> Map;
  extern __shared__ __align__(16) unsigned char smem[];
  Map* const maps = reinterpret_cast<Map*>(smem);
  const int h = blockIdx.y, c = mlcg_lane() & 15, v0 = 16 * wave_number();
  const bool live = v0 < a.dvp;
  const int first = uniform(a.seg_first[blockIdx.x]);
  const int n = uniform(a.seg_first[blockIdx.x + 1]) - first;
  const int chain = uniform(a.segs[first]).x;
  f32x4 S[B], next[B];
  load_state<B>(S, e.init + ((int64_t)chain * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                a.dk, e.init && v0 + c < a.dv);
  const auto seg_at = [&](int j) {
    return (int64_t)(first + (BACK ? n - 1 - j : j)) * a.heads + h;
  };
  const auto fetch = [&](int j) {
    if (j + 1 >= n) return;  // nothing comes behind the last segment
    const int64_t at = seg_at(j);
    send_to_lds<Map::units, WAVES>(maps[j % buffers].x, e.seg_map + at * (Map::units * 64));
    load_state<B>(next, e.seg_last + at * (DK * a.dvp) + (live ? v0 : 0), a.dvp, DK, true);
  };
#pragma unroll
  for (int b = 0; b < B; ++b) next[b] = f32x4{};
  fetch(0);
  for (int j = 0; j < n; ++j) {
    wait_for_memory();
    lds_barrier();
    Frag<NM> s[KS];
    split_rows<NM>(s, S);
    if (live) store_padded<B>(S, seg_init + seg_at(j) * (DK * a.dvp) + v0, a.dvp);
    if (j + 1 >= n) return;
#pragma unroll
    for (int b = 0; b < B; ++b) S[b] = next[b];
    // all have read the map of j - 1, which was in the place of that of j + 1
    if (buffers == 2) fetch(j + 1);
    const Map& m = maps[j % buffers];
    if (BACK) {
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int i = 0; i < KS; ++i) mma(S[b], m.rows(b * KS + i), s[i]);
    } else {
      columns_product(S, m, s);
    }
    if (buffers == 1) {
      lds_barrier();
      fetch(j + 1);
    }
  }
}

// The state's gradient along the chunks of a segment, the last one first.  512 x 100
// beads, 4 heads of 32 in bf16: 46 us, 4.5 TB/s, near a copy's rate; 2 x 4099, 8 heads of
// 64 on 4: 37 us, 3.5 TB/s, and alone 24 us, 2.8 TB/s.
template <typename T, int DK, int WAVES, bool ALONE>
__global__ __launch_bounds__(64 * WAVES, (scan_waves<T, DK>())) void delta_scan_back(
    DeltaArgs a, DeltaBack o, DeltaEnds e, int buffers) {
  constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid, KS = DK / 32, B = DK / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  typedef ScanTiles<T, DK> Tiles;
  const int4 seg = uniform(a.segs[blockIdx.x]);
  const int h = blockIdx.y, w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const int v0 = 16 * w, col = min(v0 + c, a.dv - 1);
  const bool live = v0 < a.dvp;
  const T* const grad = (const T*)o.grad + h * a.dv;
  const int row = a.heads * a.dv;  // of do and dv
  f32x4 D[B];
  if (ALONE) {
#pragma unroll
    for (int b = 0; b < B; ++b) D[b] = f32x4{};
  } else if (e.seg_init) {
    load_state<B>(D, e.seg_init + ((int64_t)blockIdx.x * a.heads + h) * (DK * a.dvp) + v0, a.dvp,
                  DK, live);
  } else {
    load_state<B>(D, e.init + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0, a.dv,
                  a.dk, e.init && v0 + c < a.dv);
  }
  const Walk walk(a, seg.y);
  Columns<T> gn;
  const auto tiles = [&](int n) {
    return reinterpret_cast<Tiles*>(smem + (n % buffers) * Tiles::bytes(true));
  };
  const int top = seg.z - 1;
  ChunkEnd end;
  end.load(a, seg.y + top, h);
  if (buffers == 2) tiles(top)->template send<WAVES, true>(a, seg.y + top, h);
  gn.load(walk.chunk(a, kDeltaRows * top), grad, row, col);
  for (int n = top; n >= 0; --n) {
    const int tile = seg.y + n;
    Tiles& sh = *tiles(n);
    if (buffers == 1) {
      if (n < top) lds_barrier();
      sh.template send<WAVES, true>(a, tile, h);
    }
    wait_for_memory();
    lds_barrier();
    const Chunk ch = walk.chunk(a, kDeltaRows * n);
    f32x4 G[4], X[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) G[b] = gn.rows(b);
    if (ch.n < kDeltaRows)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (16 * (r / 4) + 4 * g + r % 4 >= ch.n) G[r / 4][r % 4] = 0.0f;
    if (a.dv != a.dvp && v0 + c >= a.dv)
#pragma unroll
      for (int b = 0; b < 4; ++b) G[b] = f32x4{};
    const float decay = exp2_of(end.hi, end.lo);
    if (n > 0) {
      end.load(a, tile - 1, h);
      if (buffers == 2) tiles(n - 1)->template send<WAVES, true>(a, tile - 1, h);
      gn.load(walk.chunk(a, kDeltaRows * (n - 1)), grad, row, col);
    }
    if (!live) continue;
    const int64_t at = (int64_t)tile * a.heads + h;
    Frag<NM> x[2];
    {
      Frag<NM> d[KS];
      split_rows<NM>(d, D);
      if (!ALONE) store_operand<NM, KS>(o.D, at, a.dvp / 16, w, d);
      rows_product<false>(X, sh.k, d);
    }
    // du
#pragma unroll
    for (int b = 0; b < 4; ++b) X[b] *= row_factor(sh.fac[kFacWrite], b);
    {
      Frag<NI> go[2];
      split_rows<NI>(go, G);
      upper_product<false>(X, sh.p, go);
    }
    split_rows<NM>(x, X);
    // dr
#pragma unroll
    for (int b = 0; b < 4; ++b) X[b] = f32x4{};
    upper_product<false>(X, sh.t, x);
    if (!ALONE) {
      // its transpose: four columns of one bead in a lane
      f32x4 R[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) R[b] = f32x4{};
      upper_product<true>(R, sh.t, x);
      const int el = v0 + 4 * g;
      if (el < a.dv) {
        typedef typename loose<T, 4>::type vec;
        if (ch.n == kDeltaRows) {
          const Lines l(o.dv, ch.base, ch.step, row * (int)sizeof(T), c, 15,
                        (h * a.dv + el) * (int)sizeof(T));
#pragma unroll
          for (int b = 0; b < 4; ++b)
            l.row<vec>(16 * b) = __builtin_convertvector(R[b] * sh.fac[kFacBeta][16 * b + c], vec);
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (16 * b + c < ch.n)
              store4<T>((T*)o.dv + ch.bead(16 * b + c) * row + h * a.dv, el, a.dv,
                        R[b] * sh.fac[kFacBeta][16 * b + c]);
        }
      }
      store_half<NM>(o.dR, at, a.dvp / 32, w, R);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      X[b] *= row_factor(sh.fac[kFacBeta], b) * -row_factor(sh.fac[kFacRead], b);
      G[b] *= row_factor(sh.fac[kFacOut], b);
    }
#pragma unroll
    for (int b = 0; b < B; ++b) D[b] *= decay;
    split_rows<NM>(x, X);
    columns_product(D, sh.k, x);
    split_rows<NM>(x, G);
    columns_product(D, sh.q, x);
  }
  if (!live) return;
  if (ALONE)
    store_padded<B>(D, e.seg_last + ((int64_t)blockIdx.x * a.heads + h) * (DK * a.dvp) + v0,
                    a.dvp);
  else if (o.dstate && (seg.w & 1))
    store_state<B>(D, o.dstate + ((int64_t)seg.x * a.heads + h) * ((int64_t)a.dk * a.dv) + v0,
                   a.dv, a.dk, v0 + c < a.dv);
}

// ---------------------------------------------------------------------------
// The gradients of q, k, beta and g of a chunk's beads, for the heads of one
// key head; a wave has 16 beads, as columns.  Bound by neither memory nor products but by
// how few waves its registers leave: 512 x 100 beads, 4 heads of 32 in bf16, 71 us, 2.6
// TB/s, matrix instructions 11 % of the time; 2 x 4099, 8 heads of 64 on 4, 70 us, 3.5
// TB/s, with 40 registers spilled.

// What a chunk's gradients need in LDS, one after the other in one or two places:
// u, dr (and do, in the other); k and q; S0; D.
template <typename T, int DK, int KV>
struct GradTiles {
  static constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid;
  typedef Image<NM, 4 * KV> Rows;              // 64 beads x dv
  typedef Image<NI, 4 * KV> Given;             // the same of do
  typedef Image<NM, 2 * KV*(DK / 32)> State;   // dv x DK
  typedef Image<NI, DK / 8> Keys;              // 64 beads x DK
  static constexpr size_t rows = 2 * sizeof(Rows), keys = 2 * sizeof(Keys);
  static constexpr size_t even = rows > sizeof(State) ? rows : sizeof(State);
  // k and q come to their place while do behind them is still read
  static constexpr size_t behind = keys + sizeof(Given);
  static constexpr size_t odd = behind > sizeof(State) ? behind : sizeof(State);
  // in one place do lies behind u and dr
  static constexpr size_t one = rows + sizeof(Given) > keys ? rows + sizeof(Given) : keys;
  static constexpr size_t bytes(int places) {
    return places == 2 ? even + odd : one > sizeof(State) ? one : sizeof(State);
  }
  struct Small {
    float fac[kDeltaFactors][kDeltaRows];
    float dG[kDeltaRows];
    float ends[4];
  };
};

// waves a SIMD: two where the registers of half of it are enough
template <typename T, int DK, int KV>
constexpr int grad_waves() {
  return sizeof(T) == 2 ? (DK <= 64 && KV <= 2 ? 2 : 1) : (DK == 32 && KV == 1 ? 2 : 1);
}

// MANY: several heads to a key head, whose gradients are summed
template <typename T, int DK, int KV, bool MANY>
__global__ __launch_bounds__(kDeltaThreads, (grad_waves<T, DK, KV>())) void delta_grad(
    DeltaArgs a, DeltaBack o, int places) {
  typedef GradTiles<T, DK, KV> Tiles;
  typedef typename Tiles::Rows Rows;
  typedef typename Tiles::Given Given;
  typedef typename Tiles::State State;
  typedef typename Tiles::Keys Keys;
  constexpr int NI = Pieces<T>::in, NM = Pieces<T>::mid, B = DK / 16, KS = DK / 32;
  extern __shared__ __align__(16) unsigned char smem[];
  typename Tiles::Small& sh =
      *reinterpret_cast<typename Tiles::Small*>(smem + Tiles::bytes(places));
  unsigned char* const even = smem;
  unsigned char* const odd = smem + (places - 1) * Tiles::even;
  const int tile = blockIdx.x, kh = blockIdx.y;
  const int w = wave_number(), lane = mlcg_lane(), c = lane & 15, g = lane >> 4;
  const Chunk ch(a, tile);
  const int row = 16 * w + c;
  const bool in = row < ch.n;
  const int64_t bead = ch.bead(min(row, ch.n - 1));
  const bool there = in && (!a.keep || a.keep[bead]);
  f32x4 dq[B], dk[B];
#pragma unroll
  for (int b = 0; b < B; ++b) dq[b] = dk[b] = f32x4{};
  float rq = 0.0f, rk = 0.0f;

  const auto send_state = [&](unsigned char* to, const float4* from, int64_t at) {
    send_to_lds<State::units, 4>(reinterpret_cast<float4*>(to), from + at * (State::units * 64));
  };
  const int64_t kat = ((int64_t)tile * a.keys + kh) * (Keys::units * 64);
  const auto send_keys = [&](unsigned char* to) {
    send_to_lds<Keys::units, 4>(reinterpret_cast<float4*>(to), a.K + kat);
    send_to_lds<Keys::units, 4>(reinterpret_cast<float4*>(to + sizeof(Keys)), a.Q + kat);
  };
  // elements 32 i + 4 g .. and 32 i + 16 + 4 g .. of this wave's rows of k or q
  const auto own_row = [&](const float4* from, int i) {
    Frag<NI> f;
#pragma unroll
    for (int j = 0; j < NI; ++j)
      f.p[j] = __builtin_bit_cast(
          bf16x8, from[kat + (j * (DK / 8) + w * KS + i) * 64 + Keys::slot()]);
    return whole(f);
  };
  // with one place, what comes next is sent for when all are done with the last
  const auto wait_for = [&](auto send) {
    if (places == 1) {
      lds_barrier();
      send();
    }
    wait_for_memory();
    lds_barrier();
  };
  for (int h = kh * a.group; h < (kh + 1) * a.group; ++h) {
    const int64_t at = (int64_t)tile * a.heads + h;
    if (h > kh * a.group) lds_barrier();  // what the last head left has been read
    Rows& U = *reinterpret_cast<Rows*>(even);
    Rows& R = *reinterpret_cast<Rows*>(even + sizeof(Rows));
    Given& G = *reinterpret_cast<Given*>(places == 2 ? odd + Tiles::keys : even + Tiles::rows);
    send_to_lds<Rows::units, 4>(U.x, a.U + at * (Rows::units * 64));
    send_to_lds<Rows::units, 4>(R.x, o.dR + at * (Rows::units * 64));
    send_to_lds<2, 4>(reinterpret_cast<float4*>(sh.fac),
                      reinterpret_cast<const float4*>(a.fac +
                                                      at * (kDeltaFactors * kDeltaRows)));
    // this wave's beads, as columns: do, and v for dr.v
    Frag<NI> gb[KV];
    f32x8 vr[KV];
    {
      const T* const go = (const T*)o.grad + (bead * a.heads + h) * a.dv;
      const T* const v = (const T*)a.v + bead * a.v_row + h * a.v_head;
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        v4<T> x[2], y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          x[j] = load4<T>(go, 32 * i + 16 * j + 4 * g, a.dv);
          y[j] = load4<T>(v, 32 * i + 16 * j + 4 * g, a.dv);
        }
        v8<T> u = __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7);
        v8<T> z = __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7);
        if (!in) u = v8<T>{};
        if (!there) z = v8<T>{};
        gb[i] = split_raw<NI, T>(u);
        vr[i] = __builtin_convertvector(z, f32x8);
#pragma unroll
        for (int j = 0; j < NI; ++j)
          G.x[(j * (4 * KV) + w * KV + i) * 64 + G.slot()] =
              __builtin_bit_cast(float4, gb[i].p[j]);
      }
    }
    wait_for_memory();
    lds_barrier();
    if (places == 2) send_keys(odd);

    // Products by beads with this wave's, s its row's or column's: of blocks before
    // do_t.u_s and dr_t.u_s, [s][this wave's t]; of blocks behind the same, [t][this
    // wave's s]; of its own both, the second apart.
    Frag<NM> ub[KV], rb[KV];
    f32x4 ou[4], ru[4], od{}, rd{};
    float rv = 0.0f;  // dr.v
#pragma unroll
    for (int i = 0; i < KV; ++i) {
      ub[i] = U.rows(w * KV + i);
      rb[i] = R.rows(w * KV + i);
      const f32x8 r = whole(rb[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) rv = fmaf(r[j], vr[i][j], rv);
    }
    // factors of this wave's beads
    const float th = sh.fac[kFacHi][row], tl = sh.fac[kFacLo][row];
    const float ch_hi = sh.fac[kFacHi][63], ch_lo = sh.fac[kFacLo][63];
    const float first = exp2_of(th, tl), rest = exp2_of(ch_hi - th, ch_lo - tl);
    const float beta = sh.fac[kFacBeta][row];
    rk = sh.fac[kFacK][row];
    rq = sh.fac[kFacQ][row];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const f32x4 hi = row_factor(sh.fac[kFacHi], m), lo = row_factor(sh.fac[kFacLo], m);
      const f32x4 xk = row_factor(sh.fac[kFacK], m);
      ou[m] = ru[m] = f32x4{};
      if (m <= w) {
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          const Frag<NM> f = U.rows(m * KV + i);
          mma(ou[m], f, gb[i]);
          mma(ru[m], f, rb[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * m + 4 * g + i;
          const float e = r <= row ? exp2_of(th - hi[i], tl - lo[i]) * xk[i] : 0.0f;
          ou[m][i] = r <= row ? e * ou[m][i] : 0.0f;
          ru[m][i] = r < row ? -e * ru[m][i] : 0.0f;
        }
      }
      if (m >= w) {
        const f32x4 xb = row_factor(sh.fac[kFacBeta], m), xq = row_factor(sh.fac[kFacQ], m);
        f32x4 x{}, y{};
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          mma(x, G.rows(m * KV + i), ub[i]);
          mma(y, R.rows(m * KV + i), ub[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * m + 4 * g + i;
          const float e = r >= row ? exp2_of(hi[i] - th, lo[i] - tl) : 0.0f;
          x[i] = r >= row ? e * xq[i] * a.scale * x[i] : 0.0f;
          y[i] = r > row ? -e * xk[i] * xb[i] * y[i] : 0.0f;
        }
        if (m == w) {
          od = x;
          rd = y;
        } else {
          ou[m] = x;
          ru[m] = y;
        }
      }
    }
    // inside the chunk
    f32x4 hq[B], hr[B], hw[B];
#pragma unroll
    for (int b = 0; b < B; ++b) hq[b] = hr[b] = hw[b] = f32x4{};
    wait_for([&] { send_keys(odd); });
    if (places == 2) send_state(even, a.S0, at);
    {
      const Keys& K = *reinterpret_cast<const Keys*>(odd);
      const Keys& Q = *reinterpret_cast<const Keys*>(odd + sizeof(Keys));
      const f32x4 none{};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i <= w / 2) {  // beads up to this wave's
          const Frag<NM> of = split44<NM>(ou[2 * i], 2 * i + 1 <= w ? ou[2 * i + 1] : none);
          const Frag<NM> rf = split44<NM>(ru[2 * i], 2 * i + 1 <= w ? ru[2 * i + 1] : none);
#pragma unroll
          for (int b = 0; b < B; b += 2) {
            const int b0 = 2 * i * KS + b / 2, b1 = b0 + KS;
            Frag<NI> k[2];
            K.columns_now(b0, b1, k);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma(hq[b + j], k[j], of);
              mma(hr[b + j], k[j], rf);
            }
          }
        }
        if (i >= w / 2) {
          const f32x4 o0 = 2 * i == w ? od : 2 * i > w ? ou[2 * i] : none;
          const f32x4 r0 = 2 * i == w ? rd : 2 * i > w ? ru[2 * i] : none;
          const Frag<NM> of = split44<NM>(o0, 2 * i + 1 == w ? od : ou[2 * i + 1]);
          const Frag<NM> rf = split44<NM>(r0, 2 * i + 1 == w ? rd : ru[2 * i + 1]);
#pragma unroll
          for (int b = 0; b < B; b += 2) {
            const int b0 = 2 * i * KS + b / 2, b1 = b0 + KS;
            Frag<NI> k[2], q[2];
            K.columns_now(b0, b1, k);
            Q.columns_now(b0, b1, q);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              mma(hw[b + j], q[j], of);
              mma(hw[b + j], k[j], rf);
            }
          }
        }
      }
    }
    // S0 do and S0 dr
    wait_for([&] { send_state(even, a.S0, at); });
    if (places == 2) send_state(odd, o.D, at);
    {
      const State& S = *reinterpret_cast<const State*>(even);
#pragma unroll
      for (int b = 0; b < B; b += 2) {
        f32x4 q0{}, q1{}, r0{}, r1{};
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          const int b0 = 2 * i * KS + b / 2;
          Frag<NM> s[2];
          S.columns_now(b0, b0 + KS, s);
          mma(q0, s[0], gb[i]);
          mma(r0, s[0], rb[i]);
          mma(q1, s[1], gb[i]);
          mma(r1, s[1], rb[i]);
        }
        hq[b] += first * q0;
        hq[b + 1] += first * q1;
        hr[b] -= first * r0;
        hr[b + 1] -= first * r1;
      }
    }
    // D u, and this wave's part of <S0, D>
    wait_for([&] { send_state(odd, o.D, at); });
    float sd = 0.0f, kd = 0.0f;  // kd: k.(e^(G_C - G) D u)
    {
      const State& D = *reinterpret_cast<const State*>(odd);
      const float4* const s0 = a.S0 + at * (State::units * 64) + State::slot();
#pragma unroll
      for (int u = 0; u < (2 * KV * KS + 3) / 4; ++u) {
        const int block = 4 * u + w;
        if (block >= 2 * KV * KS) continue;
        Frag<NM> f;
#pragma unroll
        for (int j = 0; j < NM; ++j)
          f.p[j] = __builtin_bit_cast(bf16x8, s0[(j * (2 * KV * KS) + block) * 64]);
        const f32x8 x = whole(f), y = whole(D.rows(block));
#pragma unroll
        for (int j = 0; j < 8; ++j) sd = fmaf(x[j], y[j], sd);
      }
#pragma unroll
      for (int b = 0; b < B; b += 2) {
        const f32x8 x = own_row(a.K, b / 2) * (rk * rest);
        f32x4 w0{}, w1{};
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          const int b0 = 2 * i * KS + b / 2;
          Frag<NM> d[2];
          D.columns_now(b0, b0 + KS, d);
          mma(w0, d[0], ub[i]);
          mma(w1, d[1], ub[i]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kd = fmaf(x[j], w0[j], kd);
          kd = fmaf(x[4 + j], w1[j], kd);
        }
        hw[b] += rest * w0;
        hw[b + 1] += rest * w1;
      }
    }
    float qd = 0.0f, kr = 0.0f, kw = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const f32x8 x = own_row(a.K, i) * rk, y = own_row(a.Q, i) * rq;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int b = 2 * i + j / 4;
        qd = fmaf(y[j], hq[b][j % 4], qd);
        kr = fmaf(x[j], hr[b][j % 4], kr);
        kw = fmaf(x[j], hw[b][j % 4], kw);
      }
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (MANY) {
        dq[b] += hq[b];
        dk[b] += beta * hr[b] + hw[b];
      } else {
        dq[b] = hq[b];
        dk[b] = beta * hr[b] + hw[b];
      }
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
    lds_barrier();
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
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const f32x8 x = own_row(a.K, i) * rk, y = own_row(a.Q, i) * rq;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      pq = fmaf(y[j], dq[2 * i + j / 4][j % 4], pq);
      pk = fmaf(x[j], dk[2 * i + j / 4][j % 4], pk);
    }
  }
  pq = quarter_sum(pq);
  pk = quarter_sum(pk);
  if (!a.normalize) pq = pk = 0.0f;
  if (!in) return;
  T* const oq = (T*)o.dq + (bead * a.keys + kh) * a.dk;
  T* const ok = (T*)o.dk + (bead * a.keys + kh) * a.dk;
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const f32x8 x = own_row(a.K, i) * (rk * pk), y = own_row(a.Q, i) * (rq * pq);
    const int el = 32 * i + 4 * g;
    store4<T>(oq, el, a.dk, (dq[2 * i] - half_of<0>(y)) * (a.scale * rq));
    store4<T>(oq, el + 16, a.dk, (dq[2 * i + 1] - half_of<1>(y)) * (a.scale * rq));
    store4<T>(ok, el, a.dk, (dk[2 * i] - half_of<0>(x)) * rk);
    store4<T>(ok, el + 16, a.dk, (dk[2 * i + 1] - half_of<1>(x)) * rk);
  }
}

constexpr size_t kDeltaLds = 160 * 1024;
constexpr int kDeltaUnits = 256;  // compute units

template <typename T, int DK, int KV, bool MANY>
int grad_kernel(const DeltaArgs& a, const DeltaBack& o, hipStream_t s) {
  typedef GradTiles<T, DK, KV> Tiles;
  constexpr size_t small = sizeof(typename Tiles::Small);
  const int places = Tiles::bytes(2) + small <= kDeltaLds ? 2 : 1;
  const size_t bytes = Tiles::bytes(places) + small;
  const auto f = delta_grad<T, DK, KV, MANY>;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(f),
                          hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess)
    return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(f, dim3(a.n_tiles, a.keys), dim3(kDeltaThreads), bytes, s, a, o, places);
  return mlcg_launch_status();
}

// ---------------------------------------------------------------------------

inline bool lds_limit(const void* f, size_t bytes) {
  return hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) ==
         hipSuccess;
}

// Two buffers of a chunk in LDS where there is room for them and no more
// workgroups than compute units, which then have the LDS for one each.  Forward, 16 x
// 500 beads, 8 heads of 64 in bf16: 53 us with two, 57 with one; 4 x 500: 46 and 50.
// With more workgroups the scan alone, 512 x 100, 8 heads of 32: 68 and 50; 48 x 268,
// 8 heads of 16 in fp32: 45 and 33.
// The limit that is set is that of two in either case: calls of several threads may
// differ in it.
inline size_t scan_most(size_t bytes) { return 2 * bytes <= kDeltaLds ? 2 * bytes : bytes; }
inline int scan_buffers(size_t bytes, int64_t groups) {
  return 2 * bytes <= kDeltaLds && groups <= kDeltaUnits ? 2 : 1;
}

template <typename T, int DK, int WAVES, bool BACK>
int join(const DeltaArgs& a, const DeltaEnds& e, float* ws, hipStream_t s) {
  const auto f = delta_join<T, DK, WAVES, BACK>;
  const size_t one = sizeof(Image<Pieces<T>::mid, DK * DK / 512>);
  const int buffers = 2 * one <= kDeltaLds ? 2 : 1;
  if (!lds_limit(reinterpret_cast<const void*>(f), buffers * one)) return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(f, dim3(a.n_whole, a.heads), dim3(64 * WAVES), buffers * one, s, a, e, ws,
                     buffers);
  return MLCG_OK;
}

template <typename T, int DK, int WAVES>
int forward_waves(const DeltaArgs& a, T* out, DeltaEnds e, float* ws, hipStream_t s) {
  const auto chunk = delta_chunk<T, DK>;
  if (!lds_limit(reinterpret_cast<const void*>(chunk), sizeof(ChunkTiles<T, DK>)))
    return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(chunk, dim3(a.n_tiles, a.keys), dim3(kDeltaThreads),
                     sizeof(ChunkTiles<T, DK>), s, a);
  const int64_t groups = (int64_t)a.n_segs * a.heads;
  if (e.seg_last) {
    constexpr int W = 16 * WAVES < DK ? DK / 16 : WAVES;  // all unit vectors
    const auto alone = delta_scan<T, DK, W, true>;
    const size_t bytes = ScanTiles<T, DK>::bytes(false);
    const int buffers = scan_buffers(bytes, 2 * groups);
    if (!lds_limit(reinterpret_cast<const void*>(alone), scan_most(bytes))) return MLCG_ERR_LAUNCH;
    hipLaunchKernelGGL(alone, dim3(a.n_segs, a.heads, 2), dim3(64 * W), buffers * bytes, s, a, e,
                       out, buffers);
    const int status = join<T, DK, WAVES, false>(a, e, ws, s);
    if (status != MLCG_OK) return status;
    e.seg_init = ws;
  }
  const auto scan = delta_scan<T, DK, WAVES, false>;
  const size_t bytes = ScanTiles<T, DK>::bytes(true);
  const int buffers = scan_buffers(bytes, groups);
  if (!lds_limit(reinterpret_cast<const void*>(scan), scan_most(bytes))) return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(scan, dim3(a.n_segs, a.heads), dim3(64 * WAVES), buffers * bytes, s, a, e, out,
                     buffers);
  return mlcg_launch_status();
}

template <typename T, int DK, int WAVES>
int backward_waves(const DeltaArgs& a, const DeltaBack& o, DeltaEnds e, float* ws, hipStream_t s) {
  const size_t bytes = ScanTiles<T, DK>::bytes(true);
  const int buffers = scan_buffers(bytes, (int64_t)a.n_segs * a.heads);
  const dim3 grid(a.n_segs, a.heads), block(64 * WAVES);
  if (e.seg_last) {
    const auto alone = delta_scan_back<T, DK, WAVES, true>;
    if (!lds_limit(reinterpret_cast<const void*>(alone), scan_most(bytes))) return MLCG_ERR_LAUNCH;
    hipLaunchKernelGGL(alone, grid, block, buffers * bytes, s, a, o, e, buffers);
    const int status = join<T, DK, WAVES, true>(a, e, ws, s);
    if (status != MLCG_OK) return status;
    e.seg_init = ws;
  }
  const auto scan = delta_scan_back<T, DK, WAVES, false>;
  if (!lds_limit(reinterpret_cast<const void*>(scan), scan_most(bytes))) return MLCG_ERR_LAUNCH;
  hipLaunchKernelGGL(scan, grid, block, buffers * bytes, s, a, o, e, buffers);
  const int kv = a.dvp / 32;
  if (a.group == 1)
    return kv == 1   ? grad_kernel<T, DK, 1, false>(a, o, s)
           : kv == 2 ? grad_kernel<T, DK, 2, false>(a, o, s)
           : kv == 3 ? grad_kernel<T, DK, 3, false>(a, o, s)
                     : grad_kernel<T, DK, 4, false>(a, o, s);
  return kv == 1   ? grad_kernel<T, DK, 1, true>(a, o, s)
         : kv == 2 ? grad_kernel<T, DK, 2, true>(a, o, s)
         : kv == 3 ? grad_kernel<T, DK, 3, true>(a, o, s)
                   : grad_kernel<T, DK, 4, true>(a, o, s);
}

template <typename T, int DK>
int forward_dk(const DeltaArgs& a, T* out, const DeltaEnds& e, float* ws, hipStream_t s) {
  return a.dvp <= 64 ? forward_waves<T, DK, 4>(a, out, e, ws, s)
                    : forward_waves<T, DK, 8>(a, out, e, ws, s);
}
template <typename T, int DK>
int backward_dk(const DeltaArgs& a, const DeltaBack& b, const DeltaEnds& e, float* ws,
                hipStream_t s) {
  return a.dvp <= 64 ? backward_waves<T, DK, 4>(a, b, e, ws, s)
                    : backward_waves<T, DK, 8>(a, b, e, ws, s);
}

}  // namespace

template <>
int delta_forward<MLCG_DELTA_TYPE>(const DeltaArgs& a, void* out, const DeltaEnds& e, float* ws,
                                   hipStream_t s) {
  typedef MLCG_DELTA_TYPE T;
  switch (delta_dk(a.dk)) {
    case 32: return forward_dk<T, 32>(a, (T*)out, e, ws, s);
    case 64: return forward_dk<T, 64>(a, (T*)out, e, ws, s);
    default: return forward_dk<T, 128>(a, (T*)out, e, ws, s);
  }
}

template <>
int delta_backward<MLCG_DELTA_TYPE>(const DeltaArgs& a, const DeltaBack& b, const DeltaEnds& e,
                                    float* ws, hipStream_t s) {
  typedef MLCG_DELTA_TYPE T;
  switch (delta_dk(a.dk)) {
    case 32: return backward_dk<T, 32>(a, b, e, ws, s);
    case 64: return backward_dk<T, 64>(a, b, e, ws, s);
    default: return backward_dk<T, 128>(a, b, e, ws, s);
  }
}

#endif  // MLCG_DELTA_TYPE
