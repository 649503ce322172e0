// Attention of the beads of a chain to each other with a learned bias by
// relative position (gfx950): the kernels, one file of instantiations for
// each element type (attention_f32.hip, attention_f16.hip,
// attention_bf16.hip), the entry points in attention.hip.
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
// keeps a running maximum m and sum l of every row (base-2 exponents), apart,
// from which the backward passes form P = exp2(l_ij log2(e) - m) / l again: in
// one number with m, log2 l would be lost beside a large bias that all of a
// row's keys have in common.
//
// Tiles: a wave owns 32 queries (forward, dq) or 32 keys (dk, dv) as the
// columns of 32 x 32 MFMA tiles, so a lane is one query (key) and the softmax
// statistics are lane values; the other side comes in tiles of KT rows
// through LDS.  The 16 accumulators of a lane are rows 8 a + 4 g + c (g the
// lane's half): as the contraction over them is free to be permuted, they are
// used as the B operand of the next product as they are, and the A operand
// takes the tile's columns with its rows in that order: in 16 bits by the
// transposing LDS read (4 rows of a column a lane), in 32 bits by single
// values.  So every operand has one LDS tile, row by row, for both products.
// In 16 bits a step of 16 is one v_mfma_f32_32x32x16, in 32 bits eight
// v_mfma_f32_32x32x2.
//
// A workgroup is NQ x NK waves: NQ blocks of 32 columns, and NK parts of the
// rows, each wave its own KT rows of a staged tile of NK KT; the parts are
// joined through LDS at the end.  The next tile's rows are loaded into
// registers while the present one is used, and written to the other of two
// buffers: one barrier a tile.
//
// LDS rows hold 16-byte chunks, exchanged by row (xor), so that the 16-byte
// reads of 8 consecutive rows and the transposing reads fall on all banks (of
// all LDS instructions, the writes among them, 0.8 to 1.2 conflict cycles each
// are counted in 16 bits, of 4 to 5 that they take).
//
// The bias of an offset is one LDS value a head: an array over the offsets
// from -(R + M) to R + M, M beyond the largest span of a tile, so that a tile
// that touches the band |offset| < R needs no clipping; a block of 32 rows
// outside of it has one value.  The table's gradient is summed by offset into
// the same kind of array, one a wave:
//   index positions: the block of 32 x 32 dS goes through LDS, [query][key]
//   with a gap of zeros behind each row, at once or in two halves, and lane n
//   adds the diagonal offset n - 31 (32 reads a lane, no test: past an end
//   stand zeros);
//   given positions: LDS adds of integers, dS scaled by a power of two and cut
//   in two parts of 15 bits (LDS adds of floats take about 200 cycles a wave
//   against 6, and their order would change the last bits);
// then by bucket, then over the workgroups in a fixed order.
#pragma once

#include <type_traits>

#include "chain.h"

constexpr int kAttnQ = 32;               // columns of a wave
constexpr int kAttnWaves = 4;            // waves of columns of a workgroup, at most
constexpr int kAttnSpan = 96;            // offsets beyond the reach that a block can touch
constexpr float kAttnLog2e = 1.4426950408889634f;
constexpr float kAttnLazy = 8.0f;        // the running maximum may lag by this many powers of two
// A tile whose logits exceed the running maximum by more than this, or lie as
// far below 0 when there was none, is formed once more about the new one: a
// difference of 2^6 is rounded by 2^-18, as logits of that size are themselves,
// but from a bias of -1e9 to an ordinary key nothing of the key would be left.
constexpr float kAttnJump = 64.0f;

struct AttnArgs {
  const void *q, *k, *v, *table, *out, *grad;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  int64_t beads;
  const int32_t* bucket_of;  // [2 reach + 1]
  const int4* tiles;         // (chain's first row, its length, tile's first row in it, chain)
  const uint8_t* keep;
  const int32_t* pos;
  float* lse;  // [2][heads][beads]: m, +inf for a row without keys, and l
  int n_tiles, heads, group, dim, reach, buckets;
  float scale;
  void* rest;  // what the rounding of out leaves out, or NULL
};

// Whether positions are given: known when the kernel is built, or (kEither, in
// the form without 16-byte loads) when it runs.
enum { kIndex = 0, kGiven = 1, kEither = 2 };

// What dq leaves for dk and dv of every row [heads][beads], and of every wave of
// queries [heads][tiles][waves].
struct AttnRows {
  float *delta, *start;  // do . o;  -(m + log2 l) / c, in 16 bits
  float* apart;          // whether m is too large for start to take its place
};

struct AttnGrads {
  void *dq, *dk, *dv, *dtable;
  float* ws;
  const int32_t *order, *first;
};

// shape: waves of columns and of rows, 10 NQ + NK
template <typename T>
int attn_forward(AttnArgs a, int shape, void* out, hipStream_t s);
template <typename T>
int attn_backward(AttnArgs a, int shape, const AttnGrads& o, hipStream_t s);

#ifdef MLCG_ATTENTION_TYPE

namespace {

// rows of a part of a staged tile: 64, or 32 of the widest and, backward, of
// 32-bit elements (the accumulators and blocks of 64 leave two waves a SIMD)
template <typename T, int DP>
constexpr int part_rows() {
  return sizeof(T) * DP <= 128 ? 64 : 32;
}
template <typename T, int DP>
constexpr int part_rows_bwd() {
  return sizeof(T) == 2 ? part_rows<T, DP>() : 32;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// what row r's chunks are exchanged by, in a tile of N chunks a row: the 16
// bytes of 8 consecutive rows, and the 32 bytes of 4 that 16 lanes of the
// transposing read take, fall on all banks
template <int N>
__device__ __forceinline__ constexpr int chunk_swap(int r) {
  static_assert(N >= 4, "a row holds at least four chunks");
  return N >= 8 ? ((r & 3) << 1) | ((r >> 2) & 1) : (r & 2) | ((r >> 2) & 1);
}

// element offset of (row, el) in an LDS tile of LEN elements a row
template <typename T, int LEN>
__device__ __forceinline__ int tile_at(int row, int el) {
  constexpr int EPC = 16 / sizeof(T);
  return row * LEN + (((el / EPC) ^ chunk_swap<LEN / EPC>(row)) * EPC) + el % EPC;
}

// A operand of a step over the columns: row `row`, elements 16 k + 8 g ..
template <typename T, int LEN>
__device__ __forceinline__ v8<T> row_frag(const T* tile, int row, int el) {
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const v8<T>*>(tile + tile_at<T, LEN>(row, el));
  } else {
    const v4<T> a = *reinterpret_cast<const v4<T>*>(tile + tile_at<T, LEN>(row, el));
    const v4<T> b = *reinterpret_cast<const v4<T>*>(tile + tile_at<T, LEN>(row, el + 4));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// A operand of a step over the rows: column 32 n + (lane & 31), rows 16 u +
// 4 g + 0..3 and 16 u + 8 + 4 g + 0..3
template <typename T, int LEN>
__device__ __forceinline__ v8<T> column_frag(const T* tile, int u, int n) {
  const int lane = threadIdx.x & 63, g = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    // 16 lanes give the places of 4 rows x 16 columns, lane i those of row
    // i / 4, and get a column's 4 rows each
    const int el = 32 * n + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const int row = 16 * u + 4 * g + ((lane & 15) >> 2);
    s16x4 x[2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
      x[a] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4*)(tile + tile_at<T, LEN>(row + 8 * a, el)));
    const auto both = __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(v8<T>, both);
  } else {
    v8<T> r;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      r[e] = tile[tile_at<T, LEN>(16 * u + 8 * (e / 4) + 4 * g + e % 4, 32 * n + (lane & 31))];
    return r;
  }
}

// the wave's number in its workgroup, as the one value that it is
__device__ __forceinline__ int wave_number() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

// the row of a lane's accumulator i % 16 of block i / 16
__device__ __forceinline__ constexpr int acc_row(int i, int g) {
  return 8 * (i / 4) + 4 * g + i % 4;  // 32 a block
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

// 8 elements of a row at el: a B operand's fragment, zeros where !ok and past
// dim.  VEC: rows begin at multiples of 16 bytes and dim is one.
template <typename T, bool VEC>
__device__ __forceinline__ v8<T> load8(const T* row, int el, bool ok, int dim) {
  v8<T> r{};
  if (!ok) return r;
  if constexpr (VEC) {
    v4<T> a{}, b{};
    if (el < dim) a = *reinterpret_cast<const v4<T>*>(row + el);
    if (el + 4 < dim) b = *reinterpret_cast<const v4<T>*>(row + el + 4);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (el + e < dim) r[e] = row[el + e];
    return r;
  }
}

// ROWS rows on their way from memory to LDS, a thread PER chunks of 16 bytes.
// A chunk's place is the tile's first row plus an offset that stays the same
// from tile to tile.  Rows past the chain's end are read as its last one; like
// absent ones they are replaced by zeros (0 P would not be 0 where they hold
// no number).  Columns past dim repeat the last ones: they meet zeros of the
// other operand or accumulators that nothing reads.
template <typename T, int DP, int ROWS, int NT, bool VEC>
struct Stage {
  static constexpr int EPC = 16 / sizeof(T), NCH = DP / EPC, PER = ROWS * NCH / NT;
  static_assert(ROWS * NCH % NT == 0, "whole chunks a thread");
  typedef T chunk __attribute__((ext_vector_type(EPC)));
  chunk x[PER];
  uint32_t off[PER];  // bytes
  int stride;

  __device__ __forceinline__ static int row(int p) { return (threadIdx.x + p * NT) / NCH; }
  __device__ __forceinline__ static int column(int p) { return threadIdx.x % NCH * EPC; }

  __device__ __forceinline__ void init(int row_stride, int dim) {
    static_assert(NT % NCH == 0, "a thread's chunks stand in one column");
    stride = row_stride;
#pragma unroll
    for (int p = 0; p < PER; ++p)
      off[p] = (uint32_t)(row(p) * stride + min(column(p), dim - (VEC ? EPC : 1))) * sizeof(T);
  }
  // src: the tile's first row; rows: those of the chain from there on
  __device__ __forceinline__ void load(const T* src, int rows, int dim) {
    const char* at = reinterpret_cast<const char*>(src);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      uint32_t o = off[p];
      if (rows < ROWS) o -= (uint32_t)max(row(p) - (rows - 1), 0) * stride * sizeof(T);
      if constexpr (VEC) {
        x[p] = *reinterpret_cast<const chunk*>(at + o);
      } else {
        const T* e = reinterpret_cast<const T*>(at + o);
        x[p] = chunk{};
#pragma unroll
        for (int j = 0; j < EPC; ++j)
          if (column(p) + j < dim) x[p][j] = e[j];
      }
    }
  }
  // The rows of the thread's chunks that are past the end or absent, in two
  // steps: the bytes of `keep` (may be NULL) are sent for with a tile's rows
  // and looked at with them, as loads return in order.
  struct Rows {
    uint8_t keep[PER];
    int rows;
    __device__ __forceinline__ void load(const uint8_t* bytes, int n) {
      rows = n;
#pragma unroll
      for (int p = 0; p < PER; ++p) keep[p] = bytes ? bytes[min(row(p), n - 1)] : 1;
    }
    __device__ __forceinline__ bool absent(int p) const { return row(p) >= rows || !keep[p]; }
  };
  __device__ __forceinline__ void drop(const Rows& r) {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      if (r.absent(p)) x[p] = chunk{};
  }
  __device__ __forceinline__ void put(T* tile) const {
#pragma unroll
    for (int p = 0; p < PER; ++p)
      *reinterpret_cast<chunk*>(tile + tile_at<T, DP>(row(p), column(p))) = x[p];
  }
};

// ext[n] = log2(e) bias of the offset n - (reach + kAttnSpan), clipped; a bias
// of the type's lowest or highest value stays a number.  Of index positions in a
// chain of `len`, offsets that no pair has, but rows past the end do, have 0:
// the table may hold anything there, and -inf + inf is not -inf.
template <typename T>
__device__ __forceinline__ void fill_bias(const AttnArgs& a, int head, int len, bool given,
                                          float* ext) {
  const int n = 2 * (a.reach + kAttnSpan) + 1;
  const T* table = (const T*)a.table;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int d = min(max(i - kAttnSpan, 0), 2 * a.reach);
    const float b = (float)table[(int64_t)a.bucket_of[d] * a.heads + head];
    const float e = kAttnLog2e * b;
    ext[i] = fabsf(e) > 3.0e38f && fabsf(b) != INFINITY ? copysignf(3.0e38f, b) : e;
    if (!given && abs(i - (a.reach + kAttnSpan)) >= len) ext[i] = 0.0f;
  }
}

// clipped offset p_j - p_i as an index of ext, for any int32 positions
__device__ __forceinline__ int offset_cell(int pj, int pi, int reach) {
  return min(max(__builtin_elementwise_sub_sat(pj, pi), -reach), reach) + reach + kAttnSpan;
}

// v, rounded to fp32 where it is a product, as T.  hipcc may otherwise fold a
// product into the conversion to fp16 (one rounding in place of two) in one
// form of a kernel and not in another, and equal calls differ by a bit.
template <typename T>
__device__ __forceinline__ T round_to(float v) {
  if constexpr (std::is_same<T, _Float16>::value) asm("" : "+v"(v));
  return (T)v;
}

// The probabilities and dS, in fp32 until here, take the elements' type as
// operands of the products with v, do, k and q, as the matrix instructions ask
// for, and are each off by half a unit of that type, as their other factor is:
// the probabilities below 2^kAttnLazy relative to the row's base (forward) or at
// most 1 (backward), dS, which has the size of the gradients, in fp16 times a
// power of two (OperandScale).  The sums that follow, of the row, of o, dq, dk,
// dv and of the table, stay in fp32, and the row's sum and the table take the
// values before this rounding.
template <typename T>
__device__ __forceinline__ v8<T> pack8(const float* p) {
  v8<T> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = round_to<T>(p[e]);
  return r;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
}

// s[n] += the wave's 32 columns of  tile . B  for the rows 32 n .. 32 n + 31.
// Of 16 channels in 32 bits the padding is passed over (48 chains of up to 268
// beads, 8 heads: dq 59 us against 72, dk and dv 54 against 69).
template <typename T, int DP, int N>
__device__ __forceinline__ void row_product(const T* tile, const v8<T> (&b)[DP / 16], int dim,
                                            f32x16 (&s)[N]) {
  const int col = threadIdx.x & 31, g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    if (sizeof(T) == 2 || DP > 32 || k == 0 || dim > 16)
#pragma unroll
      for (int n = 0; n < N; ++n)
        mma(s[n], row_frag<T, DP>(tile + 32 * n * DP, col, 16 * k + 8 * g), b[k]);
}

// Keeps the reads of the above two ahead of the products that take them (in 16
// bits, where a product is shorter than the read's latency): hipcc otherwise
// orders them read, wait, product.  READS: the 16-byte reads before the first.
template <typename T, int DP, int N, int READS>
__device__ __forceinline__ void reads_ahead() {
  if constexpr (sizeof(T) == 2) {
    constexpr int products = DP / 16 * N;
    __builtin_amdgcn_sched_group_barrier(0x100, READS + 2, 0);  // LDS reads
#pragma unroll
    for (int i = 0; i < products; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix instructions
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  }
}

// acc += tile^T . P  with P the 32 N rows of a lane's column
template <typename T, int DP, int N>
__device__ __forceinline__ void column_product(const T* tile, const float (&p)[16 * N],
                                               f32x16 (&acc)[DP / 32]) {
#pragma unroll
  for (int u = 0; u < 2 * N; ++u) {
    const v8<T> b = pack8<T>(p + 8 * u);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) mma(acc[n], column_frag<T, DP>(tile, u, n), b);
  }
}

// a lane's rows of one value a row
template <int N>
__device__ __forceinline__ void load_rows(const float* rows, f32x16 (&s)[N]) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int i = 0; i < 16 * N; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(rows + acc_row(i, g));
    s[i / 16][i % 16] = v.x;
    s[i / 16][i % 16 + 1] = v.y;
    s[i / 16][i % 16 + 2] = v.z;
    s[i / 16][i % 16 + 3] = v.w;
  }
}

// a lane's column (the accumulators of DP rows) as a row of dst
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void store_column(T* dst, const f32x16 (&acc)[DP / 32], float f,
                                             int dim) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * n + 8 * a + 4 * g;
      v4<T> o;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = round_to<T>(acc[n][4 * a + c] * f);
      if constexpr (VEC) {
        if (d < dim) *reinterpret_cast<v4<T>*>(dst + d) = o;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (d + c < dim) dst[d + c] = o[c];
      }
    }
}

// what the rounding of a column leaves out, rounded itself
template <typename T, int DP, bool VEC>
__device__ __forceinline__ void store_rest(T* dst, const f32x16 (&acc)[DP / 32], float f,
                                           int dim) {
  const int g = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int d = 32 * n + 8 * a + 4 * g;
      v4<T> o;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v = acc[n][4 * a + c] * f;
        asm("" : "+v"(v));  // as store_column rounds it
        o[c] = (T)(v - (float)(T)v);
      }
      if constexpr (VEC) {
        if (d < dim) *reinterpret_cast<v4<T>*>(dst + d) = o;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (d + c < dim) dst[d + c] = o[c];
      }
    }
}

// The power of two that a lane's column of dS is multiplied by before it becomes
// an operand in fp16, whose range the gradients of a scaled loss, or of a long
// chain, leave at either end: the largest value so far lies between 2^13 and
// 2^15, so that values down to 2^-28 of it keep their bits.  It is taken out of
// the accumulators where they are stored.  The other types need none.
template <typename T>
struct OperandScale {
  static constexpr bool kOn = std::is_same<T, _Float16>::value;
  float up = 0.0f;  // 0 before the first value

  template <int M, int NA>
  __device__ __forceinline__ void fit(float (&x)[M], f32x16 (&acc)[NA]) {
    if constexpr (kOn) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < M; ++i) top = fmaxf(top, fabsf(x[i]));
      if (__any(top * up > 32768.0f || (up == 0.0f && top > 0.0f))) {
        top = fmaxf(top, other_half(top));
        float alpha = 1.0f;
        if (!(top <= 3.0e38f)) {  // infinite: it may as well be so in fp16
          up = up == 0.0f ? 1.0f : up;
        } else if (top * up > 32768.0f || (up == 0.0f && top > 0.0f)) {
          int e;
          (void)frexpf(top, &e);  // top < 2^e
          const float next = ldexpf(1.0f, 14 - max(e, -100));
          alpha = up == 0.0f ? 1.0f : next / up;
          up = next;
        }
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[n][r] *= alpha;
      }
#pragma unroll
      for (int i = 0; i < M; ++i) x[i] *= up;
    }
  }
  // the NK parts on the smallest of their scales; buf: 32 NQ NK values
  template <int NQ, int NK, int NA>
  __device__ __forceinline__ void join(f32x16 (&acc)[NA], float* buf) {
    if constexpr (kOn && NK > 1) {
      const int lane = threadIdx.x & 63, wave = wave_number(), wq = wave % NQ;
      __syncthreads();
      if (lane < 32) buf[32 * wave + lane] = up;
      __syncthreads();
      float least = 0.0f;
#pragma unroll
      for (int p = 0; p < NK; ++p) {
        const float u = buf[32 * (p * NQ + wq) + (lane & 31)];
        if (u != 0.0f) least = least == 0.0f ? u : fminf(least, u);
      }
      const float alpha = up == 0.0f ? 1.0f : least / up;
      up = least;
#pragma unroll
      for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[n][r] *= alpha;
    }
  }
  __device__ __forceinline__ float undo() const { return kOn && up != 0.0f ? 1.0f / up : 1.0f; }
};

// acc of the NK waves of a column block, joined in the order of the parts;
// the sums are part 0's.  buf: (NK - 1) NQ 64 values for each accumulator.
template <int DP, int NQ, int NK>
__device__ __forceinline__ void join_parts(f32x16 (&acc)[DP / 32], float* buf) {
  if constexpr (NK > 1) {
    const int lane = threadIdx.x & 63, wave = wave_number(), wq = wave % NQ, wk = wave / NQ;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) {
      __syncthreads();
      if (wk > 0)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          buf[(((wk - 1) * NQ + wq) * 16 + r) * 64 + lane] = acc[n][r];
      __syncthreads();
      if (wk == 0)
#pragma unroll
        for (int p = 1; p < NK; ++p)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[n][r] += buf[(((p - 1) * NQ + wq) * 16 + r) * 64 + lane];
    }
  }
}

// scale log2(e); a scale of 0 is one that leaves nothing of the products (sums
// begin with values divided by it)
__device__ __forceinline__ float logit_factor(const AttnArgs& a) {
  return fabsf(a.scale) < 1e-30f ? 1e-30f : a.scale * kAttnLog2e;
}

// Where `rows` rows lie to the wave's 32 columns: all offsets at or past the
// reach (1), at or before its negative (-1), or neither (0).
__device__ __forceinline__ int block_side(int d_min, int d_max, int R) {
  return d_min >= R ? 1 : d_max <= -R ? -1 : 0;
}

template <int POS>
__device__ __forceinline__ bool given_positions(const AttnArgs& a) {
  return POS == kEither ? a.pos != nullptr : POS == kGiven;
}

// What stands for the keys of a tile in LDS: the value that their products'
// sums begin with (0, or for an absent key what makes the logit -inf), and
// their positions (past the end another bead's, so that their offsets are
// pairs').  Thread i loads row i's.
struct KeyInfo {
  bool in;
  uint8_t keep;
  int pos;
  template <int POS>
  __device__ __forceinline__ void load(const AttnArgs& a, const int4& t, int k0, int rows) {
    const int i = threadIdx.x;
    in = i < rows && k0 + i < t.y;
    keep = 1;
    pos = 0;
    if (in) {
      const int64_t row = (int64_t)t.x + k0 + i;
      if (a.keep) keep = a.keep[row];
      if (given_positions<POS>(a)) pos = a.pos[row];
    }
  }
  template <int POS>
  __device__ __forceinline__ void put(const AttnArgs& a, int rows, int other, float* caps,
                                      int* kpos) const {
    if ((int)threadIdx.x < rows) {
      const float none = logit_factor(a) > 0.0f ? -INFINITY : INFINITY;
      caps[threadIdx.x] = in && keep ? 0.0f : none;
      if (POS != kIndex) kpos[threadIdx.x] = in ? pos : other;
    }
  }
};

// A wave of queries: its first one, the lane's, and the positions of the
// lane's and of the wave's ends.
struct QueryPlace {
  int first, mine, pos, lo, hi;
  bool ok;
  __device__ __forceinline__ QueryPlace(const AttnArgs& a, bool given, const int4& t, int begin)
      : first(begin), mine(begin + (threadIdx.x & 31)), pos(0), lo(0), hi(0) {
    ok = mine < t.y;
    if (given) {
      pos = a.pos[(int64_t)t.x + min(mine, t.y - 1)];
      lo = wave_min(pos);
      hi = wave_max(pos);
    }
  }
};

// The size of a row's shift from which on the logits are rounded before it is
// taken off.  Below, it is taken off the bias first, so that a large bias that
// all keys of a row have in common cancels and the products stay (the logits
// then lie within half a spacing of the shift of 0: 2^6 in 32 bits, 1 in
// fp16, whose probabilities have to fit it); beyond, the products vanish beside
// a bias, or are themselves that large.
template <typename T>
constexpr float kAttnFar = std::is_same<T, _Float16>::value ? 0x1p24f : 0x1p31f;

template <typename T>
__device__ __forceinline__ bool far_shift(float shift) {
  return fabsf(shift) >= kAttnFar<T> && fabsf(shift) < INFINITY;
}

// The logits (base 2) less `shift` of 32 N keys from kb on (rows) and the
// wave's queries (lanes); returns the keys' side.  A shift of +inf: -inf.
// any_far: whether far_shift holds for any of the wave's rows.
template <typename T, int N, int POS>
__device__ __forceinline__ int query_logits(const AttnArgs& a, const f32x16 (&s)[N],
                                            const float* ext, const float* cap, const int* kpos,
                                            int kb, const QueryPlace& q, float shift,
                                            bool any_far, float (&x)[16 * N]) {
  const int lane = threadIdx.x & 63, g = lane >> 5;
  const float c = logit_factor(a);
  const int R = a.reach;
  float near = shift;
  if (__builtin_expect(any_far, 0)) near = far_shift<T>(shift) ? 0.0f : shift;
  int side;
  if (given_positions<POS>(a)) {
    const int kp = kpos[lane % (32 * N)];
    const bool absent = cap[lane % (32 * N)] != 0.0f;
    side = __all(absent || __builtin_elementwise_sub_sat(kp, q.hi) >= R)    ? 1
           : __all(absent || __builtin_elementwise_sub_sat(kp, q.lo) <= -R) ? -1
                                                                            : 0;
  } else {
    side = block_side(kb - (q.first + 31), kb + 32 * N - 1 - q.first, R);
  }
  if (side) {
    const float b = ext[side > 0 ? 2 * R + kAttnSpan : kAttnSpan] - near;
#pragma unroll
    for (int i = 0; i < 16 * N; ++i) x[i] = fmaf(s[i / 16][i % 16], c, b);
  } else if (given_positions<POS>(a)) {
#pragma unroll
    for (int i = 0; i < 16 * N; ++i)
      x[i] = fmaf(s[i / 16][i % 16], c, ext[offset_cell(kpos[acc_row(i, g)], q.pos, R)] - near);
  } else {
    const float* e = ext + (kb - q.mine + 4 * g + R + kAttnSpan);
#pragma unroll
    for (int i = 0; i < 16 * N; ++i) x[i] = fmaf(s[i / 16][i % 16], c, e[acc_row(i, 0)] - near);
  }
  if (__builtin_expect(any_far, 0)) {
    const float rest = far_shift<T>(shift) ? shift : 0.0f;
#pragma unroll
    for (int i = 0; i < 16 * N; ++i) x[i] -= rest;
  }
  return side;
}

// Waves a SIMD that the registers of a kernel are limited for: `values` 32-bit
// values of fragments and accumulators, and about 70 more.
constexpr int waves_for(int values) {
  return values <= 24 ? 3 : values < 192 ? 2 : 1;
}

template <typename T, int DP, int NQ, int NK>
struct FwdLds {
  static constexpr int KS = part_rows<T, DP>() * NK;
  T k[2][KS * DP], v[2][KS * DP];
  float cap[2][KS];
  int kpos[2][KS];
  float ext[1];  // 2 (reach + kAttnSpan) + 1
};

// a query's fragments and an accumulator of DP rows; one wave more where a
// workgroup of four waves has few chunks to hold (2 x 4099 beads of 64 channels
// in bf16: 133 us against 167, as all workgroups then run at once)
template <typename T, int DP, int NQ, int NK>
constexpr int fwd_waves() {
  constexpr int values = DP * (int)sizeof(T) / 8 + DP / 2;
  return waves_for(values) + (NQ == 4 && NK == 1 && values <= 48 ? 1 : 0);
}

// Forward; lanes are queries, the tiles hold keys.  Bound by the issue of its
// matrix and vector instructions, which overlap between the waves of a SIMD
// alone: at 8191 beads, 8 heads of 64 on 2 in bf16 a logit costs 6.9 vector
// instructions (one of them exp2, at a quarter of the rate), so that they take
// about 60 % of the SIMDs' cycles and the products 25 %.  211 us, 652 TFLOP/s,
// 56 % of a large library product's rate.  4 chains of 1031, 4 heads of 32 in
// fp32: 47 us (46 TFLOP/s), 144 workgroups of 128 queries on 256 compute units.
// 512 chains of up to 100, 4 heads of 32 in bf16, with rest: 19 us, one or two
// tiles a workgroup, bound by the latency of its first loads.
template <typename T, int DP, int NQ, int NK, bool VEC, int POS>
__global__ __launch_bounds__(64 * NQ * NK, (fwd_waves<T, DP, NQ, NK>())) void attn_fwd_kernel(
    AttnArgs a, T* __restrict__ out) {
  constexpr int RT = part_rows<T, DP>(), N = RT / 32, KS = RT * NK, NT = 64 * NQ * NK;
  using Lds = FwdLds<T, DP, NQ, NK>;
  extern __shared__ __align__(16) unsigned char smem[];
  Lds& L = *reinterpret_cast<Lds*>(smem);
  float* ext = L.ext;

  const int head = blockIdx.x % a.heads, kv = head / a.group;
  const int4 t = a.tiles[blockIdx.x / a.heads];
  const int lane = threadIdx.x & 63, g = lane >> 5, wave = wave_number();
  const int wq = wave % NQ, wk = wave / NQ;
  const T* kbase = (const T*)a.k + (int64_t)t.x * a.k_row + kv * a.k_head;
  const T* vbase = (const T*)a.v + (int64_t)t.x * a.v_row + kv * a.v_head;
  const uint8_t* keep = a.keep ? a.keep + t.x : nullptr;
  Stage<T, DP, KS, NT, VEC> ks, vs;
  KeyInfo info;
  ks.init((int)a.k_row, a.dim);
  vs.init((int)a.v_row, a.dim);
  ks.load(kbase, t.y, a.dim);
  vs.load(vbase, t.y, a.dim);
  typename Stage<T, DP, KS, NT, VEC>::Rows absent;
  absent.load(keep, t.y);
  info.template load<POS>(a, t, 0, KS);

  const bool given = given_positions<POS>(a);
  const QueryPlace qi(a, given, t, t.z + kAttnQ * wq);
  const T* q = (const T*)a.q + ((int64_t)t.x + qi.mine) * a.q_row + head * a.q_head;
  v8<T> qf[DP / 16];
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) qf[k] = load8<T, VEC>(q, 16 * k + 8 * g, qi.ok, a.dim);
  fill_bias<T>(a, head, t.y, given, ext);

  f32x16 acc[DP / 32] = {};
  // the exponents are relative to base, the row's maximum so far or up to
  // kAttnLazy below it; 0 before the row's first key
  bool first = true, any_far = false;
  float base = 0.0f, l = 0.0f;
  int buf = 0;
  // puts the tile of k0 into LDS and sends for the next one
  auto next_tile = [&](int k0) {
    if (keep || k0 + KS > t.y) {
      ks.drop(absent);
      vs.drop(absent);
    }
    ks.put(L.k[buf]);
    vs.put(L.v[buf]);
    info.template put<POS>(a, KS, qi.lo, L.cap[buf], L.kpos[buf]);
    const int kn = k0 + KS;
    if (kn < t.y) {
      ks.load(kbase + kn * a.k_row, t.y - kn, a.dim);
      vs.load(vbase + kn * a.v_row, t.y - kn, a.dim);
      if (keep || kn + KS > t.y) absent.load(keep ? keep + kn : keep, t.y - kn);
      info.template load<POS>(a, t, kn, KS);
    }
    __syncthreads();
  };
  if (qi.first >= t.y)  // no queries: this wave only loads
    for (int k0 = 0; k0 < t.y; k0 += KS, buf ^= 1) next_tile(k0);
  else for (int k0 = 0; k0 < t.y; k0 += KS, buf ^= 1) {
    next_tile(k0);
    const int kb = k0 + RT * wk;
    if (kb >= t.y) continue;
    const T* vt = L.v[buf] + RT * wk * DP;
    const float* cap = L.cap[buf] + RT * wk;
    float x[16 * N];
    // a jump is known to a spacing of its larger end, at the second turn to a
    // spacing of what is left, and at the third it is gone
    constexpr int kAttnTurns = 3;
#pragma unroll 1
    for (int turn = 1;; ++turn) {
      // nothing of the tile is kept in registers for another turn (hipcc would,
      // and spill: 1053 us in place of 211 at 8191 beads)
      asm volatile("" ::: "memory");
      f32x16 s[N];
      load_rows<N>(cap, s);
      row_product<T, DP, N>(L.k[buf] + RT * wk * DP, qf, a.dim, s);
      reads_ahead<T, DP, N, 4 * N>();
      query_logits<T, N, POS>(a, s, ext, cap, L.kpos[buf] + RT * wk, kb, qi, base,
                              any_far, x);
      float top = x[0];
#pragma unroll
      for (int i = 1; i < 16 * N; ++i) top = fmaxf(top, x[i]);
      // the base follows only where the maximum has grown by more than
      // 2^kAttnLazy (or there was none): the exponentials stay below
      // 2^kAttnLazy, and most tiles leave the sums alone
      if (__builtin_expect(!__any(top > kAttnLazy || (first && top > -INFINITY)), 1)) break;
      top = fmaxf(top, other_half(top));
      const bool none = top == -INFINITY;  // no key so far: exp2(-inf) = 0
      const float next = none ? base : first ? top : fmaxf(base, base + top);
      // the difference of the two as they are kept, which the next tiles see
      const float grown = next - base;
      base = next;
      any_far = __any(far_shift<T>(base));
      // nothing to scale before the first key, where the base may have to fall
      const float alpha = grown < 0.0f ? 0.0f : __builtin_amdgcn_exp2f(-grown);
      first = first && none;
      l *= alpha;
#pragma unroll
      for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[n][r] *= alpha;
      if (__builtin_expect(turn < kAttnTurns && __any(fabsf(grown) > kAttnJump), 0)) continue;
#pragma unroll
      for (int i = 0; i < 16 * N; ++i) x[i] -= grown;
      break;
    }
    float sum[4] = {};
#pragma unroll
    for (int i = 0; i < 16 * N; ++i) {
      x[i] = __builtin_amdgcn_exp2f(x[i]);
      sum[i % 4] += x[i];
    }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    column_product<T, DP, N>(vt, x, acc);
  }
  l += other_half(l);
  if constexpr (NK > 1) {
    // the parts on one maximum, then summed
    __shared__ float ms[NK][NQ][kAttnQ], ls[NK][NQ][kAttnQ];
    if (g == 0) {
      ms[wk][wq][lane] = first ? -INFINITY : base;
      ls[wk][wq][lane] = l;
    }
    __syncthreads();
    const int c = lane & 31;
    float top = ms[0][wq][c];
#pragma unroll
    for (int p = 1; p < NK; ++p) top = fmaxf(top, ms[p][wq][c]);
    const float mine = base;
    base = top == -INFINITY ? 0.0f : top;
    l = 0.0f;
#pragma unroll
    for (int p = 0; p < NK; ++p)
      l = fmaf(ls[p][wq][c], __builtin_amdgcn_exp2f(ms[p][wq][c] - base), l);
    const float f = first ? 0.0f : __builtin_amdgcn_exp2f(mine - base);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[n][r] *= f;
    join_parts<DP, NQ, NK>(acc, reinterpret_cast<float*>(smem));
  }
  if (wk > 0 || !qi.ok) return;
  const int64_t row = (int64_t)t.x + qi.mine;
  const int64_t flat = (row * a.heads + head) * a.dim;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  store_column<T, DP, VEC>(out + flat, acc, inv, a.dim);
  // a row's dS sum to what delta = do . o is off, so that the rounding of o
  // would be the table's largest error (2 chains of 4099 beads in bf16: 4.3e-3
  // of its gradient against 1.7e-3)
  if constexpr (sizeof(T) == 2)
    if (a.rest) store_rest<T, DP, VEC>((T*)a.rest + flat, acc, inv, a.dim);
  if (a.lse && g == 0) {
    a.lse[head * a.beads + row] = l == 0.0f ? INFINITY : base;
    a.lse[(a.heads + head) * a.beads + row] = l;
  }
}

// Whether a chain has one present key at most, of up to 64 beads.  The softmax
// over one key is constant: the backward passes then write dq = dk = 0 and dv
// the sum of do over the rows that have the key (a bias of -inf may take it from
// a row: l = 0), not what the roundings of their sums would leave of them.  A
// row whose l is no number makes them none, too: l - l.
__device__ __forceinline__ bool lone_key(const uint8_t* keep, int len) {
  if (len > 64) return false;
  const int lane = threadIdx.x & 63;
  return __popcll(__ballot(lane < len && (!keep || keep[lane]))) <= 1;
}

// ---------------------------------------------------------------------------
// The table's gradient

constexpr int kDiagPitch = 68;  // 32 values and the gap of zeros; 16-byte rows
// queries that pass through the block at a time: half of them where the
// registers allow three waves a SIMD, which the whole block's LDS would not
// (512 chains of up to 100 beads, 4 heads of 32 in bf16: dq 37 us against 47)
template <int DP>
constexpr int diag_rows() {
  return DP == 32 ? 16 : 32;
}
template <int DP>
constexpr int diag_floats() {
  return 32 + diag_rows<DP>() * kDiagPitch;
}

// mine[cell of offset d0 + n - 31] += diagonal n of the block whose lanes are
// queries 0..31 and whose rows are keys 0..31, d0 = first key - first query.
template <int DP>
__device__ __forceinline__ void add_diagonals(const float* x, float* scratch, float* at_d0) {
  constexpr int QR = diag_rows<DP>();
  const int lane = threadIdx.x & 63, q = lane & 31, g = lane >> 5;
  float* row = scratch + 32 + (q % QR) * kDiagPitch + 4 * g;
  float t[4] = {};
#pragma unroll
  for (int q0 = 0; q0 < 32; q0 += QR) {
    if (q / QR == q0 / QR)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<float4*>(row + 8 * a) =
            make_float4(x[4 * a], x[4 * a + 1], x[4 * a + 2], x[4 * a + 3]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const float* d = scratch + 32 + lane - 31 + q0;
#pragma unroll
    for (int r = 0; r < QR; ++r) t[r % 4] += d[r * (kDiagPitch + 1)];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  at_d0[lane - 31] += (t[0] + t[1]) + (t[2] + t[3]);
}

// Sums by offset for given positions: integers of dS 2^e, a high part of at
// most 2^15 a value and 15 bits below it, 16 tiles (up to 2^11 values each)
// before they are moved to the wave's float array.
struct OffsetInts {
  int *hi, *lo;
  float scale, inverse;  // 2^e, or 0 before the first tile
  int tiles;
  bool poison;
  int cells;
  float* mine;  // of the offset -reach

  __device__ __forceinline__ void init(int* space, int reach, float* at) {
    cells = 2 * reach + 1;
    hi = space;
    lo = space + cells;
    scale = inverse = 0.0f;
    tiles = 0;
    poison = false;
    mine = at;
    for (int i = threadIdx.x & 63; i < 2 * cells; i += 64) space[i] = 0;
  }
  __device__ __forceinline__ void flush() {
    for (int i = threadIdx.x & 63; i < cells; i += 64) {
      float v = ((float)hi[i] + (float)lo[i] * 0x1p-15f) * inverse;
      if (poison) v = NAN;
      mine[i] += v;
      hi[i] = lo[i] = 0;
    }
    tiles = 0;
  }
  // makes room for a tile of values up to `top`
  __device__ __forceinline__ void prepare(float top) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (!(top <= 3.0e38f)) {
      poison = true;
      top = 0.0f;
    }
    if (tiles == 16 || !(top * scale <= 32768.0f) || (scale == 0.0f && top > 0.0f)) {
      if (scale != 0.0f) flush();
      if (top > 0.0f) {
        int e;
        (void)frexpf(top, &e);  // top < 2^e
        e = max(e, -100);
        scale = ldexpf(1.0f, 15 - e);
        inverse = ldexpf(1.0f, e - 15);
      }
      tiles = 0;
    }
    ++tiles;
  }
  __device__ __forceinline__ void add(int cell, float v) {
    const float y = v * scale, h = rintf(y);
    atomicAdd(hi + cell, (int)h);
    atomicAdd(lo + cell, (int)rintf((y - h) * 32768.0f));
  }
};

// The waves' sums by offset (dd, one array of `cells` a wave and one more) to
// buckets.
template <int NT>
__device__ __forceinline__ void flush_offsets(const AttnArgs& a, float* dd, int cells,
                                              const int32_t* order, const int32_t* first,
                                              float* out) {
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < cells; i += NT) {
    float t = dd[i];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) t += dd[w * cells + i];
    dd[i] = t;
  }
  __syncthreads();
  if (tid < 64) {  // the cells beyond the reach belong to its ends
    float lo = 0.0f, hi = 0.0f;
    for (int i = tid; i <= kAttnSpan; i += 64) {
      lo += dd[i];
      hi += dd[cells - 1 - i];
    }
    lo = mlcg_wave_sum(lo);
    hi = mlcg_wave_sum(hi);
    if (tid == 0) {
      dd[kAttnSpan] = lo;
      dd[cells - 1 - kAttnSpan] = hi;
    }
  }
  __syncthreads();
  // by bucket in the second array (the ends' cells are free now), all loads of
  // the order at once; then 8 lanes a bucket
  const int n = 2 * a.reach + 1;
  float* sorted = dd + cells;
  for (int i = tid; i < n; i += NT) sorted[i] = dd[kAttnSpan + order[i]];
  __syncthreads();
  for (int b = tid >> 3; b < a.buckets; b += NT / 8) {
    const int end = first[b + 1];
    float t = 0.0f;
    for (int i = first[b] + (tid & 7); i < end; i += 8) t += sorted[i];
    t += __shfl_xor(t, 1, 64);
    t += __shfl_xor(t, 2, 64);
    t += __shfl_xor(t, 4, 64);
    if ((tid & 7) == 0) out[b] = t;
  }
}

// floats of a wave's scratch: the diagonals' block or the integers
template <int DP>
__host__ __device__ __forceinline__ int scratch_floats(int reach, bool positions) {
  return positions ? (2 * (2 * reach + 1) + 3) & ~3 : diag_floats<DP>();
}

// In 16 bits, up to this |m|, the sums that dk and dv form a row's logits from
// begin with -(m + log2 l) / c, so that they leave nothing to subtract (rounded
// by 2^-16 there, below a factor's 2^-12).  In 32 bits every step of these sums
// would be rounded at that size (1031 beads of 32 channels: P off by 1.0e-6
// against 2.2e-7), and the products bound the kernel, not the subtraction.
constexpr float kAttnFold = 512.0f;

template <typename T, int DP, int NQ, int NK>
struct DqLds {
  static constexpr int KS = part_rows_bwd<T, DP>() * NK;
  T k[2][KS * DP], v[2][KS * DP];
  float cap[2][KS];
  int kpos[2][KS];
  float rest[4];  // scratch of the waves, ext, dd of the waves
};

// fragments of q and do, an accumulator
template <typename T, int DP>
constexpr int dq_waves() {
  return waves_for(2 * (DP * (int)sizeof(T) / 8) + DP / 2);
}

// dq, delta and the workgroup's part of the table's gradient; lanes are
// queries as in the forward pass.  2 chains of 4099 beads, 8 heads of 64 in
// bf16: 220 us (469 TFLOP/s over three products), vector instructions 39 % of
// the SIMDs' cycles, products 19 %, the diagonals' LDS round trips in the band
// and the waits at the tiles' barrier the rest.  48 chains of up to 268, 8
// heads of 16 in fp32, positions given: 59 us, of which the sums by offset
// about 30 (14 more with the diagonals' block kept beside the integers: two
// workgroups a compute unit instead of three).  4 chains of 1031, 4 heads of 32
// in fp32: 71 us.
template <typename T, int DP, int NQ, int NK, bool VEC, int POS>
__global__ __launch_bounds__(64 * NQ * NK, (dq_waves<T, DP>())) void attn_dq_kernel(
    AttnArgs a, T* __restrict__ dq, AttnRows rows_out, const int32_t* __restrict__ order,
    const int32_t* __restrict__ first, float* __restrict__ dtable_part) {
  constexpr int RT = part_rows_bwd<T, DP>(), N = RT / 32, KS = RT * NK, NW = NQ * NK, NT = 64 * NW;
  using Lds = DqLds<T, DP, NQ, NK>;
  extern __shared__ __align__(16) unsigned char smem[];
  Lds& L = *reinterpret_cast<Lds*>(smem);
  const int R = a.reach, cells = 2 * (R + kAttnSpan) + 1;
  const int sf = scratch_floats<DP>(R, given_positions<POS>(a));
  float* ext = L.rest + NW * sf;
  float* dd = ext + cells;

  const int head = blockIdx.x % a.heads, kv = head / a.group, tile = blockIdx.x / a.heads;
  const int4 t = a.tiles[tile];
  const int lane = threadIdx.x & 63, g = lane >> 5, wave = wave_number();
  const int wq = wave % NQ, wk = wave / NQ;
  const T* kbase = (const T*)a.k + (int64_t)t.x * a.k_row + kv * a.k_head;
  const T* vbase = (const T*)a.v + (int64_t)t.x * a.v_row + kv * a.v_head;
  const uint8_t* keep = a.keep ? a.keep + t.x : nullptr;
  float* part = dtable_part + ((int64_t)head * a.n_tiles + tile) * a.buckets;
  if (lone_key(keep, t.y)) {
    for (int i = threadIdx.x; i < min(kAttnQ * NQ, t.y - t.z) * a.dim; i += NT) {
      const int64_t r = t.x + t.z + i / a.dim;
      const float l = a.lse[(a.heads + head) * a.beads + r];
      dq[(r * a.heads + head) * a.dim + i % a.dim] = (T)(l - l);
    }
    for (int i = threadIdx.x; i < a.buckets; i += NT) part[i] = 0.0f;
    return;
  }
  Stage<T, DP, KS, NT, VEC> ks, vs;
  KeyInfo info;
  ks.init((int)a.k_row, a.dim);
  vs.init((int)a.v_row, a.dim);
  ks.load(kbase, t.y, a.dim);
  vs.load(vbase, t.y, a.dim);
  typename Stage<T, DP, KS, NT, VEC>::Rows absent;
  absent.load(keep, t.y);
  info.template load<POS>(a, t, 0, KS);

  const bool given = given_positions<POS>(a);
  const QueryPlace qi(a, given, t, t.z + kAttnQ * wq);
  const int64_t row = (int64_t)t.x + qi.mine;
  const T* q = (const T*)a.q + row * a.q_row + head * a.q_head;
  const int64_t flat = (row * a.heads + head) * a.dim;
  v8<T> qf[DP / 16], gf[DP / 16];
  float delta = 0.0f;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    qf[k] = load8<T, VEC>(q, 16 * k + 8 * g, qi.ok, a.dim);
    gf[k] = load8<T, VEC>((const T*)a.grad + flat, 16 * k + 8 * g, qi.ok, a.dim);
    const v8<T> of = load8<T, VEC>((const T*)a.out + flat, 16 * k + 8 * g, qi.ok, a.dim);
    v8<T> rf = {};
    if (sizeof(T) == 2 && a.rest)
      rf = load8<T, VEC>((const T*)a.rest + flat, 16 * k + 8 * g, qi.ok, a.dim);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      delta = fmaf((float)gf[k][e], (float)of[e] + (float)rf[e], delta);
  }
  delta += other_half(delta);
  const float m = qi.ok ? a.lse[head * a.beads + row] : INFINITY;
  const float l = qi.ok ? a.lse[(a.heads + head) * a.beads + row] : 0.0f;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l, delta_inv = delta * inv;
  const bool any_far = __any(far_shift<T>(m));
  fill_bias<T>(a, head, t.y, given, ext);
  for (int i = threadIdx.x; i < NW * cells; i += NT) dd[i] = 0.0f;
  float* mine = dd + wave * cells;
  float* scratch = L.rest + wave * sf;
  OffsetInts ints;
  if (given)
    ints.init(reinterpret_cast<int*>(scratch), R, mine + kAttnSpan);
  else
    for (int i = lane; i < diag_floats<DP>(); i += 64) scratch[i] = 0.0f;
  float far_lo = 0.0f, far_hi = 0.0f;
  f32x16 acc[DP / 32] = {};
  OperandScale<T> up;
  int buf = 0;
  // puts the tile of k0 into LDS and sends for the next one
  auto next_tile = [&](int k0) {
    if (keep || k0 + KS > t.y) {
      ks.drop(absent);
      vs.drop(absent);
    }
    ks.put(L.k[buf]);
    vs.put(L.v[buf]);
    info.template put<POS>(a, KS, qi.lo, L.cap[buf], L.kpos[buf]);
    const int kn = k0 + KS;
    if (kn < t.y) {
      ks.load(kbase + kn * a.k_row, t.y - kn, a.dim);
      vs.load(vbase + kn * a.v_row, t.y - kn, a.dim);
      if (keep || kn + KS > t.y) absent.load(keep ? keep + kn : keep, t.y - kn);
      info.template load<POS>(a, t, kn, KS);
    }
    __syncthreads();
  };
  if (qi.first >= t.y)  // no queries: this wave only loads
    for (int k0 = 0; k0 < t.y; k0 += KS, buf ^= 1) next_tile(k0);
  else for (int k0 = 0; k0 < t.y; k0 += KS, buf ^= 1) {
    next_tile(k0);
    const int kb = k0 + RT * wk;
    if (kb >= t.y) continue;
    const T* kt = L.k[buf] + RT * wk * DP;
    const float* cap = L.cap[buf] + RT * wk;
    const int* kpos = L.kpos[buf] + RT * wk;
    f32x16 s[N];
    load_rows<N>(cap, s);
    row_product<T, DP, N>(kt, qf, a.dim, s);
    float x[16 * N];
    const int side = query_logits<T, N, POS>(a, s, ext, cap, kpos, kb, qi, m, any_far, x);
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = f32x16{};
    row_product<T, DP, N>(L.v[buf] + RT * wk * DP, gf, a.dim, s);  // dP
#pragma unroll
    for (int i = 0; i < 16 * N; ++i)
      x[i] = __builtin_amdgcn_exp2f(x[i]) * fmaf(s[i / 16][i % 16], inv, -delta_inv);
    if (side) {
      float sum[4] = {};
#pragma unroll
      for (int i = 0; i < 16 * N; ++i) sum[i % 4] += x[i];
      const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if (side > 0)
        far_hi += all;
      else
        far_lo += all;
    } else if (!given) {
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (kb + 32 * n < t.y)
          add_diagonals<DP>(x + 16 * n, scratch,
                            mine + (kb + 32 * n - qi.first + R + kAttnSpan));
    } else {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 16 * N; ++i) top = fmaxf(top, fabsf(x[i]));
      // NaN does not survive the maximum
#pragma unroll
      for (int i = 0; i < 16 * N; ++i) top = x[i] != x[i] ? INFINITY : top;
      ints.prepare(top);
      // beads of one residue follow each other: one sum for equal neighbours (48
      // chains of up to 268 beads, 2.5 to a residue, 8 heads of 16: about 18 us
      // less)
#pragma unroll
      for (int i = 0; i < 16 * N; i += 4) {
        const int4 p = *reinterpret_cast<const int4*>(kpos + acc_row(i, g));
        const int pc[4] = {p.x, p.y, p.z, p.w};
        float run = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          run += x[i + c];
          if (c == 3 || pc[c] != pc[c + 1]) {
            ints.add(offset_cell(pc[c], qi.pos, R) - kAttnSpan, run);
            run = 0.0f;
          }
        }
      }
    }
    up.fit(x, acc);
    column_product<T, DP, N>(kt, x, acc);
  }
  if (given) ints.flush();
  far_lo = mlcg_wave_sum(far_lo);
  far_hi = mlcg_wave_sum(far_hi);
  if (lane == 0) {
    mine[0] += far_lo;
    mine[cells - 1] += far_hi;
  }
  up.template join<NQ, NK>(acc, reinterpret_cast<float*>(smem));
  join_parts<DP, NQ, NK>(acc, reinterpret_cast<float*>(smem));
  if (qi.ok && wk == 0) {
    store_column<T, DP, VEC>(dq + flat, acc, a.scale * up.undo(), a.dim);
    if (g == 0) {
      rows_out.delta[head * a.beads + row] = delta;
      if constexpr (sizeof(T) == 2) {  // -inf logits for a row without keys
        const float sum = l == 0.0f ? -INFINITY : -(m + __builtin_amdgcn_logf(l));
        rows_out.start[head * a.beads + row] = sum / logit_factor(a);
      }
    }
  }
  if (wk == 0) {
    const bool any = __any(fabsf(m) >= kAttnFold && m < INFINITY);
    if (lane == 0)
      rows_out.apart[((int64_t)head * a.n_tiles + tile) * NQ + wq] = any ? 1.0f : 0.0f;
  }
  flush_offsets<NT>(a, dd, cells, order, first, part);
}

template <typename T, int DP, int NQ, int NK>
struct DkvLds {
  static constexpr int KS = part_rows_bwd<T, DP>() * NK;
  T q[2][KS * DP], g[2][KS * DP];
  float start[2][KS];             // of the sums, or
  float m[2][KS], inv[2][KS];     // m and 1 / l
  float delta[2][KS];
  int qpos[2][KS];
  float ext[1];
};

// fragments of k and v and two accumulators
template <typename T, int DP>
constexpr int dkv_waves() {
  return waves_for(2 * (DP * (int)sizeof(T) / 8) + DP);
}

// dk and dv; lanes are keys, the tiles hold queries.  The query heads that
// share a key/value head are taken one after the other, so their gradients are
// summed in one wave's registers, in order.  2 chains of 4099 beads, 8 heads
// of 64 in bf16: 209 us (658 TFLOP/s over four products), products 27 % of
// the SIMDs' cycles, vector instructions 31 %; two waves a SIMD (128 fragments
// and accumulators a lane) do not cover the LDS reads between them.  4 chains
// of 1031, 4 heads of 32 in fp32: 80 us (54 TFLOP/s; 144 workgroups).
template <typename T, int DP, int NQ, int NK, bool VEC, int POS>
__global__ __launch_bounds__(64 * NQ * NK, (dkv_waves<T, DP>())) void attn_dkv_kernel(
    AttnArgs a, AttnRows rows_in, T* __restrict__ dk, T* __restrict__ dv) {
  constexpr int RT = part_rows_bwd<T, DP>(), N = RT / 32, KS = RT * NK, NT = 64 * NQ * NK;
  using Lds = DkvLds<T, DP, NQ, NK>;
  extern __shared__ __align__(16) unsigned char smem[];
  Lds& L = *reinterpret_cast<Lds*>(smem);
  float* ext = L.ext;

  const int kv_heads = a.heads / a.group;
  const int kv = blockIdx.x % kv_heads;
  const int tile = blockIdx.x / kv_heads;
  const int4 t = a.tiles[tile];
  const int lane = threadIdx.x & 63, g = lane >> 5, wave = wave_number();
  const int wq = wave % NQ, wk = wave / NQ;
  const int kw = t.z + kAttnQ * wq, ki = kw + (lane & 31);
  const int64_t row = (int64_t)t.x + ki;
  const bool in = ki < t.y, k_ok = in && (!a.keep || a.keep[row]);
  if (lone_key(a.keep ? a.keep + t.x : nullptr, t.y)) {
    for (int i = threadIdx.x; i < min(kAttnQ * NQ, t.y - t.z) * a.dim; i += NT) {
      const int64_t r = t.x + t.z + i / a.dim;
      const int d = i % a.dim;
      float sum = 0.0f, zero = 0.0f;
      if (!a.keep || a.keep[r])
        for (int j = 0; j < t.y; ++j)
          for (int h = 0; h < a.group; ++h) {
            const int head = kv * a.group + h;
            const float l = a.lse[(a.heads + head) * a.beads + t.x + j];
            zero += l - l;
            if (l != 0.0f)
              sum += (float)((const T*)a.grad)[((int64_t)(t.x + j) * a.heads + head) * a.dim + d];
          }
      dk[(r * kv_heads + kv) * a.dim + d] = (T)zero;
      dv[(r * kv_heads + kv) * a.dim + d] = (T)(sum + zero);
    }
    return;
  }
  // the sums of dP begin with -delta
  const float c = logit_factor(a);
  const int R = a.reach;

  Stage<T, DP, KS, NT, VEC> qs, gs;
  qs.init((int)a.q_row, a.dim);
  gs.init(a.heads * a.dim, a.dim);
  typename Stage<T, DP, KS, NT, VEC>::Rows absent;
  const bool given = given_positions<POS>(a);
  float start_n = 0.0f, m_n = 0.0f, l_n = 0.0f, delta_n = 0.0f;
  int pos_n = 0;
  auto load = [&](int head, int q0, bool folded, bool apart) {
    const int64_t row0 = (int64_t)t.x + q0;
    qs.load((const T*)a.q + row0 * a.q_row + head * a.q_head, t.y - q0, a.dim);
    gs.load((const T*)a.grad + (row0 * a.heads + head) * a.dim, t.y - q0, a.dim);
    if (q0 + KS > t.y) absent.load(nullptr, t.y - q0);
    const int i = threadIdx.x;
    // exp2(-inf) = 0 for the rows past the end
    start_n = c > 0.0f ? -INFINITY : INFINITY;
    m_n = INFINITY;
    l_n = delta_n = 0.0f;
    if (i < KS && q0 + i < t.y) {
      const int64_t at = head * a.beads + row0 + i;
      if (folded) start_n = rows_in.start[at];
      if (apart) {
        m_n = a.lse[at];
        l_n = a.lse[a.heads * a.beads + at];
      }
      delta_n = rows_in.delta[at];
      if (given) pos_n = a.pos[row0 + i];
    }
  };
  load(kv * a.group, 0, sizeof(T) == 2, true);
  // any large m among the chain's queries of these heads
  float large = 0.0f;
  for (int h = 0; h < a.group; ++h) {
    const int64_t at = (int64_t)(kv * a.group + h) * a.n_tiles + tile - t.z / (kAttnQ * NQ);
    for (int i = lane; i < (t.y + kAttnQ - 1) / kAttnQ; i += 64)
      large = fmaxf(large, rows_in.apart[at * NQ + i]);
  }

  const T* k = (const T*)a.k + row * a.k_row + kv * a.k_head;
  const T* v = (const T*)a.v + row * a.v_row + kv * a.v_head;
  v8<T> kf[DP / 16], vf[DP / 16];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i) {
    kf[i] = load8<T, VEC>(k, 16 * i + 8 * g, k_ok, a.dim);
    vf[i] = load8<T, VEC>(v, 16 * i + 8 * g, k_ok, a.dim);
  }
  int kp = 0, klo = 0, khi = 0;
  if (given) {
    kp = a.pos[(int64_t)t.x + min(ki, t.y - 1)];
    klo = wave_min(kp);
    khi = wave_max(kp);
  }

  f32x16 dka[DP / 32] = {}, dva[DP / 32] = {};
  OperandScale<T> up;
  int buf = 0;
  // FOLD: sums that begin with start.  FAR: some m may be far_shift's.
  auto all_queries = [&](auto fold, auto far) {
    constexpr bool FOLD = decltype(fold)::value, FAR = decltype(far)::value;
    // puts the tile of q0 into LDS and sends for the next one
    auto next_tile = [&](int h, int q0) {
      if (q0 + KS > t.y) {
        qs.drop(absent);
        gs.drop(absent);
      }
      qs.put(L.q[buf]);
      gs.put(L.g[buf]);
      if ((int)threadIdx.x < KS) {
        if (FOLD) {
          L.start[buf][threadIdx.x] = start_n;
        } else {
          L.m[buf][threadIdx.x] = m_n;
          L.inv[buf][threadIdx.x] = l_n == 0.0f ? 0.0f : 1.0f / l_n;
        }
        L.delta[buf][threadIdx.x] = -delta_n;
        // past the end a bead's of the chain, so that the offsets are pairs'
        if (POS != kIndex) L.qpos[buf][threadIdx.x] = q0 + (int)threadIdx.x < t.y ? pos_n : klo;
      }
      if (q0 + KS < t.y)
        load(kv * a.group + h, q0 + KS, FOLD, !FOLD);
      else if (h + 1 < a.group)
        load(kv * a.group + h + 1, 0, FOLD, !FOLD);
      __syncthreads();
    };
    for (int h = 0; h < a.group; ++h) {
      const int head = kv * a.group + h;
      if (h > 0) __syncthreads();
      fill_bias<T>(a, head, t.y, given, ext);
      if (kw >= t.y)  // no keys: this wave only loads
        for (int q0 = 0; q0 < t.y; q0 += KS, buf ^= 1) next_tile(h, q0);
      else for (int q0 = 0; q0 < t.y; q0 += KS, buf ^= 1) {
        next_tile(h, q0);
        const int qb = q0 + RT * wk;
        if (qb >= t.y) continue;
        const T* qt = L.q[buf] + RT * wk * DP;
        const T* gt = L.g[buf] + RT * wk * DP;
        const int* qpos = L.qpos[buf] + RT * wk;
        const float* mrow = L.m[buf] + RT * wk;
        f32x16 s[N] = {};
        if constexpr (FOLD) load_rows<N>(L.start[buf] + RT * wk, s);
        row_product<T, DP, N>(qt, kf, a.dim, s);
        float x[16 * N];
        // from the bias of row i
        auto logits = [&](auto bias) {
          if constexpr (FOLD) {
#pragma unroll
            for (int i = 0; i < 16 * N; ++i) x[i] = fmaf(s[i / 16][i % 16], c, bias(i));
          } else {
#pragma unroll
            for (int i = 0; i < 16 * N; ++i) {
              const float m = mrow[acc_row(i, g)], b = bias(i);
              x[i] = FAR && far_shift<T>(m) ? fmaf(s[i / 16][i % 16], c, b) - m
                                            : fmaf(s[i / 16][i % 16], c, b - m);
            }
          }
        };
        int side;
        if (given) {
          const int qp = qpos[lane % RT];
          const bool past = qb + lane % RT >= t.y;
          side = __all(past || __builtin_elementwise_sub_sat(klo, qp) >= R)    ? 1
                 : __all(past || __builtin_elementwise_sub_sat(khi, qp) <= -R) ? -1
                                                                               : 0;
        } else {
          side = block_side(kw - (qb + RT - 1), kw + 31 - qb, R);
        }
        if (side) {
          const float b = ext[side > 0 ? 2 * R + kAttnSpan : kAttnSpan];
          logits([=](int) { return b; });
        } else if (given) {
          logits([=](int i) { return ext[offset_cell(kp, qpos[acc_row(i, g)], R)]; });
        } else {
          const float* e = ext + (ki - qb - 4 * g + R + kAttnSpan);
          logits([=](int i) { return e[-acc_row(i, 0)]; });
        }
        load_rows<N>(L.delta[buf] + RT * wk, s);
        row_product<T, DP, N>(gt, vf, a.dim, s);  // dP - delta
#pragma unroll
        for (int i = 0; i < 16 * N; ++i) x[i] = __builtin_amdgcn_exp2f(x[i]);
        if constexpr (!FOLD) {
#pragma unroll
          for (int i = 0; i < 16 * N; ++i) x[i] *= L.inv[buf][RT * wk + acc_row(i, g)];
        }
        column_product<T, DP, N>(gt, x, dva);
#pragma unroll
        for (int i = 0; i < 16 * N; ++i) x[i] *= s[i / 16][i % 16];
        up.fit(x, dka);
        column_product<T, DP, N>(qt, x, dka);
      }
    }
  };
  if (__any(large != 0.0f))
    all_queries(std::false_type(), std::true_type());
  else
    all_queries(std::bool_constant<sizeof(T) == 2>(), std::false_type());
  up.template join<NQ, NK>(dka, reinterpret_cast<float*>(smem));
  join_parts<DP, NQ, NK>(dka, reinterpret_cast<float*>(smem));
  join_parts<DP, NQ, NK>(dva, reinterpret_cast<float*>(smem));
  if (!in || wk > 0) return;
  const int64_t flat = (row * kv_heads + kv) * a.dim;
  if (!k_ok) {  // an absent key takes part in nothing
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) dka[n] = dva[n] = f32x16{};
  }
  store_column<T, DP, VEC>(dk + flat, dka, a.scale * up.undo(), a.dim);
  store_column<T, DP, VEC>(dv + flat, dva, 1.0f, a.dim);
}

// dtable[b][head] = sum of the workgroups' parts [head][tile][b]: 8 buckets x
// 32 slices of the tiles a workgroup, joined in order.  5 us, a launch's own
// latency; a last workgroup that joins them would need an ordered counter.
template <typename T>
__global__ __launch_bounds__(256) void attn_dtable_kernel(const float* __restrict__ part,
                                                          int n_tiles, int buckets, int heads,
                                                          T* __restrict__ dtable) {
  __shared__ float red[32][9];
  const int b = blockIdx.x * 8 + (threadIdx.x & 7), slice = threadIdx.x >> 3, head = blockIdx.y;
  float s = 0.0f;
  if (b < buckets)
    for (int i = slice; i < n_tiles; i += 32)
      s += part[((int64_t)head * n_tiles + i) * buckets + b];
  red[slice][threadIdx.x & 7] = s;
  __syncthreads();
  if (slice == 0 && b < buckets) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += red[i][threadIdx.x];
    dtable[(int64_t)b * heads + head] = (T)t;
  }
}

// LDS above 64 KiB has to be asked for.
int allow_lds(const void* f, unsigned bytes) {
  if (bytes > 163840u) return MLCG_ERR_UNSUPPORTED;
  if (bytes <= 65536u) return MLCG_OK;
  return hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) ==
                 hipSuccess
             ? MLCG_OK
             : MLCG_ERR_LAUNCH;
}

template <typename T, int DP, int NQ, int NK, bool VEC, int POS>
int launch_fwd(const AttnArgs& a, void* out, hipStream_t s) {
  const unsigned cells = 2 * (a.reach + kAttnSpan) + 1;
  const unsigned lds = sizeof(FwdLds<T, DP, NQ, NK>) + 4 * cells;
  auto f = attn_fwd_kernel<T, DP, NQ, NK, VEC, POS>;
  if (int e = allow_lds(reinterpret_cast<const void*>(f), lds)) return e;
  hipLaunchKernelGGL(f, dim3((unsigned)(a.n_tiles * a.heads)), dim3(64 * NQ * NK), lds, s, a,
                     (T*)out);
  return mlcg_launch_status();
}

template <typename T, int DP, int NQ, int NK, bool VEC, int POS>
int launch_dq(const AttnArgs& a, const AttnGrads& o, const AttnRows& rows, float* part,
              hipStream_t s) {
  constexpr unsigned NW = NQ * NK;
  const unsigned cells = 2 * (a.reach + kAttnSpan) + 1;
  const unsigned lds = sizeof(DqLds<T, DP, NQ, NK>) +
                       4 * (NW * scratch_floats<DP>(a.reach, a.pos != nullptr) + (NW + 2) * cells);
  auto f = attn_dq_kernel<T, DP, NQ, NK, VEC, POS>;
  if (int e = allow_lds(reinterpret_cast<const void*>(f), lds)) return e;
  hipLaunchKernelGGL(f, dim3((unsigned)(a.n_tiles * a.heads)), dim3(64 * NW), lds, s, a,
                     (T*)o.dq, rows, o.order, o.first, part);
  return mlcg_launch_status();
}

template <typename T, int DP, int NQ, int NK, bool VEC, int POS>
int launch_dkv(const AttnArgs& a, const AttnGrads& o, const AttnRows& rows, hipStream_t s) {
  const unsigned cells = 2 * (a.reach + kAttnSpan) + 1;
  const unsigned lds = sizeof(DkvLds<T, DP, NQ, NK>) + 4 * cells;
  auto f = attn_dkv_kernel<T, DP, NQ, NK, VEC, POS>;
  if (int e = allow_lds(reinterpret_cast<const void*>(f), lds)) return e;
  hipLaunchKernelGGL(f, dim3((unsigned)(a.n_tiles * (a.heads / a.group))), dim3(64 * NQ * NK), lds,
                     s, a, rows, (T*)o.dk, (T*)o.dv);
  return mlcg_launch_status();
}

// 16-byte loads and stores: every row and head starts at a multiple of them
bool attn_vec(const AttnArgs& a, int size) {
  const void* p[] = {a.q, a.k, a.v, a.out, a.grad, a.rest};
  for (const void* x : p)
    if (!chain_aligned16(x)) return false;
  const int64_t st[] = {a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head, a.dim};
  for (int64_t x : st)
    if (x * size % 16) return false;
  return true;
}

// four parts: of the forward pass alone (the backward's tiles and sums by
// offset of eight waves would not fit the LDS)
template <int size_of, bool FORWARD, typename F>
int by_shape(const AttnArgs& a, int shape, F f) {
  using std::integral_constant;
  using One = integral_constant<int, 1>;
  using Two = integral_constant<int, 2>;
  using Four = integral_constant<int, 4>;
  auto with = [&](auto dp, auto vec, auto pos) {
    constexpr bool split = decltype(dp)::value <= 64;
    const int nk = split ? shape % 10 : 1, nq = shape / 10;
    if constexpr (split && FORWARD)
      if (nk == 4) return f(dp, Two(), Four(), vec, pos);
    if (nk == 2) {
      if constexpr (split) {
        if (nq == 2) return f(dp, Two(), Two(), vec, pos);
        if (nq == 4) return f(dp, Four(), Two(), vec, pos);
      }
    }
    if (nq == 1) return f(dp, One(), One(), vec, pos);
    if (nq == 2) return f(dp, Two(), One(), vec, pos);
    return f(dp, Four(), One(), vec, pos);
  };
  auto either = [&](auto dp) {
    using std::bool_constant;
    if (!attn_vec(a, size_of))
      return with(dp, bool_constant<false>(), integral_constant<int, kEither>());
    return a.pos ? with(dp, bool_constant<true>(), integral_constant<int, kGiven>())
                 : with(dp, bool_constant<true>(), integral_constant<int, kIndex>());
  };
  if (a.dim <= 32) return either(integral_constant<int, 32>());
  if (a.dim <= 64) return either(integral_constant<int, 64>());
  return either(integral_constant<int, 128>());
}

}  // namespace

template <>
int attn_forward<MLCG_ATTENTION_TYPE>(AttnArgs a, int shape, void* out, hipStream_t s) {
  using T = MLCG_ATTENTION_TYPE;
  return by_shape<(int)sizeof(T), true>(a, shape, [&](auto dp, auto nq, auto nk, auto vec,
                                                       auto pos) {
    return launch_fwd<T, decltype(dp)::value, decltype(nq)::value, decltype(nk)::value,
                      decltype(vec)::value, decltype(pos)::value>(a, out, s);
  });
}

template <>
int attn_backward<MLCG_ATTENTION_TYPE>(AttnArgs a, int shape, const AttnGrads& o, hipStream_t s) {
  using T = MLCG_ATTENTION_TYPE;
  const int64_t n = a.heads * a.beads, tiles = (int64_t)a.heads * a.n_tiles;
  const AttnRows rows{o.ws, o.ws + n, o.ws + 2 * n};
  float* part = rows.apart + kAttnWaves * tiles;
  if (int e = by_shape<(int)sizeof(T), false>(a, shape, [&](auto dp, auto nq, auto nk, auto vec,
                                                            auto pos) {
        return launch_dq<T, decltype(dp)::value, decltype(nq)::value, decltype(nk)::value,
                         decltype(vec)::value, decltype(pos)::value>(a, o, rows, part, s);
      }))
    return e;
  // keys of shared heads give fewer workgroups than queries: where they are no
  // more than the compute units, two waves share a block of keys (8191 beads,
  // 8 heads on 2 key heads in bf16: both passes 735 us against 1009)
  const int64_t groups = (int64_t)a.n_tiles * (a.heads / a.group);
  const int kv_shape = shape >= 20 && groups <= 256 ? shape / 10 * 10 + 2 : shape;
  if (int e = by_shape<(int)sizeof(T), false>(a, kv_shape, [&](auto dp, auto nq, auto nk,
                                                               auto vec, auto pos) {
        return launch_dkv<T, decltype(dp)::value, decltype(nq)::value, decltype(nk)::value,
                          decltype(vec)::value, decltype(pos)::value>(a, o, rows, s);
      }))
    return e;
  hipLaunchKernelGGL(attn_dtable_kernel<T>, dim3(mlcg_div_up(a.buckets, 8), a.heads), dim3(256), 0,
                     s, part, a.n_tiles, a.buckets, a.heads, (T*)o.dtable);
  return mlcg_launch_status();
}

#endif  // MLCG_ATTENTION_TYPE
