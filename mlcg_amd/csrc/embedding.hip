// Embedding lookup with a factor, and its gradient by sorted tokens (gfx950):
//   y_n = s T[tok_n],   dT_v = s sum over n with tok_n = v of dy_n.
//
// The rows' order by token (stable: rows of one token stay in order) comes from
// a radix sort, 8 bits of the token a pass, of three kernels: how many of each
// digit a block of rows has; for every digit, by a workgroup of its own, the
// exclusive sum over the blocks; every row to its place, ranked in its block by
// ballots, after the digits before it.
//
// The gradient: slabs of the ordered rows, a row's channels over 8 to 64 lanes.
// Runs of one token that begin and end in a slab are done there; of a longer one
// every slab leaves its sum, which a workgroup at the run's first slab adds in
// order.  No floating-point atomics: equal calls give equal bits.
//
// Both are bound by memory where there are many rows, by the latency of their
// launches where there are few.  548864 rows of 256 channels in bf16, 8000 tokens:
// the look-up 70 us (4.1 TB/s, nearly all of it written); the order 45 us in two
// passes; the sums 118 us, of which the gradient's 281 MB are 58 at a copy's rate:
// rows are read in the tokens' order, 512 bytes at a time.  17920 rows of 128 in
// fp32, 25 tokens: 6 us, 14 us and 17 us.
#include <type_traits>

#include "chain.h"

namespace {

constexpr int kEmbThreads = 256;
constexpr int kEmbWaves = kEmbThreads / MLCG_WAVE;
constexpr int kSortItems = 8;                           // a lane
constexpr int kSortRows = kEmbThreads * kSortItems;     // a block
constexpr int kEmbRows = 4;                             // rows of a lane in the look-up
constexpr int kEmbMaxWidth = 8192;

// kEmbRows rows over `lanes` lanes; a token outside the table gives zeros and a flag.
template <typename T>
__global__ __launch_bounds__(kEmbThreads) void embedding_forward(
    const T* __restrict__ table, int rows, const int64_t* __restrict__ tokens, int64_t n, int width,
    int lanes, float scale, T* __restrict__ out, unsigned* __restrict__ flags) {
  const int per = kEmbThreads / lanes, l = threadIdx.x % lanes;
  const int64_t i0 = (chain_group() * per + threadIdx.x / lanes) * kEmbRows;
  int64_t tok[kEmbRows];
  bool ok[kEmbRows], bad = false;
#pragma unroll
  for (int r = 0; r < kEmbRows; ++r) {
    tok[r] = i0 + r < n ? tokens[i0 + r] : 0;
    ok[r] = tok[r] >= 0 && tok[r] < rows;
    bad = bad || !ok[r];
    if (!ok[r]) tok[r] = 0;
  }
  if (bad && l == 0) atomicOr(flags, kFlagTypeRange);
  for (int el = 8 * l; el < width; el += 8 * lanes) {
    f32x8 x[kEmbRows];
#pragma unroll
    for (int r = 0; r < kEmbRows; ++r) x[r] = load_row8<T>(table + tok[r] * width, el, width);
#pragma unroll
    for (int r = 0; r < kEmbRows; ++r)
      if (i0 + r < n)
        store_row8<T>(out + (i0 + r) * width, el, width, ok[r] ? x[r] * scale : f32x8{});
  }
}

// ---------------------------------------------------------------------------
// order by token

// the key of row i in the first pass: its token, or `rows` outside the table
__device__ __forceinline__ int token_key(const int64_t* tokens, const int* keys, int64_t i,
                                         int rows) {
  if (keys) return keys[i];
  const int64_t t = tokens[i];
  return t < 0 || t >= rows ? rows : (int)t;
}

__global__ __launch_bounds__(kEmbThreads) void sort_count(const int64_t* __restrict__ tokens,
                                                          const int* __restrict__ keys, int64_t n,
                                                          int rows, int shift, int blocks,
                                                          int* __restrict__ counts,
                                                          unsigned* __restrict__ flags) {
  __shared__ int hist[256];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortRows;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * kEmbThreads + threadIdx.x;
    if (i >= n) continue;
    const int key = token_key(tokens, keys, i, rows);
    bad = bad || key == rows;
    atomicAdd(&hist[(key >> shift) & 255], 1);  // whole numbers: any order
  }
  if (bad && !keys) atomicOr(flags, kFlagTypeRange);
  __syncthreads();
  counts[(int64_t)threadIdx.x * blocks + blockIdx.x] = hist[threadIdx.x];
}

// The exclusive sum of a digit's counts over the blocks, in place, and its total.
__global__ __launch_bounds__(kEmbThreads) void sort_scan(int* __restrict__ counts, int blocks,
                                                         int* __restrict__ totals) {
  __shared__ int sums[kEmbWaves];
  constexpr int kItems = 4;
  int* const row = counts + (int64_t)blockIdx.x * blocks;
  int carry = 0;
  const int l = mlcg_lane(), w = threadIdx.x / MLCG_WAVE;
  for (int b = 0; b < blocks; b += kEmbThreads * kItems) {
    int v[kItems], own = 0;
    const int at = b + threadIdx.x * kItems;
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      v[j] = at + j < blocks ? row[at + j] : 0;
      own += v[j];
    }
    int s = own;
#pragma unroll
    for (int o = 1; o < MLCG_WAVE; o <<= 1) {
      const int up = __shfl_up(s, o, MLCG_WAVE);
      if (l >= o) s += up;
    }
    if (l == MLCG_WAVE - 1) sums[w] = s;
    __syncthreads();
    int before = carry + s - own;
#pragma unroll
    for (int j = 0; j < kEmbWaves; ++j) {
      if (j < w) before += sums[j];
      carry += sums[j];
    }
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      if (at + j < blocks) row[at + j] = before;
      before += v[j];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// A wave has kSortItems x 64 rows in a row.
__global__ __launch_bounds__(kEmbThreads) void sort_place(
    const int64_t* __restrict__ tokens, const int* __restrict__ keys,
    const int* __restrict__ index, int64_t n, int rows, int shift, int blocks,
    const int* __restrict__ counts, const int* __restrict__ totals, int* __restrict__ keys_out,
    int* __restrict__ index_out) {
  __shared__ int seen[kEmbWaves][256];
  __shared__ int sums[kEmbWaves];
  const int l = mlcg_lane(), w = threadIdx.x / MLCG_WAVE;
  for (int i = l; i < 256; i += MLCG_WAVE) seen[w][i] = 0;
  const uint64_t below = l == 0 ? 0ull : ~0ull >> (MLCG_WAVE - l);
  const int64_t base = (int64_t)blockIdx.x * kSortRows + w * (kSortItems * MLCG_WAVE) + l;
  int key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * MLCG_WAVE;
    key[j] = i < n ? token_key(tokens, keys, i, rows) : -1;
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const bool in = key[j] >= 0;
    const int d = (key[j] >> shift) & 255;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t m = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? m : ~m;
    }
    // rows of one digit in this step: the first of them moves the count on
    int before = 0;
    if (in) before = seen[w][d];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && (same & below) == 0) seen[w][d] = before + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    rank[j] = before + __popcll(same & below);
  }
  // rows of the digits before this thread's
  const int own = totals[threadIdx.x];
  int s = own;
#pragma unroll
  for (int o = 1; o < MLCG_WAVE; o <<= 1) {
    const int up = __shfl_up(s, o, MLCG_WAVE);
    if (l >= o) s += up;
  }
  if (l == MLCG_WAVE - 1) sums[w] = s;
  __syncthreads();
  {
    int at = counts[(int64_t)threadIdx.x * blocks + blockIdx.x] + s - own;
#pragma unroll
    for (int v = 0; v < kEmbWaves; ++v)
      if (v < w) at += sums[v];
#pragma unroll
    for (int v = 0; v < kEmbWaves; ++v) {
      const int c = seen[v][threadIdx.x];
      seen[v][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    if (key[j] < 0) continue;
    const int64_t i = base + j * MLCG_WAVE;
    const int at = seen[w][(key[j] >> shift) & 255] + rank[j];
    keys_out[at] = key[j];
    index_out[at] = index ? index[i] : (int)i;
  }
}

// ---------------------------------------------------------------------------
// sums of the ordered rows

template <typename T>
__global__ __launch_bounds__(kEmbThreads) void embedding_zero(T* __restrict__ out, int64_t n) {
  typedef T chunk __attribute__((ext_vector_type(16 / sizeof(T))));
  constexpr int per = 16 / sizeof(T);
  const int64_t step = (int64_t)gridDim.x * kEmbThreads;
  int64_t i = (int64_t)blockIdx.x * kEmbThreads + threadIdx.x;
  const int64_t whole = n / per;  // a tensor of its own: 16-byte aligned
  for (int64_t c = i; c < whole; c += step) reinterpret_cast<chunk*>(out)[c] = chunk{};
  for (int64_t e = whole * per + i; e < n; e += step) out[e] = (T)0.0f;
}

// A slab's rows over `lanes` lanes and, on the grid's second axis, 8 lanes
// channels each.  head[slab]: the sum of the rows of the run that comes from
// before; tail[slab]: of the run that goes on behind and begins here.  The slabs'
// keys and rows come to LDS first, so that the loads of rows wait for none.
template <typename T, int SLAB>
__global__ __launch_bounds__(kEmbThreads) void embedding_slab(
    const T* __restrict__ grad, const int* __restrict__ keys, const int* __restrict__ index,
    int64_t n, int rows, int width, int lanes, float scale, T* __restrict__ out,
    float* __restrict__ head, float* __restrict__ tail) {
  constexpr int kBatch = 8, kMost = kEmbThreads / 8 * SLAB;
  __shared__ int key_of[kMost + 1], row_of[kMost];
  const int per = kEmbThreads / lanes, l = threadIdx.x % lanes, p = threadIdx.x / lanes;
  const int64_t base = chain_group() * per * SLAB;
  for (int i = threadIdx.x; i <= per * SLAB; i += kEmbThreads) {
    key_of[i] = base + i < n ? keys[base + i] : -1;
    if (i < per * SLAB) row_of[i] = base + i < n ? index[base + i] : 0;
  }
  __syncthreads();
  const int64_t slab = chain_group() * per + p, begin = slab * SLAB;
  const int el = 8 * (blockIdx.y * lanes + l);
  if (begin >= n || el >= width) return;
  const int count = (int)min((int64_t)SLAB, n - begin);
  const int* const key = key_of + p * SLAB;
  const int* const row = row_of + p * SLAB;
  // the run comes from the slab before
  bool first = begin > 0 && keys[begin - 1] == key[0];
  f32x8 s{};
  for (int r0 = 0; r0 < count; r0 += kBatch) {
    f32x8 x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      x[j] = load_row8<T>(grad + (int64_t)row[min(r0 + j, count - 1)] * width, el, width);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (r0 + j >= count) break;
      s += x[j];
      const int k = key[r0 + j], next = key[r0 + j + 1];  // -1 behind the last row
      const bool last = r0 + j + 1 == count;
      if (k == next && !last) continue;
      if (first) {
        store_row8<float>(head + slab * width, el, width, s);
      } else if (k == next) {
        store_row8<float>(tail + slab * width, el, width, s);
      } else if (k < rows) {
        store_row8<T>(out + (int64_t)k * width, el, width, s * scale);
      }
      first = false;
      s = f32x8{};
    }
  }
}

// Runs over several slabs: the workgroup of the slab that one begins in.
template <typename T, int SLAB>
__global__ __launch_bounds__(kEmbThreads) void embedding_join(
    const int* __restrict__ keys, int64_t n, int rows, int width, int lanes, float scale,
    const float* __restrict__ head, const float* __restrict__ tail, T* __restrict__ out) {
  const int64_t slab = chain_group(), slabs = (n + SLAB - 1) / SLAB;
  const int64_t end = slab * SLAB + SLAB;
  if (end >= n) return;
  const int key = keys[end - 1];
  if (key >= rows || keys[end] != key) return;  // ends here
  // begins here, not before this slab
  const int64_t begin = slab * SLAB;
  if (begin > 0 && keys[begin] == key && keys[begin - 1] == key) return;
  __shared__ int stop;
  __shared__ float sum[kEmbThreads * 8];
  int64_t last = slab + 1;  // the last slab that the run reaches
  for (int64_t s0 = slab + 2;; s0 += kEmbThreads) {
    if (threadIdx.x == 0) stop = kEmbThreads;
    __syncthreads();
    const int64_t s = s0 + threadIdx.x;
    if (s >= slabs || keys[s * SLAB] != key) atomicMin(&stop, (int)threadIdx.x);
    __syncthreads();
    const int more = stop;
    __syncthreads();
    last += more;
    if (more < kEmbThreads) break;
  }
  // equal parts of the slabs to the groups of lanes
  const int per = kEmbThreads / lanes, p = threadIdx.x / lanes, l = threadIdx.x % lanes;
  const int64_t share = (last - slab + per - 1) / per;
  const int64_t a = slab + 1 + p * share, b = min(a + share, last + 1);
  const int el = 8 * (blockIdx.y * lanes + l);
  f32x8 s{};
  if (el < width) {
    if (p == 0) s = load_row8<float>(tail + slab * width, el, width);
    int64_t i = a;
    for (; i + 4 <= b; i += 4) {
      f32x8 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = load_row8<float>(head + (i + j) * width, el, width);
#pragma unroll
      for (int j = 0; j < 4; ++j) s += x[j];
    }
    for (; i < b; ++i) s += load_row8<float>(head + i * width, el, width);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[threadIdx.x * 8 + j] = s[j];
  __syncthreads();
  if (p == 0 && el < width) {
    for (int q = 1; q < per; ++q)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += sum[(q * lanes + l) * 8 + j];
    store_row8<T>(out + (int64_t)key * width, el, width, s * scale);
  }
}

int emb_lanes(int width) {
  int lanes = 8;
  while (lanes < MLCG_WAVE && 8 * lanes < width) lanes *= 2;
  return lanes;
}

template <typename T>
int emb_forward(const void* table, int rows, const int64_t* tokens, int64_t n, int width,
                float scale, void* out, unsigned* flags, hipStream_t s) {
  const int lanes = emb_lanes(width);
  const dim3 grid = chain_grid(mlcg_div_up(n, kEmbThreads / lanes * kEmbRows));
  hipLaunchKernelGGL((embedding_forward<T>), grid, dim3(kEmbThreads), 0, s, (const T*)table, rows,
                     tokens, n, width, lanes, scale, (T*)out, flags);
  return mlcg_launch_status();
}

// Rows of a slab: long ones leave less to be joined, short ones more to do at the
// same time: 64 where the gradient has 24 Mi elements in fp32, 96 Mi in 16 bits.  Sums
// and joins with 32 and 64 rows, us, 25 and 8000 tokens: fp32, 65536 x 128 19 and 26
// against 26 and 31; 262144 x 64 (16 Mi) 30 and 49 against 32 and 44; 262144 x 128 39 and
// 57 against 36 and 45; 131072 x 512 59 and 68 against 52 and 60; bf16, 131072 x 256 31
// and 40 against 43 and 47; 262144 x 256 (64 Mi) 42 and 57 against 48 and 56; 548864 x
// 128 50 and 66 against 53 and 71; 548864 x 256 89 and 106 against 74 and 97.  128 rows
// (548864 x 256) took 112 + 19 us, sums and joins, where 64 took 88 + 33.
int slab_rows(int64_t n, int width, bool fp32) {
  return n * width >= (int64_t(fp32 ? 24 : 96) << 20) ? 64 : 32;
}

template <typename T, int SLAB>
int emb_sums(const void* grad, const int* keys, const int* index, int64_t n, int rows, int width,
             float scale, void* out, float* ws, hipStream_t s) {
  const int lanes = emb_lanes(width);
  const int64_t slabs = (n + SLAB - 1) / SLAB;
  const unsigned parts = mlcg_div_up(width, 8 * lanes);
  float *head = ws, *tail = ws + slabs * width;
  hipLaunchKernelGGL((embedding_slab<T, SLAB>),
                     chain_grid(mlcg_div_up(slabs, kEmbThreads / lanes), parts), dim3(kEmbThreads),
                     0, s, (const T*)grad, keys, index, n, rows, width, lanes, scale, (T*)out,
                     head, tail);
  hipLaunchKernelGGL((embedding_join<T, SLAB>), chain_grid(slabs, parts), dim3(kEmbThreads), 0, s,
                     keys, n, rows, width, lanes, scale, head, tail, (T*)out);
  return mlcg_launch_status();
}

template <typename T>
int emb_backward(const void* grad, const int* keys, const int* index, int64_t n, int rows,
                 int width, float scale, void* out, float* ws, hipStream_t s) {
  const int64_t total = (int64_t)rows * width;
  hipLaunchKernelGGL((embedding_zero<T>),
                     dim3(mlcg_persistent_groups(mlcg_div_up(total, 16 * kEmbThreads), 8)),
                     dim3(kEmbThreads), 0, s, (T*)out, total);
  if (n == 0) return mlcg_launch_status();
  return slab_rows(n, width, sizeof(T) == 4) == 32
             ? emb_sums<T, 32>(grad, keys, index, n, rows, width, scale, out, ws, s)
             : emb_sums<T, 64>(grad, keys, index, n, rows, width, scale, out, ws, s);
}

bool emb_ok(int64_t rows, int64_t n, int width) {
  return rows >= 1 && rows < (int64_t(1) << 30) && n >= 0 && n < (int64_t(1) << 31) &&
         width >= 1 && width <= kEmbMaxWidth;
}

}  // namespace

extern "C" int mlcg_scaled_embedding(const void* table, int64_t rows, const int64_t* tokens,
                                     int64_t n, int width, int dtype, float scale, void* out,
                                     void* stream) {
  MLCG_REQUIRE(emb_ok(rows, n, width));
  if (n == 0) return MLCG_OK;
  MLCG_REQUIRE(table && tokens && out);
  unsigned* const flags = mlcg_numerics_word_ptr();
  if (!flags) return MLCG_ERR_LAUNCH;
  hipStream_t s = mlcg_stream(stream);
  switch (dtype) {
    case MLCG_DTYPE_F32:
      return emb_forward<float>(table, (int)rows, tokens, n, width, scale, out, flags, s);
    case MLCG_DTYPE_F16:
      return emb_forward<_Float16>(table, (int)rows, tokens, n, width, scale, out, flags, s);
    case MLCG_DTYPE_BF16:
      return emb_forward<__bf16>(table, (int)rows, tokens, n, width, scale, out, flags, s);
    default: return MLCG_ERR_ARGUMENT;
  }
}

extern "C" int64_t mlcg_token_order_workspace_ints(int64_t n, int64_t rows) {
  if (!emb_ok(rows, n, 1)) return -1;
  return 2 * n + 256 + 256 * ((n + kSortRows - 1) / kSortRows);
}

extern "C" int mlcg_token_order(const int64_t* tokens, int64_t n, int64_t rows, int* keys,
                                int* index, int* workspace, int64_t workspace_ints, void* stream) {
  MLCG_REQUIRE(emb_ok(rows, n, 1));
  if (n == 0) return MLCG_OK;
  MLCG_REQUIRE(tokens && keys && index && workspace &&
               workspace_ints >= mlcg_token_order_workspace_ints(n, rows));
  unsigned* const flags = mlcg_numerics_word_ptr();
  if (!flags) return MLCG_ERR_LAUNCH;
  hipStream_t s = mlcg_stream(stream);
  const int blocks = (int)((n + kSortRows - 1) / kSortRows);
  int bits = 1;  // of the largest key, `rows`
  while ((rows >> bits) != 0) ++bits;
  const int passes = (bits + 7) / 8;
  int *keys2 = workspace, *index2 = workspace + n, *totals = workspace + 2 * n;
  int* const counts = totals + 256;
  const int *kin = nullptr, *iin = nullptr;
  for (int p = 0; p < passes; ++p) {
    const bool here = (passes - 1 - p) % 2 == 0;  // the last pass ends in the outputs
    int *ko = here ? keys : keys2, *io = here ? index : index2;
    hipLaunchKernelGGL(sort_count, dim3(blocks), dim3(kEmbThreads), 0, s, tokens, kin, n,
                       (int)rows, 8 * p, blocks, counts, flags);
    hipLaunchKernelGGL(sort_scan, dim3(256), dim3(kEmbThreads), 0, s, counts, blocks, totals);
    hipLaunchKernelGGL(sort_place, dim3(blocks), dim3(kEmbThreads), 0, s, tokens, kin, iin, n,
                       (int)rows, 8 * p, blocks, counts, totals, ko, io);
    kin = ko;
    iin = io;
  }
  return mlcg_launch_status();
}

extern "C" int64_t mlcg_scaled_embedding_workspace_floats(int64_t n, int width) {
  if (!emb_ok(1, n, width)) return -1;
  const int slab = slab_rows(n, width, false);  // the shorter of both types'
  return 2 * ((n + slab - 1) / slab) * width;
}

extern "C" int mlcg_scaled_embedding_backward(const void* grad, const int* keys, const int* index,
                                              int64_t n, int64_t rows, int width, int dtype,
                                              float scale, void* grad_table, float* workspace,
                                              int64_t workspace_floats, void* stream) {
  MLCG_REQUIRE(emb_ok(rows, n, width) && grad_table && chain_aligned16(grad_table));
  MLCG_REQUIRE(n == 0 || (grad && keys && index && workspace &&
                          workspace_floats >= mlcg_scaled_embedding_workspace_floats(n, width)));
  hipStream_t s = mlcg_stream(stream);
  const int v = (int)rows;
  switch (dtype) {
    case MLCG_DTYPE_F32:
      return emb_backward<float>(grad, keys, index, n, v, width, scale, grad_table, workspace, s);
    case MLCG_DTYPE_F16:
      return emb_backward<_Float16>(grad, keys, index, n, v, width, scale, grad_table, workspace,
                                    s);
    case MLCG_DTYPE_BF16:
      return emb_backward<__bf16>(grad, keys, index, n, v, width, scale, grad_table, workspace, s);
    default: return MLCG_ERR_ARGUMENT;
  }
}
