// Dropout with a residual sum, the mask from a counter (gfx950):
//   out[e] = residual[e] + (u16(e) >= t ? x[e] * 65536 / (65536 - t) : 0)
// The mask is never stored: u16(e) is half-word e % 8 of the 128 bits that
// Philox4x32-10 (philox.h) gives for the key `seed` and the counter (e / 8,
// step), so the backward pass is the same kernel on the gradient, without a
// residual.  The step may live in device memory: a recorded graph then draws a
// new mask on every replay.
//
// The drop probability is held in 16 bits (t = round(65536 p)), and the kept
// values are scaled by the probability that is drawn, so the expectation is
// exact for every p.  One counter serves eight elements instead of four: ten
// rounds are 20 products of 32 x 32 bits, which would take about as long as
// the memory traffic of the four 16-bit elements that 32 bits each allow.
//
// Bound by memory: 548864 x 128 in bf16, forward with a residual and backward,
// 133 us for 703 MB (5.3 TB/s, the rate of a large copy); 17920 x 128 in fp32
// 5.8 us a pass.
#include "chain.h"
#include "philox.h"

namespace {

constexpr int kDropThreads = 256;

// the half-word of element j of the eight that a counter serves
__device__ __forceinline__ uint32_t half_word(const Philox& r, int j) {
  return (j & 1) ? r.w[j >> 1] >> 16 : r.w[j >> 1] & 0xFFFFu;
}

template <typename T>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(
    const T* __restrict__ x, const T* __restrict__ residual, int64_t n, uint32_t t, float scale,
    uint64_t seed, const int64_t* __restrict__ step_dev, int64_t step_value, int vec,
    T* __restrict__ out) {
  const uint64_t step = (uint64_t)(step_dev ? *step_dev : step_value);
  const int64_t groups = (n + 7) / 8;
  for (int64_t c = (int64_t)blockIdx.x * kDropThreads + threadIdx.x; c < groups;
       c += (int64_t)gridDim.x * kDropThreads) {
    const int64_t e = 8 * c;
    if (vec && e + 8 <= n) {
      const v8<T> xv = *reinterpret_cast<const v8<T>*>(x + e);
      v8<T> rv{};
      if (residual) rv = *reinterpret_cast<const v8<T>*>(residual + e);
      const Philox h = mlcg_philox(seed, (uint64_t)c, step);
      v8<T> y;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        y[j] = (T)((float)rv[j] + (half_word(h, j) >= t ? (float)xv[j] * scale : 0.0f));
      *reinterpret_cast<v8<T>*>(out + e) = y;
    } else {
      const Philox h = mlcg_philox(seed, (uint64_t)c, step);
      for (int j = 0; j < 8 && e + j < n; ++j)
        out[e + j] = (T)((residual ? (float)residual[e + j] : 0.0f) +
                         (half_word(h, j) >= t ? (float)x[e + j] * scale : 0.0f));
    }
  }
}

template <typename T>
int launch_dropout(const void* x, const void* residual, int64_t n, uint32_t t, uint64_t seed,
                   const int64_t* step_dev, int64_t step, void* out, hipStream_t s) {
  const int vec = chain_aligned16(x) && chain_aligned16(residual) && chain_aligned16(out);
  const unsigned groups =
      mlcg_persistent_groups((n + 8 * kDropThreads - 1) / (8 * kDropThreads), 16);
  hipLaunchKernelGGL(dropout_kernel<T>, dim3(groups), dim3(kDropThreads), 0, s, (const T*)x,
                     (const T*)residual, n, t, 65536.0f / (float)(65536u - t), seed, step_dev,
                     step, vec, (T*)out);
  return mlcg_launch_status();
}

}  // namespace

extern "C" int mlcg_dropout_add(const void* x, const void* residual, int64_t n, int dtype,
                                int threshold, uint64_t seed, const int64_t* step_dev,
                                int64_t step, void* out, void* stream) {
  MLCG_REQUIRE(n >= 0 && n <= (int64_t(1) << 40) && threshold >= 0 && threshold < 65536);
  MLCG_REQUIRE(n == 0 || (x && out));
  if (n == 0) return MLCG_OK;
  hipStream_t s = mlcg_stream(stream);
  const uint32_t t = (uint32_t)threshold;
  auto launch = [&](auto zero) {
    return launch_dropout<decltype(zero)>(x, residual, n, t, seed, step_dev, step, out, s);
  };
  switch (dtype) {
    case MLCG_DTYPE_F32: return launch(float{});
    case MLCG_DTYPE_F16: return launch(_Float16{});
    case MLCG_DTYPE_BF16: return launch(__bf16{});
  }
  return MLCG_ERR_UNSUPPORTED;
}
