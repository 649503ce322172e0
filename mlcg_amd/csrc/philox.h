// Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw
// ("Parallel random numbers: as easy as 1, 2, 3", SC 2011): 128 random bits for
// a 64-bit key and a 128-bit counter, here (index, step).
#pragma once

#include "common.h"

struct Philox {
  uint32_t w[4];
};

__device__ __forceinline__ Philox mlcg_philox(uint64_t seed, uint64_t index, uint64_t step) {
  uint32_t x0 = (uint32_t)index, x1 = (uint32_t)(index >> 32);
  uint32_t x2 = (uint32_t)step, x3 = (uint32_t)(step >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * x0;
    const uint64_t b = (uint64_t)0xCD9E8D57u * x2;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ k0;
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ k1;
    x3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox{{x0, x1, x2, x3}};
}
