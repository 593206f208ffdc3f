// The counter-based generator of dropout and of the adapters' dropped inputs (see dropout.hip
// for how its words become a mask).
#pragma once

#include "common.h"

namespace mirl {

struct DropoutArgs {
  uint64_t seed;
  const int64_t* seed_dev;  // or null: the seed is read from the device instead
  uint64_t offset;
  uint32_t threshold;       // of 65536
  float scale;
  __device__ __forceinline__ uint64_t seed_of() const { return seed_dev != nullptr ? (uint64_t)*seed_dev : seed; }
};

inline DropoutArgs dropout_args(double p, int64_t seed, const int64_t* seed_dev, int64_t offset) {
  const double t = std::floor(p * 65536.0 + 0.5);
  const uint32_t T = t > 65536.0 ? 65536u : (uint32_t)t;
  return DropoutArgs{(uint64_t)seed, seed_dev, (uint64_t)offset, T, T < 65536u ? (float)(65536.0 / (double)(65536u - T)) : 0.f};
}

// Bit e of the result: element e of block q is kept.
__device__ __forceinline__ uint32_t dropout_keep8(uint64_t seed, uint64_t offset, uint64_t q, uint32_t threshold) {
  uint32_t c0 = (uint32_t)q, c1 = (uint32_t)(q >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t keep = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    keep |= ((w[j] & 0xffffu) >= threshold ? 1u : 0u) << (2 * j);
    keep |= ((w[j] >> 16) >= threshold ? 2u : 0u) << (2 * j);
  }
  return keep;
}

}  // namespace mirl
