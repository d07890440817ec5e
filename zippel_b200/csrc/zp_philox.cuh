// Counter-based random bits: Philox-4x32 with ten rounds (J. K. Salmon, M. A. Moraes, R. O. Dror,
// D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
//
// Dropout's use of it: `state` holds (seed, offset).  Element i of a tensor in row-major order belongs
// to counter (i / 8, offset) under key seed and takes the (i % 8)-th 16-bit half of the four words that
// come out, low half first.  Which elements are kept is a function of (seed, offset, i) alone: not of
// the type, the strides, the launch, or whether the call is a forward or a VJP.  Sixteen bits an element,
// not thirty-two: ten rounds are about 60 integer instructions, and with four elements a counter they,
// not the memory, set the time of a 16-bit tensor.  The price is that p is rounded to a multiple of
// 2^-16; the factor of what is kept is one over the rounded share, so the mean stays right.
#pragma once

#include <stdint.h>

struct ZpPhiloxKey {
  uint32_t k0, k1, c2, c3;
};

__device__ __forceinline__ ZpPhiloxKey zp_philox_key(const int64_t *__restrict__ state) {
  const uint64_t seed = (uint64_t)state[0], offset = (uint64_t)state[1];
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
}

// the 128 bits of elements 8 * group .. 8 * group + 7
__device__ __forceinline__ uint4 zp_philox(const ZpPhiloxKey &key, uint64_t group) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = key.c2, c3 = key.c3;
  uint32_t k0 = key.k0, k1 = key.k1;
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
  return make_uint4(c0, c1, c2, c3);
}

// bit j set: element 8 * group + j is kept (its 16 bits are at least `threshold`)
__device__ __forceinline__ uint32_t zp_philox_kept(const ZpPhiloxKey &key, uint64_t group,
                                                   uint32_t threshold) {
  const uint4 w = zp_philox(key, group);
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  uint32_t kept = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kept |= ((words[j] & 0xFFFFu) >= threshold ? 1u : 0u) << (2 * j);
    kept |= ((words[j] >> 16) >= threshold ? 1u : 0u) << (2 * j + 1);
  }
  return kept;
}
