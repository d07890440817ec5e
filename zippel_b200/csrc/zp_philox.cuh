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

// The key of a call: the words of its ten rounds and the upper half of the counter.  kKept: all twenty words
// worked out once, in registers; else from the first two each time, where registers are short.
template <bool kKept> struct ZpPhiloxKey {
  uint32_t k0[kKept ? 10 : 1], k1[kKept ? 10 : 1], c2, c3;
};

template <bool kKept> __device__ __forceinline__ ZpPhiloxKey<kKept> zp_philox_key(const int64_t *__restrict__ state) {
  const uint64_t seed = (uint64_t)state[0], offset = (uint64_t)state[1];
  ZpPhiloxKey<kKept> key;
#pragma unroll
  for (int i = 0; i < (kKept ? 10 : 1); ++i) {
    key.k0[i] = (uint32_t)seed + i * 0x9E3779B9u;
    key.k1[i] = (uint32_t)(seed >> 32) + i * 0xBB67AE85u;
  }
  key.c2 = (uint32_t)offset;
  key.c3 = (uint32_t)(offset >> 32);
  return key;
}

// the 128 bits of elements 8 * group .. 8 * group + 7
template <bool kKept> __device__ __forceinline__ uint4 zp_philox(const ZpPhiloxKey<kKept> &key, uint64_t group) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = key.c2, c3 = key.c3;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ (kKept ? key.k0[kKept ? i : 0] : key.k0[0] + i * 0x9E3779B9u);
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ (kKept ? key.k1[kKept ? i : 0] : key.k1[0] + i * 0xBB67AE85u);
    c3 = (uint32_t)a;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The two elements of a word, kept (times scale) or zero: 16 bits h are at least the threshold t exactly if
// h 2^16 > limit = t 2^16 - 1, which for the upper half needs no shift.  1 <= t <= 2^16.
__device__ __forceinline__ uint32_t zp_drop_limit(uint32_t threshold) { return (threshold << 16) - 1; }
__device__ __forceinline__ float2 zp_drop_pair(float2 v, uint32_t word, uint32_t limit, float scale) {
  const float2 by = __fmul2_rn(v, make_float2(scale, scale));
  return make_float2((word << 16) > limit ? by.x : 0.f, word > limit ? by.y : 0.f);
}

// bit j set: element j of a counter's eight is kept
__device__ __forceinline__ uint32_t zp_kept_of(const uint4 &w, uint32_t limit) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  uint32_t kept = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kept |= ((words[j] << 16) > limit ? 1u : 0u) << (2 * j);
    kept |= (words[j] > limit ? 1u : 0u) << (2 * j + 1);
  }
  return kept;
}
template <bool kKept>
__device__ __forceinline__ uint32_t zp_philox_kept(const ZpPhiloxKey<kKept> &key, uint64_t group, uint32_t limit) {
  return zp_kept_of(zp_philox(key, group), limit);
}
