// Operators over the rows of a matrix: what their kernels share.
//
// A row is worked on by a team of 2 to 512 threads, eight elements (or 16, or 32) to a thread; teams of a
// warp or less add up by shuffles, larger ones through shared memory and a named barrier of their own.
// Rows come in through a ring in shared memory that asynchronous copies keep filled several rows ahead: a
// row of 128 to 4096 elements is 0.25 to 16 KB, and the 6.5 TB/s of the memory want some 40 KB in flight
// on every SM, which registers do not hold beside the sums.
//   aligned rows   a thread copies the 16-byte pieces that it works on itself: nobody waits for anybody
//   other rows     the 16-byte pieces that the row lies in, whose they may be; a barrier, and every thread
//                  reads its elements from wherever they fell
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "zp_common.cuh"
#include "zp_philox.cuh"
#include "zippel_b200.h"

struct ZpDrop {                     // dropout of a call; state null: nothing is dropped
  const int64_t *state;
  uint32_t threshold;
  float scale;
};

// One call of a norm, or of the join (res / sum, dsum / dres) in front of it, in either direction
struct ZpNormCall {
  int64_t rows, width;
  const void *x, *res, *w, *b, *dy, *dsum;
  int64_t ldx, ldr, ldy, lds;
  ZpDrop drop;
  float eps;
  const float *mean_in, *rstd_in;
  void *sum, *y, *dx, *dres, *dw, *db;
  float *mean, *rstd, *partial;
  int dtype, param_dtype;
};

// The kernels of teams (zp_rowwise_fwd.cu, zp_rowwise_bwd.cu); `taken` false: the call is not for them
// and nothing was launched.  The backward leaves `parts` rows of partial sums {gw, gb} in c.partial, at
// most ZP_ROWWISE_PARTS.
#define ZP_ROWWISE_PARTS 148
int zp_launch_norm_fwd(const ZpNormCall &c, bool &taken, cudaStream_t st);
int zp_launch_norm_bwd(const ZpNormCall &c, bool &taken, int &parts, cudaStream_t st);

__device__ __forceinline__ float zp_float(float v) { return v; }
__device__ __forceinline__ float zp_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float zp_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T zp_rounded(float v);
template <> __device__ __forceinline__ float zp_rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ __half zp_rounded<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 zp_rounded<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

template <typename T> constexpr int kZpVec = 16 / (int)sizeof(T);      // elements of a 16-byte piece

// 16 bytes of T to floats and back
template <typename T> __device__ __forceinline__ void zp_unpack(const uint4 &q, float (&v)[kZpVec<T>]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      v[k] = __uint_as_float(w[k]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
      v[2 * k] = f.x; v[2 * k + 1] = f.y;
    } else {
      v[2 * k] = __uint_as_float(w[k] << 16);
      v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
    }
  }
}
template <typename T> __device__ __forceinline__ uint4 zp_pack(const float (&v)[kZpVec<T>]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      w[k] = __float_as_uint(v[k]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t *>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// element c of a parameter vector of type ZP_F32 (`wide`) or T
template <typename T>
__device__ __forceinline__ float zp_param(const void *w, bool wide, int64_t c, float otherwise) {
  if (!w) return otherwise;
  return wide ? static_cast<const float *>(w)[c] : zp_float(static_cast<const T *>(w)[c]);
}

// ---- teams ----------------------------------------------------------------------------------------

constexpr int kZpTeamThreads = 512;            // of a block

// Where a thread stands.  A "walker" is what goes through rows by itself: a warp, with one or several
// teams in it, or a team of several warps.  It takes `per` rows at a time, one for each of its teams.
struct ZpTeam {
  int size, lane;                              // threads of a team, this one's place in it
  int index;                                   // of the team in the block
  int per, sub;                                // rows of a walker, this team's among them
  int walker, walkers;
  float2 *red;                                 // [2][warps of the block], for teams of several warps

  __device__ __forceinline__ ZpTeam(int team_size, float2 *red_) {
    size = team_size;
    const int tid = threadIdx.x, wide = size > 32 ? size : 32;
    lane = tid & (size - 1);
    index = tid / size;
    per = wide / size;
    walker = tid / wide;
    walkers = kZpTeamThreads / wide;
    sub = index - walker * per;
    red = red_;
  }
  __device__ __forceinline__ void sync() const {
    if (size <= 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + index), "r"(size) : "memory");
  }
  // sums over the team, the same in all of it; `turn` alternates from sum to sum (a buffer that is
  // written again has been read by all: the other's barrier lies in between)
  __device__ __forceinline__ float2 sum(float2 v, int turn) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (o >= size) continue;
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (size <= 32) return v;
    float2 *at = red + (turn & 1) * (kZpTeamThreads / 32);
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    sync();
    const int n = size >> 5;                   // warps: each adds up all of them, in the same order
    v = at[index * n + (threadIdx.x & (n - 1))];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      if (o >= n) continue;
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
  }
  __device__ __forceinline__ float sum(float v, int turn) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      if (o < size) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (size <= 32) return v;
    float *at = reinterpret_cast<float *>(red + (turn & 1) * (kZpTeamThreads / 32));
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    sync();
    const int n = size >> 5;
    v = at[index * n + (threadIdx.x & (n - 1))];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
      if (o < n) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
};

// ---- the ring -------------------------------------------------------------------------------------

__device__ __forceinline__ void zp_copy16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void zp_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until of this thread's latest groups at most `stages` - 2 are on their way (stages: 2 or 4)
__device__ __forceinline__ void zp_copy_wait(int stages) {
  if (stages == 4) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// One of the arrays that a ring brings in: the next row to fetch, and the addresses that may be read.
struct ZpSource {
  const char *row, *begin, *end;
  int64_t step;                                // bytes from a team's row to its next
  int place, turn;                             // of the row that is worked on within 16 bytes; added per row
  __device__ __forceinline__ ZpSource(const void *base, int64_t ld, int64_t rows, int64_t width, int size,
                                      int64_t first, int64_t rows_per_step) {
    begin = static_cast<const char *>(base);
    end = begin + ((rows - 1) * ld + width) * size;
    row = begin + first * ld * size;
    step = rows_per_step * ld * size;
    place = (int)(reinterpret_cast<uintptr_t>(row) & 15);
    turn = (int)(step & 15);
  }
  __device__ __forceinline__ void advance() { place = (place + turn) & 15; }
};

// The next row of `width` elements of T into a slot.  kAligned: element c goes to byte c * sizeof(T), each
// thread copies its own.  Else the row keeps its place within 16 bytes.
template <typename T, bool kAligned, int E>
__device__ __forceinline__ void zp_fetch_row(const ZpTeam &t, char *slot, ZpSource &s, bool live, int width) {
  const char *const row = s.row;
  s.row += s.step;
  if (!live) return;
  if constexpr (kAligned) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(slot) + 16 * t.lane;
    const char *const from = row + 16 * t.lane;
#pragma unroll
    for (int i = 0; i < E / kZpVec<T>; ++i) {
      const int piece = t.lane + i * t.size;
      if (piece * kZpVec<T> < width) zp_copy16(to + 16 * i * t.size, from + 16 * i * t.size);
    }
  } else {
    const char *from = reinterpret_cast<const char *>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)15);
    const char *end = row + width * (int)sizeof(T);
    for (const char *p = from + 16 * t.lane; p < end; p += 16 * t.size) {
      char *to = slot + (p - from);
      if (p >= s.begin && p + 16 <= s.end) {
        zp_copy16((uint32_t)__cvta_generic_to_shared(to), p);
      } else {                                 // the ends of the array: what lies outside is not read
        for (int k = 0; k < 16; k += sizeof(T))
          if (p + k >= row && p + k < end)
            *reinterpret_cast<T *>(to + k) = *reinterpret_cast<const T *>(p + k);
      }
    }
  }
}

// A thread's V elements number i of a row in a slot (kAligned: a piece of 16 bytes, else one element)
template <typename T, bool kAligned> constexpr int kZpStep = kAligned ? kZpVec<T> : 1;
template <typename T, bool kAligned>
__device__ __forceinline__ void zp_read(const ZpTeam &t, const char *slot, int i,
                                        float (&v)[kZpStep<T, kAligned>]) {
  if constexpr (kAligned) zp_unpack<T>(*reinterpret_cast<const uint4 *>(slot + 16 * (t.lane + i * t.size)), v);
  else v[0] = zp_float(*reinterpret_cast<const T *>(slot + sizeof(T) * (t.lane + i * t.size)));
}
// ... and to memory (or back to the slot): `row` is the address of the row's first element
template <typename T, bool kAligned>
__device__ __forceinline__ void zp_write(const ZpTeam &t, void *row, int i, const float (&v)[kZpStep<T, kAligned>]) {
  if constexpr (kAligned) static_cast<uint4 *>(row)[t.lane + i * t.size] = zp_pack<T>(v);
  else static_cast<T *>(row)[t.lane + i * t.size] = zp_rounded<T>(v[0]);
}

// ---- which of a thread's elements are kept ----------------------------------------------------------
// Bit e of the result: the thread's element e (of E, V of them side by side) of row r is kept.
//   aligned, 16-bit   a piece is one counter's eight elements
//   aligned, fp32     a piece is half of them: of two neighbours each works out one of two counters, and
//                     they swap
//   other rows        the team works out the row's counters, eight bits each into `bytes`
//                     [width / 8 + 2], and every thread looks up its own
// All threads of a warp come here together.
template <typename T, bool kAligned, int E>
__device__ __forceinline__ uint32_t zp_kept_bits(const ZpTeam &t, const ZpPhiloxKey &key, uint32_t threshold,
                                                 int64_t r, int width, uint8_t *bytes) {
  uint32_t bits = 0;
  if constexpr (kAligned && sizeof(T) == 2) {
    const uint64_t first = (uint64_t)r * (uint32_t)(width / 8);
#pragma unroll
    for (int i = 0; i < E / 8; ++i)
      bits |= zp_philox_kept(key, first + t.lane + i * t.size, threshold) << (8 * i);
  } else if constexpr (kAligned) {
    const uint64_t first = (uint64_t)r * (uint32_t)(width / 8);
    const int odd = t.lane & 1;
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
      const uint32_t mine = zp_philox_kept(key, first + (t.lane + (2 * i + odd) * t.size) / 2, threshold);
      const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
      // piece 2i: the even lane's counter, piece 2i + 1: the odd one's; low half for the even lane
      const uint32_t lo = odd ? other >> 4 : mine & 15, hi = odd ? mine >> 4 : other & 15;
      bits |= (lo | hi << 4) << (8 * i);
    }
  } else {
    const uint64_t e0 = (uint64_t)r * (uint64_t)width;
    const int groups = (int)((e0 + width - 1) / 8 - e0 / 8) + 1, place = (int)(e0 & 7);
    t.sync();                                  // the last row's have been looked up
    for (int g = t.lane; g < groups; g += t.size) bytes[g] = (uint8_t)zp_philox_kept(key, e0 / 8 + g, threshold);
    t.sync();
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int c = t.lane + i * t.size;
      if (c < width) bits |= (uint32_t)(bytes[(place + c) >> 3] >> ((place + c) & 7) & 1) << i;
    }
  }
  return bits;
}

// ---- launches ---------------------------------------------------------------------------------------

// How a call's rows are shared out: elements per thread, the team's size, whether pieces of 16 bytes are
// aligned, and the ring's sizes.
struct ZpTeamPlan {
  int team, elements;
  bool aligned;
  int slot, bytes, stages;                     // bytes of a slot, of the counters' bits of a team
  size_t smem;
  unsigned blocks;
};
// `arrays` come in per row; `last_per_element`: bytes of shared memory per element of a block's teams that
// the kernel needs when the ring is done with; `most`: elements of a thread where there are rows enough.
// False: the rows are too wide.
inline bool zp_team_plan(const ZpNormCall &c, bool aligned, int arrays, size_t last_per_element, int most,
                         ZpTeamPlan &p) {
  const int64_t size = c.dtype == ZP_F32 ? 4 : 2;
  if (c.width > kZpTeamThreads * 32) return false;
  p.aligned = aligned;
  for (p.elements = 8; p.elements < 32; p.elements *= 2) {
    if (c.width > (int64_t)kZpTeamThreads * p.elements) continue;
    if (p.elements >= most || c.rows * c.width < (int64_t)148 * kZpTeamThreads * 2 * p.elements) break;
  }
  const int64_t need = zp_ceil_div(c.width, p.elements);
  for (p.team = 2; p.team < need; p.team *= 2) {}
  const int teams = kZpTeamThreads / p.team;
  p.slot = (int)zp_align_up((size_t)(p.team * p.elements * size) + (aligned ? 0 : 16), 16);
  p.bytes = aligned || !c.drop.state ? 0 : (int)zp_align_up((size_t)c.width / 8 + 2, 16);
  const size_t red = 2 * sizeof(float2) * (kZpTeamThreads / 32), fixed = red + (size_t)p.bytes * teams;
  const size_t last = last_per_element * kZpTeamThreads * p.elements;
  const size_t stage = (size_t)arrays * p.slot * teams;
  const size_t room = 226 * 1024;
  p.stages = fixed + 4 * stage <= room ? 4 : 2;
  if (fixed + p.stages * stage > room || fixed + last > room) return false;
  p.smem = fixed + (p.stages * stage > last ? p.stages * stage : last);
  const int64_t units = zp_ceil_div(c.rows, p.team < 32 ? 32 / p.team : 1);
  p.blocks = (unsigned)(units < 148 ? units : 148);
  return true;
}
inline bool zp_piece_aligned(const void *p, int64_t ld, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ((size_t)ld * size) % 16 == 0;
}
