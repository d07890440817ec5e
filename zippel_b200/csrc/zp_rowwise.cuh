// Operators over the rows of a matrix: what their kernels share.
//
// A row is worked on by a team of 2 to 512 threads, or by a cluster of blocks of 512, E elements to a thread in
// pieces of 16 bytes; a team takes R rows at a time, so that what a row costs beside its elements (the joining of
// sums, barriers, addresses) is shared.  Teams of a warp or less add up by shuffles, larger ones through shared
// memory and a named barrier of their own, clusters through each other's shared memory.  Arithmetic on the elements goes by pairs (one instruction for two): these
// kernels have 20 to 35 instruction slots for an element at the memory's speed, and spend 11 to 20, or 28 to 41 with
// dropout.
//
// Rows come in through a ring in shared memory that asynchronous copies keep filled: the 6.5 TB/s of the
// memory want some 40 KB in flight on every SM, which registers do not hold beside the sums.
//   aligned rows   a thread copies the pieces that it works on itself: nobody waits for anybody
//   cycled rows    of a width that eight does not divide, in arrays from end to end: row r begins r * width
//                  mod 8 elements behind a border of eight, the same for every eighth row at least.  A team
//                  takes rows of one such class alone, and its pieces are those of memory, the first and the last
//                  shared with the neighbours: everything else is as with aligned rows
//   shifted rows   all others.  The 16-byte pieces that the row lies in come as they are; after a barrier a
//                  thread puts its pieces together from two of them, and results go the same way back
#pragma once

#include <cmath>
#include <initializer_list>
#include <utility>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "zp_common.cuh"
#include "zp_philox.cuh"
#include "zippel_b200.h"

struct ZpDrop {                     // dropout of a call; state null: nothing is dropped
  const int64_t *state;
  uint32_t threshold;               // of 65536
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
// most ZP_ROWWISE_PARTS and seven more than there are rows.
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

// 16 bytes of T to pairs of floats and back
template <typename T> __device__ __forceinline__ void zp_unpack(const uint4 &q, float2 (&v)[kZpVec<T> / 2]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 2; ++k) v[k] = make_float2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, __half>::value)
        v[k] = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
      else
        v[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
    }
  }
}
template <typename T> __device__ __forceinline__ uint4 zp_pack(const float2 (&v)[kZpVec<T> / 2]) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __float22half2_rn(v[k]);
        w[k] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __float22bfloat162_rn(v[k]);
        w[k] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// element c of a parameter vector of type ZP_F32 (`wide`) or T
template <typename T>
__device__ __forceinline__ float zp_param(const void *w, bool wide, int64_t c, float otherwise) {
  if (!w) return otherwise;
  return wide ? static_cast<const float *>(w)[c] : zp_float(static_cast<const T *>(w)[c]);
}

// elements c .. c + V - 1 of one (`otherwise` where there is none); vectors: they lie in aligned pieces of 16 bytes
template <typename T>
__device__ __forceinline__ void zp_params(const void *w, bool wide, bool vectors, int c, int width, float otherwise,
                                          float2 (&v)[kZpVec<T> / 2]) {
  constexpr int V = kZpVec<T>;
  if (!w || c >= width) {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) v[k] = make_float2(otherwise, otherwise);
  } else if (vectors && wide) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      const float4 q = reinterpret_cast<const float4 *>(static_cast<const float *>(w) + c)[k];
      v[2 * k] = make_float2(q.x, q.y);
      v[2 * k + 1] = make_float2(q.z, q.w);
    }
  } else if (vectors) {
    zp_unpack<T>(*reinterpret_cast<const uint4 *>(static_cast<const T *>(w) + c), v);
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k)
      v[k] = make_float2((unsigned)(c + 2 * k) < (unsigned)width ? zp_param<T>(w, wide, c + 2 * k, 0.f) : otherwise,
                         (unsigned)(c + 2 * k + 1) < (unsigned)width ? zp_param<T>(w, wide, c + 2 * k + 1, 0.f) : otherwise);
  }
}

// ---- teams ----------------------------------------------------------------------------------------

constexpr int kZpTeamThreads = 512;            // of a block
constexpr int kZpTeamWarps = kZpTeamThreads / 32;

constexpr int kZpMostRanks = 8;                // blocks of a cluster
// shared memory in front of the rings: room for two turns' sums of warps, and of blocks
constexpr int kZpSumsBytes = sizeof(float) * 2 * 4 * (kZpTeamWarps + kZpMostRanks);

// Where a thread stands.  A "walker" is what goes through rows by itself: a warp, with one or several
// teams in it, or a team of several warps.  kWide: the team is a cluster of blocks, each with pieces of its own
// of every row.
template <bool kWide> struct ZpTeam {
  int size, lane;                              // threads of a team (in the block), this one's place among them
  int index;                                   // of the team in the block
  int per, sub;                                // teams of a walker, this one among them
  int walker, walkers;
  int ranks, rank;                             // blocks of the team, this one's place among them
  float *red;                                  // [2][warps of the block][4], then [2][blocks][4]

  __device__ __forceinline__ ZpTeam(int team_size, int blocks, float *red_) {
    size = team_size;
    const int tid = threadIdx.x, wide = size > 32 ? size : 32;
    lane = tid & (size - 1);
    index = tid / size;
    per = wide / size;
    walker = tid / wide;
    walkers = kZpTeamThreads / wide;
    sub = index - walker * per;
    red = red_;
    ranks = kWide ? blocks : 1;
    rank = 0;
    if constexpr (kWide) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  }
  // number of this thread's piece i of a row, and the pieces from one to the next
  __device__ __forceinline__ int piece(int i) const { return kWide ? lane + (i * ranks + rank) * size : lane + i * size; }
  __device__ __forceinline__ int apart() const { return kWide ? ranks * size : size; }
  __device__ __forceinline__ int64_t block() const { return kWide ? blockIdx.x / ranks : blockIdx.x; }
  __device__ __forceinline__ int64_t blocks() const { return kWide ? gridDim.x / ranks : gridDim.x; }
  // all blocks of the team; what they wrote in each other's shared memory is there
  __device__ __forceinline__ void meet() const {
    if constexpr (kWide) {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
  }
  __device__ __forceinline__ void sync() const {
    if (size <= 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + index), "r"(size) : "memory");
  }
  // Sums of K values over the team, the same in all of it.  `turn` alternates from call to call (a buffer
  // that is written again has been read by all: the other's barrier lies in between); `order`: what
  // was read and written in shared memory before is ordered against what comes after.
  // Over a warp, K values take 5 + K - 1 exchanges instead of 5 K: lanes send away the values that
  // they will not add up further.
  template <int K> __device__ __forceinline__ void sum(float (&v)[K], int turn, bool order) const {
    static_assert(K == 1 || K == 2 || K == 4, "");
    if (size < 32) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        if (o >= size) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
      }
      if (order) __syncwarp();
      return;
    }
    const int at = threadIdx.x & 31;
    constexpr int kOwn = 32 / K;               // lanes that add up one value
    float s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = v[k];
#pragma unroll
    for (int left = K / 2, o = 16; left > 0; left /= 2, o /= 2) {
      const bool up = at & o;
#pragma unroll
      for (int k = 0; k < left; ++k)
        s[k] = (up ? s[k + left] : s[k]) + __shfl_xor_sync(0xffffffffu, up ? s[k] : s[k + left], o);
    }
    float one = s[0];                          // of value at / kOwn
#pragma unroll
    for (int o = kOwn / 2; o > 0; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
    if (size > 32) {
      float *const buf = red + (turn & 1) * (kZpTeamWarps * 4);
      if (at % kOwn == 0) buf[(threadIdx.x >> 5) * K + at / kOwn] = one;
      sync();
      const int n = size >> 5, first = index * n;            // warps of the team
      const float *from = buf + at / kOwn;
      one = from[(first + (at % kOwn & (n - 1))) * K];
#pragma unroll
      for (int w = kOwn; w < kZpTeamWarps; w += kOwn)
        if (w < n) one += from[(first + at % kOwn + w) * K];
#pragma unroll
      for (int o = kOwn / 2; o > 0; o >>= 1)
        if (o < n) one += __shfl_xor_sync(0xffffffffu, one, o);
    } else if (order) {
      __syncwarp();
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = K == 1 ? one : __shfl_sync(0xffffffffu, one, k * kOwn);
    if constexpr (kWide) {                     // the blocks' sums, added by each in the same order
      float *const buf = red + 2 * 4 * kZpTeamWarps + (turn & 1) * (kZpMostRanks * 4);
      if (lane < ranks * K) {
        const int k = lane % K;
        float one = v[0];
#pragma unroll
        for (int i = 1; i < K; ++i) one = k == i ? v[i] : one;
        const uint32_t own = (uint32_t)__cvta_generic_to_shared(buf + rank * 4 + k);
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(own), "r"(lane / K));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(one) : "memory");
      }
      meet();
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = 0.f;
      for (int b = 0; b < ranks; ++b) {
        const float4 q = *reinterpret_cast<const float4 *>(buf + 4 * b);
        const float each[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += each[k];
      }
    }
  }
};

// ---- the ring -------------------------------------------------------------------------------------

__device__ __forceinline__ void zp_copy16(uint32_t to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void zp_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until of this thread's latest groups at most `stages` - 2 are on their way (stages: 2, 3 or 4)
__device__ __forceinline__ void zp_copy_wait(int stages) {
  if (stages == 4) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (stages == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

__device__ __forceinline__ uint32_t zp_shared(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint4 zp_lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 zp_lds8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ void zp_sts16(uint32_t at, const uint4 &v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

enum ZpLying { kZpShifted, kZpAligned, kZpCycled };

// A team's rows in a call: the first, how far from its rows of one turn to the next, from row to row within a
// turn (kZpCycled: the cycle), in how many turns it has its row j and how many turns its warp makes; and how many
// elements of its first piece lie before the row.
template <int kLying, int R> struct ZpTeamRows {
  int64_t first, step;
  int next, turns, before;
  int n[R];
  template <bool kWide>
  __device__ __forceinline__ ZpTeamRows(const ZpTeam<kWide> &t, int64_t rows, int width, int cycle_) {
    const int cycle = kLying == kZpCycled ? cycle_ : 1;
    const int64_t teams = t.blocks() * t.walkers * t.per;                    // a multiple of the cycle
    const int64_t team = (t.walker * t.blocks() + t.block()) * t.per;
    auto first_of = [&](int64_t u) { return kLying == kZpCycled ? u % cycle + u / cycle * cycle * R : u * R; };
    first = first_of(team + t.sub);
    step = teams * R;
    next = cycle;
#pragma unroll
    for (int j = 0; j < R; ++j) n[j] = steps(rows, first + j * next);
    turns = steps(rows, first_of(team));                                      // (a warp's teams go on together)
    before = kLying == kZpCycled ? (int)(first * width & 7) : 0;
  }
  __device__ __forceinline__ int steps(int64_t rows, int64_t r) const {
    return r < rows ? (int)((rows - r + step - 1) / step) : 0;
  }
};

// One of the arrays that a ring brings in: the first of the next rows to fetch (and, but for shifted rows, this
// thread's first piece of it), and the addresses that may be read.
template <int kLying> struct ZpSource {
  static constexpr bool kShifted = kLying == kZpShifted;
  const char *row, *begin, *end;
  int64_t step, next;                          // bytes from a team's rows to its next ones, and from row to row
  int place;                                   // within 16 bytes, of the first of the rows that are worked on
  template <bool kWide, int R>
  __device__ __forceinline__ ZpSource(const ZpTeam<kWide> &t, const void *base, int64_t ld, int64_t rows, int64_t width,
                                      int size, const ZpTeamRows<kLying, R> &own) {
    begin = static_cast<const char *>(base);
    end = begin + ((rows - 1) * ld + width) * size;
    row = begin + (own.first * ld - own.before) * size + (kShifted ? 0 : 16 * t.piece(0));
    step = own.step * ld * size;
    next = own.next * ld * size;
    place = kShifted ? (int)(reinterpret_cast<uintptr_t>(row) & 15) : 0;
  }
  __device__ __forceinline__ int place_of(int j) const { return kShifted ? (place + j * (int)(next & 15)) & 15 : 0; }
  __device__ __forceinline__ void advance() {
    if (kShifted) place = (place + (int)(step & 15)) & 15;
  }
};

// Row j of the next rows, `width` elements of T, into a slot.  Each thread copies its own pieces (kFull: it has
// them all), so that the row begins `before` elements behind the slot's begin; shifted rows keep their place
// within 16 bytes.
template <typename T, int kLying, bool kFull, int M, bool kWide>
__device__ __forceinline__ void zp_fetch_row(const ZpTeam<kWide> &t, uint32_t slot, const ZpSource<kLying> &s, int j,
                                             int width, int before) {
  constexpr int V = kZpVec<T>;
  const char *const row = j ? s.row + j * s.next : s.row;
  if constexpr (kLying != kZpShifted) {
    const uint32_t to = slot + 16 * t.lane;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      const int c = t.piece(i) * V - before;
      if (kFull || (c < width && (kLying == kZpAligned || c + V > 0))) {
        const char *const from = row + 16 * i * t.apart();
        if (kLying == kZpAligned || from + 16 <= s.end)
          zp_copy16(to + 16 * i * t.size, from);
        else                                   // the array's last piece: nothing is read behind its end
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + 16 * i * t.size), "l"(from),
                       "r"((int)(s.end - from)) : "memory");
      }
    }
  } else {
    const int place = (int)(reinterpret_cast<uintptr_t>(row) & 15), span = place + width * (int)sizeof(T);
    const char *const from = row - place;
    if (from >= s.begin && from + ((span + 15) & ~15) <= s.end) {
#pragma unroll
      for (int i = 0; i <= M; ++i) {
        const int at = 16 * (t.lane + i * t.size);
        if (at < span) zp_copy16(slot + at, from + at);
      }
    } else {                                   // the ends of the array: what lies outside is not read
      for (int c = t.lane; c < width; c += t.size) {
        const uint32_t to = slot + place + c * (int)sizeof(T);
        if constexpr (sizeof(T) == 4)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(reinterpret_cast<const uint32_t *>(row)[c]) : "memory");
        else
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(to), "h"(reinterpret_cast<const uint16_t *>(row)[c]) : "memory");
      }
    }
  }
}

// Zeroes for the pieces of a thread that rows do not have, in all `slots` slots from `ring` on: nothing is fetched
// there, so that they are read like the others and add nothing (with branches around each piece 30 011 x 1000 fp16
// took 29 us forward, so 27).
template <int M, bool kWide, typename Has>
__device__ __forceinline__ void zp_clear_pieces(const ZpTeam<kWide> &t, uint32_t ring, int slots, int slot_bytes, Has has) {
#pragma unroll
  for (int i = 0; i < M; ++i)
    if (!has(i))
      for (int s = 0; s < slots; ++s)
        zp_sts16(ring + s * slot_bytes + 16 * (t.lane + i * t.size), make_uint4(0, 0, 0, 0));
}

// bytes place .. place + 15 (place 0 .. 15, a multiple of kSize) of two pieces of 16 side by side
template <int kSize> __device__ __forceinline__ uint4 zp_shifted(const uint32_t (&w)[6], int place) {
  uint32_t y[5];
#pragma unroll
  for (int k = 0; k < 5; ++k) y[k] = place & 4 ? w[k + 1] : w[k];
  if constexpr (kSize == 2) {
    const int half = (place & 2) * 8;
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = __funnelshift_r(y[k], y[k + 1], half);
  }
  return make_uint4(y[0], y[1], y[2], y[3]);
}
template <int kSize> __device__ __forceinline__ uint4 zp_between(const uint4 &a, const uint4 &b, int place) {
  const bool two = place & 8;
  const uint32_t w[6] = {two ? a.z : a.x, two ? a.w : a.y, two ? b.x : a.z, two ? b.y : a.w, two ? b.z : b.x,
                         two ? b.w : b.y};
  return zp_shifted<kSize>(w, place);
}
// ... in shared memory, from `at` (a multiple of 16) on
template <int kSize> __device__ __forceinline__ uint4 zp_read_between(uint32_t at, int place) {
  at += place & 8;
  const uint2 a = zp_lds8(at), b = zp_lds8(at + 8), c = zp_lds8(at + 16);
  const uint32_t w[6] = {a.x, a.y, b.x, b.y, c.x, c.y};
  return zp_shifted<kSize>(w, place);
}

// Piece number i of a thread, of a row in a slot.
template <typename T, int kLying, bool kWide>
__device__ __forceinline__ void zp_read(const ZpTeam<kWide> &t, uint32_t slot, int place, int i, float2 (&v)[kZpVec<T> / 2]) {
  const uint32_t at = slot + 16 * (t.lane + i * t.size);
  zp_unpack<T>(kLying == kZpShifted ? zp_read_between<sizeof(T)>(at, place) : zp_lds16(at), v);
}
// `otherwise` in place of what of a piece from column c on lies outside the row
template <typename T> __device__ __forceinline__ void zp_cut(int c, int width, float2 (&v)[kZpVec<T> / 2], float otherwise) {
#pragma unroll
  for (int k = 0; k < kZpVec<T> / 2; ++k) {
    if ((unsigned)(c + 2 * k) >= (unsigned)width) v[k].x = otherwise;
    if ((unsigned)(c + 2 * k + 1) >= (unsigned)width) v[k].y = otherwise;
  }
}
// Results, piece i from column c on.  `row`: where the team's first piece of the row goes; of a piece that the
// row shares (`edge`: the thread may have one) its own elements alone are written.  Shifted rows go into a slot, 16
// bytes from its start, from where zp_store_row takes them once the whole team has written.
template <typename T, int kLying, bool kWide>
__device__ __forceinline__ void zp_write(const ZpTeam<kWide> &t, char *row, uint32_t slot, int i, int c, int width, bool edge,
                                         const float2 (&v)[kZpVec<T> / 2]) {
  const int q = t.piece(i);
  const uint4 packed = zp_pack<T>(v);
  if constexpr (kLying == kZpShifted) {        // (the rows of a block)
    zp_sts16(slot + 16 * q + 16, packed);
  } else if (kLying == kZpAligned || !edge || (c >= 0 && c + kZpVec<T> <= width)) {
    reinterpret_cast<uint4 *>(row)[q] = packed;
  } else {
    const uint32_t w[4] = {packed.x, packed.y, packed.z, packed.w};
    T *const to = reinterpret_cast<T *>(row) + (size_t)q * kZpVec<T>;
#pragma unroll
    for (int k = 0; k < kZpVec<T>; ++k) {
      if ((unsigned)(c + k) >= (unsigned)width) continue;
      if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t *>(to)[k] = w[k];
      else reinterpret_cast<uint16_t *>(to)[k] = (uint16_t)(w[k / 2] >> (16 * (k & 1)));
    }
  }
}
template <typename T, int M, bool kWide>
__device__ __forceinline__ void zp_store_row(const ZpTeam<kWide> &t, char *row, uint32_t slot, int width) {
  const int place = (int)(reinterpret_cast<uintptr_t>(row) & 15), end = place + width * (int)sizeof(T);
  char *const to = row - place;
  const uint32_t from = place ? slot : slot + 16;
  const int shift = (16 - place) & 15;
#pragma unroll
  for (int i = 0; i <= M; ++i) {
    const int at = 16 * (t.lane + i * t.size);
    if (i == M && 16 * M * t.size >= end) break;
    if (at >= place && at + 16 <= end)
      *reinterpret_cast<uint4 *>(to + at) = zp_read_between<sizeof(T)>(from + at, shift);
  }
  // what the row has of the pieces that it shares, element by element
  constexpr int V = kZpVec<T>;
  for (int k = t.lane; k < 2 * V; k += t.size) {
    const int at = k < V ? k * (int)sizeof(T) : (end & ~15) + (k - V) * (int)sizeof(T);
    const bool mine = k < V ? place && at >= place && at < end : (end & 15) && at >= (place ? 16 : 0) && at < end;
    if (!mine) continue;
    const uint32_t at_slot = slot + 16 + at - place;
    if constexpr (sizeof(T) == 4) {
      uint32_t v;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at_slot));
      *reinterpret_cast<uint32_t *>(to + at) = v;
    } else {
      uint16_t v;
      asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at_slot));
      *reinterpret_cast<uint16_t *>(to + at) = v;
    }
  }
}

// ---- which of a thread's elements are kept ----------------------------------------------------------
// For each pair of elements of each piece:
//   16-bit            a piece is one counter's eight elements, a pair one of its words
//   fp32              a piece is half of them: of two neighbours each works out one of two counters, and
//                     they swap words
//   shifted rows      the team works out the row's counters, eight bits each into `bytes`
//                     [width / 8 + 3], and every thread looks up its own
// kWords: kept as words, which saves two instructions an element; else as a bit per element, where registers
// are short.
template <typename T, int kLying, bool kWords, int E> struct ZpKept {
  static_assert(kLying != kZpShifted || !kWords, "");
  static constexpr int H = kZpVec<T> / 2;
  uint32_t w[kWords ? E / 2 : 1];

  // (all threads of a warp come here together)
  template <bool kWide>
  __device__ __forceinline__ void find(const ZpTeam<kWide> &t, const ZpPhiloxKey<false> &key, uint32_t limit, int64_t r, int width,
                                       uint8_t *bytes) {
    if constexpr (kLying != kZpShifted) {
      if (!kWords) w[0] = 0;
      const uint64_t first = (uint64_t)r * (uint32_t)width / 8;               // counter of the first piece
      const int odd = t.lane & 1;
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        // fp32: of pieces 2i and 2i + 1 the even lane works out the first one's counter, the odd one the other's
        const int place = sizeof(T) == 2 ? t.piece(i) : t.piece(2 * i + odd) / 2;
        uint4 q = zp_philox(key, first + place);
        if constexpr (kWords) {
          if constexpr (sizeof(T) == 4) {      // first half of a counter for the even lane
            const uint32_t a = __shfl_xor_sync(0xffffffffu, odd ? q.x : q.z, 1);
            const uint32_t b = __shfl_xor_sync(0xffffffffu, odd ? q.y : q.w, 1);
            q = odd ? make_uint4(a, b, q.z, q.w) : make_uint4(q.x, q.y, a, b);
          }
          w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
        } else {
          uint32_t mine = zp_kept_of(q, limit);
          if constexpr (sizeof(T) == 4) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
            mine = odd ? other >> 4 | (mine & 0xf0) : (mine & 15) | (other & 15) << 4;
          }
          w[0] |= mine << (8 * i);
        }
      }
    } else {
      constexpr int V = kZpVec<T>;
      const uint64_t e0 = (uint64_t)r * (uint64_t)width;
      const int groups = (int)((e0 + width - 1) / 8 - e0 / 8) + 1, place = (int)(e0 & 7);
      t.sync();                                // the last row's have been looked up
      for (int g = t.lane; g < groups; g += t.size) bytes[g] = (uint8_t)zp_philox_kept(key, e0 / 8 + g, limit);
      t.sync();
      w[0] = 0;
#pragma unroll
      for (int i = 0; i < E / V; ++i) {
        const int c = (t.lane + i * t.size) * V, at = (place + c) >> 3;
        if (c < width) {
          const uint32_t two = bytes[at] | (uint32_t)bytes[at + 1] << 8;
          w[0] |= (two >> ((place + c) & 7) & ((1u << V) - 1)) << (i * V);
        }
      }
    }
  }
  // pair k of piece i
  __device__ __forceinline__ float2 drop(float2 v, int i, int k, uint32_t limit, float scale) const {
    if constexpr (kWords) {
      return zp_drop_pair(v, w[i * H + k], limit, scale);
    } else {
      const uint32_t two = w[0] >> (2 * (i * H + k));
      return make_float2(two & 1 ? v.x * scale : 0.f, two & 2 ? v.y * scale : 0.f);
    }
  }
};

// ---- launches ---------------------------------------------------------------------------------------

// One over a width as a float and what that lacks: `one` is off by at most half a step, 1 - one W is a float (fmaf gives
// it without a rounding), and one + rest is 1/W within 2^-47.  So a sum that is the width times a float gives
// exactly that float: with `one` alone rows of equal values had z 0.02 in place of 0 (1000 columns, or 41, of 1000.0).
struct ZpOver {
  float one, rest;
  __host__ __device__ __forceinline__ float of(float sum) const { return fmaf(sum, one, sum * rest); }
};
inline ZpOver zp_over(int64_t width) {
  const float one = 1.f / (float)width;
  return {one, fmaf(-one, (float)width, 1.f) * one};
}

// How a call's rows are shared out: elements per thread and rows at a time, the team's size, how the rows
// lie, whether every thread has all its pieces, whether weight and bias lie in aligned ones, and the ring's sizes.
struct ZpTeamPlan {
  int team, elements, rows;
  int ranks;                                   // blocks of a team; above one it is a cluster
  int lying, cycle;                            // rows of a class are `cycle` apart
  bool full, vectors;
  int slot, bytes, stages;                     // bytes of a slot, of the counters' bits of a team
  size_t smem;
  ZpOver over;                                 // one over the width
  unsigned blocks;                             // 0 once a device has been found to run none of the plan's clusters
};
// The largest number of teams up to `most` of which every class of the cycle has as many
inline int64_t zp_whole_cycles(const ZpTeamPlan &p, int64_t most) {
  const int teams = kZpTeamThreads / p.team;
  const int64_t by = p.cycle > teams ? p.cycle / teams : 1;
  return most / by * by;
}
// Elements of a row's pieces
inline int64_t zp_span(const ZpNormCall &c, int lying) { return lying == kZpCycled ? c.width + 7 : c.width; }
// `arrays` come in per row; `last_per_element`: bytes of shared memory per element of a block's teams that
// the kernel needs when the ring is done with.  False: this does not fit.
inline bool zp_team_plan(const ZpNormCall &c, int lying, int arrays, size_t last_per_element, int elements, int rows,
                         ZpTeamPlan &p) {
  const int64_t size = c.dtype == ZP_F32 ? 4 : 2;
  const int64_t span = zp_span(c, lying);
  p.ranks = 1;
  while (span > (int64_t)kZpTeamThreads * elements * p.ranks && p.ranks <= kZpMostRanks) p.ranks *= 2;
  // (pieces of a shifted row that lie in two blocks would have to be put together across them)
  if (p.ranks > kZpMostRanks || (p.ranks > 1 && lying == kZpShifted)) return false;
  p.lying = lying;
  p.cycle = lying != kZpCycled ? 1 : c.width % 2 ? 8 : c.width % 4 ? 4 : 2;
  p.vectors = lying != kZpCycled && c.width % (16 / size) == 0 && reinterpret_cast<uintptr_t>(c.w) % 16 == 0 &&
              reinterpret_cast<uintptr_t>(c.b) % 16 == 0;
  p.over = zp_over(c.width);
  p.elements = elements;
  p.rows = rows;
  const int64_t need = p.ranks > 1 ? kZpTeamThreads : zp_ceil_div(span, elements);
  for (p.team = 2; p.team < need; p.team *= 2) {}
  p.full = lying == kZpAligned && (int64_t)p.team * elements * p.ranks == c.width;
  const int teams = kZpTeamThreads / p.team;
  p.slot = (int)(p.team * elements * size) + (lying == kZpShifted ? 48 : 0);
  p.bytes = lying != kZpShifted || !c.drop.state ? 0 : (int)zp_align_up((size_t)c.width / 8 + 3, 16);
  const size_t fixed = kZpSumsBytes + (size_t)p.bytes * teams;
  const size_t last = last_per_element * kZpTeamThreads * elements, room = 226 * 1024;
  const size_t stage = (size_t)arrays * rows * p.slot * teams;
  p.stages = fixed + 4 * stage <= room ? 4 : fixed + 3 * stage <= room ? 3 : 2;
  if (fixed + p.stages * stage > room || fixed + last > room) return false;
  p.smem = fixed + (p.stages * stage > last ? p.stages * stage : last);
  const int64_t units = zp_ceil_div(c.rows, rows * (p.team < 32 ? 32 / p.team : 1)), all = 148 / p.ranks;
  int64_t own = zp_whole_cycles(p, all);
  if (units < own) {                           // as few as there is work for
    const int64_t by = zp_whole_cycles(p, units);
    own = by == units ? units : by + (p.cycle > teams ? p.cycle / teams : 1);
  }
  p.blocks = (unsigned)(own * p.ranks);
  return true;
}
// Clusters of `kernel` that run at the same time, looked up once per device and size (0: none, asked for anew)
struct ZpClusters {
  std::mutex lock;
  int most[64][4] = {};
};
// The plan's blocks as far as the device runs their clusters at the same time.  None: not even one of every class of
// the cycle.
template <typename Kernel> int zp_fit_clusters(Kernel kernel, ZpTeamPlan &p, ZpClusters &state) {
  int dev = 0, log = p.ranks == 2 ? 1 : p.ranks == 4 ? 2 : 3;
  ZP_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return ZP_ERR_UNSUPPORTED;
  std::lock_guard<std::mutex> hold(state.lock);
  int &most = state.most[dev][log];
  if (most == 0) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(148 / p.ranks * p.ranks); cfg.blockDim = dim3(kZpTeamThreads); cfg.dynamicSmemBytes = 227 * 1024;
    cfg.attrs = attr; cfg.numAttrs = 1;
    ZP_CUDA(cudaOccupancyMaxActiveClusters(&most, kernel, &cfg));
  }
  if ((int64_t)p.blocks > (int64_t)most * p.ranks) p.blocks = (unsigned)(zp_whole_cycles(p, most) * p.ranks);
  return ZP_OK;
}
// One kernel of teams; kWide: teams are clusters.  A plan that is left without blocks is not launched.
template <bool kWide, typename Kernel>
int zp_launch_teams(Kernel kernel, const char *name, const ZpNormCall &c, ZpTeamPlan &p, ZpSmemOptIn &opt_in,
                    ZpClusters &clusters, cudaStream_t st) {
  if (int rc = zp_ensure_smem(kernel, kWide ? 227 * 1024 : p.smem, opt_in)) return rc;
  if constexpr (kWide) {
    if (int rc = zp_fit_clusters(kernel, p, clusters)) return rc;
    if (p.blocks == 0) return ZP_OK;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.ranks; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.blocks); cfg.blockDim = dim3(kZpTeamThreads); cfg.dynamicSmemBytes = p.smem; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = kWide ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, c, (const ZpTeamPlan)p);                       // errors: ZP_LAUNCH_CHECK
  ZP_LAUNCH_CHECK(name);
  return ZP_OK;
}
// How the rows of an array of a call lie; the call's are shifted where one array's are
inline int zp_lying(const ZpNormCall &c, const void *p, int64_t ld) {
  const int64_t size = c.dtype == ZP_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p) % 16) return kZpShifted;
  if (c.width * size % 16 == 0 && ld * size % 16 == 0 && (!c.drop.state || c.width % 8 == 0)) return kZpAligned;
  return ld == c.width && c.width % 8 ? kZpCycled : kZpShifted;
}
inline int zp_lying(const ZpNormCall &c, std::initializer_list<std::pair<const void *, int64_t>> arrays) {
  int found = -1;                              // (one width makes no array aligned and another cycled)
  for (const auto &a : arrays)
    if (a.first && found != kZpShifted) found = zp_lying(c, a.first, a.second);
  return found;
}
