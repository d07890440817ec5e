// Operators over the rows of a matrix, each in fp32, fp16 and bf16 with sums in fp32:
//
//   layer norm   mean = sum x / W;  rstd = rsqrt(sum (x - mean)^2 / W + eps);  z = (x - mean) rstd
//                y = z w + b
//     its VJP    gz = gy w;  gx = rstd (gz - mean(gz) - z mean(gz z));  gw = sum_rows gy z;  gb = sum_rows gy
//   dropout      y = x / keep where the element is kept, 0 where not (zp_philox.cuh); its VJP is itself
//   joined       s = residual + dropout(x), rounded to the type;  y = layer norm of s as it is returned
//     its VJP    gs' = layer norm's VJP of gy + gs;  gresidual = gs';  gx = dropout(gs')
#include <algorithm>
#include <cmath>

#include "zp_rowwise.cuh"

namespace {

bool misplaced(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// sum over a block of kThreads, the same in every thread
constexpr int kThreads = 256;
__device__ __forceinline__ float block_sum(float v, float *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) s += red[w];
  __syncthreads();
  return s;
}

// Dropout.  Each thread writes pieces of 16 bytes, kAhead of them 32 apart, whose loads are on the way together.
// Bound by memory, with the generator close behind: of some 60 integer instructions for eight elements 20
// are wide products.  B200 (share of 6 450 GB/s): 16384 x 8192 bf16 87 to 90 us (0.93 to 0.96), 60000 x 128 fp32 11.0
// (0.86), 20011 x 1023 fp16 14.8 (0.86) and, 1030 apart, 30.8 (0.41: each piece from two, and where it lies).
// In fp32 a piece is half of a counter's elements: of two neighbouring lanes each works out the counter of one of
// two pieces, and they swap words.
//   kFlat    one row of aligned pieces from end to end
//   kRows    `per_row` aligned pieces a row
//   kGather  y lies row behind row; a piece of x is put together from the two that it lies in, at the end of
//            a row (or of x) from its elements
enum { kFlat, kRows, kGather };
// The words of kAhead pieces of a lane.
template <typename T, int kAhead>
__device__ __forceinline__ void kept_words(const ZpPhiloxKey<true> &key, int64_t p0, int lane,
                                           uint32_t (&w)[kAhead][kZpVec<T> / 2]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint4 q = zp_philox(key, p0 + 32 * i + lane);
      w[i][0] = q.x; w[i][1] = q.y; w[i][2] = q.z; w[i][3] = q.w;
    }
  } else {
    const bool odd = lane & 1;
#pragma unroll
    for (int i = 0; i < kAhead; i += 2) {
      const uint4 q = zp_philox(key, (p0 + 32 * (i + odd) + lane) / 2);
      const uint32_t a = __shfl_xor_sync(0xffffffffu, odd ? q.x : q.z, 1);
      const uint32_t b = __shfl_xor_sync(0xffffffffu, odd ? q.y : q.w, 1);
      w[i][0] = odd ? a : q.x; w[i][1] = odd ? b : q.y;
      w[i + 1][0] = odd ? q.z : a; w[i + 1][1] = odd ? q.w : b;
    }
  }
}

template <typename T, int kHow>
__global__ void __launch_bounds__(kThreads, 4)
dropout_pieces_kernel(int64_t pieces, int rest, int64_t per_row, int64_t rows, int64_t width,
                      const T *__restrict__ x, int64_t ldx, ZpDrop drop, T *__restrict__ y, int64_t ldy) {
  zp_after_previous();
  constexpr int kAhead = 4, V = kZpVec<T>;
  const ZpPhiloxKey<true> key = zp_philox_key<true>(drop.state);
  const uint32_t limit = zp_drop_limit(drop.threshold);
  const int lane = threadIdx.x % 32;
  const int64_t step = (int64_t)gridDim.x * kThreads * kAhead;
  const bool small = rows * width <= 0xffffffffll;
  if (blockIdx.x == 0 && threadIdx.x < rest) {                                 // behind the last whole counter
    const int64_t e = pieces * V + threadIdx.x, r = e / width;
    const uint32_t kept = zp_philox_kept(key, e / 8, limit) >> threadIdx.x & 1;
    y[e] = zp_rounded<T>(kept ? zp_float(x[r * ldx + e - r * width]) * drop.scale : 0.f);
  }
  for (int64_t p0 = (int64_t)(blockIdx.x * kThreads + threadIdx.x - lane) * kAhead; p0 < pieces; p0 += step) {
    uint4 in[kAhead];
    T *to[kHow == kRows ? kAhead : 1];
    const int left = (int)(pieces - p0 < 32 * kAhead ? pieces - p0 : 32 * kAhead) - lane;       // of this lane's
    if constexpr (kHow == kFlat) {
      const uint4 *const from = reinterpret_cast<const uint4 *>(x) + p0 + lane;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (32 * i < left) in[i] = __ldcs(from + 32 * i);
    } else if constexpr (kHow == kRows) {
      int64_t q = p0 + lane;                   // piece of its row
      const int64_t r = small ? (uint32_t)q / (uint32_t)per_row : q / per_row;
      q -= r * per_row;
      const T *from = x + r * ldx + q * V;
      to[0] = y + r * ldy + q * V;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (32 * i < left) in[i] = __ldcs(reinterpret_cast<const uint4 *>(from));
        if (i + 1 == kAhead) break;
        q += 32;
        from += 32 * V;
        to[i + 1] = to[i] + 32 * V;
        if (q >= per_row) {                    // rows further on
          const int64_t more = per_row >= 32 ? 1 : q / per_row;
          q -= more * per_row;
          from += more * (ldx - width);
          to[i + 1] += more * (ldy - width);
        }
      }
    } else {
      const int64_t e = (p0 + lane) * V;
      int64_t r = small ? (uint32_t)e / (uint32_t)width : e / width, c = e - r * width;      // row, column of a piece
#pragma unroll
      for (int i = 0; i < kAhead; ++i, c += 32 * V) {
        if (c >= width) {
          const int64_t more = width >= 32 * V ? 1 : c / width;
          r += more;
          c -= more * width;
        }
        if (32 * i >= left) continue;
        const char *const at = reinterpret_cast<const char *>(x + r * ldx + c);
        const int place = (int)(reinterpret_cast<uintptr_t>(at) & 15);
        const char *const from = at - place;
        const char *const end = reinterpret_cast<const char *>(x + (rows - 1) * ldx + width);
        if (c + V <= width && from >= reinterpret_cast<const char *>(x) && from + 32 <= end) {
          const uint4 a = *reinterpret_cast<const uint4 *>(from), b = *reinterpret_cast<const uint4 *>(from + 16);
          in[i] = zp_between<sizeof(T)>(a, b, place);
        } else {
          uint32_t w[4] = {0, 0, 0, 0};
          int64_t rr = r, cc = c;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const T v = x[rr * ldx + cc];
            if constexpr (sizeof(T) == 4) w[k] = *reinterpret_cast<const uint32_t *>(&v);
            else w[k / 2] |= (uint32_t)*reinterpret_cast<const uint16_t *>(&v) << (16 * (k & 1));
            if (++cc == width) { cc = 0; ++rr; }
          }
          in[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    uint32_t words[kAhead][V / 2];
    kept_words<T, kAhead>(key, p0, lane, words);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (32 * i >= left) continue;
      float2 v[V / 2];
      zp_unpack<T>(in[i], v);
#pragma unroll
      for (int k = 0; k < V / 2; ++k) v[k] = zp_drop_pair(v[k], words[i][k], limit, drop.scale);
      uint4 *const out = reinterpret_cast<uint4 *>(kHow == kRows ? to[kHow == kRows ? i : 0] : y + (p0 + lane) * V);
      __stcs(kHow == kRows ? out : out + 32 * i, zp_pack<T>(v));
    }
  }
}

// Elements wherever they lie, for results that are not row behind row or are fewer than eight.  A warp goes
// through 256 of them, works out the 32 counters and hands each lane its bits.
template <typename T>
__global__ void __launch_bounds__(kThreads)
dropout_elements_kernel(int64_t rows, int64_t width, const T *__restrict__ x, int64_t ldx, ZpDrop drop,
                        T *__restrict__ y, int64_t ldy) {
  zp_after_previous();
  const ZpPhiloxKey<true> key = zp_philox_key<true>(drop.state);
  const uint32_t limit = zp_drop_limit(drop.threshold);
  const int lane = threadIdx.x % 32;
  const int64_t n = rows * width, step = (int64_t)gridDim.x * kThreads * 8;
  for (int64_t e0 = (int64_t)(blockIdx.x * kThreads + threadIdx.x - lane) * 8; e0 < n; e0 += step) {
    const uint32_t mine = zp_philox_kept(key, e0 / 8 + lane, limit);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t kept = __shfl_sync(0xffffffffu, mine, 4 * j + lane / 8) >> (lane % 8) & 1;
      const int64_t e = e0 + 32 * j + lane;
      if (e >= n) continue;
      const int64_t r = e / width, c = e - r * width;
      y[r * ldy + c] = zp_rounded<T>(kept ? zp_float(x[r * ldx + c]) * drop.scale : 0.f);
    }
  }
}

template <typename P>
__device__ __forceinline__ float param(const P *w, int64_t c, float otherwise) {
  return w ? zp_float(w[c]) : otherwise;
}

// Rows that no team holds (above 65536 elements, 32768 in the backward; shifted ones above 8192): one block
// per row, passes over global memory.
template <typename T, typename P>
__global__ void __launch_bounds__(kThreads)
norm_fwd_kernel(int64_t rows, int64_t width, const T *__restrict__ x, int64_t ldx, const T *__restrict__ res,
                int64_t ldr, ZpDrop drop, const P *__restrict__ w, const P *__restrict__ b, float eps,
                T *__restrict__ sum, T *__restrict__ y, float *__restrict__ mean_out, float *__restrict__ rstd_out) {
  zp_after_previous();
  __shared__ float red[kThreads / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *in = x + r * ldx;
    if (res) {
      const ZpPhiloxKey<false> key = drop.state ? zp_philox_key<false>(drop.state) : ZpPhiloxKey<false>{};
      for (int64_t c = threadIdx.x; c < width; c += kThreads) {
        const uint64_t i = (uint64_t)(r * width + c);
        const bool kept = !drop.state || (zp_philox_kept(key, i / 8, zp_drop_limit(drop.threshold)) >> (i % 8) & 1);
        sum[r * width + c] = zp_rounded<T>(zp_float(res[r * ldr + c]) +
                                           (kept ? zp_float(in[c]) * drop.scale : 0.f));
      }
      in = sum + r * width;                    // (each thread reads again what it has written)
    }
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += kThreads) s += zp_float(in[c]);
    const float mean = block_sum(s, red) / (float)width;
    float q = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
      const float d = zp_float(in[c]) - mean;
      q += d * d;
    }
    const float rstd = rsqrtf(block_sum(q, red) / (float)width + eps);
    for (int64_t c = threadIdx.x; c < width; c += kThreads)
      y[r * width + c] = zp_rounded<T>((zp_float(in[c]) - mean) * rstd * param(w, c, 1.f) + param(b, c, 0.f));
    if (mean_out && threadIdx.x == 0) { mean_out[r] = mean; rstd_out[r] = rstd; }
  }
}

// gradient of the rows: dsum is added, dres takes the sum, dx what dropout leaves of it
template <typename T, typename P>
__global__ void __launch_bounds__(kThreads)
norm_bwd_kernel(int64_t rows, int64_t width, const T *__restrict__ x, int64_t ldx, const P *__restrict__ w,
                const float *__restrict__ mean_in, const float *__restrict__ rstd_in, const T *__restrict__ dy,
                int64_t ldy, const T *__restrict__ dsum, int64_t lds, ZpDrop drop, T *__restrict__ dx,
                T *__restrict__ dres) {
  zp_after_previous();
  __shared__ float red[kThreads / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mean = mean_in[r], rstd = rstd_in[r];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; dy && c < width; c += kThreads) {
      const float gz = zp_float(dy[r * ldy + c]) * param(w, c, 1.f);
      s1 += gz;
      s2 += gz * ((zp_float(x[r * ldx + c]) - mean) * rstd);
    }
    const float m1 = block_sum(s1, red) / (float)width, m2 = block_sum(s2, red) / (float)width;
    const ZpPhiloxKey<false> key = drop.state ? zp_philox_key<false>(drop.state) : ZpPhiloxKey<false>{};
    for (int64_t c = threadIdx.x; c < width; c += kThreads) {
      float g = 0.f;
      if (dy) {
        const float z = (zp_float(x[r * ldx + c]) - mean) * rstd;
        g = rstd * (zp_float(dy[r * ldy + c]) * param(w, c, 1.f) - m1 - z * m2);
      }
      if (dsum) g += zp_float(dsum[r * lds + c]);
      if (dres) dres[r * width + c] = zp_rounded<T>(g);
      if (dx) {
        const uint64_t i = (uint64_t)(r * width + c);
        const bool kept = !drop.state || (zp_philox_kept(key, i / 8, zp_drop_limit(drop.threshold)) >> (i % 8) & 1);
        dx[r * width + c] = zp_rounded<T>(kept ? g * drop.scale : 0.f);
      }
    }
  }
}

// partial sums of the parameters' gradients over the rows of blockIdx.y, then over those
template <typename T>
__global__ void __launch_bounds__(kThreads)
norm_params_kernel(int64_t rows, int64_t width, const T *__restrict__ x, int64_t ldx,
                   const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                   const T *__restrict__ dy, int64_t ldy, float *__restrict__ partial) {
  zp_after_previous();
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= width) return;
  float gw = 0.f, gb = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = zp_float(dy[r * ldy + c]);
    gw += g * ((zp_float(x[r * ldx + c]) - mean_in[r]) * rstd_in[r]);
    gb += g;
  }
  partial[(2 * (int64_t)blockIdx.y) * width + c] = gw;
  partial[(2 * (int64_t)blockIdx.y + 1) * width + c] = gb;
}

// the last sums: 32 columns to a block, the parts dealt out to 32 threads each
template <typename P>
__global__ void __launch_bounds__(1024)
norm_params_last_kernel(int64_t width, int parts, const float *__restrict__ partial, P *__restrict__ dw,
                        P *__restrict__ db) {
  zp_after_previous();
  __shared__ float red[32][33];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;           // of {gw, gb} side by side
  float s = 0.f;
#pragma unroll 4
  for (int i = ty; i < parts; i += 32) s += c < 2 * width ? partial[(int64_t)i * 2 * width + c] : 0.f;
  red[ty][tx] = s;
  __syncthreads();
  if (ty != 0 || c >= 2 * width) return;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += red[i][tx];
  P *const out = c < width ? dw : db;
  if (out) out[c < width ? c : c - width] = zp_rounded<P>(s);
}


// dropout of probability p (0 <= p <= 1), rounded to a multiple of 2^-16
bool make_drop(double p, const int64_t *state, ZpDrop &drop) {
  drop = {nullptr, 0, 1.f};
  if (!(p >= 0.0 && p <= 1.0)) return false;
  drop.threshold = (uint32_t)std::floor(65536.0 * p + 0.5);
  if (drop.threshold == 0) return true;
  drop.state = state;
  drop.scale = drop.threshold < 65536 ? (float)(65536.0 / (65536 - drop.threshold)) : 0.f;
  return state != nullptr && !misplaced(state, 8);
}

size_t type_bytes(int dtype) { return dtype == ZP_F32 ? 4 : dtype == ZP_F16 || dtype == ZP_BF16 ? 2 : 0; }

// a matrix of rows `ld` elements apart: its address a multiple of an element's size
bool bad_rows(const void *p, int64_t rows, int64_t width, int64_t ld, int dtype) {
  return !p || ld < width || (rows > 1 && ld > INT64_MAX / rows / 4) ||
         misplaced(p, type_bytes(dtype));
}

int check_sizes(int64_t rows, int64_t width, int dtype) {
  if (rows < 0 || width < 1) return ZP_ERR_INVALID_ARG;
  if (!type_bytes(dtype)) return ZP_ERR_UNSUPPORTED;
  return rows > INT64_MAX / width / 4 ? ZP_ERR_UNSUPPORTED : ZP_OK;
}

unsigned blocks_for(int64_t n, int64_t most) { return (unsigned)std::max<int64_t>(1, std::min(n, most)); }

template <typename T> int run_dropout(int64_t rows, int64_t width, const void *x, int64_t ldx, const ZpDrop &drop,
                                      void *y, int64_t ldy, cudaStream_t st) {
  constexpr int V = kZpVec<T>;
  const T *in = static_cast<const T *>(x);
  T *out = static_cast<T *>(y);
  const bool behind = ldy == width || rows == 1;             // y lies row behind row
  if (behind && (ldx == width || rows == 1)) {               // one row from end to end
    width *= rows;
    rows = 1;
    ldx = ldy = width;
  }
  const bool whole = !misplaced(x, 16) && !misplaced(y, 16) &&
                     (rows == 1 || (width % 8 == 0 && ldx % V == 0 && ldy % V == 0));
  if (whole || (behind && !misplaced(y, 16))) {
    const int64_t first = rows * width / 8 * 8;              // elements that go by pieces, whole counters of them
    const int64_t pieces = first / V;
    const unsigned blocks = blocks_for(zp_ceil_div(pieces, 4 * kThreads), 148 * 8);
    if (pieces > 0) {
      const auto kernel = !whole      ? dropout_pieces_kernel<T, kGather>
                          : rows == 1 ? dropout_pieces_kernel<T, kFlat>
                                      : dropout_pieces_kernel<T, kRows>;
      const int rest = (int)(rows * width - first);          // (none where rows are whole counters)
      zp_launch(kernel, blocks, kThreads, 0, st, pieces, rest, width / V, rows, width, in, ldx, drop, out, ldy);
      ZP_LAUNCH_CHECK("dropout_pieces_kernel");
      return ZP_OK;
    }
  }
  zp_launch(dropout_elements_kernel<T>, blocks_for(zp_ceil_div(rows * width, 8 * kThreads), 148 * 8), kThreads, 0, st,
            rows, width, in, ldx, drop, out, ldy);
  ZP_LAUNCH_CHECK("dropout_elements_kernel");
  return ZP_OK;
}

template <typename T, typename P> int run_fwd(const ZpNormCall &c, cudaStream_t st) {
  bool taken = false;
  if (int rc = zp_launch_norm_fwd(c, taken, st)) return rc;
  if (taken) return ZP_OK;
  zp_launch(norm_fwd_kernel<T, P>, blocks_for(c.rows, 148 * 8), kThreads, 0, st, c.rows, c.width,
            static_cast<const T *>(c.x), c.ldx, static_cast<const T *>(c.res), c.ldr, c.drop,
            static_cast<const P *>(c.w), static_cast<const P *>(c.b), c.eps, static_cast<T *>(c.sum),
            static_cast<T *>(c.y), c.mean, c.rstd);
  ZP_LAUNCH_CHECK("norm_fwd_kernel");
  return ZP_OK;
}

template <typename T, typename P> int run_bwd(const ZpNormCall &c, cudaStream_t st) {
  const T *x = static_cast<const T *>(c.x), *dy = static_cast<const T *>(c.dy);
  bool taken = false;
  int parts = 0;
  if (int rc = zp_launch_norm_bwd(c, taken, parts, st)) return rc;
  if (!taken && (c.dx || c.dres)) {
    zp_launch(norm_bwd_kernel<T, P>, blocks_for(c.rows, 148 * 8), kThreads, 0, st, c.rows, c.width, x, c.ldx,
              static_cast<const P *>(c.w), c.mean_in, c.rstd_in, dy, c.ldy, static_cast<const T *>(c.dsum), c.lds,
              c.drop, static_cast<T *>(c.dx), static_cast<T *>(c.dres));
    ZP_LAUNCH_CHECK("norm_bwd_kernel");
  }
  if (!c.partial) return ZP_OK;
  if (!taken) {
    parts = (int)blocks_for(c.rows, ZP_ROWWISE_PARTS);
    zp_launch(norm_params_kernel<T>, dim3((unsigned)zp_ceil_div(c.width, kThreads), parts), kThreads, 0, st, c.rows,
              c.width, x, c.ldx, c.mean_in, c.rstd_in, dy, c.ldy, c.partial);
    ZP_LAUNCH_CHECK("norm_params_kernel");
  }
  zp_launch(norm_params_last_kernel<P>, (unsigned)zp_ceil_div(2 * c.width, 32), 1024, 0, st, c.width, parts, c.partial,
            static_cast<P *>(c.dw), static_cast<P *>(c.db));
  ZP_LAUNCH_CHECK("norm_params_last_kernel");
  return ZP_OK;
}

#define BY_TYPES(CALL)                                                              \
  switch (dtype) {                                                                  \
    case ZP_F32: return CALL<float, float>(c, st);                                  \
    case ZP_F16:                                                                    \
      return param_dtype == ZP_F32 ? CALL<__half, float>(c, st) : CALL<__half, __half>(c, st); \
    default:                                                                        \
      return param_dtype == ZP_F32 ? CALL<__nv_bfloat16, float>(c, st)              \
                                   : CALL<__nv_bfloat16, __nv_bfloat16>(c, st);     \
  }

int norm_fwd(ZpNormCall &c, int dtype, int param_dtype, cudaStream_t st) {
  c.dtype = dtype;
  c.param_dtype = param_dtype;
  BY_TYPES(run_fwd)
}
int norm_bwd(ZpNormCall &c, int dtype, int param_dtype, void *work, cudaStream_t st) {
  c.dtype = dtype;
  c.param_dtype = param_dtype;
  c.partial = c.dw || c.db ? static_cast<float *>(work) : nullptr;
  BY_TYPES(run_bwd)
}
#undef BY_TYPES

bool bad_param_type(int dtype, int param_dtype) { return param_dtype != dtype && param_dtype != ZP_F32; }

int check_fwd(const ZpNormCall &c, int dtype, int param_dtype) {
  if (bad_param_type(dtype, param_dtype)) return ZP_ERR_UNSUPPORTED;
  if (bad_rows(c.x, c.rows, c.width, c.ldx, dtype) || bad_rows(c.y, c.rows, c.width, c.width, dtype) ||
      misplaced(c.w, type_bytes(param_dtype)) || misplaced(c.b, type_bytes(param_dtype)) ||
      (c.mean == nullptr) != (c.rstd == nullptr) || misplaced(c.mean, 4) || misplaced(c.rstd, 4))
    return ZP_ERR_INVALID_ARG;
  return ZP_OK;
}

int zero_params(const ZpNormCall &c, int param_dtype, cudaStream_t st) {
  const size_t bytes = (size_t)c.width * type_bytes(param_dtype);
  if (c.dw) ZP_CUDA(cudaMemsetAsync(c.dw, 0, bytes, st));
  if (c.db) ZP_CUDA(cudaMemsetAsync(c.db, 0, bytes, st));
  return ZP_OK;
}

int check_bwd(const ZpNormCall &c, int dtype, int param_dtype, const void *work, size_t work_bytes) {
  const size_t size = type_bytes(dtype), psize = type_bytes(param_dtype);
  if (bad_rows(c.x, c.rows, c.width, c.ldx, dtype) || (c.dy && bad_rows(c.dy, c.rows, c.width, c.ldy, dtype)) ||
      !c.mean_in || !c.rstd_in || misplaced(c.mean_in, 4) || misplaced(c.rstd_in, 4) || misplaced(c.w, psize) ||
      misplaced(c.dx, size) || misplaced(c.dres, size) || misplaced(c.dw, psize) || misplaced(c.db, psize))
    return ZP_ERR_INVALID_ARG;
  if (c.dw || c.db) {
    if (!work || misplaced(work, 16)) return ZP_ERR_INVALID_ARG;
    if (work_bytes < zp_rowwise_work_bytes(c.rows, c.width)) return ZP_ERR_WORKSPACE;
  }
  return ZP_OK;
}

}  // namespace

extern "C" {

int zp_dropout(int64_t rows, int64_t width, int dtype, const void *x, int64_t ldx, double p, const int64_t *state,
               void *y, int64_t ldy, void *stream) {
  if (int rc = check_sizes(rows, width, dtype)) return rc;
  ZpDrop drop;
  if (rows == 0) return p >= 0.0 && p <= 1.0 ? ZP_OK : ZP_ERR_INVALID_ARG;
  if (!make_drop(p, state, drop) || !state || misplaced(state, 8) || bad_rows(x, rows, width, ldx, dtype) ||
      bad_rows(y, rows, width, ldy, dtype))
    return ZP_ERR_INVALID_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const size_t size = type_bytes(dtype);
  if (!drop.state) {                           // nothing is dropped
    if ((ldx == width && ldy == width) || rows == 1)
      ZP_CUDA(cudaMemcpyAsync(y, x, rows * width * size, cudaMemcpyDeviceToDevice, st));
    else
      ZP_CUDA(cudaMemcpy2DAsync(y, ldy * size, x, ldx * size, width * size, rows, cudaMemcpyDeviceToDevice, st));
    return ZP_OK;
  }
  if (dtype == ZP_F32) return run_dropout<float>(rows, width, x, ldx, drop, y, ldy, st);
  if (dtype == ZP_F16) return run_dropout<__half>(rows, width, x, ldx, drop, y, ldy, st);
  return run_dropout<__nv_bfloat16>(rows, width, x, ldx, drop, y, ldy, st);
}

size_t zp_rowwise_work_bytes(int64_t rows, int64_t width) {
  return rows > 0 && width > 0 ? sizeof(float) * 2 * (size_t)std::min<int64_t>(rows + 7, ZP_ROWWISE_PARTS) * (size_t)width : 0;
}

int zp_layernorm_forward(int64_t rows, int64_t width, int dtype, const void *x, int64_t ldx, int param_dtype,
                         const void *weight, const void *bias, float eps, void *y, float *mean, float *rstd,
                         void *stream) {
  if (int rc = check_sizes(rows, width, dtype)) return rc;
  if (rows == 0) return ZP_OK;
  ZpNormCall c = {};
  c.rows = rows; c.width = width; c.x = x; c.ldx = ldx; c.w = weight; c.b = bias; c.eps = eps; c.y = y;
  c.mean = mean; c.rstd = rstd; c.drop.scale = 1.f;
  if (int rc = check_fwd(c, dtype, param_dtype)) return rc;
  return norm_fwd(c, dtype, param_dtype, (cudaStream_t)stream);
}

int zp_layernorm_backward(int64_t rows, int64_t width, int dtype, const void *x, int64_t ldx, int param_dtype,
                          const void *weight, const float *mean, const float *rstd, const void *dy, int64_t ldy,
                          void *dx, void *dweight, void *dbias, void *work, size_t work_bytes, void *stream) {
  if (int rc = check_sizes(rows, width, dtype)) return rc;
  if (bad_param_type(dtype, param_dtype)) return ZP_ERR_UNSUPPORTED;
  ZpNormCall c = {};
  c.rows = rows; c.width = width; c.x = x; c.ldx = ldx; c.w = weight; c.mean_in = mean; c.rstd_in = rstd;
  c.dy = dy; c.ldy = ldy; c.dx = dx; c.dw = dweight; c.db = dbias;
  c.drop.scale = 1.f;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) return zero_params(c, param_dtype, st);
  if (!dy) return ZP_ERR_INVALID_ARG;
  if (int rc = check_bwd(c, dtype, param_dtype, work, work_bytes)) return rc;
  return norm_bwd(c, dtype, param_dtype, work, st);
}

int zp_add_layernorm_forward(int64_t rows, int64_t width, int dtype, const void *x, int64_t ldx,
                             const void *residual, int64_t ldr, double p, const int64_t *state, int param_dtype,
                             const void *weight, const void *bias, float eps, void *sum, void *y, float *mean,
                             float *rstd, void *stream) {
  if (int rc = check_sizes(rows, width, dtype)) return rc;
  ZpNormCall c = {};
  if (rows == 0) return p >= 0.0 && p <= 1.0 ? ZP_OK : ZP_ERR_INVALID_ARG;
  if (!make_drop(p, state, c.drop)) return ZP_ERR_INVALID_ARG;
  c.rows = rows; c.width = width; c.x = x; c.ldx = ldx; c.res = residual; c.ldr = ldr; c.w = weight; c.b = bias;
  c.eps = eps; c.sum = sum; c.y = y; c.mean = mean; c.rstd = rstd;
  if (bad_rows(residual, rows, width, ldr, dtype) || bad_rows(sum, rows, width, width, dtype))
    return ZP_ERR_INVALID_ARG;
  if (int rc = check_fwd(c, dtype, param_dtype)) return rc;
  return norm_fwd(c, dtype, param_dtype, (cudaStream_t)stream);
}

int zp_add_layernorm_backward(int64_t rows, int64_t width, int dtype, const void *sum, int param_dtype,
                              const void *weight, const float *mean, const float *rstd, const void *dy, int64_t ldy,
                              const void *dsum, int64_t lds, double p, const int64_t *state, void *dx,
                              void *dresidual, void *dweight, void *dbias, void *work, size_t work_bytes,
                              void *stream) {
  if (int rc = check_sizes(rows, width, dtype)) return rc;
  if (bad_param_type(dtype, param_dtype)) return ZP_ERR_UNSUPPORTED;
  ZpNormCall c = {};
  c.rows = rows; c.width = width; c.x = sum; c.ldx = width; c.w = weight; c.mean_in = mean; c.rstd_in = rstd;
  c.dy = dy; c.ldy = ldy; c.dsum = dsum; c.lds = lds; c.dx = dx; c.dres = dresidual; c.dw = dweight; c.db = dbias;
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) return p >= 0.0 && p <= 1.0 ? zero_params(c, param_dtype, st) : (int)ZP_ERR_INVALID_ARG;
  if (!make_drop(p, state, c.drop)) return ZP_ERR_INVALID_ARG;
  if (!dy && !dsum) return ZP_ERR_INVALID_ARG;
  if (dsum && bad_rows(dsum, rows, width, lds, dtype)) return ZP_ERR_INVALID_ARG;
  if (int rc = check_bwd(c, dtype, param_dtype, work, work_bytes)) return rc;
  if (!dy) {                                   // the sum alone went on: nothing reaches the parameters
    if (int rc = zero_params(c, param_dtype, st)) return rc;
    c.dw = c.db = nullptr;
    if (!dx && !dresidual) return ZP_OK;
  }
  return norm_bwd(c, dtype, param_dtype, work, st);
}

}  // extern "C"
