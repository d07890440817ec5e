// Backward of the layer norm over rows, alone and with the residual sum and dropout in front of it: the
// rows' gradient and, from the same reading of the rows, partial sums of the parameters' gradients.
//
// A thread has the same columns in every row of its team, so the sums over rows stay in its registers;
// at the end the teams of a block add theirs up in a fixed order and the block writes one partial row of
// each, which a second kernel adds in block order.
#include "zp_rowwise.cuh"

namespace {

template <typename T, bool kAligned, int E, int R, bool kJoin>
__global__ void __launch_bounds__(kZpTeamThreads, 1)
norm_bwd_team_kernel(const ZpNormCall c, const ZpTeamPlan p) {
  zp_after_previous();
  constexpr int V = kZpVec<T>, H = V / 2, M = E / V;
  constexpr bool kHeld = E <= 16;              // the weight, z and gy w stay in registers
  extern __shared__ __align__(16) char smem[];
  const ZpTeam t(p.team, reinterpret_cast<float *>(smem));
  const int width = (int)c.width, teams = kZpTeamThreads / p.team, stages = p.stages;
  char *const after_red = smem + sizeof(float) * 2 * 4 * kZpTeamWarps;
  uint8_t *const bytes = reinterpret_cast<uint8_t *>(after_red) + t.index * p.bytes;
  char *const rings = after_red + p.bytes * teams;
  const int A = kJoin && c.dsum ? 3 : 2;
  char *const ring = rings + (size_t)t.index * stages * A * R * p.slot;
  const int64_t step = (int64_t)gridDim.x * t.walkers * t.per * R;
  const int64_t first = ((int64_t)t.walker * gridDim.x + blockIdx.x) * t.per * R + t.sub;
  ZpSource sx(c.x, c.ldx, c.rows, c.width, sizeof(T), first, step, t.per);
  ZpSource sy(c.dy, c.ldy, c.rows, c.width, sizeof(T), first, step, t.per);
  ZpSource ss(c.dsum, c.lds, c.rows, c.width, sizeof(T), first, step, t.per);
  int64_t coming = first;
  auto fetch = [&](int stage) {
    char *to = ring + stage * A * R * p.slot;
#pragma unroll
    for (int j = 0; j < R; ++j, to += A * p.slot) {
      if (coming + j * t.per >= c.rows) continue;
      zp_fetch_row<T, kAligned, M>(t, to, sx, sx.row + j * sx.next, width);
      zp_fetch_row<T, kAligned, M>(t, to + p.slot, sy, sy.row + j * sy.next, width);
      if (kJoin && A == 3) zp_fetch_row<T, kAligned, M>(t, to + 2 * p.slot, ss, ss.row + j * ss.next, width);
    }
    sx.row += sx.step;
    sy.row += sy.step;
    ss.row += ss.step;
    coming += step;
    zp_copy_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(s);

  const bool wide = c.param_dtype == ZP_F32;
  auto column = [&](int i) { return (t.lane + i * t.size) * V; };
  float2 w[kHeld ? M : 1][H], gw[M][H], gb[M][H];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    if constexpr (kHeld) zp_params<T>(c.w, wide, p.vectors, column(i), width, 1.f, w[i]);
#pragma unroll
    for (int k = 0; k < H; ++k) gw[i][k] = gb[i][k] = make_float2(0.f, 0.f);
  }
  const ZpPhiloxKey key = kJoin && c.drop.state ? zp_philox_key(c.drop.state) : ZpPhiloxKey{};
  const float inv_w = 1.f / (float)width;
  const int64_t row_bytes = c.width * (int64_t)sizeof(T);
  float next_mean[R], next_rstd[R];
  auto load_stats = [&](int64_t r0) {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (r0 + j * t.per < c.rows) {
        next_mean[j] = c.mean_in[r0 + j * t.per];
        next_rstd[j] = c.rstd_in[r0 + j * t.per];
      }
  };
#pragma unroll
  for (int j = 0; j < R; ++j) next_mean[j] = next_rstd[j] = 0.f;
  load_stats(first);
  int stage = 0, turn = 0;
  for (int64_t r0 = first; r0 - t.sub < c.rows; r0 += step) {
    float mean[R], rstd[R], s[2 * R];
#pragma unroll
    for (int j = 0; j < R; ++j) { mean[j] = next_mean[j]; rstd[j] = next_rstd[j]; }
    zp_copy_wait(stages);
    if (!kAligned) t.sync();
    fetch(stage == 0 ? stages - 1 : stage - 1);
    load_stats(r0 + step);
    char *const slots = ring + stage * A * R * p.slot;
    stage = stage + 1 == stages ? 0 : stage + 1;
    float2 z[kHeld ? R : 1][M][H], g[kHeld ? R : 1][M][H];
    int mine[R];
    // z and gy w of row j, piece i, from the slots
    auto load = [&](int j, int i, float2 (&zz)[H], float2 (&gy)[H]) {
      zp_read<T, kAligned>(t, slots + j * A * p.slot, sx.place_of(j), i, width, zz);
      zp_read<T, kAligned>(t, slots + (j * A + 1) * p.slot, sy.place_of(j), i, width, gy);
      const float2 minus = make_float2(-mean[j], -mean[j]), by = make_float2(rstd[j], rstd[j]);
#pragma unroll
      for (int k = 0; k < H; ++k) zz[k] = __fmul2_rn(__fadd2_rn(zz[k], minus), by);
    };
#pragma unroll
    for (int j = 0; j < R; ++j) {
      mine[j] = r0 + j * t.per < c.rows ? width : 0;
      float2 s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (column(i) >= mine[j]) continue;
        float2 (&zz)[H] = z[kHeld ? j : 0][i], (&gz)[H] = g[kHeld ? j : 0][i];
        load(j, i, zz, gz);
        float2 ww[H];
        if constexpr (!kHeld) zp_params<T>(c.w, wide, p.vectors, column(i), width, 1.f, ww);
#pragma unroll
        for (int k = 0; k < H; ++k) {
          gw[i][k] = __ffma2_rn(gz[k], zz[k], gw[i][k]);
          gb[i][k] = __fadd2_rn(gb[i][k], gz[k]);
          gz[k] = __fmul2_rn(gz[k], kHeld ? w[kHeld ? i : 0][k] : ww[k]);
          s1 = __fadd2_rn(s1, gz[k]);
          s2 = __ffma2_rn(gz[k], zz[k], s2);
        }
      }
      s[2 * j] = s1.x + s1.y;
      s[2 * j + 1] = s2.x + s2.y;
    }
    t.sum(s, turn++, !kAligned);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t r = r0 + j * t.per;
      uint32_t kept = 0xffffffffu;
      if (kJoin && c.drop.state)
        kept = zp_kept_bits<T, kAligned, E>(t, key, c.drop.threshold, mine[j] ? r : 0, width, bytes);
      const float2 minus1 = make_float2(-s[2 * j] * inv_w, -s[2 * j] * inv_w);
      const float2 minus2 = make_float2(-s[2 * j + 1] * inv_w, -s[2 * j + 1] * inv_w);
      const float2 by = make_float2(rstd[j], rstd[j]);
      char *const slot = slots + j * A * p.slot;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (column(i) >= mine[j]) continue;
        float2 o[H], q[H];
        if constexpr (kHeld) {
#pragma unroll
          for (int k = 0; k < H; ++k)
            o[k] = __fmul2_rn(__ffma2_rn(z[j][i][k], minus2, __fadd2_rn(g[j][i][k], minus1)), by);
        } else {
          float2 zz[H], ww[H];
          load(j, i, zz, q);
          zp_params<T>(c.w, wide, p.vectors, column(i), width, 1.f, ww);
#pragma unroll
          for (int k = 0; k < H; ++k)
            o[k] = __fmul2_rn(__ffma2_rn(zz[k], minus2, __ffma2_rn(q[k], ww[k], minus1)), by);
        }
        if constexpr (!kJoin) {
          if (c.dx) zp_write<T, kAligned>(t, static_cast<char *>(c.dx) + r * row_bytes, slot, i, o);
          continue;
        }
        if (A == 3) {
          zp_read<T, kAligned>(t, slot + 2 * p.slot, ss.place_of(j), i, width, q);
#pragma unroll
          for (int k = 0; k < H; ++k) o[k] = __fadd2_rn(o[k], q[k]);
        }
        if (c.dres) zp_write<T, kAligned>(t, static_cast<char *>(c.dres) + r * row_bytes, slot, i, o);
        if (!c.dx) continue;
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const uint32_t two = kept >> (i * V + 2 * k);
          o[k] = make_float2(two & 1 ? o[k].x * c.drop.scale : 0.f, two & 2 ? o[k].y * c.drop.scale : 0.f);
        }
        zp_write<T, kAligned>(t, static_cast<char *>(c.dx) + r * row_bytes, slot + p.slot, i, o);
      }
    }
    if constexpr (!kAligned) {
      t.sync();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int64_t r = r0 + j * t.per;
        if (!mine[j]) continue;
        char *const slot = slots + j * A * p.slot;
        if (kJoin && c.dres) zp_store_row<T>(t, static_cast<char *>(c.dres) + r * row_bytes, slot, width);
        if (c.dx) zp_store_row<T>(t, static_cast<char *>(c.dx) + r * row_bytes, slot + (kJoin ? p.slot : 0), width);
      }
    }
    sx.advance();
    sy.advance();
    ss.advance();
  }
  zp_copy_wait(2);
  if (!c.partial) return;
  // teams within a warp first, then those of the block (`copies` of them) through shared memory, in order
  for (int o = t.size; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int k = 0; k < H; ++k) {
        gw[i][k].x += __shfl_xor_sync(0xffffffffu, gw[i][k].x, o);
        gw[i][k].y += __shfl_xor_sync(0xffffffffu, gw[i][k].y, o);
        gb[i][k].x += __shfl_xor_sync(0xffffffffu, gb[i][k].x, o);
        gb[i][k].y += __shfl_xor_sync(0xffffffffu, gb[i][k].y, o);
      }
  }
  float *const all = reinterpret_cast<float *>(rings);           // [copies][2][row]
  const int row = t.size * E, copies = t.walkers;
  __syncthreads();                                               // the rings are done with
  if (t.sub == 0) {
    float *const mine = all + (size_t)t.walker * 2 * row;
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int k = 0; k < H; ++k) {
        *reinterpret_cast<float2 *>(mine + column(i) + 2 * k) = gw[i][k];
        *reinterpret_cast<float2 *>(mine + row + column(i) + 2 * k) = gb[i][k];
      }
  }
  __syncthreads();
  float *const out = c.partial + (size_t)blockIdx.x * 2 * c.width;
  for (int i = threadIdx.x; i < 2 * width; i += kZpTeamThreads) {
    const int at = i < width ? i : row + (i - width);
    float sum = 0.f;
    for (int k = 0; k < copies; ++k) sum += all[(size_t)k * 2 * row + at];
    out[i] = sum;
  }
}

template <typename T, bool kAligned, int E, int R, bool kJoin>
int launch(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  static ZpSmemOptIn opt_in;
  if (int rc = zp_ensure_smem(norm_bwd_team_kernel<T, kAligned, E, R, kJoin>, p.smem, opt_in)) return rc;
  zp_launch(norm_bwd_team_kernel<T, kAligned, E, R, kJoin>, p.blocks, kZpTeamThreads, p.smem, st, c, p);
  ZP_LAUNCH_CHECK("norm_bwd_team_kernel");
  return ZP_OK;
}
template <typename T, bool kAligned, bool kJoin>
int by_elements(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  if (p.elements == 8) return p.rows == 1 ? launch<T, kAligned, 8, 1, kJoin>(c, p, st) : launch<T, kAligned, 8, 2, kJoin>(c, p, st);
  return p.elements == 16 ? launch<T, kAligned, 16, 1, kJoin>(c, p, st) : launch<T, kAligned, 32, 1, kJoin>(c, p, st);
}
template <typename T> int by_kind(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  if (c.dsum || c.dres || c.drop.state)
    return p.aligned ? by_elements<T, true, true>(c, p, st) : by_elements<T, false, true>(c, p, st);
  return p.aligned ? by_elements<T, true, false>(c, p, st) : by_elements<T, false, false>(c, p, st);
}

}  // namespace

int zp_launch_norm_bwd(const ZpNormCall &c, bool &taken, int &parts, cudaStream_t st) {
  const size_t size = c.dtype == ZP_F32 ? 4 : 2;
  const bool aligned = (c.width * size) % 16 == 0 && zp_piece_aligned(c.x, c.ldx, size) &&
                       zp_piece_aligned(c.dy, c.ldy, size) && (!c.dsum || zp_piece_aligned(c.dsum, c.lds, size)) &&
                       (!c.dx || zp_piece_aligned(c.dx, c.width, size)) &&
                       (!c.dres || zp_piece_aligned(c.dres, c.width, size)) &&
                       (!c.drop.state || c.width % 8 == 0);
  const int64_t n = c.rows * c.width, threads = (int64_t)148 * kZpTeamThreads;
  const int arrays = c.dsum ? 3 : 2;
  const size_t last = c.partial ? 2 * sizeof(float) : 0;
  ZpTeamPlan p;
  taken = c.dy && ((n >= threads * 32 && zp_team_plan(c, aligned, arrays, last, 8, 2, p)) ||
                   zp_team_plan(c, aligned, arrays, last, 8, 1, p) || zp_team_plan(c, aligned, arrays, last, 16, 1, p) ||
                   zp_team_plan(c, aligned, arrays, last, 32, 1, p));
  if (!taken) return ZP_OK;
  parts = (int)p.blocks;
  if (c.dtype == ZP_F32) return by_kind<float>(c, p, st);
  if (c.dtype == ZP_F16) return by_kind<__half>(c, p, st);
  return by_kind<__nv_bfloat16>(c, p, st);
}
