// Backward of the layer norm over rows, alone and with the residual sum and dropout in front of it: the
// rows' gradient and, from the same reading of the rows, partial sums of the parameters' gradients.
//
// A thread has the same columns in every row of its team, so the sums over rows stay in its registers;
// at the end the teams of a block add theirs up in a fixed order and the block writes one partial row of
// each, which a second kernel adds in block order (148 rows at most: 2 % of what 16384 x 4096 bf16 moves; that
// kernel takes 1.9 us by itself).
//
// B200, both kernels (share of 6 450 GB/s): 8192 x 4096 fp32 66 us (0.94), 16384 x 4096 bf16 74 (0.85; 20 instructions
// an element, 55 % of the issue slots at sixteen warps: their registers hold the rows, the sums and the weight), joined
// with dropout 132 (0.79; 41 instructions), 60000 x 128 fp32 19.7 (0.72), 30011 x 1001 fp16 52 (0.54).
#include "zp_rowwise.cuh"

namespace {

template <typename T, int kLying, bool kFull, int E, int R, bool kJoin, bool kWide>
__global__ void __launch_bounds__(kZpTeamThreads, 1)
norm_bwd_team_kernel(const __grid_constant__ ZpNormCall c, const __grid_constant__ ZpTeamPlan p) {
  zp_after_previous();
  constexpr int V = kZpVec<T>, H = V / 2, M = E / V;
  extern __shared__ __align__(16) char smem[];
  const ZpTeam<kWide> t(p.team, p.ranks, reinterpret_cast<float *>(smem));
  const int width = (int)c.width, stages = p.stages;
  char *const after_red = smem + kZpSumsBytes;
  uint8_t *const bytes = reinterpret_cast<uint8_t *>(after_red) + t.index * p.bytes;
  char *const rings = after_red + p.bytes * (kZpTeamThreads / p.team);
  const bool third = kJoin && c.dsum;          // of the arrays that come in
  const uint32_t row_slots = (third ? 3 : 2) * p.slot, stage_bytes = R * row_slots, ring_bytes = stages * stage_bytes;
  const uint32_t ring = zp_shared(rings) + t.index * ring_bytes;
  const ZpTeamRows<kLying, R> own(t, c.rows, width, p.cycle);
  ZpSource<kLying> sx(t, c.x, c.ldx, c.rows, c.width, sizeof(T), own);
  ZpSource<kLying> sy(t, c.dy, c.ldy, c.rows, c.width, sizeof(T), own);
  ZpSource<kLying> ss(t, c.dsum, c.lds, c.rows, c.width, sizeof(T), own);
  auto fetch = [&](int turn, uint32_t to) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (turn >= own.n[j]) continue;
      const uint32_t slot = to + j * row_slots;
      zp_fetch_row<T, kLying, kFull, M>(t, slot, sx, j, width, own.before);
      zp_fetch_row<T, kLying, kFull, M>(t, slot + p.slot, sy, j, width, own.before);
      if (third) zp_fetch_row<T, kLying, kFull, M>(t, slot + 2 * p.slot, ss, j, width, own.before);
    }
    sx.row += sx.step;
    sy.row += sy.step;
    if (kJoin) ss.row += ss.step;
    zp_copy_commit();
  };
  auto column = [&](int i) { return t.piece(i) * V - own.before; };
  // whether the row has any of a thread's piece, and whether there may be a piece that it does not fill
  auto has = [&](int i) { return kFull || (column(i) < width && (kLying != kZpCycled || column(i) + V > 0)); };
  // whether a thread reads its piece i: but for shifted rows it has zeroes in place of what a row does not have
  auto reads = [&](int i) { return kLying != kZpShifted || has(i); };
  if (kLying != kZpShifted && !kFull) zp_clear_pieces<M>(t, ring, ring_bytes / p.slot, p.slot, has);
  for (int s = 0; s < stages - 1; ++s) fetch(s, ring + s * stage_bytes);

  const bool wide = c.param_dtype == ZP_F32;
  bool edge = false;
#pragma unroll
  for (int i = 0; i < M && kLying != kZpAligned; ++i) edge = edge || (has(i) && (column(i) < 0 || column(i) + V > width));
  float2 w[M][H], gw[M][H], gb[M][H];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    zp_params<T>(c.w, wide, p.vectors, column(i), width, 1.f, w[i]);
#pragma unroll
    for (int k = 0; k < H; ++k) gw[i][k] = gb[i][k] = make_float2(0.f, 0.f);
  }
  const bool drops = kJoin && c.drop.state;
  const ZpPhiloxKey<false> key = drops ? zp_philox_key<false>(c.drop.state) : ZpPhiloxKey<false>{};
  const uint32_t limit = zp_drop_limit(c.drop.threshold);
  const float inv_w = 1.f / (float)width;
  const int64_t row_bytes = c.width * (int64_t)sizeof(T), next = own.next * row_bytes;
  float next_mean[R], next_rstd[R];
  const float *mean_at = c.mean_in + own.first, *rstd_at = c.rstd_in + own.first;
  auto load_stats = [&](int turn) {
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (turn < own.n[j]) {
        next_mean[j] = mean_at[j * own.next];
        next_rstd[j] = rstd_at[j * own.next];
      }
    mean_at += own.step;
    rstd_at += own.step;
  };
#pragma unroll
  for (int j = 0; j < R; ++j) next_mean[j] = next_rstd[j] = 0.f;
  load_stats(0);
  int64_t out = own.first * row_bytes - own.before * (int)sizeof(T);        // of the rows that are worked on, in every result
  t.meet();                                    // the team's blocks run
  uint32_t slots = ring, behind = ring + (stages - 1) * stage_bytes;
  for (int turn = 0; turn < own.turns; ++turn) {
    float mean[R], rstd[R], s[2 * R];
#pragma unroll
    for (int j = 0; j < R; ++j) { mean[j] = next_mean[j]; rstd[j] = next_rstd[j]; }
    zp_copy_wait(stages);
    if (kLying == kZpShifted) t.sync();                   // others' pieces are there; the last rows have been read
    fetch(turn + stages - 1, behind);
    load_stats(turn + 1);
    float2 z[R][M][H], g[R][M][H];             // normalised rows, and gy w
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const float2 minus = make_float2(-mean[j], -mean[j]);
      const uint32_t slot = slots + j * row_slots;
      float2 s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (turn >= own.n[j] || !reads(i)) continue;
        zp_read<T, kLying>(t, slot, sx.place_of(j), i, z[j][i]);
        zp_read<T, kLying>(t, slot + p.slot, sy.place_of(j), i, g[j][i]);
        if (kLying != kZpAligned && edge) {    // (a neighbour's elements, or nothing's)
          zp_cut<T>(column(i), width, z[j][i], mean[j]);
          zp_cut<T>(column(i), width, g[j][i], 0.f);
        }
        // (z is 0 where the row has nothing: mean times rstd of large and equal values may be infinite)
        const float scale = has(i) ? rstd[j] : 0.f;
        const float2 by = make_float2(scale, scale);
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const float2 zz = __fmul2_rn(__fadd2_rn(z[j][i][k], minus), by), gy = g[j][i][k], gz = __fmul2_rn(gy, w[i][k]);
          gw[i][k] = __ffma2_rn(gy, zz, gw[i][k]);
          gb[i][k] = __fadd2_rn(gb[i][k], gy);
          s1 = __fadd2_rn(s1, gz);
          s2 = __ffma2_rn(gz, zz, s2);
          z[j][i][k] = zz;
          g[j][i][k] = gz;
        }
      }
      s[2 * j] = s1.x + s1.y;
      s[2 * j + 1] = s2.x + s2.y;
    }
    t.sum(s, turn, kLying == kZpShifted);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      ZpKept<T, kLying, false, E> kept;
      if (drops) kept.find(t, key, limit, turn < own.n[j] ? own.first + turn * own.step + j * own.next : 0, width, bytes);
      const float2 minus1 = make_float2(-s[2 * j] * inv_w, -s[2 * j] * inv_w);
      const float2 minus2 = make_float2(-s[2 * j + 1] * inv_w, -s[2 * j + 1] * inv_w);
      const float2 by = make_float2(rstd[j], rstd[j]);
      const uint32_t slot = slots + j * row_slots;
      const int64_t at = out + j * next;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (turn >= own.n[j] || !reads(i)) continue;
        float2 o[H], q[H];
#pragma unroll
        for (int k = 0; k < H; ++k)
          o[k] = __fmul2_rn(__ffma2_rn(z[j][i][k], minus2, __fadd2_rn(g[j][i][k], minus1)), by);
        if constexpr (!kJoin) {
          if (c.dx && has(i)) zp_write<T, kLying>(t, static_cast<char *>(c.dx) + at, slot, i, column(i), width, edge, o);
          continue;
        }
        if (third) {
          zp_read<T, kLying>(t, slot + 2 * p.slot, ss.place_of(j), i, q);
#pragma unroll
          for (int k = 0; k < H; ++k) o[k] = __fadd2_rn(o[k], q[k]);
        }
        if (c.dres && has(i)) zp_write<T, kLying>(t, static_cast<char *>(c.dres) + at, slot, i, column(i), width, edge, o);
        if (!c.dx) continue;
#pragma unroll
        for (int k = 0; k < H && drops; ++k) o[k] = kept.drop(o[k], i, k, limit, c.drop.scale);
        if (has(i)) zp_write<T, kLying>(t, static_cast<char *>(c.dx) + at, slot + p.slot, i, column(i), width, edge, o);
      }
    }
    if constexpr (kLying == kZpShifted) {
      t.sync();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (turn >= own.n[j]) continue;
        const int64_t at = out + j * next;
        const uint32_t from = slots + j * row_slots;
        if (kJoin && c.dres) zp_store_row<T, M>(t, static_cast<char *>(c.dres) + at, from, width);
        if (c.dx) zp_store_row<T, M>(t, static_cast<char *>(c.dx) + at, kJoin ? from + p.slot : from, width);
      }
      sx.advance();
      sy.advance();
      ss.advance();
    }
    out += own.step * row_bytes;
    behind = slots;
    slots = slots + stage_bytes == ring + ring_bytes ? ring : slots + stage_bytes;
  }
  zp_copy_wait(2);
  t.meet();                                    // (nobody writes to a block that has gone)
  if (!c.partial) return;
  float *const part = c.partial + (size_t)t.block() * 2 * c.width;
  if constexpr (kWide) {                       // each thread has columns that nobody else has
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const int at = column(i) + 2 * k;
        if ((unsigned)at < (unsigned)width) { part[at] = gw[i][k].x; part[c.width + at] = gb[i][k].x; }
        if ((unsigned)(at + 1) < (unsigned)width) { part[at + 1] = gw[i][k].y; part[c.width + at + 1] = gb[i][k].y; }
      }
    return;
  }
  // The teams' sums through shared memory, in order; of aligned rows those within a warp first, which have the same
  // columns (of cycled rows each class has its own)
  constexpr bool kByWarp = kLying != kZpCycled;
  for (int o = t.size; kByWarp && o < 32; o <<= 1) {
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
  const int row = t.size * E, copies = kByWarp ? t.walkers : kZpTeamThreads / t.size;
  __syncthreads();                                               // the rings are done with
  if (!kByWarp || t.sub == 0) {
    float *const mine = all + (size_t)(kByWarp ? t.walker : t.index) * 2 * row;
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const int at = column(i) + 2 * k;
        if constexpr (kByWarp) {
          *reinterpret_cast<float2 *>(mine + at) = gw[i][k];
          *reinterpret_cast<float2 *>(mine + row + at) = gb[i][k];
        } else {
          if ((unsigned)at < (unsigned)width) { mine[at] = gw[i][k].x; mine[row + at] = gb[i][k].x; }
          if ((unsigned)(at + 1) < (unsigned)width) { mine[at + 1] = gw[i][k].y; mine[row + at + 1] = gb[i][k].y; }
        }
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * width; i += kZpTeamThreads) {
    const int at = i < width ? i : row + (i - width);
    float sum = 0.f;
    for (int k = 0; k < copies; ++k) sum += all[(size_t)k * 2 * row + at];
    part[i] = sum;
  }
}

bool is_join(const ZpNormCall &c) { return c.dsum || c.dres || c.drop.state; }

template <typename T, int kLying, bool kFull, int E, int R, bool kJoin, bool kWide>
int launch(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  static ZpSmemOptIn opt_in;
  static ZpClusters clusters;
  return zp_launch_teams<kWide>(norm_bwd_team_kernel<T, kLying, kFull, E, R, kJoin, kWide>, "norm_bwd_team_kernel", c, p,
                                opt_in, clusters, st);
}
template <typename T, int kLying, bool kFull, bool kJoin>
int by_elements(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  if constexpr (kLying != kZpShifted) {
    if (p.ranks > 1) return launch<T, kLying, kFull, 8, 2, kJoin, true>(c, p, st);    // rows of more than a block's elements
  }
  if constexpr (kLying == kZpShifted || (sizeof(T) == 2))
    if (p.elements == 16) return launch<T, kLying, kFull, 16, 1, kJoin, false>(c, p, st);
  if constexpr (kLying == kZpAligned || !kJoin)
    if (p.rows == 2) return launch<T, kLying, kFull, 8, 2, kJoin, false>(c, p, st);
  return launch<T, kLying, kFull, 8, 1, kJoin, false>(c, p, st);
}
template <typename T, bool kJoin> int by_lying(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  if (p.full) return by_elements<T, kZpAligned, true, kJoin>(c, p, st);
  if (p.lying == kZpAligned) return by_elements<T, kZpAligned, false, kJoin>(c, p, st);
  return p.lying == kZpCycled ? by_elements<T, kZpCycled, false, kJoin>(c, p, st)
                              : by_elements<T, kZpShifted, false, kJoin>(c, p, st);
}
template <typename T> int by_kind(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  return is_join(c) ? by_lying<T, true>(c, p, st) : by_lying<T, false>(c, p, st);
}

}  // namespace

int zp_launch_norm_bwd(const ZpNormCall &c, bool &taken, int &parts, cudaStream_t st) {
  const int lying = zp_lying(c, {{c.x, c.ldx}, {c.dy, c.ldy}, {c.dsum, c.lds}, {c.dx, c.width}, {c.dres, c.width}});
  const int64_t each = c.rows * c.width / ((int64_t)148 * kZpTeamThreads);       // elements a thread
  const int arrays = c.dsum ? 3 : 2;
  const bool join = is_join(c);
  const size_t last = c.partial ? 2 * sizeof(float) : 0;
  // Two rows at a time, as in the forward: 16384 x 4096 bf16 93 us -> 76, joined 153 -> 132, 400000 x 32 23 -> 20.
  // Joined rows of a warp or less (60000 x 128 fp32 29 -> 31) or that are not aligned (30011 x 1001 fp16 91 -> 105:
  // registers) are better one by one.
  const bool two = each >= 32 && (!join || (lying == kZpAligned && c.width > 256));
  // Rows of more than 4096 elements: sixteen to a thread up to 8192 in 16 bits (8192 x 8192 bf16 91 us, by clusters 121;
  // joined 160, 196), else a cluster a row (2048 x 8192 fp32 joined 76 us, sixteen to a thread 88).
  const bool over = zp_span(c, lying) > 8 * kZpTeamThreads;
  const bool many = over && (lying == kZpShifted || c.dtype != ZP_F32), wide = over && lying != kZpShifted;
  ZpTeamPlan p;
  taken = c.dy && ((many && zp_team_plan(c, lying, arrays, last, 16, 1, p) && p.ranks == 1) ||
                   ((two || wide) && zp_team_plan(c, lying, arrays, last, 8, 2, p)) ||
                   (!wide && zp_team_plan(c, lying, arrays, last, 8, 1, p)));
  if (!taken) return ZP_OK;
  const int rc = c.dtype == ZP_F32   ? by_kind<float>(c, p, st)
                 : c.dtype == ZP_F16 ? by_kind<__half>(c, p, st)
                                     : by_kind<__nv_bfloat16>(c, p, st);
  taken = p.blocks > 0;
  parts = (int)p.blocks / p.ranks;
  return rc;
}
