// Forward of the layer norm over rows, alone and behind a residual sum with dropout.
//
// Memory bound: a row is read once and the results are written once.  Mean and variance take two passes
// over the row in registers, the variance from differences to the mean: sums of squares would lose a mean
// that is large against the spread.
//
// B200, one kernel (share of 6 450 GB/s): 8192 x 4096 fp32 43 us (0.97), 16384 x 4096 bf16 48 (0.87; 11.3
// instructions an element, 46 % of the issue slots: the waits of sixteen warps for each other's sums are what is
// left), joined with dropout 96 (0.86; 28 instructions, half of them the generator), 60000 x 128 fp32 11.9 (0.80, of it two
// for the launch and a turn that not every warp has), 30011 x 1001 fp16 39 (0.48: the ends of the rows are the
// work of two lanes while the others wait).
#include "zp_rowwise.cuh"

namespace {

// E elements of a thread in each of R rows at a time
template <typename T, int kLying, bool kFull, int E, int R, bool kJoin, bool kWide>
__global__ void __launch_bounds__(kZpTeamThreads, 1)
norm_fwd_team_kernel(const __grid_constant__ ZpNormCall c, const __grid_constant__ ZpTeamPlan p) {
  zp_after_previous();
  constexpr int V = kZpVec<T>, H = V / 2, M = E / V, A = kJoin ? 2 : 1;
  extern __shared__ __align__(16) char smem[];
  const ZpTeam<kWide> t(p.team, p.ranks, reinterpret_cast<float *>(smem));
  const int width = (int)c.width, stages = p.stages;
  char *const after_red = smem + kZpSumsBytes;
  uint8_t *const bytes = reinterpret_cast<uint8_t *>(after_red) + t.index * p.bytes;
  const uint32_t stage_bytes = A * R * p.slot, ring_bytes = stages * stage_bytes;
  const uint32_t ring = zp_shared(after_red) + p.bytes * (kZpTeamThreads / p.team) + t.index * ring_bytes;
  const ZpTeamRows<kLying, R> own(t, c.rows, width, p.cycle);
  ZpSource<kLying> sx(t, c.x, c.ldx, c.rows, c.width, sizeof(T), own);
  ZpSource<kLying> sr(t, c.res, c.ldr, c.rows, c.width, sizeof(T), own);
  auto fetch = [&](int turn, uint32_t to) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (turn >= own.n[j]) continue;
      zp_fetch_row<T, kLying, kFull, M>(t, to + j * A * p.slot, sx, j, width, own.before);
      if (kJoin) zp_fetch_row<T, kLying, kFull, M>(t, to + (j * A + 1) * p.slot, sr, j, width, own.before);
    }
    sx.row += sx.step;
    if (kJoin) sr.row += sr.step;
    zp_copy_commit();
  };
  auto column = [&](int i) { return t.piece(i) * V - own.before; };
  // whether the row has any of a thread's piece, and whether there may be a piece that it does not fill
  auto has = [&](int i) { return kFull || (column(i) < width && (kLying != kZpCycled || column(i) + V > 0)); };
  // whether a thread reads its piece i: but for shifted rows it has zeroes in place of what a row does not have
  auto reads = [&](int i) { return kLying != kZpShifted || has(i); };
  if (kLying != kZpShifted && !kFull) zp_clear_pieces<M>(t, ring, stages * A * R, p.slot, has);
  for (int s = 0; s < stages - 1; ++s) fetch(s, ring + s * stage_bytes);

  const bool wide = c.param_dtype == ZP_F32;
  bool edge = false;
#pragma unroll
  for (int i = 0; i < M && kLying != kZpAligned; ++i) edge = edge || (has(i) && (column(i) < 0 || column(i) + V > width));
  constexpr bool kHeld = E <= 16;              // weight and bias stay in registers
  float2 w[kHeld ? M : 1][H], b[kHeld ? M : 1][H];
#pragma unroll
  for (int i = 0; i < (kHeld ? M : 0); ++i) {
    zp_params<T>(c.w, wide, p.vectors, column(i), width, 1.f, w[i]);
    zp_params<T>(c.b, wide, p.vectors, column(i), width, 0.f, b[i]);
  }
  auto cut = [&](float2 (&v)[M][H]) {
    if (kLying == kZpAligned || !edge) return;
#pragma unroll
    for (int i = 0; i < M; ++i) zp_cut<T>(column(i), width, v[i], 0.f);
  };
  const bool drops = kJoin && c.drop.state;
  const ZpPhiloxKey<false> key = drops ? zp_philox_key<false>(c.drop.state) : ZpPhiloxKey<false>{};
  const uint32_t limit = zp_drop_limit(c.drop.threshold);
  // (in fp32 worked out here: read from the parameters it makes odd widths 3 % slower, 20000 x 1001 32.4 us -> 33.2; in 16
  // bits read from there: worked out it costs 2 %, 16384 x 4096 47.2 us -> 48.4)
  const ZpOver over = {sizeof(T) == 4 ? 1.f / (float)width : p.over.one, p.over.rest};
  const int64_t row_bytes = c.width * (int64_t)sizeof(T), next = own.next * row_bytes;
  int64_t out = own.first * row_bytes - own.before * (int)sizeof(T);        // of the rows that are worked on, in every result
  t.meet();                                    // the team's blocks run
  uint32_t slots = ring, behind = ring + (stages - 1) * stage_bytes;
  for (int turn = 0; turn < own.turns; ++turn) {
    zp_copy_wait(stages);
    if (kLying == kZpShifted) t.sync();                   // others' pieces are there; the last rows have been read
    fetch(turn + stages - 1, behind);
    float2 v[R][M][H];
    float s[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool mine = turn < own.n[j];
      const uint32_t x = slots + j * A * p.slot, res = x + p.slot;
      ZpKept<T, kLying, kLying != kZpShifted, E> kept;
      if (drops) kept.find(t, key, limit, mine ? own.first + turn * own.step + j * own.next : 0, width, bytes);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (!mine || !reads(i)) continue;
        zp_read<T, kLying>(t, x, sx.place_of(j), i, v[j][i]);
        if constexpr (kJoin) {
          float2 q[H];
          zp_read<T, kLying>(t, res, sr.place_of(j), i, q);
#pragma unroll
          for (int k = 0; k < H; ++k) {
            const float2 f = drops ? kept.drop(v[j][i][k], i, k, limit, c.drop.scale) : v[j][i][k];
            v[j][i][k] = __fadd2_rn(q[k], f);
          }
          // rounded: what follows works on the sum as it is returned
          const uint4 packed = zp_pack<T>(v[j][i]);
          zp_unpack<T>(packed, v[j][i]);
          if (kLying != kZpShifted && has(i))
            zp_write<T, kLying>(t, static_cast<char *>(c.sum) + out + j * next, 0, i, column(i), width, edge, v[j][i]);
        }
      }
      cut(v[j]);
#pragma unroll
      for (int i = 0; i < M; ++i)
        if (mine && reads(i)) {
#pragma unroll
          for (int k = 0; k < H; ++k) sum = __fadd2_rn(sum, v[j][i][k]);
        }
      s[j] = sum.x + sum.y;
    }
    t.sum(s, 0, kLying == kZpShifted);
    float q[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      s[j] = over.of(s[j]);
      float2 sq = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (turn >= own.n[j] || !reads(i)) continue;
        const float less = has(i) ? -s[j] : 0.f;
        const float2 minus = make_float2(less, less);
        if constexpr (kJoin && kLying == kZpShifted)      // (the team has read all of this slot)
          zp_write<T, kLying>(t, nullptr, slots + j * A * p.slot, i, 0, 0, false, v[j][i]);
#pragma unroll
        for (int k = 0; k < H; ++k) v[j][i][k] = __fadd2_rn(v[j][i][k], minus);
      }
      cut(v[j]);
#pragma unroll
      for (int i = 0; i < M; ++i)
        if (turn < own.n[j] && reads(i)) {
#pragma unroll
          for (int k = 0; k < H; ++k) sq = __ffma2_rn(v[j][i][k], v[j][i][k], sq);
        }
      q[j] = sq.x + sq.y;
    }
    t.sum(q, 1, kLying == kZpShifted);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const float rstd = rsqrtf(q[j] * over.one + c.eps);
      const float2 both = make_float2(rstd, rstd);
      char *const y = static_cast<char *>(c.y) + out + j * next;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (turn >= own.n[j] || !reads(i)) continue;
        float2 (&ww)[H] = w[kHeld ? i : 0], (&bb)[H] = b[kHeld ? i : 0];
        if constexpr (!kHeld) {
          zp_params<T>(c.w, wide, p.vectors, column(i), width, 1.f, ww);
          zp_params<T>(c.b, wide, p.vectors, column(i), width, 0.f, bb);
        }
#pragma unroll
        for (int k = 0; k < H; ++k) v[j][i][k] = __ffma2_rn(__fmul2_rn(v[j][i][k], both), ww[k], bb[k]);
        if (has(i))
          zp_write<T, kLying>(t, y, slots + (j * A + A - 1) * p.slot, i, column(i), width, edge, v[j][i]);
      }
      if (t.piece(0) == 0 && c.mean && turn < own.n[j]) {
        const int64_t r = own.first + turn * own.step + j * own.next;
        c.mean[r] = s[j];
        c.rstd[r] = rstd;
      }
    }
    if constexpr (kLying == kZpShifted) {
      t.sync();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (turn >= own.n[j]) continue;
        const int64_t at = out + j * next;
        zp_store_row<T, M>(t, static_cast<char *>(c.y) + at, slots + (j * A + A - 1) * p.slot, width);
        if (kJoin) zp_store_row<T, M>(t, static_cast<char *>(c.sum) + at, slots + j * A * p.slot, width);
      }
      sx.advance();
      sr.advance();
    }
    out += own.step * row_bytes;
    behind = slots;
    slots = slots + stage_bytes == ring + ring_bytes ? ring : slots + stage_bytes;
  }
  zp_copy_wait(2);
  t.meet();                                    // (nobody writes to a block that has gone)
}

template <typename T, int kLying, bool kFull, int E, int R, bool kJoin, bool kWide>
int launch(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  static ZpSmemOptIn opt_in;
  static ZpClusters clusters;
  return zp_launch_teams<kWide>(norm_fwd_team_kernel<T, kLying, kFull, E, R, kJoin, kWide>, "norm_fwd_team_kernel", c, p,
                                opt_in, clusters, st);
}
template <typename T, int kLying, bool kFull, bool kJoin>
int by_elements(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  if (p.ranks > 1) {                           // rows of more than a block's elements
    if constexpr (kLying != kZpShifted) return launch<T, kLying, kFull, 16, sizeof(T) == 2 ? 2 : 1, kJoin, true>(c, p, st);
  }
  if constexpr (kLying == kZpAligned)
    if (p.elements == 32) return launch<T, kLying, kFull, 32, 1, kJoin, false>(c, p, st);
  if (p.elements == 8) return launch<T, kLying, kFull, 8, 1, kJoin, false>(c, p, st);
  if constexpr (sizeof(T) == 2 && (!kJoin || kLying == kZpAligned))
    if (p.rows == 2) return launch<T, kLying, kFull, 16, 2, kJoin, false>(c, p, st);
  return launch<T, kLying, kFull, 16, 1, kJoin, false>(c, p, st);
}
template <typename T, bool kJoin> int by_lying(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  if (p.full) return by_elements<T, kZpAligned, true, kJoin>(c, p, st);
  if (p.lying == kZpAligned) return by_elements<T, kZpAligned, false, kJoin>(c, p, st);
  return p.lying == kZpCycled ? by_elements<T, kZpCycled, false, kJoin>(c, p, st)
                              : by_elements<T, kZpShifted, false, kJoin>(c, p, st);
}
template <typename T> int by_kind(const ZpNormCall &c, ZpTeamPlan &p, cudaStream_t st) {
  return c.res ? by_lying<T, true>(c, p, st) : by_lying<T, false>(c, p, st);
}

}  // namespace

int zp_launch_norm_fwd(const ZpNormCall &c, bool &taken, cudaStream_t st) {
  const size_t size = c.dtype == ZP_F32 ? 4 : 2;
  const int lying = zp_lying(c, {{c.x, c.ldx}, {c.y, c.width}, {c.res, c.ldr}, {c.sum, c.width}});
  // Two rows at a time halve what joining the sums of a team of several warps costs (16384 x 4096 bf16 59 us ->
  // 49), and leave the ring fewer stages (fp32 42 -> 50, joined without dropout 92 -> 99), the blocks fewer
  // turns to share out (60000 x 128 bf16 9.5 -> 10.4) and joined rows that are not aligned too few registers (30011 x
  // 1001 fp16 72 -> 92).  Few elements are spread over more threads.
  const int64_t each = c.rows * c.width / ((int64_t)148 * kZpTeamThreads);       // elements a thread
  const int arrays = c.res ? 2 : 1;
  const int64_t span = zp_span(c, lying);
  const bool wide = span > 16 * kZpTeamThreads;
  const bool two = size == 2 &&
                   (wide || (each >= 64 && c.width > 512 && (!c.res || (c.drop.state && lying == kZpAligned))));
  // Rows of more than 8192 elements: a cluster a row, which waits for its blocks' sums, or up to 16384, aligned and
  // where the ring has room for them, 32 elements to a thread (4096 x 16384 bf16 79 us, by clusters 94)
  ZpTeamPlan p;
  taken = (wide && lying == kZpAligned && zp_team_plan(c, lying, arrays, 0, 32, 1, p) && p.ranks == 1) ||
          (two && zp_team_plan(c, lying, arrays, 0, 16, 2, p)) ||
          ((wide || each >= 32 || span > 8 * kZpTeamThreads) && zp_team_plan(c, lying, arrays, 0, 16, 1, p)) ||
          (!wide && zp_team_plan(c, lying, arrays, 0, 8, 1, p) && p.ranks == 1);
  if (!taken) return ZP_OK;
  const int rc = c.dtype == ZP_F32   ? by_kind<float>(c, p, st)
                 : c.dtype == ZP_F16 ? by_kind<__half>(c, p, st)
                                     : by_kind<__nv_bfloat16>(c, p, st);
  taken = p.blocks > 0;
  return rc;
}
