// Backward of the layer norm over rows, alone and with the residual sum and dropout in front of it: the
// rows' gradient and, from the same reading of the rows, partial sums of the parameters' gradients.
//
// A thread has the same columns in every row of its team, so the sums over rows stay in its registers;
// at the end the teams of a block add theirs up in a fixed order and the block writes one partial row of
// each, which a second kernel adds in block order.
#include "zp_rowwise.cuh"

namespace {

template <typename T, bool kAligned, int E, bool kJoin>
__global__ void __launch_bounds__(kZpTeamThreads, 1)
norm_bwd_team_kernel(const ZpNormCall c, const ZpTeamPlan p) {
  zp_after_previous();
  constexpr int V = kZpStep<T, kAligned>, M = E / V;
  constexpr bool kHeld = E <= 16, kKept = E <= 16;
  extern __shared__ __align__(16) char smem[];
  const ZpTeam t(p.team, reinterpret_cast<float2 *>(smem));
  const int width = (int)c.width, teams = kZpTeamThreads / p.team, stages = p.stages;
  char *const after_red = smem + 2 * sizeof(float2) * (kZpTeamThreads / 32);
  uint8_t *const bytes = reinterpret_cast<uint8_t *>(after_red) + t.index * p.bytes;
  char *const rings = after_red + p.bytes * teams;
  const int A = kJoin && c.dsum ? 3 : 2;
  char *const ring = rings + (size_t)t.index * stages * A * p.slot;
  const int64_t step = (int64_t)gridDim.x * t.walkers * t.per;
  const int64_t first = ((int64_t)t.walker * gridDim.x + blockIdx.x) * t.per + t.sub;
  ZpSource sx(c.x, c.ldx, c.rows, c.width, sizeof(T), first, step);
  ZpSource sy(c.dy, c.ldy, c.rows, c.width, sizeof(T), first, step);
  ZpSource ss(c.dsum, c.lds, c.rows, c.width, sizeof(T), first, step);
  int64_t coming = first;
  auto fetch = [&](int stage) {
    char *const to = ring + stage * A * p.slot;
    const bool live = coming < c.rows;
    zp_fetch_row<T, kAligned, E>(t, to, sx, live, width);
    zp_fetch_row<T, kAligned, E>(t, to + p.slot, sy, live, width);
    if (kJoin && A == 3) zp_fetch_row<T, kAligned, E>(t, to + 2 * p.slot, ss, live, width);
    coming += step;
    zp_copy_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(s);

  const bool wide = c.param_dtype == ZP_F32;
  auto column = [&](int i, int k) { return (t.lane + i * t.size) * V + k; };
  float w[kHeld ? E : 1], gw[E], gb[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int col = column(e / V, e % V);
    if constexpr (kHeld) w[e] = col < width ? zp_param<T>(c.w, wide, col, 1.f) : 0.f;
    gw[e] = gb[e] = 0.f;
  }
  auto weight = [&](int i, int k) { return kHeld ? w[kHeld ? i * V + k : 0] : zp_param<T>(c.w, wide, column(i, k), 1.f); };
  const ZpPhiloxKey key = kJoin && c.drop.state ? zp_philox_key(c.drop.state) : ZpPhiloxKey{};
  const float inv_w = 1.f / (float)width;
  float next_mean = first < c.rows ? c.mean_in[first] : 0.f, next_rstd = first < c.rows ? c.rstd_in[first] : 0.f;
  int stage = 0, turn = 0;
  for (int64_t base = first - t.sub; base < c.rows; base += step) {
    const int64_t r = base + t.sub;
    const bool live = r < c.rows;
    const float mean = next_mean, rstd = next_rstd;
    zp_copy_wait(stages);
    if (!kAligned) t.sync();
    fetch(stage == 0 ? stages - 1 : stage - 1);
    if (r + step < c.rows) { next_mean = c.mean_in[r + step]; next_rstd = c.rstd_in[r + step]; }
    const char *const slot = ring + stage * A * p.slot;
    const char *const x = slot + (kAligned ? 0 : sx.place);
    const char *const dy = slot + p.slot + (kAligned ? 0 : sy.place);
    const char *const ds = slot + 2 * p.slot + (kAligned ? 0 : ss.place);
    sx.advance();
    sy.advance();
    ss.advance();
    stage = stage + 1 == stages ? 0 : stage + 1;
    const int mine = live ? width : 0;
    float2 s = make_float2(0.f, 0.f);
    float zs[kKept ? E : 1], gs[kKept ? E : 1];          // z and gy w, where there are registers for them
#pragma unroll
    for (int i = 0; i < M; ++i) {
      if (column(i, 0) >= mine) continue;
      float v[V], g[V];
      zp_read<T, kAligned>(t, x, i, v);
      zp_read<T, kAligned>(t, dy, i, g);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float z = (v[k] - mean) * rstd, gz = g[k] * weight(i, k);
        gw[i * V + k] += g[k] * z;
        gb[i * V + k] += g[k];
        s.x += gz;
        s.y += gz * z;
        if constexpr (kKept) { zs[i * V + k] = z; gs[i * V + k] = gz; }
      }
    }
    s = t.sum(s, turn++);
    const float m1 = s.x * inv_w, m2 = s.y * inv_w;
    uint32_t kept = 0xffffffffu;
    if (kJoin && c.drop.state)
      kept = zp_kept_bits<T, kAligned, E>(t, key, c.drop.threshold, live ? r : 0, width, bytes);
#pragma unroll
    for (int i = 0; i < M; ++i) {
      if (column(i, 0) >= mine) continue;
      float v[V], g[V];
      if constexpr (kKept) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = rstd * (gs[i * V + k] - m1 - zs[i * V + k] * m2);
      } else {
        zp_read<T, kAligned>(t, x, i, v);
        zp_read<T, kAligned>(t, dy, i, g);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = rstd * (g[k] * weight(i, k) - m1 - (v[k] - mean) * rstd * m2);
      }
      if constexpr (kJoin) {
        if (A == 3) {
          zp_read<T, kAligned>(t, ds, i, g);
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] += g[k];
        }
        if (c.dres) zp_write<T, kAligned>(t, static_cast<T *>(c.dres) + r * c.width, i, v);
        if (!c.dx) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = kept >> (i * V + k) & 1 ? v[k] * c.drop.scale : 0.f;
        zp_write<T, kAligned>(t, static_cast<T *>(c.dx) + r * c.width, i, v);
      } else if (c.dx) {
        zp_write<T, kAligned>(t, static_cast<T *>(c.dx) + r * c.width, i, v);
      }
    }
  }
  zp_copy_wait(2);
  if (!c.partial) return;
  // teams within a warp first, then those of the block (`copies` of them) through shared memory, in order
  for (int o = t.size; o < 32; o <<= 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      gw[e] += __shfl_xor_sync(0xffffffffu, gw[e], o);
      gb[e] += __shfl_xor_sync(0xffffffffu, gb[e], o);
    }
  }
  float *const all = reinterpret_cast<float *>(rings);           // [copies][2][row]
  const int row = t.size * E, copies = t.walkers;
  __syncthreads();                                               // the rings are done with
  if (t.sub == 0) {
    float *mine = all + (size_t)t.walker * 2 * row;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int col = column(e / V, e % V);
      mine[col] = gw[e];
      mine[row + col] = gb[e];
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

template <typename T, bool kAligned, int E, bool kJoin>
int launch(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  static ZpSmemOptIn opt_in;
  if (int rc = zp_ensure_smem(norm_bwd_team_kernel<T, kAligned, E, kJoin>, p.smem, opt_in)) return rc;
  zp_launch(norm_bwd_team_kernel<T, kAligned, E, kJoin>, p.blocks, kZpTeamThreads, p.smem, st, c, p);
  ZP_LAUNCH_CHECK("norm_bwd_team_kernel");
  return ZP_OK;
}
template <typename T, bool kAligned, int E>
int by_join(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  const bool join = c.dsum || c.dres || c.drop.state;
  return join ? launch<T, kAligned, E, true>(c, p, st) : launch<T, kAligned, E, false>(c, p, st);
}
template <typename T, bool kAligned> int by_elements(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  return p.elements == 8    ? by_join<T, kAligned, 8>(c, p, st)
         : p.elements == 16 ? by_join<T, kAligned, 16>(c, p, st)
                            : by_join<T, kAligned, 32>(c, p, st);
}
template <typename T> int by_alignment(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  return p.aligned ? by_elements<T, true>(c, p, st) : by_elements<T, false>(c, p, st);
}

}  // namespace

int zp_launch_norm_bwd(const ZpNormCall &c, bool &taken, int &parts, cudaStream_t st) {
  const size_t size = c.dtype == ZP_F32 ? 4 : 2;
  const bool aligned = (c.width * size) % 16 == 0 && zp_piece_aligned(c.x, c.ldx, size) && zp_piece_aligned(c.dy, c.ldy, size) &&
                       (!c.dsum || zp_piece_aligned(c.dsum, c.lds, size)) &&
                       (!c.dx || zp_piece_aligned(c.dx, c.width, size)) &&
                       (!c.dres || zp_piece_aligned(c.dres, c.width, size)) &&
                       (!c.drop.state || c.width % 8 == 0);
  ZpTeamPlan p;
  taken = c.dy && zp_team_plan(c, aligned, c.dsum ? 3 : 2, c.partial ? 2 * sizeof(float) : 0, 16, p);
  if (!taken) return ZP_OK;
  parts = (int)p.blocks;
  if (c.dtype == ZP_F32) return by_alignment<float>(c, p, st);
  if (c.dtype == ZP_F16) return by_alignment<__half>(c, p, st);
  return by_alignment<__nv_bfloat16>(c, p, st);
}
