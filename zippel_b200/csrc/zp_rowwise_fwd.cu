// Forward of the layer norm over rows, alone and behind a residual sum with dropout.
//
// Memory bound: a row is read once and the results are written once; between lie about ten instructions
// per element (and eight for the random bits).  Mean and variance take two passes over the row in shared
// memory, the variance from differences to the mean: sums of squares would lose a mean that is large
// against the spread.
#include "zp_rowwise.cuh"

namespace {

template <typename T, bool kAligned, int E, bool kJoin>
__global__ void __launch_bounds__(kZpTeamThreads, 1)
norm_fwd_team_kernel(const ZpNormCall c, const ZpTeamPlan p) {
  zp_after_previous();
  constexpr int V = kZpStep<T, kAligned>, M = E / V, A = kJoin ? 2 : 1;
  extern __shared__ __align__(16) char smem[];
  const ZpTeam t(p.team, reinterpret_cast<float2 *>(smem));
  const int width = (int)c.width, teams = kZpTeamThreads / p.team, stages = p.stages;
  char *const after_red = smem + 2 * sizeof(float2) * (kZpTeamThreads / 32);
  uint8_t *const bytes = reinterpret_cast<uint8_t *>(after_red) + t.index * p.bytes;
  char *const ring = after_red + p.bytes * teams + (size_t)t.index * stages * A * p.slot;
  const int64_t step = (int64_t)gridDim.x * t.walkers * t.per;
  const int64_t first = ((int64_t)t.walker * gridDim.x + blockIdx.x) * t.per + t.sub;
  ZpSource sx(c.x, c.ldx, c.rows, c.width, sizeof(T), first, step);
  ZpSource sr(c.res, c.ldr, c.rows, c.width, sizeof(T), first, step);
  int64_t coming = first;
  auto fetch = [&](int stage) {
    char *const to = ring + stage * A * p.slot;
    zp_fetch_row<T, kAligned, E>(t, to, sx, coming < c.rows, width);
    if (kJoin) zp_fetch_row<T, kAligned, E>(t, to + p.slot, sr, coming < c.rows, width);
    coming += step;
    zp_copy_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(s);

  const bool wide = c.param_dtype == ZP_F32;
  auto column = [&](int i, int k) { return (t.lane + i * t.size) * V + k; };
  constexpr bool kHeld = E <= 16;              // weight and bias stay in registers
  float w[kHeld ? E : 1], b[kHeld ? E : 1];
#pragma unroll
  for (int e = 0; e < (kHeld ? E : 0); ++e) {
    const int col = column(e / V, e % V);
    w[e] = col < width ? zp_param<T>(c.w, wide, col, 1.f) : 0.f;
    b[e] = col < width ? zp_param<T>(c.b, wide, col, 0.f) : 0.f;
  }
  const ZpPhiloxKey key = kJoin && c.drop.state ? zp_philox_key(c.drop.state) : ZpPhiloxKey{};
  const float inv_w = 1.f / (float)width;
  int stage = 0;
  for (int64_t base = first - t.sub; base < c.rows; base += step) {      // (a warp's teams go on together)
    const int64_t r = base + t.sub;
    const bool live = r < c.rows;
    zp_copy_wait(stages);
    if (!kAligned) t.sync();                   // others' pieces are there; the last row has been read
    fetch(stage == 0 ? stages - 1 : stage - 1);
    const char *const slot = ring + stage * A * p.slot;
    const char *const x = slot + (kAligned ? 0 : sx.place), *const res = slot + p.slot + (kAligned ? 0 : sr.place);
    sx.advance();
    sr.advance();
    stage = stage + 1 == stages ? 0 : stage + 1;
    const int mine = live ? width : 0;
    uint32_t kept = 0xffffffffu;
    if (kJoin && c.drop.state)
      kept = zp_kept_bits<T, kAligned, E>(t, key, c.drop.threshold, live ? r : 0, width, bytes);
    float v[E], s = 0.f;
#pragma unroll
    for (int i = 0; i < M; ++i) {
      float u[V] = {};
      if (column(i, 0) < mine) {
        zp_read<T, kAligned>(t, x, i, u);
        if constexpr (kJoin) {
          float q[V];
          zp_read<T, kAligned>(t, res, i, q);
#pragma unroll
          for (int k = 0; k < V; ++k)          // rounded: what follows works on the sum as it is returned
            u[k] = zp_float(zp_rounded<T>(q[k] + (kept >> (i * V + k) & 1 ? u[k] * c.drop.scale : 0.f)));
          zp_write<T, kAligned>(t, static_cast<T *>(c.sum) + r * c.width, i, u);
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[i * V + k] = u[k];
        s += u[k];
      }
    }
    const float mean = t.sum(s, 0) * inv_w;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < M; ++i)
      if (column(i, 0) < mine) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          v[i * V + k] -= mean;
          q += v[i * V + k] * v[i * V + k];
        }
      }
    const float rstd = rsqrtf(t.sum(q, 1) * inv_w + c.eps);
    T *const y = static_cast<T *>(c.y) + r * c.width;
#pragma unroll
    for (int i = 0; i < M; ++i)
      if (column(i, 0) < mine) {
        float u[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float ww = kHeld ? w[kHeld ? i * V + k : 0] : zp_param<T>(c.w, wide, column(i, k), 1.f);
          const float bb = kHeld ? b[kHeld ? i * V + k : 0] : zp_param<T>(c.b, wide, column(i, k), 0.f);
          u[k] = v[i * V + k] * rstd * ww + bb;
        }
        zp_write<T, kAligned>(t, y, i, u);
      }
    if (c.mean && live && t.lane == 0) { c.mean[r] = mean; c.rstd[r] = rstd; }
  }
  zp_copy_wait(2);
}

template <typename T, bool kAligned, int E, bool kJoin>
int launch(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  static ZpSmemOptIn opt_in;
  if (int rc = zp_ensure_smem(norm_fwd_team_kernel<T, kAligned, E, kJoin>, p.smem, opt_in)) return rc;
  zp_launch(norm_fwd_team_kernel<T, kAligned, E, kJoin>, p.blocks, kZpTeamThreads, p.smem, st, c, p);
  ZP_LAUNCH_CHECK("norm_fwd_team_kernel");
  return ZP_OK;
}
template <typename T, bool kAligned, int E>
int by_join(const ZpNormCall &c, const ZpTeamPlan &p, cudaStream_t st) {
  return c.res ? launch<T, kAligned, E, true>(c, p, st) : launch<T, kAligned, E, false>(c, p, st);
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

int zp_launch_norm_fwd(const ZpNormCall &c, bool &taken, cudaStream_t st) {
  const size_t size = c.dtype == ZP_F32 ? 4 : 2;
  // (results lie row behind row; the counters of dropout go by eight elements)
  const bool aligned = (c.width * size) % 16 == 0 && zp_piece_aligned(c.x, c.ldx, size) && zp_piece_aligned(c.y, c.width, size) &&
                       (!c.res || (zp_piece_aligned(c.res, c.ldr, size) && zp_piece_aligned(c.sum, c.width, size))) &&
                       (!c.drop.state || c.width % 8 == 0);
  ZpTeamPlan p;
  taken = zp_team_plan(c, aligned, c.res ? 2 : 1, 0, 16, p);
  if (!taken) return ZP_OK;
  if (c.dtype == ZP_F32) return by_alignment<float>(c, p, st);
  if (c.dtype == ZP_F16) return by_alignment<__half>(c, p, st);
  return by_alignment<__nv_bfloat16>(c, p, st);
}
