// The launches of wide rows where a device runs few clusters at a time: this program stands in for the runtime's
// occupancy query and its launch, and calls the library's functions.  Arguments: clusters at a time.
#include <cstdio>
#include <cstdlib>

#include <cuda_runtime.h>

#include "zippel_b200.h"

static int g_most, g_queries;
static struct { int launches, clusters, empty; } g_seen;

extern "C" {
cudaError_t cudaGetDevice(int *dev) { *dev = 0; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaOccupancyMaxActiveClusters(int *most, const void *, const cudaLaunchConfig_t *) {
  ++g_queries;
  *most = g_most;
  return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t *cfg, const void *, void **) {
  int size = 1;
  for (unsigned i = 0; i < cfg->numAttrs; ++i)
    if (cfg->attrs[i].id == cudaLaunchAttributeClusterDimension) size = cfg->attrs[i].val.clusterDim.x;
  ++g_seen.launches;
  g_seen.clusters += size > 1;
  g_seen.empty += cfg->gridDim.x == 0 || cfg->gridDim.x % size != 0 || (size > 1 && (int)cfg->gridDim.x / size > g_most);
  return cudaSuccess;
}
}
static int64_t g_count;
int64_t &zp_launch_counter() { return g_count; }
void zp_set_cuda_error(cudaError_t, const char *) {}

int main(int, char **argv) {
  g_most = std::atoi(argv[1]);
  void *const a = reinterpret_cast<void *>(uintptr_t(1) << 20);        // (nothing is read: nothing runs)
  float *const f = static_cast<float *>(a);
  const int64_t *const state = static_cast<const int64_t *>(a);
  for (int again = 0; again < 3; ++again)
    for (int64_t width : {9999, 9998, 9996, 12000, 16377, 16384, 30000, 32761, 65529})
      for (int64_t rows : {1, 7, 300})
        for (int dtype : {ZP_F32, ZP_F16})
          for (double p : {0.0, 0.5}) {
            const size_t work = zp_rowwise_work_bytes(rows, width);
            int rc[4];
            g_seen = {};
            rc[0] = zp_layernorm_forward(rows, width, dtype, a, width, dtype, a, a, 1e-5f, a, f, f, nullptr);
            rc[1] = zp_layernorm_backward(rows, width, dtype, a, width, dtype, a, f, f, a, width, a, a, a, a, work, nullptr);
            rc[2] = zp_add_layernorm_forward(rows, width, dtype, a, width, a, width, p, state, dtype, a, a, 1e-5f, a, a, f, f, nullptr);
            rc[3] = zp_add_layernorm_backward(rows, width, dtype, a, dtype, a, f, f, a, width, a, width, p, state, a, a, a, a, a, work, nullptr);
            for (int i = 0; i < 4; ++i)
              if (rc[i]) return std::printf("%lld x %lld, type %d: call %d gives status %d\n", (long long)rows, (long long)width, dtype, i, rc[i]), 1;
            if (g_seen.empty) return std::printf("%lld x %lld, type %d: %d launches of no blocks or of too many\n", (long long)rows, (long long)width, dtype, g_seen.empty), 1;
            if (g_most == 0 && g_seen.clusters) return std::puts("clusters that do not run"), 1;
            if (g_most >= 8 && !g_seen.clusters && width > 32768) return std::puts("no clusters"), 1;
          }
  std::puts("ok");
}
