// relbias.hip — learned relative position bias by buckets: table [buckets, heads] -> one fp32 row per head over the distances -reach .. reach,
// and its gradient.  The row is what the attention kernels read (they never see a [queries, keys] bias) and what their gradient returns.
//
// Bound: launch latency (a few kilobytes).  Expansion: one thread per (head, distance), a gather.  Gradient: one wave per (bucket, head) adds the
// distances of its bucket — lane i takes i, i + 64, ... in fp64, then a fixed exchange order — so equal inputs give equal bits.
#include "common.h"

namespace {

__global__ void rel_bias_kernel(const float* __restrict__ table, const int32_t* __restrict__ index, float* __restrict__ rel, const int buckets,
                                const int heads, const int n) {
  const int i = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  if (i >= n) return;
  const int b = index[i];
  rel[(int64_t)h * n + i] = b >= 0 && b < buckets ? table[(int64_t)b * heads + h] : 0.f;
}

__global__ __launch_bounds__(64) void rel_bias_grad_kernel(const float* __restrict__ drel, const int32_t* __restrict__ index,
                                                           float* __restrict__ dtable, const int heads, const int n) {
  const int h = blockIdx.x, b = blockIdx.y;
  double t = 0.;
  for (int i = threadIdx.x; i < n; i += 64)
    if (index[i] == b) t += (double)drel[(int64_t)h * n + i];
  t = wave_sum_d(t);
  if (threadIdx.x == 0) dtable[(int64_t)b * heads + h] = (float)t;
}

}  // namespace

extern "C" int mgld_rel_bias(const float* table, const int32_t* index, float* rel, int buckets, int heads, int n, void* stream) {
  MGLD_REQUIRE(table && index && rel && buckets > 0 && heads > 0 && heads <= 65535 && n > 0, "rel_bias: bad args");
  rel_bias_kernel<<<dim3(cdiv(n, 256), heads), 256, 0, (hipStream_t)stream>>>(table, index, rel, buckets, heads, n);
  return mgld_check_launch("rel_bias");
}

extern "C" int mgld_rel_bias_grad(const float* drel, const int32_t* index, float* dtable, int buckets, int heads, int n, void* stream) {
  MGLD_REQUIRE(drel && index && dtable && buckets > 0 && buckets <= 65535 && heads > 0 && n > 0, "rel_bias_grad: bad args");
  rel_bias_grad_kernel<<<dim3(heads, buckets), 64, 0, (hipStream_t)stream>>>(drel, index, dtable, heads, n);
  return mgld_check_launch("rel_bias_grad");
}
