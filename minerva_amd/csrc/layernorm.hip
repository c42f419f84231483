// Layer norm over dimension 0 of {features, count}, forward and backward.
//   xh = (x - mean) * r, r = 1 / sqrt(var + eps);  y = gamma * xh + beta
//   dx = r * (g - mean(g) - xh * mean(g * xh)), g = gamma * dy;  dgamma = sum dy * xh;  dbeta = sum dy
// The variance is the mean of squared differences from the mean (two passes over a column), never a
// difference of squares, so a large mean costs no digits.
// Roofline: HBM bandwidth, 8 bytes per element forward and 12 backward.
#include <math.h>

#include "mnv_common.h"

namespace {

#define MNV_LN_THREADS 256

// Sum over the workgroup, the same bits in every thread; lds: one float per wavefront.
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = mnv_wave_sum(v);
  __syncthreads();
  if (threadIdx.x % MNV_WAVE == 0) lds[threadIdx.x / MNV_WAVE] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < MNV_LN_THREADS / MNV_WAVE; ++w) v += lds[w];
  return v;
}

__device__ __forceinline__ void column_stats(const float* x, int features, float eps, float* lds, float* mean,
                                             float* r) {
  float s = 0.f;
  for (int f = threadIdx.x; f < features; f += MNV_LN_THREADS) s += x[f];
  *mean = block_sum(s, lds) / features;
  s = 0.f;
  for (int f = threadIdx.x; f < features; f += MNV_LN_THREADS) {
    const float d = x[f] - *mean;
    s += d * d;
  }
  *r = 1.f / sqrtf(block_sum(s, lds) / features + eps);
}

__global__ __launch_bounds__(MNV_LN_THREADS) void mnv_layernorm_fwd_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta,
    float* __restrict__ y, int features, int count, float eps) {
  __shared__ float lds[MNV_LN_THREADS / MNV_WAVE];
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    const float* xc = x + (size_t)c * features;
    float* yc = y + (size_t)c * features;
    float mean, r;
    column_stats(xc, features, eps, lds, &mean, &r);
    for (int f = threadIdx.x; f < features; f += MNV_LN_THREADS) yc[f] = gamma[f] * ((xc[f] - mean) * r) + beta[f];
  }
}

// parts: [gridDim.x][2][features] partial sums over the columns of each workgroup, dgamma then dbeta.
__global__ __launch_bounds__(MNV_LN_THREADS) void mnv_layernorm_bwd_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ dy,
    float* __restrict__ dx, float* __restrict__ parts_gamma, float* __restrict__ parts_beta, size_t part_pitch,
    int features, int count, float eps) {
  __shared__ float lds[MNV_LN_THREADS / MNV_WAVE];
  float* pg = parts_gamma + blockIdx.x * part_pitch;
  float* pb = parts_beta + blockIdx.x * part_pitch;
  for (int f = threadIdx.x; f < features; f += MNV_LN_THREADS) pg[f] = pb[f] = 0.f;
  for (int c = blockIdx.x; c < count; c += gridDim.x) {
    const float* xc = x + (size_t)c * features;
    const float* dyc = dy + (size_t)c * features;
    float* dxc = dx + (size_t)c * features;
    float mean, r;
    column_stats(xc, features, eps, lds, &mean, &r);
    float sg = 0.f, sgx = 0.f;
    for (int f = threadIdx.x; f < features; f += MNV_LN_THREADS) {
      const float g = gamma[f] * dyc[f];
      sg += g;
      sgx += g * ((xc[f] - mean) * r);
    }
    sg = block_sum(sg, lds) / features;
    sgx = block_sum(sgx, lds) / features;
    for (int f = threadIdx.x; f < features; f += MNV_LN_THREADS) {
      const float d = dyc[f], xh = (xc[f] - mean) * r;
      dxc[f] = r * (gamma[f] * d - sg - xh * sgx);
      pg[f] += d * xh;  // each thread has its own features throughout
      pb[f] += d;
    }
  }
}

__global__ __launch_bounds__(MNV_LN_THREADS) void mnv_layernorm_sums_kernel(const float* __restrict__ parts, int num,
                                                                            float* __restrict__ dgamma,
                                                                            float* __restrict__ dbeta, int features) {
  const int f = blockIdx.x * MNV_LN_THREADS + threadIdx.x;
  if (f >= features) return;
  float* out = blockIdx.y ? dbeta : dgamma;
  const float* p = parts + (size_t)blockIdx.y * features + f;
  float s = 0.f;
  for (int i = 0; i < num; ++i) s += p[(size_t)i * 2 * features];
  out[f] = s;
}

bool sizes_ok(int features, int count, float eps) {
  return features > 0 && count > 0 && (long long)features * count <= 0x7fffffffLL && eps >= 0.f && eps <= 3e38f;
}

int bwd_workgroups(int count) { return count < 512 ? count : 512; }

}  // namespace

extern "C" {

int mnv_layernorm_fwd(const float* x, const float* gamma, const float* beta, float* y, int features, int count,
                      float eps, mnv_stream_t stream) {
  if (!x || !gamma || !beta || !y || !sizes_ok(features, count, eps)) return MNV_ERR_INVALID;
  const unsigned grid = count < (int)MNV_MAX_STREAM_BLOCKS ? count : MNV_MAX_STREAM_BLOCKS;
  hipLaunchKernelGGL(mnv_layernorm_fwd_kernel, dim3(grid), dim3(MNV_LN_THREADS), 0, mnv_stream(stream), x, gamma,
                     beta, y, features, count, eps);
  return MNV_LAUNCH_STATUS();
}

size_t mnv_layernorm_bwd_workspace_bytes(int features, int count) {
  if (!sizes_ok(features, count, 0.f)) return 0;
  return (size_t)bwd_workgroups(count) * 2 * features * sizeof(float);
}

int mnv_layernorm_bwd(const float* x, const float* gamma, const float* dy, float* dx, float* dgamma, float* dbeta,
                      int features, int count, float eps, void* workspace, size_t workspace_bytes,
                      mnv_stream_t stream) {
  if (!x || !gamma || !dy || !dx || !dgamma || !dbeta || !sizes_ok(features, count, eps)) return MNV_ERR_INVALID;
  const hipStream_t s = mnv_stream(stream);
  const size_t part = (size_t)2 * features * sizeof(float);
  size_t groups = workspace ? workspace_bytes / part : 0;
  if (groups > (size_t)bwd_workgroups(count)) groups = bwd_workgroups(count);
  if (groups < 2) {  // one workgroup sums straight into the results
    hipLaunchKernelGGL(mnv_layernorm_bwd_kernel, dim3(1), dim3(MNV_LN_THREADS), 0, s, x, gamma, dy, dx, dgamma,
                       dbeta, (size_t)0, features, count, eps);
    return MNV_LAUNCH_STATUS();
  }
  float* parts = static_cast<float*>(workspace);
  hipLaunchKernelGGL(mnv_layernorm_bwd_kernel, dim3((unsigned)groups), dim3(MNV_LN_THREADS), 0, s, x, gamma, dy, dx,
                     parts, parts + features, (size_t)2 * features, features, count, eps);
  MNV_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(mnv_layernorm_sums_kernel, dim3((unsigned)mnv_ceil_div(features, MNV_LN_THREADS), 2),
                     dim3(MNV_LN_THREADS), 0, s, parts, (int)groups, dgamma, dbeta, features);
  return MNV_LAUNCH_STATUS();
}

}  // extern "C"
