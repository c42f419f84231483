// Layer norm over dimension 0 of {features, count}, forward and backward.
//   xh = (x - mean) * r, r = 1 / sqrt(var + eps);  y = gamma * xh + beta
//   dx = r * (g - mean(g) - xh * mean(g * xh)), g = gamma * dy;  dgamma = sum dy * xh;  dbeta = sum dy
// The variance is the mean of squared differences from the mean (two passes over a column), never a
// difference of squares.  A mean in fp32 is off by up to half a step of its own size and a sum's roundings, far more than the
// values' differences may bear (mean 10^5, deviation 1: results off by 0.05, those of a constant column by 1), but the
// differences from it are exact where it is large; so their own mean is summed with their squares, and taken off.
// Bound by HBM, 8 bytes per element forward and 12 backward: a column of up to 16384 values is held in registers
// between the passes, so it is read once, by as few threads as hold it with 4 to 16 values each (16 lanes to 64 features,
// 512 threads to 8192; 32 values backward of more), and a group of threads goes from column to column.  backward sums dgamma and dbeta in
// registers over the columns of a group, each thread its own features, and leaves one partial sum per
// workgroup to a second kernel.  4096 x 8192 forward: 41.2 us again and again on the same 268 MB, which the
// caches partly hold, 50.2 us on other data from call to call = 5.3 TB/s (a large copy: 4.7, an addition 5.9); backward of
// 512 x 65536: 65.8 us and 6 for the second kernel, 79 us on other data = 5.1 TB/s; 999 x 4099: 14.9 and 4 us.
// Small ones are a launch (256 x 4: 1.9 us).
#include <math.h>

#include "mnv_common.h"

namespace {

// v + its neighbour's by a row shift or broadcast of the vector unit itself, no trip through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ float add_dpp(float v) {
  const int other = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false);
  return v + __builtin_bit_cast(float, other);
}
// Sum over a wavefront, in a scalar register.
__device__ __forceinline__ float wave_total(float v) {
  v = add_dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8: lane 15 of each row of 16 has the row's sum
  v = add_dpp<0x112, 0xf>(v);
  v = add_dpp<0x114, 0xf>(v);
  v = add_dpp<0x118, 0xf>(v);
  v = add_dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3, row_bcast:31 into rows 2 and 3
  v = add_dpp<0x143, 0xc>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// Sums over GROUP neighbouring threads, the same bits in each of them; lds: N floats per wavefront.
template <int GROUP, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* lds) {
  if (GROUP < MNV_WAVE) {
#pragma unroll
    for (int o = GROUP / 2; o > 0; o >>= 1)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], o, MNV_WAVE);
    return;
  }
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = wave_total(v[n]);
  if (GROUP > MNV_WAVE) {
    constexpr int W = GROUP / MNV_WAVE;
    __syncthreads();
    if (threadIdx.x % MNV_WAVE == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) lds[n * W + threadIdx.x / MNV_WAVE] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = lds[n * W];
#pragma unroll
      for (int w = 1; w < W; ++w) v[n] += lds[n * W + w];
    }
  }
}
template <int GROUP>
__device__ __forceinline__ float group_sum(float v, float* lds) {
  float a[1] = {v};
  group_sum<GROUP, 1>(a, lds);
  return a[0];
}
template <int GROUP>
__device__ __forceinline__ void group_sum2(float& a, float& b, float* lds) {
  float v[2] = {a, b};
  group_sum<GROUP, 2>(v, lds);
  a = v[0];
  b = v[1];
}

// Four values from p on, of which `left` (1 or more) exist; 0 for the others.  VEC: all or none exist.
template <bool VEC, bool NT>
__device__ __forceinline__ mnv_f4 load4(const float* p, int left) {
  if (VEC || left >= 4) return mnv_ldx4u<NT>(p);
  return mnv_f4{p[0], left > 1 ? p[1] : 0.f, left > 2 ? p[2] : 0.f, 0.f};
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, int left, mnv_f4 v) {
  if (VEC || left >= 4) {
    if (VEC) __builtin_nontemporal_store(v, reinterpret_cast<mnv_f4u*>(p));
    else *reinterpret_cast<mnv_f4u*>(p) = v;
    return;
  }
  p[0] = v.x;
  if (left > 1) p[1] = v.y;
  if (left > 2) p[2] = v.z;
}

// 1 / sqrt(var + eps) from the mean of squared differences from a mean that is off by d, the differences' own mean.
__device__ __forceinline__ float inverse_deviation(float squares, float d, float eps) {
  const float var = squares - d * d;
  return 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);
}

// One column per GROUP threads of a workgroup, CACHE vectors of four values per thread.
template <int GROUP, int CACHE>
struct Column {
  mnv_f4 x[CACHE];
  float r;
  int t, features;  // the thread's first feature, and the number of all

  __device__ __forceinline__ int left(int u) const { return features - (t + 4 * u * GROUP); }

  template <bool VEC, bool NT>
  __device__ __forceinline__ void load(mnv_f4 (&v)[CACHE], const float* column) const {
#pragma unroll
    for (int u = 0; u < CACHE; ++u) v[u] = left(u) > 0 ? load4<VEC, NT>(column + t + 4 * u * GROUP, left(u)) : mnv_f4{0.f, 0.f, 0.f, 0.f};
  }
  // What stands in x becomes its difference from the mean (0 behind the last feature).
  __device__ __forceinline__ void centre(float eps, float* lds) {
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < CACHE; ++u) s += (x[u].x + x[u].y) + (x[u].z + x[u].w);
    const float mean = group_sum<GROUP>(s, lds) / features;
    float d = 0.f, sq = 0.f;
#pragma unroll
    for (int u = 0; u < CACHE; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[u][e] = left(u) > e ? x[u][e] - mean : 0.f;
        d += x[u][e];
        sq = fmaf(x[u][e], x[u][e], sq);
      }
    group_sum2<GROUP>(d, sq, lds);
    d /= features;
    r = inverse_deviation(sq / features, d, eps);
#pragma unroll
    for (int u = 0; u < CACHE; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[u][e] = left(u) > e ? x[u][e] - d : 0.f;
  }
};

template <int GROUP, int CACHE, int NTH, bool VEC, bool NT>
__global__ __launch_bounds__(NTH) void mnv_layernorm_fwd_kernel(const float* __restrict__ x, const float* __restrict__ gamma,
                                                                const float* __restrict__ beta, float* __restrict__ y,
                                                                int features, unsigned count, float eps) {
  __shared__ float lds[GROUP > MNV_WAVE ? 2 * NTH / MNV_WAVE : 1];
  constexpr int PER = NTH / GROUP;
  Column<GROUP, CACHE> c;
  c.t = threadIdx.x % GROUP * 4;
  c.features = features;
  mnv_f4 g[CACHE], b[CACHE];
  c.template load<VEC, false>(g, gamma);
  c.template load<VEC, false>(b, beta);
  // the next column is fetched while this one is summed (behind the last that one again)
  mnv_f4 next[CACHE];
  const unsigned first = blockIdx.x * PER + (PER > 1 ? threadIdx.x / GROUP : 0), step = gridDim.x * PER;
  if (first < count) c.template load<VEC, NT>(next, x + (size_t)first * features);
  for (unsigned i = first; i < count; i += step) {
#pragma unroll
    for (int u = 0; u < CACHE; ++u) c.x[u] = next[u];
    c.template load<VEC, NT>(next, x + (size_t)(i + step < count ? i + step : i) * features);
    c.centre(eps, lds);
    float* out = y + (size_t)i * features + c.t;
#pragma unroll
    for (int u = 0; u < CACHE; ++u) {
      if (c.left(u) <= 0) continue;
      mnv_f4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = g[u][e] * (c.x[u][e] * c.r) + b[u][e];
      store4<VEC>(out + 4 * u * GROUP, c.left(u), o);
    }
  }
}

// parts: 2 x features sums of each workgroup, dgamma then dbeta.
template <int GROUP, int CACHE, int NTH, bool VEC, bool NT>
__global__ __launch_bounds__(NTH) void mnv_layernorm_bwd_kernel(const float* __restrict__ x, const float* __restrict__ gamma,
                                                                const float* __restrict__ dy, float* __restrict__ dx,
                                                                float* __restrict__ parts_gamma,
                                                                float* __restrict__ parts_beta, size_t part_pitch,
                                                                int features, unsigned count, float eps) {
  constexpr int PER = NTH / GROUP;
  __shared__ float lds[GROUP > MNV_WAVE ? 2 * NTH / MNV_WAVE : 1];
  __shared__ mnv_f4 joined[PER > 1 ? NTH : 1];
  Column<GROUP, CACHE> c;
  c.t = threadIdx.x % GROUP * 4;
  c.features = features;
  mnv_f4 g[CACHE], sg[CACHE], sb[CACHE];
  c.template load<VEC, false>(g, gamma);
#pragma unroll
  for (int u = 0; u < CACHE; ++u) sg[u] = sb[u] = mnv_f4{0.f, 0.f, 0.f, 0.f};
  // the next column is fetched while this one is summed (behind the last that one again); of wider ones it costs
  // registers that more workgroups to a CU use better (4096 x 8192: 85 us with, 80 without; 8192 x 1000: 38 and 32)
  constexpr bool AHEAD = CACHE <= 2;
  mnv_f4 next_x[CACHE], next_d[CACHE];
  const unsigned first = blockIdx.x * PER + (PER > 1 ? threadIdx.x / GROUP : 0), step = gridDim.x * PER;
  if (AHEAD && first < count) {
    c.template load<VEC, NT>(next_x, x + (size_t)first * features);
    c.template load<VEC, NT>(next_d, dy + (size_t)first * features);
  }
  for (unsigned i = first; i < count; i += step) {
    mnv_f4 d[CACHE];
    if (AHEAD) {
#pragma unroll
      for (int u = 0; u < CACHE; ++u) {
        c.x[u] = next_x[u];
        d[u] = next_d[u];
      }
      const size_t at = (size_t)(i + step < count ? i + step : i) * features;
      c.template load<VEC, NT>(next_x, x + at);
      c.template load<VEC, NT>(next_d, dy + at);
    } else {
      c.template load<VEC, NT>(c.x, x + (size_t)i * features);
      c.template load<VEC, NT>(d, dy + (size_t)i * features);
    }
    c.centre(eps, lds);
    float s = 0.f, sx = 0.f;
#pragma unroll
    for (int u = 0; u < CACHE; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c.x[u][e] *= c.r;  // xh
        const float gd = g[u][e] * d[u][e];
        s += gd;
        sx = fmaf(gd, c.x[u][e], sx);
        sg[u][e] = fmaf(d[u][e], c.x[u][e], sg[u][e]);
        sb[u][e] += d[u][e];
      }
    group_sum2<GROUP>(s, sx, lds);
    s /= features;
    sx /= features;
    float* out = dx + (size_t)i * features + c.t;
#pragma unroll
    for (int u = 0; u < CACHE; ++u) {
      if (c.left(u) <= 0) continue;
      mnv_f4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = c.r * (g[u][e] * d[u][e] - s - c.x[u][e] * sx);
      store4<VEC>(out + 4 * u * GROUP, c.left(u), o);
    }
  }
  float* pg = parts_gamma + blockIdx.x * part_pitch + c.t;
  float* pb = parts_beta + blockIdx.x * part_pitch + c.t;
#pragma unroll
  for (int u = 0; u < CACHE; ++u) {
    if (PER > 1) {  // the groups' sums, one after the other
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        mnv_f4& mine = which ? sb[u] : sg[u];
        __syncthreads();
        joined[threadIdx.x] = mine;
        __syncthreads();
        if (threadIdx.x < GROUP) {
#pragma unroll
          for (int q = 1; q < PER; ++q) mine += joined[threadIdx.x + q * GROUP];
        }
      }
      if (threadIdx.x >= GROUP) continue;
    }
    if (c.left(u) <= 0) continue;
    store4<false>(pg + 4 * u * GROUP, c.left(u), sg[u]);
    store4<false>(pb + 4 * u * GROUP, c.left(u), sb[u]);
  }
}

// Columns of more values than the register forms hold: each pass reads the column again, value by value, three times forward
// and four times backward, where the sums of dgamma and dbeta go through memory with every column (20001 x 1000: 49 and 177 us).
#define MNV_LN_WIDE 1024
// A column's mean is a first one and the mean of the differences from it.
struct WideStats {
  float mean, rest, r;
  __device__ __forceinline__ float xh(float x) const { return (x - mean - rest) * r; }
};
__device__ __forceinline__ WideStats wide_stats(const float* x, unsigned features, float eps, float* lds) {  // lds: 2 floats per wavefront
  WideStats w;
  float s = 0.f;
  for (unsigned f = threadIdx.x; f < features; f += MNV_LN_WIDE) s += x[f];
  w.mean = group_sum<MNV_LN_WIDE>(s, lds) / features;
  float sum = 0.f, sq = 0.f;
  for (unsigned f = threadIdx.x; f < features; f += MNV_LN_WIDE) {
    const float d = x[f] - w.mean;
    sum += d;
    sq = fmaf(d, d, sq);
  }
  group_sum2<MNV_LN_WIDE>(sum, sq, lds);
  w.rest = sum / features;
  w.r = inverse_deviation(sq / features, w.rest, eps);
  return w;
}
__global__ __launch_bounds__(MNV_LN_WIDE) void mnv_layernorm_fwd_wide_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta, float* __restrict__ y,
    unsigned features, unsigned count, float eps) {
  __shared__ float lds[2 * MNV_LN_WIDE / MNV_WAVE];
  for (unsigned i = blockIdx.x; i < count; i += gridDim.x) {
    const float* xc = x + (size_t)i * features;
    float* yc = y + (size_t)i * features;
    const WideStats w = wide_stats(xc, features, eps, lds);
    for (unsigned f = threadIdx.x; f < features; f += MNV_LN_WIDE) yc[f] = gamma[f] * w.xh(xc[f]) + beta[f];
  }
}
__global__ __launch_bounds__(MNV_LN_WIDE) void mnv_layernorm_bwd_wide_kernel(
    const float* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ dy, float* __restrict__ dx,
    float* __restrict__ parts_gamma, float* __restrict__ parts_beta, size_t part_pitch, unsigned features, unsigned count, float eps) {
  __shared__ float lds[2 * MNV_LN_WIDE / MNV_WAVE];
  float* pg = parts_gamma + blockIdx.x * part_pitch;
  float* pb = parts_beta + blockIdx.x * part_pitch;
  for (unsigned f = threadIdx.x; f < features; f += MNV_LN_WIDE) pg[f] = pb[f] = 0.f;
  for (unsigned i = blockIdx.x; i < count; i += gridDim.x) {
    const float* xc = x + (size_t)i * features;
    const float* dyc = dy + (size_t)i * features;
    float* dxc = dx + (size_t)i * features;
    const WideStats w = wide_stats(xc, features, eps, lds);
    float s = 0.f, sx = 0.f;
    for (unsigned f = threadIdx.x; f < features; f += MNV_LN_WIDE) {
      const float gd = gamma[f] * dyc[f];
      s += gd;
      sx = fmaf(gd, w.xh(xc[f]), sx);
    }
    group_sum2<MNV_LN_WIDE>(s, sx, lds);
    s /= features;
    sx /= features;
    for (unsigned f = threadIdx.x; f < features; f += MNV_LN_WIDE) {
      const float d = dyc[f], xh = w.xh(xc[f]);
      dxc[f] = w.r * (gamma[f] * d - s - xh * sx);
      pg[f] = fmaf(d, xh, pg[f]);  // each thread has its own features throughout
      pb[f] += d;
    }
  }
}

// dgamma, dbeta (blockIdx.y) = the sums of the workgroups' parts: 16 features to a workgroup, 64 threads to a feature, each with
// every 64th part (768 parts of 512 features: 3 loads in a row per chain).
__global__ __launch_bounds__(1024) void mnv_layernorm_sums_kernel(const float* __restrict__ parts, int num,
                                                                  float* __restrict__ dgamma, float* __restrict__ dbeta,
                                                                  unsigned features) {
  __shared__ float lds[64][17];
  const int lane = threadIdx.x % 16, q = threadIdx.x / 16;
  for (unsigned f0 = blockIdx.x * 16; f0 < features; f0 += gridDim.x * 16) {
    const unsigned f = f0 + lane;
    float chain[4] = {0.f, 0.f, 0.f, 0.f};
    if (f < features) {
      const float* p = parts + (size_t)blockIdx.y * features + f;
      for (int i = q; i < num; i += 256) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (i + 64 * c < num) chain[c] += p[(size_t)(i + 64 * c) * 2 * features];
      }
    }
    lds[q][lane] = (chain[0] + chain[1]) + (chain[2] + chain[3]);
    __syncthreads();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      if (q < o) lds[q][lane] += lds[q + o][lane];
      __syncthreads();
    }
    if (q == 0 && f < features) (blockIdx.y ? dbeta : dgamma)[f] = lds[0][lane];
  }
}

bool sizes_ok(int features, int count, float eps) {
  return features > 0 && count > 0 && (long long)features * count <= 0x7fffffffLL && eps >= 0.f && eps <= 3e38f;
}

struct Norm {
  const float *x, *gamma, *beta, *dy;
  float *y, *dx, *pg, *pb;  // backward: the parts, or the results themselves
  size_t part_pitch;
  int features, count;
  float eps;
  unsigned groups;  // backward: workgroups
  hipStream_t s;
};

// Columns that a workgroup has at a time.
int columns_at_once(int features) {
  return features <= 64 ? 16 : features <= 128 ? 8 : features <= 1024 ? 4 : 1;
}

template <int GROUP, int CACHE, int NTH, bool VEC, bool NT>
int launch(const Norm& n) {
  if (n.dy) {
    hipLaunchKernelGGL((mnv_layernorm_bwd_kernel<GROUP, CACHE, NTH, VEC, NT>), dim3(n.groups), dim3(NTH), 0, n.s, n.x,
                       n.gamma, n.dy, n.dx, n.pg, n.pb, n.part_pitch, n.features, n.count, n.eps);
  } else {
    const size_t blocks = mnv_ceil_div(n.count, NTH / GROUP);
    const size_t most = (size_t)mnv_cu_count() * (2048 / NTH);  // what the chip holds at once
    hipLaunchKernelGGL((mnv_layernorm_fwd_kernel<GROUP, CACHE, NTH, VEC, NT>), dim3((unsigned)(blocks < most ? blocks : most)),
                       dim3(NTH), 0, n.s, n.x, n.gamma, n.beta, n.y, n.features, n.count, n.eps);
  }
  return MNV_LAUNCH_STATUS();
}
template <bool VEC, bool NT>
int by_width(const Norm& n) {
  const int f = n.features;
  if (f <= 64) return launch<16, 1, 256, VEC, NT>(n);
  if (f <= 128) return launch<32, 1, 256, VEC, NT>(n);
  if (f <= 256) return launch<64, 1, 256, VEC, NT>(n);
  if (f <= 512) return launch<64, 2, 256, VEC, NT>(n);
  if (f <= 1024) return launch<64, 4, 256, VEC, NT>(n);
  if (f <= 2048) return launch<256, 2, 256, VEC, NT>(n);
  if (f <= 4096) return launch<256, 4, 256, VEC, NT>(n);
  if (f <= 8192) return launch<512, 4, 512, VEC, NT>(n);
  // 16384 x 2048: forward 46 us (before the differences' mean was summed 43, and 54 of 512 threads); backward, whose sums take
  // registers too, 113 of 512 threads and 170 of 1024
  return n.dy ? launch<512, 8, 512, VEC, NT>(n) : launch<1024, 4, 1024, VEC, NT>(n);
}
int run(const Norm& n) {
  if (n.features > 16384) {
    if (n.dy)
      hipLaunchKernelGGL(mnv_layernorm_bwd_wide_kernel, dim3(n.groups), dim3(MNV_LN_WIDE), 0, n.s, n.x, n.gamma, n.dy,
                         n.dx, n.pg, n.pb, n.part_pitch, n.features, n.count, n.eps);
    else
      hipLaunchKernelGGL(mnv_layernorm_fwd_wide_kernel, dim3(n.count < 512 ? n.count : 512), dim3(MNV_LN_WIDE), 0, n.s,
                         n.x, n.gamma, n.beta, n.y, n.features, n.count, n.eps);
    return MNV_LAUNCH_STATUS();
  }
  // past the caches: 8192 x 16384 forward 176 us, 188 through them; backward 304 and 328.  4096 x 8192 fits them: 41 us,
  // and 49 past them
  const bool vec = n.features % 4 == 0, nt = (size_t)n.features * n.count * sizeof(float) >= MNV_PAST_CACHE_BYTES;
  if (vec) return nt ? by_width<true, true>(n) : by_width<true, false>(n);
  return nt ? by_width<false, true>(n) : by_width<false, false>(n);
}

// Workgroups of the backward pass: 3 or 2 to a CU are enough to keep the memory busy, and leave fewer partial sums (512 x
// 65536: 72 us, of 8 to a CU 77; 4096 x 8192: 70, of 4 to a CU 78), and fewer of them where a group would have few
// columns to its sums (2048 x 1000: 14.0 us of two columns or more, 12.7 of four; 64 x 100: 8.1 and 8.6).
// Of very many columns there are more of them, so that no sum of a thread has more than MNV_LN_CHAIN terms (2^28 columns of one
// feature, gradients of 1.1, whose additions all round the same way: dbeta off by 1.1e-5, 2.1e-4 with 21845 in a row).
#define MNV_LN_CHAIN 1024
unsigned bwd_workgroups(int features, int count) {
  const size_t full = (size_t)mnv_cu_count() * (features <= 512 ? 3 : 2);
  const size_t chains = mnv_ceil_div(count, (size_t)columns_at_once(features) * MNV_LN_CHAIN);
  const size_t most = full > chains ? full : chains;
  const size_t groups = mnv_ceil_div(count, (size_t)columns_at_once(features) * (features <= 512 ? 2 : 4));
  return (unsigned)(groups < most ? groups : most);
}

}  // namespace

extern "C" {

int mnv_layernorm_fwd(const float* x, const float* gamma, const float* beta, float* y, int features, int count,
                      float eps, mnv_stream_t stream) {
  if (!x || !gamma || !beta || !y || !sizes_ok(features, count, eps)) return MNV_ERR_INVALID;
  return run(Norm{x, gamma, beta, nullptr, y, nullptr, nullptr, nullptr, 0, features, count, eps, 0, mnv_stream(stream)});
}

size_t mnv_layernorm_bwd_workspace_bytes(int features, int count) {
  if (!sizes_ok(features, count, 0.f)) return 0;
  const size_t groups = bwd_workgroups(features, count);
  return groups > 1 ? groups * 2 * features * sizeof(float) : 0;
}

int mnv_layernorm_bwd(const float* x, const float* gamma, const float* dy, float* dx, float* dgamma, float* dbeta,
                      int features, int count, float eps, void* workspace, size_t workspace_bytes,
                      mnv_stream_t stream) {
  if (!x || !gamma || !dy || !dx || !dgamma || !dbeta || !sizes_ok(features, count, eps)) return MNV_ERR_INVALID;
  const size_t part = (size_t)2 * features * sizeof(float);
  size_t groups = workspace ? workspace_bytes / part : 0;
  const unsigned wanted = bwd_workgroups(features, count);
  if (groups > wanted) groups = wanted;
  Norm n = {x, gamma, nullptr, dy, nullptr, dx, dgamma, dbeta, 0, features, count, eps, 1, mnv_stream(stream)};
  if (groups < 2) return run(n);  // one workgroup sums straight into the results
  float* parts = static_cast<float*>(workspace);
  n.pg = parts;
  n.pb = parts + features;
  n.part_pitch = (size_t)2 * features;
  n.groups = (unsigned)groups;
  const int rc = run(n);
  if (rc) return rc;
  const size_t sums = mnv_ceil_div(features, 16);
  hipLaunchKernelGGL(mnv_layernorm_sums_kernel, dim3((unsigned)(sums < 65536 ? sums : 65536), 2), dim3(1024), 0, n.s, parts,
                     (int)groups, dgamma, dbeta, features);
  return MNV_LAUNCH_STATUS();
}

}  // extern "C"
