// Learned relative position bias by buckets, forward and backward.
//   bias[o][h] = table[bucket(r)][h] for every offset o = j - i + q_len - 1 between key j and query i,
//   r = j - i - q_start;  dtable[u][h] = sum of dbias over the offsets of bucket u.
// A bucket is a run of distances, so its offsets are a run of the bias's elements: the buckets'
// borders are computed once per call on the host (in 64 bits, whole numbers afterwards) and go to the kernels
// by value.  Forward: one thread per offset finds its bucket by bisection and copies; backward: one
// workgroup per bucket and head sums its run in a fixed order, so the bits do not depend on chance.
// Bound by launch latency: 16 heads of 32767 offsets are 2 MB, forward 4.1 us, backward 9.9 (a workgroup goes through the
// 15000 offsets of the farthest bucket); 12 heads of 511 offsets about 3 us each.
#include <math.h>

#include "mnv_common.h"

namespace {

#define MNV_RB_MAX_BUCKETS 256

// Distances of bucket u of one direction: from[u] <= n < from[u + 1].
struct RelativeBuckets {
  int from[MNV_RB_MAX_BUCKETS + 1];
  int each;       // buckets of one direction
  int both_ways;
  int zero;       // the offset o with r = 0 (may lie outside the bias)
  int offsets;
};

// A whole number of 32 bits to a word, the lowest first, for products of powers.
struct WholeNumber {
  unsigned words[MNV_RB_MAX_BUCKETS / 2 + 2] = {1};  // of up to 128 factors below 2^31
  int used = 1;
  void times(unsigned x) {
    unsigned long long carry = 0;
    for (int i = 0; i < used; ++i) {
      carry += (unsigned long long)words[i] * x;
      words[i] = (unsigned)carry;
      carry >>= 32;
    }
    if (carry) words[used++] = (unsigned)carry;
  }
  bool at_least(const WholeNumber& o) const {
    if (used != o.used) return used > o.used;
    for (int i = used; i-- > 0;)
      if (words[i] != o.words[i]) return words[i] > o.words[i];
    return true;
  }
};
// Whether n >= exact * (max_distance / exact)^(u / steps), as powers: n^steps >= max_distance^u exact^(steps - u).
bool reaches_border(int n, int exact, int max_distance, int u, int steps) {
  WholeNumber a, b;
  for (int i = 0; i < steps; ++i) {
    a.times((unsigned)n);
    b.times((unsigned)(i < u ? max_distance : exact));
  }
  return a.at_least(b);
}

// Fills b; false for arguments that the header does not allow.
bool make_buckets(RelativeBuckets* b, int buckets, int heads, int q_len, int k_len, int q_start,
                  int max_distance, int both_ways) {
  if (heads < 1 || q_len < 1 || k_len < 1 || q_start < -(1 << 30) || q_start > (1 << 30)) return false;
  if (buckets < (both_ways ? 4 : 2) || buckets > MNV_RB_MAX_BUCKETS || (both_ways && buckets % 2)) return false;
  const long long offsets = (long long)q_len + k_len - 1;
  if (offsets * heads > 0x7fffffffLL) return false;
  b->each = both_ways ? buckets / 2 : buckets;
  b->both_ways = both_ways != 0;
  const int exact = b->each / 2, steps = b->each - exact;
  if (max_distance <= exact) return false;
  for (int u = 0; u <= exact; ++u) b->from[u] = u;
  for (int u = 1; u < steps; ++u) {
    const double at = exact * pow((double)max_distance / exact, (double)u / steps);
    // next to a whole number, where the rounding of pow could put it on either side, whole numbers decide
    const double whole = rint(at);
    if (fabs(at - whole) <= 1e-12 * at)
      b->from[exact + u] = (int)whole + (reaches_border((int)whole, exact, max_distance, u, steps) ? 0 : 1);
    else
      b->from[exact + u] = (int)ceil(at);
  }
  b->from[b->each] = 0x7fffffff;
  b->offsets = (int)offsets;
  const long long zero = (long long)q_len - 1 + q_start;
  if (zero < -0x7fffffffLL || zero > 0x7fffffffLL) return false;
  b->zero = (int)zero;
  return true;
}

__global__ __launch_bounds__(256) void mnv_relative_bias_fwd_kernel(const float* __restrict__ table,
                                                                    float* __restrict__ bias, RelativeBuckets b,
                                                                    int heads) {
  const unsigned o = blockIdx.x * 256u + threadIdx.x;
  if (o >= (unsigned)b.offsets) return;
  const long long r = (long long)o - b.zero;
  int first = 0;
  long long n = -r;
  if (r > 0) {
    first = b.both_ways ? b.each : 0;
    n = b.both_ways ? r : 0;
  }
  // the last u with from[u] <= n
  int low = 0, high = b.each;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (b.from[mid] <= n) low = mid;
    else high = mid;
  }
  const float* row = table + (size_t)(first + low) * heads;
  for (int h = blockIdx.y; h < heads; h += gridDim.y) bias[(size_t)h * b.offsets + o] = row[h];
}

__global__ __launch_bounds__(256) void mnv_relative_bias_bwd_kernel(const float* __restrict__ dbias,
                                                                    float* __restrict__ dtable, RelativeBuckets b,
                                                                    int heads) {
  __shared__ float lds[4];
  const int u = blockIdx.x % b.each;
  const bool above = blockIdx.x >= (unsigned)b.each;
  // the run [begin, end) of offsets whose distance lies in the bucket
  const long long from = b.from[u], to = u + 1 < b.each ? b.from[u + 1] : (1LL << 40);
  long long begin, end;
  if (above) {
    begin = b.zero + (from > 1 ? from : 1);  // r > 0
    end = b.zero + to;
  } else {
    begin = b.zero - to + 1;  // -to < r <= -from
    end = b.zero - from + 1;
    if (u == 0 && !b.both_ways) end = b.offsets;  // r >= 0 all have distance 0
  }
  if (begin < 0) begin = 0;
  if (end > b.offsets) end = b.offsets;
  for (int h = blockIdx.y; h < heads; h += gridDim.y) {
    const float* d = dbias + (size_t)h * b.offsets;
    // four chains: as many loads in flight, and shorter sums; none of more than 1024 offsets, whose sums are added up by
    // themselves (2^26 offsets with gradients of 1.1: off by 1.1e-5, 6.6e-4 with one chain for all)
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    for (long long first = begin; first < end; first += 1 << 20) {
      const long long last = first + (1 << 20) < end ? first + (1 << 20) : end;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      for (long long o = first + threadIdx.x; o < last; o += 1024) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (o + 256 * c < last) sum[c] += d[o + 256 * c];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) total[c] += sum[c];
    }
    const float s = mnv_wave_sum((total[0] + total[1]) + (total[2] + total[3]));
    __syncthreads();
    if (threadIdx.x % MNV_WAVE == 0) lds[threadIdx.x / MNV_WAVE] = s;
    __syncthreads();
    if (threadIdx.x == 0)
      dtable[(size_t)blockIdx.x * heads + h] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
}

}  // namespace

extern "C" {

int mnv_relative_bias_fwd(const float* table, float* bias, int buckets, int heads, int q_len, int k_len,
                          int q_start, int max_distance, int both_ways, mnv_stream_t stream) {
  RelativeBuckets b;
  if (!table || !bias || !make_buckets(&b, buckets, heads, q_len, k_len, q_start, max_distance, both_ways))
    return MNV_ERR_INVALID;
  const dim3 grid((unsigned)mnv_ceil_div(b.offsets, 256), heads < 65535 ? heads : 65535);
  hipLaunchKernelGGL(mnv_relative_bias_fwd_kernel, grid, dim3(256), 0, mnv_stream(stream), table, bias, b, heads);
  return MNV_LAUNCH_STATUS();
}

int mnv_relative_bias_bwd(const float* dbias, float* dtable, int buckets, int heads, int q_len,
                          int k_len, int q_start, int max_distance, int both_ways, mnv_stream_t stream) {
  RelativeBuckets b;
  if (!dbias || !dtable || !make_buckets(&b, buckets, heads, q_len, k_len, q_start, max_distance, both_ways))
    return MNV_ERR_INVALID;
  const dim3 grid(buckets, heads < 65535 ? heads : 65535);
  hipLaunchKernelGGL(mnv_relative_bias_bwd_kernel, grid, dim3(256), 0, mnv_stream(stream), dbias, dtable, b, heads);
  return MNV_LAUNCH_STATUS();
}

}  // extern "C"
