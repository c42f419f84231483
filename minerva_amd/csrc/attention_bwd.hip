// Attention of queries to the states of another sequence (or their own), forward and backward.
//   t_ij = scale * q_i.k_j + bias[j - i + q_len - 1] (j < lengths[b]),  m_i = max t_ij,  l_i = sum exp(t_ij - m_i)
//   out_i = sum_j exp(t_ij - m_i) / l_i * v_j
//   p_ij = exp(t_ij - m_i) / l_i,  ds_ij = p_ij * (dout_i.v_j - dout_i.out_i)
//   dq_i = scale * sum_j ds_ij k_j,  dk_j = scale * sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
//   dbias[o] = sum of ds_ij with j - i + q_len - 1 = o
// A row that sees no key has m = -inf, l = 0, out = 0.  The pair (m, l) is kept and not m + ln l: where the bias is the
// type's lowest value for a whole row, ln l would be lost in the sum.
#include "attention_core.h"

namespace {

__device__ __forceinline__ size_t q_row(const AttentionSizes& z, int b, int i, int h) {
  return ((size_t)b * z.q_len + i) * z.heads + h;
}
__device__ __forceinline__ size_t k_row(const AttentionSizes& z, int b, int j, int h) {
  return ((size_t)b * z.k_len + j) * z.kv_heads + h;
}

__device__ __forceinline__ float dot(const float* a, const float* b, int n) {
  float s = 0.f;
  for (int d = 0; d < n; ++d) s = fmaf(a[d], b[d], s);
  return s;
}

__device__ __forceinline__ float score(const AttentionSizes& z, const float* q, const float* k, const float* bias,
                                       int h, int i, int j) {
  const float t = z.scale * dot(q, k, z.dim);
  return bias ? t + bias[(size_t)h * ((size_t)z.q_len + z.k_len - 1) + (j - i + z.q_len - 1)] : t;
}

// exp(t - m), and 0 for a hidden t = -inf where hidden ones alone leave m at -inf too
__device__ __forceinline__ float weight(float t, float m) { return expf(t - (m == -INFINITY ? 0.f : m)); }
struct AttentionGrads {
  const float *q, *k, *v, *bias, *lengths, *out, *stats, *dout;
};

// p_ij and ds_ij of one query and one visible key
__device__ __forceinline__ void pair(const AttentionSizes& z, const AttentionGrads& a, int b, int h, int kh, int i, int j,
                                     float* p, float* ds) {
  const size_t row = q_row(z, b, i, h), key = k_row(z, b, j, kh);
  const float e = weight(score(z, a.q + row * z.dim, a.k + key * z.dim, a.bias, h, i, j), a.stats[2 * row]);
  *p = e * mnv_inverse(a.stats[2 * row + 1]);
  *ds = *p * (dot(a.dout + row * z.dim, a.v + key * z.dim, z.dim) - dot(a.dout + row * z.dim, a.out + row * z.dim, z.dim));
}

// One wavefront per query.
__global__ __launch_bounds__(MNV_WAVE) void mnv_attention_dq_kernel(AttentionGrads a, float* __restrict__ dq,
                                                                    AttentionSizes z) {
  const int lane = threadIdx.x;
  const size_t rows = (size_t)z.batch * z.q_len * z.heads;
  for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int h = (int)(row % z.heads), i = (int)(row / z.heads % z.q_len), b = (int)(row / z.heads / z.q_len);
    const int kh = h / (z.heads / z.kv_heads), n = mnv_visible(a.lengths, b, z.k_len);
    float acc[2] = {0.f, 0.f};
    for (int j0 = 0; j0 < n; j0 += MNV_WAVE) {
      float p = 0.f, ds = 0.f;
      if (j0 + lane < n) pair(z, a, b, h, kh, i, j0 + lane, &p, &ds);
      for (int u = 0; u < MNV_WAVE && j0 + u < n; ++u) {
        const float du = __shfl(ds, u, MNV_WAVE);
        const float* kj = a.k + k_row(z, b, j0 + u, kh) * z.dim;
        if (lane < z.dim) acc[0] = fmaf(du, kj[lane], acc[0]);
        if (lane + MNV_WAVE < z.dim) acc[1] = fmaf(du, kj[lane + MNV_WAVE], acc[1]);
      }
    }
    for (int u = 0; u < 2; ++u)
      if (lane + u * MNV_WAVE < z.dim) dq[row * z.dim + lane + u * MNV_WAVE] = z.scale * acc[u];
  }
}

// One wavefront per key.
__global__ __launch_bounds__(MNV_WAVE) void mnv_attention_dkv_kernel(AttentionGrads a, float* __restrict__ dk,
                                                                     float* __restrict__ dv, AttentionSizes z) {
  const int lane = threadIdx.x;
  const size_t rows = (size_t)z.batch * z.k_len * z.kv_heads;
  const int group = z.heads / z.kv_heads;
  for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const int kh = (int)(row % z.kv_heads), j = (int)(row / z.kv_heads % z.k_len), b = (int)(row / z.kv_heads / z.k_len);
    float sk[2] = {0.f, 0.f}, sv[2] = {0.f, 0.f};
    const int queries = j < mnv_visible(a.lengths, b, z.k_len) ? z.q_len : 0;
    for (int h = kh * group; h < (kh + 1) * group; ++h)
      for (int i0 = 0; i0 < queries; i0 += MNV_WAVE) {
        float p = 0.f, ds = 0.f;
        if (i0 + lane < queries) pair(z, a, b, h, kh, i0 + lane, j, &p, &ds);
        for (int u = 0; u < MNV_WAVE && i0 + u < queries; ++u) {
          const float pu = __shfl(p, u, MNV_WAVE), du = __shfl(ds, u, MNV_WAVE);
          const size_t at = q_row(z, b, i0 + u, h) * z.dim;
          for (int c = 0; c < 2; ++c) {
            const int d = lane + c * MNV_WAVE;
            if (d >= z.dim) continue;
            sv[c] = fmaf(pu, a.dout[at + d], sv[c]);
            sk[c] = fmaf(du, a.q[at + d], sk[c]);
          }
        }
      }
    for (int c = 0; c < 2; ++c) {
      const int d = lane + c * MNV_WAVE;
      if (d >= z.dim) continue;
      dk[row * z.dim + d] = z.scale * sk[c];
      dv[row * z.dim + d] = sv[c];
    }
  }
}

// One wavefront per head and offset.
__global__ __launch_bounds__(MNV_WAVE) void mnv_attention_dbias_kernel(AttentionGrads a, float* __restrict__ dbias,
                                                                       AttentionSizes z) {
  const long long offsets = (long long)z.q_len + z.k_len - 1;
  for (long long at = blockIdx.x; at < offsets * z.heads; at += gridDim.x) {
    const int h = (int)(at / offsets), o = (int)(at % offsets);
    const int kh = h / (z.heads / z.kv_heads);
    float s = 0.f;
    for (int b = 0; b < z.batch; ++b) {
      const int n = mnv_visible(a.lengths, b, z.k_len);
      for (int i = threadIdx.x; i < z.q_len; i += MNV_WAVE) {
        const int j = o + i - (z.q_len - 1);
        if (j < 0 || j >= n) continue;
        float p, ds;
        pair(z, a, b, h, kh, i, j, &p, &ds);
        s += ds;
      }
    }
    s = mnv_wave_sum(s);
    if (threadIdx.x == 0) dbias[at] = s;
  }
}

unsigned row_grid(size_t rows) { return (unsigned)(rows < (1u << 20) ? rows : (1u << 20)); }

}  // namespace

extern "C" {

size_t mnv_attention_bwd_workspace_bytes(int, int, int, int, int, int, int) { return 0; }

int mnv_attention_bwd(const float* q, const float* k, const float* v, const float* bias, const float* lengths,
                      const float* out, const float* stats, const float* dout, float* dq, float* dk, float* dv,
                      float* dbias, int batch, int heads, int kv_heads, int q_len, int k_len, int head_dim, float scale,
                      void*, size_t, mnv_stream_t stream) {
  const AttentionSizes z = {batch, heads, kv_heads, q_len, k_len, head_dim, scale};
  if (!q || !k || !v || !out || !stats || !dout || !dq || !dk || !dv || (bias && !dbias) || !mnv_attention_sizes_ok(z))
    return MNV_ERR_INVALID;
  const hipStream_t s = mnv_stream(stream);
  const AttentionGrads a = {q, k, v, bias, lengths, out, stats, dout};
  hipLaunchKernelGGL(mnv_attention_dq_kernel, dim3(row_grid((size_t)batch * q_len * heads)), dim3(MNV_WAVE), 0, s, a,
                     dq, z);
  MNV_HIP_TRY(hipGetLastError());
  hipLaunchKernelGGL(mnv_attention_dkv_kernel, dim3(row_grid((size_t)batch * k_len * kv_heads)), dim3(MNV_WAVE), 0, s,
                     a, dk, dv, z);
  MNV_HIP_TRY(hipGetLastError());
  if (bias)
    hipLaunchKernelGGL(mnv_attention_dbias_kernel, dim3(row_grid(((size_t)q_len + k_len - 1) * heads)), dim3(MNV_WAVE),
                       0, s, a, dbias, z);
  return MNV_LAUNCH_STATUS();
}

}  // extern "C"
