// One step of Adam with decoupled weight decay, over many tensors in one launch.
//   m' = beta1 m + (1 - beta1) g,  v' = beta2 v + (1 - beta2) g^2
//   p' = p - rate (m' / (1 - beta1^t) / (sqrt(v' / (1 - beta2^t)) + eps) + decay p)
// Moments are held in 32 bits, or in 8: 256 neighbouring values then share the largest of them (`top`, 32 bits), and a code c
// stands for top (c / 127)^3 of m, -127 to 127, or top (c / 255)^4 of v, 0 to 255: fine near 0, where Adam's
// quotient is made of small numbers.
//   m is rounded to the nearest value: beta1 moves it by several codes' steps.
//   v is not: beta2 = 0.999 moves it by a thousandth, a code's step is 1.6% of it or more, and rounded to the nearest v
//   would never fall.  It goes up where it is more than u of the way to the next code, and u walks evenly through 0 to 1
//   from step to step (u = i 0x85EBCA6B + t 0x9E3779B9 in 32 bits, the golden section's sequence in t): v moves
//   in the mean.  A v above 0 is never rounded to 0, where the quotient would have no bound.
// Codes are chosen in 64 bits, so that they are the definition's and no other rounding decides between two of them; a
// block that holds an infinity or a NaN has `top` NaN, and so has every value of it.
// Bound by HBM: 28 bytes a value with 32-bit moments, 16.06 with 8-bit ones.
#include <math.h>

#include "mnv_common.h"

namespace {

constexpr int BLOCK = 256, WORDS = BLOCK / 4 + 1;  // values of a block; its floats: codes and top
constexpr int CHUNK = 4096;                        // values of a workgroup
constexpr int TENSORS = 48;                        // of a launch: their table is its argument (at most 4 KB)

struct Table {
  const float* p[TENSORS];
  const float* g[TENSORS];
  const float* m[TENSORS];
  const float* v[TENSORS];
  float* p_out[TENSORS];
  float* m_out[TENSORS];
  float* v_out[TENSORS];
  size_t n[TENSORS];
  float rate[TENSORS], decay[TENSORS];  // factors of the step's rate and decay
  int first[TENSORS + 1];               // first workgroup of each; of the tensors that are not there, the grid's size
};
struct Step {
  double beta1, beta2, eps, decay, scale;
  double rate, correct1, correct2;  // 1 / (1 - beta^t)
  unsigned t;
  const float* schedule;  // rate and t instead, as they are when the kernel runs; or null
};
static_assert(sizeof(Table) + sizeof(Step) <= 4096, "a launch's arguments");

// beta^t by squaring
__host__ __device__ inline double power(double beta, unsigned t) {
  double r = 1.0;
  for (; t; t >>= 1, beta *= beta)
    if (t & 1) r *= beta;
  return r;
}

__device__ __forceinline__ int tensor_of(const Table& z, int wg) {
  int low = 0;
#pragma unroll
  for (int half = 32; half > 0; half >>= 1)
    if (low + half < TENSORS && z.first[low + half] <= wg) low += half;
  return low;
}

// The step's factors in 32 bits.
struct Factors {
  float rate, decay, eps, correct1, correct2;
};
__device__ __forceinline__ Factors factors(const Table& z, const Step& s, int tensor, unsigned& t) {
  double rate = s.rate, c1 = s.correct1, c2 = s.correct2;
  t = s.t;
  if (s.schedule) {
    rate = s.schedule[0];
    t = (unsigned)s.schedule[1];
    c1 = 1.0 / (1.0 - power(s.beta1, t));
    c2 = 1.0 / (1.0 - power(s.beta2, t));
  }
  return {(float)(rate * z.rate[tensor]), (float)(s.decay * z.decay[tensor]), (float)s.eps, (float)c1, (float)c2};
}
__device__ __forceinline__ float updated(const Factors& f, float p, float m, float v) {
  const float quotient = m * f.correct1 / (sqrtf(v * f.correct2) + f.eps);
  return p - f.rate * (quotient + f.decay * p);
}

// ---- 32-bit moments: four vectors of four values a thread

template <bool NT>
__device__ __forceinline__ void put4(float* p, mnv_f4 v) {
  if (NT) __builtin_nontemporal_store(v, reinterpret_cast<mnv_f4u*>(p));
  else *reinterpret_cast<mnv_f4u*>(p) = v;
}

template <bool NT>
__global__ __launch_bounds__(256) void adamw_kernel(Table z, Step s) {
  const int tensor = tensor_of(z, (int)blockIdx.x);
  const size_t at = (size_t)((int)blockIdx.x - z.first[tensor]) * CHUNK, n = z.n[tensor];
  const float* __restrict__ p = z.p[tensor];
  const float* __restrict__ g = z.g[tensor];
  const float* __restrict__ m = z.m[tensor];
  const float* __restrict__ v = z.v[tensor];
  unsigned t;
  const Factors f = factors(z, s, tensor, t);
  const float b1 = (float)s.beta1, b2 = (float)s.beta2, a1 = (float)(1.0 - s.beta1), a2 = (float)(1.0 - s.beta2), scale = (float)s.scale;
  auto moments = [&](float gi, float& mi, float& vi) {
    gi *= scale;
    mi = b1 * mi + a1 * gi;
    vi = b2 * vi + a2 * gi * gi;
  };
  if (at + CHUNK <= n) {
    mnv_f4 pv[4], gv[4], mv[4], vv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const size_t i = at + u * 1024 + threadIdx.x * 4;
      gv[u] = mnv_ldx4u<NT>(g + i);
      mv[u] = mnv_ldx4u<NT>(m + i);
      vv[u] = mnv_ldx4u<NT>(v + i);
      pv[u] = mnv_ldx4u<NT>(p + i);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const size_t i = at + u * 1024 + threadIdx.x * 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float mi = mv[u][q], vi = vv[u][q];
        moments(gv[u][q], mi, vi);
        pv[u][q] = updated(f, pv[u][q], mi, vi);
        mv[u][q] = mi;
        vv[u][q] = vi;
      }
      put4<NT>(z.m_out[tensor] + i, mv[u]);
      put4<NT>(z.v_out[tensor] + i, vv[u]);
      put4<NT>(z.p_out[tensor] + i, pv[u]);
    }
  } else {
    for (size_t i = at + threadIdx.x; i < n; i += 256) {
      float mi = m[i], vi = v[i];
      moments(g[i], mi, vi);
      z.p_out[tensor][i] = updated(f, p[i], mi, vi);
      z.m_out[tensor][i] = mi;
      z.v_out[tensor][i] = vi;
    }
  }
}

// ---- 8-bit moments: a wavefront to a block, four values a lane

template <bool SECOND>
struct Code {
  static constexpr int MOST = SECOND ? 255 : 127;
  static constexpr double UNIT = SECOND ? 1.0 / 4228250625.0 : 1.0 / 2048383.0;  // 255^-4, 127^-3
  __device__ static double powers(int c) {
    if (SECOND) {
      const unsigned s = (unsigned)c * (unsigned)c;
      return (double)(s * s);  // 255^4 < 2^32
    }
    return (double)(c * c * c);
  }
  // code q of four
  __device__ static int get(unsigned word, int q) { return SECOND ? (word >> (8 * q)) & 255 : (int)(word << (24 - 8 * q)) >> 24; }
  // The size x's code, between 0 and MOST: unit * powers(code) is the block's value for it.
  __device__ static int choose(float x, float top, double unit, double u) {
    if (!(x > 0.f)) return 0;
    const float share = x / top;
    const float root = SECOND ? sqrtf(sqrtf(share)) : cbrtf(share);
    int c = (int)(root * MOST);
    const double size = x;
    // the root in 32 bits may be off by one code
    if (unit * powers(c) > size) --c;
    else if (c < MOST && unit * powers(c + 1) <= size) ++c;
    const double low = unit * powers(c), high = unit * powers(c + 1);
    if (c < MOST && size - low > u * (high - low)) ++c;
    return SECOND && c == 0 ? 1 : c;
  }
};

// The largest size over a wavefront; NaN where one is an infinity or NaN.
__device__ __forceinline__ float top_of(const float (&x)[4]) {
  // sizes of floats are in the order of their bits, infinities and NaN last
  unsigned most = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const unsigned b = __builtin_bit_cast(unsigned, x[q]) & 0x7fffffffu;
    most = b > most ? b : most;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned b = (unsigned)__shfl_xor((int)most, o, MNV_WAVE);
    most = b > most ? b : most;
  }
  return __builtin_bit_cast(float, most >= 0x7f800000u ? 0x7fc00000u : most);
}

template <bool SECOND>
__device__ __forceinline__ void decode(unsigned word, float top, float (&x)[4]) {
  const double unit = (double)top * Code<SECOND>::UNIT;
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = (float)(unit * Code<SECOND>::powers(Code<SECOND>::get(word, q)));
}

__global__ __launch_bounds__(256) void adamw8_kernel(Table z, Step s) {
  const int tensor = tensor_of(z, (int)blockIdx.x), lane = threadIdx.x % MNV_WAVE;
  const size_t at = (size_t)((int)blockIdx.x - z.first[tensor]) * CHUNK, n = z.n[tensor];
  unsigned t;
  const Factors f = factors(z, s, tensor, t);
  const double a1 = 1.0 - s.beta1, a2 = 1.0 - s.beta2;
  for (int b = threadIdx.x / MNV_WAVE; b < CHUNK / BLOCK; b += 4) {
    const size_t i = at + (size_t)b * BLOCK + lane * 4, block = at / BLOCK + b;
    if (block * BLOCK >= n) return;
    const int left = i >= n ? 0 : n - i < 4 ? (int)(n - i) : 4;
    const float* m = z.m[tensor] + block * WORDS;
    const float* v = z.v[tensor] + block * WORDS;
    float mi[4], vi[4], g[4], p[4];
    decode<false>(__builtin_bit_cast(unsigned, m[lane]), m[BLOCK / 4], mi);
    decode<true>(__builtin_bit_cast(unsigned, v[lane]), v[BLOCK / 4], vi);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      g[q] = q < left ? z.g[tensor][i + q] : 0.f;
      p[q] = q < left ? z.p[tensor][i + q] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const double gi = (double)g[q] * s.scale;
      mi[q] = q < left ? (float)(s.beta1 * (double)mi[q] + a1 * gi) : 0.f;
      vi[q] = q < left ? (float)(s.beta2 * (double)vi[q] + a2 * (gi * gi)) : 0.f;
      if (q < left) z.p_out[tensor][i + q] = updated(f, p[q], mi[q], vi[q]);
    }
    const float mt = top_of(mi), vt = top_of(vi);
    const double mu = (double)mt * Code<false>::UNIT, vu = (double)vt * Code<true>::UNIT;
    unsigned mw = 0, vw = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = Code<false>::choose(fabsf(mi[q]), mt, mu, 0.5);
      const unsigned walk = (unsigned)(i + q) * 0x85EBCA6Bu + t * 0x9E3779B9u;
      mw |= (unsigned)((mi[q] < 0.f ? -c : c) & 255) << (8 * q);
      vw |= (unsigned)Code<true>::choose(vi[q], vt, vu, (double)walk * 2.3283064365386963e-10) << (8 * q);
    }
    float* mo = z.m_out[tensor] + block * WORDS;
    float* vo = z.v_out[tensor] + block * WORDS;
    mo[lane] = __builtin_bit_cast(float, mw);
    vo[lane] = __builtin_bit_cast(float, vw);
    if (lane == 0) {
      mo[BLOCK / 4] = mt;
      vo[BLOCK / 4] = vt;
    }
  }
}

// The values that both moments' codes stand for, in m_out and v_out.
__global__ __launch_bounds__(256) void values_kernel(Table z) {
  const int tensor = tensor_of(z, (int)blockIdx.x), lane = threadIdx.x % MNV_WAVE;
  const size_t at = (size_t)((int)blockIdx.x - z.first[tensor]) * CHUNK, n = z.n[tensor];
  for (int b = threadIdx.x / MNV_WAVE; b < CHUNK / BLOCK; b += 4) {
    const size_t i = at + (size_t)b * BLOCK + lane * 4, block = at / BLOCK + b;
    if (i >= n) return;
    const float* m = z.m[tensor] + block * WORDS;
    const float* v = z.v[tensor] + block * WORDS;
    float mi[4], vi[4];
    decode<false>(__builtin_bit_cast(unsigned, m[lane]), m[BLOCK / 4], mi);
    decode<true>(__builtin_bit_cast(unsigned, v[lane]), v[BLOCK / 4], vi);
    if (n - i >= 4) {
      put4<false>(z.m_out[tensor] + i, mnv_f4{mi[0], mi[1], mi[2], mi[3]});
      put4<false>(z.v_out[tensor] + i, mnv_f4{vi[0], vi[1], vi[2], vi[3]});
    } else {
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (i + q < n) {
          z.m_out[tensor][i + q] = mi[q];
          z.v_out[tensor][i + q] = vi[q];
        }
    }
  }
}

// Goes through the tensors that have values, as many to a launch as its table holds and as a grid has workgroups.
template <class Fill, class Launch>
int for_tables(int count, const size_t* sizes, Fill fill, Launch launch) {
  Table z;
  int used = 0;
  long long groups = 0;
  auto flush = [&]() {
    if (!used) return MNV_OK;
    for (int i = used; i <= TENSORS; ++i) z.first[i] = (int)groups;
    const int rc = launch(z, (unsigned)groups);
    used = 0;
    groups = 0;
    return rc;
  };
  for (int i = 0; i < count; ++i) {
    const size_t chunks = (sizes[i] + CHUNK - 1) / CHUNK;
    if (!chunks) continue;
    if (used == TENSORS || groups + (long long)chunks > 0x7fffffffLL) {
      const int rc = flush();
      if (rc) return rc;
    }
    fill(z, used, i);
    z.n[used] = sizes[i];
    z.first[used++] = (int)groups;
    groups += (long long)chunks;
  }
  return flush();
}

bool in_range(double x, double low, double high) { return x >= low && x < high; }

}  // namespace

extern "C" {

size_t mnv_adamw_moment_floats(size_t n, int bits) {
  if (bits == 32) return n;
  return bits == 8 ? (n / BLOCK + (n % BLOCK != 0)) * WORDS : 0;
}

int mnv_adamw_step(int count, const float* const* params, const float* const* grads, const float* const* m, const float* const* v,
                   float* const* params_out, float* const* m_out, float* const* v_out, const size_t* sizes, const float* rates,
                   const float* decays, int bits, double rate, double beta1, double beta2, double eps, double weight_decay,
                   double grad_scale, int step, const float* schedule, mnv_stream_t stream) {
  if (count < 0 || (bits != 8 && bits != 32)) return MNV_ERR_INVALID;
  if (!in_range(beta1, 0.0, 1.0) || !in_range(beta2, 0.0, 1.0) || !in_range(eps, 0.0, INFINITY) || !isfinite(weight_decay) ||
      !isfinite(grad_scale))
    return MNV_ERR_INVALID;
  if (!schedule && (!isfinite(rate) || step < 1)) return MNV_ERR_INVALID;
  if (count == 0) return MNV_OK;
  if (!params || !grads || !m || !v || !params_out || !m_out || !v_out || !sizes) return MNV_ERR_INVALID;
  size_t total = 0;
  for (int i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    if (!params[i] || !grads[i] || !m[i] || !v[i] || !params_out[i] || !m_out[i] || !v_out[i]) return MNV_ERR_INVALID;
    if (sizes[i] > ((size_t)1 << 40) || (rates && !isfinite(rates[i])) || (decays && !isfinite(decays[i]))) return MNV_ERR_INVALID;
    total += sizes[i];
  }
  Step s;
  s.beta1 = beta1; s.beta2 = beta2; s.eps = eps; s.decay = weight_decay; s.scale = grad_scale;
  s.rate = rate; s.t = (unsigned)step; s.schedule = schedule;
  s.correct1 = schedule ? 1.0 : 1.0 / (1.0 - power(beta1, s.t));
  s.correct2 = schedule ? 1.0 : 1.0 / (1.0 - power(beta2, s.t));
  hipStream_t stm = mnv_stream(stream);
  const bool nt = total * 28 >= 2 * MNV_PAST_CACHE_BYTES;
  return for_tables(
      count, sizes,
      [&](Table& z, int at, int i) {
        z.p[at] = params[i]; z.g[at] = grads[i]; z.m[at] = m[i]; z.v[at] = v[i];
        z.p_out[at] = params_out[i]; z.m_out[at] = m_out[i]; z.v_out[at] = v_out[i];
        z.rate[at] = rates ? rates[i] : 1.f;
        z.decay[at] = decays ? decays[i] : 1.f;
      },
      [&](const Table& z, unsigned groups) {
        if (bits == 8) hipLaunchKernelGGL(adamw8_kernel, dim3(groups), dim3(256), 0, stm, z, s);
        else if (nt) hipLaunchKernelGGL(adamw_kernel<true>, dim3(groups), dim3(256), 0, stm, z, s);
        else hipLaunchKernelGGL(adamw_kernel<false>, dim3(groups), dim3(256), 0, stm, z, s);
        return MNV_LAUNCH_STATUS();
      });
}

int mnv_adamw_values(int count, const float* const* m, const float* const* v, float* const* m_values, float* const* v_values,
                     const size_t* sizes, mnv_stream_t stream) {
  if (count < 0) return MNV_ERR_INVALID;
  if (count == 0) return MNV_OK;
  if (!m || !v || !m_values || !v_values || !sizes) return MNV_ERR_INVALID;
  for (int i = 0; i < count; ++i)
    if (sizes[i] && (!m[i] || !v[i] || !m_values[i] || !v_values[i] || sizes[i] > ((size_t)1 << 40))) return MNV_ERR_INVALID;
  return for_tables(
      count, sizes,
      [&](Table& z, int at, int i) {
        z.m[at] = m[i]; z.v[at] = v[i];
        z.m_out[at] = m_values[i]; z.v_out[at] = v_values[i];
      },
      [&](const Table& z, unsigned groups) {
        hipLaunchKernelGGL(values_kernel, dim3(groups), dim3(256), 0, mnv_stream(stream), z);
        return MNV_LAUNCH_STATUS();
      });
}

}  // extern "C"
