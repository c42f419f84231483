// Rotary positions: pairs of a head's values turned by an angle that grows with the token's position.
//   (y1, y2) = magnitude * (x1 cos a - x2 sin a, x1 sin a + x2 cos a),  a = position * f_i,  f_i = base^(-2 i / rotary_dim)
// The gradient is the turn by -a.  For contexts longer than the angles were made for, f_i is divided by `factor` where
// it makes few turns within the old context, and kept where it makes many.
// Angles are counted in whole turns in 64 bits (a position of 10^6 would cost 32 bits all but one digit of the
// fastest angle), and their cosines and sines, times the magnitude, are rounded to 32 bits once.
// Bound by HBM, 8 bytes a value: 2 x 16384 tokens of 16 heads of 128 93 us, 5.8 TB/s; few tokens by the launch (3 us).
#include <math.h>

#include "mnv_common.h"

namespace {

struct RotaryAngles {
  double log2_step;        // f_i / (2 pi) = exp2(i * log2_step) / (2 pi) turns a position
  double inverse_factor;   // 1: not scaled
  double context, low, inverse_range;  // weight of the unscaled frequency: (context * turns - low) * inverse_range, cut to 0 .. 1
  double magnitude;
};
struct RotaryShape {
  const float* x;
  const float* positions;
  float* y;
  size_t x_pitch, y_pitch;
  long long start;
  int head_dim, heads, length, tokens, half;
  int head_chunk;  // heads of a workgroup
  int per_wg;      // its tokens
  MnvFastDiv vecs_div, heads_div, half_div, length_div;
  int vecs;        // vectors of a head: pairs', and behind them those that are copied
  float sign;      // -1: the gradient
};

// Turns that a position adds to pair i.
__device__ __forceinline__ double frequency(const RotaryAngles& a, int i) {
  double f = exp2(i * a.log2_step) * 0.15915494309189535;  // 1 / (2 pi)
  if (a.inverse_factor != 1.0) {
    double w = (a.context * f - a.low) * a.inverse_range;
    w = w < 0.0 ? 0.0 : w > 1.0 ? 1.0 : w;
    f *= w + (1.0 - w) * a.inverse_factor;
  }
  return f;
}

// Cosine and sine of so many turns: brought to an eighth of a turn by the nearest quarter, where the series' next terms, t^17 / 17! and
// t^16 / 16!, are below 2^-49.
__device__ __forceinline__ void cosine_sine(double turns, double& c, double& s) {
  const double quarters = rint(4.0 * turns), t = (turns - 0.25 * quarters) * 6.283185307179586, u = t * t;
  double x = -1.0 / 1307674368000.0, y = -1.0 / 87178291200.0;
  x = fma(u, x, 1.0 / 6227020800.0);
  y = fma(u, y, 1.0 / 479001600.0);
  x = fma(u, x, -1.0 / 39916800.0);
  y = fma(u, y, -1.0 / 3628800.0);
  x = fma(u, x, 1.0 / 362880.0);
  y = fma(u, y, 1.0 / 40320.0);
  x = fma(u, x, -1.0 / 5040.0);
  y = fma(u, y, -1.0 / 720.0);
  x = fma(u, x, 1.0 / 120.0);
  y = fma(u, y, 1.0 / 24.0);
  x = fma(u, x, -1.0 / 6.0);
  y = fma(u, y, -0.5);
  x = fma(u * t, x, t);
  y = fma(u, y, 1.0);
  const int q = (int)(quarters - 4.0 * floor(0.25 * quarters));  // 0 .. 3
  const double cq = q & 1 ? -x : y, sq = q & 1 ? y : x;
  c = q & 2 ? -cq : cq;
  s = q & 2 ? -sq : sq;
}

template <int W>
struct Vec {
  typedef float T __attribute__((ext_vector_type(W), aligned(4)));
};

// A workgroup turns `per_wg` tokens' `head_chunk` heads: first the angles' cosines and sines of its tokens into LDS, each
// once, then the values, neighbouring threads at neighbouring vectors.
// Half layout: vectors of V values i and half + i.  PAIRED: a vector of 2 V neighbours holds V pairs.  What is not turned
// is copied in vectors of C.
template <int V, bool PAIRED, int C>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryShape z, RotaryAngles angles) {
  extern __shared__ __align__(16) float lds[];  // cosines [per_wg][half], sines
  const long long first = ((long long)blockIdx.z * gridDim.x + blockIdx.x) * z.per_wg;
  if (first >= z.tokens) return;
  const int token0 = (int)first, head0 = blockIdx.y * z.head_chunk;
  const int count = z.tokens - token0 < z.per_wg ? z.tokens - token0 : z.per_wg;
  const int heads = z.heads - head0 < z.head_chunk ? z.heads - head0 : z.head_chunk;
  float* const cosines = lds;
  float* const sines = lds + z.per_wg * z.half;
  int pair = -1;
  double f = 0.0;
  for (int e = threadIdx.x; e < count * z.half; e += 256) {
    const int t = mnv_fastdiv(e, z.half_div), i = e - t * z.half, token = token0 + t;
    if (i != pair) {  // (a thread has the same one for all of its tokens where `half` divides 256)
      f = frequency(angles, i);
      pair = i;
    }
    const double position =
        z.positions ? (double)z.positions[token] : (double)(z.start + (token - mnv_fastdiv(token, z.length_div) * z.length));
    double s, c;
    cosine_sine(position * f, c, s);
    cosines[e] = (float)(c * angles.magnitude);
    sines[e] = (float)(s * angles.magnitude) * z.sign;
  }
  __syncthreads();
  constexpr int W = PAIRED ? 2 * V : V;  // values of a load
  typedef typename Vec<W>::T Load;
  const int pairs = z.half / V;  // vectors of pairs
  const int items = count * heads * z.vecs;
  for (int e = threadIdx.x; e < items; e += 256) {
    const int th = mnv_fastdiv(e, z.vecs_div), j = e - th * z.vecs;
    const int t = z.per_wg == 1 ? 0 : mnv_fastdiv(th, z.heads_div), h = th - t * z.heads;
    const size_t head = (size_t)(head0 + h) * z.head_dim;
    const float* x = z.x + (token0 + t) * z.x_pitch + head;
    float* y = z.y + (token0 + t) * z.y_pitch + head;
    if (j < pairs) {
      const float* c = cosines + t * z.half + j * V;
      const float* s = sines + t * z.half + j * V;
      if constexpr (PAIRED) {
        Load v = *reinterpret_cast<const Load*>(x + j * W);
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float x1 = v[2 * q], x2 = v[2 * q + 1];
          v[2 * q] = x1 * c[q] - x2 * s[q];
          v[2 * q + 1] = x1 * s[q] + x2 * c[q];
        }
        *reinterpret_cast<Load*>(y + j * W) = v;
      } else {
        Load v1 = *reinterpret_cast<const Load*>(x + j * V), v2 = *reinterpret_cast<const Load*>(x + z.half + j * V);
#pragma unroll
        for (int q = 0; q < V; ++q) {
          const float x1 = v1[q], x2 = v2[q];
          v1[q] = x1 * c[q] - x2 * s[q];
          v2[q] = x1 * s[q] + x2 * c[q];
        }
        *reinterpret_cast<Load*>(y + j * V) = v1;
        *reinterpret_cast<Load*>(y + z.half + j * V) = v2;
      }
    } else {  // behind what is turned
      typedef typename Vec<C>::T Copy;
      const int at = 2 * z.half + (j - pairs) * C;
      *reinterpret_cast<Copy*>(y + at) = *reinterpret_cast<const Copy*>(x + at);
    }
  }
}

template <int V, bool PAIRED, int C>
int launch(RotaryShape z, const RotaryAngles& a, hipStream_t s) {
  const int copied = z.x == z.y ? 0 : (z.head_dim - 2 * z.half) / C;  // in place nothing is
  z.vecs = z.half / V + copied;
  z.vecs_div = mnv_fastdiv_make(z.vecs);
  z.heads_div = mnv_fastdiv_make(z.heads);
  z.half_div = mnv_fastdiv_make(z.half);
  z.length_div = mnv_fastdiv_make(z.length);
  const int cus = mnv_cu_count();
  // About 2048 values to a workgroup, fewer where that leaves CUs without one: then single tokens, and parts of their heads.  us of both
  // passes with 1024 / 2048 / 4096 / 8192: 2 x 16384 tokens of 16 heads of 128 185 / 185 / 189 / 195, 8 x 4096 of 20 of 24 heads of 64
  // 118 / 118 / 125 / 133, 8 x 16384 of one 33 / 31 / 33 / 36.
  long long per = 2048 / ((long long)z.heads * z.head_dim);
  const long long lds_most = 8192 / (2LL * z.half);  // 32 KB
  if (per > lds_most) per = lds_most;
  if (per > z.tokens / (2LL * cus)) per = z.tokens / (2LL * cus);
  if (per < 1) per = 1;
  z.per_wg = (int)per;
  z.head_chunk = z.heads;
  const long long groups = (z.tokens + per - 1) / per;
  if (per == 1) {
    const int most = z.head_dim >= 8192 ? 1 : 8192 / z.head_dim;
    if (z.head_chunk > most) z.head_chunk = most;
    const long long parts = groups >= cus ? 1 : cus / groups;
    const int least = (256 + z.vecs - 1) / z.vecs;  // a vector for every thread
    int chunk = (int)((z.heads + parts - 1) / parts);
    if (chunk < least) chunk = least;
    if (chunk < z.head_chunk) z.head_chunk = chunk;
  }
  // A grid has 65535 chunks at most, and less than 2^32 threads along x: groups past 2^23 are dealt out along z.
  const int most_chunks = 65535;
  if ((z.heads - 1) / z.head_chunk >= most_chunks) z.head_chunk = (z.heads - 1) / most_chunks + 1;
  const long long across = groups < 1 << 23 ? groups : 1 << 23;
  const dim3 grid((unsigned)across, (z.heads - 1) / z.head_chunk + 1, (unsigned)((groups + across - 1) / across));
  const size_t lds = (size_t)z.per_wg * z.half * 2 * sizeof(float);
  hipLaunchKernelGGL((rotary_kernel<V, PAIRED, C>), grid, dim3(256), lds, s, z, a);
  return MNV_LAUNCH_STATUS();
}

int rotary(const float* x, const float* positions, float* y, int head_dim, int heads, int length, int batch, int x_pitch, int y_pitch,
           int rotary_dim, int interleaved, int start, double base, double factor, int context, double low_turns, double high_turns,
           double magnitude, bool back, mnv_stream_t stream) {
  if (!x || !y || head_dim <= 0 || heads <= 0 || length <= 0 || batch <= 0) return MNV_ERR_INVALID;
  const long long tokens = (long long)length * batch, width = (long long)heads * head_dim;
  // (a workgroup counts its vectors in 32 bits)
  if (width > 1 << 30 || width > x_pitch || width > y_pitch || tokens > 0x7fffffffLL || (x == y && x_pitch != y_pitch)) return MNV_ERR_INVALID;
  if (rotary_dim < 2 || rotary_dim % 2 || rotary_dim > head_dim || rotary_dim > 4096) return MNV_ERR_INVALID;
  if (!(base > 0.0) || !(factor > 0.0) || !isfinite(base) || !isfinite(factor) || !isfinite(magnitude)) return MNV_ERR_INVALID;
  if (!(low_turns >= 0.0) || !isfinite(high_turns) || context < 0) return MNV_ERR_INVALID;
  if (!(high_turns == 0.0 && low_turns == 0.0) && !(high_turns > low_turns)) return MNV_ERR_INVALID;
  RotaryShape z{};
  z.x = x; z.positions = positions; z.y = y;
  z.x_pitch = x_pitch; z.y_pitch = y_pitch;
  z.start = start;
  z.head_dim = head_dim; z.heads = heads; z.length = length; z.tokens = (int)tokens;
  z.half = rotary_dim / 2;
  z.sign = back ? -1.f : 1.f;
  RotaryAngles a;
  a.log2_step = -2.0 * log2(base) / rotary_dim;
  a.inverse_factor = 1.0 / factor;
  a.context = context;
  a.low = low_turns;
  a.inverse_range = high_turns > low_turns ? 1.0 / (high_turns - low_turns) : 0.0;  // 0: all are divided
  a.magnitude = magnitude;
  hipStream_t s = mnv_stream(stream);
  const bool copy4 = (head_dim - rotary_dim) % 4 == 0;
  if (interleaved) {
    if (rotary_dim % 4 == 0) return copy4 ? launch<2, true, 4>(z, a, s) : launch<2, true, 1>(z, a, s);
    return copy4 ? launch<1, true, 4>(z, a, s) : launch<1, true, 1>(z, a, s);
  }
  if (z.half % 4 == 0) return copy4 ? launch<4, false, 4>(z, a, s) : launch<4, false, 1>(z, a, s);
  return copy4 ? launch<1, false, 4>(z, a, s) : launch<1, false, 1>(z, a, s);
}

}  // namespace

extern "C" {

int mnv_rotary_fwd(const float* x, const float* positions, float* y, int head_dim, int heads, int length, int batch, int x_pitch,
                   int y_pitch, int rotary_dim, int interleaved, int start, double base, double factor, int context, double low_turns,
                   double high_turns, double magnitude, mnv_stream_t stream) {
  return rotary(x, positions, y, head_dim, heads, length, batch, x_pitch, y_pitch, rotary_dim, interleaved, start, base, factor, context,
                low_turns, high_turns, magnitude, false, stream);
}

int mnv_rotary_bwd(const float* dy, const float* positions, float* dx, int head_dim, int heads, int length, int batch, int dy_pitch,
                   int dx_pitch, int rotary_dim, int interleaved, int start, double base, double factor, int context, double low_turns,
                   double high_turns, double magnitude, mnv_stream_t stream) {
  return rotary(dy, positions, dx, head_dim, heads, length, batch, dy_pitch, dx_pitch, rotary_dim, interleaved, start, base, factor,
                context, low_turns, high_turns, magnitude, true, stream);
}

}  // extern "C"
