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
// Bound by HBM, 28 bytes a value with 32-bit moments (92.6 million values in 432 us, 6.0 TB/s); 16.06 bytes with 8-bit ones, where
// 95 vector instructions a value take longer (330 to 348 us, 4.5 TB/s); their values 10 bytes (185 us, 5.0 TB/s).
#include <math.h>

#include "mnv_common.h"

namespace {

constexpr int BLOCK = 256, WORDS = BLOCK / 4 + 1;  // values of a block; its floats: codes and top
constexpr int LONG = 4096, SHORT = 1024;           // values of a workgroup
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

// The tensor of a workgroup: every lane looks at one of them.
__device__ __forceinline__ int tensor_of(const Table& z, int wg) {
  const int lane = threadIdx.x % MNV_WAVE;
  return __popcll(__ballot(lane < TENSORS && z.first[lane < TENSORS ? lane : 0] <= wg)) - 1;
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
// With root and reciprocal of the vector unit, each within 2^-23 of itself.  Its root of a denormal number is 0: of one below 2^-63,
// which is nothing beside eps (`normal`: 2^-38 or more); with a smaller eps it is taken of v * 2^64.
__device__ __forceinline__ float updated_fast(const Factors& f, bool normal, float p, float m, float v) {
  float x = v * f.correct2;
  if (normal) {
    x = __builtin_amdgcn_sqrtf(x);
  } else {
    const bool small = x < 0x1p-96f;
    x = ldexpf(__builtin_amdgcn_sqrtf(ldexpf(x, small ? 64 : 0)), small ? -32 : 0);
  }
  const float quotient = m * f.correct1 * __builtin_amdgcn_rcpf(x + f.eps);
  return p - f.rate * (quotient + f.decay * p);
}

// ---- 32-bit moments: four vectors of four values a thread

template <bool NT>
__device__ __forceinline__ void put4(float* p, mnv_f4 v) {
  if (NT) __builtin_nontemporal_store(v, reinterpret_cast<mnv_f4u*>(p));
  else *reinterpret_cast<mnv_f4u*>(p) = v;
}

template <int CHUNK, bool NT>
__global__ __launch_bounds__(256) void adamw_kernel(Table z, Step s) {
  constexpr int V = CHUNK / 1024;  // vectors of a thread
  const int tensor = tensor_of(z, (int)blockIdx.x);
  const size_t at = (size_t)((int)blockIdx.x - z.first[tensor]) * CHUNK, n = z.n[tensor];
  const float* __restrict__ p = z.p[tensor];
  const float* __restrict__ g = z.g[tensor];
  const float* __restrict__ m = z.m[tensor];
  const float* __restrict__ v = z.v[tensor];
  const float b1 = (float)s.beta1, b2 = (float)s.beta2, a1 = (float)(1.0 - s.beta1), a2 = (float)(1.0 - s.beta2), scale = (float)s.scale;
  auto moments = [&](float gi, float& mi, float& vi) {
    gi *= scale;
    mi = b1 * mi + a1 * gi;
    vi = b2 * vi + a2 * gi * gi;
  };
  unsigned t;
  if (at + CHUNK <= n) {
    mnv_f4 pv[V], gv[V], mv[V], vv[V];
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const size_t i = at + u * 1024 + threadIdx.x * 4;
      gv[u] = mnv_ldx4u<NT>(g + i);
      mv[u] = mnv_ldx4u<NT>(m + i);
      vv[u] = mnv_ldx4u<NT>(v + i);
      pv[u] = mnv_ldx4u<NT>(p + i);
    }
    const Factors f = factors(z, s, tensor, t);
#pragma unroll
    for (int u = 0; u < V; ++u) {
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
    const Factors f = factors(z, s, tensor, t);
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

// Code c's power, exact: 127^3 < 2^21, 255^4 < 2^32.
template <bool SECOND>
__device__ __forceinline__ double powers(double c) {
  const double square = c * c;
  return SECOND ? square * square : square * c;
}
template <bool SECOND>
struct Code {
  static constexpr float MOST = SECOND ? 255.f : 127.f;
  static constexpr double UNIT = SECOND ? 1.0 / 4228250625.0 : 1.0 / 2048383.0;  // 255^-4, 127^-3
};
// A block's top, as the choice of codes wants it.
template <bool SECOND>
struct Top {
  double unit;        // unit * powers(c) is code c's value
  float lift, scale;  // x * lift * scale counts in units; lift is 1 but for tops whose reciprocal is no normal number
  __device__ explicit Top(float top) {
    unit = (double)top * Code<SECOND>::UNIT;
    const float down = top > 1.f ? 0x1p-64f : 1.f;
    lift = top < 0x1p-90f ? 0x1p80f : 1.f;
    scale = top != 0.f ? (float)(1.0 / Code<SECOND>::UNIT) * __builtin_amdgcn_rcpf(top * lift * down) * down : 0.f;
  }
  // The code of a size x (times lift) between 0 and the top: that below it, c, or the next one if x is more than u = `walk` 2^-32 of
  // the way there (m: half).  In 32 bits, where y is off by less than 2^-20 of itself and of the border between c and c + 1, the definition's
  // 64 bits decide, for one value in some thousands.  (All in 64 bits, with IEEE roots and quotients: 185 instructions a value instead of 100.)
  // That c itself may be wrong next to a code's value costs nothing: just above it c, past the border to c + 1, gives the same code as
  // c + 1 before its own border, if that is 2^-12 of the way or more behind it and from the code after: of v other u go the long way, too.
  __device__ int choose(float x, unsigned walk) const {
    const float y = x * scale;
    const float c = fminf(floorf(__builtin_amdgcn_exp2f(__builtin_amdgcn_logf(y) * (SECOND ? 0.25f : 0.33333333f))), Code<SECOND>::MOST - 1.f);
    const float square = c * c, in = y - (SECOND ? square * square : square * c);
    float past;  // the border
    bool near;
    if (SECOND) {
      // (c + 1)^4 - c^4, times 2^-32
      const float gap = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(0x1p-30f, c, 6 * 0x1p-32f), c, 0x1p-30f), c, 0x1p-32f);
      past = __builtin_fmaf(-(float)walk, gap, in);
      near = walk + (1u << 20) < (1u << 21);
    } else {
      past = __builtin_fmaf(-1.5f, square + c, in) - 0.5f;
      near = false;
    }
    near |= !(fabsf(past) >= y * 0x1p-20f);  // (not less: y may be a NaN)
    int code = (int)c + (past > 0.f);
    if (near) code = exact(x, c, SECOND ? (double)walk * 0x1p-32 : 0.5);
    return SECOND ? max(code, (int)min(__builtin_bit_cast(unsigned, x), 1u)) : code;
  }
  // c: at most one off the code below x
  __device__ int exact(float x, float c, double u) const {
    if (!(x > 0.f)) return 0;
    const double size = (double)x / lift, most = Code<SECOND>::MOST;
    double at = c;
    if (unit * powers<SECOND>(at) > size) at -= 1.0;
    else if (at < most && unit * powers<SECOND>(at + 1.0) <= size) at += 1.0;
    const double low = unit * powers<SECOND>(at), high = unit * powers<SECOND>(at + 1.0);
    return (int)at + ((at < most) & (size - low > u * (high - low)));
  }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned max_dpp(unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false));
}
// The largest size over a wavefront; NaN where one is an infinity or NaN.
__device__ __forceinline__ float top_of(const float (&x)[4]) {
  // sizes of floats are in the order of their bits, infinities and NaN last
  unsigned most = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const unsigned b = __builtin_bit_cast(unsigned, x[q]) & 0x7fffffffu;
    most = b > most ? b : most;
  }
  most = max_dpp<0x111, 0xf>(most);  // row_shr:1, 2, 4, 8: lane 15 of each row of 16 has the row's
  most = max_dpp<0x112, 0xf>(most);
  most = max_dpp<0x114, 0xf>(most);
  most = max_dpp<0x118, 0xf>(most);
  most = max_dpp<0x142, 0xa>(most);  // row_bcast:15 into rows 1 and 3, row_bcast:31 into rows 2 and 3
  most = max_dpp<0x143, 0xc>(most);
  most = (unsigned)__builtin_amdgcn_readlane((int)most, 63);
  return __builtin_bit_cast(float, most >= 0x7f800000u ? 0x7fc00000u : most);
}

template <bool SECOND>
__device__ __forceinline__ void decode(unsigned word, float top, float (&x)[4]) {
  const double unit = (double)top * Code<SECOND>::UNIT;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = SECOND ? (int)((word >> (8 * q)) & 255) : (int)(word << (24 - 8 * q)) >> 24;
    x[q] = (float)(unit * powers<SECOND>((double)c));
  }
}

// A wavefront's values of a block: four a lane, of which `left` exist.
__device__ __forceinline__ mnv_f4 get_rows(const float* p, int left) {
  if (left >= 4) return *reinterpret_cast<const mnv_f4u*>(p);
  return mnv_f4{left > 0 ? p[0] : 0.f, left > 1 ? p[1] : 0.f, left > 2 ? p[2] : 0.f, 0.f};
}
__device__ __forceinline__ void put_rows(float* p, int left, mnv_f4 x) {
  if (left >= 4) {
    *reinterpret_cast<mnv_f4u*>(p) = x;
  } else {
    if (left > 0) p[0] = x[0];
    if (left > 1) p[1] = x[1];
    if (left > 2) p[2] = x[2];
  }
}

// One block's step.  FULL: all its values exist.
struct Moments8 {
  mnv_f4 g, p;
  unsigned mw, vw;
  float mt, vt;
};
template <bool FULL>
__device__ __forceinline__ void load8(const Table& z, int tensor, size_t block, int lane, int left, Moments8& x) {
  const float* m = z.m[tensor] + block * WORDS;
  const float* v = z.v[tensor] + block * WORDS;
  const size_t i = block * BLOCK + lane * 4;
  x.mw = __builtin_bit_cast(unsigned, m[lane]);
  x.vw = __builtin_bit_cast(unsigned, v[lane]);
  x.mt = m[BLOCK / 4];
  x.vt = v[BLOCK / 4];
  x.g = get_rows(z.g[tensor] + i, FULL ? 4 : left);
  x.p = get_rows(z.p[tensor] + i, FULL ? 4 : left);
}
template <bool FULL>
__device__ __forceinline__ void step8(const Table& z, const Step& s, const Factors& f, unsigned t, int tensor, size_t block, int lane, int left,
                                      Moments8& x) {
  const size_t i = block * BLOCK + lane * 4;
  const double a1 = 1.0 - s.beta1, a2 = 1.0 - s.beta2;
  float mi[4], vi[4];
  decode<false>(x.mw, x.mt, mi);
  decode<true>(x.vw, x.vt, vi);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const double gi = (double)x.g[q] * s.scale;
    mi[q] = (float)(s.beta1 * (double)mi[q] + a1 * gi);
    vi[q] = (float)(s.beta2 * (double)vi[q] + a2 * (gi * gi));
    if (!FULL && q >= left) mi[q] = vi[q] = 0.f;
  }
  if (f.eps >= 0x1p-38f) {
#pragma unroll
    for (int q = 0; q < 4; ++q) x.p[q] = updated_fast(f, true, x.p[q], mi[q], vi[q]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) x.p[q] = updated_fast(f, false, x.p[q], mi[q], vi[q]);
  }
  put_rows(z.p_out[tensor] + i, FULL ? 4 : left, x.p);
  const float mtop = top_of(mi), vtop = top_of(vi);
  const Top<false> mc(mtop);
  const Top<true> vc(vtop);
  unsigned mo = 0, vo = 0;
  if (mc.lift != 1.f) {
#pragma unroll
    for (int q = 0; q < 4; ++q) mi[q] *= mc.lift;
  }
  if (vc.lift != 1.f) {
#pragma unroll
    for (int q = 0; q < 4; ++q) vi[q] *= vc.lift;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int c = mc.choose(fabsf(mi[q]), 0);
    const unsigned walk = (unsigned)(i + q) * 0x85EBCA6Bu + t * 0x9E3779B9u;
    mo |= (unsigned)((mi[q] < 0.f ? -c : c) & 255) << (8 * q);
    vo |= (unsigned)vc.choose(vi[q], walk) << (8 * q);
  }
  float* m = z.m_out[tensor] + block * WORDS;
  float* v = z.v_out[tensor] + block * WORDS;
  m[lane] = __builtin_bit_cast(float, mo);
  v[lane] = __builtin_bit_cast(float, vo);
  if (lane == 0) {
    m[BLOCK / 4] = mtop;
    v[BLOCK / 4] = vtop;
  }
}

// The blocks of a workgroup's wavefronts, one behind the other; the next one is fetched under the present one's step.
template <int CHUNK>
__global__ __launch_bounds__(256) void adamw8_kernel(Table z, Step s) {
  constexpr int MINE = CHUNK / BLOCK / 4;
  const int tensor = tensor_of(z, (int)blockIdx.x), lane = threadIdx.x % MNV_WAVE;
  const size_t chunk = (size_t)((int)blockIdx.x - z.first[tensor]), n = z.n[tensor];
  size_t block = chunk * (CHUNK / BLOCK) + (size_t)__builtin_amdgcn_readfirstlane(threadIdx.x / MNV_WAVE) * MINE;
  unsigned t;
  if ((block + MINE) * BLOCK <= n) {
    Moments8 x[2];
    load8<true>(z, tensor, block, lane, 4, x[0]);
    const Factors f = factors(z, s, tensor, t);
#pragma unroll
    for (int b = 0; b < MINE; ++b) {
      if (b + 1 < MINE) load8<true>(z, tensor, block + b + 1, lane, 4, x[(b + 1) % 2]);
      step8<true>(z, s, f, t, tensor, block + b, lane, 4, x[b % 2]);
    }
  } else {
    const Factors f = factors(z, s, tensor, t);
    for (int b = 0; b < MINE && block * BLOCK < n; ++b, ++block) {
      const size_t i = block * BLOCK + lane * 4;
      const int left = i >= n ? 0 : n - i < 4 ? (int)(n - i) : 4;
      Moments8 x;
      load8<false>(z, tensor, block, lane, left, x);
      step8<false>(z, s, f, t, tensor, block, lane, left, x);
    }
  }
}

// The values that both moments' codes stand for, in m_out and v_out.
template <int CHUNK>
__global__ __launch_bounds__(256) void values_kernel(Table z) {
  constexpr int MINE = CHUNK / BLOCK / 4;
  const int tensor = tensor_of(z, (int)blockIdx.x), lane = threadIdx.x % MNV_WAVE;
  const size_t chunk = (size_t)((int)blockIdx.x - z.first[tensor]), n = z.n[tensor];
  const size_t first = chunk * (CHUNK / BLOCK) + (size_t)__builtin_amdgcn_readfirstlane(threadIdx.x / MNV_WAVE) * MINE;
  unsigned mw[MINE], vw[MINE];
  float mt[MINE], vt[MINE];
#pragma unroll
  for (int b = 0; b < MINE; ++b)
    if ((first + b) * BLOCK < n) {
      const float* m = z.m[tensor] + (first + b) * WORDS;
      const float* v = z.v[tensor] + (first + b) * WORDS;
      mw[b] = __builtin_bit_cast(unsigned, m[lane]);
      vw[b] = __builtin_bit_cast(unsigned, v[lane]);
      mt[b] = m[BLOCK / 4];
      vt[b] = v[BLOCK / 4];
    }
#pragma unroll
  for (int b = 0; b < MINE; ++b) {
    const size_t i = (first + b) * BLOCK + lane * 4;
    if (i >= n) return;
    const int left = n - i < 4 ? (int)(n - i) : 4;
    float mi[4], vi[4];
    decode<false>(mw[b], mt[b], mi);
    decode<true>(vw[b], vt[b], vi);
    put_rows(z.m_out[tensor] + i, left, mnv_f4{mi[0], mi[1], mi[2], mi[3]});
    put_rows(z.v_out[tensor] + i, left, mnv_f4{vi[0], vi[1], vi[2], vi[3]});
  }
}

// Goes through the tensors that have values, as many to a launch as its table holds and as a grid has workgroups.
// `chunk`: values of a workgroup.
template <class Fill, class Launch>
int for_tables(int count, const size_t* sizes, int chunk, Fill fill, Launch launch) {
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
    const size_t chunks = (sizes[i] + chunk - 1) / chunk;
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

// Values of a workgroup: short ones where long ones would leave a CU fewer than two (60 arrays of 0.3 million values 12.7 -> 8.2 us).
int chunk_of(size_t total) { return total >= (size_t)LONG * 2 * mnv_cu_count() ? LONG : SHORT; }

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
  const int chunk = chunk_of(total);
  return for_tables(
      count, sizes, chunk,
      [&](Table& z, int at, int i) {
        z.p[at] = params[i]; z.g[at] = grads[i]; z.m[at] = m[i]; z.v[at] = v[i];
        z.p_out[at] = params_out[i]; z.m_out[at] = m_out[i]; z.v_out[at] = v_out[i];
        z.rate[at] = rates ? rates[i] : 1.f;
        z.decay[at] = decays ? decays[i] : 1.f;
      },
      [&](const Table& z, unsigned groups) {
        const dim3 grid(groups), threads(256);
        if (bits == 8 && chunk == LONG) hipLaunchKernelGGL(adamw8_kernel<LONG>, grid, threads, 0, stm, z, s);
        else if (bits == 8) hipLaunchKernelGGL(adamw8_kernel<SHORT>, grid, threads, 0, stm, z, s);
        else if (nt) hipLaunchKernelGGL((adamw_kernel<LONG, true>), grid, threads, 0, stm, z, s);
        else if (chunk == LONG) hipLaunchKernelGGL((adamw_kernel<LONG, false>), grid, threads, 0, stm, z, s);
        else hipLaunchKernelGGL((adamw_kernel<SHORT, false>), grid, threads, 0, stm, z, s);
        return MNV_LAUNCH_STATUS();
      });
}

int mnv_adamw_values(int count, const float* const* m, const float* const* v, float* const* m_values, float* const* v_values,
                     const size_t* sizes, mnv_stream_t stream) {
  if (count < 0) return MNV_ERR_INVALID;
  if (count == 0) return MNV_OK;
  if (!m || !v || !m_values || !v_values || !sizes) return MNV_ERR_INVALID;
  size_t total = 0;
  for (int i = 0; i < count; ++i) {
    if (sizes[i] && (!m[i] || !v[i] || !m_values[i] || !v_values[i] || sizes[i] > ((size_t)1 << 40))) return MNV_ERR_INVALID;
    total += sizes[i];
  }
  const int chunk = chunk_of(total);
  return for_tables(
      count, sizes, chunk,
      [&](Table& z, int at, int i) {
        z.m[at] = m[i]; z.v[at] = v[i];
        z.m_out[at] = m_values[i]; z.v_out[at] = v_values[i];
      },
      [&](const Table& z, unsigned groups) {
        if (chunk == LONG) hipLaunchKernelGGL(values_kernel<LONG>, dim3(groups), dim3(256), 0, mnv_stream(stream), z);
        else hipLaunchKernelGGL(values_kernel<SHORT>, dim3(groups), dim3(256), 0, mnv_stream(stream), z);
        return MNV_LAUNCH_STATUS();
      });
}

}  // extern "C"
