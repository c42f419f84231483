// The gated feed-forward block y = w_out (act(w_gate x) * (w_up x)), with both projections in one matrix
// w_in {2 hidden, features}, and its gradients:
//   pre = w_in x,  h = act(pre_gate) * pre_up,  y = w_out h
//   dh = w_out' dy,  dpre = (dh * pre_up * act'(pre_gate), dh * act(pre_gate))
//   dx = w_in' dpre,  dw_in = dpre x',  dw_out = dy h'
// Bound by the matrix cores (6 features hidden flops a token forward, 12 backward), and for few tokens by reading the
// weights.  Products are those of the SGEMM (sgemm_core.h), large ones in pairs of fp16 numbers (pair_gemm.h), those of large
// weights and few tokens of few_gemm.h; what lies between them is done where a product is stored: the gate forward, where both projections
// of a row meet in one tile, and dpre backward, which is all that is kept of dh.
// Both passes: 8192 tokens of 2048 -> 5632 5.0 ms (340 TFLOP/s), 4096 of 1024 -> 2816 0.90 ms (236); forward: 777 of 1001 -> 2731
// 110 us (115), 4 of 1024 -> 4096 23 us (50 MB of weights, 2.2 TB/s over four launches).
#include <algorithm>
#include <atomic>

#include "few_gemm.h"
#include "pair_gemm.h"

namespace {

enum { ACT_SIGMOID, ACT_RELU, ACT_TANH, ACT_SILU, ACT_GELU, ACT_COUNT };

// 1 / d of d from 1 to 2: the vector unit's reciprocal and a step of Newton's leave at most one rounding more than a division.
__device__ __forceinline__ float reciprocal_1_to_2(float d) {
  const float guess = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, guess, 1.f), guess, guess);
}
// The activation of N values, and its slopes there.  The kind is looked at once for them all, so that their instructions
// interleave: a wavefront has its SIMD to itself where large products store (8192 tokens of 2048 -> 5632, silu, w_in's 1166 -> 1009 us, w_out's backward
// 712 -> 611, with the reciprocal below).
template <int N>
__device__ __forceinline__ void activate(int kind, const float (&x)[N], float (&value)[N], float (&slope)[N]) {
  if (kind == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      value[i] = x[i] <= 0.f ? 0.f : x[i];  // (a NaN is not below 0: it goes on)
      slope[i] = x[i] <= 0.f ? 0.f : x[i] > 0.f ? 1.f : x[i];
    }
  } else if (kind == ACT_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // 1 - tanh^2 would keep no digit from 9 on; with z = exp(-2 |x|) the slope is 4 z / (1 + z)^2 there and everywhere
      const float z = expf(-2.f * fabsf(x[i])), near = reciprocal_1_to_2(1.f + z);
      value[i] = tanhf(x[i]);
      slope[i] = 4.f * z * near * near;
    }
  } else if (kind == ACT_GELU) {
    // x times the normal distribution's share below x: erfc keeps the digits of a small share, 1 + erf does not
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float below = 0.5f * erfcf(x[i] * -0.70710678f);
      value[i] = x[i] * below;
      slope[i] = below + x[i] * (0.39894228f * expf(-0.5f * x[i] * x[i]));
    }
  } else {
    // 1 / (1 + exp(-x)) and what it lacks to 1, from the exponential that cannot overflow: neither loses digits near 0.
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float z = expf(-fabsf(x[i])), near = reciprocal_1_to_2(1.f + z), far = z * near;
      const float e = x[i] < 0.f ? far : near, rest = x[i] < 0.f ? near : far;
      value[i] = kind == ACT_SILU ? x[i] * e : e;
      slope[i] = kind == ACT_SILU ? e + value[i] * rest : e * rest;
    }
  }
}
template <int N>
__device__ __forceinline__ void gated(int kind, const float (&gate)[N], const float (&up)[N], float (&h)[N]) {
  float slope[N];
  activate(kind, gate, h, slope);
#pragma unroll
  for (int i = 0; i < N; ++i) h[i] *= up[i];
}
__device__ __forceinline__ float gated(int kind, float gate, float up) {
  float h[1];
  gated<1>(kind, {gate}, {up}, h);
  return h[0];
}

typedef float Two __attribute__((ext_vector_type(2), aligned(4)));
// Four rows from p on, of which `left` exist.
__device__ __forceinline__ void store_rows(float* p, int left, const float (&x)[4]) {
  if (left >= 4) {
    *reinterpret_cast<mnv_f4u*>(p) = mnv_f4u{x[0], x[1], x[2], x[3]};
  } else {
#pragma unroll
    for (int q = 0; q < 3; ++q)
      if (q < left) p[q] = x[q];
  }
}

// w_in x with the gate where it is stored.  The product's rows are w_in's in runs of four, gate and up in turn, so that rows
// 8 i .. 8 i + 3 are the gate's 4 i .. 4 i + 3 and the four behind them the up projection's.  A 16-byte fetch is still
// one run of w_in's column, and a tile in parts gives neighbouring lanes the two runs of one column (C_ROWS_OF_FOUR):
// they change places by a lane permutation, as do the lanes that store a small tile's sums, four rows apart.  Rows past `hidden` of the last run hold what follows in memory, or 0
// past the end, and are not stored.
template <bool K4>
struct GatedIn {
  static constexpr bool A_KFAST = false, B_KFAST = true;
  static constexpr int A_NOFF = 1, B_NOFF = 1;
  const float* __restrict__ A;
  const float* __restrict__ B;
  float* __restrict__ pre;  // may be null
  float* __restrict__ h;
  int M, N, K, total_slabs, spp, bk;
  int lda, ldb, hidden, act;
  static constexpr bool N_GROUPED = true;
  int n_group;
  struct Res {
    mnv_rsrc a, b;
  };
  struct AState {};
  struct BState {};
  __device__ void make_res(Res& r) const {
    r.a = mnv_make_rsrc(A, (unsigned)K * (unsigned)hidden * 8u);
    r.b = mnv_make_rsrc(B, (unsigned)N * (unsigned)K * 4u);
  }
  __device__ void a_init(const Res&, AState&, int) const {}
  __device__ void b_init(const Res&, BState&, int) const {}
  __device__ void a_period(const AState&, unsigned (&off)[A_NOFF], int m, int kl, int period) const {
    const int k = period * spp * bk + kl, row = m / 8 * 4;
    off[0] = ((row < hidden) & (k < K)) ? ((unsigned)k * (unsigned)hidden * 2u + (unsigned)(row + (m & 4 ? hidden : 0))) * 4u : MNV_OOB;
  }
  __device__ void a_load(const Res& r, const AState&, const unsigned (&off)[A_NOFF], int, int s, int, float (&v)[4]) const {
    mnv_fetch_vec<A_NOFF>(r.a, off, (unsigned)s * (unsigned)bk * (unsigned)hidden * 8u, v);
  }
  __device__ void b_period(const BState&, unsigned (&off)[B_NOFF], int n, int kl, int period) const {
    const int k = period * spp * bk + kl;
    off[0] = ((n < N) & (k < K)) ? ((unsigned)n * (unsigned)K + (unsigned)k) * 4u : MNV_OOB;
  }
  __device__ void b_load(const Res& r, const BState&, const unsigned (&off)[B_NOFF], int, int s, int, float (&v)[4]) const {
    mnv_fetch_vec<B_NOFF>(r.b, off, (unsigned)s * (unsigned)bk * 4u, v);
  }
  // as SgemmNN: a vector of the last, partial slab is cleared past K
  static constexpr bool B_STASH_FIX = !K4;
  __device__ void b_stash_fix(int period, int, int kl, float (&v)[4]) const {
    if (period == (K >= bk ? 1 : 0)) {
      const int rest = K % bk;
#pragma unroll
      for (int q = 1; q < 4; ++q) v[q] = kl + q < rest ? v[q] : 0.f;
    }
  }
  size_t extra_lds_bytes() const { return 0; }
  void set_bk(int b) {
    bk = b;
    spp = K >= b ? K / b : 1;
    total_slabs = (K + b - 1) / b;
  }
  __device__ void block_init(Res&, float*, int, int) const {}
  // the small tiles' view: one row of A, and one sum of a lane, whose up or gate is four lanes away
  __device__ int a_row(int m) const { return m / 8 * 4 + m % 4 + (m & 4 ? hidden : 0); }
  __device__ void c_store(int m, int n, float x) const {
    const float other = __shfl_xor(x, 4, MNV_WAVE);
    const int row = m / 8 * 4 + m % 4;
    if (row >= hidden) return;
    if (pre) pre[(size_t)n * hidden * 2 + a_row(m)] = x;
    if (!(m & 4)) h[(size_t)n * hidden + row] = gated(act, x, other);
  }
  static constexpr bool C_STORE4 = true, C_ROWS_OF_FOUR = true;
  struct Fetched {};
  __device__ Fetched c_fetch4(int, int) const { return {}; }
  __device__ void c_store4_with(int m, int n, const float (&x)[4], const Fetched&) const { c_store4(m, n, x); }
  __device__ void c_store4(int m, int n, const float (&x)[4]) const {
    const int row = m / 8 * 4, left = hidden - row;
    const bool up = m & 4;
    if (pre) store_rows(pre + (size_t)n * hidden * 2 + row + (up ? hidden : 0), left, x);
    // The lane of the gate takes rows 0 and 1, that of the up projection 2 and 3; each gives the other what it wants (quad_perm 1, 0, 3, 2).
    float gate[2], high[2], r[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float give = up ? x[q] : x[q + 2];
      const float got = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, give), 0xb1, 0xf, 0xf, true));
      gate[q] = up ? got : x[q];
      high[q] = up ? x[q + 2] : got;
    }
    gated(act, gate, high, r);
    float* const p = h + (size_t)n * hidden + row + (up ? 2 : 0);
    const int rest = left - (up ? 2 : 0);
    if (rest >= 2) *reinterpret_cast<Two*>(p) = Two{r[0], r[1]};
    else if (rest == 1) p[0] = r[0];
  }
};

// w_out' dy, stored as dpre.  dpre may be pre itself: every element is read and written by one thread.
template <bool K4>
struct GatedOutBack : SgemmNN<K4, true, false> {
  typedef SgemmNN<K4, true, false> Base;
  const float* pre;
  float* dpre;
  int hidden, act;
  __device__ void c_store(int m, int n, float dh) const {
    const size_t at = (size_t)n * hidden * 2 + m;
    const float gate = pre[at], up = pre[at + hidden];
    float value[1], slope[1];
    activate<1>(act, {gate}, value, slope);
    dpre[at] = dh * up * slope[0];
    dpre[at + hidden] = dh * value[0];
  }
  struct Fetched {
    mnv_f4u gate, up;
  };
  __device__ Fetched c_fetch4(int m, int n) const {
    const size_t at = (size_t)n * hidden * 2 + m;
    if (m + 3 < this->M) return {*reinterpret_cast<const mnv_f4u*>(pre + at), *reinterpret_cast<const mnv_f4u*>(pre + at + hidden)};
    return {};
  }
  __device__ void c_store4_with(int m, int n, const float (&dh)[4], const Fetched& f) const {
    if (m + 3 < this->M) {
      const size_t at = (size_t)n * hidden * 2 + m;
      mnv_f4u dg, du;
      float value[4], slope[4];
      activate<4>(act, {f.gate[0], f.gate[1], f.gate[2], f.gate[3]}, value, slope);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        dg[q] = dh[q] * f.up[q] * slope[q];
        du[q] = dh[q] * value[q];
      }
      *reinterpret_cast<mnv_f4u*>(dpre + at) = dg;
      *reinterpret_cast<mnv_f4u*>(dpre + at + hidden) = du;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (m + q < this->M) c_store(m + q, n, dh[q]);
    }
  }
  __device__ void c_store4(int m, int n, const float (&dh)[4]) const { c_store4_with(m, n, dh, c_fetch4(m, n)); }
};

// h = act(gate) * up from pre as a product of its own left it: four rows a thread.
__global__ __launch_bounds__(256) void gate_kernel(const float* __restrict__ pre, float* __restrict__ h, int hidden, MnvFastDiv quads,
                                                   int quads_count, size_t total, int act) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int n = total <= 0x7fffffff ? mnv_fastdiv((int)i, quads) : (int)(i / quads_count);
    const int row = (int)(i - (size_t)n * quads_count) * 4, left = hidden - row;
    const float* p = pre + (size_t)n * hidden * 2 + row;
    float r[4];
    if (left >= 4) {
      const mnv_f4u gate = *reinterpret_cast<const mnv_f4u*>(p), up = *reinterpret_cast<const mnv_f4u*>(p + hidden);
      gated<4>(act, {gate[0], gate[1], gate[2], gate[3]}, {up[0], up[1], up[2], up[3]}, r);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) r[q] = q < left ? gated(act, p[q], p[hidden + q]) : 0.f;
    }
    store_rows(h + (size_t)n * hidden + row, left, r);
  }
}

// The projections' k ranges added, and gated: `ranges` times {2 hidden, tokens}.  ZL threads share a value, each adding every
// ZL-th range.
template <int ZL>
__global__ __launch_bounds__(256) void gate_ranges_kernel(const float* __restrict__ part, float* __restrict__ pre, float* __restrict__ h, int hidden,
                                                          int tokens, int ranges, int act) {
  constexpr int QL = 256 / ZL;
  __shared__ float red[2][256];
  const int tq = threadIdx.x % QL, tz = threadIdx.x / QL;
  const size_t all = (size_t)hidden * tokens, q = (size_t)blockIdx.x * QL + tq;
  const int n = (int)(q / hidden), m = (int)(q - (size_t)n * hidden);
  float gate = 0.f, up = 0.f;
  if (q < all) {
    const float* p = part + (size_t)tz * all * 2 + (size_t)n * hidden * 2 + m;
#pragma unroll 4
    for (int r = tz; r < ranges; r += ZL, p += ZL * all * 2) {
      gate += p[0];
      up += p[hidden];
    }
  }
  red[0][threadIdx.x] = gate;
  red[1][threadIdx.x] = up;
  __syncthreads();
  if (tz || q >= all) return;
#pragma unroll
  for (int i = 1; i < ZL; ++i) {
    gate += red[0][i * QL + tq];
    up += red[1][i * QL + tq];
  }
  if (pre) {
    pre[(size_t)n * hidden * 2 + m] = gate;
    pre[(size_t)n * hidden * 2 + hidden + m] = up;
  }
  h[q] = gated(act, gate, up);
}
int launch_gate_ranges(const float* part, float* pre, float* h, int hidden, int tokens, int ranges, int act, hipStream_t s) {
  const size_t all = (size_t)hidden * tokens;
  if (ranges >= 16 && all < 65536)
    hipLaunchKernelGGL(gate_ranges_kernel<8>, dim3((unsigned)mnv_ceil_div(all, 32)), dim3(256), 0, s, part, pre, h, hidden, tokens, ranges, act);
  else if (ranges >= 4)
    hipLaunchKernelGGL(gate_ranges_kernel<2>, dim3((unsigned)mnv_ceil_div(all, 128)), dim3(256), 0, s, part, pre, h, hidden, tokens, ranges, act);
  else
    hipLaunchKernelGGL(gate_ranges_kernel<1>, dim3((unsigned)mnv_ceil_div(all, 256)), dim3(256), 0, s, part, pre, h, hidden, tokens, ranges, act);
  return MNV_LAUNCH_STATUS();
}

template <bool K4>
GatedIn<K4> make_gated_in(const float* w_in, const float* x, float* pre, float* h, int features, int hidden, int tokens, int act) {
  GatedIn<K4> p;
  p.A = w_in; p.B = x; p.pre = pre; p.h = h;
  p.M = (hidden + 3) / 4 * 8; p.N = tokens; p.K = features;
  p.hidden = hidden; p.act = act;
  p.lda = 2 * hidden; p.ldb = features;
  p.n_group = 1;
  p.set_bk(16);
  return p;
}
template <bool K4>
int launch_gated_in(const SgemmPlan& plan, const float* w_in, const float* x, float* pre, float* h, int features, int hidden, int tokens,
                    int act, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const GatedIn<K4> p = make_gated_in<K4>(w_in, x, pre, h, features, hidden, tokens, act);
  if constexpr (K4) {
    if (plan.tile) return launch_small_tiles(plan, p, s);
  }
  return launch_split(plan, p, workspace, workspace ? workspace_bytes : 0, s);
}

// Microseconds of a product on 128 x 128 tiles with a cut tail (as mnv_tail_plan prices it), or without one.
double tiles_cost(int m, int n, int k, size_t ws_floats, int cus) {
  const long long tiles = (long long)((m + 127) / 128) * ((n + 127) / 128);
  const int slabs = (k + 15) / 16;
  const MnvTailPlan t = mnv_tail_plan(tiles, slabs, 128 * 128, ws_floats, SplitPair::TAIL);
  if (t.z <= 1) return split_cost(m, n, k, 1, cus);
  const int rem = (int)(tiles - t.begin), per_cu = t.begin / cus, parts = (rem * t.z + cus - 1) / cus, len = (slabs + t.z - 1) / t.z;
  return 1.3 * per_cu * ((slabs + 1) / 2) + 3.0 * ((per_cu + 1) / 2) + SplitPair::TAIL.slab * parts * len + SplitPair::TAIL.start * (parts - 1) +
         2.0 + 0.46e-6 * sizeof(float) * rem * t.z * 128 * 128;
}
// How the projections run.  SMALL, TILES: their product gates where it stores, on small tiles or on those in bf16 parts; RANGES: by k ranges,
// which are gated where they are added; APART: as a plain product, and a kernel of its own gates.
// The product's own plan decides, but for tiles in parts where it has others: those save the gating kernel, 3 us and 12 bytes a value
// at 5 TB/s, and their cut tail, which that plan has not weighed.  us, as planned and on these tiles, both with w_out's product: 777 tokens
// of 1001 -> 2731 158 / 130, 512 of 1024 -> 2816 99 / 91, 300 of 2048 -> 5632 219 / 191; kept: 400 of 1500 -> 1500 70 / 95, 128 of 1024 -> 4096 46 / 71.
enum Way { SMALL, TILES, RANGES, APART };
Way way(SgemmPlan* plan, int features, int hidden, int tokens, size_t ws_bytes) {
  *plan = plan_sgemm(2 * hidden, tokens, features, ws_bytes / sizeof(float));
  if (plan->tile) return SMALL;
  if (plan->split && plan->splits == 1) return TILES;
  if (!plan->skinny && tokens > 64) {
    const int cus = mnv_cu_count();
    if (tiles_cost((hidden + 3) / 4 * 8, tokens, features, ws_bytes / sizeof(float), cus) < plan->us + 3.0 + 12.0 * hidden * tokens / 5e6) {
      *plan = SgemmPlan{false, 1};
      plan->split = true;
      return TILES;
    }
  }
  return plan->splits > 1 ? RANGES : APART;
}

int launch_gate(const float* pre, float* h, int hidden, int tokens, int act, hipStream_t s) {
  const int quads = (hidden + 3) / 4;
  const size_t total = (size_t)quads * tokens;
  size_t blocks = mnv_ceil_div(total, 256);
  if (blocks > MNV_MAX_STREAM_BLOCKS) blocks = MNV_MAX_STREAM_BLOCKS;
  hipLaunchKernelGGL(gate_kernel, dim3((unsigned)blocks), dim3(256), 0, s, pre, h, hidden, mnv_fastdiv_make(quads), quads, total, act);
  return MNV_LAUNCH_STATUS();
}

template <bool K4>
GatedOutBack<K4> make_out_back(const float* w_out, const float* dy, const float* pre, float* dpre, int features, int hidden, int tokens, int act) {
  GatedOutBack<K4> p;
  static_cast<SgemmNN<K4, true, false>&>(p) =
      make_sgemm<K4, true, false>(w_out, dy, nullptr, hidden, tokens, features, SgemmEpilogue{nullptr, nullptr, 0});
  p.pre = pre; p.dpre = dpre;
  p.hidden = hidden; p.act = act;
  return p;
}
template <bool K4>
int launch_out_back(const SgemmPlan& plan, const float* w_out, const float* dy, const float* pre, float* dpre, int features, int hidden,
                    int tokens, int act, void* workspace, size_t workspace_bytes, hipStream_t s) {
  const GatedOutBack<K4> p = make_out_back<K4>(w_out, dy, pre, dpre, features, hidden, tokens, act);
  if constexpr (K4) {
    if (plan.skinny) return launch_skinny_columns(plan, p, workspace, s);
    if (plan.tile) return launch_small_tiles(plan, p, s);
  }
  return launch_plan(plan, p, workspace, workspace_bytes, s);
}

// Products read matrices through 32-bit byte offsets.
bool sizes_ok(int features, int hidden, int tokens, int act) {
  const long long most = (1LL << 29) - 1;
  return features > 0 && hidden > 0 && tokens > 0 && act >= 0 && act < ACT_COUNT && 2LL * hidden <= most / features &&
         2LL * hidden <= most / tokens && features <= most / tokens;
}

// The six products.  Operands' rows are the result's rows (the left one's) and columns; a matrix lies with its rows contiguous.
struct Product {
  PairOperand a, b;
  double store_bytes;  // that its store moves for a value
};
Product product_in(const float* w_in, const float* x, int features, int hidden, int tokens) {
  return {{w_in, 2 * (size_t)hidden, (hidden + 3) / 4 * 8, features, false, hidden}, {x, (size_t)features, tokens, features, true, 0}, 6.0};
}
Product product_out(const float* w_out, const float* h, int features, int hidden, int tokens) {
  return {{w_out, (size_t)features, features, hidden, false, 0}, {h, (size_t)hidden, tokens, hidden, true, 0}, 4.0};
}
Product product_dh(const float* w_out, const float* dy, int features, int hidden, int tokens) {
  return {{w_out, (size_t)features, hidden, features, true, 0}, {dy, (size_t)features, tokens, features, true, 0}, 16.0};
}
Product product_dx(const float* w_in, const float* dpre, int features, int hidden, int tokens) {
  return {{w_in, 2 * (size_t)hidden, features, 2 * hidden, true, 0}, {dpre, 2 * (size_t)hidden, tokens, 2 * hidden, true, 0}, 4.0};
}
// dw = left right', left {rows, tokens}, right {columns, tokens}
Product product_dw(const float* left, const float* right, int rows, int columns, int tokens) {
  return {{left, (size_t)rows, rows, tokens, false, 0}, {right, (size_t)columns, columns, tokens, false, 0}, 4.0};
}
// Whether a product runs in pairs: where that is estimated at less than the SGEMM's time, and the workspace holds it.  The
// SGEMM's own estimate is 1.2 times too low where products of this size follow each other, and more where it is above 216 TFLOP/s: 180 of
// them last (both passes, without / with that: 4096 tokens of 1024 -> 2816 955 / 936, 500 of 4096 -> 8192 1511 / 1462).  It is one of a plain
// product: what the store moves beyond 4 bytes comes on top (without / with: 8192 of 768 -> 2048 1089 / 1041, 16384 of 512 -> 2048 1580 / 1512).  us, both passes, in pairs never / so: 4096 tokens
// of 1024 -> 2816 1212 / 958, 1024 of 2048 -> 5632 1203 / 921, 8192 of 2048 -> 5632 8360 / 5120, 300 of 4096 -> 8192 1202 / 1100 (all in pairs 1240).
std::atomic<int> g_pairs{1};  // mnv_gated_ffn_pairs_mode
bool in_pairs(const Product& p, int most_ranges, size_t ws_bytes, PairPlan* plan) {
  if (!g_pairs.load(std::memory_order_relaxed)) return false;
  // below 5 GFLOP the four launches of the packing alone take half of the time
  if (!pair_fits(p.a, p.b) || 2.0 * p.a.rows * p.b.rows * p.a.k < 5e9) return false;
  const int cus = mnv_cu_count();
  *plan = pair_plan(p.a, p.b, most_ranges, p.store_bytes, cus);
  const SgemmPlan other = plan_unlimited(p.a.rows, p.b.rows, p.a.k, cus);
  double us = other.us;
  if ((other.split && other.splits == 1) || p.a.gate) us = std::min(us, tiles_cost(p.a.rows, p.b.rows, p.a.k, (size_t)-1, cus));
  us = std::max(1.2 * us, 2e-6 * p.a.rows * p.b.rows * p.a.k / 180.0) + (p.store_bytes - 4.0) * 1e-6 / 5.0 * p.a.rows * p.b.rows;
  return plan->us < us && plan->bytes() <= ws_bytes;
}
size_t pair_bytes(const Product& p, int most_ranges) {
  PairPlan plan;
  return in_pairs(p, most_ranges, (size_t)-1, &plan) ? plan.bytes() : 0;
}
constexpr int RANGES_AT_MOST = 16;
// c = a b
int pair_plain(const PairPlan& plan, const Product& p, float* c, char* ws, hipStream_t s) {
  return pair_product(plan, p.a, p.b, PairStore{c, p.a.rows},
                      make_sgemm<true>(nullptr, nullptr, c, p.a.rows, p.b.rows, 1, SgemmEpilogue{nullptr, nullptr, 0}), ws, s);
}

// The products that read a weight matrix for few tokens.  The least values: below them the SGEMM's plans are as fast; of the one with
// dh, whose tiles store no ranges, 12 million (1024 -> 4096 for 16 tokens 7 / 9 us, 4096 -> 4096 31 / 18).
FewPlan few_in(int features, int hidden, int tokens, size_t ws_bytes) { return plan_few(2 * hidden, tokens, features, false, 5e6, ws_bytes); }
FewPlan few_out(int features, int hidden, int tokens, size_t ws_bytes) { return plan_few(features, tokens, hidden, false, 2.5e6, ws_bytes); }
FewPlan few_dh(int features, int hidden, int tokens, size_t ws_bytes) { return plan_few(hidden, tokens, features, true, 12e6, ws_bytes); }
FewPlan few_dx(int features, int hidden, int tokens, size_t ws_bytes) { return plan_few(features, tokens, 2 * hidden, true, 2.5e6, ws_bytes); }
template <class P>
int run_few(const FewPlan& plan, const P& p, char* ws, hipStream_t s) {
  float* const partial = reinterpret_cast<float*>(ws);
  const int rc = launch_few(plan, p, partial, s);
  return rc || plan.ranges == 1 ? rc : mnv_gemm_reduce_launch(p, partial, plan.ranges, s);
}

size_t larger(size_t a, size_t b) { return a > b ? a : b; }
// Bytes of pre where the caller keeps none and the plan does not do without it, in whole 16 bytes.
size_t pre_bytes(int hidden, int tokens) { return ((size_t)hidden * 2 * tokens * sizeof(float) + 15) / 16 * 16; }

}  // namespace

extern "C" {

size_t mnv_gated_ffn_fwd_workspace_bytes(int features, int hidden, int tokens) {
  if (!sizes_ok(features, hidden, tokens, 0)) return 0;
  SgemmPlan plan;
  const FewPlan few = few_in(features, hidden, tokens, (size_t)-1), few_y = few_out(features, hidden, tokens, (size_t)-1);
  const Way w = few.cols ? RANGES : way(&plan, features, hidden, tokens, (size_t)-1);
  const int rows = (hidden + 3) / 4 * 8;
  size_t in = few.cols ? few.bytes(2 * hidden, tokens) : mnv_sgemm_nn_workspace_bytes(2 * hidden, tokens, features);
  if (w == TILES) in = sgemm_tail_bytes(plan, rows, tokens, features);
  const size_t out = few_y.cols ? few_y.bytes(features, tokens) : mnv_sgemm_nn_workspace_bytes(features, tokens, hidden);
  const size_t others = larger(in, out) + (w == APART ? pre_bytes(hidden, tokens) : 0);
  return larger(others, larger(pair_bytes(product_in(nullptr, nullptr, features, hidden, tokens), 1),
                               pair_bytes(product_out(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST)));
}

int mnv_gated_ffn_fwd(const float* x, const float* w_in, const float* w_out, float* pre, float* h, float* y, int features, int hidden,
                      int tokens, int activation, void* workspace, size_t workspace_bytes, mnv_stream_t stream) {
  if (!x || !w_in || !w_out || !h || !y || !sizes_ok(features, hidden, tokens, activation)) return MNV_ERR_INVALID;
  hipStream_t s = mnv_stream(stream);
  char* ws = static_cast<char*>(workspace);
  size_t bytes = workspace_bytes;
  if (!ws || !mnv_aligned16(ws)) {
    ws = nullptr;
    bytes = 0;
  }
  int rc = MNV_OK, ranges = 1;
  PairPlan pair;
  const Product in = product_in(w_in, x, features, hidden, tokens), out = product_out(w_out, h, features, hidden, tokens);
  const auto product_y = [&] {
    if (in_pairs(out, RANGES_AT_MOST, bytes, &pair)) return pair_plain(pair, out, y, ws, s);
    const FewPlan few = few_out(features, hidden, tokens, bytes);
    if (few.cols) return run_few(few, make_sgemm<true>(w_out, h, y, features, tokens, hidden, SgemmEpilogue{nullptr, nullptr, 0}), ws, s);
    return mnv_sgemm_nn(w_out, h, y, features, tokens, hidden, ws, bytes, stream);
  };
  if (in_pairs(in, 1, bytes, &pair)) {
    const GatedIn<true> e = make_gated_in<true>(w_in, x, pre, h, features, hidden, tokens, activation);
    rc = pair_product(pair, in.a, in.b, e, make_sgemm<true>(nullptr, nullptr, h, 1, 1, 1, SgemmEpilogue{nullptr, nullptr, 0}), ws, s);
    return rc ? rc : product_y();
  }
  const FewPlan few = few_in(features, hidden, tokens, bytes);
  if (few.cols) {
    if (few.ranges == 1) {
      rc = launch_few(few, make_gated_in<true>(w_in, x, pre, h, features, hidden, tokens, activation), nullptr, s);
    } else {
      float* const partial = reinterpret_cast<float*>(ws);
      rc = launch_few(few, make_sgemm<true>(w_in, x, nullptr, 2 * hidden, tokens, features, SgemmEpilogue{nullptr, nullptr, 0}), partial, s);
      if (!rc) rc = launch_gate_ranges(partial, pre, h, hidden, tokens, few.ranges, activation, s);
    }
    return rc ? rc : product_y();
  }
  SgemmPlan plan;
  Way w = way(&plan, features, hidden, tokens, bytes);
  if (w == RANGES) {
    rc = mnv_sgemm_nn_ranges(w_in, x, 2 * hidden, tokens, features, ws, bytes, &ranges, s);
    if (rc) return rc;
    if (ranges > 1) rc = launch_gate_ranges(reinterpret_cast<const float*>(ws), pre, h, hidden, tokens, ranges, activation, s);
    else w = APART;
  }
  float* kept = pre;
  if (w == APART && !kept) {
    if (bytes >= pre_bytes(hidden, tokens)) {
      kept = reinterpret_cast<float*>(ws);
      ws += pre_bytes(hidden, tokens);
      bytes -= pre_bytes(hidden, tokens);
    } else {  // nowhere to leave pre: on tiles, whatever the size
      plan = SgemmPlan{false, 1};
      plan.split = true;
      w = TILES;
    }
  }
  if (w == APART) {
    rc = mnv_sgemm_nn(w_in, x, kept, 2 * hidden, tokens, features, ws, bytes, stream);
    if (!rc) rc = launch_gate(kept, h, hidden, tokens, activation, s);
  } else if (w != RANGES) {
    rc = w == SMALL || features % 4 == 0 ? launch_gated_in<true>(plan, w_in, x, pre, h, features, hidden, tokens, activation, ws, bytes, s)
                                         : launch_gated_in<false>(plan, w_in, x, pre, h, features, hidden, tokens, activation, ws, bytes, s);
  }
  return rc ? rc : product_y();
}

int mnv_gated_ffn_pairs_mode(int mode) {
  if (mode < 0 || mode > 1) return g_pairs.load(std::memory_order_relaxed);
  return g_pairs.exchange(mode, std::memory_order_relaxed);
}

int mnv_gated_ffn_plan(int features, int hidden, int tokens, size_t fwd_workspace_bytes, size_t bwd_workspace_bytes, int* pairs) {
  if (!pairs || !sizes_ok(features, hidden, tokens, 0)) return MNV_ERR_INVALID;
  const size_t f = fwd_workspace_bytes, b = bwd_workspace_bytes;
  PairPlan plan;
  *pairs = in_pairs(product_in(nullptr, nullptr, features, hidden, tokens), 1, f, &plan) << 0 |
           in_pairs(product_out(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST, f, &plan) << 1 |
           in_pairs(product_dh(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST, b, &plan) << 2 |
           in_pairs(product_dx(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST, b, &plan) << 3 |
           in_pairs(product_dw(nullptr, nullptr, 2 * hidden, features, tokens), RANGES_AT_MOST, b, &plan) << 4 |
           in_pairs(product_dw(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST, b, &plan) << 5;
  return MNV_OK;
}

size_t mnv_gated_ffn_bwd_workspace_bytes(int features, int hidden, int tokens) {
  if (!sizes_ok(features, hidden, tokens, 0)) return 0;
  const FewPlan few = few_dh(features, hidden, tokens, (size_t)-1), few_x = few_dx(features, hidden, tokens, (size_t)-1);
  const size_t others =
      larger(larger(few.cols ? few.bytes(hidden, tokens) : mnv_sgemm_nn_workspace_bytes(hidden, tokens, features),
                    few_x.cols ? few_x.bytes(features, tokens) : mnv_sgemm_nn_workspace_bytes(features, tokens, 2 * hidden)),
             larger(mnv_sgemm_nn_workspace_bytes(2 * hidden, features, tokens), mnv_sgemm_nn_workspace_bytes(features, hidden, tokens)));
  const size_t pairs = larger(larger(pair_bytes(product_dh(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST),
                                     pair_bytes(product_dx(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST)),
                              larger(pair_bytes(product_dw(nullptr, nullptr, 2 * hidden, features, tokens), RANGES_AT_MOST),
                                     pair_bytes(product_dw(nullptr, nullptr, features, hidden, tokens), RANGES_AT_MOST)));
  return larger(others, pairs);
}

int mnv_gated_ffn_bwd(const float* x, const float* w_in, const float* w_out, const float* pre, const float* h, const float* dy, float* dpre,
                      float* dx, float* dw_in, float* dw_out, int features, int hidden, int tokens, int activation, void* workspace,
                      size_t workspace_bytes, mnv_stream_t stream) {
  if (!x || !w_in || !w_out || !pre || !h || !dy || !dpre || !dw_in || !dw_out || !sizes_ok(features, hidden, tokens, activation))
    return MNV_ERR_INVALID;
  hipStream_t s = mnv_stream(stream);
  char* const ws = workspace && mnv_aligned16(workspace) ? static_cast<char*>(workspace) : nullptr;
  const size_t bytes = ws ? workspace_bytes : 0;
  int rc;
  PairPlan pair;
  const Product dh = product_dh(w_out, dy, features, hidden, tokens);
  if (in_pairs(dh, RANGES_AT_MOST, bytes, &pair)) {
    const GatedOutBack<true> e = make_out_back<true>(w_out, dy, pre, dpre, features, hidden, tokens, activation);
    rc = pair_product(pair, dh.a, dh.b, e, e, ws, s);
  } else if (const FewPlan few = few_dh(features, hidden, tokens, bytes); few.cols) {
    rc = run_few(few, make_out_back<true>(w_out, dy, pre, dpre, features, hidden, tokens, activation), ws, s);
  } else {
    const SgemmPlan plan = plan_sgemm(hidden, tokens, features, bytes / sizeof(float));
    rc = plan.skinny || plan.tile || features % 4 == 0
             ? launch_out_back<true>(plan, w_out, dy, pre, dpre, features, hidden, tokens, activation, ws, bytes, s)
             : launch_out_back<false>(plan, w_out, dy, pre, dpre, features, hidden, tokens, activation, ws, bytes, s);
  }
  if (!rc && dx) {
    const Product p = product_dx(w_in, dpre, features, hidden, tokens);
    if (in_pairs(p, RANGES_AT_MOST, bytes, &pair)) {
      rc = pair_plain(pair, p, dx, ws, s);
    } else if (const FewPlan few = few_dx(features, hidden, tokens, bytes); few.cols) {
      rc = run_few(few, make_sgemm<true, true>(w_in, dpre, dx, features, tokens, 2 * hidden, SgemmEpilogue{nullptr, nullptr, 0}), ws, s);
    } else {
      rc = mnv_sgemm_tn(w_in, dpre, nullptr, dx, features, tokens, 2 * hidden, ws, bytes, stream);
    }
  }
  if (!rc) {
    const Product p = product_dw(dpre, x, 2 * hidden, features, tokens);
    rc = in_pairs(p, RANGES_AT_MOST, bytes, &pair) ? pair_plain(pair, p, dw_in, ws, s)
                                                   : mnv_sgemm_nt(dpre, x, dw_in, 2 * hidden, features, tokens, ws, bytes, stream);
  }
  if (!rc) {
    const Product p = product_dw(dy, h, features, hidden, tokens);
    rc = in_pairs(p, RANGES_AT_MOST, bytes, &pair) ? pair_plain(pair, p, dw_out, ws, s)
                                                   : mnv_sgemm_nt(dy, h, dw_out, features, hidden, tokens, ws, bytes, stream);
  }
  return rc;
}

}  // extern "C"
