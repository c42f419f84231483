// Attention of queries to the states of another sequence (or their own), forward.
//   t_ij = scale * q_i.k_j + bias[j - i + q_len - 1] (j < lengths[b]),  m_i = max t_ij,  l_i = sum exp(t_ij - m_i)
//   out_i = sum_j exp(t_ij - m_i) / l_i * v_j
// One pass over the keys with the running maximum and sum of each query: a workgroup of four or eight wavefronts
// has 32 queries per wavefront, and tiles of 32 keys stream through LDS.  t^T = K Q^T, so a lane
// has one query and a quarter of the tile's keys; exp(t - m) goes on as the operand of out^T += V^T P^T from
// the registers it stands in (attention_core.h).  Heads that share keys are rows of the same workgroup: row r is query
// r / group, head r % group of the key head, so their keys are read and cut once.
// A row that sees no key has m = -inf, l = 0, out = 0.  The pair (m, l) is kept and not m + ln l: where the bias is the
// type's lowest value for a whole row, ln l would be lost in the sum.
#include <type_traits>

#include "attention_core.h"

namespace {

struct FwdArgs {
  const float *q, *k, *v, *bias, *lengths;
  float *out, *stats;
  AttentionSizes z;
  int rows;        // q_len * group
  int row_tiles;   // per entry and key head
  MnvFastDiv by_group;
};

template <int DP, int NW, bool BIAS, bool VEC>
__global__ __launch_bounds__(64 * NW, 2) void mnv_attention_fwd_kernel(FwdArgs a) {
  constexpr int NB = DP / 32, KS = DP / 16;
  using Stage = MnvStage<DP, 64 * NW, VEC>;
  __shared__ __align__(16) char lds[2 * Stage::BYTES];
  const AttentionSizes& z = a.z;
  const MnvAttentionPlace place = mnv_attention_place(a.row_tiles, 0, z, a.lengths);
  const int tile = place.tile, b = place.b, kh = place.kh, n = place.n;
  const int lane = threadIdx.x % MNV_WAVE, half = lane / 32;

  const int r = tile * (32 * NW) + (int)threadIdx.x / MNV_WAVE * 32 + lane % 32;
  const int rc = r < a.rows ? r : a.rows - 1;
  const int i = mnv_fastdiv(rc, a.by_group), h = kh * z.group() + (rc - i * z.group());
  const size_t row = ((size_t)b * z.q_len + i) * z.heads + h;

  mnv_f16 acc[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[c][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  if (n > 0) {
    MnvParts qp[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      float x[8];
      mnv_load8<DP>(a.q + row * z.dim, s, z.dim, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= z.scale;
      qp[s] = mnv_cut8(x);
    }
    const unsigned pitch = (unsigned)z.kv_heads * z.dim;
    const float* kb = a.k + ((size_t)b * z.k_len * z.kv_heads + kh) * z.dim;
    const float* vb = a.v + ((size_t)b * z.k_len * z.kv_heads + kh) * z.dim;
    const float* bias = BIAS ? a.bias + h * z.offsets() + (z.q_len - 1 - i) : nullptr;

    {
      Stage first;
      first.fetch(kb, vb, pitch, n, z.dim);
      first.template store<false>(lds, 1.f);
    }
    __syncthreads();

    // Two phases to a tile, each the other half's when there are eight wavefronts: while four multiply queries and
    // keys, the four that share their matrix cores have soft-max to do.
    const bool late = NW == 8 && mnv_uniform(threadIdx.x / MNV_WAVE) >= 4;
    mnv_f16 t;
    Stage stage;
    auto fetch = [&](int piece, int j1) __attribute__((always_inline)) {
      stage.fetch_piece(piece, kb + (size_t)j1 * pitch, vb + (size_t)j1 * pitch, pitch, n - j1, z.dim);
    };
    // scores of the tile in `now`; FETCH: the tile from j1 on is fetched, else that in `stage` is cut to `then`
    auto scores = [&](auto fetches, const char* now, char* then, int j1) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) t[e] = 0.f;
      MnvParts cur = Stage::by_rows(now, 0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        MnvParts ahead = cur;
        if (s + 1 < KS) ahead = Stage::by_rows(now, s + 1);
        mnv_mul(t, cur, qp[s]);
        if (decltype(fetches)::value) fetch(s, j1);
        else stage.template store_piece<false>(s, then, 1.f);
        MNV_STEP_ORDER(6);
        cur = ahead;
      }
    };
    auto results = [&](auto fetches, const char* now, char* then, int j0, int j1) __attribute__((always_inline)) {
      const bool whole = j0 + 32 <= n;
      MnvParts cur = Stage::by_cols(now + Stage::MATRIX, 0, 0);
      if (BIAS) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + 8 * u + 4 * half;
          if (whole) {
            const mnv_f4 add = mnv_ldx4u<false>(bias + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) t[4 * u + e] += add[e];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) t[4 * u + e] += bias[j + e < n ? j + e : n - 1];
          }
        }
      }
      if (!whole) {
        MNV_KEEP_BRANCH();
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (j0 + mnv_acc_row(e, half) >= n) t[e] = -INFINITY;
      }
      float top = t[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, t[e]);
      const float next = fmaxf(m, mnv_max_of_halves(top));
      const float base = mnv_finite_max(next);
      if (__any(next > m)) {
        const float shrink = mnv_weight(m, base);
        l *= shrink;
#pragma unroll
        for (int c = 0; c < NB; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[c][e] *= shrink;
        m = next;
      }
      // the second half of the weights is made, and the next tile cut, under the products of the first
      MnvCutting pc[2];
      auto cut_p = [&](int pair) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          t[2 * pair + e] = mnv_weight(t[2 * pair + e], base);
          l += t[2 * pair + e];
        }
        pc[pair / 4].pair(pair % 4, t[2 * pair], t[2 * pair + 1]);
      };
#pragma unroll
      for (int pair = 0; pair < 4; ++pair) cut_p(pair);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        MnvParts ahead = cur;
        if (s + 1 < KS) ahead = Stage::by_cols(now + Stage::MATRIX, (s + 1) % NB * 32, (s + 1) / NB);
        mnv_mul(acc[s % NB], cur, pc[s / NB].parts());
        if (s < NB) {
#pragma unroll
          for (int pair = 4 + s * 4 / NB; pair < 4 + (s + 1) * 4 / NB; ++pair) cut_p(pair);
        }
        if (decltype(fetches)::value) fetch(s, j1);
        else stage.template store_piece<false>(s, then, 1.f);
        MNV_STEP_ORDER(6);
        cur = ahead;
      }
    };
    const std::true_type fetches;
    const std::false_type cuts;
    const int last = (n - 1) / 32 * 32;  // behind it that tile again: no branch parts a phase
    char *now = lds, *then = lds + Stage::BYTES;
    if (!late) {
      for (int j0 = 0; j0 < n; j0 += 32) {
        scores(fetches, now, then, j0 < last ? j0 + 32 : last);
        if (NW == 8) __syncthreads();
        results(cuts, now, then, j0, 0);
        __syncthreads();
        char* t_ = now;
        now = then;
        then = t_;
      }
      if (NW == 8) __syncthreads();
    } else {
      // one phase behind: cuts a tile while it makes scores, which is when the others do
#pragma unroll
      for (int piece = 0; piece < Stage::PIECES; ++piece) fetch(piece, last < 32 ? last : 32);
      __syncthreads();
      for (int j0 = 0; j0 < n; j0 += 32) {
        scores(cuts, now, then, 0);
        __syncthreads();
        results(fetches, now, then, j0, j0 + 64 < last ? j0 + 64 : last);
        __syncthreads();
        char* t_ = now;
        now = then;
        then = t_;
      }
    }
    l += __shfl_xor(l, 32, MNV_WAVE);
  }
  if (r < a.rows) {
    mnv_store_column<DP>(acc, mnv_inverse(l), true, a.out + row * z.dim, z.dim);
    if (half == 0) {
      a.stats[2 * row] = m;
      a.stats[2 * row + 1] = l;
    }
  }
}

template <int DP, int NW>
int launch(FwdArgs& a, hipStream_t s) {
  a.row_tiles = (int)mnv_ceil_div(a.rows, 32 * NW);
  const size_t grid = (size_t)a.row_tiles * a.z.batch * a.z.kv_heads;
  if (grid > 0x7fffffff) return MNV_ERR_INVALID;
  const dim3 g((unsigned)grid), b(64 * NW);
  const bool vec = a.z.dim % 4 == 0;
  if (a.bias && vec) hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, true, true>), g, b, 0, s, a);
  else if (a.bias) hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, true, false>), g, b, 0, s, a);
  else if (vec) hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, false, true>), g, b, 0, s, a);
  else hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, false, false>), g, b, 0, s, a);
  return MNV_LAUNCH_STATUS();
}

}  // namespace

extern "C" {

size_t mnv_attention_fwd_workspace_bytes(int, int, int, int, int, int) { return 0; }

int mnv_attention_fwd(const float* q, const float* k, const float* v, const float* bias, const float* lengths,
                      float* out, float* stats, int batch, int heads, int kv_heads, int q_len, int k_len, int head_dim,
                      float scale, void*, size_t, mnv_stream_t stream) {
  const AttentionSizes z = {batch, heads, kv_heads, q_len, k_len, head_dim, scale};
  if (!q || !k || !v || !out || !stats || !mnv_attention_sizes_ok(z)) return MNV_ERR_INVALID;
  FwdArgs a = {q, k, v, bias, lengths, out, stats, z, q_len * z.group(), 0, mnv_fastdiv_make(z.group())};
  const hipStream_t s = mnv_stream(stream);
  if (head_dim <= 32) return launch<32, 4>(a, s);
  if (head_dim <= 64) return launch<64, 4>(a, s);
  if (head_dim <= 96) return launch<96, 8>(a, s);
  return launch<128, 8>(a, s);
}

}  // extern "C"
