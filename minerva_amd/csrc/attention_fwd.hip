// Attention of queries to the states of another sequence (or their own), forward.
//   t_ij = scale * q_i.k_j + bias[j - i + q_len - 1] (j < lengths[b]),  m_i = max t_ij,  l_i = sum exp(t_ij - m_i)
//   out_i = sum_j exp(t_ij - m_i) / l_i * v_j
// One pass over the keys with the running maximum and sum of each query: a workgroup of four or eight wavefronts
// has 32 queries per wavefront, and tiles of 32 keys stream through LDS.  t^T = K Q^T, so a lane
// has one query and a quarter of the tile's keys; exp(t - m) goes on as the operand of out^T += V^T P^T from
// the registers it stands in (attention_core.h).  Heads that share keys are rows of the same workgroup: row r is query
// r / group, head r % group of the key head, so their keys are read and cut once.  Few rows over many keys are spread
// over parts of the keys, which a second kernel joins.
// Bound by the matrix cores where there are queries enough: 2 products of 6 instructions per value.  2 x 16 heads (4 key heads) of
// 2048 x 4096, 128 wide: 0.61 ms = 225 TFLOP/s of fp32 products in calls back to back, 0.64 to 0.68 ms in a training step, cores
// busy 63% (the rest: the first operands of each phase wait for LDS, the softmax between the phases; the kernel of eight
// wavefronts and 128 columns keeps 10 to 30 registers more than there are in scratch memory); a large fp32 product of the
// library reaches 153.  8 x 16 heads of 512 x 1024, 64 wide, lengths 128 to 1024: 81 us, the longest entry's workgroups.
// For one query the memory bounds it: 16 heads of 4 key heads, 8 entries of 250 to 2000 keys: 12 us and 4 to join, of 18 MB.
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
  int chunk;       // keys of a part, a multiple of 32
  int parts;       // 1: the result itself is written
  float *part_out, *part_stats;  // [part][row of q][DP], and [2]: sums without the division by l
};

template <int DP, int NW, bool BIAS, bool VEC>
__global__ __launch_bounds__(64 * NW, DP > 64 && NW == 4 ? 1 : 2) void mnv_attention_fwd_kernel(FwdArgs a) {
  constexpr int NB = DP / 32, KS = DP / 16;
  using Stage = MnvStage<DP, 64 * NW, VEC>;
  __shared__ __align__(16) char lds[2 * Stage::BYTES];
  const AttentionSizes& z = a.z;
  const MnvAttentionPlace place = mnv_attention_place(a.row_tiles * a.parts, 0, 0, 0, z, a.lengths);
  const int part = mnv_uniform(place.tile / a.row_tiles), tile = place.tile - part * a.row_tiles, b = place.b, kh = place.kh;
  // the part's keys
  const int begin = part * a.chunk, n = place.n < begin + a.chunk ? place.n : begin + a.chunk;
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

  if (n > begin) {
    MnvParts qp[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      float x[8];
      mnv_load8<DP, VEC>(a.q + row * z.dim, s, z.dim, x);
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
      first.fetch(kb + (size_t)begin * pitch, vb + (size_t)begin * pitch, pitch, n - begin, z.dim);
      first.store(lds);
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
    // a step's share of the next tile's fetching or cutting
    auto share = [&](auto fetches, int s, char* then, int j1) __attribute__((always_inline)) {
      constexpr int EACH = (Stage::PIECES + KS - 1) / KS;
#pragma unroll
      for (int piece = s * EACH; piece < (s + 1) * EACH && piece < Stage::PIECES; ++piece) {
        if (decltype(fetches)::value) fetch(piece, j1);
        else stage.store_piece(piece, then);
      }
    };
    // scores of the tile in `now`; `fetches`: the tile from j1 on is fetched, else that in `stage` is cut into `then`
    auto scores = [&](auto fetches, const char* now, char* then, int j1) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) t[e] = 0.f;
      auto operand = [&](int s, int c) __attribute__((always_inline)) { return Stage::by_rows(now, s, c); };
      MnvParts cur = {{operand(0, 0), operand(0, 1), operand(0, 2)}};
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        auto next = [&](int c) __attribute__((always_inline)) { return operand(s + 1, c); };
        if (s + 1 < KS) mnv_step<false>(t, cur, qp[s], next);
        else mnv_step<true>(t, cur, qp[s], next);
        share(fetches, s, then, j1);
        MNV_STEP_ORDER(6);
      }
    };
    auto results = [&](auto fetches, const char* now, char* then, int j0, int j1) __attribute__((always_inline)) {
      const bool whole = j0 + 32 <= n;
      auto operand = [&](int s, int c) __attribute__((always_inline)) {
        return Stage::by_cols(now + Stage::MATRIX, s % NB * 32, s / NB, c);
      };
      MnvParts cur = {{operand(0, 0), operand(0, 1), operand(0, 2)}};
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
        auto next = [&](int c) __attribute__((always_inline)) { return operand(s + 1, c); };
        if (s + 1 < KS) mnv_step<false>(acc[s % NB], cur, pc[s / NB].parts(), next);
        else mnv_step<true>(acc[s % NB], cur, pc[s / NB].parts(), next);
        if (s < NB) {
#pragma unroll
          for (int u = 0; u < (4 + NB - 1) / NB; ++u)
            if (4 + s * 4 / NB + u < 4 + (s + 1) * 4 / NB) cut_p(4 + s * 4 / NB + u);
        }
        share(fetches, s, then, j1);
        MNV_STEP_ORDER(6);
      }
    };
    const std::true_type fetches;
    const std::false_type cuts;
    const int last = begin + (n - begin - 1) / 32 * 32;  // behind it that tile again: no branch parts a phase
    char *now = lds, *then = lds + Stage::BYTES;
    const auto turn = [&] {
      char* t_ = now;
      now = then;
      then = t_;
    };
    if (NW == 8 && !late) {
      for (int j0 = begin; j0 < n; j0 += 32) {
        scores(fetches, now, then, j0 < last ? j0 + 32 : last);
        __syncthreads();
        results(cuts, now, then, j0, 0);
        __syncthreads();
        turn();
      }
      __syncthreads();
    } else {
      // the next tile is cut under the scores, and the one after it fetched under the results; of eight wavefronts the
      // second half is a phase behind, and so cuts when the first does
#pragma unroll
      for (int piece = 0; piece < Stage::PIECES; ++piece) fetch(piece, begin < last ? begin + 32 : last);
      if (NW == 8) __syncthreads();
      // a wavefront without rows has its share of the tiles to bring, and leaves its matrix core to others (12 heads of 129
      // queries, 6 entries of 0 to 1500 keys: 34.0 us, 35.5 where it multiplies as the others do)
      const bool idle = NW == 4 && mnv_uniform(tile * (32 * NW) + (int)threadIdx.x / MNV_WAVE * 32) >= a.rows;
      for (int j0 = begin; NW == 4 && idle && j0 < n; j0 += 32) {
#pragma unroll
        for (int piece = 0; piece < Stage::PIECES; ++piece) stage.store_piece(piece, then);
#pragma unroll
        for (int piece = 0; piece < Stage::PIECES; ++piece) fetch(piece, j0 + 64 < last ? j0 + 64 : last);
        __syncthreads();
        turn();
      }
      for (int j0 = begin; !idle && j0 < n; j0 += 32) {
        scores(cuts, now, then, 0);
        if (NW == 8) __syncthreads();
        results(fetches, now, then, j0, j0 + 64 < last ? j0 + 64 : last);
        __syncthreads();
        turn();
      }
    }
    l += __shfl_xor(l, 32, MNV_WAVE);
  }
  if (r >= a.rows) return;
  if (a.parts > 1) {
    const size_t at = part * z.q_rows() + row;
    if (n > begin) mnv_store_column<DP>(acc, 1.f, true, a.part_out + at * DP, DP);
    if (half == 0) {
      a.part_stats[2 * at] = m;
      a.part_stats[2 * at + 1] = l;
    }
    return;
  }
  // of a row that sees no key 0, and not 0 times what values hold that others see
  mnv_store_column<DP>(acc, mnv_inverse(l), l != 0.f, a.out + row * z.dim, z.dim);
  if (half == 0) {
    a.stats[2 * row] = m;
    a.stats[2 * row + 1] = l;
  }
}

// out and stats of up to 64 parts: m = max m_s, l = sum l_s exp(m_s - m), out = sum out_s exp(m_s - m) / l.  A part that
// saw no key has l_s = 0, and wrote no sums.  A wavefront to a row: a lane to a part's numbers, then 16 lanes
// to the sums of every fourth part.
__global__ __launch_bounds__(256) void mnv_attention_join_kernel(const float* __restrict__ part_out,
                                                                 const float* __restrict__ part_stats,
                                                                 float* __restrict__ out, float* __restrict__ stats,
                                                                 size_t rows, int parts, int dim, int pitch) {
  const size_t row = (size_t)blockIdx.x * 4 + threadIdx.x / MNV_WAVE;
  if (row >= rows) return;
  const int lane = threadIdx.x % MNV_WAVE;
  float ms = -INFINITY, ls = 0.f;
  if (lane < parts) {
    ms = part_stats[2 * (lane * rows + row)];
    ls = part_stats[2 * (lane * rows + row) + 1];
  }
  float m = ms;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, MNV_WAVE));
  const float w = ls == 0.f ? 0.f : mnv_weight(ms, mnv_finite_max(m));
  float l = ls * w;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, MNV_WAVE);
  const float f = mnv_inverse(l);
  const unsigned long long shown = __ballot(ls != 0.f);
  for (int d0 = 0; d0 < pitch; d0 += 64) {  // all lanes stay: they hand each other the parts' numbers
    const int d = d0 + lane % 16 * 4;
    mnv_f4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += 16) {
      mnv_f4 t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = s0 + 4 * u + lane / 16;
        t[u] = mnv_f4{0.f, 0.f, 0.f, 0.f};
        if (d < pitch && s < parts && (shown >> s & 1))
          t[u] = *reinterpret_cast<const mnv_f4*>(part_out + (s * rows + row) * pitch + d);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = s0 + 4 * u + lane / 16;
        const float ws = __shfl(w, s < parts ? s : 0, MNV_WAVE);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(t[u][e], ws, acc[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[e] += __shfl_xor(acc[e], 16, MNV_WAVE);
      acc[e] += __shfl_xor(acc[e], 32, MNV_WAVE);
      if (lane < 16 && d + e < dim) out[row * dim + d + e] = acc[e] * f;
    }
  }
  if (lane < 2) stats[2 * row + lane] = lane ? l : m;
}

// The same of up to MOST parts, 16 lanes to a row, each of which works all parts' numbers out by itself: nothing is handed
// from lane to lane (9288 rows of 64 in 7 parts: 4.4 us, 7.0 by the kernel above; in 10 parts 5.0 and 7.0; where 8 do, 16
// take half a microsecond longer).
template <int MOST>
__global__ __launch_bounds__(256) void mnv_attention_join_few_kernel(const float* __restrict__ part_out,
                                                                     const float* __restrict__ part_stats,
                                                                     float* __restrict__ out, float* __restrict__ stats,
                                                                     size_t rows, int parts, int dim, int pitch) {
  const size_t row = (size_t)blockIdx.x * 16 + threadIdx.x / 16;
  if (row >= rows) return;
  const int lane = threadIdx.x % 16;
  float w[MOST], ls[MOST], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int s = 0; s < MOST; ++s) {
    const size_t at = (s < parts ? s : 0) * rows + row;
    w[s] = part_stats[2 * at];
    ls[s] = s < parts ? part_stats[2 * at + 1] : 0.f;
  }
#pragma unroll
  for (int s = 0; s < MOST; ++s) m = fmaxf(m, w[s]);
#pragma unroll
  for (int s = 0; s < MOST; ++s) {
    w[s] = ls[s] == 0.f ? 0.f : mnv_weight(w[s], mnv_finite_max(m));
    l = fmaf(ls[s], w[s], l);
  }
  const float f = mnv_inverse(l);
  for (int d = 4 * lane; d < pitch; d += 64) {
    mnv_f4 t[MOST], acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < MOST; ++s) {
      t[s] = mnv_f4{0.f, 0.f, 0.f, 0.f};
      if (ls[s] != 0.f) t[s] = *reinterpret_cast<const mnv_f4*>(part_out + (s * rows + row) * pitch + d);
    }
#pragma unroll
    for (int s = 0; s < MOST; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(t[s][e], w[s], acc[e]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < dim) out[row * dim + d + e] = acc[e] * f;
  }
  if (lane < 2) stats[2 * row + lane] = lane ? l : m;
}

// Wavefronts of a workgroup: eight, in two halves, where a workgroup has the CU to itself and rows enough (128 wide, 2 x 16
// heads of 2048 x 4096: 626 us, 707 with four; 4 x 8 heads of 512 x 2048, a quarter of the chip: 99.5 and 103; 8 heads of
// 512 x 2048: 42.7 and 39.9).  Four also for a few rows, where three of them only bring tiles: 16 heads of 4 key heads for
// one query over 2000 keys 13.2 us, with one wavefront that does all 14.9; 128 wide, over 16384 keys 48 and 80.
int wavefronts(const AttentionSizes& z) {
  const size_t rows = (size_t)z.q_len * z.group();
  return z.dim > 64 && mnv_ceil_div(rows, 256) * z.batch * z.kv_heads >= (size_t)mnv_cu_count() / 4 ? 8 : 4;
}
size_t part_bytes(const AttentionSizes& z) { return z.q_rows() * (mnv_attention_padded(z.dim) + 2) * sizeof(float); }
int parts(const AttentionSizes& z, bool lengths, size_t workspace_bytes) {
  const int nw = wavefronts(z);
  const size_t blocks = mnv_ceil_div((size_t)z.q_len * z.group(), 32 * nw) * z.batch * z.kv_heads;
  // workgroups that a CU holds, by LDS (129 x 1500, 64 wide: 32.7 us, 35.7 with two; over 64 wide 28 us of 16 heads for one
  // query over 2000 keys, 33 with two)
  const size_t places = (size_t)mnv_cu_count() * (z.dim <= 64 ? 3 : 1);
  // Where every CU has a workgroup anyway, parts of less than 512 keys cost more to join than they even out (8 x 12 heads of 512 x
  // 512: 51 us in two parts, 47 in one; of 384 x 1024: 74 and 80; 32 heads for each of 9 queries over 4000 keys: 127 and 191).
  const size_t least = blocks > (size_t)mnv_cu_count() ? 16 : 2;
  const auto fill = [&](size_t n) {
    return mnv_attention_parts(blocks, n, mnv_ceil_div(z.k_len, 32), least, part_bytes(z), workspace_bytes);
  };
  // Of parts behind an entry's keys nothing is left to do, so where there are lengths twice as many even out the
  // rest (12 heads of 129 queries, 6 entries of 0 to 1500 keys: 43 us -> 35); not where there would be one
  // otherwise, which needs no joining (16 heads of 512 queries, 8 entries of 128 to 1024 keys: 80 us, of 2 parts 66 and 35
  // to join them).
  const int once = fill(places);
  return lengths && once > 1 ? fill(2 * places) : once;
}

template <int DP, int NW>
int launch(FwdArgs& a, hipStream_t s) {
  a.row_tiles = (int)mnv_ceil_div(a.rows, 32 * NW);
  const dim3 g((unsigned)a.row_tiles * a.parts * a.z.batch * a.z.kv_heads), b(64 * NW);
  const bool vec = a.z.dim % 4 == 0;
  if (a.bias && vec) hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, true, true>), g, b, 0, s, a);
  else if (a.bias) hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, true, false>), g, b, 0, s, a);
  else if (vec) hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, false, true>), g, b, 0, s, a);
  else hipLaunchKernelGGL((mnv_attention_fwd_kernel<DP, NW, false, false>), g, b, 0, s, a);
  return MNV_LAUNCH_STATUS();
}

template <int DP>
int launch_width(FwdArgs& a, int nw, hipStream_t s) {
  if (DP > 64 && nw == 8) return launch<DP, DP <= 64 ? 4 : 8>(a, s);
  return launch<DP, 4>(a, s);
}

}  // namespace

extern "C" {

size_t mnv_attention_fwd_workspace_bytes(int batch, int heads, int kv_heads, int q_len, int k_len, int head_dim) {
  const AttentionSizes z = {batch, heads, kv_heads, q_len, k_len, head_dim, 1.f};
  if (!mnv_attention_sizes_ok(z)) return 0;
  const int full = parts(z, false, MNV_AT_ANY_WORKSPACE), ragged = parts(z, true, MNV_AT_ANY_WORKSPACE);
  const int n = full > ragged ? full : ragged;
  return n > 1 ? n * part_bytes(z) : 0;
}

int mnv_attention_fwd(const float* q, const float* k, const float* v, const float* bias, const float* lengths,
                      float* out, float* stats, int batch, int heads, int kv_heads, int q_len, int k_len, int head_dim,
                      float scale, void* workspace, size_t workspace_bytes, mnv_stream_t stream) {
  const AttentionSizes z = {batch, heads, kv_heads, q_len, k_len, head_dim, scale};
  if (!q || !k || !v || !out || !stats || !mnv_attention_sizes_ok(z)) return MNV_ERR_INVALID;
  FwdArgs a = {q, k, v, bias, lengths, out, stats, z, q_len * z.group(), 0, mnv_fastdiv_make(z.group()), 0, 1, nullptr, nullptr};
  a.parts = parts(z, lengths != nullptr, workspace && mnv_aligned16(workspace) ? workspace_bytes : 0);
  a.chunk = (int)mnv_ceil_div(mnv_ceil_div(k_len, 32), a.parts) * 32;
  a.part_out = static_cast<float*>(workspace);
  a.part_stats = a.part_out + (a.parts > 1 ? a.parts * z.q_rows() * mnv_attention_padded(head_dim) : 0);
  const hipStream_t s = mnv_stream(stream);
  const int nw = wavefronts(z), dp = mnv_attention_padded(head_dim);
  const int rc = dp == 32   ? launch_width<32>(a, nw, s)
                 : dp == 64 ? launch_width<64>(a, nw, s)
                 : dp == 96 ? launch_width<96>(a, nw, s)
                            : launch_width<128>(a, nw, s);
  if (rc || a.parts == 1) return rc;
  const auto join = a.parts <= 8    ? mnv_attention_join_few_kernel<8>
                    : a.parts <= 16 ? mnv_attention_join_few_kernel<16>
                                    : mnv_attention_join_kernel;
  hipLaunchKernelGGL(join, dim3((unsigned)mnv_ceil_div(z.q_rows(), a.parts <= 16 ? 16 : 4)), dim3(256), 0, s, a.part_out,
                     a.part_stats, out, stats, z.q_rows(), a.parts, head_dim, dp);
  return MNV_LAUNCH_STATUS();
}

}  // extern "C"
