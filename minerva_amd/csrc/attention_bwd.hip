// Attention, backward: dq, dk, dv and the bias's gradient from what the forward pass kept (m and l of each row).
//   p_ij = exp(t_ij - m_i) / l_i,  ds_ij = p_ij * (dout_i.v_j - delta_i),  delta_i = dout_i.out_i
//   dq_i = scale * sum_j ds_ij k_j,  dk_j = scale * sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
//   dbias[o] = sum of ds_ij with j - i + q_len - 1 = o
// Scores are computed again, twice: once with a workgroup's 128 keys in registers while queries and their
// gradients stream through LDS (dk, dv, dbias), once with its 128 rows of queries in registers while keys and
// values do (dq).  That is 7 products where 5 would do, but every gradient is summed by one wavefront
// in one order: no atomics, and no partial gradients in memory unless the chip is empty otherwise.  delta waits in the
// first value of each row of dq, which the last kernel overwrites, so no workspace is needed for it.
// Bound by the matrix cores, 7 products of 6 instructions per value: 2 x 16 heads (4 key heads) of 2048 x 4096, 128 wide: dk and dv
// 1.24 to 1.29 ms (213 to 222 TFLOP/s of its 4 fp32 products, cores busy 66%), dq 1.00 to 1.07 ms (192 to 206 of its 3, 59%),
// about 150 of the 5 that the algorithm needs; the clock is 1.9 GHz under such work.  The rest waits for LDS at the products'
// starts, and for vector work between dout v and dq.  8 x 16 heads of 512 x 1024, 64 wide, lengths 128 to 1024: 137 and 106 us,
// and 8 to 12 for delta.  Two workgroups to a CU leave the keys' kernel of 64 columns 256 registers, of which it has too
// few: 27 (47 with a bias; 35 and 63 of odd widths) wait in scratch memory, 104 to 256 bytes a lane, in and out in every tile (8 x 16
// heads of 512 x 1024: 81 MB written, of which 67 are results).  The other kernels of the backward pass keep theirs.
#include "attention_core.h"

namespace {

struct BwdArgs {
  const float *q, *k, *v, *bias, *lengths, *out, *stats, *dout;
  float *dq, *dk, *dv;
  float* parts;         // sums of ds along the diagonals of each wavefront's 32 keys, or NULL
  AttentionSizes z;
  int tiles;            // workgroups per entry and key head
  unsigned first_pair;  // the launch's first (entry, key head)
  int rows;             // q_len * group
  MnvFastDiv by_group;
  // The loop of a workgroup (dk, dv: over a group's heads and their tiles of queries; dq: over tiles of keys) in
  // `splits` parts of `chunk` tiles each; with more than one, sums by part in `sums`: [part][row][DP], and for
  // dk and dv those of dv behind those of dk
  int splits, chunk;
  float* sums;
};

// dq[row][0] = dout_row . out_row; 16 lanes per row.  Bound by memory (65536 rows of 64: 7.5 to 12 us).
__global__ __launch_bounds__(256) void mnv_attention_delta_kernel(const float* __restrict__ dout,
                                                                  const float* __restrict__ out,
                                                                  float* __restrict__ dq, size_t rows, int dim) {
  const size_t row = (size_t)blockIdx.x * 16 + threadIdx.x / 16;
  if (row >= rows) return;
  float s = 0.f;
  for (int d = threadIdx.x % 16; d < dim; d += 16) s = fmaf(dout[row * dim + d], out[row * dim + d], s);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 16);
  if (threadIdx.x % 16 == 0) dq[row * dim] = s;
}

// Floats of one wavefront's partial diagonal sums: those of 32 keys and the queries in tiles of 32.
__host__ __device__ inline size_t diagonal_pitch(int q_len) { return ((size_t)q_len + 31) / 32 * 32 + 32; }
__host__ __device__ inline size_t key_tiles(int k_len) { return ((size_t)k_len + 31) / 32; }

template <int DP, bool BIAS, bool VEC>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void mnv_attention_dkv_kernel(BwdArgs a) {
  constexpr int NB = DP / 32, KS = DP / 16;
  using Stage = MnvStage<DP, 256, VEC>;  // queries and their gradients
  __shared__ __align__(16) char lds[2 * Stage::BYTES];
  __shared__ __align__(16) float row_stats[2][3][32];  // m, 1 / l, delta of the tile's queries
  __shared__ float turned[BIAS ? 4 * 16 * 48 : 1];
  const AttentionSizes& z = a.z;
  const MnvAttentionPlace place =
      mnv_attention_place(a.tiles * a.splits, a.splits, DP <= 64 ? 128 : 0, a.first_pair, z, a.lengths);
  const int tile = mnv_uniform(place.tile / a.splits), split = place.tile - tile * a.splits;
  const int b = place.b, kh = place.kh, n = place.n, group = z.group();
  const int q_tiles = (z.q_len + 31) / 32, begin = split * a.chunk;
  const int end = begin + a.chunk < group * q_tiles ? begin + a.chunk : group * q_tiles;
  const int wave = mnv_uniform(threadIdx.x / MNV_WAVE), lane = threadIdx.x % MNV_WAVE, half = lane / 32;

  const int j = tile * 128 + wave * 32 + lane % 32;
  const size_t key = ((size_t)b * z.k_len + (j < z.k_len ? j : z.k_len - 1)) * z.kv_heads + kh;
  mnv_f16 dk[NB], dv[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[c][e] = dv[c][e] = 0.f;

  if (tile * 128 < n) {
    if (BIAS)
      for (int e = threadIdx.x; e < 4 * 16 * 48; e += 256) turned[e] = 0.f;
    const bool shown = j < n;
    // The matrix instruction rounds its sums down, by up to a step of the larger of sum and terms: nothing to a
    // value, but of the same sign everywhere, and a bucket's gradient sums 10^5 ds that cancel.  So every other key's
    // products dout v are made with the opposite sign (12 heads of 512 x 512: the table's gradient off
    // by 4.0e-6 without, 4.8e-7 with).  The other products keep theirs: over 16384 keys, v and dout from a ReLU, out is
    // off by 0.8e-7 and dv by 1.4e-7, in elementary fp32 operations by 3.4e-7 and 1.4e-7.
    const float sign = j % 2 ? -1.f : 1.f;
    MnvParts kp[KS], vp[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8], y[8];
      // a key that is not read may hold anything: another one stands in for it, and 0 is stored
      const size_t at = ((size_t)b * z.k_len + (shown ? j : n - 1)) * z.kv_heads + kh;
      mnv_load8<DP, VEC>(a.k + at * z.dim, s, z.dim, x);
      mnv_load8<DP, VEC>(a.v + at * z.dim, s, z.dim, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= z.scale;
        y[e] *= sign;
      }
      kp[s] = mnv_cut8(x);
      vp[s] = mnv_cut8(y);
    }
    const unsigned pitch = (unsigned)z.heads * z.dim;
    const int jb = shown ? j : n - 1;
    const int first_g = mnv_uniform(begin / q_tiles), last_g = mnv_uniform((end - 1) / q_tiles);
    for (int g = first_g; g <= last_g; ++g) {
      const int from = g == first_g ? (begin - g * q_tiles) * 32 : 0;
      const int to = g == last_g && (end - g * q_tiles) * 32 < z.q_len ? (end - g * q_tiles) * 32 : z.q_len;
      const int h = kh * group + g;
      const size_t row0 = (size_t)b * z.q_len * z.heads + h;  // rows of the head are z.heads apart
      const float* qb = a.q + row0 * z.dim;
      const float* ob = a.dout + row0 * z.dim;
      const float* bias = BIAS ? a.bias + h * z.offsets() + (jb + z.q_len - 1) : nullptr;
      float* parts = nullptr;
      if (BIAS && a.parts && tile * 128 + wave * 32 < n)  // no others are read
        parts = a.parts + (((size_t)place.pair * group + g) * key_tiles(z.k_len) + tile * 4 + wave) *
                              diagonal_pitch(z.q_len);
      float carry = 0.f;
      struct Rows {
        float m, l, delta;
      };
      auto fetch_rows = [&](Rows& next, int i0) __attribute__((always_inline)) {
        if (threadIdx.x < 32) {
          const int i = i0 + (int)threadIdx.x;
          const size_t row = row0 + (size_t)(i < z.q_len ? i : z.q_len - 1) * z.heads;
          next.m = a.stats[2 * row];
          next.l = a.stats[2 * row + 1];
          next.delta = a.dq[row * z.dim];
        }
      };
      // 1 / l is 0 for a row that sees no key, and -0 behind the last row
      auto store_rows = [&](const Rows& next, int i0, int turn) __attribute__((always_inline)) {
        if (threadIdx.x < 32) {
          const float il = i0 + (int)threadIdx.x < z.q_len ? mnv_inverse(next.l) : -0.f;
          row_stats[turn][0][threadIdx.x] = mnv_finite_max(next.m);
          row_stats[turn][1][threadIdx.x] = il;
          row_stats[turn][2][threadIdx.x] = il == 0.f ? 0.f : next.delta;
        }
      };
      // Behind the last tile comes that one again: no branch parts a tile's work.
      const int last = from + (to - from - 1) / 32 * 32;
      Stage stage;
      {
        Rows first;
        fetch_rows(first, from);
        stage.fetch(qb + (size_t)from * pitch, ob + (size_t)from * pitch, pitch, z.q_len - from, z.dim);
        stage.store(lds);
        store_rows(first, from, 0);
        const int i1 = from < last ? from + 32 : last;
        stage.fetch(qb + (size_t)i1 * pitch, ob + (size_t)i1 * pitch, pitch, z.q_len - i1, z.dim);
      }
      __syncthreads();
      int turn = 0;
      for (int i0 = from; i0 < to; i0 += 32) {
        const bool more = i0 < last;
        Rows next;
        fetch_rows(next, more ? i0 + 32 : last);
        const int i2 = i0 + 64 < last ? i0 + 64 : last;
        const char* now = lds + turn * Stage::BYTES;
        mnv_f4 add[4];
        if (BIAS) {
          if (i0 + 32 <= z.q_len) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const mnv_f4 x = mnv_ldx4u<false>(bias - (i0 + 8 * u + 4 * half + 3));
              add[u] = mnv_f4{x.w, x.z, x.y, x.x};
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int i = i0 + 8 * u + 4 * half + e;
                add[u][e] = bias[-(i < z.q_len ? i : z.q_len - 1)];
              }
          }
        }

        // Four products in a row, a step per operand: the scores, under which the next tile is cut; dout v, under which
        // the weights are made of the scores and cut; dv, under which ds is; dk, under which the tile after the
        // next is fetched.
        mnv_f16 t, dp;
#pragma unroll
        for (int e = 0; e < 16; ++e) t[e] = dp[e] = 0.f;
        MnvCutting pc[2], sc[2];
        auto operand = [&](int k, int c) __attribute__((always_inline)) {
          const int s = k % KS;
          return k < KS       ? Stage::by_rows(now, s, c)
                 : k < 2 * KS ? Stage::by_rows(now + Stage::MATRIX, s, c)
                 : k < 3 * KS ? Stage::by_cols(now + Stage::MATRIX, s % NB * 32, s / NB, c)
                              : Stage::by_cols(now, s % NB * 32, s / NB, c);
        };
        // the numbers of two queries (a pair of result registers) that a step needs, read in the step before
        constexpr int MOST = (8 + KS - 1) / KS;
        mnv_f2 rows[2][MOST];
        auto read_rows = [&](int k) __attribute__((always_inline)) {
          if (k < KS || k >= 3 * KS) return;
          const int first = k % KS * 8 / KS;
#pragma unroll
          for (int u = 0; u < MOST; ++u) {
            const int pair = first + u;
            if (pair >= (k % KS + 1) * 8 / KS) continue;
            rows[0][u] = *reinterpret_cast<const mnv_f2*>(row_stats[turn][k < 2 * KS ? 0 : 2] + mnv_acc_row(2 * pair, half));
            if (k < 2 * KS) rows[1][u] = *reinterpret_cast<const mnv_f2*>(row_stats[turn][1] + mnv_acc_row(2 * pair, half));
          }
        };
        MnvParts cur = {{operand(0, 0), operand(0, 1), operand(0, 2)}};
        // Rows of the tile that see no key, since the bias hides all: their weights are 0, their gradients may hold anything, and
        // leave LDS before the two meet.  All wavefronts see the same rows.  Asked behind the first operands' reads, whose wait it
        // shares (8 x 12 heads of 512 x 512: 134.6 us for the backward pass, 137.9 at the tile's start).
        if (BIAS && __builtin_expect(__any(__builtin_bit_cast(unsigned, row_stats[turn][1][lane % 32]) == 0), 0)) {
          char* planes = lds + turn * Stage::BYTES + Stage::MATRIX;
          const int row = threadIdx.x / 8;
          if (row_stats[turn][1][row] == 0.f)
            for (int at = threadIdx.x % 8 * 8; at < 3 * Stage::PITCH; at += 64)
              *reinterpret_cast<mnv_u2*>(planes + at / Stage::PITCH * Stage::PLANE + row * Stage::PITCH + at % Stage::PITCH) = mnv_u2{0, 0};
          __syncthreads();
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < 4 * KS; ++k) {
          const int s = k % KS;
          auto step = [&](mnv_f16& acc, const MnvParts& b) __attribute__((always_inline)) {
            auto after = [&](int c) __attribute__((always_inline)) { return operand(k + 1, c); };
            if (k + 1 < 4 * KS) mnv_step<false>(acc, cur, b, after);
            else mnv_step<true>(acc, cur, b, after);
          };
          mnv_f2 mine[2][MOST];
#pragma unroll
          for (int c = 0; c < MOST; ++c) {
            mine[0][c] = rows[0][c];
            mine[1][c] = rows[1][c];
          }
          read_rows(k + 1);
          if (k < KS) {
            step(t, kp[s]);
            stage.store_piece(s, lds + (turn ^ 1) * Stage::BYTES);
          } else if (k < 2 * KS) {
            step(dp, vp[s]);
#pragma unroll
            for (int u = 0; u < MOST; ++u) {
              const int pair = s * 8 / KS + u;
              if (pair >= (s + 1) * 8 / KS) continue;
              const mnv_f2 m = mine[0][u], il = mine[1][u];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int r = 2 * pair + e;
                if (BIAS) t[r] += add[r / 4][r % 4];
                t[r] = mnv_weight(t[r], m[e]) * il[e];
              }
              pc[pair / 4].pair(pair % 4, t[2 * pair], t[2 * pair + 1]);
            }
          } else if (k < 3 * KS) {
            step(dv[s % NB], pc[s / NB].parts());
#pragma unroll
            for (int u = 0; u < MOST; ++u) {
              const int pair = s * 8 / KS + u;
              if (pair >= (s + 1) * 8 / KS) continue;
              const mnv_f2 delta = mine[0][u];
#pragma unroll
              for (int e = 0; e < 2; ++e) dp[2 * pair + e] = t[2 * pair + e] * fmaf(dp[2 * pair + e], sign, -delta[e]);
              sc[pair / 4].pair(pair % 4, dp[2 * pair], dp[2 * pair + 1]);
            }
          } else {
            step(dk[s % NB], sc[s / NB].parts());
            stage.fetch_piece(s, qb + (size_t)i2 * pitch, ob + (size_t)i2 * pitch, pitch, z.q_len - i2, z.dim);
          }
          MNV_STEP_ORDER(6);
        }
        turn ^= 1;
        store_rows(next, i0 + 32, turn);
        if (BIAS && parts) {
          // Lane u sums the diagonal key - query = u - 31 of the 32 x 32 tile: 16 queries at a time go to LDS,
          // each shifted by its number, so that a diagonal is a column; what a row does not reach stays 0.  The
          // next tile's diagonals lie 32 lower, so those below 0 go on in the lane 32 higher; the others
          // are whole, and written.
          float* mine = turned + wave * 16 * 48;
          float sum = carry;
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int i = mnv_acc_row(e, half);
              mine[i * 47 + 15 + lane % 32] = shown ? dp[8 * part + e] : 0.f;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int u = part == 0 ? lane - 16 : lane;
            const bool in = u >= 0 && u < 47;
            const float* column = mine + (in ? u : 0);
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) x += column[i * 48];
            sum += in ? x : 0.f;
            __builtin_amdgcn_wave_barrier();
          }
          const size_t at = diagonal_pitch(z.q_len) - 64 - i0 + lane;  // place of the diagonal key - query = lane - 31
          if (lane >= 31 && lane < 63) parts[at] = sum;
          if (!more && lane < 31) parts[at] = sum;
          carry = __shfl(sum, lane - 32, MNV_WAVE);
          carry = lane >= 32 && lane < 63 ? carry : 0.f;
        }
        __syncthreads();
      }
    }
  }
  if (j < z.k_len && a.splits > 1) {
    // of keys that are not read, nothing: mnv_attention_sum_kernel knows them
    const size_t keys = (size_t)z.batch * z.k_len * z.kv_heads;
    float* to = a.sums + (split * keys + key) * DP;
    if (j < n) {
      mnv_store_column<DP>(dk, z.scale, true, to, DP);
      mnv_store_column<DP>(dv, 1.f, true, to + a.splits * keys * DP, DP);
    }
  } else if (j < z.k_len) {
    mnv_store_column<DP>(dk, z.scale, j < n, a.dk + key * z.dim, z.dim);
    mnv_store_column<DP>(dv, 1.f, j < n, a.dv + key * z.dim, z.dim);
  }
}

template <int DP, bool BIAS, bool VEC>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void mnv_attention_dq_kernel(BwdArgs a) {
  constexpr int NB = DP / 32, KS = DP / 16;
  using Stage = MnvStage<DP, 256, VEC>;  // keys and values
  __shared__ __align__(16) char lds[2 * Stage::BYTES];
  const AttentionSizes& z = a.z;
  const MnvAttentionPlace place = mnv_attention_place(a.tiles * a.splits, 0, 0, 0, z, a.lengths);
  const int split = mnv_uniform(place.tile / a.tiles), tile = place.tile - split * a.tiles, b = place.b, kh = place.kh;
  // the part's keys
  const int begin = split * a.chunk * 32, n = place.n < begin + a.chunk * 32 ? place.n : begin + a.chunk * 32;
  const int lane = threadIdx.x % MNV_WAVE, half = lane / 32;

  const int r = tile * 128 + (int)threadIdx.x / MNV_WAVE * 32 + lane % 32;
  const int rc = r < a.rows ? r : a.rows - 1;
  const int i = mnv_fastdiv(rc, a.by_group), h = kh * z.group() + (rc - i * z.group());
  const size_t row = ((size_t)b * z.q_len + i) * z.heads + h;

  mnv_f16 dq[NB];
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) dq[c][e] = 0.f;

  bool seen = false;
  if (n > begin) {
    MnvParts qp[KS], op[KS];
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8], y[8], o[8];
      mnv_load8<DP, VEC>(a.q + row * z.dim, s, z.dim, x);
      mnv_load8<DP, VEC>(a.dout + row * z.dim, s, z.dim, y);
      mnv_load8<DP, VEC>(a.out + row * z.dim, s, z.dim, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= z.scale;
        delta = fmaf(y[e], o[e], delta);
      }
      qp[s] = mnv_cut8(x);
      op[s] = mnv_cut8(y);
    }
    delta += __shfl_xor(delta, 32, MNV_WAVE);
    const float m = mnv_finite_max(a.stats[2 * row]), il = mnv_inverse(a.stats[2 * row + 1]);
    seen = il != 0.f;  // else the row's gradient may hold anything, which weights of 0 do not hide
    const unsigned pitch = (unsigned)z.kv_heads * z.dim;
    const float* kb = a.k + ((size_t)b * z.k_len * z.kv_heads + kh) * z.dim;
    const float* vb = a.v + ((size_t)b * z.k_len * z.kv_heads + kh) * z.dim;
    const float* bias = BIAS ? a.bias + h * z.offsets() + (z.q_len - 1 - i) : nullptr;

    // Behind the last tile comes that one again: no branch parts a tile's work.
    const int last = begin + (n - begin - 1) / 32 * 32;
    Stage stage;
    stage.fetch(kb + (size_t)begin * pitch, vb + (size_t)begin * pitch, pitch, n - begin, z.dim);
    stage.store(lds);
    {
      const int j1 = begin < last ? begin + 32 : last;
      stage.fetch(kb + (size_t)j1 * pitch, vb + (size_t)j1 * pitch, pitch, n - j1, z.dim);
    }
    __syncthreads();
    char* now = lds;
    for (int j0 = begin; j0 < n; j0 += 32) {
      const bool whole = j0 + 32 <= n;
      const int j2 = j0 + 64 < last ? j0 + 64 : last;
      mnv_f4 add[4];
      if (BIAS) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + 8 * u + 4 * half;
          if (whole) {
            add[u] = mnv_ldx4u<false>(bias + j);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) add[u][e] = bias[j + e < n ? j + e : n - 1];
          }
        }
      }
      char* then = lds + (now == lds ? Stage::BYTES : 0);
      // keys of the tile that are read: the others' weights become 0
      const int left = n - j0 - 4 * half;

      // Three products in a row: the scores, under which the next tile is cut; dout v, under which the weights are made
      // of the scores; dq, under which the second half of ds is made and the tile after the next fetched.
      mnv_f16 t, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) t[e] = dp[e] = 0.f;
      MnvCutting sc[2];
      auto cut_ds = [&](int pair) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) dp[2 * pair + e] = t[2 * pair + e] * (dp[2 * pair + e] - delta);
        sc[pair / 4].pair(pair % 4, dp[2 * pair], dp[2 * pair + 1]);
      };
      auto operand = [&](int k, int c) __attribute__((always_inline)) {
        const int s = k % KS;
        return k < KS       ? Stage::by_rows(now, s, c)
               : k < 2 * KS ? Stage::by_rows(now + Stage::MATRIX, s, c)
                            : Stage::by_cols(now, s % NB * 32, s / NB, c);
      };
      MnvParts cur = {{operand(0, 0), operand(0, 1), operand(0, 2)}};
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 3 * KS; ++k) {
        const int s = k % KS;
        auto step = [&](mnv_f16& acc, const MnvParts& b) __attribute__((always_inline)) {
          auto after = [&](int c) __attribute__((always_inline)) { return operand(k + 1, c); };
          if (k + 1 < 3 * KS) mnv_step<false>(acc, cur, b, after);
          else mnv_step<true>(acc, cur, b, after);
        };
        if (k < KS) {
          step(t, qp[s]);
          stage.store_piece(s, then);
        } else if (k < 2 * KS) {
          step(dp, op[s]);
#pragma unroll
          for (int u = 0; u < (16 + KS - 1) / KS; ++u) {
            const int r = s * 16 / KS + u;
            if (r >= (s + 1) * 16 / KS) continue;
            if (BIAS) t[r] += add[r / 4][r % 4];
            t[r] = mnv_acc_row(r, 0) < left ? mnv_weight(t[r], m) * il : 0.f;
          }
        } else {
          if (s == 0) {
#pragma unroll
            for (int pair = 0; pair < 4; ++pair) cut_ds(pair);
          }
          step(dq[s % NB], sc[s / NB].parts());
          if (s < NB) {
#pragma unroll
            for (int u = 0; u < (4 + NB - 1) / NB; ++u)
            if (4 + s * 4 / NB + u < 4 + (s + 1) * 4 / NB) cut_ds(4 + s * 4 / NB + u);
          }
          stage.fetch_piece(s, kb + (size_t)j2 * pitch, vb + (size_t)j2 * pitch, pitch, n - j2, z.dim);
        }
        MNV_STEP_ORDER(6);
      }
      now = then;
      __syncthreads();
    }
  }
  if (r >= a.rows) return;
  if (a.splits == 1)
    mnv_store_column<DP>(dq, z.scale, seen, a.dq + row * z.dim, z.dim);
  else if (n > begin)  // of a part without keys, nothing
    mnv_store_column<DP>(dq, 1.f, seen, a.sums + (split * z.q_rows() + row) * DP, DP);
}

// out[row] = f * the sums of a row's parts, 0 for none; 16 lanes to a row.  blockIdx.y: dk and dv.  Of queries the parts that
// have keys count, `chunk` keys to each; of keys all, for those that are read.  Bound by memory and the launch (5994 rows
// of 72 in 2 parts: 4.4 us).
__global__ __launch_bounds__(256) void mnv_attention_sum_kernel(const float* __restrict__ sums, float* __restrict__ out0,
                                                                float* __restrict__ out1,
                                                                const float* __restrict__ lengths, AttentionSizes z,
                                                                bool queries, int splits, int chunk, int pitch, float f) {
  const size_t rows = queries ? z.q_rows() : (size_t)z.batch * z.k_len * z.kv_heads;
  const size_t row = (size_t)blockIdx.x * 16 + threadIdx.x / 16;
  if (row >= rows) return;
  float* out = blockIdx.y ? out1 : out0;
  sums += (size_t)blockIdx.y * splits * rows * pitch;
  const size_t per_entry = queries ? (size_t)z.q_len * z.heads : (size_t)z.k_len * z.kv_heads;
  const int n = mnv_visible(lengths, (int)(row / per_entry), z.k_len);
  int parts = splits;
  if (queries) parts = n < splits * chunk ? (n + chunk - 1) / chunk : splits;
  else if ((int)(row % per_entry / z.kv_heads) >= n) parts = 0;
  for (int d = threadIdx.x % 16 * 4; d < z.dim; d += 64) {
    mnv_f4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += 4) {
      mnv_f4 t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        t[u] = s0 + u < parts ? *reinterpret_cast<const mnv_f4*>(sums + ((s0 + u) * rows + row) * pitch + d)
                              : mnv_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += t[u][e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < z.dim) out[row * z.dim + d + e] = acc[e] * f;
  }
}

// dbias[o] += the parts of o: of every entry among the launch's pairs and every 32 keys that have the diagonal.  64 offsets to
// a workgroup, 16 threads to an offset, each with every 16th 32 keys (8 x 12 heads of 512 x 512: 5.8 us; 25 with one thread to
// an offset).
__global__ __launch_bounds__(1024) void mnv_attention_dbias_kernel(const float* __restrict__ parts,
                                                                   const float* __restrict__ lengths,
                                                                   float* __restrict__ dbias, AttentionSizes z,
                                                                   unsigned first_pair, unsigned pairs, bool first) {
  __shared__ float lds[16][64];
  const size_t offsets = z.offsets();
  const int lane = threadIdx.x % 64, slice = threadIdx.x / 64;
  const size_t o = (size_t)blockIdx.x * 64 + lane;
  const size_t pitch = diagonal_pitch(z.q_len), per_key = key_tiles(z.k_len);
  const int group = z.group(), padded = (int)pitch - 32;
  for (int h = blockIdx.y; h < z.heads; h += gridDim.y) {
    float s = 0.f;
    // the pairs of the head's key head: one to an entry
    const unsigned kh = h / group, from_pair = (kh + z.kv_heads - first_pair % z.kv_heads) % z.kv_heads;
    // key kt + c and query 32 s + r of the part: place o - kt + padded - q_len
    const long long place = (long long)o + padded - z.q_len;
    long long from = place - (padded + 30);
    from = (from <= 0 ? 0 : (from + 31) / 32 * 32) + 32 * slice;
    if (o < offsets)
      for (unsigned p = from_pair; p < pairs; p += z.kv_heads) {
        const int n = mnv_visible(lengths, (first_pair + p) / z.kv_heads, z.k_len);
        const float* mine = parts + ((size_t)p * group + h % group) * per_key * pitch;
        for (long long kt = from; kt < n && kt <= place; kt += 32 * 16) s += mine[kt / 32 * pitch + (place - kt)];
      }
    __syncthreads();
    lds[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && o < offsets) {
      s = first ? 0.f : dbias[h * offsets + o];
#pragma unroll
      for (int u = 0; u < 16; ++u) s += lds[u][lane];
      dbias[h * offsets + o] = s;
    }
  }
}

// The bias's gradient without a workspace: one wavefront per head and offset goes through all its pairs of
// a query and a key and computes their scores again, one after the other.
__device__ __forceinline__ float dot(const float* a, const float* b, int n) {
  float s = 0.f;
  for (int d = 0; d < n; ++d) s = fmaf(a[d], b[d], s);
  return s;
}
__global__ __launch_bounds__(MNV_WAVE) void mnv_attention_dbias_alone_kernel(BwdArgs a, float* __restrict__ dbias) {
  const AttentionSizes& z = a.z;
  const size_t offsets = z.offsets();
  for (size_t at = blockIdx.x; at < offsets * z.heads; at += gridDim.x) {
    const int h = (int)(at / offsets), o = (int)(at % offsets), kh = h / z.group();
    float sum = 0.f;
    for (int b = 0; b < z.batch; ++b) {
      const int n = mnv_visible(a.lengths, b, z.k_len);
      for (int i = threadIdx.x; i < z.q_len; i += MNV_WAVE) {
        const int j = o + i - (z.q_len - 1);
        if (j < 0 || j >= n) continue;
        const size_t row = ((size_t)b * z.q_len + i) * z.heads + h;
        const float il = mnv_inverse(a.stats[2 * row + 1]);
        if (il == 0.f) continue;  // sees no key
        const float* kj = a.k + (((size_t)b * z.k_len + j) * z.kv_heads + kh) * z.dim;
        const float* vj = a.v + (((size_t)b * z.k_len + j) * z.kv_heads + kh) * z.dim;
        const float* oi = a.dout + row * z.dim;
        const float t = z.scale * dot(a.q + row * z.dim, kj, z.dim) + a.bias[at];
        const float p = mnv_weight(t, mnv_finite_max(a.stats[2 * row])) * il;
        sum += p * (dot(oi, vj, z.dim) - dot(oi, a.out + row * z.dim, z.dim));
      }
    }
    sum = mnv_wave_sum(sum);
    if (threadIdx.x == 0) dbias[at] = sum;
  }
}

// Bytes of the partial diagonal sums of one entry and key head.
size_t pair_bytes(const AttentionSizes& z) {
  return (size_t)z.group() * key_tiles(z.k_len) * diagonal_pitch(z.q_len) * sizeof(float);
}
#define MNV_AT_PARTS_BYTES ((size_t)256 << 20)  // of partial sums of diagonals at a time, where there are more

// How a call uses its workspace: the diagonals' partial sums of `pairs` pairs of an entry and a key head at a
// time (0: none) first, the parts' sums behind them.  dq's come after dk's and dv's are added up.
struct BwdPlan {
  size_t pairs, diagonal_bytes;
  int key_splits, query_splits;
  size_t bytes;
};
BwdPlan make_plan(const AttentionSizes& z, bool has_bias, size_t workspace_bytes) {
  BwdPlan p = {0, 0, 1, 1, 0};
  const size_t pairs = (size_t)z.batch * z.kv_heads, dp = mnv_attention_padded(z.dim);
  if (has_bias) {
    const size_t one = pair_bytes(z), most = workspace_bytes < MNV_AT_PARTS_BYTES ? workspace_bytes : MNV_AT_PARTS_BYTES;
    p.pairs = most / one;
    if (p.pairs == 0 && workspace_bytes >= one) p.pairs = 1;
    if (p.pairs > pairs) p.pairs = pairs;
    p.diagonal_bytes = p.pairs * one;  // a multiple of 128
  }
  // One workgroup to a CU: more parts, where a CU holds two, cost more to add up than they save (2 x 8 heads of 200 x 1000, 32
  // wide: 32.7 us, 39.0 with two; 8 heads of 1 x 4096, 64 wide: 30.4 and 33.5).
  const size_t left = workspace_bytes - p.diagonal_bytes, places = mnv_cu_count();
  // a head's diagonals are summed by one workgroup
  const size_t key_part = 2 * (size_t)z.batch * z.k_len * z.kv_heads * dp * sizeof(float);
  const size_t q_tiles = mnv_ceil_div(z.q_len, 32);
  const bool whole_heads = p.pairs > 0;
  if (p.pairs == 0 || p.pairs == pairs)
    p.key_splits = mnv_attention_parts(mnv_ceil_div(z.k_len, 128) * pairs, places, whole_heads ? z.group() : q_tiles * z.group(),
                                       whole_heads ? 1 : 2, key_part, left);
  const size_t query_part = z.q_rows() * dp * sizeof(float);
  p.query_splits = mnv_attention_parts(mnv_ceil_div((size_t)z.q_len * z.group(), 128) * pairs, places, mnv_ceil_div(z.k_len, 32),
                                       2, query_part, workspace_bytes);
  const size_t keys = p.diagonal_bytes + (p.key_splits > 1 ? p.key_splits * key_part : 0);
  const size_t queries = p.query_splits > 1 ? p.query_splits * query_part : 0;
  p.bytes = keys > queries ? keys : queries;
  return p;
}

#define MNV_AT_LAUNCH(kernel)                                                                              \
  do {                                                                                                     \
    const dim3 g(grid), b(256);                                                                            \
    const bool vec = a.z.dim % 4 == 0;                                                                     \
    if (a.bias && vec) hipLaunchKernelGGL((kernel<DP, true, true>), g, b, 0, s, a);                        \
    else if (a.bias) hipLaunchKernelGGL((kernel<DP, true, false>), g, b, 0, s, a);                         \
    else if (vec) hipLaunchKernelGGL((kernel<DP, false, true>), g, b, 0, s, a);                            \
    else hipLaunchKernelGGL((kernel<DP, false, false>), g, b, 0, s, a);                                    \
    return MNV_LAUNCH_STATUS();                                                                            \
  } while (0)
template <int DP>
int launch_dkv(const BwdArgs& a, unsigned grid, hipStream_t s) {
  MNV_AT_LAUNCH(mnv_attention_dkv_kernel);
}
template <int DP>
int launch_dq(const BwdArgs& a, unsigned grid, hipStream_t s) {
  MNV_AT_LAUNCH(mnv_attention_dq_kernel);
}
int by_dim(int dim, int (*f32)(const BwdArgs&, unsigned, hipStream_t), int (*f64)(const BwdArgs&, unsigned, hipStream_t),
           int (*f96)(const BwdArgs&, unsigned, hipStream_t), int (*f128)(const BwdArgs&, unsigned, hipStream_t),
           const BwdArgs& a, unsigned grid, hipStream_t s) {
  return (dim <= 32 ? f32 : dim <= 64 ? f64 : dim <= 96 ? f96 : f128)(a, grid, s);
}

}  // namespace

extern "C" {

size_t mnv_attention_bwd_workspace_bytes(int batch, int heads, int kv_heads, int q_len, int k_len, int head_dim,
                                         int has_bias) {
  const AttentionSizes z = {batch, heads, kv_heads, q_len, k_len, head_dim, 1.f};
  return mnv_attention_sizes_ok(z) ? make_plan(z, has_bias != 0, MNV_AT_ANY_WORKSPACE).bytes : 0;
}

int mnv_attention_bwd(const float* q, const float* k, const float* v, const float* bias, const float* lengths,
                      const float* out, const float* stats, const float* dout, float* dq, float* dk, float* dv,
                      float* dbias, int batch, int heads, int kv_heads, int q_len, int k_len, int head_dim, float scale,
                      void* workspace, size_t workspace_bytes, mnv_stream_t stream) {
  const AttentionSizes z = {batch, heads, kv_heads, q_len, k_len, head_dim, scale};
  if (!q || !k || !v || !out || !stats || !dout || !dq || !dk || !dv || (bias && !dbias) || !mnv_attention_sizes_ok(z))
    return MNV_ERR_INVALID;
  const hipStream_t s = mnv_stream(stream);
  const BwdPlan plan = make_plan(z, bias != nullptr, workspace && mnv_aligned16(workspace) ? workspace_bytes : 0);
  const int dp = mnv_attention_padded(head_dim), group = z.group();
  const size_t pairs = (size_t)batch * kv_heads, q_rows = z.q_rows(), k_rows = pairs * k_len;
  BwdArgs a = {q, k, v, bias, lengths, out, stats, dout, dq, dk, dv, nullptr, z, 0, 0, q_len * group,
               mnv_fastdiv_make(group), 1, 0, nullptr};
  hipLaunchKernelGGL(mnv_attention_delta_kernel, dim3((unsigned)mnv_ceil_div(q_rows, 16)), dim3(256), 0, s, dout, out, dq,
                     q_rows, head_dim);
  MNV_HIP_TRY(hipGetLastError());

  // keys, and with them the bias's gradient as far as the workspace holds its parts
  BwdArgs ka = a;
  ka.tiles = (int)mnv_ceil_div(k_len, 128);
  const int q_tiles = (int)mnv_ceil_div(q_len, 32), units = plan.pairs ? group : group * q_tiles;
  ka.chunk = (int)mnv_ceil_div(units, plan.key_splits) * (plan.pairs ? q_tiles : 1);
  ka.splits = plan.key_splits;
  ka.parts = plan.pairs ? static_cast<float*>(workspace) : nullptr;
  ka.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.diagonal_bytes);
  const size_t at_once = plan.pairs ? plan.pairs : pairs;
  for (size_t p = 0; p < pairs; p += at_once) {
    const unsigned now = (unsigned)(pairs - p < at_once ? pairs - p : at_once);
    ka.first_pair = (unsigned)p;
    const int rc = by_dim(head_dim, launch_dkv<32>, launch_dkv<64>, launch_dkv<96>, launch_dkv<128>, ka,
                          now * ka.tiles * ka.splits, s);
    if (rc) return rc;
    if (!ka.parts) continue;
    const dim3 grid((unsigned)mnv_ceil_div(z.offsets(), 64), heads < 65535 ? heads : 65535);
    hipLaunchKernelGGL(mnv_attention_dbias_kernel, grid, dim3(1024), 0, s, ka.parts, lengths, dbias, z, (unsigned)p, now,
                       p == 0);
    MNV_HIP_TRY(hipGetLastError());
  }
  if (ka.splits > 1) {
    hipLaunchKernelGGL(mnv_attention_sum_kernel, dim3((unsigned)mnv_ceil_div(k_rows, 16), 2), dim3(256), 0, s, ka.sums, dk, dv,
                       lengths, z, false, ka.splits, 0, dp, 1.f);
    MNV_HIP_TRY(hipGetLastError());
  }
  if (bias && !ka.parts) {
    const size_t work = z.offsets() * heads;
    hipLaunchKernelGGL(mnv_attention_dbias_alone_kernel, dim3((unsigned)(work < (1u << 20) ? work : (1u << 20))),
                       dim3(MNV_WAVE), 0, s, a, dbias);
    MNV_HIP_TRY(hipGetLastError());
  }

  a.tiles = (int)mnv_ceil_div(a.rows, 128);
  a.splits = plan.query_splits;
  a.chunk = (int)mnv_ceil_div(mnv_ceil_div(k_len, 32), a.splits);
  a.sums = static_cast<float*>(workspace);
  const int rc = by_dim(head_dim, launch_dq<32>, launch_dq<64>, launch_dq<96>, launch_dq<128>, a,
                        (unsigned)(a.tiles * a.splits * pairs), s);
  if (rc || a.splits == 1) return rc;
  hipLaunchKernelGGL(mnv_attention_sum_kernel, dim3((unsigned)mnv_ceil_div(q_rows, 16)), dim3(256), 0, s, a.sums, dq,
                     nullptr, lengths, z, true, a.splits, a.chunk * 32, dp, scale);
  return MNV_LAUNCH_STATUS();
}

}  // extern "C"
