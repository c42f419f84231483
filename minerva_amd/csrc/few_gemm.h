// Products of a large matrix with few columns: bound by reading the matrix.
#pragma once
#include <algorithm>

#include "sgemm_core.h"

namespace {

constexpr int FEW_ROWS = 64, FEW_K = 16, FEW_WAVES = 8;

// C = A B, B {K, N} with its columns contiguous, A with its rows (x-fast) or its k contiguous, through a policy's A, B, M, N, K, lda, ldb
// (floats), a_row and c_store4.  A workgroup has 64 rows, 16 COLS columns and a k range; its eight wavefronts take every eighth step of
// 16 k, and their sums are added through LDS in order.  Lane (i, h) = (lane % 16, lane / 16) fetches rows 4 i .. 4 i + 3 at k = 4 h + j
// for j of 4, or k = 4 h .. 4 h + 3 of each of these rows, and k = 4 h .. 4 h + 3 of column i.  Value j of k is then what the fp32
// instruction wants of the lane for k = {j, 4 + j, 8 + j, 12 + j}, in either order, so that the operands go from memory to the instruction without
// LDS, a fetch of an x-fast A brings 256 bytes of a column together, and a lane's sums are four neighbouring rows.
// Two workgroups fit on a CU with up to 128 registers a lane: sums, and the fetches of 4, 3 or 2 steps, which are in flight under the
// steps before (with three steps' and 141 registers for 32 columns, and so one workgroup: 2 x 5632 x 2048 for 150 columns 88 -> 103 us).
// Measured as the projections of a gated block, 2 x 5632 rows, 2048 k, with the weights read from HBM (four of them in turn, 369 MB), this
// kernel and the SGEMM's small tiles, which leave the gate to another 3 us: 13 / 16 / 32 / 48 / 64 columns 26 / 27 / 35 / 40 / 53 us (up to 16 in k
// ranges, and 5 to add and gate them) and 37 / 38 / 35 / 40 / 47; 92 MB, i.e. 3.5 TB/s up to 16 columns.  From 32 on the matrix instruction, at 0.7 of its rate,
// and how the workgroups divide on the CUs bound it.
template <class P, int COLS>
__global__ __launch_bounds__(FEW_WAVES * MNV_WAVE, 4) void few_gemm_kernel(P prob, int blocks_m, int blocks_n, int ranges, int per_range,
                                                                              float* __restrict__ partial) {
  typedef float Acc __attribute__((ext_vector_type(4)));
  constexpr int AHEAD = 5 - COLS, AT_ONCE = COLS < 2 ? COLS : 2;
  extern __shared__ __align__(16) float few_sums[];  // [wavefront][column][row]
  // an XCD has a run of these: the column blocks of the same rows next to each other, then neighbouring rows, which share lines where a
  // column is no multiple of them (dealt out one by one, 33 columns, forward, 3001 -> 9001 138 -> 132 us, 5 columns 112 -> 93), then the ranges
  const int id = mnv_tile_remap((int)blockIdx.x, (int)gridDim.x), block_n = id % blocks_n, block_m = id / blocks_n % blocks_m;
  const int range = id / (blocks_n * blocks_m);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / MNV_WAVE)), lane = threadIdx.x % MNV_WAVE, i = lane % 16, h = lane / 16;
  const int m0 = block_m * FEW_ROWS, n0 = block_n * COLS * 16;
  const int steps = (prob.K + FEW_K - 1) / FEW_K, first = range * per_range + wave, end = min(steps, (range + 1) * per_range);
  typename P::Res res;
  prob.make_res(res);
  const unsigned lda = (unsigned)prob.lda * 4u, ldb = (unsigned)prob.ldb * 4u;
  unsigned a_off[4], b_off[COLS];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = m0 + 4 * i + (P::A_KFAST ? j : 0);
    a_off[j] = m >= prob.M ? MNV_OOB : P::A_KFAST ? (unsigned)m * lda + (unsigned)h * 16u : (unsigned)prob.a_row(m) * 4u + (unsigned)(4 * h + j) * lda;
  }
#pragma unroll
  for (int t = 0; t < COLS; ++t) {
    const int n = n0 + 16 * t + i;
    b_off[t] = n < prob.N ? (unsigned)n * ldb + (unsigned)h * 16u : MNV_OOB;
  }
  float a[AHEAD][4][4], b[AHEAD][COLS][4];
  auto load = [&](int step, int u) {
    const int left = prob.K - step * FEW_K - 4 * h;  // of k from the lane's first on
    const bool on = step < end && left > 0;
    const unsigned from = step < end ? (unsigned)step * FEW_K : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned o[1] = {(P::A_KFAST ? on : on && j < left) ? a_off[j] : MNV_OOB};
      mnv_fetch_vec<1>(res.a, o, P::A_KFAST ? from * 4u : from * lda, a[u][j]);
    }
#pragma unroll
    for (int t = 0; t < COLS; ++t) {
      const unsigned o[1] = {on ? b_off[t] : MNV_OOB};
      mnv_fetch_vec<1>(res.b, o, from * 4u, b[u][t]);
    }
  };
  Acc acc[4][COLS];
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int t = 0; t < COLS; ++t) acc[q][t] = 0.f;
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) load(first + u * FEW_WAVES, u);
#pragma unroll 1
  for (int s = first; s < end; s += AHEAD * FEW_WAVES) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int step = s + u * FEW_WAVES;
      if (step >= end) break;
      if ((step + 1) * FEW_K > prob.K) {  // a vector along k may reach past it
#pragma unroll
        for (int e = 1; e < 4; ++e) {
          const bool on = step * FEW_K + 4 * h + e < prob.K;
#pragma unroll
          for (int t = 0; t < COLS; ++t) b[u][t][e] = on ? b[u][t][e] : 0.f;
          if (P::A_KFAST) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[u][j][e] = on ? a[u][j][e] : 0.f;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int t = 0; t < COLS; ++t)
            acc[q][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[u][t][j], P::A_KFAST ? a[u][q][j] : a[u][j][q], acc[q][t], 0, 0, 0);
      load(step + AHEAD * FEW_WAVES, u);
    }
  }
  // Sum r of lane (i, h): column 4 h + r of 16, row 4 i + q.  At most 32 columns at once through LDS.
#pragma unroll
  for (int t0 = 0; t0 < COLS; t0 += AT_ONCE) {
    constexpr int REGION = AT_ONCE * 16 * FEW_ROWS;
    if (t0) __syncthreads();
#pragma unroll
    for (int t = t0; t < t0 + AT_ONCE && t < COLS; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<mnv_f4*>(few_sums + wave * REGION + ((t - t0) * 16 + 4 * h + r) * FEW_ROWS + 4 * i) =
            mnv_f4{acc[0][t][r], acc[1][t][r], acc[2][t][r], acc[3][t][r]};
    __syncthreads();
    const int e = threadIdx.x, m = m0 + e % 16 * 4, n = n0 + t0 * 16 + e / 16;
    if (e / 16 >= 16 * (COLS - t0) || e * 4 >= REGION || m >= prob.M || n >= prob.N) continue;
    mnv_f4 x = *reinterpret_cast<const mnv_f4*>(few_sums + e * 4);
#pragma unroll
    for (int w = 1; w < FEW_WAVES; ++w) x += *reinterpret_cast<const mnv_f4*>(few_sums + w * REGION + e * 4);
    const float v[4] = {x[0], x[1], x[2], x[3]};
    if (ranges == 1) {
      prob.c_store4(m, n, v);
    } else {
      float* const p = partial + ((size_t)range * prob.N + n) * prob.M + m;
      if (m + 3 < prob.M) {
        *reinterpret_cast<mnv_f4u*>(p) = mnv_f4u{x[0], x[1], x[2], x[3]};
      } else {
#pragma unroll
        for (int q = 0; q < 3; ++q)
          if (m + q < prob.M) p[q] = v[q];
      }
    }
  }
}

struct FewPlan {
  int cols = 0;  // times 16 columns to a workgroup, 1 to 3; 0: another kernel
  int ranges = 1;
  size_t bytes(int m, int n) const { return ranges > 1 ? (size_t)ranges * m * n * sizeof(float) : 0; }
};

// The plan of an m x n x k product with A's k contiguous or not, or none (cols 0).  Against the SGEMM's plans on 180 products (12 shapes of
// 64 -> 172 up to 4096 -> 14000, 1 to 220 columns) and a block's passes of 10 more, even and odd: it gains from 5 columns on, where A
// has `least` values (for less, other tiles cover the chip sooner), up to 64 columns, or 160 of a matrix of up to 9 million values, whose tiles
// of the SGEMM are too few for the chip; up to 48 of one with k contiguous or from 64 million values on, where the matrix instruction
// bounds it (4096 x 8192 at 64 columns 49 / 57).  Not where the SGEMM's reads of up to 12 columns are as quick: below 9 columns from 16 million
// values on (5 columns, forward, 3001 -> 9001 72 / 78 us), below 13 of k contiguous from 64 million on (4096 x 28000 87 / 100); nor
// for more than 32 columns from 20 million values on in rows off the 128-byte grid, where 256 bytes take a third line (33 columns, forward,
// 4095 -> 4097 72 / 89 us, 4096 -> 4096 76 / 60).
// So many ranges that the workgroups are just one to a CU, of at least 128 k: 1.02 times the best number's time; two and a half for up to
// 16 columns of rows contiguous from 8 million values on, where the fetches of one are too few for HBM (16 columns, forward, 3000 -> 9000 97 -> 83 us).
FewPlan plan_few(int m, int n, int k, bool k_fast, double least, size_t ws_bytes) {
  const double values = (double)m * k;
  const bool large = values >= 64e6, cut = !k_fast && values >= 20e6 && m % 32;
  const int from = k_fast ? (large ? 13 : 5) : values >= 16e6 ? 9 : 5;
  const int most = cut ? 32 : k_fast || large ? 48 : values <= 9e6 ? 160 : 64;
  FewPlan plan;
  if (values < least || n < from || n > most) return plan;
  plan.cols = n <= 16 ? 1 : n <= 32 ? 2 : n <= 48 ? 3 : n <= 64 ? 2 : (n + 47) / 48 * 3 <= (n + 31) / 32 * 2 ? 3 : 2;
  const int blocks = (m + FEW_ROWS - 1) / FEW_ROWS * ((n + plan.cols * 16 - 1) / (plan.cols * 16)), cus = mnv_cu_count();
  const int workgroups = !k_fast && n <= 16 && values >= 8e6 ? cus * 5 / 2 : cus;
  plan.ranges = std::max(1, std::min(std::min(16, k / 128), workgroups / blocks));
  while (plan.bytes(m, n) > ws_bytes) --plan.ranges;
  return plan;
}

template <class P, int COLS>
int launch_few_cols(const FewPlan& plan, const P& p, float* partial, hipStream_t s) {
  const int blocks_m = (p.M + FEW_ROWS - 1) / FEW_ROWS, blocks_n = (p.N + COLS * 16 - 1) / (COLS * 16);
  const int steps = (p.K + FEW_K - 1) / FEW_K, per = (steps + plan.ranges - 1) / plan.ranges;
  const int lds = FEW_WAVES * (COLS < 2 ? COLS : 2) * 16 * FEW_ROWS * (int)sizeof(float);
  hipLaunchKernelGGL((few_gemm_kernel<P, COLS>), dim3((unsigned)blocks_m * blocks_n * plan.ranges), dim3(FEW_WAVES * MNV_WAVE), lds, s, p, blocks_m,
                     blocks_n, plan.ranges, per, partial);
  return MNV_LAUNCH_STATUS();
}
// The k ranges of a plan with more than one are left in `partial`, range by range as {M, N}.
template <class P>
int launch_few(const FewPlan& plan, const P& p, float* partial, hipStream_t s) {
  return plan.cols == 1 ? launch_few_cols<P, 1>(plan, p, partial, s)
         : plan.cols == 2 ? launch_few_cols<P, 2>(plan, p, partial, s)
                          : launch_few_cols<P, 3>(plan, p, partial, s);
}

}  // namespace
