// Large fp32 products on the fp16 matrix cores, every value as a pair of fp16 numbers.
//
// A value x of a row (of the left operand; of the right one, of a column) whose largest size is below 2^(e + 15) is x = 2^e (h + l), with
// h the fp16 number next to x 2^-e and l that next to what is left: 22 bits, |x - 2^e (h + l)| <= 2^-22 |x| down to 2^-17 of the row's
// largest, and 2^-39 of that below.  A product a b is then  ah bh + al bh + ah bl,  and al bl of at most 2^-22 |a b| is left
// out.  The instruction multiplies exactly and adds in fp32; 2^(ea + eb) is put on at the end, exactly.  That is half the matrix
// instructions of the six products of three bf16 parts (gemm_split.h), which hold all 24 bits and need no scale: a product here
// is within 3 x 2^-22 of itself, a sum's error is set by the roundings of its fp32 additions all the same.  Measured against
// float64 (2-norm, relative; normal values, k = 1024 / 4096 / 16384): 3.6e-7, 7.1e-7, 1.5e-6; six products of bf16 parts 1.9e-7, 4.0e-7,
// 8.2e-7; the fp32 instruction 5.7e-7, 1.2e-6, 2.3e-6.  Sums of the two small products kept apart from the large one's bring it to
// that of bf16 parts, but their 128 registers leave the fragments too few: 160 moves beside 192 matrix instructions, 6% of the time.  An infinity or NaN
// gives NaN in all that its row has a part in.
//
// The pairs are made once for a product, not while it multiplies (the cut takes 6 vector instructions a value, and there would be
// one for two matrix instructions): pair_pack_kernel writes them in the order in which a wavefront's lanes want them, 64 rows x 32 k
// as 4 fragments of 1 KB of h and 4 of l, fragment q with the rows 4 i + q, so that a lane's four sums are four consecutive rows.  12 bytes
// a value go through memory for it.
//
// pair_gemm_kernel: 256 x 128 tiles, four wavefronts with 128 x 64 each, one workgroup to a CU.  A step of 32 k is 48 KB, loaded straight
// to LDS, in a ring of three; the fragments of the next step are read under the 96 matrix instructions of the present one, and
// the barrier between two steps waits only for loads that were issued a step before.
// Measured: 2048 x 8192 x 11264 in 860 us, 440 TFLOP/s without the packing (236 us); 5632 x 8192 x 2048, which reads and stores 16 bytes for each
// result, 611 us (310).  What bounds it is power: the matrix cores are busy for 66% of the time at 1.9 GHz, and with nothing
// else to do they are for all of it, at 1.5.
#pragma once
#include "sgemm_core.h"

namespace {

typedef _Float16 PairHalf8 __attribute__((ext_vector_type(8)));
typedef float PairAcc __attribute__((ext_vector_type(4)));

constexpr int PAIR_M = 256, PAIR_N = 128, PAIR_K = 32, PAIR_GROUP = 64;
constexpr size_t PAIR_CHUNK = 8192;  // bytes of 64 rows x 32 k
constexpr int PAIR_PARTS = 32;       // parts of k whose largest sizes are found apart, at most

// One operand: `rows` rows (or columns) of `k`; value (r, i) at src[r * ld + i] (k_fast) or src[i * ld + r].
struct PairOperand {
  const float* src;
  size_t ld;
  int rows, k;
  bool k_fast;
  int gate;  // > 0: rows in runs of four of two matrices of so many rows in turn, as GatedIn has them; `rows` is then a multiple of 8
};
__device__ __forceinline__ int pair_source_row(int row, int gate) { return gate ? row / 8 * 4 + row % 4 + (row & 4 ? gate : 0) : row; }

// Bits of the largest size; infinities and NaN are larger than all others.
__device__ __forceinline__ unsigned pair_size(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

// What the kernels below do for one operand; both of a product's go into one launch, the right one's workgroups behind the left one's.
struct PairPacking {
  PairOperand o;
  int source_rows, parts, per_part;  // largest sizes: tops[part][source row]
  unsigned* tops;
  int blocks_k, per_wave, blocks_x;  // packing: blocks_x workgroups along k, four wavefronts with per_wave blocks of 32 k each
  char* out;
  int* exps;                         // [row]: the row's e
};
struct PairBoth {
  PairPacking p[2];
  int first;  // the right operand's first workgroup
};

// Largest sizes of source rows, k contiguous: a wavefront to a row.
__device__ __forceinline__ void pair_tops_k(const PairPacking& z, int block) {
  const int lane = threadIdx.x % MNV_WAVE, row = block * 4 + threadIdx.x / MNV_WAVE, k = z.o.k;
  if (row >= z.source_rows) return;
  const float* p = z.o.src + row * z.o.ld;
  unsigned most = 0;
  int i = lane * 4;
  for (; i + 768 + 4 <= k; i += 1024) {
    mnv_f4u v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const mnv_f4u*>(p + i + u * 256);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) most = max(most, pair_size(v[u][q]));
  }
  for (; i + 4 <= k; i += 256) {
    const mnv_f4u v = *reinterpret_cast<const mnv_f4u*>(p + i);
#pragma unroll
    for (int q = 0; q < 4; ++q) most = max(most, pair_size(v[q]));
  }
  if (i < k)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i + q < k) most = max(most, pair_size(p[i + q]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, o, MNV_WAVE));
  if (lane == 0) z.tops[row] = most;
}
// The same, rows contiguous: a lane has four of them, a workgroup's wavefronts every fourth k of a part.
__device__ __forceinline__ void pair_tops_x(const PairPacking& z, int block, unsigned (&red)[4][256]) {
  const int blocks = (z.source_rows + 255) / 256, part = block / blocks, first = (block - part * blocks) * 256;
  const int lane = threadIdx.x % MNV_WAVE, wave = threadIdx.x / MNV_WAVE, row = first + lane * 4, rows = z.source_rows;
  const int end = min(z.o.k, (part + 1) * z.per_part);
  unsigned most[4] = {0, 0, 0, 0};
  int i = part * z.per_part + wave;
  if (row + 4 <= rows) {
    for (; i + 12 < end; i += 16) {
      mnv_f4u v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const mnv_f4u*>(z.o.src + (size_t)(i + u * 4) * z.o.ld + row);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) most[q] = max(most[q], pair_size(v[u][q]));
    }
    for (; i < end; i += 4) {
      const mnv_f4u v = *reinterpret_cast<const mnv_f4u*>(z.o.src + (size_t)i * z.o.ld + row);
#pragma unroll
      for (int q = 0; q < 4; ++q) most[q] = max(most[q], pair_size(v[q]));
    }
  } else {
    for (; i < end; i += 4)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (row + q < rows) most[q] = max(most[q], pair_size(z.o.src[(size_t)i * z.o.ld + row + q]));
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) red[wave][lane * 4 + q] = most[q];
  __syncthreads();
  const int t = threadIdx.x;
  if (first + t < rows) z.tops[(size_t)part * rows + first + t] = max(max(red[0][t], red[1][t]), max(red[2][t], red[3][t]));
}
__global__ __launch_bounds__(256) void pair_tops_kernel(PairBoth both) {
  __shared__ unsigned red[4][256];
  const bool right = (int)blockIdx.x >= both.first;
  const PairPacking& z = both.p[right];
  const int block = (int)blockIdx.x - (right ? both.first : 0);
  if (z.o.k_fast) pair_tops_k(z, block);
  else pair_tops_x(z, block, red);
}

// A wavefront packs 64 rows x 32 k at a time.  The workgroup's have the same rows, whose largest sizes they find together: every lane of
// each over all parts, one load waiting for the other, took longer than the packing (5632 + 1024 rows of 4096 k 129 -> 38 us).
template <bool K_FAST>
__device__ __forceinline__ void pair_pack(const PairPacking& z, int block, unsigned (&red)[4][PAIR_GROUP]) {
  const int lane = threadIdx.x % MNV_WAVE, lr = lane % 16, lq = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / MNV_WAVE));
  const int group = block / z.blocks_x, bx = block - group * z.blocks_x, row = group * PAIR_GROUP + lr * 4;
  {
    const int r = group * PAIR_GROUP + lane, src = pair_source_row(r, z.o.gate);
    unsigned top = 0;
    if (r < z.o.rows && src < z.source_rows) {
#pragma unroll 8
      for (int p = wave; p < z.parts; p += 4) top = max(top, z.tops[(size_t)p * z.source_rows + src]);
    }
    red[wave][lane] = top;
  }
  __syncthreads();
  int e[4], src_row[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    src_row[q] = pair_source_row(row + q, z.o.gate);
    // of the rows that fill the last run of the gate's, what is read is not stored
    const bool on = row + q < z.o.rows && src_row[q] < z.source_rows;
    const unsigned top = max(max(red[0][lr * 4 + q], red[1][lr * 4 + q]), max(red[2][lr * 4 + q], red[3][lr * 4 + q]));
    // 2^e below the top by 14 powers of two; of tops below 2^-112 the smallest e that a factor holds
    const int power = (int)(top >> 23) - 127;
    e[q] = top == 0 ? 0 : max(power - 14, -126);
    if (!on) src_row[q] = -1;
    if (bx == 0 && wave == 0 && lq == 0) z.exps[row + q] = e[q];
  }
  const int first = (bx * 4 + wave) * z.per_wave;
  for (int kb = first; kb < first + z.per_wave && kb < z.blocks_k; ++kb) {
    const int k = kb * PAIR_K + lq * 8;
    float v[4][8];
    if constexpr (K_FAST) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float* p = z.o.src + (size_t)max(src_row[q], 0) * z.o.ld + k;
        if (k + 8 <= z.o.k) {
          const mnv_f4u a = *reinterpret_cast<const mnv_f4u*>(p), b = *reinterpret_cast<const mnv_f4u*>(p + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[q][i] = a[i];
            v[q][4 + i] = b[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[q][i] = k + i < z.o.k ? p[i] : 0.f;
        }
      }
    } else {
      const bool whole = src_row[0] >= 0 && src_row[3] == src_row[0] + 3;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* p = z.o.src + (size_t)min(k + i, z.o.k - 1) * z.o.ld;
        if (whole) {
          const mnv_f4u a = *reinterpret_cast<const mnv_f4u*>(p + src_row[0]);
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q][i] = a[q];
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q][i] = src_row[q] >= 0 ? p[src_row[q]] : 0.f;
        }
        if (k + i >= z.o.k)
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q][i] = 0.f;
      }
    }
    char* const at = z.out + ((size_t)group * z.blocks_k + kb) * PAIR_CHUNK + lane * 16;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      PairHalf8 h, l;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = src_row[q] >= 0 ? ldexpf(v[q][i], -e[q]) : 0.f;
        h[i] = (_Float16)x;
        l[i] = (_Float16)(x - (float)h[i]);
      }
      *reinterpret_cast<PairHalf8*>(at + q * 1024) = h;
      *reinterpret_cast<PairHalf8*>(at + 4096 + q * 1024) = l;
    }
  }
}
__global__ __launch_bounds__(256) void pair_pack_kernel(PairBoth both) {
  __shared__ unsigned red[4][PAIR_GROUP];
  const bool right = (int)blockIdx.x >= both.first;
  const PairPacking& z = both.p[right];
  const int block = (int)blockIdx.x - (right ? both.first : 0);
  if (z.o.k_fast) pair_pack<true>(z, block, red);
  else pair_pack<false>(z, block, red);
}

// A plain result of M rows.
struct PairStore {
  float* c;
  int M;
  struct Fetched {};
  __device__ Fetched c_fetch4(int, int) const { return {}; }
  __device__ void c_store4_with(int m, int n, const float (&x)[4], const Fetched&) const {
    float* p = c + (size_t)n * M + m;
    if (m + 3 < M) {
      *reinterpret_cast<mnv_f4u*>(p) = mnv_f4u{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (m + q < M) p[q] = x[q];
    }
  }
};

// A product of packed operands.  E stores four rows m .. m + 3 of column n < N (m a multiple of 4 below M): c_store4_with(m, n, x, fetched),
// with what c_fetch4(m, n) has read for them.
template <class E>
struct PairProblem {
  E e;
  const char* a;
  const char* b;
  const int* a_exp;
  const int* b_exp;
  int M, N, blocks_k, per_range;  // k blocks in all, and of a range (blockIdx.z)
  int tiles_m, tiles_n, group_m;
  float* partial;  // {M, N, ranges}, or null: stored by e
};

template <class E>
__global__ __launch_bounds__(256, 1) void pair_gemm_kernel(PairProblem<E> z) {
  constexpr int STAGE = 6 * (int)PAIR_CHUNK;
  extern __shared__ __align__(1024) char pair_lds[];
  typedef __attribute__((address_space(3))) char* Lds;
  const int lane = threadIdx.x % MNV_WAVE, lr = lane % 16, lq = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / MNV_WAVE)), wm = wave % 2, wn = wave / 2;
  // tiles in groups of group_m rows: what an XCD works on at a time is a block of tiles, not a row of them
  int t = mnv_tile_remap((int)blockIdx.x, z.tiles_m * z.tiles_n);
  const int per_group = z.group_m * z.tiles_n, g = t / per_group, gm = min(z.group_m, z.tiles_m - g * z.group_m);
  t -= g * per_group;
  const int tile_m = g * z.group_m + t % gm, tile_n = t / gm;
  const int begin = blockIdx.z * z.per_range, steps = min(z.per_range, z.blocks_k - begin);
  // chunks of 1 KB: a wavefront loads one group of A and half a group of B
  const size_t a_groups = 4, b_groups = 2;
  const mnv_rsrc ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(z.a) + (size_t)tile_m * a_groups * z.blocks_k * PAIR_CHUNK, 0,
                                                        (int)(a_groups * z.blocks_k * PAIR_CHUNK), 0x00020000);
  const mnv_rsrc rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(z.b) + (size_t)tile_n * b_groups * z.blocks_k * PAIR_CHUNK, 0,
                                                        (int)(b_groups * z.blocks_k * PAIR_CHUNK), 0x00020000);
  const int voff = lane * 16;
  const int a_first = (wave * z.blocks_k + begin) * (int)PAIR_CHUNK;
  const int b_first = (wave / 2 * z.blocks_k + begin) * (int)PAIR_CHUNK + wave % 2 * 4096;
  auto load_one = [&](int step, int i) {
    const Lds to = (Lds)pair_lds + step % 3 * STAGE;
    if (i < 8)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, to + wave * 8192 + i * 1024, 16, voff, a_first + step * (int)PAIR_CHUNK + i * 1024, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, to + 32768 + wave * 4096 + (i - 8) * 1024, 16, voff,
                                               b_first + step * (int)PAIR_CHUNK + (i - 8) * 1024, 0, 0);
  };
  auto load = [&](int step) {
#pragma unroll
    for (int i = 0; i < 12; ++i) load_one(step, i);
  };
  PairAcc acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = PairAcc{0.f, 0.f, 0.f, 0.f};
  struct Set {
    PairHalf8 a[8][2], b[4][2];
  };
  Set set[2];
  typedef const __attribute__((address_space(3))) PairHalf8* Frag;
  auto read_one = [&](int step, Set& s, int i) {
    const Lds from = (Lds)pair_lds + step % 3 * STAGE + lane * 16;
    if (i < 8) s.b[i / 2][i % 2] = *(Frag)(from + 32768 + wn * 8192 + i % 2 * 4096 + i / 2 * 1024);
    else s.a[i / 2 - 4][i % 2] = *(Frag)(from + wm * 16384 + (i / 2 - 4) / 4 * 8192 + i % 2 * 4096 + (i / 2 - 4) % 4 * 1024);
  };
  auto read = [&](int step, Set& s) {
#pragma unroll
    for (int i = 0; i < 24; ++i) read_one(step, s, i);
  };
  // instruction t of 96
  auto multiply_one = [&](const Set& s, int t) {
    const int i = t / 12, part = t % 12 / 4, j = t % 4;
    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(s.b[j][part == 0], s.a[i][part == 1], acc[i][j], 0, 0, 0);
  };
  auto multiply = [&](const Set& s) {
#pragma unroll
    for (int t = 0; t < 96; ++t) multiply_one(s, t);
  };
  // The loads of `ahead` steps may still be on their way; the others' wavefronts' are as far.
  auto meet = [&](auto AHEAD) {
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (decltype(AHEAD)::value == 2) asm volatile("s_waitcnt vmcnt(24) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else if constexpr (decltype(AHEAD)::value == 1) asm volatile("s_waitcnt vmcnt(12) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  typedef std::integral_constant<int, 0> None;
  typedef std::integral_constant<int, 1> One;
  if (steps > 0) load(0);
  if (steps > 1) load(1);
  if (steps > 2) load(2);
  if (steps > 2) meet(std::integral_constant<int, 2>{});
  else if (steps > 1) meet(One{});
  else meet(None{});
  if (steps > 0) read(0, set[0]);
  // Step 0 is in registers, 1 in LDS, 2 on its way.
  if (steps > 2) meet(One{});
  else meet(None{});
  // A step with everything behind it: a ring place is loaded anew and the next step's fragments are read, a load and two
  // reads for every eight matrix instructions.
  auto full = [&](int step, const Set& now, Set& next) {
#pragma unroll
    for (int c = 0; c < 12; ++c) {
      load_one(step + 3, c);
      read_one(step + 1, next, 2 * c);
      read_one(step + 1, next, 2 * c + 1);
#pragma unroll
      for (int t = 0; t < 8; ++t) multiply_one(now, 8 * c + t);
      __builtin_amdgcn_sched_barrier(0);
    }
    meet(One{});
  };
  auto last = [&](int step, const Set& now, Set& next) {
    if (step + 3 < steps) load(step + 3);
    if (step + 1 < steps) read(step + 1, next);
    multiply(now);
    meet(None{});
  };
  int step = 0;
#pragma unroll 1
  for (; step + 4 < steps; step += 2) {
    full(step, set[0], set[1]);
    full(step + 1, set[1], set[0]);
  }
#pragma unroll 1
  for (; step < steps; step += 2) {
    last(step, set[0], set[1]);
    if (step + 1 < steps) last(step + 1, set[1], set[0]);
  }

  const int m0 = tile_m * PAIR_M + wm * 128 + lr * 4, n0 = tile_n * PAIR_N + wn * 64 + lq * 16;
  int em[8], en[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) em[i] = z.a_exp[m0 + i / 4 * 64 + i % 4];
#pragma unroll
  for (int i = 0; i < 16; ++i) en[i] = z.b_exp[n0 + i];
  // The sums pass through the wavefront's own 32 KB of LDS, so that their store is one piece of code and not 32: a lane reads what it wrote.
  typedef __attribute__((address_space(3))) mnv_f4* Sums;
  const Sums mine = (Sums)((Lds)pair_lds + wave * 32768 + lane * 16);
#pragma unroll
  for (int gi = 0; gi < 2; ++gi)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mnv_f4 x;
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = ldexpf(acc[gi * 4 + q][j][r], em[gi * 4 + q] + en[4 * r + j]);
        mine[((gi * 4 + r) * 4 + j) * MNV_WAVE] = x;
      }
  constexpr int U = 8;  // whose reads are under way together
#pragma unroll 1
  for (int t = 0; t < 32; t += U) {
    const int m = m0 + t / 16 * 64, nt = n0 + t % 16;
    if (m >= z.M) continue;
    if (z.partial) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (nt + u >= z.N) break;
        const mnv_f4 sums = mine[(t + u) * MNV_WAVE];
        PairStore{z.partial + (size_t)blockIdx.z * z.N * z.M, z.M}.c_store4_with(m, nt + u, {sums[0], sums[1], sums[2], sums[3]}, {});
      }
      continue;
    }
    typename E::Fetched f[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (nt + u < z.N) f[u] = z.e.c_fetch4(m, nt + u);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (nt + u >= z.N) break;
      const mnv_f4 sums = mine[(t + u) * MNV_WAVE];
      z.e.c_store4_with(m, nt + u, {sums[0], sums[1], sums[2], sums[3]}, f[u]);
    }
  }
}

// How a product runs in pairs, by its extents.
struct PairPlan {
  int tiles_m, tiles_n, blocks_k, ranges, per_range;
  double us;  // with the packing
  size_t a_bytes, b_bytes, exps, tops_a, tops_b, partial;  // of the workspace, in this order
  size_t bytes() const { return a_bytes + b_bytes + exps + tops_a + tops_b + partial; }
};
inline size_t pair_round(size_t n) { return (n + 255) / 256 * 256; }
inline int pair_source_rows(const PairOperand& o) { return o.gate ? 2 * o.gate : o.rows; }
// Parts for two workgroups on a CU, of 32 k or more.
inline int pair_parts(const PairOperand& o) {
  if (o.k_fast) return 1;
  const int blocks = (pair_source_rows(o) + 255) / 256;
  int parts = 512 / blocks;
  if (parts > PAIR_PARTS) parts = PAIR_PARTS;
  if (parts > o.k / 32) parts = o.k / 32;
  return parts < 1 ? 1 : parts;
}
// most_ranges: 1 where the store wants whole sums.  store_bytes: what the store moves for a value.  Microseconds: 1.17 a step of 32 k and 10
// around a tile on each CU (no other workgroup multiplies meanwhile, so that the store's bytes count in full), 12 bytes a value of either
// operand to pack and 12 for its two launches, 8 bytes a value and range for k ranges, all bytes at 5 TB/s.
PairPlan pair_plan(const PairOperand& a, const PairOperand& b, int most_ranges, double store_bytes, int cus) {
  PairPlan p;
  p.tiles_m = (a.rows + PAIR_M - 1) / PAIR_M;
  p.tiles_n = (b.rows + PAIR_N - 1) / PAIR_N;
  p.blocks_k = (a.k + PAIR_K - 1) / PAIR_K;
  const long long tiles = (long long)p.tiles_m * p.tiles_n;
  p.ranges = 1;
  double best = 1e30;
  for (int z = 1; z <= most_ranges && (z == 1 || p.blocks_k / z >= 8); ++z) {
    const int per = (p.blocks_k + z - 1) / z;
    const double us = (double)((tiles * z + cus - 1) / cus) * (1.17 * per + 10.0) + (z > 1 ? 4.0 + 8e-6 / 5.0 * a.rows * b.rows * z : 0.0);
    if (us < 0.97 * best) {
      best = us;
      p.ranges = z;
      p.per_range = per;
    }
  }
  p.ranges = (p.blocks_k + p.per_range - 1) / p.per_range;
  p.us = best + store_bytes * 1e-6 / 5.0 * a.rows * b.rows + 12.0 + 12e-6 / 5.0 * ((double)a.rows + b.rows) * a.k;
  p.a_bytes = (size_t)p.tiles_m * 4 * p.blocks_k * PAIR_CHUNK;
  p.b_bytes = (size_t)p.tiles_n * 2 * p.blocks_k * PAIR_CHUNK;
  p.exps = pair_round(((size_t)p.tiles_m * PAIR_M + (size_t)p.tiles_n * PAIR_N) * sizeof(int));
  p.tops_a = pair_round((size_t)pair_source_rows(a) * pair_parts(a) * sizeof(unsigned));
  p.tops_b = pair_round((size_t)pair_source_rows(b) * pair_parts(b) * sizeof(unsigned));
  p.partial = p.ranges > 1 ? pair_round((size_t)p.ranges * a.rows * b.rows * sizeof(float)) : 0;
  return p;
}
// Extents that the kernels' grids and offsets reach.
inline bool pair_fits(const PairOperand& a, const PairOperand& b) {
  return a.k < (1 << 20) && a.rows < (1 << 21) && b.rows < (1 << 21);
}

PairPacking pair_packing(const PairOperand& o, int blocks_k, unsigned* tops, char* out, int* exps) {
  const int parts = pair_parts(o), groups = (o.rows + PAIR_GROUP - 1) / PAIR_GROUP;
  long long per_wave = (long long)blocks_k * groups / (4 * 2048);  // 2048 workgroups where there is that much
  if (per_wave < 1) per_wave = 1;
  return {o, pair_source_rows(o), parts, (o.k + parts - 1) / parts, tops, blocks_k, (int)per_wave, (int)((blocks_k + 4 * per_wave - 1) / (4 * per_wave)),
          out, exps};
}
inline int pair_tops_blocks(const PairPacking& z) { return z.o.k_fast ? (z.source_rows + 3) / 4 : (z.source_rows + 255) / 256 * z.parts; }
inline int pair_pack_blocks(const PairPacking& z) { return (z.o.rows + PAIR_GROUP - 1) / PAIR_GROUP * z.blocks_x; }

// c = a b, stored by e, or with k ranges by `reduced`, a policy of the products.  The workspace holds plan.bytes(), aligned to 16 bytes.
template <class E, class R>
int pair_product(const PairPlan& p, const PairOperand& a, const PairOperand& b, const E& e, const R& reduced, char* ws, hipStream_t s) {
  char* const pa = ws;
  char* const pb = pa + p.a_bytes;
  int* const ea = reinterpret_cast<int*>(pb + p.b_bytes);
  int* const eb = ea + (size_t)p.tiles_m * PAIR_M;
  unsigned* const ta = reinterpret_cast<unsigned*>(pb + p.b_bytes + p.exps);
  unsigned* const tb = reinterpret_cast<unsigned*>(pb + p.b_bytes + p.exps + p.tops_a);
  float* const partial = p.ranges > 1 ? reinterpret_cast<float*>(pb + p.b_bytes + p.exps + p.tops_a + p.tops_b) : nullptr;
  PairBoth both{{pair_packing(a, p.blocks_k, ta, pa, ea), pair_packing(b, p.blocks_k, tb, pb, eb)}, 0};
  both.first = pair_tops_blocks(both.p[0]);
  hipLaunchKernelGGL(pair_tops_kernel, dim3(both.first + pair_tops_blocks(both.p[1])), dim3(256), 0, s, both);
  int rc = MNV_LAUNCH_STATUS();
  if (rc) return rc;
  both.first = pair_pack_blocks(both.p[0]);
  hipLaunchKernelGGL(pair_pack_kernel, dim3(both.first + pair_pack_blocks(both.p[1])), dim3(256), 0, s, both);
  rc = MNV_LAUNCH_STATUS();
  if (rc) return rc;
  constexpr int LDS = 3 * 6 * (int)PAIR_CHUNK;
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  MNV_HIP_TRY(hipGetDevice(&dev));
  if (dev < 0 || dev >= 64) return MNV_ERR_INVALID;
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    MNV_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(&pair_gemm_kernel<E>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    attr_set[dev].store(true, std::memory_order_release);
  }
  PairProblem<E> z{e, pa, pb, ea, eb, a.rows, b.rows, p.blocks_k, p.per_range, p.tiles_m, p.tiles_n, 4, partial};
  hipLaunchKernelGGL(pair_gemm_kernel<E>, dim3(p.tiles_m * p.tiles_n, 1, p.ranges), dim3(256), LDS, s, z);
  rc = MNV_LAUNCH_STATUS();
  if (rc || p.ranges == 1) return rc;
  return mnv_gemm_reduce_launch(reduced, partial, p.ranges, s);
}

}  // namespace
