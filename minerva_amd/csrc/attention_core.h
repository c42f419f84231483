// What the attention kernels share: sizes, tiles of a sequence in LDS, and products of them on the matrix cores.
//
// Every product is one of a tile of 32 rows that streams through LDS (two matrices, fetched and cut by the whole
// workgroup, two tiles in turn, so that one is cut while the other is multiplied) and an operand that a
// wavefront holds in registers for its own 32 columns: 32 queries in the forward pass and for dq, 32 keys for dk
// and dv.  fp32 values are cut into three bf16 parts and six of the nine part products are summed
// (gemm_split.h): the bf16 matrix instruction at 6 products per value has 2.6 times the fp32 one's rate.
//
// The 32 x 32 x 16 instruction gives lane l the column l % 32 and the rows 8 (r / 4) + 4 (l / 32) + r % 4 of
// the result, r = 0..15.  As an operand, lane l holds the 8 contraction places 8 (l / 32)... of column (or
// row) l % 32.  Which rows stand in which contraction places is free as long as both operands agree, so a
// result (scores, weights) becomes the next product's operand without leaving its lane: places 8 h + e
// of step s hold the rows 16 s + 4 h + e (e < 4) and 16 s + 4 h + 8 + e - 4, and the other operand, the tile by
// columns, is read in that order: the transposing LDS read gives each of 16 lanes four rows of its column.
// So the softmax's sums run over a lane's own registers and one exchange between the two half wavefronts.
#pragma once
#include <math.h>

#include "gemm_split.h"

#define MNV_AT_MAX_DIM 128
#define MNV_AT_MAX_PITCH (1 << 24)  // heads * dim: 64 rows of it are less than 2^32 bytes
// Rows of queries or keys, and pairs of an entry and a head: every launch has fewer than 2^32 threads (a launch's
// limit), and no number of a row rounded up to tiles and parts passes 2^31.
#define MNV_AT_MAX_ROWS (1 << 26)
#define MNV_AT_MAX_PAIRS (1 << 22)

struct AttentionSizes {
  int batch, heads, kv_heads, q_len, k_len, dim;
  float scale;
  __host__ __device__ int group() const { return heads / kv_heads; }
  __host__ __device__ size_t offsets() const { return (size_t)q_len + k_len - 1; }
  __host__ __device__ size_t q_rows() const { return (size_t)batch * q_len * heads; }
};

static inline bool mnv_attention_sizes_ok(const AttentionSizes& z) {
  if (z.batch < 1 || z.heads < 1 || z.kv_heads < 1 || z.q_len < 1 || z.k_len < 1 || z.dim < 1) return false;
  if (z.dim > MNV_AT_MAX_DIM || z.heads % z.kv_heads || z.heads > MNV_AT_MAX_PITCH / z.dim) return false;
  const long long most = 0x7fffffffLL, rows = MNV_AT_MAX_ROWS < most / z.dim ? MNV_AT_MAX_ROWS : most / z.dim;
  if ((long long)z.batch * z.heads > MNV_AT_MAX_PAIRS || (long long)z.batch * z.heads * z.q_len > rows) return false;
  if ((long long)z.batch * z.kv_heads * z.k_len > rows) return false;
  return ((long long)z.q_len + z.k_len - 1) * z.heads <= most && fabsf(z.scale) <= 3e38f;
}

// Columns that the kernels' products have.
static inline int mnv_attention_padded(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : dim <= 96 ? 96 : 128; }

// Parts that a workgroup's loop over `tiles` tiles is cut into where `blocks` workgroups leave places of the chip
// empty: as many as fill them, with `least` tiles or more to a part, and no more than the workspace holds.
static inline int mnv_attention_parts(size_t blocks, size_t places, size_t tiles, size_t least, size_t part_bytes,
                                      size_t workspace_bytes) {
  size_t parts = blocks ? places / blocks : 1;
  if (parts > tiles / least) parts = tiles / least;
  if (parts > MNV_WAVE) parts = MNV_WAVE;
  if (parts > workspace_bytes / part_bytes) parts = workspace_bytes / part_bytes;
  if (parts < 2) return 1;
  const size_t each = mnv_ceil_div(tiles, parts);
  return (int)mnv_ceil_div(tiles, each);
}
#define MNV_AT_ANY_WORKSPACE ((size_t)-1)  // for the queries

#ifdef __HIPCC__
#define MNV_LOG2E 1.4426950408889634f

typedef float mnv_f16 __attribute__((ext_vector_type(16)));
typedef float mnv_f2 __attribute__((ext_vector_type(2)));

// A value that is the same in all lanes, in a scalar register: so are the addresses made from it.
__device__ __forceinline__ int mnv_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// In a branch that few tiles take: without it, its selections run for all.
#define MNV_KEEP_BRANCH() asm volatile("")

// Keys of entry b that are read.
__device__ __forceinline__ int mnv_visible(const float* lengths, int b, int k_len) {
  if (!lengths) return k_len;
  const float n = lengths[b];
  if (!(n > 0.f)) return 0;
  if (n >= (float)MNV_AT_MAX_ROWS) return k_len;
  // compared as whole numbers: k_len past 2^24 need not be one that fp32 holds
  return (int)n < k_len ? (int)n : k_len;
}

// The workgroup's place.  Workgroups go to the 8 dies in turn: all of one entry and key head go to one die, whose
// L2 then holds the keys they share, and neighbouring heads to different ones, so that entries of different lengths
// load all dies alike.  `keys`: of a pair's `tiles` workgroups the first `each` have to do with its first `keys` keys, and so
// on, and those without keys go behind all others of the die; 0: in the pairs' order.  They end at once, but in between
// they take their turns in the order in which CUs are given a second workgroup, while others have none (dk and dv and the rest of
// the backward pass of 8 x 12 heads of 512 x 512, lengths 64 to 512, where 240 of 384 workgroups have keys: 131 us, 151
// in the pairs' order; 16 x 16 heads of 1024 x 1024, 64 to 1024: 707 and 744; 128 wide, one workgroup to a CU: 482 and 454).
struct MnvAttentionPlace {
  int tile, b, kh;
  unsigned pair;  // entry and key head, from the launch's first on
  int n;          // keys of the entry
};
__device__ __forceinline__ MnvAttentionPlace mnv_attention_place(unsigned tiles, unsigned each, int keys, unsigned first_pair,
                                                                 const AttentionSizes& z, const float* lengths) {
  MnvAttentionPlace p;
  const unsigned rows = gridDim.x / tiles / 8;  // pairs of each die, but for the last few
  if (blockIdx.x < rows * 8 * tiles) {
    unsigned at = blockIdx.x / 8, row = at / tiles;
    at -= row * tiles;
    if (keys && lengths && rows > 1 && rows <= MNV_WAVE) {
      const unsigned lane = threadIdx.x % MNV_WAVE;
      unsigned mine = 0;  // workgroups of the lane's pair that have keys
      if (lane < rows) {
        const int n = mnv_visible(lengths, (first_pair + lane * 8 + blockIdx.x % 8) / z.kv_heads, z.k_len);
        const unsigned steps = ((unsigned)n + keys - 1) / keys;
        mine = steps < tiles / each ? steps * each : tiles;
      }
      unsigned before = mine;  // of the pairs up to the lane's
#pragma unroll
      for (int o = 1; o < MNV_WAVE; o <<= 1) {
        const unsigned t = __shfl_up(before, o, MNV_WAVE);
        if (lane >= (unsigned)o) before += t;
      }
      const unsigned all = __shfl(before, MNV_WAVE - 1, MNV_WAVE);
      unsigned index = blockIdx.x / 8;
      const bool none = index >= all;  // one of those without keys
      if (none) {
        index -= all;
        before = (lane + 1) * tiles - before;
        mine = tiles - mine;
      }
      const unsigned long long reached = __ballot(lane < rows && before > index);
      row = __ffsll(reached) - 1;
      const unsigned in = __shfl(mine, row, MNV_WAVE);
      at = index - (__shfl(before, row, MNV_WAVE) - in);
      if (none) at += tiles - in;  // behind those with keys
    }
    p.pair = mnv_uniform(row) * 8 + blockIdx.x % 8;
    p.tile = mnv_uniform(at);
  } else {
    p.pair = mnv_uniform(blockIdx.x / tiles);
    p.tile = blockIdx.x - p.pair * tiles;
  }
  const unsigned pair = first_pair + p.pair;
  p.b = mnv_uniform(pair / z.kv_heads);
  p.kh = pair - p.b * z.kv_heads;
  p.n = mnv_uniform(mnv_visible(lengths, p.b, z.k_len));
  return p;
}

// exp(t - m), and 0 for a hidden t = -inf where hidden ones alone leave m at -inf too (m: see mnv_finite_max).
// The difference is taken before the factor: at the type's lowest value t * log2(e) would be infinite.
__device__ __forceinline__ float mnv_weight(float t, float m) { return __builtin_amdgcn_exp2f((t - m) * MNV_LOG2E); }
__device__ __forceinline__ float mnv_finite_max(float m) { return m == -INFINITY ? 0.f : m; }
// The larger of a value and that of the lane 32 away.
__device__ __forceinline__ float mnv_max_of_halves(float x) {
  unsigned u = __builtin_bit_cast(unsigned, x), w = u;
  asm volatile("" : "+v"(w));  // of equal operands the compiler takes both results for the same
  const auto r = __builtin_amdgcn_permlane32_swap(u, w, false, false);
  unsigned low = r[0], high = r[1];
  return fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
}
// 1 / l, and 0 for a row that sees no key
__device__ __forceinline__ float mnv_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// mnv_split_pair without a factor, its halves taken by byte permutations: those the compiler does not see through (it
// would convert each half again), and no wait is put behind them as behind its empty asm.
// LIMITED: finite values from 2^128 (1 - 2^-9) on would be rounded up to an infinity: the first part stays below, the second takes
// the rest.  An infinity or a NaN makes the second or third part a NaN.  Weights, at most about 1, and their
// gradients, which have to leave room for sums anyway, do without (two more of 13 instructions to a pair; backward of 2 x 16 heads of
// 2048 x 4096, 128 wide: 2166 us without any, 2179 so, 2200 with the gradients' too).
#define MNV_LARGEST_BF16 3.3895313892515355e38f
template <bool LIMITED>
__device__ __forceinline__ void mnv_cut_pair(float x, float y, unsigned (&p)[3]) {
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    const bool limited = LIMITED && c == 0;
    const float x0 = limited ? __builtin_amdgcn_fmed3f(x, -MNV_LARGEST_BF16, MNV_LARGEST_BF16) : x;
    const float y0 = limited ? __builtin_amdgcn_fmed3f(y, -MNV_LARGEST_BF16, MNV_LARGEST_BF16) : y;
    const mnv_bf2 t = {(__bf16)x0, (__bf16)y0};
    p[c] = __builtin_bit_cast(unsigned, t);
    x -= __builtin_bit_cast(float, __builtin_amdgcn_perm(p[c], p[c], 0x05040c0cu));
    y -= __builtin_bit_cast(float, __builtin_amdgcn_perm(p[c], p[c], 0x07060c0cu));
  }
}

// Eight values of one operand as three parts.
struct MnvParts {
  mnv_bf8 p[3];
};
__device__ __forceinline__ MnvParts mnv_cut8(const float* x) {
  mnv_u4 u[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned t[3];
    mnv_cut_pair<true>(x[2 * i], x[2 * i + 1], t);
    u[0][i] = t[0];
    u[1][i] = t[1];
    u[2][i] = t[2];
  }
  MnvParts r;
#pragma unroll
  for (int c = 0; c < 3; ++c) r.p[c] = __builtin_bit_cast(mnv_bf8, u[c]);
  return r;
}

// The order of instructions.  A 32 x 32 x 16 instruction holds its matrix core for 32 cycles and the issue for 8,
// so what else a wavefront has to do (exponentials, cutting) is free if it stands between them, six vector
// instructions to one; left alone, the compiler puts all matrix instructions of a product in a row and reads
// each operand right before its use.  So a tile's work is written as steps of one operand, six matrix instructions,
// each of which reads the next step's parts as its own are done with and takes a share of the other work.
//
// acc += a * b; a becomes the next step's operand, part c of which is next(c).  The smallest terms come first as far as
// the parts' turns allow: the third part is read five matrix instructions before its use, the second four, the first three.
template <bool LAST, class Next>
__device__ __forceinline__ void mnv_step(mnv_f16& acc, MnvParts& a, const MnvParts& b, Next&& next) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], acc, 0, 0, 0);
  if (!LAST) a.p[2] = next(2);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], acc, 0, 0, 0);
  if (!LAST) a.p[1] = next(1);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], acc, 0, 0, 0);
  if (!LAST) a.p[0] = next(0);
}
// Closes a step: others: vector instructions to a matrix instruction.
#define MNV_STEP_ORDER(others)                                 \
  do {                                                         \
    _Pragma("unroll") for (int g_ = 0; g_ < 6; ++g_) {         \
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);       \
      if (g_ == 0 || g_ == 2 || g_ == 5) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0); \
      __builtin_amdgcn_sched_group_barrier(0x002, others, 0);  \
    }                                                          \
    __builtin_amdgcn_sched_barrier(0);                         \
  } while (0)

// Eight values as an operand, cut pair by pair.
struct MnvCutting {
  mnv_u4 u[3];
  __device__ __forceinline__ void pair(int i, float x, float y) {
    unsigned t[3];
    mnv_cut_pair<false>(x, y, t);
    u[0][i] = t[0];
    u[1][i] = t[1];
    u[2][i] = t[2];
  }
  __device__ __forceinline__ MnvParts parts() const {
    return {{__builtin_bit_cast(mnv_bf8, u[0]), __builtin_bit_cast(mnv_bf8, u[1]), __builtin_bit_cast(mnv_bf8, u[2])}};
  }
};

// Row of result register r, for lanes of half h.
__device__ __forceinline__ constexpr int mnv_acc_row(int r, int h) { return 8 * (r / 4) + 4 * h + r % 4; }

// 32 consecutive rows of two matrices (of up to DP columns, `pitch` floats from row to row) on their way from
// memory to LDS: fetched into registers a tile ahead, then cut into planes of parts.  A row's 16-byte chunks
// are permuted among themselves (`swap`), so that 16 chunks of one number (read by rows) and 4 rows of 64 bytes
// (read by columns) lie in different banks; with rows padded instead, one of the two reads has conflicts
// (16 bytes: 2 extra cycles on 4 by columns; 32 bytes: 4 extra on 8 by rows).
// VEC: dim is a multiple of 4 (else values are fetched one by one).
template <int DP, int NT, bool VEC>
struct MnvStage {
  static constexpr int CHUNKS = DP / 8, UNITS = 32 * CHUNKS, SLOTS = (2 * UNITS + NT - 1) / NT;
  static constexpr int PITCH = DP * 2, PLANE = 32 * PITCH, MATRIX = 3 * PLANE, BYTES = 2 * MATRIX;
  static_assert(UNITS % MNV_WAVE == 0, "a wavefront's units are all of one matrix");

  mnv_f4 v[SLOTS][2];  // a unit is eight values of a row

  struct At {
    bool any, second;  // the same for the whole wavefront
    int row, col;
  };
  __device__ static __forceinline__ At at(int s) {
    const unsigned first = s * NT + mnv_uniform(threadIdx.x / MNV_WAVE) * MNV_WAVE;
    At a;
    a.any = 2 * UNITS % NT == 0 || first < 2 * UNITS;
    a.second = UNITS % NT == 0 ? s >= UNITS / NT : first >= UNITS;
    const unsigned u = first % UNITS + threadIdx.x % MNV_WAVE;
    a.row = u / CHUNKS;
    a.col = u % CHUNKS * 8;
    return a;
  }

  // Fetches the tile from rows >= 1 rows that exist, in PIECES pieces.  In place of a row behind them comes the last
  // one, and in place of a column behind dim another of the row: what they are multiplied by is 0, and they
  // hold nothing that has no part in the result anyway, so no value is selected and nothing waits before
  // `store`.  Byte offsets within a tile fit 32 bits (MNV_AT_MAX_PITCH).
  static constexpr int PIECES = 2 * SLOTS;
  __device__ __forceinline__ void fetch_piece(int piece, const float* m0, const float* m1, unsigned pitch, int rows,
                                              int dim) {
    const int s = piece / 2;
    if (s >= SLOTS) return;
    const At a = at(s);
    if (!a.any) return;
    const float* m = UNITS % NT == 0 ? (a.second ? m1 : m0) : m0 + (ptrdiff_t)a.second * (m1 - m0);
    const unsigned mine = (unsigned)a.row * pitch, last = (unsigned)(rows - 1) * pitch, row = mine < last ? mine : last;
    const int c = a.col + piece % 2 * 4;
    if (VEC) {
      const unsigned off = (row + (unsigned)(c < dim - 4 ? c : dim - 4)) * 4;
      v[s][piece % 2] = mnv_ldx4u<false>(reinterpret_cast<const float*>(reinterpret_cast<const char*>(m) + off));
    } else {
      const float* p = m + row;
      v[s][piece % 2] = mnv_f4{p[c < dim ? c : dim - 1], p[c + 1 < dim ? c + 1 : dim - 1],
                               p[c + 2 < dim ? c + 2 : dim - 1], p[c + 3 < dim ? c + 3 : dim - 1]};
    }
  }
  __device__ __forceinline__ void fetch(const float* m0, const float* m1, unsigned pitch, int rows, int dim) {
#pragma unroll
    for (int piece = 0; piece < PIECES; ++piece) fetch_piece(piece, m0, m1, pitch, rows, dim);
  }

  // Cuts the tile into its planes, in as many pieces, each unit written with its last.
  mnv_u4 w[3];
  __device__ __forceinline__ void store_piece(int piece, char* lds) {
    const int s = piece / 2;
    if (s >= SLOTS) return;
    const At a = at(s);
    if (!a.any) return;
#pragma unroll
    for (int h = piece % 2 * 2; h < piece % 2 * 2 + 2; ++h) {
      unsigned t[3];
      mnv_cut_pair<true>(v[s][h / 2][h % 2 * 2], v[s][h / 2][h % 2 * 2 + 1], t);
#pragma unroll
      for (int p = 0; p < 3; ++p) w[p][h] = t[p];
    }
    if (piece % 2 == 0) return;
    char* to = lds + (int)a.second * MATRIX + a.row * PITCH + ((a.col / 8) ^ swap(a.row)) * 16;
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<mnv_u4*>(to + p * PLANE) = w[p];
  }
  __device__ __forceinline__ void store(char* lds) {
#pragma unroll
    for (int piece = 0; piece < PIECES; ++piece) store_piece(piece, lds);
  }

  // What a row's chunk numbers are xored with.  4 rows of 64 bytes: 128 columns put all in the same banks, 64
  // two and two, 32 and 96 none.
  static constexpr int SWAPPED = DP == 128 ? 15 : DP == 64 ? 7 : 3;  // bits of a chunk's number that change
  __device__ static __forceinline__ int swap(int row) {
    return row / 4 % 4 + (DP == 128 ? row % 4 * 4 : DP == 64 ? row / 2 % 2 * 4 : 0);
  }

  // Part c of the operand of the 32 rows, columns 16 s ... of step s, from the planes of one matrix.
  __device__ static __forceinline__ mnv_bf8 by_rows(const char* planes, int s, int c) {
    const int lane = threadIdx.x % MNV_WAVE, row = lane % 32;
    // chunk 2 s + lane / 32
    const int at = row * PITCH + (swap(row) ^ (lane / 32)) * 16;
    return *reinterpret_cast<const mnv_bf8*>(planes + (at ^ (2 * s & SWAPPED) * 16) + (2 * s & ~SWAPPED) * 16 + c * PLANE);
  }
  // Part c of the operand of the 32 columns from `col` on, rows 16 s ... of step s.
  __device__ static __forceinline__ mnv_bf8 by_cols(const char* planes, int col, int s, int c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4* lds_s4;
    const int lane = threadIdx.x % MNV_WAVE, row = lane / 32 * 4 + lane % 16 / 4;
    // chunk col / 8 + 2 (lane / 16 % 2) + lane % 4 / 2 of rows `row` and row + 8, whose numbers are swapped by 2 more
    const int at = row * PITCH + (swap(row) ^ (lane / 16 % 2 * 2 + lane % 4 / 2)) * 16 + lane % 2 * 8;
    const char* p = planes + s * 16 * PITCH + (col / 8 & ~SWAPPED) * 16 + c * PLANE;
    const int low = at ^ (col / 8 & SWAPPED) * 16, high = (low ^ 32) + 8 * PITCH;
    const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + low));
    const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + high));
    return __builtin_bit_cast(mnv_bf8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// The columns 16 s + 8 (l / 32)... of one row (the lane's own) as an operand; 0 from dim on.
template <int DP, bool VEC>
__device__ __forceinline__ void mnv_load8(const float* row, int s, int dim, float (&x)[8]) {
  const int d0 = s * 16 + (int)threadIdx.x % MNV_WAVE / 32 * 8;
  if (VEC) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d = d0 + 4 * h;
      const mnv_f4 t = mnv_ldx4u<false>(row + (d < dim - 4 ? d : dim - 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * h + e] = d < dim ? t[e] : 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = row[d0 + e < dim ? d0 + e : dim - 1];
      x[e] = d0 + e < dim ? t : 0.f;
    }
  }
}

// Writes the lane's column of a [DP x 32] result, times f, to the dim values of `row`; 0 where it is not wanted.
template <int DP>
__device__ __forceinline__ void mnv_store_column(const mnv_f16 (&acc)[DP / 32], float f, bool wanted, float* row,
                                                 int dim) {
  const int half = (int)threadIdx.x % MNV_WAVE / 32;
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = n * 32 + 8 * u + 4 * half;
      mnv_f4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = wanted ? acc[n][4 * u + e] * f : 0.f;
      if (d + 4 <= dim) {
        *reinterpret_cast<mnv_f4u*>(row + d) = t;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < dim) row[d + e] = t[e];
      }
    }
}

#endif
