// SGEMM C{m,n} = A{m,k} * B{k,n}, column-major, no transposes, alpha 1 / beta 0:
// the product Minerva's MatMult asks for (reference minerva/op/impl/basic.cpp:150-173;
// cublasSgemm call at minerva/op/impl/cuda/cuda_perform.cu:66-70).
// The kernels, their plan and launch are in sgemm_core.h; A is fetched x-fast (m contiguous), B k-fast (k
// contiguous).  Products with too few output tiles to fill 256 CUs split the k range over
// blockIdx.z when the caller lends a workspace.
#include <mutex>

#include "sgemm_core.h"

// Split-k partial sums of mnv_sgemm_nn_static: one array per GPU the library is loaded on,
// held until the process ends.  In host code the name `scratch` is only a handle for
// hipGetSymbolAddress; kernels and every other use take the address it returns.
#define MNV_SGEMM_STATIC_SCRATCH_FLOATS ((size_t)MNV_SGEMM_STATIC_SCRATCH_BYTES / sizeof(float))
static __device__ __align__(256) float scratch[MNV_SGEMM_STATIC_SCRATCH_FLOATS];

namespace {

#define MNV_MAX_DEVICES 64
std::mutex g_scratch_mutex;
float* g_scratch_ptr[MNV_MAX_DEVICES];  // device address of `scratch` on each GPU

// The address of the current device's copy of `scratch`, looked up once per device.
int scratch_address(float** out) {
  int dev = -1;
  MNV_HIP_TRY(hipGetDevice(&dev));
  if (dev < 0 || dev >= MNV_MAX_DEVICES) return MNV_ERR_INVALID;
  std::lock_guard<std::mutex> lock(g_scratch_mutex);
  if (!g_scratch_ptr[dev]) {
    void* p = nullptr;
    MNV_HIP_TRY(hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)));
    if (!p) return MNV_ERR_INVALID;
    g_scratch_ptr[dev] = static_cast<float*>(p);
  }
  *out = g_scratch_ptr[dev];
  return MNV_OK;
}

int sgemm_nn_impl(const float* a, const float* b, float* c, int m, int n, int k, void* workspace,
                  size_t workspace_bytes, hipStream_t s,
                  const SgemmEpilogue& e = SgemmEpilogue{nullptr, nullptr, 0}) {
  // a panel of larger matrices has their pitches, which the small kernel's reach is not planned for
  const SgemmPlan plan = e.lda ? plan_within(m, n, k, 0, mnv_cu_count()) : plan_sgemm(m, n, k, workspace ? workspace_bytes / sizeof(float) : 0);
  if (plan.skinny) return launch_skinny_columns(plan, make_sgemm<true>(a, b, c, m, n, k, e), workspace, s);
  if (plan.tile) return launch_small_tiles(plan, make_sgemm<true>(a, b, c, m, n, k, e), s);
  if (k % 4 == 0) return launch_plan(plan, make_sgemm<true>(a, b, c, m, n, k, e), workspace, workspace_bytes, s);
  return launch_plan(plan, make_sgemm<false>(a, b, c, m, n, k, e), workspace, workspace_bytes, s);
}

// Operands of 2^29 elements and more (up to the reference's limit, int element counts): the
// product is cut into panels whose spans fit 32-bit byte offsets -- columns of B and C, rows
// of A and C, and ranges of k, the later k ranges accumulating into C -- each panel one launch
// with the whole matrices' leading dimensions.  Slower than one launch (C is re-read per k
// range, no k ranges over workgroups), and the sum over k is taken range by range.
const long long kOperandLimit = (1LL << 29) - 1;  // elements a launch can address per operand

bool sgemm_is_large(int m, int n, int k) {
  return (long long)m * k > kOperandLimit || (long long)k * n > kOperandLimit;
}

int sgemm_nn_large(const float* a, const float* b, float* c, int m, int n, int k, hipStream_t s) {
  const long long mc = m < (1 << 28) ? m : (1 << 28);
  long long kc = (kOperandLimit - mc) / m + 1;          // ((kc-1)*m + mc) <= limit
  if (kc > k) kc = k;
  if (kc >= 16) kc -= kc % 16;
  long long nc = (kOperandLimit - kc) / k + 1;          // ((nc-1)*k + kc) <= limit
  if (nc > n) nc = n;
  if (kc < 1 || nc < 1) return MNV_ERR_INVALID;
  for (long long n0 = 0; n0 < n; n0 += nc)
    for (long long m0 = 0; m0 < m; m0 += mc)
      for (long long k0 = 0; k0 < k; k0 += kc) {
        const int mm = (int)(m - m0 < mc ? m - m0 : mc), nn = (int)(n - n0 < nc ? n - n0 : nc);
        const int kk = (int)(k - k0 < kc ? k - k0 : kc);
        SgemmEpilogue e{nullptr, nullptr, 0, m, k, m, k0 > 0};
        int rc = sgemm_nn_impl(a + (size_t)k0 * m + m0, b + (size_t)n0 * k + k0,
                               c + (size_t)n0 * m + m0, mm, nn, kk, nullptr, 0, s, e);
        if (rc) return rc;
      }
  return MNV_OK;
}

}  // namespace

int mnv_sgemm_nn_ranges(const float* a, const float* b, int m, int n, int k, void* workspace, size_t workspace_bytes, int* ranges, hipStream_t s) {
  const SgemmPlan plan = plan_sgemm(m, n, k, workspace ? workspace_bytes / sizeof(float) : 0);
  *ranges = plan.tile ? 1 : plan.splits;
  if (*ranges == 1) return MNV_OK;
  if (!plan.skinny) {  // as the launch rounds it: ranges of equal length
    const int slabs = (k + 15) / 16, per = (slabs + plan.splits - 1) / plan.splits;
    *ranges = (slabs + per - 1) / per;
    if (*ranges == 1) return MNV_OK;
  }
  auto p = make_sgemm<true>(a, b, (float*)nullptr, m, n, k, SgemmEpilogue{nullptr, nullptr, 0});
  p.leaves_ranges = true;
  if (plan.skinny) return launch_skinny_columns(plan, p, workspace, s);
  if (k % 4 == 0) return launch_plan(plan, p, workspace, workspace_bytes, s);
  auto q = make_sgemm<false>(a, b, (float*)nullptr, m, n, k, SgemmEpilogue{nullptr, nullptr, 0});
  q.leaves_ranges = true;
  return launch_plan(plan, q, workspace, workspace_bytes, s);
}

extern "C" {

size_t mnv_sgemm_nn_workspace_bytes(int m, int n, int k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const SgemmPlan plan = plan_unlimited(m, n, k, mnv_cu_count());
  return plan.splits > 1 ? (size_t)plan.splits * m * n * sizeof(float) : sgemm_tail_bytes(plan, m, n, k);
}

int mnv_sgemm_nn_plan(int m, int n, int k, size_t workspace_bytes, int* tile_rows, int* k_ranges,
                      int* groups) {
  if (m <= 0 || n <= 0 || k <= 0 || !tile_rows || !k_ranges || !groups) return MNV_ERR_INVALID;
  const SgemmPlan plan = plan_sgemm(m, n, k, workspace_bytes / sizeof(float));
  *tile_rows = plan.tall || plan.skinny ? 256 : plan.small ? 64 : 128;
  const int slabs = (k + 15) / 16, per = (slabs + plan.splits - 1) / plan.splits;
  *k_ranges = plan.skinny ? plan.splits : (slabs + per - 1) / per;  // as the launch rounds it: ranges of equal length
  *groups = plan.tile ? 1 : plan.groups;
  return MNV_OK;
}

int mnv_sgemm_nn_small_plan(int m, int n, int k, size_t workspace_bytes, int* tile_rows, int* wavefronts) {
  if (m <= 0 || n <= 0 || k <= 0 || !tile_rows || !wavefronts) return MNV_ERR_INVALID;
  const SgemmPlan plan = plan_sgemm(m, n, k, workspace_bytes / sizeof(float));
  *tile_rows = plan.tile;
  *wavefronts = plan.tile ? plan.groups : 0;
  return MNV_OK;
}

int mnv_sgemm_nn(const float* a, const float* b, float* c, int m, int n, int k, void* workspace,
                 size_t workspace_bytes, mnv_stream_t stream) {
  if (m == 0 || n == 0) return MNV_OK;
  if (!a || !b || !c || m < 0 || n < 0 || k <= 0) return MNV_ERR_INVALID;
  // every operand is at most 2^31 - 1 elements (the reference's int element counts)
  if ((long long)m * k > 0x7fffffffLL || (long long)k * n > 0x7fffffffLL ||
      (long long)m * n > 0x7fffffffLL)
    return MNV_ERR_INVALID;
  if (sgemm_is_large(m, n, k)) return sgemm_nn_large(a, b, c, m, n, k, mnv_stream(stream));
  return sgemm_nn_impl(a, b, c, m, n, k, workspace, workspace_bytes, mnv_stream(stream));
}

int mnv_sgemm_nn_bias(const float* a, const float* b, const float* bias, float* c, int m, int n,
                      int k, int relu, void* workspace, size_t workspace_bytes,
                      mnv_stream_t stream) {
  if (m == 0 || n == 0) return MNV_OK;
  if (!a || !b || !bias || !c || m < 0 || n < 0 || k <= 0) return MNV_ERR_INVALID;
  if ((long long)m * k >= (1LL << 29) || (long long)k * n >= (1LL << 29)) return MNV_ERR_INVALID;
  return sgemm_nn_impl(a, b, c, m, n, k, workspace, workspace_bytes, mnv_stream(stream),
                       SgemmEpilogue{bias, nullptr, relu != 0});
}

int mnv_sgemm_nn_relu_bwd(const float* a, const float* b, const float* bottom, float* c, int m,
                          int n, int k, void* workspace, size_t workspace_bytes,
                          mnv_stream_t stream) {
  if (m == 0 || n == 0) return MNV_OK;
  if (!a || !b || !bottom || !c || m < 0 || n < 0 || k <= 0) return MNV_ERR_INVALID;
  if ((long long)m * k >= (1LL << 29) || (long long)k * n >= (1LL << 29)) return MNV_ERR_INVALID;
  return sgemm_nn_impl(a, b, c, m, n, k, workspace, workspace_bytes, mnv_stream(stream),
                       SgemmEpilogue{nullptr, bottom, 0});
}

int mnv_sgemm_tn(const float* at, const float* b, const float* gate, float* c, int m, int n, int k,
                 void* workspace, size_t workspace_bytes, mnv_stream_t stream) {
  if (m == 0 || n == 0) return MNV_OK;
  if (!at || !b || !c || m < 0 || n < 0 || k <= 0) return MNV_ERR_INVALID;
  if ((long long)m * k >= (1LL << 29) || (long long)k * n >= (1LL << 29)) return MNV_ERR_INVALID;
  return sgemm_t_impl<true, false>(at, b, c, m, n, k, workspace, workspace_bytes, mnv_stream(stream),
                                   SgemmEpilogue{nullptr, gate, 0});
}

int mnv_sgemm_nt(const float* a, const float* bt, float* c, int m, int n, int k, void* workspace,
                 size_t workspace_bytes, mnv_stream_t stream) {
  if (m == 0 || n == 0) return MNV_OK;
  if (!a || !bt || !c || m < 0 || n < 0 || k <= 0) return MNV_ERR_INVALID;
  if ((long long)m * k >= (1LL << 29) || (long long)k * n >= (1LL << 29)) return MNV_ERR_INVALID;
  return sgemm_t_impl<false, true>(a, bt, c, m, n, k, workspace, workspace_bytes, mnv_stream(stream),
                                   SgemmEpilogue{nullptr, nullptr, 0});
}

int mnv_sgemm_nt_sgd(const float* a, const float* bt, const float* w, float scale, float* w_out,
                     int m, int n, int k, void* workspace, size_t workspace_bytes,
                     mnv_stream_t stream) {
  if (m == 0 || n == 0) return MNV_OK;
  if (!a || !bt || !w || !w_out || m < 0 || n < 0 || k <= 0) return MNV_ERR_INVALID;
  if ((long long)m * k >= (1LL << 29) || (long long)k * n >= (1LL << 29)) return MNV_ERR_INVALID;
  SgemmEpilogue e{nullptr, nullptr, 0};
  e.sgd_w = w;
  e.sgd_scale = scale;
  return sgemm_t_impl<false, true>(a, bt, w_out, m, n, k, workspace, workspace_bytes,
                                   mnv_stream(stream), e);
}

int mnv_sgemm_nn_static(const float* a, const float* b, float* c, int m, int n, int k,
                        mnv_stream_t stream) {
  if (m == 0 || n == 0) return MNV_OK;
  if (!a || !b || !c || m < 0 || n < 0 || k <= 0) return MNV_ERR_INVALID;
  if ((long long)m * k >= (1LL << 29) || (long long)k * n >= (1LL << 29)) return MNV_ERR_INVALID;
  // at least two k ranges of partial sums must fit the static array
  if ((unsigned long long)m * (unsigned long long)n * 2ull > MNV_SGEMM_STATIC_SCRATCH_FLOATS)
    return MNV_ERR_TOO_LARGE;
  float* ws = nullptr;
  int rc = scratch_address(&ws);
  if (rc) return rc;
  return sgemm_nn_impl(a, b, c, m, n, k, ws, MNV_SGEMM_STATIC_SCRATCH_BYTES, mnv_stream(stream));
}

}  // extern "C"
