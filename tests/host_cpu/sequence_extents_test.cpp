// CPU test of what the operators of networks over sequences ask of their arrays' extents
// (minerva_amd/host/hip_sequence_ops.cpp), with entry points that only count the calls that reach them.
// usage: sequence_extents_test mixed | empty.  Prints "OK" and exits 0 when every check holds.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "hip_sequence_ops.h"
#include "mnv_hip.h"

static int g_calls = 0;
extern "C" {
const char* mnv_error_string(int) { return "error"; }
int mnv_layernorm_fwd(const float*, const float*, const float*, float*, int, int, float, mnv_stream_t) { return ++g_calls, MNV_OK; }
int mnv_layernorm_bwd(const float*, const float*, const float*, float*, float*, float*, int, int, float, void*, size_t,
                      mnv_stream_t) {
  return ++g_calls, MNV_OK;
}
int mnv_attention_fwd(const float*, const float*, const float*, const float*, const float*, float*, float*, int, int, int, int,
                      int, int, float, void*, size_t, mnv_stream_t) {
  return ++g_calls, MNV_OK;
}
int mnv_attention_bwd(const float*, const float*, const float*, const float*, const float*, const float*, const float*,
                      const float*, float*, float*, float*, float*, int, int, int, int, int, int, float, void*, size_t,
                      mnv_stream_t) {
  return ++g_calls, MNV_OK;
}
int mnv_relative_bias_fwd(const float*, float*, int, int, int, int, int, int, int, mnv_stream_t) { return ++g_calls, MNV_OK; }
int mnv_relative_bias_bwd(const float*, float*, int, int, int, int, int, int, int, mnv_stream_t) { return ++g_calls, MNV_OK; }
}

using namespace minerva;

static float g_value;
static int g_failed = 0;

static DataList List(const std::vector<Scale>& sizes) {
  DataList l;
  for (const Scale& s : sizes) l.emplace_back(&g_value, s);
  return l;
}

template <class C> using Fn = void (*)(const DataList&, const DataList&, C&, const Context&);

// Calls the operator, and says where it took what it should refuse, or the reverse.
template <class C>
static void Expect(bool taken, Fn<C> fn, C closure, const std::vector<Scale>& inputs, const std::vector<Scale>& outputs,
                   const char* what) {
  Context ctx;
  const int before = g_calls;
  bool threw = false;
  try {
    fn(List(inputs), List(outputs), closure, ctx);
  } catch (const Error&) {
    threw = true;
  }
  const bool ok = taken ? !threw && g_calls == before + 1 : threw && g_calls == before;
  if (!ok) {
    std::fprintf(stderr, "%s: should be %s\n", what, taken ? "taken" : "refused");
    ++g_failed;
  }
}

// Arrays with the right number of values in another order are not read as if they were right.
static void Mixed() {
  const Scale q{8, 4, 5, 3}, k{8, 2, 6, 3}, stats{2, 4, 5, 3};
  AttentionForwardClosure f{1.f, true, false};
  const std::vector<Scale> fo{q, stats};
  Expect(true, hip::AttentionForward, f, {q, k, k, Scale{10, 4}}, fo, "bias {offsets, heads}");
  Expect(true, hip::AttentionForward, f, {q, k, k, Scale{10, 4, 1}}, fo, "bias {offsets, heads, 1}");
  Expect(false, hip::AttentionForward, f, {q, k, k, Scale{4, 10}}, fo, "bias {heads, offsets}");
  Expect(true, hip::AttentionForward, f, {q, k, k, Scale{40}}, fo, "bias {offsets * heads}");
  Expect(false, hip::AttentionForward, f, {q, k, k, Scale{39}}, fo, "bias {offsets * heads - 1}");
  Expect(false, hip::AttentionForward, f, {q, k, k, Scale{20, 2}}, fo, "bias {2 offsets, heads / 2}");
  const Scale q1{8, 1, 5, 3}, k1{8, 1, 6, 3};
  Expect(true, hip::AttentionForward, f, {q1, k1, k1, Scale{10}}, {q1, Scale{2, 1, 5, 3}}, "bias of one head");
  AttentionForwardClosure g{1.f, false, true};
  Expect(true, hip::AttentionForward, g, {q, k, k, Scale{3}}, fo, "lengths {batch}");
  Expect(true, hip::AttentionForward, g, {q, k, k, Scale{1, 3}}, fo, "lengths {1, batch}");
  AttentionBackwardClosure b{1.f, false, false};
  const std::vector<Scale> bo{q, k, k};
  Expect(true, hip::AttentionBackward, b, {q, q, k, k, q, stats}, bo, "stats {2, heads, q_len, batch}");
  Expect(false, hip::AttentionBackward, b, {q, q, k, k, q, Scale{2, 5, 4, 3}}, bo, "stats {2, q_len, heads, batch}");
  Expect(false, hip::AttentionBackward, b, {q, q, k, k, q, Scale{4, 5, 3, 2}}, bo, "stats {heads, q_len, batch, 2}");
  const Scale x{4, 6, 7};
  LayerNormForwardClosure n{1e-5f};
  for (const Scale& good : {Scale{24}, Scale{24, 1}, Scale{1, 24}, Scale{4, 6}, Scale{4, 6, 1}})
    Expect(true, hip::LayerNormForward, n, {x, good, good}, {x}, "a value per feature");
  for (const Scale& bad : {Scale{6, 4}, Scale{2, 12}, Scale{12, 2}, Scale{23}}) {
    Expect(false, hip::LayerNormForward, n, {x, bad, Scale{24}}, {x}, "gain of another order");
    Expect(false, hip::LayerNormForward, n, {x, Scale{24}, bad}, {x}, "offset of another order");
    LayerNormBackwardClosure nb{1e-5f};
    Expect(false, hip::LayerNormBackward, nb, {x, x, bad}, {x, bad, bad}, "gain of another order, backward");
  }
}

// Of an array without values nothing is divided by its number of columns.
static void Empty() {
  for (const Scale& x : {Scale{4, 0}, Scale{0, 4}, Scale{0, 0}}) {
    LayerNormForwardClosure n{1e-5f};
    Expect(false, hip::LayerNormForward, n, {x, Scale{4}, Scale{4}}, {x}, "norm of an empty array");
    LayerNormBackwardClosure nb{1e-5f};
    Expect(false, hip::LayerNormBackward, nb, {x, x, Scale{4}}, {x, Scale{4}, Scale{4}}, "norm of an empty array, backward");
  }
}

int main(int argc, char** argv) {
  if (argc == 2 && !std::strcmp(argv[1], "mixed")) Mixed();
  else if (argc == 2 && !std::strcmp(argv[1], "empty")) Empty();
  else return 2;
  if (g_failed) return 1;
  std::printf("OK\n");
  return 0;
}
