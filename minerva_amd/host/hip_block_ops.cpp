#include "hip_op_checks.h"
#include "hip_sequence_ops.h"
#include "mnv_hip.h"

namespace minerva {
namespace hip {

namespace {

template <class C>
void Rotary(const char* what, const DataList& inputs, const DataList& outputs, const C& c, bool back, const Context& ctx) {
  MNV_CHECK_EQ(inputs.size(), 1u + c.has_positions) << "(" << what << ") #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 1u) << "(" << what << ") #outputs wrong";
  const Scale& x = inputs[0].size_;
  MNV_CHECK_EQ(x.NumDims(), 4u) << "(" << what << ") takes {head_dim, heads, length, batch}";
  MNV_CHECK(c.first >= 0 && c.count > 0 && c.count <= x[1] && c.first <= x[1] - c.count) << "(" << what << ") heads out of range";
  MNV_CHECK(static_cast<long long>(x[0]) * x[1] <= 0x7fffffffLL) << "(" << what << ") heads too wide";
  const float* positions = nullptr;
  if (c.has_positions) {
    MNV_CHECK(LiesAs(inputs[1].size_, {x[2], x[3]})) << "(" << what << ") positions are {length, batch}, not " << inputs[1].size_;
    positions = inputs[1].data_;
  }
  const auto f = back ? mnv_rotary_bwd : mnv_rotary_fwd;
  Ok(f(inputs[0].data_ + static_cast<size_t>(c.first) * x[0], positions, outputs[0].data_, x[0], c.count, x[2], x[3], x[0] * x[1],
       x[0] * c.count, c.rotary_dim, c.interleaved ? 1 : 0, c.start, c.base, c.factor, c.context, c.low_turns, c.high_turns, c.magnitude,
       ctx.stream),
     what);
}

struct GatedExtents {
  int features, hidden, tokens;
};
// x {features, tokens}, in any number of dimensions whose first is `features`
GatedExtents GatedSizes(const char* what, const Scale& x, const Scale& w_in, const Scale& w_out) {
  MNV_CHECK(x.NumDims() >= 2u && x.Prod() > 0) << "(" << what << ") takes features and tokens";
  GatedExtents e;
  e.features = x[0];
  e.tokens = x.Prod() / x[0];
  MNV_CHECK(w_out.NumDims() == 2u && w_out[0] == e.features) << "(" << what << ") the second weights are {features, hidden}, not " << w_out;
  e.hidden = w_out[1];
  MNV_CHECK(w_in.NumDims() == 2u && w_in[1] == e.features && w_in[0] == 2LL * e.hidden)
      << "(" << what << ") the first weights are {2 hidden, features}, not " << w_in;
  return e;
}

}  // namespace

void RotaryForward(const DataList& inputs, const DataList& outputs, RotaryForwardClosure& c, const Context& ctx) {
  Rotary("rotary forward", inputs, outputs, c, false, ctx);
}

void RotaryBackward(const DataList& inputs, const DataList& outputs, RotaryBackwardClosure& c, const Context& ctx) {
  Rotary("rotary backward", inputs, outputs, c, true, ctx);
}

void GatedFFNForward(const DataList& inputs, const DataList& outputs, GatedFFNForwardClosure& c, const Context& ctx) {
  MNV_CHECK_EQ(inputs.size(), 3u) << "(gated ffn forward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 3u) << "(gated ffn forward) #outputs wrong";
  const GatedExtents e = GatedSizes("gated ffn forward", inputs[0].size_, inputs[1].size_, inputs[2].size_);
  Ok(mnv_gated_ffn_fwd(inputs[0].data_, inputs[1].data_, inputs[2].data_, outputs[1].data_, outputs[2].data_, outputs[0].data_, e.features,
                       e.hidden, e.tokens, static_cast<int>(c.type), ctx.workspace, ctx.workspace_bytes, ctx.stream),
     "gated ffn forward");
}

void GatedFFNBackward(const DataList& inputs, const DataList& outputs, GatedFFNBackwardClosure& c, const Context& ctx) {
  MNV_CHECK_EQ(inputs.size(), 6u) << "(gated ffn backward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 4u) << "(gated ffn backward) #outputs wrong";
  const GatedExtents e = GatedSizes("gated ffn backward", inputs[1].size_, inputs[2].size_, inputs[3].size_);
  MNV_CHECK(inputs[0].size_ == inputs[1].size_) << "(gated ffn backward) extents differ";
  MNV_CHECK(LiesAs(inputs[4].size_, {2 * e.hidden, e.tokens})) << "(gated ffn backward) pre is {2 hidden, tokens}, not " << inputs[4].size_;
  MNV_CHECK(LiesAs(inputs[5].size_, {e.hidden, e.tokens})) << "(gated ffn backward) h is {hidden, tokens}, not " << inputs[5].size_;
  Ok(mnv_gated_ffn_bwd(inputs[1].data_, inputs[2].data_, inputs[3].data_, inputs[4].data_, inputs[5].data_, inputs[0].data_, outputs[3].data_,
                       outputs[0].data_, outputs[1].data_, outputs[2].data_, e.features, e.hidden, e.tokens, static_cast<int>(c.type),
                       ctx.workspace, ctx.workspace_bytes, ctx.stream),
     "gated ffn backward");
}

void AdamWStep(const DataList& inputs, const DataList& outputs, AdamWClosure& c, const Context& ctx) {
  const size_t n = c.rates.size();
  MNV_CHECK(n > 0 && c.decays.size() == n) << "(adamw) a rate and a decay for every array";
  MNV_CHECK_EQ(inputs.size(), 4 * n) << "(adamw) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 3 * n) << "(adamw) #outputs wrong";
  std::vector<const float*> in[4];
  std::vector<float*> out[3];
  std::vector<size_t> sizes;
  for (size_t i = 0; i < n; ++i) {
    const size_t count = inputs[i].size_.Prod();
    MNV_CHECK_EQ(static_cast<size_t>(inputs[n + i].size_.Prod()), count) << "(adamw) gradient " << i << " has other extents than its array";
    for (int k = 2; k < 4; ++k)
      MNV_CHECK_EQ(static_cast<size_t>(inputs[k * n + i].size_.Prod()), mnv_adamw_moment_floats(count, c.bits))
          << "(adamw) moments of array " << i << " of another size";
    sizes.push_back(count);
    for (int k = 0; k < 4; ++k) in[k].push_back(inputs[k * n + i].data_);
    for (int k = 0; k < 3; ++k) out[k].push_back(outputs[k * n + i].data_);
  }
  Ok(mnv_adamw_step(static_cast<int>(n), in[0].data(), in[1].data(), in[2].data(), in[3].data(), out[0].data(), out[1].data(), out[2].data(),
                    sizes.data(), c.rates.data(), c.decays.data(), c.bits, c.rate, c.beta1, c.beta2, c.eps, c.weight_decay, c.grad_scale,
                    c.step, nullptr, ctx.stream),
     "adamw");
}

void AdamWValues(const DataList& inputs, const DataList& outputs, AdamWValuesClosure&, const Context& ctx) {
  const size_t n = inputs.size() / 2;
  MNV_CHECK(n > 0 && inputs.size() == 2 * n) << "(adamw values) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 2 * n) << "(adamw values) #outputs wrong";
  std::vector<const float*> in;
  std::vector<float*> out;
  std::vector<size_t> sizes;
  for (size_t i = 0; i < 2 * n; ++i) {
    const size_t count = outputs[i].size_.Prod();
    MNV_CHECK_EQ(count, static_cast<size_t>(outputs[i % n].size_.Prod())) << "(adamw values) both moments have the same number of values";
    MNV_CHECK_EQ(static_cast<size_t>(inputs[i].size_.Prod()), mnv_adamw_moment_floats(count, 8)) << "(adamw values) moment " << i << " of another size";
    in.push_back(inputs[i].data_);
    out.push_back(outputs[i].data_);
    if (i < n) sizes.push_back(count);
  }
  Ok(mnv_adamw_values(static_cast<int>(n), in.data(), in.data() + n, out.data(), out.data() + n, sizes.data(), ctx.stream), "adamw values");
}

}  // namespace hip
}  // namespace minerva
