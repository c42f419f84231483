#include "hip_sequence_ops.h"

#include "mnv_hip.h"

namespace minerva {
namespace hip {

namespace {

void Ok(int status, const char* what) {
  MNV_CHECK(status == MNV_OK) << what << ": " << mnv_error_string(status);
}

// The extents that say how values lie in memory: without those that are 1.
std::vector<int> Layout(const std::vector<int>& dims) {
  std::vector<int> r;
  for (int d : dims)
    if (d != 1) r.push_back(d);
  return r;
}
// Whether s holds values in the order of `dims`: with these extents, or flat.
bool LiesAs(const Scale& s, const std::vector<int>& dims) {
  const std::vector<int> have = Layout(s.ToVector());
  long long all = 1;
  for (int d : dims) all *= d;
  return have == Layout(dims) || (have.size() == 1 && have[0] == all);
}

// {features, count}: the last dimension counts the columns.
int Columns(const Scale& s) {
  MNV_CHECK(s.NumDims() >= 2) << "(layer norm) takes features and columns";
  MNV_CHECK(s.Prod() > 0) << "(layer norm) of an empty array " << s;
  return s[s.NumDims() - 1];
}
// A value per feature, in a column's order.
bool PerFeature(const Scale& s, const Scale& x) { return LiesAs(s, std::vector<int>(x.begin(), x.end() - 1)); }

struct AttentionExtents {
  int head_dim, heads, q_len, batch, kv_heads, k_len;
  const float *bias = nullptr, *lengths = nullptr;
};
AttentionExtents Extents(const char* what, const DataList& inputs, size_t fixed, const Scale& q, const Scale& k,
                         const Scale& v, bool has_bias, bool has_lengths) {
  MNV_CHECK_EQ(inputs.size(), fixed + has_bias + has_lengths) << "(" << what << ") #inputs wrong";
  MNV_CHECK_EQ(q.NumDims(), 4u) << "(" << what << ") queries are {head_dim, heads, q_len, batch}";
  MNV_CHECK_EQ(k.NumDims(), 4u) << "(" << what << ") keys are {head_dim, kv_heads, k_len, batch}";
  MNV_CHECK(k == v) << "(" << what << ") keys' and values' extents differ";
  MNV_CHECK(q[0] == k[0] && q[3] == k[3]) << "(" << what << ") queries' and keys' head_dim or batch differ";
  AttentionExtents e;
  e.head_dim = q[0];
  e.heads = q[1];
  e.q_len = q[2];
  e.batch = q[3];
  e.kv_heads = k[1];
  e.k_len = k[2];
  if (has_bias) {
    const DataShard& b = inputs[fixed];
    const long long offsets = static_cast<long long>(e.q_len) + e.k_len - 1;
    MNV_CHECK(offsets <= 0x7fffffffLL && LiesAs(b.size_, {static_cast<int>(offsets), e.heads}))
        << "(" << what << ") bias is {q_len + k_len - 1, heads}, not " << b.size_;
    e.bias = b.data_;
  }
  if (has_lengths) {
    const DataShard& l = inputs[fixed + has_bias];
    MNV_CHECK(LiesAs(l.size_, {e.batch})) << "(" << what << ") lengths has one value per entry of the batch, not " << l.size_;
    e.lengths = l.data_;
  }
  return e;
}

}  // namespace

void LayerNormForward(const DataList& inputs, const DataList& outputs, LayerNormForwardClosure& c, const Context& ctx) {
  MNV_CHECK_EQ(inputs.size(), 3u) << "(layer norm forward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 1u) << "(layer norm forward) #outputs wrong";
  const int count = Columns(inputs[0].size_), features = inputs[0].size_.Prod() / count;
  MNV_CHECK(PerFeature(inputs[1].size_, inputs[0].size_)) << "(layer norm forward) gain has one value per feature";
  MNV_CHECK(PerFeature(inputs[2].size_, inputs[0].size_)) << "(layer norm forward) offset has one value per feature";
  Ok(mnv_layernorm_fwd(inputs[0].data_, inputs[1].data_, inputs[2].data_, outputs[0].data_, features, count, c.eps,
                       ctx.stream),
     "layer norm forward");
}

void LayerNormBackward(const DataList& inputs, const DataList& outputs, LayerNormBackwardClosure& c, const Context& ctx) {
  MNV_CHECK_EQ(inputs.size(), 3u) << "(layer norm backward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 3u) << "(layer norm backward) #outputs wrong";
  const auto& diff = inputs[0];
  const auto& x = inputs[1];
  const auto& gamma = inputs[2];
  const int count = Columns(x.size_), features = x.size_.Prod() / count;
  MNV_CHECK(diff.size_ == x.size_) << "(layer norm backward) extents differ";
  MNV_CHECK(PerFeature(gamma.size_, x.size_)) << "(layer norm backward) gain has one value per feature";
  Ok(mnv_layernorm_bwd(x.data_, gamma.data_, diff.data_, outputs[0].data_, outputs[1].data_, outputs[2].data_, features,
                       count, c.eps, ctx.workspace, ctx.workspace_bytes, ctx.stream),
     "layer norm backward");
}

void AttentionForward(const DataList& inputs, const DataList& outputs, AttentionForwardClosure& c, const Context& ctx) {
  MNV_CHECK(inputs.size() >= 3u) << "(attention forward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 2u) << "(attention forward) #outputs wrong";
  const AttentionExtents e = Extents("attention forward", inputs, 3, inputs[0].size_, inputs[1].size_, inputs[2].size_,
                                     c.has_bias, c.has_lengths);
  Ok(mnv_attention_fwd(inputs[0].data_, inputs[1].data_, inputs[2].data_, e.bias, e.lengths, outputs[0].data_,
                       outputs[1].data_, e.batch, e.heads, e.kv_heads, e.q_len, e.k_len, e.head_dim, c.scale,
                       ctx.workspace, ctx.workspace_bytes, ctx.stream),
     "attention forward");
}

void AttentionBackward(const DataList& inputs, const DataList& outputs, AttentionBackwardClosure& c, const Context& ctx) {
  MNV_CHECK(inputs.size() >= 6u) << "(attention backward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 3u + c.has_bias) << "(attention backward) #outputs wrong";
  const AttentionExtents e = Extents("attention backward", inputs, 6, inputs[1].size_, inputs[2].size_, inputs[3].size_,
                                     c.has_bias, c.has_lengths);
  MNV_CHECK(inputs[0].size_ == inputs[1].size_ && inputs[4].size_ == inputs[1].size_)
      << "(attention backward) queries', results' and gradients' extents differ";
  MNV_CHECK(LiesAs(inputs[5].size_, {2, e.heads, e.q_len, e.batch}))
      << "(attention backward) stats are {2, heads, q_len, batch}, not " << inputs[5].size_;
  Ok(mnv_attention_bwd(inputs[1].data_, inputs[2].data_, inputs[3].data_, e.bias, e.lengths, inputs[4].data_,
                       inputs[5].data_, inputs[0].data_, outputs[0].data_, outputs[1].data_, outputs[2].data_,
                       c.has_bias ? outputs[3].data_ : nullptr, e.batch, e.heads, e.kv_heads, e.q_len, e.k_len, e.head_dim,
                       c.scale, ctx.workspace, ctx.workspace_bytes, ctx.stream),
     "attention backward");
}

void RelativeBiasForward(const DataList& inputs, const DataList& outputs, RelativeBiasForwardClosure& c,
                         const Context& ctx) {
  MNV_CHECK_EQ(inputs.size(), 1u) << "(relative bias forward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 1u) << "(relative bias forward) #outputs wrong";
  MNV_CHECK_EQ(inputs[0].size_.NumDims(), 2u) << "(relative bias forward) the table is {heads, buckets}";
  MNV_CHECK_EQ(inputs[0].size_[1], c.buckets) << "(relative bias forward) the table is {heads, buckets}";
  Ok(mnv_relative_bias_fwd(inputs[0].data_, outputs[0].data_, c.buckets, inputs[0].size_[0], c.q_len, c.k_len, c.q_start,
                           c.max_distance, c.both_ways ? 1 : 0, ctx.stream),
     "relative bias forward");
}

void RelativeBiasBackward(const DataList& inputs, const DataList& outputs, RelativeBiasBackwardClosure& c,
                          const Context& ctx) {
  MNV_CHECK_EQ(inputs.size(), 1u) << "(relative bias backward) #inputs wrong";
  MNV_CHECK_EQ(outputs.size(), 1u) << "(relative bias backward) #outputs wrong";
  MNV_CHECK_EQ(inputs[0].size_.NumDims(), 2u) << "(relative bias backward) the gradient is {q_len + k_len - 1, heads}";
  MNV_CHECK_EQ(static_cast<long long>(inputs[0].size_[0]), static_cast<long long>(c.q_len) + c.k_len - 1)
      << "(relative bias backward) the gradient is {q_len + k_len - 1, heads}";
  Ok(mnv_relative_bias_bwd(inputs[0].data_, outputs[0].data_, c.buckets, inputs[0].size_[1], c.q_len, c.k_len, c.q_start,
                           c.max_distance, c.both_ways ? 1 : 0, ctx.stream),
     "relative bias backward");
}

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
