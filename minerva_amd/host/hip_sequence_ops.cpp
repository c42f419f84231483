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

}  // namespace hip
}  // namespace minerva
