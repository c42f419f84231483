// Operators of networks over sequences: layer norm, attention to the states of another (or the same)
// sequence, and the learned relative position bias that enters it.  The reference has none of them; closures and
// functions follow the conventions of its own (DataList inputs, DataList outputs, closure, context).  Attention's
// optional inputs follow the others in the order bias, lengths, as far as the closure says they are there.
#pragma once
#include "minerva_types.h"

namespace minerva {

// out = gamma * (x - mean) / sqrt(var + eps) + beta over all but the last dimension; inputs {x, gamma, beta}
struct LayerNormForwardClosure {
  float eps;
};
// outputs {dx, dgamma, dbeta}; inputs {diff, x, gamma}
struct LayerNormBackwardClosure {
  float eps;
};
// outputs {out, stats}; inputs {q, k, v [, bias] [, lengths]}
struct AttentionForwardClosure {
  float scale;
  bool has_bias, has_lengths;
};
// outputs {dq, dk, dv [, dbias]}; inputs {diff, q, k, v, out, stats [, bias] [, lengths]}
struct AttentionBackwardClosure {
  float scale;
  bool has_bias, has_lengths;
};
// forward: out = bias by offset, inputs {table}; backward: out = the table's gradient, inputs {the bias's gradient}
template <int i> struct RelativeBiasClosure {
  int buckets, q_len, k_len, q_start, max_distance;
  bool both_ways;
};
typedef RelativeBiasClosure<0> RelativeBiasForwardClosure;
typedef RelativeBiasClosure<1> RelativeBiasBackwardClosure;

namespace hip {

void LayerNormForward(const DataList&, const DataList&, LayerNormForwardClosure&, const Context&);
void LayerNormBackward(const DataList&, const DataList&, LayerNormBackwardClosure&, const Context&);
void AttentionForward(const DataList&, const DataList&, AttentionForwardClosure&, const Context&);
void AttentionBackward(const DataList&, const DataList&, AttentionBackwardClosure&, const Context&);
void RelativeBiasForward(const DataList&, const DataList&, RelativeBiasForwardClosure&, const Context&);
void RelativeBiasBackward(const DataList&, const DataList&, RelativeBiasBackwardClosure&, const Context&);

}  // namespace hip
}  // namespace minerva
