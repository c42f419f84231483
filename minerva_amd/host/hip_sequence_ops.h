// Operators of networks over sequences: layer norm, attention to the states of another (or the same)
// sequence, the learned relative position bias that enters it, rotary positions, the gated feed-forward block, and the
// AdamW step over many arrays that trains such networks.  The reference has none of them; closures and
// functions follow the conventions of its own (DataList inputs, DataList outputs, closure, context).  Attention's
// optional inputs follow the others in the order bias, lengths, as far as the closure says they are there.
#pragma once
#include <vector>

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
// out = the heads [first, first + count) of x {head_dim, heads, length, batch}, turned by their positions' angles, or back (the
// gradient); inputs {x [, positions {length, batch}]}.  Backward takes the turned heads' gradient, whose heads they all are.
template <int i> struct RotaryClosure {
  int first, count, rotary_dim, start, context;
  bool interleaved, has_positions;
  double base, factor, low_turns, high_turns, magnitude;
};
typedef RotaryClosure<0> RotaryForwardClosure;
typedef RotaryClosure<1> RotaryBackwardClosure;
enum class GateType { kSigmoid = 0, kRelu, kTanh, kSilu, kGelu };
// outputs {y, pre, h}; inputs {x, w_in, w_out}
struct GatedFFNForwardClosure {
  GateType type;
};
// outputs {dx, dw_in, dw_out, dpre}; inputs {diff, x, w_in, w_out, pre, h}
struct GatedFFNBackwardClosure {
  GateType type;
};
// outputs {params..., m..., v...}; inputs {params..., grads..., m..., v...}, `rates` and `decays` one per array
struct AdamWClosure {
  int bits, step;
  double rate, beta1, beta2, eps, weight_decay, grad_scale;
  std::vector<float> rates, decays;
};
// outputs {m..., v...}: the values that 8-bit moments stand for; inputs {m..., v...}
struct AdamWValuesClosure {};

namespace hip {

void LayerNormForward(const DataList&, const DataList&, LayerNormForwardClosure&, const Context&);
void LayerNormBackward(const DataList&, const DataList&, LayerNormBackwardClosure&, const Context&);
void AttentionForward(const DataList&, const DataList&, AttentionForwardClosure&, const Context&);
void AttentionBackward(const DataList&, const DataList&, AttentionBackwardClosure&, const Context&);
void RelativeBiasForward(const DataList&, const DataList&, RelativeBiasForwardClosure&, const Context&);
void RelativeBiasBackward(const DataList&, const DataList&, RelativeBiasBackwardClosure&, const Context&);
void RotaryForward(const DataList&, const DataList&, RotaryForwardClosure&, const Context&);
void RotaryBackward(const DataList&, const DataList&, RotaryBackwardClosure&, const Context&);
void GatedFFNForward(const DataList&, const DataList&, GatedFFNForwardClosure&, const Context&);
void GatedFFNBackward(const DataList&, const DataList&, GatedFFNBackwardClosure&, const Context&);
void AdamWStep(const DataList&, const DataList&, AdamWClosure&, const Context&);
void AdamWValues(const DataList&, const DataList&, AdamWValuesClosure&, const Context&);

}  // namespace hip
}  // namespace minerva
