// Launchers of the decoder operators around the matrix products (checked arguments, current stream);
// csrc/decoder_ops.cpp has the entry points that check, allocate and record gradients.
#pragma once

#include <ATen/core/Tensor.h>
#include <c10/util/Optional.h>

#include <vector>

namespace mtorus {

using OptTensor = c10::optional<at::Tensor>;

// Rotary positions. Each segment: x [B, S, heads, D] (last stride 1) -> out (last stride 1), which may be x itself.
// The first heads_rot heads are rotated, the others copied (left alone in place).
struct RotarySegment {
  at::Tensor in, out;
  int64_t heads_rot;
};
struct RotaryArgs {
  at::Tensor turns;  // int64 [rot_dim / 2]: revolutions per position of each pair times 2^64, modulo 2^64
  int64_t rot_dim;
  bool interleaved;
  double scale;         // factor on the rotated values
  OptTensor positions;  // int32 / int64 [B, S], any strides; none: offset + index in the sequence
  int64_t offset;
  bool inverse;
  bool in_place;  // every segment's out is its in
};
void rotary_launch(const std::vector<RotarySegment>& segs, const RotaryArgs& a);

// Residual update with norms: y = beta x + alpha g * norm(h; post), n = norm(y; pre).
enum GateKind : int { kGateNone = 0, kGateChannel = 1, kGateRow = 2, kGateFull = 3 };
struct ResidualNormArgs {
  at::Tensor x;     // [T, d], last stride 1
  OptTensor h;      // [T, d], last stride 1; none: y = x (beta = 1), which is not written
  OptTensor pre, post, gate;
  int gate_kind = kGateNone;
  double beta = 1.0, alpha = 1.0, eps = 1e-6;
};
// y, n: [T, d] contiguous (undefined: not written); rstd_h, rstd_y: fp32 [T] (undefined: not written).
void residual_norm_fwd_launch(const ResidualNormArgs& a, const at::Tensor& y, const at::Tensor& n,
                              const at::Tensor& rstd_h, const at::Tensor& rstd_y);
// dy, dn: [T, d] last stride 1, either may be undefined (zero). Outputs: dx, dh [T, d] contiguous; dgate of the
// gate's type and shape; dpre, dpost fp32 [d]. Undefined outputs are not computed.
void residual_norm_bwd_launch(const ResidualNormArgs& a, const at::Tensor& rstd_h, const at::Tensor& rstd_y,
                              const at::Tensor& dy, const at::Tensor& dn, const at::Tensor& dx, const at::Tensor& dh,
                              const at::Tensor& dgate, const at::Tensor& dpre, const at::Tensor& dpost);

// Log probabilities of given tokens. logits [T, V] (last stride 1), tokens int64 [T].
// stats fp32 [T, 2]: a reference m, at most 8 / c below the row's maximum (c = log2(e) / temperature), and log2 of the sum
// of the exponentials relative to it; entropy, top_lp, top_ids may be undefined.
void token_logprobs_fwd_launch(const at::Tensor& logits, const at::Tensor& tokens, double inv_tau, int64_t top,
                               const at::Tensor& logprob, const at::Tensor& stats, const at::Tensor& entropy,
                               const at::Tensor& top_lp, const at::Tensor& top_ids);
// g_*: fp32 contiguous or undefined (zero).
void token_logprobs_bwd_launch(const at::Tensor& logits, const at::Tensor& tokens, double inv_tau, int64_t top,
                               const at::Tensor& stats, const at::Tensor& entropy, const at::Tensor& top_ids,
                               const at::Tensor& g_logprob, const at::Tensor& g_entropy, const at::Tensor& g_top,
                               const at::Tensor& dlogits);

}  // namespace mtorus
