// Log probabilities of tokens on torch tensors: checks of the arguments, outputs, one b200q_* call on the current stream.  Shared by the
// torch.library shim (torch_ops.cpp) and the native Python calls (python_calls.cpp).
#pragma once

#include "paged_calls.h"

namespace b200q_calls {
namespace {

using Scores = std::tuple<Tensor, Tensor, Tensor, Tensor>;

Scores score_outputs(const Tensor& logits, int64_t top) {
  const char* op = "b200_token_log_probs";
  TORCH_CHECK(logits.dim() >= 1, op, ": expected logits [.., vocabulary], got ", logits.sizes());
  TORCH_CHECK_VALUE(top >= 0 && top <= 64 && top <= logits.size(-1), op, ": the most likely tokens are up to 64 of the vocabulary (", logits.size(-1), "), got ", top);
  auto shape = logits.sizes().vec();
  shape.pop_back();
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor log_probs = at::empty(shape, f32), entropy = at::empty(shape, f32);
  shape.push_back(top);
  return {log_probs, entropy, at::empty(shape, f32), at::empty(shape, f32.dtype(at::kInt))};
}

Scores token_log_probs(const Tensor& logits, const std::optional<Tensor>& tokens, int64_t top, double scale) {
  const char* op = "b200_token_log_probs";
  TORCH_CHECK(logits.is_cuda(), op, ": b200q operates on CUDA tensors only; there is no CPU implementation");
  TORCH_CHECK_VALUE(logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kHalf || logits.scalar_type() == at::kBFloat16, op, " received an input of ",
                    logits.scalar_type(), " type. Supported types: float32 | float16 | bfloat16");
  TORCH_CHECK_VALUE(scale > 0.0 && std::isfinite(static_cast<float>(scale)) && static_cast<float>(scale) > 0.0f, op, ": scale must be positive and finite, got ", scale);
  c10::cuda::CUDAGuard guard(logits.device());
  Scores out = score_outputs(logits, top);
  TORCH_CHECK_VALUE(logits.size(-1) > 0, op, ": the vocabulary is empty, got logits ", logits.sizes());
  Tensor t;
  if (tokens.has_value()) {
    TORCH_CHECK(tokens->sizes() == std::get<0>(out).sizes() && tokens->device() == logits.device() &&
                    (tokens->scalar_type() == at::kInt || tokens->scalar_type() == at::kLong),
                op, ": tokens must be int32 or int64 ", std::get<0>(out).sizes(), " on the device of the logits, got ", tokens->sizes(), " of ", tokens->scalar_type());
    t = tokens->contiguous();
  } else {
    std::get<0>(out).zero_();                            // no token anywhere
  }
  if (std::get<0>(out).numel() == 0) return out;
  // rows one stride apart, a row contiguous
  Tensor x = logits.dim() == 2 ? logits : logits.reshape({-1, logits.size(-1)});
  if (x.size(1) > 1 && x.stride(1) != 1) x = x.contiguous();
  const int dt = x.scalar_type() == at::kFloat ? B200Q_F32 : (x.scalar_type() == at::kHalf ? B200Q_F16 : B200Q_BF16);
  must_be_ok(b200q_token_log_probs(x.data_ptr(), dt, x.size(0), x.size(1), outer_stride(x, 0), t.defined() ? t.data_ptr() : nullptr,
                                   t.defined() && t.scalar_type() == at::kLong ? 8 : 4, static_cast<float>(scale),
                                   t.defined() ? std::get<0>(out).data_ptr<float>() : nullptr, std::get<1>(out).data_ptr<float>(), top,
                                   top > 0 ? std::get<2>(out).data_ptr<float>() : nullptr, top > 0 ? std::get<3>(out).data_ptr<int32_t>() : nullptr, stream_of_call()),
             "b200q_token_log_probs");
  return out;
}

}  // namespace
}  // namespace b200q_calls
