// The operators of torch_ops.cpp and torch_layer_ops.cpp as C++ functions, for the Python binding in torch_bind.cpp.
#pragma once

#include <ATen/ATen.h>

#include <optional>
#include <vector>

namespace t2fw_ops {

// {outputs [B,T,D], ckpt_states [B,slots,D,K]}
std::vector<at::Tensor> lfw_forward(const at::Tensor &x, const at::Tensor &f, const at::Tensor &query,
                                    const at::Tensor &key, const at::Tensor &f_key, const at::Tensor &state);
// {d_x, d_f, d_query, d_key, d_f_key, d_state}; `outputs` is only checked for its shape
std::vector<at::Tensor> lfw_backward(const at::Tensor &grad_output, const at::Tensor &grad_state,
                                     const at::Tensor &value, const at::Tensor &forget, const at::Tensor &query,
                                     const at::Tensor &key, const at::Tensor &f_key, const at::Tensor &outputs,
                                     const at::Tensor &state, const at::Tensor &ckpt_states);
void lfw_decode_step(const at::Tensor &x, const at::Tensor &f, const at::Tensor &query, const at::Tensor &key,
                     const at::Tensor &f_key, const at::Tensor &state_in, const at::Tensor &state_out,
                     const at::Tensor &outputs);
bool lfw_decode_ring(const at::Tensor &x, const at::Tensor &f, const at::Tensor &query, const at::Tensor &key,
                     const at::Tensor &f_key, const at::Tensor &state, const at::Tensor &outputs);
std::vector<at::Tensor> lfw_fused_forward(const at::Tensor &qkvg, const at::Tensor &state, int64_t n_head);
std::vector<at::Tensor> lfw_fused_backward(const at::Tensor &grad_output, const at::Tensor &grad_state,
                                           const at::Tensor &qkvg, const at::Tensor &state,
                                           const at::Tensor &ckpt_states, int64_t n_head);
// {outputs, final_state, delta}
std::vector<at::Tensor> dfw_forward(const at::Tensor &query, const at::Tensor &key, const at::Tensor &value,
                                    const at::Tensor &state);
// {d_query, d_key, d_value, d_state}
std::vector<at::Tensor> dfw_backward(const at::Tensor &grad_output, const at::Tensor &grad_state,
                                     const at::Tensor &query, const at::Tensor &key, const at::Tensor &delta_value,
                                     const at::Tensor &final_state);

// ---- torch_layer_ops.cpp ----
// {outputs [B,T,D], next_state [B,D]}
std::vector<at::Tensor> glr_forward(const at::Tensor &value, const at::Tensor &forget, const at::Tensor &state);
// {d_value, d_forget, d_state}; grad_state may be absent
std::vector<at::Tensor> glr_backward(const at::Tensor &grad_output, const std::optional<at::Tensor> &grad_state,
                                     const at::Tensor &forget, const at::Tensor &outputs, const at::Tensor &state);
std::vector<at::Tensor> glr_fused_forward(const at::Tensor &vg, const at::Tensor &state);
// {d_vg, d_state}
std::vector<at::Tensor> glr_fused_backward(const at::Tensor &grad_output, const std::optional<at::Tensor> &grad_state,
                                           const at::Tensor &vg, const at::Tensor &outputs, const at::Tensor &state);
void glr_decode_step(const at::Tensor &value, const at::Tensor &forget, const at::Tensor &state_in,
                     const at::Tensor &state_out, const at::Tensor &outputs);
// {y}, or {y, sum} with a residual
std::vector<at::Tensor> rms_forward(const at::Tensor &x, const std::optional<at::Tensor> &residual, const at::Tensor &weight,
                                    double eps);
// {d_s, d_weight}; grad_sum may be absent
std::vector<at::Tensor> rms_backward(const at::Tensor &grad_y, const std::optional<at::Tensor> &grad_sum, const at::Tensor &s,
                                     const at::Tensor &weight, double eps);
// {q, scale}, or {q, scale, sum}
std::vector<at::Tensor> rms_e4m3(const at::Tensor &x, const std::optional<at::Tensor> &residual, const at::Tensor &weight,
                                 double eps);
at::Tensor grad_norm(const std::vector<at::Tensor> &tensors);
// {total, clipped tensors ...}
std::vector<at::Tensor> grad_clip(const std::vector<at::Tensor> &tensors, double max_norm);
at::Tensor grad_clip_(const std::vector<at::Tensor> &tensors, double max_norm);

}  // namespace t2fw_ops
