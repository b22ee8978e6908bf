// torch.ops.glr, torch.ops.rms and torch.ops.gradclip: the operators that stand around the recurrences in a model, as
// adapters to the C ABI (include/t2fw_b200.h).  None has a counterpart in the reference.
#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "torch_ops.h"
#include "torch_util.h"

namespace t2fw_ops {

// ---- gated linear recurrence ---------------------------------------------------------------------
namespace {

// Bytes [a, a + size) of two dense tensors that share some.
bool overlap(const at::Tensor &a, const at::Tensor &b) {
  const auto pa = reinterpret_cast<uintptr_t>(a.data_ptr()), pb = reinterpret_cast<uintptr_t>(b.data_ptr());
  return pa < pb + b.nbytes() && pb < pa + a.nbytes();
}

const void *opt_ptr(const std::optional<at::Tensor> &t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

void check_grad_state(const std::optional<at::Tensor> &grad_state, const at::Tensor &state) {
  if (opt_ptr(grad_state) == nullptr) return;
  T2FW_CHECK_INPUT(*grad_state);
  TORCH_CHECK(grad_state->sizes() == state.sizes(), "grad_state must have state's shape");
  check_same(*grad_state, state, "grad_state");
}

}  // namespace

std::vector<at::Tensor> glr_forward(const at::Tensor &value, const at::Tensor &forget, const at::Tensor &state) {
  T2FW_CHECK_INPUT(value);
  T2FW_CHECK_INPUT(forget);
  T2FW_CHECK_INPUT(state);
  TORCH_CHECK(value.dim() == 3 && state.dim() == 2, "expected value [B,T,D], state [B,D]");
  const int64_t B = value.size(0), T = value.size(1), D = value.size(2);
  TORCH_CHECK(forget.sizes() == value.sizes(), "forget must have value's shape");
  TORCH_CHECK(state.size(0) == B && state.size(1) == D, "state must be [B,D]");
  check_same(forget, value, "forget");
  check_same(state, value, "state");
  TORCH_CHECK(B > 0 && T > 0 && D > 0, "empty tensors are not supported");
  const c10::cuda::CUDAGuard guard(value.device());
  at::Tensor outputs = new_like(value), next = new_like(state);
  check_status(t2fw_glr_forward(value.data_ptr(), forget.data_ptr(), state.data_ptr(), outputs.data_ptr(), next.data_ptr(),
                                B, T, D, dtype_code(value), at::cuda::getCurrentCUDAStream().stream()),
               "glr.forward");
  return {outputs, next};
}

std::vector<at::Tensor> glr_backward(const at::Tensor &grad_output, const std::optional<at::Tensor> &grad_state,
                                     const at::Tensor &forget, const at::Tensor &outputs, const at::Tensor &state) {
  T2FW_CHECK_INPUT(grad_output);
  T2FW_CHECK_INPUT(forget);
  T2FW_CHECK_INPUT(outputs);
  T2FW_CHECK_INPUT(state);
  TORCH_CHECK(forget.dim() == 3 && state.dim() == 2, "expected forget [B,T,D], state [B,D]");
  const int64_t B = forget.size(0), T = forget.size(1), D = forget.size(2);
  TORCH_CHECK(grad_output.sizes() == forget.sizes() && outputs.sizes() == forget.sizes(),
              "grad_output and outputs must have forget's shape");
  TORCH_CHECK(state.size(0) == B && state.size(1) == D, "state must be [B,D]");
  check_same(grad_output, forget, "grad_output");
  check_same(outputs, forget, "outputs");
  check_same(state, forget, "state");
  check_grad_state(grad_state, state);
  TORCH_CHECK(B > 0 && T > 0 && D > 0, "empty tensors are not supported");
  const c10::cuda::CUDAGuard guard(forget.device());
  at::Tensor d_value = new_like(forget), d_forget = new_like(forget), d_state = new_like(state);
  check_status(t2fw_glr_backward(grad_output.data_ptr(), opt_ptr(grad_state), forget.data_ptr(), outputs.data_ptr(),
                                 state.data_ptr(), d_value.data_ptr(), d_forget.data_ptr(), d_state.data_ptr(), B, T, D,
                                 dtype_code(forget), at::cuda::getCurrentCUDAStream().stream()),
               "glr.backward");
  return {d_value, d_forget, d_state};
}

std::vector<at::Tensor> glr_fused_forward(const at::Tensor &vg, const at::Tensor &state) {
  T2FW_CHECK_INPUT(vg);
  T2FW_CHECK_INPUT(state);
  TORCH_CHECK(vg.dim() == 3 && state.dim() == 2, "expected vg [B,T,2*D], state [B,D]");
  const int64_t B = vg.size(0), T = vg.size(1), D = state.size(1);
  TORCH_CHECK(vg.size(2) % 2 == 0 && vg.size(2) / 2 == D, "vg must be [B,T,2*D]");
  TORCH_CHECK(state.size(0) == B, "state must be [B,D]");
  check_same(state, vg, "state");
  TORCH_CHECK(B > 0 && T > 0 && D > 0, "empty tensors are not supported");
  const c10::cuda::CUDAGuard guard(vg.device());
  at::Tensor outputs = new_tensor({B, T, D}, vg.scalar_type(), vg), next = new_like(state);
  check_status(t2fw_glr_fused_forward(vg.data_ptr(), state.data_ptr(), outputs.data_ptr(), next.data_ptr(), B, T, D,
                                      dtype_code(vg), at::cuda::getCurrentCUDAStream().stream()),
               "glr.fused_forward");
  return {outputs, next};
}

std::vector<at::Tensor> glr_fused_backward(const at::Tensor &grad_output, const std::optional<at::Tensor> &grad_state,
                                           const at::Tensor &vg, const at::Tensor &outputs, const at::Tensor &state) {
  T2FW_CHECK_INPUT(grad_output);
  T2FW_CHECK_INPUT(vg);
  T2FW_CHECK_INPUT(outputs);
  T2FW_CHECK_INPUT(state);
  TORCH_CHECK(vg.dim() == 3 && state.dim() == 2 && outputs.dim() == 3, "expected vg [B,T,2*D], outputs [B,T,D], state [B,D]");
  const int64_t B = vg.size(0), T = vg.size(1), D = state.size(1);
  TORCH_CHECK(vg.size(2) % 2 == 0 && vg.size(2) / 2 == D, "vg must be [B,T,2*D]");
  TORCH_CHECK(state.size(0) == B, "state must be [B,D]");
  TORCH_CHECK(outputs.size(0) == B && outputs.size(1) == T && outputs.size(2) == D, "outputs must be [B,T,D]");
  TORCH_CHECK(grad_output.sizes() == outputs.sizes(), "grad_output must have outputs' shape");
  check_same(grad_output, vg, "grad_output");
  check_same(outputs, vg, "outputs");
  check_same(state, vg, "state");
  check_grad_state(grad_state, state);
  TORCH_CHECK(B > 0 && T > 0 && D > 0, "empty tensors are not supported");
  const c10::cuda::CUDAGuard guard(vg.device());
  at::Tensor d_vg = new_like(vg), d_state = new_like(state);
  check_status(t2fw_glr_fused_backward(grad_output.data_ptr(), opt_ptr(grad_state), vg.data_ptr(), outputs.data_ptr(),
                                       state.data_ptr(), d_vg.data_ptr(), d_state.data_ptr(), B, T, D, dtype_code(vg),
                                       at::cuda::getCurrentCUDAStream().stream()),
               "glr.fused_backward");
  return {d_vg, d_state};
}

// One step into caller-owned buffers.  state_out may be state_in itself; nothing else that is written may share memory
// with anything.
void glr_decode_step(const at::Tensor &value, const at::Tensor &forget, const at::Tensor &state_in,
                     const at::Tensor &state_out, const at::Tensor &outputs) {
  T2FW_CHECK_INPUT(value);
  T2FW_CHECK_INPUT(forget);
  T2FW_CHECK_INPUT(state_in);
  T2FW_CHECK_INPUT(state_out);
  T2FW_CHECK_INPUT(outputs);
  TORCH_CHECK(value.dim() == 3 && value.size(1) == 1 && state_in.dim() == 2, "expected value [B,1,D], state [B,D]");
  const int64_t B = value.size(0), D = value.size(2);
  TORCH_CHECK(forget.sizes() == value.sizes() && outputs.sizes() == value.sizes(), "forget and outputs must have value's shape");
  TORCH_CHECK(state_in.size(0) == B && state_in.size(1) == D, "state_in must be [B,D]");
  TORCH_CHECK(state_out.sizes() == state_in.sizes(), "state_out must have state_in's shape");
  check_same(forget, value, "forget");
  check_same(state_in, value, "state_in");
  check_same(state_out, value, "state_out");
  check_same(outputs, value, "outputs");
  TORCH_CHECK(B > 0 && D > 0, "empty tensors are not supported");
  TORCH_CHECK(state_out.data_ptr() == state_in.data_ptr() || !overlap(state_out, state_in),
              "state_out must be state_in or another buffer");
  TORCH_CHECK(!overlap(outputs, value) && !overlap(outputs, forget) && !overlap(outputs, state_in) &&
                  !overlap(outputs, state_out) && !overlap(state_out, value) && !overlap(state_out, forget),
              "outputs and state_out must not share memory with another argument");
  const c10::cuda::CUDAGuard guard(value.device());
  mark_changed(state_out);
  mark_changed(outputs);
  check_status(t2fw_glr_forward(value.data_ptr(), forget.data_ptr(), state_in.data_ptr(), outputs.data_ptr(),
                                state_out.data_ptr(), B, 1, D, dtype_code(value),
                                at::cuda::getCurrentCUDAStream().stream()),
               "glr.decode_step");
}

// ---- root-mean-square norm ------------------------------------------------------------------------
namespace {

// rows of x, after the checks that all forms share
int64_t check_rms(const at::Tensor &x, const std::optional<at::Tensor> &residual, const at::Tensor &weight, double eps) {
  T2FW_CHECK_INPUT(x);
  T2FW_CHECK_INPUT(weight);
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 1 && x.size(-1) == weight.size(0), "expected x [..., D], weight [D]");
  check_same(weight, x, "weight");
  if (opt_ptr(residual) != nullptr) {
    T2FW_CHECK_INPUT(*residual);
    TORCH_CHECK(residual->sizes() == x.sizes(), "residual must have x's shape");
    check_same(*residual, x, "residual");
  }
  TORCH_CHECK(x.numel() > 0, "empty tensors are not supported");
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  return x.numel() / weight.size(0);
}

}  // namespace

std::vector<at::Tensor> rms_forward(const at::Tensor &x, const std::optional<at::Tensor> &residual, const at::Tensor &weight,
                                    double eps) {
  const int64_t rows = check_rms(x, residual, weight, eps);
  const c10::cuda::CUDAGuard guard(x.device());
  const void *r = opt_ptr(residual);
  at::Tensor y = new_like(x), sum = r != nullptr ? new_like(x) : at::Tensor();
  check_status(t2fw_rms_norm_forward(x.data_ptr(), r, weight.data_ptr(), y.data_ptr(), r != nullptr ? sum.data_ptr() : nullptr,
                                     rows, weight.size(0), eps, dtype_code(x), at::cuda::getCurrentCUDAStream().stream()),
               "rms.forward");
  if (r != nullptr) return {y, sum};
  return {y};
}

std::vector<at::Tensor> rms_backward(const at::Tensor &grad_y, const std::optional<at::Tensor> &grad_sum, const at::Tensor &s,
                                     const at::Tensor &weight, double eps) {
  const int64_t rows = check_rms(s, grad_sum, weight, eps), D = weight.size(0);
  T2FW_CHECK_INPUT(grad_y);
  TORCH_CHECK(grad_y.sizes() == s.sizes(), "grad_y must have s's shape");
  check_same(grad_y, s, "grad_y");
  const c10::cuda::CUDAGuard guard(s.device());
  at::Tensor d_s = new_like(s), d_w = new_like(weight);
  const int dt = dtype_code(s);
  const size_t sb = t2fw_rms_norm_backward_scratch_bytes(rows, D, dt);
  const c10::DataPtr scratch = make_scratch(sb);
  check_status(t2fw_rms_norm_backward(grad_y.data_ptr(), opt_ptr(grad_sum), s.data_ptr(), weight.data_ptr(), d_s.data_ptr(),
                                      d_w.data_ptr(), rows, D, eps, dt, scratch.get(), sb,
                                      at::cuda::getCurrentCUDAStream().stream()),
               "rms.backward");
  return {d_s, d_w};
}

std::vector<at::Tensor> rms_e4m3(const at::Tensor &x, const std::optional<at::Tensor> &residual, const at::Tensor &weight,
                                 double eps) {
  const int64_t rows = check_rms(x, residual, weight, eps);
  const c10::cuda::CUDAGuard guard(x.device());
  const void *r = opt_ptr(residual);
  std::vector<int64_t> one(x.sizes().begin(), x.sizes().end());
  one.back() = 1;
  at::Tensor q = new_tensor(x.sizes(), at::kFloat8_e4m3fn, x), scale = new_tensor(one, at::kFloat, x);
  at::Tensor sum = r != nullptr ? new_like(x) : at::Tensor();
  check_status(t2fw_rms_norm_e4m3(x.data_ptr(), r, weight.data_ptr(), q.data_ptr(), scale.data_ptr<float>(),
                                  r != nullptr ? sum.data_ptr() : nullptr, rows, weight.size(0), eps, dtype_code(x),
                                  at::cuda::getCurrentCUDAStream().stream()),
               "rms.e4m3");
  if (r != nullptr) return {q, scale, sum};
  return {q, scale};
}

// ---- gradient norm and clipping ---------------------------------------------------------------------
namespace {

struct List {
  std::vector<const void *> in;
  std::vector<void *> out;
  std::vector<int64_t> numel;
  std::vector<int> dtype;
  std::vector<int64_t> at;      // place in the caller's list
  bool any64 = false;
};

// The tensors that hold anything, checked.
List gather(const std::vector<at::Tensor> &tensors) {
  TORCH_CHECK(!tensors.empty(), "gradclip: no tensors");
  List l;
  for (size_t i = 0; i < tensors.size(); ++i) {
    const at::Tensor &t = tensors[i];
    TORCH_CHECK(t.defined(), "gradclip: tensor ", i, " is undefined");
    TORCH_CHECK(t.device().is_cuda(), "gradclip: tensor ", i, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == tensors[0].device(), "gradclip: tensor ", i, ": device differs from the first tensor's");
    TORCH_CHECK(t.layout() == at::kStrided && t.is_non_overlapping_and_dense() && !t.is_neg(),
                "gradclip: tensor ", i, " must be dense (each element of its memory once)");
    const int dt = dtype_code(t);
    l.any64 = l.any64 || dt == T2FW_F64;
    if (t.numel() == 0) continue;
    l.in.push_back(t.data_ptr());
    l.numel.push_back(t.numel());
    l.dtype.push_back(dt);
    l.at.push_back((int64_t)i);
  }
  return l;
}

void check_max_norm(double max_norm) { TORCH_CHECK(max_norm >= 0, "gradclip: max_norm must not be negative or NaN"); }

// Scaling in place: two tensors on the same memory would be scaled twice, by blocks that do not wait for one another.
void check_disjoint(const List &l, const std::vector<at::Tensor> &tensors) {
  std::vector<std::pair<uintptr_t, uintptr_t>> span;
  span.reserve(l.in.size());
  for (size_t i = 0; i < l.in.size(); ++i) {
    const auto p = reinterpret_cast<uintptr_t>(l.in[i]);
    span.emplace_back(p, p + tensors[l.at[i]].nbytes());
  }
  if (!std::is_sorted(span.begin(), span.end())) std::sort(span.begin(), span.end());
  for (size_t i = 1; i < span.size(); ++i)
    TORCH_CHECK(span[i].first >= span[i - 1].second, "gradclip: tensors that are scaled in place must not share memory");
}

at::Tensor call(List &l, const at::Tensor &like, double max_norm, bool scale) {
  at::Tensor total = new_tensor({}, l.any64 ? at::kDouble : at::kFloat, like);
  if (l.in.empty()) return total.zero_();
  const int64_t n = (int64_t)l.in.size();
  const size_t sb = t2fw_grad_clip_scratch_bytes(n);
  const c10::DataPtr scratch = make_scratch(sb);
  auto stream = at::cuda::getCurrentCUDAStream();
  const int tdt = l.any64 ? T2FW_F64 : T2FW_F32;
  check_status(scale ? t2fw_grad_clip(l.in.data(), l.out.data(), l.numel.data(), l.dtype.data(), n, max_norm,
                                      total.data_ptr(), tdt, scratch.get(), sb, stream.stream())
                     : t2fw_grad_norm(l.in.data(), l.numel.data(), l.dtype.data(), n, total.data_ptr(), tdt, scratch.get(),
                                      sb, stream.stream()),
               scale ? "gradclip.clip" : "gradclip.norm");
  return total;
}

}  // namespace

at::Tensor grad_norm(const std::vector<at::Tensor> &tensors) {
  List l = gather(tensors);
  const c10::cuda::CUDAGuard guard(tensors[0].device());
  return call(l, tensors[0], 0, false);
}

std::vector<at::Tensor> grad_clip(const std::vector<at::Tensor> &tensors, double max_norm) {
  List l = gather(tensors);
  check_max_norm(max_norm);
  const c10::cuda::CUDAGuard guard(tensors[0].device());
  // One allocation for all results, each at a multiple of 512 bytes: one from the allocator for each took 21 of 29 us for 28
  // small tensors.  They are tensors of their own on one storage, not views of one another.
  std::vector<at::Tensor> r(1);
  r.reserve(tensors.size() + 1);
  size_t bytes = 0;
  auto room = [](const at::Tensor &t) { return (t.nbytes() + 511) / 512 * 512; };
  for (const at::Tensor &t : tensors) bytes += room(t);
  auto *allocator = c10::cuda::CUDACachingAllocator::get();
  const c10::Storage storage(c10::Storage::use_byte_size_t(), bytes, allocator->allocate(bytes), allocator, /*resizable=*/false);
  size_t at = 0;
  for (const at::Tensor &t : tensors) {
    r.emplace_back(at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage), c10::DispatchKeySet(c10::DispatchKey::CUDA),
                                                            t.dtype()));
    r.back().unsafeGetTensorImpl()->set_sizes_and_strides(t.sizes(), t.strides(), (int64_t)(at / t.itemsize()));
    at += room(t);
  }
  for (const int64_t i : l.at) l.out.push_back(r[i + 1].data_ptr());
  r[0] = call(l, tensors[0], max_norm, true);
  return r;
}

at::Tensor grad_clip_(const std::vector<at::Tensor> &tensors, double max_norm) {
  List l = gather(tensors);
  check_max_norm(max_norm);
  check_disjoint(l, tensors);
  const c10::cuda::CUDAGuard guard(tensors[0].device());
  for (const int64_t i : l.at) l.out.push_back(tensors[i].data_ptr());
  // what saved one of these tensors for a backward pass is to notice
  for (const at::Tensor &t : tensors) t.unsafeGetTensorImpl()->bump_version();
  return call(l, tensors[0], max_norm, true);
}

}  // namespace t2fw_ops

using namespace t2fw_ops;

TORCH_LIBRARY(glr, m) {
  m.def("forward", glr_forward);
  m.def("backward", glr_backward);
  m.def("fused_forward", glr_fused_forward);
  m.def("fused_backward", glr_fused_backward);
  m.def("decode_step(Tensor value, Tensor forget, Tensor state_in, Tensor(a!) state_out, Tensor(b!) outputs) -> ()",
        glr_decode_step);
}

TORCH_LIBRARY(rms, m) {
  m.def("forward", rms_forward);
  m.def("backward", rms_backward);
  m.def("e4m3", rms_e4m3);
}

TORCH_LIBRARY(gradclip, m) {
  m.def("norm", grad_norm);
  m.def("clip", grad_clip);
  m.def("clip_(Tensor(a!)[] tensors, float max_norm) -> Tensor", grad_clip_);
}
