// Bindings of the kernels that pass over lists of tensors (gradclip.hip,
// lamb.hip).  Everything that a kernel assumes about its tensors is checked
// here, before the first launch: nothing has been written when a call raises.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "tensor_span.h"

int64_t grad_norm_partials(const std::vector<TensorSpan>& spans,
                           SpanType type);
void launch_grad_norm_partial(const std::vector<TensorSpan>& spans,
                              SpanType type, bool inf, double* partial,
                              hipStream_t stream);
void launch_grad_norm_finish(const double* partial, int64_t n, bool inf,
                             double bound, float* out, hipStream_t stream);
void launch_grad_scale(const std::vector<TensorSpan>& spans, SpanType type,
                       const float* factor, hipStream_t stream);
void launch_grad_clamp(const std::vector<TensorSpan>& spans, SpanType type,
                       float bound, hipStream_t stream);
int64_t lamb_workspace_doubles();
void launch_lamb_step(const std::vector<LambTensor>& tensors, SpanType type,
                      double lr, double beta1, double beta2, double eps,
                      int64_t step, const float* norm, double max_norm,
                      double* workspace, hipStream_t stream);

namespace {

using Tensors = std::vector<torch::Tensor>;
using Range = std::pair<uintptr_t, uintptr_t>;

SpanType span_type(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SpanType::kF32;
    case at::kBFloat16: return SpanType::kBF16;
    case at::kHalf: return SpanType::kF16;
    default:
      TORCH_CHECK_TYPE(false, "expected fp32, bf16 or fp16 tensors, got ",
                       t.scalar_type());
  }
}

// What every list has to be; the same device comes last, so that the other
// refusals are the same with and without a GPU.
void check_list(const Tensors& list, const char* what) {
  for (const auto& t : list) {
    TORCH_CHECK_TYPE(t.defined() && t.layout() == at::kStrided, what,
                     ": expected dense (strided) tensors");
    span_type(t);
  }
}

void check_device(const Tensors& list, const char* what,
                  const torch::Device& device) {
  for (const auto& t : list)
    TORCH_CHECK_VALUE(t.device() == device, what, ": expected all tensors on ",
                      device, ", got one on ", t.device());
  TORCH_CHECK_VALUE(device.is_cuda(), what, ": expected GPU tensors");
}

void add_range(std::vector<Range>& ranges, const torch::Tensor& t) {
  if (t.numel() == 0) return;
  // the addresses that a strided tensor reaches, strides being >= 0
  int64_t reach = 1;
  for (int64_t d = 0; d < t.dim(); ++d) reach += (t.size(d) - 1) * t.stride(d);
  const auto begin = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  ranges.emplace_back(begin, begin + reach * t.element_size());
}

void check_disjoint(std::vector<Range>& ranges, const char* what) {
  if (!std::is_sorted(ranges.begin(), ranges.end()))
    std::sort(ranges.begin(), ranges.end());
  for (size_t i = 1; i < ranges.size(); ++i)
    TORCH_CHECK_VALUE(ranges[i - 1].second <= ranges[i].first, what,
                      ": a tensor is listed twice, or two share memory");
}

// `t` is only read, but from none of the (sorted, disjoint) ranges.
void check_apart(const std::vector<Range>& ranges, const torch::Tensor& t,
                 const char* what) {
  std::vector<Range> own;
  add_range(own, t);
  if (own.empty() || ranges.empty()) return;
  auto it = std::lower_bound(ranges.begin(), ranges.end(),
                             Range(own[0].second, 0));
  TORCH_CHECK_VALUE(
      it == ranges.begin() || (it - 1)->second <= own[0].first, what,
      ": a gradient shares memory with a parameter or a moment");
}

// Whether two tensors of one shape lay their elements out alike; the stride of
// a dimension of length one says nothing.
bool same_layout(const torch::Tensor& a, const torch::Tensor& b) {
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// A list as spans.  Neighbours in memory that are neighbours in the list are
// one span: the flat gradient buffer's views are a single one.
struct Spans {
  SpanType type;
  std::vector<TensorSpan> spans;
};

std::vector<Spans> spans_by_type(const Tensors& list) {
  std::vector<Spans> out;
  for (const auto& t : list) {
    int64_t left = t.numel();
    if (left == 0) continue;
    const SpanType type = span_type(t);
    auto it = std::find_if(out.begin(), out.end(),
                           [&](const Spans& s) { return s.type == type; });
    if (it == out.end()) {
      out.push_back({type, {}});
      it = out.end() - 1;
    }
    const int64_t size = t.element_size();
    auto* ptr = static_cast<char*>(const_cast<void*>(t.const_data_ptr()));
    if (!it->spans.empty()) {
      TensorSpan& last = it->spans.back();
      if (static_cast<char*>(last.ptr) + last.len * size == ptr) {
        const int64_t more = std::min(left, kMaxSpanLen - last.len);
        last.len += more;
        ptr += more * size;
        left -= more;
      }
    }
    while (left > 0) {
      const int64_t n = std::min(left, kMaxSpanLen);
      it->spans.push_back({ptr, n});
      ptr += n * size;
      left -= n;
    }
  }
  return out;
}

// Tensors whose elements do not fill one range of memory are worked on in a
// dense copy; `back` holds (tensor, copy) to be written back.
Tensors dense_list(const Tensors& list,
                   std::vector<std::pair<torch::Tensor, torch::Tensor>>* back) {
  Tensors out;
  out.reserve(list.size());
  for (const auto& t : list) {
    if (t.is_non_overlapping_and_dense()) {
      out.push_back(t);
    } else {
      out.push_back(t.contiguous());
      if (back != nullptr) back->emplace_back(t, out.back());
    }
  }
  return out;
}

// The kernels write through raw pointers: tell autograd, as an in-place
// operation does.
void mark_written(const Tensors& list) {
  for (const auto& t : list)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_writable(const Tensors& list, const char* what) {
  std::vector<Range> ranges;
  ranges.reserve(list.size());
  for (const auto& t : list) {
    TORCH_CHECK_VALUE(
        at::has_internal_overlap(t) != at::MemOverlap::Yes, what,
        ": elements of a tensor share memory (an expanded view); it cannot "
        "be written in place");
    add_range(ranges, t);
  }
  check_disjoint(ranges, what);
}

// [norm, factor] of a non-empty list
torch::Tensor norm_and_factor(const Tensors& dense, bool inf, double bound) {
  const auto stream = at::hip::getCurrentHIPStream();
  const auto groups = spans_by_type(dense);
  int64_t n = 0;
  for (const auto& g : groups) n += grad_norm_partials(g.spans, g.type);
  const auto options = dense[0].options().requires_grad(false);
  auto partial = torch::empty({n}, options.dtype(at::kDouble));
  auto out = torch::empty({2}, options.dtype(at::kFloat));
  double* at = partial.data_ptr<double>();
  for (const auto& g : groups) {
    launch_grad_norm_partial(g.spans, g.type, inf, at, stream);
    at += grad_norm_partials(g.spans, g.type);
  }
  launch_grad_norm_finish(partial.data_ptr<double>(), n, inf, bound,
                          out.data_ptr<float>(), stream);
  C10_HIP_CHECK(hipGetLastError());
  return out;
}

torch::Tensor grad_norm(const Tensors& grads, bool inf) {
  const char* what = "global_grad_norm";
  TORCH_CHECK_VALUE(!grads.empty(), what, ": no tensors");
  check_list(grads, what);
  check_device(grads, what, grads[0].device());
  const c10::DeviceGuard guard(grads[0].device());
  const auto dense = dense_list(grads, nullptr);
  return norm_and_factor(dense, inf, 0.0).select(0, 0);
}

torch::Tensor grad_clip_norm(const Tensors& grads, double max_norm, bool inf) {
  const char* what = "clip_grads_by_norm_";
  TORCH_CHECK_VALUE(!grads.empty(), what, ": no tensors");
  TORCH_CHECK_VALUE(max_norm >= 0.0, what, ": max_norm must be >= 0, got ",
                    max_norm);
  check_list(grads, what);
  check_writable(grads, what);
  check_device(grads, what, grads[0].device());
  const c10::DeviceGuard guard(grads[0].device());
  std::vector<std::pair<torch::Tensor, torch::Tensor>> back;
  const auto dense = dense_list(grads, &back);
  auto out = norm_and_factor(dense, inf, max_norm);
  const auto stream = at::hip::getCurrentHIPStream();
  for (const auto& g : spans_by_type(dense))
    launch_grad_scale(g.spans, g.type, out.data_ptr<float>() + 1, stream);
  C10_HIP_CHECK(hipGetLastError());
  for (auto& pair : back) pair.first.detach().copy_(pair.second);
  mark_written(grads);
  return out.select(0, 0);
}

void grad_clip_value(const Tensors& grads, double clip_value) {
  const char* what = "clip_grads_by_value_";
  TORCH_CHECK_VALUE(clip_value >= 0.0, what,
                    ": clip_value must be >= 0, got ", clip_value);
  if (grads.empty()) return;
  check_list(grads, what);
  check_writable(grads, what);
  check_device(grads, what, grads[0].device());
  const c10::DeviceGuard guard(grads[0].device());
  std::vector<std::pair<torch::Tensor, torch::Tensor>> back;
  const auto dense = dense_list(grads, &back);
  const auto stream = at::hip::getCurrentHIPStream();
  for (const auto& g : spans_by_type(dense))
    launch_grad_clamp(g.spans, g.type, static_cast<float>(clip_value), stream);
  C10_HIP_CHECK(hipGetLastError());
  for (auto& pair : back) pair.first.detach().copy_(pair.second);
  mark_written(grads);
}

void lamb_step(const Tensors& params, const Tensors& grads,
               const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
               const std::vector<double>& decay, int64_t step, double lr,
               double beta1, double beta2, double eps, double max_norm,
               const c10::optional<torch::Tensor>& norm) {
  const char* what = "fused_lamb_step";
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && exp_avgs.size() == n &&
                        exp_avg_sqs.size() == n && decay.size() == n,
                    what, ": lists of different lengths");
  TORCH_CHECK_VALUE(step >= 1, what, ": step counts from 1, got ", step);
  if (n == 0) return;
  std::vector<Range> ranges;
  ranges.reserve(4 * n);
  for (const auto* list : {&params, &exp_avgs, &exp_avg_sqs}) {
    check_list(*list, what);
    for (size_t i = 0; i < n; ++i) {
      const auto& t = (*list)[i];
      TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, what,
                       ": parameters and moments must be fp32, got ",
                       t.scalar_type());
      TORCH_CHECK_VALUE(t.is_non_overlapping_and_dense(), what,
                        ": parameters and moments must be dense");
      TORCH_CHECK_VALUE(t.numel() < (int64_t(1) << 31), what,
                        ": a parameter has 2^31 elements or more");
      TORCH_CHECK_VALUE(
          t.sizes() == params[i].sizes() && same_layout(t, params[i]),
          what, ": moments must have their parameter's shape and strides");
      add_range(ranges, t);
    }
  }
  check_list(grads, what);
  for (size_t i = 0; i < n; ++i) {
    TORCH_CHECK_VALUE(grads[i].sizes() == params[i].sizes(), what,
                      ": a gradient has another shape than its parameter");
    TORCH_CHECK_TYPE(grads[i].scalar_type() == grads[0].scalar_type(), what,
                     ": gradients of different types");
  }
  check_disjoint(ranges, what);
  for (const auto& g : grads) check_apart(ranges, g, what);
  const auto device = params[0].device();
  for (const auto* list : {&params, &grads, &exp_avgs, &exp_avg_sqs})
    check_device(*list, what, device);
  const float* norm_ptr = nullptr;
  if (norm.has_value()) {
    TORCH_CHECK_VALUE(norm->numel() == 1 &&
                          norm->scalar_type() == at::kFloat &&
                          norm->device() == device,
                      what, ": grad_norm must be one fp32 value on ", device);
    norm_ptr = norm->data_ptr<float>();
  }
  const c10::DeviceGuard guard(device);
  Tensors held;  // gradients in the parameters' layout, until the launches
  std::vector<LambTensor> list;
  list.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const auto& p = params[i];
    if (p.numel() == 0) continue;
    torch::Tensor g = grads[i];
    if (!same_layout(g, p)) {
      g = torch::empty_strided(p.sizes(), p.strides(), g.options()
                                   .requires_grad(false))
              .copy_(g.detach());
      held.push_back(g);
    }
    list.push_back({p.data_ptr<float>(), g.const_data_ptr(),
                    exp_avgs[i].data_ptr<float>(),
                    exp_avg_sqs[i].data_ptr<float>(), p.numel(),
                    static_cast<float>(decay[i])});
  }
  if (list.empty()) return;
  auto workspace = torch::empty(
      {lamb_workspace_doubles()},
      params[0].options().dtype(at::kDouble).requires_grad(false));
  launch_lamb_step(list, span_type(grads[0]), lr, beta1, beta2, eps, step,
                   norm_ptr, max_norm, workspace.data_ptr<double>(),
                   at::hip::getCurrentHIPStream());
  C10_HIP_CHECK(hipGetLastError());
  mark_written(params);
  mark_written(exp_avgs);
  mark_written(exp_avg_sqs);
}

}  // namespace

void bind_optim(pybind11::module& mod) {
  mod.def("grad_norm", &grad_norm, "global gradient norm (gfx950)");
  mod.def("grad_clip_norm", &grad_clip_norm,
          "clip gradients by their global norm (gfx950)");
  mod.def("grad_clip_value", &grad_clip_value,
          "clip gradients by value (gfx950)");
  mod.def("lamb_step", &lamb_step, "multi-tensor LAMB step (gfx950)",
          pybind11::arg("params"), pybind11::arg("grads"),
          pybind11::arg("exp_avgs"), pybind11::arg("exp_avg_sqs"),
          pybind11::arg("decay"), pybind11::arg("step"), pybind11::arg("lr"),
          pybind11::arg("beta1"), pybind11::arg("beta2"),
          pybind11::arg("eps"), pybind11::arg("max_norm"),
          pybind11::arg("norm") = pybind11::none());
}
