// Bindings of the kernels that pass over lists of tensors (gradclip.hip,
// lamb.hip).  Everything that a kernel assumes about its tensors is checked
// here, before the first launch: nothing has been written when a call raises.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPFunctions.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "tensor_span.h"

void make_tables(SpanGroup& group);
void launch_grad_norm_partial(const SpanGroup& group, bool inf,
                              double* partial, int64_t at, int64_t all,
                              const NormPlaces& places, int64_t wait_ticks,
                              double* full, float* rounded,
                              hipStream_t stream);
void launch_grad_norm_finish(const double* partial, int64_t n, bool inf,
                             double* full, float* rounded, hipStream_t stream);
void launch_grad_scale(const SpanGroup& group, const double* norm,
                       double bound, hipStream_t stream);
void launch_grad_clamp(const SpanGroup& group, float bound,
                       hipStream_t stream);
LambPlan lamb_plan(const std::vector<LambTensor>& tensors);
int64_t lamb_workspace_bytes(int64_t count, int64_t chunks);
void launch_lamb_step(std::vector<LambTensor>& tensors, const LambPlan& plan,
                      SpanType type, double lr, double beta1, double beta2,
                      double eps, int64_t step, const float* norm,
                      double max_norm, int64_t wait_ticks, void* workspace,
                      hipStream_t stream);

namespace {

using Range = std::pair<uintptr_t, uintptr_t>;

// A Python list of tensors, borrowed: the caller's list keeps them alive.
class TensorList {
 public:
  TensorList(const pybind11::list& list, const char* what) {
    PyObject* items = list.ptr();
    const Py_ssize_t n = PyList_GET_SIZE(items);
    refs_.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* item = PyList_GET_ITEM(items, i);
      TORCH_CHECK_TYPE(THPVariable_Check(item), what,
                       ": expected tensors, got ", Py_TYPE(item)->tp_name);
      refs_.push_back(&THPVariable_Unpack(item));
    }
  }
  size_t size() const { return refs_.size(); }
  bool empty() const { return refs_.empty(); }
  const torch::Tensor& operator[](size_t i) const { return *refs_[i]; }

 private:
  std::vector<const torch::Tensor*> refs_;
};

SpanType span_type(const torch::Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.layout() == at::kStrided, what,
                   ": expected dense (strided) tensors");
  switch (t.scalar_type()) {
    case at::kFloat: return SpanType::kF32;
    case at::kBFloat16: return SpanType::kBF16;
    case at::kHalf: return SpanType::kF16;
    default:
      TORCH_CHECK_TYPE(false, what,
                       ": expected fp32, bf16 or fp16 tensors, got ",
                       t.scalar_type());
  }
}

// Checked after everything else, so that the other refusals are the same with
// and without a GPU.
void check_device(const TensorList& list, const char* what,
                  const torch::Device& device) {
  for (size_t i = 0; i < list.size(); ++i)
    TORCH_CHECK_VALUE(list[i].device() == device, what,
                      ": expected all tensors on ", device, ", got one on ",
                      list[i].device());
  TORCH_CHECK_VALUE(device.is_cuda(), what, ": expected GPU tensors");
}

// The memory that tensors reach, to see whether any two share some.
class Ranges {
 public:
  explicit Ranges(size_t n) { ranges_.reserve(n); }

  static Range of(const torch::Tensor& t) {
    int64_t reach = 1;  // in elements, strides being >= 0
    if (t.is_non_overlapping_and_dense()) {
      reach = t.numel();
    } else {
      for (int64_t d = 0; d < t.dim(); ++d)
        reach += (t.size(d) - 1) * t.stride(d);
    }
    const auto begin = reinterpret_cast<uintptr_t>(t.const_data_ptr());
    return {begin, begin + reach * t.element_size()};
  }

  void add(const torch::Tensor& t) {
    if (t.numel() == 0) return;
    const Range r = of(t);
    ordered_ = ordered_ && (ranges_.empty() || ranges_.back() < r);
    ranges_.push_back(r);
  }

  // Sorts the ranges; whether no two of them meet.
  bool disjoint() {
    if (!ordered_) std::sort(ranges_.begin(), ranges_.end());
    ordered_ = true;
    for (size_t i = 1; i < ranges_.size(); ++i)
      if (ranges_[i - 1].second > ranges_[i].first) return false;
    return true;
  }

  // Whether none of the (disjoint) ranges reaches into `t`'s.
  bool apart_from(const torch::Tensor& t) const {
    if (t.numel() == 0) return true;
    const Range r = of(t);
    const auto it =
        std::lower_bound(ranges_.begin(), ranges_.end(), Range(r.second, 0));
    return it == ranges_.begin() || (it - 1)->second <= r.first;
  }

 private:
  std::vector<Range> ranges_;
  bool ordered_ = true;
};

// Whether two tensors of one shape lay their elements out alike; the stride of
// a dimension of length one says nothing.
bool same_layout(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.strides() == b.strides()) return true;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

// A view may stand for its memory's values negated (is_neg).  The norm and both
// clippings are the same for the two signs; the LAMB step is not.

// The kernels write through raw pointers: tell autograd, as an in-place
// operation does.
void mark_written(const TensorList& list) {
  for (size_t i = 0; i < list.size(); ++i)
    if (!list[i].is_inference()) list[i].unsafeGetTensorImpl()->bump_version();
}

// A checked list of gradients as spans of memory, by type.  Neighbours in
// memory that are neighbours in the list are one span: the flat gradient
// buffer's views are a single one.  Tensors whose elements do not fill one
// range of memory are worked on in a dense copy.
class Gradients {
 public:
  Gradients(const TensorList& list, const char* what, bool write)
      : device_(list[0].device()) {
    const size_t n = list.size();
    Ranges ranges(write ? n : 0);
    std::vector<SpanType> types(n);
    for (size_t i = 0; i < n; ++i) {
      types[i] = span_type(list[i], what);
      if (!write) continue;
      TORCH_CHECK_VALUE(
          list[i].is_non_overlapping_and_dense() ||
              at::has_internal_overlap(list[i]) != at::MemOverlap::Yes,
          what, ": elements of a tensor share memory (an expanded view); it "
          "cannot be written in place");
      ranges.add(list[i]);
    }
    TORCH_CHECK_VALUE(!write || ranges.disjoint(), what,
                      ": a tensor is listed twice, or two share memory");
    check_device(list, what, device_);
    const c10::DeviceGuard guard(device_);
    for (size_t i = 0; i < n; ++i) {
      const auto& t = list[i];
      if (t.numel() == 0) continue;
      if (t.is_non_overlapping_and_dense()) {
        add(t, types[i]);
      } else {
        copies_.emplace_back(&t, t.detach().contiguous());
        add(copies_.back().second, types[i]);
      }
    }
    for (SpanGroup& g : groups_) make_tables(g);
  }

  const std::vector<SpanGroup>& groups() const { return groups_; }
  const torch::Device& device() const { return device_; }

  void write_copies_back() const {
    for (const auto& pair : copies_) pair.first->detach().copy_(pair.second);
  }

 private:
  void add(const torch::Tensor& t, SpanType type) {
    SpanGroup* group = nullptr;
    for (SpanGroup& g : groups_)
      if (g.type == type) group = &g;
    if (group == nullptr) {
      groups_.push_back({type, {}, {}});
      group = &groups_.back();
    }
    auto& spans = group->spans;
    int64_t left = t.numel();
    const int64_t size = t.element_size();
    auto* ptr = static_cast<char*>(const_cast<void*>(t.const_data_ptr()));
    if (!spans.empty()) {
      TensorSpan& last = spans.back();
      if (static_cast<char*>(last.ptr) + last.len * size == ptr) {
        const int64_t more = std::min(left, kMaxSpanLen - last.len);
        last.len += more;
        ptr += more * size;
        left -= more;
      }
    }
    while (left > 0) {
      const int64_t n = std::min(left, kMaxSpanLen);
      spans.push_back({ptr, n});
      ptr += n * size;
      left -= n;
    }
  }

  torch::Device device_;
  std::vector<SpanGroup> groups_;
  std::vector<std::pair<const torch::Tensor*, torch::Tensor>> copies_;
};

// Places for the sums that a norm's blocks tell each other, for the current
// stream of the current device: two sets that calls take in turn, "none" in all
// of a set when a call takes it, as the call between has cleared it.  Calls on
// one stream follow each other, so they share the sets; calls on other streams
// have their own, and graphs, which may be replayed on any stream, have none.
// The sets of so many streams are kept, those of the least recent call go: a
// program may make and drop streams without end.  The memory returns to its
// stream's pool, behind the calls that use it.
class StreamSums {
 public:
  static NormPlaces get(hipStream_t stream, int64_t n) {
    const std::lock_guard<std::mutex> lock(mutex());
    const int device = c10::hip::current_device();
    if (all().size() == kStreams && all().count({device, stream}) == 0)
      all().erase(std::min_element(
          all().begin(), all().end(), [](const auto& a, const auto& b) {
            return a.second.turn < b.second.turn;
          }));
    Sets& sets = all()[{device, stream}];
    static uint64_t turns = 0;
    sets.turn = ++turns;
    if (!sets.sums.defined() || sets.size < n) {
      const int64_t size = std::max<int64_t>(2 * n, 4096);
      sets.sums = torch::full(
          {2 * size}, -1,
          torch::TensorOptions().dtype(at::kLong).device(at::kCUDA, device));
      sets.size = size;  // not if there was no memory for them
      sets.used = 0;
    }
    auto* base = reinterpret_cast<uint64_t*>(sets.sums.data_ptr<int64_t>());
    sets.next ^= 1;
    const NormPlaces places = {base + sets.next * sets.size,
                               base + (sets.next ^ 1) * sets.size, sets.used};
    sets.used = n;
    return places;
  }

  static size_t count() {
    const std::lock_guard<std::mutex> lock(mutex());
    return all().size();
  }

  // After a launch that failed: some places may be taken.
  static void forget(hipStream_t stream) {
    const std::lock_guard<std::mutex> lock(mutex());
    all().erase({c10::hip::current_device(), stream});
  }

 private:
  static constexpr size_t kStreams = 16;
  struct Sets {
    torch::Tensor sums;
    int64_t size = 0;  // of one set
    int64_t used = 0;  // places that the last call took
    int next = 0;      // the set that it took them from
    uint64_t turn = 0;
  };
  using Map = std::map<std::pair<int, hipStream_t>, Sets>;
  static std::mutex& mutex() {
    static std::mutex m;
    return m;
  }
  static Map& all() {
    static auto* map = new Map;  // never freed, so not after the runtime's end
    return *map;
  }
};

bool is_capturing(hipStream_t stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  C10_HIP_CHECK(hipStreamIsCapturing(stream, &status));
  return status != hipStreamCaptureStatusNone;
}

// The norm of a list, rounded to fp32 and, at the end of its buffer, in full.
struct Norm {
  torch::Tensor rounded;
  torch::Tensor buffer;
  const double* full;
};

// How long the block that joins a norm's sums waits for them, in 10 ns units.
constexpr int64_t kNormWaitTicks = 1000000;

Norm norm_of(const Gradients& grads, bool inf, hipStream_t stream,
             int64_t wait_ticks = kNormWaitTicks) {
  int64_t n = 0;
  for (const auto& g : grads.groups()) n += g.chunks();
  const auto options = torch::TensorOptions().device(grads.device());
  Norm norm;
  norm.rounded = torch::empty({}, options.dtype(at::kFloat));
  norm.buffer = torch::empty({n + 1}, options.dtype(at::kDouble));
  float* rounded = norm.rounded.data_ptr<float>();
  double* parts = norm.buffer.data_ptr<double>();
  double* full = parts + n;
  norm.full = full;
  NormPlaces places = {nullptr, nullptr, 0};
  if (n > 0 && !is_capturing(stream)) places = StreamSums::get(stream, n);
  int64_t at = 0;
  for (const auto& g : grads.groups()) {
    launch_grad_norm_partial(g, inf, parts, at, n, places, wait_ticks, full,
                             rounded, stream);
    at += g.chunks();
  }
  if (places.sums == nullptr)
    launch_grad_norm_finish(parts, n, inf, full, rounded, stream);
  const hipError_t launched = hipGetLastError();
  if (launched != hipSuccess && places.sums != nullptr)
    StreamSums::forget(stream);
  C10_HIP_CHECK(launched);
  return norm;
}

torch::Tensor grad_norm(const pybind11::list& list, bool inf,
                        int64_t wait_ticks) {
  const char* what = "global_grad_norm";
  TORCH_CHECK_VALUE(wait_ticks >= 0 && wait_ticks <= kNormWaitTicks, what,
                    ": wait_ticks must be 0 to ", kNormWaitTicks, ", got ",
                    wait_ticks);
  const TensorList tensors(list, what);
  TORCH_CHECK_VALUE(!tensors.empty(), what, ": no tensors");
  const Gradients grads(tensors, what, false);
  const c10::DeviceGuard guard(grads.device());
  return norm_of(grads, inf, at::hip::getCurrentHIPStream(), wait_ticks)
      .rounded;
}

torch::Tensor grad_clip_norm(const pybind11::list& list, double max_norm,
                             bool inf) {
  const char* what = "clip_grads_by_norm_";
  const TensorList tensors(list, what);
  TORCH_CHECK_VALUE(!tensors.empty(), what, ": no tensors");
  TORCH_CHECK_VALUE(max_norm >= 0.0, what, ": max_norm must be >= 0, got ",
                    max_norm);
  const Gradients grads(tensors, what, true);
  const c10::DeviceGuard guard(grads.device());
  const auto stream = at::hip::getCurrentHIPStream();
  const Norm norm = norm_of(grads, inf, stream);
  const auto& groups = grads.groups();
  for (auto g = groups.rbegin(); g != groups.rend(); ++g)
    launch_grad_scale(*g, norm.full, max_norm, stream);
  C10_HIP_CHECK(hipGetLastError());
  grads.write_copies_back();
  mark_written(tensors);
  return norm.rounded;
}

void grad_clip_value(const pybind11::list& list, double clip_value) {
  const char* what = "clip_grads_by_value_";
  const TensorList tensors(list, what);
  TORCH_CHECK_VALUE(clip_value >= 0.0, what,
                    ": clip_value must be >= 0, got ", clip_value);
  if (tensors.empty()) return;
  const Gradients grads(tensors, what, true);
  const c10::DeviceGuard guard(grads.device());
  const auto stream = at::hip::getCurrentHIPStream();
  for (const auto& g : grads.groups())
    launch_grad_clamp(g, static_cast<float>(clip_value), stream);
  C10_HIP_CHECK(hipGetLastError());
  grads.write_copies_back();
  mark_written(tensors);
}

// Whether lamb_step takes these lists together, types, layouts and devices
// being what they are; it still refuses tensors that share memory.
bool lamb_fits(const pybind11::list& param_list,
               const pybind11::list& grad_list,
               const pybind11::list& exp_avg_list,
               const pybind11::list& exp_avg_sq_list) {
  const char* what = "lamb_fits";
  const TensorList params(param_list, what), grads(grad_list, what),
      exp_avgs(exp_avg_list, what), exp_avg_sqs(exp_avg_sq_list, what);
  const size_t n = params.size();
  if (n == 0 || grads.size() != n || exp_avgs.size() != n ||
      exp_avg_sqs.size() != n)
    return false;
  const auto device = params[0].device();
  const auto grad_type = grads[0].scalar_type();
  if (!device.is_cuda() ||
      (grad_type != at::kFloat && grad_type != at::kBFloat16 &&
       grad_type != at::kHalf))
    return false;
  for (size_t i = 0; i < n; ++i) {
    const auto &p = params[i], &g = grads[i];
    if (p.numel() >= (int64_t(1) << 31) || g.device() != device ||
        g.layout() != at::kStrided || g.scalar_type() != grad_type ||
        g.sizes() != p.sizes())
      return false;
    for (const auto* t : {&p, &exp_avgs[i], &exp_avg_sqs[i]})
      if (t->layout() != at::kStrided || t->scalar_type() != at::kFloat ||
          t->device() != device || !t->is_non_overlapping_and_dense() ||
          t->is_neg() ||
          t->sizes() != p.sizes() || !same_layout(*t, p))
        return false;
  }
  return true;
}

// Returns false, and has written nothing, where tensors share memory, if that
// is not to raise.
bool lamb_step(const pybind11::list& param_list,
               const pybind11::list& grad_list,
               const pybind11::list& exp_avg_list,
               const pybind11::list& exp_avg_sq_list,
               const std::vector<double>& decay, int64_t step, double lr,
               double beta1, double beta2, double eps, double max_norm,
               const c10::optional<torch::Tensor>& norm, int64_t wait_ticks,
               bool refuse_shared) {
  const char* what = "fused_lamb_step";
  const TensorList params(param_list, what), grads(grad_list, what),
      exp_avgs(exp_avg_list, what), exp_avg_sqs(exp_avg_sq_list, what);
  const size_t n = params.size();
  TORCH_CHECK_VALUE(grads.size() == n && exp_avgs.size() == n &&
                        exp_avg_sqs.size() == n && decay.size() == n,
                    what, ": lists of different lengths");
  TORCH_CHECK_VALUE(step >= 1, what, ": step counts from 1, got ", step);
  TORCH_CHECK_VALUE(wait_ticks >= 0 && wait_ticks <= 100000, what,
                    ": wait_ticks must be 0 to 100000, got ", wait_ticks);
  if (n == 0) return true;
  Ranges written(3 * n);
  for (const auto* list : {&params, &exp_avgs, &exp_avg_sqs}) {
    for (size_t i = 0; i < n; ++i) {
      const auto& t = (*list)[i];
      const auto& p = params[i];
      TORCH_CHECK_TYPE(span_type(t, what) == SpanType::kF32, what,
                       ": parameters and moments must be fp32, got ",
                       t.scalar_type());
      TORCH_CHECK_VALUE(t.is_non_overlapping_and_dense() && !t.is_neg(), what,
                        ": parameters and moments must be dense");
      TORCH_CHECK_VALUE(t.numel() < (int64_t(1) << 31), what,
                        ": a parameter has 2^31 elements or more");
      TORCH_CHECK_VALUE(t.sizes() == p.sizes() && same_layout(t, p), what,
                        ": moments must have their parameter's shape and "
                        "strides");
      written.add(t);
    }
  }
  const SpanType grad_type = span_type(grads[0], what);
  for (size_t i = 0; i < n; ++i) {
    TORCH_CHECK_TYPE(span_type(grads[i], what) == grad_type, what,
                     ": gradients of different types");
    TORCH_CHECK_VALUE(grads[i].sizes() == params[i].sizes(), what,
                      ": a gradient has another shape than its parameter");
  }
  if (!written.disjoint()) {
    TORCH_CHECK_VALUE(!refuse_shared, what,
                      ": a tensor is listed twice, or two share memory");
    return false;
  }
  for (size_t i = 0; i < n; ++i) {
    if (written.apart_from(grads[i])) continue;
    TORCH_CHECK_VALUE(!refuse_shared, what,
                      ": a gradient shares memory with a parameter or a "
                      "moment");
    return false;
  }
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
  // gradients in their parameters' layout, with the signs that they stand for
  std::vector<torch::Tensor> held;
  std::vector<LambTensor> list;
  list.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const auto& p = params[i];
    if (p.numel() == 0) continue;
    const void* g = grads[i].const_data_ptr();
    if (!same_layout(grads[i], p) || grads[i].is_neg()) {
      held.push_back(torch::empty_strided(
          p.sizes(), p.strides(), grads[i].options().requires_grad(false)));
      held.back().copy_(grads[i].detach());
      g = held.back().const_data_ptr();
    }
    list.push_back({p.data_ptr<float>(), g, exp_avgs[i].data_ptr<float>(),
                    exp_avg_sqs[i].data_ptr<float>(), p.numel(),
                    static_cast<float>(decay[i])});
  }
  if (list.empty()) return true;
  const LambPlan plan = lamb_plan(list);
  TORCH_CHECK_VALUE(plan.chunks < (int64_t(1) << 30), what, ": too many elements");
  auto workspace = torch::empty(
      {lamb_workspace_bytes(static_cast<int64_t>(list.size()),
                            plan.chunks)},
      torch::TensorOptions().dtype(at::kByte).device(device));
  launch_lamb_step(list, plan, grad_type, lr, beta1, beta2, eps, step,
                   norm_ptr, max_norm, wait_ticks, workspace.data_ptr(),
                   at::hip::getCurrentHIPStream());
  C10_HIP_CHECK(hipGetLastError());
  mark_written(params);
  mark_written(exp_avgs);
  mark_written(exp_avg_sqs);
  return true;
}

}  // namespace

void bind_optim(pybind11::module& mod) {
  mod.def("grad_norm", &grad_norm, "global gradient norm (gfx950)",
          pybind11::arg("grads"), pybind11::arg("inf"),
          pybind11::arg("wait_ticks") = kNormWaitTicks);
  mod.def("grad_norm_streams", &StreamSums::count,
          "streams that places for a norm's sums are kept for");
  mod.def("grad_clip_norm", &grad_clip_norm,
          "clip gradients by their global norm (gfx950)");
  mod.def("grad_clip_value", &grad_clip_value,
          "clip gradients by value (gfx950)");
  mod.def("lamb_fits", &lamb_fits, "whether lamb_step takes these lists");
  mod.def("lamb_step", &lamb_step, "multi-tensor LAMB step (gfx950)",
          pybind11::arg("params"), pybind11::arg("grads"),
          pybind11::arg("exp_avgs"), pybind11::arg("exp_avg_sqs"),
          pybind11::arg("decay"), pybind11::arg("step"), pybind11::arg("lr"),
          pybind11::arg("beta1"), pybind11::arg("beta2"),
          pybind11::arg("eps"), pybind11::arg("max_norm"),
          pybind11::arg("norm") = pybind11::none(),
          // how long a block waits for the others of its tensor, in 10 ns
          // units; without a wait all long tensors take the second pass
          pybind11::arg("wait_ticks") = 20000,
          pybind11::arg("refuse_shared") = true);
}
