// What the bindings hand to the kernels over lists of tensors.
#pragma once

#include <cstdint>

// One dense run of elements; `ptr` needs only the element's own alignment.
struct TensorSpan {
  void* ptr;
  int64_t len;
};

// A parameter with its gradient and moments; fp32 but for the gradient.
struct LambTensor {
  float* p;
  const void* g;
  float* m;
  float* v;
  int64_t len;
  float decay;
};

// Element types of a span, as the bindings name them.
enum class SpanType { kF32, kBF16, kF16 };

// A span's length and the offsets inside of it are 32-bit; longer tensors are
// cut into several spans on the host.
constexpr int64_t kMaxSpanLen = int64_t(1) << 30;
