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

// A list is worked on in tables of so many spans, each in about so many
// chunks, one block for each.  Of 512 to 8192 chunks 1536 measured best or
// within 2% of it over lists of 46 to 160 MB: fewer leave too few loads in
// flight (161 MB of fp16: 43 us with 1024, 38 us with 1536), more add sums to
// join (46 MB of fp32, clipped: 24 us with 1536, 34 us with 8192).  Each
// further table costs a launch that the one before has to drain for, about
// 7 us: so a table holds as many spans as an argument of 4 KB can.
constexpr int kMaxSpans = 352;
constexpr int kTableChunks = 1536;

// Up to so many partial results of a norm, those of one table, are joined by
// every block of the scaling pass (8 KB from L2, and a launch less: 19 us for
// 22 us on 68 MB below the bound); more are joined in a launch of their own.
constexpr int64_t kMaxJoinedPartials = kTableChunks + kMaxSpans;
