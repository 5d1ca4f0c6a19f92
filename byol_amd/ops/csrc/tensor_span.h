// What the bindings hand to the kernels over lists of tensors.
#pragma once

#include <cstdint>
#include <vector>

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

// How a LAMB step cuts its tensors: 2048 elements times `packs` for a block.
struct LambPlan {
  int packs;
  int64_t chunks;
};

// Where the blocks of a norm tell each other their sums: a call's own places,
// or null, and those of the call before it on the stream, to be cleared.
struct NormPlaces {
  uint64_t* sums;
  uint64_t* clear;
  int64_t cleared;
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
// join (46 MB of fp32, clipped: 26 us with 1536, 34 us with 8192).  Each
// further table costs a launch that the one before has to drain for, about
// 7 us.  352 spans of 10 bytes leave 500 of the 4 KB that a kernel's arguments
// may have for the others and for those that the compiler adds.
constexpr int kMaxSpans = 352;
constexpr int kTableChunks = 1536;

// A table as a kernel argument (under 4 KB).
struct SpanTable {
  char* base;  // the lowest address; offsets are in elements
  uint32_t offset[kMaxSpans];
  uint32_t len[kMaxSpans];
  uint16_t first[kMaxSpans + 1];  // a span's first chunk; [count] = all chunks
  int count;
  uint32_t chunk;  // elements, a multiple of kLineBytes
};

// Spans of one type, and their tables.
struct SpanGroup {
  SpanType type;
  std::vector<TensorSpan> spans;
  std::vector<SpanTable> tables;

  int64_t chunks() const {
    int64_t n = 0;
    for (const SpanTable& t : tables) n += t.first[t.count];
    return n;
  }
};
