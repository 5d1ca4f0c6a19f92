// Lists of tensors as kernel arguments, for the kernels that pass once over
// all gradients or parameters of a model (gradclip.hip, lamb.hip).
//
// A list travels inside kernels' own argument blocks, so a step copies nothing
// from host memory, keeps nothing of its inputs between calls, and a captured
// graph holds its own copy.  The argument block is kept under 4 KB, hence the
// table sizes; longer lists take several launches.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <vector>

#include "common.h"
#include "tensor_span.h"

inline int element_size(SpanType type) {
  return type == SpanType::kF32 ? 4 : 2;
}

// f(value of the element type): the type of the argument picks the kernel.
template <typename F>
void with_element_type(SpanType type, F f) {
  if (type == SpanType::kF32)
    f(float());
  else if (type == SpanType::kBF16)
    f(__bf16());
  else
    f(_Float16());
}

constexpr int kSpanBlock = 256;

// Addresses that are all within 2^32 elements of the lowest, so that a table
// can hold their distances from it.
struct Reach {
  uintptr_t low = UINTPTR_MAX, high = 0;

  bool fits(const void* at, int64_t size) const {
    const auto a = reinterpret_cast<uintptr_t>(at);
    const uintptr_t l = a < low ? a : low, h = a > high ? a : high;
    return (h - l) / size <= UINT32_MAX;
  }
  void add(const void* at) {
    const auto a = reinterpret_cast<uintptr_t>(at);
    low = a < low ? a : low;
    high = a > high ? a : high;
  }
  uint32_t distance(const void* at, int64_t size) const {
    return static_cast<uint32_t>((reinterpret_cast<uintptr_t>(at) - low) /
                                 size);
  }
};

// A span is cut into chunks at multiples of the chunk's size from the cache
// line that it begins in, so that every access of a wave covers whole lines:
// stores that share lines cost 15% (152 MB clamped: 66 us for 58 us), loads at
// odd 2-byte addresses 20%.
constexpr int kLineBytes = 128;

// Elements between a line's start and the address.
template <typename T>
__host__ __device__ __forceinline__ uint32_t line_offset(const T* at) {
  return static_cast<uint32_t>(
      (reinterpret_cast<uintptr_t>(at) & (kLineBytes - 1)) / sizeof(T));
}

// 16 bytes of elements, loaded and stored as one access.
template <typename T>
struct Pack {
  static constexpr int kLen = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};

// The span that chunk `c` lies in: spans are in chunk order, so it is the
// number of spans that begin at or before `c`, less one.  Each lane looks at
// count/64 entries, which costs one memory latency instead of a search's
// eight.  All lanes of the wave have to be active.
template <typename Index>
__device__ __forceinline__ int span_of_chunk(const Index* first, int count,
                                             int c) {
  const int lane = threadIdx.x & (WAVE_SIZE - 1);
  int below = 0;
  for (int j = 0; j < count; j += WAVE_SIZE) {
    const int k = j + lane;
    below += __popcll(__ballot(k < count && first[k] <= c));
  }
  return __builtin_amdgcn_readfirstlane(below - 1);
}

// The chunk of a second pass's block, which takes the chunks in the opposite
// order of the first: it begins with what was read last, and each chunk is on
// the XCD (blocks go to the 8 of them in turn) whose L2 has read it.  46 MB are
// clipped in 24 us so, in 31 us in the plain opposite order.  The grid is a
// multiple of 8; a chunk past the last one is none.
__device__ __forceinline__ int mirrored_chunk() {
  return int(gridDim.x) - 8 - int(blockIdx.x & ~7u) + int(blockIdx.x & 7u);
}

// Block sum in 64 bits, for blocks of kThreads; valid in all threads.
template <int kThreads>
__device__ __forceinline__ double block_sum_f64(double v, double* scratch) {
  #pragma unroll
  for (int off = WAVE_SIZE / 2; off > 0; off >>= 1)
    v += __shfl_xor(v, off, WAVE_SIZE);
  const int wid = threadIdx.x / WAVE_SIZE;
  if ((threadIdx.x & (WAVE_SIZE - 1)) == 0) scratch[wid] = v;
  __syncthreads();
  double out = scratch[0];
  #pragma unroll
  for (int w = 1; w < kThreads / WAVE_SIZE; ++w) out += scratch[w];
  __syncthreads();
  return out;
}

// Sums that blocks tell each other while they run: 64 bits that are written
// and read past the XCDs' own L2, and valid by themselves, so that no order
// between other accesses is needed (a release or acquire at this scope writes
// back or drops a whole L2: 1536 of them cost 70 us).
//
// A sum that is not there yet; no sum has these bits, as a NaN that comes from
// 32-bit values has zeros at its end.
constexpr uint64_t kNoSum = ~uint64_t(0);

__device__ __forceinline__ uint64_t load_sum(const uint64_t* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void store_sum(uint64_t* at, double v) {
  __hip_atomic_store(at, static_cast<uint64_t>(__double_as_longlong(v)),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ void store_no_sum(uint64_t* at) {
  __hip_atomic_store(at, kNoSum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ double sum_value(uint64_t bits) {
  return __longlong_as_double(static_cast<long long>(bits));
}
