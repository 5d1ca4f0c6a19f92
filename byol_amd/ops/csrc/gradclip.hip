// Global norm of a list of gradient tensors, and clipping by it or by value.
//
//   N = sqrt(sum_t sum_i g[t][i]^2)   or   N = max_t max_i |g[t][i]|
//   c = min(1, bound / (N + 1e-6)),   g <- round(c * g)
//
// One block takes one chunk of one tensor and writes one partial result, a
// single block joins the partials, and the scaling pass reads the joined
// factor from memory: nothing waits for the host and no atomics are used, so
// the same list gives the same bits.  Squares are summed in 64 bits: the sum
// neither overflows for large fp32 gradients nor loses small ones, and the
// pass stays bound by memory (two 64-bit operations for four bytes).
#include "multi_tensor.h"

#include <cmath>

namespace {

// |x| as ordered bits: NaN lies above infinity, so a maximum keeps it.
__device__ __forceinline__ uint32_t magnitude_bits(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

struct SumOfSquares {
  double acc = 0.0;
  __device__ __forceinline__ void add(float x) {
    const double d = x;
    acc = fma(d, d, acc);
  }
  __device__ __forceinline__ double join(double* scratch) {
    return block_sum_f64(acc, scratch);
  }
};

struct LargestMagnitude {
  uint32_t acc = 0;
  __device__ __forceinline__ void add(float x) {
    const uint32_t b = magnitude_bits(x);
    acc = b > acc ? b : acc;
  }
  __device__ __forceinline__ double join(double* scratch) {
    uint32_t v = acc;
    #pragma unroll
    for (int off = WAVE_SIZE / 2; off > 0; off >>= 1) {
      const uint32_t o = __shfl_xor(v, off, WAVE_SIZE);
      v = o > v ? o : v;
    }
    uint32_t* s = reinterpret_cast<uint32_t*>(scratch);
    if ((threadIdx.x & (WAVE_SIZE - 1)) == 0) s[threadIdx.x / WAVE_SIZE] = v;
    __syncthreads();
    v = s[0];
    #pragma unroll
    for (int w = 1; w < kSpanBlock / WAVE_SIZE; ++w) v = s[w] > v ? s[w] : v;
    __syncthreads();
    return static_cast<double>(__uint_as_float(v));
  }
};

template <typename T, typename Reduce>
__global__ __launch_bounds__(kSpanBlock) void grad_norm_partial_kernel(
    const SpanTable table, double* __restrict__ partial) {
  __shared__ double scratch[kSpanBlock / WAVE_SIZE];
  using V = typename Pack<T>::type;
  constexpr int L = Pack<T>::kLen;
  const int c = blockIdx.x;
  const int s = span_of_chunk(table.first, table.count, c);
  const uint32_t begin = uint32_t(c - table.first[s]) * table.chunk;
  const uint32_t left = table.len[s] - begin;
  const uint32_t n = left < table.chunk ? left : table.chunk;
  const T* g = static_cast<const T*>(table.ptr[s]) + begin;
  const V* gv = reinterpret_cast<const V*>(g);
  const uint32_t nv = n / L;
  Reduce red;
  for (uint32_t i = threadIdx.x; i < nv; i += kSpanBlock) {
    const V v = gv[i];
    #pragma unroll
    for (int j = 0; j < L; ++j) red.add(static_cast<float>(v[j]));
  }
  const uint32_t t = nv * L + threadIdx.x;
  if (t < n) red.add(static_cast<float>(g[t]));
  const double sum = red.join(scratch);
  if (threadIdx.x == 0) partial[c] = sum;
}

// out[0] = norm, out[1] = the factor for a bound (if bound >= 0)
template <bool kInf>
__global__ __launch_bounds__(kSpanBlock) void grad_norm_finish_kernel(
    const double* __restrict__ partial, int n, double bound,
    float* __restrict__ out) {
  __shared__ double scratch[kSpanBlock / WAVE_SIZE];
  double norm;
  if (kInf) {
    LargestMagnitude red;
    for (int i = threadIdx.x; i < n; i += kSpanBlock)
      red.add(static_cast<float>(partial[i]));
    norm = red.join(scratch);
  } else {
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += kSpanBlock) acc += partial[i];
    norm = sqrt(block_sum_f64(acc, scratch));
  }
  if (threadIdx.x == 0) {
    out[0] = static_cast<float>(norm);
    const double c = bound / (norm + 1e-6);
    out[1] = c >= 1.0 ? 1.f : static_cast<float>(c);  // NaN stays
  }
}

// Both clipping passes: `f` maps one value.
template <typename T, typename F>
__device__ __forceinline__ void map_chunk(const SpanTable& table, F f) {
  using V = typename Pack<T>::type;
  constexpr int L = Pack<T>::kLen;
  const int c = blockIdx.x;
  const int s = span_of_chunk(table.first, table.count, c);
  const uint32_t begin = uint32_t(c - table.first[s]) * table.chunk;
  const uint32_t left = table.len[s] - begin;
  const uint32_t n = left < table.chunk ? left : table.chunk;
  T* g = static_cast<T*>(table.ptr[s]) + begin;
  V* gv = reinterpret_cast<V*>(g);
  const uint32_t nv = n / L;
  for (uint32_t i = threadIdx.x; i < nv; i += kSpanBlock) {
    V v = gv[i];
    #pragma unroll
    for (int j = 0; j < L; ++j)
      v[j] = static_cast<T>(f(static_cast<float>(v[j])));
    gv[i] = v;
  }
  const uint32_t t = nv * L + threadIdx.x;
  if (t < n) g[t] = static_cast<T>(f(static_cast<float>(g[t])));
}

template <typename T>
__global__ __launch_bounds__(kSpanBlock) void grad_scale_kernel(
    const SpanTable table, const float* __restrict__ factor) {
  const float c = *factor;
  if (c == 1.f) return;  // nothing to clip
  map_chunk<T>(table, [c](float x) { return c * x; });
}

template <typename T>
__global__ __launch_bounds__(kSpanBlock) void grad_clamp_kernel(
    const SpanTable table, float bound) {
  // comparisons with NaN are false, so NaN stays
  map_chunk<T>(table, [bound](float x) {
    return x > bound ? bound : x < -bound ? -bound : x;
  });
}

// Elements of a chunk, the same for all launches of one call.
int64_t chunk_elements(const std::vector<TensorSpan>& spans, int elem) {
  int64_t total = 0;
  for (const TensorSpan& s : spans) total += s.len;
  const int64_t step = kSpanBlock * (16 / elem);
  const int64_t want = (total + 2047) / 2048;
  const int64_t least = 2 * step;
  const int64_t chunk = (want + step - 1) / step * step;
  const int64_t most = kMaxSpanLen;
  return chunk < least ? least : chunk > most ? most : chunk;
}

// Calls `launch(table, chunks, chunks of the launches before)` for as many
// tables as the list takes; returns the number of chunks.
template <typename Launch>
int for_tables(const std::vector<TensorSpan>& spans, int64_t chunk,
               Launch launch) {
  SpanTable table;
  table.chunk = static_cast<uint32_t>(chunk);
  table.count = 0;
  table.first[0] = 0;
  int done = 0;
  auto flush = [&]() {
    if (table.count == 0) return;
    const int chunks = table.first[table.count];
    launch(table, chunks, done);
    done += chunks;
    table.count = 0;
  };
  for (const TensorSpan& s : spans) {
    const int at = table.count++;
    table.ptr[at] = s.ptr;
    table.len[at] = static_cast<uint32_t>(s.len);
    table.first[at + 1] =
        table.first[at] + static_cast<int>((s.len + chunk - 1) / chunk);
    if (table.count == kMaxSpans) flush();
  }
  flush();
  return done;
}

template <typename Reduce>
int launch_partials(const std::vector<TensorSpan>& spans, SpanType type,
                    double* partial, hipStream_t stream) {
  return for_tables(
      spans, chunk_elements(spans, element_size(type)),
      [&](const SpanTable& t, int chunks, int done) {
        with_element_type(type, [&](auto value) {
          using T = decltype(value);
          hipLaunchKernelGGL((grad_norm_partial_kernel<T, Reduce>),
                             dim3(chunks), dim3(kSpanBlock), 0, stream, t,
                             partial + done);
        });
      });
}

}  // namespace

// Partial results that launch_grad_norm_partial writes for this list.
int64_t grad_norm_partials(const std::vector<TensorSpan>& spans,
                           SpanType type) {
  const int64_t chunk = chunk_elements(spans, element_size(type));
  int64_t n = 0;
  for (const TensorSpan& s : spans) n += (s.len + chunk - 1) / chunk;
  return n;
}

void launch_grad_norm_partial(const std::vector<TensorSpan>& spans,
                              SpanType type, bool inf, double* partial,
                              hipStream_t stream) {
  if (inf)
    launch_partials<LargestMagnitude>(spans, type, partial, stream);
  else
    launch_partials<SumOfSquares>(spans, type, partial, stream);
}

void launch_grad_norm_finish(const double* partial, int64_t n, bool inf,
                             double bound, float* out, hipStream_t stream) {
  if (inf)
    hipLaunchKernelGGL((grad_norm_finish_kernel<true>), dim3(1),
                       dim3(kSpanBlock), 0, stream, partial, (int)n, bound,
                       out);
  else
    hipLaunchKernelGGL((grad_norm_finish_kernel<false>), dim3(1),
                       dim3(kSpanBlock), 0, stream, partial, (int)n, bound,
                       out);
}

void launch_grad_scale(const std::vector<TensorSpan>& spans, SpanType type,
                       const float* factor, hipStream_t stream) {
  for_tables(spans, chunk_elements(spans, element_size(type)),
             [&](const SpanTable& t, int chunks, int) {
    with_element_type(type, [&](auto value) {
      hipLaunchKernelGGL((grad_scale_kernel<decltype(value)>), dim3(chunks),
                         dim3(kSpanBlock), 0, stream, t, factor);
    });
  });
}

void launch_grad_clamp(const std::vector<TensorSpan>& spans, SpanType type,
                       float bound, hipStream_t stream) {
  for_tables(spans, chunk_elements(spans, element_size(type)),
             [&](const SpanTable& t, int chunks, int) {
    with_element_type(type, [&](auto value) {
      hipLaunchKernelGGL((grad_clamp_kernel<decltype(value)>), dim3(chunks),
                         dim3(kSpanBlock), 0, stream, t, bound);
    });
  });
}
