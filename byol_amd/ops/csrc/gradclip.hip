// Global norm of a list of gradient tensors, and clipping by it or by value.
//
//   N = sqrt(sum_t sum_i g[t][i]^2)   or   N = max_t max_i |g[t][i]|
//   c = min(1, bound / (N + 1e-6)),   g <- round(c * g)
//
// A block takes one chunk of one tensor and leaves one partial result; the last
// block joins them in a fixed order, and the scaling pass reads the norm from
// memory.  Nothing waits for the host, and no result depends on the order in
// which blocks run: a list in the same memory gives the same bits every time.
// A captured graph joins in a launch of its own, with more threads and so in
// another fixed order; that can change the last of the 64 bits.
//
// Squares are summed in 64 bits: the sum neither overflows for large fp32
// gradients nor loses small ones.  All passes are bound by memory: the norm of
// 148 MB takes 28 us (5.3 TB/s, launch and all), clamping 305 MB 100 us (6.1
// TB/s of reads and writes).  Clipping by norm has to read everything twice;
// 148 MB take 70 us, of which the second reading, which finds the latest 32 MB
// in the XCDs' L2 and most of the rest in the memory-side cache, and the
// writing take 43 us.
#include "multi_tensor.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

// |x| as ordered bits: NaN lies above infinity, so a maximum keeps it.
__device__ __forceinline__ uint32_t magnitude_bits(float x) {
  return __float_as_uint(x) & 0x7fffffffu;
}

// Four running results each, so that one value's operation does not wait for
// the one before it.
struct SumOfSquares {
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  __device__ __forceinline__ void add(float x, int j) {
    const double d = x;
    acc[j & 3] = fma(d, d, acc[j & 3]);
  }
  __device__ __forceinline__ void merge(double sum, int j) {
    acc[j & 3] += sum;
  }
  template <int kThreads>
  __device__ __forceinline__ double join(double* scratch) {
    return block_sum_f64<kThreads>((acc[0] + acc[1]) + (acc[2] + acc[3]),
                                   scratch);
  }
  static __device__ __forceinline__ double norm(double sum) {
    return sqrt(sum);
  }
};

struct LargestMagnitude {
  uint32_t acc[4] = {0, 0, 0, 0};
  __device__ __forceinline__ void add(float x, int j) {
    acc[j & 3] = max(acc[j & 3], magnitude_bits(x));
  }
  __device__ __forceinline__ void merge(double largest, int j) {
    add(static_cast<float>(largest), j);
  }
  template <int kThreads>
  __device__ __forceinline__ double join(double* scratch) {
    uint32_t v = max(max(acc[0], acc[1]), max(acc[2], acc[3]));
    #pragma unroll
    for (int off = WAVE_SIZE / 2; off > 0; off >>= 1)
      v = max(v, static_cast<uint32_t>(__shfl_xor(v, off, WAVE_SIZE)));
    uint32_t* s = reinterpret_cast<uint32_t*>(scratch);
    if ((threadIdx.x & (WAVE_SIZE - 1)) == 0) s[threadIdx.x / WAVE_SIZE] = v;
    __syncthreads();
    v = s[0];
    #pragma unroll
    for (int w = 1; w < kThreads / WAVE_SIZE; ++w) v = max(v, s[w]);
    __syncthreads();
    return static_cast<double>(__uint_as_float(v));
  }
  static __device__ __forceinline__ double norm(double largest) {
    return largest;
  }
};

// The part of a span that one block works on: `data` begins at a line's start,
// elements [begin, end) of it are the block's.
template <typename T>
struct Chunk {
  static constexpr uint32_t kLen = Pack<T>::kLen;
  T* data;
  uint32_t begin, end;

  __device__ __forceinline__ Chunk(const SpanTable& table, int c) {
    const int s = span_of_chunk(table.first, table.count, c);
    T* span = reinterpret_cast<T*>(table.base) + table.offset[s];
    const uint32_t before = line_offset(span);
    const uint32_t at = uint32_t(c - table.first[s]) * table.chunk;
    const uint32_t stop = before + table.len[s] - at;
    data = span - before + at;
    begin = at == 0 ? before : 0;
    end = stop < table.chunk ? stop : table.chunk;
  }

  // f(i) for the packs of this thread, four at a time where there are as many
  // (f4), and g(i) for single elements before the first and behind the last.
  template <typename F4, typename F, typename G>
  __device__ __forceinline__ void each(F4 f4, F f, G g) const {
    const uint32_t first = (begin + kLen - 1) / kLen, last = end / kLen;
    uint32_t i = threadIdx.x + (threadIdx.x < first ? kSpanBlock : 0);
    for (; i + 3 * kSpanBlock < last; i += 4 * kSpanBlock) f4(i);
    for (; i < last; i += kSpanBlock) f(i);
    // a chunk within one pack has no whole one: all of it is head or tail
    const uint32_t head = first * kLen < end ? first * kLen : end;
    const uint32_t tail = last > first ? last * kLen : head;
    const uint32_t t = threadIdx.x;
    if (begin + t < head) g(begin + t);
    if (tail + t < end && t < kLen) g(tail + t);
  }
};

// Above this size a list does not stay in the 256 MB memory-side cache
// between two steps.
constexpr int64_t kCachedBytes = 128 << 20;

// The single block that joins all partial results.
constexpr int kJoinBlock = 1024;

// Joins n partial results in a fixed order, for blocks of kThreads:
// load(i, v, count) gets a thread those of i, i + kThreads, ....  Returns the
// sum of squares or the largest magnitude, in all threads.
template <typename Reduce, int kThreads, typename Load>
__device__ __forceinline__ double join_partials(int n, double* scratch,
                                                Load load) {
  Reduce red;
  int i = threadIdx.x;
  for (; i + 3 * kThreads < n; i += 4 * kThreads) {
    double v[4];
    load(i, v, 4);
    #pragma unroll
    for (int k = 0; k < 4; ++k) red.merge(v[k], k);
  }
  for (; i < n; i += kThreads) {
    double v[1];
    load(i, v, 1);
    red.merge(v[0], 0);
  }
  return red.template join<kThreads>(scratch);
}

// From launches that have ended.
template <int kThreads>
struct LoadPartials {
  const double* partial;
  __device__ __forceinline__ void operator()(int i, double* v, int n) const {
    #pragma unroll
    for (int k = 0; k < n; ++k) v[k] = partial[i + k * kThreads];
  }
};

// From blocks that may still run: waits for each sum.  `missing` becomes the
// lowest place that has none when the time is up; the place is looked at once
// more then, as the block itself may have stood still.
template <int kThreads>
struct AwaitPartials {
  const uint64_t* sums;
  uint64_t until;
  int* missing;
  __device__ __forceinline__ void operator()(int i, double* v, int n) const {
    uint64_t bits[4];
    #pragma unroll
    for (int k = 0; k < n; ++k) bits[k] = load_sum(sums + i + k * kThreads);
    #pragma unroll
    for (int k = 0; k < n; ++k) {
      const int place = i + k * kThreads;
      bool late = false;
      while (bits[k] == kNoSum && !late) {
        late = wall_clock64() >= until;
        __builtin_amdgcn_s_sleep(1);
        bits[k] = load_sum(sums + place);
      }
      if (bits[k] == kNoSum && place < *missing) *missing = place;
      v[k] = sum_value(bits[k]);
    }
  }
};

// Where a norm goes: as the scaling pass reads it, and as it is returned.
struct NormOut {
  double* full;
  float* rounded;

  __device__ __forceinline__ void write(double norm) const {
    *full = norm;
    *rounded = static_cast<float>(norm);
  }
};

// How partial results become a norm.  With `sums`, the last block of the
// call's last launch joins them as they come in: a launch less, 3 us for the
// host and 4 us for the GPU.  It waits only for blocks that wait for nothing
// themselves, and only for a time: it then computes what is missing itself,
// with the same bits.
//
// A block that was late writes its sum all the same, after it was read for the
// last time.  So calls take two sets of places in turn, and each call clears
// the set of the call before it, whose blocks have all ended.
struct NormEnd {
  uint64_t* sums;   // this call's places, kNoSum in all before it; or null
  uint64_t* clear;  // the places of the call before, and how many it used
  int cleared;
  int all;          // blocks of all launches of the call
  uint64_t wait_ticks;  // of 10 ns
  NormOut out;
};

// With `partial`, `at` and the 256 bytes that the compiler adds.
static_assert(sizeof(SpanTable) + sizeof(NormEnd) + 16 + 256 <= 4096,
              "kernel arguments are at most 4 KB");

// A block's share of a norm: four packs of a thread at a time, or one (kWide
// false), in the same order and so with the same bits.
template <typename T, typename Reduce, bool kWide>
__device__ __forceinline__ double chunk_sum(const Chunk<const T>& chunk,
                                            double* scratch) {
  using V = typename Pack<T>::type;
  constexpr int L = Pack<T>::kLen;
  const V* packs = reinterpret_cast<const V*>(chunk.data);
  Reduce red;
  auto add = [&](const V& v) {
    #pragma unroll
    for (int j = 0; j < L; ++j) red.add(static_cast<float>(v[j]), j);
  };
  chunk.each(
      [&](uint32_t i) {
        if (kWide) {
          V v[4];
          #pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = packs[i + k * kSpanBlock];
          #pragma unroll
          for (int k = 0; k < 4; ++k) add(v[k]);
        } else {
          #pragma unroll 1
          for (int k = 0; k < 4; ++k) add(packs[i + k * kSpanBlock]);
        }
      },
      [&](uint32_t i) { add(packs[i]); },
      [&](uint32_t i) { red.add(static_cast<float>(chunk.data[i]), 0); });
  return red.template join<kSpanBlock>(scratch);
}

// Leaves what it reads in the caches, though streaming past them is faster by
// itself (148 MB: 26 us for 29): the step that follows reads the gradients
// again, and LAMB with its clipping takes 220 us so and 239 otherwise.
template <typename T, typename Reduce>
__global__ __launch_bounds__(kSpanBlock) void grad_norm_partial_kernel(
    const SpanTable table, double* __restrict__ partial, int at,
    const NormEnd end) {
  __shared__ double scratch[kSpanBlock / WAVE_SIZE];
  const int own = at + blockIdx.x;
  if (threadIdx.x == 0)  // here its latency is hidden, at the end it is not
    for (int i = own; i < end.cleared; i += end.all)
      store_no_sum(end.clear + i);
  const double sum = chunk_sum<T, Reduce, true>(
      Chunk<const T>(table, blockIdx.x), scratch);
  if (end.sums == nullptr) {
    if (threadIdx.x == 0) partial[own] = sum;
    return;
  }
  if (threadIdx.x == 0) store_sum(end.sums + own, sum);
  if (own != end.all - 1) return;
  const uint64_t until = wall_clock64() + end.wait_ticks;
  for (;;) {
    int missing = end.all;
    const double all = join_partials<Reduce, kSpanBlock>(
        end.all, scratch,
        AwaitPartials<kSpanBlock>{end.sums, until, &missing});
    if (!__syncthreads_or(missing < end.all)) {
      if (threadIdx.x == 0) end.out.write(Reduce::norm(all));
      return;
    }
    // launches before this one have ended, so what is missing is this one's
    int* least = reinterpret_cast<int*>(scratch);
    if (threadIdx.x == 0) *least = end.all;
    __syncthreads();
    atomicMin(least, missing);
    __syncthreads();
    const int place = *least;
    __syncthreads();
    const double late = chunk_sum<T, Reduce, false>(
        Chunk<const T>(table, place - at), scratch);
    if (threadIdx.x == 0) store_sum(end.sums + place, late);
  }
}

// The same from partial results of launches that have ended, in one block.
template <typename Reduce>
__global__ __launch_bounds__(kJoinBlock) void grad_norm_finish_kernel(
    const double* __restrict__ partial, int n, const NormOut out) {
  __shared__ double scratch[kJoinBlock / WAVE_SIZE];
  const double all = join_partials<Reduce, kJoinBlock>(
      n, scratch, LoadPartials<kJoinBlock>{partial});
  if (threadIdx.x == 0) out.write(Reduce::norm(all));
}

// Both clipping passes: `f` maps one value.
template <typename T, bool kStream, typename F>
__device__ __forceinline__ void map_chunk(const Chunk<T>& chunk, F f) {
  using V = typename Pack<T>::type;
  constexpr int L = Pack<T>::kLen;
  V* packs = reinterpret_cast<V*>(chunk.data);
  auto map = [&](V v) {
    #pragma unroll
    for (int j = 0; j < L; ++j)
      v[j] = static_cast<T>(f(static_cast<float>(v[j])));
    return v;
  };
  chunk.each(
      [&](uint32_t i) {
        V v[4];
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
          V* at = packs + i + k * kSpanBlock;
          v[k] = kStream ? __builtin_nontemporal_load(at) : *at;
        }
        #pragma unroll
        for (int k = 0; k < 4; ++k) {
          V* at = packs + i + k * kSpanBlock;
          if (kStream)
            __builtin_nontemporal_store(map(v[k]), at);
          else
            *at = map(v[k]);
        }
      },
      [&](uint32_t i) { packs[i] = map(packs[i]); },
      [&](uint32_t i) {
        chunk.data[i] = static_cast<T>(f(static_cast<float>(chunk.data[i])));
      });
}

// Streams past the caches, which 70 us for 148 MB need (95 us otherwise, 93
// with only the loads or only the stores so); what the optimizer then reads
// does not fit them in any case.
template <typename T>
__global__ __launch_bounds__(kSpanBlock) void grad_scale_kernel(
    const SpanTable table, const double* __restrict__ norm, double bound) {
  const double ratio = bound / (*norm + 1e-6);
  if (ratio >= 1.0) return;  // not for NaN
  const float f = static_cast<float>(ratio);
  const int c = mirrored_chunk();
  if (f == 1.f || c >= table.first[table.count]) return;
  map_chunk<T, true>(Chunk<T>(table, c), [f](float x) { return f * x; });
}

// Streams past the caches where the list does not fit them: 148 MB take 49 us
// so and 59 us otherwise, 74 MB 26 and 25 us.
template <typename T, bool kStream>
__global__ __launch_bounds__(kSpanBlock) void grad_clamp_kernel(
    const SpanTable table, float bound) {
  // comparisons with NaN are false, so NaN stays
  map_chunk<T, kStream>(Chunk<T>(table, blockIdx.x), [bound](float x) {
    return x > bound ? bound : x < -bound ? -bound : x;
  });
}

// A table's chunk, in elements: about kTableChunks chunks, but no less than
// two packs for each thread.
int64_t chunk_elements(int64_t total, SpanType type) {
  const int64_t step = kSpanBlock * (16 / element_size(type));
  const int64_t want = (total + kTableChunks - 1) / kTableChunks;
  return std::max(2 * step, (want + step - 1) / step * step);
}

template <typename Reduce>
void launch_partials(const SpanGroup& group, double* partial, int64_t at,
                     const NormEnd& end, hipStream_t stream) {
  for (const SpanTable& t : group.tables) {
    const int chunks = t.first[t.count];
    with_element_type(group.type, [&](auto value) {
      hipLaunchKernelGGL(
          (grad_norm_partial_kernel<decltype(value), Reduce>), dim3(chunks),
          dim3(kSpanBlock), 0, stream, t, partial, static_cast<int>(at), end);
    });
    at += chunks;
  }
}

}  // namespace

// Fills in the tables of a group's spans.
void make_tables(SpanGroup& group) {
  const auto& spans = group.spans;
  const int64_t size = element_size(group.type);
  for (size_t at = 0, next; at < spans.size(); at = next) {
    Reach reach;
    int64_t total = 0;
    for (next = at; next < spans.size() && next - at < kMaxSpans; ++next) {
      if (!reach.fits(spans[next].ptr, size)) break;
      reach.add(spans[next].ptr);
      total += spans[next].len;
    }
    group.tables.emplace_back();
    SpanTable& table = group.tables.back();
    table.base = reinterpret_cast<char*>(reach.low);
    table.count = static_cast<int>(next - at);
    const int64_t chunk = chunk_elements(total, group.type);
    table.chunk = static_cast<uint32_t>(chunk);
    int chunks = 0;
    for (int i = 0; i < table.count; ++i) {
      const TensorSpan& s = spans[at + i];
      const int64_t before =
          (reinterpret_cast<uintptr_t>(s.ptr) & (kLineBytes - 1)) / size;
      table.offset[i] = reach.distance(s.ptr, size);
      table.len[i] = static_cast<uint32_t>(s.len);
      table.first[i] = static_cast<uint16_t>(chunks);
      chunks += static_cast<int>((before + s.len + chunk - 1) / chunk);
    }
    table.first[table.count] = static_cast<uint16_t>(chunks);
  }
}

// Leaves one partial result for each chunk, from partial[at] on or in
// `places`.
void launch_grad_norm_partial(const SpanGroup& group, bool inf,
                              double* partial, int64_t at, int64_t all,
                              const NormPlaces& places, int64_t wait_ticks,
                              double* full, float* rounded,
                              hipStream_t stream) {
  const NormEnd end = {places.sums,
                       places.clear,
                       static_cast<int>(places.cleared),
                       static_cast<int>(all),
                       static_cast<uint64_t>(wait_ticks),
                       {full, rounded}};
  if (inf)
    launch_partials<LargestMagnitude>(group, partial, at, end, stream);
  else
    launch_partials<SumOfSquares>(group, partial, at, end, stream);
}

void launch_grad_norm_finish(const double* partial, int64_t n, bool inf,
                             double* full, float* rounded,
                             hipStream_t stream) {
  const NormOut out = {full, rounded};
  const int count = static_cast<int>(n);
  if (inf)
    hipLaunchKernelGGL((grad_norm_finish_kernel<LargestMagnitude>), dim3(1),
                       dim3(kJoinBlock), 0, stream, partial, count, out);
  else
    hipLaunchKernelGGL((grad_norm_finish_kernel<SumOfSquares>), dim3(1),
                       dim3(kJoinBlock), 0, stream, partial, count, out);
}

void launch_grad_scale(const SpanGroup& group, const double* norm,
                       double bound, hipStream_t stream) {
  // the tables, too, in the opposite order of the norm's pass
  for (auto t = group.tables.rbegin(); t != group.tables.rend(); ++t) {
    const int chunks = t->first[t->count];
    with_element_type(group.type, [&](auto value) {
      hipLaunchKernelGGL((grad_scale_kernel<decltype(value)>),
                         dim3((chunks + 7) / 8 * 8), dim3(kSpanBlock), 0,
                         stream, *t, norm, bound);
    });
  }
}

void launch_grad_clamp(const SpanGroup& group, float bound,
                       hipStream_t stream) {
  int64_t total = 0;
  for (const TensorSpan& s : group.spans) total += s.len;
  const bool streamed = total * element_size(group.type) > kCachedBytes;
  for (const SpanTable& t : group.tables) {
    with_element_type(group.type, [&](auto value) {
      using T = decltype(value);
      const dim3 grid(t.first[t.count]), block(kSpanBlock);
      if (streamed)
        hipLaunchKernelGGL((grad_clamp_kernel<T, true>), grid, block, 0,
                           stream, t, bound);
      else
        hipLaunchKernelGGL((grad_clamp_kernel<T, false>), grid, block, 0,
                           stream, t, bound);
    });
  }
}
