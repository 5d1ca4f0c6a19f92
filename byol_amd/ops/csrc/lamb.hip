// One LAMB step over a list of parameters (You et al., arXiv:1904.00962):
//
//   g' = c g                    c: the global-norm clipping factor, or 1
//   m  = b1 m + (1 - b1) g'     v = b2 v + (1 - b2) g'^2
//   u  = (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps) + wd p
//   r  = |p| / |u| over the tensor, 1 where either norm is not above 0
//   p  = p - lr r u
//
// r needs all of u before the first value of p may change.  Reading a tensor
// twice for that moves 40 bytes for each fp32 element in the place of 28, so a
// block keeps its chunk on the chip instead: u in registers, p in LDS.  It
// publishes its sums of p^2 and u^2, waits until all chunks of its tensor have,
// and then updates p, which is read once and written once.
//
// The wait needs the other blocks to run at the same time, which nothing
// guarantees: a tensor may have more chunks than fit the chip, and other work
// may hold it.  So only the last chunks of a tensor wait: one for each CU (8.4 M
// elements), or two of the smaller ones of a short list (4.2 M).  A wait ends
// after a set time, and a block that does not wait, or gave up, leaves its part
// of p to a second pass, which reads p, m and v again and computes the same
// values.
//
// Bound by memory: 37 M parameters (ResNet-50 with its heads) take 202 us in
// one launch, 5.1 TB/s, 76 M (ResNet-200) 373 us, 5.7 TB/s.  Two passes over all
// tensors took 257 us for the first.  All of p, m and v is read and written past
// the caches, where nothing is left of it until the next step (262 us for 250
// without that, at 8192 elements a block).
#include "multi_tensor.h"

#include <algorithm>
#include <cmath>

namespace {

// A block of 512 threads keeps 32768 elements: 64 values of u and 28 of p in
// a thread's registers, 36 of p in 72 KB of LDS, so that two blocks share a CU
// and 16.7 M elements are on the chip at a time.  The more, the less the
// blocks of a large tensor stand still: ResNet-50's step (37 M elements, one
// tensor of 8.4 M) takes 250 us with 8192 elements in each of 5 blocks of 256
// threads, 232 us with 16384 in each of 3, and 229 us so; ResNet-200's with its
// clipping 519, 489 and 462 us (in the order of the modules, see below).
//
// Short lists would leave CUs idle at that size: their blocks take 8192, all in
// registers.  2 M elements took 22 us so and 33 us otherwise, 4.1 M 32 and 36,
// 5 M (where not all blocks of a tensor may wait any more) 48 and 38.
constexpr int kLambBlock = 512;
constexpr int kLongPacks = 16;  // packs of 4 elements of one thread
constexpr int kShortPacks = 4;
constexpr int64_t kShortList = int64_t(1) << 22;  // elements

// Of a thread's packs, those with p in LDS, the others in registers.
constexpr int lds_packs(int packs) { return packs == kLongPacks ? 9 : 0; }

// Blocks that share a CU: by LDS and 128 registers, or by 80 registers.
constexpr int blocks_per_cu(int packs) { return packs == kLongPacks ? 2 : 3; }

// Elements of a block.
constexpr int chunk_of(int packs) { return kLambBlock * 4 * packs; }

// The tensors of a step in device memory, and what its blocks tell each other.
struct LambList {
  float** p;
  const void** g;
  float** m;
  float** v;
  uint32_t* len;
  int* first;
  float* decay;
  int count;       // tensors
  int chunks;      // of all of them
  uint32_t chunk;  // elements
  int max_wait;    // the most chunks of a tensor that wait for each other
  uint64_t* sums;  // 2 for each chunk: of p^2, of u^2, as bits of doubles
  double* totals;  // 2 for each tensor of more than kMaxJoined chunks
  int* done;       // for each chunk: p is updated
  int* undone;     // whether any chunk is left to the second pass
};

// A piece of the list as a kernel argument (under 4 KB): each array's tensors
// by their distance in elements from the lowest of them.
constexpr int kPieceTensors = 126;

struct LambPiece {
  float* p;
  const char* g;
  float* m;
  float* v;
  uint32_t to_p[kPieceTensors];
  uint32_t to_g[kPieceTensors];
  uint32_t to_m[kPieceTensors];
  uint32_t to_v[kPieceTensors];
  uint32_t len[kPieceTensors];
  int first[kPieceTensors];
  float decay[kPieceTensors];
  int at, count, grad_size;
};

struct LambRates {
  float beta1, beta2, rest1, rest2;  // rest = 1 - beta
  float unbias1, unbias2;            // 1 / (1 - beta^t)
  float eps, lr;
};

typedef float Pack4 __attribute__((ext_vector_type(4), aligned(4)));

// Writes a piece of the list; the first piece's launch also clears what the
// blocks tell each other.
__global__ __launch_bounds__(kLambBlock) void lamb_list_kernel(
    const LambPiece piece, LambList list) {
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < piece.count; i += kLambBlock) {
      const int k = piece.at + i;
      list.p[k] = piece.p + piece.to_p[i];
      list.g[k] = piece.g + size_t(piece.to_g[i]) * piece.grad_size;
      list.m[k] = piece.m + piece.to_m[i];
      list.v[k] = piece.v + piece.to_v[i];
      list.len[k] = piece.len[i];
      list.first[k] = piece.first[i];
      list.decay[k] = piece.decay[i];
    }
  }
  if (piece.at != 0) return;
  const int i0 = blockIdx.x * kLambBlock + threadIdx.x;
  if (i0 == 0) {
    *list.undone = 0;
    list.first[list.count] = list.chunks;
  }
  for (int i = i0; i < list.chunks; i += gridDim.x * kLambBlock) {
    list.sums[2 * i] = kNoSum;
    list.sums[2 * i + 1] = kNoSum;
    list.done[i] = 0;
  }
}

__device__ __forceinline__ float lamb_rate(float p, float m, float v,
                                           float decay, const LambRates& r) {
  return fmaf(decay, p,
              (m * r.unbias1) / (sqrtf(v * r.unbias2) + r.eps));
}

// -lr |p| / |u| from the sums of squares
__device__ __forceinline__ float lamb_factor(double pp, double uu, float lr) {
  const double ratio = (pp > 0.0 && uu > 0.0) ? sqrt(pp) / sqrt(uu) : 1.0;
  return -static_cast<float>(lr * ratio);
}

// Adds up the sums of chunks [c0, c1) over the block, in a fixed order.  Each
// sum is valid by itself (it is not kNoSum), so no other order between blocks
// is needed.  With kWait, sums that are missing are waited for until the time
// is up; returns whether all were there, the same in all threads.
template <bool kWait>
__device__ __forceinline__ bool join_sums(const uint64_t* sums, int c0, int c1,
                                          uint64_t wait_ticks, double* scratch,
                                          double* pp, double* uu) {
  const uint64_t start = kWait ? wall_clock64() : 0;
  bool all = true;
  double p = 0.0, u = 0.0;
  for (int k = c0 + (int)threadIdx.x; k < c1 && all; k += kLambBlock) {
    uint64_t a = load_sum(sums + 2 * k), b = load_sum(sums + 2 * k + 1);
    while (a == kNoSum || b == kNoSum) {
      if (!kWait || wall_clock64() - start > wait_ticks) {
        all = false;
        break;
      }
      __builtin_amdgcn_s_sleep(4);
      a = load_sum(sums + 2 * k);
      b = load_sum(sums + 2 * k + 1);
    }
    p += sum_value(a);
    u += sum_value(b);
  }
  all = __syncthreads_and(all);
  *pp = block_sum_f64<kLambBlock>(p, scratch);
  *uu = block_sum_f64<kLambBlock>(u, scratch);
  return all;
}

// The part of a tensor that one block works on, cut at multiples of the
// chunk's size from the line that its parameter begins in.  Pointers are to
// that place in each array; elements [begin, end) are the block's.
struct LambChunk {
  int tensor, c0, c1;  // and the tensor's chunks
  uint32_t begin, end;
  uint32_t first, last;  // whole packs
  uint32_t edge;  // this thread's single element before or behind, or kNone
  static constexpr uint32_t kNone = ~0u;
  float *p, *m, *v;
  const void* g;
  float decay;

  __device__ __forceinline__ LambChunk(const LambList& list, int c,
                                       int grad_size) {
    const int s = span_of_chunk(list.first, list.count, c);
    tensor = s;
    c0 = list.first[s];
    c1 = list.first[s + 1];
    const uint32_t before = line_offset(list.p[s]);
    const uint32_t at = uint32_t(c - c0) * list.chunk;
    const uint32_t stop = before + list.len[s] - at;
    begin = at == 0 ? before : 0;
    end = stop < list.chunk ? stop : list.chunk;
    const int64_t move = int64_t(at) - before;
    p = list.p[s] + move;
    m = list.m[s] + move;
    v = list.v[s] + move;
    g = static_cast<const char*>(list.g[s]) + move * grad_size;
    decay = list.decay[s];
    first = (begin + 3) / 4;
    last = end / 4;
    // before the first pack (threads 0 to 3), behind the last (4 to 7)
    const uint32_t head = first * 4 < end ? first * 4 : end;
    const uint32_t tail = last > first ? last * 4 : head;
    const uint32_t t = threadIdx.x;
    const uint32_t e = t < 4 ? begin + t : tail + t - 4;
    edge = t < 8 && e < (t < 4 ? head : end) ? e : kNone;
  }
  __device__ __forceinline__ bool whole(uint32_t size) const {
    return begin == 0 && end == size;
  }
  __device__ __forceinline__ bool has(uint32_t pack) const {
    return pack >= first && pack < last;
  }
};

constexpr int waves_per_simd(int packs) {
  return blocks_per_cu(packs) * kLambBlock / (4 * WAVE_SIZE);
}

template <typename G, int kPacks>
__global__
__launch_bounds__(kLambBlock, waves_per_simd(kPacks)) void lamb_step_kernel(
    const LambList list, LambRates r, const float* __restrict__ norm,
    double max_norm, uint64_t wait_ticks) {
  constexpr int kLdsPacks = lds_packs(kPacks);
  __shared__ Pack4 kept[kLdsPacks > 0 ? kLdsPacks * kLambBlock : 1];
  __shared__ float2 edge[8];  // p and u of single elements
  __shared__ double scratch[kLambBlock / WAVE_SIZE];
  typedef G PackG __attribute__((ext_vector_type(4), aligned(sizeof(G))));
  const int c = blockIdx.x;
  const LambChunk chunk(list, c, sizeof(G));
  const float decay = chunk.decay;
  float *p = chunk.p, *m = chunk.m, *v = chunk.v;
  const G* g = static_cast<const G*>(chunk.g);
  float factor = 1.f;
  if (norm != nullptr) {
    const double f = max_norm / (static_cast<double>(*norm) + 1e-6);
    factor = f >= 1.0 ? 1.f : static_cast<float>(f);  // NaN stays
  }
  double pp = 0.0, uu = 0.0;
  auto one = [&](float pv, float gv, float& mv, float& vv) {
    gv *= factor;
    mv = fmaf(r.beta1, mv, r.rest1 * gv);
    vv = fmaf(r.beta2, vv, r.rest2 * gv * gv);
    const float u = lamb_rate(pv, mv, vv, decay, r);
    const double pd = pv, ud = u;
    pp = fma(pd, pd, pp);
    uu = fma(ud, ud, uu);
    return u;
  };
  Pack4 u[kPacks], last[kPacks - kLdsPacks];
  auto pack = [&](int k) {
    const uint32_t i = threadIdx.x + k * kLambBlock;
    const Pack4 pv =
        __builtin_nontemporal_load(reinterpret_cast<const Pack4*>(p) + i);
    const PackG gv =
        __builtin_nontemporal_load(reinterpret_cast<const PackG*>(g) + i);
    Pack4* mi = reinterpret_cast<Pack4*>(m) + i;
    Pack4* vi = reinterpret_cast<Pack4*>(v) + i;
    Pack4 mv = __builtin_nontemporal_load(mi);
    Pack4 vv = __builtin_nontemporal_load(vi);
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      float mj = mv[j], vj = vv[j];
      u[k][j] = one(pv[j], static_cast<float>(gv[j]), mj, vj);
      mv[j] = mj;
      vv[j] = vj;
    }
    __builtin_nontemporal_store(mv, mi);
    __builtin_nontemporal_store(vv, vi);
    if (k < kLdsPacks)
      kept[k * kLambBlock + threadIdx.x] = pv;
    else
      last[k - kLdsPacks] = pv;
  };
  if (chunk.whole(chunk_of(kPacks))) {
    #pragma unroll
    for (int k = 0; k < kPacks; ++k) pack(k);
  } else {
    #pragma unroll
    for (int k = 0; k < kPacks; ++k)
      if (chunk.has(threadIdx.x + k * kLambBlock)) pack(k);
    if (chunk.edge != LambChunk::kNone) {
      const uint32_t e = chunk.edge;
      float mj = m[e], vj = v[e];
      const float pj = p[e];
      edge[threadIdx.x] =
          make_float2(pj, one(pj, static_cast<float>(g[e]), mj, vj));
      m[e] = mj;
      v[e] = vj;
    }
  }
  const int c0 = chunk.c0, c1 = chunk.c1;
  pp = block_sum_f64<kLambBlock>(pp, scratch);
  uu = block_sum_f64<kLambBlock>(uu, scratch);
  if (c1 - c0 > 1) {
    if (threadIdx.x == 0) {
      store_sum(list.sums + 2 * c, pp);
      store_sum(list.sums + 2 * c + 1, uu);
    }
    const bool waits = c1 - c <= list.max_wait && wait_ticks > 0;
    if (!waits || !join_sums<true>(list.sums, c0, c1, wait_ticks, scratch,
                                   &pp, &uu)) {
      if (threadIdx.x == 0)
        __hip_atomic_store(list.undone, 1, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
      return;  // the whole block
    }
  }
  const float step = lamb_factor(pp, uu, r.lr);
  auto update = [&](int k) {
    Pack4 pv = k < kLdsPacks ? kept[k * kLambBlock + threadIdx.x]
                             : last[k - kLdsPacks];
    #pragma unroll
    for (int j = 0; j < 4; ++j) pv[j] = fmaf(step, u[k][j], pv[j]);
    __builtin_nontemporal_store(
        pv, reinterpret_cast<Pack4*>(p) + threadIdx.x + k * kLambBlock);
  };
  if (chunk.whole(chunk_of(kPacks))) {
    #pragma unroll
    for (int k = 0; k < kPacks; ++k) update(k);
  } else {
    #pragma unroll
    for (int k = 0; k < kPacks; ++k)
      if (chunk.has(threadIdx.x + k * kLambBlock)) update(k);
    if (chunk.edge != LambChunk::kNone) {
      const float2 d = edge[threadIdx.x];
      p[chunk.edge] = fmaf(step, d.y, d.x);
    }
  }
  if (threadIdx.x == 0) list.done[c] = 1;
}

// A tensor of more chunks than this has its sums joined once before the second
// pass, where otherwise every block of it joins them (up to 32 KB).
constexpr int kMaxJoined = 2048;

__global__ __launch_bounds__(kLambBlock) void lamb_totals_kernel(
    const LambList list) {
  __shared__ double scratch[kLambBlock / WAVE_SIZE];
  const int s = blockIdx.x;
  const int c0 = list.first[s], c1 = list.first[s + 1];
  if (c1 - c0 <= kMaxJoined) return;
  double pp, uu;
  join_sums<false>(list.sums, c0, c1, 0, scratch, &pp, &uu);
  if (threadIdx.x != 0) return;
  list.totals[2 * s] = pp;
  list.totals[2 * s + 1] = uu;
}

// Updates p of the chunks that the step left undone.
__global__ __launch_bounds__(kLambBlock) void lamb_rest_kernel(
    const LambList list, LambRates r) {
  __shared__ double scratch[kLambBlock / WAVE_SIZE];
  if (*list.undone == 0) return;
  for (int c = blockIdx.x; c < list.chunks; c += gridDim.x) {
    if (list.done[c]) continue;
    const LambChunk chunk(list, c, 0);
    const int s = chunk.tensor, c0 = chunk.c0, c1 = chunk.c1;
    const float decay = chunk.decay;
    float* p = chunk.p;
    const float *m = chunk.m, *v = chunk.v;
    double pp, uu;
    if (c1 - c0 > kMaxJoined) {
      pp = list.totals[2 * s];
      uu = list.totals[2 * s + 1];
    } else {
      join_sums<false>(list.sums, c0, c1, 0, scratch, &pp, &uu);
    }
    const float step = lamb_factor(pp, uu, r.lr);
    #pragma unroll 2
    for (uint32_t i = threadIdx.x; i < chunk.last; i += kLambBlock) {
      if (i < chunk.first) continue;
      Pack4* at = reinterpret_cast<Pack4*>(p) + i;
      Pack4 pv = __builtin_nontemporal_load(at);
      const Pack4 mv =
          __builtin_nontemporal_load(reinterpret_cast<const Pack4*>(m) + i);
      const Pack4 vv =
          __builtin_nontemporal_load(reinterpret_cast<const Pack4*>(v) + i);
      #pragma unroll
      for (int j = 0; j < 4; ++j)
        pv[j] = fmaf(step, lamb_rate(pv[j], mv[j], vv[j], decay, r), pv[j]);
      __builtin_nontemporal_store(pv, at);
    }
    if (chunk.edge != LambChunk::kNone) {
      const uint32_t e = chunk.edge;
      p[e] = fmaf(step, lamb_rate(p[e], m[e], v[e], decay, r), p[e]);
    }
  }
}

// One block less for each CU than have room.  Where blocks that wait and blocks
// that do not share the chip, a CU's last place sometimes stays empty while a
// block that is waited for has not started.  On a list of 28 M elements, 20 M
// of them in one tensor, a step in two ran into the time limit with 409 of 512
// blocks waiting, one in a hundred with 320, none with 256; it takes 195 us so,
// and 230 us if none wait.
int max_wait_chunks(int packs) {
  static int cus[64] = {};
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64)
    return 0;
  if (cus[device] == 0)
    (void)hipDeviceGetAttribute(&cus[device],
                                hipDeviceAttributeMultiprocessorCount, device);
  return (blocks_per_cu(packs) - 1) * cus[device];
}

int64_t chunks_of(const LambTensor& t, int packs) {
  return (line_offset(t.p) + t.len + chunk_of(packs) - 1) / chunk_of(packs);
}

// The list's arrays one after the other in `bytes` of workspace.
LambList lay_out(char* at, int count, int chunks, size_t* bytes) {
  size_t used = 0;
  auto take = [&](size_t size) {
    char* here = at + used;
    used += (size + 15) / 16 * 16;
    return here;
  };
  LambList list;
  list.count = count;
  list.chunks = chunks;
  list.chunk = 0;
  list.max_wait = 0;
  list.p = reinterpret_cast<float**>(take(count * sizeof(float*)));
  list.g = reinterpret_cast<const void**>(take(count * sizeof(void*)));
  list.m = reinterpret_cast<float**>(take(count * sizeof(float*)));
  list.v = reinterpret_cast<float**>(take(count * sizeof(float*)));
  list.len = reinterpret_cast<uint32_t*>(take(count * sizeof(uint32_t)));
  list.first = reinterpret_cast<int*>(take((count + 1) * sizeof(int)));
  list.decay = reinterpret_cast<float*>(take(count * sizeof(float)));
  list.sums = reinterpret_cast<uint64_t*>(take(chunks * 2 * sizeof(uint64_t)));
  list.totals = reinterpret_cast<double*>(take(count * 2 * sizeof(double)));
  list.done = reinterpret_cast<int*>(take(chunks * sizeof(int)));
  list.undone = reinterpret_cast<int*>(take(sizeof(int)));
  *bytes = used;
  return list;
}

}  // namespace

LambPlan lamb_plan(const std::vector<LambTensor>& tensors) {
  int64_t total = 0;
  for (const LambTensor& t : tensors) total += t.len;
  LambPlan plan = {total <= kShortList ? kShortPacks : kLongPacks, 0};
  for (const LambTensor& t : tensors) plan.chunks += chunks_of(t, plan.packs);
  return plan;
}

int64_t lamb_workspace_bytes(int64_t count, int64_t chunks) {
  size_t bytes;
  lay_out(nullptr, static_cast<int>(count), static_cast<int>(chunks), &bytes);
  return static_cast<int64_t>(bytes);
}

void launch_lamb_step(std::vector<LambTensor>& tensors, const LambPlan& plan,
                      SpanType type, double lr, double beta1, double beta2,
                      double eps, int64_t step, const float* norm,
                      double max_norm, int64_t wait_ticks, void* workspace,
                      hipStream_t stream) {
  // The largest tensor last: its blocks all wait for one another, and nothing
  // is behind them that could have run in their place (214 us for 229 us in
  // the order of ResNet-50's modules, 226 us with the largest first).
  std::stable_sort(tensors.begin(), tensors.end(),
                   [](const LambTensor& a, const LambTensor& b) {
                     return a.len < b.len;
                   });
  LambRates r;
  r.beta1 = static_cast<float>(beta1);
  r.beta2 = static_cast<float>(beta2);
  r.rest1 = static_cast<float>(1.0 - beta1);
  r.rest2 = static_cast<float>(1.0 - beta2);
  r.unbias1 = static_cast<float>(1.0 / (1.0 - std::pow(beta1, step)));
  r.unbias2 = static_cast<float>(1.0 / (1.0 - std::pow(beta2, step)));
  r.eps = static_cast<float>(eps);
  r.lr = static_cast<float>(lr);
  const int count = static_cast<int>(tensors.size());
  const int n = static_cast<int>(plan.chunks);
  size_t bytes;
  LambList list = lay_out(static_cast<char*>(workspace), count, n, &bytes);
  list.chunk = chunk_of(plan.packs);
  list.max_wait = max_wait_chunks(plan.packs);
  const dim3 block(kLambBlock);
  bool long_tensors = false;
  int first = 0;
  const int grad_size = element_size(type);
  for (int at = 0, next; at < count; at = next) {
    Reach p, g, m, v;
    for (next = at; next < count && next - at < kPieceTensors; ++next) {
      const LambTensor& t = tensors[next];
      // all four, or none of them
      if (!p.fits(t.p, 4) || !g.fits(t.g, grad_size) || !m.fits(t.m, 4) ||
          !v.fits(t.v, 4))
        break;
      p.add(t.p);
      g.add(t.g);
      m.add(t.m);
      v.add(t.v);
    }
    LambPiece piece;
    piece.p = reinterpret_cast<float*>(p.low);
    piece.g = reinterpret_cast<const char*>(g.low);
    piece.m = reinterpret_cast<float*>(m.low);
    piece.v = reinterpret_cast<float*>(v.low);
    piece.at = at;
    piece.count = next - at;
    piece.grad_size = grad_size;
    for (int i = 0; i < piece.count; ++i) {
      const LambTensor& t = tensors[at + i];
      piece.to_p[i] = p.distance(t.p, 4);
      piece.to_g[i] = g.distance(t.g, grad_size);
      piece.to_m[i] = m.distance(t.m, 4);
      piece.to_v[i] = v.distance(t.v, 4);
      piece.len[i] = static_cast<uint32_t>(t.len);
      piece.first[i] = first;
      piece.decay[i] = t.decay;
      const int own = static_cast<int>(chunks_of(t, plan.packs));
      first += own;
      long_tensors = long_tensors || own > kMaxJoined;
    }
    const int blocks = at == 0 ? grid_1d(n, kLambBlock, 64) : 1;
    hipLaunchKernelGGL(lamb_list_kernel, dim3(blocks), block, 0, stream, piece,
                       list);
  }
  with_element_type(type, [&](auto value) {
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(n), block, 0, stream, list, r, norm,
                         max_norm, static_cast<uint64_t>(wait_ticks));
    };
    using G = decltype(value);
    if (plan.packs == kShortPacks)
      launch(lamb_step_kernel<G, kShortPacks>);
    else
      launch(lamb_step_kernel<G, kLongPacks>);
  });
  if (long_tensors)
    hipLaunchKernelGGL(lamb_totals_kernel, dim3(count), block, 0, stream,
                       list);
  if (n > count)  // some tensor has more than one chunk
    hipLaunchKernelGGL(lamb_rest_kernel, dim3(std::min(n, 1024)), block, 0,
                       stream, list, r);
}
