// One LAMB step over a list of parameters (You et al., arXiv:1904.00962):
//
//   g' = c g                    c: the global-norm clipping factor, or 1
//   m  = b1 m + (1 - b1) g'     v = b2 v + (1 - b2) g'^2
//   u  = (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps) + wd p
//   r  = |p| / |u| over the tensor, 1 where either norm is not above 0
//   p  = p - lr r u
//
// r needs all of u before the first value of p may change, so a tensor takes
// two passes: the first updates the moments and leaves sum p^2 and sum u^2 of
// each chunk, the second joins its tensor's chunks, forms u again from p, m
// and v, and updates p.  Forming u again reads as much as storing it in the
// first pass and reading it back would move, and takes no workspace.
#include "multi_tensor.h"

#include <algorithm>
#include <cmath>

namespace {

// 44 bytes for each tensor: see multi_tensor.h for the limit.
constexpr int kMaxLambSpans = 80;

struct LambTable {
  float* p[kMaxLambSpans];
  const void* g[kMaxLambSpans];
  float* m[kMaxLambSpans];
  float* v[kMaxLambSpans];
  uint32_t len[kMaxLambSpans];
  int first[kMaxLambSpans + 1];
  float decay[kMaxLambSpans];
  int count;
  uint32_t chunk;
};

struct LambRates {
  float beta1, beta2, rest1, rest2;  // rest = 1 - beta
  float unbias1, unbias2;            // 1 / (1 - beta^t)
  float eps, lr;
};

__device__ __forceinline__ float lamb_rate(float p, float m, float v,
                                           float decay, const LambRates& r) {
  return fmaf(decay, p,
              (m * r.unbias1) / (sqrtf(v * r.unbias2) + r.eps));
}

template <typename G>
__global__ __launch_bounds__(kSpanBlock) void lamb_moments_kernel(
    const LambTable table, LambRates r, const float* __restrict__ norm,
    double max_norm, double2* __restrict__ sums) {
  __shared__ double scratch[kSpanBlock / WAVE_SIZE];
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
  typedef G VG __attribute__((ext_vector_type(4), aligned(sizeof(G))));
  const int c = blockIdx.x;
  const int s = span_of_chunk(table.first, table.count, c);
  const uint32_t begin = uint32_t(c - table.first[s]) * table.chunk;
  const uint32_t left = table.len[s] - begin;
  const uint32_t n = left < table.chunk ? left : table.chunk;
  const float decay = table.decay[s];
  const float* p = table.p[s] + begin;
  const G* g = static_cast<const G*>(table.g[s]) + begin;
  float* m = table.m[s] + begin;
  float* v = table.v[s] + begin;
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
  };
  const uint32_t nv = n / 4;
  for (uint32_t i = threadIdx.x; i < nv; i += kSpanBlock) {
    const V pv = reinterpret_cast<const V*>(p)[i];
    const VG gv =
        __builtin_nontemporal_load(reinterpret_cast<const VG*>(g) + i);
    V mv = reinterpret_cast<const V*>(m)[i];
    V vv = reinterpret_cast<const V*>(v)[i];
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      float mj = mv[j], vj = vv[j];
      one(pv[j], static_cast<float>(gv[j]), mj, vj);
      mv[j] = mj;
      vv[j] = vj;
    }
    reinterpret_cast<V*>(m)[i] = mv;
    reinterpret_cast<V*>(v)[i] = vv;
  }
  const uint32_t t = nv * 4 + threadIdx.x;
  if (t < n) {
    float mj = m[t], vj = v[t];
    one(p[t], static_cast<float>(g[t]), mj, vj);
    m[t] = mj;
    v[t] = vj;
  }
  const double psum = block_sum_f64<kSpanBlock>(pp, scratch);
  const double usum = block_sum_f64<kSpanBlock>(uu, scratch);
  if (threadIdx.x == 0) sums[c] = make_double2(psum, usum);
}

__global__ __launch_bounds__(kSpanBlock) void lamb_update_kernel(
    const LambTable table, LambRates r, const double2* __restrict__ sums) {
  __shared__ double scratch[kSpanBlock / WAVE_SIZE];
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
  const int c = mirrored_chunk();
  if (c >= table.first[table.count]) return;
  const int s = span_of_chunk(table.first, table.count, c);
  const int chunk0 = table.first[s], chunk1 = table.first[s + 1];
  const uint32_t begin = uint32_t(c - chunk0) * table.chunk;
  const uint32_t left = table.len[s] - begin;
  const uint32_t n = left < table.chunk ? left : table.chunk;
  const float decay = table.decay[s];
  float* p = table.p[s] + begin;
  const float* m = table.m[s] + begin;
  const float* v = table.v[s] + begin;
  double pp = 0.0, uu = 0.0;
  for (int k = chunk0 + (int)threadIdx.x; k < chunk1; k += kSpanBlock) {
    const double2 d = sums[k];
    pp += d.x;
    uu += d.y;
  }
  pp = block_sum_f64<kSpanBlock>(pp, scratch);
  uu = block_sum_f64<kSpanBlock>(uu, scratch);
  const double ratio = (pp > 0.0 && uu > 0.0) ? sqrt(pp) / sqrt(uu) : 1.0;
  const float step = -static_cast<float>(r.lr * ratio);
  const uint32_t nv = n / 4;
  for (uint32_t i = threadIdx.x; i < nv; i += kSpanBlock) {
    V* at = reinterpret_cast<V*>(p) + i;
    V pv = __builtin_nontemporal_load(at);
    const V mv =
        __builtin_nontemporal_load(reinterpret_cast<const V*>(m) + i);
    const V vv =
        __builtin_nontemporal_load(reinterpret_cast<const V*>(v) + i);
    #pragma unroll
    for (int j = 0; j < 4; ++j)
      pv[j] = fmaf(step, lamb_rate(pv[j], mv[j], vv[j], decay, r), pv[j]);
    __builtin_nontemporal_store(pv, at);
  }
  const uint32_t t = nv * 4 + threadIdx.x;
  if (t < n) p[t] = fmaf(step, lamb_rate(p[t], m[t], v[t], decay, r), p[t]);
}

// A block's least share; longer lists get larger shares, so that a tensor's
// sums, which every block of its second pass joins, stay few.
constexpr int64_t kLambChunk = 4096;
constexpr int64_t kLambChunks = 4096;

}  // namespace

int64_t lamb_workspace_doubles() { return 2 * (kLambChunks + kMaxLambSpans); }

void launch_lamb_step(const std::vector<LambTensor>& tensors, SpanType type,
                      double lr, double beta1, double beta2, double eps,
                      int64_t step, const float* norm, double max_norm,
                      double* workspace, hipStream_t stream) {
  LambRates r;
  r.beta1 = static_cast<float>(beta1);
  r.beta2 = static_cast<float>(beta2);
  r.rest1 = static_cast<float>(1.0 - beta1);
  r.rest2 = static_cast<float>(1.0 - beta2);
  r.unbias1 = static_cast<float>(1.0 / (1.0 - std::pow(beta1, step)));
  r.unbias2 = static_cast<float>(1.0 / (1.0 - std::pow(beta2, step)));
  r.eps = static_cast<float>(eps);
  r.lr = static_cast<float>(lr);
  double2* sums = reinterpret_cast<double2*>(workspace);
  for (size_t at = 0; at < tensors.size(); at += kMaxLambSpans) {
    const int count =
        static_cast<int>(std::min<size_t>(kMaxLambSpans, tensors.size() - at));
    LambTable table;
    int64_t total = 0;
    for (int i = 0; i < count; ++i) total += tensors[at + i].len;
    const int64_t share =
        (total + kLambChunks - 1) / kLambChunks + kSpanBlock * 4 - 1;
    const int64_t chunk =
        std::max(kLambChunk, share / (kSpanBlock * 4) * (kSpanBlock * 4));
    table.count = count;
    table.chunk = static_cast<uint32_t>(chunk);
    table.first[0] = 0;
    for (int i = 0; i < count; ++i) {
      const LambTensor& t = tensors[at + i];
      table.p[i] = t.p;
      table.g[i] = t.g;
      table.m[i] = t.m;
      table.v[i] = t.v;
      table.len[i] = static_cast<uint32_t>(t.len);
      table.decay[i] = t.decay;
      table.first[i + 1] =
          table.first[i] + static_cast<int>((t.len + chunk - 1) / chunk);
    }
    const dim3 grid(table.first[count]), block(kSpanBlock);
    with_element_type(type, [&](auto value) {
      hipLaunchKernelGGL((lamb_moments_kernel<decltype(value)>), grid, block,
                         0, stream, table, r, norm, max_norm, sums);
    });
    hipLaunchKernelGGL(lamb_update_kernel, dim3((grid.x + 7) / 8 * 8), block,
                       0, stream, table, r, sums);
  }
}
