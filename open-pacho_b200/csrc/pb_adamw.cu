// AdamW over many tensors at once (HBM-bound: 4 values read and 3 written per
// parameter).
//
// One launch serves up to kMany tensors: their pointers and sizes travel in the
// kernel's parameters, so nothing is uploaded and nothing has to live on
// the device between calls.  Blocks take equal chunks of values; a block finds
// its tensor by bisection in the table of first chunks, a few broadcast
// reads of the constant bank.
#include <algorithm>
#include <new>

#include "pb_layers.cuh"

namespace pb {
namespace {

constexpr int kThreads = 256;
constexpr int kFew = 48, kMany = 512;
constexpr int kUnroll = 2;  // packs of 16 bytes per thread and stream

template <typename T>
struct Hyper {
  T beta1, rest1, beta2, rest2;  // rest = 1 - beta, rounded from float64
  T keep;                        // 1 - lr * weight_decay
  T rate;                        // lr / (1 - beta1^step)
  T root;                        // 1 / sqrt(1 - beta2^step)
  T eps;
};

template <typename T, int N>
struct Table {
  T* p[N];
  const T* g[N];
  T* m[N];
  T* v[N];
  int64_t n[N];
  uint32_t first[N + 1];  // chunk numbers
  int count;
  Hyper<T> h;
  const T* scale;
};

__device__ __forceinline__ float root_of(float x) { return sqrtf(x); }
__device__ __forceinline__ double root_of(double x) { return sqrt(x); }

template <typename T>
__device__ __forceinline__ void update(const Hyper<T>& h, T s, T& p, T g, T& m, T& v) {
  g *= s;
  m = fma(h.beta1, m, h.rest1 * g);
  v = fma(h.beta2, v, h.rest2 * (g * g));
  p = h.keep * p - h.rate * (m / fma(root_of(v), h.root, h.eps));
}

template <typename T, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<T, N> t) {
  constexpr int V = 16 / (int)sizeof(T);
  constexpr int kChunk = kThreads * V * kUnroll;
  int lo = 0, hi = t.count;  // first[lo] <= block < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const int64_t begin = (int64_t)(blockIdx.x - t.first[lo]) * kChunk;
  const int64_t n = t.n[lo];
  T* const p = t.p[lo];
  const T* const g = t.g[lo];
  T* const m = t.m[lo];
  T* const v = t.v[lo];
  const T s = t.scale ? __ldg(t.scale) : T(1);
  const Hyper<T> h = t.h;
  const bool aligned = (((uintptr_t)p | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15) == 0;
  if (aligned && begin + kChunk <= n) {
    Pack<T, V> P[kUnroll], G[kUnroll], M[kUnroll], W[kUnroll];
    const int64_t at = begin + threadIdx.x * V;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = at + u * kThreads * V;
      G[u] = load_pack<T, V>(g + i);
      P[u] = *reinterpret_cast<const Pack<T, V>*>(p + i);
      M[u] = *reinterpret_cast<const Pack<T, V>*>(m + i);
      W[u] = *reinterpret_cast<const Pack<T, V>*>(v + i);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = at + u * kThreads * V;
#pragma unroll
      for (int k = 0; k < V; ++k) update(h, s, P[u].v[k], G[u].v[k], M[u].v[k], W[u].v[k]);
      store_pack<T, V>(p + i, P[u]);
      store_pack<T, V>(m + i, M[u]);
      store_pack<T, V>(v + i, W[u]);
    }
    return;
  }
  const int64_t end = begin + kChunk < n ? begin + kChunk : n;
  for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) {
    T pi = p[i], mi = m[i], vi = v[i];
    update(h, s, pi, __ldg(g + i), mi, vi);
    p[i] = pi;
    m[i] = mi;
    v[i] = vi;
  }
}

struct Lists {
  void* const* p;
  const void* const* g;
  void* const* m;
  void* const* v;
  const int64_t* n;
  int64_t count;
};

// One launch for tensors [from, to), the empty ones left out.
template <typename T, int N>
int launch(Device* d, const Lists& l, int64_t from, int64_t to, const Hyper<T>& h, const T* scale) {
  constexpr int64_t chunk = (int64_t)kThreads * (16 / sizeof(T)) * kUnroll;
  Table<T, N> t;
  t.count = 0;
  t.h = h;
  t.scale = scale;
  uint64_t blocks = 0;
  for (int64_t j = from; j < to; ++j) {
    if (!l.n[j]) continue;
    const int k = t.count++;
    t.p[k] = static_cast<T*>(l.p[j]);
    t.g[k] = static_cast<const T*>(l.g[j]);
    t.m[k] = static_cast<T*>(l.m[j]);
    t.v[k] = static_cast<T*>(l.v[j]);
    t.n[k] = l.n[j];
    t.first[k] = (uint32_t)blocks;
    blocks += (uint64_t)ceil_div(l.n[j], chunk);
    if (blocks > INT32_MAX) PB_FAIL(PB_ERR_UNSUPPORTED, "too many values in one AdamW launch");
  }
  if (!blocks) return PB_OK;
  t.first[t.count] = (uint32_t)blocks;
  adamw_kernel<T, N><<<(unsigned)blocks, kThreads, 0, d->stream>>>(t);
  PB_LAUNCHED(d);
  return PB_OK;
}

template <typename T>
int run(Device* d, const Lists& l, double lr, double beta1, double beta2, double eps, double weight_decay,
        int64_t step, const T* scale) {
  Hyper<T> h;
  h.beta1 = (T)beta1;
  h.rest1 = (T)(1.0 - beta1);
  h.beta2 = (T)beta2;
  h.rest2 = (T)(1.0 - beta2);
  h.keep = (T)(1.0 - lr * weight_decay);
  h.rate = (T)(lr / (1.0 - pow(beta1, (double)step)));
  h.root = (T)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  h.eps = (T)eps;
  PB_CHECK(kt_begin(d));
  for (int64_t j = 0; j < l.count; j += kMany) {
    const int64_t to = std::min(l.count, j + kMany);
    if (to - j <= kFew) PB_CHECK((launch<T, kFew>(d, l, j, to, h, scale)));
    else PB_CHECK((launch<T, kMany>(d, l, j, to, h, scale)));
  }
  return kt_end(d);
}

// Whether a written range overlaps another written range or a gradient.
bool conflicts(const Lists& l, size_t item, const void* scale, bool* out_of_memory) {
  struct Range {
    uintptr_t at, end;
    bool operator<(const Range& o) const { return at < o.at; }
  };
  *out_of_memory = false;
  std::vector<Range> w;
  try {
    w.reserve((size_t)l.count * 3);
  } catch (...) {
    *out_of_memory = true;
    return false;
  }
  for (int64_t j = 0; j < l.count; ++j) {
    if (!l.n[j]) continue;
    const size_t bytes = (size_t)l.n[j] * item;
    for (const void* q : {(const void*)l.p[j], (const void*)l.m[j], (const void*)l.v[j]})
      w.push_back({(uintptr_t)q, (uintptr_t)q + bytes});
  }
  std::sort(w.begin(), w.end());
  for (size_t i = 1; i < w.size(); ++i)
    if (w[i].at < w[i - 1].end) return true;
  auto hits = [&](const void* q, size_t bytes) {
    const uintptr_t at = (uintptr_t)q, end = at + bytes;
    // The last written range that starts before `end` is the only one that can
    // reach into [at, end): the ranges are disjoint.
    auto it = std::lower_bound(w.begin(), w.end(), Range{end, end});
    return it != w.begin() && (it - 1)->end > at;
  };
  for (int64_t j = 0; j < l.count; ++j)
    if (l.n[j] && hits(l.g[j], (size_t)l.n[j] * item)) return true;
  return scale && hits(scale, item);
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" {

int pb_adamw(pb_ctx* ctx, int dev, int dtype, int64_t count, void* const* params, const void* const* grads,
             void* const* exp_avg, void* const* exp_avg_sq, const int64_t* sizes, double lr, double beta1,
             double beta2, double eps, double weight_decay, int64_t step, const void* grad_scale) {
  if (!ctx) PB_FAIL(PB_ERR_INVALID, "null context");
  if (dtype != PB_F32 && dtype != PB_F64) PB_FAIL(PB_ERR_INVALID, "AdamW takes float32 or float64");
  if (count < 0 || count > INT32_MAX) PB_FAIL(PB_ERR_INVALID, "bad tensor count");
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0))
    PB_FAIL(PB_ERR_INVALID, "betas lie in [0, 1)");
  if (!(eps >= 0.0) || !(lr >= 0.0) || !(weight_decay >= 0.0))
    PB_FAIL(PB_ERR_INVALID, "lr, eps and weight_decay are not negative");
  if (step < 1) PB_FAIL(PB_ERR_INVALID, "step counts from 1");
  if (!count) return PB_OK;
  const size_t item = dtype == PB_F32 ? 4 : 8;
  if (!params || !grads || !exp_avg || !exp_avg_sq || !sizes) PB_FAIL(PB_ERR_INVALID, "null table");
  for (int64_t j = 0; j < count; ++j) {
    if (sizes[j] < 0 || sizes[j] > (int64_t(1) << 58)) PB_FAIL(PB_ERR_INVALID, "bad size of tensor %lld", (long long)j);
    if (sizes[j] && (!params[j] || !grads[j] || !exp_avg[j] || !exp_avg_sq[j]))
      PB_FAIL(PB_ERR_INVALID, "null pointer of tensor %lld", (long long)j);
    if (((uintptr_t)params[j] | (uintptr_t)grads[j] | (uintptr_t)exp_avg[j] | (uintptr_t)exp_avg_sq[j]) % item)
      PB_FAIL(PB_ERR_INVALID, "a pointer of tensor %lld is not aligned to its type", (long long)j);
  }
  if ((uintptr_t)grad_scale % item) PB_FAIL(PB_ERR_INVALID, "grad_scale is not aligned to its type");
  const Lists l = {params, grads, exp_avg, exp_avg_sq, sizes, count};
  bool out_of_memory;
  if (conflicts(l, item, grad_scale, &out_of_memory))
    PB_FAIL(PB_ERR_INVALID, "a parameter or moment overlaps another array of the step");
  if (out_of_memory) PB_FAIL(PB_ERR_OOM, "no host memory for %lld tensors", (long long)count);
  std::lock_guard<std::recursive_mutex> g(ctx->mu);
  Device* d;
  PB_CHECK(enter(ctx, dev, &d));
  if (d->capturing) PB_FAIL(PB_ERR_UNSUPPORTED, "a captured AdamW step would repeat its step number and lr");
  if (dtype == PB_F32)
    return run<float>(d, l, lr, beta1, beta2, eps, weight_decay, step, static_cast<const float*>(grad_scale));
  return run<double>(d, l, lr, beta1, beta2, eps, weight_decay, step, static_cast<const double*>(grad_scale));
}

}  // extern "C"
