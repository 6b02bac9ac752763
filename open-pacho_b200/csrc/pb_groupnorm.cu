// Group norm with an activation, channels last, and its gradients (HBM-bound:
// forward 2 values moved per element, backward 3).
//
// x is (N, S, C), C = G groups of m channels; a group's set is its m channels
// over the S positions of one sample.  Channels are contiguous, so lanes run
// over channels and every sum over positions is a sum down a column:
//   sums   adds up two numbers per channel in float64 over a run of positions of
//          one sample (forward: x - k and (x - k)^2 with the shift k = the group's
//          first value, which keeps the variance of values far from zero;
//          backward: dz and dz * xhat), then over the channels of each group.  The
//          block that finishes a sample last adds its runs' sums in a fixed
//          order, so the result is deterministic.
//   apply  reads the run again and writes the result.
// One launch does both: resident blocks take sums and apply items from a counter
// whose order interleaves them, a sample's apply items following its sums by
// about one item per block.  The second read then finds the sample in L2
// (up to about half of its 126 MB) while the next sample's first read keeps HBM busy.
//
// A small group (all of one with S = 1, a norm of each token) fits into the
// registers of a part of a warp, a warp or a block: one pass reads it, forms its
// sums and writes the result.  Such a part of the block stays with one group and
// walks over the samples, so that weight and bias stay in registers and the sums of
// dweight and dbias are its own.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "pb_layers.cuh"

namespace pb {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct NormArgs {
  const T *x, *dy, *weight, *bias;
  T* out;             // y or dx
  T *mean, *rstd;     // forward: outputs, may be null; backward: inputs
  T *dweight, *dbias; // may be null
  double2* chan;      // per-channel sums: of each (n, chunk), or of each block of the ring
  double2* part;      // (N, chunks, G): per-group sums
  double2* group;     // (N, G): forward (mean, rstd); backward (mean of w dz, mean of w dz xhat)
  unsigned* words;    // see pb_layers.cuh: a flag per sample
  int* err;
  unsigned* arrivals; // N words, zero on entry and exit
  int64_t N, S, C, G, m;
  int64_t rows;       // positions per item
  int64_t chunks;     // items per sample
  FastDiv by_chunks, by_m;
  double eps;
};

// Phi(z), the normal distribution's, and phi(z), its density, each to a few roundings
// of its own size wherever the density is a normal number.
//
// float32: Phi(-a) = phi(a) R(a) for a >= 0, with Mills' ratio R as a polynomial in
// t = 1 / (1 + p a), the form of Abramowitz and Stegun, Handbook of Mathematical
// Functions, 7.1.26, of degree 8 and with coefficients fitted to R on [0, 20] for the least
// relative error, 8.6e-8.  The density's exponent is formed in two parts, as in
// sigmoid_pair: the roundings of z^2 and of its product would be z^2 of the result's.
// Beyond |z| = 20 the density is zero; the minimum keeps a NaN.  32768 x 2048 forward: 145 us;
// 7.1.26 itself, off by 1e-3 of Phi at z = -5, 130; erfcf and expf, off by z^2 roundings, 198.
__device__ __forceinline__ void normal(float z, float* Phi, float* phi) {
  constexpr float kHalfLog2e = 0.721347511f, kHalfLog2eLow = 9.62981515e-9f, kLn2 = 0.693147182f;
  float a;
  asm("min.NaN.f32 %0, %1, 0f41A00000;" : "=f"(a) : "f"(fabsf(z)));
  const float s = a * a, k = s * -kHalfLog2e;
  const float r = fmaf(-s, kHalfLog2eLow, fmaf(fmaf(a, a, -s), -kHalfLog2e, fmaf(-s, kHalfLog2e, -k)));
  float e = exp2_unit(k);  // e^(-z^2 / 2)
  e = fmaf(e, r * kLn2, e);
  const float t = reciprocal_unit(fmaf(0.3f, a, 1.0f));
  float q = fmaf(0.0376731381f, t, -0.166167408f);
  q = fmaf(q, t, 0.223319471f);
  q = fmaf(q, t, -0.0713290721f);
  q = fmaf(q, t, 0.139563337f);
  q = fmaf(q, t, 0.0957120657f);
  q = fmaf(q, t, 0.121712156f);
  q = fmaf(q, t, 0.119510069f);
  q = fmaf(q, t, 6.19924685e-06f);
  const float tail = q * e;
  *Phi = z < 0.0f ? tail : 1.0f - tail;
  *phi = e * 0.39894228f;
}
__device__ __forceinline__ void normal(double z, double* Phi, double* phi) {
  *Phi = 0.5 * erfc(z * -0.70710678118654752);  // accurate for negative z, where 1 + erf would cancel
  *phi = exp(-0.5 * z * z) * 0.39894228040143268;
}

template <typename T, int ACT>
__device__ __forceinline__ T activate(T z) {
  if constexpr (ACT == PB_ACT_RELU) return z < T(0) ? T(0) : z;
  if constexpr (ACT == PB_ACT_SILU) return z * sigmoid(z);
  if constexpr (ACT == PB_ACT_GELU) {
    T Phi, phi;
    normal(z, &Phi, &phi);
    return z * Phi;
  }
  return z;
}

template <typename T, int ACT>
__device__ __forceinline__ T slope(T z) {
  if constexpr (ACT == PB_ACT_RELU) return z > T(0) ? T(1) : T(0);
  if constexpr (ACT == PB_ACT_SILU) {
    const T s = sigmoid(z);
    return fma(s * z, T(1) - s, s);
  }
  if constexpr (ACT == PB_ACT_GELU) {
    T Phi, phi;
    normal(z, &Phi, &phi);
    return fma(z, phi, Phi);
  }
  return T(1);
}

// The shift of a group's sums: its first value, or 0 where that is not finite
// (a non-finite shift would hide which of NaN and Inf the mean is).
template <typename T>
__device__ __forceinline__ double shift_of(const NormArgs<T>& p, int64_t n, int64_t g) {
  const double k = (double)__ldg(p.x + n * p.S * p.C + g * p.m);
  return isfinite(k) ? k : 0.0;
}

// Channels whose sums a block holds in shared memory.
constexpr int64_t kSharedChannels = 1024;

// What a thread needs of its V channels c, c + step, ...: the sums of one pass over
// positions.  Channels from C on have sums that nobody reads.
// Backward, the second sum is of dz xhat, xhat = (x - mean) rstd: dz (x - mean), with
// the factor rstd at the end, would leave float32's range where x is far from 1.
// Two positions at a time: their terms are added in T and the pair in float64, which
// halves the conversions (they share a unit of a sixteenth of the rate with the
// exponential) for one rounding more.
template <typename T, int V, int ACT, bool BWD>
struct ChannelSums {
  double s1[V], s2[V];
  double k[BWD ? 1 : V];
  T mean[BWD ? V : 1], rstd[BWD ? V : 1], w[BWD ? V : 1], b[BWD ? V : 1];

  __device__ __forceinline__ void begin(const NormArgs<T>& p, int64_t n, int64_t c, bool on, int step = 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s1[i] = s2[i] = 0.0;
      const int64_t ch = c + i * step;
      const bool here = on && ch < p.C;
      const int64_t g = here ? fdiv(ch, p.by_m) : 0;
      if constexpr (BWD) {
        mean[i] = __ldg(p.mean + n * p.G + g);
        rstd[i] = __ldg(p.rstd + n * p.G + g);
        w[i] = here && p.weight ? __ldg(p.weight + ch) : T(1);
        b[i] = here && p.bias ? __ldg(p.bias + ch) : T(0);
      } else {
        k[i] = shift_of(p, n, g);
      }
    }
  }
  __device__ __forceinline__ void term(int i, T x, T dy, T* dz, T* product) const {
    const T xhat = (x - mean[i]) * rstd[i];
    *dz = dy * slope<T, ACT>(fma(xhat, w[i], b[i]));
    *product = *dz * xhat;
  }
  // Backward, dy becomes dz.
  __device__ __forceinline__ void add(const Pack<T, V>& x, Pack<T, V>& dy) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (BWD) {
        T dz, product;
        term(i, x.v[i], dy.v[i], &dz, &product);
        s1[i] += (double)dz;
        s2[i] += (double)product;
        dy.v[i] = dz;
      } else {
        const double v = (double)x.v[i] - k[i];
        s1[i] += v;
        s2[i] = fma(v, v, s2[i]);
      }
    }
  }
  __device__ __forceinline__ void add2(const Pack<T, V>& x0, Pack<T, V>& dy0, const Pack<T, V>& x1, Pack<T, V>& dy1) {
    if constexpr (BWD) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        T z0, z1, q0, q1;
        term(i, x0.v[i], dy0.v[i], &z0, &q0);
        term(i, x1.v[i], dy1.v[i], &z1, &q1);
        s1[i] += (double)(z0 + z1);
        s2[i] += (double)(q0 + q1);
        dy0.v[i] = z0;
        dy1.v[i] = z1;
      }
    } else {
      add(x0, dy0);
      add(x1, dy1);
    }
  }
};

// ... and its results, y = act((x - mean) rw + b) with rw = rstd w, and
// dx = rstd (w dz - m1 - xhat m2).  Backward every factor stays apart: rstd^2 m2 leaves
// float32's range where x is far from 1, and z has the bits that the sums had.
template <typename T, int V, int ACT, bool BWD>
struct ChannelResults {
  T mean[V], w[V], b[V];   // forward: w becomes rw
  T r1[V];                 // backward: -m1; forward: the mean's low part, so that its rounding does not show
  T rstd[BWD ? V : 1], r2[BWD ? V : 1];  // r2 = -m2

  // What does not depend on the sums of sample n.
  __device__ __forceinline__ void begin(const NormArgs<T>& p, int64_t n, int64_t c, bool on, int step = 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int64_t ch = c + i * step;
      const bool here = on && ch < p.C;
      w[i] = here && p.weight ? __ldg(p.weight + ch) : T(1);
      b[i] = here && p.bias ? __ldg(p.bias + ch) : T(0);
      if constexpr (BWD) {
        const int64_t g = here ? fdiv(ch, p.by_m) : 0;
        mean[i] = __ldg(p.mean + n * p.G + g);
        rstd[i] = __ldg(p.rstd + n * p.G + g);
      }
    }
  }
  // The statistics, at `stats` or in p.group.
  __device__ __forceinline__ void end(const NormArgs<T>& p, int64_t n, int64_t c, bool on, const double2* stats,
                                      int step = 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int64_t ch = c + i * step;
      const int64_t g = on && ch < p.C ? fdiv(ch, p.by_m) : 0;
      const double2 t = stats ? stats[g] : __ldcg(p.group + n * p.G + g);
      if constexpr (BWD) {
        r1[i] = (T)-t.x;
        r2[i] = (T)-t.y;
      } else {
        mean[i] = (T)t.x;
        r1[i] = (T)(t.x - (double)mean[i]);
        w[i] = (T)(t.y * (double)w[i]);
      }
    }
  }
  // dx where dz and xhat are known.
  __device__ __forceinline__ T gradient(int i, T dz, T xhat) const {
    return rstd[BWD ? i : 0] * fma(w[i], dz, fma(xhat, r2[BWD ? i : 0], r1[i]));
  }
  __device__ __forceinline__ Pack<T, V> of_dz(const Pack<T, V>& x, const Pack<T, V>& dz) const {
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = gradient(i, dz.v[i], (x.v[i] - mean[i]) * rstd[BWD ? i : 0]);
    return o;
  }
  __device__ __forceinline__ Pack<T, V> of(const Pack<T, V>& x, const Pack<T, V>& dy) const {
    Pack<T, V> o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const T d = x.v[i] - mean[i];
      if constexpr (BWD) {
        const T xhat = d * rstd[i];
        o.v[i] = gradient(i, dy.v[i] * slope<T, ACT>(fma(xhat, w[i], b[i])), xhat);
      } else {
        o.v[i] = activate<T, ACT>(fma(d - r1[i], w[i], b[i]));
      }
    }
    return o;
  }
};

// Over the ty rows of threads, in row order: the sums of tx * V channels from c0
// on, to `out` and, where it is another place, to `copy`.
template <typename T, int V, typename S>
__device__ __forceinline__ void sum_rows(const NormArgs<T>& p, const S& sums, int64_t c0, int tx, int ty, double2* red,
                                         double2* out, double2* copy) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    red[threadIdx.x] = make_double2(sums.s1[i], sums.s2[i]);
    __syncthreads();
    const int64_t c = c0 + (int64_t)threadIdx.x * V + i;
    if ((int)threadIdx.x < tx && c < p.C) {
      double2 t = red[threadIdx.x];
      for (int y = 1; y < ty; ++y) {
        t.x += red[y * tx + threadIdx.x].x;
        t.y += red[y * tx + threadIdx.x].y;
      }
      out[c] = t;
      if (copy && copy != out) copy[c] = t;
    }
    __syncthreads();
  }
}

// Over the channels of each group: a thread each, or a warp where they are many.
template <typename T, bool BWD>
__device__ __forceinline__ void sum_groups(const NormArgs<T>& p, const double2* channels, double2* part) {
  const int64_t lanes = p.m <= 16 ? 1 : 32;
  for (int64_t g = threadIdx.x / lanes; g < p.G; g += kThreads / lanes) {
    double2 t = make_double2(0.0, 0.0);
    for (int64_t c = g * p.m + threadIdx.x % lanes; c < (g + 1) * p.m; c += lanes) {
      const double2 v = channels[c];
      const double w = BWD && p.weight ? (double)__ldg(p.weight + c) : 1.0;
      t.x = fma(w, v.x, t.x);
      t.y = fma(w, v.y, t.y);
    }
    for (int o = (int)lanes / 2; o > 0; o >>= 1) {
      t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
      t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
    }
    if (threadIdx.x % lanes == 0) part[g] = t;
  }
}

// The group sums of one item: threads form tx lanes over packs of V channels
// and ty rows.
template <typename T, int V, int ACT, bool BWD>
__device__ __forceinline__ void sums_item(const NormArgs<T>& p, int64_t unit, int tx, int ty, double2* red, double2* shared) {
  const int lx = threadIdx.x % tx, ly = threadIdx.x / tx;
  const int64_t n = fdiv(unit, p.by_chunks), chunk = unit - n * p.chunks;
  const int64_t r0 = chunk * p.rows, r1 = min(p.S, r0 + p.rows);
  double2* const out = p.C <= kSharedChannels ? shared : p.chan + unit * p.C;
  for (int64_t c0 = 0; c0 < p.C; c0 += (int64_t)tx * V) {
    const int64_t c = c0 + (int64_t)lx * V;
    const bool on = ly < ty && c < p.C;
    ChannelSums<T, V, ACT, BWD> sums;
    sums.begin(p, n, c, on);
    if (on) {
      int64_t at = (n * p.S + r0 + ly) * p.C + c;
#pragma unroll 4
      for (int64_t r = r0 + ly; r < r1; r += ty, at += ty * p.C) {
        const Pack<T, V> x = load_pack<T, V>(p.x + at);
        Pack<T, V> dy;
        if constexpr (BWD) dy = load_pack<T, V>(p.dy + at);
        sums.add(x, dy);
      }
    }
    sum_rows<T, V>(p, sums, c0, tx, ty, red, out, BWD && p.chan ? p.chan + unit * p.C : nullptr);
  }
  sum_groups<T, BWD>(p, out, p.part + unit * p.G);
}

// Mean and rstd (forward) or the two means (backward) of a group from its sums.
template <typename T, bool BWD>
__device__ __forceinline__ double2 statistics(const NormArgs<T>& p, int64_t n, int64_t g, double2 t) {
  const double count = (double)p.S * (double)p.m;
  t.x /= count;
  t.y /= count;
  if constexpr (!BWD) {
    // A set with NaN or Inf in it has a NaN variance (fmax alone would drop
    // it); finite float64 values whose squares overflow have an infinite one.
    const double var = isinf(t.y) ? t.y : fmax(fma(-t.x, t.x, t.y), 0.0);
    const double rstd = isfinite(t.x) ? 1.0 / sqrt(var + p.eps) : t.x - t.x;
    t = make_double2(t.x + shift_of(p, n, g), rstd);
  }
  return t;
}

// The statistics of a sample from its items' group sums.  The threads take
// (group, every lanes-th item) and meet in shared memory.
template <typename T, bool BWD>
__device__ __forceinline__ void merge_sample(const NormArgs<T>& p, int64_t n, double2* red) {
  const int wide = p.G < kThreads ? (int)p.G : kThreads, lanes = kThreads / wide;
  const int lg = threadIdx.x % wide, lk = threadIdx.x / wide;
  for (int64_t g0 = 0; g0 < p.G; g0 += wide) {
    const int64_t g = g0 + lg;
    double2 t = make_double2(0.0, 0.0);
    if (g < p.G && lk < lanes) {
      const double2* q = p.part + (n * p.chunks + lk) * p.G + g;
#pragma unroll 16
      for (int64_t k = lk; k < p.chunks; k += lanes, q += (int64_t)lanes * p.G) {
        const double2 v = __ldcg(q);
        t.x += v.x;
        t.y += v.y;
      }
    }
    __syncthreads();
    red[threadIdx.x] = t;
    __syncthreads();
    if (lk == 0 && g < p.G) {
      for (int k = 1; k < lanes; ++k) {
        t.x += red[k * wide + lg].x;
        t.y += red[k * wide + lg].y;
      }
      t = statistics<T, BWD>(p, n, g, t);
      if constexpr (!BWD) {
        if (p.mean) p.mean[n * p.G + g] = (T)t.x;
        if (p.rstd) p.rstd[n * p.G + g] = (T)t.y;
      }
      p.group[n * p.G + g] = t;
    }
  }
}

template <typename T, int V, int ACT, bool BWD>
__device__ __forceinline__ void apply_item(const NormArgs<T>& p, int64_t unit, int tx, int ty) {
  const int lx = threadIdx.x % tx, ly = threadIdx.x / tx;
  const int64_t n = fdiv(unit, p.by_chunks), chunk = unit - n * p.chunks;
  const int64_t r0 = chunk * p.rows, r1 = min(p.S, r0 + p.rows);
  for (int64_t c = (int64_t)lx * V; c < p.C && ly < ty; c += (int64_t)tx * V) {
    ChannelResults<T, V, ACT, BWD> results;
    results.begin(p, n, c, true);
    results.end(p, n, c, true, nullptr);
    int64_t at = (n * p.S + r0 + ly) * p.C + c;
#pragma unroll 4
    for (int64_t r = r0 + ly; r < r1; r += ty, at += ty * p.C) {
      const Pack<T, V> x = load_pack<T, V>(p.x + at);
      Pack<T, V> dy;
      if constexpr (BWD) dy = load_pack<T, V>(p.dy + at);
      store_pack<T, V>(p.out + at, results.of(x, dy));
    }
  }
}

// Items in the order of their numbers: `lead` sums, then apply and sums in
// turn, then the rest of apply.  lead is a sample's items and two per block (the
// one it works on and the one it holds), so apply item j comes behind all sums of its
// sample.
template <typename T, int V, int ACT, bool BWD>
__global__ void __launch_bounds__(kThreads, BWD ? 2 : 3) norm_samples_kernel(const NormArgs<T> p, int tx, int ty, unsigned units,
                                                                   unsigned lead) {
  __shared__ double2 red[kThreads];
  __shared__ double2 channels[kSharedChannels];
  __shared__ unsigned item_s, epoch_s;
  __shared__ bool last;
  __shared__ int failed;
  if (threadIdx.x == 0) {
    failed = 0;
    item_s = atomicAdd(p.words, 1u);
    epoch_s = load_acquire(p.words + 2) + 1;
  }
  __syncthreads();
  const unsigned epoch = epoch_s;
  for (unsigned item = item_s; item < 2 * units; item = item_s) {
    // The next item is asked for now; it is read behind this one's end.
    unsigned next = 0;
    if (threadIdx.x == 0) next = atomicAdd(p.words, 1u);
    const unsigned turn = item - lead;  // used from item `lead` on
    bool sums;
    unsigned unit;
    if (item < lead) sums = true, unit = item;
    else if (turn < 2 * (units - lead)) sums = turn & 1u, unit = turn / 2 + (sums ? lead : 0u);
    else sums = false, unit = turn - (units - lead);
    const int64_t n = fdiv(unit, p.by_chunks);
    if (sums) {
      sums_item<T, V, ACT, BWD>(p, unit, tx, ty, red, channels);
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0)
        last = p.chunks == 1 || atomicAdd(&p.arrivals[n], 1u) == (unsigned)p.chunks - 1;
      __syncthreads();
      if (last) {
        __threadfence();
        merge_sample<T, BWD>(p, n, red);
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
          if (p.chunks > 1) p.arrivals[n] = 0;
          store_release(p.words + kFlagWords + n, epoch);
        }
      }
    } else {
      if (threadIdx.x == 0) wait_until([&] { return load_acquire(p.words + kFlagWords + n) == epoch; }, &failed, p.err);
      __syncthreads();
      apply_item<T, V, ACT, BWD>(p, unit, tx, ty);
    }
    __syncthreads();
    if (threadIdx.x == 0) item_s = next;
    __syncthreads();
  }
  if (threadIdx.x == 0) finish_words(p.words, epoch, gridDim.x);
}

// ---- the same, fed by bulk copies ----------------------------------------
//
// Positions of a sample are one run of memory, so where rows are whole 16-byte
// pieces one thread of each block copies them into a ring of shared-memory stages,
// ahead of the block across the ends of runs and passes.  There is one block per SM,
// all resident (a cooperative launch).  They work on `together` samples at a
// time, `chunks` blocks for each: a block forms the sums of its run of positions,
// waits until all blocks of the sample have theirs, adds them up and applies the
// statistics to the same run, of which the last stages are still in shared memory
// and the others come from L2.  What is left besides the copies is the chain
// between the passes (sums over the block's rows and groups, publishing,
// waiting, adding up), about 5 us for each round of samples.
//
// SPREAD: rows of any size.  A stage's values start and end anywhere, its copy on
// the 16-byte boundaries around them, the last values of the array apart; a thread's
// channels lie tx apart, so that lanes move neighbours one value at a time.
// 8 x 4096 x 319 float32 forward 33 us (plain loads of norm_samples_kernel: 69; 320
// channels: 31), backward 60 (124; 55); 6 x 3001 x 1107 forward 64 (125).
constexpr int kRingThreads = 480;  // and a warp that copies: 16 warps, 128 registers each thread
constexpr int kRingWarps = kRingThreads / 32;
constexpr int kRing = 8;
constexpr size_t kRingSmem = 220 * 1024;
// Up to so many (block, group) sums of a sample every block adds up for itself;
// beyond, each block does some of the groups and all meet once more.
constexpr int64_t kOwnSums = 8192, kOwnGroups = 512;

__device__ __forceinline__ void ring_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kRingThreads) : "memory");
}

// Wait (the whole block) until `count` blocks have arrived at *counter.
__device__ __forceinline__ void arrive_and_wait(unsigned* counter, unsigned count, volatile int* failed, int* err) {
  __threadfence();
  ring_sync();
  if (threadIdx.x == 0) {
    atomicAdd(counter, 1u);
    wait_until([&] { return load_acquire(counter) >= count; }, failed, err);
  }
  ring_sync();
}

// Values of one array of a stage.
template <typename T, bool SPREAD>
__host__ __device__ __forceinline__ int64_t ring_array(int64_t stage_rows, int64_t C) {
  constexpr int A = 16 / (int)sizeof(T);
  return SPREAD ? (stage_rows * C + 2 * A - 2) / A * A : stage_rows * C;
}

template <typename T, int V, int ACT, bool BWD, bool SPREAD>
__global__ void __launch_bounds__(kRingThreads + 32, 1) norm_ring_kernel(const NormArgs<T> p, int tx, int ty,
                                                                       int stage_rows, int64_t together) {
  constexpr int kArrays = BWD ? 2 : 1;
  constexpr int A = 16 / (int)sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t full[kRing], empty[kRing];
  __shared__ int failed;
  __shared__ bool last;
  const int C = (int)p.C, G = (int)p.G, m = (int)p.m;
  const int array = (int)ring_array<T, SPREAD>(stage_rows, C);
  T* const ring = reinterpret_cast<T*>(smem);
  double2* const red = reinterpret_cast<double2*>(ring + (size_t)kRing * kArrays * array);  // [V * kRingThreads]
  double2* const channels = red + V * kRingThreads;                                          // [C]
  double2* const stats = channels + C;  // [G] where a block adds up for itself
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      barrier_init(full + s, 1);
      barrier_init(empty + s, kRingWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
  }
  __syncthreads();
  const int64_t place = blockIdx.x / p.chunks, chunk = blockIdx.x - place * p.chunks;
  const int64_t r0 = chunk * p.rows, r1 = min(p.S, r0 + p.rows);
  const int stages = (int)((r1 - r0 + stage_rows - 1) / stage_rows);
  // The sums leave the last `held` stages where they are; the second pass takes
  // those first and then the others, in order.
  const int held = min(stages, kRing);
  unsigned turn = 0;  // copies so far: stage turn % kRing, its use number turn / kRing

  if (threadIdx.x >= kRingThreads) {
    if (threadIdx.x > kRingThreads) return;
    bool ok = true;
    for (int64_t n = place; n < p.N && ok; n += together) {
      for (int k = 0; k < 2 * stages - held && ok; ++k, ++turn) {
        const int s = turn % kRing;
        if (turn >= kRing) ok = barrier_wait(empty + s, (turn / kRing - 1) & 1, &failed, p.err);
        if (!ok) break;
        const int64_t r = r0 + (int64_t)(k < stages ? k : k - stages) * stage_rows;
        const int rows = (int)min((int64_t)stage_rows, r1 - r);
        int64_t at = (n * p.S + r) * p.C, end = at + (int64_t)rows * C;
        T* const to = ring + (size_t)s * kArrays * array;
        if constexpr (SPREAD) {
          const int64_t all = p.N * p.S * p.C, stop = min((end + A - 1) & -(int64_t)A, all & -(int64_t)A);
          at &= -(int64_t)A;
          if (end > stop) {
            for (int64_t e = max(stop, at); e < end; ++e) {
              to[e - at] = __ldg(p.x + e);
              if constexpr (BWD) to[array + (e - at)] = __ldg(p.dy + e);
            }
            // A later copy to this stage comes behind these writes.
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          end = max(stop, at);
        }
        const unsigned bytes = (unsigned)(end - at) * (unsigned)sizeof(T);
        barrier_expect(full + s, bytes * kArrays);
        if (!SPREAD || bytes) {
          bulk_copy(to, p.x + at, bytes, full + s);
          if constexpr (BWD) bulk_copy(to + array, p.dy + at, bytes, full + s);
        }
      }
    }
    // Nothing may be on its way when the block ends.
    for (unsigned q = turn > kRing ? turn - kRing : 0; q < turn; ++q)
      barrier_wait(full + q % kRing, (q / kRing) & 1, &failed, p.err);
    return;
  }

  const int lx = threadIdx.x % tx, ly = threadIdx.x / tx;
  const int c = SPREAD ? lx : lx * V, apart = SPREAD ? tx : 1;  // the first channel, and how far the others are
  const bool on = ly < ty;
  // Packs of this thread's channels in shared memory, and the result's.
  auto get = [&](const T* from) {
    Pack<T, V> o;
    if constexpr (SPREAD) {
#pragma unroll
      for (int i = 0; i < V; ++i) o.v[i] = from[i * tx];
    } else {
      o = *reinterpret_cast<const Pack<T, V>*>(from);
    }
    return o;
  };
  auto put = [&](T* to, const Pack<T, V>& o) {
    if constexpr (SPREAD) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i * tx < C) to[i * tx] = o.v[i];
    } else {
      *reinterpret_cast<Pack<T, V>*>(to) = o;
    }
  };
  // Stage k of the run, as copied in turn t: `two` takes two of its positions,
  // `one` the last of an odd number.  With `keep` the dy that they have changed (to
  // dz) goes back to the stage.
  auto take = [&](unsigned t, int k, int64_t n, bool wait, bool keep, bool release, auto&& two, auto&& one) {
    const int s = t % kRing;
    if (wait) barrier_wait(full + s, (t / kRing) & 1, &failed, p.err);
    const int64_t r = r0 + (int64_t)k * stage_rows;
    const int rows = on ? (int)min((int64_t)stage_rows, r1 - r) : 0;
    const int64_t at = (n * p.S + r) * p.C + c;
    T* const from = ring + (size_t)s * kArrays * array + c + (SPREAD ? (int)((at - c) & (A - 1)) : 0);
    int q = ly;
    for (; q + ty < rows; q += 2 * ty) {
      T* const f0 = from + q * C;
      T* const f1 = f0 + ty * C;
      const Pack<T, V> x0 = get(f0), x1 = get(f1);
      Pack<T, V> d0, d1;
      if constexpr (BWD) {
        d0 = get(f0 + array);
        d1 = get(f1 + array);
      }
      two(x0, d0, x1, d1, at + q * C, at + (q + ty) * C);
      if (BWD && keep) {
        put(f0 + array, d0);
        put(f1 + array, d1);
      }
    }
    if (q < rows) {
      T* const f0 = from + q * C;
      const Pack<T, V> x0 = get(f0);
      Pack<T, V> d0;
      if constexpr (BWD) d0 = get(f0 + array);
      one(x0, d0, at + q * C);
      if (BWD && keep) put(f0 + array, d0);
    }
    if (release) {
      // Behind this thread's own writes to the stage comes a copy of the other kind.
      if (BWD && !wait) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if ((threadIdx.x & 31) == 0) barrier_arrive(empty + s);
    }
  };
  auto store = [&](int64_t a, const Pack<T, V>& o) { put(p.out + a, o); };
  using P = const Pack<T, V>&;
  using D = Pack<T, V>&;
  const bool own = p.chunks * G <= kOwnSums && G <= kOwnGroups;
  const int lanes = tx * V;                                          // channels that the threads cover, C or a little more
  const int parts = lanes < kRingThreads ? kRingThreads / lanes : 1;  // threads per channel in the sums over rows
  for (int64_t n = place; n < p.N; n += together) {
    const int64_t unit = n * p.chunks + chunk;
    {
      ChannelSums<T, V, ACT, BWD> sums;
      sums.begin(p, n, c, on, apart);
      for (int k = 0; k < stages; ++k)
        take(turn + k, k, n, true, k >= stages - held, k < stages - held,
             [&](P x0, D d0, P x1, D d1, int64_t, int64_t) { sums.add2(x0, d0, x1, d1); },
             [&](P x, D dy, int64_t) { sums.add(x, dy); });
        // Over the rows of threads: red is [ty][tx * V], `parts` threads per channel.
      if (on) {
#pragma unroll
        for (int i = 0; i < V; ++i) red[(ly * V + i) * tx + lx] = make_double2(sums.s1[i], sums.s2[i]);
      }
    }
    ring_sync();
    if ((int)threadIdx.x < parts * lanes) {
      const int q = threadIdx.x % lanes, part = threadIdx.x / lanes;
      double2 t = make_double2(0.0, 0.0);
      for (int y = part; y < ty; y += parts) {
        const double2 v = red[y * lanes + q];
        t.x += v.x;
        t.y += v.y;
      }
      if (part < ty) red[part * lanes + q] = t;
    }
    for (int q = threadIdx.x + kRingThreads; q < lanes; q += kRingThreads) {  // more channels than threads: parts is 1
      for (int y = 1; y < ty; ++y) {
        red[q].x += red[y * lanes + q].x;
        red[q].y += red[y * lanes + q].y;
      }
    }
    ring_sync();
    for (int q = threadIdx.x; q < lanes; q += kRingThreads) {
      double2 t = red[q];
      for (int k = 1; k < parts && k < ty; ++k) {
        t.x += red[k * lanes + q].x;
        t.y += red[k * lanes + q].y;
      }
      const int ch = SPREAD ? q : q % tx * V + q / tx;
      if (ch < C) {
        if (BWD && p.chan) {
          double2* const all = p.chan + (int64_t)blockIdx.x * C + ch;  // over the block's samples
          const double2 before = n == place ? make_double2(0.0, 0.0) : *all;
          *all = make_double2(before.x + t.x, before.y + t.y);
        }
        if (BWD && p.weight) {
          const double w = (double)__ldg(p.weight + ch);
          t.x *= w;
          t.y *= w;
        }
        channels[ch] = t;
      }
    }
    ring_sync();
    // Over the channels of each group: a thread each, or a warp where they are many.
    if (m <= 16) {
      for (int g = threadIdx.x; g < G; g += kRingThreads) {
        double2 t = channels[g * m];
        for (int k = 1; k < m; ++k) {
          t.x += channels[g * m + k].x;
          t.y += channels[g * m + k].y;
        }
        __stcg(p.part + unit * G + g, t);
      }
    } else {
      for (int g = threadIdx.x / 32; g < G; g += kRingWarps) {
        double2 t = make_double2(0.0, 0.0);
        for (int k = threadIdx.x & 31; k < m; k += 32) {
          t.x += channels[g * m + k].x;
          t.y += channels[g * m + k].y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
          t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
        }
        if ((threadIdx.x & 31) == 0) __stcg(p.part + unit * G + g, t);
      }
    }
    ChannelResults<T, V, ACT, BWD> results;
    results.begin(p, n, c, on, apart);
    // Over the blocks of the sample.
    if (p.chunks > 1) arrive_and_wait(p.arrivals + n, (unsigned)p.chunks, &failed, p.err);
    else ring_sync();
    const int wide = min(G, kRingThreads), rows = kRingThreads / wide;
    const int first = own ? 0 : (int)chunk, step = own ? 1 : (int)p.chunks;  // groups this block adds up
    for (int g0 = 0; g0 * step + first < G; g0 += wide) {
      const int g = (g0 + (int)threadIdx.x % wide) * step + first, row = threadIdx.x / wide;
      double2 t = make_double2(0.0, 0.0);
      if (g < G && row < rows) {
        const double2* q = p.part + (n * p.chunks + row) * G + g;
#pragma unroll 8
        for (int64_t k = row; k < p.chunks; k += rows, q += (int64_t)rows * G) {
          const double2 v = __ldcg(q);
          t.x += v.x;
          t.y += v.y;
        }
      }
      red[threadIdx.x] = t;
      ring_sync();
      if (row == 0 && g < G) {
        for (int k = 1; k < rows; ++k) {
          t.x += red[k * wide + threadIdx.x].x;
          t.y += red[k * wide + threadIdx.x].y;
        }
        t = statistics<T, BWD>(p, n, g, t);
        if (own) stats[g] = t;
        else __stcg(p.group + n * G + g, t);
        if (!BWD && (!own || chunk == 0)) {
          if (p.mean) p.mean[n * G + g] = (T)t.x;
          if (p.rstd) p.rstd[n * G + g] = (T)t.y;
        }
      }
      ring_sync();
    }
    if (!own) {
      if (p.chunks > 1) arrive_and_wait(p.arrivals + n, 2 * (unsigned)p.chunks, &failed, p.err);
      else {
        __threadfence();
        ring_sync();
      }
    }
    results.end(p, n, c, on, own ? stats : nullptr, apart);
    for (int k = stages - held; k < stages; ++k)
      take(turn + k, k, n, false, false, true,
           [&](P x0, P d0, P x1, P d1, int64_t a0, int64_t a1) {
             store(a0, BWD ? results.of_dz(x0, d0) : results.of(x0, d0));
             store(a1, BWD ? results.of_dz(x1, d1) : results.of(x1, d1));
           },
           [&](P x, P dz, int64_t a) { store(a, BWD ? results.of_dz(x, dz) : results.of(x, dz)); });
    for (int k = 0; k < stages - held; ++k)
      take(turn + stages + k, k, n, true, false, true,
           [&](P x0, P d0, P x1, P d1, int64_t a0, int64_t a1) {
             store(a0, results.of(x0, d0));
             store(a1, results.of(x1, d1));
           },
           [&](P x, P dy, int64_t a) { store(a, results.of(x, dy)); });
    turn += 2 * stages - held;
  }
  // The last block to finish leaves the counters at zero.
  if (p.chunks > 1) {
    if (threadIdx.x == 0) {
      __threadfence();
      last = atomicAdd(p.words + 1, 1u) == gridDim.x - 1;
    }
    ring_sync();
    if (last) {
      for (int64_t n = threadIdx.x; n < p.N; n += kRingThreads) p.arrivals[n] = 0;
      if (threadIdx.x == 0) p.words[1] = 0;
    }
  }
}

// use(ACT) of the activation that a launch has.
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& use) {
  switch (act) {
    case PB_ACT_RELU: use(std::integral_constant<int, PB_ACT_RELU>{}); break;
    case PB_ACT_SILU: use(std::integral_constant<int, PB_ACT_SILU>{}); break;
    case PB_ACT_GELU: use(std::integral_constant<int, PB_ACT_GELU>{}); break;
    default: use(std::integral_constant<int, PB_ACT_NONE>{});
  }
}

__device__ __forceinline__ double plus(double a, double b) { return a + b; }
__device__ __forceinline__ double2 plus(double2 a, double2 b) { return make_double2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ double across(double t, int o) { return __shfl_xor_sync(0xffffffffu, t, o); }
__device__ __forceinline__ double2 across(double2 t, int o) { return make_double2(across(t.x, o), across(t.y, o)); }

// Sums (double or double2) over the LANES threads that share a row, the same in
// each of them and in a fixed order.
template <int LANES, typename S>
__device__ __forceinline__ S row_sum(S t) {
  constexpr int kRowWarps = LANES / 32;
#pragma unroll
  for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) t = plus(t, across(t, o));
  if constexpr (LANES > 32) {
    __shared__ S part[kRowWarps];
    __syncthreads();  // the last use of `part` is over
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = t;
    __syncthreads();
    t = part[0];
#pragma unroll
    for (int w = 1; w < kRowWarps; ++w) t = plus(t, part[w]);
  }
  return t;
}

// A group's S * m values in the registers of LANES threads, ITEMS packs of V
// values each (a "row": with S = 1 it is contiguous, else S runs of m).
// Threads are numbered in units of a warp, or of a block of LANES where a row takes
// more than a warp; a unit works on group u % G of samples chunk * rows ...
// FLAT: S is 1.  What limits it is registers: backward, above 32 bytes of a row per
// thread weight and bias are read again for each row (they stay in L1) and the next
// row is not fetched ahead.
//
// 16384 x 2048 in 16 groups, float32, silu, backward: 83 us, 4.9 TB/s or 76 % of the
// copy rate; forward 32768 x 2048 104 us, 80 %; a layer norm of 65536 x 1024 99 us, 84 %.
template <int LANES>
constexpr int kRowThreads = LANES > 32 ? LANES : kThreads;
template <int BYTES, int LANES, bool BWD>  // BYTES of a row in each thread
constexpr int kRowBlocks = (BYTES > 64 ? 256 : BWD || BYTES > 32 ? 512 : 768) / kRowThreads<LANES> > 1
                               ? (BYTES > 64 ? 256 : BWD || BYTES > 32 ? 512 : 768) / kRowThreads<LANES>
                               : 1;
template <typename T, int V, int LANES, int ITEMS, bool BWD>
constexpr bool kRowApart = BWD && V * ITEMS * sizeof(T) <= 32 && sizeof(T) == 4;

template <typename T, int V, int LANES, int ITEMS, bool BWD, bool FLAT>
__global__ void __launch_bounds__(kRowThreads<LANES>, kRowBlocks<V * ITEMS * sizeof(T), LANES, BWD>)
    norm_rows_kernel(const NormArgs<T> p, int act) {
  constexpr int UNIT = LANES < 32 ? 32 : LANES, SUBS = UNIT / LANES;
  constexpr bool KEEP = !BWD || V * ITEMS * sizeof(T) <= 32, AHEAD = KEEP;
  const int64_t unit = (int64_t)blockIdx.x * (kRowThreads<LANES> / UNIT) + threadIdx.x / UNIT;
  if (unit >= p.G * p.chunks) return;  // whole units only
  const int64_t g = unit % p.G, chunk = unit / p.G;
  const int lane = threadIdx.x % LANES, sub = threadIdx.x % UNIT / LANES;
  const int64_t n0 = chunk * p.rows, n1 = min(p.N, n0 + p.rows), sample = p.S * p.C;
  // Of each pack's first value: the channel within the group, and the distance
  // from the group's first value (below 2^31).
  const int packs = (int)(p.m / V);  // in a run
  bool on[ITEMS];
  int channel[ITEMS], place[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int q = k * LANES + lane, s = FLAT ? 0 : q / packs;
    on[k] = FLAT ? q < packs : s < (int)p.S;
    channel[k] = (q - s * packs) * V;
    place[k] = FLAT ? q * V : s * (int)p.C + channel[k];
  }
  // weight and bias of pack k
  auto affine = [&](int k, T* w, T* b) {
    Pack<T, V> q;
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = T(1), b[i] = T(0);
    if (!on[k]) return;
    if (p.weight) {
      q = load_pack<T, V>(p.weight + g * p.m + channel[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = q.v[i];
    }
    if (p.bias) {
      q = load_pack<T, V>(p.bias + g * p.m + channel[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = q.v[i];
    }
  };
  T kept_w[KEEP ? ITEMS : 1][V], kept_b[KEEP ? ITEMS : 1][V];
  if constexpr (KEEP) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) affine(k, kept_w[k], kept_b[k]);
  }
  // In float32 the sums of dweight and dbias go FEW rows at a time in T and then in
  // float64, which lie in shared memory, each thread's own: to convert and add every
  // value took more of the special-function unit than the activation, and the
  // registers of the next row.
  constexpr bool APART = kRowApart<T, V, LANES, ITEMS, BWD>;
  constexpr int FEW = 4;
  using Sum = std::conditional_t<APART, T, double>;
  Sum dw[BWD ? ITEMS : 1][V], db[BWD ? ITEMS : 1][V];
  extern __shared__ double2 whole[];  // [ITEMS * V][kRowThreads]
  auto apart = [&](int k, int i) -> double2& { return whole[(k * V + i) * kRowThreads<LANES> + threadIdx.x]; };
  if constexpr (BWD) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dw[k][i] = db[k][i] = Sum(0);
        if constexpr (APART) apart(k, i) = make_double2(0.0, 0.0);
      }
  }
  auto fetch = [&](const T* from, int64_t n, Pack<T, V>* to) {
    from += n * sample + g * p.m;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      to[k] = Pack<T, V>{};
      if (on[k] && n < n1) to[k] = load_pack<T, V>(from + place[k]);
    }
  };
  const double share = 1.0 / ((double)p.S * (double)p.m);
  Pack<T, V> x[ITEMS], e[BWD ? ITEMS : 1], x1[AHEAD ? ITEMS : 1], e1[BWD && AHEAD ? ITEMS : 1];
  T mean1 = T(0), rstd1 = T(0);
  auto fetch_row = [&](int64_t n, Pack<T, V>* to, Pack<T, V>* to_e) {
    fetch(p.x, n, to);
    if constexpr (BWD) {
      fetch(p.dy, n, to_e);
      if (n < n1) {
        mean1 = __ldg(p.mean + n * p.G + g);
        rstd1 = __ldg(p.rstd + n * p.G + g);
      }
    }
  };
  if constexpr (AHEAD) fetch_row(n0 + sub, x1, e1);
  // Every part of a unit makes the same number of turns: row_sum is theirs together.
  for (int64_t n = n0 + sub, turns = (n1 - n0 + SUBS - 1) / SUBS; turns > 0; --turns, n += SUBS) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        x[k] = x1[k];
        if constexpr (BWD) e[k] = e1[k];
      }
    } else {
      fetch_row(n, x, e);
    }
    const T mean = mean1, rstd = rstd1;
    if constexpr (AHEAD)
      if (turns > 1) fetch_row(n + SUBS, x1, e1);
    T* const out = p.out + n * sample + g * p.m;
    if constexpr (!BWD) {
      double t = 0.0;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) t += (double)x[k].v[i];
      const double mu = row_sum<LANES>(t) * share;
      // The mean in two parts: x - high is exact near the mean.  The squares are float64:
      // those of float32 deviations beyond 1e19 or below 1e-19 leave float32's range (32768 x
      // 2048: 103.5 us; pair by pair in float32 102).
      const T high = (T)mu, low = (T)(mu - (double)high);
      t = 0.0;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[k].v[i] = (x[k].v[i] - high) - low;
          if (on[k]) t = fma((double)x[k].v[i], (double)x[k].v[i], t);
        }
      }
      const T r = (T)rsqrt(row_sum<LANES>(t) * share + p.eps);
      if (n < n1) {
        if (lane == 0) {
          if (p.mean) p.mean[n * p.G + g] = (T)mu;
          if (p.rstd) p.rstd[n * p.G + g] = r;
        }
        with_activation(act, [&](auto which) {
#pragma unroll
          for (int k = 0; k < ITEMS; ++k) {
            if (!on[k]) continue;
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i)
              o.v[i] = activate<T, decltype(which)::value>(fma(x[k].v[i] * r, kept_w[k][i], kept_b[k][i]));
            store_pack<T, V>(out + place[k], o);
          }
        });
      }
    } else {
      // x becomes xhat, e becomes w dz.  The row's sums go pair by pair in T and
      // then in float64 (see ChannelSums).  Packs and rows that are not there have
      // dy = 0, and mean and rstd of 0 so that 0 times them cannot be NaN.
      double2 t = make_double2(0.0, 0.0);
      with_activation(act, [&](auto which) {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
          const bool there = on[k] && n < n1;
          const T mu = there ? mean : T(0), r = there ? rstd : T(0);
          T w[V], b[V];
          if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = kept_w[k][i], b[i] = kept_b[k][i];
          } else {
            affine(k, w, b);
          }
#pragma unroll
          for (int i = 0; i < V; i += V > 1 ? 2 : 1) {
            T z = T(0), q = T(0);
#pragma unroll
            for (int j = i; j < i + (V > 1 ? 2 : 1); ++j) {
              const T xh = (x[k].v[j] - mu) * r;
              const T dz = e[k].v[j] * slope<T, decltype(which)::value>(fma(xh, w[j], b[j])), product = dz * xh;
              db[k][j] += (Sum)dz;
              dw[k][j] += (Sum)product;
              x[k].v[j] = xh;
              e[k].v[j] = w[j] * dz;
              z = j == i ? e[k].v[j] : z + e[k].v[j];
              q = j == i ? w[j] * product : fma(w[j], product, q);
            }
            t.x += (double)z;
            t.y += (double)q;
          }
        }
      });
      if constexpr (APART) {
        if (turns % FEW == 1) {  // the last turn among them
#pragma unroll
          for (int k = 0; k < ITEMS; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              double2& sum = apart(k, i);
              sum = make_double2(sum.x + (double)db[k][i], sum.y + (double)dw[k][i]);
              db[k][i] = dw[k][i] = Sum(0);
            }
        }
      }
      t = row_sum<LANES>(t);
      // dx = rstd (w dz - m1 - xhat m2)
      const T m1 = (T)(t.x * share), m2 = (T)(t.y * share);
      if (n < n1) {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
          if (!on[k]) continue;
          Pack<T, V> o;
#pragma unroll
          for (int i = 0; i < V; ++i) o.v[i] = rstd * ((e[k].v[i] - m1) - x[k].v[i] * m2);
          store_pack<T, V>(out + place[k], o);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (!p.part) return;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        double2 t = make_double2((double)db[k][i], (double)dw[k][i]);
        if constexpr (APART) t = apart(k, i);
#pragma unroll
        for (int o = LANES; o < UNIT; o <<= 1) {
          t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
          t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
        }
        if (on[k] && sub == 0) p.part[chunk * sample + g * p.m + place[k] + i] = t;
      }
  }
}

// dweight and dbias: `rows` rows of per-channel sums, added in a fixed order.  A
// few hundred rows for each channel: 32 threads share them, since the reads'
// latency is what this takes.
constexpr int kAffineWarps = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kAffineWarps) norm_affine_kernel(const double2* sums, int64_t rows, int64_t C,
                                                                        T* dweight, T* dbias) {
  __shared__ double2 red[kAffineWarps][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  double2 t = make_double2(0.0, 0.0);
  if (c < C) {
#pragma unroll 8
    for (int64_t r = warp; r < rows; r += kAffineWarps) {
      const double2 v = __ldg(sums + r * C + c);
      t.x += v.x;
      t.y += v.y;
    }
  }
  red[warp][lane] = t;
  __syncthreads();
  // Warp w adds up channel w over the lanes.
  t = red[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
    t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
  }
  const int64_t mine = (int64_t)blockIdx.x * 32 + warp;
  if (lane == 0 && mine < C) {
    if (dbias) dbias[mine] = (T)t.x;
    if (dweight) dweight[mine] = (T)t.y;
  }
}

template <typename T>
int launch_affine(Device* d, const double2* sums, int64_t rows, const NormArgs<T>& p) {
  const int64_t blocks = ceil_div(p.C, (int64_t)32);
  if (blocks > INT32_MAX) PB_FAIL(PB_ERR_UNSUPPORTED, "too many channels");
  norm_affine_kernel<T><<<(unsigned)blocks, 32 * kAffineWarps, 0, d->stream>>>(sums, rows, p.C, p.dweight, p.dbias);
  PB_LAUNCHED(d);
  return PB_OK;
}

template <typename T, int V, int LANES, int ITEMS, bool BWD, bool FLAT>
int launch_rows(Device* d, int act, NormArgs<T> p) {
  constexpr int UNIT = LANES < 32 ? 32 : LANES, SUBS = UNIT / LANES;
  const void* kernel = (const void*)norm_rows_kernel<T, V, LANES, ITEMS, BWD, FLAT>;
  // One wave of units.  Backward, each has 16 rows per part at least, so that the
  // sums it writes are little beside what it reads; two where the card were idle else.
  const size_t smem = kRowApart<T, V, LANES, ITEMS, BWD> ? sizeof(double2) * V * ITEMS * kRowThreads<LANES> : 0;
  if (smem > 48 * 1024) PB_CHECK(allow_smem(d, kernel, smem));
  const int64_t wave = resident_blocks(d, kernel, kRowThreads<LANES>, smem) * (kRowThreads<LANES> / UNIT);
  int64_t chunks = ceil_div(wave, p.G);
  const bool sums = BWD && (p.dweight || p.dbias);
  int64_t most = ceil_div(p.N, (int64_t)SUBS * (sums ? 16 : 1));
  if (sums && most * p.G < wave) most = ceil_div(p.N, (int64_t)SUBS * 2);
  // With S > 1 a unit writes S rows of sums, which take norm_affine_kernel 6 ns each, and a
  // sample takes a unit 1.5 us: the least of 1.5 N / (SUBS chunks) + 0.006 S chunks.  2048 x 64 x 8
  // 57 us, 418 with a unit for every two samples; 100 x 64 x 256 23 and 29; 16 x 64 x 1280 19 and 19.
  if (sums && p.S > 1) most = std::min(most, (int64_t)std::ceil(std::sqrt(240.0 * (double)p.N / (double)(p.S * SUBS))));
  if (chunks > most) chunks = most;
  p.rows = ceil_div(p.N, chunks);
  p.chunks = ceil_div(p.N, p.rows);
  p.part = nullptr;
  if (sums) {
    size_t bytes;
    const int64_t e[] = {p.chunks, p.S, p.C};
    if (!array_bytes(e, 3, sizeof(double2), &bytes)) PB_FAIL(PB_ERR_INVALID, "extents too large");
    void* ws;
    PB_CHECK(scratch(d, bytes, &ws));
    p.part = static_cast<double2*>(ws);
  }
  const int64_t blocks = ceil_div(p.G * p.chunks, (int64_t)(kRowThreads<LANES> / UNIT));
  if (blocks > INT32_MAX) PB_FAIL(PB_ERR_UNSUPPORTED, "too many groups");
  PB_CHECK(kt_begin(d));
  norm_rows_kernel<T, V, LANES, ITEMS, BWD, FLAT><<<(unsigned)blocks, kRowThreads<LANES>, smem, d->stream>>>(p, act);
  PB_LAUNCHED(d);
  if (sums) PB_CHECK(launch_affine<T>(d, p.part, p.chunks * p.S, p));
  return kt_end(d);
}

// Packs of 16 bytes of a row that fit the rows kernel.
constexpr int64_t kRowPacks = 2048;

// Of 65 packs on.  Backward, two packs of 16 bytes are what a thread holds beside
// the sums of their channels (16384 x 4 groups of 512: four 134 us, two 85 us).
// Forward, four cost a barrier less often (8192 x 4096: two 83 us, four 52 us).
// Single values (V = 1): as many as two packs hold, so that a warp does up to 256
// (4547 x 42 groups of 169 forward: a block of 128 threads 261 us, a warp 66 us).
template <typename T, int V, bool BWD, bool FLAT>
int launch_wide_rows(Device* d, int act, const NormArgs<T>& p, int64_t packs) {
  constexpr bool TWO = BWD && V > 1;
  constexpr int K = V > 1 ? 2 : 32 / (int)sizeof(T);  // 32 bytes of a row to a thread
  if constexpr (V > 1) {
    if (packs <= 128) return launch_rows<T, V, TWO ? 64 : 32, TWO ? 2 : 4, BWD, FLAT>(d, act, p);
    if (packs <= 256) return launch_rows<T, V, 128, 2, BWD, FLAT>(d, act, p);
    if (packs <= 512) return launch_rows<T, V, 256, 2, BWD, FLAT>(d, act, p);
    if (packs <= 1024) return launch_rows<T, V, TWO ? 512 : 256, TWO ? 2 : 4, BWD, FLAT>(d, act, p);
    return launch_rows<T, V, 512, 4, BWD, FLAT>(d, act, p);
  } else {
    if (packs <= 128) return launch_rows<T, V, 32, 4, BWD, FLAT>(d, act, p);
    if (packs <= 256) return launch_rows<T, V, 256 / K, K, BWD, FLAT>(d, act, p);
    if (packs <= 512) return launch_rows<T, V, 512 / K, K, BWD, FLAT>(d, act, p);
    if (packs <= 1024) return launch_rows<T, V, 1024 / K, K, BWD, FLAT>(d, act, p);
    if (packs <= 2048) return launch_rows<T, V, 2048 / K, K, BWD, FLAT>(d, act, p);
    if (K * 512 > 2048 && packs <= K * 512) return launch_rows<T, V, 512, K, BWD, FLAT>(d, act, p);
    return launch_rows<T, V, 512, 2 * K, BWD, FLAT>(d, act, p);
  }
}

template <typename T, int V, bool BWD>
int launch_rows_of(Device* d, int act, const NormArgs<T>& p) {
  const int64_t packs = p.S * (p.m / V);
  if (p.S > 1) {
    if (packs <= 8) return launch_rows<T, V, 8, 1, BWD, false>(d, act, p);
    if (packs <= 64) return launch_rows<T, V, 32, 2, BWD, false>(d, act, p);
    return launch_wide_rows<T, V, BWD, false>(d, act, p, packs);
  }
  if (packs <= 2) return launch_rows<T, V, 2, 1, BWD, true>(d, act, p);
  if (packs <= 4) return launch_rows<T, V, 4, 1, BWD, true>(d, act, p);
  if (packs <= 8) return launch_rows<T, V, 8, 1, BWD, true>(d, act, p);
  if constexpr (V > 1) {
    if (packs <= 16) return launch_rows<T, V, 8, 2, BWD, true>(d, act, p);
    if (packs <= 32) return launch_rows<T, V, 16, 2, BWD, true>(d, act, p);
    if (packs <= 64) return launch_rows<T, V, 32, 2, BWD, true>(d, act, p);
  } else {
    if (packs <= 16) return launch_rows<T, V, 4, 4, BWD, true>(d, act, p);
    if (packs <= 32) return launch_rows<T, V, 8, 4, BWD, true>(d, act, p);
    if (packs <= 64) return launch_rows<T, V, 16, 4, BWD, true>(d, act, p);
  }
  return launch_wide_rows<T, V, BWD, true>(d, act, p, packs);
}

// Scratch, counters and flags of the samples kernels for p.N * p.chunks units and
// that many rows of per-channel sums.
template <typename T, bool BWD>
int sample_workspace(Device* d, NormArgs<T>& p, bool shared_channels, int64_t channel_sums) {
  const int64_t units = p.N * p.chunks;
  if (units >= (int64_t(1) << 30)) PB_FAIL(PB_ERR_UNSUPPORTED, "more than 2^30 samples");
  const bool by_channel = (BWD && (p.dweight || p.dbias)) || !shared_channels;
  size_t chan = 0, part, group;
  const int64_t e1[] = {channel_sums, p.C}, e2[] = {units, p.G}, e3[] = {p.N, p.G};
  if ((by_channel && !array_bytes(e1, 2, sizeof(double2), &chan)) || !array_bytes(e2, 2, sizeof(double2), &part) ||
      !array_bytes(e3, 2, sizeof(double2), &group))
    PB_FAIL(PB_ERR_INVALID, "extents too large");
  void* ws;
  PB_CHECK(scratch(d, part + chan + group, &ws));
  p.part = static_cast<double2*>(ws);
  p.group = p.part + part / sizeof(double2);
  p.chan = by_channel ? p.group + group / sizeof(double2) : nullptr;
  if (p.chunks > 1) PB_CHECK(counters(d, (size_t)p.N, &p.arrivals));
  PB_CHECK(epoch_words(d, kFlagWords + (size_t)p.N, &p.words));
  p.err = d->err_dev;
  p.by_chunks = make_fastdiv(p.chunks);
  p.by_m = make_fastdiv(p.m);
  return PB_OK;
}

template <typename T, int V, int ACT, bool BWD>
int launch_items(Device* d, NormArgs<T> p, int tx, int ty) {
  const void* kernel = (const void*)norm_samples_kernel<T, V, ACT, BWD>;
  const int64_t wave = resident_blocks(d, kernel, kThreads);
  int64_t chunks = ceil_div(wave * 2, p.N);
  const int64_t most = ceil_div(p.S, (int64_t)ty * 4);
  const int64_t least = ceil_div(p.S, (int64_t)ty * 64);
  if (chunks < least) chunks = least;
  if (chunks > most) chunks = most;
  p.rows = ceil_div(p.S, chunks);
  p.chunks = ceil_div(p.S, p.rows);
  PB_CHECK((sample_workspace<T, BWD>(d, p, p.C <= kSharedChannels, p.N * p.chunks)));
  const int64_t units = p.N * p.chunks;
  const int64_t grid = 2 * units < wave ? 2 * units : wave;
  const int64_t lead = p.chunks + 2 * grid < units ? p.chunks + 2 * grid : units;
  PB_CHECK(kt_begin(d));
  norm_samples_kernel<T, V, ACT, BWD>
      <<<(unsigned)grid, kThreads, 0, d->stream>>>(p, tx, ty, (unsigned)units, (unsigned)lead);
  PB_LAUNCHED(d);
  if (BWD && (p.dweight || p.dbias)) PB_CHECK(launch_affine<T>(d, p.chan, units, p));
  return kt_end(d);
}

template <typename T, int V, int ACT, bool BWD, bool SPREAD>
int launch_ring(Device* d, NormArgs<T> p) {
  constexpr int kArrays = BWD ? 2 : 1;
  const int tx = (int)ceil_div(p.C, (int64_t)V), ty = kRingThreads / tx;
  const int64_t row_bytes = p.C * (int64_t)sizeof(T) * kArrays;
  const int64_t fixed = (int64_t)sizeof(double2) * (V * kRingThreads + p.C + (p.G <= kOwnGroups ? p.G : 0));
  // The ring takes what is left of shared memory; positions per stage in
  // pairs per thread where they fit.
  int64_t stage_rows = ((int64_t)kRingSmem - fixed) / kRing / row_bytes;
  if (SPREAD) stage_rows = ((int64_t)kRingSmem - fixed - kRing * kArrays * 32) / kRing / row_bytes;  // two boundaries
  if (stage_rows > 2 * ty) stage_rows = stage_rows / (2 * ty) * (2 * ty);
  const void* kernel = (const void*)norm_ring_kernel<T, V, ACT, BWD, SPREAD>;
  const size_t bytes = (size_t)(kRing * kArrays * ring_array<T, SPREAD>(stage_rows, p.C) * (int64_t)sizeof(T) + fixed);
  PB_CHECK(allow_smem(d, kernel, kRingSmem));
  const int64_t wave = d->sm_count;
  // Samples worked on together: their operands stay in L2 between the passes,
  // and a block has at least two positions per thread.
  const int64_t most = ceil_div(p.S, (int64_t)ty * 2);
  int64_t together = (int64_t(48) << 20) / (p.S * row_bytes);
  if (together < ceil_div(wave, most)) together = ceil_div(wave, most);
  if (together < 1) together = 1;
  if (together > wave) together = wave;
  if (together > p.N) together = p.N;
  together = ceil_div(p.N, ceil_div(p.N, together));  // rounds of equal size
  int64_t chunks = wave / together;
  if (chunks > most) chunks = most;
  p.rows = ceil_div(p.S, chunks);
  p.chunks = ceil_div(p.S, p.rows);
  PB_CHECK((sample_workspace<T, BWD>(d, p, true, together * p.chunks)));
  PB_CHECK(kt_begin(d));
  int rows = (int)stage_rows, lanes = tx, thread_rows = ty;
  void* args[] = {&p, &lanes, &thread_rows, &rows, &together};
  PB_CUDA(cudaLaunchCooperativeKernel(kernel, dim3((unsigned)(together * p.chunks)), dim3(kRingThreads + 32), args,
                                      bytes, d->stream));
  PB_LAUNCHED(d);
  if (BWD && (p.dweight || p.dbias)) PB_CHECK(launch_affine<T>(d, p.chan, together * p.chunks, p));
  return kt_end(d);
}

// The ring takes rows that its threads span, of whole 16-byte pieces or not.
template <typename T>
bool ring_takes(const NormArgs<T>& p) {
  return (((uintptr_t)p.x | (uintptr_t)p.dy) & 15) == 0 && ceil_div(p.C, (int64_t)Vec16<T>::n) <= kRingThreads;
}

template <typename T, int V, int ACT, bool BWD>
int launch(Device* d, const NormArgs<T>& p) {
  const int64_t lanes = ceil_div(p.C, (int64_t)V);
  const int tx = (int)(lanes < kThreads ? lanes : kThreads), ty = kThreads / tx;
  if (ring_takes(p)) return launch_ring<T, Vec16<T>::n, ACT, BWD, V == 1>(d, p);
  return launch_items<T, V, ACT, BWD>(d, p, tx, ty);
}

template <typename T, int V, bool BWD>
int launch_act(Device* d, int act, const NormArgs<T>& p) {
  switch (act) {
    case PB_ACT_RELU: return launch<T, V, PB_ACT_RELU, BWD>(d, p);
    case PB_ACT_SILU: return launch<T, V, PB_ACT_SILU, BWD>(d, p);
    case PB_ACT_GELU: return launch<T, V, PB_ACT_GELU, BWD>(d, p);
    default: return launch<T, V, PB_ACT_NONE, BWD>(d, p);
  }
}

// Whether a group that fits the registers of a block is read there, once, rather than by
// the ring.  Times in us, rows and ring, silu, float32.
template <typename T, bool BWD>
bool rows_pay(Device* d, const NormArgs<T>& p) {
  if (p.S == 1 || !ring_takes(p)) return true;
  const int64_t run = p.m * (int64_t)sizeof(T), sample = p.S * p.C * (int64_t)sizeof(T);
  const double rounds = (double)ceil_div(p.N, (int64_t)d->sm_count);
  const bool sums = BWD && (p.dweight || p.dbias);
  // Runs of less than the 32 bytes that memory moves at once: the rows read some 0.6 TB/s
  // (1.3 from 16 bytes on) and the ring, which copies whole positions, 4, but it takes 6.5 us
  // more for each round of a sample per block.  Forward, groups of one channel: 16 x 512 x 64
  // 10.6 and 12.7, 8 x 4096 x 320 163 and 31, 1000 x 64 x 640 495 and 118 (of four 154 and 101),
  // 10000 x 64 x 64 402 and 380, 40000 x 65 x 32 849 and 1385.  Gradients with sums for each
  // position: 2000 x 200 x 32 of four 166 and 118, 20000 x 100 x 64 2033 and 1002.
  if (run < 32) {
    if (sums && p.S > 64) return false;
    const double moved = (BWD ? 3.0 : 2.0) * (double)p.N * (double)sample;
    return moved / (run < 16 ? 0.6e6 : 1.3e6) <= 10.0 + 6.5 * rounds + moved / 4e6;
  }
  // The rows give a row of sums for dweight and dbias for each position: with many
  // positions the ring's sums of whole runs are less to add up, unless it takes many
  // rounds over small samples.  Gradients, groups of eight: 1000 x 64 x 256 73 and 85, 1000 x 65 x
  // 256 114 and 85, 148 x 65 x 64 46 and 16, 1500 x 100 x 64 89 and 95, 5000 x 65 x 64 126 and 253, 20000 x
  // 128 x 64 546 and 1087, 5000 x 65 x 256 510 and 352.
  if (!sums) return true;
  return p.S <= 64 || (p.S <= 128 && rounds > 8 && sample <= kRowPacks * 16);
}

struct Pointers {
  const void *x, *dy, *weight, *bias;
  void *out, *mean, *rstd, *dweight, *dbias;
};

template <typename T, bool BWD>
int dispatch(Device* d, int act, int64_t N, int64_t S, int64_t C, int64_t G, double eps, const Pointers& q) {
  NormArgs<T> p = {};
  p.x = static_cast<const T*>(q.x);
  p.dy = static_cast<const T*>(q.dy);
  p.weight = static_cast<const T*>(q.weight);
  p.bias = static_cast<const T*>(q.bias);
  p.out = static_cast<T*>(q.out);
  p.mean = static_cast<T*>(q.mean);
  p.rstd = static_cast<T*>(q.rstd);
  p.dweight = static_cast<T*>(q.dweight);
  p.dbias = static_cast<T*>(q.dbias);
  p.N = N;
  p.S = S;
  p.C = C;
  p.G = G;
  p.m = C / G;
  p.eps = eps;
  constexpr int V = Vec16<T>::n;
  const bool aligned = (((uintptr_t)q.x | (uintptr_t)q.dy | (uintptr_t)q.out | (uintptr_t)q.weight | (uintptr_t)q.bias) & 15) == 0;
  if (S <= kRowPacks * V && S * C < (int64_t(1) << 31) && S * p.m <= kRowPacks * V && rows_pay<T, BWD>(d, p))
    return aligned && p.m % V == 0 ? launch_rows_of<T, V, BWD>(d, act, p) : launch_rows_of<T, 1, BWD>(d, act, p);
  return aligned && C % V == 0 ? launch_act<T, V, BWD>(d, act, p) : launch_act<T, 1, BWD>(d, act, p);
}

// Checks common to both directions; the bytes of x and of one sample's statistics.
int check_view(pb_ctx* ctx, int dtype, int act, int64_t N, int64_t S, int64_t C, int64_t G, size_t* bytes,
               size_t* stats) {
  if (!ctx) PB_FAIL(PB_ERR_INVALID, "null context");
  if (dtype != PB_F32 && dtype != PB_F64) PB_FAIL(PB_ERR_INVALID, "group norm takes float32 or float64");
  if (act < PB_ACT_NONE || act > PB_ACT_GELU) PB_FAIL(PB_ERR_INVALID, "unknown activation %d", act);
  if (N < 0 || S < 0 || C < 0) PB_FAIL(PB_ERR_INVALID, "negative extent");
  if (G < 1 || C % G) PB_FAIL(PB_ERR_INVALID, "%lld channels do not divide into %lld groups", (long long)C, (long long)G);
  if (!S || !C) PB_FAIL(PB_ERR_INVALID, "group norm of an empty set");
  const size_t item = dtype == PB_F32 ? 4 : 8;
  const int64_t all[3] = {N, S, C}, ends[2] = {N, G};
  if (!array_bytes(all, 3, item, bytes) || !array_bytes(ends, 2, item, stats))
    PB_FAIL(PB_ERR_INVALID, "extents too large");
  return PB_OK;
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" {

int pb_group_norm(pb_ctx* ctx, int dev, int dtype, int act, int64_t N, int64_t S, int64_t C, int64_t G, double eps,
                  const void* x, const void* weight, const void* bias, void* y, void* mean, void* rstd) {
  size_t bytes, stats;
  PB_CHECK(check_view(ctx, dtype, act, N, S, C, G, &bytes, &stats));
  if (!(eps >= 0.0)) PB_FAIL(PB_ERR_INVALID, "eps is negative or NaN");
  if (!N) return PB_OK;
  if (!x || !y) PB_FAIL(PB_ERR_INVALID, "null operand");
  const size_t item = dtype == PB_F32 ? 4 : 8, line = (size_t)C * item;
  const Span in[] = {{x, bytes}, {weight, line}, {bias, line}};
  const Span out[] = {{y, bytes}, {mean, stats}, {rstd, stats}};
  PB_CHECK(check_operands(out, 3, in, 3, item));
  std::lock_guard<std::recursive_mutex> g(ctx->mu);
  Device* d;
  PB_CHECK(enter(ctx, dev, &d));
  const Pointers q = {x, nullptr, weight, bias, y, mean, rstd, nullptr, nullptr};
  return dtype == PB_F32 ? dispatch<float, false>(d, act, N, S, C, G, eps, q)
                         : dispatch<double, false>(d, act, N, S, C, G, eps, q);
}

int pb_group_norm_backward(pb_ctx* ctx, int dev, int dtype, int act, int64_t N, int64_t S, int64_t C, int64_t G,
                           const void* dy, const void* x, const void* mean, const void* rstd, const void* weight,
                           const void* bias, void* dx, void* dweight, void* dbias) {
  size_t bytes, stats;
  PB_CHECK(check_view(ctx, dtype, act, N, S, C, G, &bytes, &stats));
  const size_t item = dtype == PB_F32 ? 4 : 8, line = (size_t)C * item;
  if (N && (!dy || !x || !mean || !rstd || !dx)) PB_FAIL(PB_ERR_INVALID, "null operand");
  const Span in[] = {{dy, bytes}, {x, bytes}, {mean, stats}, {rstd, stats}, {weight, line}, {bias, line}};
  const Span out[] = {{dx, bytes}, {dweight, line}, {dbias, line}};
  PB_CHECK(check_operands(out, 3, in, 6, item));
  std::lock_guard<std::recursive_mutex> g(ctx->mu);
  Device* d;
  PB_CHECK(enter(ctx, dev, &d));
  if (!N) {
    for (void* q : {dweight, dbias})
      if (q) PB_CHECK(fill_device(d, dtype, q, (size_t)C, 0.0));
    return PB_OK;
  }
  const Pointers q = {x, dy, weight, bias, dx, const_cast<void*>(mean), const_cast<void*>(rstd), dweight, dbias};
  return dtype == PB_F32 ? dispatch<float, true>(d, act, N, S, C, G, 0.0, q)
                         : dispatch<double, true>(d, act, N, S, C, G, 0.0, q);
}

}  // extern "C"
