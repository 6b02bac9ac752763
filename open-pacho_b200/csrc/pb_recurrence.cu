// Gated linear recurrence h_t = alpha_t h_{t-1} + u_t along an axis, and its
// gradients (HBM-bound: forward 3 values moved per element, backward 5 or 6).
//
// The backward pass is the same recurrence run from the last step to the
// first, g_t = alpha_{t+1} g_{t+1} + dh_t, so the same kernels serve both: step s
// of the chain is t = s forward and t = length - 1 - s backward.
//
// A column is one (outer, inner) pair; neighbouring columns are neighbours in
// memory, so lanes run over columns and a warp's access is a row segment.  A lane
// walks its chain in order, and nothing but the bytes on their way limits it: each
// warp is a block of its own with a ring of stages in shared memory that
// asynchronous copies fill ahead of it, so about 500 warps with 16 KiB each
// under way keep HBM busy and no block ever waits for another.
//
// Fewer columns than that: the chain is cut into segments of equal length, and a
// lane walks one segment of one column.  n steps map x to P x + H, with P the
// product of their coefficients and H their result from 0; a first pass forms
// the maps of the segments, and each lane of the second composes those before
// its own to find its start.  The first pass walks each segment from its end to
// its start (H += P u, P *= c), so that L2 holds the steps that the second
// pass reads first (1 x 16381 x 1024 float32: 57 of 134 MB).  P and H are float64: a product of thousands of gates
// neither over- nor underflows where a float32 recurrence does not.  Every
// composition has a fixed order, so results do not depend on timing.
//
// Few steps, or columns enough to fill the card with threads: a thread per column
// reads directly (recurrence_columns_kernel).
#include <type_traits>

#include "pb_layers.cuh"

namespace pb {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 16;        // chain steps per stage
constexpr int kInlineMaps = 32;  // segments up to which a lane composes the maps before its own itself

template <typename T>
struct ScanArgs {
  const T *a, *b, *h, *dh;   // h, dh: backward only
  const T* start;            // forward: state; backward: dfinal; may be null
  const T* state;            // backward: h[-1]; may be null
  T* out0;                   // forward: h; backward: da
  T* out1;                   // backward: db
  T* last;                   // forward: final; backward: dstate; may be null
  int64_t length, inner, columns;
  FastDiv by_inner, by_columns;
  int wide;                  // 16-byte copies are aligned
  int64_t segments, steps;   // segments of `steps` chain steps (the last may be shorter)
  double2* maps;             // [segment][column]: (P, H)
  double* starts;            // [segment][column]: the value before the segment (many segments)
};

template <typename T>
__device__ __forceinline__ int64_t column_base(const ScanArgs<T>& p, int64_t col) {
  const int64_t o = fdiv(col, p.by_inner);
  return o * p.length * p.inner + (col - o * p.inner);
}

// The value `e` elements (of the type that addresses this array) into it.  A
// 32-bit I serves arrays below 4 GiB: one offset for all operands of a step.
template <typename T, typename I>
__device__ __forceinline__ const T* at(const T* p, I e) {
  if constexpr (sizeof(I) == 4) return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + e * (I)sizeof(T));
  else return p + e;
}
template <typename T, typename I>
__device__ __forceinline__ T* at(T* p, I e) {
  return const_cast<T*>(at(static_cast<const T*>(p), e));
}

// Element of chain step s of a column.
template <bool BWD, typename I, typename T>
__device__ __forceinline__ I element(const ScanArgs<T>& p, I base, int64_t s) {
  return base + (I)(BWD ? p.length - 1 - s : s) * (I)p.inner;
}

// One chain step.  Backward, the own gate gives the outputs and is the
// coefficient of the next step.
template <typename T, int GATE, bool BWD>
struct Step;

template <typename T, int GATE>
struct Step<T, GATE, false> {
  __device__ __forceinline__ static void operands(T a, T b, T* c, T* u) {
    if constexpr (GATE == PB_GATE_SIGMOID) {
      T rest;
      sigmoid_pair(a, c, &rest);
      *u = rest * b;
    } else {
      *c = a;
      *u = b;
    }
  }
};

template <typename T, int GATE>
struct Step<T, GATE, true> {
  __device__ __forceinline__ static T gate(T a, T* rest) {
    if constexpr (GATE == PB_GATE_SIGMOID) {
      T s;
      sigmoid_pair(a, &s, rest);
      return s;
    } else {
      return a;
    }
  }
  // da and db of a step with the chain value g.
  __device__ __forceinline__ static void outputs(T g, T alpha, T rest, T before, T b, T* da, T* db) {
    if constexpr (GATE == PB_GATE_SIGMOID) {
      *db = g * rest;
      *da = g * (before - b) * (alpha * rest);
    } else {
      *db = g;
      *da = g * before;
    }
  }
};

// A thread per column, the whole chain in order; the loads of kAhead steps are
// issued together.
template <typename T, typename I, int GATE, bool BWD>
__global__ void __launch_bounds__(kThreads) recurrence_columns_kernel(const ScanArgs<T> p) {
  constexpr int kAhead = 16;
  const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (col >= p.columns) return;
  const I base = (I)column_base(p, col), step = (I)p.inner;
  T x = p.start ? p.start[col] : T(0);
  T c = T(1);  // backward: the coefficient of the next step
  // kAhead steps (FULL), or the `left` last ones.
  auto walk = [&](auto full, int64_t s0, int left) {
    constexpr bool FULL = decltype(full)::value;
    const I e = element<BWD>(p, base, s0);
    T a[kAhead], b[kAhead], g[BWD ? kAhead : 1], before[BWD ? kAhead : 1];
    I q = e;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (FULL || i < left) {
        a[i] = __ldg(at(p.a, q));
        if (!BWD || GATE == PB_GATE_SIGMOID) b[i] = __ldg(at(p.b, q));
        if constexpr (BWD) {
          g[i] = __ldg(at(p.dh, q));
          if (FULL || i + 1 < left) before[i] = __ldg(at(p.h, (I)(q - step)));
          else before[i] = p.state ? p.state[col] : T(0);
        }
        q = BWD ? (I)(q - step) : (I)(q + step);
      }
    }
    q = e;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (FULL || i < left) {
        if constexpr (!BWD) {
          T u;
          Step<T, GATE, false>::operands(a[i], b[i], &c, &u);
          x = fma(c, x, u);
          *at(p.out0, q) = x;
        } else {
          x = fma(c, x, g[i]);
          T rest = T(0), da, db;
          c = Step<T, GATE, true>::gate(a[i], &rest);
          Step<T, GATE, true>::outputs(x, c, rest, before[i], b[i], &da, &db);
          *at(p.out1, q) = db;
          *at(p.out0, q) = da;
        }
        q = BWD ? (I)(q - step) : (I)(q + step);
      }
    }
  };
  // The last steps go apart: t = 0, whose h[t - 1] is the state, is among them.
  int64_t s0 = 0;
  for (; s0 + kAhead < p.length; s0 += kAhead) walk(std::true_type{}, s0, kAhead);
  if (s0 < p.length) walk(std::false_type{}, s0, (int)(p.length - s0));
  if (p.last) p.last[col] = BWD ? c * x : x;
}

// Maps x -> P x + H.  A product of finite factors that overflows is +-Inf, and a zero
// wins over it: a value of 0, or a gate of 0 (a reset).  A factor that is not
// finite makes P NaN, over which nothing wins.
__device__ __forceinline__ bool bounded(double P) { return fabs(P) <= 1.7976931348623157e308; }
// P v + H
__device__ __forceinline__ double apply(double P, double v, double H) {
  if (bounded(P)) return fma(P, v, H);
  return v == 0.0 && isinf(P) ? H : fma(P, v, H);
}
// P c
__device__ __forceinline__ double extend(double P, double c) {
  const double q = P * c;
  if (bounded(q)) return q;
  if (!isfinite(c)) return c - c;
  return c == 0.0 && isinf(P) ? 0.0 : q;
}
__device__ __forceinline__ double apply(const double2& map, double x) { return apply(map.x, x, map.y); }
// The map of `a` followed by `b`.
__device__ __forceinline__ double2 compose(const double2& a, const double2& b) {
  const double P = a.x * b.x;
  return make_double2(P != P && (a.x == 0.0 || b.x == 0.0) && !(isnan(a.x) || isnan(b.x)) ? 0.0 : P, apply(b, a.y));
}

// Asynchronous copy of BYTES into shared memory; zeros where `there` is false
// (nothing is read then).
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool there) {
  const unsigned s = shared_address(to);
  const int n = there ? BYTES : 0;
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(from), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(s), "l"(from), "n"(BYTES), "r"(n) : "memory");
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  const unsigned s = shared_address(to);
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(s), "l"(from), "n"(BYTES) : "memory");
}

// The operands of a stage: forward a, b; backward a, dh and, unless only maps
// are formed, h[t - 1] and (sigmoid) b.
template <int GATE, bool BWD, bool MAPS>
constexpr int stream_arrays() {
  return !BWD || MAPS ? 2 : GATE == PB_GATE_SIGMOID ? 4 : 3;
}

// A warp: lane l takes (segment, column) number blockIdx.x * 32 + l.  MAPS: the
// first pass (from the segment's end to its start), else the outputs.
template <typename T, typename I, int GATE, bool BWD, bool MAPS, int STAGES>
__global__ void __launch_bounds__(32) recurrence_stream_kernel(const ScanArgs<T> p) {
  constexpr int kArrays = stream_arrays<GATE, BWD, MAPS>();
  constexpr int V = 16 / (int)sizeof(T), kLanes = 32 / V;  // lanes that copy a row of 32 values
  extern __shared__ __align__(16) unsigned char smem[];
  T* const ring = reinterpret_cast<T*>(smem);  // [STAGES][kArrays][kRows][32]
  const int lane = threadIdx.x;
  const int64_t item = (int64_t)blockIdx.x * 32 + lane;
  const int64_t total = (MAPS ? p.segments - 1 : p.segments) * p.columns;
  const bool on = item < total;
  const int64_t segment = on ? fdiv(item, p.by_columns) : 0, col = on ? item - segment * p.columns : 0;
  const int64_t s0 = segment * p.steps;
  const int64_t n = on ? min(p.steps, p.length - s0) : 0;  // this lane's steps
  const I base = (I)column_base(p, col), step = (I)p.inner;
  // Row r of the walk is chain step s0 + r, or from the segment's end s0 + n - 1 - r.
  constexpr bool kUp = BWD == MAPS;  // memory offsets grow along the walk
  const I first = element<BWD>(p, base, MAPS ? s0 + n - 1 : s0);
  // What this lane copies: its own column value by value, or 16 bytes of the
  // column pack of lane (lane % kLanes) * V.
  const bool wide = p.wide;
  const int source = wide ? lane % kLanes * V : lane;
  const I from = (I)__shfl_sync(0xffffffffu, first, source);
  const int64_t count = __shfl_sync(0xffffffffu, n, source);
  const int row0 = wide ? lane / kLanes : 0, rows = wide ? V : 1;
  // Where backward's h[t - 1] of the last step is the state, nothing is copied.
  const int64_t zero = BWD && !MAPS ? p.length - 1 - s0 : -1;  // the row of t = 0, if it is one of this lane's
  const int64_t from_zero = BWD && !MAPS ? __shfl_sync(0xffffffffu, zero, source) : -1;
  int64_t most = n;  // the longest of the warp
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max(most, (int64_t)__shfl_xor_sync(0xffffffffu, most, o));
  const int64_t stages = (most + kRows - 1) / kRows;

  constexpr int kStage = kArrays * kRows * 32;  // values
  int copy_slot = 0, slot = 0;                  // where the next copy goes, and the stage at hand is
  auto copy = [&](int64_t k) {
    if (k < stages) {
      T* const to = ring + copy_slot * kStage + source;
      copy_slot = copy_slot + 1 == STAGES ? 0 : copy_slot + 1;
      const I ahead = (I)(k * kRows + row0) * step;
      I e = kUp ? (I)(from + ahead) : (I)(from - ahead);
      const I de = kUp ? (I)((I)rows * step) : (I)(I(0) - (I)rows * step);
      const int64_t left = count - k * kRows, none = from_zero - k * kRows;
      // A stage whose rows are all there needs no sizes; `bytes` of a copy else.
      auto some = [&](auto whole, auto bytes, int r) {
        constexpr bool WHOLE = decltype(whole)::value;
        constexpr int N = decltype(bytes)::value;
        const bool there = WHOLE || r < left;
        auto put = [&](int array, const T* src, bool now) {
          T* const q = to + (array * kRows + r) * 32;
          if constexpr (WHOLE) copy_async<N>(q, src);
          else copy_async<N>(q, now ? src : p.a, now);
        };
        put(0, at(p.a, e), there);
        put(1, at(BWD ? p.dh : p.b, e), there);
        if constexpr (kArrays > 2) put(2, at(p.h, (I)(e - step)), there && r != none);
        if constexpr (kArrays > 3) put(3, at(p.b, e), there);
        e += de;
      };
      auto all = [&](auto whole) {
        if (wide) {
#pragma unroll
          for (int r = 0; r < kRows / V; ++r) some(whole, std::integral_constant<int, 16>{}, row0 + r * V);
        } else {
#pragma unroll
          for (int r = 0; r < kRows; ++r) some(whole, std::integral_constant<int, (int)sizeof(T)>{}, r);
        }
      };
      if (__all_sync(0xffffffffu, left >= kRows && !(kArrays > 2 && none >= 0 && none < kRows))) all(std::true_type{});
      else all(std::false_type{});
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int k = 0; k < STAGES - 1; ++k) copy(k);

  // The value before the segment.
  T x = T(0);
  if constexpr (!MAPS) {
    if (on) {
      if (p.starts) {
        x = (T)p.starts[item];
      } else {
        double v = p.start ? (double)p.start[col] : 0.0;
        for (int64_t k = 0; k < segment; k += 8) {
          double2 m[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (k + i < segment) m[i] = p.maps[(k + i) * p.columns + col];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (k + i < segment) v = apply(m[i], v);
        }
        x = (T)v;
      }
    }
  }
  // Backward: the coefficient of the next step, at first that of the segment's
  // first one: the gate at t + 1, or 1 at the end of the sequence.
  T c = T(1);
  const T state = BWD && !MAPS && on && p.state ? __ldg(p.state + col) : T(0);
  if constexpr (BWD && !MAPS) {
    if (on && s0 > 0) {
      T unused = T(0);
      c = Step<T, GATE, true>::gate(__ldg(at(p.a, (I)(first + step))), &unused);
    }
  }
  double P = 1.0, H = 0.0;
  I e = first;
  for (int64_t k = 0; k < stages; ++k) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();  // every lane's copies are there, and every lane has left the stage that is filled next
    copy(k + STAGES - 1);
    const T* const q = ring + slot * kStage + lane;
    slot = slot + 1 == STAGES ? 0 : slot + 1;
    const int64_t left = n - k * kRows;
    // `careful`: a product may be unbounded.
    auto one = [&](auto careful, int i) {
      constexpr bool CAREFUL = decltype(careful)::value;
      const T a = q[i * 32], b = q[(kRows + i) * 32];
      if constexpr (MAPS && !BWD) {
        T c1, u;
        Step<T, GATE, false>::operands(a, b, &c1, &u);
        H = CAREFUL ? apply(P, (double)u, H) : fma(P, (double)u, H);
        P = CAREFUL ? extend(P, (double)c1) : P * (double)c1;
      } else if constexpr (MAPS) {
        // Walking towards the chain's start: the gate of a step is the
        // coefficient of the step behind it, which came before.
        T unused = T(0);
        if (k * kRows + i > 0) {
          const double c1 = (double)Step<T, GATE, true>::gate(a, &unused);
          P = CAREFUL ? extend(P, c1) : P * c1;
        }
        H = CAREFUL ? apply(P, (double)b, H) : fma(P, (double)b, H);
      } else if constexpr (!BWD) {
        T c1, u;
        Step<T, GATE, false>::operands(a, b, &c1, &u);
        x = fma(c1, x, u);
        *at(p.out0, e) = x;
        e += step;
      } else {
        x = fma(c, x, b);
        T rest = T(0), da, db;
        c = Step<T, GATE, true>::gate(a, &rest);
        T before = q[(2 * kRows + i) * 32], put = T(0);
        if (k * kRows + i == zero) before = state;
        if constexpr (kArrays > 3) put = q[(3 * kRows + i) * 32];
        Step<T, GATE, true>::outputs(x, c, rest, before, put, &da, &db);
        *at(p.out1, e) = db;
        *at(p.out0, e) = da;
        e -= step;
      }
    };
    // Once a product has left float64's range, or met a NaN, it stays there: one
    // look at the end of a stage tells whether it has to be walked with care.
    const double P0 = P, H0 = H;
    bool done = false;
    if (left >= kRows) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) one(std::false_type{}, i);
      done = !MAPS || bounded(P);
    }
    if (!done) {
      P = P0;
      H = H0;
      for (int i = 0; i < min(left, (int64_t)kRows); ++i) one(std::true_type{}, i);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (!on) return;
  if constexpr (MAPS) {
    if constexpr (BWD) {
      // The first step's own coefficient.
      if (s0 > 0) {
        T unused = T(0);
        const T a = __ldg(at(p.a, (I)(element<true>(p, base, s0) + step)));
        P = extend(P, (double)Step<T, GATE, true>::gate(a, &unused));
      }
    }
    p.maps[item] = make_double2(P, H);
  } else if (p.last && s0 + n == p.length) {
    p.last[col] = BWD ? c * x : x;
  }
}

// The value before each segment of a column, where segments are many: a warp
// per column, its lanes composing consecutive runs of maps.
template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_starts_kernel(const ScanArgs<T> p) {
  const int64_t col = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  if (col >= p.columns) return;
  const int lane = threadIdx.x & 31;
  const int64_t run = (p.segments + 31) / 32, k0 = lane * run, k1 = min(p.segments, k0 + run);
  double2 map = make_double2(1.0, 0.0);
#pragma unroll 4
  for (int64_t k = k0; k < k1 && k < p.segments - 1; ++k) map = compose(map, p.maps[k * p.columns + col]);
  // Over the lanes, in order.
  double x = p.start ? (double)p.start[col] : 0.0, mine = x;
  for (int l = 0; l < 31; ++l) {
    double2 m;
    m.x = __shfl_sync(0xffffffffu, map.x, l);
    m.y = __shfl_sync(0xffffffffu, map.y, l);
    x = apply(m, x);
    if (lane == l + 1) mine = x;
  }
  for (int64_t k = k0; k < k1; ++k) {
    p.starts[k * p.columns + col] = mine;
    if (k < p.segments - 1) mine = apply(p.maps[k * p.columns + col], mine);
  }
}

template <typename T, typename I, int GATE, bool BWD, bool MAPS, int STAGES>
int launch_ring(Device* d, const ScanArgs<T>& p, int64_t warps) {
  constexpr size_t bytes = sizeof(T) * STAGES * stream_arrays<GATE, BWD, MAPS>() * kRows * 32;
  PB_CHECK(allow_smem(d, (const void*)recurrence_stream_kernel<T, I, GATE, BWD, MAPS, STAGES>, bytes));
  recurrence_stream_kernel<T, I, GATE, BWD, MAPS, STAGES><<<(unsigned)warps, 32, bytes, d->stream>>>(p);
  PB_LAUNCHED(d);
  return PB_OK;
}

template <typename T, typename I, int GATE, bool BWD, bool MAPS>
int launch_stream(Device* d, const ScanArgs<T>& p) {
  constexpr int kArrays = stream_arrays<GATE, BWD, MAPS>();
  const int64_t warps = ceil_div((MAPS ? p.segments - 1 : p.segments) * p.columns, (int64_t)32);
  // Few warps: what keeps HBM busy is on its way for each (float32: 32 KiB
  // forward, 24 backward).  Many: less, so that more of them fit an SM.  8 x
  // 4096 x 2048 float32, 512 warps: forward 127 us with eight stages, 139 with four;
  // backward 249 with three of four arrays, 300 with six, 334 with two.
  // 3 x 1000 x 515 float64 backward, 435 warps: 26 us with eight stages for the maps and
  // four for the outputs, 29 with five and four, 30 with eight and six.
  const int64_t per_sm = ceil_div(warps, (int64_t)d->sm_count);
  if constexpr (kArrays == 2) {
    if (per_sm > (sizeof(T) == 4 ? 6 : 3))
      return launch_ring<T, I, GATE, BWD, MAPS, (sizeof(T) == 4 ? 5 : 3)>(d, p, warps);
    return launch_ring<T, I, GATE, BWD, MAPS, 8>(d, p, warps);
  } else {
    return launch_ring<T, I, GATE, BWD, MAPS, (kArrays == 3 ? 4 : 3)>(d, p, warps);
  }
}

template <typename T, typename I, int GATE, bool BWD>
int launch(Device* d, ScanArgs<T>& p) {
  // Columns from which uncut chains keep HBM busy, the lanes of cut ones (16381 x 1024
  // float32: 57 us with 18432 lanes, 61 with 13500 or 36864; 3 x 1000 x 515 float64
  // backward: 25 us with 13500 lanes, 29 with 18432).
  constexpr int64_t kEnough = 8192, kLanes = sizeof(T) == 4 ? 18432 : 13500;
  constexpr int V = 16 / (int)sizeof(T);
  p.wide = p.inner % V == 0 && (((uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.h | (uintptr_t)p.dh) & 15) == 0;
  // 16 x 1024 x 4096 float32: 133 us as streams, 157 directly; 32 x 512 x 4096: 153
  // and 132; 30 x 500 x 4001 sigmoid (copies of one value): 218 and 131; 16 x 500 x
  // 4096 float64 sigmoid: 174 and 138.
  const int64_t many = sizeof(T) == 4 && p.wide ? 98304 : 49152;
  if (p.length <= 2 * kRows || p.columns >= many) {
    const int64_t blocks = ceil_div(p.columns, (int64_t)kThreads);
    if (blocks > INT32_MAX) PB_FAIL(PB_ERR_UNSUPPORTED, "recurrence over more than 2^39 columns");
    PB_CHECK(kt_begin(d));
    recurrence_columns_kernel<T, I, GATE, BWD><<<(unsigned)blocks, kThreads, 0, d->stream>>>(p);
    PB_LAUNCHED(d);
    return kt_end(d);
  }
  p.by_columns = make_fastdiv(p.columns);
  int64_t segments = p.columns >= kEnough ? 1 : ceil_div(kLanes, p.columns);
  const int64_t most = ceil_div(p.length, (int64_t)4 * kRows);
  if (segments > most) segments = most;
  p.steps = ceil_div(p.length, segments);
  p.segments = ceil_div(p.length, p.steps);
  if (p.segments > 1) {
    void* ws;
    const size_t cells = (size_t)p.segments * p.columns;
    // Lanes that take their start from `state` must not meet the one that writes
    // `final` over it: then the starts are formed first, too.
    const bool starts = p.segments > kInlineMaps || (p.last && p.last == p.start);
    PB_CHECK(scratch(d, cells * (sizeof(double2) + (starts ? sizeof(double) : 0)), &ws));
    p.maps = static_cast<double2*>(ws);
    p.starts = starts ? reinterpret_cast<double*>(p.maps + cells) : nullptr;
  }
  PB_CHECK(kt_begin(d));
  if (p.segments > 1) {
    PB_CHECK((launch_stream<T, I, GATE, BWD, true>(d, p)));
    if (p.starts) {
      recurrence_starts_kernel<T><<<(unsigned)ceil_div(p.columns, (int64_t)(kThreads / 32)), kThreads, 0, d->stream>>>(p);
      PB_LAUNCHED(d);
    }
  }
  PB_CHECK((launch_stream<T, I, GATE, BWD, false>(d, p)));
  return kt_end(d);
}

template <typename T, bool BWD>
int launch_gate(Device* d, int gate, ScanArgs<T> p, size_t bytes) {
  const bool narrow = bytes < (size_t(1) << 32);
  if (gate == PB_GATE_SIGMOID)
    return narrow ? launch<T, uint32_t, PB_GATE_SIGMOID, BWD>(d, p) : launch<T, int64_t, PB_GATE_SIGMOID, BWD>(d, p);
  return narrow ? launch<T, uint32_t, PB_GATE_LINEAR, BWD>(d, p) : launch<T, int64_t, PB_GATE_LINEAR, BWD>(d, p);
}

// Checks common to both directions; the array's bytes and those of a state.
int check_view(pb_ctx* ctx, int dtype, int gate, int64_t outer, int64_t length, int64_t inner, size_t* bytes,
               size_t* state_bytes) {
  if (!ctx) PB_FAIL(PB_ERR_INVALID, "null context");
  if (dtype != PB_F32 && dtype != PB_F64) PB_FAIL(PB_ERR_INVALID, "recurrence takes float32 or float64");
  if (gate != PB_GATE_LINEAR && gate != PB_GATE_SIGMOID) PB_FAIL(PB_ERR_INVALID, "unknown gate %d", gate);
  if (outer < 0 || length < 0 || inner < 0) PB_FAIL(PB_ERR_INVALID, "negative extent");
  const size_t item = dtype == PB_F32 ? 4 : 8;
  const int64_t all[3] = {outer, length, inner}, ends[2] = {outer, inner};
  if (!array_bytes(ends, 2, item, state_bytes)) PB_FAIL(PB_ERR_INVALID, "extents too large");
  if (!*state_bytes) {
    *bytes = 0;
    return PB_OK;
  }
  if (!array_bytes(all, 3, item, bytes)) PB_FAIL(PB_ERR_INVALID, "extents too large");
  return PB_OK;
}

template <typename T, bool BWD>
ScanArgs<T> make_args(int64_t outer, int64_t length, int64_t inner, const void* a, const void* b, const void* h,
                      const void* dh, const void* start, const void* state, void* out0, void* out1, void* last) {
  ScanArgs<T> p = {};
  p.a = static_cast<const T*>(a);
  p.b = static_cast<const T*>(b);
  p.h = static_cast<const T*>(h);
  p.dh = static_cast<const T*>(dh);
  p.start = static_cast<const T*>(start);
  p.state = static_cast<const T*>(state);
  p.out0 = static_cast<T*>(out0);
  p.out1 = static_cast<T*>(out1);
  p.last = static_cast<T*>(last);
  p.length = length;
  p.inner = inner;
  p.by_inner = make_fastdiv(inner);
  p.columns = outer * inner;
  return p;
}

}  // namespace
}  // namespace pb

using namespace pb;

extern "C" {

int pb_recurrence(pb_ctx* ctx, int dev, int dtype, int gate, int64_t outer, int64_t length, int64_t inner,
                  const void* a, const void* b, const void* state, void* h, void* final) {
  size_t bytes, ends;
  PB_CHECK(check_view(ctx, dtype, gate, outer, length, inner, &bytes, &ends));
  if (!ends) return PB_OK;
  if (bytes && (!a || !b || !h)) PB_FAIL(PB_ERR_INVALID, "null operand");
  const Span in[] = {{a, bytes}, {b, bytes}, {state == final ? nullptr : state, ends}};
  const Span out[] = {{h, bytes}, {final, ends}};
  PB_CHECK(check_operands(out, 2, in, 3, dtype == PB_F32 ? 4 : 8));
  std::lock_guard<std::recursive_mutex> g(ctx->mu);
  Device* d;
  PB_CHECK(enter(ctx, dev, &d));
  if (dtype == PB_F32)
    return launch_gate<float, false>(d, gate, make_args<float, false>(outer, length, inner, a, b, nullptr, nullptr,
                                                                      state, nullptr, h, nullptr, final), bytes);
  return launch_gate<double, false>(d, gate, make_args<double, false>(outer, length, inner, a, b, nullptr, nullptr,
                                                                      state, nullptr, h, nullptr, final), bytes);
}

int pb_recurrence_backward(pb_ctx* ctx, int dev, int dtype, int gate, int64_t outer, int64_t length, int64_t inner,
                           const void* a, const void* b, const void* h, const void* dh, const void* state,
                           const void* dfinal, void* da, void* db, void* dstate) {
  size_t bytes, ends;
  PB_CHECK(check_view(ctx, dtype, gate, outer, length, inner, &bytes, &ends));
  if (!ends) return PB_OK;
  if (bytes && (!a || !h || !dh || !da || !db)) PB_FAIL(PB_ERR_INVALID, "null operand");
  if (bytes && gate == PB_GATE_SIGMOID && !b) PB_FAIL(PB_ERR_INVALID, "the sigmoid gate's gradients need b");
  const Span in[] = {{a, bytes}, {b, bytes}, {h, bytes}, {dh, bytes}, {state, ends}, {dfinal, ends}};
  const Span out[] = {{da, bytes}, {db, bytes}, {dstate, ends}};
  PB_CHECK(check_operands(out, 3, in, 6, dtype == PB_F32 ? 4 : 8));
  std::lock_guard<std::recursive_mutex> g(ctx->mu);
  Device* d;
  PB_CHECK(enter(ctx, dev, &d));
  if (dtype == PB_F32)
    return launch_gate<float, true>(d, gate, make_args<float, true>(outer, length, inner, a, b, h, dh, dfinal, state,
                                                                    da, db, dstate), bytes);
  return launch_gate<double, true>(d, gate, make_args<double, true>(outer, length, inner, a, b, h, dh, dfinal, state,
                                                                    da, db, dstate), bytes);
}

}  // extern "C"
