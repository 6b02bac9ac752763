// Gated linear recurrence h_t = alpha_t h_{t-1} + u_t along an axis, and its
// gradients (HBM-bound: forward 3 values moved per element, backward 5 or 6).
//
// The backward pass is the same recurrence run from the last step to the
// first, g_t = alpha_{t+1} g_{t+1} + dh_t, so the same kernels serve both: step s
// of the chain is t = s forward and t = length - 1 - s backward.
//
// A column is one (outer, inner) pair; neighbouring columns are neighbours in
// memory, so lanes run over columns and a warp's access is a row segment.
//
// Many columns or few steps: a thread per column walks the chain.  Few columns
// and many steps: the chain is cut.  n steps map x to P x + H, with P the product
// of their coefficients and H their result from 0; both are known without the
// value x before them, and two such maps compose to one.  A thread takes
// L steps of a column in registers, reduces them to (P, H), and the block
// composes its threads' maps; the block's own map goes to memory for the
// blocks behind it, which compose the maps of the chunks before them.  With the
// true value before its steps each thread then runs them again from registers:
// every input is read once.
//
// Every composition has a fixed order (chunks in groups of kGroup: the value at
// the end of the group before, then the chunks of the own group one by one), so
// the result does not depend on timing.  P and the composed values are float64:
// a product of thousands of gates neither over- nor underflows where the
// recurrence itself does not.
#include <type_traits>

#include "pb_layers.cuh"

namespace pb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kGroup = 16;  // chunks per group

template <typename T>
struct ScanArgs {
  const T *a, *b, *h, *dh;   // h, dh: backward only
  const T* start;            // forward: state; backward: dfinal; may be null
  const T* state;            // backward: h[-1]; may be null
  T* out0;                   // forward: h; backward: da
  T* out1;                   // backward: db
  T* last;                   // forward: final; backward: dstate; may be null
  int64_t length, inner, columns;
  // The cut chain (recurrence_chunks_kernel).
  int lanes_log2;            // lanes of a warp along columns
  unsigned tiles, chunks;    // column tiles, chunks along the chain
  double2* maps;             // [chunk][column]: (P, H)
  double* ends;              // [group][column]: the value at a group's end
  unsigned* words;           // ticket, finished blocks, epoch, -, then a flag per (tile, chunk) and per (tile, group)
  int* err;
};

__device__ __forceinline__ int64_t column_base(int64_t col, int64_t length, int64_t inner) {
  const int64_t o = col / inner;
  return o * length * inner + (col - o * inner);
}

// L consecutive chain steps of one column in registers.  Steps past the end
// are the identity.
template <typename T, int GATE, bool BWD, int L>
struct Steps;

template <typename T, int GATE, int L>
struct Steps<T, GATE, false, L> {
  T c[L], u[L];

  __device__ __forceinline__ void load(const ScanArgs<T>& p, int64_t base, int64_t, int64_t s0) {
    const int left = (int)max((int64_t)0, min((int64_t)L, p.length - s0));
    const T* a = p.a + base + s0 * p.inner;
    const T* b = p.b + base + s0 * p.inner;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      c[i] = T(1);
      u[i] = T(0);
      if (i < left) {
        c[i] = __ldg(a);
        u[i] = __ldg(b);
      }
      a += p.inner;
      b += p.inner;
    }
    if constexpr (GATE == PB_GATE_SIGMOID) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        T s, rest;
        sigmoid_pair(c[i], &s, &rest);
        c[i] = i < left ? s : T(1);
        u[i] *= rest;
      }
    }
  }
  __device__ __forceinline__ T coefficient(int i) const { return c[i]; }
  __device__ __forceinline__ T input(int i) const { return u[i]; }

  // The outputs of these steps from the value `x` before the first of them;
  // returns the value after the last.
  __device__ __forceinline__ T run(const ScanArgs<T>& p, int64_t base, int64_t col, int64_t s0, T x) const {
    const int64_t left = p.length - s0;
    T* h = p.out0 + base + s0 * p.inner;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      x = fma(c[i], x, u[i]);
      if (i < left) *h = x;
      h += p.inner;
    }
    if (p.last && left > 0 && left <= L) p.last[col] = x;
    return x;
  }
};

// Backward: step i of the chain is t = t0 - i.  Its own gate gives the outputs
// and is the coefficient of step i + 1; the first step's coefficient is the
// gate at t0 + 1, or 1 at the end of the sequence (dfinal as it is).
template <typename T, int GATE, int L>
struct Steps<T, GATE, true, L> {
  T first, alpha[L], g[L], before[L];
  T rest[GATE == PB_GATE_SIGMOID ? L : 1], put[GATE == PB_GATE_SIGMOID ? L : 1];

  __device__ __forceinline__ void load(const ScanArgs<T>& p, int64_t base, int64_t col, int64_t s0) {
    const int left = (int)max((int64_t)0, min((int64_t)L, p.length - s0));
    const int64_t t0 = p.length - 1 - s0;
    int64_t e = base + t0 * p.inner;
    first = T(1);
    if (left > 0 && s0 > 0) first = __ldg(p.a + e + p.inner);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      alpha[i] = T(1);
      g[i] = before[i] = T(0);
      if (i < left) {
        alpha[i] = __ldg(p.a + e);
        g[i] = __ldg(p.dh + e);
        if (t0 > i) before[i] = __ldg(p.h + e - p.inner);
        else if (p.state) before[i] = __ldg(p.state + col);
        if constexpr (GATE == PB_GATE_SIGMOID) put[i] = __ldg(p.b + e);
      }
      e -= p.inner;
    }
    if constexpr (GATE == PB_GATE_SIGMOID) {
      T unused;
      if (s0 > 0) sigmoid_pair(first, &first, &unused);
#pragma unroll
      for (int i = 0; i < L; ++i) {
        T s;
        sigmoid_pair(alpha[i], &s, &rest[i]);
        alpha[i] = i < left ? s : T(1);
      }
    }
  }
  __device__ __forceinline__ T coefficient(int i) const { return i ? alpha[i - 1] : first; }
  __device__ __forceinline__ T input(int i) const { return g[i]; }

  __device__ __forceinline__ T run(const ScanArgs<T>& p, int64_t base, int64_t col, int64_t s0, T x) const {
    const int64_t left = p.length - s0;
    int64_t e = base + (left - 1) * p.inner;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      x = fma(coefficient(i), x, g[i]);
      if (i < left) {
        if constexpr (GATE == PB_GATE_SIGMOID) {
          p.out1[e] = x * rest[i];
          p.out0[e] = x * (before[i] - put[i]) * (alpha[i] * rest[i]);
        } else {
          p.out1[e] = x;
          p.out0[e] = x * before[i];
        }
        if (p.last && left == i + 1) p.last[col] = alpha[i] * x;
      }
      e -= p.inner;
    }
    return x;
  }
};

// A thread per column, the whole chain in order.
template <typename T, int GATE, bool BWD, int L>
__global__ void __launch_bounds__(kThreads) recurrence_columns_kernel(const ScanArgs<T> p) {
  const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (col >= p.columns) return;
  const int64_t base = column_base(col, p.length, p.inner);
  T x = p.start ? p.start[col] : T(0);
  if (p.length == 0) {
    if (p.last) p.last[col] = x;
    return;
  }
  for (int64_t s0 = 0; s0 < p.length; s0 += L) {
    Steps<T, GATE, BWD, L> st;
    st.load(p, base, col, s0);
    x = st.run(p, base, col, s0, x);
  }
}

// x -> P x + H.  0 maps to H even where P has overflowed.
__device__ __forceinline__ double apply(const double2& map, double x) {
  return x == 0.0 ? map.y : fma(map.x, x, map.y);
}
// The map of `a` followed by `b`.
__device__ __forceinline__ double2 compose(const double2& a, const double2& b) {
  return make_double2(a.x * b.x, apply(b, a.y));
}

// One block per (column tile, chunk).  A warp covers 2^lanes_log2 columns and
// 32 >> lanes_log2 consecutive pieces of L steps, the block kWarps times that.
// Blocks take their chunk from a counter, chunk by chunk over the column
// tiles, so every chunk that a block waits for is already running or done.
template <typename T, int GATE, bool BWD, int L>
__global__ void __launch_bounds__(kThreads, BWD ? (sizeof(T) == 4 ? 3 : 2) : 4) recurrence_chunks_kernel(const ScanArgs<T> p) {
  __shared__ double2 warp_map[kWarps][32];
  __shared__ double2 earlier[kGroup - 1][32];
  __shared__ double carry[32];
  __shared__ unsigned ticket_s, epoch_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    ticket_s = atomicAdd(p.words, 1u);
    epoch_s = load_acquire(p.words + 2) + 1;
  }
  __syncthreads();
  const unsigned chunk = ticket_s / p.tiles, tile = ticket_s % p.tiles, epoch = epoch_s;
  const int width = 1 << p.lanes_log2, pieces = 32 >> p.lanes_log2;
  const int lc = lane & (width - 1), piece = lane >> p.lanes_log2;
  const int64_t col = (int64_t)tile * width + lc;
  const bool on = col < p.columns;
  const int64_t base = on ? column_base(col, p.length, p.inner) : 0;
  const int64_t s0 = (int64_t)chunk * (kWarps * L) * pieces + (int64_t)(warp * pieces + piece) * L;
  Steps<T, GATE, BWD, L> st;
  st.load(p, base, on ? col : 0, on ? s0 : p.length);

  // This thread's map, and the composition of the pieces before it in the warp.
  double2 map;
  {
    double P = (double)st.coefficient(0);
    T H = fma(st.coefficient(0), T(0), st.input(0));
#pragma unroll
    for (int i = 1; i < L; ++i) {
      P *= (double)st.coefficient(i);
      H = fma(st.coefficient(i), H, st.input(i));
    }
    map = make_double2(P, (double)H);
  }
  double2 before = make_double2(1.0, 0.0);
  for (int k = 1; k < pieces; k <<= 1) {
    // Inclusive scan over the pieces, each composition in a fixed order.
    double2 prev;
    prev.x = __shfl_up_sync(0xffffffffu, map.x, k * width);
    prev.y = __shfl_up_sync(0xffffffffu, map.y, k * width);
    if (piece >= k) map = compose(prev, map);
  }
  if (pieces > 1) {
    double2 prev;
    prev.x = __shfl_up_sync(0xffffffffu, map.x, width);
    prev.y = __shfl_up_sync(0xffffffffu, map.y, width);
    if (piece > 0) before = prev;
  }
  if (piece == pieces - 1) warp_map[warp][lc] = map;
  __syncthreads();

  const unsigned groups = (p.chunks + kGroup - 1) / kGroup;
  unsigned* const chunk_flag = p.words + kFlagWords + (size_t)tile * p.chunks;
  unsigned* const group_flag = p.words + kFlagWords + (size_t)p.tiles * p.chunks + (size_t)tile * groups;
  const unsigned group = chunk / kGroup, place = chunk % kGroup;
  const bool behind = chunk + 1 < p.chunks;  // some chunk waits for this one
  const bool writer = piece == 0 && on;
  double2 all;  // the block's map (warp 0)
  if (warp == 0) {
    all = warp_map[0][lc];
    for (int w = 1; w < kWarps; ++w) all = compose(all, warp_map[w][lc]);
    if (behind && place != kGroup - 1) {
      if (writer) __stcg(p.maps + (int64_t)chunk * p.columns + col, all);
      __syncwarp();
      if (lane == 0) {
        __threadfence();
        store_release(chunk_flag + chunk, epoch);
      }
    }
  }
  // The maps of the group's chunks before this one, a warp for each (so that
  // their latencies overlap), and the value at the end of the group before.
  for (unsigned k = warp; k < place; k += kWarps) {
    if (lane == 0) wait_flag(chunk_flag + group * kGroup + k, epoch, p.err);
    __syncwarp();
    if (writer) earlier[k][lc] = __ldcg(p.maps + (int64_t)(group * kGroup + k) * p.columns + col);
  }
  if (warp == kWarps - 1) {
    double x = 0.0;
    if (group == 0) {
      if (p.start && on) x = (double)p.start[col];
    } else {
      if (lane == 0) wait_flag(group_flag + group - 1, epoch, p.err);
      __syncwarp();
      if (on) x = __ldcg(p.ends + (int64_t)(group - 1) * p.columns + col);
    }
    if (piece == 0) carry[lc] = x;
  }
  __syncthreads();
  double x = carry[lc];
  for (unsigned k = 0; k < place; ++k) x = apply(earlier[k][lc], x);
  if (warp == 0 && behind && place == kGroup - 1) {
    if (writer) __stcg(p.ends + (int64_t)group * p.columns + col, apply(all, x));
    __syncwarp();
    if (lane == 0) {
      __threadfence();
      store_release(group_flag + group, epoch);
    }
  }
  for (int w = 0; w < warp; ++w) x = apply(warp_map[w][lc], x);
  x = apply(before, x);
  if (on && s0 < p.length) st.run(p, base, col, s0, (T)x);

  if (threadIdx.x == 0) finish_words(p.words, epoch, p.tiles * p.chunks);
}

template <typename T, int GATE, bool BWD>
int launch(Device* d, ScanArgs<T>& p) {
  // Steps per thread: what keeps the registers of one thread near 64.
  constexpr int L = BWD ? 8 : sizeof(T) == 4 ? 16 : 8;
  int lanes = 0;
  while (lanes < 5 && (int64_t(1) << lanes) < p.columns) ++lanes;
  const int64_t tiles = ceil_div(p.columns, int64_t(1) << lanes);
  const int64_t chunks = ceil_div(p.length, (int64_t)(kWarps * L) << (5 - lanes));
  const int64_t groups = ceil_div(chunks, (int64_t)kGroup);
  const bool cut = p.length > 2 * L && p.columns < (int64_t)d->sm_count * 1024 &&
                   tiles * (chunks + groups) < (int64_t(1) << 26);
  if (cut) {
    void* ws;
    const size_t maps = (size_t)chunks * p.columns, ends = (size_t)groups * p.columns;
    PB_CHECK(scratch(d, maps * sizeof(double2) + ends * sizeof(double), &ws));
    p.maps = static_cast<double2*>(ws);
    p.ends = reinterpret_cast<double*>(p.maps + maps);
    PB_CHECK(epoch_words(d, kFlagWords + (size_t)(tiles * (chunks + groups)), &p.words));
    p.lanes_log2 = lanes;
    p.tiles = (unsigned)tiles;
    p.chunks = (unsigned)chunks;
    p.err = d->err_dev;
    PB_CHECK(kt_begin(d));
    recurrence_chunks_kernel<T, GATE, BWD, L><<<(unsigned)(tiles * chunks), kThreads, 0, d->stream>>>(p);
    PB_LAUNCHED(d);
    return kt_end(d);
  }
  const int64_t blocks = ceil_div(p.columns, (int64_t)kThreads);
  if (blocks > INT32_MAX) PB_FAIL(PB_ERR_UNSUPPORTED, "recurrence over more than 2^39 columns");
  PB_CHECK(kt_begin(d));
  recurrence_columns_kernel<T, GATE, BWD, 8><<<(unsigned)blocks, kThreads, 0, d->stream>>>(p);
  PB_LAUNCHED(d);
  return kt_end(d);
}

template <typename T, bool BWD>
int launch_gate(Device* d, int gate, ScanArgs<T> p) {
  return gate == PB_GATE_SIGMOID ? launch<T, PB_GATE_SIGMOID, BWD>(d, p) : launch<T, PB_GATE_LINEAR, BWD>(d, p);
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
                                                                      state, nullptr, h, nullptr, final));
  return launch_gate<double, false>(d, gate, make_args<double, false>(outer, length, inner, a, b, nullptr, nullptr,
                                                                      state, nullptr, h, nullptr, final));
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
                                                                    da, db, dstate));
  return launch_gate<double, true>(d, gate, make_args<double, true>(outer, length, inner, a, b, h, dh, dfinal, state,
                                                                    da, db, dstate));
}

}  // extern "C"
