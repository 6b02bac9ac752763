// Gated linear recurrence h_t = alpha_t h_{t-1} + u_t along an axis, and its
// gradients (HBM-bound: forward 3 values moved per element, backward 5 or 6).
//
// The backward pass is the same recurrence run from the last step to the
// first, g_t = alpha_{t+1} g_{t+1} + dh_t, so one kernel serves both: step s of
// the chain is t = s forward and t = length - 1 - s backward.
//
// A column is one (outer, inner) pair; neighbouring columns are neighbours in
// memory, so lanes run over columns and a warp's access is a row segment.
#include <type_traits>

#include "pb_layers.cuh"

namespace pb {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct ScanArgs {
  const T *a, *b, *h, *dh;   // h, dh: backward only
  const T* start;            // forward: state; backward: dfinal; may be null
  const T* state;            // backward: h[-1]; may be null
  T* out0;                   // forward: h; backward: da
  T* out1;                   // backward: db
  T* last;                   // forward: final; backward: dstate; may be null
  int64_t length, inner, columns;
};

// L consecutive chain steps of one column in registers: their coefficients
// and inputs.  Steps past the end are the identity (1, 0).
template <typename T, int GATE, bool BWD, int L>
struct Steps {
  T c[L], u[L];

  __device__ __forceinline__ void load(const ScanArgs<T>& p, int64_t base, int64_t s0) {
    const int64_t left = p.length - s0;
    if constexpr (!BWD) {
      const T* a = p.a + base + s0 * p.inner;
      const T* b = p.b + base + s0 * p.inner;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        c[i] = T(1);
        u[i] = T(0);
        if (i < left) {
          c[i] = __ldg(a + i * p.inner);
          u[i] = __ldg(b + i * p.inner);
        }
      }
      if constexpr (GATE == PB_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
          if (i < left) {
            T rest;
            sigmoid_pair(c[i], &c[i], &rest);
            u[i] *= rest;
          }
        }
      }
    } else {
      // The coefficient of chain step s is alpha[t + 1]; the first step's is 1
      // (it takes dfinal as it is).
      const int64_t t0 = p.length - 1 - s0;
      const T* a = p.a + base + (t0 + 1) * p.inner;
      const T* g = p.dh + base + t0 * p.inner;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        c[i] = T(1);
        u[i] = T(0);
        if (i < left) {
          if (s0 + i > 0) c[i] = __ldg(a - i * p.inner);
          u[i] = __ldg(g - i * p.inner);
        }
      }
      if constexpr (GATE == PB_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
          if (i < left && s0 + i > 0) {
            T rest;
            sigmoid_pair(c[i], &c[i], &rest);
          }
        }
      }
    }
  }

  // The outputs of these steps from the value `x` before the first of them;
  // returns the value after the last.
  __device__ __forceinline__ T run(const ScanArgs<T>& p, int64_t base, int64_t col, int64_t s0, T x) const {
    const int64_t left = p.length - s0;
    if constexpr (!BWD) {
      T* h = p.out0 + base + s0 * p.inner;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        x = fma(c[i], x, u[i]);
        if (i < left) h[i * p.inner] = x;
      }
      if (p.last && left > 0 && left <= L) p.last[col] = x;
    } else {
      const int64_t t0 = p.length - 1 - s0;
      const int64_t at = base + t0 * p.inner;
#pragma unroll
      for (int i = 0; i < L; ++i) {
        x = fma(c[i], x, u[i]);
        if (i < left) {
          const int64_t e = at - i * p.inner;
          T before = T(0);
          if (t0 > i) before = __ldg(p.h + e - p.inner);
          else if (p.state) before = p.state[col];
          if constexpr (GATE == PB_GATE_SIGMOID) {
            T alpha, rest;
            sigmoid_pair(__ldg(p.a + e), &alpha, &rest);
            p.out1[e] = x * rest;
            p.out0[e] = x * (before - __ldg(p.b + e)) * (alpha * rest);
            if (t0 == i && p.last) p.last[col] = alpha * x;
          } else {
            p.out1[e] = x;
            p.out0[e] = x * before;
            if (t0 == i && p.last) p.last[col] = __ldg(p.a + e) * x;
          }
        }
      }
    }
    return x;
  }
};

// One thread per column, the whole chain in order.
template <typename T, int GATE, bool BWD, int L>
__global__ void __launch_bounds__(kThreads) recurrence_columns_kernel(const ScanArgs<T> p) {
  const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (col >= p.columns) return;
  const int64_t base = col / p.inner * p.length * p.inner + col % p.inner;
  T x = p.start ? p.start[col] : T(0);
  if (p.length == 0) {
    if (p.last) p.last[col] = x;
    return;
  }
  for (int64_t s0 = 0; s0 < p.length; s0 += L) {
    Steps<T, GATE, BWD, L> st;
    st.load(p, base, s0);
    x = st.run(p, base, col, s0, x);
  }
}

template <typename T, int GATE, bool BWD>
int launch(Device* d, const ScanArgs<T>& p) {
  constexpr int L = 8;
  const int64_t blocks = ceil_div(p.columns, (int64_t)kThreads);
  if (blocks > INT32_MAX) PB_FAIL(PB_ERR_UNSUPPORTED, "recurrence over more than 2^39 columns");
  PB_CHECK(kt_begin(d));
  recurrence_columns_kernel<T, GATE, BWD, L><<<(unsigned)blocks, kThreads, 0, d->stream>>>(p);
  PB_LAUNCHED(d);
  return kt_end(d);
}

template <typename T, bool BWD>
int launch_gate(Device* d, int gate, const ScanArgs<T>& p) {
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
