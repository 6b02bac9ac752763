// Helpers shared by the layer kernels (recurrence, group norm, AdamW).
#pragma once

#include "pb_internal.cuh"

namespace pb {

template <typename T> struct Vec16;
template <> struct Vec16<float> { using type = float4; static constexpr int n = 4; };
template <> struct Vec16<double> { using type = double2; static constexpr int n = 2; };

// V values of T in registers, moved with one access when V * sizeof(T) is 16
// (the address then has to be 16-byte aligned) and value by value otherwise.
template <typename T, int V>
struct alignas(V * sizeof(T) == 16 ? 16 : sizeof(T)) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* __restrict__ p) {
  Pack<T, V> r;
  if constexpr (V * sizeof(T) == 16) {
    const typename Vec16<T>::type q = __ldg(reinterpret_cast<const typename Vec16<T>::type*>(p));
    __builtin_memcpy(&r, &q, 16);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = __ldg(p + i);
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r) {
  if constexpr (V * sizeof(T) == 16) {
    typename Vec16<T>::type q;
    __builtin_memcpy(&q, &r, 16);
    *reinterpret_cast<typename Vec16<T>::type*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = r.v[i];
  }
}

// 2^x and 1/x of the special-function unit: within 2 ulp and 1 ulp, results and
// operands below 2^-126 as zero.
__device__ __forceinline__ float exp2_unit(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float reciprocal_unit(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// s = 1 / (1 + e^-z) and rest = 1 - s, each to a few roundings of its own size:
// with e = e^-|z| <= 1 the two are 1/(1+e) and e/(1+e), so neither is the
// difference of two nearly equal numbers.
__device__ __forceinline__ void sigmoid_pair(float z, float* s, float* rest) {
  // e = 2^(t + r) with t = -|z| log2 e rounded and r what the rounding lost (log2 e
  // in two parts): 2^t (1 + r ln 2), r being below 2^-17.  From |z| = 126 on, e is
  // zero; the minimum keeps a NaN.
  constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596303e-8f, kLn2 = 0.693147182f;
  float a;
  asm("min.NaN.f32 %0, %1, 0f42FC0000;" : "=f"(a) : "f"(fabsf(z)));
  const float t = a * -kLog2e;
  const float r = fmaf(-a, kLog2eLow, fmaf(-a, kLog2e, -t));
  float e = exp2_unit(t);
  e = fmaf(e, r * kLn2, e);
  const float big = reciprocal_unit(1.0f + e), small = e * big;
  *s = z < 0.0f ? small : big;
  *rest = z < 0.0f ? big : small;
}
__device__ __forceinline__ void sigmoid_pair(double z, double* s, double* rest) {
  const double e = exp(-fabs(z)), big = 1.0 / (1.0 + e), small = e * big;
  *s = z < 0.0 ? small : big;
  *rest = z < 0.0 ? big : small;
}

// s alone, off by 8 + 1.3 |z| roundings of itself, for an activation: z s is then off by
// less than two roundings of 1 beyond its own, since z^2 e^z <= 0.54 for negative z.  Its
// slope takes 1 - s, off by roundings of 1, times s z.  Compensated as above, which is
// felt in the tail alone: 32768 x 2048 forward 108 us instead of 105, 4547 x 42 groups of 169
// 85 instead of 76, 4 x 65536 x 128 gradients 133 instead of 124.
__device__ __forceinline__ float sigmoid(float z) { return reciprocal_unit(1.0f + exp2_unit(z * -1.44269502f)); }
__device__ __forceinline__ double sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

// ---- flags between the blocks of one launch (words of epoch_words()) ----
//
// words[0] counts the work items handed out, words[1] the blocks that are done,
// words[2] is the number of launches so far; flags follow from kFlagWords on.
// An item waits only for flags of items with lower numbers, which are running or
// done when it gets its own, so every wait ends.
constexpr int kFlagWords = 4;
constexpr unsigned long long kFlagWaitNs = 4ull * 1000 * 1000 * 1000, kShortWaitNs = 1000 * 1000;

__device__ __forceinline__ unsigned load_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(unsigned* p, unsigned v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
// Wait until reached(): after kFlagWaitNs the error word and `failed` (the block's)
// are set and the kernel goes on to its end (with wrong values), its further waits
// being short.
template <typename F>
__device__ __forceinline__ void wait_until(F&& reached, volatile int* failed, int* err) {
  if (reached()) return;
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  const unsigned long long limit = *failed ? kShortWaitNs : kFlagWaitNs;
  while (!reached()) {
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > limit) {
      *failed = 1;
      atomicExch(err, KERR_WAIT_TIMEOUT);
      return;
    }
  }
}

// The last block to finish readies the words for the next launch: flags need no
// clearing, the next epoch's value is another.  One thread of each block, after
// the block's last use of the words.
__device__ __forceinline__ void finish_words(unsigned* words, unsigned epoch, unsigned blocks) {
  __threadfence();
  if (atomicAdd(words + 1, 1u) == blocks - 1) {
    words[0] = 0;
    words[1] = 0;
    words[2] = epoch;
  }
}

// ---- runs of memory on their way into shared memory ------------------------
//
// Bulk copies that report to an mbarrier.  Every wait is bounded, as above.
__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void barrier_init(uint64_t* bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(bar)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint64_t* bar, unsigned parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(shared_address(bar)), "r"(parity), "r"(20000)  // sleep for up to 20 us
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool barrier_wait(uint64_t* bar, unsigned parity, volatile int* failed, int* err) {
  bool done = false;
  wait_until([&] { return done = barrier_try(bar, parity); }, failed, err);
  return done;
}
// `bytes` (a multiple of 16) from global to shared memory, both 16-byte aligned.
__device__ __forceinline__ void bulk_copy(void* to, const void* from, unsigned bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared_address(to)),
      "l"(from), "r"(bytes), "r"(shared_address(bar))
      : "memory");
}

// Whether [p, p + pn) and [q, q + qn) share a byte (NULL shares none).
inline bool overlap(const void* p, size_t pn, const void* q, size_t qn) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && pn && qn && a < b + qn && b < a + pn;
}

struct Span {
  const void* p;
  size_t n;
};
// Refuses an output that overlaps another output or an input, and an operand
// that does not start on a whole element.
inline int check_operands(const Span* out, int nout, const Span* in, int nin, size_t item) {
  for (int i = 0; i < nout; ++i) {
    for (int j = i + 1; j < nout; ++j)
      if (overlap(out[i].p, out[i].n, out[j].p, out[j].n)) PB_FAIL(PB_ERR_INVALID, "two outputs overlap");
    for (int j = 0; j < nin; ++j)
      if (overlap(out[i].p, out[i].n, in[j].p, in[j].n)) PB_FAIL(PB_ERR_INVALID, "an output overlaps an input");
    if ((uintptr_t)out[i].p % item) PB_FAIL(PB_ERR_INVALID, "a pointer is not aligned to its type");
  }
  for (int j = 0; j < nin; ++j)
    if ((uintptr_t)in[j].p % item) PB_FAIL(PB_ERR_INVALID, "a pointer is not aligned to its type");
  return PB_OK;
}

// Product of extents of one array in bytes; false when it passes 2^62.
inline bool array_bytes(const int64_t* extents, int n, size_t item, size_t* bytes) {
  unsigned __int128 t = item;
  for (int i = 0; i < n; ++i) {
    t *= (uint64_t)extents[i];
    if (t > ((unsigned __int128)1 << 62)) return false;
  }
  *bytes = (size_t)t;
  return true;
}

}  // namespace pb
