// Device code shared by the operators that read rows of logits (logits.cu): element access, the
// running maximum and sum of a softmax, and their join across threads.
//
// A row x[0..vocab) of logits at temperature t has z = x / t. Every kernel keeps, for the part of
// the row that it has seen, m = max x and s = sum exp((x - m) / t); two parts join into
// M = max(m1, m2), S = s1 exp((m1 - M) / t) + s2 exp((m2 - M) / t), so a row can be cut anywhere.
// The difference x - m is formed before the product with 1 / t: a row whose logits all have the
// type's lowest value then has differences of 0 and is uniform, where a product taken first would
// overflow.
//
// Sums are float (double for float64 logits): a row's sum is a tree of at most a few hundred
// sequential additions per thread, its rounding error about 1e-6 at worst and 1e-7 as a rule.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tiso {

template <typename T>
struct AccOf {
  using type = float;
};
template <>
struct AccOf<double> {
  using type = double;
};

__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }

template <typename T>
__device__ __forceinline__ T from_acc(typename AccOf<T>::type v);
template <>
__device__ __forceinline__ __half from_acc<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float from_acc<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ double from_acc<double>(double v) {
  return v;
}

template <typename A>
__device__ __forceinline__ A lowest();
template <>
__device__ __forceinline__ float lowest<float>() {
  return __int_as_float(static_cast<int>(0xff800000u));
}
template <>
__device__ __forceinline__ double lowest<double>() {
  return __longlong_as_double(static_cast<long long>(0xfff0000000000000ULL));
}
__device__ __forceinline__ float nan_of(float) { return __int_as_float(0x7fc00000); }
__device__ __forceinline__ double nan_of(double) {
  return __longlong_as_double(0x7ff8000000000000LL);
}

// exp((x - m) / t): `k` is log2(e) / t in float (one ex2, 2 units in the last place), 1 / t in
// double.
__device__ __forceinline__ float scaled_exp(float d, float k) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * k));
  return r;
}
__device__ __forceinline__ double scaled_exp(double d, double k) { return exp(d * k); }

// max(a, b) with a NaN ignored: the NaN reaches the sum through its own exponential.
__device__ __forceinline__ float max_acc(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double max_acc(double a, double b) { return fmax(a, b); }

// The point that exponentials are taken from: the maximum, or 0 where nothing but -infinity has
// been seen (-infinity minus itself is NaN; every exponential is then 0).
template <typename A>
__device__ __forceinline__ A base_of(A m) {
  return m == lowest<A>() ? A(0) : m;
}

template <typename A>
struct Part {
  A m, s;
};

template <typename A>
__device__ __forceinline__ Part<A> join(const Part<A>& a, const Part<A>& b, A k) {
  const A m = max_acc(a.m, b.m);
  const A base = base_of(m);
  // a part that holds the maximum keeps its sum as it is (its exponent is exactly 0)
  return {m, a.s * scaled_exp(a.m == m ? A(0) : a.m - base, k) +
                 b.s * scaled_exp(b.m == m ? A(0) : b.m - base, k)};
}

template <typename A>
__device__ __forceinline__ Part<A> join_warp(Part<A> p, A k) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const Part<A> q{__shfl_xor_sync(0xffffffffu, p.m, d), __shfl_xor_sync(0xffffffffu, p.s, d)};
    p = join(p, q, k);
  }
  return p;
}

}  // namespace tiso
