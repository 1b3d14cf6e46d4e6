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

#include <type_traits>

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
__device__ __forceinline__ double scaled_exp(double d, double k) { return exp(__dmul_rn(d, k)); }

// max(a, b) with a NaN ignored: the NaN reaches the sum through its own exponential.
__device__ __forceinline__ float max_acc(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double max_acc(double a, double b) { return fmax(a, b); }

// Products and sums that are not contracted into one operation.
__device__ __forceinline__ float mul_rn(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ double mul_rn(double a, double b) { return __dmul_rn(a, b); }
__device__ __forceinline__ float add_rn(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ double add_rn(double a, double b) { return __dadd_rn(a, b); }

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

// ---------------------------------------------------------------------------------------------
// A row in 16-byte vectors. Rows start anywhere (an odd vocabulary, a cut tensor), so a row is a
// body of whole vectors and at most 4 E - 1 single elements around it (E to a vector). The body is
// aligned for the row that is written, g; where the row read, x, is off that by `shift` elements,
// a vector of x is put together from the two aligned ones that hold it. No load leaves the row.

template <typename T>
struct RowView {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  T* g;
  int head, vectors, edges, shift;

  // `address`: the written row's; where none is written, what decides the cut
  __device__ __forceinline__ RowView(const T* x_, T* g_, uintptr_t address, int vocab)
      : x(x_), g(g_) {
    head = static_cast<int>((16 - (address & 15)) & 15) / static_cast<int>(sizeof(T));
    shift = static_cast<int>((reinterpret_cast<uintptr_t>(x_ + head) & 15) / sizeof(T));
    if (shift > head) head += E;
    head = min(head, vocab);
    // with a shift, vector v also reads the aligned vector after its own
    vectors = max(0, (vocab - head + shift) / E - (shift ? 1 : 0));
    edges = vocab - vectors * E;
  }

  // the e-th single element's index in the row
  __device__ __forceinline__ int edge(int e) const { return e < head ? e : vectors * E + e; }
  __device__ __forceinline__ int element(int v) const { return head + v * E; }
};

template <int kBytes>
__device__ __forceinline__ void shift_words(uint32_t (&w)[8], bool on) {
  if constexpr (kBytes >= 4) {
#pragma unroll
    for (int i = 0; i + kBytes / 4 < 8; ++i) w[i] = on ? w[i + kBytes / 4] : w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i) w[i] = on ? __funnelshift_r(w[i], w[i + 1], 8 * kBytes) : w[i];
  }
}

__device__ __forceinline__ uint4 load_once(const void* p) {  // read once: keeps out of L1
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// kN vectors of the row read, v, v + kStep, ...
template <int kN, int kStep, typename T>
__device__ __forceinline__ void load_vectors(const RowView<T>& r, int v, uint4 (&q)[kN]) {
  const uint4* at = reinterpret_cast<const uint4*>(r.x + r.head - r.shift) + v;
  if (r.shift == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) q[i] = load_once(at + i * kStep);
    return;
  }
  const int bytes = r.shift * static_cast<int>(sizeof(T));
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const uint4 a = __ldg(at + i * kStep), b = __ldg(at + i * kStep + 1);
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    shift_words<8>(w, bytes & 8);
    if constexpr (sizeof(T) <= 4) shift_words<4>(w, bytes & 4);
    if constexpr (sizeof(T) <= 2) shift_words<2>(w, bytes & 2);
    q[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T>
__device__ __forceinline__ uint4 load_vector(const RowView<T>& r, int v) {
  uint4 q[1];
  load_vectors<1, 1>(r, v, q);
  return q[0];
}

// A vector of -infinity: what a thread holds where the row has no vector for it.
template <typename T>
__device__ __forceinline__ uint4 no_vector() {
  if constexpr (sizeof(T) == 8) {
    return make_uint4(0, 0xfff00000u, 0, 0xfff00000u);
  } else {
    const uint32_t w = std::is_same_v<T, __half>          ? 0xfc00fc00u
                       : std::is_same_v<T, __nv_bfloat16> ? 0xff80ff80u
                                                          : 0xff800000u;
    return make_uint4(w, w, w, w);
  }
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& q, typename AccOf<T>::type (&x)[16 / sizeof(T)]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else if constexpr (std::is_same_v<T, __half>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  } else {
    x[0] = __hiloint2double(static_cast<int>(w[1]), static_cast<int>(w[0]));
    x[1] = __hiloint2double(static_cast<int>(w[3]), static_cast<int>(w[2]));
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const typename AccOf<T>::type (&x)[16 / sizeof(T)]) {
  uint32_t w[4];
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else if constexpr (std::is_same_v<T, __half>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[2 * i] = static_cast<uint32_t>(__double2loint(x[i]));
      w[2 * i + 1] = static_cast<uint32_t>(__double2hiint(x[i]));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest element of kN vectors (a NaN is ignored; it reaches the sum).
template <typename T, int kN>
__device__ __forceinline__ typename AccOf<T>::type vector_max(const uint4 (&q)[kN]) {
  using A = typename AccOf<T>::type;
  if constexpr (sizeof(T) == 2) {
    using H2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const uint4 none = no_vector<T>();
    H2 m = *reinterpret_cast<const H2*>(&none.x);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const H2* h = reinterpret_cast<const H2*>(&q[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) m = __hmax2(m, h[j]);
    }
    return fmaxf(to_acc(m.x), to_acc(m.y));
  } else {
    A m = lowest<A>();
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      A x[16 / sizeof(T)];
      unpack<T>(q[i], x);
#pragma unroll
      for (int j = 0; j < static_cast<int>(16 / sizeof(T)); ++j) m = max_acc(m, x[j]);
    }
    return m;
  }
}

// Pairs of floats in one 64-bit register, for the instructions that take two at a time.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair_of(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float exp2_of(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp((x - base) / t) of a vector's elements, in place.
template <int kE>
__device__ __forceinline__ void exponentials(float (&x)[kE], float base, float k) {
  const Pair minus = pair_of(-base, -base), factor = pair_of(k, k);
#pragma unroll
  for (int j = 0; j < kE; j += 2) {
    float a, b;
    split(mul2(add2(pair_of(x[j], x[j + 1]), minus), factor), a, b);
    x[j] = exp2_of(a);
    x[j + 1] = exp2_of(b);
  }
}
template <int kE>
__device__ __forceinline__ void exponentials(double (&x)[kE], double base, double k) {
#pragma unroll
  for (int j = 0; j < kE; ++j) x[j] = exp(mul_rn(x[j] - base, k));
}

// The elements times a number, in place.
template <int kE>
__device__ __forceinline__ void scale_by(float (&x)[kE], float c) {
  const Pair factor = pair_of(c, c);
#pragma unroll
  for (int j = 0; j < kE; j += 2) split(mul2(pair_of(x[j], x[j + 1]), factor), x[j], x[j + 1]);
}
template <int kE>
__device__ __forceinline__ void scale_by(double (&x)[kE], double c) {
#pragma unroll
  for (int j = 0; j < kE; ++j) x[j] = mul_rn(x[j], c);
}

// The sum of a vector's elements.
template <int kE>
__device__ __forceinline__ float total(const float (&x)[kE]) {
  Pair s = pair_of(x[0], x[1]);
#pragma unroll
  for (int j = 2; j < kE; j += 2) s = add2(s, pair_of(x[j], x[j + 1]));
  float a, b;
  split(s, a, b);
  return a + b;
}
template <int kE>
__device__ __forceinline__ double total(const double (&x)[kE]) {
  return x[0] + x[1];
}

__device__ __forceinline__ void store_once(void* p, const uint4& v) {
  __stcs(reinterpret_cast<uint4*>(p), v);
}

// Copies of 16 bytes to shared memory that a thread starts, closes a group of, and waits for until
// no more than kOpen groups are open.
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from)
               : "memory");
}
__device__ __forceinline__ void close_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kOpen>
__device__ __forceinline__ void wait_groups() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kOpen) : "memory");
}

// The parts of kLanes neighbouring lanes joined: the same bits in each of them (sums pair by pair
// do not depend on the order of the two).
template <int kLanes>
__device__ __forceinline__ float max_of_lanes(float m) {
  if constexpr (kLanes == 32) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(m));
    return r;
  } else {
#pragma unroll
    for (int d = kLanes / 2; d; d >>= 1) m = max_acc(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
  }
}
template <int kLanes>
__device__ __forceinline__ double max_of_lanes(double m) {
#pragma unroll
  for (int d = kLanes / 2; d; d >>= 1) m = max_acc(m, __shfl_xor_sync(0xffffffffu, m, d));
  return m;
}

template <int kLanes, typename A>
__device__ __forceinline__ Part<A> join_lanes(const Part<A>& p, A k) {
  const A m = max_of_lanes<kLanes>(p.m);
  // a part that holds the maximum keeps its sum as it is
  A s = p.m == m ? p.s : mul_rn(p.s, scaled_exp(p.m - base_of(m), k));
#pragma unroll
  for (int d = kLanes / 2; d; d >>= 1) s = add_rn(s, __shfl_xor_sync(0xffffffffu, s, d));
  return {m, s};
}

}  // namespace tiso
