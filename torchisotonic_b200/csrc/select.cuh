// Choosing the k largest of n numbers exactly, equal ones by their place (the lowest first), by the
// threads of a warp or of a CTA.
//
// Numbers are compared as unsigned integers in their order (ordered()). The k-th largest is found
// digit by digit from the top (a radix selection): a histogram of 256 bins over the numbers that
// agree with the digits found so far, and the bin in which the k-th lies. It ends as soon as a bin
// is wanted whole; where the k-th has equals beyond it, the digits of the places decide. No data
// makes it take more than sizeof(key) + 4 rounds.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace tiso {

template <int kThreads>
struct Team {
  int tid;
  __device__ __forceinline__ void sync() const {
    if constexpr (kThreads == 32) {
      __syncwarp();
    } else {
      __syncthreads();
    }
  }
};

// Larger numbers have larger keys; -0 has 0's and NaN that of -infinity.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = x == x ? __float_as_uint(x + 0.0f) : 0xff800000u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t b = x == x ? static_cast<uint64_t>(__double_as_longlong(x + 0.0))
                            : 0xfff0000000000000ULL;
  return b >> 63 ? ~b : b | 0x8000000000000000ULL;
}

template <typename A>
using KeyOf = std::conditional_t<sizeof(A) == 4, uint32_t, uint64_t>;

// What is chosen: keys above `key`, and those equal to it whose place is at most `place`.
template <typename A>
struct Cut {
  KeyOf<A> key;
  uint32_t place;
  __device__ __forceinline__ bool takes(KeyOf<A> k, uint32_t p) const {
    return k > key || (k == key && p <= place);
  }
};

constexpr int kBins = 256, kHistogram = kBins + 4;  // words of shared memory for a selection

// The digit in which the need-th largest of the digits lies (-1: not one of them), how many lie
// above it, and how many in it.
struct Digit {
  int bin, above, inside;
};

template <int kThreads, typename F>
__device__ __forceinline__ Digit find_digit(const Team<kThreads>& team, int n, int need,
                                            const F& digit, unsigned* histogram) {
  for (int i = team.tid; i < kBins; i += kThreads) histogram[i] = 0;
  team.sync();
  for (int i = team.tid; i < n; i += kThreads) {
    const int d = digit(i);
    if (d >= 0) atomicAdd(histogram + d, 1u);
  }
  team.sync();
  if (team.tid < 32) {
    constexpr int kEach = kBins / 32;
    const int top = kBins - 1 - kEach * team.tid;  // this lane's bins, from the largest down
    int own = 0;
    for (int j = 0; j < kEach; ++j) own += static_cast<int>(histogram[top - j]);
    int upto = own;
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, d);
      if (team.tid >= d) upto += other;
    }
    int above = upto - own;
    if (above < need && need <= upto) {
      int j = 0;
      while (above + static_cast<int>(histogram[top - j]) < need)
        above += static_cast<int>(histogram[top - j++]);
      histogram[kBins] = static_cast<unsigned>(top - j);
      histogram[kBins + 1] = static_cast<unsigned>(above);
      histogram[kBins + 2] = histogram[top - j];
    }
  }
  team.sync();
  const Digit r{static_cast<int>(histogram[kBins]), static_cast<int>(histogram[kBins + 1]),
                static_cast<int>(histogram[kBins + 2])};
  team.sync();  // the bins are zeroed next
  return r;
}

// The cut that takes k of n > k numbers: key(i), and place(i), different for each.
template <int kThreads, typename A, typename F, typename G>
__device__ __forceinline__ Cut<A> find_cut(const Team<kThreads>& team, int n, int k, const F& key,
                                           const G& place, unsigned* histogram) {
  using U = KeyOf<A>;
  U found = 0, mask = 0;
  int need = k;
  for (int shift = 8 * sizeof(U) - 8; shift >= 0; shift -= 8) {
    const Digit d = find_digit<kThreads>(
        team, n, need,
        [&](int i) {
          const U v = key(i);
          return (v & mask) == found ? static_cast<int>(v >> shift & 255) : -1;
        },
        histogram);
    found |= static_cast<U>(d.bin) << shift;
    mask |= static_cast<U>(255) << shift;
    need -= d.above;
    if (need == d.inside) return {found, 0xffffffffu};
  }
  // equal numbers: the first `need` places, by the digits of their complement
  uint32_t low = 0, low_mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    const Digit d = find_digit<kThreads>(
        team, n, need,
        [&](int i) {
          const uint32_t v = ~place(i);
          return key(i) == found && (v & low_mask) == low ? static_cast<int>(v >> shift & 255) : -1;
        },
        histogram);
    low |= static_cast<uint32_t>(d.bin) << shift;
    low_mask |= 255u << shift;
    need -= d.above;
    if (need == d.inside) break;
  }
  return {found, ~low};  // complements from `low` on
}

}  // namespace tiso
