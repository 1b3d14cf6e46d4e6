// Operators on rows of logits (include/tiso.h: tiso_logprobs*, tiso_policy*): the log-probability
// of one token per row and its gradient, and the clipped policy loss with its gradient.
//
// All are streams over the logits: an exponential and about four other instructions an element and
// pass, no contraction. Times below are of one B200 (copy bandwidth 6545 GB/s measured), bf16.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <mutex>
#include <set>
#include <string>
#include <utility>

#include "cta.cuh"
#include "entry.cuh"
#include "logits.cuh"

namespace tiso {
namespace {

namespace cg = cooperative_groups;

constexpr int kBatch = 4;       // vectors a thread loads before it uses the first
constexpr int kRowWarps = 8;    // rows to a CTA where a warp takes a row
constexpr int kMostRows = 1 << 28;
constexpr int kNoEdge = 1 << 30;

int logits_fail(cudaError_t e, const char* what) {
  return report_error(TISO_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// Rows of logits: row r starts at x + (r / inner) * outer_stride + (r % inner) * inner_stride.
struct Rows {
  const void* x;
  int64_t rows, inner, outer_stride, inner_stride;
  int vocab;
  const int64_t* targets;
  int64_t ignore;
};

template <typename T>
__device__ __forceinline__ const T* row_at(const Rows& a, int64_t r) {
  const T* x = static_cast<const T*>(a.x);
  if (r < a.inner) return x + r * a.inner_stride;  // one stride: no division
  return x + (r / a.inner) * a.outer_stride + (r % a.inner) * a.inner_stride;
}

// Who works on a row: a warp (kThreads 32; kRowWarps rows to a CTA), a CTA, or a cluster of CTAs
// (kThreads > 32; the row's index is the cluster's). A row's vectors are cut into tiles of kBatch
// vectors a thread; the CTAs of a cluster take tiles in turn.
template <int kThreads>
struct Place {
  int64_t row;
  int tid, cta, ctas;

  __device__ __forceinline__ Place() {
    if constexpr (kThreads == 32) {
      row = static_cast<int64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
      tid = threadIdx.x & 31;
      cta = 0;
      ctas = 1;
    } else {
      ctas = static_cast<int>(cg::this_cluster().num_blocks());
      row = blockIdx.x / ctas;
      cta = static_cast<int>(blockIdx.x % ctas);
      tid = threadIdx.x;
    }
  }
  __device__ __forceinline__ bool first() const { return tid == 0 && cta == 0; }
  // this thread's number for a row's single elements; none but the first CTA takes them
  __device__ __forceinline__ int edge() const { return cta == 0 ? tid : kNoEdge; }
};

// Adds vectors to what a thread has seen.
template <typename T, int kN, typename A>
__device__ __forceinline__ void add_vectors(Part<A>& p, const uint4 (&q)[kN], A k) {
  const A m = max_acc(p.m, vector_max<T>(q));
  const A base = base_of(m);
  p.s *= scaled_exp(p.m == m ? A(0) : p.m - base, k);
  p.m = m;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    A x[RowView<T>::E];
    unpack<T>(q[i], x);
    exponentials(x, base, k);
    p.s += total(x);
  }
}

// The part of a row that a thread sees: of a CTA's tiles (every ctas-th), those from vector `first`
// on, and one of the single elements.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ Part<A> thread_part(const RowView<T>& r, const Place<kThreads>& place,
                                               int first, A k) {
  constexpr int kTile = kBatch * kThreads;
  // loaded ahead of the vectors, used behind them
  const A edge = place.edge() < r.edges ? to_acc(r.x[r.edge(place.edge())]) : lowest<A>();
  Part<A> p{lowest<A>(), A(0)};
  for (int tile = first; tile < r.vectors; tile += place.ctas * kTile) {
    const int v = tile + place.tid;
    uint4 q[kBatch];
    if (tile + kTile <= r.vectors) {
      load_vectors<kBatch, kThreads>(r, v, q);
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        q[i] = v + i * kThreads < r.vectors ? load_vector(r, v + i * kThreads) : no_vector<T>();
    }
    add_vectors<T>(p, q, k);
  }
  const A m = max_acc(p.m, edge), base = base_of(m);
  p.s = (p.m == m ? p.s : p.s * scaled_exp(p.m - base, k)) + scaled_exp(edge - base, k);
  p.m = m;
  return p;
}

// The part of a row that a warp sees.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ Part<A> warp_part(const RowView<T>& r, const Place<kThreads>& place, A k) {
  return join_lanes<32>(thread_part(r, place, place.cta * kBatch * kThreads, k), k);
}

// The parts of all of a row's warps joined (a warp's lanes hold the same); every thread gets the
// result. Called once by a CTA (its shared memory is not used again), by all of its threads, after
// cluster_started.
template <int kThreads, typename A>
__device__ __forceinline__ Part<A> join_warps(Part<A> p, A k) {
  if constexpr (kThreads > 32) {
    constexpr int kWarps = kThreads / 32, kMostCtas = 8;
    __shared__ Part<A> of_warp[kWarps], of_cta[kMostCtas];
    const int lane = threadIdx.x & 31;
    if (lane == 0) of_warp[threadIdx.x >> 5] = p;
    __syncthreads();
    p = join_lanes<kWarps>(of_warp[lane % kWarps], k);
    auto cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks());
    if (ctas > 1) {
      wait_for_start();
      if (threadIdx.x < ctas)
        *cluster.map_shared_rank(&of_cta[cluster.block_rank()], threadIdx.x) = p;
      cluster.sync();
      p = {lowest<A>(), A(0)};
      if (lane % kMostCtas < ctas) p = of_cta[lane % kMostCtas];
      p = join_lanes<kMostCtas>(p, k);
    }
  }
  return p;
}

// log softmax(x / t) at the target from its logit. The steps after the sum are in double: in float,
// rounding x - m - log s near 10 would cost more than the whole sum did, and a policy's ratio is
// the exponential of a difference of two such numbers.
template <typename A>
__device__ __forceinline__ double logp_of(A x, const Part<A>& p, double inv_temp) {
  return (static_cast<double>(x) - static_cast<double>(base_of(p.m))) * inv_temp -
         log(static_cast<double>(p.s));
}

template <typename T, typename A>
__device__ __forceinline__ A target_logit(const T* x, int vocab, int64_t target) {
  return target < 0 || target >= vocab ? nan_of(A(0)) : to_acc(x[target]);
}

// What a row's gradient is made of: c / t (1[v = target] - softmax), the softmax from the row's
// base and sum, c already divided by t. A target out of range gives NaN throughout. Each product
// and sum is rounded on its own, so that every kernel that writes it writes the same bits.
template <typename A>
struct Slope {
  A base, scale, k;
  int target;
  double c;  // the target's own gradient, c (1 - p), is rounded once

  __device__ __forceinline__ Slope(A base_, A s, double c_, A k_, int64_t target_, int vocab)
      : base(base_), k(k_), c(c_) {
    const bool in = target_ >= 0 && target_ < vocab;
    target = in ? static_cast<int>(target_) : -1;
    scale = in ? -static_cast<A>(c_) / s : nan_of(A(0));
  }
  // (a coefficient that the type has no room for is infinite in its own direction)
  __device__ __forceinline__ A at_target(A d) const {
    return static_cast<A>(isinf(d) ? c : __dadd_rn(c, static_cast<double>(d)));
  }
  __device__ __forceinline__ A at(A x, int v) const {
    const A d = mul_rn(scaled_exp(x - base, k), scale);
    return v == target ? at_target(d) : d;
  }
};

// The gradient of a vector's elements as if none was the target.
template <typename T, typename A>
__device__ __forceinline__ uint4 slope_vector(const uint4& q, const Slope<A>& slope) {
  A x[RowView<T>::E];
  unpack<T>(q, x);
  exponentials(x, slope.base, slope.k);
  scale_by(x, slope.scale);
  return pack<T>(x);
}

// The target's gradient, where the tile of kTile vectors from `tile` on has it, by the thread that
// wrote its vector (vector v by thread v % kThreads).
template <int kThreads, int kTile, typename T, typename A>
__device__ __forceinline__ void write_target_of_tile(const RowView<T>& r, int tile, int tid,
                                                     const Slope<A>& slope) {
  const int v = (slope.target - r.head) / RowView<T>::E, in_tile = v - tile;
  if (slope.target >= r.head && in_tile >= 0 && in_tile < kTile && in_tile % kThreads == tid &&
      v < r.vectors)
    r.g[slope.target] = from_acc<T>(slope.at(to_acc(r.x[slope.target]), slope.target));
}

template <typename T, typename A>
__device__ __forceinline__ void write_edge(const RowView<T>& r, int edge, const Slope<A>& slope) {
  if (edge < r.edges) {
    const int v = r.edge(edge);
    r.g[v] = from_acc<T>(slope.at(to_acc(r.x[v]), v));
  }
}

// The gradient of one tile's vectors.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void write_tile(const RowView<T>& r, int tile, int tid,
                                           const Slope<A>& slope) {
  constexpr int kTile = kBatch * kThreads;
  const int v = tile + tid;
  uint4* to = reinterpret_cast<uint4*>(r.g + r.head) + v;
  if (tile + kTile <= r.vectors) {
    uint4 q[kBatch];
    load_vectors<kBatch, kThreads>(r, v, q);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) store_once(to + i * kThreads, slope_vector<T>(q[i], slope));
  } else {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (v + i * kThreads < r.vectors)
        store_once(to + i * kThreads, slope_vector<T>(load_vector(r, v + i * kThreads), slope));
  }
  write_target_of_tile<kThreads, kTile>(r, tile, tid, slope);
}

template <int kThreads, typename T>
__device__ __forceinline__ void zero_tile(const RowView<T>& r, int tile, int tid) {
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int v = tile + i * kThreads + tid;
    if (v < r.vectors) store_once(r.g + r.element(v), make_uint4(0, 0, 0, 0));
  }
}

template <typename T>
__device__ __forceinline__ void zero_edge(const RowView<T>& r, int edge) {
  if (edge < r.edges) r.g[r.edge(edge)] = from_acc<T>(typename AccOf<T>::type(0));
}

// A row that is left out (its target is the ignored index, or its weight is 0) is marked by a
// negative sum in stats: its gradient is zeros and its logits are not read.
constexpr int kLeftOut = -1;

template <typename A>
__device__ __forceinline__ void write_logp(int64_t r, A logit, const Part<A>& p, double inv_temp,
                                           A* logps, A* stats) {
  logps[r] = static_cast<A>(logp_of(logit, p, inv_temp));
  if (stats) {
    stats[2 * r] = base_of(p.m);
    stats[2 * r + 1] = p.s;
  }
}

template <typename A>
__device__ __forceinline__ void write_ignored(int64_t r, A* logps, A* stats) {
  logps[r] = A(0);
  if (stats) stats[2 * r + 1] = A(kLeftOut);
}

// logps[r] = (x[r, y] - m) / t - log s, m and s the row's maximum and sum of exponentials. One pass:
// a thread keeps its own maximum and sum, rescaled once for every four vectors, the row's are
// joined at its end. Bound by memory: 4096 x 131072 in 150 us (0.97 GB read, 99 % of the copy
// bandwidth), 4 x 1023 x 50021 in 78 us (80 %: a CTA's start and join are a larger part of a row of
// 100 KB). A row takes a CTA, or where rows are few a cluster.
template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(kThreads)
    logprobs_kernel(Rows a, double inv_temp, A k, A* logps, A* stats) {
  const Place<kThreads> place;
  const int64_t r = place.row, target = a.targets[r];
  if (target == a.ignore) {
    if (place.first()) write_ignored(r, logps, stats);
    return;
  }
  cluster_started(place.ctas);
  const T* x = row_at<T>(a, r);
  A at_target = A(0);
  if (place.first()) at_target = target_logit<T, A>(x, a.vocab, target);
  const RowView<T> view(x, nullptr, reinterpret_cast<uintptr_t>(x), a.vocab);
  const Part<A> p = join_warps<kThreads>(warp_part(view, place, k), k);
  if (place.first()) write_logp(r, at_target, p, inv_temp, logps, stats);
}

// A warp to a row; the steps after the sums by a lane for each of the CTA's rows.
template <typename T, typename A>
__global__ void __launch_bounds__(32 * kRowWarps)
    logprobs_warp_kernel(Rows a, double inv_temp, A k, A* logps, A* stats) {
  __shared__ Part<A> parts[kRowWarps];
  __shared__ A logits[kRowWarps];
  __shared__ bool read[kRowWarps];
  const Place<32> place;
  const int64_t r = place.row;
  const int warp = threadIdx.x / 32;
  const int64_t target = r < a.rows ? a.targets[r] : a.ignore;
  if (place.tid == 0) read[warp] = target != a.ignore;
  if (target != a.ignore) {
    const T* x = row_at<T>(a, r);
    if (place.tid == 0) logits[warp] = target_logit<T, A>(x, a.vocab, target);
    const RowView<T> view(x, nullptr, reinterpret_cast<uintptr_t>(x), a.vocab);
    const Part<A> p = warp_part(view, place, k);
    if (place.tid == 0) parts[warp] = p;
  }
  __syncthreads();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowWarps + threadIdx.x;
  if (threadIdx.x < kRowWarps && row < a.rows) {
    if (read[threadIdx.x]) {
      write_logp(row, logits[threadIdx.x], parts[threadIdx.x], inv_temp, logps, stats);
    } else {
      write_ignored(row, logps, stats);
    }
  }
}

// g[r, v] = coef[r] / t (1[v = y] - exp((x[r, v] - m) / t) / s): one more read of the logits, from
// the sums that the forward kept. Bound by memory: 4 x 1023 x 50021 in 138 us (0.82 GB, 91 %), 147
// us where three quarters of the rows are read and written at different alignments (85 %).
// coef: per row, d loss / d logp. upstream (may be NULL): a scalar that multiplies it, and where
// it is 1 nothing is written. A warp or a CTA (kThreads) takes a tile, `tiles` to the row.
template <typename T, typename A, typename C, int kThreads>
__global__ void __launch_bounds__(256)
    logprobs_grad_kernel(Rows a, double inv_temp, A k, const A* stats, const C* coef,
                         const A* upstream, T* grad, int tiles) {
  const A up = upstream ? *upstream : A(1);
  if (upstream && up == A(1)) return;
  constexpr int kGroups = 256 / kThreads, kTile = kBatch * kThreads;
  const int tid = threadIdx.x % kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kThreads;
       i < a.rows * tiles; i += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t r = i / tiles;
    const int tile = static_cast<int>(i % tiles) * kTile;
    T* g = grad + r * a.vocab;
    const RowView<T> view(row_at<T>(a, r), g, reinterpret_cast<uintptr_t>(g), a.vocab);
    const int edge = tile == 0 ? tid : kNoEdge;
    const A sum = stats[2 * r + 1];
    if (sum < A(0)) {
      zero_edge(view, edge);
      zero_tile<kThreads>(view, tile, tid);
    } else {
      const Slope<A> slope(stats[2 * r], sum, static_cast<double>(coef[r]) * up * inv_temp,
                           k, a.targets[r], a.vocab);
      write_edge(view, edge, slope);
      write_tile<kThreads>(view, tile, tid, slope);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// The clipped policy loss

enum WeightKind { kNoWeight = 0, kByteWeight = 1, kAccWeight = 2 };

template <typename A>
struct PolicyArgs {
  const A *old_logps, *ref_logps, *advantages;
  const void* weight;
  int weight_kind;
  double lo, hi, kl_coef;  // lo, hi: the clip's edges 1 - clip_low and 1 + clip_high
  A* logps;           // per row
  double* coef;       // per row, d loss / d logp
  A* stats;           // per row, maximum and sum
  A* terms;           // per unit (a row, or a CTA's rows), w loss, w kl and w [clipped]
  A* out;             // loss, kl, clip fraction
  double* total;      // sum of the weights
  unsigned* done;     // units whose results are written
};

template <typename A>
__device__ __forceinline__ A weight_of(const Rows& a, const PolicyArgs<A>& p, int64_t r) {
  const int64_t target = a.targets[r];  // both loads in flight together
  A w = A(1);
  if (p.weight_kind == kByteWeight) {
    w = static_cast<const uint8_t*>(p.weight)[r] ? A(1) : A(0);
  } else if (p.weight_kind == kAccWeight) {
    w = static_cast<const A*>(p.weight)[r];
  }
  return target == a.ignore ? A(0) : w;
}

// The sum of the weights, by a CTA, or a cluster of them where there are many rows, ahead of the
// rows. The rows' kernel starts meanwhile (a programmatic launch): what it needs of this one it reads
// after waiting for it.
constexpr int kTotalThreads = 1024, kTotalCtas = 8;

template <typename A>
__global__ void __launch_bounds__(kTotalThreads) policy_total_kernel(Rows a, PolicyArgs<A> p) {
  cudaTriggerProgrammaticLaunchCompletion();
  constexpr int kAhead = 4;
  __shared__ double shared[32], sums[kTotalCtas];
  auto cluster = cg::this_cluster();
  cluster_started(gridDim.x);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTotalThreads;
  double sum = 0;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kTotalThreads + threadIdx.x; r < a.rows;
       r += kAhead * step) {
    A w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      w[i] = r + i * step < a.rows ? weight_of(a, p, r + i * step) : A(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) sum += static_cast<double>(w[i]);
  }
  sum = block_sum(sum, shared);
  if (gridDim.x > 1) {
    wait_for_start();
    if (threadIdx.x == 0) *cluster.map_shared_rank(&sums[blockIdx.x], 0) = sum;
    cluster.sync();
    sum = 0;
    for (unsigned i = 0; i < gridDim.x; ++i) sum += sums[i];  // the first CTA's are the sums
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *p.total = sum;
    *p.done = 0;
    if (a.rows == 0) p.out[0] = p.out[1] = p.out[2] = A(0);
  }
}

// Called by one thread of each unit (a row, or a CTA's rows) once its results are written: whether it
// was the last of them.
template <typename A>
__device__ __forceinline__ bool last_unit(const PolicyArgs<A>& p, int64_t units) {
  __threadfence();
  return atomicAdd(p.done, 1u) == static_cast<unsigned>(units - 1);
}

// The means over the tokens by the CTA of the last unit: in a fixed order whichever it is; 0 when the
// weights sum to 0.
template <typename A>
__device__ void write_means(const PolicyArgs<A>& p, int64_t units) {
  constexpr int kAhead = 4;
  __shared__ double shared[32];
  __threadfence();
  double s[3] = {0, 0, 0};
  const int64_t step = blockDim.x;
  for (int64_t u = threadIdx.x; u < units; u += kAhead * step) {
    A q[kAhead][3];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int j = 0; j < 3; ++j)
        q[i][j] = u + i * step < units ? __ldcg(p.terms + 3 * (u + i * step) + j) : A(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int j = 0; j < 3; ++j) s[j] += static_cast<double>(q[i][j]);
  }
  const double total = *p.total;
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    const double v = block_sum(s[j], shared);
    if (threadIdx.x == 0) p.out[j] = total == 0 ? A(0) : static_cast<A>(v / total);
  }
}

// What the policy loss needs of a token beside its row.
template <typename A>
struct TokenInput {
  int64_t target;
  A w, old, adv, ref, logit;
  double total;  // of the weights

  __device__ __forceinline__ void read(const Rows& a, const PolicyArgs<A>& p, int64_t r,
                                       A logit_) {
    target = a.targets[r];
    old = p.old_logps[r];
    adv = p.advantages[r];
    ref = p.ref_logps ? p.ref_logps[r] : A(0);
    logit = logit_;
    cudaGridDependencySynchronize();  // the total's kernel is done
    total = *p.total;
  }
};

// exp of a double to the accumulation type's precision (in float: of its float, times 1 + the rest;
// for |d| < kFar).
__device__ __forceinline__ float exp_as(float, double d) {
  const float hi = static_cast<float>(d);
  const float lo = static_cast<double>(hi) == d ? 0.0f : static_cast<float>(d - hi);
  const float e = expf(hi);
  return __fmaf_rn(e, lo, e);
}
__device__ __forceinline__ double exp_as(double, double d) { return exp(d); }

// exp(d) / s and exp(d) s, s a row's sum (up to 2^30). Beyond e^+-60 float has no room for them, nor
// for exp(d) on the way: a token that the old policy all but excluded has a ratio of any size, which
// the clip then cuts.
constexpr double kFar = 60.0;
template <typename A>
__device__ __forceinline__ double exp_over(double d, A s) {
  if (fabs(d) < kFar) return exp_as(A(0), d) / s;
  return exp(d - log(static_cast<double>(s)));
}
template <typename A>
__device__ __forceinline__ double exp_times(double d, A s) {
  if (fabs(d) < kFar) return exp_as(A(0), d) * s;
  return exp(d + log(static_cast<double>(s)));
}

// A token's loss and its slope d loss / d logp (both without the token's weight):
//   rho = exp(logp - old);  loss = -min(rho A, clip(rho) A) + kl_coef kl,
//   kl = exp(d) - d - 1, d = ref - logp;
//   slope = -rho A where rho A <= clip(rho) A, else 0, plus kl_coef (1 - exp(d)).
// With t = (x - base) / temperature at the target and s the row's sum, logp = t - log s, so that
// rho = exp(t - old) / s and exp(d) = exp(ref - t) s: the slope, which a row's gradient waits for,
// needs no logarithm. t is in double: rounding it near 10 would be the largest error of all.
template <typename A>
struct Token {
  double t, ratio, free_side, held;
  double coef;  // d loss / d logp with the weight's share

  __device__ __forceinline__ Token(const PolicyArgs<A>& p, const TokenInput<A>& in,
                                   const Part<A>& part, double inv_temp) {
    t = (static_cast<double>(in.logit) - static_cast<double>(base_of(part.m))) * inv_temp;
    ratio = exp_over(t - static_cast<double>(in.old), part.s);
    // a factor of 0 leaves its term out, whatever overflowed in the other one
    free_side = in.adv == A(0) && isinf(ratio) ? 0.0 : ratio * static_cast<double>(in.adv);
    held = (ratio < p.lo ? p.lo : ratio > p.hi ? p.hi : ratio) * static_cast<double>(in.adv);
    double slope = free_side > held ? 0.0 : -free_side;
    if (p.ref_logps && p.kl_coef != 0)
      slope += p.kl_coef * (1.0 - exp_times(static_cast<double>(in.ref) - t, part.s));
    coef = in.total != 0 ? static_cast<double>(in.w) / in.total * slope : 0.0;
  }

  // the row's results, and in `terms` what the means sum
  __device__ __forceinline__ void write(const PolicyArgs<A>& p, int64_t r, const TokenInput<A>& in,
                                        const Part<A>& part, A (&terms)[3]) const {
    const double lp = t - log(static_cast<double>(part.s));
    double loss = -(free_side > held ? held : free_side), kl = 0.0;
    if (p.ref_logps) {
      const double d = static_cast<double>(in.ref) - lp;
      kl = isinf(d) ? static_cast<double>(INFINITY) : expm1(d) - d;
      if (p.kl_coef != 0) loss += p.kl_coef * kl;
    }
    p.logps[r] = static_cast<A>(lp);
    p.coef[r] = coef;
    p.stats[2 * r] = base_of(part.m);
    p.stats[2 * r + 1] = part.s;
    terms[0] = static_cast<A>(in.w * loss);
    terms[1] = static_cast<A>(in.w * kl);
    terms[2] = free_side > held ? in.w : A(0);
  }
};

template <typename A>
__device__ __forceinline__ void write_terms(const PolicyArgs<A>& p, int64_t unit,
                                            const A (&terms)[3]) {
#pragma unroll
  for (int j = 0; j < 3; ++j) p.terms[3 * unit + j] = terms[j];
}

// The row's cut is as for a gradient in a buffer on a vector's boundary, also where no gradient is
// written (grad NULL): the loss is the same bits.
template <typename T>
__device__ __forceinline__ RowView<T> policy_view(const Rows& a, int64_t r, T* grad) {
  T* g = grad + r * a.vocab;
  return RowView<T>(row_at<T>(a, r), g, reinterpret_cast<uintptr_t>(g), a.vocab);
}

template <typename A>
__device__ __forceinline__ void write_left_out(const PolicyArgs<A>& p, int64_t r) {
  p.logps[r] = A(0);
  p.coef[r] = 0;
  p.stats[2 * r + 1] = A(kLeftOut);
}

// Short rows: a warp to a row, which it reads twice; the tokens' steps between by a lane for each of
// the CTA's rows (by every warp for its own row they cost as much as 2000 logits).
template <typename T, typename A>
__global__ void __launch_bounds__(32 * kRowWarps)
    policy_warp_kernel(Rows a, PolicyArgs<A> p, double inv_temp, A k, T* grad) {
  __shared__ Part<A> parts[kRowWarps];
  __shared__ TokenInput<A> tokens[kRowWarps];  // of weight 0: a row that is left out, or none
  __shared__ double coefs[kRowWarps];
  __shared__ bool last;
  const Place<32> place;
  const int64_t r = place.row, first_row = static_cast<int64_t>(blockIdx.x) * kRowWarps;
  const int warp = threadIdx.x / 32;
  const bool is_row = r < a.rows;
  const RowView<T> view = policy_view(a, is_row ? r : first_row, grad);
  const A w = is_row ? weight_of(a, p, r) : A(0);
  if (w != A(0)) {
    TokenInput<A> token;
    if (place.tid == 0)  // in flight with the row's own loads
      token.read(a, p, r, target_logit<T, A>(view.x, a.vocab, a.targets[r]));
    const Part<A> part = warp_part(view, place, k);
    if (place.tid == 0) {
      token.w = w;
      tokens[warp] = token;
      parts[warp] = part;
    }
  } else if (place.tid == 0) {
    tokens[warp].w = w;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    const int64_t row = first_row + threadIdx.x;
    A terms[3] = {};
    if (threadIdx.x < kRowWarps && row < a.rows) {
      const TokenInput<A>& token = tokens[threadIdx.x];
      if (token.w != A(0)) {
        const Token<A> result(p, token, parts[threadIdx.x], inv_temp);
        result.write(p, row, token, parts[threadIdx.x], terms);
        coefs[threadIdx.x] = result.coef;
      } else {
        write_left_out(p, row);
      }
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
#pragma unroll
      for (int d = kRowWarps / 2; d; d >>= 1) terms[j] += __shfl_xor_sync(0xffffffffu, terms[j], d);
    if (threadIdx.x == 0) write_terms(p, blockIdx.x, terms);
  }
  __syncthreads();
  if (grad && is_row) {
    if (w != A(0)) {
      const Slope<A> slope(base_of(parts[warp].m), parts[warp].s, coefs[warp] * inv_temp, k,
                           tokens[warp].target, a.vocab);
      write_edge(view, place.edge(), slope);
      for (int tile = 0; tile < view.vectors; tile += kBatch * 32)
        write_tile<32>(view, tile, place.tid, slope);
    } else {
      zero_edge(view, place.edge());
      for (int tile = 0; tile < view.vectors; tile += kBatch * 32)
        zero_tile<32>(view, tile, place.tid);
    }
  }
  if (threadIdx.x == 0) {
    cudaGridDependencySynchronize();
    last = last_unit(p, gridDim.x);
  }
  __syncthreads();
  if (last) write_means(p, gridDim.x);
}

// Loss and gradient in one launch: the row's sum, the token's coefficient, then the row's gradient
// from a second read that does not reach memory. 4000 x 131072, a tenth of them left out, in 376 us:
// 2.04 GB of DRAM traffic, 3 % over each byte once, at 83 % of the copy bandwidth; 8192 rows in 840 to
// 880 us. The exponential unit is busy 63 % of the time, and what is missing are the joins between a
// row's two passes (of a CTA's 20 us about 5), which two other CTAs of the SM fill in part.
//
// A cluster's CTAs take a row's tiles in turn, a tile kBatch vectors a thread. Tiles come through
// kStages places of shared memory, each thread copying and reading its own vectors there (no
// barrier), so that kStages tiles are in flight. The gradient takes them in the reverse order: the
// last kStages are still there, and the others, if few enough rows are in work at a time, in L2.
// A last tile that is cut goes this way too: loaded directly it is waited for twice (32000 to the
// row: 306 us for 800 MB of bf16 logits, 320 with it loaded). The tiles of a row that is read and
// written at different alignments are loaded directly, from two vectors each.
constexpr int kStages = 2;
constexpr int kSmThreads = 1536;  // resident at 40 registers a thread (spills: double 96 bytes, 16-bit types 8)

template <int kThreads, typename T, typename A>
__device__ __forceinline__ void policy_row(const Rows& a, const PolicyArgs<A>& p, double inv_temp,
                                           A k, T* grad, bool& last) {
  constexpr int kTile = kBatch * kThreads;
  extern __shared__ uint4 stages[];  // [kStages][kTile]
  __shared__ TokenInput<A> token;    // read after the join's barrier
  const Place<kThreads> place;
  const int64_t r = place.row;
  const RowView<T> view = policy_view(a, r, grad);
  const A w = weight_of(a, p, r);
  if (w == A(0)) {
    if (place.first()) {
      write_left_out(p, r);
      write_terms(p, r, {A(0), A(0), A(0)});
      cudaGridDependencySynchronize();
      last = last_unit(p, a.rows);
    }
    if (!grad) return;
    zero_edge(view, place.edge());
    for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile)
      zero_tile<kThreads>(view, tile, place.tid);
    return;
  }
  cluster_started(place.ctas);
  // this CTA's tiles that go through shared memory: its j-th is tile cta + j ctas; the row's last
  // tile may be cut
  const int staged = view.shift == 0 ? view.vectors : 0;
  const int tiles = (staged + kTile - 1) / kTile;
  const int mine = tiles > place.cta ? (tiles - place.cta + place.ctas - 1) / place.ctas : 0;
  const bool cut = staged % kTile != 0 && (tiles - 1) % place.ctas == place.cta;
  const int whole = mine - cut;
  const int stride = place.ctas * kTile;
  const int own = place.cta * kTile + place.tid;
  const uint4* from = reinterpret_cast<const uint4*>(view.x + view.head) + own;
  uint4* to = reinterpret_cast<uint4*>(view.g + view.head) + own;
  const auto has = [&](int i) { return own + whole * stride + i * kThreads < staged; };  // if cut
  const auto copy = [&](int j) {
    uint4* at = stages + static_cast<unsigned>(j) % kStages * kTile + place.tid;
    if (j >= 0 && j < whole) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        copy_async(at + i * kThreads, from + static_cast<int64_t>(j) * stride + i * kThreads);
    } else if (cut && j == whole) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (has(i))
          copy_async(at + i * kThreads, from + static_cast<int64_t>(j) * stride + i * kThreads);
    }
    close_group();
  };
  const auto fetch = [&](int j, uint4 (&q)[kBatch]) {
    wait_groups<kStages - 1>();  // tile j's, closed kStages - 1 groups before the last
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      q[i] = stages[static_cast<unsigned>(j) % kStages * kTile + i * kThreads + place.tid];
  };
#pragma unroll
  for (int j = 0; j < kStages; ++j) copy(j);
  if (place.tid == 0) {
    token.w = w;
    token.read(a, p, r, target_logit<T, A>(view.x, a.vocab, a.targets[r]));
  }

  // the tiles that are loaded directly, and the single elements
  Part<A> part = thread_part(view, place, staged ? staged : place.cta * kTile, k);
  for (int j = 0; j < whole; ++j) {
    uint4 q[kBatch];
    fetch(j, q);
    copy(j + kStages);
    add_vectors<T>(part, q, k);
  }
  if (cut) {
    uint4 q[kBatch];
    fetch(whole, q);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (!has(i)) q[i] = no_vector<T>();
    add_vectors<T>(part, q, k);
    close_group();
  }
  part = join_warps<kThreads>(join_lanes<32>(part, k), k);
  // every warp takes the few steps to the coefficient by itself: one more barrier takes longer
  const Token<A> result(p, token, part, inv_temp);
  if (place.first()) {
    A terms[3];
    result.write(p, r, token, part, terms);
    write_terms(p, r, terms);
    last = last_unit(p, a.rows);
  }
  if (!grad) return;
  const Slope<A> slope(base_of(part.m), part.s, result.coef * inv_temp, k, token.target, a.vocab);
  const auto write_target = [&](int j) {
    write_target_of_tile<kThreads, kTile>(view, own - place.tid + j * stride, place.tid, slope);
  };
  if (cut) {
    uint4 q[kBatch];
    fetch(whole, q);
    copy(whole - kStages);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (has(i))
        store_once(to + static_cast<int64_t>(whole) * stride + i * kThreads,
                   slope_vector<T>(q[i], slope));
    write_target(whole);
  }
  for (int j = whole - 1; j >= 0; --j) {
    uint4 q[kBatch];
    fetch(j, q);
    copy(j - kStages);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      store_once(to + static_cast<int64_t>(j) * stride + i * kThreads,
                 slope_vector<T>(q[i], slope));
    write_target(j);
  }
  write_edge(view, place.edge(), slope);
  if (staged == 0)
    for (int tile = place.cta * kTile; tile < view.vectors; tile += stride)
      write_tile<kThreads>(view, tile, place.tid, slope);
}

template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(kThreads, kSmThreads / kThreads)
    policy_kernel(Rows a, PolicyArgs<A> p, double inv_temp, A k, T* grad) {
  __shared__ bool last;  // written by thread 0 alone
  if (threadIdx.x == 0) last = false;
  policy_row<kThreads>(a, p, inv_temp, k, grad, last);
  __syncthreads();
  if (last) write_means(p, a.rows);
}

// ---------------------------------------------------------------------------------------------
// Host side

// grad: NULL, or the gradient that the call writes
int check_rows(int dtype, const tiso_rows* x, const int64_t* targets, const void* grad) {
  if (dtype < TISO_F16 || dtype > TISO_F64)
    return report_error(TISO_ERR_ARGUMENT, "dtype must be a tiso_dtype");
  if (!x) return report_error(TISO_ERR_ARGUMENT, "rows is NULL");
  if (x->rows < 0 || x->vocab < 1 || x->inner < 1)
    return report_error(TISO_ERR_ARGUMENT, "need rows >= 0, vocab >= 1 and inner >= 1");
  if (x->outer_stride < 0 || x->inner_stride < 0)
    return report_error(TISO_ERR_ARGUMENT, "strides must not be negative");
  if (x->rows > kMostRows || x->vocab > int64_t{1} << 30)
    return report_error(TISO_ERR_ARGUMENT, "more than 2^28 rows or a vocabulary of more than 2^30");
  if (x->rows && (!x->data || !targets))
    return report_error(TISO_ERR_ARGUMENT, "logits and targets must not be NULL");
  const int size = dtype == TISO_F64 ? 8 : dtype == TISO_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x->data) | reinterpret_cast<uintptr_t>(grad)) % size)
    return report_error(TISO_ERR_ARGUMENT, "logits and grad must be aligned to their elements");
  return TISO_OK;
}

Rows rows_of(const tiso_rows* x, const int64_t* targets, int64_t ignore) {
  return {x->data,         x->rows,          x->inner,
          x->outer_stride, x->inner_stride,  static_cast<int>(x->vocab),
          targets,         ignore};
}

// log2(e) / t for the exponentials in float, 1 / t for those in double
float exp_factor(float, double inv_temp) {
  return static_cast<float>(inv_temp * 1.4426950408889634);
}
double exp_factor(double, double inv_temp) { return inv_temp; }

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TISO_OK : logits_fail(e, what);
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Allows a kernel more than 48 KB of dynamic shared memory: once per kernel and device.
int allow_shared(const void* kernel, size_t bytes) {
  static std::mutex mutex;
  static std::set<std::pair<const void*, int>> done;
  if (bytes <= 48 * 1024) return TISO_OK;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return logits_fail(e, "cudaGetDevice");
  std::lock_guard<std::mutex> lock(mutex);
  if (done.count({kernel, dev})) return TISO_OK;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(bytes));
  if (e != cudaSuccess) return logits_fail(e, "cudaFuncSetAttribute");
  done.insert({kernel, dev});
  return TISO_OK;
}

// A launch of `clusters` clusters of `ctas` CTAs (a power of two up to 8) of `threads`. early: it may
// start before the kernel ahead of it in the stream is done, and waits for it itself.
template <typename... P, typename... Q>
int launch_clusters(void (*kernel)(P...), int64_t clusters, int ctas, int threads, size_t shared,
                    bool early, cudaStream_t st, const char* what, Q... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(clusters * ctas));
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = shared;
  config.stream = st;
  cudaLaunchAttribute attributes[2]{};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = early ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
  return e == cudaSuccess ? TISO_OK : logits_fail(e, what);
}

// A kernel over rows, a warp to each.
template <typename... P, typename... Q>
int launch_warps(void (*kernel)(P...), int64_t rows, cudaStream_t st, const char* what, Q... args) {
  kernel<<<static_cast<unsigned>((rows + kRowWarps - 1) / kRowWarps), 32 * kRowWarps, 0, st>>>(
      args...);
  return launched(what);
}

// Rows of at most kWarpVectors vectors go to a warp each; of up to `most` of them where there are
// enough rows to fill the GPU with warps. A CTA's start and join cost as much as some 1000 vectors:
// 97656 x 4096 bf16, log-probabilities 126 us by warps and 342 by CTAs of 256 threads, their gradient
// 272 and 358, the policy loss 380 and 779; 976 x 8192: 11.2 and 10.2 us.
constexpr int kWarpVectors = 256;

bool by_warps(int64_t rows, int64_t vectors, int64_t most, int sms) {
  return vectors <= kWarpVectors || (vectors <= most && rows >= int64_t{16} * sms);
}

// Bytes of rows in work at once that L2 is to hold from a row's first read to its
// second. Rows of 256 KB: one CTA to a row (116 MB) reads 1.8 GB where two (58 MB) read 1.06 and
// four 0.95 (0.94 is each byte once); two are fastest (828, 874 and 931 us with 2, 1 and 4).
constexpr int64_t kRowsInL2 = 80 << 20;

// CTAs of `threads` to a row: doubled while rows are too few to fill the GPU and a CTA would have
// more than a batch for each thread.
int ctas_for(int64_t rows, int64_t vectors, int threads, int sms) {
  int ctas = 1;
  while (ctas < 8 && rows * ctas < 2 * sms && vectors > int64_t{ctas} * threads * kBatch) ctas *= 2;
  return ctas;
}

template <typename T>
int run_logprobs(const Rows& a, double inv_temp, void* logps, void* stats, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int vectors = a.vocab / RowView<T>::E;
  const A k = exp_factor(A(0), inv_temp);
  const int sms = sm_count();
  if (by_warps(a.rows, vectors, 2048, sms))  // 24414 x 16384 bf16: 125 us, by CTAs 140
    return launch_warps(logprobs_warp_kernel<T, A>, a.rows, st, "logprobs_warp_kernel launch",
                        a, inv_temp, k, static_cast<A*>(logps), static_cast<A*>(stats));
  return launch_clusters(logprobs_kernel<T, A, 256>, a.rows,
                         ctas_for(a.rows, vectors, 256, sms), 256, 0, false, st,
                         "logprobs_kernel launch", a, inv_temp, k, static_cast<A*>(logps),
                         static_cast<A*>(stats));
}

template <typename T, typename C>
int run_logprobs_grad(const Rows& a, double inv_temp, const void* stats, const void* coef,
                      const void* upstream, void* grad, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int vectors = a.vocab / RowView<T>::E;
  const int sms = sm_count();
  const bool by_warp = by_warps(a.rows, vectors, 768, sms);  // 48828 x 8192: 262 us, by CTAs 250
  const int tile = kBatch * (by_warp ? 32 : 256);
  const int tiles = vectors > tile ? (vectors + tile - 1) / tile : 1;
  const int64_t all = (a.rows * tiles + (by_warp ? 7 : 0)) / (by_warp ? 8 : 1);
  // where the launch may have nothing to do (upstream is 1), no more CTAs than are resident
  const int64_t most = upstream ? int64_t{sms} * 8 : int64_t{1} << 30;
  const unsigned grid = static_cast<unsigned>(all < most ? all : most);
  const A k = exp_factor(A(0), inv_temp);
  auto kernel = by_warp ? logprobs_grad_kernel<T, A, C, 32> : logprobs_grad_kernel<T, A, C, 256>;
  kernel<<<grid, 256, 0, st>>>(a, inv_temp, k, static_cast<const A*>(stats),
                               static_cast<const C*>(coef), static_cast<const A*>(upstream),
                               static_cast<T*>(grad), tiles);
  return launched("logprobs_grad_kernel launch");
}

template <typename T, int kThreads>
int launch_policy_rows(const Rows& a, const PolicyArgs<typename AccOf<T>::type>& p, double inv_temp,
                       T* grad, int sms, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr size_t kShared = size_t{kStages} * kBatch * kThreads * 16;
  const int64_t vectors = a.vocab / RowView<T>::E;
  int ctas = ctas_for(a.rows, vectors, kThreads, sms);
  while (ctas < 8 && int64_t{sms} * (kSmThreads / kThreads) * vectors * 16 / ctas > kRowsInL2)
    ctas *= 2;
  const auto kernel = policy_kernel<T, A, kThreads>;
  const int rc = allow_shared(reinterpret_cast<const void*>(kernel), kShared);
  if (rc) return rc;
  return launch_clusters(kernel, a.rows, ctas, kThreads, kShared, true, st, "policy_kernel launch",
                         a, p, inv_temp, exp_factor(A(0), inv_temp), grad);
}

// By warps, or in CTAs of the more threads the longer the row: smaller ones have more rows in work,
// which hides a row's start and join, larger ones less of both. 800 MB of bf16 logits, us: 8192 to
// the row by warps 374, by 128 threads 415; 10000: 394, 435; 12000: 394, 391; 16384: 375, 312. By
// 128, 256 and 512 threads 16384: 312, 314, 431, 32000: 312, 294, 333, 50021: 347, 314, 323, 65536:
// 303, 303, 277, 131072: 297, 302, 290. Rows whose last tile is cut lose more with 512 (100003: 311
// with 256, 337 with 512).
template <typename T>
int launch_policy(const Rows& a, const PolicyArgs<typename AccOf<T>::type>& p, double inv_temp,
                  T* grad, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int64_t vectors = a.vocab / RowView<T>::E;
  const int sms = sm_count();
  if (by_warps(a.rows, vectors, 1536, sms))
    return launch_clusters(policy_warp_kernel<T, A>, (a.rows + kRowWarps - 1) / kRowWarps, 1,
                           32 * kRowWarps, 0, true, st, "policy_warp_kernel launch", a, p, inv_temp,
                           exp_factor(A(0), inv_temp), grad);
  if (vectors <= 2560) return launch_policy_rows<T, 128>(a, p, inv_temp, grad, sms, st);
  if (vectors >= 8192 && vectors % (kBatch * 512) == 0)
    return launch_policy_rows<T, 512>(a, p, inv_temp, grad, sms, st);
  return launch_policy_rows<T, 256>(a, p, inv_temp, grad, sms, st);
}

template <typename T>
int run_policy(const Rows& a, const tiso_policy_args* q, double inv_temp, void* logps, double* coef,
               void* stats, void* out, void* grad, void* workspace, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  PolicyArgs<A> p{};
  p.old_logps = static_cast<const A*>(q->old_logps);
  p.ref_logps = static_cast<const A*>(q->ref_logps);
  p.advantages = static_cast<const A*>(q->advantages);
  p.weight = q->weight;
  p.weight_kind = !q->weight ? kNoWeight : q->weight_is_byte ? kByteWeight : kAccWeight;
  p.lo = 1.0 - q->clip_low;
  p.hi = 1.0 + q->clip_high;
  p.kl_coef = q->kl_coef;
  p.logps = static_cast<A*>(logps);
  p.coef = coef;
  p.stats = static_cast<A*>(stats);
  p.out = static_cast<A*>(out);
  p.total = static_cast<double*>(workspace);
  p.done = reinterpret_cast<unsigned*>(p.total + 1);
  p.terms = reinterpret_cast<A*>(p.total + 2);
  // 8192 rows: 7 us by one CTA
  const int ctas = a.rows > 8 * kTotalThreads ? kTotalCtas : 1;
  const int rc = launch_clusters(policy_total_kernel<A>, 1, ctas, kTotalThreads, 0, false, st,
                                 "policy_total_kernel launch", a, p);
  if (rc || a.rows == 0) return rc;
  return launch_policy<T>(a, p, inv_temp, static_cast<T*>(grad), st);
}

// fn(T{}) with T the element type of dtype
template <typename F>
int by_type(int dtype, F&& fn) {
  switch (dtype) {
    case TISO_F16: return fn(__half{});
    case TISO_BF16: return fn(__nv_bfloat16{});
    case TISO_F32: return fn(float{});
    default: return fn(double{});
  }
}

}  // namespace
}  // namespace tiso

using namespace tiso;

extern "C" {

int tiso_logprobs(int dtype, const tiso_rows* x, const int64_t* targets, int64_t ignore_index,
                  double temperature, void* logps, void* stats, void* stream) {
  return guarded([&]() -> int {
    const int rc = check_rows(dtype, x, targets, nullptr);
    if (rc) return rc;
    if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
    if (x->rows == 0) return TISO_OK;
    if (!logps) return report_error(TISO_ERR_ARGUMENT, "logps must not be NULL");
    const Rows a = rows_of(x, targets, ignore_index);
    return by_type(dtype, [&](auto t) {
      return run_logprobs<decltype(t)>(a, 1.0 / temperature, logps, stats,
                                       static_cast<cudaStream_t>(stream));
    });
  });
}

int tiso_logprobs_grad(int dtype, const tiso_rows* x, const int64_t* targets, double temperature,
                       const void* stats, int coef_dtype, const void* coef,
                       const void* upstream, void* grad, void* stream) {
  return guarded([&]() -> int {
    const int rc = check_rows(dtype, x, targets, grad);
    if (rc) return rc;
    if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
    if (x->rows == 0) return TISO_OK;
    if (!stats || !coef || !grad)
      return report_error(TISO_ERR_ARGUMENT, "stats, coef and grad must not be NULL");
    if (coef_dtype != TISO_F64 && (coef_dtype != TISO_F32 || dtype == TISO_F64))
      return report_error(TISO_ERR_ARGUMENT, "coef_dtype must be the accumulation type or TISO_F64");
    const Rows a = rows_of(x, targets, 0);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (coef_dtype == TISO_F64)
        return run_logprobs_grad<T, double>(a, 1.0 / temperature, stats, coef, upstream, grad, st);
      return run_logprobs_grad<T, typename AccOf<T>::type>(a, 1.0 / temperature, stats, coef,
                                                           upstream, grad, st);
    });
  });
}

int tiso_policy_workspace_size(int dtype, int64_t rows, size_t* bytes) {
  return guarded([&]() -> int {
    if (!bytes) return report_error(TISO_ERR_ARGUMENT, "bytes is NULL");
    *bytes = 0;
    if (dtype < TISO_F16 || dtype > TISO_F64)
      return report_error(TISO_ERR_ARGUMENT, "dtype must be a tiso_dtype");
    if (rows < 0) return report_error(TISO_ERR_ARGUMENT, "need rows >= 0");
    *bytes = 16 + static_cast<size_t>(rows) * 3 * (dtype == TISO_F64 ? 8 : 4);
    return TISO_OK;
  });
}

int tiso_policy(int dtype, const tiso_rows* x, const int64_t* targets, int64_t ignore_index,
                double temperature, const tiso_policy_args* args, void* logps, double* coef,
                void* stats, void* out, void* grad, void* workspace, size_t workspace_bytes,
                void* stream) {
  return guarded([&]() -> int {
    int rc = check_rows(dtype, x, targets, grad);
    if (rc) return rc;
    if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
    if (!args) return report_error(TISO_ERR_ARGUMENT, "args is NULL");
    if (!(args->clip_low >= 0 && args->clip_high >= 0))
      return report_error(TISO_ERR_ARGUMENT, "clip_low and clip_high must not be negative");
    if (x->rows && (!args->old_logps || !args->advantages || !logps || !coef || !stats))
      return report_error(TISO_ERR_ARGUMENT,
                          "old_logps, advantages, logps, coef and stats must not be NULL");
    if (!out) return report_error(TISO_ERR_ARGUMENT, "out must not be NULL");
    size_t need = 0;
    rc = tiso_policy_workspace_size(dtype, x->rows, &need);
    if (rc) return rc;
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))
      return report_error(TISO_ERR_WORKSPACE,
                          "workspace missing, unaligned or smaller than tiso_policy_workspace_size");
    const Rows a = rows_of(x, targets, ignore_index);
    return by_type(dtype, [&](auto t) {
      return run_policy<decltype(t)>(a, args, 1.0 / temperature, logps, coef, stats, out, grad,
                                     workspace, static_cast<cudaStream_t>(stream));
    });
  });
}

}  // extern "C"
