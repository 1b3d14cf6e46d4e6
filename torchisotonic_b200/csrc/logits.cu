// Operators on rows of logits (include/tiso.h: tiso_logprobs*, tiso_policy*): the log-probability
// of one token per row and its gradient, and the clipped policy loss with its gradient.
//
// All are streams over the logits: an exponential and about four other instructions an element and
// pass, no contraction. Times below are of one B200 (copy bandwidth 6545 GB/s measured), bf16.
#include "rows.cuh"

namespace tiso {
namespace {

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

template <typename A>
struct PolicyArgs {
  const A *old_logps, *ref_logps, *advantages;
  TokenWeights<A> weights;
  double lo, hi, kl_coef;  // lo, hi: the clip's edges 1 - clip_low and 1 + clip_high
  A* logps;           // per row
  double* coef;       // per row, d loss / d logp
  A* stats;           // per row, maximum and sum
  A* terms;           // per unit (a row, or a CTA's rows), w loss, w kl and w [clipped]
  A* out;             // loss, kl, clip fraction
  double* total;      // sum of the weights
  unsigned* done;     // units whose results are written
};

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
  const A w = is_row ? p.weights.of(a.targets[r], r) : A(0);
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
    last = last_unit(p.done, gridDim.x);
  }
  __syncthreads();
  if (last) write_means<3>(p.terms, *p.total, p.out, gridDim.x);
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
constexpr int kSmThreads = 1536;  // resident at 40 registers a thread (spills: double 108 bytes)

template <int kThreads, typename T, typename A>
__device__ __forceinline__ void policy_row(const Rows& a, const PolicyArgs<A>& p, double inv_temp,
                                           A k, T* grad, bool& last) {
  constexpr int kTile = kBatch * kThreads;
  extern __shared__ uint4 stages[];  // [kStages][kTile]
  __shared__ TokenInput<A> token;    // read after the join's barrier
  const Place<kThreads> place;
  const int64_t r = place.row;
  const RowView<T> view = policy_view(a, r, grad);
  const TokenWeights<A> weights = p.weights;  // (by way of p: 50021 to the row in 129.5 us, not 127.6)
  const A w = weights.of(weights.marks[r], r);
  if (w == A(0)) {
    if (place.first()) {
      write_left_out(p, r);
      write_terms(p, r, {A(0), A(0), A(0)});
      cudaGridDependencySynchronize();
      last = last_unit(p.done, a.rows);
    }
    if (!grad) return;
    zero_edge(view, place.edge());
    for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile)
      zero_tile<kThreads>(view, tile, place.tid);
    return;
  }
  cluster_started(place.ctas);
  const StagedTiles<kThreads, T> tiles(view, place, stages);
#pragma unroll
  for (int j = 0; j < kStages; ++j) tiles.copy(j);
  if (place.tid == 0) {
    token.w = w;
    token.read(a, p, r, target_logit<T, A>(view.x, a.vocab, a.targets[r]));
  }

  // the tiles that are loaded directly, and the single elements
  Part<A> part = thread_part(view, place, tiles.staged ? tiles.staged : place.cta * kTile, k);
  for (int j = 0; j < tiles.whole; ++j) {
    uint4 q[kBatch];
    tiles.fetch(j, q);
    tiles.copy(j + kStages);
    add_vectors<T>(part, q, k);
  }
  if (tiles.cut) {
    uint4 q[kBatch];
    tiles.arrived();
    tiles.read_cut(q);
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
    last = last_unit(p.done, a.rows);
  }
  if (!grad) return;
  const Slope<A> slope(base_of(part.m), part.s, result.coef * inv_temp, k, token.target, a.vocab);
  const auto write_target = [&](int j) {
    write_target_of_tile<kThreads, kTile>(view, tiles.tile(j), place.tid, slope);
  };
  if (tiles.cut) {
    uint4 q[kBatch];
    tiles.fetch(tiles.whole, q);
    tiles.copy(tiles.whole - kStages);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (tiles.has(i)) store_once(tiles.to(tiles.whole) + i * kThreads, slope_vector<T>(q[i], slope));
    write_target(tiles.whole);
  }
  for (int j = tiles.whole - 1; j >= 0; --j) {
    uint4 q[kBatch];
    tiles.fetch(j, q);
    tiles.copy(j - kStages);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      store_once(tiles.to(j) + i * kThreads, slope_vector<T>(q[i], slope));
    write_target(j);
  }
  write_edge(view, place.edge(), slope);
  if (tiles.staged == 0)
    for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile)
      write_tile<kThreads>(view, tile, place.tid, slope);
}

template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(kThreads, kSmThreads / kThreads)
    policy_kernel(Rows a, PolicyArgs<A> p, double inv_temp, A k, T* grad) {
  __shared__ bool last;  // written by thread 0 alone
  if (threadIdx.x == 0) last = false;
  policy_row<kThreads>(a, p, inv_temp, k, grad, last);
  __syncthreads();
  if (last) write_means<3>(p.terms, *p.total, p.out, a.rows);
}

// ---------------------------------------------------------------------------------------------
// Host side

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
  p.weights = weights_of<A>(a.targets, 1, a.ignore, q->weight, q->weight_is_byte);
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
  const int rc = launch_total(p.weights, a.rows, 8 * kTotalThreads, p.total, p.done, p.out, 3, st);
  if (rc || a.rows == 0) return rc;
  return launch_policy<T>(a, p, inv_temp, static_cast<T*>(grad), st);
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
