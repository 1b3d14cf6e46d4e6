// The preference loss (include/tiso.h: tiso_preference*): paired log ratios of packed sequences
// of token log-probabilities, forward and backward.
//
// With sequences 0..P-1 the chosen and P..2P-1 the rejected answers,
//   s_k = sum over the sequence's unmasked tokens of (logp - ref)  (their mean with `average`),
//   u_i = beta (s_i - s_{P+i}) - margin,  loss = mean of l(u_i),
//   d loss / d logp_t = +-beta l'(u) / P (1 / count with `average`), + for chosen.
// Sums are double, in a fixed order.
//
// Three launches: the sequences' sums, one CTA over the pairs, and in the backward the tokens. All
// are small (8 bytes a token): up to some 100,000 tokens they take 3 to 7 us each, the latency of a
// launch and a few dependent loads; 2e6 tokens in 512 answers 13, 5 and 11 us (18 MB, 2.8 us at the
// copy bandwidth). A pass through autograd costs more host time (70 us) than all of that.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <string>

#include "cta.cuh"
#include "entry.cuh"

namespace tiso {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kManyThreads = 1024;

template <typename A>
struct PrefArgs {
  const A *logps, *refs;
  const uint8_t* mask;
  const int64_t* offsets;
  int64_t tokens, pairs;
  int kind, average;
  double beta, smoothing, margin;
  double *sums, *counts;  // per sequence
  A *loss, *rewards, *coef;
};

// Offsets are the caller's numbers on the device: cut to the tokens there are.
__device__ __forceinline__ int64_t cut(int64_t v, int64_t lo, int64_t hi) {
  return v < lo ? lo : v > hi ? hi : v;
}

// A cluster of CTAs (one, where there are many sequences) to a sequence: the sum and number of its
// unmasked tokens. A masked token is read but not used in any way (its value may be NaN).
template <typename A, int kT>
__global__ void __launch_bounds__(kT) pref_sum_kernel(PrefArgs<A> a) {
  constexpr int kAhead = 4, kMostCtas = 8;
  __shared__ double shared[32], sums[kMostCtas], counts[kMostCtas];
  auto cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  cluster_started(ctas);
  const int64_t k = blockIdx.x / ctas;
  const int64_t begin = cut(a.offsets[k], 0, a.tokens);
  const int64_t end = cut(a.offsets[k + 1], begin, a.tokens);
  const int64_t step = static_cast<int64_t>(ctas) * kT;
  double sum = 0, count = 0;
  for (int64_t t = begin + rank * kT + threadIdx.x; t < end; t += kAhead * step) {
    A x[kAhead], ref[kAhead];
    bool used[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t u = t + i * step;
      used[i] = u < end;
      x[i] = ref[i] = A(0);
      if (u < end) {
        if (a.mask) used[i] = a.mask[u] != 0;
        x[i] = a.logps[u];
        if (a.refs) ref[i] = a.refs[u];
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      sum += used[i] ? static_cast<double>(x[i]) - static_cast<double>(ref[i]) : 0.0;
      count += used[i] ? 1.0 : 0.0;
    }
  }
  sum = block_sum(sum, shared);
  count = block_sum(count, shared);
  if (ctas > 1) {
    wait_for_start();
    if (threadIdx.x == 0) {
      *cluster.map_shared_rank(&sums[rank], 0) = sum;
      *cluster.map_shared_rank(&counts[rank], 0) = count;
    }
    cluster.sync();
    if (rank != 0) return;
    sum = count = 0;
    for (int i = 0; i < ctas; ++i) {
      sum += sums[i];
      count += counts[i];
    }
  }
  if (threadIdx.x == 0) {
    a.sums[k] = sum;
    a.counts[k] = count;
  }
}

// log(1 + exp(-u)) without overflow
__device__ __forceinline__ double softplus_neg(double u) {
  return log1p(exp(-fabs(u))) + (u < 0 ? -u : 0.0);
}

__device__ void pair_loss(int kind, double u, double smoothing, double beta, double* loss,
                          double* slope) {
  if (kind == TISO_PREF_LOGISTIC) {
    *loss = (1 - smoothing) * softplus_neg(u);
    if (smoothing != 0) *loss += smoothing * softplus_neg(-u);  // an infinite u stays out of it
    // e / (1 + exp(-u)) - (1 - e) / (1 + exp(u)): a difference from 1 would leave nothing of the slope
    // of a pair that is far on the right side
    const double z = exp(-fabs(u)), near = 1 / (1 + z), far = z / (1 + z);
    *slope = smoothing * (u < 0 ? far : near) - (1 - smoothing) * (u < 0 ? near : far);
  } else if (kind == TISO_PREF_HINGE) {
    *loss = u < 1 ? 1 - u : u >= 1 ? 0.0 : u;  // NaN stays
    *slope = u < 1 ? -1.0 : u >= 1 ? 0.0 : u;
  } else {
    const double d = u - 0.5;
    *loss = d * d / (beta * beta);
    *slope = 2 * d / (beta * beta);
  }
}

// One CTA over the pairs: their losses and rewards, the mean, the tokens' coefficients.
template <typename A>
__global__ void __launch_bounds__(kThreads) pref_pair_kernel(PrefArgs<A> a) {
  __shared__ double shared[32];
  double total = 0;
  for (int64_t i = threadIdx.x; i < a.pairs; i += kThreads) {
    const int64_t j = a.pairs + i;
    double each_i = 1, each_j = 1;
    if (a.average) {
      each_i = 1 / fmax(a.counts[i], 1.0);
      each_j = 1 / fmax(a.counts[j], 1.0);
    }
    const double chosen = a.beta * a.sums[i] * each_i, rejected = a.beta * a.sums[j] * each_j;
    double loss, slope;
    pair_loss(a.kind, chosen - rejected - a.margin, a.smoothing, a.beta, &loss, &slope);
    slope *= a.beta / static_cast<double>(a.pairs);
    total += loss;
    a.rewards[i] = static_cast<A>(chosen);
    a.rewards[j] = static_cast<A>(rejected);
    a.coef[i] = static_cast<A>(slope * each_i);
    a.coef[j] = static_cast<A>(-slope * each_j);
  }
  total = block_sum(total, shared);
  if (threadIdx.x == 0) *a.loss = static_cast<A>(total / static_cast<double>(a.pairs));
}

// A thread takes 4 tokens in a row: the first one's sequence by a binary search (the last k with
// offsets[k] <= t), the others' from there on. Tokens of no sequence and masked ones get 0.
constexpr int kEach = 4;

template <typename A>
__global__ void __launch_bounds__(kThreads)
    pref_grad_kernel(const uint8_t* mask, const int64_t* offsets, int64_t tokens, int64_t sequences,
                     const A* coef, const A* upstream, A* grad, A* grad_ref, bool aligned) {
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kEach;
  if (first >= tokens) return;
  const A up = *upstream;
  int64_t lo = 0, hi = sequences + 1;  // offsets[lo - 1] <= first < offsets[hi], as if -inf and inf
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (offsets[mid] <= first) {
      lo = mid + 1;
    } else {
      hi = mid;
    }
  }
  A g[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int64_t t = first + i;
    g[i] = A(0);
    if (t < tokens) {
      while (lo <= sequences && offsets[lo] <= t) ++lo;
      if (lo > 0 && lo <= sequences && (!mask || mask[t])) g[i] = coef[lo - 1] * up;
    }
  }
  struct alignas(kEach * sizeof(A) < 16 ? kEach * sizeof(A) : 16) Four {
    A x[kEach];
  };
  if (aligned && first + kEach <= tokens) {
    if (grad) *reinterpret_cast<Four*>(grad + first) = Four{{g[0], g[1], g[2], g[3]}};
    if (grad_ref) *reinterpret_cast<Four*>(grad_ref + first) = Four{{-g[0], -g[1], -g[2], -g[3]}};
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (first + i >= tokens) break;
      if (grad) grad[first + i] = g[i];
      if (grad_ref) grad_ref[first + i] = -g[i];
    }
  }
}

int pref_launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess
             ? TISO_OK
             : report_error(TISO_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

template <typename A>
int run_preference(const tiso_preference_args* q, void* loss, void* rewards, void* coef,
                   void* workspace, cudaStream_t st) {
  PrefArgs<A> a{};
  a.logps = static_cast<const A*>(q->logps);
  a.refs = static_cast<const A*>(q->ref_logps);
  a.mask = q->mask;
  a.offsets = q->offsets;
  a.tokens = q->tokens;
  a.pairs = q->pairs;
  a.kind = q->kind;
  a.average = q->average;
  a.beta = q->beta;
  a.smoothing = q->label_smoothing;
  a.margin = q->margin;
  a.sums = static_cast<double*>(workspace);
  a.counts = a.sums + 2 * q->pairs;
  a.loss = static_cast<A*>(loss);
  a.rewards = static_cast<A*>(rewards);
  a.coef = static_cast<A*>(coef);
  // more CTAs, then larger ones, to a sequence while there are few of them and each has over 4096
  // tokens to read (two answers of 670,000 tokens: 1028 us with one CTA of 256 threads each, 102 with
  // 8 of them, 36 with 8 of 1024)
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  int ctas = 1;
  while (ctas < 8 && 2 * q->pairs * ctas < 2 * sms && q->tokens > 2 * q->pairs * ctas * 4096)
    ctas *= 2;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(2 * q->pairs * ctas));
  const bool many = ctas == 8 && q->tokens > 2 * q->pairs * ctas * 4096;
  config.blockDim = dim3(many ? kManyThreads : kThreads);
  config.stream = st;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = static_cast<unsigned>(ctas);
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(
      &config, many ? pref_sum_kernel<A, kManyThreads> : pref_sum_kernel<A, kThreads>, a);
  if (e != cudaSuccess)
    return report_error(TISO_ERR_CUDA,
                        std::string("pref_sum_kernel launch: ") + cudaGetErrorString(e));
  pref_pair_kernel<A><<<1, kThreads, 0, st>>>(a);
  return pref_launched("preference kernels launch");
}

template <typename A>
int run_preference_grad(const tiso_preference_args* q, const void* coef, const void* upstream,
                        void* grad, void* grad_ref, cudaStream_t st) {
  const int64_t ctas = (q->tokens + kThreads * kEach - 1) / (kThreads * kEach);
  const bool aligned =
      ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(grad_ref)) & 15) == 0;
  pref_grad_kernel<A><<<static_cast<unsigned>(ctas), kThreads, 0, st>>>(
      q->mask, q->offsets, q->tokens, 2 * q->pairs, static_cast<const A*>(coef),
      static_cast<const A*>(upstream), static_cast<A*>(grad), static_cast<A*>(grad_ref), aligned);
  return pref_launched("pref_grad_kernel launch");
}

int check_preference(int dtype, const tiso_preference_args* q) {
  if (dtype != TISO_F32 && dtype != TISO_F64)
    return report_error(TISO_ERR_ARGUMENT, "dtype must be TISO_F32 or TISO_F64");
  if (!q) return report_error(TISO_ERR_ARGUMENT, "args is NULL");
  if (q->pairs < 1 || q->pairs > int64_t{1} << 28)
    return report_error(TISO_ERR_ARGUMENT, "pairs must be in [1, 2^28]");
  if (q->tokens < 0 || q->tokens > int64_t{1} << 38)
    return report_error(TISO_ERR_ARGUMENT, "tokens must be in [0, 2^38]");
  if (!q->offsets || (q->tokens && !q->logps))
    return report_error(TISO_ERR_ARGUMENT, "logps and offsets must not be NULL");
  if (q->kind < TISO_PREF_LOGISTIC || q->kind > TISO_PREF_SQUARE)
    return report_error(TISO_ERR_ARGUMENT, "kind must be a tiso_preference_kind");
  if (!(q->beta > 0)) return report_error(TISO_ERR_ARGUMENT, "beta must be > 0");
  if (!(q->label_smoothing >= 0 && q->label_smoothing < 0.5))
    return report_error(TISO_ERR_ARGUMENT, "label_smoothing must be in [0, 0.5)");
  return TISO_OK;
}

}  // namespace
}  // namespace tiso

using namespace tiso;

extern "C" {

int tiso_preference_workspace_size(int64_t pairs, size_t* bytes) {
  return guarded([&]() -> int {
    if (!bytes) return report_error(TISO_ERR_ARGUMENT, "bytes is NULL");
    *bytes = 0;
    if (pairs < 1 || pairs > int64_t{1} << 28)
      return report_error(TISO_ERR_ARGUMENT, "pairs must be in [1, 2^28]");
    *bytes = static_cast<size_t>(pairs) * 4 * sizeof(double);
    return TISO_OK;
  });
}

int tiso_preference(int dtype, const tiso_preference_args* args, void* loss, void* rewards,
                    void* coef, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&]() -> int {
    const int rc = check_preference(dtype, args);
    if (rc) return rc;
    if (!loss || !rewards || !coef)
      return report_error(TISO_ERR_ARGUMENT, "loss, rewards and coef must not be NULL");
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 7) ||
        workspace_bytes < static_cast<size_t>(args->pairs) * 4 * sizeof(double))
      return report_error(TISO_ERR_WORKSPACE, "workspace missing, unaligned or smaller than "
                                              "tiso_preference_workspace_size");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == TISO_F32 ? run_preference<float>(args, loss, rewards, coef, workspace, st)
                             : run_preference<double>(args, loss, rewards, coef, workspace, st);
  });
}

int tiso_preference_grad(int dtype, const tiso_preference_args* args, const void* coef,
                         const void* upstream, void* grad, void* grad_ref, void* stream) {
  return guarded([&]() -> int {
    const int rc = check_preference(dtype, args);
    if (rc) return rc;
    if (!coef || !upstream)
      return report_error(TISO_ERR_ARGUMENT, "coef and upstream must not be NULL");
    if (args->tokens == 0 || (!grad && !grad_ref)) return TISO_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == TISO_F32
               ? run_preference_grad<float>(args, coef, upstream, grad, grad_ref, st)
               : run_preference_grad<double>(args, coef, upstream, grad, grad_ref, st);
  });
}

}  // extern "C"
