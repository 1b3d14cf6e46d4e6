// The preference loss (include/tiso.h: tiso_preference*): paired log ratios of packed sequences
// of token log-probabilities, forward and backward.
//
// With sequences 0..P-1 the chosen and P..2P-1 the rejected answers,
//   s_k = sum over the sequence's unmasked tokens of (logp - ref)  (their mean with `average`),
//   u_i = beta (s_i - s_{P+i}) - margin,  loss = mean of l(u_i),
//   d loss / d logp_t = +-beta l'(u) / P (1 / count with `average`), + for chosen.
// Sums are double, in a fixed order.
#include <cuda_runtime.h>

#include <string>

#include "entry.cuh"

namespace tiso {

namespace {

constexpr int kThreads = 256;

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

__device__ double block_sum(double v, double* shared) {
  for (int d = 16; d; d >>= 1) v += __shfl_down_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < blockDim.x / 32 ? shared[threadIdx.x] : 0.0;
  if (threadIdx.x < 32)
    for (int d = 16; d; d >>= 1) v += __shfl_down_sync(0xffffffffu, v, d);
  __syncthreads();
  return v;
}

// A CTA per sequence: the sum and number of its unmasked tokens. A masked token is not used in
// any way (its value may be NaN).
template <typename A>
__global__ void __launch_bounds__(kThreads) pref_sum_kernel(PrefArgs<A> a) {
  __shared__ double shared[32];
  const int64_t k = blockIdx.x;
  const int64_t begin = cut(a.offsets[k], 0, a.tokens);
  const int64_t end = cut(a.offsets[k + 1], begin, a.tokens);
  double sum = 0, count = 0;
  for (int64_t t = begin + threadIdx.x; t < end; t += kThreads) {
    if (a.mask && !a.mask[t]) continue;
    sum += static_cast<double>(a.logps[t]) - (a.refs ? static_cast<double>(a.refs[t]) : 0.0);
    count += 1;
  }
  sum = block_sum(sum, shared);
  count = block_sum(count, shared);
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
    *slope = 1 / (1 + exp(-u)) - (1 - smoothing);
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

// A token's sequence by a binary search: the last k with offsets[k] <= t. Tokens of no sequence
// and masked ones get 0.
template <typename A>
__global__ void __launch_bounds__(kThreads)
    pref_grad_kernel(const uint8_t* mask, const int64_t* offsets, int64_t tokens, int64_t sequences,
                     const A* coef, const A* upstream, A* grad, A* grad_ref) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (t >= tokens) return;
  int64_t lo = 0, hi = sequences + 1;  // offsets[lo - 1] <= t < offsets[hi], as if -inf and inf
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (offsets[mid] <= t) {
      lo = mid + 1;
    } else {
      hi = mid;
    }
  }
  const int64_t k = lo - 1;
  A g = A(0);
  if (k >= 0 && k < sequences && (!mask || mask[t])) g = coef[k] * *upstream;
  if (grad) grad[t] = g;
  if (grad_ref) grad_ref[t] = -g;
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
  pref_sum_kernel<A><<<static_cast<unsigned>(2 * q->pairs), kThreads, 0, st>>>(a);
  pref_pair_kernel<A><<<1, kThreads, 0, st>>>(a);
  return pref_launched("preference kernels launch");
}

template <typename A>
int run_preference_grad(const tiso_preference_args* q, const void* coef, const void* upstream,
                        void* grad, void* grad_ref, cudaStream_t st) {
  pref_grad_kernel<A><<<static_cast<unsigned>((q->tokens + kThreads - 1) / kThreads), kThreads, 0,
                        st>>>(q->mask, q->offsets, q->tokens, 2 * q->pairs,
                              static_cast<const A*>(coef), static_cast<const A*>(upstream),
                              static_cast<A*>(grad), static_cast<A*>(grad_ref));
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
