// Operators on rows of logits (include/tiso.h: tiso_logprobs*, tiso_policy*): the log-probability
// of one token per row and its gradient, and the clipped policy loss with its gradient.
#include <cuda_runtime.h>

#include <string>

#include "../../include/tiso.h"
#include "logits.cuh"

namespace tiso {

int report_error(int code, const std::string& msg);

namespace {

constexpr int kThreads = 512;

int logits_fail(cudaError_t e, const char* what) {
  return report_error(TISO_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// Rows of logits: row r starts at x + (r / inner) * outer_stride + (r % inner) * inner_stride.
struct Rows {
  const void* x;
  int64_t rows, inner, outer_stride, inner_stride, vocab;
  const int64_t* targets;
  int64_t ignore;
};

template <typename T>
__device__ __forceinline__ const T* row_at(const Rows& a, int64_t r) {
  return static_cast<const T*>(a.x) + (r / a.inner) * a.outer_stride +
         (r % a.inner) * a.inner_stride;
}

// The maximum and sum of a row, by all threads of the CTA; every thread gets them.
template <typename T, typename A>
__device__ Part<A> row_part(const T* x, int64_t vocab, A k) {
  __shared__ Part<A> warp_part[kThreads / 32];
  Part<A> p{lowest<A>(), A(0)};
  for (int64_t v = threadIdx.x; v < vocab; v += kThreads) {
    const A z = to_acc(x[v]);
    const A m = max_acc(p.m, z);
    const A base = base_of(m);
    p.s = p.s * scaled_exp(p.m == m ? A(0) : p.m - base, k) + scaled_exp(z - base, k);
    p.m = m;
  }
  p = join_warp(p, k);
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = p;
  __syncthreads();
  p = warp_part[0];
  for (int i = 1; i < kThreads / 32; ++i) p = join(p, warp_part[i], k);
  __syncthreads();
  return p;
}

// log softmax(x / t) at the target. The steps after the sum are in double: in float, rounding
// x - m - log s near 10 would cost more than the whole sum did.
template <typename T, typename A>
__device__ __forceinline__ double logp_of(const T* x, int64_t vocab, int64_t target, const Part<A>& p,
                                     double inv_temp) {
  if (target < 0 || target >= vocab) return nan_of(0.0);
  const double m = base_of(p.m);
  return (static_cast<double>(to_acc(x[target])) - m) * inv_temp - log(static_cast<double>(p.s));
}

// d/dx of c * logp(x / t): c / t (1[v = target] - softmax), c already divided by t. An index out
// of range gives NaN throughout.
template <typename T, typename A>
__device__ void write_grad(const T* x, T* g, int64_t vocab, int64_t target, A base, A s, A c, A k) {
  const A scale = target < 0 || target >= vocab ? nan_of(A(0)) : -c / s;
  for (int64_t v = threadIdx.x; v < vocab; v += kThreads) {
    A d = scaled_exp(to_acc(x[v]) - base, k) * scale;
    if (v == target) d += c;
    g[v] = from_acc<T>(d);
  }
}

template <typename T>
__device__ void write_zeros(T* g, int64_t vocab) {
  for (int64_t v = threadIdx.x; v < vocab; v += kThreads)
    g[v] = from_acc<T>(typename AccOf<T>::type(0));
}

// A row that is left out (its target is the ignored index, or its weight is 0) is marked by a
// negative sum in stats: its gradient is zeros and its logits are not read.
constexpr int kLeftOut = -1;

template <typename T, typename A>
__global__ void __launch_bounds__(kThreads)
    logprobs_kernel(Rows a, double inv_temp, A k, A* logps, A* stats) {
  const int64_t r = blockIdx.x;
  const int64_t target = a.targets[r];
  if (target == a.ignore) {
    if (threadIdx.x == 0) {
      logps[r] = A(0);
      if (stats) stats[2 * r + 1] = A(kLeftOut);
    }
    return;
  }
  const T* x = row_at<T>(a, r);
  const Part<A> p = row_part(x, a.vocab, k);
  if (threadIdx.x == 0) {
    logps[r] = static_cast<A>(logp_of(x, a.vocab, target, p, inv_temp));
    if (stats) {
      stats[2 * r] = base_of(p.m);
      stats[2 * r + 1] = p.s;
    }
  }
}

// coef: per row, d loss / d logp. upstream (may be NULL): a scalar that multiplies it, and where
// it is 1 nothing is written.
template <typename T, typename A>
__global__ void __launch_bounds__(kThreads)
    logprobs_grad_kernel(Rows a, double inv_temp, A k, const A* stats, const A* coef,
                         const A* upstream, T* grad) {
  const A up = upstream ? *upstream : A(1);
  if (upstream && up == A(1)) return;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    T* g = grad + r * a.vocab;
    const A sum = stats[2 * r + 1];
    if (sum < A(0)) {
      write_zeros(g, a.vocab);
    } else {
      write_grad(row_at<T>(a, r), g, a.vocab, a.targets[r], stats[2 * r], sum,
                 static_cast<A>(coef[r] * up * inv_temp), k);
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
  A* coef;            // per row, d loss / d logp
  A* stats;           // per row, maximum and sum
  A* terms;           // per row, w loss, w kl and w [clipped]
  A* out;             // loss, kl, clip fraction
  double* total;      // sum of the weights
};

template <typename A>
__device__ __forceinline__ A weight_of(const Rows& a, const PolicyArgs<A>& p, int64_t r) {
  if (a.targets[r] == a.ignore) return A(0);
  if (p.weight_kind == kNoWeight) return A(1);
  if (p.weight_kind == kByteWeight)
    return static_cast<const uint8_t*>(p.weight)[r] ? A(1) : A(0);
  return static_cast<const A*>(p.weight)[r];
}

// The sum of v over the CTA in a fixed order (thread 0 has it).
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

template <typename A>
__global__ void __launch_bounds__(1024) policy_total_kernel(Rows a, PolicyArgs<A> p) {
  __shared__ double shared[32];
  double sum = 0;
  for (int64_t r = threadIdx.x; r < a.rows; r += blockDim.x)
    sum += static_cast<double>(weight_of(a, p, r));
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) *p.total = sum;
}

// The loss of one token and its slope d loss / d logp (both without the token's weight):
//   rho = exp(logp - old);  loss = -min(rho A, clip(rho) A) + kl_coef kl,
//   kl = exp(d) - d - 1, d = ref - logp;
//   slope = -rho A where rho A <= clip(rho) A, else 0, plus kl_coef (1 - exp(d)).
// In double: one thread a row does it, and the ratio's exponent is a difference of numbers
// near 10 whose float rounding would be the largest error of the loss.
template <typename A>
__device__ void policy_token(const PolicyArgs<A>& p, int64_t r, double lp, double* loss,
                             double* slope, double* kl, bool* clipped) {
  const double adv = p.advantages[r];
  const double ratio = exp(lp - static_cast<double>(p.old_logps[r]));
  const double held = (ratio < p.lo ? p.lo : ratio > p.hi ? p.hi : ratio) * adv;
  const double free_side = ratio * adv;
  *clipped = free_side > held;
  *loss = -(free_side > held ? held : free_side);
  *slope = free_side > held ? 0.0 : -free_side;
  *kl = 0;
  if (p.ref_logps) {
    const double d = static_cast<double>(p.ref_logps[r]) - lp;
    const double e = expm1(d);
    *kl = e - d;
    *loss += p.kl_coef * *kl;
    *slope -= p.kl_coef * e;
  }
}

template <typename T, typename A>
__global__ void __launch_bounds__(kThreads)
    policy_kernel(Rows a, PolicyArgs<A> p, double inv_temp, A k, T* grad) {
  __shared__ A shared_coef;
  const int64_t r = blockIdx.x;
  T* g = grad + r * a.vocab;
  const A w = weight_of(a, p, r);
  if (w == A(0)) {
    if (threadIdx.x == 0) {
      p.logps[r] = p.coef[r] = A(0);
      p.stats[2 * r + 1] = A(kLeftOut);
      p.terms[3 * r] = p.terms[3 * r + 1] = p.terms[3 * r + 2] = A(0);
    }
    if (grad) write_zeros(g, a.vocab);
    return;
  }
  const T* x = row_at<T>(a, r);
  const Part<A> part = row_part(x, a.vocab, k);
  const int64_t target = a.targets[r];
  if (threadIdx.x == 0) {
    const double lp = logp_of(x, a.vocab, target, part, inv_temp);
    double loss, slope, kl;
    bool clipped;
    policy_token(p, r, lp, &loss, &slope, &kl, &clipped);
    const double total = *p.total;
    const A coef = total == 0 ? A(0) : static_cast<A>(w * slope / total);
    p.logps[r] = static_cast<A>(lp);
    p.coef[r] = shared_coef = coef;
    p.stats[2 * r] = base_of(part.m);
    p.stats[2 * r + 1] = part.s;
    p.terms[3 * r] = static_cast<A>(w * loss);
    p.terms[3 * r + 1] = static_cast<A>(w * kl);
    p.terms[3 * r + 2] = clipped ? w : A(0);
  }
  if (!grad) return;
  __syncthreads();
  write_grad(x, g, a.vocab, target, base_of(part.m), part.s,
             static_cast<A>(shared_coef * inv_temp), k);
}

// The means over the tokens, in a fixed order; 0 when the weights sum to 0.
template <typename A>
__global__ void __launch_bounds__(1024) policy_means_kernel(int64_t rows, PolicyArgs<A> p) {
  __shared__ double shared[32];
  double s[3] = {0, 0, 0};
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x)
    for (int j = 0; j < 3; ++j) s[j] += static_cast<double>(p.terms[3 * r + j]);
  const double total = *p.total;
  for (int j = 0; j < 3; ++j) {
    const double v = block_sum(s[j], shared);
    if (threadIdx.x == 0) p.out[j] = total == 0 ? A(0) : static_cast<A>(v / total);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side

int check_rows(int dtype, const tiso_rows* x, const int64_t* targets) {
  if (dtype < TISO_F16 || dtype > TISO_F64)
    return report_error(TISO_ERR_ARGUMENT, "dtype must be a tiso_dtype");
  if (!x) return report_error(TISO_ERR_ARGUMENT, "rows is NULL");
  if (x->rows < 0 || x->vocab < 1 || x->inner < 1)
    return report_error(TISO_ERR_ARGUMENT, "need rows >= 0, vocab >= 1 and inner >= 1");
  if (x->outer_stride < 0 || x->inner_stride < 0)
    return report_error(TISO_ERR_ARGUMENT, "strides must not be negative");
  if (x->rows > int64_t{2147483647})
    return report_error(TISO_ERR_ARGUMENT, "more than 2^31 - 1 rows");
  if (x->rows && (!x->data || !targets))
    return report_error(TISO_ERR_ARGUMENT, "logits and targets must not be NULL");
  return TISO_OK;
}

Rows rows_of(const tiso_rows* x, const int64_t* targets, int64_t ignore) {
  return {x->data, x->rows, x->inner, x->outer_stride, x->inner_stride, x->vocab, targets, ignore};
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

template <typename T>
int run_logprobs(const Rows& a, double inv_temp, void* logps, void* stats, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  logprobs_kernel<T, A><<<static_cast<unsigned>(a.rows), kThreads, 0, st>>>(
      a, inv_temp, exp_factor(A(0), inv_temp), static_cast<A*>(logps), static_cast<A*>(stats));
  return launched("logprobs_kernel launch");
}

int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

template <typename T>
int run_logprobs_grad(const Rows& a, double inv_temp, const void* stats, const void* coef,
                      const void* upstream, void* grad, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int64_t most = int64_t{sm_count()} * 4;
  logprobs_grad_kernel<T, A><<<static_cast<unsigned>(a.rows < most ? a.rows : most), kThreads, 0,
                               st>>>(a, inv_temp, exp_factor(A(0), inv_temp),
                                     static_cast<const A*>(stats), static_cast<const A*>(coef),
                                     static_cast<const A*>(upstream), static_cast<T*>(grad));
  return launched("logprobs_grad_kernel launch");
}

template <typename T>
int run_policy(const Rows& a, const tiso_policy_args* q, double inv_temp, void* logps, void* coef,
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
  p.coef = static_cast<A*>(coef);
  p.stats = static_cast<A*>(stats);
  p.out = static_cast<A*>(out);
  p.total = static_cast<double*>(workspace);
  p.terms = reinterpret_cast<A*>(p.total + 1);
  policy_total_kernel<A><<<1, 1024, 0, st>>>(a, p);
  if (a.rows > 0)
    policy_kernel<T, A><<<static_cast<unsigned>(a.rows), kThreads, 0, st>>>(
        a, p, inv_temp, exp_factor(A(0), inv_temp), static_cast<T*>(grad));
  policy_means_kernel<A><<<1, 1024, 0, st>>>(a.rows, p);
  return launched("policy kernels launch");
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
  const int rc = check_rows(dtype, x, targets);
  if (rc) return rc;
  if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
  if (x->rows == 0) return TISO_OK;
  if (!logps) return report_error(TISO_ERR_ARGUMENT, "logps must not be NULL");
  const Rows a = rows_of(x, targets, ignore_index);
  return by_type(dtype, [&](auto t) {
    return run_logprobs<decltype(t)>(a, 1.0 / temperature, logps, stats,
                                     static_cast<cudaStream_t>(stream));
  });
}

int tiso_logprobs_grad(int dtype, const tiso_rows* x, const int64_t* targets, double temperature,
                       const void* stats, const void* coef, const void* upstream, void* grad,
                       void* stream) {
  const int rc = check_rows(dtype, x, targets);
  if (rc) return rc;
  if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
  if (x->rows == 0) return TISO_OK;
  if (!stats || !coef || !grad)
    return report_error(TISO_ERR_ARGUMENT, "stats, coef and grad must not be NULL");
  const Rows a = rows_of(x, targets, 0);
  return by_type(dtype, [&](auto t) {
    return run_logprobs_grad<decltype(t)>(a, 1.0 / temperature, stats, coef, upstream, grad,
                                          static_cast<cudaStream_t>(stream));
  });
}

int tiso_policy_workspace_size(int dtype, int64_t rows, size_t* bytes) {
  if (!bytes) return report_error(TISO_ERR_ARGUMENT, "bytes is NULL");
  *bytes = 0;
  if (dtype < TISO_F16 || dtype > TISO_F64)
    return report_error(TISO_ERR_ARGUMENT, "dtype must be a tiso_dtype");
  if (rows < 0) return report_error(TISO_ERR_ARGUMENT, "need rows >= 0");
  *bytes = 8 + static_cast<size_t>(rows) * 3 * (dtype == TISO_F64 ? 8 : 4);
  return TISO_OK;
}

int tiso_policy(int dtype, const tiso_rows* x, const int64_t* targets, int64_t ignore_index,
                double temperature, const tiso_policy_args* args, void* logps, void* coef,
                void* stats, void* out, void* grad, void* workspace, size_t workspace_bytes,
                void* stream) {
  int rc = check_rows(dtype, x, targets);
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
}

}  // extern "C"
