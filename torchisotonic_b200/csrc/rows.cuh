// What the operators on rows of logits share (logits.cu, scores.cu, distill.cu): where a row lies and who
// works on it, the softmax parts of threads, warps and CTAs and their joins, the writing of a
// gradient, and the launches.
#pragma once

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

inline int logits_fail(cudaError_t e, const char* what) {
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

// Where the CTA of that rank in the cluster has its copy of a shared value. Called by all threads of a
// CTA, after cluster_started; first: the start has not been waited for yet.
template <typename V>
__device__ __forceinline__ V* of_peer(V* own, int rank, bool first) {
  if (first) wait_for_start();
  return cg::this_cluster().map_shared_rank(own, rank);
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
      const int rank = min(static_cast<int>(threadIdx.x), ctas - 1);
      Part<A>* there = of_peer(&of_cta[cluster.block_rank()], rank, true);
      if (threadIdx.x < ctas) *there = p;
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
template <int kThreads, int kTile, typename T, typename S>
__device__ __forceinline__ void write_target_of_tile(const RowView<T>& r, int tile, int tid,
                                                     const S& slope) {
  const int v = (slope.target - r.head) / RowView<T>::E, in_tile = v - tile;
  if (slope.target >= r.head && in_tile >= 0 && in_tile < kTile && in_tile % kThreads == tid &&
      v < r.vectors)
    r.g[slope.target] = from_acc<T>(slope.at(to_acc(r.x[slope.target]), slope.target));
}

template <typename T, typename S>
__device__ __forceinline__ void write_edge(const RowView<T>& r, int edge, const S& slope) {
  if (edge < r.edges) {
    const int v = r.edge(edge);
    r.g[v] = from_acc<T>(slope.at(to_acc(r.x[v]), v));
  }
}

// The gradient of one tile's vectors. S: Slope, or another gradient with its slope_vector.
template <int kThreads, typename T, typename S>
__device__ __forceinline__ void write_tile(const RowView<T>& r, int tile, int tid,
                                           const S& slope) {
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

// A CTA's tiles of a row that is read twice, for its sum and then in the reverse order: through kStages
// places of shared memory, each thread copying and reading its own vectors there (no barrier). The
// row's last tile may be cut. A row that is read and written at different alignments has none.
constexpr int kStages = 2;

template <int kThreads, typename T>
struct StagedTiles {
  static constexpr int kTile = kBatch * kThreads;
  uint4* stages;  // [kStages][kTile]
  const uint4* from;
  uint4* first;
  int staged, whole, stride, own, tid;
  bool cut;

  // this CTA's j-th tile is tile cta + j ctas
  __device__ __forceinline__ StagedTiles(const RowView<T>& view, const Place<kThreads>& place,
                                         uint4* stages_)
      : stages(stages_), tid(place.tid) {
    staged = view.shift == 0 ? view.vectors : 0;
    const int tiles = (staged + kTile - 1) / kTile;
    const int mine = tiles > place.cta ? (tiles - place.cta + place.ctas - 1) / place.ctas : 0;
    cut = staged % kTile != 0 && (tiles - 1) % place.ctas == place.cta;
    whole = mine - cut;
    stride = place.ctas * kTile;
    own = place.cta * kTile + place.tid;
    from = reinterpret_cast<const uint4*>(view.x + view.head) + own;
    first = reinterpret_cast<uint4*>(view.g + view.head) + own;
  }
  __device__ __forceinline__ int tile(int j) const { return own - tid + j * stride; }
  __device__ __forceinline__ uint4* to(int j) const {
    return first + static_cast<int64_t>(j) * stride;
  }
  // whether this thread has an i-th vector in the cut tile
  __device__ __forceinline__ bool has(int i) const {
    return own + whole * stride + i * kThreads < staged;
  }
  __device__ __forceinline__ void copy(int j) const {
    uint4* at = this->at(j);
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
  }
  // waits for the tile that is read next: kStages - 1 groups were closed after its own
  __device__ __forceinline__ void arrived() const { wait_groups<kStages - 1>(); }
  // this thread's vectors of tile j in shared memory, kThreads apart
  __device__ __forceinline__ uint4* at(int j) const {
    return stages + static_cast<unsigned>(j) % kStages * kTile + tid;
  }
  __device__ __forceinline__ void read(int j, uint4 (&q)[kBatch]) const {
#pragma unroll
    for (int i = 0; i < kBatch; ++i)  // (from at(j) the policy's kernel needs a register more, and spills)
      q[i] = stages[static_cast<unsigned>(j) % kStages * kTile + i * kThreads + tid];
  }
  __device__ __forceinline__ void read_cut(uint4 (&q)[kBatch]) const {
    read(whole, q);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (!has(i)) q[i] = no_vector<T>();
  }
  __device__ __forceinline__ void fetch(int j, uint4 (&q)[kBatch]) const {
    arrived();
    read(j, q);
  }
};

// A row that is left out (its target is the ignored index, or its weight is 0) is marked by a
// negative sum in stats: its gradient is zeros and its logits are not read.
constexpr int kLeftOut = -1;

// ---------------------------------------------------------------------------------------------
// Weighted means over a batch's tokens: the sum of the weights ahead of the rows, the means by the
// CTA of the last row

enum WeightKind { kNoWeight = 0, kByteWeight = 1, kAccWeight = 2 };

// How much a token counts: its weight, or nothing where its mark is the ignored one.
template <typename A>
struct TokenWeights {
  const int64_t* marks;
  int64_t stride, ignore;
  const void* weight;
  int kind;

  __device__ __forceinline__ A at(int64_t r) const { return of(marks[r * stride], r); }
  // (token r's mark may still be on its way: both loads are in flight together)
  __device__ __forceinline__ A of(int64_t mark, int64_t r) const {
    A w = A(1);
    if (kind == kByteWeight) {
      w = static_cast<const uint8_t*>(weight)[r] ? A(1) : A(0);
    } else if (kind == kAccWeight) {
      w = static_cast<const A*>(weight)[r];
    }
    return mark == ignore ? A(0) : w;
  }
};

// The sum of the weights, by a CTA, or a cluster of them where there are many rows, ahead of the
// rows. The rows' kernel starts meanwhile (a programmatic launch): what it needs of this one it reads
// after waiting for it. Without rows the means are 0.
constexpr int kTotalThreads = 1024, kTotalCtas = 8;

template <typename A>
__global__ void __launch_bounds__(kTotalThreads)
    weights_total_kernel(TokenWeights<A> weights, int64_t rows, double* total, unsigned* done, A* out,
                         int means) {
  cudaTriggerProgrammaticLaunchCompletion();
  constexpr int kAhead = 4;
  __shared__ double shared[32], sums[kTotalCtas];
  auto cluster = cg::this_cluster();
  cluster_started(gridDim.x);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTotalThreads;
  double sum = 0;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kTotalThreads + threadIdx.x; r < rows;
       r += kAhead * step) {
    A w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) w[i] = r + i * step < rows ? weights.at(r + i * step) : A(0);
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
    *total = sum;
    *done = 0;
    for (int i = 0; i < means && rows == 0; ++i) out[i] = A(0);
  }
}

// Called by one thread of each unit (a row, or a CTA's rows) once its results are written: whether it
// was the last of them.
__device__ __forceinline__ bool last_unit(unsigned* done, int64_t units) {
  __threadfence();
  return atomicAdd(done, 1u) == static_cast<unsigned>(units - 1);
}

// The means over the tokens by the CTA of the last unit, from kMeans terms of each unit: in a fixed
// order whichever it is; 0 when the weights sum to 0.
template <int kMeans, typename A>
__device__ void write_means(const A* terms, double total, A* out, int64_t units) {
  constexpr int kAhead = 4;
  __shared__ double shared[32];
  __threadfence();
  double s[kMeans] = {};
  const int64_t step = blockDim.x;
  for (int64_t u = threadIdx.x; u < units; u += kAhead * step) {
    A q[kAhead][kMeans];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int j = 0; j < kMeans; ++j)
        q[i][j] = u + i * step < units ? __ldcg(terms + kMeans * (u + i * step) + j) : A(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int j = 0; j < kMeans; ++j) s[j] += static_cast<double>(q[i][j]);
  }
#pragma unroll
  for (int j = 0; j < kMeans; ++j) {
    const double v = block_sum(s[j], shared);
    if (threadIdx.x == 0) out[j] = total == 0 ? A(0) : static_cast<A>(v / total);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side

// grad: NULL, or the gradient that the call writes
inline int check_rows(int dtype, const tiso_rows* x, const int64_t* targets, const void* grad,
                      bool needs_targets = true) {
  if (dtype < TISO_F16 || dtype > TISO_F64)
    return report_error(TISO_ERR_ARGUMENT, "dtype must be a tiso_dtype");
  if (!x) return report_error(TISO_ERR_ARGUMENT, "rows is NULL");
  if (x->rows < 0 || x->vocab < 1 || x->inner < 1)
    return report_error(TISO_ERR_ARGUMENT, "need rows >= 0, vocab >= 1 and inner >= 1");
  if (x->outer_stride < 0 || x->inner_stride < 0)
    return report_error(TISO_ERR_ARGUMENT, "strides must not be negative");
  if (x->rows > kMostRows || x->vocab > int64_t{1} << 30)
    return report_error(TISO_ERR_ARGUMENT, "more than 2^28 rows or a vocabulary of more than 2^30");
  if (x->rows && (!x->data || (needs_targets && !targets)))
    return report_error(TISO_ERR_ARGUMENT, "logits and targets must not be NULL");
  const int size = dtype == TISO_F64 ? 8 : dtype == TISO_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x->data) | reinterpret_cast<uintptr_t>(grad)) % size)
    return report_error(TISO_ERR_ARGUMENT, "logits and grad must be aligned to their elements");
  return TISO_OK;
}

inline Rows rows_of(const tiso_rows* x, const int64_t* targets, int64_t ignore) {
  return {x->data,         x->rows,          x->inner,
          x->outer_stride, x->inner_stride,  static_cast<int>(x->vocab),
          targets,         ignore};
}

// log2(e) / t for the exponentials in float, 1 / t for those in double
inline float exp_factor(float, double inv_temp) {
  return static_cast<float>(inv_temp * 1.4426950408889634);
}
inline double exp_factor(double, double inv_temp) { return inv_temp; }

inline int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TISO_OK : logits_fail(e, what);
}

inline int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess)
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

// Allows a kernel more than 48 KB of dynamic shared memory: once per kernel and device.
inline int allow_shared(const void* kernel, size_t bytes) {
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

template <typename A>
TokenWeights<A> weights_of(const int64_t* marks, int64_t stride, int64_t ignore, const void* weight,
                           int weight_is_byte) {
  return {marks, stride, ignore, weight,
          !weight ? kNoWeight : weight_is_byte ? kByteWeight : kAccWeight};
}

// `alone`: up to so many rows by one CTA (8192 rows: 7 us)
template <typename A>
int launch_total(const TokenWeights<A>& weights, int64_t rows, int64_t alone, double* total,
                 unsigned* done, A* out, int means, cudaStream_t st) {
  return launch_clusters(weights_total_kernel<A>, 1, rows > alone ? kTotalCtas : 1, kTotalThreads, 0,
                         false, st, "weights_total_kernel launch", weights, rows, total, done, out,
                         means);
}

// Rows of at most kWarpVectors vectors go to a warp each; of up to `most` of them where there are
// enough rows to fill the GPU with warps. A CTA's start and join cost as much as some 1000 vectors:
// 97656 x 4096 bf16, log-probabilities 126 us by warps and 342 by CTAs of 256 threads, their gradient
// 272 and 358, the policy loss 380 and 779; 976 x 8192: 11.2 and 10.2 us.
constexpr int kWarpVectors = 256;

inline bool by_warps(int64_t rows, int64_t vectors, int64_t most, int sms) {
  return vectors <= kWarpVectors || (vectors <= most && rows >= int64_t{16} * sms);
}

// Bytes of rows in work at once that L2 is to hold from a row's first read to its
// second. Rows of 256 KB: one CTA to a row (116 MB) reads 1.8 GB where two (58 MB) read 1.06 and
// four 0.95 (0.94 is each byte once); two are fastest (828, 874 and 931 us with 2, 1 and 4).
constexpr int64_t kRowsInL2 = 80 << 20;

// CTAs of `threads` to a row: doubled while rows are too few to fill the GPU and a CTA would have
// more than a batch for each thread.
inline int ctas_for(int64_t rows, int64_t vectors, int threads, int sms) {
  int ctas = 1;
  while (ctas < 8 && rows * ctas < 2 * sms && vectors > int64_t{ctas} * threads * kBatch) ctas *= 2;
  return ctas;
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
