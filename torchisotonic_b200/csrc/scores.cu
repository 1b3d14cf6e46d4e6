// A token's scores from rows of logits (include/tiso.h: tiso_scores*): the log-probability of a given
// token, the entropy and the top alternatives, in one pass over the logits; and the gradient of the
// first two.
//
// With z = (x - m) / t, m the row's maximum, s = sum exp(z) and u = sum exp(z) z:
//   log p_v = z_v - log s,  entropy = log s - u / s,
// neither a difference of large numbers (s >= 1, u <= 0). Parts of a row join as for s alone: with
// d = (m1 - M) / t, s1 and u1 become s1 exp(d) and exp(d) (u1 + d s1).
//
// Top alternatives: the row's body is cut into groups of neighbouring vectors, whose maxima the pass
// leaves in shared memory. The k best groups (equal maxima: the first) hold the k largest elements,
// for each of the others has an element in each of these before it. Those groups are read again and
// their elements, all at least the k-th maximum, are ranked.
#include "rows.cuh"
#include "select.cuh"

namespace tiso {
namespace {

constexpr int kMostTop = 128;
constexpr size_t kSharedForTop = 160 * 1024;

// What a thread has seen of a row; u in the exponent's unit (log 2 in float, 1 in double).
template <typename A>
struct Scored {
  A m, s, u;
};

__device__ __forceinline__ double unit_of(float) { return 0.6931471805599453; }
__device__ __forceinline__ double unit_of(double) { return 1.0; }

// Arguments of exponentials are raised to at least this, whose exponential is 0: an element of
// -infinity then adds 0 times a number.
__device__ __forceinline__ float least_argument(float) { return -300.0f; }
__device__ __forceinline__ double least_argument(double) { return -2000.0; }
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return a != a || a > b ? a : b; }
__device__ __forceinline__ float exp_of(float a) { return exp2_of(a); }
__device__ __forceinline__ double exp_of(double a) { return exp(a); }

// (x - base) k of a vector's elements, in place.
template <int kE>
__device__ __forceinline__ void arguments(float (&x)[kE], float base, float k) {
  const Pair minus = pair_of(-base, -base), factor = pair_of(k, k);
#pragma unroll
  for (int j = 0; j < kE; j += 2) {
    split(mul2(add2(pair_of(x[j], x[j + 1]), minus), factor), x[j], x[j + 1]);
    x[j] = max_nan(x[j], least_argument(base));
    x[j + 1] = max_nan(x[j + 1], least_argument(base));
  }
}
template <int kE>
__device__ __forceinline__ void arguments(double (&x)[kE], double base, double k) {
#pragma unroll
  for (int j = 0; j < kE; ++j) x[j] = max_nan(mul_rn(x[j] - base, k), least_argument(base));
}

// Adds the exponentials of a vector's arguments, and their products with them.
template <int kE>
__device__ __forceinline__ void add_scores(const float (&a)[kE], float& s, float& u) {
  Pair sum = 0, weighted = 0;
#pragma unroll
  for (int j = 0; j < kE; j += 2) {
    const Pair e = pair_of(exp_of(a[j]), exp_of(a[j + 1]));
    sum = j ? add2(sum, e) : e;
    weighted = j ? fma2(e, pair_of(a[j], a[j + 1]), weighted) : mul2(e, pair_of(a[j], a[j + 1]));
  }
  float p, q;
  split(sum, p, q);
  s += p + q;
  split(weighted, p, q);
  u += p + q;
}
template <int kE>
__device__ __forceinline__ void add_scores(const double (&a)[kE], double& s, double& u) {
#pragma unroll
  for (int j = 0; j < kE; ++j) {
    const double e = exp_of(a[j]);
    s += e;
    u += e * a[j];
  }
}

// Takes a part's exponentials from another base, M >= p.m.
template <typename A>
__device__ __forceinline__ void move_base(Scored<A>& p, A m, A k) {
  const A d = p.m == m ? A(0) : max_nan(mul_rn(p.m - base_of(m), k), least_argument(k));
  const A f = exp_of(d);
  p.u = f * (p.u + d * p.s);
  p.s *= f;
  p.m = m;
}

template <int kLanes, typename A>
__device__ __forceinline__ Scored<A> join_scores(Scored<A> p, A k) {
  move_base(p, max_of_lanes<kLanes>(p.m), k);
#pragma unroll
  for (int d = kLanes / 2; d; d >>= 1) {
    p.s = add_rn(p.s, __shfl_xor_sync(0xffffffffu, p.s, d));
    p.u = add_rn(p.u, __shfl_xor_sync(0xffffffffu, p.u, d));
  }
  return p;
}

// As join_warps of rows.cuh.
template <int kThreads, typename A>
__device__ __forceinline__ Scored<A> join_scores_of_warps(Scored<A> p, A k) {
  if constexpr (kThreads > 32) {
    constexpr int kWarps = kThreads / 32, kMostCtas = 8;
    __shared__ Scored<A> of_warp[kWarps], of_cta[kMostCtas];
    const int lane = threadIdx.x & 31;
    if (lane == 0) of_warp[threadIdx.x >> 5] = p;
    __syncthreads();
    p = join_scores<kWarps>(of_warp[lane % kWarps], k);
    auto cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks());
    if (ctas > 1) {
      const int rank = min(static_cast<int>(threadIdx.x), ctas - 1);
      Scored<A>* there = of_peer(&of_cta[cluster.block_rank()], rank, true);
      if (threadIdx.x < ctas) *there = p;
      cluster.sync();
      p = {lowest<A>(), A(0), A(0)};
      if (lane % kMostCtas < ctas) p = of_cta[lane % kMostCtas];
      p = join_scores<kMostCtas>(p, k);
    }
  }
  return p;
}

// ---------------------------------------------------------------------------------------------
// Top alternatives

// A row's element; the larger one, of equal ones the first, is before the other.
template <typename A>
struct Element {
  A value;
  int at;
  __device__ __forceinline__ bool before(const Element& o) const {
    return value > o.value || (value == o.value && at < o.at);
  }
};

// Shared memory of the threads that work on a row (a cluster's CTAs have one each).
template <typename A>
struct TopSpace {
  Element<A>* candidates;  // 8 top + 32
  Element<A>* best;        // top; of the first CTA of a cluster top for each CTA
  A* maxima;               // of the groups; 32 top at least
  int* picked;             // top
  unsigned* histogram;
  int* count;              // 2

  static size_t bytes(int top, int groups, int ctas) {
    const size_t numbers = groups > 32 * top ? groups : 32 * top;
    return sizeof(Element<A>) * (8 * top + 32 + static_cast<size_t>(top) * ctas) +
           sizeof(A) * ((numbers + 3) / 4 * 4) + sizeof(int) * ((top + 3) / 4 * 4 + kHistogram + 4);
  }

  __device__ TopSpace(void* at, int top, int groups, int ctas) {
    const int numbers = max(groups, 32 * top);
    candidates = static_cast<Element<A>*>(at);
    best = candidates + 8 * top + 32;
    maxima = reinterpret_cast<A*>(best + top * ctas);
    histogram = reinterpret_cast<unsigned*>(maxima + (numbers + 3) / 4 * 4);
    picked = reinterpret_cast<int*>(histogram + kHistogram);
    count = picked + (top + 3) / 4 * 4;
  }
};

// How a CTA's share of a row's vectors is numbered: local vector l, ascending with the vectors.
template <int kThreads>
struct Share {
  int cta, ctas;
  __device__ __forceinline__ int vector(int l) const {
    constexpr int kTile = kBatch * kThreads;
    return (l / kTile * ctas + cta) * kTile + l % kTile;
  }
};

template <typename A>
__device__ __forceinline__ A number_of(A x) {  // NaN in the order of -infinity
  return x == x ? x : lowest<A>();
}

// The row's `top` best elements of this CTA's share to space.best, in order; elements that are not
// there (a share of fewer) stand at the end, at an impossible place. kGroup: vectors to a maximum (32
// or 1), `groups` of them. The maxima are written and the threads have met.
template <int kGroup, int kThreads, typename T, typename A>
__device__ __forceinline__ void choose_top(const RowView<T>& r, const Place<kThreads>& place, int top,
                                           int groups, const TopSpace<A>& space) {
  constexpr int E = RowView<T>::E;
  const Team<kThreads> team{place.tid};
  const Share<kThreads> share{place.cta, place.ctas};
  const int room = 8 * top;
  Cut<A> cut{0, 0xffffffffu};
  if (team.tid < 2) space.count[team.tid] = 0;
  if (groups > top)
    cut = find_cut<2, kThreads, A>(
        team, groups, top, [&](int i) { return ordered(space.maxima[i]); },
        [](int i) { return static_cast<uint32_t>(i); }, space.histogram);
  team.sync();
  for (int i = team.tid; i < groups; i += kThreads)
    if (cut.takes(ordered(space.maxima[i]), static_cast<uint32_t>(i)))
      space.picked[atomicAdd(space.count + 1, 1)] = i;
  team.sync();
  const int picked = space.count[1];
  const auto add = [&](int v, KeyOf<A> least) {  // a vector's elements from `least` on
    A x[E];
    unpack<T>(load_vector(r, v), x);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      x[j] = number_of(x[j]);
      if (ordered(x[j]) >= least) {
        const int slot = atomicAdd(space.count, 1);
        if (slot < room) space.candidates[slot] = {x[j], r.element(v) + j};
      }
    }
  };
  for (int i = team.tid; i < picked * kGroup; i += kThreads) {
    const int v = share.vector(space.picked[i / kGroup] * kGroup + i % kGroup);
    if (v < r.vectors) add(v, cut.key);
  }
  team.sync();
  if (kGroup > 1 && space.count[0] > room) {
    // more than 8 elements each: the best vectors of these groups first
    for (int i = team.tid; i < picked * kGroup; i += kThreads) {
      const int v = share.vector(space.picked[i / kGroup] * kGroup + i % kGroup);
      A most = lowest<A>();
      if (v < r.vectors) {
        uint4 q[1] = {load_vector(r, v)};
        most = vector_max<T>(q);
      }
      space.maxima[i] = most;
    }
    const auto key = [&](int i) { return ordered(space.maxima[i]); };
    const auto at = [&](int i) {
      return static_cast<uint32_t>(space.picked[i / kGroup] * kGroup + i % kGroup);
    };
    if (team.tid == 0) space.count[0] = 0;
    team.sync();
    const Cut<A> best = find_cut<4, kThreads, A>(team, picked * kGroup, top, key, at, space.histogram);
    for (int i = team.tid; i < picked * kGroup; i += kThreads) {
      const int v = share.vector(static_cast<int>(at(i)));
      if (v < r.vectors && best.takes(key(i), at(i))) add(v, 0);
    }
    team.sync();
  }
  const int body = space.count[0];
  if (place.cta == 0) {
    for (int e = team.tid; e < r.edges; e += kThreads)
      space.candidates[body + e] = {number_of(to_acc(r.x[r.edge(e)])), r.edge(e)};
    team.sync();
  }
  const int n = body + (place.cta == 0 ? r.edges : 0);
  Cut<A> last{0, 0xffffffffu};
  const auto key = [&](int i) { return ordered(space.candidates[i].value); };
  const auto at = [&](int i) { return static_cast<uint32_t>(space.candidates[i].at); };
  if (n > top) last = find_cut<4, kThreads, A>(team, n, top, key, at, space.histogram);
  for (int i = team.tid; i < n; i += kThreads) {
    if (!last.takes(key(i), at(i))) continue;
    const Element<A> own = space.candidates[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += space.candidates[j].before(own);
    space.best[rank] = own;
  }
  for (int i = n + team.tid; i < top; i += kThreads) space.best[i] = {lowest<A>(), 0x7fffffff};
  team.sync();
}

// ---------------------------------------------------------------------------------------------
// Kernels

template <typename A>
struct ScoresArgs {
  int top, groups;     // of a CTA
  A *logps, *entropy;  // logps may be NULL (no targets)
  A* top_logps;
  int64_t* top_ids;
  A* stats;  // NULL, or per row the base, the sum and the mean of z
};

template <typename A>
__device__ __forceinline__ void write_scores(const ScoresArgs<A>& p, int64_t r, A logit,
                                             const Scored<A>& part, double inv_temp) {
  const double s = part.s, mean = part.u * unit_of(part.u) / s;
  if (p.logps) p.logps[r] = static_cast<A>(logp_of(logit, Part<A>{part.m, part.s}, inv_temp));
  p.entropy[r] = static_cast<A>(log(s) - mean);
  if (p.stats) {
    p.stats[3 * r] = base_of(part.m);
    p.stats[3 * r + 1] = part.s;
    p.stats[3 * r + 2] = static_cast<A>(mean);
  }
}

// One pass over a row by a CTA, or where rows are few by a cluster. kGroup: 0 where no alternatives
// are asked for, else the vectors to a maximum.
template <typename T, typename A, int kThreads, int kGroup>
__global__ void __launch_bounds__(kThreads)
    scores_kernel(Rows a, ScoresArgs<A> p, double inv_temp, A k) {
  constexpr int kTile = kBatch * kThreads, kWarps = kThreads / 32;
  extern __shared__ uint4 shared[];
  const Place<kThreads> place;
  const int64_t r = place.row;
  const int64_t target = a.targets ? a.targets[r] : 0;
  if (a.targets && target == a.ignore) {
    if (place.first()) {
      p.logps[r] = A(0);
      p.entropy[r] = A(0);
      if (p.stats) p.stats[3 * r + 1] = A(kLeftOut);
    }
    if (place.cta == 0)
      for (int i = place.tid; i < p.top; i += kThreads) {
        p.top_logps[r * p.top + i] = A(0);
        p.top_ids[r * p.top + i] = a.ignore;
      }
    return;
  }
  cluster_started(place.ctas);
  const T* x = row_at<T>(a, r);
  const RowView<T> view(x, nullptr, reinterpret_cast<uintptr_t>(x), a.vocab);
  A logit = A(0);
  if (place.first() && a.targets) logit = target_logit<T, A>(x, a.vocab, target);
  const TopSpace<A> space(shared, p.top, p.groups, place.ctas);

  const A edge = place.edge() < view.edges ? to_acc(x[view.edge(place.edge())]) : lowest<A>();
  Scored<A> part{lowest<A>(), A(0), A(0)};
  int local = 0, groups = 0;
  for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile) {
    const int v = tile + place.tid;
    uint4 q[kBatch];
    if (tile + kTile <= view.vectors) {
      load_vectors<kBatch, kThreads>(view, v, q);
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        q[i] = v + i * kThreads < view.vectors ? load_vector(view, v + i * kThreads) : no_vector<T>();
    }
    A m = part.m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint4 one[1] = {q[i]};
      A most = vector_max<T>(one);
      m = max_acc(m, most);
      if constexpr (kGroup == 1) space.maxima[local + i * kThreads + place.tid] = most;
      if constexpr (kGroup == 32) {
        most = max_of_lanes<32>(most);
        if ((place.tid & 31) == 0)
          space.maxima[(local + i * kThreads) / 32 + place.tid / 32] = most;
      }
    }
    local += kTile;
    groups += kBatch * (kGroup == 32 ? kWarps : kThreads);
    move_base(part, m, k);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      A z[RowView<T>::E];
      unpack<T>(q[i], z);
      arguments(z, base_of(m), k);
      add_scores(z, part.s, part.u);
    }
  }
  move_base(part, max_acc(part.m, edge), k);
  if (place.edge() < view.edges) {
    const A z = max_nan(mul_rn(edge - base_of(part.m), k), least_argument(k)), e = exp_of(z);
    part.s += e;
    part.u += e * z;
  }
  part = join_scores_of_warps<kThreads>(join_scores<32>(part, k), k);
  if (place.first()) write_scores(p, r, logit, part, inv_temp);
  if constexpr (kGroup > 0) {
    choose_top<kGroup>(view, place, p.top, groups, space);
    const auto write = [&](int rank, const Element<A>& e) {
      p.top_logps[r * p.top + rank] =
          static_cast<A>(logp_of(e.value, Part<A>{part.m, part.s}, inv_temp));
      p.top_ids[r * p.top + rank] = e.at;
    };
    if (place.ctas == 1) {
      for (int i = place.tid; i < p.top; i += kThreads) write(i, space.best[i]);
    } else {
      // the CTAs' lists to the first CTA, where an element's rank is its place in its own list and
      // what of the others is before it
      auto cluster = cg::this_cluster();
      Element<A>* to = of_peer(space.best, 0, false) + place.cta * p.top;
      if (place.cta != 0)
        for (int i = place.tid; i < p.top; i += kThreads) to[i] = space.best[i];
      cluster.sync();
      if (place.cta == 0)
        for (int i = place.tid; i < p.top * place.ctas; i += kThreads) {
          const Element<A> own = space.best[i];
          const int list = i / p.top;
          int rank = i % p.top;
          for (int other = 0; other < place.ctas; ++other) {
            if (other == list) continue;
            const Element<A>* of = space.best + other * p.top;
            int low = 0, high = p.top;  // the first that is not before it
            while (low < high) {
              const int mid = (low + high) / 2;
              if (of[mid].before(own)) {
                low = mid + 1;
              } else {
                high = mid;
              }
            }
            rank += low;
          }
          if (rank < p.top && own.at != 0x7fffffff) write(rank, own);
        }
    }
  }
}

// The gradient of c log p_y + h entropy, both divided by t: exp(z) (alpha + beta z), and c at the
// target: alpha = (-c + h mean) / s, beta = -h / s.
template <typename A>
struct ScoresSlope {
  A base, alpha, beta, k;
  int target;
  double c;

  // target_ < 0 and `wanted` false: no target
  __device__ __forceinline__ ScoresSlope(const A* stats, double c_, double h, A k_, bool wanted,
                                         int64_t target_, int vocab)
      : base(stats[0]), k(k_), c(c_) {
    const bool in = target_ >= 0 && target_ < vocab;
    const double s = stats[1], mean = stats[2];
    target = in && wanted ? static_cast<int>(target_) : -1;
    alpha = in || !wanted ? static_cast<A>((h * mean - c) / s) : nan_of(A(0));
    beta = static_cast<A>(-h * unit_of(k_) / s);
  }
  __device__ __forceinline__ A at(A x, int v) const {
    const A z = max_nan(mul_rn(x - base, k), least_argument(k));
    const A d = mul_rn(exp_of(z), add_rn(mul_rn(z, beta), alpha));
    return v == target ? static_cast<A>(isinf(d) ? c : __dadd_rn(c, static_cast<double>(d))) : d;
  }
};

template <typename T, typename A>
__device__ __forceinline__ uint4 slope_vector(const uint4& q, const ScoresSlope<A>& slope) {
  A x[RowView<T>::E];
  unpack<T>(q, x);
  arguments(x, slope.base, slope.k);
#pragma unroll
  for (int j = 0; j < RowView<T>::E; ++j)
    x[j] = mul_rn(exp_of(x[j]), add_rn(mul_rn(x[j], slope.beta), slope.alpha));
  return pack<T>(x);
}

// coef_logp, coef_entropy: per row, may be NULL. A warp or a CTA takes a tile, `tiles` to the row.
template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(256)
    scores_grad_kernel(Rows a, double inv_temp, A k, const A* stats, const A* coef_logp,
                       const A* coef_entropy, T* grad, int tiles) {
  constexpr int kGroups = 256 / kThreads, kTile = kBatch * kThreads;
  const int tid = threadIdx.x % kThreads;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kThreads;
  if (i >= a.rows * tiles) return;
  const int64_t r = i / tiles;
  const int tile = static_cast<int>(i % tiles) * kTile;
  T* g = grad + r * a.vocab;
  const RowView<T> view(row_at<T>(a, r), g, reinterpret_cast<uintptr_t>(g), a.vocab);
  const int edge = tile == 0 ? tid : kNoEdge;
  if (stats[3 * r + 1] < A(0)) {
    zero_edge(view, edge);
    zero_tile<kThreads>(view, tile, tid);
  } else {
    const double c = coef_logp ? coef_logp[r] * inv_temp : 0.0;
    const double h = coef_entropy ? coef_entropy[r] * inv_temp : 0.0;
    const ScoresSlope<A> slope(stats + 3 * r, c, h, k, a.targets != nullptr,
                               a.targets ? a.targets[r] : -1, a.vocab);
    write_edge(view, edge, slope);
    write_tile<kThreads>(view, tile, tid, slope);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side

template <typename T, int kGroup>
int launch_scores(const Rows& a, ScoresArgs<typename AccOf<T>::type> p, double inv_temp, int ctas,
                  cudaStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr int kThreads = 256;
  const auto kernel = scores_kernel<T, A, kThreads, kGroup>;
  const size_t shared = kGroup ? TopSpace<A>::bytes(p.top, p.groups, ctas) : 0;
  const int rc = allow_shared(reinterpret_cast<const void*>(kernel), kSharedForTop);
  if (rc) return rc;
  return launch_clusters(kernel, a.rows, ctas, kThreads, shared, false, st, "scores_kernel launch", a,
                         p, inv_temp, exp_factor(A(0), inv_temp));
}

template <typename T>
int run_scores(const Rows& a, int top, double inv_temp, void* logps, void* entropy, void* top_logps,
               int64_t* top_ids, void* stats, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr int kTile = kBatch * 256;
  const int64_t vectors = a.vocab / RowView<T>::E, tiles = (vectors + kTile - 1) / kTile;
  int ctas = ctas_for(a.rows, vectors, 256, sm_count());
  ScoresArgs<A> p{top,
                  0,
                  static_cast<A*>(logps),
                  static_cast<A*>(entropy),
                  static_cast<A*>(top_logps),
                  top_ids,
                  static_cast<A*>(stats)};
  if (top == 0) return launch_scores<T, 0>(a, p, inv_temp, ctas, st);
  const auto share = [&] { return (tiles + ctas - 1) / ctas * kTile; };  // vectors of a CTA
  // maxima of whole groups of 32 vectors where there are enough of them to choose from
  const auto whole = [&] { return share() / 32 >= 2 * top; };
  const auto fits = [&] {
    const int64_t groups = whole() ? share() / 32 : share();
    return groups < 1 << 16 &&
           TopSpace<A>::bytes(top, static_cast<int>(groups), ctas) <= kSharedForTop;
  };
  while (ctas < 8 && !fits()) ctas *= 2;
  if (!fits())
    return report_error(TISO_ERR_ARGUMENT, "a vocabulary too large for top alternatives");
  p.groups = static_cast<int>(whole() ? share() / 32 : share());
  return whole() ? launch_scores<T, 32>(a, p, inv_temp, ctas, st)
                 : launch_scores<T, 1>(a, p, inv_temp, ctas, st);
}

template <typename T>
int run_scores_grad(const Rows& a, double inv_temp, const void* stats, const void* coef_logp,
                    const void* coef_entropy, void* grad, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int vectors = a.vocab / RowView<T>::E;
  const bool by_warp = by_warps(a.rows, vectors, 768, sm_count());
  const int tile = kBatch * (by_warp ? 32 : 256);
  const int tiles = vectors > tile ? (vectors + tile - 1) / tile : 1;
  const int64_t grid = by_warp ? (a.rows * tiles + 7) / 8 : a.rows * tiles;
  if (grid > 0x7fffffff) return report_error(TISO_ERR_ARGUMENT, "too many logits for one gradient");
  const auto kernel = by_warp ? scores_grad_kernel<T, A, 32> : scores_grad_kernel<T, A, 256>;
  kernel<<<static_cast<unsigned>(grid), 256, 0, st>>>(
      a, inv_temp, exp_factor(A(0), inv_temp), static_cast<const A*>(stats),
      static_cast<const A*>(coef_logp), static_cast<const A*>(coef_entropy), static_cast<T*>(grad),
      tiles);
  return launched("scores_grad_kernel launch");
}

}  // namespace
}  // namespace tiso

using namespace tiso;

extern "C" {

int tiso_scores(int dtype, const tiso_rows* x, const int64_t* targets, int64_t ignore_index,
                double temperature, int64_t top, void* logps, void* entropy, void* top_logps,
                int64_t* top_ids, void* stats, void* stream) {
  return guarded([&]() -> int {
    const int rc = check_rows(dtype, x, targets, nullptr, false);
    if (rc) return rc;
    if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
    if (top < 0 || top > kMostTop || top > x->vocab)
      return report_error(TISO_ERR_ARGUMENT, "top must be from 0 to 128 and to the vocabulary");
    if (x->rows == 0) return TISO_OK;
    if (!entropy || (targets && !logps) || (top && (!top_logps || !top_ids)))
      return report_error(TISO_ERR_ARGUMENT,
                          "entropy, logps and the alternatives' arrays must not be NULL");
    const Rows a = rows_of(x, targets, ignore_index);
    return by_type(dtype, [&](auto t) {
      return run_scores<decltype(t)>(a, static_cast<int>(top), 1.0 / temperature,
                                     targets ? logps : nullptr, entropy, top_logps, top_ids, stats,
                                     static_cast<cudaStream_t>(stream));
    });
  });
}

int tiso_scores_grad(int dtype, const tiso_rows* x, const int64_t* targets, double temperature,
                     const void* stats, const void* coef_logp, const void* coef_entropy, void* grad,
                     void* stream) {
  return guarded([&]() -> int {
    const int rc = check_rows(dtype, x, targets, grad, false);
    if (rc) return rc;
    if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
    if (x->rows == 0) return TISO_OK;
    if (!stats || !grad) return report_error(TISO_ERR_ARGUMENT, "stats and grad must not be NULL");
    if (coef_logp && !targets)
      return report_error(TISO_ERR_ARGUMENT, "coef_logp goes with targets");
    const Rows a = rows_of(x, targets, 0);
    return by_type(dtype, [&](auto t) {
      return run_scores_grad<decltype(t)>(a, 1.0 / temperature, stats, coef_logp, coef_entropy, grad,
                                          static_cast<cudaStream_t>(stream));
    });
  });
}

}  // extern "C"
