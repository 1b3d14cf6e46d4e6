// A token's scores from rows of logits (include/tiso.h: tiso_scores*): the log-probability of a given
// token, the entropy and the top alternatives, in one pass over the logits; and the gradient of the
// first two.
//
// With z = (x - m) / t, m the row's maximum, s = sum exp(z) and u = sum exp(z) z:
//   log p_v = z_v - log s,  entropy = log s - u / s,
// neither a difference of large numbers (s >= 1, u <= 0). Parts of a row join as for s alone: with
// d = (m1 - M) / t, s1 and u1 become s1 exp(d) and exp(d) (u1 + d s1).
//
// Top alternatives: the upper 16 bits of a number's key (its order as an integer) make it coarse. The
// pass leaves the coarse maximum of each unit of vectors in shared memory and finds a bound that `top`
// units reach at least: the alternatives are then among the elements that reach it. The units that do
// are read again, and what is found there, once or twice `top` elements as a rule, is sorted. The bound
// is the least of what the warps find for themselves, the q-th largest of their lanes' maxima, q = top
// / warps rounded up; where a warp alone has a row and q is large the top-th largest of the units'
// maxima, by bisection.
// Where more elements reach the bound than there is room for (equal logits, rows in order) the
// selection is by groups instead: the row is read again for the maxima of groups of neighbouring
// vectors; the `top` best groups (equal maxima: the first) hold the top elements, for each of the
// others has an element in each of these before it; and so on with their vectors and elements, each
// step an exact selection that no data makes longer.
#include "rows.cuh"
#include "select.cuh"

namespace tiso {
namespace {

constexpr int kMostTop = 128;
constexpr int kSharedForTop = 160 * 1024;

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

// The parts of a row's threads joined, first in each CTA (the threads have met then), and from there
// across a cluster in two steps: the CTAs send their parts, and wait for one another's later. Called
// by all threads, after cluster_started.
template <int kThreads, typename A>
struct JoinScores {
  static constexpr int kMostCtas = 8;
  Scored<A>* of_cta;  // kMostCtas, shared
  int ctas;

  __device__ __forceinline__ Scored<A> send(Scored<A> p, A k) const {
    p = join_scores<32>(p, k);
    if constexpr (kThreads > 32) {
      constexpr int kWarps = kThreads / 32;
      __shared__ Scored<A> of_warp[kWarps];
      const int lane = threadIdx.x & 31;
      if (lane == 0) of_warp[threadIdx.x >> 5] = p;
      __syncthreads();
      p = join_scores<kWarps>(of_warp[lane % kWarps], k);
      if (ctas > 1) {
        auto cluster = cg::this_cluster();
        const int rank = min(static_cast<int>(threadIdx.x), ctas - 1);
        Scored<A>* there = of_peer(&of_cta[cluster.block_rank()], rank, true);
        if (threadIdx.x < ctas) *there = p;
        cluster.barrier_arrive();
      }
    } else {
      __syncwarp();
    }
    return p;
  }
  __device__ __forceinline__ Scored<A> receive(Scored<A> p, A k) const {
    if (kThreads > 32 && ctas > 1) {
      cg::this_cluster().barrier_wait();
      const int at = threadIdx.x % kMostCtas;
      p = {lowest<A>(), A(0), A(0)};
      if (at < ctas) p = of_cta[at];
      p = join_scores<kMostCtas>(p, k);
    }
    return p;
  }
};

// ---------------------------------------------------------------------------------------------
// Top alternatives

// A row's element: the larger one, of equal ones the first, is before the other. In float as one
// integer, the number's key over the complement of its place.
template <typename A>
struct Ranked;
template <>
struct Ranked<float> {
  uint64_t key;
  Ranked() = default;
  __device__ __forceinline__ Ranked(float value, int at)
      : key(static_cast<uint64_t>(ordered(value)) << 32 | (0xffffffffu - static_cast<unsigned>(at))) {}
  __device__ __forceinline__ bool before(const Ranked& o) const { return key > o.key; }
  __device__ __forceinline__ float value() const {
    const uint32_t b = static_cast<uint32_t>(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
  }
  __device__ __forceinline__ int at() const {
    return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
  }
};
template <>
struct Ranked<double> {
  uint64_t key;
  int place;
  Ranked() = default;
  __device__ __forceinline__ Ranked(double value, int at) : key(ordered(value)), place(at) {}
  __device__ __forceinline__ bool before(const Ranked& o) const {
    return key > o.key || (key == o.key && place < o.place);
  }
  __device__ __forceinline__ double value() const {
    return __longlong_as_double(
        static_cast<long long>(key >> 63 ? key & 0x7fffffffffffffffULL : ~key));
  }
  __device__ __forceinline__ int at() const { return place; }
};

constexpr int kNowhere = 0x7fffffff;  // the place of an element that is not there

template <typename A>
__device__ __forceinline__ A number_of(A x) {  // NaN in the order of -infinity
  return x == x ? x : lowest<A>();
}

// The upper 16 bits of a number's key.
__device__ __forceinline__ uint32_t coarse(float x) { return ordered(x) >> 16; }
__device__ __forceinline__ uint32_t coarse(double x) {
  return static_cast<uint32_t>(ordered(x) >> 48);
}

// The least number of a coarse key, or of all.
__device__ __forceinline__ float least_of(uint32_t key, float) {
  const uint32_t b = key << 16;
  return key <= 0x7fu ? lowest<float>() : __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ double least_of(uint32_t key, double) {
  const uint64_t b = static_cast<uint64_t>(key) << 48;
  return key <= 0xfu ? lowest<double>()
                     : __longlong_as_double(static_cast<long long>(
                           b >> 63 ? b & 0x7fffffffffffffffULL : ~b));
}

constexpr int kMostUnits = 16;  // of a warp's lane

// What the threads that work on a row have to choose from (a cluster's CTAs each for their share).
struct TopSizes {
  int top, tiles;  // of this CTA's share, at most
  int groups;      // and groups of vectors
  bool whole;      // 32 vectors to a group, else one
  bool fine;       // a unit is one vector, else a batch of a thread's

  __host__ __device__ int rows() const { return fine ? tiles * kBatch : tiles; }  // of units
  __host__ __device__ int room() const { return 3 * top + 128; }
  __host__ __device__ int units() const { return (3 * top + 99) / 4 * 4; }
  // of a selection by groups
  __host__ __device__ int numbers() const { return whole && groups < 32 * top ? 32 * top : groups; }
};

// Their shared memory.
template <typename A, int kThreads>
struct TopSpace {
  static constexpr int kWarps = kThreads / 32;
  Ranked<A>* candidates;  // room, and up to a multiple of 32
  Ranked<A>* best;        // in the first CTA of a cluster top for each CTA
  double* log_s;
  unsigned* kth;          // of each warp
  int* picked;            // units, or top groups
  int* count;             // 2: candidates, picked
  unsigned* histogram;
  uint16_t* unit_max;     // rows of units x threads
  A* maxima;              // of the groups: in the same place

  static __host__ __device__ int rounded(const TopSizes& z) { return (z.room() + 31) / 32 * 32; }
  static __host__ __device__ int bytes(const TopSizes& z, int ctas) {
    const int maxima = z.numbers() * static_cast<int>(sizeof(A)), units = z.rows() * kThreads * 2;
    return static_cast<int>(sizeof(Ranked<A>)) * (rounded(z) + (z.top + 1) / 2 * 2 * ctas) + 16 +
           4 * ((kWarps + 3) / 4 * 4 + z.units() + 4 + kHistogram) +
           ((maxima > units ? maxima : units) + 15) / 16 * 16;
  }

  __device__ TopSpace(void* at, const TopSizes& z, int ctas) {
    candidates = static_cast<Ranked<A>*>(at);
    best = candidates + rounded(z);
    log_s = reinterpret_cast<double*>(best + (z.top + 1) / 2 * 2 * ctas);
    kth = reinterpret_cast<unsigned*>(log_s + 2);
    picked = reinterpret_cast<int*>(kth + (kWarps + 3) / 4 * 4);
    count = picked + z.units();
    histogram = reinterpret_cast<unsigned*>(count + 4);
    maxima = reinterpret_cast<A*>(histogram + kHistogram);
    unit_max = reinterpret_cast<uint16_t*>(maxima);
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

// The q-th largest of a warp's numbers (1 <= q <= 32): by taking out the largest, or by sorting.
__device__ __forceinline__ unsigned largest_of_warp(unsigned v, int q) {
  const int lane = threadIdx.x & 31;
  if (q <= 6) {
    unsigned most = 0;
    for (int i = 0; i < q; ++i) {
      most = __reduce_max_sync(0xffffffffu, v);
      if (lane == __ffs(__ballot_sync(0xffffffffu, v == most)) - 1) v = 0;
    }
    return most;
  }
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int d = size / 2; d; d /= 2) {
      const unsigned other = __shfl_xor_sync(0xffffffffu, v, d);
      const bool first = (lane & d) == 0, down = (lane & size) == 0;
      v = first == down ? max(v, other) : min(v, other);
    }
  return __shfl_sync(0xffffffffu, v, q - 1);
}

// A number that `top` of a warp's units' maxima reach, 0 where they are fewer: the top-th largest, or
// less where no more reach it.
__device__ __forceinline__ unsigned bound_of_warp(const uint16_t* unit_max, int rows, int top) {
  unsigned v[kMostUnits];
#pragma unroll
  for (int i = 0; i < kMostUnits; ++i)
    v[i] = i < rows ? unit_max[32 * i + (threadIdx.x & 31)] : 0u;
  unsigned bound = 0;
#pragma unroll 1
  for (int bit = 15; bit >= 0; --bit) {
    const unsigned more = bound | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int i = 0; i < kMostUnits; ++i) reach += v[i] >= more;
    reach = __reduce_add_sync(0xffffffffu, reach);
    if (reach >= top) bound = more;
    if (reach == top) break;
  }
  return bound;
}

// Up to so many alternatives a warp alone takes its bound from its lanes. 200000 x 2048 bf16, 16, 20, 24 and 28
// of them: 343, 391, 454 and 531 us so, 470, 483, 491 and 503 by bisection over the units; 50000 x 8192, 20 and 24:
// 257 and 290, 262 and 272.
constexpr int kMostByLanes = 20;

// For more alternatives than this a warp keeps the maximum of each vector of a short row, else that of a
// lane's batches: 200000 x 2048 bf16, 1, 5, 10 and 16 alternatives 288, 306, 325 and 343 us by vectors, 261,
// 280, 322 and 372 by batches; 200000 x 777 float32 247, 272, 287 and 300, 230, 253, 288 and 329.
constexpr int kMostByBatches = 8;

// How many of each warp's lanes are to reach the bound, over the warps whose lanes all have a vector;
// 0 where these are too few to give one.
template <int kThreads, typename T>
__device__ __forceinline__ int quota_of(const RowView<T>& r, const Place<kThreads>& place, int top,
                                        int& warps) {
  const int own = r.vectors - place.cta * kBatch * kThreads;
  warps = kThreads / 32;
  if (own >= kThreads) return (top + warps - 1) / warps;
  warps = max(own, 0) / 32;
  const int q = warps > 0 ? (top + warps - 1) / warps : 33;
  return q <= 32 ? q : 0;
}

// The `top` best elements of this CTA's share (all, if fewer), for any data: to space.candidates, not in
// order; returns how many.
template <int kGroup, int kThreads, typename T, typename A>
__device__ __noinline__ int choose_by_groups(const RowView<T> r, const Place<kThreads> place, int top,
                                             const TopSpace<A, kThreads> space) {
  constexpr int E = RowView<T>::E, kTile = kBatch * kThreads;
  const Team<kThreads> team{place.tid};
  const Share<kThreads> share{place.cta, place.ctas};
  int groups = 0;
  for (int tile = place.cta * kTile, l = 0; tile < r.vectors; tile += place.ctas * kTile, l += kTile) {
    for (int i = 0; i < kBatch; ++i) {
      const int v = tile + i * kThreads + place.tid;
      const uint4 q[1] = {v < r.vectors ? load_vector(r, v) : no_vector<T>()};
      A most = vector_max<T>(q);
      if (kGroup == 1) {
        space.maxima[l + i * kThreads + place.tid] = most;
      } else {
        most = max_of_lanes<32>(most);
        if (place.tid % 32 == 0) space.maxima[(l + i * kThreads + place.tid) / 32] = most;
      }
    }
    groups += kTile / kGroup;
  }
  if (team.tid < 2) space.count[team.tid] = 0;
  team.sync();
  // puts down the places of the numbers that are among the `top` largest of n
  const auto choose = [&](int n, const auto& key, const auto& at, int* places, int* count) {
    Cut<A> cut{0, 0xffffffffu};
    if (n > top) cut = find_cut<kThreads, A>(team, n, top, key, at, space.histogram);
    for (int i = team.tid; i < n; i += kThreads)
      if (cut.takes(key(i), at(i))) places[atomicAdd(count, 1)] = static_cast<int>(at(i));
    team.sync();
    return min(n, top);
  };
  const auto maximum = [&](int i) { return ordered(space.maxima[i]); };
  int picked = choose(groups, maximum, [](int i) { return static_cast<uint32_t>(i); }, space.picked,
                      space.count);
  const int* vectors = space.picked;  // local ones
  if constexpr (kGroup > 1) {
    for (int i = team.tid; i < picked * kGroup; i += kThreads) {
      const int v = share.vector(space.picked[i / kGroup] * kGroup + i % kGroup);
      A most = lowest<A>();
      if (v < r.vectors) {
        const uint4 q[1] = {load_vector(r, v)};
        most = vector_max<T>(q);
      }
      space.maxima[i] = most;
    }
    team.sync();
    int* chosen = reinterpret_cast<int*>(space.candidates);
    picked = choose(picked * kGroup, maximum,
                    [&](int i) {
                      return static_cast<uint32_t>(space.picked[i / kGroup] * kGroup + i % kGroup);
                    },
                    chosen, space.count + 1);
    for (int i = team.tid; i < picked; i += kThreads) space.picked[i] = chosen[i];
    team.sync();
  }
  // their elements, and the single ones
  if (team.tid == 0) *space.count = 0;
  const int body = picked * E, edges = place.cta == 0 ? r.edges : 0, n = body + edges;
  const auto element = [&](int i) {
    if (i >= body) return r.edge(i - body);
    const int v = share.vector(vectors[i / E]);
    return v < r.vectors ? r.element(v) + i % E : kNowhere - i;  // distinct, behind all others
  };
  const auto number = [&](int i) {
    const int at = element(i);
    return at <= kNowhere - n ? number_of(to_acc(r.x[at])) : lowest<A>();
  };
  Cut<A> cut{0, 0xffffffffu};
  if (n > top)
    cut = find_cut<kThreads, A>(
        team, n, top, [&](int i) { return ordered(number(i)); },
        [&](int i) { return static_cast<uint32_t>(element(i)); }, space.histogram);
  team.sync();
  for (int i = team.tid; i < n; i += kThreads) {
    const int at = element(i);
    if (at > kNowhere - n || !cut.takes(ordered(number(i)), static_cast<uint32_t>(at))) continue;
    space.candidates[atomicAdd(space.count, 1)] = Ranked<A>(number(i), at);
  }
  team.sync();
  return *space.count;
}

// The elements of this CTA's share among which its `top` best are, to space.candidates; returns how
// many. tiles: of the share; own: the thread's coarse maximum; edge: its single element. The maxima, the
// warps' bounds and counts of 0 are written and the threads have met. meanwhile() is called between two more meetings.
template <int kThreads, typename T, typename A, typename F>
__device__ __forceinline__ int choose_top(const RowView<T>& r, const Place<kThreads>& place,
                                          const TopSizes& z, int tiles, unsigned own, A edge,
                                          const TopSpace<A, kThreads>& space, const F& meanwhile) {
  constexpr int E = RowView<T>::E, kTile = kBatch * kThreads;
  const Team<kThreads> team{place.tid};
  const Share<kThreads> share{place.cta, place.ctas};
  const int rows = kThreads == 32 && z.fine ? tiles * kBatch : tiles;  // of units
  unsigned bound = 0;
  if (kThreads == 32 && z.top > kMostByLanes) {
    bound = bound_of_warp(space.unit_max, rows, z.top);
  } else {
    int warps;
    if (quota_of(r, place, z.top, warps) > 0) {
      bound = space.kth[0];
      for (int i = 1; i < warps; ++i) bound = min(bound, space.kth[i]);
    }
  }
  const auto add = [&](A x, int at) {
    const int slot = atomicAdd(space.count, 1);
    if (slot < z.room()) space.candidates[slot] = Ranked<A>(x, at);
  };
  // a unit's first vector; a batch's others are kThreads apart
  const bool fine = kThreads == 32 && z.fine;
  const int each = fine ? 1 : kBatch, log_each = fine ? 0 : 2;
  static_assert(kBatch == 4, "log_each");
  const auto first = [&](int unit) {
    return share.vector(fine ? unit : unit / kThreads * kTile + unit % kThreads);
  };
  const A least = least_of(bound, A(0));
  if (own >= bound) {
    constexpr int kAhead = 4;
    for (int row = 0; row < rows; row += kAhead) {
      unsigned most[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        most[i] = row + i < rows ? space.unit_max[(row + i) * kThreads + team.tid] : 0u;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int unit = (row + i) * kThreads + team.tid;
        if (most[i] == 0 || most[i] < bound || row + i >= rows) continue;  // 0: no vector
        const int slot = atomicAdd(space.count + 1, 1);
        if (slot < z.units()) space.picked[slot] = unit;
      }
    }
  }
  if (place.edge() < r.edges && !(edge < least)) add(number_of(edge), r.edge(place.edge()));
  team.sync();
  const int picked = space.count[1];
  if (picked <= z.units()) {
    for (int i = team.tid; i < picked << log_each; i += kThreads) {
      const int v = first(space.picked[i >> log_each]) + (i & (each - 1)) * kThreads;
      if (v >= r.vectors) continue;
      A x[E];
      unpack<T>(load_vector(r, v), x);
#pragma unroll
      for (int c = 0; c < E; ++c)
        if (!(x[c] < least)) add(number_of(x[c]), r.element(v) + c);
    }
  }
  meanwhile();
  team.sync();
  const int n = space.count[0];
  if (picked <= z.units() && n <= z.room()) return n;
  team.sync();  // the counts have been read
  return z.whole ? choose_by_groups<32>(r, place, z.top, space)
                 : choose_by_groups<1>(r, place, z.top, space);
}

template <typename A>
__device__ __forceinline__ Ranked<A> of_lane(const Ranked<A>& v, int d) {
  Ranked<A> r = v;
  r.key = __shfl_xor_sync(0xffffffffu, v.key, d);
  if constexpr (sizeof(A) == 8) r.place = __shfl_xor_sync(0xffffffffu, v.place, d);
  return r;
}

// Calls fn(rank, element) for the `top` best of the n candidates, each by one thread. Few are counted
// through; of more 32 at a time are sorted by a warp, and a rank is the place among these and, by
// halving, what of the others is before it.
constexpr int kFewCandidates = 48;

template <int kThreads, typename A, typename F>
__device__ __forceinline__ void rank_candidates(const Team<kThreads>& team, int n, int top,
                                                const TopSpace<A, kThreads>& space, const F& fn) {
  if (n <= kFewCandidates) {
    for (int i = team.tid; i < n; i += kThreads) {
      const Ranked<A> own = space.candidates[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += space.candidates[j].before(own);
      if (rank < top) fn(rank, own);
    }
    return;
  }
  const int lane = team.tid & 31, runs = (n + 31) / 32;
  for (int run = team.tid / 32; run < runs; run += kThreads / 32) {
    const int i = 32 * run + lane;
    Ranked<A> v = i < n ? space.candidates[i] : Ranked<A>(lowest<A>(), kNowhere);
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
      for (int d = size / 2; d; d /= 2) {
        const Ranked<A> other = of_lane(v, d);
        const bool first = (lane & d) == 0, down = (lane & size) == 0;
        if (other.before(v) == (first == down)) v = other;
      }
    space.candidates[i] = v;
  }
  team.sync();
  for (int i = team.tid; i < 32 * runs; i += kThreads) {
    const Ranked<A> own = space.candidates[i];
    int rank = lane;
    for (int run = 0; run < runs && rank < top; ++run) {
      if (run == i / 32) continue;
      const Ranked<A>* of = space.candidates + 32 * run;
      int before = 0;
#pragma unroll
      for (int d = 16; d; d /= 2) before += of[before + d - 1].before(own) ? d : 0;
      rank += before + of[before].before(own);
    }
    if (rank < top && own.at() != kNowhere) fn(rank, own);
  }
}

// ---------------------------------------------------------------------------------------------
// Kernels

template <typename A>
struct ScoresArgs {
  TopSizes sizes;
  A *logps, *entropy;  // logps may be NULL (no targets)
  A* top_logps;
  int64_t* top_ids;
  A* stats;  // NULL, or per row the base, the sum and the mean of z
};

// By one thread; returns log s.
template <typename A>
__device__ __forceinline__ double write_scores(const ScoresArgs<A>& p, int64_t r, A logit,
                                               const Scored<A>& part, double inv_temp) {
  const double s = part.s, mean = part.u * unit_of(part.u) / s, log_s = log(s);
  if (p.logps)
    p.logps[r] = static_cast<A>(
        (static_cast<double>(logit) - static_cast<double>(base_of(part.m))) * inv_temp - log_s);
  p.entropy[r] = static_cast<A>(log_s - mean);
  if (p.stats) {
    p.stats[3 * r] = base_of(part.m);
    p.stats[3 * r + 1] = part.s;
    p.stats[3 * r + 2] = static_cast<A>(mean);
  }
  return log_s;
}

// A row that is left out.
template <int kThreads, typename A>
__device__ __forceinline__ void write_no_scores(const Rows& a, const ScoresArgs<A>& p,
                                                const Place<kThreads>& place) {
  const int64_t r = place.row;
  const int top = p.sizes.top;
  if (place.first()) {
    p.logps[r] = A(0);
    p.entropy[r] = A(0);
    if (p.stats) p.stats[3 * r + 1] = A(kLeftOut);
  }
  if (place.cta == 0)
    for (int i = place.tid; i < top; i += kThreads) {
      p.top_logps[r * top + i] = A(0);
      p.top_ids[r * top + i] = a.ignore;
    }
}

// One pass over a row by a warp, a CTA or a cluster; its alternatives if kTop. 4096 x 131072 bf16 in 164 us
// without alternatives (the copy bandwidth; 7.1 instructions an element where the log-probability
// alone takes 5.1), 191, 199 and 220 us with 1, 20 and 64 of them: 168 us of it are the pass, 8 to find
// the batches that reach the bound, 15 to 34 to read them again (L2's latency under load), 6 to 13 to
// rank what they hold. 50021 to the row, 2865 of 4092 rows read, in 60 us (71 % of the copy bandwidth).
template <bool kTop, int kThreads, typename T, typename A>
__device__ __forceinline__ void scores_row(const Rows& a, const ScoresArgs<A>& p, double inv_temp, A k,
                                           const Place<kThreads>& place, int64_t target, void* shared) {
  constexpr int kTile = kBatch * kThreads;
  const Team<kThreads> team{place.tid};
  const int64_t r = place.row;
  const T* x = row_at<T>(a, r);
  const RowView<T> view(x, nullptr, reinterpret_cast<uintptr_t>(x), a.vocab);
  A logit = A(0);
  if (place.cta == 0 && place.tid == kThreads - 1 && a.targets)
    logit = target_logit<T, A>(x, a.vocab, target);
  const TopSpace<A, kThreads> space(shared, p.sizes, place.ctas);
  if (kTop && team.tid < 2) space.count[team.tid] = 0;

  const A edge = place.edge() < view.edges ? to_acc(x[view.edge(place.edge())]) : lowest<A>();
  Scored<A> part{lowest<A>(), A(0), A(0)};
  int j = 0;
  for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile, ++j) {
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
    if (kTop && kThreads == 32 && p.sizes.fine) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint4 one[1] = {q[i]};
        const A most = vector_max<T>(one);
        space.unit_max[(j * kBatch + i) * kThreads + place.tid] =
            v + i * kThreads < view.vectors ? coarse(most) : 0u;
        m = max_acc(m, most);
      }
    } else {
      const A most = vector_max<T>(q);
      if constexpr (kTop)
        space.unit_max[j * kThreads + place.tid] = v < view.vectors ? coarse(most) : 0u;
      m = max_acc(m, most);
    }
    move_base(part, m, k);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      A z[RowView<T>::E];
      unpack<T>(q[i], z);
      arguments(z, base_of(m), k);
      add_scores(z, part.s, part.u);
    }
  }
  const unsigned own = coarse(part.m);
  if constexpr (kTop) {
    int warps;
    const int quota = quota_of(view, place, p.sizes.top, warps);
    if (quota > 0 && (kThreads > 32 || p.sizes.top <= kMostByLanes)) {
      const unsigned kth = largest_of_warp(own, quota);
      if (team.tid % 32 == 0) space.kth[team.tid / 32] = kth;
    }
  }
  move_base(part, max_acc(part.m, edge), k);
  if (place.edge() < view.edges) {
    const A z = max_nan(mul_rn(edge - base_of(part.m), k), least_argument(k)), e = exp_of(z);
    part.s += e;
    part.u += e * z;
  }
  __shared__ Scored<A> of_cta[JoinScores<kThreads, A>::kMostCtas];
  const JoinScores<kThreads, A> join{of_cta, place.ctas};
  part = join.send(part, k);
  const auto write_first = [&] {
    part = join.receive(part, k);
    if (place.cta == 0 && place.tid == kThreads - 1) {
      const double log_s = write_scores(p, r, logit, part, inv_temp);
      if (kTop) *space.log_s = log_s;
    }
  };
  if constexpr (!kTop) {
    write_first();
  } else {
    const int top = p.sizes.top;
    const int n = choose_top(view, place, p.sizes, j, own, edge, space, write_first);
    const double base = base_of(part.m);
    const auto write = [&](int rank, const Ranked<A>& e) {
      p.top_logps[r * top + rank] =
          static_cast<A>((static_cast<double>(e.value()) - base) * inv_temp - *space.log_s);
      p.top_ids[r * top + rank] = e.at();
    };
    if (place.ctas == 1) {
      rank_candidates(team, n, top, space, write);
    } else if constexpr (kThreads > 32) {
      // the CTAs' lists to the first CTA, where an element's rank is its place in its own list and
      // what of the others is before it
      auto cluster = cg::this_cluster();
      Ranked<A>* to = of_peer(space.best, 0, false) + place.cta * top;
      rank_candidates(team, n, top, space, [&](int rank, const Ranked<A>& e) { to[rank] = e; });
      for (int i = n + place.tid; i < top; i += kThreads) to[i] = Ranked<A>(lowest<A>(), kNowhere);
      cluster.sync();
      if (place.cta == 0)
        for (int i = place.tid; i < top * place.ctas; i += kThreads) {
          const Ranked<A> own_element = space.best[i];
          const int list = i / top;
          int rank = i % top;
          for (int other = 0; other < place.ctas; ++other) {
            if (other == list) continue;
            const Ranked<A>* of = space.best + other * top;
            int low = 0, high = top;  // the first that is not before it
            while (low < high) {
              const int mid = (low + high) / 2;
              if (of[mid].before(own_element)) {
                low = mid + 1;
              } else {
                high = mid;
              }
            }
            rank += low;
          }
          if (rank < top && own_element.at() != kNowhere) write(rank, own_element);
        }
    }
  }
}

// Resident at 48 registers a thread; with alternatives 8 bytes are spilled for 16 bits, 36 in float32 (stores;
// float64, with twice the registers, nothing; by groups 64 in float32).
constexpr int kSmThreads = 1280;

template <typename T, typename A, int kThreads, bool kTop>
__global__ void __launch_bounds__(kThreads, kSmThreads / kThreads / (sizeof(T) == 8 ? 2 : 1))
    scores_kernel(Rows a, ScoresArgs<A> p, double inv_temp, A k) {
  extern __shared__ uint4 shared[];
  const Place<kThreads> place;
  const int64_t target = a.targets ? a.targets[place.row] : 0;
  if (a.targets && target == a.ignore) {
    write_no_scores(a, p, place);
    return;
  }
  cluster_started(place.ctas);
  scores_row<kTop, kThreads, T>(a, p, inv_temp, k, place, target, shared);
}

// Short rows: a warp to a row.
template <typename T, typename A, bool kTop>
__global__ void __launch_bounds__(32 * kRowWarps)
    scores_warp_kernel(Rows a, ScoresArgs<A> p, double inv_temp, A k) {
  extern __shared__ uint4 shared[];
  const Place<32> place;
  if (place.row >= a.rows) return;
  const int64_t target = a.targets ? a.targets[place.row] : 0;
  if (a.targets && target == a.ignore) {
    write_no_scores(a, p, place);
    return;
  }
  char* own = reinterpret_cast<char*>(shared) +
              static_cast<int>(threadIdx.x / 32) * TopSpace<A, 32>::bytes(p.sizes, 1);
  scores_row<kTop, 32, T>(a, p, inv_temp, k, place, target, own);
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
    const A s = stats[1], mean = stats[2], of_entropy = static_cast<A>(h);
    target = in && wanted ? static_cast<int>(target_) : -1;
    // (not in double: two divisions a thread would be a third of a tile's instructions)
    alpha = in || !wanted ? (of_entropy * mean - static_cast<A>(c)) / s : nan_of(A(0));
    beta = -of_entropy * static_cast<A>(unit_of(k_)) / s;
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

// One more read of the logits. Bound by memory: 4 x 1023 of 1024 x 50021 bf16, 30 % left out, in 132 us (0.70 GB,
// 80 % of the copy bandwidth; three quarters of the rows are read and written at different alignments).
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

// What there is to choose from where `threads` threads and `ctas` CTAs take a row.
template <typename T>
TopSizes top_sizes(int top, int64_t vectors, int threads, int ctas) {
  const int64_t tile = int64_t{kBatch} * threads, tiles = (vectors + tile - 1) / tile;
  const int64_t share = (tiles + ctas - 1) / ctas;
  const bool whole = share * tile > 1024 && share * tile / 32 >= 2 * top;
  const int64_t groups = whole ? share * tile / 32 : share * tile;
  const bool fine = threads == 32 && top > kMostByBatches && share * kBatch <= kMostUnits;
  return {top, static_cast<int>(share), static_cast<int>(groups), whole, fine};
}

// By CTAs of kThreads, or clusters of them.
template <typename T, bool kTop, int kThreads>
int launch_score_rows(const Rows& a, ScoresArgs<typename AccOf<T>::type> p, double inv_temp, int sms,
                      cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int64_t vectors = a.vocab / RowView<T>::E;
  int ctas = ctas_for(a.rows, vectors, kThreads, sms);
  const auto fits = [&] {
    p.sizes = top_sizes<T>(p.sizes.top, vectors, kThreads, ctas);
    return !kTop || (p.sizes.groups < 1 << 16 && p.sizes.tiles < 1 << 15 &&
                     TopSpace<A, kThreads>::bytes(p.sizes, ctas) <= kSharedForTop);
  };
  while (!fits() && ctas < 8) ctas *= 2;
  if (!fits())
    return report_error(TISO_ERR_ARGUMENT, "a vocabulary too large for top alternatives");
  const auto kernel = scores_kernel<T, A, kThreads, kTop>;
  const int rc = allow_shared(reinterpret_cast<const void*>(kernel), kSharedForTop);
  if (rc) return rc;
  const size_t shared = kTop ? TopSpace<A, kThreads>::bytes(p.sizes, ctas) : 0;
  return launch_clusters(kernel, a.rows, ctas, kThreads, shared, false, st, "scores_kernel launch", a,
                         p, inv_temp, exp_factor(A(0), inv_temp));
}

// Rows of up to kFewVectors vectors, where there are many, take CTAs of 128 threads for up to 64
// alternatives: the few steps after a row's sum are short of work, and more rows hide them. 16384 x
// 32000 bf16, 1, 20 and 64 alternatives: 232, 257 and 338 us by 128 threads, 279, 307 and 373 by 256;
// 4096 x 131072, 64: 237 and 228. (More alternatives than half the threads, and the bound is loose.)
constexpr int kFewVectors = 8192, kMostByHalf = 64;

template <typename T, bool kTop>
int launch_scores(const Rows& a, ScoresArgs<typename AccOf<T>::type> p, double inv_temp,
                  cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int64_t vectors = a.vocab / RowView<T>::E;
  const int top = p.sizes.top, sms = sm_count();
  if (by_warps(a.rows, vectors, 2048, sms)) {
    p.sizes = top_sizes<T>(top, vectors, 32, 1);
    const int64_t shared = kTop ? int64_t{kRowWarps} * TopSpace<A, 32>::bytes(p.sizes, 1) : 0;
    if (shared <= kSharedForTop) {
      const auto kernel = scores_warp_kernel<T, A, kTop>;
      const int rc = allow_shared(reinterpret_cast<const void*>(kernel), kSharedForTop);
      if (rc) return rc;
      return launch_clusters(kernel, (a.rows + kRowWarps - 1) / kRowWarps, 1, 32 * kRowWarps, shared,
                             false, st, "scores_warp_kernel launch", a, p, inv_temp,
                             exp_factor(A(0), inv_temp));
    }
  }
  if constexpr (kTop)
    if (vectors <= kFewVectors && top <= kMostByHalf && a.rows >= int64_t{16} * sms)
      return launch_score_rows<T, kTop, 128>(a, p, inv_temp, sms, st);
  return launch_score_rows<T, kTop, 256>(a, p, inv_temp, sms, st);
}

template <typename T>
int run_scores(const Rows& a, int top, double inv_temp, void* logps, void* entropy, void* top_logps,
               int64_t* top_ids, void* stats, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  ScoresArgs<A> p{};
  p.sizes.top = top;
  p.logps = static_cast<A*>(logps);
  p.entropy = static_cast<A*>(entropy);
  p.top_logps = static_cast<A*>(top_logps);
  p.top_ids = top_ids;
  p.stats = static_cast<A*>(stats);
  return top ? launch_scores<T, true>(a, p, inv_temp, st) : launch_scores<T, false>(a, p, inv_temp, st);
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
