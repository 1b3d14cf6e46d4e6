// Distillation from a teacher's top lists (include/tiso.h: tiso_distill*): a divergence between the
// teacher's and the student's probabilities of the listed tokens and of the rest as one, with its
// gradient in the student's logits.
//
// Over the buckets b (the listed tokens, and the rest) with the student's P and the teacher's Q:
//   forward  D = sum Q log(Q / P)
//   reverse  D = sum P log(P / Q)
//   jensen   D = a sum Q log(Q / M) + (1 - a) sum P log(P / M),  M = a Q + (1 - a) P
// and with f = dD / dP of each bucket, dD / dz_v = p_v (f_b - sum P f): every token of the rest has
// its probability times one factor, so a row is read for its sum, the few steps over the list give
// the factors, and a second read writes the gradient.
//
// The rest's probability is summed from the rest's own exponentials, taken from the rest's own
// maximum: as the row's sum less the listed ones it would cancel where the list holds nearly all, and
// taken from the row's maximum it would underflow where the student is sure of a listed token. The
// row's pass leaves the listed tokens out by a bit for each of its elements in shared memory.
#include "rows.cuh"
#include "select.cuh"

namespace tiso {
namespace {

constexpr int kMostListed = 128;
constexpr int kSmThreads = 1536;  // resident at 40 registers a thread
constexpr int kSharedForBits = 160 * 1024;
// the teacher's rest where it is divided by: a list's float log-probabilities say no less
constexpr double kLeastRest = 1.0 / (1 << 24);

template <typename A>
struct DistillArgs {
  TokenWeights<A> weights;
  const int64_t* ids;
  const A* logps;
  int top, kind;
  bool drop;
  double mix, upstream;
  A* divergence;  // per row
  double* coef;   // NULL, or per row the rest's factor for an upstream gradient of 1
  A* stats;       // per row the rest's base, and -1 where the row is left out
  A* listed;      // per row and entry the gradient for an upstream gradient of 1
  A* terms;       // per unit (a row, or a CTA's rows) w D
  A* out;
  double* total;
  unsigned* done;
};

// Sums over the list's tokens: of q, q log q, q z, e = exp(z) and e (z - log q), z the logits from the
// list's own maximum, over t; and how many tokens there are.
struct ListSums {
  double q, q_log_q, q_z, e, e_far;
  int tokens;
};

// What the gradient of the list is made of, once the row's sum is known.
struct Settled {
  double c;      // the row's share of the loss, over t
  double p;      // of an e: its probability
  double log_p;  // of a z: its logarithm
  double mean;   // sum P f
  double list_q, whole;
};

constexpr int kListWarps = kMostListed / 32;

// Shared memory of the threads that work on a row.
template <typename A>
struct ListSpace {
  double *q, *log_q, *e;  // the teacher's probabilities; exp(z)
  ListSums* sums;         // of each warp that has entries
  Settled* settled;
  A *logit, *gradient;
  A* most;                // of each of these warps, the largest logit
  int *id, *lead;         // -1: no entry; the first entry of its id
  int *bad, *twice;       // an id out of range; an id listed again
  unsigned* edge_bits;    // of the single elements
  unsigned* bits;         // of this CTA's share of the vectors: a bit an element

  static __host__ __device__ int entries(int top) { return (top + 3) / 4 * 4; }
  static __host__ __device__ int bytes(int top, int bits) {
    return entries(top) * static_cast<int>(3 * sizeof(double) + 2 * sizeof(A) + 2 * sizeof(int)) +
           static_cast<int>(kListWarps * sizeof(ListSums) + sizeof(Settled) + kListWarps * sizeof(A)) +
           16 + (bits + 15) / 16 * 16;
  }

  __device__ ListSpace(void* at, int top) {
    const int n = entries(top);
    q = static_cast<double*>(at);
    log_q = q + n;
    e = log_q + n;
    sums = reinterpret_cast<ListSums*>(e + n);
    settled = reinterpret_cast<Settled*>(sums + kListWarps);
    logit = reinterpret_cast<A*>(settled + 1);
    gradient = logit + n;
    most = gradient + n;
    id = reinterpret_cast<int*>(most + kListWarps);
    lead = id + n;
    bad = lead + n;
    twice = bad + 1;
    edge_bits = reinterpret_cast<unsigned*>(bad + 2);
    bits = edge_bits + 2;
  }
};

// Where an element lies among those of the threads that work on a row.
template <int kThreads, typename T>
struct Spot {
  int cta, bit;  // of the bits of that CTA, or with `edge` of the edges'
  bool edge;

  __device__ __forceinline__ Spot(const RowView<T>& r, int ctas, int element) {
    constexpr int E = RowView<T>::E, kTile = kBatch * kThreads;
    edge = element < r.head || element >= r.head + r.vectors * E;
    if (edge) {
      cta = 0;
      bit = element < r.head ? element : element - r.vectors * E;
    } else {
      const int v = (element - r.head) / E, tile = v / kTile, in = v % kTile;
      cta = tile % ctas;
      bit = ((tile / ctas * kThreads + in % kThreads) * kBatch + in / kThreads) * E +
            (element - r.head) % E;
    }
  }
};

// The bits of the vectors that a thread takes of its CTA's tile `local`.
template <int kThreads, typename T>
__device__ __forceinline__ unsigned bits_of_tile(const unsigned* bits, int local, int tid) {
  const int at = local * kThreads + tid;
  if constexpr (RowView<T>::E == 8) return bits[at];
  if constexpr (RowView<T>::E == 4) return reinterpret_cast<const uint16_t*>(bits)[at];
  return reinterpret_cast<const uint8_t*>(bits)[at];
}

// -infinity for the elements whose bits are set.
template <typename T>
__device__ __forceinline__ void hide(uint4& q, unsigned bits) {
  const uint4 none = no_vector<T>();
  uint32_t* w = reinterpret_cast<uint32_t*>(&q);
  const uint32_t* n = reinterpret_cast<const uint32_t*>(&none);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t gone = (bits >> 2 * i & 1 ? 0xffffu : 0u) | (bits >> 2 * i & 2 ? 0xffff0000u : 0u);
      w[i] = (w[i] & ~gone) | (n[i] & gone);
    } else if constexpr (sizeof(T) == 4) {
      if (bits >> i & 1) w[i] = n[i];
    } else {
      if (bits >> (i / 2) & 1) w[i] = n[i];
    }
  }
}

// Adds a tile's vectors but for the listed tokens.
template <typename T, typename A>
__device__ __forceinline__ void add_rest(Part<A>& p, uint4 (&q)[kBatch], unsigned bits, A k) {
  constexpr int E = RowView<T>::E;
  if (bits) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const unsigned own = bits >> i * E & ((1u << E) - 1);
      if (own) hide<T>(q[i], own);
    }
  }
  add_vectors<T>(p, q, k);
}

// Adds one of the single elements, unless it is listed.
template <typename T, int kThreads, typename A>
__device__ __forceinline__ void add_edge(Part<A>& p, const RowView<T>& r, const Place<kThreads>& place,
                                         unsigned edge_bits, A k) {
  const int e = place.edge();
  const A edge = e < r.edges && !(edge_bits >> e & 1) ? to_acc(r.x[r.edge(e)]) : lowest<A>();
  const A m = max_acc(p.m, edge), base = base_of(m);
  p.s = (p.m == m ? p.s : p.s * scaled_exp(p.m - base, k)) + scaled_exp(edge - base, k);
  p.m = m;
}

__device__ __forceinline__ double sum_of_warp(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ __forceinline__ double product(double x, double y) { return x == 0 ? 0.0 : x * y; }

// Warps with entries of a list, and the largest of its logits.
template <int kThreads>
__device__ __forceinline__ int warps_of(int top) {
  return min((top + 31) / 32, kThreads / 32);
}
template <int kThreads, typename A>
__device__ __forceinline__ A most_of(const ListSpace<A>& space, int top) {
  A most = space.most[0];
  for (int i = 1; i < warps_of<kThreads>(top); ++i) most = max_acc(most, space.most[i]);
  return most;
}

// The list of row r into shared memory, its bits, and its sums (after the next meeting of the
// threads).
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void read_list(const Rows& a, const DistillArgs<A>& p, int64_t r,
                                          const RowView<T>& view, const Place<kThreads>& place,
                                          int bit_words, double inv_temp, const ListSpace<A>& space) {
  const Team<kThreads> team{place.tid};
  for (int i = team.tid; i < bit_words; i += kThreads) space.bits[i] = 0;
  if (team.tid == 0) *space.bad = *space.twice = static_cast<int>(*space.edge_bits = 0u);
  team.sync();
  const bool has_entries = team.tid / 32 * 32 < p.top;  // this warp
  A most = lowest<A>();
  for (int k = team.tid; k < p.top; k += kThreads) {
    const int64_t id = p.ids[r * p.top + k];
    const bool listed = id != a.ignore, in = id >= 0 && id < a.vocab;
    if (listed && !in) *space.bad = 1;
    space.id[k] = space.lead[k] = -1;
    space.gradient[k] = A(0);
    if (!listed || !in) continue;
    const double log_q = static_cast<double>(p.logps[r * p.top + k]);
    const A logit = to_acc(view.x[id]);
    const Spot<kThreads, T> spot(view, place.ctas, static_cast<int>(id));
    if (spot.cta == place.cta) {
      unsigned* word = spot.edge ? space.edge_bits : space.bits + spot.bit / 32;
      if (atomicOr(word, 1u << spot.bit % 32) >> spot.bit % 32 & 1) *space.twice = 1;
    }
    space.id[k] = static_cast<int>(id);
    space.lead[k] = k;
    space.logit[k] = logit;
    space.log_q[k] = log_q;
    space.q[k] = exp(log_q);
    most = max_acc(most, logit);
  }
  if (has_entries) {
    most = max_of_lanes<32>(most);
    if (team.tid % 32 == 0) space.most[team.tid / 32] = most;
  }
  team.sync();
  if (place.ctas > 1 || *space.twice) {
    // the same id again: its probabilities are added up in its first entry. (A CTA of a cluster sees
    // only its own elements' bits, and looks through the list.)
    for (int k = team.tid; k < p.top; k += kThreads) {
      const int id = space.id[k];
      if (id < 0) continue;
      int first = k;
      for (int j = k - 1; j >= 0; --j)
        if (space.id[j] == id) first = j;
      space.lead[k] = first;
    }
    team.sync();
    for (int k = team.tid; k < p.top; k += kThreads) {
      if (space.lead[k] != k) continue;
      double q = space.q[k];
      bool more = false;
      for (int j = k + 1; j < p.top; ++j)
        if (space.lead[j] == k) {
          q += space.q[j];
          more = true;
        }
      if (more) {
        space.q[k] = q;
        space.log_q[k] = log(q);
      }
    }
    team.sync();
  }
  if (!has_entries) return;
  const double base = base_of(most_of<kThreads>(space, p.top));
  ListSums sums{};
  for (int k = team.tid; k < p.top; k += kThreads) {
    if (space.lead[k] != k) continue;
    const double q = space.q[k], log_q = space.log_q[k];
    const double z = (static_cast<double>(space.logit[k]) - base) * inv_temp, e = exp(z);
    space.e[k] = e;
    sums.q += q;
    sums.q_log_q += product(q, log_q);
    sums.q_z += product(q, z);
    sums.e += e;
    sums.e_far += product(e, z - log_q);
    ++sums.tokens;
  }
  sums.q = sum_of_warp(sums.q);
  sums.q_log_q = sum_of_warp(sums.q_log_q);
  sums.q_z = sum_of_warp(sums.q_z);
  sums.e = sum_of_warp(sums.e);
  sums.e_far = sum_of_warp(sums.e_far);
  sums.tokens = __reduce_add_sync(0xffffffffu, sums.tokens);
  if (team.tid % 32 == 0) space.sums[team.tid / 32] = sums;
}

// The teacher's probabilities of the list and of the rest.
struct Teacher {
  double list_q, rest_q, whole;
  __device__ __forceinline__ Teacher(double q, int tokens, int vocab, int kind, bool drop)
      : list_q(q) {
    rest_q = tokens == vocab ? 0.0 : fmax(1.0 - q, kind == TISO_DISTILL_REVERSE ? kLeastRest : 0.0);
    if (drop) rest_q = 0.0;
    if (q != q) rest_q = q;  // NaN
    whole = drop ? (q > 0 ? 1.0 : 0.0) : q + rest_q;
  }
};

// The student's, from the parts' sums and maxima.
template <typename A>
struct Student {
  double rest_z, list_z;  // the parts' maxima less the row's, over t
  A s, rest_p, list_p;    // list_p: the probability of an e of 1

  __device__ __forceinline__ Student(const Part<A>& rest, A most, double list_e, double inv_temp) {
    const double base = base_of(max_acc(rest.m, most));
    rest_z = (static_cast<double>(base_of(rest.m)) - base) * inv_temp;
    list_z = (static_cast<double>(base_of(most)) - base) * inv_temp;
    // a part that is empty, or hidden, has a sum of 0 and no maximum
    const A of_rest = rest.s == A(0) ? A(0) : exp_as(A(0), rest_z) * rest.s;
    const A of_list = list_e == 0 ? A(0) : exp_as(A(0), list_z);
    s = of_rest + of_list * static_cast<A>(list_e);
    rest_p = of_rest / s;
    list_p = of_list / s;
  }
};

// An entry's q, log q and log m (m the mixture of both), the q's renormalised where the rest is
// dropped.
template <typename A>
__device__ __forceinline__ void entry_of(const DistillArgs<A>& p, const ListSpace<A>& space, int k,
                                         const Settled& row, double prob, double& q, double& log_q,
                                         double& log_m) {
  q = space.q[k];
  log_q = space.log_q[k];
  if (p.drop && row.list_q > 0) {
    q /= row.list_q;
    log_q -= log(row.list_q);
  }
  log_m = p.kind == TISO_DISTILL_JENSEN ? log(p.mix * q + (1 - p.mix) * prob) : log_q;
}

// The steps after a row's sum, by a warp: the row's divergence, what the list's gradient is made of
// into `settled`, and the rest's factor.
template <int kThreads, typename A>
__device__ __forceinline__ double settle(const DistillArgs<A>& p, const ListSpace<A>& space,
                                         const Part<A>& rest, int vocab, double inv_temp,
                                         double& factor) {
  ListSums sums = space.sums[0];
  for (int i = 1; i < warps_of<kThreads>(p.top); ++i) {
    const ListSums& more = space.sums[i];
    sums.q += more.q;
    sums.q_log_q += more.q_log_q;
    sums.q_z += more.q_z;
    sums.e += more.e;
    sums.e_far += more.e_far;
    sums.tokens += more.tokens;
  }
  const Teacher teacher(sums.q, sums.tokens, vocab, p.kind, p.drop);
  const A most = most_of<kThreads>(space, p.top);
  const Student<A> student(rest, most, sums.e, inv_temp);
  const double log_s = log(static_cast<double>(student.s));
  const double rest_log_p = student.rest_z + log(static_cast<double>(rest.s)) - log_s;
  const double rest_log_q = log(teacher.rest_q), rest_p = student.rest_p;
  const double unknown = *space.bad || student.s == A(0) ? nan_of(0.0) : 0.0;
  Settled row{space.settled->c + unknown, student.list_p, student.list_z - log_s, 0.0, sums.q,
              teacher.whole};
  double d;
  if (p.drop && sums.q == 0) {  // nothing to compare with
    d = factor = row.c = unknown;
  } else if (p.kind == TISO_DISTILL_FORWARD) {
    // p_v (f - sum P f) = p_v whole - q_v
    const double each = p.drop ? 1 / sums.q : 1.0, shift = p.drop ? log(sums.q) : 0.0;
    d = each * (sums.q_log_q - sums.q_z) - each * sums.q * (shift + row.log_p) +
        product(teacher.rest_q, rest_log_q - rest_log_p);
    factor = teacher.whole * rest_p - teacher.rest_q;
  } else if (p.kind == TISO_DISTILL_REVERSE) {
    const double rest_f = rest_log_p - rest_log_q;
    d = row.mean = row.p * (sums.e_far + sums.e * row.log_p) + product(rest_p, rest_f);
    factor = product(rest_p, rest_f - row.mean);
  } else {
    const double base = base_of(most);
    double mean = 0, cross = 0;
    for (int k = threadIdx.x & 31; k < p.top; k += 32) {
      if (space.lead[k] != k) continue;
      const double prob = space.e[k] * row.p;
      const double log_p = (static_cast<double>(space.logit[k]) - base) * inv_temp + row.log_p;
      double q, log_q, log_m;
      entry_of(p, space, k, row, prob, q, log_q, log_m);
      mean += product(prob, (1 - p.mix) * (log_p - log_m));
      cross += product(q, log_q - log_m);
    }
    const double log_m = log(p.mix * teacher.rest_q + (1 - p.mix) * rest_p);
    const double rest_f = (1 - p.mix) * (rest_log_p - log_m);
    row.mean = sum_of_warp(mean) + product(rest_p, rest_f);
    d = row.mean + p.mix * (sum_of_warp(cross) + product(teacher.rest_q, rest_log_q - log_m));
    factor = product(rest_p, rest_f - row.mean);
  }
  factor = rest.s == A(0) ? unknown : row.c * factor / static_cast<double>(rest.s);
  __syncwarp();  // every lane has read the share
  if ((threadIdx.x & 31) == 0) *space.settled = row;
  return d + unknown;
}

// The gradient of an entry's token.
template <typename A>
__device__ __forceinline__ A gradient_of(const DistillArgs<A>& p, const ListSpace<A>& space, int k,
                                         const Settled& row, A most, double inv_temp) {
  const double prob = space.e[k] * row.p;
  double q, log_q, log_m;
  if (p.kind == TISO_DISTILL_FORWARD) {
    q = space.q[k];
    if (p.drop && row.list_q > 0) q /= row.list_q;
    return static_cast<A>(row.c * (prob * row.whole - q));
  }
  entry_of(p, space, k, row, prob, q, log_q, log_m);
  const double z = (static_cast<double>(space.logit[k]) - static_cast<double>(base_of(most))) * inv_temp;
  const double f = (p.kind == TISO_DISTILL_JENSEN ? 1 - p.mix : 1.0) * (z + row.log_p - log_m);
  return static_cast<A>(row.c * product(prob, f - row.mean));
}

// The gradient of the rest: exp((x - base) / t) scale.
template <typename A>
struct RestSlope {
  A base, scale, k;
  __device__ __forceinline__ A at(A x, int) const { return mul_rn(scaled_exp(x - base, k), scale); }
};

template <typename T, typename A>
__device__ __forceinline__ uint4 slope_vector(const uint4& q, const RestSlope<A>& slope) {
  A x[RowView<T>::E];
  unpack<T>(q, x);
  exponentials(x, slope.base, slope.k);
  scale_by(x, slope.scale);
  return pack<T>(x);
}

template <int kThreads, typename T, typename A>
__device__ __forceinline__ void write_rest_of_tile(const RowView<T>& r, int tile, int tid,
                                                   const RestSlope<A>& slope) {
  const int v = tile + tid;
  uint4* to = reinterpret_cast<uint4*>(r.g + r.head) + v;
#pragma unroll
  for (int i = 0; i < kBatch; ++i)
    if (v + i * kThreads < r.vectors)
      store_once(to + i * kThreads, slope_vector<T>(load_vector(r, v + i * kThreads), slope));
}

// The list's gradients, over what the pass wrote in their places. The threads have met since.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void write_list(const Rows& a, const DistillArgs<A>& p, int64_t r,
                                           const RowView<T>& view, const Place<kThreads>& place,
                                           double inv_temp, bool with_grad,
                                           const ListSpace<A>& space) {
  const Team<kThreads> team{place.tid};
  const Settled row = *space.settled;
  const A most = most_of<kThreads>(space, p.top);
  for (int k = team.tid; k < p.top; k += kThreads) {
    if (space.lead[k] != k) continue;
    const A value = gradient_of(p, space, k, row, most, inv_temp);
    space.gradient[k] = value;
    const Spot<kThreads, T> spot(view, place.ctas, space.id[k]);
    if (with_grad && spot.cta == place.cta)
      view.g[space.id[k]] = from_acc<T>(static_cast<A>(value * p.upstream));
  }
  if (!p.listed || place.cta != 0) return;
  team.sync();
  for (int k = team.tid; k < p.top; k += kThreads)
    p.listed[r * p.top + k] = space.lead[k] < 0 ? A(0) : space.gradient[space.lead[k]];
}

// A row's results but for the means' terms.
template <typename A>
__device__ __forceinline__ void write_row(const DistillArgs<A>& p, int64_t r, const Part<A>& rest,
                                          double d, double factor) {
  p.divergence[r] = static_cast<A>(d);
  if (p.coef) {
    p.coef[r] = factor;
    p.stats[2 * r] = base_of(rest.m);
    p.stats[2 * r + 1] = A(0);
  }
}

template <typename A>
__device__ __forceinline__ void write_left_out(const DistillArgs<A>& p, int64_t r) {
  p.divergence[r] = A(0);
  if (p.coef) p.stats[2 * r + 1] = A(kLeftOut);
}

// The row's share of the loss, into `settled`, by one thread while the row is read.
template <typename A>
__device__ __forceinline__ void read_share(const DistillArgs<A>& p, A w, double inv_temp,
                                           const ListSpace<A>& space) {
  cudaGridDependencySynchronize();  // the total's kernel is done
  const double total = *p.total;
  space.settled->c = total != 0 ? static_cast<double>(w) / total * inv_temp : 0.0;
}

template <typename T, typename A>
__device__ __forceinline__ RowView<T> distill_view(const Rows& a, int64_t r, T* grad) {
  T* g = grad + r * a.vocab;
  return RowView<T>(row_at<T>(a, r), g, reinterpret_cast<uintptr_t>(g), a.vocab);
}

// Loss and gradient of a row by a CTA, or a cluster of them.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void distill_row(const Rows& a, const DistillArgs<A>& p, double inv_temp,
                                            A k, T* grad, int bit_words, bool& last) {
  constexpr int kTile = kBatch * kThreads;
  extern __shared__ uint4 shared[];
  __shared__ A slope_of[2];
  const Place<kThreads> place;
  const int64_t r = place.row;
  const RowView<T> view = distill_view<T, A>(a, r, grad);
  const A w = p.weights.at(r);
  if (w == A(0)) {
    if (place.first()) {
      write_left_out(p, r);
      p.terms[r] = A(0);
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
  const StagedTiles<kThreads, T> tiles(view, place, shared);
#pragma unroll
  for (int j = 0; j < kStages; ++j) tiles.copy(j);
  const ListSpace<A> space(shared + kStages * kTile, p.top);
  read_list(a, p, r, view, place, bit_words, inv_temp, space);
  if (place.tid == 0) read_share(p, w, inv_temp, space);

  Part<A> rest{lowest<A>(), A(0)};
  add_edge(rest, view, place, *space.edge_bits, k);
  if (tiles.staged == 0)
    for (int tile = place.cta * kTile, j = 0; tile < view.vectors; tile += place.ctas * kTile, ++j) {
      uint4 q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int v = tile + i * kThreads + place.tid;
        q[i] = v < view.vectors ? load_vector(view, v) : no_vector<T>();
      }
      add_rest<T>(rest, q, bits_of_tile<kThreads, T>(space.bits, j, place.tid), k);
    }
  for (int j = 0; j < tiles.whole; ++j) {
    uint4 q[kBatch];
    tiles.fetch(j, q);
    tiles.copy(j + kStages);
    add_rest<T>(rest, q, bits_of_tile<kThreads, T>(space.bits, j, place.tid), k);
  }
  if (tiles.cut) {
    uint4 q[kBatch];
    tiles.fetch_cut(q);
    add_rest<T>(rest, q, bits_of_tile<kThreads, T>(space.bits, tiles.whole, place.tid), k);
    close_group();
  }
  rest = join_warps<kThreads>(join_lanes<32>(rest, k), k);
  if (threadIdx.x < 32) {
    double factor;
    const double d = settle<kThreads>(p, space, rest, a.vocab, inv_temp, factor);
    if (place.tid == 0) {
      slope_of[0] = base_of(rest.m);
      slope_of[1] = static_cast<A>(factor * p.upstream);
    }
    if (place.first()) {
      write_row(p, r, rest, d, factor);
      p.terms[r] = static_cast<A>(static_cast<double>(w) * d);
      last = last_unit(p.done, a.rows);
    }
  }
  if (!grad && !p.listed) return;
  __syncthreads();
  if (grad) {
    const RestSlope<A> slope{slope_of[0], slope_of[1], k};
    if (tiles.cut) {
      uint4 q[kBatch];
      tiles.fetch(tiles.whole, q);
      tiles.copy(tiles.whole - kStages);
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (tiles.has(i))
          store_once(tiles.to(tiles.whole) + i * kThreads, slope_vector<T>(q[i], slope));
    }
    for (int j = tiles.whole - 1; j >= 0; --j) {
      uint4 q[kBatch];
      tiles.fetch(j, q);
      tiles.copy(j - kStages);
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        store_once(tiles.to(j) + i * kThreads, slope_vector<T>(q[i], slope));
    }
    write_edge(view, place.edge(), slope);
    if (tiles.staged == 0)
      for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile)
        write_rest_of_tile<kThreads>(view, tile, place.tid, slope);
    __syncthreads();
  }
  write_list(a, p, r, view, place, inv_temp, grad != nullptr, space);
}

template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(kThreads, kSmThreads / kThreads)
    distill_kernel(Rows a, DistillArgs<A> p, double inv_temp, A k, T* grad, int bit_words) {
  __shared__ bool last;  // written by thread 0 alone
  if (threadIdx.x == 0) last = false;
  distill_row<kThreads>(a, p, inv_temp, k, grad, bit_words, last);
  __syncthreads();
  if (last) write_means<1>(p.terms, *p.total, p.out, a.rows);
}

// Short rows: a warp to a row.
template <typename T, typename A>
__global__ void __launch_bounds__(32 * kRowWarps)
    distill_warp_kernel(Rows a, DistillArgs<A> p, double inv_temp, A k, T* grad, int bit_words) {
  constexpr int kTile = kBatch * 32;
  extern __shared__ uint4 shared[];
  __shared__ A terms[kRowWarps];
  __shared__ bool last;
  const Place<32> place;
  const int64_t r = place.row;
  const int warp = threadIdx.x / 32;
  const A w = r < a.rows ? p.weights.at(r) : A(0);
  if (place.tid == 0) terms[warp] = A(0);
  if (w != A(0)) {
    const RowView<T> view = distill_view<T, A>(a, r, grad);
    const ListSpace<A> space(
        reinterpret_cast<char*>(shared) + warp * ListSpace<A>::bytes(p.top, 4 * bit_words), p.top);
    read_list(a, p, r, view, place, bit_words, inv_temp, space);
    if (place.tid == 0) read_share(p, w, inv_temp, space);
    Part<A> rest{lowest<A>(), A(0)};
    add_edge(rest, view, place, *space.edge_bits, k);
    for (int tile = 0, j = 0; tile < view.vectors; tile += kTile, ++j) {
      uint4 q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int v = tile + i * 32 + place.tid;
        q[i] = v < view.vectors ? load_vector(view, v) : no_vector<T>();
      }
      add_rest<T>(rest, q, bits_of_tile<32, T>(space.bits, j, place.tid), k);
    }
    rest = join_lanes<32>(rest, k);
    __syncwarp();
    double factor;
    const double d = settle<32>(p, space, rest, a.vocab, inv_temp, factor);
    if (place.tid == 0) {
      write_row(p, r, rest, d, factor);
      terms[warp] = static_cast<A>(static_cast<double>(w) * d);
    }
    if (grad) {
      const RestSlope<A> slope{base_of(rest.m), static_cast<A>(factor * p.upstream), k};
      write_edge(view, place.edge(), slope);
      for (int tile = 0; tile < view.vectors; tile += kTile)
        write_rest_of_tile<32>(view, tile, place.tid, slope);
    }
    __syncwarp();
    if (grad || p.listed) write_list(a, p, r, view, place, inv_temp, grad != nullptr, space);
  } else if (r < a.rows) {
    if (place.tid == 0) write_left_out(p, r);
    if (grad) {
      const RowView<T> view = distill_view<T, A>(a, r, grad);
      zero_edge(view, place.edge());
      for (int tile = 0; tile < view.vectors; tile += kTile) zero_tile<32>(view, tile, place.tid);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    A sum = A(0);
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) sum += terms[i];
    p.terms[blockIdx.x] = sum;
    cudaGridDependencySynchronize();
    last = last_unit(p.done, gridDim.x);
  }
  __syncthreads();
  if (last) write_means<1>(p.terms, *p.total, p.out, gridDim.x);
}

// The gradient for another upstream gradient than the expected one, from what the loss left; nothing
// is written where it is that one. A warp or a CTA (kThreads) takes a tile, `tiles` to the row.
template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(256)
    distill_grad_kernel(Rows a, const int64_t* ids, int top, A k, const double* coef, const A* stats,
                        const A* listed, double expected, const A* upstream, T* grad, int tiles) {
  const A up = *upstream;
  if (up == static_cast<A>(expected)) return;
  constexpr int kGroups = 256 / kThreads, kTile = kBatch * kThreads, E = RowView<T>::E;
  const Team<kThreads> team{static_cast<int>(threadIdx.x % kThreads)};
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kGroups + threadIdx.x / kThreads;
       i < a.rows * tiles; i += static_cast<int64_t>(gridDim.x) * kGroups) {
    const int64_t r = i / tiles;
    const int tile = static_cast<int>(i % tiles) * kTile;
    T* g = grad + r * a.vocab;
    const RowView<T> view(row_at<T>(a, r), g, reinterpret_cast<uintptr_t>(g), a.vocab);
    const int edge = tile == 0 ? team.tid : kNoEdge;
    if (stats[2 * r + 1] < A(0)) {
      zero_edge(view, edge);
      zero_tile<kThreads>(view, tile, team.tid);
      continue;
    }
    const RestSlope<A> slope{stats[2 * r], static_cast<A>(coef[r] * up), k};
    write_edge(view, edge, slope);
    write_rest_of_tile<kThreads>(view, tile, team.tid, slope);
    team.sync();
    for (int j = team.tid; j < top; j += kThreads) {
      const int64_t id = ids[r * top + j];
      if (id == a.ignore || id < 0 || id >= a.vocab) continue;
      const int v = static_cast<int>(id) - view.head;
      const bool single = v < 0 || v >= view.vectors * E;
      if (single ? tile == 0 : v / E / kTile * kTile == tile)
        view.g[id] = from_acc<T>(static_cast<A>(listed[r * top + j] * static_cast<double>(up)));
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Host side

// Bits of the vectors of a CTA's share of `vectors`, in bytes.
template <typename T>
int64_t bit_bytes(int64_t vectors, int threads, int ctas) {
  const int64_t tile = int64_t{kBatch} * threads, tiles = (vectors + tile - 1) / tile;
  return (tiles + ctas - 1) / ctas * tile * RowView<T>::E / 8;
}

template <typename T, int kThreads>
int launch_distill_rows(const Rows& a, const DistillArgs<typename AccOf<T>::type>& p,
                        double inv_temp, T* grad, int sms, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr int64_t kStaged = int64_t{kStages} * kBatch * kThreads * 16;
  const int64_t vectors = a.vocab / RowView<T>::E;
  int ctas = ctas_for(a.rows, vectors, kThreads, sms);
  while (ctas < 8 && int64_t{sms} * (kSmThreads / kThreads) * vectors * 16 / ctas > kRowsInL2)
    ctas *= 2;
  while (ctas < 8 && bit_bytes<T>(vectors, kThreads, ctas) > kSharedForBits) ctas *= 2;
  const int64_t bits = bit_bytes<T>(vectors, kThreads, ctas);
  if (bits > kSharedForBits)
    return report_error(TISO_ERR_ARGUMENT, "a vocabulary too large for the distillation loss");
  const size_t shared = kStaged + ListSpace<A>::bytes(p.top, static_cast<int>(bits));
  const auto kernel = distill_kernel<T, A, kThreads>;
  const int rc = allow_shared(reinterpret_cast<const void*>(kernel),
                              kStaged + ListSpace<A>::bytes(kMostListed, kSharedForBits));
  if (rc) return rc;
  return launch_clusters(kernel, a.rows, ctas, kThreads, shared, true, st, "distill_kernel launch", a,
                         p, inv_temp, exp_factor(A(0), inv_temp), grad, static_cast<int>(bits / 4));
}

template <typename T>
int launch_distill(const Rows& a, const DistillArgs<typename AccOf<T>::type>& p, double inv_temp,
                   T* grad, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int64_t vectors = a.vocab / RowView<T>::E;
  const int sms = sm_count();
  if (by_warps(a.rows, vectors, 1536, sms)) {
    const int bits = static_cast<int>(bit_bytes<T>(vectors, 32, 1));
    const size_t shared = size_t{kRowWarps} * ListSpace<A>::bytes(p.top, bits);
    const auto kernel = distill_warp_kernel<T, A>;
    const int rc = allow_shared(reinterpret_cast<const void*>(kernel),
                                size_t{kRowWarps} * ListSpace<A>::bytes(kMostListed, 1536 * 16 / 8));
    if (rc) return rc;
    return launch_clusters(kernel, (a.rows + kRowWarps - 1) / kRowWarps, 1, 32 * kRowWarps, shared,
                           true, st, "distill_warp_kernel launch", a, p, inv_temp,
                           exp_factor(A(0), inv_temp), grad, bits / 4);
  }
  return launch_distill_rows<T, 256>(a, p, inv_temp, grad, sms, st);
}

template <typename T>
int run_distill(const Rows& a, const tiso_distill_args* q, double inv_temp, void* divergence,
                double* coef, void* stats, void* listed, void* out, void* grad, void* workspace,
                cudaStream_t st) {
  using A = typename AccOf<T>::type;
  DistillArgs<A> p{};
  p.weights = weights_of<A>(q->ids, q->top, a.ignore, q->weight, q->weight_is_byte);
  p.ids = q->ids;
  p.logps = static_cast<const A*>(q->logps);
  p.top = static_cast<int>(q->top);
  p.kind = q->kind;
  p.drop = q->drop != 0;
  p.mix = q->mix;
  p.upstream = static_cast<A>(q->upstream);
  p.divergence = static_cast<A*>(divergence);
  p.coef = coef;
  p.stats = static_cast<A*>(stats);
  p.listed = static_cast<A*>(listed);
  p.out = static_cast<A*>(out);
  p.total = static_cast<double*>(workspace);
  p.done = reinterpret_cast<unsigned*>(p.total + 1);
  p.terms = reinterpret_cast<A*>(p.total + 2);
  int rc = launch_total(p.weights, a.rows, p.total, p.done, p.out, 1, st);
  if (rc || a.rows == 0) return rc;
  return launch_distill<T>(a, p, inv_temp, static_cast<T*>(grad), st);
}

template <typename T>
int run_distill_grad(const Rows& a, const int64_t* ids, int top, double inv_temp, const double* coef,
                     const void* stats, const void* listed, double expected, const void* upstream,
                     void* grad, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int vectors = a.vocab / RowView<T>::E;
  const int sms = sm_count();
  const bool by_warp = by_warps(a.rows, vectors, 768, sms);
  const int tile = kBatch * (by_warp ? 32 : 256);
  const int tiles = vectors > tile ? (vectors + tile - 1) / tile : 1;
  const int64_t all = (a.rows * tiles + (by_warp ? 7 : 0)) / (by_warp ? 8 : 1);
  // the launch may have nothing to do: no more CTAs than are resident
  const int64_t most = int64_t{sms} * 8;
  auto kernel = by_warp ? distill_grad_kernel<T, A, 32> : distill_grad_kernel<T, A, 256>;
  kernel<<<static_cast<unsigned>(all < most ? all : most), 256, 0, st>>>(
      a, ids, top, exp_factor(A(0), inv_temp), coef, static_cast<const A*>(stats),
      static_cast<const A*>(listed), expected, static_cast<const A*>(upstream),
      static_cast<T*>(grad), tiles);
  return launched("distill_grad_kernel launch");
}

int check_list(const tiso_rows* x, const int64_t* ids, int64_t top) {
  if (top < 1 || top > kMostListed)
    return report_error(TISO_ERR_ARGUMENT, "a list must have 1 to 128 entries");
  if (x->rows && !ids) return report_error(TISO_ERR_ARGUMENT, "ids must not be NULL");
  return TISO_OK;
}

}  // namespace
}  // namespace tiso

using namespace tiso;

extern "C" {

int tiso_distill_workspace_size(int dtype, int64_t rows, size_t* bytes) {
  return guarded([&]() -> int {
    if (!bytes) return report_error(TISO_ERR_ARGUMENT, "bytes is NULL");
    *bytes = 0;
    if (dtype < TISO_F16 || dtype > TISO_F64)
      return report_error(TISO_ERR_ARGUMENT, "dtype must be a tiso_dtype");
    if (rows < 0) return report_error(TISO_ERR_ARGUMENT, "need rows >= 0");
    *bytes = 16 + static_cast<size_t>(rows) * (dtype == TISO_F64 ? 8 : 4);
    return TISO_OK;
  });
}

int tiso_distill(int dtype, const tiso_rows* x, int64_t ignore_index, double temperature,
                 const tiso_distill_args* args, void* divergence, double* coef, void* stats,
                 void* listed, void* out, void* grad, void* workspace, size_t workspace_bytes,
                 void* stream) {
  return guarded([&]() -> int {
    int rc = check_rows(dtype, x, nullptr, grad, false);
    if (rc) return rc;
    if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
    if (!args) return report_error(TISO_ERR_ARGUMENT, "args is NULL");
    rc = check_list(x, args->ids, args->top);
    if (rc) return rc;
    if (args->kind < TISO_DISTILL_FORWARD || args->kind > TISO_DISTILL_JENSEN)
      return report_error(TISO_ERR_ARGUMENT, "kind must be a tiso_distill_kind");
    if (args->kind == TISO_DISTILL_REVERSE && args->drop)
      return report_error(TISO_ERR_ARGUMENT, "the reverse divergence needs the rest");
    if (args->kind == TISO_DISTILL_JENSEN && !(args->mix > 0 && args->mix < 1))
      return report_error(TISO_ERR_ARGUMENT, "mix must be between 0 and 1");
    if (x->rows && (!args->logps || !divergence))
      return report_error(TISO_ERR_ARGUMENT, "logps and divergence must not be NULL");
    if (x->rows && (!coef != !stats || !coef != !listed))
      return report_error(TISO_ERR_ARGUMENT, "coef, stats and listed go together");
    if (!out) return report_error(TISO_ERR_ARGUMENT, "out must not be NULL");
    size_t need = 0;
    rc = tiso_distill_workspace_size(dtype, x->rows, &need);
    if (rc) return rc;
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))
      return report_error(TISO_ERR_WORKSPACE,
                          "workspace missing, unaligned or smaller than tiso_distill_workspace_size");
    const Rows a = rows_of(x, nullptr, ignore_index);
    return by_type(dtype, [&](auto t) {
      return run_distill<decltype(t)>(a, args, 1.0 / temperature, divergence, coef, stats, listed, out,
                                      grad, workspace, static_cast<cudaStream_t>(stream));
    });
  });
}

int tiso_distill_grad(int dtype, const tiso_rows* x, int64_t ignore_index, double temperature,
                      const int64_t* ids, int64_t top, const double* coef, const void* stats,
                      const void* listed, double expected, const void* upstream, void* grad,
                      void* stream) {
  return guarded([&]() -> int {
    int rc = check_rows(dtype, x, nullptr, grad, false);
    if (rc) return rc;
    if (!(temperature > 0)) return report_error(TISO_ERR_ARGUMENT, "temperature must be > 0");
    rc = check_list(x, ids, top);
    if (rc) return rc;
    if (x->rows == 0) return TISO_OK;
    if (!coef || !stats || !listed || !upstream || !grad)
      return report_error(TISO_ERR_ARGUMENT,
                          "coef, stats, listed, upstream and grad must not be NULL");
    const Rows a = rows_of(x, nullptr, ignore_index);
    return by_type(dtype, [&](auto t) {
      return run_distill_grad<decltype(t)>(a, ids, static_cast<int>(top), 1.0 / temperature, coef,
                                           stats, listed, expected, upstream, grad,
                                           static_cast<cudaStream_t>(stream));
    });
  });
}

}  // extern "C"
