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
constexpr size_t kSharedForBits = 160 * 1024;
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
  A* terms;       // per row w D
  A* out;
  double* total;
  unsigned* done;
};

// Shared memory of the threads that work on a row.
template <typename A>
struct ListSpace {
  double *q, *log_q;     // the teacher's
  A *logit, *gradient;
  int *id, *lead;        // -1: no entry; the first entry of its id
  unsigned* bits;        // of this CTA's share of the vectors: a bit an element
  unsigned* edge_bits;   // of the single elements
  int *bad, *twice;      // an id out of range; an id listed again
  A *base, *scale;       // of the rest's gradient

  static size_t bytes(int top, size_t bits) {
    const size_t n = (top + 3) / 4 * 4;
    return n * (2 * sizeof(double) + 2 * sizeof(A) + 2 * sizeof(int)) + 4 * sizeof(double) +
           (bits + 15) / 16 * 16;
  }

  __device__ ListSpace(void* at, int top) {
    const int n = (top + 3) / 4 * 4;
    q = static_cast<double*>(at);
    log_q = q + n;
    A* numbers = reinterpret_cast<A*>(log_q + n);
    base = numbers;
    scale = numbers + 1;
    logit = numbers + (sizeof(A) == 4 ? 4 : 2);  // 16 bytes on
    gradient = logit + n;
    id = reinterpret_cast<int*>(gradient + n);
    lead = id + n;
    bad = lead + n;
    twice = bad + 1;
    edge_bits = reinterpret_cast<unsigned*>(bad + 2);
    bits = reinterpret_cast<unsigned*>(bad + 4);
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

// The part of the rest that a thread sees.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ Part<A> rest_part(const RowView<T>& r, const Place<kThreads>& place,
                                             const ListSpace<A>& space, A k) {
  constexpr int E = RowView<T>::E, kTile = kBatch * kThreads;
  const int e = place.edge();
  const A edge = e < r.edges && !(*space.edge_bits >> e & 1) ? to_acc(r.x[r.edge(e)]) : lowest<A>();
  Part<A> p{lowest<A>(), A(0)};
  int local = 0;
  for (int tile = place.cta * kTile; tile < r.vectors; tile += place.ctas * kTile, ++local) {
    const int v = tile + place.tid;
    uint4 q[kBatch];
    if (tile + kTile <= r.vectors) {
      load_vectors<kBatch, kThreads>(r, v, q);
    } else {
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        q[i] = v + i * kThreads < r.vectors ? load_vector(r, v + i * kThreads) : no_vector<T>();
    }
    const unsigned bits = bits_of_tile<kThreads, T>(space.bits, local, place.tid);
    if (bits) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) hide<T>(q[i], bits >> i * E & ((1u << E) - 1));
    }
    add_vectors<T>(p, q, k);
  }
  const A m = max_acc(p.m, edge), base = base_of(m);
  p.s = (p.m == m ? p.s : p.s * scaled_exp(p.m - base, k)) + scaled_exp(edge - base, k);
  p.m = m;
  return p;
}

__device__ __forceinline__ double sum_of_warp(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ __forceinline__ double product(double x, double y) { return x == 0 ? 0.0 : x * y; }

// The steps over the list by a warp, in double: the divergence, and in `space` the gradient of the
// listed tokens and the base and scale of the rest's, all times c.
template <typename A>
__device__ __forceinline__ double settle(const DistillArgs<A>& p, const ListSpace<A>& space,
                                         const Part<A>& rest, int vocab, double inv_temp, double c,
                                         double& scale) {
  constexpr int kEach = kMostListed / 32;
  const int lane = threadIdx.x & 31;
  double q[kEach], log_q[kEach], z[kEach];
  bool there[kEach];
  A m = rest.m;
  double listed_q = 0;
  int tokens = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int k = lane + 32 * i;
    there[i] = k < p.top && space.lead[k] == k;
    q[i] = there[i] ? space.q[k] : 0.0;
    log_q[i] = there[i] ? space.log_q[k] : 0.0;
    z[i] = there[i] ? static_cast<double>(space.logit[k]) : static_cast<double>(lowest<A>());
    m = max_acc(m, static_cast<A>(z[i]));
    listed_q += q[i];
    tokens += __popc(__ballot_sync(0xffffffffu, there[i]));
  }
  m = max_of_lanes<32>(m);
  listed_q = sum_of_warp(listed_q);
  // the student: z relative to the maximum, logarithms less log s
  const double base = static_cast<double>(base_of(m));
  double e[kEach], s = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    z[i] = (z[i] - base) * inv_temp;
    e[i] = there[i] ? exp(z[i]) : 0.0;
    s += e[i];
  }
  const double rest_z = (static_cast<double>(rest.m) - base) * inv_temp;
  const double rest_e = rest.s == A(0) ? 0.0 : exp(rest_z) * static_cast<double>(rest.s);
  s = sum_of_warp(s) + rest_e;
  const double log_s = log(s), rest_p = rest_e / s;
  const double rest_log_p = rest_z + log(static_cast<double>(rest.s)) - log_s;
  // the teacher
  double rest_q = tokens == vocab ? 0.0 : fmax(1.0 - listed_q, 0.0), whole = listed_q + rest_q;
  if (p.drop) {
    rest_q = 0.0;
    whole = listed_q > 0 ? 1.0 : 0.0;
    const double log_listed = log(listed_q);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      log_q[i] = q[i] > 0 ? log_q[i] - log_listed : log_q[i];
      q[i] = q[i] > 0 ? q[i] / listed_q : q[i];
    }
  } else if (p.kind == TISO_DISTILL_REVERSE && tokens < vocab) {
    rest_q = fmax(rest_q, kLeastRest);
  }
  if (listed_q != listed_q) rest_q = listed_q;  // NaN
  const double rest_log_q = log(rest_q);
  double d = 0, factor;
  if (p.kind == TISO_DISTILL_FORWARD) {
    // p_v (f - sum P f) = p_v whole - q_v
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      d += product(q[i], log_q[i] - (z[i] - log_s));
      if (there[i]) e[i] = e[i] / s * whole - q[i];
    }
    d = sum_of_warp(d) + product(rest_q, rest_log_q - rest_log_p);
    factor = rest_p * whole - rest_q;
  } else {
    const double a = p.kind == TISO_DISTILL_REVERSE ? 0.0 : p.mix;
    double f[kEach], mean = 0, cross = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const double prob = e[i] / s, log_p = z[i] - log_s;
      const double log_m = a == 0 ? log_q[i] : log(a * q[i] + (1 - a) * prob);
      e[i] = prob;
      f[i] = (1 - a) * (log_p - log_m);
      if (there[i]) {
        mean += product(prob, f[i]);
        cross += product(q[i], log_q[i] - log_m);
      }
    }
    const double log_m = a == 0 ? rest_log_q : log(a * rest_q + (1 - a) * rest_p);
    const double rest_f = (1 - a) * (rest_log_p - log_m);
    mean = sum_of_warp(mean) + product(rest_p, rest_f);
    d = mean + a * (sum_of_warp(cross) + product(rest_q, rest_log_q - log_m));
    if (a == 0) d = mean;
#pragma unroll
    for (int i = 0; i < kEach; ++i) e[i] = product(e[i], f[i] - mean);
    factor = product(rest_p, rest_f - mean);
  }
  const bool none = p.drop && listed_q == 0;  // nothing to compare with
  const double unknown = *space.bad || s == 0 ? nan_of(0.0) : 0.0;
  if (none) d = factor = 0;
  d += unknown;
  scale = rest.s == A(0) ? unknown : c * factor / static_cast<double>(rest.s) + unknown;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int k = lane + 32 * i;
    if (there[i]) space.gradient[k] = static_cast<A>(none ? unknown : c * e[i] + unknown);
  }
  if (lane == 0) {
    *space.base = base_of(rest.m);
    *space.scale = static_cast<A>(scale * p.upstream);
  }
  __syncwarp();
  return d;
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

// The list of row r into shared memory, and its bits. The threads have met when it returns.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void read_list(const Rows& a, const DistillArgs<A>& p, int64_t r,
                                          const RowView<T>& view, const Place<kThreads>& place,
                                          int bit_words, const ListSpace<A>& space) {
  const Team<kThreads> team{place.tid};
  for (int i = team.tid; i < bit_words; i += kThreads) space.bits[i] = 0;
  if (team.tid == 0) *space.bad = *space.twice = static_cast<int>(*space.edge_bits = 0u);
  team.sync();
  for (int k = team.tid; k < p.top; k += kThreads) {
    const int64_t id = p.ids[r * p.top + k];
    const bool listed = id != a.ignore, in = id >= 0 && id < a.vocab;
    if (listed && !in) *space.bad = 1;
    const double log_q = listed && in ? static_cast<double>(p.logps[r * p.top + k])
                                      : static_cast<double>(lowest<A>());
    space.id[k] = space.lead[k] = -1;
    space.log_q[k] = log_q;
    space.q[k] = exp(log_q);
    space.gradient[k] = A(0);
    if (!listed || !in) continue;
    space.id[k] = static_cast<int>(id);
    space.lead[k] = k;
    space.logit[k] = to_acc(view.x[id]);
    const Spot<kThreads, T> spot(view, place.ctas, static_cast<int>(id));
    if (spot.cta != place.cta) continue;
    unsigned* word = spot.edge ? space.edge_bits : space.bits + spot.bit / 32;
    if (atomicOr(word, 1u << spot.bit % 32) >> spot.bit % 32 & 1) *space.twice = 1;
  }
  team.sync();
  // the same id again: its probabilities are added up in its first entry. (A CTA of a cluster sees
  // only its own elements' bits, and looks through the list.)
  if (place.ctas == 1 && !*space.twice) return;
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

// Loss and gradient of a row by a CTA, or a cluster of them.
template <typename T, typename A, int kThreads>
__device__ __forceinline__ void distill_row(const Rows& a, const DistillArgs<A>& p, double inv_temp,
                                            A k, T* grad, int bit_words, bool& last) {
  constexpr int kTile = kBatch * kThreads;
  extern __shared__ uint4 shared[];
  const Place<kThreads> place;
  const Team<kThreads> team{place.tid};
  const int64_t r = place.row;
  T* g = grad + r * a.vocab;
  const RowView<T> view(row_at<T>(a, r), g, reinterpret_cast<uintptr_t>(g), a.vocab);
  const A w = p.weights.at(r);
  if (w == A(0)) {
    if (place.first()) {
      p.divergence[r] = p.terms[r] = A(0);
      if (p.coef) p.stats[2 * r + 1] = A(kLeftOut);
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
  const ListSpace<A> space(shared, p.top);
  read_list(a, p, r, view, place, bit_words, space);
  const Part<A> rest =
      join_warps<kThreads>(join_lanes<32>(rest_part<kThreads>(view, place, space, k), k), k);
  if (threadIdx.x < 32) {
    cudaGridDependencySynchronize();
    const double total = *p.total, c = total != 0 ? static_cast<double>(w) / total * inv_temp : 0.0;
    double scale;
    const double d = settle(p, space, rest, a.vocab, inv_temp, c, scale);
    if (place.first()) {
      p.divergence[r] = static_cast<A>(d);
      p.terms[r] = static_cast<A>(static_cast<double>(w) * d);
      if (p.coef) {
        p.coef[r] = scale;
        p.stats[2 * r] = base_of(rest.m);
        p.stats[2 * r + 1] = A(0);
      }
      last = last_unit(p.done, a.rows);
    }
  }
  if (!grad && !p.listed) return;
  team.sync();
  if (p.listed && place.cta == 0)
    for (int i = team.tid; i < p.top; i += kThreads)
      p.listed[r * p.top + i] = space.lead[i] < 0 ? A(0) : space.gradient[space.lead[i]];
  if (!grad) return;
  const RestSlope<A> slope{*space.base, *space.scale, k};
  if (place.edge() < view.edges) write_edge(view, place.edge(), slope);
  for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile)
    write_rest_of_tile<kThreads>(view, tile, place.tid, slope);
  team.sync();  // the listed tokens' gradients over what the pass wrote there
  for (int i = team.tid; i < p.top; i += kThreads) {
    if (space.lead[i] < 0) continue;
    const Spot<kThreads, T> spot(view, place.ctas, space.id[i]);
    if (spot.cta == place.cta && space.lead[i] == i)
      view.g[space.id[i]] = from_acc<T>(static_cast<A>(space.gradient[i] * p.upstream));
  }
}

template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(kThreads)
    distill_kernel(Rows a, DistillArgs<A> p, double inv_temp, A k, T* grad, int bit_words) {
  __shared__ bool last;  // written by thread 0 alone
  if (threadIdx.x == 0) last = false;
  distill_row<T, A, kThreads>(a, p, inv_temp, k, grad, bit_words, last);
  __syncthreads();
  if (last) write_means<1>(p.terms, *p.total, p.out, a.rows);
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

template <typename T>
int run_distill(const Rows& a, const tiso_distill_args* q, double inv_temp, void* divergence,
                double* coef, void* stats, void* listed, void* out, void* grad, void* workspace,
                cudaStream_t st) {
  using A = typename AccOf<T>::type;
  constexpr int kThreads = 256, kTile = kBatch * kThreads, E = RowView<T>::E;
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
  const int64_t vectors = a.vocab / E, tiles = (vectors + kTile - 1) / kTile;
  int ctas = ctas_for(a.rows, vectors, kThreads, sm_count());
  const auto bits = [&] { return static_cast<size_t>((tiles + ctas - 1) / ctas) * kTile * E / 8; };
  while (ctas < 8 && ListSpace<A>::bytes(p.top, bits()) > kSharedForBits) ctas *= 2;
  const size_t shared = ListSpace<A>::bytes(p.top, bits());
  if (shared > kSharedForBits)
    return report_error(TISO_ERR_ARGUMENT, "a vocabulary too large for the distillation loss");
  const auto kernel = distill_kernel<T, A, kThreads>;
  rc = allow_shared(reinterpret_cast<const void*>(kernel), kSharedForBits);
  if (rc) return rc;
  return launch_clusters(kernel, a.rows, ctas, kThreads, shared, true, st, "distill_kernel launch", a,
                         p, inv_temp, exp_factor(A(0), inv_temp), static_cast<T*>(grad),
                         static_cast<int>(bits() / 4));
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
