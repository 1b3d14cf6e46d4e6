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
// taken from the row's maximum it would underflow where the student is sure of a listed token. Each
// listed token is handed to the thread that reads its element, which puts -infinity in its place.
#include "rows.cuh"
#include "select.cuh"

namespace tiso {
namespace {

constexpr int kMostListed = 128;
// Resident at 48 registers a thread, which spill: 48 bytes of stores and 88 of loads for 16 bits, 104 and 112
// in float32. (A warp to a row, at 64: 40 and 80, 64 and 148.)
constexpr int kSmThreads = 1280;
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

__device__ __forceinline__ double sum_of_warp(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

__device__ __forceinline__ double product(double x, double y) { return x == 0 ? 0.0 : x * y; }

// Sums over the list's tokens, of a warp's entries: of q and of e = exp(z), z the logits from the
// largest of them, over t; `far` of q (log q - z), in the reverse divergence of e (z - log q).
template <typename A>
struct ListSums {
  double q, far, e;
  A most;
  int tokens;
};

// What the gradients are made of, once the row's sum is known.
struct Settled {
  double c;         // the row's share of the loss, over t
  double each;      // what the teacher's probabilities are multiplied with
  double log_each;  // its logarithm
  double whole;     // their sum with the rest's
  double p;         // of an exp(z), z from the largest logit of the list: its probability
  double log_p;     // of a z: its logarithm
  double mean;      // sum P f
  double factor;    // of the rest's gradient
};

constexpr int kListWarps = kMostListed / 32;

// The forward divergence's gradient has the differences p_v sum Q - q_v and P_rest sum Q - Q_rest, small
// beside their terms where the student is near its teacher: with the terms in float, rows that agree to
// 0.01 lose two digits of it. So float32 logits have them in double (4096 x 32000, lists of 128: 245 us
// for 239; 4096 x 131072, 64: 920 for 905). Logits of 16 bits have them in float: their own steps and the
// gradient's rounding are larger (in double 156 us for 149, and 8192 x 131072 935 for 900).
template <typename T>
constexpr bool kWide = sizeof(T) == 4;

// Shared memory of the kThreads threads that work on a row. An entry is handed to the thread that
// reads and writes its token's element (its owner): each thread has a chain of its entries.
template <typename A, int kThreads>
struct ListSpace {
  double *q, *log_q;     // the teacher's probabilities
  double* e;             // kWide, forward: in log_q's place the student's exp(z), z as in the warp's sums
  double* share;         // the row's share of the loss, over t
  ListSums<A>* sums;     // of each warp that has entries
  Settled* settled;
  A *logit, *gradient;
  int *id, *lead;        // -1: no entry; the first entry of its id
  int *next, *place;     // in its owner's chain; where among the owner's elements
  int* head;             // of each thread's chain
  int *bad, *twice;      // an id out of range; a token that is listed again

  static __host__ __device__ constexpr int entries(int top) { return (top + 3) / 4 * 4; }
  static __host__ __device__ constexpr int bytes(int top) {
    return entries(top) * static_cast<int>(2 * sizeof(double) + 2 * sizeof(A) + 4 * sizeof(int)) +
           static_cast<int>(kListWarps * sizeof(ListSums<A>) + sizeof(Settled)) + 16 +
           kThreads * 4 + 16;
  }

  __device__ ListSpace(void* at, int top) {
    const int n = entries(top);
    q = static_cast<double*>(at);
    e = log_q = q + n;
    share = log_q + n;
    sums = reinterpret_cast<ListSums<A>*>(share + 2);
    settled = reinterpret_cast<Settled*>(sums + kListWarps);
    logit = reinterpret_cast<A*>(settled + 1);
    gradient = logit + n;
    id = reinterpret_cast<int*>(gradient + n);
    lead = id + n;
    next = lead + n;
    place = next + n;
    head = place + n;
    bad = head + kThreads;
    twice = bad + 1;
  }
};

// The same with the staged tiles, in bytes (whole vectors).
template <typename A, int kThreads>
__host__ __device__ constexpr int row_bytes(int top) {
  return (kStages * kBatch * kThreads * 16 + ListSpace<A, kThreads>::bytes(top) + 15) / 16 * 16;
}

// An element's owner: of a CTA's tiles (every ctas-th) the thread that has its vector, of the single
// elements the thread of their number in the first CTA. place: its number among the owner's elements.
constexpr int kNoPlace = -1, kEdgePlace = -2;

template <int kThreads, typename T>
__device__ __forceinline__ int owner_of(const RowView<T>& r, const Place<kThreads>& place, int element,
                                        int& number) {
  constexpr int E = RowView<T>::E, kTile = kBatch * kThreads;
  if (element < r.head || element >= r.head + r.vectors * E) {
    number = place.cta == 0 ? kEdgePlace : kNoPlace;
    return element < r.head ? element : element - r.vectors * E;
  }
  const int v = (element - r.head) / E, tile = v / kTile, in = v % kTile;
  const int local = tile / place.ctas;
  number = tile - local * place.ctas == place.cta
               ? (local * kBatch + in / kThreads) * E + (element - r.head) % E
               : kNoPlace;
  return in % kThreads;
}

// A thread's listed elements: in which tiles (bit j mod 32), and whether its single element is one.
struct Own {
  unsigned tiles;
  bool edge;
};

// Calls fn(k, place) for the entries of a thread that this CTA has.
template <int kThreads, typename A, typename F>
__device__ __forceinline__ void for_own(const ListSpace<A, kThreads>& space, int tid, const F& fn) {
  for (int k = space.head[tid]; k >= 0; k = space.next[k])
    if (space.place[k] != kNoPlace) fn(k, space.place[k]);
}

// Row r's list is handed out. The threads have met when it returns.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ Own hand_out(const Rows& a, const DistillArgs<A>& p, int64_t r,
                                        const RowView<T>& view, const Place<kThreads>& place,
                                        const ListSpace<A, kThreads>& space) {
  constexpr int kOfTile = kBatch * RowView<T>::E;
  const Team<kThreads> team{place.tid};
  space.head[team.tid] = -1;
  if (team.tid == 0) *space.bad = *space.twice = 0;
  for (int k = team.tid; k < p.top; k += kThreads) {
    const int64_t id = p.ids[r * p.top + k];
    space.id[k] = id == a.ignore ? -1 : id >= 0 && id < a.vocab ? static_cast<int>(id) : -2;
  }
  team.sync();
  for (int k = team.tid; k < p.top; k += kThreads) {
    const int id = space.id[k];
    if (id == -2) *space.bad = 1;
    if (id < 0) continue;
    int number;
    const int owner = owner_of<kThreads>(view, place, id, number);
    space.place[k] = number;
    space.next[k] = atomicExch(space.head + owner, k);
  }
  team.sync();
  Own own{0, false};
  for (int k = space.head[team.tid]; k >= 0; k = space.next[k])
    for (int j = space.next[k]; j >= 0; j = space.next[j])
      if (space.id[j] == space.id[k]) *space.twice = 1;
  for_own(space, team.tid, [&](int, int number) {
    if (number == kEdgePlace) {
      own.edge = true;
    } else {
      own.tiles |= 1u << number / kOfTile % 32;
    }
  });
  return own;
}

// Warps with entries of a list.
template <int kThreads>
__device__ __forceinline__ int warps_of(int top) {
  return min((top + 31) / 32, kThreads / 32);
}

// The list's numbers and their sums, by each warp for its own entries (the others' are known after
// the threads' next meeting). kAgain: tokens are listed more than once, each counts in its first entry
// with the sum of its probabilities.
template <bool kAgain, int kThreads, typename T, typename A>
__device__ __forceinline__ void read_list(const DistillArgs<A>& p, int64_t r, const RowView<T>& view,
                                          const Place<kThreads>& place, double inv_temp,
                                          const ListSpace<A, kThreads>& space) {
  if (place.tid / 32 * 32 >= p.top) return;
  A most = lowest<A>();
  for (int i = place.tid; i < p.top; i += kThreads) {
    const int id = space.id[i];
    int lead = -1;
    if (id >= 0) {
      const A logit = to_acc(view.x[id]);
      double log_q = static_cast<double>(p.logps[r * p.top + i]), q = exp(log_q);
      lead = i;
      if constexpr (kAgain) {
        bool more = false;
        for (int j = 0; j < p.top; ++j) {
          if (space.id[j] != id || j == i) continue;
          if (j < i) {
            lead = min(lead, j);
          } else {
            q += exp(static_cast<double>(p.logps[r * p.top + j]));
            more = true;
          }
        }
        if (more) log_q = log(q);
      }
      space.logit[i] = logit;
      space.log_q[i] = log_q;
      space.q[i] = q;
      most = max_acc(most, logit);
    }
    space.lead[i] = lead;
  }
  most = max_of_lanes<32>(most);
  const double base = base_of(most);
  ListSums<A> sums{};
  for (int i = place.tid; i < p.top; i += kThreads) {
    if (space.lead[i] != i) continue;
    const double q = space.q[i], log_q = space.log_q[i];
    const double z = (static_cast<double>(space.logit[i]) - base) * inv_temp, e = exp(z);
    sums.q += q;
    sums.far += p.kind == TISO_DISTILL_REVERSE ? product(e, z - log_q) : product(q, log_q - z);
    sums.e += e;
    ++sums.tokens;
    if (kWide<T> && p.kind == TISO_DISTILL_FORWARD) space.e[i] = e;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    sums.q += __shfl_xor_sync(0xffffffffu, sums.q, d);
    sums.far += __shfl_xor_sync(0xffffffffu, sums.far, d);
    sums.e += __shfl_xor_sync(0xffffffffu, sums.e, d);
  }
  sums.tokens = __reduce_add_sync(0xffffffffu, sums.tokens);
  sums.most = most;
  if (place.tid % 32 == 0) space.sums[place.tid / 32] = sums;
}

// What the first steps need of the whole list: the sums of q and of exp(z), z from its largest logit,
// this one in the accumulation type.
template <typename A>
struct WholeList {
  double q;
  A e, most;
  int tokens;

  template <int kThreads>
  __device__ __forceinline__ WholeList(const ListSpace<A, kThreads>& space, int top, A k) {
    const ListSums<A>* sums = space.sums;
    const int warps = warps_of<kThreads>(top);
    q = sums[0].q;
    e = static_cast<A>(sums[0].e);
    most = sums[0].most;
    tokens = sums[0].tokens;
    if (warps > 1) {
      for (int i = 1; i < warps; ++i) {
        most = max_acc(most, sums[i].most);
        q += sums[i].q;
        tokens += sums[i].tokens;
      }
      e = A(0);
      for (int i = 0; i < warps; ++i)
        if (sums[i].e != 0)  // (a part that is hidden has no maximum)
          e += static_cast<A>(sums[i].e) * scaled_exp(base_of(sums[i].most) - base_of(most), k);
    }
  }
};

// The teacher's probabilities of the list and of the rest.
struct Teacher {
  double rest_q, whole;
  __device__ __forceinline__ Teacher(double q, int tokens, int vocab, int kind, bool drop) {
    rest_q = tokens == vocab ? 0.0 : fmax(1.0 - q, kind == TISO_DISTILL_REVERSE ? kLeastRest : 0.0);
    if (drop) rest_q = 0.0;
    if (q != q) rest_q = q;  // NaN
    whole = drop ? (q > 0 ? 1.0 : 0.0) : q + rest_q;
  }
};

// The student's, from the parts' sums and maxima; a part that is empty, or hidden, has a sum of 0 and no
// maximum. list_p: the probability of an e of 1.
template <typename A>
struct Student {
  A base, s, rest_p, list_p;

  __device__ __forceinline__ Student(const Part<A>& rest, A most, A list_e, A k)
      : base(base_of(max_acc(rest.m, most))) {
    const A of_rest = rest.s == A(0) ? A(0) : scaled_exp(base_of(rest.m) - base, k) * rest.s;
    const A of_list = list_e == A(0) ? A(0) : scaled_exp(base_of(most) - base, k);
    s = of_rest + of_list * list_e;
    rest_p = of_rest / s;
    list_p = of_list / s;
  }
};

// The same in double (kWide), by a warp: each exponential by a lane of its own, one quotient. own: the part
// of the list of this warp's entries. factor: (P_rest sum Q - Q_rest) / rest.s.
struct WideStudent {
  double list_p, part, factor;

  template <typename A, int kThreads>
  __device__ __forceinline__ WideStudent(const Teacher& teacher, const Part<A>& rest, A most,
                                         const ListSpace<A, kThreads>& space, int top, int own,
                                         double inv_temp) {
    const int lane = threadIdx.x & 31, parts = warps_of<kThreads>(top);
    const ListSums<A>& sums = space.sums[lane < parts ? lane : 0];
    const double base = base_of(most), d = (static_cast<double>(base_of(rest.m)) - base) * inv_temp;
    const double z = (static_cast<double>(base_of(sums.most)) - base) * inv_temp;
    const double e = exp(lane < kListWarps ? z : -fabs(d));
    // (a part that is hidden has no maximum)
    double list_e = lane >= parts || sums.e == 0 ? 0.0 : e * sums.e;
#pragma unroll
    for (int i = kListWarps / 2; i; i /= 2) list_e += __shfl_xor_sync(0xffffffffu, list_e, i);
    list_e = __shfl_sync(0xffffffffu, list_e, 0);
    part = __shfl_sync(0xffffffffu, sums.e == 0 ? 0.0 : e, own % kListWarps);
    const double less = __shfl_sync(0xffffffffu, e, kListWarps);
    const double rest_s = rest.s;
    const double of_rest = rest_s == 0 ? 0.0 : d < 0 && list_e != 0 ? less : 1.0;
    const double of_list = list_e == 0 ? 0.0 : d > 0 && rest_s != 0 ? less : 1.0;
    const double rest_e = of_rest * rest_s, s = rest_e + of_list * list_e;
    const double one = rest_s == 0 ? 1.0 : rest_s, r = 1 / (s * one);
    list_p = of_list * one * r;
    factor = rest_s == 0 ? 0.0 : (teacher.whole * rest_e - teacher.rest_q * s) * r;
  }
};

// The first steps after a row's sum, by every warp: what a gradient of the forward divergence is made
// of; without a logarithm, and in double only what cancels. part (kWide): what takes this warp's entries'
// exponentials from their largest logit to the list's.
template <typename T, typename A, int kThreads>
__device__ __forceinline__ Settled settle(const DistillArgs<A>& p, const ListSpace<A, kThreads>& space,
                                          const WholeList<A>& list, const Part<A>& rest, int vocab,
                                          const Place<kThreads>& place, double inv_temp, A k,
                                          double& part) {
  const Teacher teacher(list.q, list.tokens, vocab, p.kind, p.drop);
  const auto settled = [&](bool nothing) {
    Settled row{};
    row.c = *space.share;
    if (*space.bad || nothing) row.c = nan_of(0.0);
    row.each = p.drop ? (list.q > 0 ? 1 / list.q : list.q) : 1.0;  // nothing to compare with: 0
    row.whole = teacher.whole;
    return row;
  };
  // p_v (f - sum P f) = p_v whole - q_v
  if constexpr (kWide<T>) {
    Settled row = settled(rest.s == A(0) && list.e == A(0));
    if (p.kind != TISO_DISTILL_FORWARD) return row;
    const WideStudent student(teacher, rest, list.most, space, p.top, place.tid / 32, inv_temp);
    row.p = student.list_p;
    part = student.part;
    row.factor = row.c * student.factor;
    return row;
  } else {
    const Student<A> student(rest, list.most, list.e, k);
    Settled row = settled(student.s == A(0));
    row.p = student.list_p;
    const A factor = static_cast<A>(teacher.whole) * student.rest_p - static_cast<A>(teacher.rest_q);
    row.factor = static_cast<A>(row.c) * (rest.s == A(0) ? A(0) : factor / rest.s);
    return row;
  }
}

// The steps to the divergence, by a warp, in double (it is small beside its terms where the student is
// near the teacher); and what the gradients of the others than the forward one are made of. A lane for
// each exponential and logarithm that can be taken at once.
template <typename A, int kThreads>
__device__ __forceinline__ double settle_logs(const DistillArgs<A>& p,
                                              const ListSpace<A, kThreads>& space,
                                              const WholeList<A>& list, const Part<A>& rest, int vocab,
                                              double inv_temp, Settled& row) {
  const Teacher teacher(list.q, list.tokens, vocab, p.kind, p.drop);
  const int lane = threadIdx.x & 31;
  const auto of_lane = [](double v, int from) { return __shfl_sync(0xffffffffu, v, from); };
  const double most = base_of(list.most);
  // the list's sums with z from its largest logit
  double far = 0, e = 0;
  if (lane < warps_of<kThreads>(p.top)) {
    const ListSums<A> part = space.sums[lane];
    far = part.far;
    e = part.e;
    const double d = (static_cast<double>(base_of(part.most)) - most) * inv_temp;
    if (part.tokens > 0 && part.most != list.most) {
      const double f = e == 0 ? 0.0 : exp(d);
      if (p.kind == TISO_DISTILL_REVERSE) {
        far = f == 0 ? 0.0 : f * (far + d * e);
      } else if (part.q != 0) {
        far -= part.q * d;
      }
      e *= f;
    }
  }
#pragma unroll
  for (int d = kListWarps / 2; d; d /= 2) {
    far += __shfl_xor_sync(0xffffffffu, far, d);
    e += __shfl_xor_sync(0xffffffffu, e, d);
  }
  far = of_lane(far, 0);
  e = of_lane(e, 0);
  // both parts' sums from the row's maximum
  const double base = base_of(max_acc(rest.m, list.most)), rest_s = rest.s;
  const double rest_z = (static_cast<double>(base_of(rest.m)) - base) * inv_temp;
  const double list_z = (most - base) * inv_temp;
  const double z = lane == 0 ? rest_z : list_z, from_base = z == 0 ? 1.0 : exp(z);
  const double of_rest = rest_s == 0 ? 0.0 : of_lane(from_base, 0) * rest_s;
  const double of_list = e == 0 ? 0.0 : of_lane(from_base, 1), s = of_rest + of_list * e;
  const double rest_p = of_rest / s;
  const double logarithm = log(lane == 0 ? s : lane == 1 ? rest_s : lane == 2 ? teacher.rest_q : list.q);
  const double log_s = of_lane(logarithm, 0), rest_log_p = rest_z + of_lane(logarithm, 1) - log_s;
  const double rest_log_q = of_lane(logarithm, 2);
  row.log_each = p.drop ? -of_lane(logarithm, 3) : 0.0;
  row.log_p = list_z - log_s;
  double d, factor = 0;
  if (p.drop && list.q == 0) {  // nothing to compare with: 0, or NaN where the row's sum is
    row.c *= 0 * s;
    row.factor = row.c;
    return row.c;
  }
  if (p.kind == TISO_DISTILL_FORWARD) {
    d = row.each * far + row.each * list.q * (row.log_each - row.log_p) +
        product(teacher.rest_q, rest_log_q - rest_log_p);
    return row.c == row.c ? d : row.c;
  }
  if (p.kind == TISO_DISTILL_REVERSE) {
    const double rest_f = rest_log_p - rest_log_q;
    // (where the list has no probability log_p may be as far as the type's lowest value)
    d = row.mean = product(of_list / s, far + e * row.log_p) + product(rest_p, rest_f);
    factor = product(rest_p, rest_f - row.mean);
  } else {
    double mean = 0, cross = 0;
    for (int i = lane; i < p.top; i += 32) {
      if (space.lead[i] != i) continue;
      const double log_p = (static_cast<double>(space.logit[i]) - most) * inv_temp + row.log_p;
      const double prob = exp(log_p), q = space.q[i] * row.each;
      const double log_m = log(p.mix * q + (1 - p.mix) * prob);
      mean += product(prob, (1 - p.mix) * (log_p - log_m));
      cross += product(q, space.log_q[i] + row.log_each - log_m);
    }
    const double log_m = log(p.mix * teacher.rest_q + (1 - p.mix) * rest_p);
    const double rest_f = (1 - p.mix) * (rest_log_p - log_m);
    row.mean = sum_of_warp(mean) + product(rest_p, rest_f);
    d = row.mean + p.mix * (sum_of_warp(cross) + product(teacher.rest_q, rest_log_q - log_m));
    factor = product(rest_p, rest_f - row.mean);
  }
  row.factor = rest.s == A(0) ? 0 * row.c : row.c * factor / rest_s;
  return row.c == row.c ? d : row.c;
}

// The gradients of the list's tokens, by the threads of their entries.
template <typename T, int kThreads, typename A>
__device__ __forceinline__ void list_gradients(const DistillArgs<A>& p, int64_t r,
                                               const Place<kThreads>& place, double inv_temp, A k,
                                               const Settled& row, double part, A most,
                                               const ListSpace<A, kThreads>& space) {
  for (int i = place.tid; i < p.top; i += kThreads) {
    const int lead = space.lead[i];
    A value = A(0);
    if (lead >= 0) {
      const A z = space.logit[lead] - base_of(most);
      const double q = space.q[lead] * row.each;
      if (p.kind == TISO_DISTILL_FORWARD) {
        double e;
        if constexpr (!kWide<T>) {
          e = scaled_exp(z, k);
        } else if (kThreads == 32 || lead / 32 == place.tid / 32) {
          e = space.e[lead] * part;
        } else {  // listed again, first among another warp's entries
          e = exp((static_cast<double>(space.logit[lead]) - static_cast<double>(base_of(most))) * inv_temp);
        }
        value = static_cast<A>(row.c * (e * row.p * row.whole - q));
      } else {
        const double log_p =
            (static_cast<double>(space.logit[lead]) - static_cast<double>(base_of(most))) * inv_temp +
            row.log_p;
        const double prob = exp(log_p);
        const double f = p.kind == TISO_DISTILL_REVERSE
                             ? log_p - space.log_q[lead]
                             : (1 - p.mix) * (log_p - log(p.mix * q + (1 - p.mix) * prob));
        value = static_cast<A>(row.c * product(prob, f - row.mean));
      }
    }
    space.gradient[i] = value;
    if (p.listed && place.cta == 0) p.listed[r * p.top + i] = value;
  }
}

// Over what the pass wrote in their places. The threads have met since.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void write_list(const DistillArgs<A>& p, const RowView<T>& view,
                                           const Place<kThreads>& place,
                                           const ListSpace<A, kThreads>& space) {
  for (int i = place.tid; i < p.top; i += kThreads)
    if (space.lead[i] == i && space.place[i] != kNoPlace)
      view.g[space.id[i]] = from_acc<T>(static_cast<A>(space.gradient[i] * p.upstream));
}

// ---------------------------------------------------------------------------------------------
// The row's passes

// -infinity for the listed elements of a tile that came through shared memory.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void hide_staged(const StagedTiles<kThreads, T>& tiles, int j, const Own& own,
                                            const ListSpace<A, kThreads>& space) {
  constexpr int E = RowView<T>::E, kOfTile = kBatch * E;
  if (!(own.tiles >> j % 32 & 1)) return;
  for_own(space, tiles.tid, [&](int, int number) {
    if (number < 0 || number / kOfTile != j) return;
    const T none = from_acc<T>(lowest<A>());
    char* vector = reinterpret_cast<char*>(tiles.at(j) + number % kOfTile / E * kThreads);
    memcpy(vector + number % E * sizeof(T), &none, sizeof(T));
  });
}

// The same for a tile's vectors in registers.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void hide_loaded(uint4 (&q)[kBatch], int tid, int j, const Own& own,
                                            const ListSpace<A, kThreads>& space) {
  constexpr int E = RowView<T>::E, kOfTile = kBatch * E;
  if (!(own.tiles >> j % 32 & 1)) return;
  const uint4 none = no_vector<T>();
  const uint32_t* n = reinterpret_cast<const uint32_t*>(&none);
  for_own(space, tid, [&](int, int number) {
    if (number < 0 || number / kOfTile != j) return;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&q[i]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (sizeof(T) == 2) {
          const uint32_t gone = number % 2 ? 0xffff0000u : 0xffffu;
          if (number % kOfTile / 2 == 4 * i + c) w[c] = (w[c] & ~gone) | (n[c] & gone);
        } else if constexpr (sizeof(T) == 4) {
          if (number % kOfTile == 4 * i + c) w[c] = n[c];
        } else {
          if (number % kOfTile == 2 * i + c / 2) w[c] = n[c];
        }
      }
    }
  });
}

// The rest's sum over tiles that are loaded directly.
template <int kThreads, typename T, typename A>
__device__ __forceinline__ void add_loaded(Part<A>& rest, const RowView<T>& view,
                                           const Place<kThreads>& place, const Own& own,
                                           const ListSpace<A, kThreads>& space, A k) {
  constexpr int kTile = kBatch * kThreads;
  for (int tile = place.cta * kTile, j = 0; tile < view.vectors; tile += place.ctas * kTile, ++j) {
    uint4 q[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int v = tile + i * kThreads + place.tid;
      q[i] = v < view.vectors ? load_vector(view, v) : no_vector<T>();
    }
    hide_loaded<kThreads, T>(q, place.tid, j, own, space);
    add_vectors<T>(rest, q, k);
  }
}

// Adds one of the single elements, unless it is listed.
template <typename T, int kThreads, typename A>
__device__ __forceinline__ void add_edge(Part<A>& p, const RowView<T>& r, const Place<kThreads>& place,
                                         const Own& own, A k) {
  const int e = place.edge();
  const A edge = e < r.edges && !own.edge ? to_acc(r.x[r.edge(e)]) : lowest<A>();
  const A m = max_acc(p.m, edge), base = base_of(m);
  p.s = (p.m == m ? p.s : p.s * scaled_exp(p.m - base, k)) + scaled_exp(edge - base, k);
  p.m = m;
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

// A row's results but for the means' terms. factor: of the rest's gradient for an upstream one of 1.
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

// The row's share of the loss, by one thread while the row is read.
template <typename A, int kThreads>
__device__ __forceinline__ void read_share(const DistillArgs<A>& p, A w, double inv_temp,
                                           const ListSpace<A, kThreads>& space) {
  cudaGridDependencySynchronize();  // the total's kernel is done
  const double total = *p.total;
  *space.share = total != 0 ? static_cast<double>(w) / total * inv_temp : 0.0;
}

template <typename T>
__device__ __forceinline__ RowView<T> distill_view(const Rows& a, int64_t r, T* grad) {
  T* g = grad + r * a.vocab;
  return RowView<T>(row_at<T>(a, r), g, reinterpret_cast<uintptr_t>(g), a.vocab);
}

// A row that is left out: its gradient is zeros.
template <int kThreads, typename T>
__device__ __forceinline__ void zero_row(const RowView<T>& view, const Place<kThreads>& place) {
  constexpr int kTile = kBatch * kThreads;
  zero_edge(view, place.edge());
  for (int tile = place.cta * kTile; tile < view.vectors; tile += place.ctas * kTile)
    zero_tile<kThreads>(view, tile, place.tid);
}

// Loss and gradient of a row by a warp, a CTA, or a cluster of them: the rest's sum, the few steps over
// the list, the gradient from a second read that does not reach memory. 8192 x 131072 bf16, lists of 64, a
// tenth left out, in 855 us: 0.73 of the copy bandwidth for each byte once, DRAM traffic 3 % over that; 108
// M warp instructions for 1350 such rows, 64 % of the issue slots and 59 % of the exponential unit
// busy, a quarter of the warps' time at the CTA's meetings. In CTAs of 256: 128 and 512 threads took 955 and 900
// us where these took 839; of five CTAs to the SM, six (40 registers) 888. finish(d) is called by one thread
// with the row's divergence, after the row's other results are written.
template <int kThreads, typename T, typename A, typename F>
__device__ __forceinline__ void distill_row(const Rows& a, const DistillArgs<A>& p, double inv_temp,
                                            A k, T* grad, const Place<kThreads>& place, A w,
                                            uint4* shared, const F& finish) {
  constexpr int kTile = kBatch * kThreads;
  const Team<kThreads> team{place.tid};
  const int64_t r = place.row;
  const RowView<T> view = distill_view<T>(a, r, grad);
  const StagedTiles<kThreads, T> tiles(view, place, shared);
#pragma unroll
  for (int j = 0; j < kStages; ++j) tiles.copy(j);
  const ListSpace<A, kThreads> space(shared + kStages * kTile, p.top);
  const Own own = hand_out(a, p, r, view, place, space);
  read_list<false>(p, r, view, place, inv_temp, space);
  if (place.tid == kThreads - 1) read_share(p, w, inv_temp, space);

  Part<A> rest{lowest<A>(), A(0)};
  add_edge(rest, view, place, own, k);
  if (tiles.staged == 0) add_loaded(rest, view, place, own, space, k);
  for (int j = 0; j < tiles.whole; ++j) {
    uint4 q[kBatch];
    tiles.arrived();
    hide_staged(tiles, j, own, space);
    tiles.read(j, q);
    tiles.copy(j + kStages);
    add_vectors<T>(rest, q, k);
  }
  if (tiles.cut) {
    uint4 q[kBatch];
    tiles.arrived();
    hide_staged(tiles, tiles.whole, own, space);
    tiles.read_cut(q);
    add_vectors<T>(rest, q, k);
    close_group();
  }
  rest = join_warps<kThreads>(join_lanes<32>(rest, k), k);
  if constexpr (kThreads == 32) team.sync();
  if (*space.twice) {
    read_list<true>(p, r, view, place, inv_temp, space);
    team.sync();
  }
  const WholeList<A> list(space, p.top, k);
  // every warp takes the few steps to the rest's factor by itself, where they need no logarithm
  double part = 1;
  Settled row = settle<T>(p, space, list, rest, a.vocab, place, inv_temp, k, part);
  const auto write_results = [&](double d) {
    write_row(p, r, rest, d, row.factor);
    finish(d);
  };
  if (p.kind != TISO_DISTILL_FORWARD) {
    double d = 0;
    if (place.tid < 32) {
      d = settle_logs(p, space, list, rest, a.vocab, inv_temp, row);
      if (place.tid == 0) *space.settled = row;
    }
    team.sync();
    row = *space.settled;
    if (place.first()) write_results(d);
  }
  if (grad || p.listed) list_gradients<T>(p, r, place, inv_temp, k, row, part, list.most, space);
  if (p.kind == TISO_DISTILL_FORWARD && place.tid >= kThreads - 32 && place.cta == 0) {
    // by the last warp: the first ones have the list
    Settled all = row;
    const double d = settle_logs(p, space, list, rest, a.vocab, inv_temp, all);
    if (place.tid == kThreads - 32) write_results(d);
  }
  if (!grad) return;
  const RestSlope<A> slope{base_of(rest.m), static_cast<A>(row.factor * p.upstream), k};
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
  team.sync();
  write_list(p, view, place, space);
}

template <typename T, typename A, int kThreads>
__global__ void __launch_bounds__(kThreads, kSmThreads / kThreads / (sizeof(T) == 8 ? 2 : 1))
    distill_kernel(Rows a, DistillArgs<A> p, double inv_temp, A k, T* grad) {
  extern __shared__ uint4 shared[];
  __shared__ bool last;  // written by one thread of a CTA, after its start
  if (threadIdx.x == 0) last = false;
  const Place<kThreads> place;
  const int64_t r = place.row;
  const A w = p.weights.at(r);
  if (w != A(0)) {
    cluster_started(place.ctas);
    distill_row(a, p, inv_temp, k, grad, place, w, shared, [&](double d) {
      p.terms[r] = static_cast<A>(static_cast<double>(w) * d);
      last = last_unit(p.done, a.rows);
    });
  } else {
    if (place.first()) {
      write_left_out(p, r);
      p.terms[r] = A(0);
      cudaGridDependencySynchronize();
      last = last_unit(p.done, a.rows);
    }
    if (grad) zero_row(distill_view<T>(a, r, grad), place);
  }
  __syncthreads();
  if (last) write_means<1>(p.terms, *p.total, p.out, a.rows);
}

// Short rows: a warp to a row.
template <typename T, typename A>
__global__ void __launch_bounds__(32 * kRowWarps, sizeof(T) == 8 ? 2 : 4)
    distill_warp_kernel(Rows a, DistillArgs<A> p, double inv_temp, A k, T* grad) {
  extern __shared__ uint4 shared[];
  __shared__ A terms[kRowWarps];
  __shared__ bool last;
  const Place<32> place;
  const int64_t r = place.row;
  const int warp = threadIdx.x / 32;
  const A w = r < a.rows ? p.weights.at(r) : A(0);
  if (place.tid == 0) terms[warp] = A(0);
  if (w != A(0)) {
    uint4* own = shared + warp * (row_bytes<A, 32>(p.top) / 16);
    distill_row(a, p, inv_temp, k, grad, place, w, own,
                [&](double d) { terms[warp] = static_cast<A>(static_cast<double>(w) * d); });
  } else if (r < a.rows) {
    if (place.tid == 0) write_left_out(p, r);
    if (grad) zero_row(distill_view<T>(a, r, grad), place);
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

template <typename T, int kThreads>
int launch_distill_rows(const Rows& a, const DistillArgs<typename AccOf<T>::type>& p,
                        double inv_temp, T* grad, int sms, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int64_t vectors = a.vocab / RowView<T>::E;
  int ctas = ctas_for(a.rows, vectors, kThreads, sms);
  while (ctas < 8 && int64_t{sms} * (kSmThreads / kThreads) * vectors * 16 / ctas > kRowsInL2)
    ctas *= 2;
  const auto kernel = distill_kernel<T, A, kThreads>;
  const int rc =
      allow_shared(reinterpret_cast<const void*>(kernel), row_bytes<A, kThreads>(kMostListed));
  if (rc) return rc;
  return launch_clusters(kernel, a.rows, ctas, kThreads, row_bytes<A, kThreads>(p.top), true, st,
                         "distill_kernel launch", a, p, inv_temp, exp_factor(A(0), inv_temp), grad);
}

template <typename T>
int launch_distill(const Rows& a, const DistillArgs<typename AccOf<T>::type>& p, double inv_temp,
                   T* grad, cudaStream_t st) {
  using A = typename AccOf<T>::type;
  const int64_t vectors = a.vocab / RowView<T>::E;
  const int sms = sm_count();
  if (by_warps(a.rows, vectors, 1536, sms)) {
    const auto kernel = distill_warp_kernel<T, A>;
    const int rc = allow_shared(reinterpret_cast<const void*>(kernel),
                                kRowWarps * row_bytes<A, 32>(kMostListed));
    if (rc) return rc;
    return launch_clusters(kernel, (a.rows + kRowWarps - 1) / kRowWarps, 1, 32 * kRowWarps,
                           kRowWarps * row_bytes<A, 32>(p.top), true, st,
                           "distill_warp_kernel launch", a, p, inv_temp, exp_factor(A(0), inv_temp),
                           grad);
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
  int rc = launch_total(p.weights, a.rows, kTotalThreads, p.total, p.done, p.out, 1, st);
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
