// Log probabilities of given tokens, with the entropy and the best alternatives of each row of logits, forward and
// backward (vocab.h has the formulas).
//
// Memory bounds them: the forward pass reads the logits once (4096x32768 float32 in 89 us, 6.0 TB/s, where a plain read
// reaches 6.2), the backward pass reads them once more and writes as much (2047x50021 float32: 819 MB in 136 us, 6.0
// TB/s). What little there is to do for a row of a decoding step is bound by latency: reading a share, a ticket,
// joining the shares (1x32768: 7 us, 10 with five alternatives; 48x131072 float16 with twenty: 18 us, 8 with
// none).
#include "vocab.h"

#include <climits>
#include <type_traits>

namespace {

using tt::kUnroll;
using tt::kWave;
using tt::LogitRow;
using tt::Pack;
using tt::Share;
using tt::Stat;
using tt::Words;

constexpr int kThreads = 256;
constexpr tt::Scale kPlain = {(float)tt::kLog2e, 1.f, 1.f};
constexpr int kMostTop = 64;
constexpr int kMostSplitRows = 255;     // rows that may be shared by blocks

// ---- the best alternatives -------------------------------------------------------------------------
//
// One pass keeps, beside the sums, each thread's largest value.  Of the G threads' largest values the K-th largest is a
// bound: K threads reach it, and what no thread's largest value reaches is no candidate.  So the packs of these K
// owners alone are read again, a few thousand values of a row that has just come through the cache, and what reaches
// the bound (K values and few more, unless the row is laid out against it) is ranked by counting.  Values and places
// make keys without ties, so the answer does not depend on the order in which candidates arrive.  (512 rows of 131072
// in float32: 47 us with no alternatives, 56 with five, 73 with twenty.)

typedef unsigned long long Key;

// A value as a number that orders alike, above zero.  -0 counts as 0.
__device__ __forceinline__ unsigned order_of(float z) {
  const unsigned b = __float_as_uint(z + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
// A value and its place as one number that orders by value, then by the lower place.
__device__ __forceinline__ Key make_key(float z, int place) {
  return ((Key)order_of(z) << 32) | (0xffffffffu - (unsigned)place);
}
// The value that a bound of keys has at least.  (Orders below that of -inf belong to no value.)
__device__ __forceinline__ float least_value(unsigned order) {
  return order <= 0x007fffffu ? -INFINITY : __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int key_place(Key k) { return (int)(0xffffffffu - (unsigned)k); }
__device__ __forceinline__ float key_value(Key k) {
  const unsigned order = (unsigned)(k >> 32);
  return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu));
}

constexpr int most(int a, int b) { return a > b ? a : b; }
// how many of these lanes come before this one
__device__ __forceinline__ int lanes_below(unsigned long long who) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0));
}

// More than K owners do no harm; up to this many more may be named, as halves, which are often equal, tend to.
constexpr int kMore = 32;

template <int G, int n>
struct TopSpace {
  // what one round can add to K kept candidates; what the lists of the splits can add up to
  static constexpr int room = most(G * n + kMostTop, G == kWave ? 0 : kMostTop * (kMostTop + 1) / 2);
  Key cand[room];
  Key heads[G];
  alignas(16) unsigned largest[G];
  Key best[kMostTop];
  int owner[kMostTop + kMore];
  int count, owners;
  Key bound;
};
struct NoSpace {};

// Of `count` keys in `cand` the K largest, largest first, to `best` (zeros where there are fewer).
template <int G, int n>
__device__ __forceinline__ void rank_candidates(TopSpace<G, n>& s, int lane, int count, int K) {
  for (int k = lane; k < K; k += G) s.best[k] = 0;
  tt::sync_row<G>();
  if (G == kWave && count <= kWave) {       // a key to a lane
    const Key mine = lane < count ? s.cand[lane] : 0;
    int rank = 0;
    for (int k = 0; k < count; ++k) rank += tt::lane_value(mine, k) > mine;
    if (lane < count && rank < K) s.best[rank] = mine;
  } else {
    for (int i = lane; i < count; i += G) {
      const Key mine = s.cand[i];
      int rank = 0;
      for (int k = 0; k < count; ++k) rank += s.cand[k] > mine;
      if (rank < K) s.best[rank] = mine;
    }
  }
  tt::sync_row<G>();
}

// The key of a thread's best value; `best` is what scan() says.
template <typename T, int G>
__device__ __forceinline__ Key best_key(const T* x, const LogitRow<T>& r, const Share& h, int lane, int best) {
  Key mine = 0;
  const int from = best == tt::kNothing ? h.p0 + lane : best;
#pragma unroll 1
  for (int j = from; j < from + kUnroll * G && j < h.p1; j += G) {
    float z[Pack<T>::n];
    tt::unpack<T>(z, r.pack(j));
#pragma unroll
    for (int i = 0; i < Pack<T>::n; ++i) {
      const Key k = make_key(z[i], r.column(j) + i);
      mine = k > mine ? k : mine;
    }
  }
  if (lane < h.head + h.tail) {
    const int i = tt::loose_column(r, h, lane);
    const Key k = make_key(tt::widen(x[r.start + i]), i);
    mine = k > mine ? k : mine;
  }
  return mine;
}

// What K of the numbers reach, LISTS of a lane: built bit by bit from the top, each time counting those that reach it,
// some 12 steps of a few scalar instructions, where sorting them took 21 of exchanges through LDS. `have` is how many
// do: K alone do most often after some bits, which is near enough unless K is most of them.
template <typename T, int LISTS>
__device__ __forceinline__ unsigned reached_by(const unsigned (&v)[LISTS], int K, int& have) {
  constexpr int kLowest = sizeof(T) == 2 ? 13 : 0;     // (a widened half has 13 bits alike below)
  unsigned reach = 0;
  have = LISTS * kWave;
  for (int bit = 31; bit >= kLowest && (have != K || 2 * K > LISTS * kWave); --bit) {
    const unsigned next = reach | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < LISTS; ++i) n += __popcll(__ballot(v[i] >= next));
    if (n >= K) {
      reach = next;
      have = n;
    }
  }
  return reach;
}

// Names the owners in s.owner, as many as it returns, and leaves the bound in `bound`.
template <typename T, int G>
__device__ __forceinline__ int name_owners(TopSpace<G, Pack<T>::n>& s, const T* x, const LogitRow<T>& r, const Share& h,
                                           int lane, float largest, int best, int K, Key& bound) {
  constexpr int kLists = G / kWave;
  const int in_wave = lane & (kWave - 1);
  const bool any = h.p0 + lane < h.p1 || lane < h.head + h.tail;
  const unsigned own = any ? order_of(largest) : 0u;
  unsigned v[kLists] = {own};
  if (lane == 0) s.count = s.owners = 0;
  if constexpr (G > kWave) {
    static_assert(kLists == 4, "a wave reads the block's values as 16 bytes a lane");
    s.largest[lane] = own;
    tt::sync_row<G>();
    const uint4 all = *reinterpret_cast<const uint4*>(&s.largest[in_wave * kLists]);
    v[0] = all.x, v[1] = all.y, v[2] = all.z, v[3] = all.w;
  }
  int have;
  unsigned reach = reached_by<T, kLists>(v, K, have);
  bound = (Key)reach << 32;
  if (have <= K + kMore || reach == 0) {
    reach = reach ? reach : 1u;         // (0: fewer than K threads have values at all, and each of those is an owner)
    int at = 0;
#pragma unroll
    for (int i = 0; i < kLists; ++i) {
      const unsigned long long who = __ballot(v[i] >= reach);
      const int slot = at + lanes_below(who);
      if (v[i] >= reach && lane < kWave) s.owner[slot] = in_wave * kLists + i;
      at += __popcll(who);
    }
    tt::sync_row<G>();
    return at;
  }
  // many threads reach the K-th largest value: those with the lowest places are the owners
  const Key mine = own >= reach ? best_key<T, G>(x, r, h, lane, best) : 0;
  s.heads[lane] = mine;
  tt::sync_row<G>();
  if (mine != 0) {
    int rank = 0;
    for (int i = 0; i < G; ++i) rank += s.heads[i] > mine;
    if (rank < K) s.owner[rank] = lane;
    if (rank == K - 1) s.bound = mine;
  }
  tt::sync_row<G>();
  bound = s.bound;
  return K;
}

// The owners' packs and loose columns, numbered: an owner's have numbers from its own on, up to a power of two.
template <typename T, int G>
struct Again {
  static constexpr int n = Pack<T>::n, kNone = INT_MIN;
  int rounds, shift, all;
  __device__ __forceinline__ Again(const Share& h, int owners) : rounds((h.p1 - h.p0 + G - 1) / G) {
    shift = 32 - __builtin_clz(rounds | 1);       // 2^shift > rounds
    all = owners << shift;
  }
  // what number q is: a pack, or -1 - c for a column, or kNone
  __device__ __forceinline__ int place(const TopSpace<G, n>& s, const LogitRow<T>& r, const Share& h, int q) const {
    if (q >= all) return kNone;
    const int owner = s.owner[q >> shift], step = q & ((1 << shift) - 1);
    if (step == rounds) return owner < h.head + h.tail ? -1 - tt::loose_column(r, h, owner) : kNone;
    const int j = h.p0 + owner + step * G;
    return step < rounds && j < h.p1 ? j : kNone;
  }
  // Appends the keys that reach the bound.  A wave of its own counts them in a register.
  static __device__ __forceinline__ void offer(TopSpace<G, n>& s, int& count, bool any, float z, int column,
                                               Key bound) {
    const Key k = make_key(z, column);
    const bool is = any && k >= bound;
    if constexpr (G == kWave) {
      const unsigned long long who = __ballot(is);
      if (who == 0) return;
      const int at = count + lanes_below(who);
      if (is && at < TopSpace<G, n>::room) s.cand[at] = k;
      count += __popcll(who);
    } else if (is) {
      const int at = atomicAdd(&s.count, 1);
      if (at < TopSpace<G, n>::room) s.cand[at] = k;
    }
  }
  static __device__ __forceinline__ void collect(TopSpace<G, n>& s, int& count, const T* x, const LogitRow<T>& r,
                                                 int at, const Words& p, Key bound) {
    float z[n];
    tt::unpack<T>(z, p);
#pragma unroll
    for (int i = 0; i < n; ++i) offer(s, count, at >= 0, z[i], r.column(at) + i, bound);
    const bool loose = at < 0 && at != kNone;
    offer(s, count, loose, loose ? tt::widen(x[r.start - 1 - at]) : 0.f, -1 - at, bound);
  }
};

// Leaves the K best of a share in s.best; `largest` is this thread's largest value and `best` what scan() says of it.
template <typename T, int G>
__device__ __forceinline__ void select_top(TopSpace<G, Pack<T>::n>& s, const T* x, const LogitRow<T>& r, const Share& h,
                                           int lane, float largest, int best, int K) {
  Key bound;
  const Again<T, G> again(h, name_owners<T, G>(s, x, r, h, lane, largest, best, K, bound));
  int count = 0;
  constexpr int kAgain = 2;       // packs on their way at once
  // If there is no room for all candidates, the second time keeps the K best after each step.
  for (bool careful = false;; careful = true) {
    for (int q0 = 0; q0 < again.all; q0 += kAgain * G) {
      int at[kAgain];
      Words p[kAgain];
#pragma unroll
      for (int u = 0; u < kAgain; ++u) {
        at[u] = again.place(s, r, h, q0 + u * G + lane);
        p[u] = Words(Pack<T>::lowest);
        if (at[u] >= 0) p[u] = r.pack(at[u]);
      }
#pragma unroll
      for (int u = 0; u < kAgain; ++u) {
        if (q0 + u * G >= again.all) continue;
        Again<T, G>::collect(s, count, x, r, at[u], p[u], bound);
        if (!careful) continue;
        tt::sync_row<G>();
        if (G > kWave) count = s.count;
        if (count > kMostTop) {
          rank_candidates(s, lane, count, K);
          for (int k = lane; k < K; k += G) s.cand[k] = s.best[k];
          bound = s.best[K - 1] > bound ? s.best[K - 1] : bound;
          if (lane == 0) s.count = K;
          count = K;
        }
        tt::sync_row<G>();
      }
    }
    tt::sync_row<G>();
    if (G > kWave) count = s.count;
    if (count <= TopSpace<G, Pack<T>::n>::room) break;
    tt::sync_row<G>();
    if (lane == 0) s.count = 0;
    count = 0;
    tt::sync_row<G>();
  }
  rank_candidates(s, lane, count, K);
}

// The same for a row that a wave keeps in registers, `kept` packs and one loose value to a lane: all that reach the
// bound are at hand, and nothing is read again.
template <typename T, int NV>
__device__ __forceinline__ void select_kept(TopSpace<kWave, Pack<T>::n>& s, const T* x, const LogitRow<T>& r,
                                            const Share& h, int lane, const Words (&kept)[NV], float loose, float largest,
                                            int best, int K) {
  constexpr int n = Pack<T>::n;
  const bool any = h.p0 + lane < h.p1 || lane < h.head + h.tail;
  const unsigned v[1] = {any ? order_of(largest) : 0u};
  int have, count = 0;
  const float least = least_value(reached_by<T, 1>(v, K, have));
  auto offer = [&](bool is, float z, int column) {
    const unsigned long long who = __ballot(is);
    if (who == 0) return;
    const int at = count + lanes_below(who);
    if (is && at < TopSpace<kWave, n>::room) s.cand[at] = make_key(z, column);
    count += __popcll(who);
  };
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int j = h.p0 + lane + u * kWave;
    const bool has = j < h.p1 && tt::pack_max<T, 1>(&kept[u]) >= least;
    if (__ballot(has) == 0) continue;
    float z[n];
    tt::unpack<T>(z, kept[u]);
#pragma unroll
    for (int i = 0; i < n; ++i) offer(has && z[i] >= least, z[i], r.column(j) + i);
  }
  offer(lane < h.head + h.tail && loose >= least, loose, tt::loose_column(r, h, lane));
  if (count > TopSpace<kWave, n>::room) return select_top<T, kWave>(s, x, r, h, lane, largest, best, K);
  rank_candidates(s, lane, count, K);
}

// The K best of `splits` sorted lists of K keys.  The list whose head has rank i holds at most K - i of them, and those
// reach the K-th head: at most K (K + 1) / 2 candidates.
template <int G, int n>
__device__ __forceinline__ void join_top(TopSpace<G, n>& s, const Key* lists, int splits, int lane, int K) {
  const Key head = lane < splits ? tt::shared(lists + (size_t)lane * K) : 0;
  s.heads[lane] = head;
  if (lane == 0) {
    s.count = s.owners = 0;
    s.bound = 0;
  }
  __syncthreads();
  if (head != 0) {
    int rank = 0;
    for (int i = 0; i < splits; ++i) rank += s.heads[i] > head;
    if (rank < K) {
      s.owner[rank] = lane;
      atomicAdd(&s.owners, 1);
      if (rank == K - 1) s.bound = head;
    }
  }
  __syncthreads();
  for (int q = lane; q < s.owners * K; q += G) {
    const int rank = q / K, k = q % K;
    if (k < K - rank) {
      const Key key = tt::shared(lists + (size_t)s.owner[rank] * K + k);
      if (key != 0 && key >= s.bound) s.cand[atomicAdd(&s.count, 1)] = key;
    }
  }
  __syncthreads();
  rank_candidates(s, lane, s.count, K);
}

// ---- forward ---------------------------------------------------------------------------------------

struct ForwardOut {
  const void* tokens;
  int wide;
  float* logp;
  float* entropy;
  float* top_logp;
  long long* top_index;
  float2* stats;
  long long ignored;
};

// A token as given, counted from the end where it is negative; -1 where it is no token.
__device__ __forceinline__ long long token_place(long long t, int V) {
  if (t < 0) t += V;
  return t >= 0 && t < V ? t : -1;
}

template <int G>
__device__ __forceinline__ void write_ignored(const ForwardOut& o, size_t row, int lane, int K) {
  if (lane == 0) {
    o.logp[row] = 0.f;
    o.entropy[row] = 0.f;
    if (o.stats) o.stats[row] = make_float2(0.f, 0.f);
  }
  for (int k = lane; k < K; k += G) {
    o.top_logp[row * K + k] = 0.f;
    o.top_index[row * K + k] = -1;
  }
}

template <typename T, int G>
__device__ __forceinline__ void write_row(const ForwardOut& o, size_t row, int lane, const Stat& a, bool is_token,
                                          float z_token, const Key* best, int K) {
  const float log_s = tt::log_sum(a), m = tt::anchor(a.m);
  if (lane == 0) {
    o.logp[row] = is_token ? tt::log_p<T>(z_token, m, log_s, kPlain) : NAN;
    o.entropy[row] = a.s == 0.f ? 0.f : (log_s - a.t / a.s) * tt::kLn2;
    if (o.stats) o.stats[row] = make_float2(a.m, log_s);
  }
  const bool fine = a.s == a.s;
  for (int k = lane; k < K; k += G) {
    o.top_logp[row * K + k] = fine ? tt::log_p<T>(key_value(best[k]), m, log_s, kPlain) : NAN;
    o.top_index[row * K + k] = fine ? key_place(best[k]) : -1;
  }
}

// NV > 0: a wave keeps its row, NV packs to a lane.
template <typename T, int G, bool TOP, int NV = 0>
__global__ __launch_bounds__(kThreads) void logp_rows(const T* __restrict__ x, ForwardOut o, int R, int V, int K) {
  constexpr int kRows = kThreads / G, kKept = NV < kUnroll ? NV : kUnroll;      // (of a lane's packs taken together)
  __shared__ float part[kRows][tt::parts_of(G, 3)];
  __shared__ std::conditional_t<TOP, TopSpace<G, Pack<T>::n>, NoSpace> space[kRows];
  const int lane = threadIdx.x % G, sub = tt::row_of_block<G>();
  const float c = (float)tt::kLog2e;
  for (long long row = (long long)blockIdx.x * kRows + sub; row < R; row += (long long)gridDim.x * kRows) {
    const LogitRow<T> r(x, row, V);
    const Share h(r, 0, 1);
    Words kept[NV ? NV : 1];            // (on their way together with the token)
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      kept[u] = Words(Pack<T>::lowest);
      if (h.p0 + lane + u * G < h.p1) kept[u] = r.pack(h.p0 + lane + u * G);
    }
    float loose = -INFINITY;
    if (NV > 0 && lane < h.head + h.tail) loose = tt::widen(x[r.start + tt::loose_column(r, h, lane)]);
    const long long t0 = tt::read_index(o.tokens, row, o.wide);
    if (t0 == o.ignored) {
      write_ignored<G>(o, row, lane, K);
      continue;
    }
    const long long t = token_place(t0, V);
    const float z_token = lane == 0 && t >= 0 ? tt::widen(x[r.start + t]) : 0.f;
    Stat a = {-INFINITY, 0.f, 0.f};
    int best = tt::kNothing;
    if constexpr (NV > 0) {
#pragma unroll
      for (int u = 0; u < NV; u += kKept)
        if (h.p0 + u * G < h.p1 && tt::add_packs<T, kKept, true>(a, kept + u, c)) best = h.p0 + lane + u * G;
      tt::add_value<T, true>(a, loose, c);
    } else {
      tt::scan<T, G, true>(a, best, x, r, h, lane, c);
    }
    const float largest = a.m;
    a = tt::row_join<T, G, true>(a, c, part[sub]);
    if constexpr (NV > 0) {
      select_kept<T, NV>(space[sub], x, r, h, lane, kept, loose, largest, best, K);
      write_row<T, G>(o, row, lane, a, t >= 0, z_token, space[sub].best, K);
    } else if constexpr (TOP) {
      select_top<T, G>(space[sub], x, r, h, lane, largest, best, K);
      write_row<T, G>(o, row, lane, a, t >= 0, z_token, space[sub].best, K);
    } else {
      write_row<T, G>(o, row, lane, a, t >= 0, z_token, nullptr, 0);
    }
    tt::sync_row<G>();
  }
}

__device__ tt::Ticket logp_tickets[kMostSplitRows];       // the splits of each row that are done

// Few long rows: `splits` blocks to a row, each with its share; the one that comes last puts the shares together.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void logp_split(const T* __restrict__ x, ForwardOut o, float* stat_part,
                                                       Key* key_part, int splits, int V, int K) {
  constexpr int G = kThreads;
  __shared__ float part[3 * (G / kWave)];
  __shared__ float more[3 * (G / kWave)];
  __shared__ std::conditional_t<TOP, TopSpace<G, Pack<T>::n>, NoSpace> space;
  __shared__ bool last;
  const float c = (float)tt::kLog2e;
  const int split = blockIdx.x % splits, lane = threadIdx.x;
  const size_t row = blockIdx.x / splits;
  const long long t0 = tt::read_index(o.tokens, row, o.wide);
  if (t0 == o.ignored) {
    if (split == 0) write_ignored<G>(o, row, lane, K);
    return;
  }
  const LogitRow<T> r(x, row, V);
  const Share h(r, split, splits);
  Stat a = {-INFINITY, 0.f, 0.f};
  int best = tt::kNothing;
  tt::scan<T, G, true>(a, best, x, r, h, lane, c);
  const float largest = a.m;
  a = tt::row_join<T, G, true>(a, c, part);
  if constexpr (TOP) select_top<T, G>(space, x, r, h, lane, largest, best, K);
  if (lane < kWave) {
    float* mine_part = stat_part + (size_t)blockIdx.x * 3;
    if (lane < 3) tt::share(mine_part + lane, lane == 0 ? a.m : lane == 1 ? a.s : a.t);
    if constexpr (TOP)
      if (lane < K) tt::share(key_part + (size_t)blockIdx.x * K + lane, space.best[lane]);
    tt::stores_done();
    if (lane == 0) last = tt::last_ticket(logp_tickets + row, splits);
  }
  __syncthreads();
  if (!last) return;
  const long long t = token_place(t0, V);
  const float z_token = lane == 0 && t >= 0 ? tt::widen(x[r.start + t]) : 0.f;
  Stat all = {-INFINITY, 0.f, 0.f};
  if (lane < splits) {
    const float* p = stat_part + (row * splits + lane) * 3;
    all.m = tt::shared(p);
    all.s = tt::shared(p + 1);
    all.t = tt::shared(p + 2);
  }
  all = tt::row_join<T, G, true>(all, c, more);
  if constexpr (TOP) {
    join_top(space, key_part + row * (size_t)splits * K, splits, lane, K);
    write_row<T, G>(o, row, lane, all, t >= 0, z_token, space.best, K);
  } else {
    write_row<T, G>(o, row, lane, all, t >= 0, z_token, nullptr, 0);
  }
}

// ---- backward --------------------------------------------------------------------------------------

struct BackwardIn {
  const void* tokens;
  int wide;
  const float2* stats;
  const float* entropy;
  const long long* top_index;
  const float* g_logp;
  const float* g_entropy;
  const float* g_top;
  long long ignored;
};

// dz_j = -p_j (a + sum_k c_k + h (log p_j + H)) + a [j = t] + sum_k c_k [j = i_k]
template <typename T>
struct RowGradient {
  float m, log_s, total, h, H;
  __device__ __forceinline__ float operator()(float z, float extra) const {
    const float d = tt::bits<T>(z, m, (float)tt::kLog2e) - log_s;
    return fmaf(-tt::pow2(d), fmaf(h, fmaf(tt::floor_at(d), tt::kLn2, H), total), extra);
  }
};

// G threads write a share of a row without the last two terms, and then the few values that have them once more.
// Rows go last to first: what the forward pass read last may still be in the memory-side cache.
template <typename T, int G>
__global__ __launch_bounds__(kThreads) void logp_bwd(const T* __restrict__ x, BackwardIn in, T* dx, int splits, int R,
                                                     int V, int K) {
  constexpr int kRows = kThreads / G, n = Pack<T>::n;
  const int lane = threadIdx.x % G, sub = tt::row_of_block<G>();
  const long long items = (long long)R * splits;
  for (long long item = (long long)blockIdx.x * kRows + sub; item < items; item += (long long)gridDim.x * kRows) {
    const size_t row = R - 1 - item / splits;
    const LogitRow<T> r(x, row, V);
    const Share s(r, (int)(item % splits), splits);
    const long long t0 = tt::read_index(in.tokens, row, in.wide), t = token_place(t0, V);
    const float2 st = in.stats[row];
    const bool none = t0 == in.ignored || tt::is_empty(st.x, st.y), given = in.g_logp && t >= 0;
    RowGradient<T> g = {st.x, st.y, 0.f, 0.f, 0.f};
    float a = 0.f;
    if (!none) {
      a = in.g_logp ? in.g_logp[row] : 0.f;
      g.h = in.g_entropy ? in.g_entropy[row] : 0.f;
      g.H = in.entropy[row];
      g.total = in.g_logp && t < 0 ? NAN : a;
      if (in.g_top) {
        constexpr int kLanes = G < kWave ? G : kWave;
        float sum = 0.f;
        for (int k = lane % kLanes; k < K; k += kLanes) sum += in.g_top[row * K + k];
        g.total += tt::lanes_reduce<kLanes>(sum, tt::Plus());
      }
    }
    for (int j = s.p0 + lane; j < s.p1; j += kUnroll * G) {
      tt::Words p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (!none && j + u * G < s.p1) p[u] = r.pack(j + u * G);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (j + u * G >= s.p1) continue;
        float z[n];
        tt::unpack<T>(z, p[u]);
#pragma unroll
        for (int i = 0; i < n; ++i) z[i] = g(z[i], 0.f);
        tt::write_pack(r, dx, j + u * G, none ? tt::Words(0u) : tt::pack<T>(z));
      }
    }
    for (int i = lane; i < s.head + s.tail; i += G) {
      const size_t at = r.start + tt::loose_column(r, s, i);
      dx[at] = none ? (T)0.f : (T)g(tt::widen(x[at]), 0.f);
    }
    const int fixes = none ? 0 : (given ? 1 : 0) + (in.g_top ? K : 0);
    if (fixes == 0) continue;
    // what is stored below goes over what was stored above: that has to have left first
    tt::stores_done();
    tt::sync_row<G>();
    for (int f = lane; f < fixes; f += G) {
      const long long j = given && f == 0 ? t : in.top_index[row * K + f - (given ? 1 : 0)];
      const int pack = (int)((j + r.skip) / n);
      const bool here = j < r.head ? s.head > 0 : j >= r.tail_at ? s.tail > 0 : pack >= s.p0 && pack < s.p1;
      if (j < 0 || j >= V || !here) continue;       // (the places are the caller's memory by now)
      float extra = given && j == t ? a : 0.f;      // summed first: what cancels here leaves no rounding behind
      if (in.g_top)
        for (int k = 0; k < K; ++k)
          if (in.top_index[row * K + k] == j) extra += in.g_top[row * K + k];
      dx[r.start + j] = (T)g(tt::widen(x[r.start + j]), extra);
    }
    tt::sync_row<G>();
  }
}

// ---- launches --------------------------------------------------------------------------------------

int check(const char* fn, int dtype, int index_bits, long long R, int V, int K) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_F16, "%s: unknown type %d", fn, dtype);
  TT_REQUIRE(index_bits == 32 || index_bits == 64, "%s: indexes have 32 or 64 bits (got %d)", fn, index_bits);
  TT_REQUIRE(R > 0 && R <= (1 << 30), "%s: rows must be in 1..2^30 (got %lld)", fn, R);
  TT_REQUIRE(V > 0 && V <= (1 << 30), "%s: the vocabulary must have 1..2^30 entries (got %d)", fn, V);
  TT_REQUIRE(K >= 0 && K <= kMostTop && K <= V, "%s: alternatives must be in 0..min(%d, %d) (got %d)", fn, kMostTop, V,
             K);
  return 0;
}

unsigned grid_for(long long blocks) { return (unsigned)(blocks < (1 << 22) ? blocks : (1 << 22)); }

// Rows of up to kWavePacks packs go to a wave each, short ones to some of its lanes, so that a wave has several rows on
// their way; longer ones go to a block.  131072 rows of float32, a wave against eight lanes: of 10 values 47 and 8 us,
// of 300 values 64 and 31 us forward; and backward, where more lanes store wider pieces, 8 against 16 lanes: of 37
// values 17 and 24 us, of 100 values 31 and 29 us, of 300 values 109 and 80 us (a wave: 120 us); 67108 rows of 1000 take
// 54 and 52 us forward, 107 by waves and 131 by sixteen lanes backward.  22369 rows of 3000 with five alternatives 64 us by
// waves and 127 by blocks; with more than kWaveTop a block, of four times as many threads, has a closer bound (with 32 93
// and 156 us, with 64 428 and 182).
constexpr int kLanesPacks = 128, kFewPacks = 16, kWavePacks = 1024, kWaveTop = 32;
template <int G>
unsigned row_grid(long long R) {
  return grid_for((R + kThreads / G - 1) / (kThreads / G));
}

// Rows shared by blocks, where they are fewer than units: two blocks to a unit, with kUnroll packs to a thread at least
// (200 rows of 50021 with twenty alternatives take 19 us, with eight blocks to a unit 24; 250 of 131072 with five 31, 40 if
// they stay whole; one row of 32768 4.6 and 6.0). From 256 rows on they stay whole (1000 rows of 9000 with ten 14 us and 22
// shared by two, 512 of 131072 with five 54 and 57). The join costs few rows of few packs more than it saves (100 rows of
// 9000 with ten take 10 us, 7 if they stay whole).
int forward_splits(long long R, int packs) {
  if (packs <= kWavePacks || R > kMostSplitRows) return 1;
  return tt::splits_for(R, packs, kThreads, 2, kUnroll * kThreads);
}
// The blocks of the backward pass share nothing, and more of them end more evenly: 32 to a unit, of twice as many
// packs, where that is more (1300 rows of 50021: 118 -> 98 us; 8000 rows of 8191, which stay whole, take 102 us, shared
// by two 105).
int backward_splits(long long R, int packs) {
  const int few = tt::splits_for(R, packs, kThreads, 8, kUnroll * kThreads);
  const int many = tt::splits_for(R, packs, kThreads, 32, 2 * kUnroll * kThreads);
  return few > many ? few : many;
}

template <typename T>
int forward(const T* x, const ForwardOut& o, int R, int V, int K) {
  hipStream_t st = tt::stream();
  const int packs = (V + Pack<T>::n - 1) / Pack<T>::n;
  const int splits = forward_splits(R, packs);
  if (splits > 1) {
    void* ws;
    const size_t parts = (size_t)R * splits, stat_bytes = (parts * 3 * sizeof(float) + 255) / 256 * 256;
    if (tt::workspace(stat_bytes + parts * K * sizeof(Key), &ws)) return -1;
    Key* keys = (Key*)((char*)ws + stat_bytes);
    if (K) logp_split<T, true><<<(unsigned)parts, kThreads, 0, st>>>(x, o, (float*)ws, keys, splits, V, K);
    else logp_split<T, false><<<(unsigned)parts, kThreads, 0, st>>>(x, o, (float*)ws, keys, splits, V, K);
  } else if (packs <= kLanesPacks && K == 0) {
    logp_rows<T, 8, false><<<row_grid<8>(R), kThreads, 0, st>>>(x, o, R, V, K);
  } else if (packs <= kWavePacks && K <= kWaveTop) {
    const unsigned grid = row_grid<kWave>(R);
    if (K && packs <= 2 * kWave) logp_rows<T, kWave, true, 2><<<grid, kThreads, 0, st>>>(x, o, R, V, K);
    else if (K && packs <= 4 * kWave) logp_rows<T, kWave, true, 4><<<grid, kThreads, 0, st>>>(x, o, R, V, K);
    else if (K) logp_rows<T, kWave, true><<<grid, kThreads, 0, st>>>(x, o, R, V, K);
    else logp_rows<T, kWave, false><<<grid, kThreads, 0, st>>>(x, o, R, V, K);
  } else {
    if (K) logp_rows<T, kThreads, true><<<grid_for(R), kThreads, 0, st>>>(x, o, R, V, K);
    else logp_rows<T, kThreads, false><<<grid_for(R), kThreads, 0, st>>>(x, o, R, V, K);
  }
  TT_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int backward(const T* x, const BackwardIn& in, T* dx, int R, int V, int K) {
  hipStream_t st = tt::stream();
  const int packs = (V + Pack<T>::n - 1) / Pack<T>::n;
  if (packs <= kFewPacks) {
    logp_bwd<T, 8><<<row_grid<8>(R), kThreads, 0, st>>>(x, in, dx, 1, R, V, K);
  } else if (packs <= kLanesPacks) {
    logp_bwd<T, 16><<<row_grid<16>(R), kThreads, 0, st>>>(x, in, dx, 1, R, V, K);
  } else if (packs <= kWavePacks) {
    logp_bwd<T, kWave><<<row_grid<kWave>(R), kThreads, 0, st>>>(x, in, dx, 1, R, V, K);
  } else {
    const int splits = backward_splits(R, packs);
    logp_bwd<T, kThreads><<<grid_for((long long)R * splits), kThreads, 0, st>>>(x, in, dx, splits, R, V, K);
  }
  TT_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" {

int tt_token_log_prob_fwd(const void* x, const void* tokens, float* logp, float* entropy, float* top_logp,
                          long long* top_index, float* stats, int dtype, int token_bits, long long ignore_index,
                          long long R, int V, int K) {
  TT_REQUIRE_INIT();
  const char* fn = "tt_token_log_prob_fwd";
  TT_REQUIRE(x && tokens && logp && entropy, "%s: null pointer", fn);
  if (int rc = check(fn, dtype, token_bits, R, V, K)) return rc;
  TT_REQUIRE(K == 0 || (top_logp && top_index), "%s: null pointer for the alternatives", fn);
  TT_REQUIRE_ALIGNED(fn, x, stats);
  const ForwardOut o = {tokens, token_bits == 64, logp, entropy, top_logp, top_index, (float2*)stats, ignore_index};
  if (dtype == TT_F32) return forward((const float*)x, o, (int)R, V, K);
  return forward((const _Float16*)x, o, (int)R, V, K);
}

int tt_token_log_prob_bwd(const void* x, const void* tokens, const float* stats, const float* entropy,
                          const long long* top_index, const float* g_logp, const float* g_entropy, const float* g_top,
                          void* dx, int dtype, int token_bits, long long ignore_index, long long R, int V, int K) {
  TT_REQUIRE_INIT();
  const char* fn = "tt_token_log_prob_bwd";
  TT_REQUIRE(x && tokens && stats && entropy && dx, "%s: null pointer", fn);
  if (int rc = check(fn, dtype, token_bits, R, V, K)) return rc;
  TT_REQUIRE(g_top == nullptr || (K > 0 && top_index), "%s: a gradient of the alternatives needs their indexes", fn);
  TT_REQUIRE_ALIGNED(fn, x, dx, stats);
  const BackwardIn in = {tokens, token_bits == 64, (const float2*)stats, entropy, top_index, g_logp, g_entropy, g_top,
                         ignore_index};
  if (dtype == TT_F32) return backward((const float*)x, in, (float*)dx, (int)R, V, K);
  return backward((const _Float16*)x, in, (_Float16*)dx, (int)R, V, K);
}

}  // extern "C"
