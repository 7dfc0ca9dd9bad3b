// Log probabilities of given tokens, with the entropy and the best alternatives of each row of logits, forward and
// backward (vocab.h has the formulas).
#include "vocab.h"

namespace {

using tt::kWave;
using tt::LogitRow;
using tt::Pack;
using tt::Stat;

constexpr int kThreads = 256;
constexpr int kMostTop = 64;
constexpr int kUnroll = 4;

// ---- the best alternatives -------------------------------------------------------------------------
//
// One pass keeps, beside the sums, each thread's largest value and where it stood first.  Of the G threads' best values
// the K largest name K owners, and the K-th of them is a bound: a value above it lies with an owner, for every other
// thread's best is below.  So the owners' packs alone are read again, a few thousand values of a row that has just come
// through the cache, and what reaches the bound (K values and few more, unless the row is laid out against it) is
// ranked by counting.  Values and places make keys without ties, so the answer does not depend on the order in which
// candidates arrive.

typedef unsigned long long Key;

// A value and its place as one number that orders by value, then by the lower place.  -0 counts as 0.
__device__ __forceinline__ Key make_key(float z, int place) {
  const unsigned b = __float_as_uint(z + 0.f);
  const unsigned order = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((Key)order << 32) | (0xffffffffu - (unsigned)place);
}
__device__ __forceinline__ int key_place(Key k) { return (int)(0xffffffffu - (unsigned)k); }
__device__ __forceinline__ float key_value(Key k) {
  const unsigned order = (unsigned)(k >> 32);
  return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu));
}

// The keys of a wave, largest first.
__device__ __forceinline__ Key wave_sort(Key k) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int size = 2; size <= kWave; size <<= 1) {
#pragma unroll
    for (int off = size >> 1; off > 0; off >>= 1) {
      const Key o = __shfl_xor(k, off, kWave);
      const bool lower = (lane & off) == 0, down = (lane & size) == 0;
      k = (o > k) == (lower == down) ? o : k;
    }
  }
  return k;
}

template <int G, int n>
struct TopSpace {
  static constexpr int room = G * n + kMostTop;     // what one round can add to K kept candidates
  Key cand[room];
  Key heads[G / kWave * kMostTop];
  Key best[kMostTop];
  int owner[kMostTop];
  int count, owners;
  Key bound;
};

// Of `count` keys in `cand` the K largest, largest first, to `best` (zeros where there are fewer).
template <int G, int n>
__device__ __forceinline__ void rank_candidates(TopSpace<G, n>& s, int lane, int count, int K) {
  for (int k = lane; k < K; k += G) s.best[k] = 0;
  tt::sync_row<G>();
  for (int i = lane; i < count; i += G) {
    const Key mine = s.cand[i];
    int rank = 0;
    for (int k = 0; k < count; ++k) rank += s.cand[k] > mine;
    if (rank < K) s.best[rank] = mine;
  }
  tt::sync_row<G>();
}

// Packs [v0, v1) of the row by the G threads, thread `lane` on v0 + lane + i G; `mine` is the key of its best value, or
// zero.  Leaves the K best in s.best.
template <typename T, int G>
__device__ __forceinline__ void select_top(TopSpace<G, Pack<T>::n>& s, const LogitRow<T>& r, int v0, int v1, int lane,
                                           Key mine, int K) {
  constexpr int n = Pack<T>::n;
  const Key sorted = wave_sort(mine);
  const int in_wave = lane & (kWave - 1), lists = G / kWave;
  if (in_wave < K) s.heads[(lane >> 6) * K + in_wave] = sorted;
  if (lane == 0) {
    s.count = s.owners = 0;
    s.bound = 0;
  }
  tt::sync_row<G>();
  for (int i = lane; i < lists * K; i += G) {       // (at most one each: K <= 64)
    const Key k = s.heads[i];
    int rank = 0;
    for (int o = 0; o < lists * K; ++o) rank += s.heads[o] > k;
    if (k != 0 && rank < K) {
      s.owner[rank] = ((key_place(k) + r.skip) / n - v0) % G;
      atomicAdd(&s.owners, 1);
      if (rank == K - 1) s.bound = k;
    }
  }
  tt::sync_row<G>();
  const int rounds = (v1 - v0 + G - 1) / G, pairs = s.owners * rounds;
  Key bound = s.bound;
  int count = 0;
  for (int p0 = 0; p0 < pairs; p0 += G) {
    const int p = p0 + lane;
    if (p < pairs) {
      const int j = v0 + s.owner[p / rounds] + p % rounds * G;
      if (j < v1) {
        const typename Pack<T>::type q = r.read(j);
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const int c = r.column(j) + i;
          const Key k = make_key(tt::widen(q[i]), c);
          if (c >= 0 && c < r.V && k >= bound) s.cand[atomicAdd(&s.count, 1)] = k;
        }
      }
    }
    tt::sync_row<G>();
    count = s.count;
    if (count > kMostTop && p0 + G < pairs) {       // another round might not fit: keep the K best of these
      rank_candidates(s, lane, count, K);
      for (int k = lane; k < K; k += G) s.cand[k] = s.best[k];
      bound = s.best[K - 1] > bound ? s.best[K - 1] : bound;
      if (lane == 0) s.count = K;
    }
    tt::sync_row<G>();
  }
  rank_candidates(s, lane, count, K);
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

template <int G>
__device__ __forceinline__ void write_row(const ForwardOut& o, size_t row, int lane, const Stat& a, bool is_token,
                                          float z_token, const Key* best, int K) {
  const float log_s = tt::log_sum(a), m = tt::anchor(a.m);
  if (lane == 0) {
    o.logp[row] = is_token ? (z_token - m) - log_s * tt::kLn2 : NAN;
    o.entropy[row] = a.s == 0.f ? 0.f : (log_s - a.t / a.s) * tt::kLn2;
    if (o.stats) o.stats[row] = make_float2(a.m, log_s);
  }
  const bool fine = a.s == a.s;
  for (int k = lane; k < K; k += G) {
    o.top_logp[row * K + k] = fine ? (key_value(best[k]) - m) - log_s * tt::kLn2 : NAN;
    o.top_index[row * K + k] = fine ? key_place(best[k]) : -1;
  }
}

// The statistics of packs [v0, v1), and with TOP the key of this thread's best value.
template <typename T, int G, bool TOP>
__device__ __forceinline__ Stat scan(const LogitRow<T>& r, int v0, int v1, int lane, float c, Key& mine) {
  constexpr int n = Pack<T>::n;
  typedef typename Pack<T>::type P;
  Stat a = {-INFINITY, 0.f, 0.f};
  int best = -1;
  const int whole1 = v1 < r.whole1 ? v1 : r.whole1;
  for (int j = v0 + lane; j < v1; j += kUnroll * G) {
    P p[kUnroll];
    if (j >= r.whole0 && j + (kUnroll - 1) * G < whole1) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) p[u] = r.at[j + u * G];
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) p[u] = j + u * G < v1 ? r.read(j + u * G) : P((T)-INFINITY);
    }
    float z[kUnroll * n];
#pragma unroll
    for (int i = 0; i < kUnroll * n; ++i) z[i] = tt::widen(p[i / n][i % n]);
    const bool rises = tt::add_values<kUnroll * n, true>(a, z, c);
    if (TOP && (rises || best < 0)) best = j;
  }
  if (TOP) {
    mine = 0;
    if (best >= 0) {
#pragma unroll
      for (int u = kUnroll - 1; u >= 0; --u) {
        const int j = best + u * G;
        if (j < v1) {
          const P p = r.read(j);
#pragma unroll
          for (int i = n - 1; i >= 0; --i) {
            const int col = r.column(j) + i;
            const Key k = make_key(tt::widen(p[i]), col);
            if (col >= 0 && col < r.V && k > mine) mine = k;
          }
        }
      }
    }
  }
  return a;
}

template <typename T, int G, bool TOP>
__global__ __launch_bounds__(kThreads) void logp_rows(const T* __restrict__ x, ForwardOut o, int R, int V, int K) {
  constexpr int kRows = kThreads / G;
  __shared__ float part[kRows][3 * (G / kWave)];
  __shared__ TopSpace<TOP ? G : kWave, TOP ? Pack<T>::n : 1> space[TOP ? kRows : 1];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const float c = (float)tt::kLog2e;
  for (long long row = (long long)blockIdx.x * kRows + sub; row < R; row += (long long)gridDim.x * kRows) {
    const long long t0 = tt::read_index(o.tokens, row, o.wide);
    if (t0 == o.ignored) {
      write_ignored<G>(o, row, lane, K);
      continue;
    }
    const LogitRow<T> r(x, row, V);
    const long long t = token_place(t0, V);
    const float z_token = lane == 0 && t >= 0 ? tt::widen(x[row * (size_t)V + t]) : 0.f;
    Key mine;
    Stat a = scan<T, G, TOP>(r, 0, r.packs, lane, c, mine);
    a = tt::row_join<G, true>(a, c, part[sub]);
    if constexpr (TOP) select_top<T, G>(space[sub], r, 0, r.packs, lane, mine, K);
    if constexpr (TOP) write_row<G>(o, row, lane, a, t >= 0, z_token, space[sub].best, K);
    else write_row<G>(o, row, lane, a, t >= 0, z_token, nullptr, 0);
    tt::sync_row<G>();
  }
}

// Few long rows: `splits` blocks to a row, each with its share of the packs; logp_join puts them together.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void logp_split(const T* __restrict__ x, const void* __restrict__ tokens,
                                                       int wide, long long ignored, Stat* __restrict__ stat_part,
                                                       Key* __restrict__ key_part, int splits, int V, int K) {
  constexpr int G = kThreads;
  __shared__ float part[3 * (G / kWave)];
  __shared__ TopSpace<TOP ? G : kWave, TOP ? Pack<T>::n : 1> space;
  const int row = blockIdx.x / splits, split = blockIdx.x % splits, lane = threadIdx.x;
  if (tt::read_index(tokens, row, wide) == ignored) return;
  const LogitRow<T> r(x, row, V);
  const int per = (r.packs + splits - 1) / splits;
  const int v0 = split * per, v1 = v0 + per < r.packs ? v0 + per : r.packs;     // (v0 may lie behind the last pack)
  Key mine;
  Stat a = scan<T, G, TOP>(r, v0, v1, lane, (float)tt::kLog2e, mine);
  a = tt::row_join<G, true>(a, (float)tt::kLog2e, part);
  if (lane == 0) stat_part[blockIdx.x] = a;
  if constexpr (TOP) {
    select_top<T, G>(space, r, v0, v1, lane, mine, K);
    for (int k = lane; k < K; k += G) key_part[(size_t)blockIdx.x * K + k] = space.best[k];
  }
}

// One block to a row.  The splits' lists of keys are sorted, so the list whose head has rank i holds at most K - i of
// the K best, and those reach the K-th head: at most K (K + 1) / 2 candidates.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void logp_join(const T* __restrict__ x, ForwardOut o,
                                                      const Stat* __restrict__ stat_part,
                                                      const Key* __restrict__ key_part, int splits, int V, int K) {
  constexpr int G = kThreads;
  __shared__ float part[3 * (G / kWave)];
  __shared__ Key heads[TOP ? G : 1];
  typedef TopSpace<TOP ? G : kWave, TOP ? 8 : 1> Space;
  static_assert(!TOP || kMostTop * (kMostTop + 1) / 2 <= Space::room, "the lists' candidates fit");
  __shared__ Space space;
  const int lane = threadIdx.x;
  const size_t row = blockIdx.x;
  const long long t0 = tt::read_index(o.tokens, row, o.wide);
  if (t0 == o.ignored) {
    write_ignored<G>(o, row, lane, K);
    return;
  }
  const long long t = token_place(t0, V);
  const float z_token = lane == 0 && t >= 0 ? tt::widen(x[row * (size_t)V + t]) : 0.f;
  Stat a = {-INFINITY, 0.f, 0.f};
  if (lane < splits) a = stat_part[row * splits + lane];
  a = tt::row_join<G, true>(a, (float)tt::kLog2e, part);
  if constexpr (TOP) {
    const Key* keys = key_part + row * (size_t)splits * K;
    const Key head = lane < splits ? keys[(size_t)lane * K] : 0;
    heads[lane] = head;
    if (lane == 0) {
      space.count = 0;
      space.bound = 0;
    }
    __syncthreads();
    int rank = 0;
    for (int i = 0; i < splits; ++i) rank += heads[i] > head;
    if (head != 0 && rank == K - 1) space.bound = head;
    __syncthreads();
    if (head != 0 && rank < K)
      for (int k = 0; k < K - rank; ++k) {
        const Key key = keys[(size_t)lane * K + k];
        if (key == 0 || key < space.bound) break;
        space.cand[atomicAdd(&space.count, 1)] = key;
      }
    __syncthreads();
    rank_candidates(space, lane, space.count, K);
    write_row<G>(o, row, lane, a, t >= 0, z_token, space.best, K);
  } else {
    write_row<G>(o, row, lane, a, t >= 0, z_token, nullptr, 0);
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

// dz_j = -p_j (a + sum_k c_k + h (log p_j + H)) + a [j = t] + sum_k c_k [j = i_k].
// A block (or wave, G = 64) writes packs [v0, v1) of a row without the last two terms, and then the few values that
// have them once more.
template <typename T, int G>
__global__ __launch_bounds__(kThreads) void logp_bwd(const T* __restrict__ x, BackwardIn in, T* __restrict__ dx,
                                                     int splits, int R, int V, int K) {
  constexpr int kRows = kThreads / G, n = Pack<T>::n;
  typedef typename Pack<T>::type P;
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  const float c = (float)tt::kLog2e;
  const long long items = (long long)R * splits;
  for (long long item = (long long)blockIdx.x * kRows + sub; item < items; item += (long long)gridDim.x * kRows) {
    const long long row = item / splits;
    const int split = (int)(item % splits);
    const LogitRow<T> r(x, row, V);
    T* out = tt::packs_of(dx, row, V);
    const int per = (r.packs + splits - 1) / splits;
    const int v0 = split * per, v1 = v0 + per < r.packs ? v0 + per : r.packs;
    const long long t0 = tt::read_index(in.tokens, row, in.wide), t = token_place(t0, V);
    const float2 st = in.stats[row];
    if (t0 == in.ignored || st.x == -INFINITY) {
      for (int j = v0 + lane; j < v1; j += G) tt::write_pack(r, out, j, P((T)0.f));
      continue;
    }
    const float a = in.g_logp ? in.g_logp[row] : 0.f, h = in.g_entropy ? in.g_entropy[row] : 0.f;
    const float H = in.entropy[row];
    float total = in.g_logp && t < 0 ? NAN : a;
    if (in.g_top) {
      const int at = threadIdx.x & (kWave - 1);
      total += tt::wave_sum(at < K ? in.g_top[row * K + at] : 0.f);
    }
    for (int j = v0 + lane; j < v1; j += kUnroll * G) {
      P p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u * G < v1) p[u] = r.read(j + u * G);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (j + u * G >= v1) continue;
        P q;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float d = (tt::widen(p[u][i]) - st.x) * c - st.y;
          q[i] = (T)(-tt::pow2(d) * fmaf(h, fmaf(tt::floor_at(d), tt::kLn2, H), total));
        }
        tt::write_pack(r, out, j + u * G, q);
      }
    }
    const int fixes = (in.g_logp && t >= 0 ? 1 : 0) + (in.g_top ? K : 0);
    if (fixes == 0) continue;
    // what is stored below goes over what was stored above: that has to have left first
    tt::stores_done();
    tt::sync_row<G>();
    for (int f = lane; f < fixes; f += G) {
      const bool given = in.g_logp && t >= 0;
      const long long j = given && f == 0 ? t : in.top_index[row * K + f - (given ? 1 : 0)];
      const int pack = (int)((j + r.skip) / n);
      if (j < 0 || pack < v0 || pack >= v1) continue;
      float extra = given && j == t ? a : 0.f;      // summed first: what cancels here leaves no rounding behind
      if (in.g_top)
        for (int k = 0; k < K; ++k)
          if (in.top_index[row * K + k] == j) extra += in.g_top[row * K + k];
      const float d = (tt::widen(x[row * (size_t)V + j]) - st.x) * c - st.y;
      dx[row * (size_t)V + j] = (T)fmaf(-tt::pow2(d), fmaf(h, fmaf(tt::floor_at(d), tt::kLn2, H), total), extra);
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

// Rows of up to this many packs go to a wave each, longer ones to a block.
constexpr int kWavePacks = 1024;

// How many blocks share a row: as many as fill the device eight times, each with kUnroll packs to a thread at least.
int splits_for(long long R, int packs) {
  long long want = (8LL * tt::compute_units() + R - 1) / R;
  const long long most = (packs + kUnroll * kThreads - 1) / (kUnroll * kThreads);
  if (want > most) want = most;
  if (want > kThreads) want = kThreads;
  return want < 1 ? 1 : (int)want;
}

template <typename T>
int forward(const T* x, const ForwardOut& o, int R, int V, int K) {
  hipStream_t st = tt::stream();
  const int packs = (V + Pack<T>::n - 1) / Pack<T>::n;
  const int splits = packs <= kWavePacks ? 1 : splits_for(R, packs);
  if (splits > 1) {
    void* ws;
    const size_t parts = (size_t)R * splits, stat_bytes = (parts * sizeof(Stat) + 255) / 256 * 256;
    if (tt::workspace(stat_bytes + parts * K * sizeof(Key), &ws)) return -1;
    Stat* stat_part = (Stat*)ws;
    Key* key_part = (Key*)((char*)ws + stat_bytes);
    if (K) {
      logp_split<T, true><<<(unsigned)parts, kThreads, 0, st>>>(x, o.tokens, o.wide, o.ignored, stat_part, key_part,
                                                                splits, V, K);
      TT_LAUNCH_CHECK();
      logp_join<T, true><<<R, kThreads, 0, st>>>(x, o, stat_part, key_part, splits, V, K);
    } else {
      logp_split<T, false><<<(unsigned)parts, kThreads, 0, st>>>(x, o.tokens, o.wide, o.ignored, stat_part, key_part,
                                                                 splits, V, K);
      TT_LAUNCH_CHECK();
      logp_join<T, false><<<R, kThreads, 0, st>>>(x, o, stat_part, key_part, splits, V, K);
    }
  } else if (packs <= kWavePacks) {
    const unsigned grid = grid_for((R + 3LL) / 4);
    if (K) logp_rows<T, kWave, true><<<grid, kThreads, 0, st>>>(x, o, R, V, K);
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
  if (packs <= kWavePacks) {
    logp_bwd<T, kWave><<<grid_for((R + 3LL) / 4), kThreads, 0, st>>>(x, in, dx, 1, R, V, K);
  } else {
    const int splits = splits_for(R, packs);
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
