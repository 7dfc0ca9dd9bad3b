// Distillation of a student's logits from the K best of a teacher, forward and backward (vocab.h has the statistics):
//   q = softmax(teacher / T) over a row's entries,  p = softmax(x / T) over all V
//   loss_r = T^2 sum_k q_k (log q_k - log p_(i_k)),   dx_j = g T (p_j - sum_(k: i_k = j) q_k)
//
// The loss is formed as the difference of sum q log q, which needs the teacher alone, and sum q log p: it is off by some
// 2^-23 T^2 of the size of those two (the logarithm of V at most, as a rule), however small the divergence itself is.
//
// Memory bounds them, and the fewest bytes are one read and one write of the row: the gradient for an incoming gradient
// of one is written in the visit that reads the row for the loss (4096x32768 float32 with 32 entries: 1074 MB in 205
// us, 5.2 TB/s, where a large copy reaches 5.0 to 5.6).  Of rows longer than registers and LDS hold the rest is read
// twice (1024x131072 float16 with 64 entries: 604 MB instead of 537, in 116 us, 5.2 TB/s; the vector units are busy for
// 38 % of that).  Short rows are bound by the latency of their teacher: index, then the logit there (131072 rows of 100
// with 32 entries: 34 us, 58 with the gradient).
#include "vocab.h"

namespace tt {

// A half that is divided by a temperature below kCold, where logits times c are too large for the rounded products that
// halves take as a rule (vocab.h): a row of -65504 alone at 1e-6 would sum to 2^4096.  Its differences are taken first, as
// float32 does it, which costs the halves of warmer calls up to 18 % (at 1e-4, where both would do, 22369x3000 with 32
// entries and the gradient take 61.7 us and 54.7 by products, 300x50021 21.8 and 18.5).
struct ColdHalf {
  _Float16 v;
  ColdHalf() = default;
  __device__ explicit ColdHalf(float z) : v((_Float16)z) {}
};
constexpr double kCold = 1.0 / 8192;
template <>
struct Pack<ColdHalf> : Pack<_Float16> {};
__device__ __forceinline__ float widen(ColdHalf z) { return widen(z.v); }

}  // namespace tt

namespace {

using tt::kUnroll;
using tt::kWave;
using tt::LogitRow;
using tt::Pack;
using tt::Scale;
using tt::Share;
using tt::Stat;
using tt::Words;

constexpr int kThreads = 256;
constexpr int kMostTeacher = 1024;
constexpr int kMostSplitRows = 255;     // rows that may be shared by blocks

struct Teacher {
  const void* logits;
  const void* index;
  int half, wide, K;
};

// The teacher's entry k of a row: its logit, -inf where there is none, NaN for an index behind the vocabulary.
__device__ __forceinline__ float teacher_entry(const Teacher& te, size_t at, int V, int* place) {
  const long long i = tt::read_index(te.index, at, te.wide);
  *place = i < 0 || i >= V ? 0 : (int)i;
  return i < 0 ? -INFINITY : i >= V ? NAN : tt::read_value(te.logits, at, te.half);
}

// A row's teacher in LDS, K entries each: their probabilities q, their places, the student's logits there, and a
// queue for each of the G threads that write the row's gradient (below).
struct Entries {
  float* weight;
  int* place;
  float* logit;
  int* next;
  int* queue;
};
// K rounded up, so that places can be read sixteen bytes at a time.
__host__ __device__ __forceinline__ int whole(int K) { return (K + 3) / 4 * 4; }

template <int G>
__device__ __forceinline__ Entries entries_of(float* lds, int K, int sub) {
  const int n = whole(K);
  float* at = lds + (size_t)sub * (4 * n + G);
  return {at, (int*)(at + n), at + 2 * n, (int*)(at + 3 * n), (int*)(at + 4 * n)};
}
template <int G>
size_t entries_bytes(int K, int rows) {
  return ((size_t)whole(K) * 4 + G) * sizeof(float) * rows;
}

struct TeacherSum {
  float s;            // at least 1: the row has a teacher; 0: it has none; NaN: it cannot be computed
  float q_log_q;      // sum_k q_k log2 q_k
};

template <typename T, int G>
__device__ __forceinline__ TeacherSum read_teacher(const Teacher& te, const T* x, const LogitRow<T>& r, size_t row,
                                                   float c, int lane, const Entries& e, float* part) {
  Stat a = {-INFINITY, 0.f, 0.f};
  e.queue[lane] = -1;
  if (lane < whole(te.K) - te.K) e.place[te.K + lane] = -1;
  for (int k = lane; k < te.K; k += G) {
    int i;
    const float z = teacher_entry(te, row * te.K + k, r.V, &i);
    e.weight[k] = z;
    e.place[k] = i;
    e.logit[k] = tt::widen(x[r.start + i]);
    tt::add_value<float, true>(a, z, c);
  }
  a = tt::row_join<float, G, true>(a, c, part);
  const float log_s = tt::log_sum(a), m = tt::anchor(a.m);
  for (int k = lane; k < te.K; k += G) e.weight[k] = a.s == 0.f ? 0.f : tt::pow2((e.weight[k] - m) * c - log_s);
  tt::sync_row<G>();
  return {a.s, a.s == 0.f ? 0.f : a.t / a.s - log_s};
}

// This thread's part of sum_k q_k (-log p_(i_k)).
template <typename T, int G>
__device__ __forceinline__ float cross_entropy(const Entries& e, int K, int lane, const Stat& a, float log_s,
                                               const Scale& sc) {
  float s = 0.f;
  for (int k = lane; k < K; k += G) {
    const float w = e.weight[k];
    if (w != 0.f) s -= w * tt::log_p<T>(e.logit[k], tt::anchor(a.m), log_s, sc);
  }
  return s;
}

// The gradient at the teacher's entries has q in it, which the threads that write a row's packs do not know.  Each such
// value is queued for the thread that writes its pack, which stores it after that: a thread's own stores stay in order,
// so nobody waits for them.  The values go where the logits were.
template <typename T, int G>
__device__ __forceinline__ void queue_entries(const Entries& e, const LogitRow<T>& r, const Share& s, int K, int lane,
                                              float m, float log_s, float c, float scale) {
  for (int k = lane; k < K; k += G) {
    const int j = e.place[k], pack = (j + r.skip) / Pack<T>::n;
    if (e.weight[k] == 0.f) continue;
    int owner;
    if (j < r.head) {
      if (s.head == 0) continue;
      owner = j % G;
    } else if (j >= r.tail_at) {
      if (s.tail == 0) continue;
      owner = (s.head + j - r.tail_at) % G;
    } else {
      if (pack < s.p0 || pack >= s.p1) continue;
      owner = (pack - s.p0) % G;
    }
    int same = 0;
    for (int i = 0; i < K; i += 4) {
      const int4 p = *reinterpret_cast<const int4*>(e.place + i);
      same += (p.x == j) + (p.y == j) + (p.z == j) + (p.w == j);
    }
    float q = e.weight[k];
    if (same > 1) {
      q = 0.f;
      for (int i = 0; i < K; ++i) q += e.place[i] == j ? e.weight[i] : 0.f;
    }
    e.logit[k] = scale * (tt::pow2(tt::bits<T>(e.logit[k], m, c) - log_s) - q);
    e.next[k] = atomicExch(&e.queue[owner], k);
  }
  tt::sync_row<G>();
}
// Of its queue a thread takes the first P entries of packs into registers, and into the packs as it writes them; `rest`
// is stored behind the packs.  (A lone value costs memory a piece of 64 bytes: 131072 rows of 300 with 32 entries take
// 103 us with P = 4 and 137 us with none, 67108 of 1000 with P = 2 118 and 180; but of 100 57 and 54.  Of long rows they are few, so P = 0.)
template <int G>
constexpr int kPatches = G < kWave ? 4 : G == kWave ? 2 : 0;
template <int P>
struct Patches {
  int at[P ? P : 1];
  float value[P ? P : 1];
  int rest;
};
template <typename T, int P>
__device__ __forceinline__ Patches<P> take_queued(const Entries& e, const LogitRow<T>& r, int lane) {
  Patches<P> t;
  int k = e.queue[lane];
  t.rest = k;
  if constexpr (P > 0) {
    t.rest = -1;
#pragma unroll
    for (int i = 0; i < P; ++i) t.at[i] = -1;
    for (int taken = 0; k >= 0;) {
      const int j = e.place[k], next = e.next[k];
      if (taken < P && j >= r.head && j < r.tail_at) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          t.at[i] = i == taken ? j + r.skip : t.at[i];
          t.value[i] = i == taken ? e.logit[k] : t.value[i];
        }
        ++taken;
      } else {
        e.next[k] = t.rest;
        t.rest = k;
      }
      k = next;
    }
  }
  return t;
}
template <typename T, int P>
__device__ __forceinline__ void patch(float (&z)[Pack<T>::n], const Patches<P>& t, int j) {
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int i0 = t.at[p] - j * Pack<T>::n;
#pragma unroll
    for (int i = 0; i < Pack<T>::n; ++i) z[i] = i0 == i ? t.value[p] : z[i];
  }
}
template <typename T>
__device__ __forceinline__ void store_rest(const Entries& e, T* dx, const LogitRow<T>& r, int rest) {
  asm volatile("" ::: "memory");      // (behind the packs' stores for the compiler too, to which they are another type)
  for (int k = rest; k >= 0; k = e.next[k]) dx[r.start + e.place[k]] = (T)e.logit[k];
}

// What the rows leave behind, and what the last block makes of it.
struct Out {
  float* loss;        // of each row, where that is wanted
  float2* stats;      // for the backward pass
  double* sums;       // of each block's rows: their losses, and how many have a teacher
  float* total;       // the rows' sum, or over the count for the mean; NULL: not wanted
  float* count;       // how many rows have a teacher
  int mean;
};

// A row without a teacher is an empty one for the backward pass, as one without any possible class: no gradient.
__device__ __forceinline__ double write_row(const Out& o, size_t row, const Stat& a, float log_s, const TeacherSum& te,
                                            float cross, const Scale& sc) {
  const bool none = te.s == 0.f;
  const float loss = none ? 0.f : fmaf(te.q_log_q, tt::kLn2, cross) * (sc.temperature * sc.temperature);
  if (o.loss) o.loss[row] = loss;
  o.stats[row] = none || tt::is_empty(a.m, a.s) ? make_float2(-INFINITY, 0.f)
                                                : make_float2(a.m, te.s == te.s ? log_s : te.s);
  return loss;
}

// The block's number `at` of `all` is done with its rows.  The one that comes last adds up what they all leave, in 64
// bits and in an order that the sizes alone decide.  `part` is LDS of 2 BLOCK / 64 values.
template <int BLOCK>
__device__ __forceinline__ void add_up(const Out& o, tt::Ticket* done, unsigned at, unsigned all, double loss,
                                       double rows, double* part) {
  __shared__ bool last;
  loss = tt::row_sum<BLOCK>(loss, part);
  rows = tt::row_sum<BLOCK>(rows, part + BLOCK / kWave);
  if (threadIdx.x == 0) {
    tt::share(o.sums + 2 * (size_t)at, loss);
    tt::share(o.sums + 2 * (size_t)at + 1, rows);
    tt::stores_done();
    last = tt::last_ticket(done, at, all);
  }
  __syncthreads();
  if (!last) return;
  loss = rows = 0.0;
  for (unsigned i = threadIdx.x; i < all; i += BLOCK) {
    loss += tt::shared(o.sums + 2 * (size_t)i);
    rows += tt::shared(o.sums + 2 * (size_t)i + 1);
  }
  loss = tt::row_sum<BLOCK>(loss, part);
  rows = tt::row_sum<BLOCK>(rows, part + BLOCK / kWave);
  if (threadIdx.x == 0) {
    if (o.total) o.total[0] = (float)(o.mean ? loss / rows : loss);
    o.count[0] = (float)rows;
  }
}

// scale p of the values of pack j, and the patches.  (log2(scale) in the exponent would spare halves a product: 1024x131072
// with 64 entries 106 us where this takes 109.  But a sum of it with m c is rounded at the size of m c, 2e-3 of the
// gradient in a row of -65504 alone, and added to the difference it is no faster.)
template <typename T, int P>
__device__ __forceinline__ Words gradient_pack(const Words& p, const Patches<P>& t, int j, float m, float log_s,
                                               float c, float scale) {
  float z[Pack<T>::n];
  tt::unpack<T>(z, p);
#pragma unroll
  for (int i = 0; i < Pack<T>::n; ++i) z[i] = scale * tt::pow2(tt::bits<T>(z[i], m, c) - log_s);
  patch<T, P>(z, t, j);
  return tt::pack<T>(z);
}

// The values of NV packs, or the first `packs` of them: their maximum first, then their sum, so that there is no chain
// of rescaled sums. The packs are opaque to the compiler in between, which would otherwise hold all their widened
// values from one loop to the other.
template <typename T, int NV>
__device__ __forceinline__ void add_kept(Stat& a, Words (&kept)[NV], int packs, float c) {
  constexpr int n = Pack<T>::n;
  const float most = tt::pack_max<T, NV>(kept);
  if (most > a.m) tt::rescale<T, false>(a, most, c);
  const float m = tt::anchor(a.m);
  float s[4] = {};
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    asm volatile("" : "+v"(kept[u]));
    if (u >= packs) continue;
    float z[n];
    tt::unpack<T>(z, kept[u]);
#pragma unroll
    for (int i = 0; i < n; ++i) s[i % 4] += tt::pow2(tt::bits<T>(z[i], m, c));
    __builtin_amdgcn_sched_barrier(0);
  }
  a.s += (s[0] + s[1]) + (s[2] + s[3]);
}

template <typename T, int G>
__device__ __forceinline__ void write_loose(const T* x, T* dx, const LogitRow<T>& r, const Share& s, int lane,
                                            bool none, float m, float log_s, float c, float scale) {
  for (int i = lane; i < s.head + s.tail; i += G) {
    const size_t at = r.start + tt::loose_column(r, s, i);
    dx[at] = none ? (T)0.f : (T)(scale * tt::pow2(tt::bits<T>(tt::widen(x[at]), m, c) - log_s));
  }
}

__device__ __forceinline__ bool has_teacher(const Teacher& te, size_t row, int V) {
  for (int k = 0; k < te.K; ++k) {        // (the first entry decides, as a rule)
    int i;
    if (teacher_entry(te, row * te.K + k, V, &i) != -INFINITY) return true;
  }
  return false;
}

// How many rows have a teacher, in parts: one whole number for each block.
constexpr int kCountBlocks = 256;
__global__ __launch_bounds__(kThreads) void distill_count(Teacher te, int* __restrict__ parts, int R, int V) {
  constexpr int kLanes = 16;              // to a row
  __shared__ int part[kThreads / kWave];
  const int lane = threadIdx.x % kLanes, shift = (threadIdx.x & (kWave - 1)) / kLanes * kLanes;
  int n = 0;
  for (long long row = ((long long)blockIdx.x * kThreads + threadIdx.x) / kLanes; row < R;
       row += (long long)gridDim.x * (kThreads / kLanes)) {
    bool any = false;
    for (int k = lane; k < te.K; k += kLanes) {
      int i;
      any |= teacher_entry(te, row * te.K + k, V, &i) != -INFINITY;
    }
    const unsigned long long rows = __ballot(any);
    if (lane == 0 && (rows >> shift & 0xffffu) != 0) ++n;
  }
  n = tt::row_sum<kThreads>(n, part);
  if (threadIdx.x == 0) parts[blockIdx.x] = n;
}

__device__ tt::Ticket distill_done[1 + tt::kBranches], distill_tickets[kMostSplitRows];

// Of a longer row than the registers hold, LDS takes this many packs more of each thread (1024x131072 float16: 126 us
// without, 117 with them); the loop over them and what is left has few registers.
constexpr int kShelf = 8, kPair = 2;

// Rows of G threads each: loss, statistics and, with GRAD, the gradient for an incoming gradient of one. For that the
// row is kept in registers, NV packs to a thread, and costs one read and one write; of a longer row (LONG) kShelf packs
// more go to LDS and the rest is read a second time. For the mean's gradient the rows with a teacher are counted first:
// by each block, or from `count_parts`.
template <typename T, int G, int NV, bool LONG, bool GRAD>
__global__ __launch_bounds__(G < kThreads ? kThreads : G, G == 512 ? 4 : 1) void distill_rows(
    const T* __restrict__ x, Teacher te, Out o, T* dx, const int* __restrict__ count_parts, Scale sc, int R, int V) {
  constexpr int kBlock = G < kThreads ? kThreads : G, kRows = kBlock / G;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float part[kRows][tt::parts_of(G, 3)];
  __shared__ float more[kRows][tt::parts_of(G, 4)];
  __shared__ double sums[2 * (kBlock / kWave)];
  const int lane = threadIdx.x % G, sub = tt::row_of_block<G>();
  Words* shelf = reinterpret_cast<Words*>(lds);
  const Entries e = entries_of<G>(lds + (LONG && GRAD ? kShelf * G * 4 : 0), te.K, sub);
  double losses = 0.0, rows = 0.0;
  float scale = sc.temperature;
  if (GRAD && o.mean) {
    int n = 0;
    if (count_parts) {
      for (int i = threadIdx.x; i < kCountBlocks; i += kBlock) n += count_parts[i];
    } else {
      for (int i = threadIdx.x; i < R; i += kBlock) n += has_teacher(te, i, V) ? 1 : 0;
    }
    scale /= (float)tt::row_sum<kBlock>(n, (int*)sums);
  }
  for (long long row = (long long)blockIdx.x * kRows + sub; row < R; row += (long long)gridDim.x * kRows) {
    const LogitRow<T> r(x, row, V);
    const Share all(r, 0, 1);
    Words kept[NV ? NV : 1];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      kept[u] = Words(Pack<T>::lowest);
      if (all.p0 + lane + u * G < all.p1) kept[u] = r.pack(all.p0 + lane + u * G);
    }
    const TeacherSum ts = read_teacher<T, G>(te, x, r, row, sc.c, lane, e, part[sub]);
    Stat a = {-INFINITY, 0.f, 0.f};
    Share rest = all;
    rest.p0 = LONG && all.p0 + NV * G < all.p1 ? all.p0 + NV * G : all.p1;
    int best;
    tt::scan<T, G, false, LONG && !GRAD>(a, best, x, r, rest, lane, sc.c);
    if constexpr (NV > 0) add_kept<T, NV>(a, kept, G > kWave ? NV : (all.p1 - all.p0 + G - 1) / G, sc.c);
    if constexpr (LONG && GRAD)
      for (int j = rest.p0 + lane, i = 0; j < rest.p1; j += kPair * G, i += kPair) {
        Words p[kPair];
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
          p[u] = Words(Pack<T>::lowest);
          if (j + u * G < rest.p1) p[u] = r.pack(j + u * G);
        }
        if (i < kShelf) {
#pragma unroll
          for (int u = 0; u < kPair; ++u) shelf[(i + u) * G + lane] = p[u];
        }
        tt::add_packs<T, kPair, false>(a, p, sc.c);
      }
    a = tt::row_join<T, G, false>(a, sc.c, more[sub]);
    const float log_s = tt::log_sum(a);
    float cross = cross_entropy<T, G>(e, te.K, lane, a, log_s, sc);
    if constexpr (GRAD) {
      const bool none = ts.s == 0.f || tt::is_empty(a.m, a.s);
      const float by = ts.s == ts.s ? scale : ts.s;
      if (!none) queue_entries<T, G>(e, r, all, te.K, lane, a.m, log_s, sc.c, by);
      const Patches<kPatches<G>> patches = take_queued<T, kPatches<G>>(e, r, lane);
      int own = all.p0 + lane;        // (opaque as the packs are: no address is held from the reads to here)
      asm volatile("" : "+v"(own));
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        asm volatile("" : "+v"(kept[u]));
        const int j = own + u * G;
        if (j < all.p1) {
          const Words q = none ? Words(0u) : gradient_pack<T>(kept[u], patches, j, a.m, log_s, sc.c, by);
          tt::write_pack(r, dx, j, q);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (LONG)
        for (int j = rest.p0 + lane, i = 0; j < rest.p1; j += kPair * G, i += kPair) {
          Words p[kPair];
#pragma unroll
          for (int u = 0; u < kPair; ++u)
            if (j + u * G < rest.p1) p[u] = i < kShelf ? shelf[(i + u) * G + lane] : r.pack(j + u * G);
#pragma unroll
          for (int u = 0; u < kPair; ++u)
            if (j + u * G < rest.p1)
              tt::write_pack(r, dx, j + u * G,
                             none ? Words(0u) : gradient_pack<T>(p[u], patches, j + u * G, a.m, log_s, sc.c, by));
        }
      write_loose<T, G>(x, dx, r, all, lane, none, a.m, log_s, sc.c, by);
      store_rest(e, dx, r, patches.rest);
    }
    cross = tt::row_sum<G>(cross, more[sub] + tt::parts_of(G, 3) % tt::parts_of(G, 4));
    if (lane == 0) {
      losses += write_row(o, row, a, log_s, ts, cross, sc);
      rows += ts.s == 0.f ? 0.0 : 1.0;
    }
    tt::sync_row<G>();
  }
  __syncthreads();
  add_up<kBlock>(o, distill_done, blockIdx.x, gridDim.x, losses, rows, sums);
}

// Few long rows: `splits` blocks to a row, each with the sums of its share; the one that comes last puts them together,
// and the one whose row is the last of all adds up the rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void distill_split(const T* __restrict__ x, Teacher te, Out o, float* stat_part,
                                                          Scale sc, int splits, int R, int V) {
  constexpr int G = kThreads;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float part[3 * (G / kWave)];
  __shared__ float more[4 * (G / kWave)];
  __shared__ double sums[2 * (G / kWave)];
  __shared__ bool last;
  const int split = blockIdx.x % splits, lane = threadIdx.x;
  const size_t row = blockIdx.x / splits;
  const Entries e = entries_of<G>(lds, te.K, 0);
  const LogitRow<T> r(x, row, V);
  Stat a = {-INFINITY, 0.f, 0.f};
  int best;
  tt::scan<T, G, false>(a, best, x, r, Share(r, split, splits), lane, sc.c);
  a = tt::row_join<T, G, false>(a, sc.c, part);
  if (lane == 0) {
    tt::share(stat_part + (size_t)blockIdx.x * 2, a.m);
    tt::share(stat_part + (size_t)blockIdx.x * 2 + 1, a.s);
    tt::stores_done();
    last = tt::last_ticket(distill_tickets + row, splits);
  }
  __syncthreads();
  if (!last) return;
  Stat whole = {-INFINITY, 0.f, 0.f};
  if (lane < splits) {
    whole.m = tt::shared(stat_part + (row * splits + lane) * 2);
    whole.s = tt::shared(stat_part + (row * splits + lane) * 2 + 1);
  }
  const TeacherSum ts = read_teacher<T, G>(te, x, r, row, sc.c, lane, e, part);
  whole = tt::row_join<T, G, false>(whole, sc.c, more);
  const float log_s = tt::log_sum(whole);
  const float cross = tt::row_sum<G>(cross_entropy<T, G>(e, te.K, lane, whole, log_s, sc), more + 3 * (G / kWave));
  const double loss = lane == 0 ? write_row(o, row, whole, log_s, ts, cross, sc) : 0.0;
  add_up<G>(o, distill_done, row, R, loss, lane == 0 && ts.s != 0.f ? 1.0 : 0.0, sums);
}

// The gradient from the kept statistics.  With `ahead` the forward pass has written it for an incoming gradient of one
// already: then that is looked at first, and only another one makes work.
template <typename T, int G>
__global__ __launch_bounds__(kThreads) void distill_bwd(const T* __restrict__ x, Teacher te,
                                                        const float2* __restrict__ stats,
                                                        const float* __restrict__ count, const float* __restrict__ g,
                                                        T* dx, Scale sc, int reduction, int ahead, int splits, int R,
                                                        int V) {
  constexpr int kRows = kThreads / G;
  if (ahead && g[0] == 1.f) return;
  extern __shared__ __attribute__((aligned(16))) float lds[];
  __shared__ float part[kRows][tt::parts_of(G, 3)];
  const int lane = threadIdx.x % G, sub = tt::row_of_block<G>();
  const Entries e = entries_of<G>(lds, te.K, sub);
  const long long items = (long long)R * splits;
  for (long long item = (long long)blockIdx.x * kRows + sub; item < items; item += (long long)gridDim.x * kRows) {
    const size_t row = R - 1 - item / splits;     // (what the forward pass read last may still be cached)
    const LogitRow<T> r(x, row, V);
    const Share s(r, (int)(item % splits), splits);
    const float2 st = stats[row];
    const bool none = tt::is_empty(st.x, st.y);
    float scale = sc.temperature * (reduction == 0 ? g[row] : g[0]);
    if (reduction == 2) scale /= count[0];
    if (none) {
      e.queue[lane] = -1;
    } else {
      read_teacher<T, G>(te, x, r, row, sc.c, lane, e, part[sub]);
      queue_entries<T, G>(e, r, s, te.K, lane, st.x, st.y, sc.c, scale);
    }
    const Patches<kPatches<G>> patches = take_queued<T, kPatches<G>>(e, r, lane);
    for (int j = s.p0 + lane; j < s.p1; j += kUnroll * G) {
      Words p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (!none && j + u * G < s.p1) p[u] = r.pack(j + u * G);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u * G < s.p1)
          tt::write_pack(r, dx, j + u * G,
                         none ? Words(0u) : gradient_pack<T>(p[u], patches, j + u * G, st.x, st.y, sc.c, scale));
    }
    write_loose<T, G>(x, dx, r, s, lane, none, st.x, st.y, sc.c, scale);
    store_rest(e, dx, r, patches.rest);
    tt::sync_row<G>();
  }
}

// ---- launches --------------------------------------------------------------------------------------

int check(const char* fn, int dtype, int teacher_dtype, int index_bits, double temperature, int reduction, long long R,
          int V, int K) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_F16, "%s: unknown type %d", fn, dtype);
  TT_REQUIRE(teacher_dtype == TT_F32 || teacher_dtype == TT_F16, "%s: unknown type %d", fn, teacher_dtype);
  TT_REQUIRE(index_bits == 32 || index_bits == 64, "%s: indexes have 32 or 64 bits (got %d)", fn, index_bits);
  TT_REQUIRE(temperature >= 1e-6 && temperature <= 1e6, "%s: temperature must be in 1e-6..1e6 (got %g)", fn,
             temperature);
  TT_REQUIRE(reduction >= 0 && reduction <= 2, "%s: reduction must be 0 (none), 1 (sum) or 2 (mean)", fn);
  TT_REQUIRE(R > 0 && R <= (1 << 30), "%s: rows must be in 1..2^30 (got %lld)", fn, R);
  TT_REQUIRE(V > 0 && V <= (1 << 30), "%s: the vocabulary must have 1..2^30 entries (got %d)", fn, V);
  TT_REQUIRE(K >= 1 && K <= kMostTeacher, "%s: teacher entries must be in 1..%d (got %d)", fn, kMostTeacher, K);
  return 0;
}

constexpr long long kMostBlocks = 16;      // of a launch, to a compute unit; they take rows in turn
unsigned grid_for(long long blocks, long long most) { return (unsigned)(blocks < most ? blocks : most); }

// Rows of up to kWavePacks packs go to a wave each, which keeps them in registers; four of them share a block's LDS,
// where the teacher's entries have to fit. (22369 rows of 3000 in float32 with 32 entries and their gradient: 114 us,
// by blocks 134.) Short ones go to kLanes lanes each: 131072 rows of 300 with 32 entries take 101 us, by waves 144.
constexpr int kWavePacks = 16 * kWave, kWaveEntries = 256;
bool by_waves(int packs, int K) { return packs <= kWavePacks && K <= kWaveEntries; }
constexpr int kLanes = 16, kLanesPacks = 8 * kLanes, kLanesEntries = 64;
bool by_lanes(int packs, int K) { return packs <= kLanesPacks && K <= kLanesEntries; }

int packs_for(int V, int dtype) { return dtype == TT_F32 ? (V + 3) / 4 : (V + 7) / 8; }

// Rows shared by blocks, where they are fewer than units: the block that joins a row reads its teacher last. (300 rows
// of 50021 take 15.6 us whole and 16.7 shared, 512 of 131072 49 and 52; 100 of 131072 25 and 15 us.)
int forward_splits(long long R, int packs) {
  if (packs <= kWavePacks || R > kMostSplitRows) return 1;
  return tt::splits_for(R, packs, kThreads, 2, kUnroll * kThreads);
}
// Where the backward pass has more than those, it has fewer than that of log probabilities, for each block reads the
// row's teacher (1300 rows of 50021 with 32 entries: 120 -> 110 us, with as many as there 103; but of 2047 in float16 96 us,
// with as many 99).
int backward_splits(long long R, int packs) {
  const int few = tt::splits_for(R, packs, kThreads, 8, kUnroll * kThreads);
  const int many = tt::splits_for(R, packs, kThreads, 16, 4 * kUnroll * kThreads);
  return few > many ? few : many;
}

// A row to a block, loss and gradient in one visit: while it fits the registers, which saves two launches (20 rows of
// 10000: 10 us, 13 us shared by blocks), and longer ones from half as many rows as there are units on (140 rows of
// 131072 42 and 45 us, 80 rows 34 and 32 us).
bool whole_rows(long long R, int packs) { return packs <= 16 * 512 || 2 * R >= tt::compute_units(); }

// Whether the forward pass writes the gradient too, for an incoming gradient of one: where a row's own block does it
// (the row is then read once for both), and that gradient is the likely one.  A loss for each row is weighted by its
// user, and float16 gradients of a mean have to be scaled to be held at all, so those wait for the backward pass.
bool ahead(int dtype, int reduction, long long R, int V) {
  return whole_rows(R, packs_for(V, dtype)) && (reduction == 1 || (reduction == 2 && dtype == TT_F32));
}

template <typename T, bool GRAD>
int launch_rows(const T* x, const Teacher& te, const Out& o, T* dx, const int* count_parts, const Scale& sc, int R,
                int V, int packs) {
  hipStream_t st = tt::stream();
  const long long most = kMostBlocks * tt::compute_units();
  const size_t wave_lds = entries_bytes<kWave>(te.K, kThreads / kWave);
  constexpr int kRows = kThreads / kLanes;
  if (GRAD && by_lanes(packs, te.K) && packs <= 2 * kLanes) {
    distill_rows<T, kLanes, 2, false, true>
        <<<grid_for((R + kRows - 1LL) / kRows, most), kThreads, entries_bytes<kLanes>(te.K, kRows), st>>>(
            x, te, o, dx, count_parts, sc, R, V);
  } else if (by_lanes(packs, te.K)) {
    distill_rows<T, kLanes, GRAD ? 8 : 0, !GRAD, GRAD>
        <<<grid_for((R + kRows - 1LL) / kRows, most), kThreads, entries_bytes<kLanes>(te.K, kRows), st>>>(
            x, te, o, dx, count_parts, sc, R, V);
  } else if constexpr (!GRAD) {
    if (by_waves(packs, te.K))
      distill_rows<T, kWave, 0, true, false><<<grid_for((R + 3LL) / 4, most), kThreads, wave_lds, st>>>(
          x, te, o, dx, count_parts, sc, R, V);
    else
      distill_rows<T, 256, 0, true, false><<<grid_for(R, most), 256, entries_bytes<256>(te.K, 1), st>>>(
          x, te, o, dx, count_parts, sc, R, V);
  } else if (by_waves(packs, te.K) && packs > 8 * kWave) {
    distill_rows<T, kWave, 16, false, true><<<grid_for((R + 3LL) / 4, most), kThreads, wave_lds, st>>>(
        x, te, o, dx, count_parts, sc, R, V);
  } else if (by_waves(packs, te.K)) {
    distill_rows<T, kWave, 8, false, true><<<grid_for((R + 3LL) / 4, most), kThreads, wave_lds, st>>>(
        x, te, o, dx, count_parts, sc, R, V);
  } else if (packs <= 8 * 256) {
    distill_rows<T, 256, 8, false, true><<<grid_for(R, most), 256, entries_bytes<256>(te.K, 1), st>>>(
        x, te, o, dx, count_parts, sc, R, V);
  } else if (packs <= 16 * 512) {
    distill_rows<T, 512, 16, false, true><<<grid_for(R, most), 512, entries_bytes<512>(te.K, 1), st>>>(
        x, te, o, dx, count_parts, sc, R, V);
  } else {
    const size_t lds = entries_bytes<512>(te.K, 1) + kShelf * 512 * sizeof(Words);
    distill_rows<T, 512, 16, true, true><<<grid_for(R, most), 512, lds, st>>>(x, te, o, dx, count_parts, sc, R, V);
  }
  TT_LAUNCH_CHECK();
  return 0;
}

Scale scale_for(double temperature) {
  return {(float)(tt::kLog2e / temperature), (float)(1.0 / temperature), (float)temperature};
}

template <typename T>
int forward(const T* x, const Teacher& te, float* loss, float* stats, float* count, T* dx, double temperature,
            int reduction, int R, int V) {
  hipStream_t st = tt::stream();
  const Scale sc = scale_for(temperature);
  const int packs = (V + Pack<T>::n - 1) / Pack<T>::n;
  const int splits = dx ? 1 : forward_splits(R, packs);
  const size_t blocks = splits > 1 ? R : kMostBlocks * (size_t)tt::compute_units();
  const size_t words = kCountBlocks + (size_t)R * splits * 2;
  void* ws;
  if (tt::workspace(blocks * 2 * sizeof(double) + words * sizeof(float), &ws)) return -1;
  double* sums = (double*)ws;
  int* parts = (int*)(sums + 2 * blocks);
  float* stat_part = (float*)(parts + kCountBlocks);
  const Out o = {reduction == 0 ? loss : nullptr, (float2*)stats, sums, reduction == 0 ? nullptr : loss, count,
                 reduction == 2};
  if (splits > 1) {
    distill_split<T><<<(unsigned)(R * splits), kThreads, entries_bytes<kThreads>(te.K, 1), st>>>(
        x, te, o, stat_part, sc, splits, R, V);
    TT_LAUNCH_CHECK();
    return 0;
  }
  if (!dx) return launch_rows<T, false>(x, te, o, dx, nullptr, sc, R, V, packs);
  // each block counts this many rows by itself in the time of a launch (900 rows of 1000: 9.6 and 10.7 us, 1500 rows
  // 11.2 and 11.5, 4096 rows 21 and 15)
  const bool counts_itself = R <= 1024;
  if (reduction == 2 && !counts_itself) {
    distill_count<<<kCountBlocks, kThreads, 0, st>>>(te, parts, R, V);
    TT_LAUNCH_CHECK();
  }
  return launch_rows<T, true>(x, te, o, dx, counts_itself ? nullptr : parts, sc, R, V, packs);
}

template <typename T>
int backward(const T* x, const Teacher& te, const float* stats, const float* count, const float* g, T* dx,
             double temperature, int reduction, int is_ahead, int R, int V) {
  hipStream_t st = tt::stream();
  const Scale sc = scale_for(temperature);
  const int packs = (V + Pack<T>::n - 1) / Pack<T>::n;
  if (by_lanes(packs, te.K)) {
    constexpr int kRows = kThreads / kLanes;
    distill_bwd<T, kLanes><<<grid_for((R + kRows - 1LL) / kRows, kMostBlocks * tt::compute_units()), kThreads,
                             entries_bytes<kLanes>(te.K, kRows), st>>>(
        x, te, (const float2*)stats, count, g, dx, sc, reduction, is_ahead, 1, R, V);
  } else if (by_waves(packs, te.K)) {
    distill_bwd<T, kWave><<<grid_for((R + 3LL) / 4, kMostBlocks * tt::compute_units()), kThreads,
                            entries_bytes<kWave>(te.K, kThreads / kWave), st>>>(
        x, te, (const float2*)stats, count, g, dx, sc, reduction, is_ahead, 1, R, V);
  } else {
    const int splits = backward_splits(R, packs);
    distill_bwd<T, kThreads><<<grid_for((long long)R * splits, kMostBlocks * tt::compute_units()), kThreads,
                               entries_bytes<kThreads>(te.K, 1), st>>>(
        x, te, (const float2*)stats, count, g, dx, sc, reduction, is_ahead, splits, R, V);
  }
  TT_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" {

int tt_distill_ahead(int* yes, int dtype, int reduction, long long R, int V) {
  TT_REQUIRE_INIT();
  TT_REQUIRE(yes != nullptr, "tt_distill_ahead: null pointer");
  *yes = ahead(dtype, reduction, R, V) ? 1 : 0;
  return 0;
}

int tt_distill_fwd(const void* x, const void* teacher, const void* index, float* loss, float* stats, float* count,
                   void* dx, double temperature, int reduction, int dtype, int teacher_dtype, int index_bits,
                   long long R, int V, int K) {
  TT_REQUIRE_INIT();
  const char* fn = "tt_distill_fwd";
  TT_REQUIRE(x && teacher && index && loss && stats && count, "%s: null pointer", fn);
  if (int rc = check(fn, dtype, teacher_dtype, index_bits, temperature, reduction, R, V, K)) return rc;
  TT_REQUIRE(dx == nullptr || ahead(dtype, reduction, R, V), "%s: the gradient is not written ahead of this call", fn);
  TT_REQUIRE_ALIGNED(fn, x, stats, dx);
  const Teacher te = {teacher, index, teacher_dtype == TT_F16, index_bits == 64, K};
  if (dtype == TT_F32)
    return forward((const float*)x, te, loss, stats, count, (float*)dx, temperature, reduction, (int)R, V);
  if (temperature < tt::kCold)
    return forward((const tt::ColdHalf*)x, te, loss, stats, count, (tt::ColdHalf*)dx, temperature, reduction, (int)R, V);
  return forward((const _Float16*)x, te, loss, stats, count, (_Float16*)dx, temperature, reduction, (int)R, V);
}

int tt_distill_bwd(const void* x, const void* teacher, const void* index, const float* stats, const float* count,
                   const float* g, void* dx, double temperature, int reduction, int is_ahead, int dtype,
                   int teacher_dtype, int index_bits, long long R, int V, int K) {
  TT_REQUIRE_INIT();
  const char* fn = "tt_distill_bwd";
  TT_REQUIRE(x && teacher && index && stats && count && g && dx, "%s: null pointer", fn);
  if (int rc = check(fn, dtype, teacher_dtype, index_bits, temperature, reduction, R, V, K)) return rc;
  TT_REQUIRE(!is_ahead || ahead(dtype, reduction, R, V), "%s: the gradient was not written ahead of this call", fn);
  TT_REQUIRE_ALIGNED(fn, x, dx, stats);
  const Teacher te = {teacher, index, teacher_dtype == TT_F16, index_bits == 64, K};
  if (dtype == TT_F32)
    return backward((const float*)x, te, stats, count, g, (float*)dx, temperature, reduction, is_ahead, (int)R, V);
  if (temperature < tt::kCold)
    return backward((const tt::ColdHalf*)x, te, stats, count, g, (tt::ColdHalf*)dx, temperature, reduction, is_ahead,
                    (int)R, V);
  return backward((const _Float16*)x, te, stats, count, g, (_Float16*)dx, temperature, reduction, is_ahead, (int)R, V);
}

}  // extern "C"
