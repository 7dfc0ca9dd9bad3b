// Distillation of a student's logits from the K best of a teacher, forward and backward (vocab.h has the statistics):
//   q = softmax(teacher / T) over a row's entries,  p = softmax(x / T) over all V
//   loss_r = T^2 sum_k q_k (log q_k - log p_(i_k)),   dx_j = g T (p_j - sum_(k: i_k = j) q_k)
#include "vocab.h"

namespace {

using tt::kWave;
using tt::LogitRow;
using tt::Pack;
using tt::Stat;

constexpr int kThreads = 256;
constexpr int kMostTeacher = 1024;
constexpr int kUnroll = 4;
constexpr int kCountBlocks = 256;

struct Teacher {
  const void* logits;
  const void* index;
  int half, wide, K;
};

struct Scale {
  float c;            // log2(e) / T
  float inverse;      // 1 / T
  float temperature;
};

// The teacher's entry k of a row: its logit, -inf where there is none, NaN for an index behind the vocabulary.
__device__ __forceinline__ float teacher_entry(const Teacher& te, size_t at, int V, int* place) {
  const long long i = tt::read_index(te.index, at, te.wide);
  *place = i < 0 || i >= V ? 0 : (int)i;
  return i < 0 ? -INFINITY : i >= V ? NAN : tt::read_value(te.logits, at, te.half);
}

// The teacher's distribution of a row: weight[k] = q_k and place[k], LDS of K each.
struct TeacherSum {
  float s;            // at least 1: the row has a teacher; 0: it has none; NaN: it cannot be computed
  float q_log_q;      // sum_k q_k log2 q_k
};

template <int G>
__device__ __forceinline__ TeacherSum read_teacher(const Teacher& te, size_t row, int V, float c, int lane,
                                                   float* weight, int* place, float* part) {
  Stat a = {-INFINITY, 0.f, 0.f};
  for (int k = lane; k < te.K; k += G) {
    int i;
    const float z[1] = {teacher_entry(te, row * te.K + k, V, &i)};
    weight[k] = z[0];
    place[k] = i;
    tt::add_values<1, true>(a, z, c);
  }
  a = tt::row_join<G, true>(a, c, part);
  const float log_s = tt::log_sum(a), m = tt::anchor(a.m);
  for (int k = lane; k < te.K; k += G) weight[k] = a.s == 0.f ? 0.f : tt::pow2((weight[k] - m) * c - log_s);
  tt::sync_row<G>();
  return {a.s, a.s == 0.f ? 0.f : a.t / a.s - log_s};
}

// sum_k q_k (-log p_(i_k)) of a row; every thread gets it.
template <typename T, int G>
__device__ __forceinline__ float cross_entropy(const T* x, size_t row, int V, const Stat& a, float log_s, float inverse,
                                               int K, int lane, const float* weight, const int* place, float* part) {
  float s = 0.f;
  for (int k = lane; k < K; k += G) {
    const float w = weight[k];
    if (w != 0.f)
      s -= w * ((tt::widen(x[row * (size_t)V + place[k]]) - tt::anchor(a.m)) * inverse - log_s * tt::kLn2);
  }
  return tt::row_sum<G>(s, part);
}

// What a row leaves behind: its loss, whether it counts, and what the backward pass needs.  A row without a teacher has
// m = -inf there, as one without any possible class: no gradient.
__device__ __forceinline__ void write_row(float* loss, float* counted, float2* stats, size_t row, const Stat& a,
                                          float log_s, const TeacherSum& te, float cross, const Scale& sc) {
  const bool none = te.s == 0.f;
  loss[row] = none ? 0.f : fmaf(te.q_log_q, tt::kLn2, cross) * (sc.temperature * sc.temperature);
  counted[row] = none ? 0.f : 1.f;
  stats[row] = make_float2(none ? -INFINITY : a.m, te.s == te.s ? log_s : te.s);
}

// The gradient at the teacher's entries, over what has been written there without q: of a row's packs [v0, v1).
template <typename T, int G>
__device__ __forceinline__ void fix_entries(const T* x, T* dx, const LogitRow<T>& r, size_t row, int v0, int v1, int K,
                                            int lane, const float* weight, const int* place, float m, float log_s,
                                            float c, float scale) {
  tt::stores_done();
  tt::sync_row<G>();
  for (int k = lane; k < K; k += G) {
    const int j = place[k], pack = (j + r.skip) / Pack<T>::n;
    if (pack < v0 || pack >= v1 || weight[k] == 0.f) continue;
    float q = 0.f;
    for (int i = 0; i < K; ++i) q += place[i] == j ? weight[i] : 0.f;
    const size_t at = row * (size_t)r.V + j;
    dx[at] = (T)(scale * (tt::pow2((tt::widen(x[at]) - m) * c - log_s) - q));
  }
}

template <typename T>
__device__ __forceinline__ typename Pack<T>::type gradient_pack(const typename Pack<T>::type& p, float m, float log_s,
                                                                float c, float scale) {
  typename Pack<T>::type q;
#pragma unroll
  for (int i = 0; i < Pack<T>::n; ++i) q[i] = (T)(scale * tt::pow2((tt::widen(p[i]) - m) * c - log_s));
  return q;
}

// Adds packs j, j + G, ... (N of them, those below v1) to the statistics.
template <typename T, int N>
__device__ __forceinline__ void add_packs(Stat& a, const typename Pack<T>::type (&p)[N], float c) {
  constexpr int n = Pack<T>::n;
  float z[N * n];
#pragma unroll
  for (int i = 0; i < N * n; ++i) z[i] = tt::widen(p[i / n][i % n]);
  tt::add_values<N * n, false>(a, z, c);
}

template <typename T, int G>
__device__ __forceinline__ void scan(Stat& a, const LogitRow<T>& r, int v0, int v1, int lane, float c) {
  typedef typename Pack<T>::type P;
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
    add_packs<T, kUnroll>(a, p, c);
  }
}

// How many rows have a teacher, in parts: one whole number for each block.
__global__ __launch_bounds__(kThreads) void distill_count(Teacher te, int* __restrict__ parts, int R, int V) {
  __shared__ int part[kThreads / kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  int n = 0;
  for (long long row = (long long)blockIdx.x * 4 + wave; row < R; row += (long long)gridDim.x * 4) {
    bool any = false;
    for (int k = lane; k < te.K; k += kWave) {
      int i;
      any |= teacher_entry(te, row * te.K + k, V, &i) != -INFINITY;
    }
    n += __any(any) ? 1 : 0;
  }
  if (lane == 0) part[wave] = n;
  __syncthreads();
  if (threadIdx.x == 0) parts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// Rows of G threads each, kept in registers as far as NV packs to a thread reach: loss, statistics and, with GRAD, the
// gradient for an incoming gradient of one, which then costs one read and one write of the row.  `count_parts`: for
// the mean.
template <typename T, int G, int NV, bool GRAD>
__global__ __launch_bounds__(G < kThreads ? kThreads : G) void distill_rows(const T* __restrict__ x, Teacher te,
                                                                           float* __restrict__ loss,
                                                                           float* __restrict__ counted,
                                                                           float2* __restrict__ stats, T* dx,
                                                                           const int* __restrict__ count_parts,
                                                                           Scale sc, int R, int V) {
  constexpr int kBlock = G < kThreads ? kThreads : G, kRows = kBlock / G;
  typedef typename Pack<T>::type P;
  extern __shared__ float lds[];
  __shared__ float part[kRows][3 * (G / kWave)];
  __shared__ float more[kRows][4 * (G / kWave)];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float* weight = lds + sub * 2 * te.K;
  int* place = (int*)(weight + te.K);
  float scale = sc.temperature;
  if (GRAD && count_parts) {
    int n = 0;
    for (int i = lane; i < kCountBlocks; i += G) n += count_parts[i];
    scale /= (float)tt::row_sum<G>(n, (int*)part[sub]);
    tt::sync_row<G>();
  }
  for (long long row = (long long)blockIdx.x * kRows + sub; row < R; row += (long long)gridDim.x * kRows) {
    const LogitRow<T> r(x, row, V);
    P kept[NV];
    // (a thread's packs beyond the row are -inf, which adds nothing)
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int j = lane + u * G;
      kept[u] = j < r.packs ? r.read(j) : P((T)-INFINITY);
    }
    const TeacherSum ts = read_teacher<G>(te, row, V, sc.c, lane, weight, place, part[sub]);
    Stat a = {-INFINITY, 0.f, 0.f};
    if constexpr (NV % 4 == 0) {
#pragma unroll
      for (int u = 0; u < NV; u += 4) add_packs<T, 4>(a, reinterpret_cast<const P(&)[4]>(kept[u]), sc.c);
    } else {
      add_packs<T, NV>(a, kept, sc.c);
    }
    scan<T, G>(a, r, NV * G, r.packs, lane, sc.c);
    a = tt::row_join<G, false>(a, sc.c, more[sub]);
    const float log_s = tt::log_sum(a);
    const float cross = cross_entropy<T, G>(x, row, V, a, log_s, sc.inverse, te.K, lane, weight, place,
                                            more[sub] + 3 * (G / kWave));
    if (lane == 0) write_row(loss, counted, stats, row, a, log_s, ts, cross, sc);
    if constexpr (GRAD) {
      T* out = tt::packs_of(dx, row, V);
      const bool none = ts.s == 0.f || a.m == -INFINITY;
      const float by = ts.s == ts.s ? scale : ts.s, l = log_s;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int j = lane + u * G;
        if (j < r.packs) tt::write_pack(r, out, j, none ? P((T)0.f) : gradient_pack<T>(kept[u], a.m, l, sc.c, by));
      }
      for (int j = lane + NV * G; j < r.packs; j += G)
        tt::write_pack(r, out, j, none ? P((T)0.f) : gradient_pack<T>(r.read(j), a.m, l, sc.c, by));
      if (!none) fix_entries<T, G>(x, dx, r, row, 0, r.packs, te.K, lane, weight, place, a.m, l, sc.c, by);
    }
    tt::sync_row<G>();
  }
}

// Few long rows: `splits` blocks to a row, each with the sums of its share of the packs; distill_join puts them
// together.
template <typename T>
__global__ __launch_bounds__(kThreads) void distill_split(const T* __restrict__ x, float2* __restrict__ stat_part,
                                                          Scale sc, int splits, int V) {
  __shared__ float part[3 * (kThreads / kWave)];
  const int row = blockIdx.x / splits, split = blockIdx.x % splits;
  const LogitRow<T> r(x, row, V);
  const int per = (r.packs + splits - 1) / splits;
  const int v0 = split * per, v1 = v0 + per < r.packs ? v0 + per : r.packs;
  Stat a = {-INFINITY, 0.f, 0.f};
  scan<T, kThreads>(a, r, v0, v1, threadIdx.x, sc.c);
  a = tt::row_join<kThreads, false>(a, sc.c, part);
  if (threadIdx.x == 0) stat_part[blockIdx.x] = make_float2(a.m, a.s);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_join(const T* __restrict__ x, Teacher te,
                                                         const float2* __restrict__ stat_part,
                                                         float* __restrict__ loss, float* __restrict__ counted,
                                                         float2* __restrict__ stats, Scale sc, int splits, int V) {
  constexpr int G = kThreads;
  extern __shared__ float lds[];
  __shared__ float part[3 * (G / kWave)];
  __shared__ float more[4 * (G / kWave)];
  const size_t row = blockIdx.x;
  float* weight = lds;
  int* place = (int*)(lds + te.K);
  Stat a = {-INFINITY, 0.f, 0.f};
  if (threadIdx.x < splits) {
    const float2 v = stat_part[row * splits + threadIdx.x];
    a.m = v.x;
    a.s = v.y;
  }
  const TeacherSum ts = read_teacher<G>(te, row, V, sc.c, threadIdx.x, weight, place, part);
  a = tt::row_join<G, false>(a, sc.c, more);
  const float log_s = tt::log_sum(a);
  const float cross = cross_entropy<T, G>(x, row, V, a, log_s, sc.inverse, te.K, threadIdx.x, weight, place,
                                          more + 3 * (G / kWave));
  if (threadIdx.x == 0) write_row(loss, counted, stats, row, a, log_s, ts, cross, sc);
}

// out[0] = sum of the rows' losses, over count[0], the number of rows with a teacher, if `mean`.  One block.
__global__ __launch_bounds__(1024) void distill_total(const float* __restrict__ loss, const float* __restrict__ counted,
                                                      float* __restrict__ out, float* __restrict__ count, int R,
                                                      int mean) {
  __shared__ double part[2][16];
  double s = 0.0, n = 0.0;
  for (int r = threadIdx.x; r < R; r += 1024) {
    s += (double)loss[r];
    n += (double)counted[r];
  }
  s = tt::row_sum<1024>(s, part[0]);
  n = tt::row_sum<1024>(n, part[1]);
  if (threadIdx.x == 0) {
    if (out) out[0] = (float)(mean ? s / n : s);
    count[0] = (float)n;
  }
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
  typedef typename Pack<T>::type P;
  if (ahead && g[0] == 1.f) return;
  extern __shared__ float lds[];
  __shared__ float part[kRows][3 * (G / kWave)];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G;
  float* weight = lds + sub * 2 * te.K;
  int* place = (int*)(weight + te.K);
  const long long items = (long long)R * splits;
  for (long long item = (long long)blockIdx.x * kRows + sub; item < items; item += (long long)gridDim.x * kRows) {
    const size_t row = item / splits;
    const int split = (int)(item % splits);
    const LogitRow<T> r(x, row, V);
    T* out = tt::packs_of(dx, row, V);
    const int per = (r.packs + splits - 1) / splits;
    const int v0 = split * per, v1 = v0 + per < r.packs ? v0 + per : r.packs;
    const float2 st = stats[row];
    if (st.x == -INFINITY) {
      for (int j = v0 + lane; j < v1; j += G) tt::write_pack(r, out, j, P((T)0.f));
      continue;
    }
    float scale = sc.temperature * (reduction == 0 ? g[row] : g[0]);
    if (reduction == 2) scale /= count[0];
    for (int j = v0 + lane; j < v1; j += kUnroll * G) {
      P p[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u * G < v1) p[u] = r.read(j + u * G);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u * G < v1) tt::write_pack(r, out, j + u * G, gradient_pack<T>(p[u], st.x, st.y, sc.c, scale));
    }
    read_teacher<G>(te, row, V, sc.c, lane, weight, place, part[sub]);
    fix_entries<T, G>(x, dx, r, row, v0, v1, te.K, lane, weight, place, st.x, st.y, sc.c, scale);
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

unsigned grid_for(long long blocks, long long most) { return (unsigned)(blocks < most ? blocks : most); }

// Rows of up to this many packs go to a wave each, which keeps them in registers.
constexpr int kWavePacks = 8 * kWave;

int packs_for(int V, int dtype) { return dtype == TT_F32 ? (V + 3) / 4 : (V + 7) / 8; }

// How many blocks share a row: as many as fill the device eight times, each with kUnroll packs to a thread at least.
int splits_for(long long R, int packs) {
  long long want = (8LL * tt::compute_units() + R - 1) / R;
  const long long most = (packs + kUnroll * kThreads - 1) / (kUnroll * kThreads);
  if (want > most) want = most;
  if (want > kThreads) want = kThreads;
  return want < 1 ? 1 : (int)want;
}

// A row to a block, or a wave, from this many rows on (two blocks of 1024 threads to a unit); fewer long rows are split.
bool whole_rows(long long R, int packs) { return packs <= kWavePacks || R >= tt::compute_units(); }

// Whether the forward pass writes the gradient too, for an incoming gradient of one: where a row's own block does it
// (the row is then read once for both), and that gradient is the likely one.  A loss for each row is weighted by its
// user, and float16 gradients of a mean have to be scaled to be held at all, so those wait for the backward pass.
bool ahead(int dtype, int reduction, long long R, int V) {
  return whole_rows(R, packs_for(V, dtype)) && (reduction == 1 || (reduction == 2 && dtype == TT_F32));
}

template <typename T, bool GRAD>
int launch_rows(const T* x, const Teacher& te, float* loss, float* counted, float* stats, T* dx, const int* count_parts,
                const Scale& sc, int R, int V, int packs) {
  hipStream_t st = tt::stream();
  float2* s = (float2*)stats;
  const size_t lds = (size_t)te.K * 8;
  const int cus = tt::compute_units();
  if (packs <= kWavePacks)
    distill_rows<T, kWave, 8, GRAD><<<grid_for((R + 3LL) / 4, 16 * cus), kThreads, 4 * lds, st>>>(
        x, te, loss, counted, s, dx, count_parts, sc, R, V);
  else if (packs <= 8 * 256)
    distill_rows<T, 256, 8, GRAD><<<grid_for(R, 16 * cus), 256, lds, st>>>(x, te, loss, counted, s, dx, count_parts, sc,
                                                                          R, V);
  else
    distill_rows<T, 1024, 8, GRAD><<<grid_for(R, 16 * cus), 1024, lds, st>>>(x, te, loss, counted, s, dx, count_parts,
                                                                            sc, R, V);
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
  const int splits = whole_rows(R, packs) ? 1 : splits_for(R, packs);
  void* ws;
  if (tt::workspace(((size_t)R * 2 + kCountBlocks) * sizeof(float) + (size_t)R * splits * sizeof(float2), &ws))
    return -1;
  float2* stat_part = (float2*)ws;
  float* counted = (float*)(stat_part + (size_t)R * splits);
  int* parts = (int*)(counted + R);
  float* rows = reduction == 0 ? loss : (float*)(parts + kCountBlocks);
  if (splits > 1) {
    distill_split<T><<<(unsigned)(R * splits), kThreads, 0, st>>>(x, stat_part, sc, splits, V);
    TT_LAUNCH_CHECK();
    distill_join<T><<<R, kThreads, (size_t)te.K * 8, st>>>(x, te, stat_part, rows, counted, (float2*)stats, sc, splits,
                                                           V);
    TT_LAUNCH_CHECK();
  } else if (dx) {
    if (reduction == 2) {
      distill_count<<<kCountBlocks, kThreads, 0, st>>>(te, parts, R, V);
      TT_LAUNCH_CHECK();
    }
    if (launch_rows<T, true>(x, te, rows, counted, stats, dx, reduction == 2 ? parts : nullptr, sc, R, V, packs))
      return -1;
  } else {
    if (launch_rows<T, false>(x, te, rows, counted, stats, dx, nullptr, sc, R, V, packs)) return -1;
  }
  distill_total<<<1, 1024, 0, st>>>(rows, counted, reduction == 0 ? nullptr : loss, count, R, reduction == 2);
  TT_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int backward(const T* x, const Teacher& te, const float* stats, const float* count, const float* g, T* dx,
             double temperature, int reduction, int is_ahead, int R, int V) {
  hipStream_t st = tt::stream();
  const Scale sc = scale_for(temperature);
  const int packs = (V + Pack<T>::n - 1) / Pack<T>::n;
  const size_t lds = (size_t)te.K * 8;
  if (packs <= kWavePacks) {
    distill_bwd<T, kWave><<<grid_for((R + 3LL) / 4, 16 * tt::compute_units()), kThreads, 4 * lds, st>>>(
        x, te, (const float2*)stats, count, g, dx, sc, reduction, is_ahead, 1, R, V);
  } else {
    const int splits = splits_for(R, packs);
    distill_bwd<T, kThreads><<<grid_for((long long)R * splits, 16 * tt::compute_units()), kThreads, lds, st>>>(
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
  return backward((const _Float16*)x, te, stats, count, g, (_Float16*)dx, temperature, reduction, is_ahead, (int)R, V);
}

}  // extern "C"
