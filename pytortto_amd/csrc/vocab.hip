// Rows of logits over a vocabulary: log probabilities of given tokens with the entropy and the best alternatives, and
// distillation from a teacher's top logits, forward and backward.  Logits and their gradients are float32 or float16,
// everything else float32.
//
// With m = max z and S = sum_j 2^((z_j - m) c), c = log2(e) / temperature:
//   log p_j = (z_j - m) / temperature - ln S (in bits z_j may overflow where a mask is the type's lowest value)
//           H = (log2 S - sum_j 2^(d_j) d_j / S) ln 2,  d_j = (z_j - m) c
// The pair (m, log2 S) is kept for the backward pass.  The two are not added up: of a row that a mask has left with
// nothing but the type's lowest value, log2 S would be lost beside m.
#include "rows.h"

#include <math.h>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / tt::kWave;
constexpr int kMostTop = 64;
constexpr int kMostTeacher = 1024;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr double kLog2e = 1.44269504088896340736;

// Running maximum and sums of a softmax: s = sum 2^d, t = sum 2^d d with d = (z - m) c.  No value yet: m = -inf.
struct Stat {
  float m, s, t;
};

// Of a row of -inf alone m stays -inf; differences are then taken from zero and every 2^d is zero.
__device__ __forceinline__ float anchor(float m) { return m == -INFINITY ? 0.f : m; }
// 2^d d where d may be -inf; the clamp changes no product, for 2^-200 is zero.
__device__ __forceinline__ float floor_at(float d) { return fmaxf(d, -200.f); }

__device__ __forceinline__ void add_value(Stat& a, float z, float c) {
  if (z > a.m) {
    const float d = (a.m - z) * c, f = exp2f(d);
    a.t = f * fmaf(a.s, floor_at(d), a.t);
    a.s *= f;
    a.m = z;
  }
  const float d = (z - anchor(a.m)) * c, e = exp2f(d);
  a.s += e;
  a.t = fmaf(e, floor_at(d), a.t);
}

__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = (a.m - anchor(m)) * c, db = (b.m - anchor(m)) * c, fa = exp2f(da), fb = exp2f(db);
  Stat r;
  r.m = m;
  r.s = fmaf(a.s, fa, b.s * fb);
  r.t = fmaf(fa, fmaf(a.s, floor_at(da), a.t), fb * fmaf(b.s, floor_at(db), b.t));
  return r;
}

__device__ __forceinline__ Stat block_join(Stat a, float c, Stat* part) {
#pragma unroll
  for (int off = tt::kWave / 2; off > 0; off >>= 1) {
    Stat b;
    b.m = __shfl_xor(a.m, off, tt::kWave);
    b.s = __shfl_xor(a.s, off, tt::kWave);
    b.t = __shfl_xor(a.t, off, tt::kWave);
    a = join(a, b, c);
  }
  if ((threadIdx.x & (tt::kWave - 1)) == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  a = part[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) a = join(a, part[i], c);
  __syncthreads();
  return a;
}

// A value and its place as one number that orders by value, then by the lower place.  -0 counts as 0.
__device__ __forceinline__ unsigned long long make_key(float z, int j) {
  const unsigned b = __float_as_uint(z + 0.f);
  const unsigned order = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)order << 32) | (0xffffffffu - (unsigned)j);
}
__device__ __forceinline__ int key_place(unsigned long long k) { return (int)(0xffffffffu - (unsigned)k); }
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned order = (unsigned)(k >> 32);
  return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, unsigned long long* part) {
#pragma unroll
  for (int off = tt::kWave / 2; off > 0; off >>= 1) {
    const unsigned long long o = __shfl_xor(v, off, tt::kWave);
    v = o > v ? o : v;
  }
  if ((threadIdx.x & (tt::kWave - 1)) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) v = part[i] > v ? part[i] : v;
  __syncthreads();
  return v;
}

// A token as given, counted from the end where it is negative; -1 where it is no token.
__device__ __forceinline__ long long token_place(long long t, int V) {
  if (t < 0) t += V;
  return t >= 0 && t < V ? t : -1;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logp_fwd(const T* __restrict__ x, const void* __restrict__ tokens,
                                                     int wide, float* __restrict__ logp, float* __restrict__ entropy,
                                                     float* __restrict__ top_logp, long long* __restrict__ top_index,
                                                     float2* __restrict__ stats, long long ignored, int R, int V,
                                                     int K) {
  __shared__ Stat part[kWaves];
  __shared__ unsigned long long best[kWaves];
  const float c = (float)kLog2e;
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const long long t0 = tt::read_index(tokens, row, wide);
    const size_t out = (size_t)row * K;
    if (t0 == ignored) {
      if (threadIdx.x == 0) {
        logp[row] = 0.f;
        entropy[row] = 0.f;
        if (stats) stats[row] = make_float2(0.f, 0.f);
      }
      for (int k = threadIdx.x; k < K; k += kThreads) {
        top_logp[out + k] = 0.f;
        top_index[out + k] = -1;
      }
      continue;
    }
    const T* __restrict__ p = x + (size_t)row * V;
    Stat a = {-INFINITY, 0.f, 0.f};
    for (int j = threadIdx.x; j < V; j += kThreads) add_value(a, tt::widen(p[j]), c);
    a = block_join(a, c, part);
    const float log_s = a.s > 0.f ? log2f(a.s) : a.s;     // (an empty row: 0; NaN stays)
    if (threadIdx.x == 0) {
      const long long t = token_place(t0, V);
      logp[row] = t < 0 ? NAN : (tt::widen(p[t]) - anchor(a.m)) - log_s * kLn2;
      entropy[row] = a.s == 0.f ? 0.f : (log_s - a.t / a.s) * kLn2;
      if (stats) stats[row] = make_float2(a.m, log_s);
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < K; ++k) {
      unsigned long long v = 0;
      for (int j = threadIdx.x; j < V; j += kThreads) {
        const unsigned long long key = make_key(tt::widen(p[j]), j);
        if (key < last && key > v) v = key;
      }
      last = block_max(v, best);
      if (threadIdx.x == 0) {
        const bool fine = a.s == a.s;
        top_logp[out + k] = fine ? (key_value(last) - anchor(a.m)) - log_s * kLn2 : NAN;
        top_index[out + k] = fine ? key_place(last) : -1;
      }
    }
  }
}

// dz_j = -p_j (a + sum_k c_k + h (log p_j + H)) + a [j = t] + sum_k c_k [j = i_k]
template <typename T>
__global__ __launch_bounds__(kThreads) void logp_bwd(const T* __restrict__ x, const void* __restrict__ tokens,
                                                     int wide, const float2* __restrict__ stats,
                                                     const float* __restrict__ entropy,
                                                     const long long* __restrict__ top_index,
                                                     const float* __restrict__ g_logp,
                                                     const float* __restrict__ g_entropy,
                                                     const float* __restrict__ g_top, T* __restrict__ dx,
                                                     long long ignored, int R, int V, int K) {
  const float c = (float)kLog2e;
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const size_t base = (size_t)row * V, out = (size_t)row * K;
    const long long t0 = tt::read_index(tokens, row, wide), t = token_place(t0, V);
    const float2 st = stats[row];
    if (t0 == ignored || st.x == -INFINITY) {
      for (int j = threadIdx.x; j < V; j += kThreads) dx[base + j] = (T)0.f;
      continue;
    }
    const float a = g_logp ? g_logp[row] : 0.f, h = g_entropy ? g_entropy[row] : 0.f, H = entropy[row];
    float total = g_logp && t < 0 ? NAN : a;
    if (g_top)
      for (int k = 0; k < K; ++k) total += g_top[out + k];
    for (int j = threadIdx.x; j < V; j += kThreads) {
      const float d = (tt::widen(x[base + j]) - st.x) * c - st.y, p = exp2f(d);
      float given = j == t ? a : 0.f;     // summed first: what cancels here leaves no rounding behind
      if (g_top)
        for (int k = 0; k < K; ++k)
          if (top_index[out + k] == j) given += g_top[out + k];
      dx[base + j] = (T)fmaf(-p, fmaf(h, fmaf(floor_at(d), kLn2, H), total), given);
    }
  }
}

// The teacher's distribution over its entries, in LDS: weight[k] = q_k; returns {sum of 2^d, any entry} and the sum
// over k of q_k log2 q_k.  An index from V on leaves NaN.
struct Teacher {
  float s;            // > 0: the row has a teacher; 0: it has none; NaN: it cannot be computed
  float q_log_q;      // in bits
};

template <typename T>
__device__ __forceinline__ Teacher read_teacher(const T* __restrict__ teacher, const void* __restrict__ index, int wide,
                                                size_t at, int K, int V, float c, float* weight, int* place,
                                                Stat* part) {
  Stat a = {-INFINITY, 0.f, 0.f};
  for (int k = threadIdx.x; k < K; k += kThreads) {
    const long long i = tt::read_index(index, at + k, wide);
    const float z = i < 0 ? -INFINITY : i >= V ? NAN : tt::widen(teacher[at + k]);
    weight[k] = z;
    place[k] = i < 0 || i >= V ? 0 : (int)i;
    add_value(a, z, c);
  }
  a = block_join(a, c, part);
  const float log_s = log2f(a.s);
  Teacher r = {a.s, a.s > 0.f ? a.t / a.s - log_s : 0.f};
  for (int k = threadIdx.x; k < K; k += kThreads)
    weight[k] = a.s == 0.f ? 0.f : exp2f((weight[k] - anchor(a.m)) * c - log_s);
  __syncthreads();
  return r;
}

// The loss of each row, and (m, log2 S) of each row for the backward pass.
template <typename T, typename U>
__global__ __launch_bounds__(kThreads) void distill_rows(const T* __restrict__ x, const U* __restrict__ teacher,
                                                         const void* __restrict__ index, int wide,
                                                         float* __restrict__ loss, float* __restrict__ counted,
                                                         float2* __restrict__ stats, float c, float inverse,
                                                         float factor, int R, int V, int K) {
  __shared__ Stat part[kWaves];
  __shared__ float sums[kWaves];
  __shared__ float weight[kMostTeacher];
  __shared__ int place[kMostTeacher];
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const T* __restrict__ p = x + (size_t)row * V;
    const Teacher te = read_teacher(teacher, index, wide, (size_t)row * K, K, V, c, weight, place, part);
    Stat a = {-INFINITY, 0.f, 0.f};
    for (int j = threadIdx.x; j < V; j += kThreads) add_value(a, tt::widen(p[j]), c);
    a = block_join(a, c, part);
    const float log_s = a.s > 0.f ? log2f(a.s) : a.s;
    float cross = 0.f;
    for (int k = threadIdx.x; k < K; k += kThreads)
      if (weight[k] != 0.f) cross -= weight[k] * ((tt::widen(p[place[k]]) - anchor(a.m)) * inverse - log_s * kLn2);
    cross = tt::block_sum<kWaves>(cross, sums);
    if (threadIdx.x == 0) {
      loss[row] = te.s == 0.f ? 0.f : fmaf(te.q_log_q, kLn2, cross) * factor;
      counted[row] = te.s == 0.f ? 0.f : 1.f;
      stats[row] = make_float2(a.m, log_s);
    }
  }
}

// out[0] = sum of the rows' losses, over count[0], the number of rows with a teacher, if `mean`.  One block.
__global__ __launch_bounds__(kThreads) void distill_total(const float* __restrict__ loss,
                                                          const float* __restrict__ counted, float* __restrict__ out,
                                                          float* __restrict__ count, int R, int mean) {
  __shared__ double part[kWaves];
  double s = 0.0, n = 0.0;
  for (int r = threadIdx.x; r < R; r += kThreads) {
    s += (double)loss[r];
    n += (double)counted[r];
  }
  s = tt::block_sum<kWaves>(s, part);
  n = tt::block_sum<kWaves>(n, part);
  if (threadIdx.x == 0) {
    if (out) out[0] = (float)(mean ? s / n : s);
    count[0] = (float)n;
  }
}

// dz_j = g T (p_j - q_j), with g over the count if `mean`; zero in a row without a teacher.
template <typename T, typename U>
__global__ __launch_bounds__(kThreads) void distill_bwd(const T* __restrict__ x, const U* __restrict__ teacher,
                                                        const void* __restrict__ index, int wide,
                                                        const float2* __restrict__ stats,
                                                        const float* __restrict__ count, const float* __restrict__ g,
                                                        T* __restrict__ dx, float c, float temperature, int reduction,
                                                        int R, int V, int K) {
  __shared__ Stat part[kWaves];
  __shared__ float weight[kMostTeacher];
  __shared__ int place[kMostTeacher];
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const size_t base = (size_t)row * V;
    const Teacher te = read_teacher(teacher, index, wide, (size_t)row * K, K, V, c, weight, place, part);
    const float2 st = stats[row];
    float scale = temperature * (reduction == 0 ? g[row] : g[0]);
    if (reduction == 2) scale /= count[0];
    const bool none = te.s == 0.f || st.x == -INFINITY;
    for (int j = threadIdx.x; j < V; j += kThreads) {
      float v = 0.f;
      if (!none) {
        v = exp2f((tt::widen(x[base + j]) - st.x) * c - st.y);
        for (int k = 0; k < K; ++k)
          if (place[k] == j) v -= weight[k];
        v = te.s != te.s ? NAN : scale * v;
      }
      dx[base + j] = (T)v;
    }
    __syncthreads();
  }
}

unsigned blocks_for(long long rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

int check(const char* fn, int dtype, int index_bits, long long R, int V) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_F16, "%s: unknown type %d", fn, dtype);
  TT_REQUIRE(index_bits == 32 || index_bits == 64, "%s: indexes have 32 or 64 bits (got %d)", fn, index_bits);
  TT_REQUIRE(R > 0 && R <= (1 << 30), "%s: rows must be in 1..2^30 (got %lld)", fn, R);
  TT_REQUIRE(V > 0 && V <= (1 << 30), "%s: the vocabulary must have 1..2^30 entries (got %d)", fn, V);
  return 0;
}

int check_top(const char* fn, int K, int V) {
  TT_REQUIRE(K >= 0 && K <= kMostTop && K <= V, "%s: alternatives must be in 0..min(%d, %d) (got %d)", fn, kMostTop, V,
             K);
  return 0;
}

int check_distill(const char* fn, int teacher_dtype, double temperature, int reduction, int K) {
  TT_REQUIRE(teacher_dtype == TT_F32 || teacher_dtype == TT_F16, "%s: unknown type %d", fn, teacher_dtype);
  TT_REQUIRE(temperature >= 1e-6 && temperature <= 1e6, "%s: temperature must be in 1e-6..1e6 (got %g)", fn,
             temperature);
  TT_REQUIRE(reduction >= 0 && reduction <= 2, "%s: reduction must be 0 (none), 1 (sum) or 2 (mean)", fn);
  TT_REQUIRE(K >= 1 && K <= kMostTeacher, "%s: teacher entries must be in 1..%d (got %d)", fn, kMostTeacher, K);
  return 0;
}

template <typename T, typename U>
int distill_forward(const T* x, const U* teacher, const void* index, int wide, float* loss, float* stats, float* count,
                    double temperature, int reduction, int R, int V, int K) {
  hipStream_t st = tt::stream();
  void* ws;
  if (tt::workspace((size_t)R * 2 * sizeof(float), &ws)) return -1;
  float* rows = reduction == 0 ? loss : (float*)ws;
  float* counted = (float*)ws + R;
  distill_rows<T, U><<<blocks_for(R), kThreads, 0, st>>>(x, teacher, index, wide, rows, counted, (float2*)stats,
                                                         (float)(kLog2e / temperature), (float)(1.0 / temperature),
                                                         (float)(temperature * temperature), R, V, K);
  TT_LAUNCH_CHECK();
  distill_total<<<1, kThreads, 0, st>>>(rows, counted, reduction == 0 ? nullptr : loss, count, R, reduction == 2);
  TT_LAUNCH_CHECK();
  return 0;
}

template <typename T, typename U>
int distill_backward(const T* x, const U* teacher, const void* index, int wide, const float* stats, const float* count,
                     const float* g, T* dx, double temperature, int reduction, int R, int V, int K) {
  distill_bwd<T, U><<<blocks_for(R), kThreads, 0, tt::stream()>>>(x, teacher, index, wide, (const float2*)stats, count,
                                                                  g, dx, (float)(kLog2e / temperature),
                                                                  (float)temperature, reduction, R, V, K);
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
  if (int rc = check(fn, dtype, token_bits, R, V)) return rc;
  if (int rc = check_top(fn, K, V)) return rc;
  TT_REQUIRE(K == 0 || (top_logp && top_index), "%s: null pointer for the alternatives", fn);
  TT_REQUIRE_ALIGNED(fn, x, stats);
  const int wide = token_bits == 64;
  if (dtype == TT_F32)
    logp_fwd<float><<<blocks_for(R), kThreads, 0, tt::stream()>>>((const float*)x, tokens, wide, logp, entropy,
                                                                  top_logp, top_index, (float2*)stats, ignore_index,
                                                                  (int)R, V, K);
  else
    logp_fwd<_Float16><<<blocks_for(R), kThreads, 0, tt::stream()>>>((const _Float16*)x, tokens, wide, logp, entropy,
                                                                     top_logp, top_index, (float2*)stats, ignore_index,
                                                                     (int)R, V, K);
  TT_LAUNCH_CHECK();
  return 0;
}

int tt_token_log_prob_bwd(const void* x, const void* tokens, const float* stats, const float* entropy,
                          const long long* top_index, const float* g_logp, const float* g_entropy, const float* g_top,
                          void* dx, int dtype, int token_bits, long long ignore_index, long long R, int V, int K) {
  TT_REQUIRE_INIT();
  const char* fn = "tt_token_log_prob_bwd";
  TT_REQUIRE(x && tokens && stats && entropy && dx, "%s: null pointer", fn);
  if (int rc = check(fn, dtype, token_bits, R, V)) return rc;
  if (int rc = check_top(fn, K, V)) return rc;
  TT_REQUIRE(g_top == nullptr || (K > 0 && top_index), "%s: a gradient of the alternatives needs their indexes", fn);
  TT_REQUIRE_ALIGNED(fn, x, dx, stats);
  const int wide = token_bits == 64;
  if (dtype == TT_F32)
    logp_bwd<float><<<blocks_for(R), kThreads, 0, tt::stream()>>>((const float*)x, tokens, wide, (const float2*)stats,
                                                                  entropy, top_index, g_logp, g_entropy, g_top,
                                                                  (float*)dx, ignore_index, (int)R, V, K);
  else
    logp_bwd<_Float16><<<blocks_for(R), kThreads, 0, tt::stream()>>>((const _Float16*)x, tokens, wide,
                                                                     (const float2*)stats, entropy, top_index, g_logp,
                                                                     g_entropy, g_top, (_Float16*)dx, ignore_index,
                                                                     (int)R, V, K);
  TT_LAUNCH_CHECK();
  return 0;
}

int tt_distill_fwd(const void* x, const void* teacher, const void* index, float* loss, float* stats, float* count,
                   double temperature, int reduction, int dtype, int teacher_dtype, int index_bits, long long R, int V,
                   int K) {
  TT_REQUIRE_INIT();
  const char* fn = "tt_distill_fwd";
  TT_REQUIRE(x && teacher && index && loss && stats && count, "%s: null pointer", fn);
  if (int rc = check(fn, dtype, index_bits, R, V)) return rc;
  if (int rc = check_distill(fn, teacher_dtype, temperature, reduction, K)) return rc;
  TT_REQUIRE_ALIGNED(fn, x, stats);
  const int wide = index_bits == 64, r = (int)R;
  typedef _Float16 h;
  if (dtype == TT_F32 && teacher_dtype == TT_F32)
    return distill_forward((const float*)x, (const float*)teacher, index, wide, loss, stats, count, temperature,
                           reduction, r, V, K);
  if (dtype == TT_F32)
    return distill_forward((const float*)x, (const h*)teacher, index, wide, loss, stats, count, temperature, reduction,
                           r, V, K);
  if (teacher_dtype == TT_F32)
    return distill_forward((const h*)x, (const float*)teacher, index, wide, loss, stats, count, temperature, reduction,
                           r, V, K);
  return distill_forward((const h*)x, (const h*)teacher, index, wide, loss, stats, count, temperature, reduction, r, V,
                         K);
}

int tt_distill_bwd(const void* x, const void* teacher, const void* index, const float* stats, const float* count,
                   const float* g, void* dx, double temperature, int reduction, int dtype, int teacher_dtype,
                   int index_bits, long long R, int V, int K) {
  TT_REQUIRE_INIT();
  const char* fn = "tt_distill_bwd";
  TT_REQUIRE(x && teacher && index && stats && count && g && dx, "%s: null pointer", fn);
  if (int rc = check(fn, dtype, index_bits, R, V)) return rc;
  if (int rc = check_distill(fn, teacher_dtype, temperature, reduction, K)) return rc;
  TT_REQUIRE_ALIGNED(fn, x, dx, stats);
  const int wide = index_bits == 64, r = (int)R;
  typedef _Float16 h;
  if (dtype == TT_F32 && teacher_dtype == TT_F32)
    return distill_backward((const float*)x, (const float*)teacher, index, wide, stats, count, g, (float*)dx,
                            temperature, reduction, r, V, K);
  if (dtype == TT_F32)
    return distill_backward((const float*)x, (const h*)teacher, index, wide, stats, count, g, (float*)dx, temperature,
                            reduction, r, V, K);
  if (teacher_dtype == TT_F32)
    return distill_backward((const h*)x, (const float*)teacher, index, wide, stats, count, g, (h*)dx, temperature,
                            reduction, r, V, K);
  return distill_backward((const h*)x, (const h*)teacher, index, wide, stats, count, g, (h*)dx, temperature, reduction,
                          r, V, K);
}

}  // extern "C"
