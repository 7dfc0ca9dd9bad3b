// Device code shared by the operators over a vocabulary (vocab_logp.hip, vocab_distill.hip): a row of logits as
// aligned sixteen-byte packs, and the running statistics of its softmax.
//
// With m = max z and S = sum_j 2^(d_j), d_j = (z_j - m) c, c = log2(e) / temperature:
//   log p_j = (z_j - m) / temperature - ln S          H = (log2 S - sum_j 2^(d_j) d_j / S) ln 2
// The pair (m, log2 S) is kept for the backward pass.  The two are not added up: of a row that a mask has left with
// nothing but the type's lowest value, log2 S would be lost beside m.
#pragma once
#include "rows.h"

namespace tt {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr double kLog2e = 1.44269504088896340736;

// Rows begin at any multiple of the type: a row is read as the aligned packs that cover it.  Element i of pack j is
// column j * n + i - skip; the first and the last pack may hold columns of the neighbours, and those two are then read
// value by value, so that nothing outside the row is touched.
template <typename T>
struct LogitRow {
  typedef typename Pack<T>::type P;
  static constexpr int n = Pack<T>::n;
  const P* at;        // the pack that holds column 0
  int skip, V;
  int packs;          // that cover the row
  int whole0, whole1; // [whole0, whole1): the packs that lie in the row altogether

  __device__ __forceinline__ LogitRow(const T* x, size_t row, int V_) : V(V_) {
    const size_t first = row * (size_t)V;       // (x itself is 16-byte aligned)
    skip = (int)(first % n);
    at = reinterpret_cast<const P*>(x) + first / n;
    packs = (V + skip + n - 1) / n;
    whole0 = skip ? 1 : 0;
    whole1 = (V + skip) / n;
  }
  __device__ __forceinline__ int column(int j) const { return j * n - skip; }
  __device__ __forceinline__ P read(int j) const {
    if (j >= whole0 && j < whole1) return at[j];
    P p;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int c = column(j) + i;
      p[i] = c >= 0 && c < V ? reinterpret_cast<const T*>(at)[(ptrdiff_t)c + skip] : (T)-INFINITY;
    }
    return p;
  }
};

template <typename T>
__device__ __forceinline__ void write_pack(const LogitRow<T>& r, T* dx_at, int j, const typename Pack<T>::type& p) {
  if (j >= r.whole0 && j < r.whole1) {
    __builtin_nontemporal_store(p, reinterpret_cast<typename Pack<T>::type*>(dx_at) + j);
    return;
  }
#pragma unroll
  for (int i = 0; i < Pack<T>::n; ++i) {
    const int c = r.column(j) + i;
    if (c >= 0 && c < r.V) dx_at[(ptrdiff_t)c + r.skip] = p[i];
  }
}

// Where the aligned packs of a row begin in an array laid out like the logits.
template <typename T>
__device__ __forceinline__ T* packs_of(T* dx, size_t row, int V) {
  return dx + (row * (size_t)V) / Pack<T>::n * Pack<T>::n;
}

// Running maximum and sums of a softmax: s = sum 2^d, t = sum 2^d d with d = (z - m) c.  No value yet: m = -inf.
struct Stat {
  float m, s, t;
};

// v_exp_f32: results below 2^-126 are zero, which no sum or gradient of float32 here can tell
__device__ __forceinline__ float pow2(float d) { return __builtin_amdgcn_exp2f(d); }
// Of a row of -inf alone m stays -inf; differences are then taken from zero and every 2^d is zero.
__device__ __forceinline__ float anchor(float m) { return m == -INFINITY ? 0.f : m; }
// 2^d d where d may be -inf; the clamp changes no product, for 2^-200 is zero.
__device__ __forceinline__ float floor_at(float d) { return fmaxf(d, -200.f); }

// Moves the sums of `a` to another, larger maximum.
template <bool ENTROPY>
__device__ __forceinline__ void rescale(Stat& a, float m, float c) {
  const float d = (a.m - anchor(m)) * c, f = pow2(d);
  if (ENTROPY) a.t = f * fmaf(a.s, floor_at(d), a.t);
  a.s *= f;
  a.m = m;
}

// N values at once: one comparison of maxima and at most one rescaling for all of them.  A NaN, or an infinity, which
// is taken from itself, ends up in s.
template <int N, bool ENTROPY>
__device__ __forceinline__ bool add_values(Stat& a, const float (&z)[N], float c) {
  float most = z[0];
#pragma unroll
  for (int i = 1; i < N; ++i) most = fmaxf(most, z[i]);
  const bool rises = most > a.m;
  if (rises) rescale<ENTROPY>(a, most, c);
  const float m = anchor(a.m);
  float s0 = 0.f, s1 = 0.f, t0 = 0.f, t1 = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float d0 = (z[i] - m) * c, e0 = pow2(d0);
    s0 += e0;
    if (ENTROPY) t0 = fmaf(e0, floor_at(d0), t0);
    if (i + 1 < N) {
      const float d1 = (z[i + 1] - m) * c, e1 = pow2(d1);
      s1 += e1;
      if (ENTROPY) t1 = fmaf(e1, floor_at(d1), t1);
    }
  }
  a.s += s0 + s1;
  if (ENTROPY) a.t += t0 + t1;
  return rises;
}

// The statistics of all G threads of a row: first the maximum, then each thread's sums moved to it and added up.
// part: LDS of 3 * G / 64 floats.
template <int G, bool ENTROPY>
__device__ __forceinline__ Stat row_join(Stat a, float c, float* part) {
  const float m = row_max<G>(a.m, part);
  rescale<ENTROPY>(a, m, c);
  a.s = row_sum<G>(a.s, part + G / kWave);
  if (ENTROPY) a.t = row_sum<G>(a.t, part + 2 * (G / kWave));
  return a;
}

// log2 of the sum, 0 for an empty row; a NaN stays.
__device__ __forceinline__ float log_sum(const Stat& a) { return a.s > 0.f ? log2f(a.s) : a.s; }

}  // namespace tt
