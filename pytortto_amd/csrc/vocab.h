// Device code shared by the operators over a vocabulary (vocab_logp.hip, vocab_distill.hip): a row of logits as
// aligned sixteen-byte packs, and the running statistics of its softmax.
//
// With m = max z and S = sum_j 2^(d_j), d_j = (z_j - m) c, c = log2(e) / temperature:
//   log p_j = (z_j - m) / temperature - ln S          H = (log2 S - sum_j 2^(d_j) d_j / S) ln 2
// The pair (m, log2 S) is kept for the backward pass.  The two are not added up: of a row that a mask has left with
// nothing but the type's lowest value, log2 S would be lost beside m.
// One pass keeps a thread's maximum and its sums to that maximum.  A thread takes kUnroll packs at a time, so a
// rescaling costs one exponential for 16 or 32 values, and the sums of G threads move to the row's maximum at the end.
#pragma once
#include "rows.h"

namespace tt {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr double kLog2e = 1.44269504088896340736;

// Rows begin at any multiple of the type.  The aligned packs that lie in a row altogether, [first, end), are read and
// written whole; element i of pack j is column j n + i - skip.  The columns in front of them (`head`, n - 1 at most)
// and behind them (`tail`, from tail_at on) go one by one, so nothing outside the row is touched.
template <typename T>
struct LogitRow {
  static constexpr int n = Pack<T>::n;
  const char* at;     // where pack 0, which holds column 0, begins
  size_t start;       // element offset of column 0
  int skip, V;
  int first, end;
  int head, tail, tail_at;

  __device__ __forceinline__ LogitRow(const T* x, size_t row, int V_) : start(row * (size_t)V_), V(V_) {
    skip = (int)(start % n);                    // (x itself is 16-byte aligned)
    at = reinterpret_cast<const char*>(x + (start - skip));
    first = skip ? 1 : 0;
    end = (V + skip) / n;
    head = skip ? n - skip : 0;
    head = head < V ? head : V;
    tail_at = end * n - skip;
    tail_at = tail_at > head ? tail_at : head;
    tail = V - tail_at;
  }
  __device__ __forceinline__ Words pack(int j) const {
    return *reinterpret_cast<const Words*>(at + (unsigned)j * 16u);
  }
  __device__ __forceinline__ int column(int j) const { return j * n - skip; }
};

template <typename T>
__device__ __forceinline__ void write_pack(const LogitRow<T>& r, T* dx, int j, const Words& p) {
  char* at = reinterpret_cast<char*>(dx + (r.start - r.skip));
  __builtin_nontemporal_store(p, reinterpret_cast<Words*>(at + (unsigned)j * 16u));
}

// The part of a row that split `split` of `splits` works on: whole packs [p0, p1), the head with the first split, the
// tail with the last.
struct Share {
  int p0, p1;
  int head, tail;
  template <typename T>
  __device__ __forceinline__ Share(const LogitRow<T>& r, int split, int splits) {
    const int packs = r.end > r.first ? r.end - r.first : 0, per = (packs + splits - 1) / splits;
    p0 = r.first + (split * per < packs ? split * per : packs);
    p1 = r.first + ((split + 1) * per < packs ? (split + 1) * per : packs);
    head = split == 0 ? r.head : 0;
    tail = split == splits - 1 ? r.tail : 0;
  }
};

// Running maximum and sums of a softmax: s = sum 2^d, t = sum 2^d d with d = (z - m) c.  No value yet: m = -inf.
struct Stat {
  float m, s, t;
};

// v_exp_f32: results below 2^-126 are zero, which no sum or gradient of float32 here can tell.  Its argument is a rounded
// product, so the result is off by up to |d| 2^-24 of itself, which an exponential of z - m would not be: the price of one
// instruction for it.  It weighs where the result is small: 2e-6 of a probability of 1e-12.
__device__ __forceinline__ float pow2(float d) { return __builtin_amdgcn_exp2f(d); }
// Of a row of -inf alone m stays -inf; differences are then taken from zero and every 2^d is zero.
__device__ __forceinline__ float anchor(float m) { return m == -INFINITY ? 0.f : m; }
// 2^d d where d may be -inf; the clamp changes no product, for 2^-200 is zero.
__device__ __forceinline__ float floor_at(float d) { return fmaxf(d, -200.f); }

// d of a value, (z - m) c.  Halves cannot overflow z c, and take one instruction for their widening, the product and
// the difference; every d of a row has the same rounded m c then, which drops out of all that is made of them.  (Where c
// is below 2^14: m c is below 2^30 then, and what it is rounded by below 2^5, a factor of 2^32 for all sums of the row.)
template <typename T>
constexpr bool by_product = false;
template <>
inline constexpr bool by_product<_Float16> = true;
__device__ __forceinline__ float rounded(float m, float c) {
#pragma clang fp contract(off)
  return m * c;
}
__device__ __forceinline__ float rounded_between(float m, float to, float c) {
#pragma clang fp contract(off)
  return m * c - to * c;        // (fused, equal ones would differ by the rounding)
}
template <typename T>
__device__ __forceinline__ float bits(float z, float m, float c) {
  return by_product<T> ? fmaf(z, c, -rounded(m, c)) : (z - m) * c;
}

// Moves the sums of `a` to another, larger maximum.
template <typename T, bool ENTROPY>
__device__ __forceinline__ void rescale(Stat& a, float m, float c) {
  const float to = anchor(m), d = by_product<T> ? rounded_between(a.m, to, c) : (a.m - to) * c, f = pow2(d);
  if (ENTROPY) a.t = f * fmaf(a.s, floor_at(d), a.t);
  a.s *= f;
  a.m = m;
}

// Adds N values of which `most` is the largest: at most one rescaling for all of them.  A NaN, or an infinity, which is
// taken from itself, ends up in s.  Returns whether the maximum rose.
template <typename T, int N, bool ENTROPY>
__device__ __forceinline__ bool add_values(Stat& a, const float (&z)[N], float most, float c) {
  const bool rises = most > a.m;
  if (rises) rescale<T, ENTROPY>(a, most, c);
  const float m = anchor(a.m);
  float s[2] = {}, t[2] = {};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = bits<T>(z[i], m, c), e = pow2(d);
    s[i % 2] += e;
    if (ENTROPY) t[i % 2] = fmaf(e, floor_at(d), t[i % 2]);
  }
  a.s += s[0] + s[1];
  if (ENTROPY) a.t += t[0] + t[1];
  return rises;
}

template <typename T, int N, bool ENTROPY>
__device__ __forceinline__ bool add_packs(Stat& a, const Words* p, float c) {
  constexpr int n = Pack<T>::n;
  float z[N * n];
#pragma unroll
  for (int i = 0; i < N; ++i) unpack<T>(z + i * n, p[i]);
  return add_values<T, N * n, ENTROPY>(a, z, pack_max<T, N>(p), c);
}
template <typename T, bool ENTROPY>
__device__ __forceinline__ bool add_value(Stat& a, float value, float c) {
  const float z[1] = {value};
  return add_values<T, 1, ENTROPY>(a, z, value, c);
}

constexpr int kUnroll = 4;      // packs that a thread has on their way at once in the streaming loops

// How many blocks of `threads` share a row: as many as come to `fill` for each compute unit, each with `least` packs.
inline int splits_for(long long R, int packs, int threads, int fill, int least) {
  long long want = ((long long)fill * compute_units() + R - 1) / R;
  const long long most = (packs + least - 1) / least;
  if (want > most) want = most;
  if (want > threads) want = threads;
  return want < 1 ? 1 : (int)want;
}

// The columns outside the whole packs, of which thread `lane` of G takes lane, lane + G, ...
template <typename T>
__device__ __forceinline__ int loose_column(const LogitRow<T>& r, const Share& h, int i) {
  return i < h.head ? i : r.tail_at + i - h.head;
}

// A thread's share of a row: packs p0 + lane + i G in ascending order, then its loose columns (PACKS = false: these
// only).  `best` is told the first pack of those, kUnroll at most and G apart, that hold the first of the packs'
// largest values; kNothing: none is above -inf.
constexpr int kNothing = -1;

template <typename T, int G, bool ENTROPY, bool PACKS = true>
__device__ __forceinline__ void scan(Stat& a, int& best, const T* x, const LogitRow<T>& r, const Share& h, int lane,
                                     float c) {
  for (int j0 = h.p0; PACKS && j0 < h.p1; j0 += kUnroll * G) {
    const int j = j0 + lane;
    Words p[kUnroll];
    if (j0 + kUnroll * G <= h.p1) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) p[u] = r.pack(j + u * G);
      if (add_packs<T, kUnroll, ENTROPY>(a, p, c)) best = j;
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        p[u] = Words(Pack<T>::lowest);
        if (j + u * G < h.p1) p[u] = r.pack(j + u * G);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j0 + u * G < h.p1 && add_packs<T, 1, ENTROPY>(a, p + u, c)) best = j + u * G;
    }
  }
  for (int i = lane; i < h.head + h.tail; i += G)
    add_value<T, ENTROPY>(a, widen(x[r.start + loose_column(r, h, i)]), c);
}

// The statistics of all G threads of a row: first the maximum, then each thread's sums moved to it and added up.
// part: LDS of 3 G / 64 floats.
template <typename T, int G, bool ENTROPY>
__device__ __forceinline__ Stat row_join(Stat a, float c, float* part) {
  constexpr int kParts = G > kWave ? G / kWave : 0;
  const float m = row_max<G>(a.m, part);
  rescale<T, ENTROPY>(a, m, c);
  a.s = row_sum<G>(a.s, part + kParts);
  if (ENTROPY) a.t = row_sum<G>(a.t, part + 2 * kParts);
  return a;
}

struct Scale {
  float c;            // log2(e) / temperature
  float inverse;      // 1 / temperature
  float temperature;
};

// log p of a value, in nats.  (In bits a float32 that is its type's lowest would overflow.)
template <typename T>
__device__ __forceinline__ float log_p(float z, float m, float log_s, const Scale& sc) {
  return (by_product<T> ? bits<T>(z, m, sc.c) * kLn2 : (z - m) * sc.inverse) - log_s * kLn2;
}

// LDS floats of `sums` sums over a row.
constexpr int parts_of(int G, int sums) { return G > kWave ? sums * (G / kWave) : 1; }

// log2 of the sum, 0 for an empty row; a NaN stays.
__device__ __forceinline__ float log_sum(const Stat& a) { return a.s > 0.f ? log2f(a.s) : a.s; }
// Whether a row has no value above -inf, by its maximum and its sum or the sum's logarithm.  The maximum passes over
// NaN, so that a row of nothing else has -inf too; its sum is NaN then.
__device__ __forceinline__ bool is_empty(float m, float s) { return m == -INFINITY && s == s; }

}  // namespace tt
