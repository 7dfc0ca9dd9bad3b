// What the kernels over rows of float32 or float16 values share: layer normalisation (layernorm.hip), token log
// probabilities and distillation (vocab_logp.hip, vocab_distill.hip).  Values are widened to float32 as they are read;
// sums and statistics are float32 or wider, and a result is rounded once, to its own type, as it is stored.
#pragma once
#include "tt_common.h"

#include <math.h>

namespace tt {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }

// Sixteen bytes of a row.  They are kept as four words until their values are wanted: as a vector of halves the
// compiler would give every value a register of its own.
typedef unsigned Words __attribute__((ext_vector_type(4)));
template <typename T>
struct Pack;
template <>
struct Pack<float> {
  typedef float value;
  typedef float vector __attribute__((ext_vector_type(4)));
  static constexpr int n = 4;
  static constexpr unsigned lowest = 0xff800000u;      // -inf, as often as a word holds it
};
template <>
struct Pack<_Float16> {
  typedef _Float16 value;
  typedef _Float16 vector __attribute__((ext_vector_type(8)));
  static constexpr int n = 8;
  static constexpr unsigned lowest = 0xfc00fc00u;
};
template <typename T>
__device__ __forceinline__ void unpack(float* z, const Words& p) {
  const typename Pack<T>::vector v = __builtin_bit_cast(typename Pack<T>::vector, p);
#pragma unroll
  for (int i = 0; i < Pack<T>::n; ++i) z[i] = widen(v[i]);
}
// The largest of N packs' values, two halves to an instruction.  (NaN counts for nothing.)
template <typename T, int N>
__device__ __forceinline__ float pack_max(const Words* p) {
  typedef typename Pack<T>::vector V;
  V m = __builtin_bit_cast(V, p[0]);
#pragma unroll
  for (int i = 1; i < N; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(V, p[i]));
  float most = widen(m[0]);
#pragma unroll
  for (int i = 1; i < Pack<T>::n; ++i) most = fmaxf(most, widen(m[i]));
  return most;
}
template <typename T>
__device__ __forceinline__ Words pack(const float* z) {
  typename Pack<T>::vector v;
#pragma unroll
  for (int i = 0; i < Pack<T>::n; ++i) v[i] = (typename Pack<T>::value)z[i];
  return __builtin_bit_cast(Words, v);
}

// G threads work on a row: a part of a wave, a wave, or a block of G threads.
template <int G>
__device__ __forceinline__ void sync_row() {
  if (G <= kWave) {
    // LDS operations of one wave run in order: only the compiler has to keep them so
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// Which row of its block a thread works on; the compiler is told where that is the same for a whole wave.
template <int G>
__device__ __forceinline__ int row_of_block() {
  const int sub = threadIdx.x / G;
  return G < kWave ? sub : __builtin_amdgcn_readfirstlane(sub);
}

// Waits until this wave's stores have left for memory.
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

struct Plus {
  template <typename V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Larger {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// The value of another lane of the sixteen, by a cross-lane move of the vector unit (a tenth of the time that one
// through LDS takes): 0xB1 and 0x4E exchange neighbours and pairs, 0x141 and 0x140 mirror eight and sixteen lanes.
template <int CTRL, typename V>
__device__ __forceinline__ V across(V v) {
  static_assert(sizeof(V) == 4 || sizeof(V) == 8, "words");
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
  } else {
    const int2 w = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(V, make_int2(__builtin_amdgcn_mov_dpp(w.x, CTRL, 0xf, 0xf, true),
                                           __builtin_amdgcn_mov_dpp(w.y, CTRL, 0xf, 0xf, true)));
  }
}
template <typename V>
__device__ __forceinline__ V lane_value(V v, int lane) {
  if constexpr (sizeof(V) == 4) {
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else {
    const int2 w = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(V, make_int2(__builtin_amdgcn_readlane(w.x, lane), __builtin_amdgcn_readlane(w.y, lane)));
  }
}

// v of G lanes of a wave together (G a power of two to 64), in an order that is the same for all of them.
template <int G, typename V, typename Op>
__device__ __forceinline__ V lanes_reduce(V v, Op op) {
  if (G >= 2) v = op(v, across<0xB1>(v));
  if (G >= 4) v = op(v, across<0x4E>(v));
  if (G >= 8) v = op(v, across<0x141>(v));
  if (G >= 16) v = op(v, across<0x140>(v));
  if (G == 32) v = op(v, __shfl_xor(v, 16, kWave));
  if (G == 64) v = op(op(lane_value(v, 0), lane_value(v, 16)), op(lane_value(v, 32), lane_value(v, 48)));
  return v;
}

// The same over the G threads of a row.  `part` is LDS of G / 64 values of this row's own (none for G <= 64); it is
// written before and read after one barrier, so two calls in a row need different ones.
template <int G, typename V, typename Op>
__device__ __forceinline__ V row_reduce(V v, V* part, Op op) {
  v = lanes_reduce<(G < kWave ? G : kWave)>(v, op);
  if (G <= kWave) return v;
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  V s = part[0];
#pragma unroll
  for (int i = 1; i < G / kWave; ++i) s = op(s, part[i]);
  return s;
}
template <int G, typename V>
__device__ __forceinline__ V row_sum(V v, V* part) {
  return row_reduce<G>(v, part, Plus());
}
template <int G>
__device__ __forceinline__ float row_max(float v, float* part) {
  return row_reduce<G>(v, part, Larger());
}

// What blocks of one launch leave for the block that comes last.  The stores and loads are device-wide ones, which go
// past the caches that the compute dies do not share; stores_done() stands between a wave's stores and the ticket.
template <typename V>
__device__ __forceinline__ void share(V* p, V v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V>
__device__ __forceinline__ V shared(const V* p) {
  return __hip_atomic_load(const_cast<V*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A counter of blocks that are done, zero between launches.  Blocks that count at one address wait for each other, some
// 9 ns each (4096 of them 38 us), so counters stand in lines of their own, and blocks of one large launch count in two
// steps, in kBranches groups and then the groups (3 us).
struct alignas(128) Ticket {
  unsigned n;
};
constexpr unsigned kBranches = 32;
// True for the last of `all` callers, for whom everything the others shared is there; the counter is zero again then.
// One thread of a block calls it, after what the block shares.
__device__ __forceinline__ bool last_ticket(Ticket* t, unsigned all) {
  asm volatile("" ::: "memory");
  const bool last = atomicInc(&t->n, all - 1) == all - 1;
  asm volatile("" ::: "memory");
  return last;
}
// The same for caller number `at`, with 1 + kBranches counters.
__device__ __forceinline__ bool last_ticket(Ticket* t, unsigned at, unsigned all) {
  const unsigned groups = all < kBranches ? all : kBranches, group = at % groups;
  return last_ticket(t + 1 + group, all / groups + (group < all % groups ? 1 : 0)) && last_ticket(t, groups);
}

// An index array of 64 or 32 bits, and a value array of float16 or float32.
__device__ __forceinline__ long long read_index(const void* p, size_t i, int wide) {
  return wide ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}
__device__ __forceinline__ float read_value(const void* p, size_t i, int half) {
  return half ? (float)reinterpret_cast<const _Float16*>(p)[i] : reinterpret_cast<const float*>(p)[i];
}

}  // namespace tt
