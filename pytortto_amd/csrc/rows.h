// What the kernels over rows of float32 or float16 values share: layer normalisation (layernorm.hip), token
// log probabilities and distillation (vocab.hip).  Values are widened to float32 as they are read; sums and
// statistics are float32 or wider, and a result is rounded once, to its own type, as it is stored.
//
// G threads work on a row: a wave (G = 64, several rows to a block, no block barrier) or a block.
#pragma once
#include "tt_common.h"

#include <math.h>

namespace tt {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }

// Sixteen bytes of a row.  They are kept as four words until their values are wanted: as a vector of halves the compiler
// would give every value a register of its own.
typedef unsigned Words __attribute__((ext_vector_type(4)));
template <typename T>
struct Pack;
template <>
struct Pack<float> {
  typedef float vector __attribute__((ext_vector_type(4)));
  static constexpr int n = 4;
  static constexpr unsigned lowest = 0xff800000u;      // -inf, as often as a word holds it
};
template <>
struct Pack<_Float16> {
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
  for (int i = 0; i < Pack<T>::n; ++i) v[i] = (T)z[i];
  return __builtin_bit_cast(Words, v);
}

// Whether the threads of a row are a wave of a larger block or the block itself.
template <int G>
__device__ __forceinline__ void sync_row() {
  if (G == kWave) {
    // LDS operations of one wave run in order: only the compiler has to keep them so
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// Waits until this wave's stores have left for memory: what another wave of the block stores to the same place after
// the next sync_row comes later.
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, kWave));
  return v;
}

// Sum over the G threads of a row; every thread gets it.  `part` is LDS of G / 64 values of this row's own; it is
// written before and read after one barrier, so two calls in a row need different ones.
template <int G, typename V>
__device__ __forceinline__ V row_sum(V v, V* part) {
  v = wave_sum(v);
  if (G == kWave) return v;
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  V s = part[0];
#pragma unroll
  for (int i = 1; i < G / kWave; ++i) s += part[i];
  return s;
}
template <int G>
__device__ __forceinline__ float row_max(float v, float* part) {
  v = wave_max(v);
  if (G == kWave) return v;
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = part[0];
#pragma unroll
  for (int i = 1; i < G / kWave; ++i) s = fmaxf(s, part[i]);
  return s;
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
// True for the last of `all` callers, for whom everything the others shared is there; the counter is zero again then.
// One thread of a block calls it, after what the block shares.
__device__ __forceinline__ bool last_ticket(unsigned* counter, unsigned all) {
  asm volatile("" ::: "memory");
  const bool last = atomicInc(counter, all - 1) == all - 1;
  asm volatile("" ::: "memory");
  return last;
}

// An index array of 64 or 32 bits, and a value array of float16 or float32.
__device__ __forceinline__ long long read_index(const void* p, size_t i, int wide) {
  return wide ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}
__device__ __forceinline__ float read_value(const void* p, size_t i, int half) {
  return half ? (float)reinterpret_cast<const _Float16*>(p)[i] : reinterpret_cast<const float*>(p)[i];
}

}  // namespace tt
