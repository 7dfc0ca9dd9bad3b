// What the kernels over rows of float32 or float16 values share: layer normalisation (layernorm.hip), token
// log probabilities and distillation (vocab.hip).  Values are widened to float32 as they are read; sums and
// statistics are float32 or wider, and a result is rounded once, to its own type, as it is stored.
//
// G threads work on a row: a wave (G = 64, several rows to a block, no block barrier) or a block.
#pragma once
#include "tt_common.h"

#include <math.h>

namespace tt {

// Sixteen bytes of a row.
template <typename T>
struct Pack;
template <>
struct Pack<float> {
  typedef float type __attribute__((ext_vector_type(4)));
  static constexpr int n = 4;
};
template <>
struct Pack<_Float16> {
  typedef _Float16 type __attribute__((ext_vector_type(8)));
  static constexpr int n = 8;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }

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

// An index array of 64 or 32 bits, and a value array of float16 or float32.
__device__ __forceinline__ long long read_index(const void* p, size_t i, int wide) {
  return wide ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}
__device__ __forceinline__ float read_value(const void* p, size_t i, int half) {
  return half ? (float)reinterpret_cast<const _Float16*>(p)[i] : reinterpret_cast<const float*>(p)[i];
}

}  // namespace tt
