// What the kernels over rows of float32 or float16 values share: layer normalisation (layernorm.hip), token
// log probabilities and distillation (vocab.hip).  Values are widened to float32 as they are read; sums and
// statistics are float32 or wider, and a result is rounded once, to its own type, as it is stored.
#pragma once
#include "tt_common.h"

namespace tt {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// Sum over a block of kWaves waves; every thread gets it.  `part` is LDS of kWaves values, free again on return.
template <int kWaves, typename V>
__device__ __forceinline__ V block_sum(V v, V* part) {
  v = wave_sum(v);
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  V s = part[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) s += part[i];
  __syncthreads();
  return s;
}

// An index array of 64 or 32 bits.
__device__ __forceinline__ long long read_index(const void* p, size_t i, int wide) {
  return wide ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

}  // namespace tt
