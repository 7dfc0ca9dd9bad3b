// Layer normalisation of rows: y = (x - mean) / sqrt(var + eps) * w + b, its gradient dx and the reductions over the
// rows that give dw and db. x, y, dy and dx are float32 or float16, everything else float32.
//
//   n = (x - mean) rstd,  h = dy w,  dx = rstd (h - mean(h) - n mean(h n)),  dw = sum_rows dy n,  db = sum_rows dy
//
// G threads hold a row in registers, NV sixteen-byte packs each, so a row is read once whatever is summed over it: the
// variance is that of the values less their mean, not a difference of squares. The backward kernel walks a block's rows
// and keeps each thread's columns of dw and db in registers on the way; they are added up over the rows of a block in
// LDS, and over the blocks by ln_join. Rows longer than the registers hold are read again (the *_long kernels).
//
// Memory bounds them: 2^25 float32 values take 47 to 57 us forward and 76 to 84 us backward (4.7 to 5.7 and 4.8 to 5.3
// TB/s, a large copy 5.0 to 5.6) in rows of 24 to 8192; float16 23 to 37 us and 43 to 63 us (3.6 to 5.8 and 3.2 to 4.7
// TB/s), the longer ones where rows begin off sixteen bytes.  Rows longer than a block holds read twice or three times
// take 74 and 157 us (20001 columns).  What is left to lose are idle lanes, where a row's packs do not fill its waves, and
// the blocks' sums.
#include "rows.h"

namespace {

using tt::kWave;

// Columns [q n, q n + n) of a row that begins at any multiple of its type (the memory instructions take that).
template <typename T>
struct Loose;
template <>
struct Loose<float> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4)));
  static constexpr int n = 4;
};
template <>
struct Loose<_Float16> {
  typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2)));
  static constexpr int n = 8;
};

// Behind the last column: zeros, or (REPEAT) the pack's first value again, whose normalised value is as finite as the row's.
template <bool REPEAT = false, typename T>
__device__ __forceinline__ typename Loose<T>::type read_columns(const T* row, int q, int D) {
  constexpr int n = Loose<T>::n;
  if (q * n + n <= D) return *reinterpret_cast<const typename Loose<T>::type*>(row + (size_t)q * n);
  typename Loose<T>::type p;
  p[0] = row[(size_t)q * n];
#pragma unroll
  for (int i = 1; i < n; ++i) p[i] = q * n + i < D ? row[(size_t)q * n + i] : REPEAT ? p[0] : (T)0.f;
  return p;
}
template <typename T>
__device__ __forceinline__ bool whole_lines(int D) {
  return D % (128 / (int)sizeof(T)) == 0;
}
// `passing`: on its way to memory at once, past the caches, which then hold more of what is read. Float32 rows of the
// forward pass that end inside a line of memory and have a part of a wave each, so that its pieces come from several
// instructions, are better left to the cache, which puts them together (2^27 values: 72 columns 199 us, 390 passing, 260
// columns 191 and 236). Rows that come from one instruction pass (20 columns 256 us and 249), and so do those of a wave or
// a block (2500 columns 196 and 188), halves (385 columns at 2^25 values 37 and 36) and the backward pass, which has more to
// read (2^25 values: 60 columns 82 us and 79, 2500 columns 82 and 79; 2^27 values: 319 and 298 at 2500, level within 7 %
// in shorter rows).
template <typename T>
__device__ __forceinline__ void write_columns(T* row, int q, int D, const typename Loose<T>::type& p,
                                              bool passing = true) {
  constexpr int n = Loose<T>::n;
  if (q * n + n <= D) {
    typename Loose<T>::type* at = reinterpret_cast<typename Loose<T>::type*>(row + (size_t)q * n);
    if (sizeof(T) == 2) {
      __builtin_nontemporal_store(p, at);
    } else if (passing) {
      asm volatile("" ::: "memory");        // (or the compiler makes one store of the two, that does not pass)
      __builtin_nontemporal_store(p, at);
      asm volatile("" ::: "memory");
    } else {
      *at = p;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < n; ++i)
    if (q * n + i < D) row[(size_t)q * n + i] = p[i];
}
// n parameters from column q n on; `other` where there are none
template <int n>
__device__ __forceinline__ void read_parameters(float (&v)[n], const float* w, int q, int D, float other) {
  if (w && q * n + n <= D) {
#pragma unroll
    for (int i = 0; i < n; i += 4) {
      const float4 p = *reinterpret_cast<const float4*>(w + (size_t)q * n + i);
      v[i] = p.x;
      v[i + 1] = p.y;
      v[i + 2] = p.z;
      v[i + 3] = p.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < n; ++i) v[i] = w && q * n + i < D ? w[(size_t)q * n + i] : other;
}

// Sums of N values over the threads of a row: G of a wave, or (G = 0) the whole waves of one y of the block.  part: LDS
// of 16 N floats of this call's own.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* part) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = tt::lanes_reduce<(G ? G : kWave)>(v[k], tt::Plus());
  if (G) return;
  const int waves = blockDim.x / kWave;
  part += threadIdx.y * waves * N;
  if ((threadIdx.x & (kWave - 1)) == 0)
#pragma unroll
    for (int k = 0; k < N; ++k) part[(threadIdx.x >> 6) * N + k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = part[k];
  for (int i = 1; i < waves; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += part[i * N + k];
}

constexpr int kFlight = 16;       // loads that a thread of the joining block has on their way
constexpr int kMostBlock = 1024, kFwdBlock = 256, kBwdBlock = 512;    // threads: G = 0 at most, G > 0 forward, backward

template <typename T, int G, int NV>
__global__ __launch_bounds__(G ? kFwdBlock : kMostBlock) void ln_fwd(const T* __restrict__ x,
                                                                    const float* __restrict__ w,
                                                                    const float* __restrict__ b, T* __restrict__ y,
                                                                    float* __restrict__ mean, float* __restrict__ rstd,
                                                                    int R, int D, float eps) {
  constexpr int n = Loose<T>::n, kRows = G ? kFwdBlock / (G ? G : 1) : 1;
  typedef typename Loose<T>::type P;
  __shared__ float part[2][G ? 1 : kMostBlock / kWave];
  const int stride = G ? G : (int)blockDim.x, lane = threadIdx.x % stride;
  const int sub = G ? tt::row_of_block<G ? G : 1>() : 0;
  const int packs = (D + n - 1) / n;
  const bool passing = G == 0 || G == kWave || NV == 1 || whole_lines<T>(D);
  for (long long row = (long long)blockIdx.x * kRows + sub; row < R; row += (long long)gridDim.x * kRows) {
    const T* __restrict__ p = x + row * (size_t)D;
    P v[NV];
    float s[1] = {}, sq[1] = {};
#pragma unroll
    for (int u = 0; u < NV; ++u) v[u] = lane + u * stride < packs ? read_columns(p, lane + u * stride, D) : P((T)0.f);
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int i = 0; i < n; ++i) s[0] += tt::widen(v[u][i]);
    group_sum<G>(s, part[0]);
    const float m = s[0] / (float)D;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int left = D - (lane + u * stride) * n;     // columns of the row from this pack on
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float d = i < left ? tt::widen(v[u][i]) - m : 0.f;
        sq[0] = fmaf(d, d, sq[0]);
      }
    }
    group_sum<G>(sq, part[1]);
    const float r = 1.f / sqrtf(sq[0] / (float)D + eps);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int q = lane + u * stride;
      if (q >= packs) break;
      float wv[n], bv[n];
      read_parameters(wv, w, q, D, 1.f);
      read_parameters(bv, b, q, D, 0.f);
      P o;
#pragma unroll
      for (int i = 0; i < n; ++i) o[i] = (T)fmaf((tt::widen(v[u][i]) - m) * r, wv[i], bv[i]);
      write_columns(y + row * (size_t)D, q, D, o, passing);
    }
    if (mean && lane == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

__device__ tt::Ticket ln_done;     // blocks of a launch that have left their sums: zero between launches

// parts: [blocks][2][D], a block's sums for dw and db (NULL when neither is wanted). One block writes dw and db itself;
// of few blocks with few columns (`joins`) the last adds them up, which saves a launch.
template <typename T, int G, int NV>
__global__ __launch_bounds__(G ? kBwdBlock : kMostBlock) void ln_bwd(const T* __restrict__ x, const T* __restrict__ dy,
                                                                    const float* __restrict__ w,
                                                                    const float* __restrict__ mean,
                                                                    const float* __restrict__ rstd, T* __restrict__ dx,
                                                                    float* parts, float* dw_out, float* db_out,
                                                                    int joins, int R, int D) {
  constexpr int n = Loose<T>::n;
  typedef typename Loose<T>::type P;
  __shared__ float part[2][G ? 1 : 2 * (kMostBlock / kWave)];
  const int stride = G ? G : (int)blockDim.x, rows = G ? kBwdBlock / (G ? G : 1) : (int)blockDim.y;
  const int lane = G ? threadIdx.x % stride : threadIdx.x;
  const int sub = G ? tt::row_of_block<G ? G : 1>() : __builtin_amdgcn_readfirstlane(threadIdx.y);
  const int thread = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  const int all_packs = (D + n - 1) / n;
  float sums[2][NV][n] = {};        // dw, db
  float wv[NV][n];
#pragma unroll
  for (int u = 0; u < NV; ++u)
    read_parameters(wv[u], lane + u * stride < all_packs ? w : nullptr, lane + u * stride, D, 1.f);
  int turn = 0;
  // (all rows of a block go round together, for the barriers: one behind the last has no packs)
  for (long long row0 = (long long)blockIdx.x * rows; row0 < R; row0 += (long long)gridDim.x * rows, turn ^= 1) {
    const long long row = row0 + sub < R ? row0 + sub : R - 1;
    const int packs = row0 + sub < R ? all_packs : 0;
    const size_t base = row * (size_t)D;
    P xv[NV], gv[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int q = lane + u * stride;
      xv[u] = q < packs ? read_columns<true>(x + base, q, D) : P((T)0.f);
      gv[u] = q < packs ? read_columns(dy + base, q, D) : P((T)0.f);
    }
    const float m = mean[row], r = rstd[row];
    float of[2] = {};                 // h, h n
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if (lane + u * stride >= packs) break;
#pragma unroll
      for (int i = 0; i < n; ++i) {       // (behind the last column dy is 0 and n finite: nothing is added)
        const float g = tt::widen(gv[u][i]), nn = (tt::widen(xv[u][i]) - m) * r, h = g * wv[u][i];
        of[0] += h;
        of[1] = fmaf(h, nn, of[1]);
        sums[0][u][i] = fmaf(g, nn, sums[0][u][i]);
        sums[1][u][i] += g;
      }
    }
    if (!dx) continue;
    group_sum<G>(of, part[turn]);     // (in turns: one barrier to a row)
    const float mh = of[0] / (float)D, mhn = of[1] / (float)D;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int q = lane + u * stride;
      if (q >= packs) break;
      P o;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float nn = (tt::widen(xv[u][i]) - m) * r;
        o[i] = (T)(r * (tt::widen(gv[u][i]) * wv[u][i] - mh - nn * mhn));
      }
      write_columns(dx + base, q, D, o);
    }
  }
  if (!dw_out && !db_out) return;
  const bool alone = gridDim.x == 1;
  float* out[2] = {alone ? dw_out : parts + (size_t)blockIdx.x * 2 * D,
                   alone ? db_out : parts + (size_t)blockIdx.x * 2 * D + D};
  auto leave = [&](int which, int c, float s) {
    if (c >= D || !out[which]) return;
    if (joins) tt::share(out[which] + c, s);
    else out[which][c] = s;
  };
  // this block's rows: one sum for each column, pack by pack
  __shared__ __attribute__((aligned(16))) float all[(G || sizeof(T) == 4 ? kBwdBlock : kMostBlock) * n];
  // (values of as many threads as have several rows)
#pragma unroll
  for (int u = 0; u < 2 * NV; ++u) {
    const int which = u & 1, first = (u >> 1) * stride;
    if (rows == 1) {
#pragma unroll
      for (int i = 0; i < n; ++i) leave(which, (lane + first) * n + i, sums[which][u >> 1][i]);
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < n; ++i) all[thread * n + i] = sums[which][u >> 1][i];
      __syncthreads();
      for (int c = thread; c < stride * n; c += threads) {
        float s = 0.f;
        for (int k = 0; k < rows; ++k) s += all[k * stride * n + c];
        leave(which, first * n + c, s);
      }
    }
  }
  if (!joins) return;
  __shared__ bool last;
  tt::stores_done();
  __syncthreads();
  if (thread == 0) last = tt::last_ticket(&ln_done, gridDim.x);
  __syncthreads();
  if (!last) return;
  // as many threads to a column as there are, each with every so manieth block's sum, kFlight on their way
  double* sums64 = reinterpret_cast<double*>(all);
  const int ways = 2 * D < threads ? threads / (2 * D) : 1, used = 2 * D < threads ? 2 * D : threads;
  for (int c0 = 0; c0 < 2 * D; c0 += used) {
    const int c = c0 + thread % used, way = thread / used;
    double s = 0.0;
    if (way < ways && c < 2 * D)
      for (int k = way; k < (int)gridDim.x; k += kFlight * ways) {
        float v[kFlight];
#pragma unroll
        for (int i = 0; i < kFlight; ++i) {
          v[i] = 0.f;
          if (k + i * ways < (int)gridDim.x) v[i] = tt::shared(parts + (size_t)(k + i * ways) * 2 * D + c);
        }
#pragma unroll
        for (int i = 0; i < kFlight; ++i) s += (double)v[i];
      }
    __syncthreads();
    sums64[thread] = s;
    __syncthreads();
    if (way || c >= 2 * D) continue;
    for (int k = 1; k < ways; ++k) s += sums64[k * used + thread];
    float* to = c < D ? dw_out : db_out;
    if (to) to[c < D ? c : c - D] = (float)s;
  }
}

// dw and db from the blocks' sums: 64 columns to a block of 16 waves, each wave every sixteenth block's, in an order
// that the sizes alone decide.
__global__ __launch_bounds__(1024) void ln_join(const float* __restrict__ parts, float* __restrict__ dw,
                                                float* __restrict__ db, int D, int blocks) {
  __shared__ double sums[16][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const size_t c = (size_t)blockIdx.x * kWave + lane;
  double s = 0.0;
  if (c < 2 * (size_t)D) {
    const float* __restrict__ p = parts + c;
    const size_t step = 2 * (size_t)D;
    int k = wave;
    for (; k + 7 * 16 < blocks; k += 8 * 16) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[(k + i * 16) * step];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += (double)v[i];
    }
    for (; k < blocks; k += 16) s += (double)p[k * step];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || c >= 2 * (size_t)D) return;
  for (int k = 1; k < 16; ++k) s += sums[k][lane];
  float* __restrict__ out = c < (size_t)D ? dw : db;
  if (out) out[c < (size_t)D ? c : c - D] = (float)s;
}

// ---- rows that no block's registers hold -----------------------------------------------------------

constexpr int kLong = 1024;

template <typename T>
__global__ __launch_bounds__(kLong) void ln_fwd_long(const T* __restrict__ x, const float* __restrict__ w,
                                                     const float* __restrict__ b, T* __restrict__ y,
                                                     float* __restrict__ mean, float* __restrict__ rstd, int R, int D,
                                                     float eps) {
  constexpr int n = Loose<T>::n;
  __shared__ float part[2][kLong / kWave];
  const int packs = (D + n - 1) / n;
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const T* __restrict__ p = x + row * (size_t)D;
    float s = 0.f;
    for (int q = threadIdx.x; q < packs; q += kLong) {
      const typename Loose<T>::type v = read_columns(p, q, D);
#pragma unroll
      for (int i = 0; i < n; ++i) s += tt::widen(v[i]);
    }
    const float m = tt::row_sum<kLong>(s, part[0]) / (float)D;
    float sq = 0.f;
    for (int q = threadIdx.x; q < packs; q += kLong) {
      const typename Loose<T>::type v = read_columns(p, q, D);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float d = q * n + i < D ? tt::widen(v[i]) - m : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float r = 1.f / sqrtf(tt::row_sum<kLong>(sq, part[1]) / (float)D + eps);
    for (int q = threadIdx.x; q < packs; q += kLong) {
      const typename Loose<T>::type v = read_columns(p, q, D);
      float wv[n], bv[n];
      read_parameters(wv, w, q, D, 1.f);
      read_parameters(bv, b, q, D, 0.f);
      typename Loose<T>::type o;
#pragma unroll
      for (int i = 0; i < n; ++i) o[i] = (T)fmaf((tt::widen(v[i]) - m) * r, wv[i], bv[i]);
      write_columns(y + row * (size_t)D, q, D, o);
    }
    if (mean && threadIdx.x == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kLong) void ln_bwd_long(const T* __restrict__ x, const T* __restrict__ dy,
                                                     const float* __restrict__ w, const float* __restrict__ mean,
                                                     const float* __restrict__ rstd, T* __restrict__ dx, int R, int D) {
  constexpr int n = Loose<T>::n;
  __shared__ float part[2][kLong / kWave];
  const int packs = (D + n - 1) / n;
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const size_t base = row * (size_t)D;
    const float m = mean[row], r = rstd[row];
    float sh = 0.f, shn = 0.f;
    for (int q = threadIdx.x; q < packs; q += kLong) {
      const typename Loose<T>::type xv = read_columns<true>(x + base, q, D), gv = read_columns(dy + base, q, D);
      float wv[n];
      read_parameters(wv, w, q, D, 1.f);
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float h = tt::widen(gv[i]) * wv[i];
        sh += h;
        shn = fmaf(h, (tt::widen(xv[i]) - m) * r, shn);
      }
    }
    __syncthreads();
    const float mh = tt::row_sum<kLong>(sh, part[0]) / (float)D, mhn = tt::row_sum<kLong>(shn, part[1]) / (float)D;
    for (int q = threadIdx.x; q < packs; q += kLong) {
      const typename Loose<T>::type xv = read_columns(x + base, q, D), gv = read_columns(dy + base, q, D);
      float wv[n];
      read_parameters(wv, w, q, D, 1.f);
      typename Loose<T>::type o;
#pragma unroll
      for (int i = 0; i < n; ++i)
        o[i] = (T)(r * (tt::widen(gv[i]) * wv[i] - mh - (tt::widen(xv[i]) - m) * r * mhn));
      write_columns(dx + base, q, D, o);
    }
  }
}

// A thread sums its pack of columns over the rows of its split: parts[split][0 | 1][column].
template <typename T>
__global__ __launch_bounds__(256) void ln_parts_long(const T* __restrict__ x, const T* __restrict__ dy,
                                                     const float* __restrict__ mean, const float* __restrict__ rstd,
                                                     float* __restrict__ parts, int R, int D, int rows_per_split) {
  constexpr int n = Loose<T>::n;
  const int q = blockIdx.x * 256 + threadIdx.x;
  if (q >= (D + n - 1) / n) return;
  const int r0 = blockIdx.y * rows_per_split;
  const int r1 = R - r0 < rows_per_split ? R : r0 + rows_per_split;
  float dw[n] = {}, db[n] = {};
  for (int row = r0; row < r1; ++row) {
    const size_t base = row * (size_t)D;
    const typename Loose<T>::type xv = read_columns(x + base, q, D), gv = read_columns(dy + base, q, D);
    const float m = mean[row], r = rstd[row];
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float g = tt::widen(gv[i]);
      dw[i] = fmaf(g, (tt::widen(xv[i]) - m) * r, dw[i]);
      db[i] += g;
    }
  }
  float* __restrict__ out = parts + (size_t)blockIdx.y * 2 * D;
#pragma unroll
  for (int i = 0; i < n; ++i)
    if (q * n + i < D) {
      out[q * n + i] = dw[i];
      out[D + q * n + i] = db[i];
    }
}

// ---- launches --------------------------------------------------------------------------------------

int check(const char* fn, int dtype, long long R, int D) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_F16, "%s: unknown type %d", fn, dtype);
  TT_REQUIRE(R > 0 && R <= (1 << 30), "%s: rows must be in 1..2^30 (got %lld)", fn, R);
  TT_REQUIRE(D > 0 && D <= (1 << 30), "%s: columns must be in 1..2^30 (got %d)", fn, D);
  return 0;
}

unsigned grid_for(long long rows, int rows_per_block, long long most) {
  const long long blocks = (rows + rows_per_block - 1) / rows_per_block;
  return (unsigned)(blocks < most ? blocks : most);
}

template <typename T, int G, int NV>
int launch_fwd(const T* x, const float* w, const float* b, T* y, float* mean, float* rstd, float eps, int R, int D) {
  const int packs = (D + Loose<T>::n - 1) / Loose<T>::n;
  const int block = G ? kFwdBlock : (packs + NV * kWave - 1) / (NV * kWave) * kWave;
  const int rows = G ? kFwdBlock / (G ? G : 1) : 1;
  ln_fwd<T, G, NV><<<grid_for(R, rows, 1 << 22), block, 0, tt::stream()>>>(x, w, b, y, mean, rstd, R, D, eps);
  TT_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int forward(const T* x, const float* w, const float* b, T* y, float* mean, float* rstd, float eps, int R, int D) {
  const int packs = (D + Loose<T>::n - 1) / Loose<T>::n;
#define TT_LN_FWD(G, NV) return launch_fwd<T, G, NV>(x, w, b, y, mean, rstd, eps, R, D)
  // The fewest lanes that hold a row in two or three packs each, which keeps several rows of a wave on their way (2^25
  // values: 64 columns of float32 48 us, on 32 lanes 77; 256 columns 48, on 64 lanes 50, of halves 24 and 41; 72 columns
  // with three packs 55, with two 59); a wave alone up to five, before the barriers of a block (1088 columns 52 us, by
  // blocks 58, of halves 2176 columns 27 and 31); then as few packs a thread as leave waves enough (2304 columns with three
  // 49 us, with two 64; 3328 with four 49, with three 57; but 2048 with two 48, with one 70).
  if (packs <= 4) TT_LN_FWD(4, 1);
  if (packs <= 8) TT_LN_FWD(8, 1);
  if (packs <= 16) TT_LN_FWD(8, 2);
  if (packs <= 24) TT_LN_FWD(8, 3);
  if (packs <= 32) TT_LN_FWD(16, 2);
  if (packs <= 48) TT_LN_FWD(16, 3);
  if (packs <= 64) TT_LN_FWD(32, 2);
  if (packs <= 96) TT_LN_FWD(32, 3);
  if (packs <= 128) TT_LN_FWD(64, 2);
  if (packs <= 192) TT_LN_FWD(64, 3);
  if (packs <= 256) TT_LN_FWD(64, 4);
  if (packs <= 320) TT_LN_FWD(64, 5);
  if (packs <= 512) TT_LN_FWD(0, 2);
  if (packs <= 768) TT_LN_FWD(0, 3);
  if (packs <= 4 * kMostBlock) TT_LN_FWD(0, 4);
#undef TT_LN_FWD
  ln_fwd_long<T><<<grid_for(R, 1, 1 << 20), kLong, 0, tt::stream()>>>(x, w, b, y, mean, rstd, R, D, eps);
  TT_LAUNCH_CHECK();
  return 0;
}

int launch_join(const float* parts, float* dw, float* db, int D, int blocks) {
  ln_join<<<(2 * (unsigned)D + kWave - 1) / kWave, 1024, 0, tt::stream()>>>(parts, dw, db, D, blocks);
  TT_LAUNCH_CHECK();
  return 0;
}

template <typename T, int G, int NV>
int launch_bwd(const T* x, const T* dy, const float* w, const float* mean, const float* rstd, T* dx, float* dw,
               float* db, int R, int D) {
  const int packs = (D + Loose<T>::n - 1) / Loose<T>::n;
  // a row's threads, and as many rows as fill the block, which leaves one set of sums. (Long rows of halves, whose sums
  // weigh as much as a dozen of them: blocks of 1024 threads, 8192 columns 55 us at 2^25 values, 64 with 512; and rows of
  // three waves, five of which leave fewer threads idle than two: 2100 columns 61 us, 68 with 512. Of float32, or of other
  // short ones, 512: 1537 columns of halves 59 us, 71 with 1024)
  const int along = G ? kBwdBlock : (packs + NV * kWave - 1) / (NV * kWave) * kWave;
  const int fill = sizeof(T) == 2 && (along > 256 || along == 192) ? kMostBlock : kBwdBlock;
  const int rows = G ? kBwdBlock / (G ? G : 1) : along < fill ? fill / along : 1;
  const dim3 block(along, G ? 1 : rows);
  // as many blocks as the device holds at once: more of them would only leave more sums
  static int resident[kMostBlock / kWave + 1];
  int& per_unit = resident[along / kWave];
  if (per_unit == 0)
    TT_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_unit, ln_bwd<T, G, NV>, block.x * block.y, 0));
  const unsigned grid = grid_for(R, rows, (long long)tt::compute_units() * (per_unit > 0 ? per_unit : 1));
  const bool sums = dw || db;
  // the last block joins what takes it a few rounds of loads: that saves a launch (1000 rows of 64: 5.2 us, 8.1 with it; 50
  // of 768, in two rounds, 8.9 and 7.8, where the host is spared its part; 300 of 512, in six rounds, 11.2 and 7.6)
  const int threads = block.x * block.y, ways = 2 * D < threads ? threads / (2 * D) : 1;
  const long long rounds = (2 * (long long)D + threads - 1) / threads * ((grid + kFlight * ways - 1) / (kFlight * ways));
  const bool joins = sums && grid > 1 && rounds <= 3;
  void* ws = nullptr;
  if (sums && grid > 1)
    if (tt::workspace((size_t)grid * 2 * D * sizeof(float), &ws)) return -1;
  ln_bwd<T, G, NV><<<grid, block, 0, tt::stream()>>>(x, dy, w, mean, rstd, dx, (float*)ws, dw, db, joins, R, D);
  TT_LAUNCH_CHECK();
  return sums && grid > 1 && !joins ? launch_join((const float*)ws, dw, db, D, grid) : 0;
}

template <typename T>
int backward(const T* x, const T* dy, const float* w, const float* mean, const float* rstd, T* dx, float* dw, float* db,
             int R, int D) {
  constexpr bool wide = sizeof(T) == 4;
  const int packs = (D + Loose<T>::n - 1) / Loose<T>::n;
#define TT_LN_BWD(G, NV) return launch_bwd<T, G, NV>(x, dy, w, mean, rstd, dx, dw, db, R, D)
  // A lane has x, dy and two sums of each column, so fewer packs than forward: one, up to 64 to a row (2^25 values: 40
  // columns of float32 77 us, with two 100; 72 columns 79, with two 85), but two or three where one would leave a third of
  // the lanes idle (288 columns with three 78, on 64 lanes with two 82; of halves 576 columns 50, by blocks 60). From 97
  // packs on a wave with two or three (577 columns of float32 81, by blocks 89, of halves 1025 columns 64, by blocks 81),
  // then blocks: with one or two packs a thread as long as the row has waves enough for few rows (20 of 1537 columns of
  // halves 8 us, with two packs 10; many rows are level within 6 %), of float32 three from there on (1088 columns 77, with
  // two 97), or four where three would leave five waves (3328 columns 81, with three 88), of halves, which are eight to a
  // pack, two (3200 columns 50, with one 63).
  if (packs <= 4) TT_LN_BWD(4, 1);
  if (packs <= 8) TT_LN_BWD(8, 1);
  if (packs <= 16) TT_LN_BWD(16, 1);
  if (packs <= 32) TT_LN_BWD(32, 1);
  if (packs <= 48) TT_LN_BWD(32, 2);
  if (packs <= 64) TT_LN_BWD(64, 1);
  if (packs <= 96) TT_LN_BWD(32, 3);
  if (packs <= 128) TT_LN_BWD(64, 2);
  if (packs <= 192) TT_LN_BWD(64, 3);
  if (packs <= 256) TT_LN_BWD(0, 1);
  if constexpr (wide) {
    if (packs > 384 && packs <= 512) TT_LN_BWD(0, 2);
    if (packs > 768 && packs <= 960) TT_LN_BWD(0, 4);
    if (packs <= 3 * kMostBlock) TT_LN_BWD(0, 3);
    if (packs <= 4 * kMostBlock) TT_LN_BWD(0, 4);
  } else {
    if (packs <= 2 * kMostBlock) TT_LN_BWD(0, 2);
  }
#undef TT_LN_BWD
  hipStream_t st = tt::stream();
  if (dx) {
    ln_bwd_long<T><<<grid_for(R, 1, 1 << 20), kLong, 0, st>>>(x, dy, w, mean, rstd, dx, R, D);
    TT_LAUNCH_CHECK();
  }
  if (dw || db) {
    const int columns = (packs + 255) / 256;
    int splits = (4 * tt::compute_units() + columns - 1) / columns;
    if (splits > R) splits = R;
    const int per = (R + splits - 1) / splits;
    splits = (R + per - 1) / per;
    void* ws;
    if (tt::workspace((size_t)splits * 2 * D * sizeof(float), &ws)) return -1;
    ln_parts_long<T><<<dim3(columns, splits), 256, 0, st>>>(x, dy, mean, rstd, (float*)ws, R, D, per);
    TT_LAUNCH_CHECK();
    return launch_join((const float*)ws, dw, db, D, splits);
  }
  return 0;
}

}  // namespace

extern "C" {

int tt_layer_norm_fwd(const void* x, const float* w, const float* b, void* y, float* mean, float* rstd, double eps,
                      int dtype, long long R, int D) {
  TT_REQUIRE_INIT();
  TT_REQUIRE(x && y, "tt_layer_norm_fwd: null pointer");
  TT_REQUIRE((mean == nullptr) == (rstd == nullptr), "tt_layer_norm_fwd: mean and rstd come together");
  if (int rc = check("tt_layer_norm_fwd", dtype, R, D)) return rc;
  TT_REQUIRE_ALIGNED("tt_layer_norm_fwd", x, w, b, y);
  if (dtype == TT_F32) return forward((const float*)x, w, b, (float*)y, mean, rstd, (float)eps, (int)R, D);
  return forward((const _Float16*)x, w, b, (_Float16*)y, mean, rstd, (float)eps, (int)R, D);
}

int tt_layer_norm_bwd(const void* x, const void* dy, const float* w, const float* mean, const float* rstd, void* dx,
                      float* dw, float* db, int dtype, long long R, int D) {
  TT_REQUIRE_INIT();
  TT_REQUIRE(x && dy && mean && rstd, "tt_layer_norm_bwd: null pointer");
  if (int rc = check("tt_layer_norm_bwd", dtype, R, D)) return rc;
  TT_REQUIRE_ALIGNED("tt_layer_norm_bwd", x, dy, w, dx, dw, db);
  if (dtype == TT_F32)
    return backward((const float*)x, (const float*)dy, w, mean, rstd, (float*)dx, dw, db, (int)R, D);
  return backward((const _Float16*)x, (const _Float16*)dy, w, mean, rstd, (_Float16*)dx, dw, db, (int)R, D);
}

}  // extern "C"
