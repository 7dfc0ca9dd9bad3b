// Layer normalisation of rows: y = (x - mean) / sqrt(var + eps) * w + b, its gradient dx and the reductions over the
// rows that give dw and db.  x, y, dy and dx are float32 or float16, everything else float32.
//
//   n = (x - mean) rstd,  h = dy w,  dx = rstd (h - mean(h) - n mean(h n)),  dw = sum_rows dy n,  db = sum_rows dy
//
// G threads hold a row in registers, NV sixteen-byte packs each, so a row is read once whatever is summed over it: the
// variance is that of the values less their mean, not a difference of squares.  The backward kernel walks a block's
// rows and keeps each thread's columns of dw and db in registers on the way; they are added up over the rows of a block
// in LDS, and over the blocks by ln_join.  Rows longer than the registers hold are read again (the *_long kernels).
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

template <typename T>
__device__ __forceinline__ typename Loose<T>::type read_columns(const T* row, int q, int D) {
  constexpr int n = Loose<T>::n;
  if (q * n + n <= D) return *reinterpret_cast<const typename Loose<T>::type*>(row + (size_t)q * n);
  typename Loose<T>::type p;
#pragma unroll
  for (int i = 0; i < n; ++i) p[i] = q * n + i < D ? row[(size_t)q * n + i] : (T)0.f;
  return p;
}
template <typename T>
__device__ __forceinline__ void write_columns(T* row, int q, int D, const typename Loose<T>::type& p) {
  constexpr int n = Loose<T>::n;
  if (q * n + n <= D) {
    __builtin_nontemporal_store(p, reinterpret_cast<typename Loose<T>::type*>(row + (size_t)q * n));
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

// Sums over the G threads of a row: a part of a wave, a wave, or a block.
template <int G>
__device__ __forceinline__ float group_sum(float v, float* part) {
  if (G > kWave) return tt::row_sum<(G > kWave ? G : kWave)>(v, part);
#pragma unroll
  for (int off = (G < kWave ? G : kWave) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

template <typename T, int G, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK) void ln_fwd(const T* __restrict__ x, const float* __restrict__ w,
                                                const float* __restrict__ b, T* __restrict__ y,
                                                float* __restrict__ mean, float* __restrict__ rstd, int R, int D,
                                                float eps) {
  constexpr int n = Loose<T>::n, kRows = BLOCK / G, kParts = G > kWave ? G / kWave : 1;
  typedef typename Loose<T>::type P;
  __shared__ float part[2][kParts];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G, packs = (D + n - 1) / n;
  for (long long row = (long long)blockIdx.x * kRows + sub; row < R; row += (long long)gridDim.x * kRows) {
    const T* __restrict__ p = x + row * (size_t)D;
    P v[NV];
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) v[u] = lane + u * G < packs ? read_columns(p, lane + u * G, D) : P((T)0.f);
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int i = 0; i < n; ++i) s += tt::widen(v[u][i]);
    const float m = group_sum<G>(s, part[0]) / (float)D;
    float sq = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int left = D - (lane + u * G) * n;      // columns of the row from this pack on
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float d = i < left ? tt::widen(v[u][i]) - m : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float r = 1.f / sqrtf(group_sum<G>(sq, part[1]) / (float)D + eps);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int q = lane + u * G;
      if (q >= packs) break;
      float wv[n], bv[n];
      read_parameters(wv, w, q, D, 1.f);
      read_parameters(bv, b, q, D, 0.f);
      P o;
#pragma unroll
      for (int i = 0; i < n; ++i) o[i] = (T)fmaf((tt::widen(v[u][i]) - m) * r, wv[i], bv[i]);
      write_columns(y + row * (size_t)D, q, D, o);
    }
    if (mean && lane == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

// parts: [blocks][2][D], a block's sums for dw and db, or NULL when neither is wanted.
template <typename T, int G, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK) void ln_bwd(const T* __restrict__ x, const T* __restrict__ dy,
                                                const float* __restrict__ w, const float* __restrict__ mean,
                                                const float* __restrict__ rstd, T* __restrict__ dx,
                                                float* __restrict__ parts, int R, int D) {
  constexpr int n = Loose<T>::n, kRows = BLOCK / G, kParts = G > kWave ? G / kWave : 1;
  typedef typename Loose<T>::type P;
  __shared__ float part[2][kParts];
  const int lane = threadIdx.x % G, sub = threadIdx.x / G, packs = (D + n - 1) / n;
  float dw[NV][n], db[NV][n];
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int i = 0; i < n; ++i) dw[u][i] = db[u][i] = 0.f;
  for (long long row = (long long)blockIdx.x * kRows + sub; row < R; row += (long long)gridDim.x * kRows) {
    const size_t base = row * (size_t)D;
    P xv[NV], gv[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int q = lane + u * G;
      xv[u] = q < packs ? read_columns(x + base, q, D) : P((T)0.f);
      gv[u] = q < packs ? read_columns(dy + base, q, D) : P((T)0.f);
    }
    const float m = mean[row], r = rstd[row];
    float sh = 0.f, shn = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int q = lane + u * G;
      if (q >= packs) break;
      float wv[n];
      read_parameters(wv, w, q, D, 1.f);
#pragma unroll
      for (int i = 0; i < n; ++i) {       // (behind the last column dy is 0 and adds nothing)
        const float g = tt::widen(gv[u][i]), nn = (tt::widen(xv[u][i]) - m) * r, h = g * wv[i];
        sh += h;
        shn = fmaf(h, nn, shn);
        dw[u][i] = fmaf(g, nn, dw[u][i]);
        db[u][i] += g;
      }
    }
    if (!dx) continue;
    const float mh = group_sum<G>(sh, part[0]) / (float)D, mhn = group_sum<G>(shn, part[1]) / (float)D;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int q = lane + u * G;
      if (q >= packs) break;
      float wv[n];
      read_parameters(wv, w, q, D, 1.f);
      P o;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float nn = (tt::widen(xv[u][i]) - m) * r;
        o[i] = (T)(r * (tt::widen(gv[u][i]) * wv[i] - mh - nn * mhn));
      }
      write_columns(dx + base, q, D, o);
    }
  }
  if (!parts) return;
  // this block's rows: one sum of dw and db for each column, pack by pack
  __shared__ float sums[kRows > 1 ? BLOCK * n : 1];
  float* __restrict__ out = parts + (size_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (kRows == 1) {
        const int q = lane + u * G;
#pragma unroll
        for (int i = 0; i < n; ++i)
          if (q * n + i < D) out[which * D + q * n + i] = which ? db[u][i] : dw[u][i];
      } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < n; ++i) sums[threadIdx.x * n + i] = which ? db[u][i] : dw[u][i];
        __syncthreads();
        for (int c = threadIdx.x; c < G * n; c += BLOCK) {
          float s = 0.f;
          for (int k = 0; k < kRows; ++k) s += sums[k * G * n + c];
          if (u * G * n + c < D) out[which * D + u * G * n + c] = s;
        }
      }
    }
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
      const typename Loose<T>::type xv = read_columns(x + base, q, D), gv = read_columns(dy + base, q, D);
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

template <typename T, int G, int NV, int BLOCK>
int launch_fwd(const T* x, const float* w, const float* b, T* y, float* mean, float* rstd, float eps, int R, int D) {
  ln_fwd<T, G, NV, BLOCK><<<grid_for(R, BLOCK / G, 1 << 22), BLOCK, 0, tt::stream()>>>(x, w, b, y, mean, rstd, R, D, eps);
  TT_LAUNCH_CHECK();
  return 0;
}

template <typename T>
int forward(const T* x, const float* w, const float* b, T* y, float* mean, float* rstd, float eps, int R, int D) {
  const int packs = (D + Loose<T>::n - 1) / Loose<T>::n;
  if (packs <= 16) return launch_fwd<T, 16, 1, 256>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 32) return launch_fwd<T, 32, 1, 256>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 64) return launch_fwd<T, 64, 1, 256>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 128) return launch_fwd<T, 64, 2, 256>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 256) return launch_fwd<T, 64, 4, 256>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 512) return launch_fwd<T, 256, 2, 256>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 1024) return launch_fwd<T, 256, 4, 256>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 2048) return launch_fwd<T, 1024, 2, 1024>(x, w, b, y, mean, rstd, eps, R, D);
  if (packs <= 4096) return launch_fwd<T, 1024, 4, 1024>(x, w, b, y, mean, rstd, eps, R, D);
  ln_fwd_long<T><<<grid_for(R, 1, 1 << 20), kLong, 0, tt::stream()>>>(x, w, b, y, mean, rstd, R, D, eps);
  TT_LAUNCH_CHECK();
  return 0;
}

template <typename T, int G, int NV, int BLOCK>
int launch_bwd(const T* x, const T* dy, const float* w, const float* mean, const float* rstd, T* dx, float* dw,
               float* db, int R, int D) {
  hipStream_t st = tt::stream();
  const unsigned grid = grid_for(R, BLOCK / G, tt::compute_units() * (1024 / BLOCK));
  void* ws = nullptr;
  if (dw || db)
    if (tt::workspace((size_t)grid * 2 * D * sizeof(float), &ws)) return -1;
  ln_bwd<T, G, NV, BLOCK><<<grid, BLOCK, 0, st>>>(x, dy, w, mean, rstd, dx, (float*)ws, R, D);
  TT_LAUNCH_CHECK();
  if (dw || db) {
    ln_join<<<(2 * D + kWave - 1) / kWave, 1024, 0, st>>>((const float*)ws, dw, db, D, grid);
    TT_LAUNCH_CHECK();
  }
  return 0;
}

template <typename T>
int backward(const T* x, const T* dy, const float* w, const float* mean, const float* rstd, T* dx, float* dw, float* db,
             int R, int D) {
  constexpr bool wide = sizeof(T) == 4;
  const int packs = (D + Loose<T>::n - 1) / Loose<T>::n;
  if (packs <= 16) return launch_bwd<T, 16, 1, 512>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if (packs <= 32) return launch_bwd<T, 32, 1, 512>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if (packs <= 64) return launch_bwd<T, 64, 1, 512>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if (packs <= 128) return launch_bwd<T, 64, 2, 512>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if (packs <= 256) return launch_bwd<T, 64, 4, 512>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if (packs <= 512) return launch_bwd<T, 512, 1, 512>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if (packs <= 1024) return launch_bwd<T, 512, 2, 512>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if (packs <= 2048) return launch_bwd<T, 1024, 2, 1024>(x, dy, w, mean, rstd, dx, dw, db, R, D);
  if constexpr (wide)
    if (packs <= 4096) return launch_bwd<T, 1024, 4, 1024>(x, dy, w, mean, rstd, dx, dw, db, R, D);
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
    ln_join<<<(2 * (unsigned)D + kWave - 1) / kWave, 1024, 0, st>>>((const float*)ws, dw, db, D, splits);
    TT_LAUNCH_CHECK();
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
