// Layer normalisation of rows: y = (x - mean) / sqrt(var + eps) * w + b, its gradient dx and the reductions over the
// rows that give dw and db.  x, y, dy and dx are float32 or float16, everything else float32.
//
//   n = (x - mean) rstd,  h = dy w,  dx = rstd (h - mean(h) - n mean(h n)),  dw = sum_rows dy n,  db = sum_rows dy
#include "rows.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / tt::kWave;

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_fwd(const T* __restrict__ x, const float* __restrict__ w,
                                                   const float* __restrict__ b, T* __restrict__ y,
                                                   float* __restrict__ mean, float* __restrict__ rstd, int R, int D,
                                                   float eps) {
  __shared__ float part[kWaves];
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const size_t base = row * (size_t)D;
    float s = 0.f;
    for (int i = threadIdx.x; i < D; i += kThreads) s += tt::widen(x[base + i]);
    const float m = tt::block_sum<kWaves>(s, part) / (float)D;
    float q = 0.f;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float c = tt::widen(x[base + i]) - m;
      q = fmaf(c, c, q);
    }
    const float r = 1.f / sqrtf(tt::block_sum<kWaves>(q, part) / (float)D + eps);
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float n = (tt::widen(x[base + i]) - m) * r;
      y[base + i] = (T)fmaf(n, w ? w[i] : 1.f, b ? b[i] : 0.f);
    }
    if (mean && threadIdx.x == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ln_bwd_dx(const T* __restrict__ x, const T* __restrict__ dy,
                                                      const float* __restrict__ w, const float* __restrict__ mean,
                                                      const float* __restrict__ rstd, T* __restrict__ dx, int R, int D) {
  __shared__ float part[kWaves];
  for (int row = blockIdx.x; row < R; row += gridDim.x) {
    const size_t base = row * (size_t)D;
    const float m = mean[row], r = rstd[row];
    float sh = 0.f, shn = 0.f;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float n = (tt::widen(x[base + i]) - m) * r, h = tt::widen(dy[base + i]) * (w ? w[i] : 1.f);
      sh += h;
      shn = fmaf(h, n, shn);
    }
    const float mh = tt::block_sum<kWaves>(sh, part) / (float)D, mhn = tt::block_sum<kWaves>(shn, part) / (float)D;
    for (int i = threadIdx.x; i < D; i += kThreads) {
      const float n = (tt::widen(x[base + i]) - m) * r, h = tt::widen(dy[base + i]) * (w ? w[i] : 1.f);
      dx[base + i] = (T)(r * (h - mh - n * mhn));
    }
  }
}

// A thread sums its column over the rows of its split: part[split][0 | 1][column].
template <typename T>
__global__ __launch_bounds__(kThreads) void ln_bwd_params(const T* __restrict__ x, const T* __restrict__ dy,
                                                          const float* __restrict__ mean,
                                                          const float* __restrict__ rstd, float* __restrict__ part,
                                                          int R, int D, int rows_per_split) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= D) return;
  const int r0 = blockIdx.y * rows_per_split;
  const int r1 = R - r0 < rows_per_split ? R : r0 + rows_per_split;
  float sw = 0.f, sb = 0.f;
  for (int r = r0; r < r1; ++r) {
    const size_t at = (size_t)r * D + c;
    const float g = tt::widen(dy[at]);
    sw = fmaf(g, (tt::widen(x[at]) - mean[r]) * rstd[r], sw);
    sb += g;
  }
  float* __restrict__ p = part + (size_t)blockIdx.y * 2 * D;
  p[c] = sw;
  p[D + c] = sb;
}

// dw and db from the splits' sums, in the order of the splits.
__global__ __launch_bounds__(kThreads) void ln_bwd_join(const float* __restrict__ part, float* __restrict__ dw,
                                                        float* __restrict__ db, int D, int splits) {
  const int c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= 2 * D) return;
  double s = 0.0;
  for (int i = 0; i < splits; ++i) s += (double)part[(size_t)i * 2 * D + c];
  float* __restrict__ out = c < D ? dw : db;
  if (out) out[c < D ? c : c - D] = (float)s;
}

unsigned blocks_for(long long rows) { return (unsigned)(rows < (1 << 20) ? rows : (1 << 20)); }

int check(const char* fn, int dtype, long long R, int D) {
  TT_REQUIRE(dtype == TT_F32 || dtype == TT_F16, "%s: unknown type %d", fn, dtype);
  TT_REQUIRE(R > 0 && R <= (1 << 30), "%s: rows must be in 1..2^30 (got %lld)", fn, R);
  TT_REQUIRE(D > 0 && D <= (1 << 30), "%s: columns must be in 1..2^30 (got %d)", fn, D);
  return 0;
}

template <typename T>
int backward(const T* x, const T* dy, const float* w, const float* mean, const float* rstd, T* dx, float* dw, float* db,
             int R, int D) {
  hipStream_t st = tt::stream();
  if (dx) {
    ln_bwd_dx<T><<<blocks_for(R), kThreads, 0, st>>>(x, dy, w, mean, rstd, dx, R, D);
    TT_LAUNCH_CHECK();
  }
  if (dw || db) {
    const int columns = (D + kThreads - 1) / kThreads;
    int splits = (4 * tt::compute_units() + columns - 1) / columns;
    if (splits > R) splits = R;
    const int per = (R + splits - 1) / splits;
    splits = (R + per - 1) / per;
    void* ws;
    if (tt::workspace((size_t)splits * 2 * D * sizeof(float), &ws)) return -1;
    ln_bwd_params<T><<<dim3(columns, splits), kThreads, 0, st>>>(x, dy, mean, rstd, (float*)ws, R, D, per);
    TT_LAUNCH_CHECK();
    ln_bwd_join<<<(2 * D + kThreads - 1) / kThreads, kThreads, 0, st>>>((const float*)ws, dw, db, D, splits);
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
  if (dtype == TT_F32)
    ln_fwd<float><<<blocks_for(R), kThreads, 0, tt::stream()>>>((const float*)x, w, b, (float*)y, mean, rstd, (int)R,
                                                              D, (float)eps);
  else
    ln_fwd<_Float16><<<blocks_for(R), kThreads, 0, tt::stream()>>>((const _Float16*)x, w, b, (_Float16*)y, mean, rstd,
                                                                 (int)R, D, (float)eps);
  TT_LAUNCH_CHECK();
  return 0;
}

int tt_layer_norm_bwd(const void* x, const void* dy, const float* w, const float* mean, const float* rstd, void* dx,
                      float* dw, float* db, int dtype, long long R, int D) {
  TT_REQUIRE_INIT();
  TT_REQUIRE(x && dy && mean && rstd, "tt_layer_norm_bwd: null pointer");
  if (int rc = check("tt_layer_norm_bwd", dtype, R, D)) return rc;
  TT_REQUIRE_ALIGNED("tt_layer_norm_bwd", x, dy, w, dx, dw, db);
  if (dtype == TT_F32)
    return backward<float>((const float*)x, (const float*)dy, w, mean, rstd, (float*)dx, dw, db, (int)R, D);
  return backward<_Float16>((const _Float16*)x, (const _Float16*)dy, w, mean, rstd, (_Float16*)dx, dw, db, (int)R, D);
}

}  // extern "C"
