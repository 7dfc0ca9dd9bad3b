// Softmax cross entropy over a vocabulary, from features and the head's weight, without keeping the logits:
//
//   z = x W^T     M_i = max_v z_iv     S_i = sum_v e^(z_iv - M_i)     loss_i = ln S_i + M_i - z_i,t(i)
//   G_iv = g_i (e^(z_iv - M_i) / S_i - [v = t(i)])        dX = G W        dW = G^T x
//
// Rows are worked on in chunks.  The first product leaves a chunk's logits in scratch memory (none without gradients)
// and, with the tile still in registers, every row's maximum and sum over 64 columns; these are joined, and one pass turns the logits
// into G where they stand.  The two other products read it there: G^T needs no copy, see product.h.  So a training step
// has three products and not a fourth for logits that it forgot, and the scratch memory is bounded whatever the batch.
//
// float16: the tensors are the products' operands as they are; G is rounded to float16 once, scaled by 2^14.
// float32: operands have two float16 terms.  Row i of x and row v of W are scaled by powers of two 2^-f_i and 2^-e_v to below
// 2^15; G, which meets W's rows and x's rows as k, carries 2^(e_v + f_i), and all of it a common 2^c that brings the largest
// to 2^15: G's entries are held to 2^-22 of themselves, and to 2^-40 of the largest.
#include "product.h"
#include "rows.h"

#include <algorithm>

namespace {

using namespace tt;

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr size_t kMostLogits = (size_t)2 << 30;     // bytes of a chunk's logits
constexpr size_t kMostStats = (size_t)256 << 20;
constexpr int kTop = 14;                            // scaled values are below 2^(kTop + 1)
constexpr int kLowest = -1000;                      // an exponent below all
constexpr int kAny = -2000;                         // that of a row of zeros: whatever suits the others

// Set at the start of a call, read by all that follows.
struct Control {
  float scale;          // of the loss and its gradients: 1 / positions for 'mean'
  int most_e, most_f;   // the largest exponents of W's rows, and of x's rows with their g
  __device__ __forceinline__ int top_e() const { return most_e == kLowest ? 0 : most_e; }
  __device__ __forceinline__ int top_f() const { return most_f == kLowest ? 0 : most_f; }
};

struct Targets {
  const void* at;
  int wide, V;
  long long ignore;
};
constexpr int kIgnored = -1, kInvalid = -2;
__device__ __forceinline__ int class_of(const Targets& t, long long i) {
  const long long v = read_index(t.at, (size_t)i, t.wide);
  if (v == t.ignore) return kIgnored;
  const long long c = v < 0 ? v + t.V : v;
  return c < 0 || c >= t.V ? kInvalid : (int)c;
}

// exponent e with |v| < 2^e; 0 and what is not finite: 0
__device__ __forceinline__ int exponent(float v) {
  int e = 0;
  if (v != 0.f && __builtin_isfinite(v)) (void)frexpf(v, &e);
  return e;
}

__global__ __launch_bounds__(1024) void lce_begin(Targets t, long long rows, int mean, int lowest_e, int lowest_f, Control* c) {
  __shared__ long long part[16];
  long long n = 0;
  for (long long i = threadIdx.x; i < rows; i += 1024) n += read_index(t.at, (size_t)i, t.wide) != t.ignore;
  n = row_sum<1024>(n, part);
  if (threadIdx.x == 0) {
    c->scale = !mean ? 1.f : n ? 1.f / (float)n : 0.f;
    c->most_e = lowest_e;
    c->most_f = lowest_f;
  }
}

// Rows of x or W as the products' operands: two terms of float32, or a copy of float16.  Rows without a target are
// zeros, whatever they hold.  A wave has a row.
template <typename T>
__global__ __launch_bounds__(256) void lce_rows(const T* __restrict__ from, char* __restrict__ to, int* __restrict__ exponents,
                                                const float* __restrict__ g, long long rows, int columns, int ld, Targets t,
                                                int* most) {
  const long long row = (long long)blockIdx.x * 4 + row_of_block<kWave>();
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  const T* x = from + (size_t)row * columns;
  char* y = to + (size_t)row * ld;
  const bool kept = !t.at || class_of(t, row) != kIgnored;
  int e = 0;
  bool counts = kept;       // among the largest exponents
  if (sizeof(T) == 4) {
    float m = 0.f;
    if (kept)
      for (int c = lane; c < columns; c += 64) m = fmaxf(m, fabsf(widen(x[c])));
    m = lanes_reduce<64>(m, Larger());
    counts = m > 0.f && __builtin_isfinite(m);
    e = counts ? exponent(m) - kTop - 1 : 0;
    for (int c = lane; c < (columns + 63) / 64 * 64; c += 64) {
      _Float16 hi, lo;
      split(kept && c < columns ? ldexpf(widen(x[c]), -e) : 0.f, &hi, &lo);
      char* p = y + at_column(c);
      *reinterpret_cast<_Float16*>(p) = hi;
      *reinterpret_cast<_Float16*>(p + kTermBytes) = lo;
    }
    if (lane == 0) exponents[row] = counts ? e : kAny;
  } else {
    for (int c = lane; c < (columns + 63) / 64 * 64; c += 64)
      *reinterpret_cast<_Float16*>(y + c * 2) = kept && c < columns ? (_Float16)x[c] : (_Float16)0.f;
  }
  if (most && lane == 0 && counts) {
    if (!g) atomicMax(most, e);
    else if (g[row] != 0.f) atomicMax(most, e + exponent(g[row]));
  }
}

struct LogitsEpilogue {
  const int* f;         // exponents of x's rows and W's, of float32
  const int* e;
  Targets t;
  long long first;      // row of the chunk's first
  float* z;             // [rows][ld] or none
  long long ld;
  float2* stats;        // [rows][blocks of 64 columns]
  float* own;           // [rows] the target's logit
  int blocks;

  template <int TERMS, typename G>
  __device__ __forceinline__ void apply(G& p, int m0, int n0, int rows, int V) const {
    constexpr int MT = sizeof(p.acc) / sizeof(p.acc[0]);
    const int c0 = n0 + G::column(), lane = threadIdx.x & 63;
    int scale[16];
    if (TERMS == 2) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int c = c0 + (j >> 2) * 16 + (j & 3);
        scale[j] = c < V ? e[c] : 0;
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = m0 + G::row() + 16 * i;
      const bool in = r < rows;
      const int fi = TERMS == 2 && in ? f[r] : 0, target = in ? class_of(t, first + r) : kIgnored;
      float v[16], most = -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int c = c0 + (j >> 2) * 16 + (j & 3);
        v[j] = p.acc[i][j >> 2][j & 3];
        if (TERMS == 2) v[j] = ldexpf(v[j], scale[j] + fi);
        if (c == target) own[r] = v[j];
        if (c < V) most = fmaxf(most, v[j]);
      }
      if (z && in) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c0 + 16 * j < ld) *reinterpret_cast<floatx4*>(z + (size_t)r * ld + c0 + 16 * j) = floatx4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
      }
      most = fmaxf(most, __shfl_xor(most, 16, kWave));
      most = fmaxf(most, __shfl_xor(most, 32, kWave));
      const float from = most == -INFINITY ? 0.f : most;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c0 + (j >> 2) * 16 + (j & 3) < V) sum += __builtin_amdgcn_exp2f((v[j] - from) * kLog2e);
      sum += __shfl_xor(sum, 16, kWave);
      sum += __shfl_xor(sum, 32, kWave);
      const int block = (c0 - (lane >> 4) * 4) >> 6;
      if (in && lane < 16 && block < blocks) stats[(size_t)r * blocks + block] = make_float2(most, sum);
    }
  }
};

template <int TERMS, int SIZE>
__global__ __launch_bounds__((Sized<TERMS, false, false, SIZE>::kThreads)) void lce_logits(Operand x, Operand w, int rows, int V,
                                                                                          int stages, LogitsEpilogue epilogue) {
  typedef Sized<TERMS, false, false, SIZE> G;
  extern __shared__ __align__(16) char lds[];
  int m, n;
  tile_of(blockIdx.x, gridDim.x, (rows + G::kM - 1) / G::kM, (V + G::kN - 1) / G::kN, &m, &n);
  G p;
  p.run(x, w, m * G::kM, n * G::kN, 0, stages, lds);
  epilogue.template apply<TERMS>(p, m * G::kM, n * G::kN, rows, V);
}

// A row's maximum and log2 of its sum from those of its blocks, and its loss.  A wave has a row.
__global__ __launch_bounds__(256) void lce_join(const float2* __restrict__ stats, const float* __restrict__ own, float2* __restrict__ of,
                                                float* __restrict__ loss, Targets t, long long first, int rows, int blocks) {
  const int r = blockIdx.x * 4 + row_of_block<kWave>();
  if (r >= rows) return;
  const int lane = threadIdx.x & 63, target = class_of(t, first + r);
  if (target == kIgnored) {
    if (lane == 0) loss[r] = 0.f;
    return;
  }
  const float2* s = stats + (size_t)r * blocks;
  float most = -INFINITY;
  for (int b = lane; b < blocks; b += 64) most = fmaxf(most, s[b].x);
  most = lanes_reduce<64>(most, Larger());
  const float from = most == -INFINITY ? 0.f : most;
  float sum = 0.f;
  for (int b = lane; b < blocks; b += 64) {
    const float2 v = s[b];
    sum += v.y * __builtin_amdgcn_exp2f(((v.x == -INFINITY ? from : v.x) - from) * kLog2e);
  }
  sum = lanes_reduce<64>(sum, Plus());
  if (lane == 0) {
    const float log_sum = log2f(sum);
    of[r] = make_float2(from, log_sum);
    loss[r] = target == kInvalid ? NAN : log_sum * kLn2 + (from - own[r]);
  }
}

// With the exponent of a row of zeros, it is the largest that leaves the row's G (times its g) in range.
__device__ __forceinline__ int exponent_of_row(int e, int top, float g) { return e == kAny ? top - exponent(g) + 1 : e; }

// The logits of a chunk become G, where they stand: 64 floats are the 64 first and 64 second terms.
template <int TERMS>
__global__ __launch_bounds__(256) void lce_gradient(float* __restrict__ z, long long ld, const float2* __restrict__ of,
                                                    const float* __restrict__ loss, const float* __restrict__ g,
                                                    const int* __restrict__ f, const int* __restrict__ e, Targets t,
                                                    long long first, int V, const Control* __restrict__ control) {
  const int r = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= ld) return;
  float* at = z + (size_t)r * ld;
  const int target = class_of(t, first + r);
  floatx4 v = {};
  if (target != kIgnored) {
    v = *reinterpret_cast<const floatx4*>(at + c);
    const float2 s = of[r];
    const float weight = g ? g[first + r] : 1.f, mine = loss[r];
    const int top_e = control->top_e();
    const int shift = kTop - top_e - control->top_f() + (TERMS == 2 ? exponent_of_row(f[r], control->top_f(), weight) : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int column = c + i;
      float p = __builtin_amdgcn_exp2f((v[i] - s.x) * kLog2e - s.y);
      if (column == target) p = expm1f(-mine);
      if (target == kInvalid) p = NAN;
      if (TERMS == 2 && column < V) p = ldexpf(p * weight, shift + exponent_of_row(e[column], top_e, 1.f));
      else p = ldexpf(p * weight, shift);
      v[i] = column < V ? p : 0.f;
    }
  }
  char* row = reinterpret_cast<char*>(at);
  if (TERMS == 2) {
    store_terms(row, c, v);
  } else {
    *reinterpret_cast<half4*>(row + at_column(c)) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  }
}

// What the two gradients' products do with their sums: take the scales back, and store them as float32 (to or on top of what is there)
// or float16; or leave partial sums for lce_sum.
struct GradientOut {
  void* to;
  const int* exponents;     // of the rows, of float32
  int top_f;                // they are x's, not W's
  const float* g;           // of the rows, if they are x's
  const Control* control;
  int half, add;
  int columns;
  __device__ __forceinline__ void store(int row, int c, floatx4 v) const {
    const float s = control->scale;
    const int top = top_f ? control->top_f() : control->top_e();
    const int e = control->top_e() + control->top_f() - kTop - (exponents ? exponent_of_row(exponents[row], top, g ? g[row] : 1.f) : 0);
    const size_t at = (size_t)row * columns + c;
    const int n = columns - c;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ldexpf(v[i] * s, e);
    if (half) {
      _Float16* p = reinterpret_cast<_Float16*>(to) + at;
      if (n >= 4 && (at & 3) == 0) {
        *reinterpret_cast<half4*>(p) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
      } else {
        for (int i = 0; i < 4 && i < n; ++i) p[i] = (_Float16)v[i];
      }
    } else {
      float* p = reinterpret_cast<float*>(to) + at;
      if (n >= 4 && (at & 3) == 0) {
        floatx4* q = reinterpret_cast<floatx4*>(p);
        *q = add ? *q + v : v;
      } else {
        for (int i = 0; i < 4 && i < n; ++i) p[i] = add ? p[i] + v[i] : v[i];
      }
    }
  }
};

template <int TERMS, bool A_ACROSS, int SIZE>
__global__ __launch_bounds__((Sized<TERMS, A_ACROSS, true, SIZE>::kThreads)) void lce_product(Operand a, Operand b, int M, int N, int stages,
                                                                                            int per, int splits, float* partial, GradientOut out) {
  typedef Sized<TERMS, A_ACROSS, true, SIZE> G;
  extern __shared__ __align__(16) char lds[];
  const int blocks = gridDim.x / splits, split = blockIdx.x / blocks;
  int m, n;
  tile_of(blockIdx.x % blocks, blocks, (M + G::kM - 1) / G::kM, (N + G::kN - 1) / G::kN, &m, &n);
  const int first = split * per, count = min(per, stages - first);
  G p;
  p.run(a, b, m * G::kM, n * G::kN, first, count, lds);
  constexpr int MT = sizeof(p.acc) / sizeof(p.acc[0]), NT = sizeof(p.acc[0]) / sizeof(p.acc[0][0]);
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = m * G::kM + G::row() + 16 * i;
    if (row >= M) continue;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int c = n * G::kN + G::column() + 16 * j;
      if (c >= N) continue;
      if (splits > 1) {
        const long long ld = (N + 3) / 4 * 4;
        *reinterpret_cast<floatx4*>(partial + ((size_t)split * M + row) * ld + c) = p.acc[i][j];
      } else {
        out.store(row, c, p.acc[i][j]);
      }
    }
  }
}

__global__ __launch_bounds__(256) void lce_sum(const float* __restrict__ partial, int splits, int M, int N, GradientOut out) {
  const int quads = (N + 3) / 4;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= (long long)M * quads) return;
  floatx4 v = {};
  for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const floatx4*>(partial + ((size_t)s * M * quads + at) * 4);
  out.store((int)(at / quads), (int)(at % quads) * 4, v);
}

__global__ __launch_bounds__(1024) void lce_loss(const float* __restrict__ loss, long long rows, int mean, Targets t, const Control* control,
                                                 float* __restrict__ out) {
  __shared__ double part[16];
  double s = 0.0;
  for (long long i = threadIdx.x; i < rows; i += 1024) s += (double)loss[i];
  s = row_sum<1024>(s, part);
  if (threadIdx.x == 0) *out = mean && control->scale == 0.f ? NAN : (float)(s * (double)control->scale);
}

// g (none: 1) times a float32 gradient, as float32 or float16.
template <typename T>
__global__ __launch_bounds__(256) void lce_scale(const float* __restrict__ from, const float* __restrict__ g, T* __restrict__ to, size_t n) {
  const float s = g ? *g : 1.f;
  const size_t packs = n / 4, step = (size_t)gridDim.x * 256;
  size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  for (size_t p = i; p < packs; p += step) {
    const floatx4 v = reinterpret_cast<const floatx4*>(from)[p] * s;
    typedef T Four __attribute__((ext_vector_type(4)));
    reinterpret_cast<Four*>(to)[p] = Four{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
  }
  if (i < n % 4) to[packs * 4 + i] = (T)(from[packs * 4 + i] * s);
}

template <typename T>
int launch_scale(const float* from, const float* g, T* to, size_t n) {
  const size_t blocks = std::min((n / 4 + 255) / 256 + 1, (size_t)compute_units() * 16);
  lce_scale<T><<<(unsigned)blocks, 256, 0, stream()>>>(from, g, to, n);
  TT_LAUNCH_CHECK();
  return 0;
}

template <int TERMS, int SIZE>
int launch_logits(const Operand& x, const Operand& w, int rows, int V, int H, const LogitsEpilogue& epilogue) {
  typedef Sized<TERMS, false, false, SIZE> G;
  TT_ALLOW_LDS((lce_logits<TERMS, SIZE>), G::kLds);
  lce_logits<TERMS, SIZE><<<(unsigned)tiles_of(rows, V, SIZE), G::kThreads, G::kLds, stream()>>>(
      x, w, rows, V, (int)(padded(H) / G::kDepth), epilogue);
  TT_LAUNCH_CHECK();
  return 0;
}
template <int TERMS>
int launch_logits(const Operand& x, const Operand& w, int rows, int V, int H, const LogitsEpilogue& epilogue) {
  switch (tile_size(rows, V)) {
    case 2: return launch_logits<TERMS, 2>(x, w, rows, V, H, epilogue);
    case 1: return launch_logits<TERMS, 1>(x, w, rows, V, H, epilogue);
    default: return launch_logits<TERMS, 0>(x, w, rows, V, H, epilogue);
  }
}

// How a gradient's product [m, n] over `stages` is cut: the size of its tiles, and how many blocks share one.
struct Plan {
  int size, per, splits;      // stages for each block, blocks
};
Plan plan_product(long long m, long long n, long long stages) {
  Plan p;
  p.size = tile_size(m, n);
  // few tiles and a long reduction: large tiles shared by several blocks
  while (p.size < 2 && stages >= 64 && tiles_of(m, n, p.size + 1) * (stages / 16) >= compute_units() && m > kTileSide[p.size] && n > kTileSide[p.size]) ++p.size;
  const long long tiles = tiles_of(m, n, p.size);
  long long splits = compute_units() / tiles;
  splits = std::max(1LL, std::min(splits, stages / 8));
  p.per = (int)((stages + splits - 1) / splits);
  p.splits = (int)((stages + p.per - 1) / p.per);
  return p;
}

template <int TERMS, bool A_ACROSS, int SIZE>
int launch_product(const Operand& a, const Operand& b, int M, int N, int stages, int per, float* partial, const GradientOut& out) {
  typedef Sized<TERMS, A_ACROSS, true, SIZE> G;
  TT_ALLOW_LDS((lce_product<TERMS, A_ACROSS, SIZE>), G::kLds);
  const int splits = (stages + per - 1) / per;      // (fewer for a chunk that is not whole)
  lce_product<TERMS, A_ACROSS, SIZE><<<(unsigned)(tiles_of(M, N, SIZE) * splits), G::kThreads, G::kLds, stream()>>>(
      a, b, M, N, stages, per, splits, partial, out);
  TT_LAUNCH_CHECK();
  if (splits > 1) {
    const long long quads = (long long)M * ((N + 3) / 4);
    lce_sum<<<(unsigned)((quads + 255) / 256), 256, 0, stream()>>>(partial, splits, M, N, out);
    TT_LAUNCH_CHECK();
  }
  return 0;
}
template <int TERMS, bool A_ACROSS>
int launch_product(const Plan& plan, const Operand& a, const Operand& b, int M, int N, int stages, float* partial, const GradientOut& out) {
  switch (plan.size) {
    case 2: return launch_product<TERMS, A_ACROSS, 2>(a, b, M, N, stages, plan.per, partial, out);
    case 1: return launch_product<TERMS, A_ACROSS, 1>(a, b, M, N, stages, plan.per, partial, out);
    default: return launch_product<TERMS, A_ACROSS, 0>(a, b, M, N, stages, plan.per, partial, out);
  }
}

// Parts of the workspace, one behind the other.
struct Carve {
  size_t bytes = 0;
  size_t take(size_t n) {
    const size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};

struct Call {
  const void *x, *w;
  Targets t;
  const float* g;
  float* loss;
  void *dx, *dw;
  int half_out, reduction, H;
  long long N;
};

template <typename T, int TERMS>
int run(const Call& q) {
  const int V = q.t.V, H = q.H, mean = q.reduction == 2;
  const long long N = q.N, Hp = padded(H), Vp = padded(V);
  const bool grad = q.dx || q.dw, copy_w = TERMS == 2 || H % 8 != 0;
  const int blocks = (int)(Vp / 64), depth = TERMS == 1 ? 64 : 32;
  long long chunk = (long long)((grad ? kMostLogits : kMostStats) / ((size_t)Vp * (grad ? 4 : 8) / (grad ? 1 : 64)));
  chunk = std::max(256LL, chunk / 256 * 256);
  chunk = std::min(chunk, N);
  const bool several = chunk < N;
  const int stagesV = (int)(Vp / depth), stagesN = (int)((chunk + depth - 1) / depth);
  const Plan plan_x = plan_product(chunk, H, stagesV), plan_w = plan_product(V, H, stagesN);

  Carve c;
  const size_t at_control = c.take(sizeof(Control)), at_f = c.take(TERMS == 2 ? 4 * N : 0), at_e = c.take(TERMS == 2 ? 4 * (size_t)V : 0);
  const size_t at_x = c.take((size_t)N * Hp * 2 * TERMS), at_w = c.take(copy_w ? (size_t)V * Hp * 2 * TERMS : 0);
  const size_t at_stats = c.take((size_t)chunk * blocks * 8), at_own = c.take(4 * chunk), at_of = c.take(8 * chunk);
  const size_t at_loss = c.take(4 * N), at_z = c.take(grad ? (size_t)chunk * Vp * 4 : 0);
  const size_t part_x = q.dx && plan_x.splits > 1 ? (size_t)plan_x.splits * chunk * ((H + 3) / 4) * 16 : 0;
  const size_t part_w = q.dw && plan_w.splits > 1 ? (size_t)plan_w.splits * V * ((H + 3) / 4) * 16 : 0;
  const size_t at_part = c.take(std::max(part_x, part_w));
  const size_t at_sum = c.take(several && q.half_out && q.dw ? (size_t)V * H * 4 : 0);
  void* ws;
  if (tt::workspace(c.bytes, &ws)) return -1;
  char* base = (char*)ws;
  Control* control = (Control*)(base + at_control);
  int *f = TERMS == 2 ? (int*)(base + at_f) : nullptr, *e = TERMS == 2 ? (int*)(base + at_e) : nullptr;
  float *z = grad ? (float*)(base + at_z) : nullptr, *partial = (float*)(base + at_part);
  float* losses = q.reduction == 0 && q.loss ? q.loss : (float*)(base + at_loss);
  float2 *stats = (float2*)(base + at_stats), *of = (float2*)(base + at_of);
  float* own = (float*)(base + at_own);

  lce_begin<<<1, 1024, 0, stream()>>>(q.t, N, mean, TERMS == 2 ? kLowest : 0, TERMS == 2 || q.g ? kLowest : 0, control);
  TT_LAUNCH_CHECK();
  const int ldx = (int)(Hp * 2 * TERMS);
  lce_rows<T><<<(unsigned)((N + 3) / 4), 256, 0, stream()>>>((const T*)q.x, base + at_x, f, q.g, N, H, ldx, q.t,
                                                             TERMS == 2 || q.g ? &control->most_f : nullptr);
  TT_LAUNCH_CHECK();
  Operand w = {(const char*)q.w, (long long)V * H * 2, H * 2, kTermBytes};
  if (copy_w) {
    lce_rows<T><<<(unsigned)((V + 3) / 4), 256, 0, stream()>>>((const T*)q.w, base + at_w, e, nullptr, V, H, ldx, Targets{nullptr, 0, 0, 0},
                                                               TERMS == 2 ? &control->most_e : nullptr);
    TT_LAUNCH_CHECK();
    w = Operand{base + at_w, (long long)V * ldx, ldx, kTermBytes * TERMS};
  }
  for (long long first = 0; first < N; first += chunk) {
    const int rows = (int)std::min(chunk, N - first);
    const Operand x = {base + at_x + (size_t)first * ldx, (long long)rows * ldx, ldx, kTermBytes * TERMS};
    const LogitsEpilogue epilogue = {f ? f + first : nullptr, e, q.t, first, z, Vp, stats, own, blocks};
    if (launch_logits<TERMS>(x, w, rows, V, H, epilogue)) return -1;
    lce_join<<<(unsigned)((rows + 3) / 4), 256, 0, stream()>>>(stats, own, of, losses + first, q.t, first, rows, blocks);
    TT_LAUNCH_CHECK();
    if (!grad) continue;
    for (int r = 0; r < rows; r += 65535) {
      const int some = std::min(rows - r, 65535);
      lce_gradient<TERMS><<<dim3((unsigned)((Vp / 4 + 255) / 256), some), 256, 0, stream()>>>(
          z + (size_t)r * Vp, Vp, of + r, losses + first + r, q.g, f ? f + first + r : nullptr, e, q.t, first + r, V, control);
      TT_LAUNCH_CHECK();
    }
    const Operand gradient = {(const char*)z, (long long)rows * Vp * 4, (int)(Vp * 4), 2 * kTermBytes};
    if (q.dx) {
      const GradientOut out = {(char*)q.dx + (size_t)first * H * (q.half_out ? 2 : 4), f ? f + first : nullptr, 1, q.g ? q.g + first : nullptr, control,
                               q.half_out, 0, H};
      if (launch_product<TERMS, false>(plan_x, gradient, w, rows, H, stagesV, partial, out)) return -1;
    }
    if (q.dw) {
      const GradientOut out = {several && q.half_out ? (void*)(base + at_sum) : q.dw, e, 0, nullptr, control, several ? 0 : q.half_out, first > 0, H};
      if (launch_product<TERMS, true>(plan_w, gradient, x, V, H, (rows + depth - 1) / depth, partial, out)) return -1;
    }
  }
  if (several && q.half_out && q.dw) {
    if (launch_scale((float*)(base + at_sum), nullptr, (_Float16*)q.dw, (size_t)V * H)) return -1;
  }
  if (q.loss && q.reduction) {
    lce_loss<<<1, 1024, 0, stream()>>>(losses, N, mean, q.t, control, q.loss);
    TT_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace

extern "C" {

int tt_linear_cross_entropy(const void* x, const void* w, const void* target, const float* g, float* loss, void* dx, void* dw,
                            int kind, int half_gradients, int index_bits, long long ignore_index, int reduction, long long N,
                            int H, int V) {
  TT_REQUIRE_INIT();
  const char* fn = "linear_cross_entropy";
  TT_REQUIRE(kind == 0 || kind == 1, "%s: unknown type %d", fn, kind);
  TT_REQUIRE(index_bits == 64 || index_bits == 32, "%s: targets are of 64 or 32 bits, got %d", fn, index_bits);
  TT_REQUIRE(reduction >= 0 && reduction <= 2, "%s: unknown reduction %d", fn, reduction);
  TT_REQUIRE(N >= 1 && N <= (1LL << 30), "%s: 1 to 2^30 positions, got %lld", fn, N);
  TT_REQUIRE(H >= 1 && H <= 1 << 20, "%s: 1 to 2^20 features, got %d", fn, H);
  TT_REQUIRE(V >= 1 && V <= 1 << 20, "%s: 1 to 2^20 classes, got %d", fn, V);
  TT_REQUIRE(x && w && target && (loss || dx || dw), "%s: null pointer", fn);
  TT_REQUIRE(!half_gradients || kind == 1, "%s: gradients of float32 tensors are float32", fn);
  TT_REQUIRE_ALIGNED(fn, x, w, g, loss, dx, dw);
  const Call q = {x, w, {target, index_bits == 64, V, ignore_index}, g, loss, dx, dw, half_gradients, reduction, H, N};
  return kind ? run<_Float16, 1>(q) : run<float, 2>(q);
}

int tt_scaled_gradient(const float* from, const float* g, void* to, int kind, size_t n) {
  TT_REQUIRE_INIT();
  TT_REQUIRE(kind == 0 || kind == 1, "scaled_gradient: unknown type %d", kind);
  TT_REQUIRE(from && g && to, "scaled_gradient: null pointer");
  TT_REQUIRE_ALIGNED("scaled_gradient", from, to);
  return kind ? launch_scale(from, g, (_Float16*)to, n) : launch_scale(from, g, (float*)to, n);
}

}  // extern "C"
