// Orthogonalised updates: Newton-Schulz products of a matrix [rows, columns], alone or inside the optimiser's step.
//
//   X <- X / max(|X|_F, eps)         steps times:  A = X X^T,  X <- a X + (b A + c A A) X
//
// takes every singular value s of X to a s + b s^3 + c s^5, and in a few steps all of them to about 1.  A is taken over the
// shorter side: X^T X, and X on the left of the sum, where there are more rows than columns, so that nothing is transposed (product.h
// reads either operand along or across its rows).
//
// All products are of two float16 terms an operand, X and A scaled by 2^14 and b A + c A A by 2^12: with singular values
// below 3.9 no entry leaves float16's range, and one is held to 2^-22 of itself or 2^-39 of the unit.
// The matrices of a step share the launches, 3 a Newton-Schulz step and two in front: a network has tens of them, most too
// small to fill the device.
#include "product.h"
#include "rows.h"

#include <algorithm>
#include <vector>

namespace {

using namespace tt;

constexpr int kMost = 24;                   // matrices of a launch
constexpr size_t kMostScratch = (size_t)4 << 30;
constexpr float kUp = 16384.f;              // the scale of X and A
constexpr int kParts = 256;                 // partial sums of a matrix's squares, at most

struct Matrix {
  const void* from;         // the gradient, or the matrix itself (float32 or float16)
  float* momentum;          // or none
  void* to;                 // the parameter, or the result
  char* scratch;
  double* parts;
  float rate;               // of a parameter: learning rate times the matrix's own scale
  int rows, columns;
};

// X twice, A, b A + c A A: rows of blocks of two terms.
struct Place {
  long long ldx, lda, x, a;         // bytes of a row of X and A, bytes of X and A
  int m;
  bool tall;
  __host__ __device__ Place(int rows, int columns) {
    tall = rows > columns;
    m = tall ? columns : rows;
    ldx = padded(columns) * 4;
    lda = padded(m) * 4;
    x = ldx * rows;
    a = lda * m;
  }
  __host__ __device__ long long bytes() const { return 2 * x + 2 * a; }
};

struct Batch {
  Matrix of[kMost];
  unsigned first[kMost + 1];        // blocks in front of each
  int count;
};
__device__ __forceinline__ int matrix_of(const Batch& b) {
  int i = 0;
  while (i + 1 < b.count && blockIdx.x >= b.first[i + 1]) ++i;
  return i;
}

// Partial sums of a matrix of n values.
__host__ __device__ inline int parts_of(size_t n) { return n > (size_t)kParts * 4096 ? kParts : (int)((n + 4095) / 4096); }

struct Rule {
  float a, b, c;
  float eps;
  float mix;                        // 1 - momentum
  float keep;                       // 1 - learning rate times weight decay
  int nesterov, half, step;
};

__device__ __forceinline__ float update_of(const Rule& q, float g, float m) { return q.nesterov ? m - q.mix * (m - g) : m; }

// The momentum, and the squares of the update's values.
__global__ __launch_bounds__(256) void muon_begin(Batch b, Rule q) {
  __shared__ double part[4];
  const int at = matrix_of(b);
  const Matrix& x = b.of[at];
  const unsigned block = blockIdx.x - b.first[at], blocks = b.first[at + 1] - b.first[at];
  const size_t n = (size_t)x.rows * x.columns;
  double s = 0.0;
  for (size_t i = (size_t)block * 256 + threadIdx.x; i < n; i += (size_t)blocks * 256) {
    float u;
    if (x.momentum) {
      const float g = reinterpret_cast<const float*>(x.from)[i], old = x.momentum[i], m = old + q.mix * (g - old);
      x.momentum[i] = m;
      u = update_of(q, g, m);
    } else {
      u = read_value(x.from, i, q.half);
    }
    s += (double)u * (double)u;
  }
  s = row_sum<256>(s, part);
  if (threadIdx.x == 0) x.parts[block] = s;
}

// X as rows of terms, divided by its norm.  Four rows a block.
__global__ __launch_bounds__(256) void muon_scale(Batch b, Rule q) {
  __shared__ double part[4];
  const int at = matrix_of(b);
  const Matrix& x = b.of[at];
  const Place p(x.rows, x.columns);
  const int parts = parts_of((size_t)x.rows * x.columns);
  const double s = row_sum<256>((int)threadIdx.x < parts ? x.parts[threadIdx.x] : 0.0, part);
  const double norm = sqrt(s);
  const float inverse = (float)(1.0 / (norm > (double)q.eps || norm != norm ? norm : (double)q.eps));
  const int row = (int)(blockIdx.x - b.first[at]) * 4 + (int)(threadIdx.x >> 6);
  if (row >= x.rows) return;
  char* to = x.scratch + row * p.ldx;
  for (int c = threadIdx.x & 63; c < (x.columns + 63) / 64 * 64; c += 64) {
    float u = 0.f;
    if (c < x.columns) {
      const size_t i = (size_t)row * x.columns + c;
      u = x.momentum ? update_of(q, reinterpret_cast<const float*>(x.from)[i], x.momentum[i]) : read_value(x.from, i, q.half);
    }
    _Float16 hi, lo;
    split(u * inverse * kUp, &hi, &lo);
    *reinterpret_cast<_Float16*>(to + at_column(c)) = hi;
    *reinterpret_cast<_Float16*>(to + at_column(c) + kTermBytes) = lo;
  }
}

constexpr int kGram = 0, kPolynomial = 1, kUpdate = 2;

// One product of a step for a tile of one matrix.
template <int WHAT, bool ACROSS, int SIZE>
__device__ __forceinline__ void muon_tile(const Matrix& x, const Rule& q, bool last, unsigned block, unsigned blocks, char* lds) {
  constexpr bool kA = WHAT == kGram && ACROSS, kB = WHAT == kGram ? ACROSS : WHAT == kUpdate && ACROSS;
  typedef Sized<2, kA, kB, SIZE> G;
  const Place p(x.rows, x.columns);
  char* x0 = x.scratch + (q.step & 1 ? p.x : 0);
  char* x1 = x.scratch + (q.step & 1 ? 0 : p.x);
  char *a = x.scratch + 2 * p.x, *s = a + p.a;
  const Operand X = {x0, p.x, (int)p.ldx, kLine}, A = {a, p.a, (int)p.lda, kLine}, S = {s, p.a, (int)p.lda, kLine};
  const int M = WHAT == kUpdate ? x.rows : p.m, N = WHAT == kUpdate ? x.columns : p.m;
  int m, n;
  tile_of((int)block, (int)blocks, (M + G::kM - 1) / G::kM, (N + G::kN - 1) / G::kN, &m, &n);
  G g;
  const int m0 = m * G::kM, n0 = n * G::kN, edge = (N + 63) / 64 * 64;
  constexpr int U = G::kAhead;
  const auto each = [&](int r, int c, int edge, auto f) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (m0 + r + u * G::kStep < M && n0 + c < edge) f(u, m0 + r + u * G::kStep, n0 + c);
  };
  if (WHAT == kGram) {
    const int k = ACROSS ? x.rows : x.columns;
    g.run(X, X, m0, n0, 0, (k + 31) / 32, lds);
    g.rows(lds, [](int, int) { return 0; }, [&](int r, int c, const floatx4 (&v)[U], int (&)[U]) {
      each(r, c, edge, [&](int u, int row, int column) { store_terms(a + row * p.lda, column, v[u] * (1.f / kUp)); });
    });
  } else if (WHAT == kPolynomial) {
    g.run(A, A, m0, n0, 0, (p.m + 31) / 32, lds);
    g.rows(lds, [&](int r, int c) { return m0 + r < M && n0 + c < edge ? load_terms(a + (m0 + r) * p.lda, n0 + c) : floatx4{}; },
           [&](int r, int c, const floatx4 (&v)[U], const floatx4 (&old)[U]) {
             each(r, c, edge, [&](int u, int row, int column) {
               store_terms(s + row * p.lda, column, old[u] * (q.b * 0.25f) + v[u] * (q.c * (0.25f / kUp)));
             });
           });
  } else {
    // wide: S X with X's rows as k;  tall: X S, S being symmetric
    if (ACROSS) g.run(S, X, m0, n0, 0, (p.m + 31) / 32, lds);
    else g.run(X, S, m0, n0, 0, (p.m + 31) / 32, lds);
    const auto old = [&](int r, int c) { return m0 + r < M && n0 + c < edge ? load_terms(x0 + (m0 + r) * p.ldx, n0 + c) : floatx4{}; };
    if (!last) {
      g.rows(lds, old, [&](int r, int c, const floatx4 (&v)[U], const floatx4 (&o)[U]) {
        each(r, c, edge, [&](int u, int row, int column) { store_terms(x1 + row * p.ldx, column, o[u] * q.a + v[u] * (1.f / 4096.f)); });
      });
      return;
    }
    const int columns = x.columns;
    const bool whole = columns % 4 == 0 && (reinterpret_cast<uintptr_t>(x.to) & 15) == 0;
    const auto put = [&](auto* to, int column, const floatx4& y) {
      typedef __typeof__(*to) T;
      typedef T Four __attribute__((ext_vector_type(4)));
      if (whole) {
        *reinterpret_cast<Four*>(to) = Four{(T)y[0], (T)y[1], (T)y[2], (T)y[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (column + i < columns) to[i] = (T)y[i];
      }
    };
    if (x.momentum) {
      float* w = reinterpret_cast<float*>(x.to);
      const float rate = x.rate;
      g.rows(lds,
             [&](int r, int c) {
               floatx4 v = {};
               if (m0 + r >= M || n0 + c >= columns) return v;
               const float* from = w + (size_t)(m0 + r) * columns + n0 + c;
               if (whole) {
                 v = *reinterpret_cast<const floatx4*>(from);
               } else {
#pragma unroll
                 for (int i = 0; i < 4; ++i)
                   if (n0 + c + i < columns) v[i] = from[i];
               }
               return v * q.keep - old(r, c) * (q.a * rate * (1.f / kUp));
             },
             [&](int r, int c, const floatx4 (&v)[U], const floatx4 (&o)[U]) {
               each(r, c, columns, [&](int u, int row, int column) {
                 put(w + (size_t)row * columns + column, column, o[u] - v[u] * (rate * (1.f / 4096.f / kUp)));
               });
             });
    } else {
      g.rows(lds, old, [&](int r, int c, const floatx4 (&v)[U], const floatx4 (&o)[U]) {
        each(r, c, columns, [&](int u, int row, int column) {
          const floatx4 y = (o[u] * q.a + v[u] * (1.f / 4096.f)) * (1.f / kUp);
          const size_t at = (size_t)row * columns + column;
          if (q.half) put(reinterpret_cast<_Float16*>(x.to) + at, column, y);
          else put(reinterpret_cast<float*>(x.to) + at, column, y);
        });
      });
    }
  }
}

template <int WHAT, int SIZE>
__global__ __launch_bounds__(256) void muon_product(Batch b, Rule q, int last) {
  extern __shared__ __align__(16) char lds[];
  const int at = matrix_of(b);
  const Matrix& x = b.of[at];
  const unsigned block = blockIdx.x - b.first[at], blocks = b.first[at + 1] - b.first[at];
  if (WHAT == kPolynomial) {
    muon_tile<WHAT, false, SIZE>(x, q, last, block, blocks, lds);
  } else if ((x.rows > x.columns) == (WHAT == kGram)) {
    muon_tile<WHAT, true, SIZE>(x, q, last, block, blocks, lds);
  } else {
    muon_tile<WHAT, false, SIZE>(x, q, last, block, blocks, lds);
  }
}

template <int WHAT, int SIZE>
int launch(const Batch& b, const Rule& q, int last) {
  typedef Sized<2, false, false, SIZE> G;
  TT_ALLOW_LDS((muon_product<WHAT, SIZE>), G::kLds);
  muon_product<WHAT, SIZE><<<b.first[b.count], G::kThreads, G::kLds, stream()>>>(b, q, last);
  TT_LAUNCH_CHECK();
  return 0;
}

template <int WHAT>
int launch(Batch& b, const Rule& q, int last) {
  int size = 2;
  for (;; --size) {
    long long tiles = 0;
    for (int i = 0; i < b.count; ++i) {
      const Place p(b.of[i].rows, b.of[i].columns);
      b.first[i] = (unsigned)tiles;
      tiles += WHAT == kUpdate ? tiles_of(b.of[i].rows, b.of[i].columns, size) : tiles_of(p.m, p.m, size);
    }
    b.first[b.count] = (unsigned)tiles;
    if (size == 0 || tiles >= compute_units() * 3 / 4) break;
  }
  return size == 2 ? launch<WHAT, 2>(b, q, last) : size == 1 ? launch<WHAT, 1>(b, q, last) : launch<WHAT, 0>(b, q, last);
}

// The matrices of one batch, all steps.  scratch: of all of them, and kParts doubles for each.
int run(Batch& b, Rule q, int steps) {
  size_t bytes = 0;
  for (int i = 0; i < b.count; ++i) bytes += ((size_t)Place(b.of[i].rows, b.of[i].columns).bytes() + 255) / 256 * 256 + kParts * sizeof(double);
  void* ws;
  if (tt::workspace(bytes, &ws)) return -1;
  char* at = (char*)ws;
  for (int i = 0; i < b.count; ++i) {
    b.of[i].parts = (double*)at;
    at += kParts * sizeof(double);
    b.of[i].scratch = at;
    at += ((size_t)Place(b.of[i].rows, b.of[i].columns).bytes() + 255) / 256 * 256;
  }
  Batch rows = b;
  b.first[0] = rows.first[0] = 0;
  for (int i = 0; i < b.count; ++i) {
    const size_t n = (size_t)b.of[i].rows * b.of[i].columns;
    b.first[i + 1] = b.first[i] + (unsigned)parts_of(n);
    rows.first[i + 1] = rows.first[i] + (unsigned)((b.of[i].rows + 3) / 4);
  }
  muon_begin<<<b.first[b.count], 256, 0, stream()>>>(b, q);
  TT_LAUNCH_CHECK();
  muon_scale<<<rows.first[b.count], 256, 0, stream()>>>(rows, q);
  TT_LAUNCH_CHECK();
  for (q.step = 0; q.step < steps; ++q.step) {
    if (launch<kGram>(b, q, 0) || launch<kPolynomial>(b, q, 0) || launch<kUpdate>(b, q, q.step == steps - 1)) return -1;
  }
  return 0;
}

// Whether singular values in [0, 1] keep every entry of X, A and b A + c A A inside its range.
bool in_range(double a, double b, double c, int steps) {
  for (int i = 0; i <= 4096; ++i) {
    double s = i / 4096.0;
    for (int k = 0; k < steps; ++k) {
      const double s2 = s * s, p = b * s2 + c * s2 * s2;
      if (!(fabs(p) <= 15.0)) return false;
      s *= a + p;
      if (!(fabs(s) <= 1.9)) return false;
    }
  }
  return true;
}

int check(const char* fn, int rows, int columns) {
  TT_REQUIRE(rows >= 1 && columns >= 1 && rows <= 1 << 20 && columns <= 1 << 20, "%s: matrices of 1 to 2^20 rows and columns, got %d x %d", fn,
             rows, columns);
  TT_REQUIRE((long long)rows * columns <= 1LL << 32, "%s: matrices of 2^32 values at most, got %d x %d", fn, rows, columns);
  return 0;
}
int check(const char* fn, double a, double b, double c, double eps, int steps) {
  TT_REQUIRE(steps >= 1 && steps <= 100, "%s: 1 to 100 steps, got %d", fn, steps);
  TT_REQUIRE(eps > 0.0 && eps <= 1e30, "%s: eps must be positive, got %g", fn, eps);
  TT_REQUIRE(in_range(a, b, c, steps), "%s: the coefficients (%g, %g, %g) let singular values grow past 1.9", fn, a, b, c);
  return 0;
}

}  // namespace

extern "C" {

int tt_orthogonalize(const void* x, void* out, int kind, int rows, int columns, int steps, double a, double b, double c, double eps) {
  TT_REQUIRE_INIT();
  TT_REQUIRE(kind == 0 || kind == 1, "orthogonalize: unknown type %d", kind);
  TT_REQUIRE(x && out, "orthogonalize: null pointer");
  if (check("orthogonalize", rows, columns) || check("orthogonalize", a, b, c, eps, steps)) return -1;
  Batch batch = {};
  batch.count = 1;
  batch.of[0] = Matrix{x, nullptr, out, nullptr, nullptr, 0.f, rows, columns};
  const Rule q = {(float)a, (float)b, (float)c, (float)eps, 0.f, 0.f, 0, kind, 0};
  return run(batch, q, steps);
}

int tt_muon_step_multi_f32(int count, float* const* params, const float* const* grads, float* const* momenta, const int* rows,
                           const int* columns, const double* scales, double lr, double momentum, double weight_decay, int nesterov,
                           int steps, double a, double b, double c, double eps) {
  TT_REQUIRE_INIT();
  const char* fn = "muon_step";
  TT_REQUIRE(count >= 0, "%s: negative count", fn);
  if (count == 0) return 0;
  TT_REQUIRE(params && grads && momenta && rows && columns && scales, "%s: null table", fn);
  if (check(fn, a, b, c, eps, steps)) return -1;
  std::vector<int> order;
  for (int i = 0; i < count; ++i) {
    if (check(fn, rows[i], columns[i])) return -1;
    TT_REQUIRE(params[i] && grads[i] && momenta[i], "%s: null pointer for matrix %d", fn, i);
    order.push_back(i);
  }
  // (large ones first: the last blocks of a launch are then small ones')
  std::stable_sort(order.begin(), order.end(), [&](int i, int j) { return (long long)rows[i] * columns[i] > (long long)rows[j] * columns[j]; });
  const Rule q = {(float)a, (float)b, (float)c, (float)eps, (float)(1.0 - momentum), (float)(1.0 - lr * weight_decay), nesterov, 0, 0};
  for (size_t done = 0; done < order.size();) {
    Batch batch = {};
    size_t bytes = 0;
    for (; done < order.size() && batch.count < kMost; ++done) {
      const int i = order[done];
      const size_t more = (size_t)Place(rows[i], columns[i]).bytes();
      if (batch.count && bytes + more > kMostScratch) break;
      bytes += more;
      batch.of[batch.count++] = Matrix{grads[i], momenta[i], params[i], nullptr, nullptr, (float)(lr * scales[i]), rows[i], columns[i]};
    }
    if (run(batch, q, steps)) return -1;
  }
  return 0;
}

}  // extern "C"
