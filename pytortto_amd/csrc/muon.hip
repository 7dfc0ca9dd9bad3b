// Orthogonalised updates: Newton-Schulz products of a matrix [rows, columns], alone or inside the optimiser's step.
//
//   X <- X / max(|X|_F, eps)         steps times:  A = X X^T,  X <- a X + (b A + c A A) X
//
// takes every singular value s of X to a s + b s^3 + c s^5, and in a few steps all of them to about 1.  A is taken over the
// shorter side: X^T X, and X on the left of the sum, where there are more rows than columns, so that nothing is transposed (product.h
// reads either operand along or across its rows).
//
// All products are of two float16 terms an operand, X and A scaled by 2^14 and a I + b A + c A A (in muon_small without a I) by 2^12: with
// singular values up to 1.9, and a and the polynomial up to 15, which calls are checked for, no entry
// leaves float16's range, and one is held to 2^-22 of itself or 2^-39 of the unit.
// The two symmetric products are made of the tiles on and above the diagonal; several blocks may share one along the reduction, and
// leave sums that muon_join adds up, in order, and mirrors.  The matrices of a step share the launches, five for each of its
// Newton-Schulz steps and two in front: a network has tens of them, most too small to fill the device.
#include "product.h"
#include "rows.h"

#include <algorithm>
#include <map>
#include <vector>

namespace {

using namespace tt;

constexpr int kMost = 48;                   // matrices of a launch (their table is a kernel's argument)
constexpr size_t kMostScratch = (size_t)4 << 30;
constexpr size_t kMostPartial = (size_t)1 << 30;
constexpr int kUpBits = 14;
constexpr float kUp = 1 << kUpBits;         // the scale of X and A
constexpr int kParts = 1024;                // partial sums of a matrix's squares, at most
constexpr int kJoin = 64;                   // columns of what a block of muon_join works on

struct Matrix {
  const void* from;         // the gradient, or the matrix itself (float32 or float16)
  float* momentum;          // or none
  void* to;                 // the parameter, or the result
  char* scratch;
  float* partial;           // sums of a symmetric product's upper tiles, `splits` times
  float rate;               // of a parameter: learning rate times the matrix's own scale
  int rows, columns, splits;
};

// In scratch memory: X twice, A, b A + c A A, each as rows of terms, and the partial sums of squares.
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
  __host__ __device__ long long bytes() const { return 2 * x + 2 * a + kParts * (long long)sizeof(double); }
  __host__ __device__ double* parts(char* scratch) const { return reinterpret_cast<double*>(scratch + 2 * x + 2 * a); }
  // floats of one set of partial sums
  __host__ __device__ long long square() const { return padded(m) * m; }
};

struct Batch {
  Matrix of[kMost];
  unsigned first[kMost + 1];        // blocks in front of each
  int count;
};
static_assert(sizeof(Batch) <= 3800, "a kernel's arguments");
__device__ __forceinline__ int matrix_of(const Batch& b) {
  int i = 0;
  while (i + 1 < b.count && blockIdx.x >= b.first[i + 1]) ++i;
  return i;
}

// Partial sums of a matrix of n values: a block has 8192 of them, or more.
__host__ __device__ inline int parts_of(size_t n) { return n > (size_t)kParts * 8192 ? kParts : (int)((n + 8191) / 8192); }

struct Rule {
  float a, b, c;
  double eps;
  float mix;                        // 1 - momentum
  float keep;                       // 1 - learning rate times weight decay
  int nesterov, half, step;
};

__device__ __forceinline__ float update_of(const Rule& q, float g, float m) { return q.nesterov ? m - q.mix * (m - g) : m; }

// kUp / max(|u|_F, eps) for a sum of squares, as 2^e m with m in (1, 2]: the quotient itself would leave float32's range for norms below 5e-35, and
// lose digits above 8e37.
struct Inverse {
  int e;
  float m;
  __device__ __forceinline__ Inverse(double squares, double eps) {
    const double norm = sqrt(squares), by = norm > eps || norm != norm ? norm : eps;
    int k = 0;
    const double part = __builtin_isfinite(by) ? frexp(by, &k) : by;
    e = kUpBits - k;
    m = (float)(1.0 / part);
  }
  __device__ __forceinline__ float operator()(float u) const { return ldexpf(u, e) * m; }
};

// n values of an array from value i on, n = 4 where the array and i allow it.
template <typename T>
__device__ __forceinline__ floatx4 read_four(const T* p, size_t i, int n, bool whole) {
  typedef T Four __attribute__((ext_vector_type(4)));
  floatx4 v = {};
  if (whole) {
    const Four f = *reinterpret_cast<const Four*>(p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = widen(f[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) v[k] = widen(p[i + k]);
  }
  return v;
}
__device__ __forceinline__ floatx4 read_from(const Matrix& x, const Rule& q, size_t i, int n, bool whole) {
  return q.half ? read_four(reinterpret_cast<const _Float16*>(x.from), i, n, whole) : read_four(reinterpret_cast<const float*>(x.from), i, n, whole);
}
__device__ __forceinline__ bool all_aligned(const Matrix& x) {
  return ((reinterpret_cast<uintptr_t>(x.from) | reinterpret_cast<uintptr_t>(x.momentum)) & 15) == 0;
}

// The momentum, and the squares of the update's values.  Bound by memory: 50 million values 105 us, 5.7 TB/s.
__global__ __launch_bounds__(256) void muon_begin(Batch b, Rule q) {
  __shared__ double part[4];
  const int at = matrix_of(b);
  const Matrix& x = b.of[at];
  const unsigned block = blockIdx.x - b.first[at], blocks = b.first[at + 1] - b.first[at];
  const size_t n = (size_t)x.rows * x.columns, step = (size_t)blocks * 1024;
  const bool aligned = all_aligned(x);
  double s = 0.0;
  for (size_t i = (size_t)block * 1024 + threadIdx.x * 4; i < n; i += step) {
    const int some = n - i < 4 ? (int)(n - i) : 4;
    const bool whole = aligned && some == 4;
    floatx4 u = read_from(x, q, i, some, whole);
    if (x.momentum) {
      const floatx4 g = u, old = read_four(x.momentum, i, some, whole), m = old + q.mix * (g - old);
      if (whole) {
        *reinterpret_cast<floatx4*>(x.momentum + i) = m;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < some) x.momentum[i + k] = m[k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = update_of(q, g[k], m[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) s += (double)u[k] * (double)u[k];
  }
  s = row_sum<256>(s, part);
  if (threadIdx.x == 0) Place(x.rows, x.columns).parts(x.scratch)[block] = s;
}

// X as rows of terms, divided by its norm.  A block has kScaled quads of columns, of one row or several.  Bound by memory: 50 million values
// 118 us, 5.1 TB/s.  (The update is formed again from gradient and momentum: a copy of it would be written and read.)
constexpr int kScaled = 2048;
__host__ __device__ inline unsigned scale_blocks(int rows, int columns) {
  return (unsigned)(((size_t)rows * (padded(columns) / 4) + kScaled - 1) / kScaled);
}
__global__ __launch_bounds__(256) void muon_scale(Batch b, Rule q) {
  __shared__ double part[4];
  const int at = matrix_of(b);
  const Matrix& x = b.of[at];
  const Place p(x.rows, x.columns);
  const int parts = parts_of((size_t)x.rows * x.columns);
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) s += p.parts(x.scratch)[i];
  s = row_sum<256>(s, part);
  const Inverse inverse(s, q.eps);
  const size_t quads = padded(x.columns) / 4, all = (size_t)x.rows * quads;
  const bool aligned = all_aligned(x) && x.columns % 4 == 0;
  size_t k = (size_t)(blockIdx.x - b.first[at]) * kScaled + threadIdx.x;
  for (const size_t end = k + kScaled < all ? k + kScaled : all; k < end; k += 256) {
    const size_t row = k / quads;
    const int c = (int)(k - row * quads) * 4, some = x.columns - c < 4 ? x.columns - c : 4;
    const size_t i = row * x.columns + c;
    floatx4 u = {};
    if (some > 0) {
      u = read_from(x, q, i, some, aligned);
      if (x.momentum) {
        const floatx4 m = read_four(x.momentum, i, some, aligned);
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = update_of(q, u[e], m[e]);
      }
    }
    store_terms(x.scratch + row * p.ldx, c, floatx4{inverse(u[0]), inverse(u[1]), inverse(u[2]), inverse(u[3])});
  }
}

constexpr int kGram = 0, kPolynomial = 1, kUpdate = 2;

// Tiles of a symmetric product on and above the diagonal, `side` in a row.
__host__ __device__ inline long long upper(long long side) { return side * (side + 1) / 2; }
__device__ __forceinline__ void upper_tile(int at, int side, int* m, int* n) {
  int row = 0;
  while (at >= side - row) at -= side - row++;
  *m = row;
  *n = row + at;
}

// One tile of one product of a step.  Bound by the matrix instructions under the power limit where there are many: a step's update of four
// matrices of 2048 x 2048 and two of 2048 x 8192 takes 466 us, 1330 TFLOP/s of three products, and their symmetric products 278 and 134 us,
// 1250 and 1300 of the tiles they have.  Small ones are bound by their tiles' beginning and end: 5001 x 777 40, 20 and 8 us.
template <int WHAT, bool ACROSS, int SIZE>
__device__ __forceinline__ void muon_tile(const Matrix& x, const Rule& q, bool last, unsigned block, unsigned blocks, char* lds) {
  constexpr bool kA = WHAT == kGram && ACROSS, kB = WHAT == kGram ? ACROSS : WHAT == kUpdate && ACROSS;
  typedef Sized<2, kA, kB, SIZE> G;
  constexpr int U = G::kAhead;
  const Place p(x.rows, x.columns);
  char* x0 = x.scratch + (q.step & 1 ? p.x : 0);
  char* x1 = x.scratch + (q.step & 1 ? 0 : p.x);
  char *a = x.scratch + 2 * p.x, *s = a + p.a;
  const Operand X = {x0, p.x, (int)p.ldx, kLine}, A = {a, p.a, (int)p.lda, kLine}, S = {s, p.a, (int)p.lda, kLine};
  int m, n;
  G g;
  if (WHAT != kUpdate) {
    // sums of a part of the reduction, for muon_join
    const int side = (p.m + G::kM - 1) / G::kM, tiles = (int)upper(side), at = xcd_remap(block, blocks), split = at / tiles;
    upper_tile(at % tiles, side, &m, &n);
    const int pairs = ((WHAT == kGram ? ACROSS ? x.rows : x.columns : p.m) + 31) / 32, per = (pairs + x.splits - 1) / x.splits;
    const int first = split * per, count = first + per < pairs ? per : pairs - first;
    const int m0 = m * G::kM, n0 = n * G::kN, edge = (int)padded(p.m);
    float* to = x.partial + split * p.square();
    if (WHAT == kGram) g.run(X, X, m0, n0, first, count, lds);
    else g.run(A, A, m0, n0, first, count, lds);
    g.rows(lds, [](int, int) { return 0; }, [&](int r, int c, const floatx4 (&v)[U], int (&)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = m0 + r + u * G::kStep;
        if (row < p.m && n0 + c < edge) *reinterpret_cast<floatx4*>(to + (long long)row * edge + n0 + c) = v[u];
      }
    });
    return;
  }
  const int M = x.rows, columns = x.columns, edge = (int)padded(columns);
  tile_at(xcd_remap(block, blocks), (M + G::kM - 1) / G::kM, (columns + G::kN - 1) / G::kN, &m, &n);
  const int m0 = m * G::kM, n0 = n * G::kN;
  const auto each = [&](int r, int c, int end, auto f) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (m0 + r + u * G::kStep < M && n0 + c < end) f(u, m0 + r + u * G::kStep, n0 + c);
  };
  // wide: S X with X's rows as k;  tall: X S, S being symmetric
  if (ACROSS) g.run(S, X, m0, n0, 0, (p.m + 31) / 32, lds);
  else g.run(X, S, m0, n0, 0, (p.m + 31) / 32, lds);
  const auto none = [](int, int) { return 0; };
  if (!last) {
    g.rows(lds, none, [&](int r, int c, const floatx4 (&v)[U], const int (&)[U]) {
      each(r, c, edge, [&](int u, int row, int column) { store_terms(x1 + row * p.ldx, column, v[u] * (1.f / 4096.f)); });
    });
    return;
  }
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
             if (m0 + r >= M || n0 + c >= columns) return floatx4{};
             const size_t at = (size_t)(m0 + r) * columns + n0 + c;
             return read_four(w, at, columns - n0 - c, whole) * q.keep;
           },
           [&](int r, int c, const floatx4 (&v)[U], const floatx4 (&o)[U]) {
             each(r, c, columns, [&](int u, int row, int column) {
               put(w + (size_t)row * columns + column, column, o[u] - v[u] * (rate * (1.f / 4096.f / kUp)));
             });
           });
  } else {
    g.rows(lds, none, [&](int r, int c, const floatx4 (&v)[U], const int (&)[U]) {
      each(r, c, columns, [&](int u, int row, int column) {
        const floatx4 y = v[u] * (1.f / 4096.f / kUp);
        const size_t at = (size_t)row * columns + column;
        if (q.half) put(reinterpret_cast<_Float16*>(x.to) + at, column, y);
        else put(reinterpret_cast<float*>(x.to) + at, column, y);
      });
    });
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

// A = X X^T, or a I + b A + c A A, from the partial sums of the upper tiles: STRIP x 64 of it, and the same on the other side of the
// diagonal.  The sums come from other dies' blocks, and what bounds few blocks is how many loads are on their way: 9 sums of 777 x 777 took 91
// blocks with 64 rows 13.7 us, and 364 with 16 rows 5.1.  Many are bound by memory, and better with whole lines on the other
// side, too: the polynomials of 6 matrices of 2048 x 2048, 3168 blocks, take 32 us with 64 rows and 38 with 16.
template <int WHAT, int STRIP>
__global__ __launch_bounds__(256) void muon_join(Batch b, Rule q) {
  __shared__ float turned[kJoin][STRIP + 1];
  constexpr int kStrips = kJoin / STRIP, kHigh = STRIP / 16, kAtOnce = 8 / kHigh;
  const int at = matrix_of(b);
  const Matrix& x = b.of[at];
  const Place p(x.rows, x.columns);
  const int edge = (int)padded(p.m), block = (int)(blockIdx.x - b.first[at]), strip = block % kStrips * STRIP;
  int m, n;
  upper_tile(block / kStrips, edge / kJoin, &m, &n);
  char *a = x.scratch + 2 * p.x, *to = WHAT == kGram ? a : a + p.a;
  const int r = threadIdx.x >> 4, r0 = m * kJoin + strip + r, c = n * kJoin + (threadIdx.x & 15) * 4;
  floatx4 v[kHigh] = {};
  const float* from[kHigh];
#pragma unroll
  for (int i = 0; i < kHigh; ++i) from[i] = x.partial + (long long)min(r0 + 16 * i, p.m - 1) * edge + c;
#pragma unroll kAtOnce
  for (int s = 0; s < x.splits; ++s) {
#pragma unroll
    for (int i = 0; i < kHigh; ++i) v[i] += *reinterpret_cast<const floatx4*>(from[i] + s * p.square());
  }
#pragma unroll
  for (int i = 0; i < kHigh; ++i) {
    const int row = r0 + 16 * i;
    if (row < p.m) {
      if (WHAT == kGram) {
        v[i] *= 1.f / kUp;
      } else {
        v[i] = load_terms(a + row * p.lda, c) * (q.b * 0.25f) + v[i] * (q.c * (0.25f / kUp));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] += row == c + e ? q.a * 4096.f : 0.f;
      }
      store_terms(to + row * p.lda, c, v[i]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) turned[(threadIdx.x & 15) * 4 + e][r + 16 * i] = row < p.m ? v[i][e] : 0.f;
  }
  if (m == n) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kHigh; ++i) {
    const int k = (threadIdx.x + i * 256) / (STRIP / 4), j = threadIdx.x % (STRIP / 4) * 4, other = n * kJoin + k;
    if (other < p.m) store_terms(to + other * p.lda, m * kJoin + strip + j, floatx4{turned[k][j], turned[k][j + 1], turned[k][j + 2], turned[k][j + 3]});
  }
}

// What a product takes, in microseconds (measured with one block on every compute unit): a pair of a tile, a tile's beginning and end.
constexpr float kPairTime[3] = {0.36f, 0.75f, 2.1f}, kTileTime[3] = {4.f, 7.f, 16.f};

template <int WHAT>
int pairs_of(const Matrix& x) {
  const int m = std::min(x.rows, x.columns), n = std::max(x.rows, x.columns);
  return ((WHAT == kGram ? n : m) + 31) / 32;
}
template <int WHAT>
long long tiles_in(const Matrix& x, int size) {
  if (WHAT == kUpdate) return tiles_of(x.rows, x.columns, size);
  return upper((std::min(x.rows, x.columns) + kTileSide[size] - 1) / kTileSide[size]);
}

// The same matrices come every step, so plans are kept by their sizes.
struct Plan {
  int size;
  std::vector<int> splits;
};
template <int WHAT>
std::map<std::vector<int>, Plan>& plans() {
  static std::map<std::vector<int>, Plan> all;
  return all;
}

// The size of the tiles, and of a symmetric product how many blocks share one (a matrix's splits): what takes the least time if all blocks
// are as long as their mean, in whole rounds over the compute units, and none is longer than that.
template <int WHAT>
Plan make_plan(const Batch& b) {
  float least = 0.f;
  int best_size = -1, best_share = 0;
  const auto splits_for = [&](const Matrix& x, int share) {
    if (WHAT == kUpdate) return 1;
    // (four pairs or more to a block, and partial sums within their memory)
    const int pairs = pairs_of<WHAT>(x), want = (pairs + share - 1) / share;
    const long long room = std::max(1LL, (long long)(kMostPartial / b.count) / (Place(x.rows, x.columns).square() * 4));
    const int splits = (int)std::max(1LL, std::min<long long>(want, room)), per = (pairs + splits - 1) / splits;
    return (pairs + per - 1) / per;
  };
  for (int size = 0; size < 3; ++size) {
    for (int share = WHAT == kUpdate ? 1 << 20 : 4; share <= 1 << 20; share = share < 512 ? share * 3 / 2 : share == 1 << 20 ? share + 1 : 1 << 20) {
      double blocks = 0.0, work = 0.0, traffic = 0.0, longest = 0.0;
      for (int i = 0; i < b.count; ++i) {
        const Matrix& x = b.of[i];
        const int splits = splits_for(x, share), pairs = pairs_of<WHAT>(x);
        const double mine = (double)tiles_in<WHAT>(x, size) * splits, time = (pairs + splits - 1) / splits * kPairTime[size] + kTileTime[size];
        blocks += mine;
        work += mine * time;
        longest = std::max(longest, time);
        if (WHAT != kUpdate) traffic += 4.0 * splits * Place(x.rows, x.columns).square();
      }
      const double rounds = ceil(blocks / compute_units()), time = std::max(longest, rounds * work / blocks) + traffic / 4e6;
      if (best_size < 0 || time < least) {
        least = (float)time;
        best_size = size;
        best_share = share;
      }
    }
  }
  Plan p{best_size, {}};
  for (int i = 0; i < b.count; ++i) p.splits.push_back(splits_for(b.of[i], best_share));
  return p;
}
template <int WHAT>
int plan(Batch& b) {
  std::vector<int> key;
  for (int i = 0; i < b.count; ++i) key.insert(key.end(), {b.of[i].rows, b.of[i].columns});
  auto& all = plans<WHAT>();
  if (all.size() >= 256) all.clear();
  auto found = all.find(key);
  if (found == all.end()) found = all.emplace(std::move(key), make_plan<WHAT>(b)).first;
  unsigned first = 0;
  for (int i = 0; i < b.count; ++i) {
    b.of[i].splits = found->second.splits[i];
    b.first[i] = first;
    first += (unsigned)(tiles_in<WHAT>(b.of[i], found->second.size) * b.of[i].splits);
  }
  b.first[b.count] = first;
  return found->second.size;
}

template <int WHAT, int SIZE>
int launch(const Batch& b, const Rule& q, int last) {
  typedef Sized<2, false, false, SIZE> G;
  TT_ALLOW_LDS((muon_product<WHAT, SIZE>), G::kLds);
  muon_product<WHAT, SIZE><<<b.first[b.count], 256, G::kLds, stream()>>>(b, q, last);
  TT_LAUNCH_CHECK();
  return 0;
}
template <int WHAT>
int launch(int size, const Batch& b, const Rule& q, int last) {
  return size == 2 ? launch<WHAT, 2>(b, q, last) : size == 1 ? launch<WHAT, 1>(b, q, last) : launch<WHAT, 0>(b, q, last);
}

// ---- small matrices --------------------------------------------------------------------------------
// A matrix of at most kShort rows or columns, and kLong of the others, stays in one block's LDS for all steps (one launch instead of 27, of some 4 us
// each; 64 x 64 24 us, 65 x 65 119; 64 x 384 92 us, 64 x 385 116): X with its shorter side as rows, A, and b A + c A A, each as
// rows of terms, kGap bytes apart so that rows stand in different banks.
constexpr int kShort = 64, kLong = 384, kGap = 16;
bool is_small(int rows, int columns) { return std::min(rows, columns) <= kShort && std::max(rows, columns) <= kLong; }

constexpr int kSquareRow = kShort * 4 + kGap;
constexpr int small_row(int n) { return n * 4 + kGap; }

// Fragments of 16 x 32 from rows of terms: k along the rows, or across them.
__device__ __forceinline__ half8 along(const char* rows, int ld, int first, int k, int term) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const half8*>(rows + (first + (lane & 15)) * ld + (k >> 5) * kLine + term * kTermBytes + (lane >> 4) * 16);
}
__device__ __forceinline__ half8 across_rows(const char* rows, int ld, int first, int k, int term) {
  const int lane = threadIdx.x & 63, j = lane & 15;
  const char* p = rows + (k + (lane >> 4) * 8 + (j >> 2)) * ld + (first >> 5) * kLine + term * kTermBytes + (first & 16) * 2 + (j & 3) * 8;
  const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<shortx4>)p);
  const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<shortx4>)(p + 4 * ld));
  return __builtin_bit_cast(half8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}
// Three products of two terms each; a lane holds row l % 16 of a, columns 4 (l / 16) .. + 3 of b.
__device__ __forceinline__ floatx4 three(const half8 (&a)[2], const half8 (&b)[2], floatx4 sum) {
  sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[0], a[0], sum, 0, 0, 0);
  sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[1], a[0], sum, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(b[0], a[1], sum, 0, 0, 0);
}

// A block has one matrix, a wave sixteen of its shorter side.  X has WIDE columns, those behind the matrix's zeros.
template <int WIDE>
__global__ __launch_bounds__(256) void muon_small(Batch b, Rule q, int steps) {
  __shared__ double part[4];
  extern __shared__ __align__(16) char lds[];
  const Matrix& x = b.of[blockIdx.x];
  const bool tall = x.rows > x.columns;
  const int size = x.rows * x.columns;
  constexpr int ld = small_row(WIDE);
  char *X = lds, *A = X + kShort * ld, *S = A + kShort * kSquareRow;
  // element i of the matrix is X[row][column]
  const auto place = [&](int i, int* row, int* column) {
    const int r = i / x.columns, c = i - r * x.columns;
    *row = tall ? c : r;
    *column = tall ? r : c;
  };
  double s = 0.0;
  for (int i = threadIdx.x; i < size; i += 256) {
    float u;
    if (x.momentum) {
      const float g = reinterpret_cast<const float*>(x.from)[i], old = x.momentum[i], now = old + q.mix * (g - old);
      x.momentum[i] = now;
      u = update_of(q, g, now);
    } else {
      u = read_value(x.from, i, q.half);
    }
    s += (double)u * (double)u;
  }
  s = row_sum<256>(s, part);
  const Inverse inverse(s, q.eps);
  for (int i = threadIdx.x; i < kShort * (ld / 16); i += 256) reinterpret_cast<floatx4*>(X)[i] = floatx4{};
  __syncthreads();
  for (int i = threadIdx.x; i < size; i += 256) {
    const float u = x.momentum ? update_of(q, reinterpret_cast<const float*>(x.from)[i], x.momentum[i]) : read_value(x.from, i, q.half);
    int row, column;
    place(i, &row, &column);
    _Float16 hi, lo;
    split(inverse(u), &hi, &lo);
    char* p = X + row * ld + at_column(column);
    *reinterpret_cast<_Float16*>(p) = hi;
    *reinterpret_cast<_Float16*>(p + kTermBytes) = lo;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, mine = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 16;
  const int row = mine + (lane & 15), c0 = (lane >> 4) * 4;
  constexpr int kSquare = kShort / 16, kPieces = WIDE / 16;
  for (int step = 0; step < steps; ++step) {
    {
      floatx4 sum[kSquare] = {};
      for (int k = 0; k < WIDE; k += 32) {
        const half8 a[2] = {along(X, ld, mine, k, 0), along(X, ld, mine, k, 1)};
#pragma unroll
        for (int j = 0; j < kSquare; ++j) {
          const half8 c[2] = {along(X, ld, j * 16, k, 0), along(X, ld, j * 16, k, 1)};
          sum[j] = three(a, c, sum[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < kSquare; ++j) store_terms(A + row * kSquareRow, j * 16 + c0, sum[j] * (1.f / kUp));
    }
    __syncthreads();
    {
      floatx4 sum[kSquare] = {};
#pragma unroll
      for (int k = 0; k < kShort; k += 32) {
        const half8 a[2] = {along(A, kSquareRow, mine, k, 0), along(A, kSquareRow, mine, k, 1)};
#pragma unroll
        for (int j = 0; j < kSquare; ++j) {
          const half8 c[2] = {along(A, kSquareRow, j * 16, k, 0), along(A, kSquareRow, j * 16, k, 1)};
          sum[j] = three(a, c, sum[j]);
        }
      }
#pragma unroll
      for (int j = 0; j < kSquare; ++j) {
        const floatx4 old = load_terms(A + row * kSquareRow, j * 16 + c0);
        store_terms(S + row * kSquareRow, j * 16 + c0, old * (q.b * 0.25f) + sum[j] * (q.c * (0.25f / kUp)));
      }
    }
    __syncthreads();
    floatx4 sum[kPieces] = {};
#pragma unroll
    for (int k = 0; k < kShort; k += 32) {
      const half8 a[2] = {along(S, kSquareRow, mine, k, 0), along(S, kSquareRow, mine, k, 1)};
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const half8 c[2] = {across_rows(X, ld, j * 16, k, 0), across_rows(X, ld, j * 16, k, 1)};
        sum[j] = three(a, c, sum[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      sum[j] = load_terms(X + row * ld, j * 16 + c0) * q.a + sum[j] * (1.f / 4096.f);
    }
    __syncthreads();          // (everybody has read X)
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      if (step < steps - 1) {
        store_terms(X + row * ld, j * 16 + c0, sum[j]);
        continue;
      }
      // the result, as it is: its own row of LDS holds as many floats as terms
      *reinterpret_cast<floatx4*>(X + row * ld + (j * 16 + c0) * 4) = sum[j] * (1.f / kUp);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < size; i += 256) {
    int r, c;
    place(i, &r, &c);
    const float o = *reinterpret_cast<const float*>(X + r * ld + c * 4);
    if (x.momentum) {
      float* w = reinterpret_cast<float*>(x.to) + i;
      *w = *w * q.keep - x.rate * o;
    } else if (q.half) {
      reinterpret_cast<_Float16*>(x.to)[i] = (_Float16)o;
    } else {
      reinterpret_cast<float*>(x.to)[i] = o;
    }
  }
}

template <int WIDE>
int launch_small(const Batch& b, const Rule& q, int steps) {
  constexpr int kBytes = kShort * small_row(WIDE) + 2 * kShort * kSquareRow;
  TT_ALLOW_LDS(muon_small<WIDE>, kBytes);
  muon_small<WIDE><<<b.count, 256, kBytes, stream()>>>(b, q, steps);
  TT_LAUNCH_CHECK();
  return 0;
}
// (The time is that of the columns there is room for: 64 x 64 24 us, 64 x 192 53, 64 x 384 92.)
int run_small(const Batch& b, const Rule& q, int steps) {
  int most = 0;
  for (int i = 0; i < b.count; ++i) most = std::max(most, std::max(b.of[i].rows, b.of[i].columns));
  return most <= 64 ? launch_small<64>(b, q, steps) : most <= 192 ? launch_small<192>(b, q, steps) : launch_small<kLong>(b, q, steps);
}

template <int WHAT>
int launch_join(bool strips, const Batch& b, const Rule& q) {
  if (strips) muon_join<WHAT, 16><<<b.first[b.count], 256, 0, stream()>>>(b, q);
  else muon_join<WHAT, 64><<<b.first[b.count], 256, 0, stream()>>>(b, q);
  TT_LAUNCH_CHECK();
  return 0;
}

// ---- batches ---------------------------------------------------------------------------------------
// The matrices of one batch, with the plans of their products.
struct Work {
  Batch gram, polynomial, update;       // (of small ones the first alone)
  int gram_size, polynomial_size, update_size;
  bool small;
  size_t bytes;                         // of scratch memory
};
size_t up(size_t n) { return (n + 255) / 256 * 256; }
size_t partial_bytes(const Work& w, int i) {
  const Matrix& x = w.gram.of[i];
  return up((size_t)std::max(x.splits, w.polynomial.of[i].splits) * Place(x.rows, x.columns).square() * 4);
}
Work prepare(const Batch& batch, bool small) {
  Work w = {batch, batch, batch, 0, 0, 0, small, 0};
  if (small) return w;
  w.gram_size = plan<kGram>(w.gram);
  w.polynomial_size = plan<kPolynomial>(w.polynomial);
  w.update_size = plan<kUpdate>(w.update);
  for (int i = 0; i < batch.count; ++i) w.bytes += up(Place(batch.of[i].rows, batch.of[i].columns).bytes()) + partial_bytes(w, i);
  return w;
}

// All steps of a batch.
int run(Work& w, Rule q, int steps) {
  if (w.small) return run_small(w.gram, q, steps);
  Batch &gram = w.gram, &polynomial = w.polynomial, &update = w.update;
  void* ws;
  if (tt::workspace(w.bytes, &ws)) return -1;
  char* at = (char*)ws;
  for (int i = 0; i < gram.count; ++i) {
    gram.of[i].scratch = polynomial.of[i].scratch = update.of[i].scratch = at;
    at += up(Place(gram.of[i].rows, gram.of[i].columns).bytes());
    gram.of[i].partial = polynomial.of[i].partial = (float*)at;
    at += partial_bytes(w, i);
  }
  Batch begin = gram, rows = gram, gram_join = gram, polynomial_join = polynomial;
  begin.first[0] = rows.first[0] = gram_join.first[0] = polynomial_join.first[0] = 0;
  for (int i = 0; i < gram.count; ++i) {
    const int r = gram.of[i].rows, c = gram.of[i].columns;
    begin.first[i + 1] = begin.first[i] + (unsigned)parts_of((size_t)r * c);
    rows.first[i + 1] = rows.first[i] + scale_blocks(r, c);
    gram_join.first[i + 1] = polynomial_join.first[i + 1] = gram_join.first[i] + (unsigned)upper(padded(std::min(r, c)) / kJoin);
  }
  const bool strips = gram_join.first[gram.count] < (unsigned)compute_units();
  for (int i = 1; strips && i <= gram.count; ++i) gram_join.first[i] = polynomial_join.first[i] = 4 * gram_join.first[i];
  muon_begin<<<begin.first[begin.count], 256, 0, stream()>>>(begin, q);
  TT_LAUNCH_CHECK();
  muon_scale<<<rows.first[rows.count], 256, 0, stream()>>>(rows, q);
  TT_LAUNCH_CHECK();
  for (q.step = 0; q.step < steps; ++q.step) {
    if (launch<kGram>(w.gram_size, gram, q, 0)) return -1;
    if (launch_join<kGram>(strips, gram_join, q)) return -1;
    if (launch<kPolynomial>(w.polynomial_size, polynomial, q, 0)) return -1;
    if (launch_join<kPolynomial>(strips, polynomial_join, q)) return -1;
    if (launch<kUpdate>(w.update_size, update, q, q.step == steps - 1)) return -1;
  }
  return 0;
}

// Whether singular values in [0, 1] keep every entry of X, A and the polynomial of A inside its range.  (It takes 30 us, more than
// all of a small matrix: the last answer is kept.)
bool try_range(double a, double b, double c, int steps) {
  for (int i = 0; i <= 4096; ++i) {
    double s = i / 4096.0;
    for (int k = 0; k < steps; ++k) {
      const double s2 = s * s, p = b * s2 + c * s2 * s2;
      if (!(fabs(p) <= 15.0 && fabs(a + p) <= 15.0)) return false;
      s *= a + p;
      if (!(fabs(s) <= 1.9)) return false;
    }
  }
  return true;
}
bool in_range(double a, double b, double c, int steps) {
  static double last[3];
  static int last_steps = 0;      // (of a good answer)
  if (steps == last_steps && a == last[0] && b == last[1] && c == last[2]) return true;
  if (!try_range(a, b, c, steps)) return false;
  last[0] = a;
  last[1] = b;
  last[2] = c;
  last_steps = steps;
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

int tt_orthogonalize(const void* x, void* out, int kind, int rows, int columns, int steps, double a, double b, double c, double eps) try {
  TT_REQUIRE_INIT();
  TT_REQUIRE(kind == 0 || kind == 1, "orthogonalize: unknown type %d", kind);
  TT_REQUIRE(x && out, "orthogonalize: null pointer");
  if (check("orthogonalize", rows, columns) || check("orthogonalize", a, b, c, eps, steps)) return -1;
  Batch batch = {};
  batch.count = 1;
  batch.of[0] = Matrix{x, nullptr, out, nullptr, nullptr, 0.f, rows, columns, 1};
  const Rule q = {(float)a, (float)b, (float)c, eps, 0.f, 0.f, 0, kind, 0};
  Work work = prepare(batch, is_small(rows, columns));
  return run(work, q, steps);
} catch (const std::exception& e) {
  return tt::fail(-1, "orthogonalize: %s", e.what());
}

int tt_muon_step_multi_f32(int count, float* const* params, const float* const* grads, float* const* momenta, const int* rows,
                           const int* columns, const double* scales, double lr, double momentum, double weight_decay, int nesterov,
                           int steps, double a, double b, double c, double eps) try {
  TT_REQUIRE_INIT();
  const char* fn = "muon_step";
  TT_REQUIRE(count >= 0, "%s: negative count", fn);
  if (count == 0) return 0;
  TT_REQUIRE((!params || (grads && momenta)) && rows && columns && scales, "%s: null table", fn);
  if (check(fn, a, b, c, eps, steps)) return -1;
  std::vector<int> order;
  for (int i = 0; i < count; ++i) {
    if (check(fn, rows[i], columns[i])) return -1;
    TT_REQUIRE(!params || (params[i] && grads[i] && momenta[i]), "%s: null pointer for matrix %d", fn, i);
    order.push_back(i);
  }
  // (large ones first: the last blocks of a launch are then small ones', and those of one block each come last)
  std::stable_sort(order.begin(), order.end(), [&](int i, int j) {
    const bool first = is_small(rows[i], columns[i]), second = is_small(rows[j], columns[j]);
    return first != second ? second : (long long)rows[i] * columns[i] > (long long)rows[j] * columns[j];
  });
  const Rule q = {(float)a, (float)b, (float)c, eps, (float)(1.0 - momentum), (float)(1.0 - lr * weight_decay), nesterov, 0, 0};
  std::vector<Work> works;
  size_t most = 0;
  for (size_t done = 0; done < order.size();) {
    Batch batch = {};
    size_t bytes = 0;
    const bool small = is_small(rows[order[done]], columns[order[done]]);
    for (; done < order.size() && batch.count < kMost; ++done) {
      const int i = order[done];
      if (is_small(rows[i], columns[i]) != small) break;
      const size_t more = (size_t)Place(rows[i], columns[i]).bytes();
      if (batch.count && bytes + more > kMostScratch) break;
      bytes += more;
      batch.of[batch.count++] = params ? Matrix{grads[i], momenta[i], params[i], nullptr, nullptr, (float)(lr * scales[i]), rows[i], columns[i], 1}
                                       : Matrix{nullptr, nullptr, nullptr, nullptr, nullptr, 0.f, rows[i], columns[i], 1};
    }
    works.push_back(prepare(batch, small));
    most = std::max(most, works.back().bytes);
  }
  // (the largest batch's memory before the first batch moves anything)
  void* ws;
  if (most && tt::workspace(most, &ws)) return -1;
  if (!params) return 0;
  for (Work& work : works) {
    if (run(work, q, steps)) return -1;
  }
  return 0;
} catch (const std::exception& e) {
  return tt::fail(-1, "muon_step: %s", e.what());
}

}  // extern "C"
