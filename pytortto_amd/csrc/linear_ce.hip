// Softmax cross entropy over a vocabulary, from features and the head's weight, without keeping the logits:
//
//   z = x W^T     M_i = max_v z_iv     S_i = sum_v e^(z_iv - M_i)     loss_i = ln S_i + M_i - z_i,t(i)
//   G_iv = g_i (e^(z_iv - M_i) / S_i - [v = t(i)])        dX = G W        dW = G^T x
//
// Positions are worked on in chunks.  Their rows come into the products' form; the first product leaves the logits in scratch memory
// (none without gradients) and, with the tile still in registers, every row's maximum and sum over a tile's columns; these are joined, and one
// pass turns the logits into G where they stand.  The two other products read it there: G^T needs no copy, see product.h.  So a
// training step has three products and not a fourth for logits that it forgot, and the scratch memory has a bound that the batch does not
// move: 2 GiB of logits, 2 GiB of features (twice that with gradients of float32), the weight's terms once or twice, and partial sums.
//
// float16: the weight is the products' operand as it is where its rows are multiples of 16 bytes, and features are but for positions without
// a target; G is rounded to float16 once, scaled by 2^14.  That is 11 bits of it: gradients are 2.3 to 3.0e-4 off (norms), of which
// 2.1 are the rounding of the result itself.  A second term would double the gradients' products, 3.5 of 6.4 ms at 4096 x 2048 x 131072.
// float32: operands have two float16 terms.  For the logits row i of x and row v of W are scaled by powers of two 2^-f_i and 2^-e_v to
// below 2^15, so that every position and every class has the digits that it would have alone.  In the gradients' products, where these rows
// are k, a scale of each row's own would have to be G's, and small rows' G would fall out of its range; there W and g x are scaled by one power
// of two each, and G is the bare softmax(z) - [v = t], times 2^15: its entries are held to 2^-22 of themselves and to 2^-40, whatever the
// rows they meet.
#include "product.h"
#include "rows.h"

#include <algorithm>

namespace {

using namespace tt;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr size_t kMostLogits = (size_t)2 << 30;     // bytes of a chunk's logits
constexpr size_t kMostStats = (size_t)256 << 20;
constexpr size_t kMostRows = (size_t)2 << 30;       // of a chunk's features in the products' form
constexpr int kTop = 14;                            // scaled values are below 2^(kTop + 1)
constexpr int kLowest = -1000;                      // an exponent below all
constexpr int kAny = -2000;                         // that of a row of zeros, or with what is not finite
constexpr int kTopGradient = 15;                    // the scale of G of float32

// Set at the start of a call, and most_f at that of a chunk, read by all that follows.
struct Control {
  double sum;           // of the losses of the chunks so far
  float scale;          // of the loss and its gradients: 1 / positions for 'mean'
  int most_e, most_f;   // the largest exponents of W's rows, and of x's rows with their g (float16: of g)
  Ticket done;
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

// Of float32, e and f are the exponents of W's rows and of those of x in the chunk.  (One block, with every row's behind each other: an atomic
// operation of each row where it is found took 9 ns of all the others, 10 us of 1064 rows.)
__global__ __launch_bounds__(1024) void lce_begin(Targets t, long long positions, long long first, long long rows, int mean, const int* __restrict__ e,
                                                  const int* __restrict__ f, const float* __restrict__ g, Control* c) {
  __shared__ long long part[16];
  __shared__ int part_e[16], part_f[16];
  long long n = 0;
  int most_e = e ? kLowest : 0, most_f = f || g ? kLowest : 0;
  const long long end = first ? first + rows : positions;
#pragma unroll 4
  for (long long i = first + threadIdx.x; i < end; i += 1024) {
    const bool kept = read_index(t.at, (size_t)i, t.wide) != t.ignore;
    n += kept;
    if (i >= first + rows) continue;
    const int own = f ? f[i - first] : 0;
    const float weight = g ? g[i] : 1.f;
    if (kept && own != kAny && weight != 0.f) most_f = max(most_f, g ? own + exponent(weight) : own);
  }
  const auto larger_int = [](int a, int b) { return max(a, b); };
  most_f = row_reduce<1024>(most_f, part_f, larger_int);
  if (first) {
    if (threadIdx.x == 0) c->most_f = most_f;
    return;
  }
  if (e) {
#pragma unroll 8
    for (int i = threadIdx.x; i < t.V; i += 1024) most_e = max(most_e, e[i]);
  }
  n = row_sum<1024>(n, part);
  most_e = row_reduce<1024>(most_e, part_e, larger_int);
  if (threadIdx.x == 0) {
    c->sum = 0.0;
    c->scale = !mean ? 1.f : n ? 1.f / (float)n : 0.f;
    c->most_e = most_e;
    c->most_f = most_f;
    c->done.n = 0;
  }
}

// Rows of x or W as the products' operands: two terms of float32, or a copy of float16.  Rows without a target are
// zeros, whatever they hold.  G threads have a row; of 16 G columns they keep it between its largest value and its terms.
// Both matrices share a launch: the first blocks have x's rows.  Bound by memory: 50021 + 777 rows of 1024 float32 69 us, 6.0 TB/s.
// A wave has a row of up to kWaveColumns, a block one of more (losses of 64 positions, 50021 float32 classes: of 512 features 83 us and 92 with a
// block, of 768 117 and 119, of 1024 158 and 151, of 2048 304 and 271).
constexpr int kWaveColumns = 768;
template <typename T>
struct Rows {
  const T* from;
  char* to;
  int* exponents;
  long long rows;
  Targets t;
  long long first;      // target of the first row
};
template <typename T, int G>
__global__ __launch_bounds__(256) void lce_rows(Rows<T> of_x, Rows<T> of_w, unsigned blocks_x, int columns, int ld) {
  __shared__ float part[256 / kWave];
  constexpr int kKept = 4;
  const bool second = blockIdx.x >= blocks_x;
  const Rows<T>& q = second ? of_w : of_x;
  const Targets t = q.t;
  const long long row = (long long)(blockIdx.x - (second ? blocks_x : 0)) * (256 / G) + row_of_block<G>();
  if (row >= q.rows) return;
  const int lane = threadIdx.x % G, quads = (columns + 63) / 64 * 16;
  const T* x = q.from + (size_t)row * columns;
  char* y = q.to + (size_t)row * ld;
  const bool kept = !t.at || class_of(t, q.first + row) != kIgnored, whole = columns % 4 == 0;
  const auto four = [&](int q) {
    typedef T Four __attribute__((ext_vector_type(4)));
    floatx4 v = {};
    if (!kept) return v;
    if (whole && q * 4 < columns) {
      const Four p = *reinterpret_cast<const Four*>(x + q * 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = widen(p[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (q * 4 + i < columns) v[i] = widen(x[q * 4 + i]);
    }
    return v;
  };
  floatx4 own[kKept];
#pragma unroll
  for (int k = 0; k < kKept; ++k) own[k] = lane + k * G < quads ? four(lane + k * G) : floatx4{};
  int e = 0;
  if (sizeof(T) == 4) {
    float m = 0.f;
    const auto look = [&](const floatx4& v) { m = fmaxf(m, fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])))); };
#pragma unroll
    for (int k = 0; k < kKept; ++k) look(own[k]);
    for (int q = lane + kKept * G; q < quads; q += G) look(four(q));
    m = row_max<G>(m, part);
    const bool counts = m > 0.f && __builtin_isfinite(m);
    e = counts ? exponent(m) - kTop - 1 : 0;
    if (lane == 0) q.exponents[row] = counts ? e : kAny;
  }
  const auto put = [&](int q, const floatx4& v) {
    if (sizeof(T) == 4) {
      store_terms(y, q * 4, floatx4{ldexpf(v[0], -e), ldexpf(v[1], -e), ldexpf(v[2], -e), ldexpf(v[3], -e)});
    } else {
      *reinterpret_cast<half4*>(y + q * 8) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    }
  };
#pragma unroll
  for (int k = 0; k < kKept; ++k)
    if (lane + k * G < quads) put(lane + k * G, own[k]);
  for (int q = lane + kKept * G; q < quads; q += G) put(q, four(q));
}

// x times g, and W, as operands of the gradients' products: float32 with one scale for the whole matrix.  G threads have a row.  Bound
// by memory: 32768 + 4096 rows of 1024 49 us, 6.1 TB/s.
struct Again {
  Rows<float> x, w;
  const float* g;       // of x's rows
  unsigned blocks_x, blocks;
  int columns, ld;
};
template <int G>
__device__ __forceinline__ void again_rows(const Again& a, unsigned block, const Control* __restrict__ control) {
  const bool second = block >= a.blocks_x;
  const Rows<float>& q = second ? a.w : a.x;
  const long long row = (long long)(block - (second ? a.blocks_x : 0)) * (256 / G) + row_of_block<G>();
  if (row >= q.rows) return;
  const float* g = a.g;
  const int columns = a.columns, ld = a.ld, quads = (columns + 63) / 64 * 16;
  const float* x = q.from + (size_t)row * columns;
  char* y = q.to + (size_t)row * ld;
  const bool kept = !q.t.at || class_of(q.t, q.first + row) != kIgnored, whole = columns % 4 == 0;
  // v 2^-first m 2^then: g's exponent is not multiplied with, so that nothing leaves the range on the way
  float m = 1.f;
  int first = 0, then = 0;
  if (second) {
    first = control->top_e();
  } else {
    first = q.exponents[row] == kAny ? 0 : q.exponents[row];
    then = first - control->top_f();
    if (g && kept) {
      m = g[row];
      const int e = exponent(m);
      m = ldexpf(m, -e);
      then += e;
    }
  }
  for (int k = threadIdx.x % G; k < quads; k += G) {
    floatx4 v = {};
    if (kept && whole && k * 4 < columns) {
      v = *reinterpret_cast<const floatx4*>(x + k * 4);
    } else if (kept) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k * 4 + i < columns) v[i] = x[k * 4 + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ldexpf(ldexpf(v[i], -first) * m, then);
    store_terms(y, k * 4, v);
  }
}

__device__ __forceinline__ void again_block(const Again& a, unsigned block, const Control* __restrict__ control) {
  if (a.columns <= kWaveColumns) again_rows<64>(a, block, control);
  else again_rows<256>(a, block, control);
}
__global__ __launch_bounds__(256) void lce_again(Again a, const Control* __restrict__ control) { again_block(a, blockIdx.x, control); }

// Columns of the logits, or rows of a gradient, that a launch has, and how many blocks of columns are in front of it.
struct Part {
  int first, end, blocks;
};

struct Logits {
  const int* f;         // exponents of x's rows and W's, of float32
  const int* e;
  Targets t;
  long long first;      // row of the chunk's first
  float* z;             // [rows][ld] or none
  long long ld;
  float2* stats;        // [rows][blocks]: of a tile's columns the largest logit, and the sum of e^(z - it) without its 1
  float* own;           // [rows] the target's logit, without z
  int blocks;
  float* partial;       // [splits][rows][ld] or none: the blocks that share a tile leave their sums here, for lce_few
  int per, splits;      // pairs for each
};

// One instruction each (fmaxf and fminf first quiet their arguments); the larger of a NaN and a number is the NaN.
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("v_maximum3_f32 %0, %1, %2, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float smaller(float a, float b) {
  float r;
  asm("v_min_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// What a lane and the one 16 (32) lanes away have, in the same order in both.
struct Pair {
  float a, b;
};
template <int APART>
__device__ __forceinline__ Pair with_lane(float v) {
  const unsigned x = __builtin_bit_cast(unsigned, v);
  const auto both = APART == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false) : __builtin_amdgcn_permlane32_swap(x, x, false, false);
  const unsigned a = both[0], b = both[1];      // (a cast of an element itself is one of the first element)
  return {__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)};
}

// A tile of logits, and its rows' maxima and sums.  Bound by the matrix instructions under the power limit, and by the logits it stores, which
// all blocks do at about the same time: 4096 x 2048 x 131072 float16 2.08 ms (1060 TFLOP/s), without a gradient to come 1.67 (1310);
// 4096 x 1024 x 32768 float32 664 us (three products counted 1240).  Dies that begin at different times, so that they store at
// different times, were 3 % slower.
template <int TERMS, int SIZE>
__global__ __launch_bounds__(256) void lce_logits(Operand x, Operand w, int rows, int V, int pairs, Logits q, Part part) {
  typedef Sized<TERMS, false, false, SIZE> G;
  extern __shared__ __align__(16) char lds[];
  int m, n;
  const int tile = xcd_remap(blockIdx.x, gridDim.x), blocks = gridDim.x / q.splits, split = tile / blocks;
  tile_at(tile % blocks, (rows + G::kM - 1) / G::kM, (part.end - part.first + G::kN - 1) / G::kN, &m, &n);
  const int m0 = m * G::kM, n0 = part.first + n * G::kN, at = threadIdx.x;
  if (SIZE == 0 && q.splits > 1) {
    const int first = split * q.per;
    float* to = q.partial + ((size_t)split * rows + m0) * q.ld + n0;
    G p;
    p.run(x, w, m0, n0, first, min(q.per, pairs - first), lds);
    p.rows(lds, [](int, int) { return 0; }, [&](int r, int c, const floatx4 (&v)[G::kAhead], int (&)[G::kAhead]) {
#pragma unroll
      for (int u = 0; u < G::kAhead; ++u)
        if (m0 + r + u * G::kStep < rows && n0 + c < q.ld) *reinterpret_cast<floatx4*>(to + (r + u * G::kStep) * q.ld + c) = v[u];
    });
    return;
  }
  // the rows' targets and exponents, and the columns' exponents
  int2 mine = make_int2(kInvalid, 0);
  int column_e = 0;
  if (at < G::kM && m0 + at < rows) mine = make_int2(class_of(q.t, q.first + m0 + at), TERMS == 2 ? q.f[m0 + at] : 0);
  if (TERMS == 2 && at < G::kN) column_e = q.e[n0 + at];      // (padded to a whole tile)
  G p;
  p.run(x, w, m0, n0, 0, pairs, lds);
  int2* about = reinterpret_cast<int2*>(lds + G::kExtra);
  int* scales = reinterpret_cast<int*>(about + G::kM);
  float2* halves = reinterpret_cast<float2*>(scales + G::kN);     // [2][kM] of a row's two waves
  if (at < G::kM) about[at] = mine;
  if (TERMS == 2 && at < G::kN) scales[at] = column_e;
  __syncthreads();
  const int c0 = G::column();
  int4 scale[G::kAcross];
  if (TERMS == 2) {
#pragma unroll
    for (int j = 0; j < G::kAcross; ++j) scale[j] = *reinterpret_cast<const int4*>(scales + c0 + j * 16);
  }
  // A row's columns in this wave are in four lanes, 4 NT of them in a thread: little is left between lanes.  (Row by row, with the row
  // across a wave, the reductions were most of 12 us that a tile of 256 x 256 took behind its product.)
#pragma unroll
  for (int i = 0; i < G::kDown; ++i) {
    const int r = G::row() + i * 16;
    const int2 it = about[r];
    float v[G::kAcross * 4];
#pragma unroll
    for (int j = 0; j < G::kAcross; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[j * 4 + e] = p.acc[i][j][e];
        if (TERMS == 2) v[j * 4 + e] = ldexpf(v[j * 4 + e], (&scale[j].x)[e] + it.y);
      }
    const int here = it.x - n0 - c0;
    if (!q.z && here >= 0 && here < G::kAcross * 16 && (here & 12) == 0) {
      float own = 0.f;
#pragma unroll
      for (int k = 0; k < G::kAcross * 4; ++k)
        if (here == (k >> 2) * 16 + (k & 3)) own = v[k];
      q.own[m0 + r] = own;
    }
    if (n0 + G::kN > V) {
#pragma unroll
      for (int k = 0; k < G::kAcross * 4; ++k)
        if (n0 + c0 + (k >> 2) * 16 + (k & 3) >= V) v[k] = -INFINITY;
    }
    // the largest goes up, and all others stay: the sum is over these
    float top = v[0];
#pragma unroll
    for (int k = 1; k < G::kAcross * 4; ++k) {
      const float other = smaller(top, v[k]);
      top = larger(top, v[k]);
      v[k] = other;
    }
    const Pair one = with_lane<16>(top), two = with_lane<32>(larger(one.a, one.b));
    const float most = larger(two.a, two.b), from = most == -INFINITY ? 0.f : most;
    float sum = 0.f;
#pragma unroll
    for (int k = 1; k < G::kAcross * 4; ++k) sum += __builtin_amdgcn_exp2f((v[k] - from) * kLog2e);
    const Pair four = with_lane<16>(sum);
    sum = four.a + four.b + __builtin_amdgcn_exp2f((smaller(one.a, one.b) - from) * kLog2e);
    const Pair all = with_lane<32>(sum);
    sum = all.a + all.b + __builtin_amdgcn_exp2f((smaller(two.a, two.b) - from) * kLog2e);
    if ((at & 48) == 0) halves[(at >> 6 & 1) * G::kM + r] = make_float2(most, sum);
  }
  __syncthreads();
  if (at < G::kM && m0 + at < rows) {
    const float2 a = halves[at], b = halves[G::kM + at];
    const float2 more = a.x < b.x ? b : a, less = a.x < b.x ? a : b;
    const float rest = more.y + (1.f + less.y) * (a.x == b.x ? 1.f : __builtin_amdgcn_exp2f((less.x - more.x) * kLog2e));
    q.stats[(size_t)(m0 + at) * q.blocks + part.blocks + n] = make_float2(more.x, rest);
  }
  if (!q.z) return;
  // (past the caches, here and in lce_product: 2047 x 1000 x 50021 float16 with gradients 1086 -> 1061 us)
  float* z = q.z + (size_t)m0 * q.ld + n0;
  const int ld = (int)q.ld;
  const int4 mine4 = TERMS == 2 ? *reinterpret_cast<const int4*>(scales + (at & 63) % G::kLanes * 4) : int4{};
  p.rows(lds, [](int, int) { return 0; }, [&](int r, int c, floatx4 (&v)[G::kAhead], int (&)[G::kAhead]) {
#pragma unroll
    for (int u = 0; u < G::kAhead; ++u) {
      const int k = r + u * G::kStep;
      if (TERMS == 2) {
        // (again: written back to the accumulators, they would need as many registers more)
        const int e = about[k].y;
        v[u] = floatx4{ldexpf(v[u][0], mine4.x + e), ldexpf(v[u][1], mine4.y + e), ldexpf(v[u][2], mine4.z + e), ldexpf(v[u][3], mine4.w + e)};
      }
      if (m0 + k < rows && n0 + c < ld) __builtin_nontemporal_store(v[u], reinterpret_cast<floatx4*>(z + (unsigned)(k * ld + c)));
    }
  });
}

// The loss of all positions, in the order of the positions: those of a chunk are added to what the chunks in front of it have left.
struct Total {
  float* to;            // or none
  long long n;
  int mean, last;       // the last chunk's
  Control* control;
};
template <int THREADS, typename L>
__device__ __forceinline__ void total(const Total& q, L loss) {
  __shared__ double part[THREADS / kWave];
  double s = 0.0;
  for (long long i = threadIdx.x; i < q.n; i += THREADS) s += (double)loss(i);
  s = row_sum<THREADS>(s, part);
  if (threadIdx.x) return;
  s += q.control->sum;
  if (!q.last) q.control->sum = s;
  else *q.to = q.mean && q.control->scale == 0.f ? NAN : (float)(s * (double)q.control->scale);
}
// The same by the last of `blocks` blocks, each of which has shared some.  (Of few: a launch less.)
__device__ __forceinline__ void total_by_last(const Total& q, const float* loss, unsigned blocks) {
  __shared__ bool last;
  stores_done();
  __syncthreads();
  if (threadIdx.x == 0) last = last_ticket(&q.control->done, blocks);
  __syncthreads();
  if (last) total<256>(q, [&](long long i) { return shared(loss + i); });
}

// The logarithm of a row's sum, without its largest term in `rest`.  With a logit of +inf, or none but -inf, there is none: inf - inf.
__device__ __forceinline__ float log_of_sum(float most, float rest) { return __builtin_isinf(most) ? NAN : log1pf(rest); }

// A row's maximum and log2 of its sum from those of its blocks, and its loss.  A wave has a row.  The sum is kept without the
// largest term, which is 1: of a target that has nearly all of the probability, the loss is what is left, and keeps its digits.
__device__ __forceinline__ void join_row(const float2* __restrict__ stats, const float* __restrict__ own, const float* __restrict__ z, long long ld,
                                         float2* __restrict__ of, float* __restrict__ loss, const Targets& t, long long first, int r, int blocks) {
  const int lane = threadIdx.x & 63, target = class_of(t, first + r);
  if (target == kIgnored) {
    if (lane == 0) share(loss + r, 0.f);
    return;
  }
  const float2* s = stats + (size_t)r * blocks;
  float most = -INFINITY;
  for (int b = lane; b < blocks; b += 64) most = fmaxf(most, s[b].x);
  most = lanes_reduce<64>(most, Larger());
  const float from = most == -INFINITY ? 0.f : most;
  float rest = 0.f;
  int largest = 0;
  for (int b = lane; b < blocks; b += 64) {
    const float2 v = s[b];
    const bool it = v.x == most;
    largest += it;
    rest += it ? v.y : (1.f + v.y) * __builtin_amdgcn_exp2f((v.x - from) * kLog2e);
  }
  rest = lanes_reduce<64>(rest, Plus()) + (float)(lanes_reduce<64>(largest, Plus()) - 1);
  if (lane == 0) {
    const float log_sum = log_of_sum(most, rest);
    of[r] = make_float2(from, log_sum * kLog2e);
    share(loss + r, target == kInvalid ? NAN : log_sum + (from - (z ? z[(size_t)r * ld + target] : own[r])));
  }
}
__global__ __launch_bounds__(256) void lce_join(const float2* __restrict__ stats, const float* __restrict__ own, const float* __restrict__ z,
                                                long long ld, float2* __restrict__ of, float* __restrict__ loss, Targets t, long long first,
                                                int rows, int blocks, Total all) {
  const int r = blockIdx.x * 4 + row_of_block<kWave>();
  if (r < rows) join_row(stats, own, z, ld, of, loss, t, first, r, blocks);
  if (all.to) total_by_last(all, loss, gridDim.x);
}
// What a row's G is multiplied with: float32's weight of the position comes in with x, or behind the product.
template <int TERMS>
__device__ __forceinline__ float factor_of(const Control* control, const float* g, long long i) {
  return TERMS == 2 ? (float)(1 << kTopGradient) : ldexpf(g ? g[i] : 1.f, kTop - control->top_f());
}

// A row of G: 32 floats of the logits' row are first and second terms, or 64 are values as halves and a gap.
template <int TERMS>
__device__ __forceinline__ void store_gradient(const floatx4& v, float* z, int c) {
  char* row = reinterpret_cast<char*>(z);
  if (TERMS == 2) store_terms(row, c, v);
  else *reinterpret_cast<half4*>(row + (c >> 6) * (2 * kLine) + (c & 63) * 2) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
}
// Four logits of a row, from column c on, become G.
template <int TERMS>
__device__ __forceinline__ void put_gradient(floatx4 v, float* z, int c, int V, int target, float most, float log_sum, float loss, float factor) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int column = c + i;
    float p = __builtin_amdgcn_exp2f((v[i] - most) * kLog2e - log_sum);
    if (column == target) p = expm1f(-loss);
    if (target == kInvalid) p = NAN;
    v[i] = column < V ? p * factor : 0.f;
  }
  store_gradient<TERMS>(v, z, c);
}

// The logits of a chunk become G, where they stand.  Bound by memory: 4096 x 131072, float16 530 us (6.1 TB/s: half of G's line stays as it is),
// 4096 x 32768 float32 165 us (6.5 TB/s).
template <int TERMS>
__global__ __launch_bounds__(256) void lce_gradient(float* __restrict__ z, long long ld, const float2* __restrict__ of,
                                                    const float* __restrict__ loss, const float* __restrict__ g, Targets t,
                                                    long long first, int V, const Control* __restrict__ control) {
  const int r = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= ld) return;
  float* at = z + (size_t)r * ld;
  const int target = class_of(t, first + r);
  if (target == kIgnored) {
    store_gradient<TERMS>(floatx4{}, at, c);
    return;
  }
  const floatx4 v = *reinterpret_cast<const floatx4*>(at + c);
  const float2 s = of[r];
  put_gradient<TERMS>(v, at, c, V, target, s.x, s.y, loss[r], factor_of<TERMS>(control, g, first + r));
}

// What lce_join and lce_gradient do, and the logits from the sums of the blocks that shared their tiles: of few rows over few classes,
// where the reduction is what there is to share out (64 x 2048 x 1000 float32: 16 tiles of 64 x 64 and the two kernels took 32 us, 128 shares
// and this 15).  A block has a row; of 4096 columns it keeps the logits in registers.
template <int TERMS>
__device__ __forceinline__ void few_row(const Logits& q, int rows, int V, const float* __restrict__ g, float* __restrict__ loss,
                                        const Control* __restrict__ control) {
  __shared__ float part[3][256 / kWave];
  __shared__ float own;
  constexpr int kKept = 4;
  const int r = blockIdx.x, target = class_of(q.t, r), quads = (int)(q.ld / 4);
  float* z = q.z ? q.z + (size_t)r * q.ld : nullptr;
  const int f = TERMS == 2 ? q.f[r] : 0;
  const auto logits = [&](int k) {
    floatx4 v = {};
#pragma unroll 4
    for (int s = 0; s < q.splits; ++s) v += *reinterpret_cast<const floatx4*>(q.partial + ((size_t)s * rows + r) * q.ld + k * 4);
    const int4 e = TERMS == 2 ? *reinterpret_cast<const int4*>(q.e + k * 4) : int4{};
    if (TERMS == 2) v = floatx4{ldexpf(v[0], e.x + f), ldexpf(v[1], e.y + f), ldexpf(v[2], e.z + f), ldexpf(v[3], e.w + f)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (k * 4 + i >= V) v[i] = -INFINITY;
      if (k * 4 + i == target) own = v[i];
    }
    return v;
  };
  floatx4 kept[kKept];
  if (target != kIgnored) {
    float most = -INFINITY, sum = 0.f;
    int largest = 0;
    const auto look = [&](const floatx4& v) { most = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), most); };
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
      kept[k] = (int)threadIdx.x + k * 256 < quads ? logits(threadIdx.x + k * 256) : floatx4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      look(kept[k]);
    }
    for (int k = threadIdx.x + kKept * 256; k < quads; k += 256) look(logits(k));
    most = row_max<256>(most, part[0]);
    const float from = most == -INFINITY ? 0.f : most;
    const auto add = [&](const floatx4& v, int k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool it = v[i] == most;
        largest += it && k * 4 + i < V;
        sum += it ? 0.f : __builtin_amdgcn_exp2f((v[i] - from) * kLog2e);
      }
    };
#pragma unroll
    for (int k = 0; k < kKept; ++k) add(kept[k], threadIdx.x + k * 256);
    for (int k = threadIdx.x + kKept * 256; k < quads; k += 256) add(logits(k), k);
    const float rest = row_sum<256>(sum, part[1]) + (float)(row_sum<256>(largest, reinterpret_cast<int*>(part[2])) - 1);
    const float log_sum = log_of_sum(most, rest), mine = target == kInvalid ? NAN : log_sum + (from - own);
    if (threadIdx.x == 0) share(loss + r, mine);
    if (!z) return;
    const float factor = factor_of<TERMS>(control, g, r);
    const auto put = [&](const floatx4& v, int k) { put_gradient<TERMS>(v, z, k * 4, V, target, from, log_sum * kLog2e, mine, factor); };
#pragma unroll
    for (int k = 0; k < kKept; ++k)
      if ((int)threadIdx.x + k * 256 < quads) put(kept[k], threadIdx.x + k * 256);
    for (int k = threadIdx.x + kKept * 256; k < quads; k += 256) put(logits(k), k);
    return;
  }
  if (threadIdx.x == 0) share(loss + r, 0.f);
  if (!z) return;
  for (int k = threadIdx.x; k < quads; k += 256) store_gradient<TERMS>(floatx4{}, z, k * 4);
}
// Blocks behind the rows' bring x and W into the form of the gradients' products: a launch less.
template <int TERMS>
__global__ __launch_bounds__(256) void lce_few(Logits q, int rows, int V, const float* __restrict__ g, float* __restrict__ loss,
                                               const Control* __restrict__ control, Total all, Again again) {
  if ((int)blockIdx.x >= rows) {
    if (TERMS == 2) again_block(again, blockIdx.x - rows, control);
    return;
  }
  few_row<TERMS>(q, rows, V, g, loss, control);
  if (all.to) total_by_last(all, loss, rows);
}

// What the two gradients' products do with their sums: take the scales back, and store them as float32 (to or on top of what is there)
// or float16; or leave partial sums for lce_sum.
enum Of { kHalf, kPositions, kClasses };      // float16 operands; rows of float32's dX; rows of its dW
struct Scale {
  float s;
  int e;
};
struct GradientOut {
  void* to;
  Of of;
  const float* g;           // of the rows, if they are positions
  Targets t;
  long long first;          // row of the first position
  const Control* control;
  int half, add;
  int columns;
  // What a row's sums are multiplied with: s 2^e.
  __device__ __forceinline__ Scale scale_of(int row) const {
    const float s = control->scale;
    if (of == kHalf) return {s, control->top_f() - kTop};
    if (of == kClasses) return {s, control->top_f() - kTopGradient};
    if (!g || class_of(t, first + row) == kIgnored) return {s, control->top_e() - kTopGradient};
    const float weight = g[row];
    const int e = exponent(weight);
    return {s * ldexpf(weight, -e), control->top_e() - kTopGradient + e};
  }
  // What stands there, to be added to.
  __device__ __forceinline__ floatx4 before(int row, int c) const {
    const size_t at = (size_t)row * columns + c;
    const float* p = reinterpret_cast<const float*>(to) + at;
    floatx4 v = {};
    if (columns - c >= 4 && (at & 3) == 0) return *reinterpret_cast<const floatx4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < columns - c) v[i] = p[i];
    return v;
  }
  __device__ __forceinline__ void store(int row, int c, floatx4 v, const Scale& q, const floatx4& old) const {
    const size_t at = (size_t)row * columns + c;
    const int n = columns - c;
    const bool whole = n >= 4 && (at & 3) == 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ldexpf(v[i] * q.s, q.e);
    v += old;
    if (half) {
      _Float16* p = reinterpret_cast<_Float16*>(to) + at;
      if (whole) {
        *reinterpret_cast<half4*>(p) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) p[i] = (_Float16)v[i];
      }
    } else {
      float* p = reinterpret_cast<float*>(to) + at;
      if (whole) {
        *reinterpret_cast<floatx4*>(p) = v;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < n) p[i] = v[i];
      }
    }
  }
};

// A tile of dX = G W or dW = G^T x.  Bound as lce_logits is: of 4096 x 2048 x 131072 float16 1.56 ms (dX, 1410 TFLOP/s) and 1.95 (dW, 1130: a
// reduction of 64 pairs, and 1.1 GB of sums to store), of 4096 x 1024 x 32768 float32 535 and 563 us (1540 and 1460).
template <int TERMS, bool A_ACROSS, int SIZE>
__global__ __launch_bounds__(256) void lce_product(Operand a, Operand b, int M, int N, int pairs, int per, int splits, float* partial,
                                                   GradientOut out, Part part) {
  typedef Sized<TERMS, A_ACROSS, true, SIZE> G;
  extern __shared__ __align__(16) char lds[];
  const int tile = xcd_remap(blockIdx.x, gridDim.x), blocks = gridDim.x / splits, split = tile / blocks;
  int m, n;
  tile_at(tile % blocks, (part.end - part.first + G::kM - 1) / G::kM, (N + G::kN - 1) / G::kN, &m, &n);
  const int first = split * per, count = min(per, pairs - first), m0 = part.first + m * G::kM, n0 = n * G::kN;
  const Scale mine = splits == 1 && threadIdx.x < G::kM && m0 + (int)threadIdx.x < M ? out.scale_of(m0 + threadIdx.x) : Scale{};
  G p;
  p.run(a, b, m0, n0, first, count, lds);
  if (splits > 1) {
    const long long ld = (N + 3) / 4 * 4;
    float* to = partial + ((size_t)split * M + m0) * ld + n0;
    p.rows(lds, [](int, int) { return 0; }, [&](int r, int c, const floatx4 (&v)[G::kAhead], int (&)[G::kAhead]) {
#pragma unroll
      for (int u = 0; u < G::kAhead; ++u)
        if (m0 + r + u * G::kStep < M && n0 + c < N) *reinterpret_cast<floatx4*>(to + (r + u * G::kStep) * ld + c) = v[u];
    });
    return;
  }
  Scale* about = reinterpret_cast<Scale*>(lds + G::kExtra);
  if (threadIdx.x < G::kM) about[threadIdx.x] = mine;
  __syncthreads();
  const auto none = [](int, int) { return 0; };
  if (out.columns % 4) {
    // rows of any alignment
    p.rows(lds, [&](int r, int c) { return out.add && m0 + r < M && n0 + c < N ? out.before(m0 + r, n0 + c) : floatx4{}; },
           [&](int r, int c, const floatx4 (&v)[G::kAhead], const floatx4 (&old)[G::kAhead]) {
#pragma unroll
             for (int u = 0; u < G::kAhead; ++u) {
               const int k = r + u * G::kStep;
               if (m0 + k < M && n0 + c < N) out.store(m0 + k, n0 + c, v[u], about[k], old[u]);
             }
           });
    return;
  }
  // of four columns all are there or none, and every four can be stored at once
  const auto scaled = [&](const floatx4& v, int k) {
    const Scale q = about[k];
    return floatx4{ldexpf(v[0] * q.s, q.e), ldexpf(v[1] * q.s, q.e), ldexpf(v[2] * q.s, q.e), ldexpf(v[3] * q.s, q.e)};
  };
  const size_t corner = (size_t)m0 * out.columns + n0;
  if (out.half) {
    _Float16* to = reinterpret_cast<_Float16*>(out.to) + corner;
    p.rows(lds, none, [&](int r, int c, const floatx4 (&v)[G::kAhead], const int (&)[G::kAhead]) {
#pragma unroll
      for (int u = 0; u < G::kAhead; ++u) {
        const int k = r + u * G::kStep;
        const floatx4 s = scaled(v[u], k);
        if (m0 + k < M && n0 + c < N)
          *reinterpret_cast<half4*>(to + (unsigned)(k * out.columns + c)) = half4{(_Float16)s[0], (_Float16)s[1], (_Float16)s[2], (_Float16)s[3]};
      }
    });
    return;
  }
  float* to = reinterpret_cast<float*>(out.to) + corner;
  if (out.add) {
    p.rows(lds,
           [&](int r, int c) {
             return m0 + r < M && n0 + c < N ? *reinterpret_cast<const floatx4*>(to + (unsigned)(r * out.columns + c)) : floatx4{};
           },
           [&](int r, int c, const floatx4 (&v)[G::kAhead], const floatx4 (&old)[G::kAhead]) {
#pragma unroll
             for (int u = 0; u < G::kAhead; ++u) {
               const int k = r + u * G::kStep;
               const floatx4 s = scaled(v[u], k) + old[u];
               if (m0 + k < M && n0 + c < N) __builtin_nontemporal_store(s, reinterpret_cast<floatx4*>(to + (unsigned)(k * out.columns + c)));
             }
           });
    return;
  }
  p.rows(lds, none, [&](int r, int c, const floatx4 (&v)[G::kAhead], const int (&)[G::kAhead]) {
#pragma unroll
    for (int u = 0; u < G::kAhead; ++u) {
      const int k = r + u * G::kStep;
      const floatx4 s = scaled(v[u], k);
      if (m0 + k < M && n0 + c < N) __builtin_nontemporal_store(s, reinterpret_cast<floatx4*>(to + (unsigned)(k * out.columns + c)));
    }
  });
}

// The sums of the blocks that shared a reduction.  (A later chunk's are added to what the chunks in front of it have left, as lce_product's are.)
__global__ __launch_bounds__(256) void lce_sum(const float* __restrict__ partial, int splits, int M, int N, GradientOut out) {
  const int quads = (N + 3) / 4;
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= (long long)M * quads) return;
  floatx4 v = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const floatx4*>(partial + ((size_t)s * M * quads + at) * 4);
  const int row = (int)(at / quads), c = (int)(at % quads) * 4;
  out.store(row, c, v, out.scale_of(row), out.add ? out.before(row, c) : floatx4{});
}

__global__ __launch_bounds__(1024) void lce_loss(const float* __restrict__ loss, Total all) {
  total<1024>(all, [&](long long i) { return loss[i]; });
}

// g (none: 1) times a float32 gradient, as float32 or float16.  Bound by memory: 131072 x 2048 to float16 5.1 TB/s.
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

template <typename T>
void launch_rows(const Rows<T>& x, const Rows<T>& w, int columns, int ld) {
  // (of kMostRows bytes of rows and 2^20 classes: below 2^32 threads, which is all that a launch can have)
  const int side = columns <= kWaveColumns ? 4 : 1;
  const unsigned blocks_x = (unsigned)((x.rows + side - 1) / side), blocks = blocks_x + (unsigned)((w.rows + side - 1) / side);
  if (side == 4) lce_rows<T, 64><<<blocks, 256, 0, stream()>>>(x, w, blocks_x, columns, ld);
  else lce_rows<T, 256><<<blocks, 256, 0, stream()>>>(x, w, blocks_x, columns, ld);
}

Again again_of(const Rows<float>& x, const Rows<float>& w, const float* g, int columns, int ld) {
  const int side = columns <= kWaveColumns ? 4 : 1;
  const unsigned blocks_x = (unsigned)((x.rows + side - 1) / side);
  return {x, w, g, blocks_x, blocks_x + (unsigned)((w.rows + side - 1) / side), columns, ld};
}

// Where the tiles are not whole rounds over the compute units and few are left for the last one, the last columns (of n, m the other side)
// are left to smaller tiles, in a launch behind the others': the first of these columns.  (777 x 1024 x 50021 float32, 784 tiles of 256 x 256:
// the logits took 283 us; 768 of them take 232 and 208 of 64 x 64 behind them 16.)  Few are a quarter of the units at most, and half of them where
// they begin with a whole column of tiles: losses of 1024 x 512 x 20000 float32, 60 left, 88 us and 106 as they are; of 5000 x 1024 x 7500 float16, 88
// left, 122 and 116 as they are.
long long first_left(long long m, long long n, int size) {
  const long long side = kTileSide[size], high = (m + side - 1) / side, wide = (n + side - 1) / side, units = compute_units();
  const long long rounds = high * wide / units, rest = high * wide % units;
  if (size == 0 || rounds == 0 || rest == 0 || rest > units / 4) return n;
  const long long kept = rounds * units / high;
  return kept > 0 && (wide - kept) * high <= units / 2 ? kept * side : n;
}
int size_left(long long m, long long n, int size) { return std::min(tile_size(m, n), size - 1); }

template <int TERMS, int SIZE>
int launch_logits(const Operand& x, const Operand& w, int rows, int V, int H, const Logits& q, const Part& part) {
  typedef Sized<TERMS, false, false, SIZE> G;
  TT_ALLOW_LDS((lce_logits<TERMS, SIZE>), G::kLds);
  lce_logits<TERMS, SIZE><<<(unsigned)(tiles_of(rows, part.end - part.first, SIZE) * q.splits), G::kThreads, G::kLds, stream()>>>(
      x, w, rows, V, (int)(padded(H) / (64 / TERMS)), q, part);
  TT_LAUNCH_CHECK();
  return 0;
}
template <int TERMS>
int launch_logits(int size, const Operand& x, const Operand& w, int rows, int V, int H, const Logits& q, const Part& part) {
  switch (size) {
    case 2: return launch_logits<TERMS, 2>(x, w, rows, V, H, q, part);
    case 1: return launch_logits<TERMS, 1>(x, w, rows, V, H, q, part);
    default: return launch_logits<TERMS, 0>(x, w, rows, V, H, q, part);
  }
}

// How a gradient's product [m, n] over `pairs` is cut: the size of its tiles, and how many blocks share one.
struct Plan {
  int size, per, splits;      // pairs for each block, blocks
};
Plan plan_product(long long m, long long n, long long pairs) {
  Plan p;
  p.size = tile_size(m, n);
  // Few tiles and a long reduction: large tiles shared by several blocks, sixteen pairs to each unit.  (Losses with gradients: of 8192 x 768 x 2000
  // float16 185 us, 217 without; of 8192 x 1024 x 512 107, 112 without or from 256 pairs on, 115 where four pairs are enough; of 1024 x 1024 x 2400
  // float32 107, 105 and 118.)
  while (p.size < 2 && pairs >= 64 && tiles_of(m, n, p.size + 1) * (pairs / 16) >= compute_units() && std::min(m, n) > kTileSide[p.size]) ++p.size;
  const long long tiles = tiles_of(m, n, p.size);
  long long splits = compute_units() / tiles;
  // (eight pairs or more to a block: of 8192 x 1024 x 512 float16 107 us, 122 with four and 113 with 32; of 4096 x 256 x 512 float32 66, 66 and 71)
  splits = std::max(1LL, std::min(splits, pairs / 8));
  p.per = (int)((pairs + splits - 1) / splits);
  p.splits = (int)((pairs + p.per - 1) / p.per);
  return p;
}

template <int TERMS, bool A_ACROSS, int SIZE>
int launch_product(const Operand& a, const Operand& b, int M, int N, int pairs, int per, float* partial, const GradientOut& out, const Part& part) {
  typedef Sized<TERMS, A_ACROSS, true, SIZE> G;
  TT_ALLOW_LDS((lce_product<TERMS, A_ACROSS, SIZE>), G::kLds);
  const int splits = (pairs + per - 1) / per;      // (fewer for a chunk that is not whole)
  lce_product<TERMS, A_ACROSS, SIZE><<<(unsigned)(tiles_of(part.end - part.first, N, SIZE) * splits), G::kThreads, G::kLds, stream()>>>(
      a, b, M, N, pairs, per, splits, partial, out, part);
  TT_LAUNCH_CHECK();
  if (splits > 1) {
    const long long quads = (long long)M * ((N + 3) / 4);
    lce_sum<<<(unsigned)((quads + 255) / 256), 256, 0, stream()>>>(partial, splits, M, N, out);
    TT_LAUNCH_CHECK();
  }
  return 0;
}
template <int TERMS, bool A_ACROSS>
int launch_product(int size, const Operand& a, const Operand& b, int M, int N, int pairs, int per, float* partial, const GradientOut& out,
                   const Part& part) {
  switch (size) {
    case 2: return launch_product<TERMS, A_ACROSS, 2>(a, b, M, N, pairs, per, partial, out, part);
    case 1: return launch_product<TERMS, A_ACROSS, 1>(a, b, M, N, pairs, per, partial, out, part);
    default: return launch_product<TERMS, A_ACROSS, 0>(a, b, M, N, pairs, per, partial, out, part);
  }
}
template <int TERMS, bool A_ACROSS>
int launch_product(const Plan& plan, const Operand& a, const Operand& b, int M, int N, int pairs, float* partial, const GradientOut& out) {
  const int end = plan.splits > 1 ? M : (int)first_left(N, M, plan.size);
  if (launch_product<TERMS, A_ACROSS>(plan.size, a, b, M, N, pairs, plan.per, partial, out, Part{0, end, 0})) return -1;
  if (end == M) return 0;
  return launch_product<TERMS, A_ACROSS>(size_left(N, M - end, plan.size), a, b, M, N, pairs, plan.per, partial, out, Part{end, M, 0});
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
  const int depth = 64 / TERMS;
  const size_t most = std::min(grad ? kMostLogits / ((size_t)Vp * 4) : kMostStats / ((size_t)Vp / 8), kMostRows / ((size_t)Hp * 2 * TERMS));
  const long long chunk = std::min(N, std::max(256LL, (long long)most / 256 * 256));
  const bool several = chunk < N;
  const int pairsV = (int)(Vp / depth), pairsN = (int)((chunk + depth - 1) / depth);
  const int size = tile_size(chunk, V), V1 = (int)first_left(chunk, V, size), left = V1 < V ? size_left(chunk, V - V1, size) : size;
  const int blocks1 = (V1 + kTileSide[size] - 1) / kTileSide[size], blocks = blocks1 + (V - V1 + kTileSide[left] - 1) / kTileSide[left];
  // (the reduction of few small tiles is shared out, eight pairs or more to a block: fewer would be loads on their way and little else, though a whole call
  // is as long with two to sixteen)
  const int pairsH = (int)(Hp / depth);
  int splits = size || several ? 1 : (int)std::max(1LL, std::min(compute_units() / tiles_of(chunk, V, 0), (long long)pairsH / 8));
  const int per = (pairsH + splits - 1) / splits;
  splits = (pairsH + per - 1) / per;
  const Plan plan_x = plan_product(chunk, H, pairsV), plan_w = plan_product(V, H, pairsN);

  Carve c;
  const size_t at_control = c.take(sizeof(Control)), at_f = c.take(TERMS == 2 ? 4 * chunk : 0), at_e = c.take(TERMS == 2 ? 4 * (size_t)(V + 256) : 0);
  const size_t at_x = c.take((size_t)chunk * Hp * 2 * TERMS), at_w = c.take(copy_w ? (size_t)V * Hp * 2 * TERMS : 0);
  const size_t at_x2 = c.take(TERMS == 2 && q.dw ? (size_t)chunk * Hp * 4 : 0), at_w2 = c.take(TERMS == 2 && q.dx ? (size_t)V * Hp * 4 : 0);
  const size_t at_stats = c.take((size_t)chunk * blocks * 8), at_own = c.take(4 * chunk), at_of = c.take(8 * chunk);
  const size_t at_loss = c.take(4 * chunk), at_z = c.take(grad ? (size_t)chunk * Vp * 4 : 0);
  const size_t part_x = q.dx && plan_x.splits > 1 ? (size_t)plan_x.splits * chunk * ((H + 3) / 4) * 16 : 0;
  const size_t part_w = q.dw && plan_w.splits > 1 ? (size_t)plan_w.splits * V * ((H + 3) / 4) * 16 : 0;
  const size_t part_z = splits > 1 ? (size_t)splits * chunk * Vp * 4 : 0;
  const size_t at_part = c.take(std::max({part_x, part_w, part_z}));
  const size_t at_sum = c.take(several && q.half_out && q.dw ? (size_t)V * H * 4 : 0);
  void* ws;
  if (tt::workspace(c.bytes, &ws)) return -1;
  char* base = (char*)ws;
  Control* control = (Control*)(base + at_control);
  int *f = TERMS == 2 ? (int*)(base + at_f) : nullptr, *e = TERMS == 2 ? (int*)(base + at_e) : nullptr;
  float *z = grad ? (float*)(base + at_z) : nullptr, *partial = (float*)(base + at_part);
  float2 *stats = (float2*)(base + at_stats), *of = (float2*)(base + at_of);
  float* own = (float*)(base + at_own);

  const int ldx = (int)(Hp * 2 * TERMS);
  const Operand w = copy_w ? Operand{base + at_w, (long long)V * ldx, ldx, kLine}
                           : Operand{(const char*)q.w, (long long)V * H * 2, H * 2, kLine, H % 64 ? H / 64 : -1, H % 64 / 8};
  Operand w_gradient = w;
  if (TERMS == 2) w_gradient.at = base + at_w2;
  // (of at most as many blocks as there are at one time: each counts itself, 9 ns of the others' time)
  const bool at_once = !several && (splits > 1 ? N : (N + 3) / 4) <= 256;
  for (long long first = 0; first < N; first += chunk) {
    const int rows = (int)std::min(chunk, N - first);
    const T* from = (const T*)q.x + (size_t)first * H;
    const Targets none = {nullptr, 0, 0, 0};
    launch_rows<T>({from, base + at_x, f, rows, q.t, first}, {(const T*)q.w, base + at_w, e, copy_w && first == 0 ? V : 0, none, 0}, H, ldx);
    TT_LAUNCH_CHECK();
    if (first == 0 || (grad && (f || q.g))) {
      lce_begin<<<1, 1024, 0, stream()>>>(q.t, N, first, rows, mean, e, f, q.g, control);
      TT_LAUNCH_CHECK();
    }
    Again again = {};
    if constexpr (TERMS == 2) {
      again = again_of({from, base + at_x2, f, q.dw ? rows : 0, q.t, first}, {(const float*)q.w, base + at_w2, nullptr, q.dx && first == 0 ? V : 0, none, 0},
                       q.g ? q.g + first : nullptr, H, ldx);
      if (again.blocks && splits == 1) lce_again<<<again.blocks, 256, 0, stream()>>>(again, control);
      TT_LAUNCH_CHECK();
    }
    const Operand x = {base + at_x, (long long)rows * ldx, ldx, kLine};
    float* losses = q.reduction == 0 && q.loss ? q.loss + first : (float*)(base + at_loss);
    const Total all = {q.reduction ? q.loss : nullptr, rows, mean, first + rows == N, control}, by_last = at_once ? all : Total{};
    const Logits logits = {f, e, q.t, first, z, Vp, stats, own, blocks, partial, per, splits};
    if (launch_logits<TERMS>(size, x, w, rows, V, H, logits, Part{0, V1, 0})) return -1;
    if (V1 < V && launch_logits<TERMS>(left, x, w, rows, V, H, logits, Part{V1, V, blocks1})) return -1;
    if (splits > 1) lce_few<TERMS><<<(unsigned)rows + again.blocks, 256, 0, stream()>>>(logits, rows, V, q.g, losses, control, by_last, again);
    else lce_join<<<(unsigned)((rows + 3) / 4), 256, 0, stream()>>>(stats, own, z, Vp, of, losses, q.t, first, rows, blocks, by_last);
    TT_LAUNCH_CHECK();
    if (all.to && !at_once) {
      lce_loss<<<1, 1024, 0, stream()>>>(losses, all);
      TT_LAUNCH_CHECK();
    }
    if (!grad) continue;
    for (int r = splits > 1 ? rows : 0; r < rows; r += 65535) {
      const int some = std::min(rows - r, 65535);
      lce_gradient<TERMS><<<dim3((unsigned)((Vp / 4 + 255) / 256), some), 256, 0, stream()>>>(
          z + (size_t)r * Vp, Vp, of + r, losses + r, q.g, q.t, first + r, V, control);
      TT_LAUNCH_CHECK();
    }
    const Operand gradient = {(const char*)z, (long long)rows * Vp * 4, (int)(Vp * 4), TERMS == 1 ? 2 * kLine : kLine};
    if (q.dx) {
      const GradientOut out = {(char*)q.dx + (size_t)first * H * (q.half_out ? 2 : 4), TERMS == 2 ? kPositions : kHalf, q.g ? q.g + first : nullptr,
                               q.t, first, control, q.half_out, 0, H};
      if (launch_product<TERMS, false>(plan_x, gradient, w_gradient, rows, H, pairsV, partial, out)) return -1;
    }
    if (q.dw) {
      const GradientOut out = {several && q.half_out ? (void*)(base + at_sum) : q.dw, TERMS == 2 ? kClasses : kHalf, nullptr, q.t, first, control,
                               several ? 0 : q.half_out, first > 0, H};
      Operand x_gradient = x;
      if (TERMS == 2) x_gradient.at = base + at_x2;
      if (launch_product<TERMS, true>(plan_w, gradient, x_gradient, V, H, (rows + depth - 1) / depth, partial, out)) return -1;
    }
  }
  if (several && q.half_out && q.dw) {
    if (launch_scale((float*)(base + at_sum), nullptr, (_Float16*)q.dw, (size_t)V * H)) return -1;
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
  TT_REQUIRE((long long)H * V <= 1LL << 32, "%s: a weight of 2^32 values at most, got %d x %d", fn, V, H);
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
