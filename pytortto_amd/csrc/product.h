// Matrix products on v_mfma_f32_16x16x32_f16 for operators that do their own work in front of and behind them: the loss
// of a vocabulary (linear_ce.hip) and orthogonalised updates (muon.hip).
//
//   D[m, n] = sum_k A(m, k) B(n, k),  float32 accumulators
//
// Operands are rows of float16 terms.  Of one term (TERMS = 1) a row is its values, 64 columns of 128 bytes after the other (with a
// distance between them, if need be); of two it is, for every 32 columns, 64 bytes of leading terms and 64 bytes of second ones.
// Two terms hold x = hi + lo with hi = f16(x) and lo = f16(x - hi), x scaled by a power of two so that neither leaves the
// type's range: 22 bits and more of the value, or 2^-25 of the scaled unit.  Three products then stand for one of float32,
//   hi_a hi_b + hi_a lo_b + lo_a hi_b,
// and what is left out, lo_a lo_b, is below 2^-22 of the term.  Where a product comes from float16 tensors TERMS = 1 has all of it.
//
// Either operand may be stored with k along its rows (the usual form: a row is one m, or one n) or with k across them
// (X^T X, G^T X: a row is one k, columns are m or n).  The first is read from LDS sixteen bytes a lane, the second by
// ds_read_b64_tr_b16, which hands sixteen lanes the columns of a 4 x 16 piece; so nothing is ever transposed in memory.
//
// A pair is what 128 bytes of every row hold: two parts of 32 k of one term, or both terms of 32 k.  It comes to LDS as two
// units, each half of the tile's rows and half of its columns, straight from memory, past the registers and by whole cache lines, into a
// ring of units, five for the largest tiles.  A step works on the fragments of one part while those of the next are read and one unit of the
// pair after the next is loaded, all three taking turns; so there is one barrier for two steps, and loads have a step and more to arrive.  Lanes
// fetch from permuted addresses, so that what lanes read together later stands in different banks.  Buffer loads check the
// offset: rows behind the last, and all that is behind the last k, come as zeros.
//
// 4096 x 4096 x 16384 takes 1381 TFLOP/s with one term and 1568 with two (all three products counted), k along the rows; what bounds it
// there is power (a short burst is faster).  Of a tile of 256 x 256 with 32 pairs of one term, 45 us are the product (1.5
// PFLOP/s), 1 to 6 the launch of a block and 7 the stores of its sums, so short reductions are worse off.
#pragma once
#include <utility>

#include "tt_common.h"

namespace tt {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

constexpr int kLine = 128;                      // bytes of 64 columns of one term, or 32 of two
constexpr int kTermBytes = 64;                  // of one term of 32 columns

// `bytes` from `at` to the end of the last row; `ld` bytes from row to row, `block` from one line of 128 bytes to the next.
// All are multiples of sixteen, and a tile's rows times ld stay below 2^31 (checked on the host).  Rows end in zeros up to a whole line, or, of the
// second operand of a product of one term with k along both, in the next row: of their line number `cut` the first `kept` pieces of sixteen bytes
// are theirs, and the others are not read.
struct Operand {
  const char* at;
  long long bytes;
  int ld, block;
  int cut = -1, kept = 0;
};

template <typename T>
using lds_ptr = __attribute__((address_space(3))) T*;

// Brings a tile's share of one operand to LDS: of a pair, ROWS / 2 rows (or, where k goes across, columns) a unit.  CUT: its rows may end in
// the next (read against zeros of the other operand, a value that is not finite there would make NaN of this row).
template <int TERMS, bool ACROSS, int ROWS, int THREADS, bool CUT = false>
struct Fetch {
  static_assert(!CUT || (TERMS == 1 && !ACROSS), "rows of one term");
  static constexpr int kHalf = ROWS / 2, kLoads = kHalf * 8 / THREADS;
  static_assert(kLoads * THREADS == kHalf * 8, "whole loads");
  static constexpr int kColumns = kLine / 2 / TERMS;            // of a line
  static constexpr int kRowBytes = kHalf * 2 * TERMS;           // of a row of k in a unit
  unsigned offset[kLoads];
  unsigned half, step;      // from a pair's first unit to its second, from a pair to the next
  const char* at;
  int left;                 // from there to the end, by sixteen bytes: 2^35 bytes at most (checked on the host)
  int bytes[2];             // what may be read of either unit
  int until, kept;          // CUT: pairs to the last of the row, and what it has of it

  // A unit holds its rows of 128 bytes one after the other, with the sixteen bytes c of row r at place c ^ (r % 8); or its rows of k, with
  // the 32-byte piece u (sixteen columns of a term) at place u ^ piece_mask(k), which differs among the rows that sixteen lanes read together.
  static __device__ __forceinline__ int piece_mask(int k) {
    constexpr int most = kHalf / 16 - 1;
    return ((k & 3) | ((k >> 1) & 4)) & most;
  }

  // Rows (or columns) from `first` on, a multiple of the tile's; pairs from `pair` on.
  __device__ __forceinline__ void begin(const Operand& o, int first, int pair) {
    const long long skip = ACROSS ? (long long)(first / kColumns) * o.block + (long long)pair * (64 / TERMS) * o.ld
                                  : (long long)first * o.ld + (long long)pair * o.block;
    at = o.at + skip;
    left = (int)((o.bytes - skip) >> 4);
    const int ld = o.ld, block = o.block;
    step = ACROSS ? (unsigned)(64 / TERMS * ld) : (unsigned)block;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    half = ACROSS ? (unsigned)(kHalf / kColumns * block) : (unsigned)(kHalf * ld);
    if (ACROSS && kHalf < kColumns) half = kHalf * 2;
    measure();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int q = (wave * kLoads + i) * 64 + lane;      // the sixteen bytes of a unit that this lane fills
      if (ACROSS) {
        constexpr int per = kRowBytes / 16, pieces = kHalf / 16;
        const int k = q / per, pos = q % per, piece = (pos >> 1) ^ piece_mask(k);
        const int column = piece % pieces * 16 + (pos & 1) * 8, term = piece / pieces;
        offset[i] = (unsigned)(k * ld + (column / kColumns) * block + (column % kColumns) * 2 + term * kTermBytes);
      } else {
        const int row = q >> 3, c = (q & 7) ^ (row & 7);
        offset[i] = (unsigned)(row * ld + c * 16);
      }
    }
    if (CUT) {
      until = o.cut - pair;
      kept = o.kept;
      if (until == 0) cut();
    }
  }
  // What is behind the row is out of what may be read.  (A lane has the same sixteen bytes of a line in all of its loads.)
  __device__ __forceinline__ void cut() {
    const int lane = threadIdx.x & 63;
    if (((lane & 7) ^ (lane >> 3)) < kept) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) offset[i] = 0x80000000u;
  }

  __device__ __forceinline__ void measure() {
#pragma unroll
    for (int unit = 0; unit < 2; ++unit) {
      int rest = left - (unit ? (int)(half >> 4) : 0);
      rest = rest < 0 ? 0 : rest;
      // (the compiler has a vector instruction for the two limits, and is told that it may come back from there)
      bytes[unit] = __builtin_amdgcn_readfirstlane(rest < 0x7ffffff ? rest : 0x7ffffff) << 4;
    }
  }
  // Load `i` of a pair's unit 0 or 1.
  __device__ __forceinline__ void load_part(char* lds, int i, int unit) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const auto srd = __builtin_amdgcn_make_buffer_rsrc((void*)(unit ? at + half : at), 0, bytes[unit], 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(srd, (lds_ptr<void>)(lds + (wave * kLoads + i) * 1024), 16, offset[i], 0, 0, 0);
  }

  // To the next pair; where there is none, loads from then on bring zeros.
  __device__ __forceinline__ void advance(bool more) {
    at += step;
    left = more ? left - (int)(step >> 4) : 0;
    measure();
    if (CUT && --until == 0) cut();
  }
};

// Fragments of 16 rows and 32 k: lane l has row l % 16 and k = 8 (l / 16) .. + 7.
template <int TERMS, bool ACROSS, int ROWS, int TILES>
struct Fragments {
  typedef Fetch<TERMS, ACROSS, ROWS, 64> Unit;
  int at[ACROSS ? TILES : 2];

  // `first`: the wave's first row of its unit
  __device__ __forceinline__ void begin(int first) {
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    if (ACROSS) {
      const int k = g * 8 + (j >> 2);
      const int mask = Unit::piece_mask(k);
#pragma unroll
      for (int i = 0; i < TILES; ++i) at[i] = k * Unit::kRowBytes + ((((first >> 4) + i) ^ mask) << 5) + ((j & 3) << 3);
    } else {
#pragma unroll
      for (int part = 0; part < 2; ++part) at[part] = (first + j) * 128 + (((part * 4 + g) ^ (j & 7)) << 4);
    }
  }
  __device__ __forceinline__ half8 read(const char* unit, int tile, int part) const {
    if (ACROSS) {
      const char* p = unit + at[tile] + part * (TERMS == 1 ? 32 * Unit::kRowBytes : Unit::kHalf * 2);
      const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<shortx4>)p);
      const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<shortx4>)(p + 4 * Unit::kRowBytes));
      return __builtin_bit_cast(half8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *reinterpret_cast<const half8*>(unit + at[part] + tile * (16 * 128));
  }
};

// A tile of 2 x 2 waves, each with MT x NT fragments of 16 x 16; AHEAD pairs are on their way or there.
template <int TERMS, bool A_ACROSS, bool B_ACROSS, int MT, int NT, int AHEAD>
struct Product {
  static constexpr int kM = 2 * MT * 16, kN = 2 * NT * 16, kThreads = 256;
  static constexpr int kUnits = 2 * AHEAD + 1, kUnit = (kM + kN) * 64, kLds = kUnits * kUnit;
  typedef Fetch<TERMS, A_ACROSS, kM, kThreads> FetchA;
  typedef Fetch<TERMS, B_ACROSS, kN, kThreads, TERMS == 1 && !A_ACROSS && !B_ACROSS> FetchB;
  static constexpr int kReads = MT + NT, kAll = MT * NT, kLoads = FetchA::kLoads + FetchB::kLoads;

  // Lane l's acc[i][j] are D[row() + 16 i][column() + 16 j + 0 .. 3].  (The fragments change places in the instruction:
  // a lane then holds neighbours of one row.)
  floatx4 acc[MT][NT];

  static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
  static __device__ __forceinline__ int row() { return (wave() >> 1) * (MT * 16) + (threadIdx.x & 15); }
  static __device__ __forceinline__ int column() { return (wave() & 1) * (NT * 16) + ((threadIdx.x & 63) >> 4) * 4; }

  // One instruction.  With 64 accumulators a wave has no registers to spare, and the compiler moves results from one to
  // another; written out, each stays where it is.
  static constexpr bool kPinned = MT * NT == 64;
  __device__ __forceinline__ void multiply(int i, int j, const half8& a, const half8& b) {
    if (kPinned) asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(acc[i][j]) : "v"(b), "v"(a));
    else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b, a, acc[i][j], 0, 0, 0);
  }

  // What a step works on: products of the fragments (a, b), while those of the next part come to (to_a, to_b).
  struct Step {
    const half8 (&a)[MT];
    const half8 (&b)[NT];
    half8 (&to_a)[MT];
    half8 (&to_b)[NT];
    const Fragments<TERMS, A_ACROSS, kM, MT>& ra;
    const Fragments<TERMS, B_ACROSS, kN, NT>& rb;
    const FetchA& fa;
    const FetchB& fb;
  };
  template <int K, int PART>
  static __device__ __forceinline__ void read_one(Step& w, const char* __restrict unit_a, const char* __restrict unit_b) {
    if constexpr (K < NT) w.to_b[K] = w.rb.read(unit_b + kM * 64, K, PART);
    else if constexpr (K < kReads) w.to_a[K - NT] = w.ra.read(unit_a, K - NT, PART);
  }
  template <int K, int UNIT>
  static __device__ __forceinline__ void load_one(const Step& w, char* __restrict to) {
    if constexpr (K < FetchA::kLoads) w.fa.load_part(to, K, UNIT);
    else if constexpr (K < kLoads) w.fb.load_part(to + kM * 64, K - FetchA::kLoads, UNIT);
  }
  // Product Q of a step, and in front of it the reads and loads whose turn it is; both in the first three quarters, so that no
  // read is waited for at the end and loads have more time.
  template <int Q, int PART, int UNIT>
  __device__ __forceinline__ void one(Step& w, const char* __restrict unit_a, const char* __restrict unit_b, char* __restrict to) {
    constexpr int early = kAll * 3 / 4 > kReads ? kAll * 3 / 4 : kAll;
    constexpr int r0 = Q < early ? Q * kReads / early : kReads, r1 = Q + 1 < early ? (Q + 1) * kReads / early : kReads;
    constexpr int l0 = Q < early ? Q * kLoads / early : kLoads, l1 = Q + 1 < early ? (Q + 1) * kLoads / early : kLoads;
    if constexpr (r1 > r0) read_one<r0, PART>(w, unit_a, unit_b);
    if constexpr (r1 > r0 + 1) read_one<r0 + 1, PART>(w, unit_a, unit_b);
    if constexpr (l1 > l0) load_one<l0, UNIT>(w, to);
    if constexpr (l1 > l0 + 1) load_one<l0 + 1, UNIT>(w, to);
    static_assert(r1 <= r0 + 2 && l1 <= l0 + 2, "reads and loads");
    __builtin_amdgcn_sched_barrier(0);
    multiply(Q / NT, Q % NT, w.a[Q / NT], w.b[Q % NT]);
    __builtin_amdgcn_sched_barrier(0);
  }
  template <int PART, int UNIT, int... Q>
  __device__ __forceinline__ void all(Step& w, const char* __restrict unit_a, const char* __restrict unit_b, char* __restrict to,
                                      std::integer_sequence<int, Q...>) {
    (one<Q, PART, UNIT>(w, unit_a, unit_b, to), ...);
  }
  template <int... Q>
  __device__ __forceinline__ void plain(const half8 (&a)[MT], const half8 (&b)[NT], std::integer_sequence<int, Q...>) {
    (multiply(Q / NT, Q % NT, a[Q / NT], b[Q % NT]), ...);
  }
  // Reads of part PART of a pair, loads of unit UNIT.  (A function of its own so that the compiler takes the units for
  // different memory, and does not wait for the loads on their way before it reads.)
  template <int PART, int UNIT>
  __device__ __forceinline__ void step(Step w, const char* __restrict unit_a, const char* __restrict unit_b, char* __restrict to) {
    all<PART, UNIT>(w, unit_a, unit_b, to, std::make_integer_sequence<int, kAll>());
  }

  // Everybody has read what the next loads overwrite, and the next pair's loads have arrived: all but those of the pairs
  // behind it and of the last step.
  static constexpr int kMayWait = (2 * (AHEAD - 2) + 1) * kLoads;
  static_assert(kMayWait + kLoads <= 63, "the counter of loads");
  static __device__ __forceinline__ void meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kMayWait) : "memory");
  }

  // `pairs` from pair `first` on (of 64 k of one term, 32 of two); lds: kLds bytes.
  __device__ __forceinline__ void run(const Operand& A, const Operand& B, int m0, int n0, int first, int pairs, char* lds) {
    FetchA fa;
    FetchB fb;
    fa.begin(A, m0, first);
    fb.begin(B, n0, first);
    Fragments<TERMS, A_ACROSS, kM, MT> ra;
    Fragments<TERMS, B_ACROSS, kN, NT> rb;
    ra.begin(0);
    rb.begin(0);
    int loaded = 0;
    const auto next_pair = [&]() {
      ++loaded;
      fa.advance(loaded < pairs);
      fb.advance(loaded < pairs);
    };
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      char* to = lds + 2 * p * kUnit;
#pragma unroll
      for (int i = 0; i < FetchA::kLoads; ++i) fa.load_part(to, i, 0);
#pragma unroll
      for (int i = 0; i < FetchB::kLoads; ++i) fb.load_part(to + kM * 64, i, 0);
#pragma unroll
      for (int i = 0; i < FetchA::kLoads; ++i) fa.load_part(to + kUnit, i, 1);
#pragma unroll
      for (int i = 0; i < FetchB::kLoads; ++i) fb.load_part(to + kUnit + kM * 64, i, 1);
      next_pair();
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = floatx4{};
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * (AHEAD - 1) * kLoads) : "memory");
    const int half_a = (wave() >> 1) * kUnit, half_b = (wave() & 1) * kUnit;      // this wave's units of a pair
    half8 a[MT], b[NT], a1[MT], b1[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) b[j] = rb.read(lds + half_b + kM * 64, j, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) a[i] = ra.read(lds + half_a, i, 0);
    int at = 0;                           // where the pair's first unit stands in the ring
    const auto around = [](int offset) { return offset >= kLds ? offset - kLds : offset; };
    // One pair more: its first part's fragments are in (a, y), its second's come to (a1, b1), and the next one's first to (a, z).
    const auto go = [&](half8(&y)[NT], half8(&z)[NT]) {
      step<1, 0>(Step{a, y, a1, b1, ra, rb, fa, fb}, lds + around(at + half_a), lds + around(at + half_b), lds + around(at + 2 * AHEAD * kUnit));
      if (TERMS == 2) plain(a, b1, std::make_integer_sequence<int, kAll>());
      meet();
      const int next = around(at + 2 * kUnit);
      if (TERMS == 1) step<0, 1>(Step{a1, b1, a, z, ra, rb, fa, fb}, lds + around(next + half_a), lds + around(next + half_b), lds + at);
      else step<0, 1>(Step{a1, y, a, z, ra, rb, fa, fb}, lds + around(next + half_a), lds + around(next + half_b), lds + at);
      at = next;
      next_pair();
    };
    if (TERMS == 1) {
#pragma unroll 1
      for (int p = 0; p < pairs; ++p) go(b, b);
    } else {
      // two at a time, so that no fragment has to be moved; one too many is zeros
      half8 b2[NT];
#pragma unroll 1
      for (int p = 0; p < pairs; p += 2) {
        go(b, b2);
        go(b2, b);
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");       // (nothing is on its way to LDS any more)
    if (kPinned) {
      // the last results may be read eighteen cycles after their instruction
      asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) asm volatile("" : "+a"(acc[i][j]));
    }
  }

  // The sums, row by row, for what is done with them: kLanes lanes have four neighbours each of a row, a wave kRows rows.
  // They change places through LDS, half of the tile's rows at a time, so that the code behind is a short loop over whole rows (written out
  // for every accumulator it did not fit the instruction cache) and what it reads and writes comes by whole lines.
  // `before(row, c)` reads what a row needs, kAhead turns early: a load that is waited for waits for all stores in front of it.
  // `f(row of the tile, column of the tile, sums, what was read)` is called for kAhead rows at a time, kStep apart, also
  // behind the last.
  static constexpr int kLanes = kN / 4, kRows = 64 / kLanes, kTurns = kM / 2 / (4 * kRows), kAhead = kTurns < 4 ? kTurns : 4;
  static constexpr int kStep = 4 * kRows, kDown = MT, kAcross = NT;
  static constexpr int kRowFloats = kN + 4, kExtra = kM / 2 * kRowFloats * 4;       // (behind it LDS is free for the caller)
  static_assert(kTurns % kAhead == 0 && kExtra + kM * 24 + kN * 4 <= kLds, "rows");
  template <typename R, typename F>
  __device__ __forceinline__ void rows(char* lds, R before, F f) {
    float* at = reinterpret_cast<float*>(lds);
    const int lane = threadIdx.x & 63, first = wave() * kRows + lane / kLanes, c = lane % kLanes * 4;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      decltype(before(0, 0)) old[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) old[u] = before(h * (kM / 2) + first + u * kStep, c);
      if (wave() >> 1 == h) {
        float* to = at + (threadIdx.x & 15) * kRowFloats + column();
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) *reinterpret_cast<floatx4*>(to + i * 16 * kRowFloats + j * 16) = acc[i][j];
      }
      __syncthreads();
#pragma unroll 1
      for (int t = 0; t < kTurns; t += kAhead) {
        const int r = first + t * kStep;
        floatx4 v[kAhead];
        decltype(before(0, 0)) was[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          v[u] = *reinterpret_cast<const floatx4*>(at + (r + u * kStep) * kRowFloats + c);
          was[u] = old[u];
          if (t + kAhead < kTurns) old[u] = before(h * (kM / 2) + r + (u + kAhead) * kStep, c);
        }
        f(h * (kM / 2) + r, c, v, was);
      }
      __syncthreads();
    }
  }
};

// Which tile a block works on.  The dies get runs of `at` (and of the parts of a reduction one after the other: a die's blocks share what they
// read only where they are at the same k), and within a run the tiles of kTogether rows of tiles follow each other, so
// that what a die's blocks read at one time is about as wide as it is high and stays in its cache.  (4096 x 131072 times 131072 x 2048 in two
// parts, float16: with both parts' blocks on every die 1.6 ms, or 1.9 where they drift apart, and this 1.55.)
__device__ __forceinline__ void tile_at(int at, int tilesM, int tilesN, int* m, int* n) {
  constexpr int kTogether = 8;
  const int run = kTogether * tilesN, first = at / run * kTogether;
  const int high = tilesM - first < kTogether ? tilesM - first : kTogether;
  *m = first + at % run % high;
  *n = at % run / high;
}

// Two terms of a value that a power of two has brought into range.  What is not finite has no second term.  (The value is a
// float32 in a register first: rounded to float16 straight from the product in front, as one instruction can do it, the
// first term could be another in one place than in the other, one unit of its last place off in one of a thousand.)
__device__ __forceinline__ void split(float v, _Float16* hi, _Float16* lo) {
  asm("" : "+v"(v));
  *hi = (_Float16)v;
  const float rest = v - (float)*hi;
  *lo = __builtin_isfinite(rest) ? (_Float16)rest : (_Float16)0.f;
}
// Where column c of a row of blocks with two terms stands, in bytes (of the first term).
__device__ __forceinline__ int at_column(int c) { return (c >> 5) * kLine + (c & 31) * 2; }
__device__ __forceinline__ void store_terms(char* row, int c, const floatx4& v) {
  half4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    _Float16 h, l;
    split(v[e], &h, &l);
    hi[e] = h;
    lo[e] = l;
  }
  char* p = row + at_column(c);
  *reinterpret_cast<half4*>(p) = hi;
  *reinterpret_cast<half4*>(p + kTermBytes) = lo;
}
__device__ __forceinline__ floatx4 load_terms(const char* row, int c) {
  const char* p = row + at_column(c);
  const half4 hi = *reinterpret_cast<const half4*>(p), lo = *reinterpret_cast<const half4*>(p + kTermBytes);
  floatx4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)hi[e] + (float)lo[e];
  return v;
}

// Columns of a row with its padding, which is zeros.
__host__ __device__ inline long long padded(long long columns) { return (columns + 63) / 64 * 64; }

// The three sizes of tiles.
template <int TERMS, bool A_ACROSS, bool B_ACROSS, int SIZE>
struct Sized;
template <int TERMS, bool A, bool B>
struct Sized<TERMS, A, B, 0> : Product<TERMS, A, B, 2, 2, 6> {};     // 64 x 64
template <int TERMS, bool A, bool B>
struct Sized<TERMS, A, B, 1> : Product<TERMS, A, B, 4, 4, 4> {};     // 128 x 128
template <int TERMS, bool A, bool B>
struct Sized<TERMS, A, B, 2> : Product<TERMS, A, B, 8, 8, 2> {};     // 256 x 256
constexpr int kTileSide[3] = {64, 128, 256};
inline long long tiles_of(long long m, long long n, int size) {
  const int side = kTileSide[size];
  return ((m + side - 1) / side) * ((n + side - 1) / side);
}
// The largest tile of which there are enough: for half of the compute units where it is filled (a loss with gradients, float32: of 1024 x 1024 x
// 2400, 152 tiles of 128 x 128 100 us, 608 of 64 x 64 131;  of 2048 x 1024 x 3400, 112 of 256 x 256 196 us, 432 of 128 x 128 179), and for three
// quarters where there are few rows, and what counts is how many read at a time (of 1 x 2048 x 32768 float16, 256 of 128 columns 47 us,
// 128 of 256 columns 57).
inline int tile_size(long long m, long long n) {
  for (int size = 2; size > 0; --size) {
    const bool filled = m >= kTileSide[size] && n >= kTileSide[size];
    if (tiles_of(m, n, size) >= (filled ? compute_units() / 2 : compute_units() * 3 / 4)) return size;
  }
  return 0;
}

}  // namespace tt

// Kernels with more LDS than 64 KB say so once.
#define TT_ALLOW_LDS(kernel, bytes)                                                                                  \
  do {                                                                                                               \
    static bool allowed = false;                                                                                     \
    if (!allowed) TT_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes)); \
    allowed = true;                                                                                                  \
  } while (0)
