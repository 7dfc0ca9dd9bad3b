// Matrix products on v_mfma_f32_16x16x32_f16 for operators that do their own work in front of and behind them: the loss
// of a vocabulary (linear_ce.hip) and orthogonalised updates (muon.hip).
//
//   D[m, n] = sum_k A(m, k) B(n, k),  float32 accumulators
//
// Operands are rows of float16 terms.  A row's columns stand in blocks of 64: 128 bytes of the values themselves (TERMS = 1),
// or of the leading terms with the 128 bytes of the second terms behind them (TERMS = 2).  Two terms hold x = hi + lo with
// hi = f16(x) and lo = f16(x - hi), x scaled by a power of two so that neither leaves the type's range: 22 bits and
// more of the value, or 2^-25 of the scaled unit.  Three products then stand for one of float32,
//   lo_a hi_b + hi_a lo_b + hi_a hi_b,
// and what is left out, lo_a lo_b, is below 2^-22 of the term.  Where a product comes from float16 tensors TERMS = 1 has all of it.
//
// Either operand may be stored with k along its rows (the usual form: a row is one m, or one n) or with k across them
// (X^T X, G^T X: a row is one k, columns are m or n).  The first is read from LDS sixteen bytes a lane, the second by
// ds_read_b64_tr_b16, which hands sixteen lanes the columns of a 4 x 16 piece; so nothing is ever transposed in memory.
//
// A stage is 128 bytes of every row and column of the tile (64 k of one term, 32 of two) and goes from memory straight
// to LDS, past the registers, into one of two buffers while the other is worked on.  Lanes fetch from permuted addresses, so that what
// lanes read together later stands in different banks.  Buffer loads check the offset: rows behind the last come as zeros.
#pragma once
#include "tt_common.h"

namespace tt {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

constexpr int kBlockColumns = 64;               // columns of a block of a row
constexpr int kTermBytes = 128;                 // of one term of a block

// `bytes` from `at` to the end of the last row; `ld` bytes from row to row, `block` from one block of 64 columns to the
// next.  All are multiples of sixteen, and a tile's rows times ld stay below 2^31 (checked on the host).
struct Operand {
  const char* at;
  long long bytes;
  int ld, block;
};

template <typename T>
using lds_ptr = __attribute__((address_space(3))) T*;

// Brings a tile's share of one operand, ROWS rows (or columns) of 128 bytes a stage, to LDS.
template <int TERMS, bool ACROSS, int ROWS, int THREADS>
struct Fetch {
  static constexpr int kDepth = TERMS == 1 ? 64 : 32;
  static constexpr int kLoads = ROWS * 8 / THREADS;
  static_assert(kLoads * THREADS == ROWS * 8, "whole loads");
  unsigned offset[kLoads];
  const char* at;
  long long left;
  int ld, block;

  // Which 32-byte unit of a row of k the unit u stands in: rows that sixteen lanes read together differ in it.
  static __device__ __forceinline__ int unit_mask(int k) {
    constexpr int most = ROWS / 16 - 1;
    return ((k & 3) | ((k >> 1) & 4)) & most;
  }

  // Rows (or columns) from `first` on, a multiple of 64 or of ROWS; from stage `stage` on.
  __device__ __forceinline__ void begin(const Operand& o, int first, int stage) {
    const long long skip =
        ACROSS ? (long long)(first / kBlockColumns) * o.block + (first % kBlockColumns) * 2 + (long long)stage * kDepth * o.ld
               : (long long)first * o.ld + (TERMS == 1 ? (long long)stage * o.block : (long long)(stage >> 1) * o.block + (stage & 1) * 64);
    at = o.at + skip;
    left = o.bytes - skip;
    ld = o.ld;
    block = o.block;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int q = (wave * kLoads + i) * 64 + lane;      // the sixteen bytes of LDS that this lane fills
      if (ACROSS) {
        constexpr int per = ROWS / 8;
        const int line = q / per, pos = q % per, k = line % kDepth, term = line / kDepth;
        const int column = (((pos >> 1) ^ unit_mask(k)) << 4) + ((pos & 1) << 3);
        offset[i] = (unsigned)(k * ld + term * kTermBytes + (column / kBlockColumns) * block + (column % kBlockColumns) * 2);
      } else {
        const int row = q >> 3, c = (q & 7) ^ (row & 7);
        offset[i] = (unsigned)(row * ld + (TERMS == 1 ? c * 16 : (c >> 2) * kTermBytes + (c & 3) * 16));
      }
    }
  }

  __device__ __forceinline__ void load(char* lds) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int records = left > 0x7fffffffLL ? 0x7fffffff : left < 0 ? 0 : (int)left;
    const __amdgpu_buffer_rsrc_t srd = __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, records, 0x00020000);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(srd, (lds_ptr<void>)(lds + (wave * kLoads + i) * 1024), 16, offset[i], 0, 0, 0);
  }

  // to stage `next`
  __device__ __forceinline__ void advance(int next) {
    const int step = ACROSS ? kDepth * ld : TERMS == 1 ? block : (next & 1) ? 64 : block - 64;
    at += step;
    left -= step;
  }
};

// Fragments of 16 rows and 32 k: lane l has row l % 16 and k = 8 (l / 16) .. + 7.
template <int TERMS, bool ACROSS, int ROWS, int TILES>
struct Fragments {
  static constexpr int kDepth = TERMS == 1 ? 64 : 32;
  int at[ACROSS ? TILES : 2];

  __device__ __forceinline__ void begin(int first) {
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    if (ACROSS) {
      const int k = g * 8 + (j >> 2);
      const int mask = Fetch<TERMS, true, ROWS, 64>::unit_mask(k);
#pragma unroll
      for (int i = 0; i < TILES; ++i) at[i] = k * (ROWS * 2) + ((((first >> 4) + i) ^ mask) << 5) + ((j & 3) << 3);
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (first + j) * 128 + (((s * 4 + g) ^ (j & 7)) << 4);
    }
  }
  // Fragment `tile` of part s: of one term the stage's k 32 s .. 32 s + 31, of two terms the term s.
  __device__ __forceinline__ half8 read(const char* lds, int tile, int s) const {
    if (ACROSS) {
      const char* p = lds + at[tile] + s * (32 * ROWS * 2);
      const shortx4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<shortx4>)p);
      const shortx4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<shortx4>)(p + 4 * ROWS * 2));
      return __builtin_bit_cast(half8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return *reinterpret_cast<const half8*>(lds + at[s] + tile * (16 * 128));
  }
};

// A tile of WM x WN waves, each with MT x NT fragments of 16 x 16.
template <int TERMS, bool A_ACROSS, bool B_ACROSS, int WM, int WN, int MT, int NT>
struct Product {
  static constexpr int kM = WM * MT * 16, kN = WN * NT * 16, kThreads = 64 * WM * WN;
  static constexpr int kDepth = TERMS == 1 ? 64 : 32;
  static constexpr int kStage = (kM + kN) * 128, kLds = 2 * kStage;
  typedef Fetch<TERMS, A_ACROSS, kM, kThreads> FetchA;
  typedef Fetch<TERMS, B_ACROSS, kN, kThreads> FetchB;

  // Lane l's acc[i][j] are D[row() + 16 i][column() + 16 j + 0 .. 3].  (The fragments change places in the instruction:
  // a lane then holds neighbours of one row.)
  floatx4 acc[MT][NT];

  static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
  static __device__ __forceinline__ int row() { return (wave() / WN) * (MT * 16) + (threadIdx.x & 15); }
  static __device__ __forceinline__ int column() { return (wave() % WN) * (NT * 16) + ((threadIdx.x & 63) >> 4) * 4; }

  struct Reads {
    Fragments<TERMS, A_ACROSS, kM, MT> a;
    Fragments<TERMS, B_ACROSS, kN, NT> b;
  };

  __device__ __forceinline__ void stage(const char* __restrict from, char* __restrict to, const Reads& r, const FetchA& fa,
                                        const FetchB& fb, bool more) {
    if (more) {
      fa.load(to);
      fb.load(to + kM * 128);
    }
    const char* fromB = from + kM * 128;
    half8 a[2][MT], b[2][NT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < MT; ++i) a[s][i] = r.a.read(from, i, s);
#pragma unroll
      for (int j = 0; j < NT; ++j) b[s][j] = r.b.read(fromB, j, s);
    }
    if (TERMS == 1) {
#pragma unroll
      for (int s = 0; s < 2; ++s) multiply(a[s], b[s]);
    } else {
      multiply(a[1], b[0]);
      multiply(a[0], b[1]);
      multiply(a[0], b[0]);
    }
  }
  __device__ __forceinline__ void multiply(const half8 (&a)[MT], const half8 (&b)[NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[j], a[i], acc[i][j], 0, 0, 0);
  }

  // `stages` of the reduction from stage `first` on; lds: kLds bytes.
  __device__ __forceinline__ void run(const Operand& A, const Operand& B, int m0, int n0, int first, int stages, char* lds) {
    FetchA fa;
    FetchB fb;
    fa.begin(A, m0, first);
    fb.begin(B, n0, first);
    Reads r;
    r.a.begin((wave() / WN) * (MT * 16));
    r.b.begin((wave() % WN) * (NT * 16));
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = floatx4{};
    fa.load(lds);
    fb.load(lds + kM * 128);
    for (int t = 0; t < stages; ++t) {
      fa.advance(first + t + 1);
      fb.advance(first + t + 1);
      __syncthreads();              // (waits for this stage's loads, too)
      stage(lds + (t & 1) * kStage, lds + ((t + 1) & 1) * kStage, r, fa, fb, t + 1 < stages);
    }
  }
};

// Which tile a block works on: the dies get runs of tiles, and within a run the tiles of kTogether rows of tiles follow
// each other, so that what a die's blocks read at one time is about as wide as it is high and stays in its cache.
__device__ __forceinline__ void tile_of(int block, int blocks, int tilesM, int tilesN, int* m, int* n) {
  constexpr int kTogether = 8;
  const int at = xcd_remap(block, blocks), run = kTogether * tilesN, first = at / run * kTogether;
  const int high = tilesM - first < kTogether ? tilesM - first : kTogether;
  *m = first + at % run % high;
  *n = at % run / high;
}

// Two terms of a value that a power of two has brought into range.  What is not finite has no second term.
__device__ __forceinline__ void split(float v, _Float16* hi, _Float16* lo) {
  *hi = (_Float16)v;
  const float rest = v - (float)*hi;
  *lo = __builtin_isfinite(rest) ? (_Float16)rest : (_Float16)0.f;
}
// Where column c of a row of blocks with two terms stands, in bytes (of the first term).
__device__ __forceinline__ int at_column(int c) { return (c >> 6) * (2 * kTermBytes) + (c & 63) * 2; }
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

inline long long padded(long long columns) { return (columns + kBlockColumns - 1) / kBlockColumns * kBlockColumns; }

// The three sizes of tiles.
template <int TERMS, bool A_ACROSS, bool B_ACROSS, int SIZE>
struct Sized;
template <int TERMS, bool A, bool B>
struct Sized<TERMS, A, B, 0> : Product<TERMS, A, B, 4, 1, 1, 4> {};     // 64 x 64
template <int TERMS, bool A, bool B>
struct Sized<TERMS, A, B, 1> : Product<TERMS, A, B, 2, 2, 4, 4> {};     // 128 x 128
template <int TERMS, bool A, bool B>
struct Sized<TERMS, A, B, 2> : Product<TERMS, A, B, 2, 4, 8, 4> {};     // 256 x 256
constexpr int kTileSide[3] = {64, 128, 256};
inline long long tiles_of(long long m, long long n, int size) {
  const int side = kTileSide[size];
  return ((m + side - 1) / side) * ((n + side - 1) / side);
}
// The largest tile of which there are enough for the compute units.
inline int tile_size(long long m, long long n) {
  for (int size = 2; size > 0; --size)
    if (tiles_of(m, n, size) >= compute_units() * 3 / 4) return size;
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
