// Matrix-core tiles of the sequence-attention kernels: element types, LDS tile layouts, operand moves (gfx950).
//
// Every product is built from 32 x 32 output tiles; lane l, r = l & 31, g = l >> 5.  An operand "chunk" is 16 bytes of one row: 8 elements
// of a 16-bit type (one v_mfma_f32_32x32x16) or 4 floats (four v_mfma_f32_32x32x2_f32).  Chunk 2 j + g of row r is lane (r, g)'s share of
// step j, for A and B alike, so the k order inside a step never matters.
//   accumulator register t of lane (r, g): row 8 (t >> 2) + 4 g + (t & 3), column r.
// A product whose LEFT operand was just accumulated reuses it in place: accumulator rows 8 u + 4 g .. + 3 are the k values of lane group g
// in step u, and the other operand is read TRANSPOSED from its row-major LDS tile in the same order (ds_read_b64_tr_b16: four rows of one
// column per lane; 32-bit: four plain reads).  No score ever travels through LDS.
#pragma once
#include "common.h"

namespace is {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

enum { TYPE_F32 = 0, TYPE_BF16 = 1, TYPE_F16 = 2 };      // the C ABI's `type` argument

// 16 bytes <-> floats
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(u32x4_t c, float (&x)[4]) {
    const f32x4 v = __builtin_bit_cast(f32x4, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  }
  static __device__ __forceinline__ u32x4_t pack(const float (&x)[4]) { return __builtin_bit_cast(u32x4_t, f32x4{x[0], x[1], x[2], x[3]}); }
};
template <typename T> struct Vec {
  static constexpr int N = 8;
  typedef T V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void unpack(u32x4_t c, float (&x)[8]) {
    const V v = __builtin_bit_cast(V, c);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  }
  static __device__ __forceinline__ u32x4_t pack(const float (&x)[8]) {
    V v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
    return __builtin_bit_cast(u32x4_t, v);
  }
};

// chunk c of a row in global memory: elements [c N, c N + N) of which the first `len` of the row exist (the rest are 0).
// VEC: rows are 16-byte aligned and `len` is a multiple of N, so a chunk is there whole or not at all.
template <typename T, bool VEC>
__device__ __forceinline__ u32x4_t load_chunk(const char* row, int c, int len) {
  constexpr int N = Vec<T>::N;
  u32x4_t out = {0u, 0u, 0u, 0u};
  if constexpr (VEC) {
    if (c * N < len) out = *reinterpret_cast<const u32x4_t*>(row + c * 16);
  } else {
    const T* p = reinterpret_cast<const T*>(row);
    T x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = c * N + i < len ? p[c * N + i] : (T)0.0f;
    __builtin_memcpy(&out, x, 16);
  }
  return out;
}

template <typename T>
__device__ __forceinline__ f32x16 mfma_chunk(u32x4_t a, u32x4_t b, f32x16 c) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, __bf16)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// Row-major LDS tile of N-element rows, each padded so that one lane address and compile-time offsets reach everything (a swizzle would cost a
// register or an instruction per read, and these kernels have neither to spare).  In 4-byte words, rows are W + pad apart with (W + pad) / 4
// odd: 16 rows of one chunk fall on 64 different banks.  The transposed reads take 4 rows x 64 bytes at a time: the pads of the 16-bit types keep
// those (nearly) apart as well; 32-bit transposed reads are at most 2-way, hidden behind their 64-cycle matrix instructions.
template <typename T, int N>
struct Tile {
  static constexpr int WORDS = N * (int)sizeof(T) / 4, CHUNKS = WORDS / 4;
  static constexpr int STRIDE = 4 * (WORDS + (sizeof(T) == 4 || WORDS <= 32 ? 4 : 20));
  static constexpr int bytes(int rows) { return rows * STRIDE; }
  static __device__ __forceinline__ int offset(int row, int chunk) { return row * STRIDE + chunk * 16; }
  // lane (r, g)'s place in rows [0, 32): chunk g of row r (step j: + 32 j)
  static __device__ __forceinline__ int rows_at(int lane) { return (lane & 31) * STRIDE + (lane >> 5) * 16; }
  // lane's place for the transposed reads of rows [0, 4) + 4 g, columns [0, 32): see mm_transposed
  static __device__ __forceinline__ int columns_at(int lane) {
    if constexpr (sizeof(T) == 4) return 4 * (lane >> 5) * STRIDE + (lane & 31) * 4;
    else return (4 * (lane >> 5) + ((lane >> 2) & 3)) * STRIDE + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  }
};

// (32 x 32) = tile rows . b: `at` = tile + rows_at(lane) of its first row, b = the register-resident other operand (N / (2 Vec::N) steps)
template <typename T, int N>
__device__ __forceinline__ f32x16 mm_tile(const char* at, const u32x4_t (&b)[N / (2 * Vec<T>::N)]) {
  f32x16 acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < N / (2 * Vec<T>::N); ++j) acc = mfma_chunk<T>(*reinterpret_cast<const u32x4_t*>(at + 32 * j), b[j], acc);
  return acc;
}
// the same with both operands in LDS
template <typename T, int N>
__device__ __forceinline__ f32x16 mm_tiles(const char* at, const char* other) {
  f32x16 acc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < N / (2 * Vec<T>::N); ++j)
    acc = mfma_chunk<T>(*reinterpret_cast<const u32x4_t*>(at + 32 * j), *reinterpret_cast<const u32x4_t*>(other + 32 * j), acc);
  return acc;
}

// acc[t] (32 x 32: rows = columns 32 t .. of the tile, columns = p's columns) += (32 tile rows)^T . p;  `at` = tile + columns_at(lane) of the first row.
// The 16-bit matrix instructions take both operands in 16 bits: p goes in as two terms, its rounding and the rounding of what that left out (2^-16 of p
// at most remains in bf16, 2^-22 in fp16), which meet the same tile read.  One term alone is off by up to
// half a step per weight, which added as much error to a result as its own rounding does (0.0025 of the norm for 0.0017 in bf16).
template <typename T, int N, int NT>
__device__ __forceinline__ void mm_transposed(f32x16 (&acc)[NT], const char* at, const f32x16& p) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          acc[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(*reinterpret_cast<const float*>(at + (8 * u + e) * Tile<T, N>::STRIDE + t * 128), p[4 * u + e], acc[t], 0, 0, 0);
  } else {
    typedef T V __attribute__((ext_vector_type(8)));
    // 16 lanes read 4 rows x 16 columns (lane i: row i / 4, columns 4 (i mod 4) ..) and receive column i of the 4 rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      V v, w;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = (T)p[8 * h + e];
        w[e] = (T)(p[8 * h + e] - (float)v[e]);
      }
      const u32x4_t b = __builtin_bit_cast(u32x4_t, v), rest = __builtin_bit_cast(u32x4_t, w);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        u32x2 half[2];
#pragma unroll
        for (int w = 0; w < 2; ++w)
          half[w] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(at + 8 * (2 * h + w) * Tile<T, N>::STRIDE + t * 64)));
        const u32x4_t a = {half[0][0], half[0][1], half[1][0], half[1][1]};
        acc[t] = mfma_chunk<T>(a, b, acc[t]);
        acc[t] = mfma_chunk<T>(a, rest, acc[t]);
      }
    }
  }
}

// ROWS rows of N elements, global -> registers -> LDS by NTHREADS threads.  Thread t handles chunk t mod CH of the rows row_of(k); their byte
// offsets from a base that is uniform over the workgroup are 32-bit (one 64-bit scalar base per tile and one 32-bit lane offset per load).
// Rows of fewer than N elements: the loads repeat the row's last chunk (no test per load), the stores put zeros in its place.
template <typename T, int N, int ROWS, int NTHREADS, bool VEC>
struct Stage {
  static constexpr int ROWS_ = ROWS, CH = Tile<T, N>::CHUNKS, TOTAL = ROWS * CH, PER = (TOTAL + NTHREADS - 1) / NTHREADS;
  static_assert(NTHREADS % CH == 0, "a thread's chunks lie whole rows apart");
  u32x4_t v[PER];
  static __device__ __forceinline__ int row_of(int tid, int k) { return (tid + k * NTHREADS) / CH; }
  static __device__ __forceinline__ bool has(int tid, int k) { return TOTAL % NTHREADS == 0 || tid + k * NTHREADS < TOTAL; }
  __device__ __forceinline__ void load(int tid, const char* base, const unsigned (&offset)[PER], int len) {
    const int c = tid % CH, most = len / Vec<T>::N - 1;
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (has(tid, k)) {
        if constexpr (VEC) v[k] = *reinterpret_cast<const u32x4_t*>(base + (offset[k] + (unsigned)(c < most ? c : most) * 16u));
        else v[k] = load_chunk<T, false>(base + offset[k], c, len);
      }
  }
  __device__ __forceinline__ void store(int tid, char* tile, int len) {
    char* at = tile + Tile<T, N>::offset(tid / CH, tid % CH);
    if (VEC && len < N) {      // (uniform)
      const bool there = (tid % CH) * Vec<T>::N < len;
#pragma unroll
      for (int k = 0; k < PER; ++k) v[k] = there ? v[k] : u32x4_t{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (has(tid, k)) *reinterpret_cast<u32x4_t*>(at + k * (NTHREADS / CH) * Tile<T, N>::STRIDE) = v[k];
  }
};

// four consecutive elements of an output row (columns [col, col + 4) of which those below `len` exist)
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* row, int col, int len, f32x4 x) {
  typedef T V4 __attribute__((ext_vector_type(4)));
  if constexpr (VEC) {
    if (col < len) {
      V4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (T)x[e];
      *reinterpret_cast<V4*>(row + col) = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < len) row[col + e] = (T)x[e];
  }
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// Order of a grid over `outer` independent problems of `units` workgroups each (units in the order they should start).  Consecutive workgroup
// ids go to the 8 XCDs in turn; every XCD gets its own problems (neighbours share its L2).  With few problems per XCD the units of all of them
// advance together, so that the heavy units of every problem start first; with many, problem after problem.
__device__ __forceinline__ void grid_order(int id, int outer, int units, int& problem, int& unit) {
  if (outer % 8 == 0) {
    const int per = outer >> 3, x = id & 7, k = id >> 3;
    if (per <= 4) {
      unit = k / per;
      problem = x * per + k - unit * per;
    } else {
      problem = k / units;
      unit = k - problem * units;
      problem += x * per;
    }
  } else if (outer <= 32) {
    unit = id / outer;
    problem = id - unit * outer;
  } else {
    const int total = outer * units, x = id & 7, k = id >> 3, q = total >> 3, rem = total & 7;
    id = x * q + (x < rem ? x : rem) + k;
    problem = id / units;
    unit = id - problem * units;
  }
}

}  // namespace is
