// leaf_mma.h — what the kernels of the leaves' linear maps share: element types and their
// matrix instructions, tiles of a leaf's rows, and tiles of operands in LDS.
#pragma once

#include "leaf_ops.h"

#include "../../include/lgbm_hip.h"

namespace lgbm {
namespace mma {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// An element type: how many of them 16 bytes hold, and the matrix instruction over
// fragments of 16 bytes a lane (lane l: row or column l % 16 and, of a step's 4 chunks of
// the contraction, chunk l / 16).  Lane l of the result holds rows 4 (l / 16) .. + 4 of the
// first operand and column l % 16 of the second.  Products and sums are float32; a 16-bit
// product is exact in it.
template <typename T>
struct El;
template <>
struct El<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ u32x4 ones() { return u32x4{0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u}; }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
};
template <>
struct El<__bf16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ u32x4 ones() { return u32x4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}; }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a),
                                                   __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  }
};
template <>
struct El<_Float16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ u32x4 ones() { return u32x4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u}; }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a),
                                                  __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
};

// The sums of a stretch of the contraction.  In float32 they start at zero and are added to
// the whole ones afterwards, so that a rounding is of a short sum's size (root mean square
// error of y, and by one chain: 100 inputs 1.1e-7, 1.8e-7, 1000 inputs 1.5e-7, 5.7e-7).  With
// 16-bit operands the stretch goes on in place: the rounding of y and dx hides that, and the
// gradients of the maps, float32 whatever their operands, add no more than CHAIN_ROWS rows
// in one chain.
template <typename T, int M, int N>
struct Parts {
  f32x4 (&at)[M][N];
  __device__ __forceinline__ Parts(f32x4 (&sums)[M][N]) : at(sums) {}
  __device__ __forceinline__ void add_to(f32x4 (&)[M][N]) {}
};
template <int M, int N>
struct Parts<float, M, N> {
  f32x4 at[M][N];
  __device__ __forceinline__ Parts(f32x4 (&)[M][N]) {
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) at[i][j] = f32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void add_to(f32x4 (&sums)[M][N]) {
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) sums[i][j] += at[i][j];
  }
};

// 16 bytes of elements p[0 .. valid), zeros behind them; nothing behind `valid` is read.
// gfx950 loads 16 bytes from any address, so rows need no alignment.
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p, int valid) {
  u32x4 v = {0, 0, 0, 0};
  if (valid >= El<T>::V) {
    __builtin_memcpy(&v, p, 16);
  } else if (valid > 0) {
    T e[El<T>::V];
#pragma unroll
    for (int j = 0; j < El<T>::V; ++j) e[j] = j < valid ? p[j] : (T)0.0f;
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

// Two results of neighbouring rows, as the 16 bits of two neighbouring columns of one: even
// lanes take the first row, odd ones the second.
template <typename T>
__device__ __forceinline__ uint32_t pair_of(float first, float second) {
  const T e[2] = {(T)first, (T)second};
  uint32_t mine;
  __builtin_memcpy(&mine, e, 4);
  const uint32_t other = (uint32_t)__builtin_amdgcn_mov_dpp((int)mine, 0xb1, 0xf, 0xf, true);  // lane ^ 1
  return __builtin_amdgcn_perm(other, mine, threadIdx.x & 1 ? 0x03020706u : 0x05040100u);
}

// ---- tiles of rows -------------------------------------------------------------------------

struct RowTile {
  int leaf;   // -1: rows of the tree that are in no leaf
  int first;  // position in the tree's order
  int rows;   // 0: there is no such tile
};

// Tile number `mt` of a tree, below MAX_TILES: the leaves' rows in tiles of `bm`, then the rows
// in no leaf.  Every thread of the block takes part; counts and begins are held within [0,
// rows], and a leaf's and a wave's tiles to MAX_TILES, so that a wrong table can neither reach
// outside the order nor have sums that wrap, by which two threads would find the tile.
constexpr int MAX_TILES = 1 << 24;  // blocks of a launch
template <int THREADS>
__device__ RowTile find_tile(const LeafGroups& g, int tree, int mt, int bm) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ int wave_tiles[THREADS / 64];
  __shared__ int wave_rows[THREADS / 64];
  __shared__ RowTile found;
  const int32_t* count = g.count + (int64_t)tree * g.leaves;
  const int32_t* begin = g.begin + (int64_t)tree * g.leaves;
  int tiles_before = 0;
  int64_t rows_before = 0;
  if (tid == 0) found = RowTile{-1, 0, 0};
  for (int l0 = 0; l0 < g.leaves; l0 += THREADS) {
    const int l = l0 + tid;
    int c = 0;
    if (l < g.leaves) c = min(max(count[l], 0), g.rows);
    // of 64 leaves at most 2^6 times 2^31 rows: held back to the rows there are, which
    // only counts that exceed them reach
    const int tiles = (int)min(((int64_t)c + bm - 1) / bm, (int64_t)MAX_TILES);
    int incl = tiles, rows = c;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(incl, d), r = __shfl_xor(rows, d);
      if (lane >= d) incl += up;
      rows = (int)min((int64_t)rows + r, (int64_t)g.rows);
    }
    __syncthreads();
    if (lane == 63) {
      wave_tiles[wave] = min(incl, MAX_TILES);
      wave_rows[wave] = rows;
    }
    __syncthreads();
    int base = tiles_before;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) base += wave_tiles[w];
      tiles_before += wave_tiles[w];
      rows_before += wave_rows[w];
    }
    const int excl = base + incl - tiles;
    if (mt >= excl && mt < excl + tiles) {
      const int b = min(max(begin[l], 0), g.rows - c), at = (mt - excl) * bm;
      found = RowTile{l, b + at, min(bm, c - at)};
    }
    if (mt < tiles_before) break;
  }
  if (mt >= tiles_before && rows_before < g.rows && tid == 0) {
    const int64_t at = rows_before + (int64_t)(mt - tiles_before) * bm;
    if (at < g.rows) found = RowTile{-1, (int)at, (int)min((int64_t)bm, g.rows - at)};
  }
  __syncthreads();
  return found;
}

// A bound of a tree's tiles: whole ones, an end for every leaf and for the rows in none, and
// no tile without a row.
__host__ __device__ inline int64_t row_tiles(const LeafGroups& g, int64_t bm) {
  const int64_t tiles = (g.rows + bm - 1) / bm + g.leaves + 1;
  return tiles < g.rows ? tiles : g.rows;
}

// How many tiles a tree has (a wrong table's counts may ask for more than there can be).
template <int THREADS>
__device__ int count_tiles(const LeafGroups& g, int tree, int bm) {
  __shared__ int64_t wave_tiles[THREADS / 64], wave_rows[THREADS / 64];
  const int32_t* count = g.count + (int64_t)tree * g.leaves;
  int64_t tiles = 0, rows = 0;
  for (int l = threadIdx.x; l < g.leaves; l += THREADS) {
    const int c = min(max(count[l], 0), g.rows);
    tiles += ((int64_t)c + bm - 1) / bm;
    rows += c;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    tiles += __shfl_xor(tiles, d);
    rows += __shfl_xor(rows, d);
  }
  if ((threadIdx.x & 63) == 0) wave_tiles[threadIdx.x >> 6] = tiles, wave_rows[threadIdx.x >> 6] = rows;
  __syncthreads();
  tiles = rows = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) tiles += wave_tiles[w], rows += wave_rows[w];
  if (rows < g.rows) tiles += (g.rows - rows + bm - 1) / bm;
  return (int)min(tiles, row_tiles(g, bm));
}

// The row at a position of a tree's order, -1 for an entry outside the matrix.
__device__ __forceinline__ int row_at(const LeafGroups& g, int tree, int position) {
  const int n = g.order[(int64_t)tree * g.rows + position];
  return n >= 0 && n < g.rows ? n : -1;
}

// ---- parts of the maps' gradients --------------------------------------------------------------

// Rows a block sums at most, 0: a leaf's rows are not split.  The parts of a leaf of more rows
// go to slots in the workspace, [tree][slots][outputs * inputs + outputs], and k_sum_slots
// adds them; a leaf of one part has its place in dw.  A part's slot follows from where it
// begins in the order: of the parts that begin in one stretch of `rows` one at most, the first of
// its leaf, is not the last of another, so two slots for a stretch are enough, whatever the
// leaves.
struct Split {
  int rows;
  int64_t parts, slots;  // of a tree, at most
};
inline Split split_by(const LeafGroups& g, int64_t rows) {
  if (rows >= g.rows) return {0, 0, 0};
  return {(int)rows, row_tiles(g, rows), 2 * ((g.rows - 1) / rows + 1)};
}
__device__ __forceinline__ int64_t slot_of(const Split& split, int first, bool first_of_leaf) {
  return 2 * (int64_t)(first / split.rows) + first_of_leaf;
}

// The longest chain of float32 adds over rows: the running sum's rounding is 8192 terms' at
// most (600000 rows of the same bfloat16 value in one chain were off by 4 in 1000).
constexpr int64_t CHAIN_ROWS = 8192;

// What a block sums, and where to.
struct DwPart {
  int tree, first, count;  // count -1: nothing
  float *dw, *db;
};
// `rows` from `first` on of a leaf.
__device__ __forceinline__ DwPart dw_part_of(const LeafProduct& p, const Split& split, int tree, int leaf, int first,
                                             int rows) {
  const int64_t size = (int64_t)p.outputs * p.inputs, at = (int64_t)tree * p.g.leaves + leaf;
  const int count = min(max(p.g.count[at], 0), p.g.rows);
  if (split.rows == 0 || count <= split.rows)
    return {tree, first, rows, p.dw + at * size, p.db ? p.db + at * p.outputs : nullptr};
  const int64_t slot = slot_of(split, first, first == min(max(p.g.begin[at], 0), p.g.rows - count));
  float* const dw = (float*)p.ws + (tree * split.slots + slot) * (size + p.outputs);
  return {tree, first, rows, dw, p.db ? dw + size : nullptr};
}
// Part number `id`: of tree blockIdx.y where leaves are split, else a leaf of the forest.
template <int THREADS>
__device__ __forceinline__ DwPart dw_part(const LeafProduct& p, const Split& split, int id) {
  if (split.rows) {
    const RowTile rt = find_tile<THREADS>(p.g, blockIdx.y, id, split.rows);
    if (rt.rows == 0 || rt.leaf < 0) return {0, 0, -1, nullptr, nullptr};
    return dw_part_of(p, split, blockIdx.y, rt.leaf, rt.first, rt.rows);
  }
  const int count = min(max(p.g.count[id], 0), p.g.rows);
  return dw_part_of(p, split, id / p.g.leaves, id % p.g.leaves, min(max(p.g.begin[id], 0), p.g.rows - count), count);
}

// The results v of column col in rows n[0 .. 4) (-1: none), to the output of one tree or to a
// tree's plane.  Neighbouring lanes have neighbouring columns, so that a store's lanes fill
// pieces of a row: lanes of different rows side by side make a request of every lane's bytes
// (y of 2M rows of 100 float32 inputs to 10 outputs: 318 us instead of 294; dx of 1M rows, 10
// outputs to 100 inputs: 23M requests of 16 bytes, 206 us instead of 199).  Every lane takes part; col of even lanes is even.
template <typename T>
__device__ __forceinline__ void store_rows(const LeafProduct& p, int tree, const int (&n)[4], int col, int cols,
                                           f32x4 v) {
  if (p.planes) {
    float* const to = (float*)p.ws + (int64_t)tree * p.g.rows * cols + col;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n[e] >= 0 && col < cols) to[(int64_t)n[e] * cols] = v[e];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n[e] >= 0 && col < cols) ((float*)p.out)[n[e] * p.ldo + col] = v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const uint32_t two = pair_of<T>(v[e], v[e + 1]);
      const int row = threadIdx.x & 1 ? n[e + 1] : n[e], first = col & ~1;
      T* const to = (T*)p.out + max(row, 0) * p.ldo + first;
      if (row >= 0 && first + 1 < cols)
        __builtin_memcpy(to, &two, 4);
      else if (row >= 0 && first < cols)
        __builtin_memcpy(to, &two, 2);
    }
  }
}

// Of 16 rows, a row in each of the first 16 lanes: those of a lane's results.
__device__ __forceinline__ void rows_of(int mine, int lane, int (&n)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) n[e] = __shfl(mine, (lane >> 4) * 4 + e);
}

template <typename T>
__device__ __forceinline__ float bias_at(const T* bias, int col, int cols) {
  return bias && col < cols ? (float)bias[col] : 0.0f;
}

// ---- tiles in LDS --------------------------------------------------------------------------

// The swizzle of a contraction-major tile: the rows that a transposing read touches at once
// land in different banks.
template <typename T>
__device__ __forceinline__ int cm_swizzle(int row) {
  return sizeof(T) == 2 ? ((row & 3) | ((row >> 1) & 4)) : ((row >> 2) & 3);
}

// Byte of a 16-byte chunk of a tile whose rows hold 128 bytes of the contraction: [ROWS][8].
__device__ __forceinline__ int kc_at(int row, int chunk) {
  return row * 128 + ((chunk ^ (row & 7)) << 4);
}
// The same for a tile stored with the contraction as the slow index: [128 bytes' worth][COLS].
template <typename T, int COLS>
__device__ __forceinline__ int cm_at(int row, int chunk) {
  constexpr int UNITS = COLS / 16, PER = sizeof(T);  // a unit: 16 columns; its chunks of 16 bytes
  const int unit = chunk / PER, in = chunk % PER;
  return row * (COLS * (int)sizeof(T)) + (((unit ^ (cm_swizzle<T>(row) & (UNITS - 1))) * PER + in) << 4);
}

// A lane's fragment of 16 rows from row0 on, half `step` of the tile's contraction.
__device__ __forceinline__ u32x4 kc_frag(const char* tile, int row0, int step, int lane) {
  return *reinterpret_cast<const u32x4*>(tile + kc_at(row0 + (lane & 15), step * 4 + (lane >> 4)));
}

template <typename T, int COLS>
__device__ __forceinline__ u32x4 cm_frag(const char* tile, int col0, int step, int lane) {
  const int q = lane >> 4, l = lane & 15, unit = col0 / 16;
  constexpr int UNITS = COLS / 16, UB = 16 * (int)sizeof(T), ROW = COLS * (int)sizeof(T);
  u32x4 out;
  if constexpr (sizeof(T) == 2) {
    // a transposing read: within 16 lanes, lane l gives row l / 4, columns 4 (l % 4) .. + 4
    // and gets column l of the four rows
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    s16x4 v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = step * 32 + q * 8 + h * 4 + (l >> 2);
      const int at = row * ROW + (unit ^ (cm_swizzle<T>(row) & (UNITS - 1))) * UB + (l & 3) * 8;
      v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)const_cast<char*>(tile + at));
    }
    __builtin_memcpy(&out, v, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = step * 16 + q * 4 + j;
      const int at = row * ROW + (unit ^ (cm_swizzle<T>(row) & (UNITS - 1))) * UB + l * 4;
      out[j] = *reinterpret_cast<const uint32_t*>(tile + at);
    }
  }
  return out;
}

}  // namespace mma

// leaf_big.hip, gradients of the maps: the parts, and whether they are taken by their length
// (those of empty leaves, their zeros, with them)
mma::Split leaf_big_split(const LeafProduct& p);
__host__ __device__ inline bool leaf_big_ranks(const LeafGroups& g) { return (int64_t)g.trees * g.leaves <= 256; }

}  // namespace lgbm
