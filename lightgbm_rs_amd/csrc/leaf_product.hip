// leaf_product.hip — the linear maps of a forest's leaves: y[n] = sum over trees of
// W[t, leaf] x[n] + b[t, leaf], and the gradients dx, dW, db.
//
// Rows come grouped by leaf (leaf_groups.hip, or the layout of a grown tree), so every leaf
// is a matrix product of its own, of as many rows as it holds: a block finds its leaf from
// the counts on the device and gathers its rows through the order.  One tree writes its
// rows directly; several write float32 planes [tree][row] that k_sum_trees adds in the
// trees' order, so results never depend on the order of blocks.
#include "leaf_ops.h"

#include <algorithm>

#include "../../include/lgbm_hip.h"

namespace lgbm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr int THREADS = 256;

// An element type: how many of them 16 bytes hold, and the matrix instruction over
// fragments of 16 bytes a lane (lane l: row or column l % 16 and, of a step's 4 chunks of
// the contraction, chunk l / 16).  Lane l of the result holds rows 4 (l / 16) .. + 4 of the
// first operand and column l % 16 of the second.
template <typename T>
struct El;
template <>
struct El<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
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
  static __device__ __forceinline__ float to(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 from(float v) { return (__bf16)v; }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a),
                                                   __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  }
};
template <>
struct El<_Float16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ float to(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from(float v) { return (_Float16)v; }
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a),
                                                  __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
};

// 16 bytes of elements p[0 .. valid), zeros behind them; nothing behind `valid` is read.
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 load16(const T* p, int valid) {
  u32x4 v = {0, 0, 0, 0};
  if (valid >= El<T>::V) {
    if (VEC)
      v = *reinterpret_cast<const u32x4*>(p);
    else
      __builtin_memcpy(&v, p, 16);
  } else if (valid > 0) {
    T e[El<T>::V];
#pragma unroll
    for (int j = 0; j < El<T>::V; ++j) e[j] = j < valid ? p[j] : (T)0.0f;
    __builtin_memcpy(&v, e, 16);
  }
  return v;
}

// ---- tiles of rows -------------------------------------------------------------------------

struct RowTile {
  int leaf;   // -1: rows of the tree that are in no leaf
  int first;  // position in the tree's order
  int rows;   // 0: there is no such tile
};

// Tile number `mt` of a tree: the leaves' rows in tiles of BM, then the rows in no leaf.
// Every thread of the block takes part; counts and begins are held within [0, rows], so
// that a wrong table cannot reach outside the order.
template <int BM>
__device__ RowTile find_tile(const LeafGroups& g, int tree, int mt, RowTile* shared) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  __shared__ int wave_tiles[THREADS / 64];
  __shared__ int wave_rows[THREADS / 64];
  const int32_t* count = g.count + (int64_t)tree * g.leaves;
  const int32_t* begin = g.begin + (int64_t)tree * g.leaves;
  int tiles_before = 0;
  int64_t rows_before = 0;
  if (tid == 0) *shared = RowTile{-1, 0, 0};
  for (int l0 = 0; l0 < g.leaves; l0 += THREADS) {
    const int l = l0 + tid;
    int c = 0;
    if (l < g.leaves) c = min(max(count[l], 0), g.rows);
    int tiles = (c + BM - 1) / BM, incl = tiles, rows = c;
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(incl, d), r = __shfl_xor(rows, d);
      if (lane >= d) incl += up;
      rows += r;  // wraps only where the counts exceed the rows: the rest is then empty
    }
    __syncthreads();
    if (lane == 63) {
      wave_tiles[wave] = incl;
      wave_rows[wave] = rows;
    }
    __syncthreads();
    int base = tiles_before;
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) base += wave_tiles[w];
      tiles_before += wave_tiles[w];
      rows_before += wave_rows[w];
    }
    const int excl = base + incl - tiles;
    if (mt >= excl && mt < excl + tiles) {
      const int b = min(max(begin[l], 0), g.rows - c), at = (mt - excl) * BM;
      *shared = RowTile{l, b + at, min(BM, c - at)};
    }
    if (mt < tiles_before) break;
  }
  if (mt >= tiles_before && rows_before >= 0 && rows_before < g.rows) {
    const int64_t at = rows_before + (int64_t)(mt - tiles_before) * BM;
    if (tid == 0 && at < g.rows) *shared = RowTile{-1, (int)at, (int)min((int64_t)BM, g.rows - at)};
  }
  __syncthreads();
  return *shared;
}

// Blocks an upper bound of tiles of a tree needs.
int64_t row_tiles(const LeafGroups& g, int bm) {
  return ((int64_t)g.rows + bm - 1) / bm + g.leaves + 1;
}

// ---- products over the inputs (y) and over the outputs (dx) ----------------------------------

// The swizzle of a contraction-major tile: the 16 rows that a transposing read touches at
// once land in different banks.
template <typename T>
__device__ __forceinline__ int cm_swizzle(int row) {
  return sizeof(T) == 2 ? ((row & 3) | ((row >> 1) & 4)) : ((row >> 2) & 3);
}

// A tile in LDS of which lanes read 16 bytes along the contraction: [ROWS][8 chunks].
__device__ __forceinline__ int kc_at(int row, int chunk) {
  return row * 128 + ((chunk ^ (row & 7)) << 4);
}
// The same, stored with the contraction as the slow index: [128 bytes' worth][COLS].
template <typename T, int COLS>
__device__ __forceinline__ int cm_at(int row, int chunk) {
  constexpr int UNITS = COLS / 16, PER = sizeof(T);  // a unit: 16 columns; its chunks of 16 bytes
  const int unit = chunk / PER, in = chunk % PER;
  return row * (COLS * (int)sizeof(T)) + (((unit ^ (cm_swizzle<T>(row) & (UNITS - 1))) * PER + in) << 4);
}

__device__ __forceinline__ u32x4 kc_frag(const char* tile, int row0, int step, int lane) {
  return *reinterpret_cast<const u32x4*>(tile + kc_at(row0 + (lane & 15), step * 4 + (lane >> 4)));
}

template <typename T, int COLS>
__device__ __forceinline__ u32x4 cm_frag(const char* tile, int col0, int step, int lane) {
  const int q = lane >> 4, l = lane & 15, unit = col0 / 16;
  constexpr int UNITS = COLS / 16, UB = 16 * (int)sizeof(T), ROW = COLS * (int)sizeof(T);
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
    u32x4 out;
    __builtin_memcpy(&out, v, 16);
    return out;
  } else {
    u32x4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = step * 16 + q * 4 + j;
      const int at = row * ROW + (unit ^ (cm_swizzle<T>(row) & (UNITS - 1))) * UB + l * 4;
      out[j] = *reinterpret_cast<const uint32_t*>(tile + at);
    }
    return out;
  }
}

// out[row][col] = sum over c of a[row][c] * B(c, col), rows gathered through the order.
// DX false: B(c, col) = w[leaf][col][c] (c: inputs, col: outputs); DX true: B(c, col) =
// w[leaf][c][col] (c: outputs, col: inputs).  BM x BN of the output a block, 128 bytes of the
// contraction a step through LDS, 4 waves in 2 x 2.
template <typename T, bool DX, bool VEC, int BM, int BN>
__global__ __launch_bounds__(THREADS) void k_leaf_tile(LeafProduct p, int length, int cols,
                                                       int col_tiles) {
  constexpr int V = El<T>::V, BK = 8 * V;  // elements of the contraction a step
  constexpr int WM = BM / 2, WN = BN / 2;
  constexpr int ACH = BM * 8 / THREADS, BCH = BN * 8 / THREADS;
  __shared__ __align__(16) char lds[2][(BM + BN) * 128];
  __shared__ int32_t row_of[BM];
  __shared__ RowTile tile;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tree = blockIdx.y;
  const int mt = blockIdx.x / col_tiles, c0 = (blockIdx.x % col_tiles) * BN;
  const RowTile rt = find_tile<BM>(p.g, tree, mt, &tile);
  if (rt.rows == 0) return;
  for (int r = tid; r < BM; r += THREADS) {
    int n = -1;
    if (r < rt.rows) n = p.g.order[(int64_t)tree * p.g.rows + rt.first + r];
    row_of[r] = (n >= 0 && n < p.g.rows) ? n : -1;
  }
  __syncthreads();
  const int64_t leaf = (int64_t)tree * p.g.leaves + rt.leaf;
  const T* const w = (const T*)p.w + (rt.leaf < 0 ? 0 : leaf * p.outputs * (int64_t)p.inputs);
  const T* const src = (const T*)(DX ? p.dy : p.x);
  const int64_t lds_src = DX ? p.lddy : p.ldx;

  f32x4 acc[WM / 16][WN / 16];
#pragma unroll
  for (int i = 0; i < WM / 16; ++i)
#pragma unroll
    for (int j = 0; j < WN / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  if (rt.leaf >= 0) {
    u32x4 ra[ACH], rb[BCH];
    const T* arow[ACH];
#pragma unroll
    for (int i = 0; i < ACH; ++i) {
      const int n = row_of[(tid + i * THREADS) >> 3];
      arow[i] = n < 0 ? nullptr : src + (int64_t)n * lds_src;
    }
    auto load = [&](int k0) {
#pragma unroll
      for (int i = 0; i < ACH; ++i) {
        const int k = k0 + (tid & 7) * V;
        ra[i] = load16<T, VEC>(arow[i] + k, arow[i] ? length - k : 0);
      }
#pragma unroll
      for (int i = 0; i < BCH; ++i) {
        const int at = tid + i * THREADS;
        if (DX) {
          constexpr int CH = BN / V;  // chunks a row
          const int row = k0 + at / CH, col = c0 + at % CH * V;
          rb[i] = load16<T, VEC>(w + (int64_t)row * cols + col, row < length ? cols - col : 0);
        } else {
          const int col = c0 + (at >> 3), k = k0 + (at & 7) * V;
          rb[i] = load16<T, VEC>(w + (int64_t)col * length + k, col < cols ? length - k : 0);
        }
      }
    };
    auto store = [&](char* buf) {
#pragma unroll
      for (int i = 0; i < ACH; ++i) {
        const int at = tid + i * THREADS;
        *reinterpret_cast<u32x4*>(buf + kc_at(at >> 3, at & 7)) = ra[i];
      }
#pragma unroll
      for (int i = 0; i < BCH; ++i) {
        const int at = tid + i * THREADS;
        constexpr int CH = BN / V;
        const int to = DX ? cm_at<T, BN>(at / CH, at % CH) : kc_at(at >> 3, at & 7);
        *reinterpret_cast<u32x4*>(buf + BM * 128 + to) = rb[i];
      }
    };
    const int m0 = (wave >> 1) * WM, n0 = (wave & 1) * WN;
    load(0);
    store(lds[0]);
    __syncthreads();
    for (int k0 = 0, b = 0; k0 < length; k0 += BK, b ^= 1) {
      const bool more = k0 + BK < length;
      if (more) load(k0 + BK);
      const char *ta = lds[b], *tb = lds[b] + BM * 128;
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        u32x4 fa[WM / 16], fb[WN / 16];
#pragma unroll
        for (int i = 0; i < WM / 16; ++i) fa[i] = kc_frag(ta, m0 + 16 * i, step, lane);
#pragma unroll
        for (int j = 0; j < WN / 16; ++j)
          fb[j] = DX ? cm_frag<T, BN>(tb, n0 + 16 * j, step, lane) : kc_frag(tb, n0 + 16 * j, step, lane);
#pragma unroll
        for (int i = 0; i < WM / 16; ++i)
#pragma unroll
          for (int j = 0; j < WN / 16; ++j) acc[i][j] = El<T>::mfma(fb[j], fa[i], acc[i][j]);
      }
      if (more) store(lds[b ^ 1]);
      __syncthreads();
    }
  }

  // lane: output row lane % 16, columns 4 (lane / 16) .. + 4 of each 16 x 16
  const bool planes = p.g.trees > 1;
  float* const plane = (float*)p.ws + (int64_t)tree * p.g.rows * cols;
  const T* const bias = (!DX && p.b && rt.leaf >= 0) ? (const T*)p.b + leaf * cols : nullptr;
#pragma unroll
  for (int i = 0; i < WM / 16; ++i) {
    const int n = row_of[(wave >> 1) * WM + i * 16 + (lane & 15)];
    if (n < 0) continue;
#pragma unroll
    for (int j = 0; j < WN / 16; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = c0 + (wave & 1) * WN + j * 16 + (lane >> 4) * 4 + e;
        if (col >= cols) continue;
        const float v = acc[i][j][e] + (bias ? El<T>::to(bias[col]) : 0.0f);
        if (planes)
          plane[(int64_t)n * cols + col] = v;
        else
          ((T*)p.out)[(int64_t)n * p.ldo + col] = El<T>::from(v);
      }
    }
  }
}

// The trees' planes added in their order, rounded once.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_sum_trees(const float* planes, int64_t rows, int cols,
                                                       int trees, T* out, int64_t ldo) {
  const int64_t total = rows * cols;
  for (int64_t e = blockIdx.x * (int64_t)THREADS + threadIdx.x; e < total;
       e += (int64_t)gridDim.x * THREADS) {
    float v = 0.0f;
    for (int t = 0; t < trees; ++t) v += planes[t * total + e];
    out[e / cols * ldo + e % cols] = El<T>::from(v);
  }
}

// ---- gradients of the maps -------------------------------------------------------------------

// dw[leaf][m][k] = sum over the leaf's rows of dy[row][m] * x[row][k]; db[leaf][m] their sum.
template <typename T, bool VEC, int BM, int BN>
__global__ __launch_bounds__(THREADS) void k_leaf_dw(LeafProduct p, int m_tiles, int k_tiles) {
  constexpr int V = El<T>::V, BK = 8 * V;  // rows a step
  constexpr int WM = BM / 2, WN = BN / 2;
  constexpr int ACH = BM * 8 / THREADS, BCH = BN * 8 / THREADS;
  __shared__ __align__(16) char lds[2][(BM + BN) * 128];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t id = blockIdx.x;
  const int k0 = (int)(id % k_tiles) * BN, m0 = (int)(id / k_tiles % m_tiles) * BM;
  const int64_t leaf = id / ((int64_t)k_tiles * m_tiles);
  const int tree = (int)(leaf / p.g.leaves);
  const int count = min(max(p.g.count[leaf], 0), p.g.rows);
  const int first = min(max(p.g.begin[leaf], 0), p.g.rows - count);
  const int32_t* const order = p.g.order + (int64_t)tree * p.g.rows + first;

  f32x4 acc[WM / 16][WN / 16];
#pragma unroll
  for (int i = 0; i < WM / 16; ++i)
#pragma unroll
    for (int j = 0; j < WN / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  float bias = 0.0f;

  u32x4 ra[ACH], rb[BCH];
  auto row_at = [&](int i) {
    if (i >= count) return -1;
    const int n = order[i];
    return n >= 0 && n < p.g.rows ? n : -1;
  };
  auto load = [&](int r0) {
    constexpr int CA = BM / V, CB = BN / V;
#pragma unroll
    for (int i = 0; i < ACH; ++i) {
      const int at = tid + i * THREADS, n = row_at(r0 + at / CA), m = m0 + at % CA * V;
      ra[i] = load16<T, VEC>((const T*)p.dy + (int64_t)n * p.lddy + m, n < 0 ? 0 : p.outputs - m);
    }
#pragma unroll
    for (int i = 0; i < BCH; ++i) {
      const int at = tid + i * THREADS, n = row_at(r0 + at / CB), k = k0 + at % CB * V;
      rb[i] = load16<T, VEC>((const T*)p.x + (int64_t)n * p.ldx + k, n < 0 ? 0 : p.inputs - k);
    }
  };
  auto store = [&](char* buf) {
    constexpr int CA = BM / V, CB = BN / V;
#pragma unroll
    for (int i = 0; i < ACH; ++i) {
      const int at = tid + i * THREADS;
      *reinterpret_cast<u32x4*>(buf + cm_at<T, BM>(at / CA, at % CA)) = ra[i];
    }
#pragma unroll
    for (int i = 0; i < BCH; ++i) {
      const int at = tid + i * THREADS;
      *reinterpret_cast<u32x4*>(buf + BM * 128 + cm_at<T, BN>(at / CB, at % CB)) = rb[i];
    }
  };
  if (count > 0) {
    load(0);
    store(lds[0]);
    __syncthreads();
    for (int r0 = 0, b = 0; r0 < count; r0 += BK, b ^= 1) {
      const bool more = r0 + BK < count;
      if (more) load(r0 + BK);
      const char *ta = lds[b], *tb = lds[b] + BM * 128;
      if (p.db && k0 == 0 && tid < BM) {
        for (int r = 0; r < BK; ++r)
          bias += El<T>::to(*reinterpret_cast<const T*>(ta + cm_at<T, BM>(r, tid / V) + tid % V * sizeof(T)));
      }
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        u32x4 fa[WM / 16], fb[WN / 16];
#pragma unroll
        for (int i = 0; i < WM / 16; ++i)
          fa[i] = cm_frag<T, BM>(ta, (wave >> 1) * WM + 16 * i, step, lane);
#pragma unroll
        for (int j = 0; j < WN / 16; ++j)
          fb[j] = cm_frag<T, BN>(tb, (wave & 1) * WN + 16 * j, step, lane);
#pragma unroll
        for (int i = 0; i < WM / 16; ++i)
#pragma unroll
          for (int j = 0; j < WN / 16; ++j) acc[i][j] = El<T>::mfma(fb[j], fa[i], acc[i][j]);
      }
      if (more) store(lds[b ^ 1]);
      __syncthreads();
    }
  }
  float* const dw = p.dw + leaf * p.outputs * (int64_t)p.inputs;
#pragma unroll
  for (int i = 0; i < WM / 16; ++i) {
    const int m = m0 + (wave >> 1) * WM + i * 16 + (lane & 15);
    if (m >= p.outputs) continue;
#pragma unroll
    for (int j = 0; j < WN / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int k = k0 + (wave & 1) * WN + j * 16 + (lane >> 4) * 4 + e;
        if (k < p.inputs) dw[(int64_t)m * p.inputs + k] = acc[i][j][e];
      }
  }
  if (p.db && k0 == 0 && tid < BM && m0 + tid < p.outputs) p.db[leaf * p.outputs + m0 + tid] = bias;
}

template <typename T, bool VEC>
void launch(const LeafProduct& p, int what, hipStream_t s) {
  constexpr int B = 64;
  if (what == LEAF_PRODUCT_DW) {
    const int mt = (p.outputs + B - 1) / B, kt = (p.inputs + B - 1) / B;
    const int64_t blocks = (int64_t)mt * kt * p.g.trees * p.g.leaves;
    k_leaf_dw<T, VEC, B, B><<<dim3((unsigned)blocks), THREADS, 0, s>>>(p, mt, kt);
    return;
  }
  const bool dx = what == LEAF_PRODUCT_DX;
  const int length = dx ? p.outputs : p.inputs, cols = dx ? p.inputs : p.outputs;
  const int ct = (cols + B - 1) / B;
  const dim3 grid((unsigned)(row_tiles(p.g, B) * ct), (unsigned)p.g.trees);
  if (dx)
    k_leaf_tile<T, true, VEC, B, B><<<grid, THREADS, 0, s>>>(p, length, cols, ct);
  else
    k_leaf_tile<T, false, VEC, B, B><<<grid, THREADS, 0, s>>>(p, length, cols, ct);
  if (p.g.trees > 1) {
    const int64_t total = (int64_t)p.g.rows * cols;
    const unsigned blocks = (unsigned)std::min<int64_t>((total + THREADS - 1) / THREADS, 4096);
    k_sum_trees<T><<<blocks, THREADS, 0, s>>>((const float*)p.ws, p.g.rows, cols, p.g.trees,
                                              (T*)p.out, p.ldo);
  }
}

// 16-byte loads: every row of every operand starts on 16 bytes.
bool aligned16(const LeafProduct& p, int what, size_t e) {
  auto ok = [&](const void* q, int64_t ld) { return ((uintptr_t)q | (uintptr_t)(ld * (int64_t)e)) % 16 == 0; };
  if (what == LEAF_PRODUCT_DW) return ok(p.dy, p.lddy) && ok(p.x, p.ldx);
  return ok(p.w, p.inputs) && (what == LEAF_PRODUCT_DX ? ok(p.dy, p.lddy) : ok(p.x, p.ldx));
}

template <typename T>
void launch_type(const LeafProduct& p, int what, hipStream_t s) {
  if (aligned16(p, what, sizeof(T)))
    launch<T, true>(p, what, s);
  else
    launch<T, false>(p, what, s);
}

}  // namespace

size_t leaf_product_workspace(const LeafProduct& p, int what) {
  if (what == LEAF_PRODUCT_DW || p.g.trees <= 1) return 0;
  return (size_t)p.g.trees * (size_t)p.g.rows * (size_t)(what == LEAF_PRODUCT_DX ? p.inputs : p.outputs) * 4;
}

int64_t leaf_product_blocks(const LeafProduct& p, int what) {
  const int64_t kt = (p.inputs + 63) / 64, mt = (p.outputs + 63) / 64;
  if (what == LEAF_PRODUCT_DW) return kt * mt * p.g.trees * p.g.leaves;
  return row_tiles(p.g, 64) * (what == LEAF_PRODUCT_DX ? kt : mt);
}

void launch_leaf_product(const LeafProduct& p, int what, hipStream_t s) {
  if (p.dtype == LGBM_HIP_DTYPE_F32)
    launch_type<float>(p, what, s);
  else if (p.dtype == LGBM_HIP_DTYPE_BF16)
    launch_type<__bf16>(p, what, s);
  else
    launch_type<_Float16>(p, what, s);
}

}  // namespace lgbm
