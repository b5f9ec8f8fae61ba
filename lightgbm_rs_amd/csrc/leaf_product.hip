// leaf_product.hip — the linear maps of a forest's leaves: y[n] = sum over trees of
// W[t, leaf] x[n] + b[t, leaf], and the gradients dx, dW, db.
//
// Rows come grouped by leaf (leaf_groups.hip, or the layout of a grown tree), so every leaf
// is a matrix product of its own, of as many rows as it holds: a block finds its leaf from
// the counts on the device and gathers its rows through the order.  One tree writes its
// rows directly; several write float32 planes [tree][row] that k_sum_trees adds, so results
// never depend on the order of blocks.  As many trees at a time as PLANES holds the planes of.
#include <algorithm>
#include <type_traits>

#include "leaf_mma.h"

namespace lgbm {
namespace {

using namespace mma;

constexpr int THREADS = 256;

// ---- products over the inputs (y) and over the outputs (dx) ----------------------------------

// out[row][col] = sum over c of a[row][c] * B(c, col), rows gathered through the order.
// DX false: B(c, col) = w[leaf][col][c] (c: inputs, col: outputs); DX true: B(c, col) =
// w[leaf][c][col] (c: outputs, col: inputs).  BM x BN of the output a block, 128 bytes of the
// contraction a step through LDS, GM x 4 / GM waves.  Rows and columns that a tile has
// more than the product only make results that are not stored, so their loads are those of
// the last ones; only the end of the contraction needs zeros.  Bound by the matrix
// instructions and, in 16 bits, by LDS (20000 x 1000 to 1000 float32 by 7 leaves: 99 TFLOP/s of
// the 142 to 155 of a library product; 40000 x 2001 to 2047 bfloat16 by 9: 483).
// REST: the parts of large tiles behind their last whole round, of which a row has col_tiles.
template <typename T, bool DX, int BM, int BN, int GM, bool REST = false>
__global__ __launch_bounds__(THREADS) void k_leaf_tile(LeafProduct p, int length, int cols,
                                                       int col_tiles) {
  constexpr int V = El<T>::V, BK = 8 * V;  // elements of the contraction a step
  constexpr int GN = 4 / GM, WM = BM / GM, WN = BN / GN;
  constexpr int ACH = BM * 8 / THREADS, BCH = BN * 8 / THREADS;
  __shared__ __align__(16) char lds[2][(BM + BN) * 128];
  __shared__ __align__(16) int32_t row_of[BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tree = blockIdx.y;
  int c0 = (blockIdx.x % col_tiles) * BN;
  const RowTile rt = REST ? rest_tile<THREADS>(p.g, tree, col_tiles, BN, &c0)
                          : find_tile<THREADS>(p.g, tree, blockIdx.x / col_tiles, BM);
  if (rt.rows == 0 || (REST && c0 >= cols)) return;
  for (int r = tid; r < BM; r += THREADS) row_of[r] = r < rt.rows ? row_at(p.g, tree, rt.first + r) : -1;
  __syncthreads();
  const int64_t leaf = (int64_t)tree * p.g.leaves + rt.leaf;
  const T* const w = (const T*)p.w + (rt.leaf < 0 ? 0 : leaf * p.outputs * (int64_t)p.inputs);
  const T* const src = DX ? (const T*)p.dy + tree * p.dy_tree : (const T*)p.x;
  const int64_t ld = DX ? p.lddy : p.ldx;
  const int m0 = (wave / GN) * WM, n0 = (wave % GN) * WN;

  f32x4 acc[WM / 16][WN / 16];
#pragma unroll
  for (int i = 0; i < WM / 16; ++i)
#pragma unroll
    for (int j = 0; j < WN / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  if (rt.leaf >= 0) {
    u32x4 ra[ACH], rb[BCH];
    const T *arow[ACH], *brow[BCH];
#pragma unroll
    for (int i = 0; i < ACH; ++i) arow[i] = src + (int64_t)max(row_of[(tid + i * THREADS) >> 3], 0) * ld;
    if (!DX)
#pragma unroll
      for (int i = 0; i < BCH; ++i)
        brow[i] = w + (int64_t)min(c0 + ((tid + i * THREADS) >> 3), cols - 1) * length;
    auto load = [&](int k0) {
      const int k = k0 + (tid & 7) * V;
      const bool whole = k0 + BK <= length;
#pragma unroll
      for (int i = 0; i < ACH; ++i) ra[i] = whole ? load16(arow[i] + k) : load16(arow[i] + k, length - k);
#pragma unroll
      for (int i = 0; i < BCH; ++i) {
        if (DX) {
          constexpr int CH = BN / V;  // chunks a row
          const int at = tid + i * THREADS, row = k0 + at / CH, col = c0 + at % CH * V;
          rb[i] = load16(w + (int64_t)row * cols + col, row < length ? cols - col : 0);
        } else {
          rb[i] = whole ? load16(brow[i] + k) : load16(brow[i] + k, length - k);
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
    load(0);
    store(lds[0]);
    __syncthreads();
    for (int k0 = 0, b = 0; k0 < length; k0 += BK, b ^= 1) {
      const bool more = k0 + BK < length;
      if (more) load(k0 + BK);
      const char *ta = lds[b], *tb = lds[b] + BM * 128;
      Parts<T, WM / 16, WN / 16> part(acc);
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        if (step == 1 && k0 + BK / 2 >= length) break;
        u32x4 fa[WM / 16], fb[WN / 16];
#pragma unroll
        for (int i = 0; i < WM / 16; ++i) fa[i] = kc_frag(ta, m0 + 16 * i, step, lane);
#pragma unroll
        for (int j = 0; j < WN / 16; ++j)
          fb[j] = DX ? cm_frag<T, BN>(tb, n0 + 16 * j, step, lane) : kc_frag(tb, n0 + 16 * j, step, lane);
#pragma unroll
        for (int i = 0; i < WM / 16; ++i)
#pragma unroll
          for (int j = 0; j < WN / 16; ++j) part.at[i][j] = El<T>::mfma(fa[i], fb[j], part.at[i][j]);
      }
      part.add_to(acc);
      if (more) store(lds[b ^ 1]);
      __syncthreads();
    }
  }

  // lane: rows 4 (lane / 16) .. + 4, column lane % 16 of each 16 x 16
  const T* const bias = (!DX && p.b && rt.leaf >= 0) ? (const T*)p.b + leaf * cols : nullptr;
#pragma unroll
  for (int j = 0; j < WN / 16; ++j) {
    if (c0 + n0 + j * 16 >= cols) continue;
    const int col = c0 + n0 + j * 16 + (lane & 15);
    const float b = bias_at(bias, col, cols);
#pragma unroll
    for (int i = 0; i < WM / 16; ++i) {
      int n[4];
      __builtin_memcpy(n, row_of + m0 + i * 16 + (lane >> 4) * 4, sizeof(n));
      store_rows<T>(p, tree, n, col, cols, acc[i][j] + b);
    }
  }
}

// The same for up to 16 NB outputs of a leaf: bound by reading x, which no wave shares with
// another, so lanes load their fragments straight from memory (16 rows x 64 bytes an
// instruction; w from the caches), UNROLL steps at a time and without a barrier.  A wave
// takes ROUNDS times 32 rows; blocks of one wave where leaves hold few rows.  2M x 100 float32 to
// 10 by 127 leaves: 294 us, 4.1 TB/s of the lines that rows spread over the table touch.
template <typename T, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void k_leaf_narrow(LeafProduct p) {
  constexpr int V = El<T>::V, UNROLL = 4, ROUNDS = 2, BM = WAVES * 32 * ROUNDS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int tree = blockIdx.y, length = p.inputs, cols = p.outputs;
  const RowTile rt = find_tile<WAVES * 64>(p.g, tree, blockIdx.x, BM);
  if (rt.rows == 0) return;
  const int64_t leaf = (int64_t)tree * p.g.leaves + rt.leaf;
  const T* const w = (const T*)p.w + (rt.leaf < 0 ? 0 : leaf * cols * (int64_t)length);
  const T* wrow[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) wrow[j] = w + (int64_t)min(j * 16 + r, cols - 1) * length;
  const T* const bias = (p.b && rt.leaf >= 0) ? (const T*)p.b + leaf * cols : nullptr;
  float b[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) b[j] = bias_at(bias, j * 16 + r, cols);
  int n[ROUNDS][2];
#pragma unroll
  for (int t = 0; t < ROUNDS; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = (t * WAVES + wave) * 32 + i * 16 + r;
      n[t][i] = at < rt.rows ? row_at(p.g, tree, rt.first + at) : -1;
    }
#pragma unroll
  for (int t = 0; t < ROUNDS; ++t) {
    if ((t * WAVES + wave) * 32 >= rt.rows) break;
    f32x4 acc[2][NB];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{b[j], b[j], b[j], b[j]};
    if (rt.leaf >= 0) {
      const T* xrow[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) xrow[i] = (const T*)p.x + (int64_t)max(n[t][i], 0) * p.ldx;
      for (int k0 = 0; k0 < length; k0 += 4 * V * UNROLL) {
        u32x4 fa[UNROLL][2], fb[UNROLL][NB];
        if (k0 + 4 * V * UNROLL <= length) {
#pragma unroll
          for (int u = 0; u < UNROLL; ++u) {
            const int k = k0 + (u * 4 + q) * V;
#pragma unroll
            for (int i = 0; i < 2; ++i) fa[u][i] = load16(xrow[i] + k);
#pragma unroll
            for (int j = 0; j < NB; ++j) fb[u][j] = load16(wrow[j] + k);
          }
        } else {
#pragma unroll
          for (int u = 0; u < UNROLL; ++u) {
            const int k = k0 + (u * 4 + q) * V;
#pragma unroll
            for (int i = 0; i < 2; ++i) fa[u][i] = load16(xrow[i] + k, length - k);
#pragma unroll
            for (int j = 0; j < NB; ++j) fb[u][j] = load16(wrow[j] + k, length - k);
          }
        }
        Parts<T, 2, NB> part(acc);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          if (k0 + u * 4 * V >= length) break;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) part.at[i][j] = El<T>::mfma(fa[u][i], fb[u][j], part.at[i][j]);
        }
        part.add_to(acc);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int rows[4];
      rows_of(n[t][i], lane, rows);
#pragma unroll
      for (int j = 0; j < NB; ++j) store_rows<T>(p, tree, rows, j * 16 + r, cols, acc[i][j]);
    }
  }
}

// y where leaves hold few rows and the inputs are many: bound by reading the maps.  A block
// makes 16 x 16 of a leaf's result; its waves take every fourth part of the inputs, straight
// from memory, and their sums are added in LDS.  16 rows, 4096 to 4096 float16: 57 to 67 us
// for the 11 to 13 maps of 34 MB that are hit.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_leaf_few(LeafProduct p, int col_tiles) {
  constexpr int V = El<T>::V, UNROLL = 4, PART = 4 * V * UNROLL;
  __shared__ f32x4 sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int tree = blockIdx.y, length = p.inputs, cols = p.outputs;
  const int c0 = (int)(blockIdx.x % col_tiles) * 16;
  const RowTile rt = find_tile<THREADS>(p.g, tree, blockIdx.x / col_tiles, 16);
  if (rt.rows == 0) return;
  const int64_t leaf = (int64_t)tree * p.g.leaves + rt.leaf;
  const int n = r < rt.rows ? row_at(p.g, tree, rt.first + r) : -1;
  f32x4 acc[1][1] = {{f32x4{0, 0, 0, 0}}};
  if (rt.leaf >= 0) {
    const T* const xrow = (const T*)p.x + (int64_t)max(n, 0) * p.ldx;
    const T* const wrow = (const T*)p.w + (leaf * cols + min(c0 + r, cols - 1)) * (int64_t)length;
    for (int k0 = wave * PART; k0 < length; k0 += 4 * PART) {
      u32x4 fx[UNROLL], fw[UNROLL];
      const bool whole = k0 + PART <= length;
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int k = k0 + (u * 4 + q) * V;
        fw[u] = whole ? load16(wrow + k) : load16(wrow + k, length - k);
        fx[u] = whole ? load16(xrow + k) : load16(xrow + k, length - k);
      }
      Parts<T, 1, 1> part(acc);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) part.at[0][0] = El<T>::mfma(fx[u], fw[u], part.at[0][0]);
      part.add_to(acc);
    }
  }
  sums[wave][lane] = acc[0][0];
  __syncthreads();
  if (wave == 0) {
    const T* const bias = (p.b && rt.leaf >= 0) ? (const T*)p.b + leaf * cols : nullptr;
    f32x4 y = acc[0][0] + bias_at(bias, c0 + r, cols);
#pragma unroll
    for (int v = 1; v < 4; ++v) y += sums[v][lane];
    int rows[4];
    rows_of(n, lane, rows);
    store_rows<T>(p, tree, rows, c0 + r, cols, y);
  }
}

// dx for up to 32 outputs of a leaf: bound by writing dx.  A wave keeps the leaf's map of 128
// inputs in registers, turned as the matrix instruction takes it, and runs over its rows, 16
// at a time: one load of dy's rows, then a product for each 16 inputs, and the rows go out
// through LDS whole.  1M rows of 10 outputs to 100 float32 inputs: 138 us where a leaf's rows lie
// side by side (by pieces of 64 bytes, of which the most lie across two lines, 170).
template <typename T, int STEPS>
__global__ __launch_bounds__(THREADS) void k_leaf_dx_narrow(LeafProduct p, int col_tiles) {
  constexpr int V = El<T>::V, FN = 8, BM = 512, PITCH = 16 * FN + 4;
  __shared__ __align__(16) float lds[THREADS / 64][16 * PITCH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int tree = blockIdx.y, cols = p.inputs, length = p.outputs;
  const int c0 = (int)(blockIdx.x % col_tiles) * (16 * FN);
  const RowTile rt = find_tile<THREADS>(p.g, tree, blockIdx.x / col_tiles, BM);
  if (wave * 16 >= rt.rows) return;
  const int64_t leaf = (int64_t)tree * p.g.leaves + rt.leaf;
  const T* const w = (const T*)p.w + (rt.leaf < 0 ? 0 : leaf * length * (int64_t)cols);
  u32x4 fw[STEPS][FN];
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      T e[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int m = (s * 4 + q) * V + v, k = c0 + j * 16 + r;
        e[v] = rt.leaf >= 0 && m < length && k < cols ? w[(int64_t)m * cols + k] : (T)0.0f;
      }
      __builtin_memcpy(&fw[s][j], e, 16);
    }
  float* const mine = lds[wave];
  // 16 rows from LDS, 16 bytes a lane
  auto store_tile = [&](auto* out, int64_t ld, int valid, int row, const float* from) {
    typedef std::remove_reference_t<decltype(*out)> O;
    constexpr int CH = 16 / (int)sizeof(O), ACROSS = 16 * FN / CH;
    const int col = lane % ACROSS * CH;
#pragma unroll
    for (int i = 0; i < 16; i += 64 / ACROSS) {
      const int at = i + lane / ACROSS, n = __shfl(row, at);
      O v[CH];
#pragma unroll
      for (int e = 0; e < CH; ++e) v[e] = (O)from[at * PITCH + col + e];
      if (n >= 0 && col + CH <= valid) {
        __builtin_memcpy(out + n * ld + col, v, 16);
      } else if (n >= 0) {
#pragma unroll
        for (int e = 0; e < CH; ++e)
          if (col + e < valid) out[n * ld + col + e] = v[e];
      }
    }
  };
  constexpr int UNROLL = 4;
  for (int r0 = wave * 16; r0 < rt.rows; r0 += 64 * UNROLL) {
    int n[UNROLL];
    u32x4 f[UNROLL][STEPS];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int at = r0 + u * 64 + r;
      n[u] = at < rt.rows ? row_at(p.g, tree, rt.first + at) : -1;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int m = (s * 4 + q) * V;
        f[u][s] = load16((const T*)p.dy + tree * p.dy_tree + (int64_t)max(n[u], 0) * p.lddy + m,
                         n[u] < 0 || rt.leaf < 0 ? 0 : length - m);
      }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if (c0 + j * 16 >= cols) break;
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < STEPS; ++s) acc = El<T>::mfma(f[u][s], fw[s][j], acc);
#pragma unroll
        for (int e = 0; e < 4; ++e) mine[(q * 4 + e) * PITCH + j * 16 + r] = acc[e];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (p.planes)
        store_tile((float*)p.ws + (int64_t)tree * p.g.rows * cols + c0, cols, cols - c0, n[u], mine);
      else
        store_tile((T*)p.out + c0, p.ldo, cols - c0, n[u], mine);
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// The planes of a run of trees added, in float64, since a forest has hundreds; the last run
// rounds once, the others leave their sums in carry [rows][cols] (null: one run).  The last
// adds a layer's residual (null: none).
struct Run {
  double* carry;
  bool first, last;
  const void* res;
  int64_t ldr;
};
template <typename T>
__device__ __forceinline__ double res_at(const Run& run, int64_t row, int64_t col) {
  return run.res ? (double)(float)((const T*)run.res)[row * run.ldr + col] : 0.0;
}
template <int V>
__device__ __forceinline__ void carry_in(const Run& run, int64_t e, double (&v)[V]) {
  if (run.first) return;
  double c[V];
  __builtin_memcpy(c, run.carry + e, sizeof(c));
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] += c[i];
}

// 64 elements a block, a quarter of the trees a wave.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_sum_trees(const float* planes, int64_t rows, int cols,
                                                       int trees, Run run, T* out, int64_t ldo) {
  __shared__ double part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t total = rows * cols;
  const int t0 = (int)((int64_t)trees * wave / 4), t1 = (int)((int64_t)trees * (wave + 1) / 4);
  for (int64_t e0 = blockIdx.x * (int64_t)64; e0 < total; e0 += (int64_t)gridDim.x * 64) {
    const int64_t e = e0 + lane;
    double v = 0;
    if (e < total) {
#pragma unroll 8
      for (int t = t0; t < t1; ++t) v += (double)planes[t * total + e];
    }
    part[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && e < total) {
      double sum[1] = {part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane]};
      carry_in(run, e, sum);
      if (run.last)
        out[e / cols * ldo + e % cols] = (T)(float)(sum[0] + res_at<T>(run, e / cols, e % cols));
      else
        run.carry[e] = sum[0];
    }
    __syncthreads();
  }
}
// Few trees: a thread an element, or four of rows without gaps.
template <typename T, int V>
__global__ __launch_bounds__(THREADS) void k_sum_few_trees(const float* planes, int64_t rows, int cols,
                                                           int trees, Run run, T* out, int64_t ldo) {
  const int64_t total = rows * cols;
  for (int64_t e = (blockIdx.x * (int64_t)THREADS + threadIdx.x) * V; e < total;
       e += (int64_t)gridDim.x * THREADS * V) {
    double v[V] = {};
#pragma unroll 4
    for (int t = 0; t < trees; ++t) {
      float x[V];
      __builtin_memcpy(x, planes + t * total + e, sizeof(x));
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += (double)x[i];
    }
    carry_in(run, e, v);
    if (!run.last) {
      __builtin_memcpy(run.carry + e, v, sizeof(v));
      continue;
    }
    if (run.res)
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] += res_at<T>(run, (e + i) / cols, (e + i) % cols);
    T o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (T)(float)v[i];
    __builtin_memcpy(out + (V > 1 ? e : e / cols * ldo + e % cols), o, sizeof(o));
  }
}

// ---- gradients of the maps -------------------------------------------------------------------

// Leaves differ in size and may be fewer than the CUs, so blocks take about a 2048th of the
// work (a thousandth is one round of blocks and a few more: ragged leaves of 2M rows, 100 float32
// inputs, 10 outputs 382 us instead of 283), or of many tiles a thousandth, which leaves more
// leaves whole (float32, by that and by a 2048th: 20000 x 1000 to 1000 by seven leaves alike 622 and 709
// us, 5000 x 2000 to 2000 by two 580 and 600; ragged 40000 x 600 to 600 by 31 547 and 472).
Split dw_split(const LeafProduct& p, int64_t tiles) {
  const int64_t work = (int64_t)p.g.rows * p.g.trees * tiles;
  int64_t rows = (work / (tiles <= 64 ? 2048 : 1024) + 255) / 256 * 256;
  rows = std::min<int64_t>(std::max<int64_t>(rows, 512), CHAIN_ROWS);
  return split_by(p.g, rows);
}

// dw[leaf][m][k] = sum over the leaf's rows of dy[row][m] * x[row][k]; db[leaf][m] their sum.
// BM x BN of a leaf's outputs x inputs a block, 128 bytes' worth of rows a step.  As
// k_leaf_tile, with both operands read across (20000 x 1000 to 1000 float32 by 7 leaves: 610 us,
// 66 TFLOP/s; 50000 x 300 to 100 float16 by two trees of 15: 89 us).
template <typename T, int BM, int BN, int GM>
__global__ __launch_bounds__(THREADS) void k_leaf_dw(LeafProduct p, int m_tiles, int k_tiles, Split split) {
  constexpr int V = El<T>::V, BK = 8 * V;  // rows a step
  constexpr int GN = 4 / GM, WM = BM / GM, WN = BN / GN;
  constexpr int ACH = (BM * 8 + THREADS - 1) / THREADS, BCH = (BN * 8 + THREADS - 1) / THREADS;
  constexpr int CA = BM / V, CB = BN / V;  // chunks a row
  __shared__ __align__(16) char lds[2][(BM + BN) * 128];
  __shared__ int32_t row_of[2][BK];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tiles = m_tiles * k_tiles, tile = (int)(blockIdx.x % tiles);
  const int k0 = tile % k_tiles * BN, m0 = tile / k_tiles * BM;
  const DwPart part_of = dw_part<T, THREADS>(p, split, (int)(blockIdx.x / tiles));
  const int tree = part_of.tree, first = part_of.first, count = part_of.count;
  if (count < 0) return;
  if (count == 0) {  // the leaf's zeros, in one piece a block
    const int64_t size = (int64_t)p.outputs * p.inputs;
    const int64_t piece = ((size + tiles - 1) / tiles + 3) / 4 * 4, to = min(size, (tile + 1) * piece);
    const int64_t word = part_of.narrow ? 2 : 4;
    for (int64_t e = tile * piece + tid * 4; e < to; e += THREADS * 4) {
      if (e + 4 <= to) {
        const f32x4 none = {0, 0, 0, 0};
        char* const at = (char*)part_of.dw + e * word;
        if (part_of.narrow)
          __builtin_memcpy(at, &none, 8);
        else
          __builtin_memcpy(at, &none, 16);
      } else {
        for (int64_t k = e; k < to; ++k) put<T>(part_of, part_of.dw, k, 0.0f);
      }
    }
    for (int m = tile * THREADS + tid; part_of.db && m < p.outputs; m += tiles * THREADS)
      put<T>(part_of, part_of.db, m, 0.0f);
    return;
  }

  f32x4 acc[WM / 16][WN / 16];
#pragma unroll
  for (int i = 0; i < WM / 16; ++i)
#pragma unroll
    for (int j = 0; j < WN / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  f32x4 bias[WM / 16][1];
#pragma unroll
  for (int i = 0; i < WM / 16; ++i) bias[i][0] = f32x4{0, 0, 0, 0};
  const bool sums = part_of.db && k0 == 0 && wave % GN == 0;  // a product with ones
  const T* const dy = (const T*)p.dy + tree * p.dy_tree;

  // rows of step s in row_of[s & 1]; the loads of a step are two steps behind its rows
  auto rows = [&](int r0) {
    if (tid < BK) row_of[(r0 / BK) & 1][tid] = r0 + tid < count ? row_at(p.g, tree, first + r0 + tid) : -1;
  };
  u32x4 ra[ACH], rb[BCH];
  auto load = [&](int r0) {
    const int32_t* const of = row_of[(r0 / BK) & 1];
#pragma unroll
    for (int i = 0; i < ACH; ++i) {
      const int at = tid + i * THREADS;
      if (BM * 8 % THREADS != 0 && at >= BM * 8) break;
      const int n = of[at / CA], m = m0 + at % CA * V;
      ra[i] = load16(dy + (int64_t)max(n, 0) * p.lddy + m, n < 0 ? 0 : p.outputs - m);
    }
#pragma unroll
    for (int i = 0; i < BCH; ++i) {
      const int at = tid + i * THREADS;
      if (BN * 8 % THREADS != 0 && at >= BN * 8) break;
      const int n = of[at / CB], k = k0 + at % CB * V;
      rb[i] = load16((const T*)p.x + (int64_t)max(n, 0) * p.ldx + k, n < 0 ? 0 : p.inputs - k);
    }
  };
  auto store = [&](char* buf) {
#pragma unroll
    for (int i = 0; i < ACH; ++i) {
      const int at = tid + i * THREADS;
      if (BM * 8 % THREADS != 0 && at >= BM * 8) break;
      *reinterpret_cast<u32x4*>(buf + cm_at<T, BM>(at / CA, at % CA)) = ra[i];
    }
#pragma unroll
    for (int i = 0; i < BCH; ++i) {
      const int at = tid + i * THREADS;
      if (BN * 8 % THREADS != 0 && at >= BN * 8) break;
      *reinterpret_cast<u32x4*>(buf + BM * 128 + cm_at<T, BN>(at / CB, at % CB)) = rb[i];
    }
  };
  if (count > 0) {
    rows(0);
    __syncthreads();
    load(0);
    rows(BK);
    store(lds[0]);
    __syncthreads();
    for (int r0 = 0, b = 0; r0 < count; r0 += BK, b ^= 1) {
      const bool more = r0 + BK < count;
      if (more) load(r0 + BK);
      rows(r0 + 2 * BK);  // into the half whose rows are loaded already
      const char *ta = lds[b], *tb = lds[b] + BM * 128;
      Parts<T, WM / 16, WN / 16> part(acc);
      Parts<T, WM / 16, 1> bias_part(bias);
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        u32x4 fa[WM / 16], fb[WN / 16];
#pragma unroll
        for (int i = 0; i < WM / 16; ++i) fa[i] = cm_frag<T, BM>(ta, (wave / GN) * WM + 16 * i, step, lane);
#pragma unroll
        for (int j = 0; j < WN / 16; ++j) fb[j] = cm_frag<T, BN>(tb, (wave % GN) * WN + 16 * j, step, lane);
        if (sums)
#pragma unroll
          for (int i = 0; i < WM / 16; ++i)
            bias_part.at[i][0] = El<T>::mfma(El<T>::ones(), fa[i], bias_part.at[i][0]);
#pragma unroll
        for (int i = 0; i < WM / 16; ++i)
#pragma unroll
          for (int j = 0; j < WN / 16; ++j) part.at[i][j] = El<T>::mfma(fa[i], fb[j], part.at[i][j]);
      }
      part.add_to(acc);
      if (sums) bias_part.add_to(bias);
      if (more) store(lds[b ^ 1]);
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < WM / 16; ++i) {
    const int mi = m0 + (wave / GN) * WM + i * 16;
    if (sums && lane < 16 && mi + lane < p.outputs) put<T>(part_of, part_of.db, mi + lane, bias[i][0][0]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int m = mi + (lane >> 4) * 4 + e;
#pragma unroll
      for (int j = 0; j < WN / 16; ++j) {
        const int k = k0 + (wave % GN) * WN + j * 16 + (lane & 15);
        if (m < p.outputs && k < p.inputs)
          put<T>(part_of, part_of.dw, (int64_t)m * p.inputs + k, acc[i][j][e]);
      }
    }
  }
}

// The same for up to 16 outputs and 16 NB inputs: bound by reading x, so waves take rows of
// their own straight from memory, 16 neighbouring columns of a row a load, without a barrier
// until their sums are added (float32, 500000 x 28 to 1 by 5 trees of 31 leaves: 121 us, by
// k_leaf_dw 273; 1M x 60 to 10 by 63: 86 and 128; 1M x 100 to 10: 135 and 150).
template <typename T, int NB>
__global__ __launch_bounds__(THREADS) void k_leaf_dw_small(LeafProduct p, Split split) {
  constexpr int V = El<T>::V, STEP = 4 * V, UNROLL = NB == 8 ? 1 : 2;
  __shared__ f32x4 sums[THREADS / 64][NB + 1][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const DwPart part_of = dw_part<T, THREADS>(p, split, (int)blockIdx.x);
  if (part_of.count < 0) return;
  f32x4 acc[1][NB + 1];  // the last: with ones
#pragma unroll
  for (int j = 0; j <= NB; ++j) acc[0][j] = f32x4{0, 0, 0, 0};
  // columns behind the last only make results that are not stored
  const T* const dy = (const T*)p.dy + part_of.tree * p.dy_tree + min(r, p.outputs - 1);
  const T* x[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) x[j] = (const T*)p.x + min(j * 16 + r, p.inputs - 1);
  for (int r0 = wave * (STEP * UNROLL); r0 < part_of.count; r0 += THREADS / 64 * (STEP * UNROLL)) {
    T fa[UNROLL][V], fb[UNROLL][NB][V];
    int n[UNROLL][V];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int at = r0 + u * STEP + q * V + e;
        n[u][e] = at < part_of.count ? row_at(p.g, part_of.tree, part_of.first + at) : -1;
      }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int64_t row = max(n[u][e], 0);
        fa[u][e] = dy[row * p.lddy];
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[u][j][e] = x[j][row * p.ldx];
      }
    Parts<T, 1, NB + 1> part(acc);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      u32x4 a, b[NB];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (n[u][e] >= 0) continue;
        fa[u][e] = (T)0.0f;
#pragma unroll
        for (int j = 0; j < NB; ++j) fb[u][j][e] = (T)0.0f;
      }
      __builtin_memcpy(&a, fa[u], 16);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        __builtin_memcpy(&b[j], fb[u][j], 16);
        part.at[0][j] = El<T>::mfma(a, b[j], part.at[0][j]);
      }
      if (part_of.db) part.at[0][NB] = El<T>::mfma(El<T>::ones(), a, part.at[0][NB]);
    }
    part.add_to(acc);
  }
#pragma unroll
  for (int j = 0; j <= NB; ++j) sums[wave][j][lane] = acc[0][j];
  __syncthreads();
  for (int j = wave; j <= NB; j += THREADS / 64) {
    f32x4 v = sums[0][j][lane];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v += sums[w][j][lane];
    if (j == NB) {
      if (part_of.db && lane < p.outputs && lane < 16) put<T>(part_of, part_of.db, lane, v[0]);
      continue;
    }
    const int k = j * 16 + r;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (q * 4 + e < p.outputs && k < p.inputs)
        put<T>(part_of, part_of.dw, (q * 4 + e) * p.inputs + k, v[e]);
  }
}

// The slots of a leaf of several parts added in their order, by `parts` blocks a leaf, in
// float64: a long leaf has hundreds.  `zeros`: and the zeros of leaves without rows.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_sum_slots(LeafProduct p, Split split, int parts, bool zeros) {
  const DwPart to{0, 0, 0, p.dw, p.db, sizeof(T) == 2 && p.narrow};
  const int64_t at = blockIdx.x / parts;  // leaf of the forest
  const int tree = (int)(at / p.g.leaves);
  const int count = min(max(p.g.count[at], 0), p.g.rows), begin = min(max(p.g.begin[at], 0), p.g.rows - count);
  if (count <= split.rows && !(count == 0 && zeros)) return;
  const int more = (int)(((int64_t)count + split.rows - 1) / split.rows) - 1;  // parts behind the first
  const int64_t map = (int64_t)p.outputs * p.inputs, size = map + p.outputs;
  const int64_t used = p.db ? size : map;
  const float* const slots = (const float*)p.ws + tree * split.slots * size;
  const float* const first = slots + slot_of(split, begin, true) * size;
  const float* const others = slots + slot_of(split, begin, false) * size;  // two slots a part
  for (int64_t e = blockIdx.x % parts * (int64_t)THREADS + threadIdx.x; e < used; e += (int64_t)parts * THREADS) {
    double v = count > 0 ? (double)first[e] : 0.0;
#pragma unroll 16
    for (int64_t s = 1; s <= more; ++s) v += (double)others[2 * s * size + e];
    if (e < map)
      put<T>(to, to.dw, at * map + e, (float)v);
    else
      put<T>(to, to.db, at * p.outputs + (e - map), (float)v);
  }
}

// ---- which kernel ------------------------------------------------------------------------------

// The tile of outputs x inputs of a leaf that a block of k_leaf_dw sums, or the whole of it by
// k_leaf_dw_small (1M rows of 128 float16 inputs to 1 by that: 72 us instead of 59, so 16
// bits stop at 64).
struct DwShape {
  int bm, bn;
  bool small;
};
DwShape dw_shape(const LeafProduct& p) {
  if (p.outputs <= 16) return {16, 128, p.inputs <= (p.dtype == LGBM_HIP_DTYPE_F32 ? 128 : 64)};
  if (p.inputs <= 16) return {128, 16, false};
  return {64, 64, false};
}

// Leaves of 16 rows at most, on average.
bool few_rows(const LeafProduct& p) { return p.g.rows <= 16 * (int64_t)p.g.leaves; }

// k_leaf_few: leaves of few rows, or few outputs of so few rows that k_leaf_narrow's blocks
// of 256 would leave CUs without work (float32, 2000 inputs to 10 outputs by k_leaf_narrow
// and by it: 1000 rows 85 and 16 us, 30000 rows 109 and 92, 60000 rows 141 and 152; to 32
// outputs 10000 rows 121 and 52, 30000 rows 138 and 151; 130 inputs to 10, 10000 rows: 16
// and 9).
bool by_maps(const LeafProduct& p) {
  if (p.outputs > 32) return p.inputs >= 512 && few_rows(p);
  return p.inputs >= 128 && (few_rows(p) || (int64_t)p.g.rows * ((p.outputs + 15) / 16) < 49152);
}

// Tiles of 128 x 128, where leaves fill them and there is one for every CU: 16-bit products
// that are not for leaf_big.hip (40000 x 2001 to 2047 bf16 by 9 leaves: y 690 us instead of
// 965, dx 945 instead of 1004).  float32 is slower by them (20000 x 1000 to 1000 by 7: 454 us,
// 423 by 64 x 64), and so are the gradients of the maps (bf16 as above, rows not split: 2518 us, 1371).
bool wide_tiles(const LeafProduct& p, int cols) {
  return p.dtype != LGBM_HIP_DTYPE_F32 && cols >= 128 && p.g.rows >= 128 * (int64_t)p.g.leaves &&
         (int64_t)p.g.rows / 128 * ((cols + 127) / 128) * p.g.trees >= 256;
}

// Leaves of one part leave most of the blocks without work (bfloat16, 60000 x 256 to 256 by 300
// leaves: 88 us of all the kernels by 2^16 blocks, 55 by 2^13).
template <typename T>
void sum_slots(const LeafProduct& p, const Split& split, bool zeros, hipStream_t s) {
  const int64_t leaves = (int64_t)p.g.trees * p.g.leaves, size = (int64_t)p.outputs * (p.inputs + 1);
  const int parts = (int)std::max<int64_t>(1, std::min((size + THREADS - 1) / THREADS, (1 << 13) / leaves));
  k_sum_slots<T><<<(unsigned)(leaves * parts), THREADS, 0, s>>>(p, split, parts, zeros);
}

template <typename T>
void launch_dw(const LeafProduct& p, hipStream_t s) {
  const DwShape d = dw_shape(p);
  const int mt = (p.outputs + d.bm - 1) / d.bm, kt = (p.inputs + d.bn - 1) / d.bn;
  const Split split = dw_split(p, (int64_t)mt * kt);
  const int64_t leaves = (int64_t)p.g.trees * p.g.leaves;
  const dim3 grid = split.rows ? dim3((unsigned)(split.parts * mt * kt), p.g.trees)
                               : dim3((unsigned)((int64_t)mt * kt * leaves));
  if (d.small && p.inputs <= 32)
    k_leaf_dw_small<T, 2><<<grid, THREADS, 0, s>>>(p, split);
  else if (d.small && p.inputs <= 64)
    k_leaf_dw_small<T, 4><<<grid, THREADS, 0, s>>>(p, split);
  else if (d.small && sizeof(T) == 4)
    k_leaf_dw_small<float, 8><<<grid, THREADS, 0, s>>>(p, split);
  else if (d.bm == 16)
    k_leaf_dw<T, 16, 128, 1><<<grid, THREADS, 0, s>>>(p, mt, kt, split);
  else if (d.bn == 16)
    k_leaf_dw<T, 128, 16, 4><<<grid, THREADS, 0, s>>>(p, mt, kt, split);
  else
    k_leaf_dw<T, 64, 64, 2><<<grid, THREADS, 0, s>>>(p, mt, kt, split);
  if (split.rows) sum_slots<T>(p, split, true, s);
}

template <typename T, bool DX, int BM, int BN>
void launch_tile(const LeafProduct& p, hipStream_t s) {
  const int length = DX ? p.outputs : p.inputs, cols = DX ? p.inputs : p.outputs;
  const int ct = (cols + BN - 1) / BN;
  const dim3 grid((unsigned)(row_tiles(p.g, BM) * ct), (unsigned)p.g.trees);
  k_leaf_tile<T, DX, BM, BN, 2><<<grid, THREADS, 0, s>>>(p, length, cols, ct);
}

template <typename T, bool DX>
void launch_tiles(const LeafProduct& p, bool wide, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (wide) return launch_tile<T, DX, 128, 128>(p, s);
  }
  launch_tile<T, DX, 64, 64>(p, s);
}

// Which kernel makes y or dx; by all the trees, however few of them are made at a time.
struct Form {
  bool big, maps, wide;
};
Form form_of(const LeafProduct& p, int what) {
  return {leaf_big_fits(p, what), what == LEAF_PRODUCT_Y && by_maps(p),
          wide_tiles(p, what == LEAF_PRODUCT_DX ? p.inputs : p.outputs)};
}

template <typename T>
void launch_product(const LeafProduct& p, int what, const Form& form, hipStream_t s) {
  const bool dx = what == LEAF_PRODUCT_DX;
  const int cols = dx ? p.inputs : p.outputs;
  if (form.big) {
    const int ct = (int)leaf_big_cols(p, what);
    LeafProduct q = p;
    q.rest = p.rest && row_tiles(p.g, BIG_ROWS) * ct > BIG_BLOCKS;
    launch_leaf_big(q, what, s);
    if constexpr (sizeof(T) == 2) {
      if (dx && q.rest)
        k_leaf_tile<T, true, PART_ROWS, PART_ROWS, 2, true>
            <<<dim3(REST_BLOCKS, (unsigned)p.g.trees), THREADS, 0, s>>>(q, p.outputs, cols, ct);
    }
  } else if (dx && p.outputs <= 32) {
    const int ct = (cols + 127) / 128;
    const dim3 grid((unsigned)(row_tiles(p.g, 512) * ct), (unsigned)p.g.trees);
    if (p.outputs <= 4 * El<T>::V)
      k_leaf_dx_narrow<T, 1><<<grid, THREADS, 0, s>>>(p, ct);
    else if constexpr (sizeof(T) == 4)
      k_leaf_dx_narrow<T, 2><<<grid, THREADS, 0, s>>>(p, ct);
  } else if (dx) {
    launch_tiles<T, true>(p, form.wide, s);
  } else if (form.maps) {
    const int ct = (cols + 15) / 16;
    k_leaf_few<T><<<dim3((unsigned)(row_tiles(p.g, 16) * ct), (unsigned)p.g.trees), THREADS, 0, s>>>(p, ct);
  } else if (cols <= 32) {
    const bool one = few_rows(p);
    const dim3 grid((unsigned)row_tiles(p.g, one ? 64 : 256), (unsigned)p.g.trees);
    if (cols <= 16 && one)
      k_leaf_narrow<T, 1, 1><<<grid, 64, 0, s>>>(p);
    else if (cols <= 16)
      k_leaf_narrow<T, 1, 4><<<grid, 256, 0, s>>>(p);
    else if (one)
      k_leaf_narrow<T, 2, 1><<<grid, 64, 0, s>>>(p);
    else
      k_leaf_narrow<T, 2, 4><<<grid, 256, 0, s>>>(p);
  } else {
    launch_tiles<T, false>(p, form.wide, s);
  }
}

// Trees made at a time: as many as have their planes within PLANES, one at least, in runs
// alike.
constexpr int64_t PLANES = (int64_t)4 << 30;
int64_t plane_bytes(const LeafProduct& p, int what) {
  return (int64_t)p.g.rows * (what == LEAF_PRODUCT_DX ? p.inputs : p.outputs) * 4;
}
int run_trees(const LeafProduct& p, int what) {
  const int64_t most = std::max<int64_t>(1, PLANES / std::max<int64_t>(1, plane_bytes(p, what)));
  const int64_t runs = (p.g.trees + most - 1) / most;
  return (int)((p.g.trees + runs - 1) / runs);
}
size_t planes_bytes(const LeafProduct& p, int what) {  // the sums carried over stand behind them
  return ((size_t)run_trees(p, what) * (size_t)plane_bytes(p, what) + 15) / 16 * 16;
}

template <typename T>
void launch(const LeafProduct& p, int what, hipStream_t s) {
  if (what == LEAF_PRODUCT_DW) {
    if (!leaf_big_fits(p, what)) return launch_dw<T>(p, s);
    launch_leaf_big(p, what, s);
    const Split split = leaf_big_split(p);
    if (split.rows) sum_slots<T>(p, split, !leaf_big_ranks(p.g), s);
    return;
  }
  const Form form = what == LEAF_LAYER ? Form{} : form_of(p, what);
  const auto make = [&](const LeafProduct& q) {
    if (what == LEAF_LAYER)
      launch_leaf_layer(q, p.g.trees, s);
    else
      launch_product<T>(q, what, form, s);
  };
  if (p.g.trees == 1) return make(p);
  const int cols = what == LEAF_PRODUCT_DX ? p.inputs : p.outputs, trees = run_trees(p, what);
  const int64_t total = (int64_t)p.g.rows * cols;
  double* const carry = trees < p.g.trees ? (double*)((char*)p.ws + planes_bytes(p, what)) : nullptr;
  for (int t = 0; t < p.g.trees; t += trees) {
    LeafProduct q = p;
    const int64_t leaves = (int64_t)t * p.g.leaves;
    q.planes = true;
    q.g.trees = std::min(trees, p.g.trees - t);
    q.g.order += (int64_t)t * p.g.rows, q.g.begin += leaves, q.g.count += leaves;
    q.w = (const T*)p.w + leaves * p.map_rows() * p.inputs;
    if (p.b) q.b = (const T*)p.b + leaves * p.map_rows();
    if (p.dy) q.dy = (const T*)p.dy + t * p.dy_tree;
    if (p.z) q.z = p.z_of<T>(t);
    make(q);
    const Run run{carry, t == 0, t + trees >= p.g.trees, p.res, p.ldr};
    const float* const planes = (const float*)p.ws;
    const auto blocks = [&](int64_t elements, int64_t most) { return (unsigned)std::min(elements, most); };
    if (q.g.trees >= 16)
      k_sum_trees<T><<<blocks((total + 63) / 64, 1 << 20), THREADS, 0, s>>>(planes, p.g.rows, cols, q.g.trees, run,
                                                                            (T*)p.out, p.ldo);
    else if (p.ldo == cols && total % 4 == 0)
      k_sum_few_trees<T, 4><<<blocks((total / 4 + THREADS - 1) / THREADS, 1 << 16), THREADS, 0, s>>>(
          planes, p.g.rows, cols, q.g.trees, run, (T*)p.out, p.ldo);
    else
      k_sum_few_trees<T, 1><<<blocks((total + THREADS - 1) / THREADS, 1 << 16), THREADS, 0, s>>>(
          planes, p.g.rows, cols, q.g.trees, run, (T*)p.out, p.ldo);
  }
}

}  // namespace

size_t leaf_product_workspace(const LeafProduct& p, int what) {
  if (what == LEAF_PRODUCT_DW) {
    // whatever the pointers' alignment, which may turn the large tiles down
    const DwShape d = dw_shape(p);
    const Split split = dw_split(p, (int64_t)((p.outputs + d.bm - 1) / d.bm) * ((p.inputs + d.bn - 1) / d.bn));
    LeafProduct any = p;
    any.x = any.dy = nullptr, any.ldx = any.lddy = 0;
    const int64_t slots = std::max(split.slots, leaf_big_fits(any, what) ? leaf_big_split(any).slots : 0);
    return (size_t)p.g.trees * (size_t)slots * (size_t)p.outputs * (size_t)(p.inputs + 1) * 4;
  }
  if (p.g.trees <= 1) return 0;
  return planes_bytes(p, what) + (run_trees(p, what) < p.g.trees ? 2 * (size_t)plane_bytes(p, what) : 0);
}

int64_t leaf_product_blocks(const LeafProduct& p, int what) {
  if (what == LEAF_LAYER) return leaf_layer_blocks(p);
  if (leaf_big_fits(p, what)) return leaf_big_blocks(p, what);
  if (what == LEAF_PRODUCT_DW) {
    const DwShape d = dw_shape(p);
    const int64_t tiles = (int64_t)((p.outputs + d.bm - 1) / d.bm) * ((p.inputs + d.bn - 1) / d.bn);
    const Split split = dw_split(p, tiles);
    const int64_t leaves = (int64_t)p.g.trees * p.g.leaves;
    return split.rows ? std::max(tiles * split.parts, leaves) : tiles * leaves;
  }
  const int64_t cols = what == LEAF_PRODUCT_DX ? p.inputs : p.outputs;
  if (what == LEAF_PRODUCT_DX && p.outputs <= 32) return row_tiles(p.g, 512) * ((cols + 127) / 128);
  if (what == LEAF_PRODUCT_Y && by_maps(p)) return row_tiles(p.g, 16) * ((cols + 15) / 16);
  return row_tiles(p.g, 64) * ((cols + 63) / 64);
}

void launch_leaf_product(const LeafProduct& p, int what, hipStream_t s) {
  if (p.dtype == LGBM_HIP_DTYPE_F32)
    launch<float>(p, what, s);
  else if (p.dtype == LGBM_HIP_DTYPE_BF16)
    launch<__bf16>(p, what, s);
  else
    launch<_Float16>(p, what, s);
}

}  // namespace lgbm
