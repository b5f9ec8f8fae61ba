// leaf_layer.hip — layers of a forest's leaves: y[n] = r[n] + sum over trees of f(z), z = W[t,
// leaf] x[n] + b[t, leaf], f an activation, or gated: the activation of z's first half times its
// second.  Rows come grouped by leaf, as for the linear maps (leaf_product.hip): the products are
// theirs, and what the layer adds is done where the sums are in registers, so that neither z
// (unless it is kept for the gradients) nor the two halves of a gated layer go through memory.
// Several trees write float32 planes that are added together with r.
#include <algorithm>
#include <type_traits>

#include "leaf_layer.h"

namespace lgbm {
namespace {

using namespace mma;

constexpr int THREADS = 256;

// ---- tiles through LDS ------------------------------------------------------------------------

// BM rows by BN rows of a leaf's map a block (half of that many results where gated), 128 bytes
// of the contraction a step through LDS (16 bits: loaded two steps ahead), GM x 4 / GM waves.
// Rows and columns that a tile has more than the layer only make results that are not stored, so
// their loads are those of the last ones; only the end of the contraction needs zeros.  The sums
// of 16 rows of a wave go through LDS to eight neighbouring results a lane, so that z, r and y are
// read and written by 16 bytes.  Short contractions are bound by the steps' latencies: 200003 x
// 100 float32 to 64 with z kept 87 us, 2.6 TB/s; wide ones as k_leaf_tile.
// REST: the parts of large tiles behind their last whole round, of which a row has col_tiles.
template <typename T, bool GATED, int BM, int BN, int GM, bool REST = false>
__global__ __launch_bounds__(THREADS) void k_layer_tile(LeafProduct p, int col_tiles) {
  constexpr int V = El<T>::V, BK = 8 * V;  // elements of the contraction a step
  constexpr int GN = 4 / GM, WM = BM / GM, WN = BN / GN, CW = GATED ? WN / 2 : WN;
  constexpr int ACH = BM * 8 / THREADS, BCH = BN * 8 / THREADS;
  // steps between a load and its use (us by one and two: the parts behind 16389 x 4096 bfloat16 to
  // 2048 47 and 37, 64 rows a leaf, 2048 to 2048 by 31 leaves 89 and 83; float32's, of 32 inputs,
  // 84 and 86)
  constexpr int AHEAD = sizeof(T) == 2 ? 2 : 1;
  constexpr int PITCH = WN + 4, STRIP = 16 * PITCH * 4;
  constexpr int STAGE = (BM + BN) * 128, LDS = 2 * STAGE > 4 * STRIP ? 2 * STAGE : 4 * STRIP;
  __shared__ __align__(16) char lds[LDS];
  __shared__ __align__(16) int32_t row_of[BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tree = blockIdx.y, length = p.inputs, cols = p.outputs;
  constexpr int CB = GATED ? BN / 2 : BN;
  int c0 = (blockIdx.x % col_tiles) * CB;
  const RowTile rt = REST ? rest_tile<THREADS>(p.g, tree, col_tiles, CB, &c0)
                          : find_tile<THREADS>(p.g, tree, blockIdx.x / col_tiles, BM);
  if (rt.rows == 0 || (REST && c0 >= cols)) return;
  for (int r = tid; r < BM; r += THREADS) row_of[r] = r < rt.rows ? row_at(p.g, tree, rt.first + r) : -1;
  __syncthreads();
  const int64_t leaf = rt.leaf < 0 ? -1 : (int64_t)tree * p.g.leaves + rt.leaf;
  const T* const w = (const T*)p.w + (leaf < 0 ? 0 : leaf * p.map_rows() * (int64_t)length);
  const int m0 = (wave / GN) * WM, n0 = (wave % GN) * WN;

  f32x4 acc[WM / 16][WN / 16];
#pragma unroll
  for (int i = 0; i < WM / 16; ++i)
#pragma unroll
    for (int j = 0; j < WN / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

  if (leaf >= 0) {
    u32x4 ra[AHEAD][ACH], rb[AHEAD][BCH];  // of even and odd steps
    const T *arow[ACH], *brow[BCH];
#pragma unroll
    for (int i = 0; i < ACH; ++i)
      arow[i] = (const T*)p.x + (int64_t)max(row_of[(tid + i * THREADS) >> 3], 0) * p.ldx + (tid & 7) * V;
#pragma unroll
    for (int i = 0; i < BCH; ++i)
      brow[i] = w + (int64_t)map_row<GATED, WN>((tid + i * THREADS) >> 3, c0, cols) * length + (tid & 7) * V;
    const auto load = [&](int k0, auto set) {
      constexpr int S = decltype(set)::value;
      if (k0 + BK <= length) {
#pragma unroll
        for (int i = 0; i < ACH; ++i) ra[S][i] = load16(arow[i] + k0);
#pragma unroll
        for (int i = 0; i < BCH; ++i) rb[S][i] = load16(brow[i] + k0);
      } else if (k0 < length) {
        const int valid = length - k0 - (tid & 7) * V;
#pragma unroll
        for (int i = 0; i < ACH; ++i) ra[S][i] = load16(arow[i] + k0, valid);
#pragma unroll
        for (int i = 0; i < BCH; ++i) rb[S][i] = load16(brow[i] + k0, valid);
      }
    };
    const auto store = [&](char* buf, auto set) {
      constexpr int S = decltype(set)::value;
#pragma unroll
      for (int i = 0; i < ACH; ++i) {
        const int at = tid + i * THREADS;
        *reinterpret_cast<u32x4*>(buf + kc_at(at >> 3, at & 7)) = ra[S][i];
      }
#pragma unroll
      for (int i = 0; i < BCH; ++i) {
        const int at = tid + i * THREADS;
        *reinterpret_cast<u32x4*>(buf + BM * 128 + kc_at(at >> 3, at & 7)) = rb[S][i];
      }
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, AHEAD - 1> odd;
    // the step at k0, whose loads were `set`, in half b of the LDS
    const auto step_at = [&](int k0, int b, auto set, auto other) {
      const bool more = k0 + BK < length;
      load(k0 + AHEAD * BK, set);
      const char *ta = lds + b * STAGE, *tb = ta + BM * 128;
      Parts<T, WM / 16, WN / 16> part(acc);
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        if (step == 1 && k0 + BK / 2 >= length) break;
        u32x4 fa[WM / 16], fb[WN / 16];
#pragma unroll
        for (int i = 0; i < WM / 16; ++i) fa[i] = kc_frag(ta, m0 + 16 * i, step, lane);
#pragma unroll
        for (int j = 0; j < WN / 16; ++j) fb[j] = kc_frag(tb, n0 + 16 * j, step, lane);
#pragma unroll
        for (int i = 0; i < WM / 16; ++i)
#pragma unroll
          for (int j = 0; j < WN / 16; ++j) part.at[i][j] = El<T>::mfma(fa[i], fb[j], part.at[i][j]);
      }
      part.add_to(acc);
      if (more) store(lds + (b ^ 1) * STAGE, other);
      __syncthreads();
    };
    load(0, even);
    if (AHEAD == 2) load(BK, odd);
    store(lds, even);
    __syncthreads();
    if constexpr (AHEAD == 2) {
      for (int k0 = 0; k0 < length; k0 += 2 * BK) {
        step_at(k0, 0, even, odd);
        if (k0 + BK < length) step_at(k0 + BK, 1, odd, even);
      }
    } else {
      for (int k0 = 0, b = 0; k0 < length; k0 += BK, b ^= 1) step_at(k0, b, even, even);
    }
  }

  // lane: rows 4 (lane / 16) .. + 4, column lane % 16 of each 16 x 16
  float* const mine = reinterpret_cast<float*>(lds + wave * STRIP);
#pragma unroll
  for (int i = 0; i < WM / 16; ++i) {
#pragma unroll
    for (int j = 0; j < WN / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[((lane >> 4) * 4 + e) * PITCH + j * 16 + (lane & 15)] = acc[i][j][e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int at = lane; at < 16 * (CW / 8); at += 64) {
      const int row = at / (CW / 8), col = at % (CW / 8) * 8;
      float a[8], u[8];
      __builtin_memcpy(a, mine + row * PITCH + col, sizeof(a));
      if (GATED) __builtin_memcpy(u, mine + row * PITCH + WN / 2 + col, sizeof(u));
      layer_end_of_sums<T, GATED>(p, tree, leaf, row_of[m0 + i * 16 + row], c0 + (wave % GN) * CW + col, a, u);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- few rows a leaf ------------------------------------------------------------------------------

// Bound by reading the maps: a block makes 16 RB rows by 16 results of a leaf (32 rows of its map
// where gated); its waves take every WAVES-th stretch of the inputs, and their sums are added in
// LDS in the waves' order.  A wave's stretch is BYTES of every row, side by side in the lanes (a
// matrix instruction takes 16 rows side by side: loads in its order touch a line for every lane,
// 64 bfloat16 rows of 4096 to 4096 23 us instead of 15), and goes through LDS to the lanes that need
// it, the next stretch on its way.  One row of 4096 to 4096 gated: 13.6 us, 4.9 TB/s; 64 rows, whose
// inputs every block reads from L2, 14.8 us; 16 rows to 2048 gated float16 by 31 leaves 56 to 75 us
// for the 11 to 13 maps of 34 MB that are hit.
template <typename T, bool GATED, int RB, int WAVES, int BYTES>
__attribute__((amdgpu_waves_per_eu(1, 4))) __global__ __launch_bounds__(WAVES * 64) void k_layer_few(LeafProduct p, int col_tiles) {
  constexpr int V = El<T>::V, NB = GATED ? 2 : 1, PART = BYTES / (int)sizeof(T), STEPS = BYTES / 64;
  constexpr int CH = BYTES / 16, PER = 64 / CH;  // chunks a row, rows a load
  constexpr int XLOADS = 16 * RB / PER, LOADS = XLOADS + 16 * NB / PER, STAGE = 16 * (RB + NB) * BYTES;
  constexpr int PITCH = 16 * NB + 4, SUMS = 16 * RB * PITCH * 4;
  __shared__ __align__(16) char lds[WAVES * (STAGE > SUMS ? STAGE : SUMS)];
  __shared__ int32_t row_of[16 * RB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  const int tree = blockIdx.y, length = p.inputs, cols = p.outputs;
  const int c0 = (int)(blockIdx.x % col_tiles) * 16;
  const RowTile rt = find_tile<WAVES * 64>(p.g, tree, blockIdx.x / col_tiles, 16 * RB);
  if (rt.rows == 0) return;
  const int64_t leaf = rt.leaf < 0 ? -1 : (int64_t)tree * p.g.leaves + rt.leaf;
  if (tid < 16 * RB) row_of[tid] = tid < rt.rows ? row_at(p.g, tree, rt.first + tid) : -1;
  __syncthreads();
  f32x4 acc[RB][NB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  if (leaf >= 0) {
    char* const mine = lds + wave * STAGE;
    const int chunk = lane % CH;
    // rows in the order of the stage: x's, the gates', the other half's
    const T* from[LOADS];
    int to[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = i * PER + lane / CH;
      if (i < XLOADS)
        from[i] = (const T*)p.x + (int64_t)max(row_of[row], 0) * p.ldx;
      else
        from[i] = (const T*)p.w + (leaf * p.map_rows() + (row - 16 * RB) / 16 * cols + min(c0 + row % 16, cols - 1)) *
                                      (int64_t)length;
      from[i] += chunk * V;
      to[i] = row * BYTES + ((chunk ^ row) & (CH - 1)) * 16;
    }
    u32x4 ahead[LOADS];
    const auto load = [&](int k0) {
      if (k0 + PART <= length) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) ahead[i] = load16(from[i] + k0);
      } else if (k0 < length) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) ahead[i] = load16(from[i] + k0, length - k0 - chunk * V);
      }
    };
    load(wave * PART);
    for (int k0 = wave * PART; k0 < length; k0 += WAVES * PART) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) *reinterpret_cast<u32x4*>(mine + to[i]) = ahead[i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      load(k0 + WAVES * PART);
      Parts<T, RB, NB> part(acc);
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        const auto frag = [&](int row0) {
          const int row = row0 + r;
          return *reinterpret_cast<const u32x4*>(mine + row * BYTES + (((u * 4 + q) ^ row) & (CH - 1)) * 16);
        };
        u32x4 fw[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) fw[j] = frag(16 * (RB + j));
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          const u32x4 fx = frag(16 * i);
#pragma unroll
          for (int j = 0; j < NB; ++j) part.at[i][j] = El<T>::mfma(fx, fw[j], part.at[i][j]);
        }
      }
      part.add_to(acc);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
  }
  float* const sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sums[wave * (SUMS / 4) + (i * 16 + q * 4 + e) * PITCH + j * 16 + r] = acc[i][j][e];
  __syncthreads();
  // eight results a thread
  for (int at = tid; at < 16 * RB * 2; at += WAVES * 64) {
    const int row = at >> 1, col = (at & 1) * 8;
    float a[8] = {}, u[8] = {};
#pragma unroll
    for (int v = 0; v < WAVES; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] += sums[v * (SUMS / 4) + row * PITCH + col + j];
        if (GATED) u[j] += sums[v * (SUMS / 4) + row * PITCH + 16 + col + j];
      }
    layer_end_of_sums<T, GATED>(p, tree, leaf, row_of[row], c0 + col, a, u);
  }
}

// ---- few outputs ----------------------------------------------------------------------------------

// Up to 16 NB outputs of a leaf: bound by reading x, which no wave shares with another, so lanes
// load their fragments straight from memory, UNROLL steps at a time and without a barrier; maps
// come from the caches.  A wave takes ROUNDS times 32 rows; blocks of one wave where leaves hold
// few rows.  Sums stay in registers to the end: lane r of 16 has column r of the outputs.  2M x 28
// float32 to 10 by 127 leaves onto a residual: 173 us for 507 MB read and written; rows of 112 and
// 40 bytes spread over the table make 9.4M requests to L2, and the address units are busy 72 % of
// the time (119 us where a leaf's rows lie side by side; whole maps in LDS and rows loaded side by
// side through LDS took as long).
template <typename T, bool GATED, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void k_layer_narrow(LeafProduct p) {
  constexpr int V = El<T>::V, UNROLL = 4, ROUNDS = 2, BM = WAVES * 32 * ROUNDS, M = GATED ? 2 * NB : NB;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int tree = blockIdx.y, length = p.inputs, cols = p.outputs, rows = p.map_rows();
  const RowTile rt = find_tile<WAVES * 64>(p.g, tree, blockIdx.x, BM);
  if (rt.rows == 0) return;
  const int64_t leaf = (int64_t)tree * p.g.leaves + rt.leaf;
  const T* const w = (const T*)p.w + (rt.leaf < 0 ? 0 : leaf * rows * (int64_t)length);
  // group j of 16 map rows: outputs 16 (j % NB) on, of the gates or the second half
  const T* wrow[M];
  float b[M];
#pragma unroll
  for (int j = 0; j < M; ++j) {
    const int at = j / NB * cols + min(j % NB * 16 + r, cols - 1);
    wrow[j] = w + (int64_t)at * length;
    b[j] = p.b && rt.leaf >= 0 ? (float)((const T*)p.b)[leaf * rows + at] : 0.0f;
  }
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
    // the rows of a lane's results, and what they have already
    int of[2][4];
    float res[2][NB][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      rows_of(n[t][i], lane, of[i]);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = j * 16 + r;
          const bool has = p.res && !p.planes && of[i][e] >= 0 && col < cols;
          res[i][j][e] = has ? (float)((const T*)p.res)[of[i][e] * p.ldr + col] : 0.0f;
        }
    }
    f32x4 acc[2][M];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < M; ++j) acc[i][j] = f32x4{b[j], b[j], b[j], b[j]};
    if (rt.leaf >= 0) {
      const T* xrow[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) xrow[i] = (const T*)p.x + (int64_t)max(n[t][i], 0) * p.ldx;
      const auto stretch = [&](int k0, auto whole) {
        u32x4 fa[UNROLL][2], fb[UNROLL][M];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          const int k = k0 + (u * 4 + q) * V;
#pragma unroll
          for (int i = 0; i < 2; ++i) fa[u][i] = whole ? load16(xrow[i] + k) : load16(xrow[i] + k, length - k);
#pragma unroll
          for (int j = 0; j < M; ++j) fb[u][j] = whole ? load16(wrow[j] + k) : load16(wrow[j] + k, length - k);
        }
        Parts<T, 2, M> part(acc);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          if (k0 + u * 4 * V >= length) break;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j) part.at[i][j] = El<T>::mfma(fa[u][i], fb[u][j], part.at[i][j]);
        }
        part.add_to(acc);
      };
      int k0 = 0;
      for (; k0 + 4 * V * UNROLL <= length; k0 += 4 * V * UNROLL) stretch(k0, std::true_type());
      if (k0 < length) stretch(k0, std::false_type());
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int col = j * 16 + r;
        float a[4], f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = acc[i][j][e];
        if (p.z) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (of[i][e] < 0 || col >= cols) continue;
            const int64_t at = (int64_t)of[i][e] * rows + col;
            if (sizeof(T) == 2 && p.z_narrow) {
              T* const z = (T*)p.z_of<T>(tree) + at;
              z[0] = (T)a[e];
              if (GATED) z[cols] = (T)acc[i][GATED ? NB + j : 0][e];
            } else {
              float* const z = (float*)p.z_of<T>(tree) + at;
              z[0] = a[e];
              if (GATED) z[cols] = acc[i][GATED ? NB + j : 0][e];
            }
          }
        }
        activate<T>(p.act, a, f);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = GATED ? f[e] * acc[i][GATED ? NB + j : 0][e] : f[e];
          if (rt.leaf < 0) v[e] = 0.0f;
          v[e] += res[i][j][e];
        }
        store_rows<T>(p, tree, of[i], col, cols, v);
      }
    }
  }
}

// ---- the gradient of z ----------------------------------------------------------------------------

// dz = dy f'(z), or where gated dy f'(z_gate) z_up and dy f(z_gate): eight neighbouring results a
// thread.  Bound by memory (16389 rows of 2048 gated bfloat16 results, z in float32: 88 us, 5.3
// TB/s).  dz is rounded to the type, as the products that take it need, and dbias is the sum of
// the same dz, which is read once for both; z, of type Z, is float32 unless the caller kept it
// rounded, so that this is the only rounding between the layer's inputs and its gradients' sums.
// (In bfloat16 it takes dx and dW from 0.0017 of their own, their last rounding's, to 0.0023.)
template <typename T, typename Z, bool GATED>
__global__ __launch_bounds__(THREADS) void k_layer_dz(LeafProduct p, int64_t pieces, T* dz) {
  const int cols = p.outputs, across = (cols + 7) / 8;
  for (int64_t i = blockIdx.x * (int64_t)THREADS + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * THREADS) {
    const int64_t at = i / across;  // tree and row
    const int col = (int)(i - at * across) * 8, valid = min(8, cols - col);
    const int64_t n = at % p.g.rows, from = at * (GATED ? 2 * (int64_t)cols : cols) + col;
    float dy[8], a[8], u[8];
    load8((const T*)p.dy + n * p.lddy + col, valid, dy);
    load8((const Z*)p.z + from, valid, a);
    if (GATED) load8((const Z*)p.z + from + cols, valid, u);
    float da[8], du[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f, d;
      slope_of<T>(p.act, a[j], f, d);
      da[j] = GATED ? dy[j] * u[j] * d : dy[j] * d;
      du[j] = dy[j] * f;
    }
    store8(dz + from, valid, da);
    if (GATED) store8(dz + from + cols, valid, du);
  }
}

// ---- which kernel ---------------------------------------------------------------------------------

// The large tiles of leaf_big.hip, by all the trees, however few of them are made at a time.
bool big_tiles(LeafProduct p, int trees) {
  p.g.trees = trees;
  return leaf_big_fits(p, LEAF_LAYER);
}

// Leaves of 16 rows at most, on average.
bool few_rows_a_leaf(const LeafProduct& p) { return p.g.rows <= 16 * (int64_t)p.g.leaves; }

// Rows a block of k_layer_few, in units of 16, 0: not for it.  Few outputs of so few rows that
// k_layer_narrow's blocks would leave CUs without work, as for the linear maps (by_maps); leaves of
// 32 rows at most, on average; and 64 x 64 tiles that are fewer than about 320 (us by it and by those
// tiles: 4096 bfloat16 inputs to 4096, one leaf, 64 rows 16.7 and 42.5, 256 rows 38 and 43.5, 384
// rows 52 and 47; to 2048 gated, 256 rows 25 and 44; float32, 256 rows 115 and 120, 512 rows 206
// and 174; 48 rows a leaf, 4096 to 4096 by seven leaves 93 and 73, 600 to 100 by 127 24 and 20).
int few_rows(const LeafProduct& p) {
  if (p.inputs >= 128 && p.outputs <= 32 && (int64_t)p.g.rows * ((p.outputs + 15) / 16) < 49152) return 1;
  if (p.inputs < 512) return 0;
  const int64_t rows = (p.g.rows + p.g.leaves - 1) / p.g.leaves;
  if (rows <= 32) return rows <= 16 ? 1 : 2;
  return ((int64_t)p.g.rows / 64 + p.g.leaves) * ((p.map_rows() + 63) / 64) <= 320 ? 4 : 0;
}

// Tiles of 128 x 128, as for the linear maps (wide_tiles).
bool wide_tiles(const LeafProduct& p, int trees) {
  const int rows = p.map_rows();
  return p.dtype != LGBM_HIP_DTYPE_F32 && rows >= 128 && p.g.rows >= 128 * (int64_t)p.g.leaves &&
         (int64_t)p.g.rows / 128 * ((rows + 127) / 128) * trees >= 256;
}

template <typename T, bool GATED, int BM, int BN>
void launch_tile(const LeafProduct& p, hipStream_t s) {
  constexpr int CB = GATED ? BN / 2 : BN;
  const int ct = (p.outputs + CB - 1) / CB;
  const dim3 grid((unsigned)(row_tiles(p.g, BM) * ct), (unsigned)p.g.trees);
  k_layer_tile<T, GATED, BM, BN, 2><<<grid, THREADS, 0, s>>>(p, ct);
}

// Large tiles, and what is behind their last whole round.
template <typename T, bool GATED>
void launch_big(LeafProduct p, hipStream_t s) {
  const int ct = (int)leaf_big_cols(p, LEAF_LAYER);
  p.rest = row_tiles(p.g, BIG_ROWS) * ct > BIG_BLOCKS;
  launch_leaf_big(p, LEAF_LAYER, s);
  if (p.rest)
    k_layer_tile<T, GATED, PART_ROWS, PART_ROWS, 2, true><<<dim3(REST_BLOCKS, (unsigned)p.g.trees), THREADS, 0, s>>>(p, ct);
}

template <typename T, bool GATED, int RB>
void launch_few(const LeafProduct& p, hipStream_t s) {
  const int ct = (p.outputs + 15) / 16;
  const dim3 grid((unsigned)(row_tiles(p.g, 16 * RB) * ct), (unsigned)p.g.trees);
  // 256 bytes a row of few rows, 128 of many (64 rows of 4096 bfloat16 inputs to 4096: 16.1 and
  // 14.7 us; one row to 4096 gated: 13.6 and 14.1)
  k_layer_few<T, GATED, RB, 4, RB == 1 ? 256 : 128><<<grid, 256, 0, s>>>(p, ct);
}

template <typename T, bool GATED>
void launch(const LeafProduct& p, int trees, hipStream_t s) {
  const int few = few_rows(p);
  if (few == 1) return launch_few<T, GATED, 1>(p, s);
  if (few == 2) return launch_few<T, GATED, 2>(p, s);
  if (few == 4) return launch_few<T, GATED, 4>(p, s);
  if (p.outputs <= 32) {
    const bool one = few_rows_a_leaf(p);
    const dim3 grid((unsigned)row_tiles(p.g, one ? 64 : 256), (unsigned)p.g.trees);
    if (p.outputs <= 16 && one)
      k_layer_narrow<T, GATED, 1, 1><<<grid, 64, 0, s>>>(p);
    else if (p.outputs <= 16)
      k_layer_narrow<T, GATED, 1, 4><<<grid, 256, 0, s>>>(p);
    else if (one)
      k_layer_narrow<T, GATED, 2, 1><<<grid, 64, 0, s>>>(p);
    else
      k_layer_narrow<T, GATED, 2, 4><<<grid, 256, 0, s>>>(p);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (big_tiles(p, trees)) return launch_big<T, GATED>(p, s);
    if (wide_tiles(p, trees)) return launch_tile<T, GATED, 128, 128>(p, s);
  }
  launch_tile<T, GATED, 64, 64>(p, s);
}

template <typename T, bool GATED>
void launch_dz(const LeafProduct& p, void* dz, hipStream_t s) {
  const int64_t pieces = (int64_t)p.g.trees * p.g.rows * ((p.outputs + 7) / 8);
  const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>((pieces + THREADS - 1) / THREADS, 1 << 16));
  if (p.z_narrow)
    k_layer_dz<T, T, GATED><<<grid, THREADS, 0, s>>>(p, pieces, (T*)dz);
  else
    k_layer_dz<T, float, GATED><<<grid, THREADS, 0, s>>>(p, pieces, (T*)dz);
}

}  // namespace

int64_t leaf_layer_blocks(const LeafProduct& p) {
  if (leaf_big_fits(p, LEAF_LAYER)) return leaf_big_blocks(p, LEAF_LAYER);
  if (const int few = few_rows(p)) return row_tiles(p.g, 16 * few) * ((p.outputs + 15) / 16);
  const int64_t cb = p.gated ? 32 : 64;
  return row_tiles(p.g, 64) * ((p.outputs + cb - 1) / cb);
}

void launch_leaf_layer(const LeafProduct& p, int trees, hipStream_t s) {
  if (p.dtype == LGBM_HIP_DTYPE_F32)
    p.gated ? launch<float, true>(p, trees, s) : launch<float, false>(p, trees, s);
  else if (p.dtype == LGBM_HIP_DTYPE_BF16)
    p.gated ? launch<__bf16, true>(p, trees, s) : launch<__bf16, false>(p, trees, s);
  else
    p.gated ? launch<_Float16, true>(p, trees, s) : launch<_Float16, false>(p, trees, s);
}

void launch_layer_dz(const LeafProduct& p, void* dz, hipStream_t s) {
  if (p.dtype == LGBM_HIP_DTYPE_F32)
    p.gated ? launch_dz<float, true>(p, dz, s) : launch_dz<float, false>(p, dz, s);
  else if (p.dtype == LGBM_HIP_DTYPE_BF16)
    p.gated ? launch_dz<__bf16, true>(p, dz, s) : launch_dz<__bf16, false>(p, dz, s);
  else
    p.gated ? launch_dz<_Float16, true>(p, dz, s) : launch_dz<_Float16, false>(p, dz, s);
}

}  // namespace lgbm
