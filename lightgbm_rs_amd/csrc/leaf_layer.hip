// leaf_layer.hip — layers of a forest's leaves: y[n] = r[n] + sum over trees of f(z), z = W[t,
// leaf] x[n] + b[t, leaf], f an activation, or gated: the activation of z's first half times its
// second.  Rows come grouped by leaf, as for the linear maps (leaf_product.hip): the products are
// theirs, and what the layer adds is done where the sums are in registers, so that neither z
// (unless it is kept for the gradients) nor the two halves of a gated layer go through memory.
// Several trees write float32 planes that are added together with r.
#include <algorithm>

#include "leaf_layer.h"

namespace lgbm {
namespace {

using namespace mma;

constexpr int THREADS = 256;

// ---- tiles through LDS ------------------------------------------------------------------------

// BM rows by BN rows of a leaf's map a block (half of that many results where gated), 128 bytes
// of the contraction a step through LDS, GM x 4 / GM waves.  Rows and columns that a tile has
// more than the layer only make results that are not stored, so their loads are those of the
// last ones; only the end of the contraction needs zeros.  The sums of 16 rows of a wave go
// through LDS to eight neighbouring results a lane, so that z, r and y are read and written by
// 16 bytes.
template <typename T, bool GATED, int BM, int BN, int GM>
__global__ __launch_bounds__(THREADS) void k_layer_tile(LeafProduct p, int col_tiles) {
  constexpr int V = El<T>::V, BK = 8 * V;  // elements of the contraction a step
  constexpr int GN = 4 / GM, WM = BM / GM, WN = BN / GN, CW = GATED ? WN / 2 : WN;
  constexpr int ACH = BM * 8 / THREADS, BCH = BN * 8 / THREADS;
  constexpr int PITCH = WN + 4, STRIP = 16 * PITCH * 4;
  constexpr int STAGE = (BM + BN) * 128, LDS = 2 * STAGE > 4 * STRIP ? 2 * STAGE : 4 * STRIP;
  __shared__ __align__(16) char lds[LDS];
  __shared__ __align__(16) int32_t row_of[BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tree = blockIdx.y, length = p.inputs, cols = p.outputs;
  const int mt = blockIdx.x / col_tiles, c0 = (blockIdx.x % col_tiles) * (GATED ? BN / 2 : BN);
  const RowTile rt = find_tile<THREADS>(p.g, tree, mt, BM);
  if (rt.rows == 0) return;
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
    u32x4 ra[ACH], rb[BCH];
    const T *arow[ACH], *brow[BCH];
#pragma unroll
    for (int i = 0; i < ACH; ++i) arow[i] = (const T*)p.x + (int64_t)max(row_of[(tid + i * THREADS) >> 3], 0) * p.ldx;
#pragma unroll
    for (int i = 0; i < BCH; ++i) brow[i] = w + (int64_t)map_row<GATED, WN>((tid + i * THREADS) >> 3, c0, cols) * length;
    auto load = [&](int k0) {
      const int k = k0 + (tid & 7) * V;
      const bool whole = k0 + BK <= length;
#pragma unroll
      for (int i = 0; i < ACH; ++i) ra[i] = whole ? load16(arow[i] + k) : load16(arow[i] + k, length - k);
#pragma unroll
      for (int i = 0; i < BCH; ++i) rb[i] = whole ? load16(brow[i] + k) : load16(brow[i] + k, length - k);
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
        *reinterpret_cast<u32x4*>(buf + BM * 128 + kc_at(at >> 3, at & 7)) = rb[i];
      }
    };
    load(0);
    store(lds);
    __syncthreads();
    for (int k0 = 0, b = 0; k0 < length; k0 += BK, b ^= 1) {
      const bool more = k0 + BK < length;
      if (more) load(k0 + BK);
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
      if (more) store(lds + (b ^ 1) * STAGE);
      __syncthreads();
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
      layer_end<T, GATED>(p, tree, leaf, row_of[m0 + i * 16 + row], c0 + (wave % GN) * CW + col, a, u);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- the gradient of z ----------------------------------------------------------------------------

// dz = dy f'(z), or where gated dy f'(z_gate) z_up and dy f(z_gate): eight neighbouring results a
// thread.  Bound by memory.  dz is rounded to the type, as the products that take it need; z, of
// type Z, is float32 unless the caller kept it rounded, so that this is the only rounding between
// the layer's inputs and its gradients' sums.
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

template <typename T, bool GATED>
void launch(const LeafProduct& p, int trees, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
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
