// leaf_big.hip — the leaves' linear maps in 16 bits where leaves hold hundreds of rows and
// wide maps: bound by the matrix cores.
//
// A block of 8 waves makes 256 x 256 of a result, a wave 128 x 64 of it in registers.  64
// elements of the contraction a step pass through LDS, in two buffers: while the matrix
// instructions work on one, loads that go to LDS directly fill the other (rows and chunks
// are addressed a lane, so the gather through the order costs nothing and the swizzle is
// made by the addresses).  A lane beyond the operand reads zeros.
#include <algorithm>

#include "leaf_mma.h"

namespace lgbm {
namespace {

using namespace mma;

constexpr int THREADS = 512, BM = 256, BN = 256, BK = 64, WM = 128, WN = 64;

__device__ __align__(16) unsigned int zeros[4];

typedef const __attribute__((address_space(1))) void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// 64 lanes x 16 bytes to `to` (wave-uniform) and the 1 KB behind it.
__device__ __forceinline__ void load_lds(const void* from, char* to) {
  __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)to, 16, 0, 0);
}

// MODE LEAF_PRODUCT_Y: a = x rows [k], b = w[leaf] [col][k]; _DX: a = dy rows [m], b = w[leaf]
// [m][col]; _DW: a = dy [row][m], b = x [row][k] over a leaf's rows.
template <typename T, int MODE>
__global__ __launch_bounds__(THREADS) void k_leaf_big(LeafProduct p, int col_tiles) {
  constexpr bool DW = MODE == LEAF_PRODUCT_DW, ACM = DW, BCM = MODE != LEAF_PRODUCT_Y;
  __shared__ __align__(1024) char a0[BM * 128], b0[BN * 128], a1[BM * 128], b1[BN * 128];
  __shared__ int32_t row_of[DW ? 1 : BM];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = (wave >> 2) * WM, wn = (wave & 3) * WN;

  // the block's part of the result, and the length of the contraction
  int tree, first = 0, length, m0 = 0, c0, cols, rows = BM;
  int64_t leaf;
  if (DW) {
    const int tiles = (p.outputs + BM - 1) / BM * col_tiles, tile = (int)(blockIdx.x % tiles);
    leaf = blockIdx.x / tiles;
    tree = (int)(leaf / p.g.leaves);
    length = min(max(p.g.count[leaf], 0), p.g.rows);
    first = min(max(p.g.begin[leaf], 0), p.g.rows - length);
    m0 = tile / col_tiles * BM, c0 = tile % col_tiles * BN, cols = p.inputs;
  } else {
    tree = blockIdx.y;
    length = MODE == LEAF_PRODUCT_Y ? p.inputs : p.outputs;
    cols = MODE == LEAF_PRODUCT_Y ? p.outputs : p.inputs;
    // neighbouring tiles to one XCD, which shares their rows and maps in its L2
    const int tiles = count_tiles<THREADS>(p.g, tree, BM) * col_tiles, share = (tiles + 7) / 8;
    const int slot = (int)(blockIdx.x >> 3), id = (int)(blockIdx.x & 7) * share + slot;
    if (slot >= share || id >= tiles) return;
    const RowTile rt = find_tile<THREADS>(p.g, tree, id / col_tiles, BM);
    c0 = id % col_tiles * BN;
    if (rt.rows == 0) return;
    rows = rt.rows;
    leaf = rt.leaf < 0 ? -1 : (int64_t)tree * p.g.leaves + rt.leaf;
    if (tid < BM) row_of[tid] = tid < rows ? row_at(p.g, tree, rt.first + tid) : -1;
    __syncthreads();
    if (leaf < 0) length = 0;
  }
  const T* const w = (const T*)p.w + (DW || leaf < 0 ? 0 : leaf * p.outputs * (int64_t)p.inputs);

  // a lane's addresses: four loads of each operand a step.  Along the contraction: row
  // 8 (4 wave + j) + lane / 8, chunk lane % 8 (swizzled); contraction-major: row 2 (4 wave +
  // j) + lane / 32, 16 bytes lane % 32 (swizzled).
  const int kc_row = wave * 32 + (lane >> 3), cm_row = wave * 8 + (lane >> 5);
  const T *abase[4], *bbase[4];
  int acol[4], bcol[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = cm_row + 2 * j, sw = cm_swizzle<T>(row);
    const int unit = ((lane & 31) >> 1) ^ sw, in = (unit * 2 + (lane & 1)) * 8;
    const int kr = kc_row + 8 * j, kchunk = ((lane & 7) ^ (kr & 7)) * 8;
    if (ACM) {
      acol[j] = m0 + in;
    } else {
      acol[j] = kchunk;
      const T* const src = (const T*)(MODE == LEAF_PRODUCT_Y ? p.x : p.dy);
      abase[j] = src + (int64_t)max(row_of[DW ? 0 : kr], 0) * (MODE == LEAF_PRODUCT_Y ? p.ldx : p.lddy) + kchunk;
    }
    if (BCM) {
      bcol[j] = c0 + in;
    } else {
      bcol[j] = kchunk;
      bbase[j] = w + (int64_t)min(c0 + kr, cols - 1) * length + kchunk;
    }
  }
  int next_row[4];  // DW: the rows of the step that is loaded next
  auto fetch_rows = [&](int k0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = k0 + cm_row + 2 * j;
      next_row[j] = at < length ? row_at(p.g, tree, first + at) : -1;
    }
  };
  auto load = [&](int k0, char* a, char* b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const void *from_a, *from_b;
      if (DW) {
        const int n = next_row[j];
        from_a = n >= 0 && acol[j] < p.outputs ? (const T*)p.dy + n * p.lddy + acol[j] : (const void*)zeros;
        from_b = n >= 0 && bcol[j] < cols ? (const T*)p.x + n * p.ldx + bcol[j] : (const void*)zeros;
      } else {
        from_a = k0 + acol[j] < length ? abase[j] + k0 : (const void*)zeros;
        if (BCM) {
          const int m = k0 + cm_row + 2 * j;
          from_b = m < length && bcol[j] < cols ? w + (int64_t)m * cols + bcol[j] : (const void*)zeros;
        } else {
          from_b = k0 + bcol[j] < length ? bbase[j] + k0 : (const void*)zeros;
        }
      }
      load_lds(from_a, a + (wave * 4 + j) * 1024);
      load_lds(from_b, b + (wave * 4 + j) * 1024);
    }
    if (DW) fetch_rows(k0 + BK);
  };

  f32x4 acc[WM / 16][WN / 16];
  float bias[DW ? WM / 16 : 1];  // of the lane's chunks
#pragma unroll
  for (int i = 0; i < WM / 16; ++i)
#pragma unroll
    for (int j = 0; j < WN / 16; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < (DW ? WM / 16 : 1); ++i) bias[i] = 0.0f;
  const bool sums = DW && p.db && c0 == 0 && wn == 0;

  auto compute = [&](const char* a, const char* b) {
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      u32x4 fa[WM / 16], fb[WN / 16];
#pragma unroll
      for (int j = 0; j < WN / 16; ++j)
        fb[j] = BCM ? cm_frag<T, BN>(b, wn + 16 * j, step, lane) : kc_frag(b, wn + 16 * j, step, lane);
#pragma unroll
      for (int i = 0; i < WM / 16; ++i)
        fa[i] = ACM ? cm_frag<T, BM>(a, wm + 16 * i, step, lane) : kc_frag(a, wm + 16 * i, step, lane);
      if (DW && sums)
#pragma unroll
        for (int i = 0; i < WM / 16; ++i) {
          T e[8];
          __builtin_memcpy(e, &fa[i], 16);
#pragma unroll
          for (int k = 0; k < 8; ++k) bias[DW ? i : 0] += (float)e[k];
        }
#pragma unroll
      for (int i = 0; i < WM / 16; ++i)
#pragma unroll
        for (int j = 0; j < WN / 16; ++j) acc[i][j] = El<T>::mfma(fb[j], fa[i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (DW) fetch_rows(0);
  if (length > 0) load(0, a0, b0);
  for (int k0 = 0; k0 < length; k0 += 2 * BK) {
    __syncthreads();  // the loads are there, and the other buffer has been read
    load(k0 + BK, a1, b1);  // behind the end: zeros
    compute(a0, b0);
    __syncthreads();
    if (k0 + 2 * BK < length) load(k0 + 2 * BK, a0, b0);
    compute(a1, b1);
  }

  // lane: row lane % 16, columns 4 (lane / 16) .. + 4 of each 16 x 16
  if (DW) {
    float* const dw = p.dw + leaf * p.outputs * (int64_t)p.inputs;
#pragma unroll
    for (int i = 0; i < WM / 16; ++i) {
      const int m = m0 + wm + i * 16 + (lane & 15);
      if (m >= p.outputs) continue;
      if (sums) {
        float b = bias[DW ? i : 0];
        b += __shfl_xor(b, 16);
        b += __shfl_xor(b, 32);
        if (lane < 16) p.db[leaf * p.outputs + m] = b;
      }
#pragma unroll
      for (int j = 0; j < WN / 16; ++j) {
        const int k = c0 + wn + j * 16 + (lane >> 4) * 4;
        if (k < cols) store4(dw + (int64_t)m * cols + k, acc[i][j], cols - k);
      }
    }
    return;
  }
  const T* const bias_of = MODE == LEAF_PRODUCT_Y && p.b && leaf >= 0 ? (const T*)p.b + leaf * cols : nullptr;
#pragma unroll
  for (int j = 0; j < WN / 16; ++j) {
    const int col = c0 + wn + j * 16 + (lane >> 4) * 4;
    if (col >= cols) continue;
    const f32x4 b = bias4(bias_of, col, cols);
#pragma unroll
    for (int i = 0; i < WM / 16; ++i) {
      const int n = row_of[DW ? 0 : wm + i * 16 + (lane & 15)];
      if (n >= 0) store_row<T>(p, tree, n, col, cols, acc[i][j] + b);
    }
  }
}

template <typename T>
void launch(const LeafProduct& p, int what, hipStream_t s) {
  const int cols = what == LEAF_PRODUCT_Y ? p.outputs : p.inputs, ct = (cols + BN - 1) / BN;
  const dim3 grid((unsigned)leaf_big_blocks(p, what), what == LEAF_PRODUCT_DW ? 1u : (unsigned)p.g.trees);
  if (what == LEAF_PRODUCT_Y)
    k_leaf_big<T, LEAF_PRODUCT_Y><<<grid, THREADS, 0, s>>>(p, ct);
  else if (what == LEAF_PRODUCT_DX)
    k_leaf_big<T, LEAF_PRODUCT_DX><<<grid, THREADS, 0, s>>>(p, ct);
  else
    k_leaf_big<T, LEAF_PRODUCT_DW><<<grid, THREADS, 0, s>>>(p, ct);
}

}  // namespace

int64_t leaf_big_blocks(const LeafProduct& p, int what) {
  const int64_t ct = ((what == LEAF_PRODUCT_Y ? p.outputs : p.inputs) + BN - 1) / BN;
  if (what == LEAF_PRODUCT_DW) return (p.outputs + BM - 1) / BM * ct * p.g.trees * p.g.leaves;
  return (row_tiles(p.g, BM) * ct + 7) / 8 * 8;
}

// Rows and maps that make whole tiles of 256 x 256 worthwhile, and 16-byte chunks that do not
// cross a row's end.
bool leaf_big_fits(const LeafProduct& p, int what) {
  if (p.dtype == LGBM_HIP_DTYPE_F32) return false;
  if (p.inputs % 8 || p.outputs % 8 || p.inputs < 192 || p.outputs < 192) return false;
  if ((int64_t)p.g.rows < 192 * (int64_t)p.g.leaves) return false;
  auto ok = [](const void* q, int64_t ld) { return (((uintptr_t)q) | (uintptr_t)(ld * 2)) % 16 == 0; };
  if (what == LEAF_PRODUCT_Y) return ok(p.x, p.ldx) && ok(p.w, p.inputs);
  if (what == LEAF_PRODUCT_DX) return ok(p.dy, p.lddy) && ok(p.w, p.inputs);
  return ok(p.x, p.ldx) && ok(p.dy, p.lddy);
}

void launch_leaf_big(const LeafProduct& p, int what, hipStream_t s) {
  if (p.dtype == LGBM_HIP_DTYPE_BF16)
    launch<__bf16>(p, what, s);
  else
    launch<_Float16>(p, what, s);
}

}  // namespace lgbm
