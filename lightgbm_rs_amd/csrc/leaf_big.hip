// leaf_big.hip — the leaves' linear maps in 16 bits where leaves hold hundreds of rows and
// wide maps: bound by the matrix cores.
//
// A block of four waves makes 256 x 256 of a result, a wave 128 x 128 of it in registers (a
// smaller wave tile reads LDS for as long as it multiplies).  64 elements of the
// contraction a stage pass through LDS, in two buffers: 128 bytes of a row, since the
// caches fetch no less (32 elements a stage: 64 KB from L2 take 1.2 us a CU instead of
// 0.8).  A further stage is on its way in registers (two gain nothing and spill), which the
// accumulators in the other half of the register file leave free.  Every lane gives its own
// address, so the gather through the order costs nothing, and what is beyond an operand
// reads zeros.
//
// Measured in bfloat16, 4096 rows to 4096 outputs (a tile a CU): 43 us for 1024 inputs, 67
// for 2048, 218 for 8192 (1262 TFLOP/s; a library product 1646): 1.57 us a stage, of which
// the matrix instructions are 0.85 at full clock, LDS 0.64, and 19 us around them.  40007
// ragged rows of 2000 in 31 leaves to 2048: 417 us, 787 TFLOP/s, six rounds of tiles of which
// the last is 0.4 full and the leaves' ends leave a tenth empty.
#include <algorithm>

#include "leaf_mma.h"

namespace lgbm {
namespace {

using namespace mma;

constexpr int THREADS = 256, BM = 256, BN = 256, BK = 64, WM = 128, WN = 128;
constexpr int A_BYTES = BM * BK * 2, STAGE = (BM + BN) * BK * 2;
constexpr int LOADS = 8;  // of 1 KB a wave, operand and stage

__device__ __align__(16) unsigned int zeros[BN / 2];  // what a row that is not there reads

typedef const __attribute__((address_space(1))) u32x4* global_vec;
typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));

// The wave's LDS accesses are done, then the block's.
__device__ __forceinline__ void turn() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// 32 x 32 of a result, 16 of the contraction: a lane's fragment is 16 bytes of row lane % 32,
// chunk lane / 32 of two.  Lane l of the result holds column l % 32 (of the second operand)
// and in element 4 a + b row 8 a + 4 (l / 32) + b (of the first).
template <typename T>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c,
                                                  0, 0, 0);
}

// Stages in LDS.  Along the contraction: [256 rows][8 chunks of 16 bytes], the chunks
// swizzled so that the eight rows that are read together lie in different banks.
__device__ __forceinline__ u32x4 kc_frag32(const char* tile, int base, int step, int lane) {
  const int row = base + (lane & 31);
  return *reinterpret_cast<const u32x4*>(tile + row * 128 + (((step * 2 + (lane >> 5)) ^ (row & 7)) << 4));
}
// Contraction-major: [64][256 columns], in units of 16 columns (32 bytes), pairs of units
// swizzled.  Transposing reads: within 16 lanes, lane l gives four columns of row l / 4 and
// gets column l of the four rows.
__device__ __forceinline__ int cm_swizzle32(int row) { return ((row & 3) | ((row >> 1) & 4)) << 1; }
__device__ __forceinline__ u32x4 cm_frag32(const char* tile, int base, int step, int lane) {
  typedef __attribute__((address_space(3))) s16x4* tr_ptr;
  const int g = lane >> 4, l = lane & 15, col = base + (g & 1) * 16 + (l & 3) * 4;
  s16x4 v[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = step * 16 + (g >> 1) * 8 + h * 4 + (l >> 2);
    const int at = row * 512 + (((col >> 4) ^ cm_swizzle32(row)) << 5) + (col & 15) * 2;
    v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr) const_cast<char*>(tile + at));
  }
  u32x4 out;
  __builtin_memcpy(&out, v, 16);
  return out;
}

// The part of the gradients that is the `rank`-th by rows, in a forest of at most THREADS
// leaves: whole parts first, then the leaves' ends by their length.  So the long blocks begin
// first, and the short ones fill the end (both gradients of two trees of 15 leaves, 16389 rows
// of 2048 to 2048: 885 us in their order, 840).
__device__ __forceinline__ DwPart part_of_rank(const LeafProduct& p, const Split& split, int rank) {
  __shared__ int fulls[THREADS], ends[THREADS];
  __shared__ int found[3];  // leaf of the forest, -1: none; first row, rows
  const int tid = threadIdx.x, leaves = p.g.trees * p.g.leaves;
  const int count = tid < leaves ? min(max(p.g.count[tid], 0), p.g.rows) : 0;
  const int full = split.rows ? count / split.rows : 0, end = count - full * split.rows;
  fulls[tid] = full, ends[tid] = end;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  int longer = 0, before = 0, all = 0;
#pragma unroll 8
  for (int l = 0; l < leaves; ++l) {
    const int f = fulls[l], e = ends[l];
    longer += e > end || (e == end && l < tid);
    all += f;
    before += l < tid ? f : 0;
  }
  // a leaf without rows is a part: its zeros
  const bool in_full = rank >= before && rank < before + full;
  if (tid < leaves && (in_full || (rank == all + longer && (end > 0 || count == 0)))) {
    const int skip = in_full ? rank - before : full;
    found[0] = tid;
    found[1] = min(max(p.g.begin[tid], 0), p.g.rows - count) + skip * split.rows;
    found[2] = in_full ? split.rows : end;
  }
  __syncthreads();
  const int at = __builtin_amdgcn_readfirstlane(found[0]);
  if (at < 0) return {0, 0, -1, nullptr, nullptr};
  return dw_part_of(p, split, at / p.g.leaves, at % p.g.leaves, __builtin_amdgcn_readfirstlane(found[1]),
                    __builtin_amdgcn_readfirstlane(found[2]));
}

// MODE LEAF_PRODUCT_Y: a = x rows [k], b = w[leaf] [col][k]; _DX: a = dy rows [m], b = w[leaf]
// [m][col]; _DW: a = dy [row][m], b = x [row][k] over a leaf's rows.  Y and DX: one block a
// CU takes tile after tile, so that what it stores drains while the next tile begins; DW:
// a block a tile of a part, since leaves differ in length.
template <typename T, int MODE>
__global__ __launch_bounds__(THREADS, 1) void k_leaf_big(LeafProduct p, int col_tiles, Split split) {
  constexpr bool DW = MODE == LEAF_PRODUCT_DW, ACM = DW, BCM = MODE != LEAF_PRODUCT_Y;
  constexpr int FM = WM / 32, FN = WN / 32, STEPS = BK / 16, ITEMS = STEPS * FM, RING = 4;
  constexpr int TURN = ITEMS - 2;
  __shared__ __align__(1024) char lds[2][STAGE];
  __shared__ int32_t row_of[DW ? 1 : BM];
  __shared__ __align__(16) uint64_t rows_at[DW ? THREADS / 64 : 1][DW ? 16 : 1][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave >> 1) * WM, wn = (wave & 1) * WN;
  const int tree_y = blockIdx.y;
  // neighbouring tiles to one XCD, which shares their rows and maps in its L2
  int tiles = 0, share = 0;
  if (!DW) {
    tiles = count_tiles<THREADS>(p.g, tree_y, BM) * col_tiles;
    share = (tiles + 7) / 8;
  }

  for (int slot = blockIdx.x >> 3;; slot += gridDim.x >> 3) {
    // the block's part of the result, and the length of the contraction
    int tree = tree_y, first = 0, length, m0 = 0, c0, cols;
    int64_t leaf;
    DwPart part{};
    if (DW) {
      const int of = (p.outputs + BM - 1) / BM * col_tiles, tile = (int)(blockIdx.x % of);
      const int id = (int)(blockIdx.x / of);
      part = leaf_big_ranks(p.g)
                 ? part_of_rank(p, split, (int)(blockIdx.y * split.parts) + id)
                 : dw_part<THREADS>(p, split, id);
      if (part.count < 0) return;
      tree = part.tree, first = part.first, length = part.count;
      leaf = 0;
      m0 = tile / col_tiles * BM, c0 = tile % col_tiles * BN, cols = p.inputs;
    } else {
      length = MODE == LEAF_PRODUCT_Y ? p.inputs : p.outputs;
      cols = MODE == LEAF_PRODUCT_Y ? p.outputs : p.inputs;
      const int id = (int)(blockIdx.x & 7) * share + slot;
      if (slot >= share || id >= tiles) return;
      const RowTile rt = find_tile<THREADS>(p.g, tree, id / col_tiles, BM);
      c0 = id % col_tiles * BN;
      if (rt.rows == 0) return;
      leaf = rt.leaf < 0 ? -1 : (int64_t)tree * p.g.leaves + rt.leaf;
      row_of[tid] = tid < rt.rows ? row_at(p.g, tree, rt.first + tid) : -1;
      __syncthreads();
      if (leaf < 0) length = 0;
    }
    const T* const w = (const T*)p.w + (DW || leaf < 0 ? 0 : leaf * p.outputs * (int64_t)p.inputs);

    // A lane's addresses.  Along the contraction: row 8 (8 wave + j) + lane / 8, chunk lane %
    // 8 (swizzled); contraction-major: row 2 (8 wave + j) + lane / 32, 16 bytes lane % 32
    // (swizzled).
    const int kc_row = wave * 64 + (lane >> 3), cm_row = wave * 16 + (lane >> 5);
    const int achunk = ((lane & 7) ^ (kc_row & 7)) * 8;
    // Offsets are in 16 bytes, which rows are whole ones of: 32 bits reach 64 GB.
    uint32_t aoff[LOADS], boff[LOADS];
    int cm_col[LOADS];
    const uint32_t ld16 = (uint32_t)((MODE == LEAF_PRODUCT_Y ? p.ldx : p.lddy) / 8);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int unit = ((lane & 31) >> 1) ^ cm_swizzle32(cm_row + 2 * j);
      cm_col[j] = (unit * 2 + (lane & 1)) * 8;
      if (!ACM) aoff[j] = (uint32_t)max(row_of[DW ? 0 : kc_row + 8 * j], 0) * ld16 + achunk / 8;
      if (MODE == LEAF_PRODUCT_Y)
        boff[j] = (uint32_t)min(c0 + kc_row + 8 * j, cols - 1) * (uint32_t)(length / 8) + achunk / 8;
      if (MODE == LEAF_PRODUCT_DX) boff[j] = (uint32_t)(cm_row + 2 * j) * (uint32_t)(cols / 8) + (c0 + cm_col[j]) / 8;
    }
    // DW: where the 16 rows of a wave's loads begin, in dy and in x at the block's columns.
    // Lanes 0 to 15 and 32 to 47 make dy's, the others x's; a load's half waves take theirs
    // from LDS, and every lane adds its column.  Columns behind the last only make results
    // that are not stored, so they read the last ones.
    const int half = lane >> 5, op = (lane >> 4) & 1;
    const T* const base = op ? (const T*)p.x + c0 : (const T*)p.dy + m0;
    const uint32_t ld_of_op = (uint32_t)(op ? p.ldx : p.lddy) * 2;
    const uint32_t a_col = (uint32_t)(min(m0 + (lane & 31) * 8, p.outputs - 8) - m0) * 2;
    const uint32_t b_col = (uint32_t)(min(c0 + (lane & 31) * 8, cols - 8) - c0) * 2;
    auto order_of = [&](int k0) {
      return p.g.order[(int64_t)tree * p.g.rows + min(first + k0 + wave * 16 + (lane & 15), p.g.rows - 1)];
    };
    auto put_rows = [&](int n, int k0) {
      const bool there = k0 + wave * 16 + (lane & 15) < length && (uint32_t)n < (uint32_t)p.g.rows;
      const uint64_t at = (uint64_t)(uintptr_t)base + (uint64_t)(uint32_t)n * ld_of_op;
      rows_at[DW ? wave : 0][DW ? lane & 15 : 0][op] = there ? at : (uint64_t)(uintptr_t)zeros;
    };
    auto get_rows = [&](int j) { return *(const u64x2*)rows_at[DW ? wave : 0][DW ? 2 * j + half : 0]; };
    u64x2 at_row[2];
    // The j-th loads of the stage at k0, and their place in its buffer.  The stage's addresses
    // are scalars that the compiler takes as new ones, or it would keep a lane's 32 in
    // registers.
    const T* const src = (const T*)(MODE == LEAF_PRODUCT_Y ? p.x : p.dy);
    const uint64_t zero_at = (uint64_t)(uintptr_t)zeros;
    struct Stage {
      uint64_t a, b;
    };
    auto stage_at = [&](int k0) {
      if (DW) return Stage{(uint64_t)(uintptr_t)p.dy, (uint64_t)(uintptr_t)p.x};
      Stage g{(uint64_t)(uintptr_t)(src + k0),
              (uint64_t)(uintptr_t)(w + (MODE == LEAF_PRODUCT_Y ? (int64_t)k0 : (int64_t)k0 * cols))};
      asm("" : "+s"(g.a), "+s"(g.b));
      return g;
    };
    auto load_a = [&](const Stage& g, int k0, int j) {
      uint64_t from;
      bool in;
      if (DW) return *(global_vec)(at_row[j & 1].x + a_col);
      in = k0 + achunk < length;
      from = g.a + (uint64_t)aoff[j] * 16;
      return *(global_vec)(in ? from : zero_at);
    };
    auto load_b = [&](const Stage& g, int k0, int j) {
      uint64_t from;
      bool in;
      if (DW) return *(global_vec)(at_row[j & 1].y + b_col);
      in = BCM ? k0 + cm_row + 2 * j < length && c0 + cm_col[j] < cols : k0 + achunk < length;
      from = g.b + (uint64_t)boff[j] * 16;
      return *(global_vec)(in ? from : zero_at);
    };
    // (DW: the column's unit swizzled by bits 0, 1 and 3 of the row, 16 wave + 2 j + half)
    const int lane_at = DW ? half * 512 + (((lane & 31) * 16) ^ (half << 6)) : lane * 16;
    auto place = [&](char* buf, int j) {
      return (u32x4*)(buf + (wave * LOADS + j) * 1024 + (DW ? lane_at ^ ((j & 1) << 7 | (j >> 2) << 8) : lane_at));
    };

    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    float bias[DW ? FM : 1];  // of the lane's chunks
#pragma unroll
    for (int i = 0; i < (DW ? FM : 1); ++i) bias[i] = 0.0f;

    // item: step FM + i of a stage
    auto frag_a = [&](const char* buf, int item) {
      const int base = wm + 32 * (item % FM), step = item / FM;
      return ACM ? cm_frag32(buf, base, step, lane) : kc_frag32(buf, base, step, lane);
    };
    auto frag_b = [&](const char* buf, int j, int step) {
      return BCM ? cm_frag32(buf + A_BYTES, wn + 32 * j, step, lane)
                 : kc_frag32(buf + A_BYTES, wn + 32 * j, step, lane);
    };
    u32x4 fa[RING], fb[2][FN], ahead[2 * LOADS];
    int next_rows = 0;  // DW: what put_rows takes next
    // sums of dy's columns cost as much again as what else the matrix instructions hide: only
    // the blocks of the first columns make them
    const bool sums = DW && part.db && c0 == 0;
    // A stage is 16 items: a fragment of rows times the four of columns, for each 16 of the
    // stage's contraction.  Fragments of rows are read three items ahead, the columns' four.
    // During items 0 to 11 the next stage goes from registers to the other buffer, and the
    // registers are loaded with the stage behind it.  Behind item 13 the wave has read all of
    // its buffer: the block turns and the first fragments of the next stage are read.
    const auto share_of = [](int t) constexpr {  // the eight shares, over items 0 to 11
      for (int j = 0; j < LOADS; ++j)
        if (j * 13 / 8 == t) return j;
      return -1;
    };
    auto stage = [&](int k0, char* cur, char* next) {
      const Stage from = stage_at(k0 + 2 * BK);
#pragma unroll
      for (int t = 0; t < ITEMS; ++t) {
        const int i = t % FM, step = t / FM;
        if (t == TURN) {
          turn();
#pragma unroll
          for (int j = 0; j < FN; ++j) fb[0][j] = frag_b(next, j, 0);
        }
        if (t < TURN - 1)
          fa[(t + RING - 1) % RING] = frag_a(cur, t + RING - 1);
        else if (t >= TURN)
          for (int u = t == TURN ? 0 : 2; u < (t == TURN ? 2 : 3); ++u) fa[u] = frag_a(next, u);
        if (step + 1 < STEPS) fb[(step + 1) % 2][i] = frag_b(cur, i, step + 1);
        const u32x4 f = fa[t % RING];
        if (DW && sums) {
          T e[8];
          __builtin_memcpy(e, &f, 16);
          bias[DW ? i : 0] += (((float)e[0] + (float)e[1]) + ((float)e[2] + (float)e[3])) +
                              (((float)e[4] + (float)e[5]) + ((float)e[6] + (float)e[7]));
        }
        if (share_of(t) >= 0) {
          const int l = share_of(t);
          *place(next, l) = ahead[2 * l];
          *place(next + A_BYTES, l) = ahead[2 * l + 1];
          ahead[2 * l] = load_a(from, k0 + 2 * BK, l);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < FN / 2; ++j) acc[i][j] = mfma32<T>(f, fb[step % 2][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
        if (t > 0 && share_of(t - 1) >= 0) {
          const int l = share_of(t - 1);
          ahead[2 * l + 1] = load_b(from, k0 + 2 * BK, l);
          if (DW && l + 2 < LOADS) at_row[l & 1] = get_rows(l + 2);
        }
#pragma unroll
        for (int j = FN / 2; j < FN; ++j) acc[i][j] = mfma32<T>(f, fb[step % 2][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
        if (t == TURN && DW) {
          put_rows(next_rows, k0 + 3 * BK);
          next_rows = order_of(k0 + 4 * BK);
          at_row[0] = get_rows(0), at_row[1] = get_rows(1);
        }
      }
    };

    if (length > 0) {
      // stage 0 to the first buffer, then stage 1 on its way, loaded in the order of a stage:
      // the compiler's waits in the loop count the loads that are younger on every way to it
      int order[3];
      if (DW) {
#pragma unroll
        for (int i = 0; i < 3; ++i) order[i] = order_of(i * BK);
        next_rows = order_of(3 * BK);
        put_rows(order[0], 0);
      }
      const Stage first_stage = stage_at(0), second = stage_at(BK);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        if (DW) at_row[j & 1] = get_rows(j);
        ahead[2 * j] = load_a(first_stage, 0, j);
        ahead[2 * j + 1] = load_b(first_stage, 0, j);
      }
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        *place(lds[0], j) = ahead[2 * j], *place(lds[0] + A_BYTES, j) = ahead[2 * j + 1];
      if (DW) {
        put_rows(order[1], BK);
        at_row[0] = get_rows(0), at_row[1] = get_rows(1);
      }
#pragma unroll
      for (int t = 0; t < ITEMS; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        if (share_of(t) >= 0) ahead[2 * share_of(t)] = load_a(second, BK, share_of(t));
        __builtin_amdgcn_sched_barrier(0);
        if (t > 0 && share_of(t - 1) >= 0) {
          const int l = share_of(t - 1);
          ahead[2 * l + 1] = load_b(second, BK, l);
          if (DW && l + 2 < LOADS) at_row[l & 1] = get_rows(l + 2);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (DW) {
        put_rows(order[2], 2 * BK);
        at_row[0] = get_rows(0), at_row[1] = get_rows(1);
      }
      turn();
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[0][j] = frag_b(lds[0], j, 0);
#pragma unroll
      for (int u = 0; u < RING - 1; ++u) fa[u] = frag_a(lds[0], u);
      int cur = 0;
      for (int k0 = 0; k0 < length; k0 += BK, cur ^= 1) stage(k0, lds[cur], lds[cur ^ 1]);
    }

    // A lane has column lane % 32 of each 32 x 32, so that a store's lanes fill 64 or 128 bytes
    // of a row (by 16 bytes of 64 rows, gradients of maps of 4096 x 4096 over 512 rows took 66
    // us instead of 32).
    const int col0 = c0 + wn + (lane & 31), row4 = (lane >> 5) * 4;
    if (DW) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int mi = m0 + wm + i * 32;
        if (sums && wn == 0) {
          const float b = bias[DW ? i : 0] + __shfl_xor(bias[DW ? i : 0], 32);
          if (lane < 32 && mi + lane < p.outputs) part.db[mi + lane] = b;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int m = mi + (e >> 2) * 8 + row4 + (e & 3);
          if (m >= p.outputs) continue;
#pragma unroll
          for (int j = 0; j < FN; ++j)
            if (col0 + j * 32 < cols) part.dw[(int64_t)m * cols + col0 + j * 32] = acc[i][j][e];
        }
      }
      return;
    }
    float b[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const bool has = MODE == LEAF_PRODUCT_Y && p.b && leaf >= 0 && col0 + j * 32 < cols;
      b[j] = has ? (float)((const T*)p.b)[leaf * cols + col0 + j * 32] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const int r = wm + i * 32 + (e >> 2) * 8 + row4 + (e & 3);
        const int n[2] = {row_of[DW ? 0 : r], row_of[DW ? 0 : r + 1]};
        if (p.planes) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (n[k] < 0) continue;
            float* const to = (float*)p.ws + ((int64_t)tree * p.g.rows + n[k]) * cols + col0;
#pragma unroll
            for (int j = 0; j < FN; ++j)
              if (col0 + j * 32 < cols) to[j * 32] = acc[i][j][e + k] + b[j];
          }
        } else {
          const int row = n[lane & 1];
          T* const to = (T*)p.out + (int64_t)max(row, 0) * p.ldo + (col0 & ~1);
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            const uint32_t v = pair_of<T>(acc[i][j][e] + b[j], acc[i][j][e + 1] + b[j]);
            if (row >= 0 && col0 + j * 32 < cols) __builtin_memcpy(to + j * 32, &v, 4);
          }
        }
      }
    __syncthreads();  // row_of is read before the next tile's
  }
}

template <typename T>
void launch(const LeafProduct& p, int what, hipStream_t s) {
  const int cols = what == LEAF_PRODUCT_Y ? p.outputs : p.inputs, ct = (cols + BN - 1) / BN;
  const Split split = what == LEAF_PRODUCT_DW ? leaf_big_split(p) : Split{0, 0, 0};
  const dim3 grid((unsigned)leaf_big_blocks(p, what),
                  what == LEAF_PRODUCT_DW && split.rows == 0 ? 1u : (unsigned)p.g.trees);
  if (what == LEAF_PRODUCT_Y)
    k_leaf_big<T, LEAF_PRODUCT_Y><<<grid, THREADS, 0, s>>>(p, ct, split);
  else if (what == LEAF_PRODUCT_DX)
    k_leaf_big<T, LEAF_PRODUCT_DX><<<grid, THREADS, 0, s>>>(p, ct, split);
  else
    k_leaf_big<T, LEAF_PRODUCT_DW><<<grid, THREADS, 0, s>>>(p, ct, split);
}

}  // namespace

// Rows a block of the maps' gradients sums at most: a 256th of the work, a part for every CU
// (bfloat16, ragged leaves, by parts of 8192 rows and by these: 100000 x 256 to 512 by 63 leaves 297
// and 104 us, 40000 x 512 to 512 by 31 295 and 90, 1M x 256 to 256 by two 320 and 223; by parts
// of a 512th the last takes 271, and 16389 x 2048 to 2048 by two trees of 15, whose long leaves
// are then in parts, 530 instead of 443).
Split leaf_big_split(const LeafProduct& p) {
  const int64_t tiles = (int64_t)((p.outputs + BM - 1) / BM) * ((p.inputs + BN - 1) / BN);
  const int64_t share = (p.g.rows * (int64_t)p.g.trees * tiles / 256 + BK - 1) / BK * BK;
  const int64_t rows = std::min<int64_t>(std::max<int64_t>(share, 512), CHAIN_ROWS);
  return split_by(p.g, rows);
}

int64_t leaf_big_blocks(const LeafProduct& p, int what) {
  const int64_t ct = ((what == LEAF_PRODUCT_Y ? p.outputs : p.inputs) + BN - 1) / BN;
  if (what == LEAF_PRODUCT_DW) {
    const Split split = leaf_big_split(p);
    return (p.outputs + BM - 1) / BM * ct * (split.rows ? split.parts : (int64_t)p.g.trees * p.g.leaves);
  }
  return std::min<int64_t>((row_tiles(p.g, BM) * ct + 7) / 8 * 8, 256);  // one a CU
}

// Rows and maps that make whole tiles of 256 x 256 worthwhile, and 16-byte chunks that do not
// cross a row's end.  The counts of the leaves are on the device, so the rule takes their
// average; tables of many small leaves and a few long ones still gain or break even (bfloat16,
// these tiles and the other kernels, us: 100000 x 512 to 512 by 500 leaves alike y 141, 202, dx 156,
// 206, dw 218, 371; with sizes as exp(3 N(0, 1)) 168, 192, 183, 188, 484, 510; 40000 x 2048 to 2048
// by 200 leaves of sizes as exp(N(0, 1)) 677, 781, 699, 696, 1512, 1967).
//
// y and dx also need tiles for the CUs, about 72 with half a tile for every leaf's end (bfloat16 by
// these tiles and by k_leaf_tile's, us):
//   tiles            y           dx
//     2..5   400 x 4096 to 200 by two leaves 92, 38; 400 x 200 to 4096 103, 43
//    39..41  1000 x 2048 to 2048 by two 57, 42 and 64, 41; 400 x 4096 to 4096 by two 96, 61 and 107, 59
//    63..66  16000 x 4096 to 200 by one 98, 80; 2000 x 2048 to 2048 by one 58, 45 and 66, 43
//    76..78  4000 x 1024 to 1024 by seven 38, 43 and 43, 42; 16000 x 4096 to 200 by 31 100, 127
//   127..139 8000 x 1024 to 1024 by one 41, 44 and 45, 42, by seven 41, 64 and 46, 60
bool leaf_big_fits(const LeafProduct& p, int what) {
  if (p.dtype == LGBM_HIP_DTYPE_F32) return false;
  if (p.inputs % 8 || p.outputs % 8 || p.inputs < 192 || p.outputs < 192) return false;
  if ((int64_t)p.g.rows < 192 * (int64_t)p.g.leaves) return false;
  const int64_t ct = ((what == LEAF_PRODUCT_Y ? p.outputs : p.inputs) + BN - 1) / BN;
  if (what != LEAF_PRODUCT_DW && (2 * (int64_t)p.g.rows / BM + p.g.leaves) * ct * p.g.trees < 2 * 72) return false;
  if (p.g.rows * std::max(p.ldx, p.lddy) >> 35 || (int64_t)p.inputs * p.outputs >> 35) return false;  // 64 GB
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
