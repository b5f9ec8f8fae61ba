// leaf_groups.hip — the rows of every leaf from the leaf of every row: a stable counting
// sort of each tree's column of leaf indices.
//
// Few rows: a block a tree does it in one launch (k_group_few).  Else the rows go in chunks,
// about eight for every CU: the leaves of every chunk are counted (k_count_leaves), each
// leaf's counts summed over the chunks before (k_sum_chunks), and the rows put in their
// places (k_order_rows), a tile of rows at a time.  Within a wave's 64 rows, the ballots
// of a leaf's bits give every row the lanes that share its leaf, and so its rank; a wave's
// counters rank it among the wave's rows, their sums among the tile's.  Nothing is decided
// by the order of atomics, so the order is stable and always the same.
//
// 4 bytes a row and tree are read twice and written once, but what bounds a large table is the
// ranking: eight ballots a wave of rows and a chain of LDS counters (10.5M rows, 255
// leaves: k_order_rows 57 us where its bytes take 17; tiles of 4096 rows 68 us).
#include <algorithm>

#include "leaf_ops.h"

namespace lgbm {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int ITEMS = 8;                 // rows a lane in a tile
constexpr int TILE = THREADS * ITEMS;    // rows a tile
constexpr int TARGET_CHUNKS = 2048;      // eight for every CU

// Rows a chunk: whole tiles.
int64_t chunk_rows(int64_t rows) {
  const int64_t tiles = (rows + TILE - 1) / TILE;
  return std::max<int64_t>((tiles + TARGET_CHUNKS - 1) / TARGET_CHUNKS, 1) * TILE;
}
int64_t num_chunks(int64_t rows) { return (rows + chunk_rows(rows) - 1) / chunk_rows(rows); }

// The chunk of a block: neighbours go to one XCD (blocks go to the eight in turn), where they
// share the cache lines of their counts and of the ends of the leaves' runs in the order.
__device__ __forceinline__ int chunk_of_block() {
  return (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
}

// The leaf of row n, `leaves` where it is in none.
__device__ __forceinline__ int leaf_of(const int32_t* leaf, int64_t ld, int64_t n, int tree, int leaves) {
  const int l = leaf[n * ld + tree];
  return l >= 0 && l < leaves ? l : leaves;
}

// The sum of a block's values before this thread's, and of all; sums: a word a wave.
__device__ __forceinline__ int block_scan(int v, int* sums, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(incl, d);
    if (lane >= d) incl += up;
  }
  __syncthreads();
  if (lane == 63) sums[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  return before + incl - v;
}

// The rows [n0, n1), at most a tile, put behind place[leaf] (which moves on): wave w takes
// the w-th quarter of a tile.  counters: [WAVES][leaves + 1].
__device__ __forceinline__ void order_tile(const int32_t* leaf, int64_t ld, int64_t n0, int64_t n1, int tree,
                                           int leaves, int bits, int32_t* counters, int32_t* place,
                                           int32_t* order) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, width = leaves + 1;
  const int64_t w0 = n0 + (int64_t)wave * (ITEMS * 64) + lane;
  int l[ITEMS], rank[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int64_t n = w0 + i * 64;
    l[i] = n < n1 ? leaf_of(leaf, ld, n, tree, leaves) : -1;
  }
  for (int i = tid; i < WAVES * width; i += THREADS) counters[i] = 0;
  __syncthreads();
  int32_t* const mine = counters + wave * width;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const uint64_t here = __ballot(l[i] >= 0);
    uint32_t lo = (uint32_t)here, hi = (uint32_t)(here >> 32);
    for (int b = 0; b < bits; ++b) {
      const uint32_t mine_set = (uint32_t)((l[i] << (31 - b)) >> 31);  // all ones or none
      const uint64_t with = __ballot(mine_set != 0);
      lo &= ~((uint32_t)with ^ mine_set);
      hi &= ~((uint32_t)(with >> 32) ^ mine_set);
    }
    if (l[i] >= 0) {
      const uint64_t same = (uint64_t)hi << 32 | lo;
      const int before = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
      rank[i] = mine[l[i]] + before;
      __builtin_amdgcn_wave_barrier();
      if ((same >> lane) == 1ull) mine[l[i]] = rank[i] + 1;  // the last of them
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  for (int i = tid; i < width; i += THREADS) {
    int32_t at = place[i];
    for (int w = 0; w < WAVES; ++w) {
      const int32_t c = counters[w * width + i];
      counters[w * width + i] = at;
      at += c;
    }
    place[i] = at;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (l[i] >= 0) order[mine[l[i]] + rank[i]] = (int32_t)(w0 + i * 64);
  __syncthreads();
}

// The leaves of rows [n0, n1) counted in LDS.
__device__ __forceinline__ void count_rows(const int32_t* leaf, int64_t ld, int64_t n0, int64_t n1, int tree,
                                           int leaves, int32_t* count) {
  for (int l = threadIdx.x; l <= leaves; l += THREADS) count[l] = 0;
  __syncthreads();
#pragma unroll 8
  for (int64_t n = n0 + threadIdx.x; n < n1; n += THREADS)
    atomicAdd(&count[leaf_of(leaf, ld, n, tree, leaves)], 1);
  __syncthreads();
}

// A tree's leaf totals to begin and count; place[l]: where leaf l starts.  total(l): of leaf
// l <= leaves.
template <typename F>
__device__ __forceinline__ void place_leaves(int leaves, int32_t* place, int32_t* begin, int32_t* count,
                                             int* sums, F total) {
  int base = 0;
  for (int l0 = 0; l0 <= leaves; l0 += THREADS) {
    const int l = l0 + (int)threadIdx.x, c = l <= leaves ? total(l) : 0;
    int all;
    const int at = base + block_scan(c, sums, all);
    base += all;
    if (l <= leaves) place[l] = at;
    if (l < leaves && begin) begin[l] = at, count[l] = c;
  }
  __syncthreads();
}

// LDS: [WAVES + 1][leaves + 1]
__global__ __launch_bounds__(THREADS) void k_group_few(const int32_t* leaf, int64_t ld, int64_t rows, int leaves,
                                                       int bits, int32_t* order, int32_t* begin, int32_t* count) {
  extern __shared__ int32_t lds[];
  __shared__ int sums[WAVES];
  const int tree = blockIdx.x, width = leaves + 1;
  int32_t* const place = lds + WAVES * width;
  count_rows(leaf, ld, 0, rows, tree, leaves, lds);
  place_leaves(leaves, place, begin + (int64_t)tree * leaves, count + (int64_t)tree * leaves, sums,
               [&](int l) { return lds[l]; });
  for (int64_t n0 = 0; n0 < rows; n0 += TILE)
    order_tile(leaf, ld, n0, min(n0 + TILE, rows), tree, leaves, bits, lds, place, order + (int64_t)tree * rows);
}

// counts[tree][leaf][chunk], leaves + 1 leaves: the last one for rows in no leaf
__global__ __launch_bounds__(THREADS) void k_count_leaves(const int32_t* leaf, int64_t ld, int64_t rows,
                                                          int64_t chunk, int leaves, int chunks, int32_t* counts) {
  extern __shared__ int32_t lds[];
  const int tree = blockIdx.y, at = chunk_of_block();
  if (at >= chunks) return;
  const int64_t n0 = at * chunk;
  count_rows(leaf, ld, n0, min(n0 + chunk, rows), tree, leaves, lds);
  for (int l = threadIdx.x; l <= leaves; l += THREADS)
    counts[((int64_t)tree * (leaves + 1) + l) * chunks + at] = lds[l];
}

// A block a leaf: counts become the sums over the chunks before, the total goes to totals.
__global__ __launch_bounds__(THREADS) void k_sum_chunks(int chunks, int32_t* counts, int32_t* totals) {
  __shared__ int sums[WAVES];
  const int64_t list = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;  // a tree's leaf
  int32_t* const c = counts + list * chunks;
  int32_t base = 0;
  for (int i0 = 0; i0 < chunks; i0 += THREADS) {
    const int i = i0 + (int)threadIdx.x;
    int all;
    const int32_t v = i < chunks ? c[i] : 0, before = block_scan(v, sums, all);
    if (i < chunks) c[i] = base + before;
    base += all;
  }
  if (threadIdx.x == 0) totals[list] = base;
}

// LDS: [WAVES + 1][leaves + 1]
__global__ __launch_bounds__(THREADS) void k_order_rows(const int32_t* leaf, int64_t ld, int64_t rows,
                                                        int64_t chunk, int leaves, int bits, int chunks,
                                                        const int32_t* counts, const int32_t* totals,
                                                        int32_t* order, int32_t* begin, int32_t* count) {
  extern __shared__ int32_t lds[];
  __shared__ int sums[WAVES];
  const int tree = blockIdx.y, width = leaves + 1, at = chunk_of_block();
  if (at >= chunks) return;
  int32_t* const place = lds + WAVES * width;
  const bool first = at == 0;
  place_leaves(leaves, place, first ? begin + (int64_t)tree * leaves : nullptr, count + (int64_t)tree * leaves,
               sums, [&](int l) { return totals[(int64_t)tree * width + l]; });
  for (int l = threadIdx.x; l < width; l += THREADS)
    place[l] += counts[((int64_t)tree * width + l) * chunks + at];
  const int64_t c0 = at * chunk, c1 = min(c0 + chunk, rows);
  for (int64_t n0 = c0; n0 < c1; n0 += TILE)
    order_tile(leaf, ld, n0, min(n0 + TILE, c1), tree, leaves, bits, lds, place, order + (int64_t)tree * rows);
}

// One launch where a tree's rows are at most two tiles.
bool few(int64_t rows) { return rows <= 2 * TILE; }

}  // namespace

size_t leaf_groups_workspace(int64_t rows, int32_t trees, int32_t leaves) {
  if (few(rows)) return 0;
  return (size_t)trees * (size_t)(leaves + 1) * (size_t)(num_chunks(rows) + 1) * 4;
}

void launch_leaf_groups(const int32_t* leaf, int64_t ld, int64_t rows, int32_t trees,
                        int32_t leaves, int32_t* order, int32_t* begin, int32_t* count, void* ws,
                        hipStream_t s) {
  int bits = 1;
  while ((leaves >> bits) != 0) ++bits;
  const size_t row = (size_t)(leaves + 1) * 4, lds = row * (WAVES + 1);
  if (few(rows)) {
    k_group_few<<<trees, THREADS, lds, s>>>(leaf, ld, rows, leaves, bits, order, begin, count);
    return;
  }
  const int chunks = (int)num_chunks(rows);
  const dim3 grid((chunks + 7) / 8 * 8, trees);
  const int64_t chunk = chunk_rows(rows), lists = (int64_t)trees * (leaves + 1);
  int32_t* const counts = (int32_t*)ws;
  int32_t* const totals = counts + lists * chunks;
  k_count_leaves<<<grid, THREADS, row, s>>>(leaf, ld, rows, chunk, leaves, chunks, counts);
  k_sum_chunks<<<dim3(leaves + 1, trees), THREADS, 0, s>>>(chunks, counts, totals);
  k_order_rows<<<grid, THREADS, lds, s>>>(leaf, ld, rows, chunk, leaves, bits, chunks, counts, totals, order, begin,
                                        count);
}

}  // namespace lgbm
