// leaf_groups.hip — the rows of every leaf from the leaf of every row: a stable counting
// sort of each tree's column of leaf indices.
//
// Three passes: the leaves of every chunk of rows counted (k_count_leaves), the counts
// of (leaf, chunk) turned into places (k_place_leaves), the rows put there
// (k_order_rows).  Rows keep their order within a leaf, since a chunk's waves take
// consecutive rows and a wave ranks its 64 rows by the ballots of their leaf's bits.
#include <algorithm>

#include "leaf_ops.h"

namespace lgbm {
namespace {

constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int CHUNK = 4096;  // rows a block

int64_t num_chunks(int64_t rows) { return (rows + CHUNK - 1) / CHUNK; }

// The leaf of row n, `leaves` where it is in none.
__device__ __forceinline__ int leaf_of(const int32_t* leaf, int64_t ld, int64_t n, int tree, int leaves) {
  const int l = leaf[n * ld + tree];
  return l >= 0 && l < leaves ? l : leaves;
}

// counts[tree][leaf][chunk], `leaves` + 1 leaves: the last one for rows in no leaf
__global__ __launch_bounds__(THREADS) void k_count_leaves(const int32_t* leaf, int64_t ld, int64_t rows,
                                                          int leaves, int chunks, int32_t* counts) {
  extern __shared__ int32_t count[];
  const int tree = blockIdx.y;
  for (int l = threadIdx.x; l <= leaves; l += THREADS) count[l] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * CHUNK, n1 = min(n0 + CHUNK, rows);
  for (int64_t n = n0 + threadIdx.x; n < n1; n += THREADS)
    atomicAdd(&count[leaf_of(leaf, ld, n, tree, leaves)], 1);
  __syncthreads();
  for (int l = threadIdx.x; l <= leaves; l += THREADS)
    counts[((int64_t)tree * (leaves + 1) + l) * chunks + blockIdx.x] = count[l];
}

// One block a tree: counts become the place of the chunk's first row of that leaf.
__global__ __launch_bounds__(1024) void k_place_leaves(int leaves, int chunks, int32_t* counts,
                                                       int32_t* begin, int32_t* count) {
  __shared__ int32_t sums[16];
  const int tree = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* const c = counts + (int64_t)tree * (leaves + 1) * chunks;
  const int64_t total = (int64_t)(leaves + 1) * chunks;
  int32_t base = 0;
  for (int64_t i0 = 0; i0 < total; i0 += 1024) {
    const int64_t i = i0 + tid;
    const int32_t v = i < total ? c[i] : 0;
    int32_t incl = v;
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int32_t before = base;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += sums[w];
      base += sums[w];
    }
    if (i < total) c[i] = before + incl - v;
    __syncthreads();
  }
  for (int l = tid; l < leaves; l += 1024) {
    const int32_t at = c[(int64_t)l * chunks], next = c[(int64_t)(l + 1) * chunks];
    begin[(int64_t)tree * leaves + l] = at;
    count[(int64_t)tree * leaves + l] = next - at;
  }
}

__global__ __launch_bounds__(THREADS) void k_order_rows(const int32_t* leaf, int64_t ld, int64_t rows,
                                                        int leaves, int bits, int chunks,
                                                        const int32_t* places, int32_t* order) {
  extern __shared__ int32_t next[];  // [WAVES][leaves + 1]
  const int tree = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int width = leaves + 1;
  for (int i = tid; i < WAVES * width; i += THREADS) next[i] = 0;
  __syncthreads();
  constexpr int PER = CHUNK / WAVES;
  const int64_t n0 = (int64_t)blockIdx.x * CHUNK + wave * PER, n1 = min(n0 + PER, rows);
  int32_t* const mine = next + wave * width;
  for (int64_t n = n0 + lane; n < n1; n += 64) atomicAdd(&mine[leaf_of(leaf, ld, n, tree, leaves)], 1);
  __syncthreads();
  for (int l = tid; l < width; l += THREADS) {
    int32_t at = places[((int64_t)tree * width + l) * chunks + blockIdx.x];
    for (int w = 0; w < WAVES; ++w) {
      const int32_t c = next[w * width + l];
      next[w * width + l] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t i0 = n0; i0 < n1; i0 += 64) {
    const int64_t n = i0 + lane;
    const bool here = n < n1;
    const int l = here ? leaf_of(leaf, ld, n, tree, leaves) : 0;
    uint64_t same = __ballot(here);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((l >> b) & 1);
      same &= ((l >> b) & 1) ? set : ~set;
    }
    if (here) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int32_t at = mine[l] + rank;
      __builtin_amdgcn_wave_barrier();
      if ((same >> lane) == 1ull) mine[l] = at + 1;  // the last of them
      order[(int64_t)tree * rows + at] = (int32_t)n;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace

size_t leaf_groups_workspace(int64_t rows, int32_t trees, int32_t leaves) {
  return (size_t)trees * (size_t)(leaves + 1) * (size_t)std::max<int64_t>(num_chunks(rows), 1) * 4;
}

void launch_leaf_groups(const int32_t* leaf, int64_t ld, int64_t rows, int32_t trees,
                        int32_t leaves, int32_t* order, int32_t* begin, int32_t* count, void* ws,
                        hipStream_t s) {
  const int chunks = (int)std::max<int64_t>(num_chunks(rows), 1);
  int bits = 1;
  while ((leaves >> bits) != 0) ++bits;
  int32_t* const counts = (int32_t*)ws;
  const size_t row = (size_t)(leaves + 1) * 4;
  k_count_leaves<<<dim3(chunks, trees), THREADS, row, s>>>(leaf, ld, rows, leaves, chunks, counts);
  k_place_leaves<<<trees, 1024, 0, s>>>(leaves, chunks, counts, begin, count);
  k_order_rows<<<dim3(chunks, trees), THREADS, row * WAVES, s>>>(leaf, ld, rows, leaves, bits, chunks,
                                                                 counts, order);
}

}  // namespace lgbm
