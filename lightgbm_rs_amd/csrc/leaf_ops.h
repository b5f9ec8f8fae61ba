// leaf_ops.h — the operators around a forest's leaves: rows grouped by leaf, the leaves'
// linear maps and their gradients, dropout and class scores.  Launchers of the kernels in
// leaf_groups.hip, leaf_product.hip, dropout.hip and scores.hip, called by the C entries
// in leaf_capi.hip, which check every argument first.  Nothing here allocates or waits, so
// every launcher can be recorded into a graph.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace lgbm {

// ---- rows by leaf ------------------------------------------------------------------

// order[t][n]: tree t's rows by their leaf; begin / count[t][l]: leaf l's range of it.
struct LeafGroups {
  const int32_t* order;
  const int32_t* begin;
  const int32_t* count;
  int32_t rows, trees, leaves;
};

size_t leaf_groups_workspace(int64_t rows, int32_t trees, int32_t leaves);
void launch_leaf_groups(const int32_t* leaf, int64_t ld, int64_t rows, int32_t trees,
                        int32_t leaves, int32_t* order, int32_t* begin, int32_t* count, void* ws,
                        hipStream_t s);

// ---- the leaves' linear maps ---------------------------------------------------------

// W[trees * leaves][outputs][inputs] and b[trees * leaves][outputs], contiguous; x, y and
// their gradients are [rows][...] with a row stride in elements.  dtype: LGBM_HIP_DTYPE_*.
struct LeafProduct {
  LeafGroups g;
  int32_t inputs, outputs, dtype;
  const void* x;
  int64_t ldx;
  const void* w;
  const void* b;   // product: may be null
  const void* dy;  // gradients
  int64_t lddy;
  void* out;  // product: y [rows][outputs]; dx: [rows][inputs]
  int64_t ldo;
  float* dw;  // [trees * leaves][outputs][inputs]
  float* db;  // [trees * leaves][outputs], may be null
  void* ws;
  // product and dx: whether a tree's results go to its float32 plane [rows][columns] in ws,
  // to be added, instead of to out
  bool planes;
};

#define LEAF_PRODUCT_Y 0
#define LEAF_PRODUCT_DX 1
#define LEAF_PRODUCT_DW 2
size_t leaf_product_workspace(const LeafProduct& p, int what);
int64_t leaf_product_blocks(const LeafProduct& p, int what);  // along x of its largest launch
void launch_leaf_product(const LeafProduct& p, int what, hipStream_t s);
// leaf_big.hip: 16-bit products of large tiles
bool leaf_big_fits(const LeafProduct& p, int what);
int64_t leaf_big_blocks(const LeafProduct& p, int what);
void launch_leaf_big(const LeafProduct& p, int what, hipStream_t s);

// ---- dropout ---------------------------------------------------------------------------

void launch_dropout(const void* x, int64_t ldx, int64_t rows, int64_t cols, int32_t dtype,
                    uint32_t threshold, uint64_t seed, uint64_t offset, int by_row, void* out,
                    int64_t ldo, hipStream_t s);

// ---- class scores ----------------------------------------------------------------------

struct ScoreArgs {
  const void* x;
  int64_t ldx, rows;
  int32_t classes, dtype, kind;
  const void* bias;          // [classes], may be null
  const uint32_t* mask;      // [masks][words], may be null
  int32_t masks;
  const int32_t* mask_rows;  // [rows], may be null: row n's mask is n (masks == rows) or 0
  const int32_t* ids;        // may be null: no history
  const int64_t* offsets;    // [rows + 1]
  int64_t num_ids;
  double repetition, frequency, presence;
  const float* penalties;  // [rows][3], may be null: the three scalars
  void* out;
  int64_t ldo;
  void* ws;
};
size_t adjust_scores_workspace(int64_t rows, int32_t classes, int32_t dtype, int32_t kind, bool history);
void launch_adjust_scores(const ScoreArgs& a, hipStream_t s);

}  // namespace lgbm
