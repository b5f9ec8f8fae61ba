// leaf_ops.h — the operators around a forest's leaves: rows grouped by leaf, the leaves'
// linear maps and layers and their gradients, clipping of gradients, dropout and class scores.
// Launchers of the kernels in leaf_groups.hip, leaf_product.hip, leaf_layer.hip, grad_norm.hip,
// dropout.hip and scores.hip, called by the C entries in leaf_capi.hip, which check every
// argument first.  Nothing here allocates or waits, so every launcher can be recorded into a
// graph.
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
  int64_t dy_tree;  // elements from a tree's dy to the next one's, 0: the trees share it
  void* out;  // product: y [rows][outputs]; dx: [rows][inputs]
  int64_t ldo;
  void* dw;  // [trees * leaves][outputs][inputs]
  void* db;  // [trees * leaves][outputs], may be null
  bool narrow;  // dw and db are of the type dtype, else float32
  void* ws;
  // product, layer and dx: whether a tree's results go to its float32 plane [rows][columns] in
  // ws, to be added, instead of to out
  bool planes;
  // layer, and dx of its gradient: whether the large tiles behind their last whole round go to
  // smaller ones (not product and dx of the linear maps, whose results stay what they were: smaller
  // tiles add in another order)
  bool rest;
  // layer: out[n] = res[n] + sum over trees of act(z), or of act(z's first half) times its
  // second half where gated; z = W x + b has map_rows() elements, `outputs` those of the layer
  int32_t act;
  bool gated;
  const void* res;  // [rows][outputs], may be null
  int64_t ldr;
  void* z;  // [trees][rows][map_rows()], may be null
  bool z_narrow;  // z is of the type dtype, else float32
  // where a tree's z begins
  template <typename T>
  __host__ __device__ void* z_of(int64_t tree) const {
    const int64_t at = tree * g.rows * map_rows();
    return z_narrow ? (void*)((T*)z + at) : (void*)((float*)z + at);
  }
  __host__ __device__ int map_rows() const { return gated ? 2 * outputs : outputs; }
};

#define LEAF_PRODUCT_Y 0
#define LEAF_PRODUCT_DX 1
#define LEAF_PRODUCT_DW 2
#define LEAF_LAYER 3
size_t leaf_product_workspace(const LeafProduct& p, int what);
int64_t leaf_product_blocks(const LeafProduct& p, int what);  // along x of its largest launch
void launch_leaf_product(const LeafProduct& p, int what, hipStream_t s);
// leaf_layer.hip: the layer of the leaves of one tree, or of several into their planes
int64_t leaf_layer_blocks(const LeafProduct& p);
void launch_leaf_layer(const LeafProduct& p, int trees, hipStream_t s);
// dz [trees][rows][map_rows()] = the gradient of z from p.dy and p.z
void launch_layer_dz(const LeafProduct& p, void* dz, hipStream_t s);
// leaf_big.hip: 16-bit products of large tiles
bool leaf_big_fits(const LeafProduct& p, int what);
int64_t leaf_big_blocks(const LeafProduct& p, int what);
int64_t leaf_big_cols(const LeafProduct& p, int what);  // tiles along the columns of a result
void launch_leaf_big(const LeafProduct& p, int what, hipStream_t s);

// ---- the norm of many tensors ------------------------------------------------------------

// Tensor i of a list: `count` elements from `in` on, without gaps; clipped into `out`.
struct GradTensor {
  const void* in;
  void* out;
  int64_t count;
  int32_t dtype;
};
size_t grad_norm_workspace(int64_t elements, int64_t num);
// norm: a float32 on the device.  clip: out = in * min(1, most / norm) too
void launch_grad_norm(const GradTensor* t, int64_t num, bool clip, double most, float* norm, void* ws,
                      hipStream_t s);

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
