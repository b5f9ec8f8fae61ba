// leaf_capi.hip — the C entries of the operators around a forest's leaves
// (include/lgbm_hip.h): every argument is checked before the device is touched, then the
// work is queued on the caller's stream, or run to its end on the context's own.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <new>
#include <vector>

#include "context.h"
#include "leaf_ops.h"

using namespace lgbm;

namespace {

// The limit of work items along x, in blocks of the products' size.
constexpr int64_t MAX_GRID_X = (int64_t)0xffffffff / 256;

int bad(lgbm_hip_ctx* c, const char* what) {
  return context_error(c, LGBM_HIP_ERR_INVALID_ARGUMENT, what);
}
int mismatch(lgbm_hip_ctx* c, const char* what) {
  return context_error(c, LGBM_HIP_ERR_LENGTH_MISMATCH, what);
}
int beyond(lgbm_hip_ctx* c, const char* what) {
  return context_error(c, LGBM_HIP_ERR_CAPABILITY, what);
}

int64_t type_size(int32_t dtype) {
  switch (dtype) {
    case LGBM_HIP_DTYPE_F32: return 4;
    case LGBM_HIP_DTYPE_F64: return 8;
    case LGBM_HIP_DTYPE_BF16:
    case LGBM_HIP_DTYPE_F16: return 2;
    default: return 0;
  }
}

struct Span {
  const void* p;
  int64_t bytes;
  int64_t row, pitch;  // of a matrix: the bytes of a row, and from row to row
};
Span matrix(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t e) {
  return {p, rows > 0 ? ((rows - 1) * ld + cols) * e : 0, cols * e, ld * e};
}
bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  if (!(a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes && y < x + (uintptr_t)a.bytes))
    return false;
  if (a.pitch <= 0 || a.pitch != b.pitch) return true;
  // matrices side by side in one table: where b's row begins within a's pitch
  const uintptr_t pitch = (uintptr_t)a.pitch;
  const uintptr_t at = y >= x ? (y - x) % pitch : (pitch - (x - y) % pitch) % pitch;
  return at < (uintptr_t)a.row || at + (uintptr_t)b.row > pitch;
}
bool overlaps(const Span& out, std::initializer_list<Span> in) {
  for (const Span& s : in)
    if (overlap(out, s)) return true;
  return false;
}
bool misaligned(const void* p, int64_t e) { return (uintptr_t)p % (uintptr_t)e != 0; }

// Rows times a stride has to stay far from the end of 64 bits.
bool huge(int64_t rows, int64_t ld) { return ld > ((int64_t)1 << 40) || (__int128)rows * ld > ((__int128)1 << 58); }

int check_ws(lgbm_hip_ctx* c, const void* ws, size_t have, size_t need) {
  if (need == 0) return LGBM_HIP_OK;
  if (!ws) return bad(c, "null workspace");
  if (have < need) return mismatch(c, "workspace smaller than its _workspace entry says");
  if (misaligned(ws, 16)) return bad(c, "workspace not 16-byte aligned");
  return LGBM_HIP_OK;
}

// Queues `work` on the caller's stream, or runs it on the context's own; the caller's
// current device is put back.
template <typename F>
int queue(lgbm_hip_ctx* c, void* const* stream, F&& work) {
  if (!c) return bad(c, "null context");
  int device = -1;
  if (hipGetDevice(&device) != hipSuccess) return context_error(c, LGBM_HIP_ERR_HIP, "hipGetDevice");
  const int own = context_device(c);
  if (device != own && hipSetDevice(own) != hipSuccess)
    return context_error(c, LGBM_HIP_ERR_HIP, "hipSetDevice");
  const hipStream_t s = stream ? (hipStream_t)*stream : context_stream(c);
  (void)hipGetLastError();  // an earlier call's
  work(s);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && !stream) e = hipStreamSynchronize(s);
  if (device != own) (void)hipSetDevice(device);
  if (e != hipSuccess) return context_error(c, LGBM_HIP_ERR_HIP, hipGetErrorString(e));
  return LGBM_HIP_OK;
}

int check_groups(lgbm_hip_ctx* c, int64_t rows, int32_t trees, int32_t leaves) {
  if (rows < 0 || trees <= 0 || leaves <= 0) return bad(c, "rows, trees or leaves out of range");
  if (rows > INT32_MAX) return beyond(c, "2^31 rows or more");
  if (trees > LGBM_HIP_MAX_GROUP_TREES) return beyond(c, "more than 65535 trees");
  return LGBM_HIP_OK;
}

int check_maps(lgbm_hip_ctx* c, const lgbm_leaf_maps* m) {
  if (!m) return bad(c, "null maps");
  const int rc = check_groups(c, m->num_rows, m->num_trees, m->num_leaves);
  if (rc) return rc;
  if (m->inputs <= 0 || m->outputs <= 0) return bad(c, "inputs or outputs not positive");
  if (m->dtype != LGBM_HIP_DTYPE_F32 && m->dtype != LGBM_HIP_DTYPE_BF16 &&
      m->dtype != LGBM_HIP_DTYPE_F16)
    return bad(c, "dtype is none of f32, bf16 and f16");
  if (!m->d_begin || !m->d_count || (m->num_rows > 0 && !m->d_order)) return bad(c, "null order, begin or count");
  if ((int64_t)m->num_trees * m->num_leaves > INT32_MAX) return beyond(c, "2^31 leaves or more");
  if (m->inputs > (1 << 24) || m->outputs > (1 << 24)) return beyond(c, "more than 2^24 inputs or outputs");
  if ((__int128)m->num_trees * m->num_leaves * m->inputs * m->outputs > ((__int128)1 << 48))
    return beyond(c, "more than 2^48 weights");
  return LGBM_HIP_OK;
}

LeafProduct product_of(const lgbm_leaf_maps* m) {
  LeafProduct p{};
  p.g = LeafGroups{m->d_order, m->d_begin, m->d_count, (int32_t)m->num_rows, m->num_trees, m->num_leaves};
  p.inputs = m->inputs;
  p.outputs = m->outputs;
  p.dtype = m->dtype;
  return p;
}

int check_grid(lgbm_hip_ctx* c, const LeafProduct& p, int what) {
  return leaf_product_blocks(p, what) > MAX_GRID_X ? beyond(c, "too many leaves times outputs for one launch")
                                                   : LGBM_HIP_OK;
}

// `rows`: of a leaf's map for each output
Span weights(const lgbm_leaf_maps* m, const void* w, int64_t e, int64_t rows = 1) {
  return {w, (int64_t)m->num_trees * m->num_leaves * m->outputs * rows * m->inputs * e};
}
Span biases(const lgbm_leaf_maps* m, const void* b, int64_t e, int64_t rows = 1) {
  return {b, (int64_t)m->num_trees * m->num_leaves * m->outputs * rows * e};
}
Span kept(const lgbm_leaf_maps* m, const void* z, int64_t e, int64_t rows) {
  return {z, (int64_t)m->num_trees * m->num_rows * m->outputs * rows * e};
}
Span order_of(const lgbm_leaf_maps* m) { return {m->d_order, (int64_t)m->num_trees * m->num_rows * 4}; }
Span table(const lgbm_leaf_maps* m, const int32_t* t) {
  return {t, (int64_t)m->num_trees * m->num_leaves * 4};
}

}  // namespace

extern "C" {

int lgbm_hip_leaf_groups_workspace(int64_t num_rows, int32_t num_trees, int32_t num_leaves,
                                   size_t* bytes) {
  const int rc = check_groups(nullptr, num_rows, num_trees, num_leaves);
  if (rc) return rc;
  if (!bytes) return bad(nullptr, "null bytes");
  *bytes = leaf_groups_workspace(num_rows, num_trees, num_leaves);
  return LGBM_HIP_OK;
}

int lgbm_hip_leaf_groups(lgbm_hip_ctx* c, const int32_t* d_leaf, int64_t ld, int64_t rows,
                         int32_t trees, int32_t leaves, int32_t* d_order, int32_t* d_begin,
                         int32_t* d_count, void* d_ws, size_t ws_bytes, void* const* stream) {
  int rc = check_groups(c, rows, trees, leaves);
  if (rc) return rc;
  if (leaves > LGBM_HIP_MAX_GROUP_LEAVES) return beyond(c, "more than 4095 leaves a tree");
  if (ld < trees || huge(rows, ld)) return bad(c, "stride of the leaf indices out of range");
  if ((rows > 0 && (!d_leaf || !d_order)) || !d_begin || !d_count)
    return bad(c, "null leaf, order, begin or count");
  if (misaligned(d_leaf, 4) || misaligned(d_order, 4) || misaligned(d_begin, 4) || misaligned(d_count, 4))
    return bad(c, "a pointer is not aligned to its type");
  const size_t need = leaf_groups_workspace(rows, trees, leaves);
  if ((rc = check_ws(c, d_ws, ws_bytes, need))) return rc;
  const Span leaf = matrix(d_leaf, rows, trees, ld, 4), order{d_order, rows * trees * 4};
  const Span begin{d_begin, (int64_t)trees * leaves * 4}, count{d_count, begin.bytes};
  const Span ws{d_ws, (int64_t)need};
  if (overlaps(order, {leaf, begin, count, ws}) || overlaps(begin, {leaf, count, ws}) ||
      overlaps(count, {leaf, ws}) || overlaps(ws, {leaf}))
    return bad(c, "outputs overlap one another, the leaf indices or the workspace");
  return queue(c, stream, [&](hipStream_t s) {
    launch_leaf_groups(d_leaf, ld, rows, trees, leaves, d_order, d_begin, d_count, d_ws, s);
  });
}

int lgbm_hip_leaf_product_workspace(const lgbm_leaf_maps* m, int32_t what, size_t* bytes) {
  const int rc = check_maps(nullptr, m);
  if (rc) return rc;
  if (what < LGBM_HIP_LEAF_PRODUCT || what > LGBM_HIP_LEAF_PRODUCT_DW) return bad(nullptr, "unknown product");
  if (!bytes) return bad(nullptr, "null bytes");
  *bytes = leaf_product_workspace(product_of(m), what);
  return LGBM_HIP_OK;
}

int lgbm_hip_leaf_product(lgbm_hip_ctx* c, const lgbm_leaf_maps* m, const void* d_x, int64_t ldx,
                          const void* d_w, const void* d_bias, void* d_y, int64_t ldy, void* d_ws,
                          size_t ws_bytes, void* const* stream) {
  int rc = check_maps(c, m);
  if (rc) return rc;
  const int64_t e = type_size(m->dtype), rows = m->num_rows;
  if (ldx < m->inputs || ldy < m->outputs || huge(rows, ldx) || huge(rows, ldy))
    return bad(c, "row stride smaller than the row, or too large");
  if (!d_w || (rows > 0 && (!d_x || !d_y))) return bad(c, "null x, w or y");
  if (misaligned(d_x, e) || misaligned(d_w, e) || misaligned(d_bias, e) || misaligned(d_y, e))
    return bad(c, "a pointer is not aligned to its type");
  LeafProduct p = product_of(m);
  const size_t need = leaf_product_workspace(p, LEAF_PRODUCT_Y);
  p.x = d_x, p.ldx = ldx, p.w = d_w, p.b = d_bias, p.out = d_y, p.ldo = ldy, p.ws = d_ws;
  if ((rc = check_ws(c, d_ws, ws_bytes, need)) || (rc = check_grid(c, p, LEAF_PRODUCT_Y))) return rc;
  const Span y = matrix(d_y, rows, m->outputs, ldy, e), ws{d_ws, (int64_t)need};
  const Span x = matrix(d_x, rows, m->inputs, ldx, e), w = weights(m, d_w, e), b = biases(m, d_bias, e);
  if (overlaps(y, {x, w, b, order_of(m), table(m, m->d_begin), table(m, m->d_count), ws}) ||
      overlaps(ws, {x, w, b, order_of(m), table(m, m->d_begin), table(m, m->d_count)}))
    return bad(c, "y or the workspace overlaps an input");
  if (rows == 0) return c ? LGBM_HIP_OK : bad(c, "null context");
  return queue(c, stream, [&](hipStream_t s) { launch_leaf_product(p, LEAF_PRODUCT_Y, s); });
}

int lgbm_hip_leaf_product_dx(lgbm_hip_ctx* c, const lgbm_leaf_maps* m, const void* d_dy, int64_t lddy,
                             const void* d_w, void* d_dx, int64_t lddx, void* d_ws, size_t ws_bytes,
                             void* const* stream) {
  int rc = check_maps(c, m);
  if (rc) return rc;
  const int64_t e = type_size(m->dtype), rows = m->num_rows;
  if (lddy < m->outputs || lddx < m->inputs || huge(rows, lddy) || huge(rows, lddx))
    return bad(c, "row stride smaller than the row, or too large");
  if (!d_w || (rows > 0 && (!d_dy || !d_dx))) return bad(c, "null dy, w or dx");
  if (misaligned(d_dy, e) || misaligned(d_w, e) || misaligned(d_dx, e))
    return bad(c, "a pointer is not aligned to its type");
  LeafProduct p = product_of(m);
  const size_t need = leaf_product_workspace(p, LEAF_PRODUCT_DX);
  p.dy = d_dy, p.lddy = lddy, p.w = d_w, p.out = d_dx, p.ldo = lddx, p.ws = d_ws;
  if ((rc = check_ws(c, d_ws, ws_bytes, need)) || (rc = check_grid(c, p, LEAF_PRODUCT_DX))) return rc;
  const Span dx = matrix(d_dx, rows, m->inputs, lddx, e), ws{d_ws, (int64_t)need};
  const Span dy = matrix(d_dy, rows, m->outputs, lddy, e), w = weights(m, d_w, e);
  if (overlaps(dx, {dy, w, order_of(m), table(m, m->d_begin), table(m, m->d_count), ws}) ||
      overlaps(ws, {dy, w, order_of(m), table(m, m->d_begin), table(m, m->d_count)}))
    return bad(c, "dx or the workspace overlaps an input");
  if (rows == 0) return c ? LGBM_HIP_OK : bad(c, "null context");
  return queue(c, stream, [&](hipStream_t s) { launch_leaf_product(p, LEAF_PRODUCT_DX, s); });
}

int lgbm_hip_leaf_product_dw(lgbm_hip_ctx* c, const lgbm_leaf_maps* m, const void* d_dy, int64_t lddy,
                             const void* d_x, int64_t ldx, float* d_dw, float* d_db, void* d_ws,
                             size_t ws_bytes, void* const* stream) {
  int rc = check_maps(c, m);
  if (rc) return rc;
  const int64_t e = type_size(m->dtype), rows = m->num_rows;
  if (lddy < m->outputs || ldx < m->inputs || huge(rows, lddy) || huge(rows, ldx))
    return bad(c, "row stride smaller than the row, or too large");
  if (!d_dw || (rows > 0 && (!d_dy || !d_x))) return bad(c, "null dy, x or dw");
  if (misaligned(d_dy, e) || misaligned(d_x, e) || misaligned(d_dw, 4) || misaligned(d_db, 4))
    return bad(c, "a pointer is not aligned to its type");
  LeafProduct p = product_of(m);
  const size_t need = leaf_product_workspace(p, LEAF_PRODUCT_DW);
  p.dy = d_dy, p.lddy = lddy, p.x = d_x, p.ldx = ldx, p.dw = d_dw, p.db = d_db, p.ws = d_ws;
  if ((rc = check_ws(c, d_ws, ws_bytes, need)) || (rc = check_grid(c, p, LEAF_PRODUCT_DW))) return rc;
  const Span dw = weights(m, d_dw, 4), db = biases(m, d_db, 4), ws{d_ws, (int64_t)need};
  const Span dy = matrix(d_dy, rows, m->outputs, lddy, e), x = matrix(d_x, rows, m->inputs, ldx, e);
  if (overlaps(dw, {dy, x, db, order_of(m), table(m, m->d_begin), table(m, m->d_count), ws}) ||
      overlaps(db, {dy, x, order_of(m), table(m, m->d_begin), table(m, m->d_count), ws}) ||
      overlaps(ws, {dy, x, order_of(m), table(m, m->d_begin), table(m, m->d_count)}))
    return bad(c, "dw, db or the workspace overlaps an input or one another");
  return queue(c, stream, [&](hipStream_t s) { launch_leaf_product(p, LEAF_PRODUCT_DW, s); });
}

// ---- layers ----------------------------------------------------------------------------

static int check_layer(lgbm_hip_ctx* c, const lgbm_leaf_maps* m, int32_t activation, int32_t gated,
                       int32_t z_dtype) {
  const int rc = check_maps(c, m);
  if (rc) return rc;
  if (activation < LGBM_HIP_ACT_NONE || activation > LGBM_HIP_ACT_SIGMOID) return bad(c, "unknown activation");
  if (gated != 0 && gated != 1) return bad(c, "gated is neither 0 nor 1");
  if (z_dtype != m->dtype && z_dtype != LGBM_HIP_DTYPE_F32) return bad(c, "z_dtype is neither the maps' nor f32");
  const int64_t rows = gated ? 2 : 1;
  if ((__int128)m->num_trees * m->num_leaves * m->inputs * m->outputs * rows > ((__int128)1 << 48))
    return beyond(c, "more than 2^48 weights");
  if (m->outputs * rows > (1 << 24)) return beyond(c, "more than 2^24 rows of a leaf's map");
  if ((__int128)m->num_trees * m->num_rows * m->outputs * rows > ((__int128)1 << 58))
    return beyond(c, "more than 2^58 elements of z");
  return LGBM_HIP_OK;
}

static LeafProduct layer_of(const lgbm_leaf_layer* a) {
  LeafProduct p = product_of(&a->maps);
  p.act = a->activation, p.gated = a->gated != 0;
  p.x = a->d_x, p.ldx = a->ldx, p.w = a->d_w, p.b = a->d_bias, p.res = a->d_residual, p.ldr = a->ldr;
  p.out = a->d_y, p.ldo = a->ldy, p.z = a->d_z, p.z_narrow = a->z_dtype != LGBM_HIP_DTYPE_F32;
  return p;
}

int lgbm_hip_leaf_layer_workspace(const lgbm_leaf_layer* a, size_t* bytes) {
  if (!a) return bad(nullptr, "null layer");
  const int rc = check_layer(nullptr, &a->maps, a->activation, a->gated, a->z_dtype);
  if (rc) return rc;
  if (!bytes) return bad(nullptr, "null bytes");
  *bytes = leaf_product_workspace(layer_of(a), LEAF_LAYER);
  return LGBM_HIP_OK;
}

int lgbm_hip_leaf_layer(lgbm_hip_ctx* c, const lgbm_leaf_layer* a, void* d_ws, size_t ws_bytes,
                        void* const* stream) {
  if (!a) return bad(c, "null layer");
  const lgbm_leaf_maps* const m = &a->maps;
  int rc = check_layer(c, m, a->activation, a->gated, a->z_dtype);
  if (rc) return rc;
  const int64_t e = type_size(m->dtype), rows = m->num_rows, of = a->gated ? 2 : 1;
  if (a->ldx < m->inputs || a->ldy < m->outputs || (a->d_residual && a->ldr < m->outputs) || huge(rows, a->ldx) ||
      huge(rows, a->ldy) || (a->d_residual && huge(rows, a->ldr)))
    return bad(c, "row stride smaller than the row, or too large");
  if (!a->d_w || (rows > 0 && (!a->d_x || !a->d_y))) return bad(c, "null x, w or y");
  if (misaligned(a->d_x, e) || misaligned(a->d_w, e) || misaligned(a->d_bias, e) || misaligned(a->d_residual, e) ||
      misaligned(a->d_y, e) || misaligned(a->d_z, type_size(a->z_dtype)))
    return bad(c, "a pointer is not aligned to its type");
  LeafProduct p = layer_of(a);
  p.ws = d_ws;
  const size_t need = leaf_product_workspace(p, LEAF_LAYER);
  if ((rc = check_ws(c, d_ws, ws_bytes, need)) || (rc = check_grid(c, p, LEAF_LAYER))) return rc;
  const Span x = matrix(a->d_x, rows, m->inputs, a->ldx, e), w = weights(m, a->d_w, e, of);
  const Span b = biases(m, a->d_bias, e, of), z = kept(m, a->d_z, type_size(a->z_dtype), of), ws{d_ws, (int64_t)need};
  const Span y = matrix(a->d_y, rows, m->outputs, a->ldy, e);
  const Span r = matrix(a->d_residual, a->d_residual ? rows : 0, m->outputs, a->ldr, e);
  const Span order = order_of(m), begin = table(m, m->d_begin), count = table(m, m->d_count);
  if (overlaps(y, {x, w, b, z, order, begin, count, ws}) || overlaps(z, {x, w, b, r, order, begin, count, ws}) ||
      overlaps(ws, {x, w, b, r, order, begin, count}))
    return bad(c, "y, z or the workspace overlaps an input or one another");
  if (!(a->d_y == a->d_residual && a->ldy == a->ldr) && overlap(y, r))
    return bad(c, "y overlaps the residual other than in place");
  if (rows == 0) return c ? LGBM_HIP_OK : bad(c, "null context");
  return queue(c, stream, [&](hipStream_t s) { launch_leaf_product(p, LEAF_LAYER, s); });
}

// dz is dy itself where the layer is a linear map.
static bool linear(const lgbm_leaf_layer_grad* a) { return a->activation == LGBM_HIP_ACT_NONE && !a->gated; }

// The products that a layer's gradients are, of dz (at `dz`) in dy's place.
static LeafProduct layer_grad_of(const lgbm_leaf_layer_grad* a, const void* dz) {
  LeafProduct p = product_of(&a->maps);
  if (a->gated) p.outputs *= 2;
  p.dy = linear(a) ? a->d_dy : dz;
  p.lddy = linear(a) ? a->lddy : p.outputs;
  p.dy_tree = linear(a) ? 0 : a->maps.num_rows * p.outputs;
  p.x = a->d_x, p.ldx = a->ldx, p.w = a->d_w, p.out = a->d_dx, p.ldo = a->lddx, p.dw = a->d_dw, p.db = a->d_dbias;
  p.narrow = a->dw_dtype != LGBM_HIP_DTYPE_F32;
  p.rest = true;
  return p;
}

static int64_t dz_bytes(const lgbm_leaf_layer_grad* a) {
  if (linear(a)) return 0;
  const int64_t n = (int64_t)a->maps.num_trees * a->maps.num_rows * a->maps.outputs * (a->gated ? 2 : 1);
  return (n * type_size(a->maps.dtype) + 255) / 256 * 256;
}

// dz, then what the products need, one after the other.
static size_t layer_grad_workspace(const lgbm_leaf_layer_grad* a) {
  const LeafProduct p = layer_grad_of(a, nullptr);
  return (size_t)dz_bytes(a) + std::max(a->d_dx ? leaf_product_workspace(p, LEAF_PRODUCT_DX) : 0,
                                        a->d_dw ? leaf_product_workspace(p, LEAF_PRODUCT_DW) : 0);
}

static int check_layer_grad(lgbm_hip_ctx* c, const lgbm_leaf_layer_grad* a) {
  if (!a) return bad(c, "null gradient");
  const int rc = check_layer(c, &a->maps, a->activation, a->gated, a->z_dtype);
  if (rc) return rc;
  if (a->dw_dtype != a->maps.dtype && a->dw_dtype != LGBM_HIP_DTYPE_F32)
    return bad(c, "dw_dtype is neither the maps' nor f32");
  if (!a->d_dx && !a->d_dw) return bad(c, "neither dx nor dw is asked for");
  if (a->d_dbias && !a->d_dw) return bad(c, "dbias without dw");
  return LGBM_HIP_OK;
}

int lgbm_hip_leaf_layer_grad_workspace(const lgbm_leaf_layer_grad* a, size_t* bytes) {
  const int rc = check_layer_grad(nullptr, a);
  if (rc) return rc;
  if (!bytes) return bad(nullptr, "null bytes");
  *bytes = layer_grad_workspace(a);
  return LGBM_HIP_OK;
}

int lgbm_hip_leaf_layer_grad(lgbm_hip_ctx* c, const lgbm_leaf_layer_grad* a, void* d_ws, size_t ws_bytes,
                             void* const* stream) {
  int rc = check_layer_grad(c, a);
  if (rc) return rc;
  const lgbm_leaf_maps* const m = &a->maps;
  const int64_t e = type_size(m->dtype), rows = m->num_rows, of = a->gated ? 2 : 1;
  const int64_t we = type_size(a->dw_dtype), ze = type_size(a->z_dtype);
  if (a->lddy < m->outputs || (a->d_dw && a->ldx < m->inputs) || (a->d_dx && a->lddx < m->inputs) ||
      huge(rows, a->lddy) || (a->d_dw && huge(rows, a->ldx)) || (a->d_dx && huge(rows, a->lddx)))
    return bad(c, "row stride smaller than the row, or too large");
  if ((rows > 0 && (!a->d_dy || (!a->d_z && !linear(a)) || (a->d_dw && !a->d_x))) || (a->d_dx && !a->d_w))
    return bad(c, "null dy, z, x or w");
  if (misaligned(a->d_dy, e) || misaligned(a->d_z, ze) || misaligned(a->d_x, e) || misaligned(a->d_w, e) ||
      misaligned(a->d_dx, e) || misaligned(a->d_dw, we) || misaligned(a->d_dbias, we))
    return bad(c, "a pointer is not aligned to its type");
  const size_t need = layer_grad_workspace(a);
  if ((rc = check_ws(c, d_ws, ws_bytes, need))) return rc;
  LeafProduct p = layer_grad_of(a, d_ws);
  p.ws = (char*)d_ws + dz_bytes(a);
  if (a->d_dx && (rc = check_grid(c, p, LEAF_PRODUCT_DX))) return rc;
  if (a->d_dw && (rc = check_grid(c, p, LEAF_PRODUCT_DW))) return rc;
  const Span dy = matrix(a->d_dy, rows, m->outputs, a->lddy, e), z = kept(m, linear(a) ? nullptr : a->d_z, ze, of);
  const Span x = matrix(a->d_x, a->d_dw ? rows : 0, m->inputs, a->ldx, e);
  const Span w = weights(m, a->d_dx ? a->d_w : nullptr, e, of), ws{d_ws, (int64_t)need};
  const Span dx = matrix(a->d_dx, a->d_dx ? rows : 0, m->inputs, a->lddx, e);
  const Span dw = weights(m, a->d_dw, we, of), db = biases(m, a->d_dbias, we, of);
  const Span order = order_of(m), begin = table(m, m->d_begin), count = table(m, m->d_count);
  if (overlaps(dx, {dy, z, x, w, dw, db, order, begin, count, ws}) ||
      overlaps(dw, {dy, z, x, w, db, order, begin, count, ws}) ||
      overlaps(db, {dy, z, x, w, order, begin, count, ws}) || overlaps(ws, {dy, z, x, w, order, begin, count}))
    return bad(c, "an output or the workspace overlaps an input or one another");
  if (rows == 0 && !a->d_dw) return c ? LGBM_HIP_OK : bad(c, "null context");
  return queue(c, stream, [&](hipStream_t s) {
    if (rows > 0 && !linear(a)) {
      LeafProduct q = product_of(m);
      q.act = a->activation, q.gated = a->gated != 0;
      q.dy = a->d_dy, q.lddy = a->lddy, q.z = const_cast<void*>(a->d_z);
      q.z_narrow = a->z_dtype != LGBM_HIP_DTYPE_F32;
      launch_layer_dz(q, d_ws, s);
    }
    if (rows > 0 && a->d_dx) launch_leaf_product(p, LEAF_PRODUCT_DX, s);
    if (a->d_dw) launch_leaf_product(p, LEAF_PRODUCT_DW, s);
  });
}

// ---- the norm of many tensors ------------------------------------------------------------

// The list as the kernels' launcher takes it; an error code, or LGBM_HIP_OK.
static int check_grads(lgbm_hip_ctx* c, const lgbm_grad* g, int64_t num, bool clip, std::vector<GradTensor>& list) {
  if (num < 0 || (num > 0 && !g)) return bad(c, "null or negative list of gradients");
  if (num > (1 << 24)) return beyond(c, "more than 2^24 gradients");
  try {
    list.reserve((size_t)num);
  } catch (const std::bad_alloc&) {
    return beyond(c, "no host memory for the list of gradients");
  }
  int64_t total = 0;
  for (int64_t i = 0; i < num; ++i) {
    if (g[i].dtype != LGBM_HIP_DTYPE_F32 && g[i].dtype != LGBM_HIP_DTYPE_BF16 && g[i].dtype != LGBM_HIP_DTYPE_F16)
      return bad(c, "dtype is none of f32, bf16 and f16");
    if (g[i].count < 0) return bad(c, "negative count");
    if (g[i].count > ((int64_t)1 << 48) || (total += g[i].count) > ((int64_t)1 << 48))
      return beyond(c, "more than 2^48 elements");
    if (g[i].count == 0) continue;
    const int64_t e = type_size(g[i].dtype);
    if (!g[i].d_in || (clip && !g[i].d_out)) return bad(c, "null gradient");
    if (misaligned(g[i].d_in, e) || (clip && misaligned(g[i].d_out, e)))
      return bad(c, "a pointer is not aligned to its type");
    list.push_back({g[i].d_in, clip ? g[i].d_out : nullptr, g[i].count, g[i].dtype});
  }
  return LGBM_HIP_OK;
}

// Whether a clipped gradient overlaps anything but its own input, or `more`.  Views of one buffer
// come in its order, so the lists are mostly sorted.
static bool clipped_overlap(const std::vector<GradTensor>& list, std::initializer_list<Span> more, bool& no_memory) {
  struct Range {
    uintptr_t from, to;
  };
  std::vector<Range> in, out;
  try {
    in.reserve(list.size());
    out.reserve(list.size() + more.size());
  } catch (const std::bad_alloc&) {
    no_memory = true;
    return false;
  }
  const auto range = [](const void* p, int64_t bytes) { return Range{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes}; };
  for (const GradTensor& t : list) {
    const int64_t bytes = t.count * type_size(t.dtype);
    out.push_back(range(t.out, bytes));
    if (t.in != t.out) in.push_back(range(t.in, bytes));
  }
  for (const Span& s : more)
    if (s.p && s.bytes > 0) out.push_back(range(s.p, s.bytes));
  const auto before = [](const Range& a, const Range& b) { return a.from < b.from; };
  for (std::vector<Range>* v : {&in, &out})
    if (!std::is_sorted(v->begin(), v->end(), before)) std::sort(v->begin(), v->end(), before);
  for (size_t k = 1; k < out.size(); ++k)
    if (out[k].from < out[k - 1].to) return true;
  // inputs may overlap one another: of those that begin in front of an output's end, the
  // furthest end
  size_t at = 0;
  uintptr_t end = 0;
  for (const Range& o : out) {
    for (; at < in.size() && in[at].from < o.to; ++at) end = std::max(end, in[at].to);
    if (end > o.from) return true;
  }
  return false;
}

int lgbm_hip_grad_norm_workspace(const lgbm_grad* g, int64_t num, size_t* bytes) {
  // sizes and types: pointers may be missing still
  if (num < 0 || (num > 0 && !g)) return bad(nullptr, "null or negative list of gradients");
  if (num > (1 << 24)) return beyond(nullptr, "more than 2^24 gradients");
  if (!bytes) return bad(nullptr, "null bytes");
  int64_t total = 0;
  for (int64_t i = 0; i < num; ++i) {
    if (g[i].count < 0) return bad(nullptr, "negative count");
    if (g[i].count > ((int64_t)1 << 48) || (total += g[i].count) > ((int64_t)1 << 48))
      return beyond(nullptr, "more than 2^48 elements");
  }
  *bytes = grad_norm_workspace(total, num);
  return LGBM_HIP_OK;
}

static int norm_and_clip(lgbm_hip_ctx* c, const lgbm_grad* g, int64_t num, bool clip, double most, float* d_norm,
                         void* d_ws, size_t ws_bytes, void* const* stream) {
  std::vector<GradTensor> list;
  int rc = check_grads(c, g, num, clip, list);
  if (rc) return rc;
  if (clip && !(most >= 0.0)) return bad(c, "max_norm is negative or NaN");
  if (!d_norm) return bad(c, "null norm");
  if (misaligned(d_norm, 4)) return bad(c, "a pointer is not aligned to its type");
  int64_t total = 0;
  for (const GradTensor& t : list) total += t.count;
  const size_t need = grad_norm_workspace(total, num);
  if ((rc = check_ws(c, d_ws, ws_bytes, need))) return rc;
  const Span norm{d_norm, 4}, ws{d_ws, (int64_t)need};
  if (clip) {
    bool no_memory = false;
    if (clipped_overlap(list, {norm, ws}, no_memory))
      return bad(c, "a clipped gradient, the norm or the workspace overlaps another tensor");
    if (no_memory) return beyond(c, "no host memory for the list of gradients");
  } else {
    bool hit = overlap(norm, ws);
    for (const GradTensor& t : list) {
      const Span in{t.in, t.count * type_size(t.dtype)};
      hit = hit || overlap(norm, in) || overlap(ws, in);
    }
    if (hit) return bad(c, "the norm or the workspace overlaps a gradient or one another");
  }
  return queue(c, stream, [&](hipStream_t s) {
    launch_grad_norm(list.data(), (int64_t)list.size(), clip, most, d_norm, d_ws, s);
  });
}

int lgbm_hip_grad_norm(lgbm_hip_ctx* c, const lgbm_grad* g, int64_t num, float* d_norm, void* d_ws,
                       size_t ws_bytes, void* const* stream) {
  return norm_and_clip(c, g, num, false, 0.0, d_norm, d_ws, ws_bytes, stream);
}

int lgbm_hip_clip_grads(lgbm_hip_ctx* c, const lgbm_grad* g, int64_t num, double max_norm, float* d_norm, void* d_ws,
                        size_t ws_bytes, void* const* stream) {
  return norm_and_clip(c, g, num, true, max_norm, d_norm, d_ws, ws_bytes, stream);
}

int lgbm_hip_dropout(lgbm_hip_ctx* c, const void* d_x, int64_t ldx, int64_t rows, int64_t cols,
                     int32_t dtype, double p, uint64_t seed, uint64_t offset, int32_t by_row,
                     void* d_out, int64_t ldo, void* const* stream) {
  if (rows < 0 || cols < 0) return bad(c, "negative rows or columns");
  if (dtype != LGBM_HIP_DTYPE_F32 && dtype != LGBM_HIP_DTYPE_BF16 && dtype != LGBM_HIP_DTYPE_F16)
    return bad(c, "dtype is none of f32, bf16 and f16");
  if (!(p >= 0.0 && p <= 1.0)) return bad(c, "p outside [0, 1]");
  if (ldx < cols || ldo < cols || huge(rows, ldx) || huge(rows, ldo))
    return bad(c, "row stride smaller than the row, or too large");
  if (cols > 0 && rows > ((int64_t)1 << 60) / cols) return beyond(c, "2^60 elements or more");
  const int64_t e = type_size(dtype);
  const bool none = rows == 0 || cols == 0;
  if (!none && (!d_x || !d_out)) return bad(c, "null x or out");
  if (misaligned(d_x, e) || misaligned(d_out, e)) return bad(c, "a pointer is not aligned to its type");
  if (!(d_x == d_out && ldx == ldo) &&
      overlap(matrix(d_x, rows, cols, ldx, e), matrix(d_out, rows, cols, ldo, e)))
    return bad(c, "out overlaps x other than in place");
  if (none) return c ? LGBM_HIP_OK : bad(c, "null context");
  const uint32_t threshold = (uint32_t)std::lround(p * 65536.0);
  return queue(c, stream, [&](hipStream_t s) {
    launch_dropout(d_x, ldx, rows, cols, dtype, threshold, seed, offset, by_row != 0, d_out, ldo, s);
  });
}

static int check_scores(lgbm_hip_ctx* c, const lgbm_score_args* a) {
  if (!a) return bad(c, "null args");
  const int64_t e = type_size(a->dtype);
  if (e == 0) return bad(c, "unknown dtype");
  if (a->kind != LGBM_HIP_PREDICT_RAW && a->kind != LGBM_HIP_PREDICT_TRANSFORMED)
    return bad(c, "kind is neither raw nor transformed");
  if (a->num_rows < 0 || a->num_classes <= 0) return bad(c, "rows or classes out of range");
  if (a->num_rows > INT32_MAX || a->num_classes > INT32_MAX / 2) return beyond(c, "too many rows or classes");
  if (a->ldx < a->num_classes || a->ldo < a->num_classes || huge(a->num_rows, a->ldx) ||
      huge(a->num_rows, a->ldo))
    return bad(c, "row stride smaller than the row, or too large");
  if (a->num_rows > 0 && (!a->d_x || !a->d_out)) return bad(c, "null x or out");
  if (a->d_mask) {
    if (a->num_masks <= 0) return bad(c, "a mask table without masks");
    if (!a->d_mask_rows && a->num_masks != 1 && a->num_masks != a->num_rows)
      return mismatch(c, "one mask, a mask for each row, or mask_rows");
  }
  if (a->d_ids || a->d_offsets || a->num_ids) {
    if (a->num_ids < 0 || !a->d_offsets || (a->num_ids > 0 && !a->d_ids))
      return bad(c, "a history needs ids and offsets");
    // in the type of the arithmetic, where a small repetition may be 0 and a large one infinite
    const bool wide = a->dtype == LGBM_HIP_DTYPE_F64;
    const auto of = [&](double v) { return wide ? v : (double)(float)v; };
    if (!a->d_penalties && !(of(a->repetition) > 0.0 && std::isfinite(of(a->repetition)) &&
                             std::isfinite(of(a->frequency)) && std::isfinite(of(a->presence))))
      return bad(c, "repetition not positive, or a penalty not finite");
  }
  if (misaligned(a->d_x, e) || misaligned(a->d_out, e) || misaligned(a->d_bias, e) ||
      misaligned(a->d_mask, 4) || misaligned(a->d_mask_rows, 4) || misaligned(a->d_ids, 4) ||
      misaligned(a->d_offsets, 8) || misaligned(a->d_penalties, 4))
    return bad(c, "a pointer is not aligned to its type");
  return LGBM_HIP_OK;
}

int lgbm_hip_adjust_scores_workspace(const lgbm_score_args* a, size_t* bytes) {
  const int rc = check_scores(nullptr, a);
  if (rc) return rc;
  if (!bytes) return bad(nullptr, "null bytes");
  *bytes = adjust_scores_workspace(a->num_rows, a->num_classes, a->dtype, a->kind, a->num_ids > 0);
  return LGBM_HIP_OK;
}

int lgbm_hip_adjust_scores(lgbm_hip_ctx* c, const lgbm_score_args* a, void* d_ws, size_t ws_bytes,
                           void* const* stream) {
  int rc = check_scores(c, a);
  if (rc) return rc;
  const size_t need = adjust_scores_workspace(a->num_rows, a->num_classes, a->dtype, a->kind, a->num_ids > 0);
  if ((rc = check_ws(c, d_ws, ws_bytes, need))) return rc;
  const int64_t e = type_size(a->dtype), rows = a->num_rows, V = a->num_classes;
  const Span x = matrix(a->d_x, rows, V, a->ldx, e), out = matrix(a->d_out, rows, V, a->ldo, e);
  const Span ws{d_ws, (int64_t)need}, bias{a->d_bias, V * e};
  const Span mask{a->d_mask, (int64_t)a->num_masks * ((V + 31) / 32) * 4};
  const Span mask_rows{a->d_mask_rows, rows * 4}, ids{a->d_ids, a->num_ids * 4};
  const Span offsets{a->d_offsets, (rows + 1) * 8}, penalties{a->d_penalties, rows * 12};
  if (!(a->d_x == a->d_out && a->ldx == a->ldo) && overlap(x, out))
    return bad(c, "out overlaps x other than in place");
  if (overlaps(out, {bias, mask, mask_rows, ids, offsets, penalties, ws}) ||
      overlaps(ws, {x, bias, mask, mask_rows, ids, offsets, penalties}))
    return bad(c, "out or the workspace overlaps an input");
  if (rows == 0) return c ? LGBM_HIP_OK : bad(c, "null context");
  ScoreArgs s{};
  s.x = a->d_x, s.ldx = a->ldx, s.rows = rows, s.classes = a->num_classes, s.dtype = a->dtype;
  s.kind = a->kind, s.bias = a->d_bias, s.mask = a->d_mask, s.masks = a->num_masks;
  s.mask_rows = a->d_mask ? a->d_mask_rows : nullptr;
  s.ids = a->num_ids > 0 ? a->d_ids : nullptr, s.offsets = a->d_offsets, s.num_ids = a->num_ids;
  s.repetition = a->repetition, s.frequency = a->frequency, s.presence = a->presence;
  s.penalties = a->d_penalties, s.out = a->d_out, s.ldo = a->ldo, s.ws = d_ws;
  return queue(c, stream, [&](hipStream_t q) { launch_adjust_scores(s, q); });
}

}  // extern "C"
