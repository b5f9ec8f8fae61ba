// leaf_capi.hip — the C entries of the operators around a forest's leaves
// (include/lgbm_hip.h): every argument is checked before the device is touched, then the
// work is queued on the caller's stream, or run to its end on the context's own.
#include <cmath>
#include <cstdint>
#include <initializer_list>

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

Span weights(const lgbm_leaf_maps* m, const void* w, int64_t e) {
  return {w, (int64_t)m->num_trees * m->num_leaves * m->outputs * m->inputs * e};
}
Span biases(const lgbm_leaf_maps* m, const void* b, int64_t e) {
  return {b, (int64_t)m->num_trees * m->num_leaves * m->outputs * e};
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
