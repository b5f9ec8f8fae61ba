// dropout.hip — elements or whole rows dropped by a counter-based generator.  The mask is a
// function of (seed, offset, unit) and is never stored: the gradient is the same call on
// the outputs' gradient.
//
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", 2011): counter (block, offset), key seed.  A block's 128 bits give eight 16-bit
// fields, so the ten rounds are shared by eight units; unit e is kept where field e % 8 of
// block e / 8 is at least threshold = round(65536 p), and what is kept is divided by the
// share that is really kept, 1 - threshold / 65536.
//
// Bound by memory: an element is read and written once; the ten rounds' twenty 32 x 32
// products for eight elements are below the time that their bytes take.  Elements without
// gaps between rows are one long row (k_dropout_flat: 32771 x 4096 bfloat16 89 us, 6.0 TB/s);
// so are whole rows of 1, 2 or 4 columns, where a thread's vector holds several
// (k_dropout_pairs: 10.5M x 2 float32 29 us, 5.8 TB/s); the rest goes row by row, eight
// elements a thread (k_dropout_rows: 32771 x 4096 of stride 4104 111 us, 4.8 TB/s; 10M x 3
// whole rows of float32 94 us, where every row makes its own block of the generator).
#include <algorithm>

#include "leaf_ops.h"

#include "../../include/lgbm_hip.h"

namespace lgbm {
namespace {

constexpr int THREADS = 256;

__device__ __forceinline__ uint4 philox(uint64_t block, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t field_of(const uint4& r, int j) {
  const uint32_t w = j < 4 ? (j < 2 ? r.x : r.y) : (j < 6 ? r.z : r.w);
  return (j & 1) ? w >> 16 : w & 0xffffu;
}

struct Dropout {
  uint32_t threshold;
  float scale;
  uint64_t seed, offset;
};

template <typename T>
__device__ __forceinline__ T kept(T x, bool keep, float scale) {
  return keep ? (T)((float)x * scale) : (T)0.0f;
}

// `total` elements in a row: a block of eight a thread, as 16-byte vectors.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_dropout_flat(const T* x, int64_t total, Dropout d, T* out) {
  const int64_t blocks = (total + 7) / 8;
  for (int64_t b = blockIdx.x * (int64_t)THREADS + threadIdx.x; b < blocks;
       b += (int64_t)gridDim.x * THREADS) {
    const uint4 r = philox((uint64_t)b, d.offset, d.seed);
    T v[8];
    if (b * 8 + 8 <= total) {
      __builtin_memcpy(v, x + b * 8, sizeof(v));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = kept(v[j], field_of(r, j) >= d.threshold, d.scale);
      __builtin_memcpy(out + b * 8, v, sizeof(v));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (b * 8 + j < total) out[b * 8 + j] = kept(x[b * 8 + j], field_of(r, j) >= d.threshold, d.scale);
    }
  }
}

// Whole rows of 1, 2 or 4 columns without gaps, a vector a thread: its rows lie in one block
// of the generator.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_dropout_pairs(const T* x, int64_t total, int col_bits,
                                                           Dropout d, T* out) {
  constexpr int V = 16 / (int)sizeof(T);
  for (int64_t i = (blockIdx.x * (int64_t)THREADS + threadIdx.x) * V; i < total;
       i += (int64_t)gridDim.x * THREADS * V) {
    const int64_t row = i >> col_bits;
    const uint4 r = philox((uint64_t)(row >> 3), d.offset, d.seed);
    const uint64_t lo = (uint64_t)r.y << 32 | r.x, hi = (uint64_t)r.w << 32 | r.z;
    T v[V];
    if (i + V <= total) {
      __builtin_memcpy(v, x + i, sizeof(v));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int j = (int)((i + e) >> col_bits) & 7;
        const uint32_t f = (uint32_t)((j < 4 ? lo : hi) >> ((j & 3) * 16)) & 0xffffu;
        v[e] = kept(v[e], f >= d.threshold, d.scale);
      }
      __builtin_memcpy(out + i, v, sizeof(v));
    } else {
      for (int e = 0; e < V && i + e < total; ++e) {
        const int j = (int)((i + e) >> col_bits) & 7;
        const uint32_t f = (uint32_t)((j < 4 ? lo : hi) >> ((j & 3) * 16)) & 0xffffu;
        out[i + e] = kept(x[i + e], f >= d.threshold, d.scale);
      }
    }
  }
}

// Rows of any columns and strides, eight elements of a row a thread, 1 << tx_bits threads
// along a row.  By element the eights are the generator's blocks, so a row may begin and end
// within one, which two rows then make.
template <typename T, bool BY_ROW>
__global__ __launch_bounds__(THREADS) void k_dropout_rows(const T* x, int64_t ldx, int64_t rows, int64_t cols,
                                                          int tx_bits, Dropout d, T* out, int64_t ldo) {
  const int tx = threadIdx.x & ((1 << tx_bits) - 1), ty = threadIdx.x >> tx_bits;
  const int64_t row_step = (int64_t)gridDim.y * (THREADS >> tx_bits), col_step = ((int64_t)gridDim.x << tx_bits) * 8;
  for (int64_t n = blockIdx.y * (int64_t)(THREADS >> tx_bits) + ty; n < rows; n += row_step) {
    const int64_t unit0 = BY_ROW ? 0 : n * cols;
    const T* const from = x + n * ldx;
    T* const to = out + n * ldo;
    const uint4 whole = BY_ROW ? philox((uint64_t)n >> 3, d.offset, d.seed) : make_uint4(0, 0, 0, 0);
    const bool keep = field_of(whole, (int)(n & 7)) >= d.threshold;
    // the column of an eight's first element, which may lie before the row
    for (int64_t c = ((((int64_t)blockIdx.x << tx_bits) + tx) * 8) - (unit0 & 7); c < cols; c += col_step) {
      const uint4 r = BY_ROW ? whole : philox((uint64_t)(unit0 + c) >> 3, d.offset, d.seed);
      if (c >= 0 && c + 8 <= cols) {
        T v[8];
        __builtin_memcpy(v, from + c, sizeof(v));
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = kept(v[j], BY_ROW ? keep : field_of(r, j) >= d.threshold, d.scale);
        __builtin_memcpy(to + c, v, sizeof(v));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j >= 0 && c + j < cols)
            to[c + j] = kept(from[c + j], BY_ROW ? keep : field_of(r, j) >= d.threshold, d.scale);
      }
    }
  }
}

unsigned grid_of(int64_t threads) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + THREADS - 1) / THREADS, 1 << 20));
}

template <typename T>
void launch(const void* x, int64_t ldx, int64_t rows, int64_t cols, const Dropout& d, int by_row,
            void* out, int64_t ldo, hipStream_t s) {
  const bool flat = ldx == cols && ldo == cols;
  constexpr int V = 16 / sizeof(T);
  if (flat && !by_row) {
    k_dropout_flat<T><<<grid_of((rows * cols + 7) / 8), THREADS, 0, s>>>((const T*)x, rows * cols, d, (T*)out);
    return;
  }
  if (flat && (cols == 1 || cols == 2 || cols == 4)) {
    k_dropout_pairs<T><<<grid_of((rows * cols + V - 1) / V), THREADS, 0, s>>>((const T*)x, rows * cols,
                                                                              (int)cols / 2, d, (T*)out);
    return;
  }
  // eights that a row reaches over
  const int64_t eights = by_row || cols % 8 == 0 ? (cols + 7) / 8 : (cols + 14) / 8;
  int bits = 0;
  while (bits < 8 && ((int64_t)1 << bits) < eights) ++bits;
  const int64_t across = (eights + (1 << bits) - 1) >> bits, down = (rows + (THREADS >> bits) - 1) / (THREADS >> bits);
  const dim3 grid((unsigned)std::min<int64_t>(across, 1 << 20), (unsigned)std::min<int64_t>(down, 65535));
  if (by_row)
    k_dropout_rows<T, true><<<grid, THREADS, 0, s>>>((const T*)x, ldx, rows, cols, bits, d, (T*)out, ldo);
  else
    k_dropout_rows<T, false><<<grid, THREADS, 0, s>>>((const T*)x, ldx, rows, cols, bits, d, (T*)out, ldo);
}

}  // namespace

void launch_dropout(const void* x, int64_t ldx, int64_t rows, int64_t cols, int32_t dtype,
                    uint32_t threshold, uint64_t seed, uint64_t offset, int by_row, void* out,
                    int64_t ldo, hipStream_t s) {
  // threshold 65536 keeps nothing: the scale is then of no effect
  const float scale = threshold < 65536 ? (float)(65536.0 / (65536.0 - (double)threshold)) : 0.0f;
  const Dropout d{threshold, scale, seed, offset};
  if (dtype == LGBM_HIP_DTYPE_F32)
    launch<float>(x, ldx, rows, cols, d, by_row, out, ldo, s);
  else if (dtype == LGBM_HIP_DTYPE_BF16)
    launch<__bf16>(x, ldx, rows, cols, d, by_row, out, ldo, s);
  else
    launch<_Float16>(x, ldx, rows, cols, d, by_row, out, ldo, s);
}

}  // namespace lgbm
