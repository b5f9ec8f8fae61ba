// dropout.hip — elements or whole rows dropped by a counter-based generator.  The mask is a
// function of (seed, offset, unit) and is never stored: the gradient is the same call on
// the outputs' gradient.
//
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2,
// 3", 2011): counter (block, offset), key seed.  A block's 128 bits give eight 16-bit
// fields, so the ten rounds are shared by eight units; unit e is kept where field e % 8 of
// block e / 8 is at least threshold = round(65536 p), and what is kept is divided by the
// share that is really kept, 1 - threshold / 65536.
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

// A block of eight units a thread.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_dropout(const T* x, int64_t ldx, int64_t rows, int64_t cols,
                                                     uint32_t threshold, float scale, uint64_t seed,
                                                     uint64_t offset, int by_row, T* out, int64_t ldo) {
  const int64_t units = by_row ? rows : rows * cols;
  const int64_t blocks = (units + 7) / 8;
  for (int64_t b = blockIdx.x * (int64_t)THREADS + threadIdx.x; b < blocks;
       b += (int64_t)gridDim.x * THREADS) {
    const uint4 r = philox((uint64_t)b, offset, seed);
    for (int j = 0; j < 8; ++j) {
      const int64_t e = b * 8 + j;
      if (e >= units) break;
      const bool keep = field_of(r, j) >= threshold;
      if (by_row) {
        for (int64_t c = 0; c < cols; ++c)
          out[e * ldo + c] = keep ? (T)((float)x[e * ldx + c] * scale) : (T)0.0f;
      } else {
        const int64_t n = e / cols, c = e % cols;
        out[n * ldo + c] = keep ? (T)((float)x[n * ldx + c] * scale) : (T)0.0f;
      }
    }
  }
}

template <typename T>
void launch(const void* x, int64_t ldx, int64_t rows, int64_t cols, uint32_t threshold, uint64_t seed,
            uint64_t offset, int by_row, void* out, int64_t ldo, hipStream_t s) {
  const int64_t blocks = ((by_row ? rows : rows * cols) + 7) / 8;
  const unsigned grid = (unsigned)std::min<int64_t>((blocks + THREADS - 1) / THREADS, 65536);
  // threshold 65536 keeps nothing: the scale is then of no effect
  const float scale = threshold < 65536 ? (float)(65536.0 / (65536.0 - (double)threshold)) : 0.0f;
  k_dropout<T><<<grid, THREADS, 0, s>>>((const T*)x, ldx, rows, cols, threshold, scale, seed, offset,
                                        by_row, (T*)out, ldo);
}

}  // namespace

void launch_dropout(const void* x, int64_t ldx, int64_t rows, int64_t cols, int32_t dtype,
                    uint32_t threshold, uint64_t seed, uint64_t offset, int by_row, void* out,
                    int64_t ldo, hipStream_t s) {
  if (dtype == LGBM_HIP_DTYPE_F32)
    launch<float>(x, ldx, rows, cols, threshold, seed, offset, by_row, out, ldo, s);
  else if (dtype == LGBM_HIP_DTYPE_BF16)
    launch<__bf16>(x, ldx, rows, cols, threshold, seed, offset, by_row, out, ldo, s);
  else
    launch<_Float16>(x, ldx, rows, cols, threshold, seed, offset, by_row, out, ldo, s);
}

}  // namespace lgbm
