// scores.hip — class scores to answers: penalties for classes that a row was given before,
// a bias for every class, the classes that a row may have, and the softmax of the rest.
//
// s = x[n][j]; where class j stands c > 0 times in the row's history, s = (s > 0 ? s / r :
// s * r) - f c - p; then + bias[j]; -inf (probability 0) where the mask's bit j is not set.
// Sums, maxima and products are float64 for float64 scores and float32 for the others.
#include <algorithm>

#include "leaf_ops.h"

#include "../../include/lgbm_hip.h"

namespace lgbm {
namespace {

constexpr int THREADS = 256;
constexpr int CHUNK = 4096;  // classes whose counts a block holds in LDS at a time

template <typename T>
struct Wide {
  typedef float type;
};
template <>
struct Wide<double> {
  typedef double type;
};

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// Maximum and sum of exponentials joined with another's; a maximum of -inf has sum 0.
template <typename A>
__device__ __forceinline__ void join(A& m, A& s, A m2, A s2) {
  const A top = m > m2 || m != m ? m : m2;  // NaN stays
  const A a = m == -INFINITY ? (A)0 : s * exp_of(m - top);
  const A b = m2 == -INFINITY ? (A)0 : s2 * exp_of(m2 - top);
  m = top;
  s = a + b;
}

// A block a row.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_scores(ScoreArgs a) {
  typedef typename Wide<T>::type A;
  __shared__ uint32_t count[CHUNK];
  __shared__ A tops[THREADS / 64], sums[THREADS / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int V = a.classes, words = (V + 31) / 32;
  for (int64_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
    const T* const x = (const T*)a.x + n * a.ldx;
    T* const out = (T*)a.out + n * a.ldo;
    const uint32_t* mask = nullptr;
    if (a.mask) {
      const int64_t m = a.mask_rows ? a.mask_rows[n] : a.masks == 1 ? 0 : n;
      if (m >= 0 && m < a.masks) mask = a.mask + m * words;
    }
    int64_t h0 = 0, h1 = 0;
    if (a.ids) {
      h0 = min(max(a.offsets[n], (int64_t)0), a.num_ids);
      h1 = min(max(a.offsets[n + 1], h0), a.num_ids);
    }
    A rep = (A)a.repetition, fre = (A)a.frequency, pre = (A)a.presence;
    if (a.penalties) {
      rep = (A)a.penalties[n * 3];
      fre = (A)a.penalties[n * 3 + 1];
      pre = (A)a.penalties[n * 3 + 2];
    }
    A top = -INFINITY, sum = 0;
    auto value = [&](int j, uint32_t c) {
      A s = (A)x[j];
      if (c) s = (s > 0 ? s / rep : s * rep) - fre * (A)c - pre;
      if (a.bias) s += (A)((const T*)a.bias)[j];
      if (mask && !((mask[j >> 5] >> (j & 31)) & 1)) s = -INFINITY;
      return s;
    };
    // kind transformed: the first sweep finds the maximum and the sum, the second writes
    for (int sweep = a.kind == LGBM_HIP_PREDICT_TRANSFORMED ? 0 : 1; sweep < 2; ++sweep) {
      for (int c0 = 0; c0 < V; c0 += CHUNK) {
        if (h1 > h0) {
          __syncthreads();
          for (int j = tid; j < CHUNK; j += THREADS) count[j] = 0;
          __syncthreads();
          for (int64_t h = h0 + tid; h < h1; h += THREADS) {
            const uint32_t j = (uint32_t)a.ids[h] - (uint32_t)c0;
            if (j < (uint32_t)CHUNK) atomicAdd(&count[j], 1u);
          }
          __syncthreads();
        }
        for (int j = tid; j < CHUNK && c0 + j < V; j += THREADS) {
          const A s = value(c0 + j, h1 > h0 ? count[j] : 0);
          if (sweep == 0)
            join(top, sum, s, (A)1);
          else if (a.kind == LGBM_HIP_PREDICT_RAW)
            out[c0 + j] = (T)s;
          else
            out[c0 + j] = (T)(top == -INFINITY ? (A)0 : exp_of(s - top) / sum);
        }
      }
      if (sweep == 0) {
        for (int d = 1; d < 64; d <<= 1) join(top, sum, (A)__shfl_xor(top, d), (A)__shfl_xor(sum, d));
        __syncthreads();
        if (lane == 0) tops[wave] = top, sums[wave] = sum;
        __syncthreads();
        top = -INFINITY, sum = 0;
        for (int w = 0; w < THREADS / 64; ++w) join(top, sum, tops[w], sums[w]);
      }
    }
  }
}

template <typename T>
void launch(const ScoreArgs& a, hipStream_t s) {
  k_scores<T><<<(unsigned)std::min<int64_t>(a.rows, 65536), THREADS, 0, s>>>(a);
}

}  // namespace

size_t adjust_scores_workspace(int64_t rows, int32_t classes, int32_t dtype, int32_t kind) { return 0; }

void launch_adjust_scores(const ScoreArgs& a, hipStream_t s) {
  if (a.dtype == LGBM_HIP_DTYPE_F64)
    launch<double>(a, s);
  else if (a.dtype == LGBM_HIP_DTYPE_F32)
    launch<float>(a, s);
  else if (a.dtype == LGBM_HIP_DTYPE_BF16)
    launch<__bf16>(a, s);
  else
    launch<_Float16>(a, s);
}

}  // namespace lgbm
