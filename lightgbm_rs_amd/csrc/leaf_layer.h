// leaf_layer.h — what the kernels of the leaves' layers share: activations and their slopes,
// and the end of a layer, from a map's sums to what is stored.
#pragma once

#include "leaf_mma.h"

namespace lgbm {
namespace mma {

// exp, 1 / v and erf: the library's in float32.  Where results are rounded to 16 bits the
// instructions' own (an ulp or two), and erf by Abramowitz and Stegun, "Handbook of
// Mathematical Functions", 7.1.26, which is off by 1.5e-7 at most.
template <typename T>
__device__ __forceinline__ float exp_of(float v) {
  if constexpr (sizeof(T) == 4) return expf(v);
  return __builtin_amdgcn_exp2f(v * 1.44269504f);
}
template <typename T>
__device__ __forceinline__ float inverse(float v) {
  if constexpr (sizeof(T) == 4) return 1.0f / v;
  return __builtin_amdgcn_rcpf(v);
}
template <typename T>
__device__ __forceinline__ float erf_of(float v) {
  if constexpr (sizeof(T) == 4) return erff(v);
  const float a = fabsf(v), t = inverse<T>(1.0f + 0.3275911f * a);
  float s = 1.061405429f;
  s = fmaf(s, t, -1.453152027f);
  s = fmaf(s, t, 1.421413741f);
  s = fmaf(s, t, -0.284496736f);
  s = fmaf(s, t, 0.254829592f);
  return copysignf(1.0f - s * t * exp_of<T>(-a * a), v);
}

constexpr float SQRT_HALF = 0.70710678f, TANH_SCALE = 0.79788456f, TANH_CUBE = 0.044715f;

template <typename T>
__device__ __forceinline__ float sigmoid_of(float z) {
  return inverse<T>(1.0f + exp_of<T>(-z));
}

// N values of an activation.
template <typename T, int N>
__device__ __forceinline__ void activate(int act, const float (&z)[N], float (&f)[N]) {
  switch (act) {
    case LGBM_HIP_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = z[i] < 0.0f ? 0.0f : z[i];  // a NaN stays
      return;
    case LGBM_HIP_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = z[i] * sigmoid_of<T>(z[i]);
      return;
    case LGBM_HIP_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = 0.5f * z[i] * (1.0f + erf_of<T>(z[i] * SQRT_HALF));
      return;
    case LGBM_HIP_ACT_GELU_TANH:  // (1 + tanh u) / 2 = sigmoid(2 u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = 2.0f * TANH_SCALE * (z[i] + TANH_CUBE * z[i] * z[i] * z[i]);
        f[i] = z[i] * sigmoid_of<T>(u);
      }
      return;
    case LGBM_HIP_ACT_SIGMOID:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = sigmoid_of<T>(z[i]);
      return;
    default:
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = z[i];
  }
}

// The activation f and its slope d at z.  Slopes are constant long before |z| = 10000, and a z
// that its type holds as an infinity has that slope too, not infinity times zero.
template <typename T>
__device__ __forceinline__ void slope_of(int act, float z, float& f, float& d) {
  const float c = z > 1e4f ? 1e4f : (z < -1e4f ? -1e4f : z);  // a NaN stays
  const float g = z < 0.0f ? c : z;
  switch (act) {
    case LGBM_HIP_ACT_RELU:
      f = z < 0.0f ? 0.0f : z;
      d = z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
      return;
    case LGBM_HIP_ACT_SILU: {
      const float p = sigmoid_of<T>(c);
      f = g * p;
      d = p * (1.0f + c * (1.0f - p));
      return;
    }
    case LGBM_HIP_ACT_GELU: {
      const float half = 0.5f * (1.0f + erf_of<T>(c * SQRT_HALF));
      f = g * half;
      d = half + c * exp_of<T>(-0.5f * c * c) * 0.39894228f;
      return;
    }
    case LGBM_HIP_ACT_GELU_TANH: {
      const float p = sigmoid_of<T>(2.0f * TANH_SCALE * (c + TANH_CUBE * c * c * c));
      f = g * p;
      d = p + c * 2.0f * p * (1.0f - p) * TANH_SCALE * (1.0f + 3.0f * TANH_CUBE * c * c);
      return;
    }
    case LGBM_HIP_ACT_SIGMOID:
      f = sigmoid_of<T>(c);
      d = f * (1.0f - f);
      return;
    default:
      f = z;
      d = 1.0f;
  }
}

// `valid` of eight elements from p on, zeros behind them, as float32; and back.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int valid, float (&v)[8]) {
  T e[8];
  if (valid >= 8) {
    __builtin_memcpy(e, p, sizeof(e));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j < valid ? p[j] : (T)0.0f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)e[j];
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int valid, const float (&v)[8]) {
  T e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = (T)v[j];
  if (valid >= 8) {
    __builtin_memcpy(p, e, sizeof(e));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) p[j] = e[j];
  }
}

// Eight neighbouring results of row n (-1: none) of a layer, from column col on: a is the map's
// sums (where gated the gates') and u the second half's.  leaf < 0: the row is in no leaf,
// nothing is added to it and its z is 0.
template <typename T, bool GATED>
__device__ __forceinline__ void layer_end(const LeafProduct& p, int tree, int64_t leaf, int n, int col, float (&a)[8],
                                          float (&u)[8]) {
  const int cols = p.outputs, valid = min(8, cols - col);
  if (n < 0 || valid <= 0) return;
  const int64_t rows = GATED ? 2 * (int64_t)cols : cols;
  if (p.b && leaf >= 0) {
    const T* const b = (const T*)p.b + leaf * rows + col;
    float v[8];
    load8(b, valid, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] += v[j];
    if (GATED) {
      load8(b + cols, valid, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] += v[j];
    }
  }
  if (p.z) {
    const int64_t at = n * rows + col;
    if (sizeof(T) == 2 && p.z_narrow) {
      T* const z = (T*)p.z_of<T>(tree) + at;
      store8(z, valid, a);
      if (GATED) store8(z + cols, valid, u);
    } else {
      float* const z = (float*)p.z_of<T>(tree) + at;
      store8(z, valid, a);
      if (GATED) store8(z + cols, valid, u);
    }
  }
  float f[8];
  activate<T>(p.act, a, f);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (GATED) f[j] *= u[j];
    if (leaf < 0) f[j] = 0.0f;
  }
  if (p.planes) {
    store8((float*)p.ws + ((int64_t)tree * p.g.rows + n) * cols + col, valid, f);
    return;
  }
  if (p.res) {
    float r[8];
    load8((const T*)p.res + (int64_t)n * p.ldr + col, valid, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] += r[j];
  }
  store8((T*)p.out + (int64_t)n * p.ldo + col, valid, f);
}

// The row of a leaf's map that column r of a tile holds, whose waves hold WN columns each: where
// gated the first half of a wave's columns are gates, the second half the same results' other
// factors.  c0: the tile's first result.  Rows behind the last are the last.
template <bool GATED, int WN>
__device__ __forceinline__ int map_row(int r, int c0, int cols) {
  if (!GATED) return min(c0 + r, cols - 1);
  const int in = r % WN, col = min(c0 + r / WN * (WN / 2) + in % (WN / 2), cols - 1);
  return in < WN / 2 ? col : cols + col;
}

}  // namespace mma
}  // namespace lgbm
