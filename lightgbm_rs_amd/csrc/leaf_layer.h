// leaf_layer.h — what the kernels of the leaves' layers share: activations and their slopes,
// and the end of a layer, from a map's sums to what is stored.
#pragma once

#include "leaf_mma.h"

namespace lgbm {
namespace mma {

// exp, 1 / v and the normal distribution below z: the library's in float32.  Where results are
// rounded to 16 bits the instructions' own (an ulp or two), and a polynomial.
constexpr float SQRT_HALF = 0.70710678f, TANH_SCALE = 0.79788456f, TANH_CUBE = 0.044715f, LOG2_E = 1.44269504f;
template <typename T>
__device__ __forceinline__ float exp_of(float v) {
  if constexpr (sizeof(T) == 4) return expf(v);
  return __builtin_amdgcn_exp2f(v * LOG2_E);
}
template <typename T>
__device__ __forceinline__ float inverse(float v) {
  if constexpr (sizeof(T) == 4) return 1.0f / v;
  return __builtin_amdgcn_rcpf(v);
}
// erfc(-z / sqrt 2) / 2, which keeps its digits where z is far below zero (1 + erf has none left
// there).  The polynomial: exp(a^2) erfc(a) / 2 by powers of t = 1 / (1 + 0.36 a), fitted by linear
// programming over 0 <= a <= 9.5 so that erfc is off by 4e-8 and by 5e-6 of itself at most, as far
// as float32 reaches (in float32 arithmetic 3.4e-7 and 1.1e-5).
constexpr float BELOW_RATE = 0.36f;
constexpr float BELOW[7] = {0.101116134f,  0.108133462f, 0.0546303386f, 0.212387595f,
                            -0.175420932f, 0.280600975f, -0.0814475543f};
template <typename T>
__device__ __forceinline__ float normal_below(float z) {
  if constexpr (sizeof(T) == 4) return 0.5f * erfcf(z * -SQRT_HALF);
  const float t = inverse<T>(fmaf(BELOW_RATE * SQRT_HALF, fabsf(z), 1.0f));
  float s = BELOW[6];
#pragma unroll
  for (int k = 5; k >= 0; --k) s = fmaf(s, t, BELOW[k]);
  s = s * t * exp_of<T>(-0.5f * z * z);
  return z < 0.0f ? s : 1.0f - s;
}

// The sigmoid of z c, c a constant; in 16 bits the exponential's base goes into c.
template <typename T>
__device__ __forceinline__ float sigmoid_of(float z, float c = 1.0f) {
  if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-(z * c)));
  return inverse<T>(1.0f + __builtin_amdgcn_exp2f(z * (c * -LOG2_E)));
}

// Activations by the code that makes them.
enum ActClass { ACT_LINE, ACT_SIGMOID, ACT_CUBIC, ACT_ERF };
__host__ __device__ inline ActClass act_class(int act) {
  if (act <= LGBM_HIP_ACT_RELU) return ACT_LINE;
  return act == LGBM_HIP_ACT_GELU ? ACT_ERF : act == LGBM_HIP_ACT_GELU_TANH ? ACT_CUBIC : ACT_SIGMOID;
}

// N values of an activation.  GELU_TANH: (1 + tanh v) / 2 = sigmoid(2 v).
template <typename T, ActClass CLASS, int N>
__device__ __forceinline__ void activate_as(int act, const float (&z)[N], float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (CLASS == ACT_LINE) {
      f[i] = act == LGBM_HIP_ACT_RELU && z[i] < 0.0f ? 0.0f : z[i];  // a NaN stays
    } else if (CLASS == ACT_ERF) {
      f[i] = z[i] * normal_below<T>(z[i]);
    } else if (CLASS == ACT_CUBIC) {
      f[i] = z[i] * sigmoid_of<T>(z[i] * fmaf(TANH_CUBE, z[i] * z[i], 1.0f), 2.0f * TANH_SCALE);
    } else {
      const float p = sigmoid_of<T>(z[i]);
      f[i] = act == LGBM_HIP_ACT_SIGMOID ? p : z[i] * p;
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void activate(int act, const float (&z)[N], float (&f)[N]) {
  switch (act_class(act)) {
    case ACT_LINE: return activate_as<T, ACT_LINE>(act, z, f);
    case ACT_ERF: return activate_as<T, ACT_ERF>(act, z, f);
    case ACT_CUBIC: return activate_as<T, ACT_CUBIC>(act, z, f);
    default: activate_as<T, ACT_SIGMOID>(act, z, f);
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
      const float p = normal_below<T>(c);
      f = g * p;
      d = p + c * exp_of<T>(-0.5f * c * c) * 0.39894228f;
      return;
    }
    case LGBM_HIP_ACT_GELU_TANH: {
      const float p = sigmoid_of<T>(2.0f * TANH_SCALE * (c + TANH_CUBE * c * c * c));
      f = g * p;
      d = p + c * 2.0f * p * (1.0f - p) * TANH_SCALE * (1.0f + 3.0f * TANH_CUBE * c * c);
      return;
    }
    case LGBM_HIP_ACT_SIGMOID: {
      // 1 - f has no digits left where f is near one, e / (1 + e)^2 keeps them
      const float e = exp_of<T>(-fabsf(c)), r = inverse<T>(1.0f + e);
      f = c >= 0.0f ? r : e * r;
      d = e * r * r;
      return;
    }
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

// Eight neighbouring results of row n (-1: none) of a layer, from column col on: a is z (where
// gated the gates') and u its second half, r what the row has already.  lost: the row is in no
// leaf, nothing is added to it.  CLASS: the activation's, where it is known.
template <typename T, bool GATED, int CLASS = -1>
__device__ __forceinline__ void layer_end(const LeafProduct& p, int tree, bool lost, int n, int col,
                                          const float (&a)[8], const float (&u)[8], const float (&r)[8]) {
  const int cols = p.outputs, valid = min(8, cols - col);
  if (n < 0 || valid <= 0) return;
  if (p.z) {
    const int64_t at = n * (GATED ? 2 * (int64_t)cols : cols) + col;
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
  if constexpr (CLASS >= 0)
    activate_as<T, (ActClass)CLASS>(p.act, a, f);
  else
    activate<T>(p.act, a, f);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (GATED) f[j] *= u[j];
    if (lost) f[j] = 0.0f;
    f[j] += r[j];
  }
  if (p.planes)
    store8((float*)p.ws + ((int64_t)tree * p.g.rows + n) * cols + col, valid, f);
  else
    store8((T*)p.out + (int64_t)n * p.ldo + col, valid, f);
}

// Bias of eight neighbouring results of a leaf (-1: none) of the map's half `half`; what row n has
// already in eight columns.  Zeros where there is none.
template <typename T>
__device__ __forceinline__ void bias8(const LeafProduct& p, int64_t leaf, int half, int col, float (&v)[8]) {
  const bool has = p.b && leaf >= 0;
  const T* const b = (const T*)p.b + (has ? leaf * p.map_rows() + half * p.outputs + col : 0);
  load8(b, has ? p.outputs - col : 0, v);
}
template <typename T>
__device__ __forceinline__ void residual8(const LeafProduct& p, int n, int col, float (&v)[8]) {
  const bool has = p.res && !p.planes && n >= 0;
  load8((const T*)p.res + (has ? (int64_t)n * p.ldr + col : 0), has ? p.outputs - col : 0, v);
}

// The same from the map's sums.
template <typename T, bool GATED>
__device__ __forceinline__ void layer_end_of_sums(const LeafProduct& p, int tree, int64_t leaf, int n, int col,
                                                  float (&a)[8], float (&u)[8]) {
  float r[8], b[8];
  residual8<T>(p, n, col, r);
  bias8<T>(p, leaf, 0, col, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] += b[j];
  if (GATED) {
    bias8<T>(p, leaf, 1, col, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] += b[j];
  }
  layer_end<T, GATED>(p, tree, leaf < 0, n, col, a, u, r);
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
