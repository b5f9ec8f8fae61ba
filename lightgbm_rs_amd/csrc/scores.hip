// scores.hip — class scores to answers: penalties for classes that a row was given before,
// a bias for every class, the classes that a row may have, and the softmax of the rest.
//
// s = x[n][j]; where class j stands c > 0 times in the row's history, s = (s > 0 ? s / r :
// s * r) - f c - p; then + bias[j]; -inf (probability 0) where the mask's bit j is not set.
// Sums, maxima and products are float64 for float64 scores and float32 for the others;
// what a row's sum is made of is added in a fixed order.
//
// Bound by memory: a pass reads and writes every score once.  Three forms, by how many
// classes a row has:
//  - up to 32: a row a thread (k_scores_thread): the rows of a block pass through LDS, so
//    that global accesses are contiguous, and no lane waits for another's maximum;
//  - up to 8192: the row in registers of a wave or a block (k_scores_row), read once;
//  - more: chunks of a row, each in a block's registers.  For probabilities the chunks'
//    maxima and sums are written first (PART) and every chunk is read again to be
//    written (FINISH); its second read mostly hits the caches.
// 2M x 10 float64 to probabilities 94 us (3.5 TB/s); 64 x 128007 bfloat16 with histories of 1000 ids
// 37 us, most of it the latency of two launches.
// Counts of a row's history are whole numbers in LDS; a chunk looks at the whole history
// and counts its own classes.
#include <algorithm>

#include "leaf_ops.h"

#include "../../include/lgbm_hip.h"

namespace lgbm {
namespace {

constexpr int THREADS = 256;
constexpr int THREAD_CLASSES = 32;
constexpr int NARROW_CLASSES = 256, WAVE_CLASSES = 512, BLOCK_CLASSES = 2048, ROW_CLASSES = 8192;

template <typename T>
struct Wide {
  typedef float type;
};
template <>
struct Wide<double> {
  typedef double type;
};

// e^v.  For 16-bit results the hardware's 2^x is enough: the product with log2(e) is off by
// |v| 2^-24, far below their rounding wherever e^v is not 0 beside the row's largest.
template <typename T>
__device__ __forceinline__ float exp_of(float v) {
  return sizeof(T) == 2 ? __builtin_amdgcn_exp2f(v * 1.44269504f) : expf(v);
}
template <typename T>
__device__ __forceinline__ double exp_of(double v) {
  return exp(v);
}
// The larger.  A NaN that is one of them comes through in float32, which has an instruction
// for it; in float64 it is passed over, and found by is_nan beside the maximum.
__device__ __forceinline__ float top_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ double top_of(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ bool is_nan(float) { return false; }
__device__ __forceinline__ bool is_nan(double a) { return a != a; }
// s, or -inf where bit e is set.
__device__ __forceinline__ float unless(uint32_t bits, int e, float s) {
  const uint32_t m = (uint32_t)((int32_t)(bits << (31 - e)) >> 31);
  return __uint_as_float((m & 0xff800000u) | (~m & __float_as_uint(s)));
}
__device__ __forceinline__ double unless(uint32_t bits, int e, double s) {
  return (bits >> e) & 1 ? -INFINITY : s;
}
// What the exponentials are relative to.  Where every class is masked their -inf stays; in a
// row of a NaN no exponential but a masked class's may be 0, so that the NaN of their sum
// reaches the others.
template <typename A>
__device__ __forceinline__ A base_of(A top) {
  const A lowest = sizeof(A) == 8 ? (A)-__DBL_MAX__ : (A)-__FLT_MAX__;
  return top == -INFINITY ? (A)0 : top != top ? lowest : top;
}

// What a row's scores are adjusted by.
template <typename A>
struct Row {
  const uint32_t* mask;  // null: every class is allowed
  int64_t h0, h1;        // its history
  A rep, fre, pre;
};

template <typename A>
__device__ __forceinline__ Row<A> row_of(const ScoreArgs& a, int64_t n) {
  Row<A> r{nullptr, 0, 0, (A)a.repetition, (A)a.frequency, (A)a.presence};
  if (a.mask) {
    const int64_t m = a.mask_rows ? a.mask_rows[n] : a.masks == 1 ? 0 : n;
    if (m >= 0 && m < a.masks) r.mask = a.mask + m * ((a.classes + 31) / 32);
  }
  if (a.ids) {
    r.h0 = min(max(a.offsets[n], (int64_t)0), a.num_ids);
    r.h1 = min(max(a.offsets[n + 1], r.h0), a.num_ids);
    if (a.penalties) {
      r.rep = (A)a.penalties[n * 3];
      r.fre = (A)a.penalties[n * 3 + 1];
      r.pre = (A)a.penalties[n * 3 + 2];
    }
  }
  return r;
}

template <typename A>
__device__ __forceinline__ A adjusted(A s, uint32_t count, const Row<A>& r, A bias, bool allowed) {
  if (count) s = (s > 0 ? s / r.rep : s * r.rep) - r.fre * (A)count - r.pre;
  s += bias;
  return allowed ? s : -INFINITY;
}

// ---- a row a thread ------------------------------------------------------------------------

// LDS: [THREADS][classes | 1] values (odd strides: a wave's rows in different banks), and
// as many counts where there is a history.  FLAT: the rows of x and of out follow each
// other without gaps, so a block's are copied as vectors of 16 bytes.
template <typename T, bool FLAT>
__global__ __launch_bounds__(THREADS) void k_scores_thread(ScoreArgs a, uint32_t inverse) {
  typedef typename Wide<T>::type A;
  constexpr int VE = FLAT ? 16 / (int)sizeof(T) : 1;
  extern __shared__ __align__(16) char lds[];
  const int V = a.classes, stride = V | 1, tid = threadIdx.x;
  A* const values = (A*)lds;
  uint32_t* const counts = (uint32_t*)(values + THREADS * stride) + tid * stride;
  A* const mine = values + tid * stride;
  const T* const bias = (const T*)a.bias;
  auto at = [&](int i) {  // element i of the block's rows in LDS
    const int r = (int)((uint32_t)i * inverse >> 19);
    return r * stride + (i - r * V);
  };
  for (int64_t n0 = blockIdx.x * (int64_t)THREADS; n0 < a.rows; n0 += (int64_t)gridDim.x * THREADS) {
    const int rows = (int)min((int64_t)THREADS, a.rows - n0), total = rows * V;
    const T* const x = (const T*)a.x + n0 * a.ldx;
    T* const out = (T*)a.out + n0 * a.ldo;
#pragma unroll 4
    for (int i = tid * VE; i + VE <= total; i += THREADS * VE) {
      T v[VE];
      if (FLAT) {
        __builtin_memcpy(v, x + i, sizeof(v));
      } else {
        const int r = (int)((uint32_t)i * inverse >> 19);
        v[0] = x[r * a.ldx + (i - r * V)];
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) values[at(i + e)] = (A)v[e];
    }
    const int tail = total - total % VE + tid;
    if (tail < total) values[at(tail)] = (A)x[tail];  // FLAT only
    __syncthreads();
    if (tid < rows) {
      const Row<A> row = row_of<A>(a, n0 + tid);
      const uint32_t allowed = row.mask ? row.mask[0] : ~0u;
      if (a.ids) {
        for (int j = 0; j < V; ++j) counts[j] = 0;
        for (int64_t h = row.h0; h < row.h1; ++h) {
          const uint32_t j = (uint32_t)a.ids[h];
          if (j < (uint32_t)V) ++counts[j];
        }
      }
      A top = -INFINITY;
      bool nan = false;
      for (int j = 0; j < V; ++j) {
        const A s = adjusted(mine[j], a.ids ? counts[j] : 0, row, bias ? (A)bias[j] : (A)0,
                             (allowed >> j) & 1);
        mine[j] = s;
        top = top_of(top, s);
        nan |= is_nan(s);
      }
      if (a.kind == LGBM_HIP_PREDICT_TRANSFORMED) {
        const A base = base_of(nan ? (A)NAN : top);
        A sum = 0;
        for (int j = 0; j < V; ++j) {
          const A e = exp_of<T>(mine[j] - base);
          mine[j] = e;
          sum += e;
        }
        const A scale = 1 / sum;
        for (int j = 0; j < V; ++j) mine[j] = mine[j] == 0 ? (A)0 : mine[j] * scale;
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int i = tid * VE; i + VE <= total; i += THREADS * VE) {
      T v[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = (T)values[at(i + e)];
      if (FLAT) {
        __builtin_memcpy(out + i, v, sizeof(v));
      } else {
        const int r = (int)((uint32_t)i * inverse >> 19);
        out[r * a.ldo + (i - r * V)] = v[0];
      }
    }
    if (tail < total) out[tail] = (T)values[at(tail)];
    __syncthreads();
  }
}

// ---- a row, or a chunk of one, in registers ----------------------------------------------------

enum { WHOLE, PART, FINISH };

// Long rows: chunks of 32 bytes a lane.
constexpr int CHUNK_BYTES = 32;

// LANES of one row, each with NV vectors of VW neighbouring classes, LANES * NV * VW classes
// from c0 on.  float64's FINISH is held to the registers of five waves a SIMD (200 x 60000 75
// us, by the 101 registers that the compiler takes else 79).
template <typename T, int LANES, int NV, int VW, int MODE>
__global__ __launch_bounds__(LANES < THREADS ? THREADS : LANES,
                             MODE == FINISH && sizeof(T) == 8 && LANES <= 512 ? 5 : 1) void k_scores_row(ScoreArgs a, int chunks) {
  typedef typename Wide<T>::type A;
  constexpr int CAP = LANES * NV * VW, TEAMS = LANES < THREADS ? THREADS / LANES : 1;
  __shared__ __align__(16) uint32_t counts[TEAMS * CAP];
  __shared__ A shared[LANES / 64], sums[LANES / 64];
  const int lane = threadIdx.x % LANES, team = threadIdx.x / LANES;
  uint32_t* const count = counts + team * CAP;
  auto sync = [&] {
    if (LANES == 64) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  // over the row's lanes; every one gets the result
  auto of_wave = [&](A v, auto join) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = join(v, (A)__shfl_xor(v, d));
    return v;
  };
  // v: already of the wave
  auto of_block = [&](A v, auto join) {
    if (LANES > 64) {
      __syncthreads();
      if (lane % 64 == 0) shared[lane / 64] = v;
      __syncthreads();
      v = shared[0];
#pragma unroll
      for (int w = 1; w < LANES / 64; ++w) v = join(v, shared[w]);
    }
    return v;
  };
  const auto plus = [](A p, A q) { return p + q; };
  const auto larger = [](A p, A q) { return top_of(p, q); };
  // the maximum over a wave, NaN where a lane's `nan` is set
  auto top_of_wave = [&](A v, bool nan) {
    v = of_wave(v, larger);
    return __any(nan) ? (A)NAN : v;
  };
  const int64_t tasks = a.rows * chunks;
  for (int64_t task = blockIdx.x * (int64_t)TEAMS + team; task < tasks;
       task += (int64_t)gridDim.x * TEAMS) {
    const int64_t n = task / chunks;
    const int c0 = (int)(task - n * chunks) * CAP;
    const int V = min(a.classes - c0, CAP);
    const T* const x = (const T*)a.x + n * a.ldx + c0;
    const T* const bias = a.bias ? (const T*)a.bias + c0 : nullptr;
    A s[NV][VW];
    T v[NV][VW], b[NV][VW];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * LANES + lane) * VW;
      const bool full = j + VW <= V;
      if (full)
        __builtin_memcpy(v[i], x + j, sizeof(v[i]));
      else
#pragma unroll
        for (int e = 0; e < VW; ++e) v[i][e] = j + e < V ? x[j + e] : (T)0.0f;
      if (bias && full)
        __builtin_memcpy(b[i], bias + j, sizeof(b[i]));
      else
#pragma unroll
        for (int e = 0; e < VW; ++e) b[i][e] = bias && j + e < V ? bias[j + e] : (T)0.0f;
    }
    const Row<A> row = row_of<A>(a, n);
    const bool seen = row.h1 > row.h0;
    const bool masked = row.mask || V < CAP;  // else every class is allowed
    uint32_t refused[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * LANES + lane) * VW;
      // VW divides 32 and c0 is a multiple of 32, so the bits are of one word
      refused[i] = row.mask && j < V ? ~(row.mask[(c0 + j) >> 5] >> (j & 31)) : 0u;
      if (j + VW > V) refused[i] |= j < V ? ~0u << (V - j) : ~0u;
    }
    if (seen) {
#pragma unroll
      for (int i = 0; i < NV; ++i) __builtin_memset(count + (i * LANES + lane) * VW, 0, 4 * VW);
      sync();
#pragma unroll 4
      for (int64_t h = row.h0 + lane; h < row.h1; h += LANES) {
        const uint32_t j = (uint32_t)a.ids[h] - (uint32_t)c0;
        if (j < (uint32_t)V) atomicAdd(&count[j], 1u);
      }
      sync();
    }
    A top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * LANES + lane) * VW;
#pragma unroll
      for (int e = 0; e < VW; ++e) s[i][e] = (A)v[i][e];
      if (seen) {
        uint32_t c[VW], any = 0;
        __builtin_memcpy(c, count + j, sizeof(c));  // behind V: zeros
#pragma unroll
        for (int e = 0; e < VW; ++e) any |= c[e];
        if (any) {
#pragma unroll
          for (int e = 0; e < VW; ++e)
            if (c[e]) s[i][e] = (s[i][e] > 0 ? s[i][e] / row.rep : s[i][e] * row.rep) - row.fre * (A)c[e] - row.pre;
        }
      }
#pragma unroll
      for (int e = 0; e < VW; ++e) s[i][e] += (A)b[i][e];
      if (masked)
#pragma unroll
        for (int e = 0; e < VW; ++e) s[i][e] = unless(refused[i], e, s[i][e]);
#pragma unroll
      for (int e = 0; e < VW; ++e) top = top_of(top, s[i][e]), nan |= is_nan(s[i][e]);
    }
    if (seen) sync();  // the counts are read before the next row's are cleared
    A scale = 1;
    const bool probabilities = a.kind == LGBM_HIP_PREDICT_TRANSFORMED;
    if (probabilities) {
      A* const parts = (A*)a.ws;  // [rows][chunks]: maximum (NaN: of a NaN), sum
      if (MODE == FINISH) {  // each wave for itself
        top = -INFINITY, nan = false;
        for (int c = lane % 64; c < chunks; c += 64) {
          const A t = parts[(n * chunks + c) * 2];
          top = top_of(top, t), nan |= is_nan(t);
        }
      }
      // a part's waves are joined at its end, in one turn of the block
      top = top_of_wave(top, nan);
      if (MODE == WHOLE && LANES > 64) {
        nan = false;
        top = of_block(top, [&](A p, A q) {
          nan |= is_nan(p) || is_nan(q);
          return top_of(p, q);
        });
        if (nan) top = NAN;
      }
      const A base = base_of(top);
      A sum = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          s[i][e] = exp_of<T>(s[i][e] - base);
          if (MODE != FINISH) sum += s[i][e];
        }
      if (MODE == FINISH) {
        for (int c = lane; c < chunks; c += LANES)
          sum += parts[(n * chunks + c) * 2 + 1] * exp_of<A>(parts[(n * chunks + c) * 2] - base);
      }
      if (MODE == PART) {
        sum = of_wave(sum, plus);
        __syncthreads();
        if (lane % 64 == 0) shared[lane / 64] = top, sums[lane / 64] = sum;
        __syncthreads();
        if (lane < 64) {
          A t = lane < LANES / 64 ? shared[lane] : (A)-INFINITY;
          top = top_of_wave(t, is_nan(t));
          sum = of_wave(lane < LANES / 64 ? sums[lane] * exp_of<A>(t - base_of(top)) : (A)0, plus);
          if (lane == 0) parts[task * 2] = top, parts[task * 2 + 1] = sum;
        }
        continue;
      }
      sum = of_block(of_wave(sum, plus), plus);
      scale = 1 / sum;
    }
    if (!(scale <= 1)) {  // of a NaN or an infinity, or of no class: 0 stays 0 beside it
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VW; ++e) s[i][e] = s[i][e] == 0 ? (A)0 : s[i][e] * scale;
      scale = 1;
    }
    T* const out = (T*)a.out + n * a.ldo + c0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = (i * LANES + lane) * VW;
      T v[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) v[e] = (T)(s[i][e] * scale);
      if (j + VW <= V)
        __builtin_memcpy(out + j, v, sizeof(v));
      else
#pragma unroll
        for (int e = 0; e < VW; ++e)
          if (j + e < V) out[j + e] = v[e];
    }
  }
}

template <typename T, int LANES, int CAP, int VW, int MODE>
void launch_row(const ScoreArgs& a, int chunks, hipStream_t s) {
  constexpr int TEAMS = LANES < THREADS ? THREADS / LANES : 1;
  const int64_t blocks = (a.rows * chunks + TEAMS - 1) / TEAMS;
  k_scores_row<T, LANES, CAP / LANES / VW, VW, MODE>
      <<<(unsigned)std::min<int64_t>(blocks, 1 << 20), TEAMS * LANES, 0, s>>>(a, chunks);
}

// Lanes of a chunk.  Small blocks overlap best (bfloat16 x 128007 without histories: 256 rows
// 90 us by 256 lanes, 97 by 512, 106 by 1024), but every block of a row looks at its whole
// history (1000 ids a row: 134, 136 and 147 us; 64 rows 39, 39 and 37), so where all blocks
// of 1024 fit the card at once those are taken; and 256 lanes where CUs would be without
// work.
int chunk_lanes(int64_t rows, int32_t classes, int e, bool history) {
  const int chunk = 1024 * (CHUNK_BYTES / e);
  const int64_t blocks = rows * ((classes + chunk - 1) / chunk);
  return !history || blocks < 256 ? 256 : blocks <= 512 ? 1024 : 512;
}

template <typename T, int LANES>
void launch_chunks(const ScoreArgs& a, hipStream_t s) {
  constexpr int VW = 16 / sizeof(T), CAP = LANES * (CHUNK_BYTES / (int)sizeof(T));
  const int chunks = (a.classes + CAP - 1) / CAP;
  if (a.kind == LGBM_HIP_PREDICT_RAW) return launch_row<T, LANES, CAP, VW, WHOLE>(a, chunks, s);
  launch_row<T, LANES, CAP, VW, PART>(a, chunks, s);
  launch_row<T, LANES, CAP, VW, FINISH>(a, chunks, s);
}

template <typename T>
void launch(const ScoreArgs& a, hipStream_t s) {
  typedef typename Wide<T>::type A;
  constexpr int VW = 16 / sizeof(T);
  const int V = a.classes;
  if (V <= THREAD_CLASSES) {
    const size_t lds = (size_t)THREADS * (V | 1) * (sizeof(A) + (a.ids ? 4 : 0));
    const int64_t blocks = (a.rows + THREADS - 1) / THREADS;
    const uint32_t inverse = ((1u << 19) + V - 1) / V;  // i / V for i < 256 V: i V < 2^19
    const unsigned grid = (unsigned)std::min<int64_t>(blocks, 1 << 20);
    if (a.ldx == V && a.ldo == V)
      k_scores_thread<T, true><<<grid, THREADS, lds, s>>>(a, inverse);
    else
      k_scores_thread<T, false><<<grid, THREADS, lds, s>>>(a, inverse);
  } else if (V <= NARROW_CLASSES) {
    launch_row<T, 64, NARROW_CLASSES, 1, WHOLE>(a, 1, s);
  } else if (V <= WAVE_CLASSES) {
    launch_row<T, 64, WAVE_CLASSES, VW, WHOLE>(a, 1, s);
  } else if (V <= BLOCK_CLASSES) {
    launch_row<T, THREADS, BLOCK_CLASSES, VW, WHOLE>(a, 1, s);
  } else if (V <= ROW_CLASSES) {
    launch_row<T, 512, ROW_CLASSES, VW, WHOLE>(a, 1, s);
  } else {
    const int lanes = chunk_lanes(a.rows, V, sizeof(T), a.num_ids > 0);
    if (lanes == 256)
      launch_chunks<T, 256>(a, s);
    else if (lanes == 512)
      launch_chunks<T, 512>(a, s);
    else
      launch_chunks<T, 1024>(a, s);
  }
}

}  // namespace

size_t adjust_scores_workspace(int64_t rows, int32_t classes, int32_t dtype, int32_t kind, bool history) {
  if (classes <= ROW_CLASSES || kind == LGBM_HIP_PREDICT_RAW) return 0;
  const int e = dtype == LGBM_HIP_DTYPE_F64 ? 8 : dtype == LGBM_HIP_DTYPE_F32 ? 4 : 2;
  const int chunk = chunk_lanes(rows, classes, e, history) * (CHUNK_BYTES / e);
  return (size_t)rows * (size_t)((classes + chunk - 1) / chunk) * (e == 8 ? 16 : 8);
}

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
