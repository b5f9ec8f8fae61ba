// grad_norm.hip — the 2-norm over all elements of many tensors, and the tensors scaled to a
// largest norm.
//
// norm = sqrt(sum of g^2); out = g * min(1, most / norm).  Squares are added in float64: those of
// float32 gradients reach over twice its exponents' range, and hundreds of millions of terms over
// its digits.  Bound by memory: every element is read once for the norm and once more for its
// scaling, and written once (400M elements, half of them bfloat16, to other tensors: 243 us, 4.9
// TB/s, and 546 us, 4.4 TB/s, of the 4.9 that a copy reaches).
//
// The tensors' pointers go to the kernels by value, LIST of them a launch, so nothing is copied
// to the device and a call can be captured.  A tensor is cut into chunks, a block each, whose
// size follows from the elements of the whole list: a chunk's sum has its place, and the sums are
// added in their order, so that results are the same every time.
#include <algorithm>
#include <cstdint>

#include "leaf_ops.h"

#include "../../include/lgbm_hip.h"

namespace lgbm {
namespace {

constexpr int THREADS = 256, LIST = 128, FINAL = 1024, FEW = 16;

// first[i]: the launch's block that begins tensor i.  count: elements times four, and the type
// (0: float32, 1: bfloat16, 2: float16).
struct List {
  const void* in[LIST];
  void* out[LIST];
  int64_t count[LIST];
  int32_t first[LIST];
  int32_t tensors;
};

struct Chunk {
  int tensor;
  int64_t from, to;
};
__device__ __forceinline__ Chunk chunk_of(const List& l, int block, int64_t chunk) {
  int lo = 0, hi = l.tensors - 1;  // the last tensor that begins at this block or before
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (l.first[mid] <= block)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int64_t from = (block - l.first[lo]) * chunk;
  return {lo, from, min(from + chunk, l.count[lo] >> 2)};
}

template <typename T>
__device__ __forceinline__ double squares(const T* in, int64_t from, int64_t to) {
  constexpr int V = 16 / (int)sizeof(T), UNROLL = 4;
  double sum[2] = {0, 0};
  auto add = [&](const T(&v)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double d = (double)(float)v[j];
      sum[j & 1] = fma(d, d, sum[j & 1]);
    }
  };
  int64_t i = from + threadIdx.x % THREADS * V;
  for (; i + (UNROLL - 1) * (int64_t)THREADS * V + V <= to; i += UNROLL * (int64_t)THREADS * V) {
    T v[UNROLL][V];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) __builtin_memcpy(v[u], in + i + u * THREADS * V, 16);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) add(v[u]);
  }
  for (; i < to; i += (int64_t)THREADS * V) {
    T v[V];
    if (i + V <= to) {
      __builtin_memcpy(v, in + i, 16);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = i + j < to ? in[i + j] : (T)0.0f;
    }
    add(v);
  }
  return sum[0] + sum[1];
}

// The sum over a block of N threads, in the first.
template <int N>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double of_wave[N / 64];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) v += of_wave[w];
  return v;
}

// A thread's part of a chunk's sum.
__device__ __forceinline__ double squares_of(const List& l, int block, int64_t chunk) {
  const Chunk c = chunk_of(l, block, chunk);
  switch (l.count[c.tensor] & 3) {
    case 0: return squares((const float*)l.in[c.tensor], c.from, c.to);
    case 1: return squares((const __bf16*)l.in[c.tensor], c.from, c.to);
    default: return squares((const _Float16*)l.in[c.tensor], c.from, c.to);
  }
}

__global__ __launch_bounds__(THREADS) void k_squares(List l, int64_t chunk, double* sums) {
  const double v = block_sum<THREADS>(squares_of(l, blockIdx.x, chunk));
  if (threadIdx.x == 0) sums[blockIdx.x] = v;
}

// What a gradient is multiplied by: first by one factor, then by the other.  The second is 1 unless
// the scale is below float32's normal numbers, where a single factor would have few digits or none;
// the product with the first is then in their range wherever that with both is not zero.
struct Scale {
  float first, second;
};

__device__ __forceinline__ void put_norm(double sum, double most, float* norm, Scale* scale) {
  const double v = sqrt(sum);
  *norm = (float)v;
  if (!scale) return;
  // a norm that is NaN gives a scale that is
  const double s = v <= most ? 1.0 : most / v;
  Scale of{(float)s, 1.0f};
  if (s > 0.0 && s < 0x1p-126) {
    int e;
    const double m = frexp(s, &e);  // (a scale below 2^-300 makes zeros of all that float32 holds)
    const int half = max(e, -300) / 2;
    of = {(float)ldexp(m, e - half), ldexpf(1.0f, half)};
  }
  *scale = of;
}

// The norm, and the scale in front of the sums.
__global__ __launch_bounds__(FINAL) void k_norm(const double* sums, int64_t n, double most, float* norm,
                                                Scale* scale) {
  double v = 0;
  for (int64_t i = threadIdx.x; i < n; i += FINAL) v += sums[i];
  v = block_sum<FINAL>(v);
  if (threadIdx.x == 0) put_norm(v, most, norm, scale);
}

// Both for a list of few chunks: one block, whose parts of THREADS take a chunk each.
__global__ __launch_bounds__(FINAL) void k_norm_of_few(List l, int64_t chunk, int chunks, double most, float* norm,
                                                       Scale* scale) {
  double v = 0;
  for (int i = threadIdx.x / THREADS; i < chunks; i += FINAL / THREADS) v += squares_of(l, i, chunk);
  v = block_sum<FINAL>(v);
  if (threadIdx.x == 0) put_norm(v, most, norm, scale);
}

// 16 bytes, as elements of 2 or 4 lie in memory.
typedef unsigned int vec16 __attribute__((ext_vector_type(4), aligned(2)));

// PASS: what is written goes by the caches, and the next kernel finds no lines in them that have
// to be written back first.
template <bool PASS, typename T>
__device__ __forceinline__ void scale_chunk(const T* in, T* out, int64_t from, int64_t to, Scale scale) {
  constexpr int V = 16 / (int)sizeof(T), UNROLL = 4;
  if (scale.first == 1.0f && in == out) return;
  int64_t i = from + threadIdx.x * V;
  for (; i + (UNROLL - 1) * (int64_t)THREADS * V + V <= to; i += UNROLL * (int64_t)THREADS * V) {
    T v[UNROLL][V];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) __builtin_memcpy(v[u], in + i + u * THREADS * V, 16);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[u][j] = (T)((float)v[u][j] * scale.first * scale.second);
      vec16 x;
      __builtin_memcpy(&x, v[u], 16);
      if constexpr (PASS)
        __builtin_nontemporal_store(x, (vec16*)(out + i + u * THREADS * V));
      else
        *(vec16*)(out + i + u * THREADS * V) = x;
    }
  }
  for (; i < to; i += (int64_t)THREADS * V)
    for (int j = 0; j < V && i + j < to; ++j) out[i + j] = (T)((float)in[i + j] * scale.first * scale.second);
}

// The chunks of a launch from the last to the first: what a list of one launch read last is still in
// the caches.  (Lists of more than LIST tensors are several launches, which go forward.)
template <bool PASS>
__global__ __launch_bounds__(THREADS) void k_scale(List l, int64_t chunk, const Scale* scale) {
  const Chunk c = chunk_of(l, gridDim.x - 1 - blockIdx.x, chunk);
  const Scale s = *scale;
  const void* const in = l.in[c.tensor];
  void* const out = l.out[c.tensor];
  switch (l.count[c.tensor] & 3) {
    case 0: scale_chunk<PASS>((const float*)in, (float*)out, c.from, c.to, s); break;
    case 1: scale_chunk<PASS>((const __bf16*)in, (__bf16*)out, c.from, c.to, s); break;
    default: scale_chunk<PASS>((const _Float16*)in, (_Float16*)out, c.from, c.to, s);
  }
}

// Elements a chunk: a list in about 4096 of them, multiples of a float32 turn of a block's vectors.
// In 16 bits a turn is twice that: where chunks are odd multiples, as in all lists of up to 16.8M
// elements, the last half turn of each goes through the loops' ends, which k_scale makes by single
// elements (10M bfloat16: 8.3 and 21.1 us; 10M float32, twice the bytes, 8.7 and 13.5).
int64_t chunk_size(int64_t total) {
  constexpr int64_t TURN = THREADS * 16;
  return std::max<int64_t>(TURN, (total / 4096 + TURN - 1) / TURN * TURN);
}
int64_t chunks_of(const GradTensor& t, int64_t chunk) { return (t.count + chunk - 1) / chunk; }

// Calls `launch` with lists of the tensors that have elements, each list's first chunk and its
// chunks, of which there are 4096 and LIST at most.
template <typename F>
void lists(const GradTensor* t, int64_t num, int64_t chunk, F&& launch) {
  List l;
  l.tensors = 0;
  int64_t done = 0, blocks = 0;
  const auto flush = [&] {
    if (l.tensors) launch(l, done, blocks);
    done += blocks, blocks = 0, l.tensors = 0;
  };
  for (int64_t i = 0; i < num; ++i) {
    if (t[i].count <= 0) continue;
    const int n = l.tensors++;
    l.in[n] = t[i].in, l.out[n] = t[i].out, l.first[n] = (int32_t)blocks;
    l.count[n] = t[i].count * 4 + (t[i].dtype == LGBM_HIP_DTYPE_F32 ? 0 : t[i].dtype == LGBM_HIP_DTYPE_BF16 ? 1 : 2);
    blocks += chunks_of(t[i], chunk);
    if (l.tensors == LIST) flush();
  }
  flush();
}

}  // namespace

// The scale in 16 bytes, then the sums of the chunks: whole ones and an end for every tensor.
size_t grad_norm_workspace(int64_t elements, int64_t num) {
  return 16 + (size_t)(elements / chunk_size(elements) + num) * sizeof(double);
}

void launch_grad_norm(const GradTensor* t, int64_t num, bool clip, double most, float* norm, void* ws,
                      hipStream_t s) {
  int64_t total = 0;
  for (int64_t i = 0; i < num; ++i) total += t[i].count;
  const int64_t chunk = chunk_size(total);
  Scale* const scale = clip ? (Scale*)ws : nullptr;
  double* const sums = (double*)ws + 2;
  int64_t chunks = 0;
  int64_t most_chunks = 0;
  for (int64_t i = 0; i < num; ++i) most_chunks += chunks_of(t[i], chunk);
  lists(t, num, chunk, [&](const List& l, int64_t done, int64_t blocks) {
    if (most_chunks <= FEW && blocks == most_chunks) {
      k_norm_of_few<<<1, FINAL, 0, s>>>(l, chunk, (int)blocks, most, norm, scale);
      chunks = -1;
      return;
    }
    k_squares<<<(unsigned)blocks, THREADS, 0, s>>>(l, chunk, sums + done);
    chunks = done + blocks;
  });
  if (chunks >= 0) k_norm<<<1, FINAL, 0, s>>>(sums, chunks, most, norm, scale);
  if (!clip) return;
  // past the caches where the list is more than half of the memory's cache of 256 MB (us of k_squares
  // and k_scale, eight float32 tensors to others, through the caches and past them: 96 MB 45.3 and
  // 44.6, 128 MB 58.5 and 57.9, 160 MB 76.5 and 71.8, 256 MB 138 and 113, 768 MB 425 and 400, most of it
  // the next call's k_squares; in place, where stores hit lines that were just read, it is all one: 160
  // MB 72.4 and 72.4, 384 MB 187 and 185, 768 MB 428 and 425)
  int64_t bytes = 0;
  for (int64_t i = 0; i < num; ++i) bytes += t[i].count * (t[i].dtype == LGBM_HIP_DTYPE_F32 ? 4 : 2);
  const bool pass = bytes > ((int64_t)128 << 20);
  lists(t, num, chunk, [&](const List& l, int64_t, int64_t blocks) {
    if (pass)
      k_scale<true><<<(unsigned)blocks, THREADS, 0, s>>>(l, chunk, scale);
    else
      k_scale<false><<<(unsigned)blocks, THREADS, 0, s>>>(l, chunk, scale);
  });
}

}  // namespace lgbm
