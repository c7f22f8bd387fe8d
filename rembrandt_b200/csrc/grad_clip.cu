// The global norm of many gradients, and clipping by it:
//   out[0] = scale (sum over all values of all tensors of g^2)^1/2
//   out[1] = min(1, max_norm / out[0]), the coefficient; 0 where out[0] is not finite
//   clipping: g = scale out[1] g; zeros where out[1] is 0, whatever g holds
// Squares are added in 64 bits, and in fp32 only among the 16 or 32 values that a thread has at a time, where that neither
// overflows nor loses any (part_squares): no fp32 values are too large or too small for it. The sums of the blocks are joined in
// a fixed order, so that the same gradients always have the same norm.
//
// Bound by memory: a norm reads each value once, clipping reads and writes it, and does nothing where the factor is 1. Measured
// (us, and at the copy rate of 6.5 TB/s): norm of 62.4 M fp32 values 37.9 (38.2), of bf16 ones 21.6 (19.1); clipping 79 (76) and
// 40.4 (38.2); both together 118 and 58, because about 25 MB of what the norm has read is still in the L2.
#include "launch.cuh"
#include "clip_factor.cuh"
#include "common.cuh"
#include "f32x2.cuh"
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <utility>
#include <string.h>

namespace rb {

constexpr int NORM_BLOCKS = 740;         // most blocks of one launch: as many sums a scratch holds
constexpr int VECTORS = 4;               // 16-byte vectors that a thread has under way
constexpr int CHUNK = 256 * VECTORS;     // vectors of a tensor that a block takes at a time

// The tensors of one launch; the table is a kernel parameter, which a captured launch keeps. A tensor is a row of 16-byte
// vectors from the boundary at or before its first value on; chunk k belongs to the last tensor whose `first` is at most k.
template <int TENSORS>
struct GradTable {
  unsigned long long at[TENSORS];        // address of the first value
  long long n[TENSORS];                  // values * 4 + type (0 fp32, 1 bf16, 2 fp16)
  int first[TENSORS];
  int count, chunks;
};

template <int TENSORS>
__device__ __forceinline__ int tensor_of(const GradTable<TENSORS>& t, int k) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= k) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// One thread's part of a chunk: vectors v + 256 i of the tensor for i < VECTORS, the first of them at `at`.
struct Part {
  char* at;
  long long v, last;      // the number of vectors
  int lead, tail, type;   // values before the first in vector 0, live values of the last vector
  bool inside;            // the chunk as a whole has neither the tensor's first vector, where that is cut, nor its last
};
template <int TENSORS>
__device__ __forceinline__ Part part_of(const GradTable<TENSORS>& t, int i, int k, int thread) {
  Part p;
  const unsigned long long at = t.at[i];
  const long long n = t.n[i];
  p.type = (int)(n & 3);
  const int shift = p.type == 0 ? 2 : 1, per = 16 >> shift;
  p.lead = (int)(at & 15) >> shift;
  const long long end = p.lead + (n >> 2), v0 = (long long)(k - t.first[i]) * CHUNK;
  p.last = (end + per - 1) >> (4 - shift);
  p.tail = (int)(end - (p.last - 1) * per);
  p.inside = (v0 > 0 || p.lead == 0) && v0 + CHUNK < p.last;
  p.v = v0 + thread;
  p.at = reinterpret_cast<char*>((at & ~15ull) + p.v * 16);
  return p;
}

template <int TYPE>
__device__ __forceinline__ float value(const uint4& v, int j) {
  const uint32_t w = reinterpret_cast<const uint32_t*>(&v)[TYPE == 0 ? j : j >> 1];
  if (TYPE == 0) return __uint_as_float(w);
  if (TYPE == 1) return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return j & 1 ? f.y : f.x;
}

// The vector at p.v + 256 i, zeros outside of the tensor. Values are read one by one where the tensor ends inside of it: what
// lies there may belong to nobody.
template <int TYPE>
__device__ __forceinline__ uint4 load_part(const Part& p, int i) {
  constexpr int PER = TYPE == 0 ? 4 : 8;
  const char* const here = p.at + 4096 * i;
  if (p.inside) return *reinterpret_cast<const uint4*>(here);
  const long long v = p.v + 256 * i;
  uint4 r = make_uint4(0, 0, 0, 0);
  if (v >= p.last) return r;
  const char* at = here;
  const int lo = v == 0 ? p.lead : 0, hi = v == p.last - 1 ? p.tail : PER;
  if (lo == 0 && hi == PER) return *reinterpret_cast<const uint4*>(at);
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (j >= lo && j < hi) {
      if (TYPE == 0) w[j] = reinterpret_cast<const uint32_t*>(at)[j];
      else w[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(at)[j] << (16 * (j & 1));
    }
  return r;
}

// Sum of the squares of a part's values (times scale^2): at most seven roundings between a square and the sum.
template <int TYPE, bool SCALED>
__device__ __forceinline__ float squares(const uint4 (&v)[VECTORS], float scale) {
  f2 s[VECTORS];
#pragma unroll
  for (int i = 0; i < VECTORS; ++i) {
    s[i] = 0;
#pragma unroll
    for (int j = 0; j < (TYPE == 0 ? 4 : 8); j += 2) {
      f2 f = both(value<TYPE>(v[i], j), value<TYPE>(v[i], j + 1));
      if (SCALED) f = mul2(f, both(scale, scale));
      s[i] = fma2(f, f, s[i]);
    }
  }
  static_assert(VECTORS == 4, "");
  const float2 t = parts(add2(add2(s[0], s[1]), add2(s[2], s[3])));
  return t.x + t.y;
}

// In fp32 while the sum lies between 2^-60 and 2^100: no square has overflown then, and what is lost of those that have gone
// below 2^-126 is less than 2^-60 of the sum. Otherwise the values are taken times a power of two that brings the largest and
// smallest ones that there are (2^128 and 2^-149) between 2^-59 and 2^60.
template <int TYPE>
__device__ __forceinline__ double part_squares(const Part& p) {
  uint4 v[VECTORS];
#pragma unroll
  for (int i = 0; i < VECTORS; ++i) v[i] = load_part<TYPE>(p, i);
  const float s = squares<TYPE, false>(v, 1.f);
  if (s >= 0x1p-60f && s <= 0x1p100f) return (double)s;
  const bool small = s < 1.f;
  const double t = squares<TYPE, true>(v, small ? 0x1p90f : 0x1p-70f);
  return t * (small ? 0x1p-180 : 0x1p140);
}

__device__ __forceinline__ double block_sum(double s, double* part) {   // valid in thread 0
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  s = part[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) s += part[i];
  return s;
}

// Five blocks an SM, with four 16-byte loads under way per thread: with eight, the last round of chunks fills less of the device
// (62.4 M fp32 values: 39.4 us against 38.4). From the last chunk to the first: what is read last, and is still in the L2, is where
// the sweep that follows begins.
// `again`: a later launch of the same norm adds to what the first has left.
template <int TENSORS>
__global__ void __launch_bounds__(256) grad_squares_kernel(const __grid_constant__ GradTable<TENSORS> t, double* __restrict__ ws,
                                                           int again) {
  pdl_prolog();
  __shared__ double part[8];
  double s = 0.0;
  int k = t.chunks - 1 - (int)blockIdx.x;
  for (int i = tensor_of(t, k); k >= 0; k -= gridDim.x) {
    while (t.first[i] > k) --i;
    const Part p = part_of(t, i, k, threadIdx.x);
    s += p.type == 0 ? part_squares<0>(p) : p.type == 1 ? part_squares<1>(p) : part_squares<2>(p);
  }
  s = block_sum(s, part);
  if (threadIdx.x == 0) ws[blockIdx.x] = again ? ws[blockIdx.x] + s : s;
  if (!again && blockIdx.x == 0)
    for (int i = gridDim.x + threadIdx.x; i < NORM_BLOCKS; i += blockDim.x) ws[i] = 0.0;
}

__device__ __forceinline__ void put_norm(double sum, double scale, float max_norm, float* out) {
  const float norm = (float)(scale * sqrt(sum));
  out[0] = norm;
  out[1] = !isfinite(norm) ? 0.f : norm > max_norm ? max_norm / norm : 1.f;
}

// All of it in one launch, for lists that a cluster of eight blocks gets through in the time of a second launch: an SM reads about
// 70 GB/s (1000 fp32 values: 2.7 us against 3.0, 85 thousand: 3.1 against 3.2, 260 thousand: 3.9 against 3.3), and a program
// that launches step by step saves the 2 us of the launch. The blocks hand their sums to the first through its shared memory.
constexpr int CLUSTER = 8, SMALL_CHUNKS = 32;
template <int TENSORS>
__global__ void __cluster_dims__(CLUSTER) __launch_bounds__(1024)
    grad_norm_small_kernel(const __grid_constant__ GradTable<TENSORS> t, float* __restrict__ out, double scale, float max_norm) {
  pdl_prolog();
  __shared__ double part[32];
  __shared__ double sums[CLUSTER];
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  auto started = cluster.barrier_arrive();
  double s = 0.0;
  int k = blockIdx.x * 4 + (threadIdx.x >> 8);
  if (k < t.chunks) {
    for (int i = tensor_of(t, k); k < t.chunks; k += CLUSTER * 4) {
      while (i + 1 < t.count && t.first[i + 1] <= k) ++i;
      const Part p = part_of(t, i, k, threadIdx.x & 255);
      s += p.type == 0 ? part_squares<0>(p) : p.type == 1 ? part_squares<1>(p) : part_squares<2>(p);
    }
  }
  s = block_sum(s, part);
  cluster.barrier_wait(std::move(started));     // the first block's shared memory is there
  if (threadIdx.x == 0) *cluster.map_shared_rank(&sums[blockIdx.x], 0) = s;
  cluster.sync();
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    s = sums[0];
    for (int i = 1; i < CLUSTER; ++i) s += sums[i];
    put_norm(s, scale, max_norm, out);
  }
}

__global__ void __launch_bounds__(256) grad_norm_kernel(const double* __restrict__ ws, float* __restrict__ out, double scale,
                                                        float max_norm) {
  pdl_prolog();
  __shared__ double part[8];
  double v[(NORM_BLOCKS + 255) / 256];
#pragma unroll
  for (int i = 0; i < (NORM_BLOCKS + 255) / 256; ++i) v[i] = i * 256 + threadIdx.x < NORM_BLOCKS ? ws[i * 256 + threadIdx.x] : 0.0;
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < (NORM_BLOCKS + 255) / 256; ++i) s += v[i];
  s = block_sum(s, part);
  if (threadIdx.x == 0) put_norm(s, scale, max_norm, out);
}

template <int TYPE, bool LOW>
__device__ __forceinline__ void scale_part(const Part& p, const ClipFactor& f, bool zero) {
  constexpr int PER = TYPE == 0 ? 4 : 8;
  uint4 v[VECTORS];
#pragma unroll
  for (int i = 0; i < VECTORS; ++i) v[i] = load_part<TYPE>(p, i);
  // value j of a vector, times the factor
  auto scaled = [&](const uint4& vec, int j) { return zero ? 0.f : LOW ? value<TYPE>(vec, j) * f.back * f.by : value<TYPE>(vec, j) * f.by; };
#pragma unroll
  for (int i = 0; i < VECTORS; ++i) {
    const long long n = p.v + 256 * i;
    if (!p.inside && n >= p.last) break;
    uint4 r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (TYPE == 0) {
        w[j] = __float_as_uint(scaled(v[i], j));
      } else {
        const float a = scaled(v[i], 2 * j), b = scaled(v[i], 2 * j + 1);
        if (TYPE == 1) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(a, b);
          w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
    char* at = p.at + 4096 * i;
    const int lo = n == 0 ? p.lead : 0, hi = n == p.last - 1 ? p.tail : PER;
    if (p.inside || (lo == 0 && hi == PER)) {
      __stcs(reinterpret_cast<uint4*>(at), r);   // not to drive out of the L2 what is still to be read
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (j >= lo && j < hi) {
          if (TYPE == 0) reinterpret_cast<uint32_t*>(at)[j] = w[j];
          else reinterpret_cast<uint16_t*>(at)[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
        }
    }
  }
}

// Blocks take runs of chunks and start in order, so that what is under way lies close together. The more blocks, the faster they
// clip, and the longer it takes them to find that there is nothing to do (62.4 M fp32 values, us for one and for the other: 888 blocks
// 87.6 and 1.3, 1776 83.3 and 2.2, 3552 79.1 and 3.7, 8000 75.8 and 8.3, one a chunk 74.4 and 16.2).
constexpr int CLIP_BLOCKS = 3552;
template <bool LOW, int TENSORS>
__device__ __forceinline__ void clip_run(const GradTable<TENSORS>& t, const ClipFactor& f, bool zero, int run) {
  int k = blockIdx.x * run;
  const int end = min(k + run, t.chunks);
  for (int i = tensor_of(t, k); k < end; ++k) {
    while (i + 1 < t.count && t.first[i + 1] <= k) ++i;
    const Part p = part_of(t, i, k, threadIdx.x);
    if (p.type == 0) scale_part<0, LOW>(p, f, zero);
    else if (p.type == 1) scale_part<1, LOW>(p, f, zero);
    else scale_part<2, LOW>(p, f, zero);
  }
}

template <int TENSORS>
__global__ void __launch_bounds__(256) clip_kernel(const __grid_constant__ GradTable<TENSORS> t, const float* __restrict__ out,
                                                   float scale, int run) {
  pdl_prolog();
  const float coef = out[1];
  const ClipFactor f = clip_factor(scale, coef);
  if (f.by == 1.f) return;
  if (f.back == 1.f) clip_run<false>(t, f, false, run);
  else clip_run<true>(t, f, coef == 0.f, run);
}

}  // namespace rb

using namespace rb;

// A table of few tensors is 2.6 KB of parameters, one of many 31 KB, which take longer to hand over.
constexpr int FEW = 128, MANY = 1536;
static_assert(sizeof(GradTable<MANY>) < 32000, "kernel parameters end at 32764 bytes");

// Calls f(table) for as many tables of TENSORS as hold the tensors. False where they are too large for a table's chunk numbers.
template <int TENSORS, class F>
static bool fill_tables(const void* const* at, const long long* n, const int* types, int count, F f) {
  GradTable<TENSORS> t;
  for (int i = 0; i < count;) {
    t.count = t.chunks = 0;
    for (; i < count && t.count < TENSORS; ++i) {
      if (n[i] == 0) continue;
      const int size = types[i] == 0 ? 4 : 2, per = 16 / size;
      const long long vectors = ((long long)((uintptr_t)at[i] & 15) / size + n[i] + per - 1) / per, chunks = (vectors + CHUNK - 1) / CHUNK;
      if (chunks > (1 << 30)) return false;
      if (t.chunks + chunks > (1 << 30)) break;
      t.at[t.count] = (unsigned long long)(uintptr_t)at[i];
      t.n[t.count] = n[i] * 4 + types[i];
      t.first[t.count++] = t.chunks;
      t.chunks += (int)chunks;
    }
    if (t.count) f(t);
  }
  return true;
}
// A list of gradients as calls hand it over: host arrays of addresses, numbers of values and types (0 fp32, 1 bf16, 2 fp16).
struct GradListRecord {
  const void* const* at;
  const long long* n;
  const int* types;
  long long count;
};
static_assert(sizeof(GradListRecord) == 32, "as ops/native_ops.py packs it");

template <class F>
static bool for_tables(const void* list, F f) {
  GradListRecord r;
  memcpy(&r, list, sizeof(r));
  const void* const* at = r.at;
  const long long* n = r.n;
  const int* types = r.types;
  const int count = r.count < 0 || r.count > 1 << 30 ? -1 : (int)r.count;
  if (count < 0 || (count && (!at || !n || !types))) return false;
  for (int i = 0; i < count; ++i) {
    if (types[i] < 0 || types[i] > 2 || n[i] < 0 || n[i] > (1ll << 40)) return false;
    if (n[i] && (!at[i] || (uintptr_t)at[i] % (types[i] == 0 ? 4 : 2))) return false;
  }
  return count <= FEW ? fill_tables<FEW>(at, n, types, count, f) : fill_tables<MANY>(at, n, types, count, f);
}

extern "C" {

// list: a packed GradListRecord; ws: 740 doubles.
int rb_grad_norm(const void* list, float scale, float max_norm, float* out, double* ws, cudaStream_t st) {
  if (!list || !out || !ws || !(max_norm > 0.f)) return -10;
  int again = 0;
  bool done = false;
  const bool ok = for_tables(list, [&](const auto& t) {
    constexpr int TENSORS = sizeof(t.first) / sizeof(int);
    if constexpr (TENSORS == FEW) {
      done = !again && t.chunks <= SMALL_CHUNKS;
      if (done) {
        launch_pdl(grad_norm_small_kernel<FEW>, CLUSTER, 1024, 0, st, t, out, (double)scale, max_norm);
        return;
      }
    }
    launch_pdl(grad_squares_kernel<TENSORS>, std::min(t.chunks, NORM_BLOCKS), 256, 0, st, t, ws, again);
    again = 1;
  });
  if (!ok) return -10;
  if (done) return RB_LAUNCH_OK();
  if (!again && cudaMemsetAsync(ws, 0, NORM_BLOCKS * sizeof(double), st) != cudaSuccess) return -1;
  launch_pdl(grad_norm_kernel, 1, 256, 0, st, (const double*)ws, out, (double)scale, max_norm);
  return RB_LAUNCH_OK();
}

int rb_clip_grads(const void* list, float scale, const float* out, cudaStream_t st) {
  if (!list || !out) return -10;
  const bool ok = for_tables(list, [&](const auto& t) {
    const int run = ceil_div(t.chunks, CLIP_BLOCKS);
    launch_pdl(clip_kernel<sizeof(t.first) / 4>, ceil_div(t.chunks, run), 256, 0, st, t, out, scale, run);
  });
  return ok ? RB_LAUNCH_OK() : -10;
}

}  // extern "C"
