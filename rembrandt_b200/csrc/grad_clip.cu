// The global norm of many gradients, and clipping by it:
//   out[0] = |scale| (sum over all values of all tensors of g^2)^1/2
//   out[1] = min(1, max_norm / out[0]), the coefficient; 0 where out[0] is not finite
//   clipping: g = scale out[1] g; zeros where out[1] is 0, whatever g holds
// The sum of squares is taken in 64 bits: it neither overflows nor vanishes for any fp32 values, and what is kept of it, a
// fp32 norm, does not depend on the number of tensors that the values are cut into. The sums of the blocks are joined in a
// fixed order, so that the same gradients always have the same norm.
#include "launch.cuh"
#include "common.cuh"
#include <cuda_fp16.h>

namespace rb {

constexpr int NORM_BLOCKS = 1184;        // most blocks of one launch: as many sums a scratch holds
constexpr int CHUNK = 4096;              // values of a tensor that a block takes at a time
constexpr int TABLE_TENSORS = 128;       // tensors of one launch (a table is a kernel parameter)

// Tensors of one launch. Chunk k belongs to the last tensor whose `first` is at most k.
struct GradTable {
  void* at[TABLE_TENSORS];
  long long n[TABLE_TENSORS];
  long long first[TABLE_TENSORS];
  uint8_t type[TABLE_TENSORS];           // 0 fp32, 1 bf16, 2 fp16
  int count;
  long long chunks;
};

__device__ __forceinline__ int tensor_of(const GradTable& t, long long k) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= k) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <class F>
__device__ __forceinline__ void each_value(const GradTable& t, F f) {
  for (long long k = blockIdx.x; k < t.chunks; k += gridDim.x) {
    const int i = tensor_of(t, k);
    const long long lo = (k - t.first[i]) * CHUNK, hi = min(t.n[i], lo + CHUNK);
    for (long long e = lo + threadIdx.x; e < hi; e += blockDim.x) f(t.at[i], t.type[i], e);
  }
}

// `again`: a later launch of the same norm adds to what the first has left.
__global__ void __launch_bounds__(256) grad_squares_kernel(const __grid_constant__ GradTable t, double* __restrict__ ws, int again) {
  pdl_prolog();
  __shared__ double part[8];
  double s = 0.0;
  each_value(t, [&](const void* p, int type, long long e) {
    const double v = type == 0 ? ((const float*)p)[e] : type == 1 ? bf2f(((const bf16*)p)[e]) : __half2float(((const __half*)p)[e]);
    s += v * v;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) s += part[i];
    ws[blockIdx.x] = again ? ws[blockIdx.x] + s : s;
  }
  if (!again && blockIdx.x == 0)
    for (int i = gridDim.x + threadIdx.x; i < NORM_BLOCKS; i += blockDim.x) ws[i] = 0.0;
}

__global__ void __launch_bounds__(256) grad_norm_kernel(const double* __restrict__ ws, float* __restrict__ out, double scale,
                                                        float max_norm) {
  pdl_prolog();
  __shared__ double part[8];
  double s = 0.0;
  for (int i = threadIdx.x; i < NORM_BLOCKS; i += 256) s += ws[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < 8; ++i) s += part[i];
  const float norm = (float)(fabs(scale) * sqrt(s));
  out[0] = norm;
  out[1] = !isfinite(norm) ? 0.f : norm > max_norm ? max_norm / norm : 1.f;
}

__global__ void __launch_bounds__(256) clip_kernel(const __grid_constant__ GradTable t, const float* __restrict__ out, float scale) {
  pdl_prolog();
  const float coef = out[1], f = scale * coef;
  if (f == 1.f) return;
  each_value(t, [&](void* p, int type, long long e) {
    if (type == 0) { float* q = (float*)p + e; *q = coef == 0.f ? 0.f : *q * f; }
    else if (type == 1) { bf16* q = (bf16*)p + e; *q = f2bf(coef == 0.f ? 0.f : bf2f(*q) * f); }
    else { __half* q = (__half*)p + e; *q = __float2half_rn(coef == 0.f ? 0.f : __half2float(*q) * f); }
  });
}

}  // namespace rb

using namespace rb;

// Calls f(table) for as many tables as hold the tensors; false where an argument is not in order.
template <class F>
static bool for_tables(const void* const* at, const long long* n, const int* types, int count, F f) {
  if (count < 0 || (count && (!at || !n || !types))) return false;
  for (int i = 0; i < count; ++i) {
    const int size = types[i] == 0 ? 4 : 2;
    if (n[i] < 0 || n[i] > (1ll << 40) || types[i] < 0 || types[i] > 2) return false;
    if (n[i] && (!at[i] || (uintptr_t)at[i] % size)) return false;
  }
  GradTable t;
  for (int i = 0; i < count;) {
    t.count = 0;
    t.chunks = 0;
    for (; i < count && t.count < TABLE_TENSORS; ++i) {
      if (n[i] == 0) continue;
      t.at[t.count] = const_cast<void*>(at[i]);
      t.n[t.count] = n[i];
      t.type[t.count] = (uint8_t)types[i];
      t.first[t.count] = t.chunks;
      t.chunks += (n[i] + CHUNK - 1) / CHUNK;
      ++t.count;
    }
    if (t.count) f(t);
  }
  return true;
}

extern "C" {

// at, n, types: host arrays of `count` addresses, numbers of values and types (0 fp32, 1 bf16, 2 fp16).
int rb_grad_norm(const void* const* at, const long long* n, const int* types, int count, float scale, float max_norm,
                 float* out, double* ws, cudaStream_t st) {
  if (!out || !ws || !(max_norm > 0.f)) return -10;
  int again = 0;
  const bool ok = for_tables(at, n, types, count, [&](const GradTable& t) {
    const unsigned blocks = (unsigned)(t.chunks < NORM_BLOCKS ? t.chunks : NORM_BLOCKS);
    launch_pdl(grad_squares_kernel, blocks, 256, 0, st, t, ws, again);
    again = 1;
  });
  if (!ok) return -10;
  if (!again && cudaMemsetAsync(ws, 0, NORM_BLOCKS * sizeof(double), st) != cudaSuccess) return -1;
  launch_pdl(grad_norm_kernel, 1, 256, 0, st, (const double*)ws, out, (double)scale, max_norm);
  return RB_LAUNCH_OK();
}

int rb_clip_grads(const void* const* at, const long long* n, const int* types, int count, float scale, const float* out,
                  cudaStream_t st) {
  if (!out) return -10;
  const bool ok = for_tables(at, n, types, count, [&](const GradTable& t) {
    const unsigned blocks = (unsigned)(t.chunks < 148 * 8 ? t.chunks : 148 * 8);
    launch_pdl(clip_kernel, blocks, 256, 0, st, t, out, scale);
  });
  return ok ? RB_LAUNCH_OK() : -10;
}

}  // extern "C"
