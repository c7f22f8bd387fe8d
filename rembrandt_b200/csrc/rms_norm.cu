// Root-mean-square normalisation over the channels of each position of an NHWC bf16 tensor ([rows][C], of which the first
// c_valid channels are live; the others count as zeros and come out as zeros):
//   forward   h = x [+ residual], rounded to bf16 as it is stored;  r = (sum h^2 / c_valid + eps)^-1/2;  y = act(gamma h r)
//   backward  from y: g = dy where gamma h r > 0 (with a ReLU), xhat = h r, m = sum g gamma xhat / c_valid:
//             dx = r (g gamma - xhat m) [+ add],  dgamma += sum over rows of g xhat
// Unlike a batch normalisation nothing here depends on the other samples of a batch, and there are no running statistics.
// All sums are in fp32; h is the rounded sum, so that backward, which reads it, differentiates what forward computed.
#include "launch.cuh"
#include "common.cuh"
#include <cuda_fp8.h>

namespace rb {

struct RmsArgs {
  const bf16* x;
  const bf16* residual;   // null: h = x
  bf16* h;                // null: not stored
  bf16* y;                // bf16 output, or null
  uint8_t* q;             // e4m3 output, with one scale per row, or null
  float* scales;
  float* rstd;            // null: not stored
  const float* gamma;
  long long rows;
  int C, c_valid;
  float eps;
  int relu;
};

__device__ __forceinline__ float max_nan(float a, float b) {   // as fmaxf, but NaN where either is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

constexpr float E4M3_MAX = 448.f;

// One warp per row; the row is read again for the output.
__global__ void __launch_bounds__(128) rms_norm_kernel(const RmsArgs a) {
  pdl_prolog();
  const int lane = threadIdx.x & 31;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= a.rows) return;
  const long long base = r * a.C;
  auto h_at = [&](int c) {
    if (c >= a.c_valid) return 0.f;
    float v = bf2f(a.x[base + c]);
    if (a.residual) v = bf2f(f2bf(v + bf2f(a.residual[base + c])));
    return v;
  };
  float s = 0.f;
  for (int c = lane; c < a.c_valid; c += 32) {
    const float v = h_at(c);
    s += v * v;
  }
  const float rstd = rsqrtf(warp_sum(s) / a.c_valid + a.eps);
  if (a.rstd && lane == 0) a.rstd[r] = rstd;
  auto y_of = [&](float h, int c) {
    if (c >= a.c_valid) return 0.f;
    const float y = h * rstd * a.gamma[c];
    return a.relu && y <= 0.f ? 0.f : y;
  };
  float inv = 1.f;
  if (a.q) {
    float m = 0.f;
    for (int c = lane; c < a.c_valid; c += 32) m = max_nan(m, fabsf(y_of(h_at(c), c)));
    m = warp_max_nan(m);
    // at least the smallest normal number, whose reciprocal is finite
    const float scale = m == 0.f ? 1.f : max_nan(m / E4M3_MAX, 1.17549435e-38f);
    inv = 1.f / scale;
    if (lane == 0) a.scales[r] = scale;
  }
  for (int c = lane; c < a.C; c += 32) {
    const float h = h_at(c), y = y_of(h, c);
    if (a.h) a.h[base + c] = f2bf(h);
    if (a.q) a.q[base + c] = __nv_cvt_float_to_fp8(y * inv, __NV_SATFINITE, __NV_E4M3);
    else a.y[base + c] = f2bf(y);
  }
}

struct RmsBackArgs {
  const bf16* h;
  const bf16* dy;
  const bf16* add;        // null: nothing is added
  bf16* dx;
  const float* rstd;
  const float* gamma;
  float* dgamma;
  long long rows;
  int C, c_valid;
  int relu;
};

__global__ void __launch_bounds__(128) rms_norm_back_kernel(const RmsBackArgs a) {
  pdl_prolog();
  const int lane = threadIdx.x & 31;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (r >= a.rows) return;
  const long long base = r * a.C;
  const float rstd = a.rstd[r];
  float m = 0.f;
  for (int c = lane; c < a.c_valid; c += 32) {
    const float xhat = bf2f(a.h[base + c]) * rstd, gamma = a.gamma[c];
    const float g = a.relu && !(gamma * xhat > 0.f) ? 0.f : bf2f(a.dy[base + c]);
    m += g * gamma * xhat;
  }
  m = warp_sum(m) / a.c_valid;
  for (int c = lane; c < a.C; c += 32) {
    float d = 0.f;
    if (c < a.c_valid) {
      const float xhat = bf2f(a.h[base + c]) * rstd, gamma = a.gamma[c];
      const float g = a.relu && !(gamma * xhat > 0.f) ? 0.f : bf2f(a.dy[base + c]);
      d = rstd * (g * gamma - xhat * m);
      if (a.add) d += bf2f(a.add[base + c]);
    }
    a.dx[base + c] = f2bf(d);
  }
}

// dgamma: one block per 32 channels, eight rows at a time, joined in a fixed order.
__global__ void __launch_bounds__(256) rms_norm_dgamma_kernel(const RmsBackArgs a) {
  pdl_prolog();
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < a.c_valid) {
    const float gamma = a.gamma[c];
    for (long long r = k; r < a.rows; r += 8) {
      const float xhat = bf2f(a.h[r * a.C + c]) * a.rstd[r];
      const float g = a.relu && !(gamma * xhat > 0.f) ? 0.f : bf2f(a.dy[r * a.C + c]);
      s += g * xhat;
    }
  }
  part[k][lane] = s;
  __syncthreads();
  if (k == 0 && c < a.c_valid) {
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    a.dgamma[c] += s;
  }
}

}  // namespace rb

using namespace rb;

static bool rms_shape_ok(long long rows, int C, int c_valid) {
  return rows >= 0 && C >= 8 && C % 8 == 0 && C <= 32768 && c_valid >= 1 && c_valid <= C && rows <= (1ll << 40) / C;
}

extern "C" {

// y (bf16), or q (e4m3) and scales: one of the two outputs is null.
int rb_rms_norm_fwd(const void* x, const void* residual, void* h, void* y, void* q, float* scales, float* rstd,
                    const float* gamma, long long rows, int C, int c_valid, float eps, int relu, cudaStream_t st) {
  if (!rms_shape_ok(rows, C, c_valid) || (y != nullptr) == (q != nullptr) || (q && !scales)) return -10;
  if (rows == 0) return 0;
  RmsArgs a{(const bf16*)x, (const bf16*)residual, (bf16*)h, (bf16*)y, (uint8_t*)q, scales, rstd, gamma, rows, C, c_valid,
            eps, relu};
  launch_pdl(rms_norm_kernel, (unsigned)((rows + 3) / 4), 128, 0, st, a);
  return RB_LAUNCH_OK();
}

int rb_rms_norm_bwd(const void* h, const void* dy, const void* add, void* dx, const float* rstd, const float* gamma,
                    float* dgamma, float* ws, long long rows, int C, int c_valid, int relu, cudaStream_t st) {
  if (!rms_shape_ok(rows, C, c_valid)) return -10;
  if (rows == 0) return 0;
  RmsBackArgs a{(const bf16*)h, (const bf16*)dy, (const bf16*)add, (bf16*)dx, rstd, gamma, dgamma, rows, C, c_valid, relu};
  // dgamma first: dx may be written over dy
  launch_pdl(rms_norm_dgamma_kernel, (unsigned)((c_valid + 31) / 32), 256, 0, st, a);
  launch_pdl(rms_norm_back_kernel, (unsigned)((rows + 3) / 4), 128, 0, st, a);
  return RB_LAUNCH_OK();
}

}  // extern "C"
