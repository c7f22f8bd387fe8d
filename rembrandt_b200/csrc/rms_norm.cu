// Root-mean-square normalisation over the channels of each position of an NHWC bf16 tensor ([rows][C], of which the first
// c_valid channels are live; the others count as zeros and come out as zeros):
//   forward   h = x [+ residual], rounded to bf16 as it is stored;  r = (sum h^2 / c_valid + eps)^-1/2;  y = act(gamma h r)
//   backward  from y: g = dy where gamma h r > 0 (with a ReLU), xhat = h r, m = sum g gamma xhat / c_valid:
//             dx = r (g gamma - xhat m) [+ add],  dgamma += sum over rows of g xhat
// Unlike a batch normalisation nothing here depends on the other samples of a batch, and there are no running statistics.
// All sums are in fp32; h is the rounded sum, so that backward, which reads it, differentiates what forward computed.
//
// A row is read once and stays in registers between its sum and its output, which is all the traffic there is: 4 bytes a value
// forward (8 with a residual that is kept, 3 into 8 bits), 6 backward (8 with `add`).
//
// How rows lie on threads. Vectors of 8 channels (16 bytes); vector v of a row belongs to lane v % lanes of the row's threads,
// so that neighbouring lanes read neighbouring 16 bytes; a lane has V of them at most.
//   narrow rows: L = 4 to 32 lanes of a warp hold one row, a warp 32 / L of them; sums are shuffles
//   wide rows:   a block holds one row (L = 0)
#include "launch.cuh"
#include "common.cuh"
#include "f32x2.cuh"
#include <algorithm>
#include <atomic>
#include <type_traits>
#include <string.h>

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
  float eps, inv_valid;
  int relu;
};

constexpr float E4M3_MAX = 448.f;

__device__ __forceinline__ float max_nan(float a, float b) {   // as fmaxf, but NaN where either is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float max_nan(float m, float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_abs_nan(float m, float a, float b) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b));
  return d;
}

struct Plus {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Most {
  __device__ __forceinline__ float operator()(float a, float b) const { return max_nan(a, b); }
};

// v of all lanes of a row (L = 0: of the block), joined in the same order everywhere. `slots`: 16 floats of shared memory that
// no other join uses between two barriers.
template <int L, class F>
__device__ __forceinline__ float join_row(float v, float* slots, F f) {
#pragma unroll
  for (int o = (L ? L : 32) >> 1; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (L) return v;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = slots[0];
  for (int w = 1; w < warps; ++w) v = f(v, slots[w]);
  return v;
}

// With two floats an instruction, constant lane counts, 32-bit offsets from a base that is the block's and masks only where channels
// are dead, a vector of eight takes 100 instructions a warp instead of 146 forward and 161 instead of 275 into 8 bits, which
// those kernels were bound by.
__device__ __forceinline__ f2 widen(uint32_t w) {   // two bf16 values
  return both(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t to_bf16(f2 a, bool relu = false) {
  const float2 v = parts(a);
  uint32_t d;
  if (relu) asm("cvt.rn.relu.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(v.y), "f"(v.x));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(v.y), "f"(v.x));
  return d;
}
__device__ __forceinline__ uint32_t to_e4m3(f2 a, f2 b, bool relu) {   // NaN stays NaN
  const float2 v = parts(a), w = parts(b);
  uint16_t lo, hi;
  if (relu) {
    asm("cvt.rn.satfinite.relu.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v.y), "f"(v.x));
    asm("cvt.rn.satfinite.relu.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(w.y), "f"(w.x));
  } else {
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v.y), "f"(v.x));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(w.y), "f"(w.x));
  }
  return lo | ((uint32_t)hi << 16);
}

// Eight bf16 values; `keep_live`: the first `live` of them, zeros behind.
struct Vec8 {
  uint32_t w[4];
};
__device__ __forceinline__ Vec8 load_vec(const bf16* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  return Vec8{{v.x, v.y, v.z, v.w}};
}
__device__ __forceinline__ void store_vec(bf16* p, const Vec8& v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
}
__device__ __forceinline__ void keep_live(Vec8& v, int live) {
  if (live >= 8) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.w[i] = live > 2 * i + 1 ? v.w[i] : live == 2 * i + 1 ? v.w[i] & 0xffffu : 0u;
}

// The vectors of one thread: channel of the first, live channels (0 to 8; -1: behind the row's end), gamma (0 in dead ones).
// Narrow rows lie on L lanes, wide ones (L = 0) on a block.
template <int L, int V>
struct RmsLane {
  int rr, c0, live[V];    // row of the block
  f2 gamma[V][4];
  __device__ __forceinline__ int lanes() const { return L ? L : blockDim.x; }
  __device__ __forceinline__ int next(int j) const { return j * lanes() * 8; }   // vector j behind the first, in channels
  __device__ __forceinline__ RmsLane(const float* g, int C, int c_valid) {
    rr = L ? threadIdx.x / (L ? L : 1) : 0;
    c0 = (L ? threadIdx.x & (L - 1) : threadIdx.x) * 8;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = c0 + next(j);
      live[j] = c >= C ? -1 : min(8, max(0, c_valid - c));
      float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
      if (live[j] >= 0) {
        lo = *reinterpret_cast<const float4*>(g + c);
        hi = *reinterpret_cast<const float4*>(g + c + 4);
      }
      float all[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      if (c_valid < C) {
#pragma unroll
        for (int k = 0; k < 8; ++k) all[k] = k < live[j] ? all[k] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) gamma[j][k] = both(all[2 * k], all[2 * k + 1]);
    }
  }
};

// Threads of a block: narrow rows 256 / L at a time, or one wide row.
template <int L>
struct RmsBlock {
  enum { most = L ? 256 : 512, rows = L ? 256 / (L ? L : 1) : 1 };
};

// A block walks down the rows; the loads of its next rows are under way while it works on the present ones. There is one copy
// of the work in the code, not one for each of several rows: short calls wait for their instructions.
template <int L, int V, bool RES, bool Q8>
__global__ void __launch_bounds__(RmsBlock<L>::most) rms_norm_kernel(const RmsArgs a) {
  pdl_prolog();
  __shared__ float slots[2][2][16];
  const RmsLane<L, V> w(a.gamma, a.C, a.c_valid);
  const unsigned off = (unsigned)(w.rr * a.C + w.c0);      // from the block's first row; less than 2^15
  const bool dead = a.c_valid < a.C;
  const long long step = (long long)gridDim.x * RmsBlock<L>::rows;
  Vec8 hn[V], rn[RES ? V : 1];
  auto fetch = [&](long long r0) {
    const bf16 *x = a.x + r0 * a.C, *res = RES ? a.residual + r0 * a.C : nullptr;
    const bool row = w.rr < a.rows - r0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!row || w.live[j] < 0) { hn[j] = Vec8{{0, 0, 0, 0}}; if (RES) rn[j] = hn[j]; continue; }
      hn[j] = load_vec(x + off + w.next(j));
      if (RES) rn[j] = load_vec(res + off + w.next(j));
    }
  };
  int turn = 0;
  long long r0 = (long long)blockIdx.x * RmsBlock<L>::rows;
  fetch(r0);
  for (; r0 < a.rows; r0 += step, turn ^= 1) {
    const bool row = w.rr < a.rows - r0;
    Vec8 hv[V];
    f2 sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      hv[j] = hn[j];
      if (RES) {
#pragma unroll
        for (int k = 0; k < 4; ++k) hv[j].w[k] = to_bf16(add2(widen(hv[j].w[k]), widen(rn[j].w[k])));
      }
      if (dead) keep_live(hv[j], w.live[j]);
    }
    fetch(r0 + step);
    if (RES && a.h) {
      bf16* h = a.h + r0 * a.C;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (row && w.live[j] >= 0) store_vec(h + off + w.next(j), hv[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f2 f = widen(hv[j].w[k]);
        sum = fma2(f, f, sum);
      }
    const float s = join_row<L>(parts(sum).x + parts(sum).y, slots[turn][0], Plus());
    const float rstd = rsqrtf(s * a.inv_valid + a.eps);
    if (a.rstd && w.c0 == 0 && row) a.rstd[r0 + w.rr] = rstd;
    // h r before gamma: neither product leaves fp32 where the output does not
    const f2 rs = both(rstd, rstd);
    f2 y[V][4];
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) y[j][k] = mul2(mul2(widen(hv[j].w[k]), rs), w.gamma[j][k]);
    if (Q8) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 t = parts(y[j][k]);
          m = a.relu ? max_nan(m, t.x, t.y) : max_abs_nan(m, t.x, t.y);
        }
      m = join_row<L>(m, slots[turn][1], Most());
      // at least the smallest normal number, whose reciprocal is finite
      const float scale = m == 0.f ? 1.f : max_nan(m * (1.f / E4M3_MAX), 1.17549435e-38f);
      const float inv = 1.f / scale;
      if (w.c0 == 0 && row) a.scales[r0 + w.rr] = scale;
      uint8_t* q = a.q + r0 * a.C;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (w.live[j] < 0 || !row) continue;
        uint2 o;
#pragma unroll
        for (int k = 0; k < 4; ++k) y[j][k] = mul2(y[j][k], both(inv, inv));
        if (a.relu) { o.x = to_e4m3(y[j][0], y[j][1], true); o.y = to_e4m3(y[j][2], y[j][3], true); }
        else { o.x = to_e4m3(y[j][0], y[j][1], false); o.y = to_e4m3(y[j][2], y[j][3], false); }
        if (dead && w.live[j] < 8) {   // a row of NaN has zeros there too
          const unsigned long long keep = (1ull << (8 * w.live[j])) - 1;
          o.x &= (uint32_t)keep;
          o.y &= (uint32_t)(keep >> 32);
        }
        *reinterpret_cast<uint2*>(q + off + w.next(j)) = o;
      }
    } else {
      bf16* to = a.y + r0 * a.C;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (w.live[j] < 0 || !row) continue;
        Vec8 o;
        if (a.relu) {
#pragma unroll
          for (int k = 0; k < 4; ++k) o.w[k] = to_bf16(y[j][k], true);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) o.w[k] = to_bf16(y[j][k], false);
        }
        if (dead) keep_live(o, w.live[j]);
        store_vec(to + off + w.next(j), o);
      }
    }
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
  float* sums;            // [blocks][C]: what each block has of dgamma
  long long rows;
  int C, c_valid;
  float inv_valid;
  int relu;
};

// Blocks of the backward kernel that the compiler has to leave room for on an SM (0: as it sees fit). Three vectors: two, which leaves
// no registers for loads ahead and is faster (40000 x 288: 20.4 us against 19.5, with a delta of h 23.7 against 20.9). Four: one,
// with all its registers (15000 x 1024: 22.5 against 20.8); two would spill (with a delta of h 25.4 against 36.5).
template <int L, int V>
struct RmsBackBlocks {
  enum { n = !L ? 0 : V == 3 ? 2 : V == 4 ? 1 : 0 };
};

// A thread has the same channels in all its rows and keeps their part of dgamma in registers; the block's rows are joined at the
// end and the blocks by rms_dgamma_kernel, both in a fixed order (atomic additions would give other last bits every time).
template <int L, int V, bool ADD>
__global__ void __launch_bounds__(RmsBlock<L>::most, RmsBackBlocks<L, V>::n) rms_norm_back_kernel(const RmsBackArgs a) {
  pdl_prolog();
  // the next rows' loads are under way where there are registers for them
  constexpr bool EARLY = L ? V != 3 : V * (ADD ? 3 : 2) <= 6;
  __shared__ float slots[2][16];
  __shared__ __align__(16) float part[L ? V * 2048 : 4];
  const RmsLane<L, V> w(a.gamma, a.C, a.c_valid);
  const unsigned off = (unsigned)(w.rr * a.C + w.c0);
  const bool dead = a.c_valid < a.C;
  f2 acc[V][4];
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[j][k] = 0;
  const long long step = (long long)gridDim.x * RmsBlock<L>::rows;
  Vec8 hn[V], gn[V], an[ADD ? V : 1];
  float rn;
  auto fetch = [&](long long r0) {
    const long long base = r0 * a.C;
    const bf16 *h = a.h + base, *dy = a.dy + base, *add = ADD ? a.add + base : nullptr;
    const bool row = w.rr < a.rows - r0;
    rn = row ? a.rstd[r0 + w.rr] : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!row || w.live[j] < 0) { hn[j] = gn[j] = Vec8{{0, 0, 0, 0}}; continue; }
      hn[j] = load_vec(h + off + w.next(j));
      gn[j] = load_vec(dy + off + w.next(j));
      if (ADD) an[j] = load_vec(add + off + w.next(j));
    }
  };
  int turn = 0;
  long long r0 = (long long)blockIdx.x * RmsBlock<L>::rows;
  if (EARLY) fetch(r0);
  for (; r0 < a.rows; r0 += step, turn ^= 1) {
    const bool row = w.rr < a.rows - r0;
    if (!EARLY) fetch(r0);
    Vec8 hv[V], gv[V], av[ADD ? V : 1];
    const float rstd = rn;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      hv[j] = hn[j];
      gv[j] = gn[j];
      if (ADD) av[j] = an[j];
    }
    if (EARLY) fetch(r0 + step);
    const f2 rs = both(rstd, rstd);
    f2 sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (dead) {
        keep_live(hv[j], w.live[j]);
        keep_live(gv[j], w.live[j]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f2 xhat = mul2(widen(hv[j].w[k]), rs), t = mul2(xhat, w.gamma[j][k]);
        if (a.relu) {
          const float2 p = parts(t);
          uint32_t& g = gv[j].w[k];
          g = (p.x > 0.f ? g & 0xffffu : 0u) | (p.y > 0.f ? g & 0xffff0000u : 0u);
        }
        const f2 g = widen(gv[j].w[k]);
        acc[j][k] = fma2(g, xhat, acc[j][k]);
        sum = fma2(g, t, sum);
      }
    }
    // dx = r (g gamma - h r m): r^2 m would leave fp32 where h is large and the deltas are small
    const float m = join_row<L>(parts(sum).x + parts(sum).y, slots[turn], Plus()) * a.inv_valid;
    const f2 by = both(-(m * rstd), -(m * rstd));
    bf16* dx = a.dx + r0 * a.C;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (w.live[j] < 0 || !row) continue;
      Vec8 d;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f2 t = fma2(widen(hv[j].w[k]), by, mul2(widen(gv[j].w[k]), w.gamma[j][k]));
        d.w[k] = to_bf16(ADD ? fma2(t, rs, widen(av[j].w[k])) : mul2(t, rs));
      }
      if (dead) keep_live(d, w.live[j]);
      store_vec(dx + off + w.next(j), d);
    }
  }
  // a block that is alone adds to dgamma itself
  const bool alone = gridDim.x == 1;
  float* mine = a.sums + (long long)blockIdx.x * a.C;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float2 p0 = parts(acc[j][0]), p1 = parts(acc[j][1]), p2 = parts(acc[j][2]), p3 = parts(acc[j][3]);
    // narrow: part[vector][row of the block][channel]
    float4* to = reinterpret_cast<float4*>(L ? part + j * 2048 + threadIdx.x * 8 : mine + w.c0 + w.next(j));
    if (!L && alone) {
      if (w.live[j] < 0) continue;
      float all[8] = {p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
      to = reinterpret_cast<float4*>(a.dgamma + w.c0 + w.next(j));
      const float4 lo = to[0], hi = to[1];
#pragma unroll
      for (int k = 0; k < 8; ++k) all[k] = k < w.live[j] ? all[k] : 0.f;
      to[0] = make_float4(lo.x + all[0], lo.y + all[1], lo.z + all[2], lo.w + all[3]);
      to[1] = make_float4(hi.x + all[4], hi.y + all[5], hi.z + all[6], hi.w + all[7]);
    } else if (L || w.live[j] >= 0) {
      to[0] = make_float4(p0.x, p0.y, p1.x, p1.y);
      to[1] = make_float4(p2.x, p2.y, p3.x, p3.y);
    }
  }
  if (L) {
    // 256 / width threads per channel add eight rows each, then the first of them what the others have
    constexpr int width = L ? L * 8 : 256;
    const int c = threadIdx.x & (width - 1), t = threadIdx.x / width;
    float s[V];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s[j] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[j] += part[j * 2048 + (t * 8 + i) * width + c];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) part[j * 256 + threadIdx.x] = s[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (t == 0 && j * width + c < a.C) {
#pragma unroll
        for (int i = 1; i < 256 / width; ++i) s[j] += part[j * 256 + i * width + c];
        if (!alone) mine[j * width + c] = s[j];
        else if (j * width + c < a.c_valid) a.dgamma[j * width + c] += s[j];
      }
    }
  }
}

// dgamma += the blocks' sums: COLS channels to a block, 1024 / COLS of the sums at a time, joined in a fixed order.
template <int COLS>
__global__ void __launch_bounds__(1024) rms_dgamma_kernel(const float* __restrict__ sums, float* __restrict__ dgamma, int blocks,
                                                          int C, int c_valid) {
  pdl_prolog();
  constexpr int AT_ONCE = 1024 / COLS;
  __shared__ float part[32][COLS + 1];
  const int k = threadIdx.x / COLS, c = blockIdx.x * COLS + threadIdx.x % COLS;
  float s = 0.f;
  if (c < C) {
#pragma unroll 5
    for (int b = k; b < blocks; b += AT_ONCE) s += sums[(long long)b * C + c];
  }
#pragma unroll
  for (int o = COLS; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) < COLS) part[threadIdx.x >> 5][threadIdx.x & 31] = s;
  __syncthreads();
  // warp w has channel w of the block, a lane each of the 32 parts
  const int ch = threadIdx.x >> 5;
  if (ch >= COLS) return;
  s = warp_sum(part[threadIdx.x & 31][ch]);
  if ((threadIdx.x & 31) == 0 && blockIdx.x * COLS + ch < c_valid) dgamma[blockIdx.x * COLS + ch] += s;
}

}  // namespace rb

using namespace rb;

// What a call hands over, in one record: ctypes takes 1.7 us to convert 14 arguments, 0.6 for a packed record and a stream.
struct RmsFwdCall {
  const bf16* x;
  const bf16* residual;
  bf16* h;
  bf16* y;           // y (bf16), or q (e4m3) and scales: one of the two outputs is null
  uint8_t* q;
  float* scales;
  float* rstd;
  const float* gamma;
  long long rows;
  int C, c_valid;
  float eps;
  int relu;
};
struct RmsBwdCall {
  const bf16* h;
  const bf16* dy;
  const bf16* add;
  bf16* dx;
  const float* rstd;
  const float* gamma;
  float* dgamma;
  float* ws;         // 592 * C floats; 1184 * C for 1032 to 2048 channels
  long long rows;
  int C, c_valid;
  int relu, unused;
};
static_assert(sizeof(RmsFwdCall) == 88 && sizeof(RmsBwdCall) == 88, "as ops/native_ops.py packs them");

static bool rms_shape_ok(long long rows, int C, int c_valid) {
  return rows >= 0 && C >= 8 && C % 8 == 0 && C <= 16384 && c_valid >= 1 && c_valid <= C && rows <= (1ll << 40) / C;
}

// Blocks of a kernel that an SM holds: grids are as large as fit at once, and the blocks walk down the rows.
template <auto KERNEL>
static int blocks_per_sm(int threads) {
  static std::atomic<int> known[17];
  int n = known[threads / 32].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, threads, 0) != cudaSuccess || n < 1) n = 1;
    known[threads / 32].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int n>
using N = std::integral_constant<int, n>;

// Calls go(L, V, threads) for rows of C channels. Up to 1024 channels: as few idle lanes as there can be with at most 4 vectors
// each, and as many lanes where that is equal. Backward passes and bf16 outputs with a residual (`TWO`) rather leave lanes idle than take
// three vectors each, whose registers leave one block on an SM (100000 x 96: forward with residual 13.7 us against 14.3, backward
// 15.3 against 15.8, with a delta of h 17.3 against 18.3; 2000 x 96 backward 3.3 against 3.8; forward alone 9.0 against 8.1). Wider rows: one
// block with two vectors a thread, more where 512 threads do not hold the row. Twice the threads with one vector each wait longer
// for one another (8000 x 2048: forward 14.8 us against 12.8, into 8 bits 19.0 against 13.5, backward 29.3 against 26.0), half of
// them with four keep less under way (6000 x 2560: backward 30.8 against 22.9).
template <bool TWO, class F>
static void rms_cover(int C, F go) {
  const int cg = C / 8;
  if (cg > 128) {
    const int V = cg <= 1024 ? 2 : cg <= 1536 ? 3 : 4, threads = (ceil_div(cg, V) + 31) / 32 * 32;
    if (V == 2) go(N<0>(), N<2>(), threads);
    else if (V == 3) go(N<0>(), N<3>(), threads);
    else go(N<0>(), N<4>(), threads);
    return;
  }
  int lanes = 0, V = 0;
  for (int l = 32; l >= 4; l >>= 1) {
    const int v = ceil_div(cg, l);
    const bool built = v == 1 || l == 32 || (v == 3 && !(TWO && cg <= 32));
    if (built && v <= 4 && (!lanes || l * v < lanes * V)) { lanes = l; V = v; }
  }
  constexpr int THREE = TWO ? 1 : 3;      // what three vectors on four or eight lanes are, where they are not built
  if (lanes == 4) V == 1 ? go(N<4>(), N<1>(), 256) : go(N<4>(), N<THREE>(), 256);
  else if (lanes == 8) V == 1 ? go(N<8>(), N<1>(), 256) : go(N<8>(), N<THREE>(), 256);
  else if (lanes == 16) V == 1 ? go(N<16>(), N<1>(), 256) : go(N<16>(), N<3>(), 256);
  else if (V == 1) go(N<32>(), N<1>(), 256);
  else if (V == 2) go(N<32>(), N<2>(), 256);
  else if (V == 3) go(N<32>(), N<3>(), 256);
  else go(N<32>(), N<4>(), 256);
}

extern "C" {

// call: a packed RmsFwdCall.
int rb_rms_norm_fwd(const void* call, cudaStream_t st) {
  RmsFwdCall c;
  memcpy(&c, call, sizeof(c));
  const long long rows = c.rows;
  if (!rms_shape_ok(rows, c.C, c.c_valid)) return -10;
  if (rows == 0) return 0;
  if ((c.y != nullptr) == (c.q != nullptr) || (c.q && !c.scales)) return -10;
  if (c.h && !c.residual) return -10;      // without a residual h is x
  const RmsArgs a{c.x, c.residual, c.h, c.y, c.q, c.scales, c.rstd, c.gamma, rows, c.C, c.c_valid, c.eps, 1.f / (float)c.c_valid, c.relu};
  auto run = [&](auto res, auto q8) {
    constexpr bool RES = decltype(res)::value, Q8 = decltype(q8)::value;
    rms_cover<RES && !Q8>(c.C, [&](auto lanes, auto vectors, int threads) {
      constexpr int L = decltype(lanes)::value;
      constexpr auto kern = rms_norm_kernel<L, decltype(vectors)::value, RES, Q8>;
      const long long need = (rows + RmsBlock<L>::rows - 1) / RmsBlock<L>::rows, most = 148ll * blocks_per_sm<kern>(threads);
      launch_pdl(kern, (unsigned)std::min(need, most), threads, 0, st, a);
    });
  };
  if (c.residual) c.q ? run(std::true_type(), std::true_type()) : run(std::true_type(), std::false_type());
  else c.q ? run(std::false_type(), std::true_type()) : run(std::false_type(), std::false_type());
  return RB_LAUNCH_OK();
}

// call: a packed RmsBwdCall.
int rb_rms_norm_bwd(const void* call, cudaStream_t st) {
  RmsBwdCall c;
  memcpy(&c, call, sizeof(c));
  const long long rows = c.rows;
  const int C = c.C, c_valid = c.c_valid;
  if (!rms_shape_ok(rows, C, c_valid)) return -10;
  if (rows == 0) return 0;
  const RmsBackArgs a{c.h, c.dy, c.add, c.dx, c.rstd, c.gamma, c.dgamma, c.ws, rows, C, c_valid, 1.f / (float)c_valid, c.relu};
  int blocks = 0;
  rms_cover<true>(C, [&](auto lanes, auto vectors, int threads) {
    constexpr int L = decltype(lanes)::value, V = decltype(vectors)::value;
    auto go = [&](auto with) {
      constexpr auto kern = rms_norm_back_kernel<L, V, decltype(with)::value>;
      const long long need = (rows + RmsBlock<L>::rows - 1) / RmsBlock<L>::rows;
      // a block for each of four resident ones, eight where they are small: fewer partial sums against more rows under way
      // (12000 x 1280, 96 threads: 32.4 us with four, 24.2 with eight)
      const int most = 148 * std::min(L || threads > 128 ? 4 : 8, blocks_per_sm<kern>(threads));
      // up to four times the rows that a block has at once, one block is as fast as several and a second launch (64 x 128: 2.9 us
      // against 3.0, 128 x 128: 4.2), but not where its vectors are many (32 x 512: 4.5 against 3.6)
      blocks = need <= (L && V == 1 ? 4 : 1) ? 1 : (int)std::min(need, (long long)most);
      launch_pdl(kern, blocks, threads, 0, st, a);
    };
    c.add ? go(std::true_type()) : go(std::false_type());
  });
  if (blocks == 1) return RB_LAUNCH_OK();
  auto finish = [&](auto cols) {
    constexpr int COLS = decltype(cols)::value;
    launch_pdl(rms_dgamma_kernel<COLS>, (unsigned)ceil_div(c_valid, COLS), 1024, 0, st, (const float*)c.ws, c.dgamma, blocks, C, c_valid);
  };
  // eight channels a block while that leaves few blocks (92416 x 128: 16.2 us both launches against 17.0), 32 from there on
  // (1500 x 9216: 23.0 against 27.3)
  C <= 2048 ? finish(N<8>()) : finish(N<32>());
  return RB_LAUNCH_OK();
}

}  // extern "C"
