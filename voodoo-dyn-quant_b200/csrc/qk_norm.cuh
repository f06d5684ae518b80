// Norm of every query and key head with the rotation of its position in the
// same pass, and its backward (HBM-bandwidth bound: one read, one write).
//
//   r = rsqrt(mean(x^2) + eps), n = x * r, y = n * (offset + w)       (per head)
//   out[j]     = y[j] * cos[j] - y[j + h] * sin[j]              j < h = R / 2
//   out[j + h] = y[j + h] * cos[j + h] + y[j] * sin[j + h]
//   out[j]     = y[j]                                          R <= j < D
// and, with g the gradient of out turned back by the transposed rotation,
//   dw = sum over heads of g * n,  gn = g * (offset + w),
//   dx = r * (gn - n * mean(gn * n)).
//
// A head is held by a team of G lanes (G = D / 16 rounded up to a power of
// two), each lane with the 8 values at a place of the first half of the
// turned part and the 8 values they turn with, so the rotation needs no
// exchange between lanes and the mean is log2(G) shuffles; the lanes past
// D / 16 of a head that is no power of two carry nothing.  Arithmetic is fp32
// from the load to the one rounding of the store.
#pragma once

#include "common.cuh"

namespace vq {
namespace qknorm {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 512;  // 32 lanes of 16 values
// Blocks of one launch at most: the rows of the weight-gradient partials.
constexpr int kMaxBlocks = 2368;

struct F8 {
  float v[8];
};

template <typename T>
__device__ __forceinline__ F8 load8(const T* p);
template <>
__device__ __forceinline__ F8 load8<float>(const float* p) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
template <>
__device__ __forceinline__ F8 load8<__nv_bfloat16>(const __nv_bfloat16* p) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    r.v[2 * i] = f.x;
    r.v[2 * i + 1] = f.y;
  }
  return r;
}
template <>
__device__ __forceinline__ F8 load8<__half>(const __half* p) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    r.v[2 * i] = f.x;
    r.v[2 * i + 1] = f.y;
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const F8& r);
template <>
__device__ __forceinline__ void store8<float>(float* p, const F8& r) {
  reinterpret_cast<float4*>(p)[0] = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(r.v[4], r.v[5], r.v[6], r.v[7]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const F8& r) {
  uint4 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(r.v[2 * i], r.v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}
template <>
__device__ __forceinline__ void store8<__half>(__half* p, const F8& r) {
  uint4 raw;
  __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(r.v[2 * i], r.v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}

// Weights and tables may be float32 beside 16-bit heads.
template <typename T>
__device__ __forceinline__ F8 load8_or_f32(const void* p, long long at, bool f32) {
  return f32 ? load8<float>(static_cast<const float*>(p) + at) : load8<T>(static_cast<const T*>(p) + at);
}

// The queries or the keys.
template <typename T>
struct Side {
  const T* x;            // [B, S, H, D], strides (xb, xs, xh), unit stride over D
  long long xb, xs, xh;
  const T* g;            // backward: the output's gradient, strides (gb, gs, gh)
  long long gb, gs, gh;
  T* out;                // forward: the turned heads; backward: dx; contiguous [B, S, H, D]
  const void* w;         // [D]
  int H;
  int chunks;            // pieces that a position's heads are split into
  int iters;             // teams of heads a piece walks
  int blocks;            // blocks of the launch that serve this side
};

struct Shape {
  const void* cos;  // [B, S, R], strides (cb, cs)
  const void* sin;
  long long cb, cs;
  long long positions;  // B * S
  int S, D, R;
  int team_log2;  // log2 of the lanes of a head
  float eps, offset;
  bool w_f32, cs_f32;
};

// One warp per (position, piece of its heads), grid-stride within a side; the
// first q.blocks blocks serve the queries, the rest the keys.
// kBackward with partials != nullptr also leaves this block's sum of
// g * n in partials[blockIdx.x][D].
template <typename T, bool kBackward>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(Side<T> q, Side<T> k, Shape sh,
                                                                float* __restrict__ partials) {
  const bool is_q = blockIdx.x < static_cast<unsigned>(q.blocks);
  const Side<T>& side = is_q ? q : k;
  const int block = is_q ? blockIdx.x : blockIdx.x - q.blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int team = 1 << sh.team_log2;
  const int per_warp = 32 >> sh.team_log2;
  const int i = lane & (team - 1), slot = lane >> sh.team_log2;
  const bool live = 16 * i < sh.D;
  const bool turned = 16 * i < sh.R;
  const int a = turned ? 8 * i : 16 * i;
  const int b = turned ? sh.R / 2 + 8 * i : 16 * i + 8;

  F8 w1, w2, dw1, dw2;
#pragma unroll
  for (int j = 0; j < 8; ++j) w1.v[j] = w2.v[j] = dw1.v[j] = dw2.v[j] = 0.f;
  if (live) {
    w1 = load8_or_f32<T>(side.w, a, sh.w_f32);
    w2 = load8_or_f32<T>(side.w, b, sh.w_f32);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w1.v[j] += sh.offset;
      w2.v[j] += sh.offset;
    }
  }
  const float inv_d = 1.f / static_cast<float>(sh.D);
  const long long items = sh.positions * side.chunks;
  for (long long item = static_cast<long long>(block) * kWarps + warp; item < items;
       item += static_cast<long long>(side.blocks) * kWarps) {
    const long long pos = item / side.chunks;
    const int chunk = static_cast<int>(item - pos * side.chunks);
    const long long bi = pos / sh.S, si = pos - bi * sh.S;
    F8 c1, c2, s1, s2;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      c1.v[j] = c2.v[j] = 1.f;
      s1.v[j] = s2.v[j] = 0.f;
    }
    if (turned) {
      const long long at = bi * sh.cb + si * sh.cs;
      c1 = load8_or_f32<T>(sh.cos, at + a, sh.cs_f32);
      c2 = load8_or_f32<T>(sh.cos, at + b, sh.cs_f32);
      s1 = load8_or_f32<T>(sh.sin, at + a, sh.cs_f32);
      s2 = load8_or_f32<T>(sh.sin, at + b, sh.cs_f32);
    }
    const T* xp = side.x + bi * side.xb + si * side.xs;
    const T* gp = kBackward ? side.g + bi * side.gb + si * side.gs : nullptr;
    T* op = side.out + pos * side.H * static_cast<long long>(sh.D);
    const int h0 = chunk * side.iters * per_warp;
    for (int it = 0; it < side.iters; ++it) {
      const int h = h0 + it * per_warp + slot;
      const bool on = live && h < side.H;
      F8 x1, x2, g1, g2;
#pragma unroll
      for (int j = 0; j < 8; ++j) x1.v[j] = x2.v[j] = g1.v[j] = g2.v[j] = 0.f;
      if (on) {
        const T* p = xp + h * side.xh;
        x1 = load8<T>(p + a);
        x2 = load8<T>(p + b);
        if (kBackward) {
          const T* e = gp + h * side.gh;
          g1 = load8<T>(e + a);
          g2 = load8<T>(e + b);
        }
      }
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x1.v[j], x1.v[j], fmaf(x2.v[j], x2.v[j], ss));
      for (int o = team >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(fmaf(ss, inv_d, sh.eps));
      F8 o1, o2;
      if (!kBackward) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y1 = x1.v[j] * r * w1.v[j], y2 = x2.v[j] * r * w2.v[j];
          o1.v[j] = turned ? fmaf(y1, c1.v[j], -y2 * s1.v[j]) : y1;
          o2.v[j] = turned ? fmaf(y2, c2.v[j], y1 * s2.v[j]) : y2;
        }
      } else {
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float t1 = turned ? fmaf(g1.v[j], c1.v[j], g2.v[j] * s2.v[j]) : g1.v[j];
          const float t2 = turned ? fmaf(g2.v[j], c2.v[j], -g1.v[j] * s1.v[j]) : g2.v[j];
          const float n1 = x1.v[j] * r, n2 = x2.v[j] * r;
          dw1.v[j] = fmaf(t1, n1, dw1.v[j]);
          dw2.v[j] = fmaf(t2, n2, dw2.v[j]);
          g1.v[j] = t1 * w1.v[j];
          g2.v[j] = t2 * w2.v[j];
          dot = fmaf(g1.v[j], n1, fmaf(g2.v[j], n2, dot));
        }
        for (int o = team >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        const float m = dot * inv_d;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o1.v[j] = r * fmaf(-(x1.v[j] * r), m, g1.v[j]);
          o2.v[j] = r * fmaf(-(x2.v[j] * r), m, g2.v[j]);
        }
      }
      if (on) {
        T* d = op + static_cast<long long>(h) * sh.D;
        store8<T>(d + a, o1);
        store8<T>(d + b, o2);
      }
    }
  }
  if (kBackward && partials != nullptr) {
    // the same column lives in this lane's place of every team of every warp
    __shared__ float red[kWarps][kMaxDim];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      for (int o = team; o < 32; o <<= 1) {
        dw1.v[j] += __shfl_xor_sync(0xffffffffu, dw1.v[j], o);
        dw2.v[j] += __shfl_xor_sync(0xffffffffu, dw2.v[j], o);
      }
    }
    if (slot == 0 && live) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        red[warp][a + j] = dw1.v[j];
        red[warp][b + j] = dw2.v[j];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < sh.D; c += kThreads) {
      float t = 0.f;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) t += red[v][c];
      partials[static_cast<long long>(blockIdx.x) * sh.D + c] = t;
    }
  }
}

// dw of both sides from the blocks' partials: 32 columns per block, the rows
// of a side summed in a fixed order in 64 bits.  blockIdx.y: 0 queries, 1 keys.
template <typename T>
__global__ void __launch_bounds__(512) qk_norm_weight_grad_kernel(const float* __restrict__ partials, int q_blocks,
                                                                  int k_blocks, int D, bool f32, void* __restrict__ dwq,
                                                                  void* __restrict__ dwk) {
  __shared__ double red[16][33];
  const bool is_q = blockIdx.y == 0;
  void* dw = is_q ? dwq : dwk;
  if (dw == nullptr) return;
  const int rows = is_q ? q_blocks : k_blocks;
  const float* p = partials + (is_q ? 0LL : static_cast<long long>(q_blocks) * D);
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  double t = 0.0;
  if (col < D)
    for (int r = part; r < rows; r += 16) t += static_cast<double>(p[static_cast<long long>(r) * D + col]);
  red[part][threadIdx.x & 31] = t;
  __syncthreads();
  if (part == 0 && col < D) {
    double s = 0.0;
#pragma unroll
    for (int v = 0; v < 16; ++v) s += red[v][threadIdx.x];
    if (f32)
      static_cast<float*>(dw)[col] = static_cast<float>(s);
    else
      static_cast<T*>(dw)[col] = static_cast<T>(static_cast<float>(s));
  }
}

}  // namespace qknorm
}  // namespace vq
