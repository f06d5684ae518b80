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
#ifndef VQ_QK_FWD_BLOCKS
#define VQ_QK_FWD_BLOCKS 6
#endif
#ifndef VQ_QK_BWD_BLOCKS
#define VQ_QK_BWD_BLOCKS 4
#endif
#ifndef VQ_QK_BWD_BLOCKS_WIDE
#define VQ_QK_BWD_BLOCKS_WIDE 3
#endif
// Resident blocks per SM; fp32 tables take twice the registers in the backward.
constexpr int kFwdBlocks = VQ_QK_FWD_BLOCKS, kBwdBlocks = VQ_QK_BWD_BLOCKS, kBwdBlocksWide = VQ_QK_BWD_BLOCKS_WIDE;
// Blocks of one launch at most: the rows of the weight-gradient partials.
constexpr int kMaxBlocks = 2368;

// Sixteen-bit values are widened two at a time and all arithmetic is on
// pairs: sm_100 runs two fp32 operations per instruction (f32x2), which is
// what keeps these kernels under the memory time.
struct F8 {
  float2 v[4];
};

__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 neg(float2 a) { return make_float2(-a.x, -a.y); }

// Eight values as they lie in memory.
template <typename T>
struct Raw8 {
  uint4 q;
  __device__ __forceinline__ void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { q = make_uint4(0, 0, 0, 0); }
  // Keeps the compiler from widening it once, ahead of the loop that uses it:
  // that would hold twice the registers for the whole loop.
  __device__ __forceinline__ void stay() { asm volatile("" : "+r"(q.x), "+r"(q.y), "+r"(q.z), "+r"(q.w)); }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void stay() {}
};

__device__ __forceinline__ F8 widen(const Raw8<float>& r) {
  return {{make_float2(r.a.x, r.a.y), make_float2(r.a.z, r.a.w), make_float2(r.b.x, r.b.y), make_float2(r.b.z, r.b.w)}};
}
__device__ __forceinline__ float2 widen2(uint32_t w, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 widen2(uint32_t w, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ F8 widen(const Raw8<T>& r) {
  const T* t = nullptr;
  return {{widen2(r.q.x, t), widen2(r.q.y, t), widen2(r.q.z, t), widen2(r.q.w, t)}};
}

__device__ __forceinline__ uint32_t narrow2(float2 f, const __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float2 f, const __half*) {
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const F8& r) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(r.v[0].x, r.v[0].y, r.v[1].x, r.v[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(r.v[2].x, r.v[2].y, r.v[3].x, r.v[3].y);
  } else {
    const T* t = nullptr;
    *reinterpret_cast<uint4*>(p) =
        make_uint4(narrow2(r.v[0], t), narrow2(r.v[1], t), narrow2(r.v[2], t), narrow2(r.v[3], t));
  }
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
  unsigned positions;  // B * S
  unsigned S;
  int D, R;
  int team_log2;  // log2 of the lanes of a head
  float eps, offset;
  bool w_f32;
};

// Eight weights from column c, with the offset.
template <typename T>
__device__ __forceinline__ F8 weights(const void* w, bool f32, int c, float offset) {
  F8 f;
  if (f32) {
    Raw8<float> r;
    r.load(static_cast<const float*>(w) + c);
    f = widen(r);
  } else {
    Raw8<T> r;
    r.load(static_cast<const T*>(w) + c);
    f = widen(r);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) f.v[j] = __fadd2_rn(f.v[j], both(offset));
  return f;
}

__device__ __forceinline__ float sum_squares(const F8& a, const F8& b) {
  float2 s = __fmul2_rn(a.v[0], a.v[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j) s = __ffma2_rn(a.v[j], a.v[j], s);
#pragma unroll
  for (int j = 0; j < 4; ++j) s = __ffma2_rn(b.v[j], b.v[j], s);
  return s.x + s.y;
}

__device__ __forceinline__ float team_sum(float v, int team) {
  for (int o = team >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What both kernels share: the lane's places in a head, and its walk over
// the items (position, piece of its heads) of its side with the heads of the
// next step on their way while this one's are computed.
template <typename T, bool kGrad>
struct Walk {
  const Side<T>& side;
  const Shape& sh;
  int team, per_warp, slot, a, b;
  bool live, turned;
  unsigned items, stride, item;
  const T *xp, *gp;  // next heads to fetch
  int h;             // the one to fetch
  long long xstep, gstep;
  Raw8<T> x1, x2, g1, g2;

  __device__ __forceinline__ Walk(const Side<T>& side_, const Shape& sh_, unsigned block) : side(side_), sh(sh_) {
    const int lane = threadIdx.x & 31;
    team = 1 << sh.team_log2;
    per_warp = 32 >> sh.team_log2;
    slot = lane >> sh.team_log2;
    const int i = lane & (team - 1);
    live = 16 * i < sh.D;
    turned = 16 * i < sh.R;
    a = turned ? 8 * i : 16 * i;
    b = turned ? sh.R / 2 + 8 * i : 16 * i + 8;
    items = sh.positions * static_cast<unsigned>(side.chunks);
    stride = static_cast<unsigned>(side.blocks) * kWarps;
    item = block * kWarps + (threadIdx.x >> 5);
    xstep = per_warp * side.xh;
    gstep = per_warp * side.gh;
  }

  // Position (batch entry, place in the sequence) and first head of an item.
  __device__ __forceinline__ void place(unsigned it, unsigned& bi, unsigned& si, int& h0) const {
    const unsigned pos = it / static_cast<unsigned>(side.chunks);
    h0 = static_cast<int>(it - pos * side.chunks) * side.iters * per_warp + slot;
    bi = pos / sh.S;
    si = pos - bi * sh.S;
  }

  __device__ __forceinline__ void aim(unsigned bi, unsigned si, int h0) {
    h = h0;
    xp = side.x + bi * side.xb + si * side.xs + h * side.xh + a;
    if (kGrad) gp = side.g + bi * side.gb + si * side.gs + h * side.gh + a;
  }

  __device__ __forceinline__ void fetch() {
    if (live && h < side.H) {
      x1.load(xp);
      x2.load(xp + (b - a));
      if (kGrad) {
        g1.load(gp);
        g2.load(gp + (b - a));
      }
    } else {
      x1.zero();
      x2.zero();
      if (kGrad) {
        g1.zero();
        g2.zero();
      }
    }
    h += per_warp;
    xp += xstep;
    if (kGrad) gp += gstep;
  }
};

// Forward.  With A = (offset + w) cos and B = the partner's (offset + w) sin,
// held for all heads of a position, a pair is r (x1 A1 - x2 B1),
// r (x2 A2 + x1 B2).  One warp per item, grid-stride within a side; the first
// q.blocks blocks serve the queries, the rest the keys.  TC: type of the tables.
template <typename T, typename TC>
__global__ void __launch_bounds__(kThreads, kFwdBlocks)
    qk_norm_rope_fwd_kernel(const __grid_constant__ Side<T> q, const __grid_constant__ Side<T> k,
                            const __grid_constant__ Shape sh) {
  const bool is_q = blockIdx.x < static_cast<unsigned>(q.blocks);
  const Side<T>& side = is_q ? q : k;
  Walk<T, false> w(side, sh, is_q ? blockIdx.x : blockIdx.x - q.blocks);
  if (w.item >= w.items) return;
  const float inv_d = 1.f / static_cast<float>(sh.D);
  unsigned bi, si;
  int h0;
  w.place(w.item, bi, si, h0);
  w.aim(bi, si, h0);
  w.fetch();
  for (;;) {
    F8 a1, a2, b1, b2;
#pragma unroll
    for (int j = 0; j < 4; ++j) a1.v[j] = a2.v[j] = b1.v[j] = b2.v[j] = both(0.f);
    if (w.live) {
      a1 = weights<T>(side.w, sh.w_f32, w.a, sh.offset);
      a2 = weights<T>(side.w, sh.w_f32, w.b, sh.offset);
      if (w.turned) {
        const long long o = bi * sh.cb + si * sh.cs;
        const TC* cp = static_cast<const TC*>(sh.cos) + o;
        const TC* sp = static_cast<const TC*>(sh.sin) + o;
        Raw8<TC> c1, c2, s1, s2;
        c1.load(cp + w.a);
        c2.load(cp + w.b);
        s1.load(sp + w.a);
        s2.load(sp + w.b);
        const F8 fc1 = widen(c1), fc2 = widen(c2), fs1 = widen(s1), fs2 = widen(s2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          b1.v[j] = neg(__fmul2_rn(a2.v[j], fs1.v[j]));
          b2.v[j] = __fmul2_rn(a1.v[j], fs2.v[j]);
          a1.v[j] = __fmul2_rn(a1.v[j], fc1.v[j]);
          a2.v[j] = __fmul2_rn(a2.v[j], fc2.v[j]);
        }
      }
    }
    int hh = h0;
    T* op = side.out + ((static_cast<long long>(bi) * sh.S + si) * side.H + hh) * sh.D + w.a;
    const long long ostep = static_cast<long long>(w.per_warp) * sh.D;
    const bool more = w.items - w.item > w.stride;
    for (int it = side.iters; it > 0; --it) {
      const Raw8<T> r1 = w.x1, r2 = w.x2;
      if (it > 1) {
        w.fetch();
      } else if (more) {
        w.item += w.stride;
        w.place(w.item, bi, si, h0);
        w.aim(bi, si, h0);
        w.fetch();
      }
      const F8 x1 = widen(r1), x2 = widen(r2);
      const float r = rsqrtf(fmaf(team_sum(sum_squares(x1, x2), w.team), inv_d, sh.eps));
      F8 o1, o2;
      if (w.turned) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o1.v[j] = __fmul2_rn(both(r), __ffma2_rn(x1.v[j], a1.v[j], __fmul2_rn(x2.v[j], b1.v[j])));
          o2.v[j] = __fmul2_rn(both(r), __ffma2_rn(x2.v[j], a2.v[j], __fmul2_rn(x1.v[j], b2.v[j])));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o1.v[j] = __fmul2_rn(both(r), __fmul2_rn(x1.v[j], a1.v[j]));
          o2.v[j] = __fmul2_rn(both(r), __fmul2_rn(x2.v[j], a2.v[j]));
        }
      }
      if (w.live && hh < side.H) {
        store8<T>(op, o1);
        store8<T>(op + (w.b - w.a), o2);
      }
      hh += w.per_warp;
      op += ostep;
    }
    if (!more) break;
  }
}

// Backward, on the same items.  kWeights: also leave this block's sum of
// g * n, of its side's weight gradient, in partials[blockIdx.x][D].
template <typename T, typename TC, bool kWeights>
__global__ void __launch_bounds__(kThreads, sizeof(TC) == 4 ? kBwdBlocksWide : kBwdBlocks)
    qk_norm_rope_bwd_kernel(const __grid_constant__ Side<T> q, const __grid_constant__ Side<T> k,
                            const __grid_constant__ Shape sh, float* __restrict__ partials) {
  const bool is_q = blockIdx.x < static_cast<unsigned>(q.blocks);
  const Side<T>& side = is_q ? q : k;
  Walk<T, true> w(side, sh, is_q ? blockIdx.x : blockIdx.x - q.blocks);
  const float inv_d = 1.f / static_cast<float>(sh.D);
  F8 w1, w2, dw1, dw2;
#pragma unroll
  for (int j = 0; j < 4; ++j) w1.v[j] = w2.v[j] = dw1.v[j] = dw2.v[j] = both(0.f);
  if (w.live) {
    w1 = weights<T>(side.w, sh.w_f32, w.a, sh.offset);
    w2 = weights<T>(side.w, sh.w_f32, w.b, sh.offset);
  }
  unsigned bi = 0, si = 0;
  int h0 = 0;
  bool more = w.item < w.items;
  if (more) {
    w.place(w.item, bi, si, h0);
    w.aim(bi, si, h0);
    w.fetch();
  }
  while (more) {
    Raw8<TC> c1r, c2r, s1r, s2r;
    c1r.zero(), c2r.zero(), s1r.zero(), s2r.zero();
    if (w.turned) {
      const long long o = bi * sh.cb + si * sh.cs;
      const TC* cp = static_cast<const TC*>(sh.cos) + o;
      const TC* sp = static_cast<const TC*>(sh.sin) + o;
      c1r.load(cp + w.a);
      c2r.load(cp + w.b);
      s1r.load(sp + w.a);
      s2r.load(sp + w.b);
    }
    int hh = h0;
    T* op = side.out + ((static_cast<long long>(bi) * sh.S + si) * side.H + hh) * sh.D + w.a;
    const long long ostep = static_cast<long long>(w.per_warp) * sh.D;
    more = w.items - w.item > w.stride;
    for (int it = side.iters; it > 0; --it) {
      const Raw8<T> r1 = w.x1, r2 = w.x2, e1 = w.g1, e2 = w.g2;
      if (it > 1) {
        w.fetch();
      } else if (more) {
        w.item += w.stride;
        w.place(w.item, bi, si, h0);
        w.aim(bi, si, h0);
        w.fetch();
      }
      F8 n1 = widen(r1), n2 = widen(r2);
      const float r = rsqrtf(fmaf(team_sum(sum_squares(n1, n2), w.team), inv_d, sh.eps));
      F8 g1 = widen(e1), g2 = widen(e2);
      if (w.turned) {
        c1r.stay(), c2r.stay(), s1r.stay(), s2r.stay();
        const F8 c1 = widen(c1r), c2 = widen(c2r), s1 = widen(s1r), s2 = widen(s2r);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 y1 = g1.v[j], y2 = g2.v[j];
          g1.v[j] = __ffma2_rn(y1, c1.v[j], __fmul2_rn(y2, s2.v[j]));
          g2.v[j] = __ffma2_rn(y2, c2.v[j], neg(__fmul2_rn(y1, s1.v[j])));
        }
      }
      float2 dot = both(0.f);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        n1.v[j] = __fmul2_rn(n1.v[j], both(r));
        n2.v[j] = __fmul2_rn(n2.v[j], both(r));
        if (kWeights) {
          dw1.v[j] = __ffma2_rn(g1.v[j], n1.v[j], dw1.v[j]);
          dw2.v[j] = __ffma2_rn(g2.v[j], n2.v[j], dw2.v[j]);
        }
        g1.v[j] = __fmul2_rn(g1.v[j], w1.v[j]);
        g2.v[j] = __fmul2_rn(g2.v[j], w2.v[j]);
        dot = __ffma2_rn(g1.v[j], n1.v[j], dot);
        dot = __ffma2_rn(g2.v[j], n2.v[j], dot);
      }
      const float m = -team_sum(dot.x + dot.y, w.team) * inv_d;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        n1.v[j] = __fmul2_rn(both(r), __ffma2_rn(n1.v[j], both(m), g1.v[j]));
        n2.v[j] = __fmul2_rn(both(r), __ffma2_rn(n2.v[j], both(m), g2.v[j]));
      }
      if (w.live && hh < side.H) {
        store8<T>(op, n1);
        store8<T>(op + (w.b - w.a), n2);
      }
      hh += w.per_warp;
      op += ostep;
    }
  }
  if (kWeights) {
    // the same column lives in this lane's place of every team of every warp
    __shared__ float red[kWarps][kMaxDim];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      for (int o = w.team; o < 32; o <<= 1) {
        dw1.v[j].x += __shfl_xor_sync(0xffffffffu, dw1.v[j].x, o);
        dw1.v[j].y += __shfl_xor_sync(0xffffffffu, dw1.v[j].y, o);
        dw2.v[j].x += __shfl_xor_sync(0xffffffffu, dw2.v[j].x, o);
        dw2.v[j].y += __shfl_xor_sync(0xffffffffu, dw2.v[j].y, o);
      }
    }
    if (w.slot == 0 && w.live) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float* r = red[threadIdx.x >> 5];
        r[w.a + 2 * j] = dw1.v[j].x, r[w.a + 2 * j + 1] = dw1.v[j].y;
        r[w.b + 2 * j] = dw2.v[j].x, r[w.b + 2 * j + 1] = dw2.v[j].y;
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
