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
//
// 16384 positions x 40 heads of 128 in bf16: forward 57 us (5.9 TB/s),
// backward with the weights' gradients 90 us (5.6 TB/s); 16384 x 24: 35 and
// 52 us (5.8 and 5.8 TB/s).  A plain copy of that size reaches 6.5.
#pragma once

#include "common.cuh"

namespace vq {
namespace qknorm {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 512;  // 32 lanes of 16 values
// Steps of the ring: one being computed, the others on their way (16384
// positions, forward and backward of 32 + 8 heads of 128: 57 and 90 us, with 2
// 55 and 88, with 8 54 and 99; of 16 + 8: 35 and 52, 35 and 55, 38 and 67).
constexpr int kDepth = 4;
// Resident blocks per SM; fp32 heads or tables take twice the registers.
constexpr int kFwdBlocks = 6, kBwdBlocks = 4, kFwdBlocksWide = 4, kBwdBlocksWide = 3;
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

// Eight weights from column c, with the offset (read once a position in the
// forward, where they would take registers from the loop: they are in L1).
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

// Sum over the lanes of a head.  kTeam: log2 of their number, -1: only known at run time.
template <int kTeam>
__device__ __forceinline__ float team_sum(float v, int team_log2) {
  if constexpr (kTeam >= 0) {
#pragma unroll
    for (int o = (1 << kTeam) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  } else {
    for (int o = (1 << team_log2) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

__device__ __forceinline__ void async_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory of a block: kDepth steps of every thread's own values, and for
// a weight gradient each warp's sums of g * n by column.
template <typename T, bool kGrad>
constexpr int kRingBytes = kDepth * (kGrad ? 4 : 2) * 8 * static_cast<int>(sizeof(T)) * kThreads;
constexpr int sums_bytes(int D) { return kWarps * D * static_cast<int>(sizeof(double)); }
// Largest D of which three blocks with the ring of float32 heads fit an SM;
// above, the launch is planned for the two that do (16 + 4 heads of 448,
// 6144 positions: 208 us, planned for three 205; 10240: 333 and 373; 4 + 4
// heads of 512, 10240 positions: 141 and 158).
constexpr int kThreeBlockDim = 352;

// Steps after which a lane's sums of g * n, held in 32 bits, go to its warp's
// in 64: summed in 32 bits to the end their error grew with the batch (1.6e-7
// of the result at 16384 positions, 1e-6 at a million).
constexpr int kFlushSteps = 32;

// What both kernels share: the lane's places in a head, and its walk over
// the items (position, piece of its heads) of its side.  A thread copies the
// values of the steps to come into a ring of its own in shared memory
// (asynchronous copies, read back by the same thread: no barrier), since the
// registers that plain loads ahead would take hold too few bytes in flight:
// at one step ahead the kernels ran at the memory's latency (72 us forward
// for 16384 x 40 heads of 128, 106 us backward).  Lanes past the end of a
// head, and teams past the last head, read one that exists and leave nothing:
// that is cheaper than holding their loads back.
template <typename T, bool kGrad, int kTeam>
struct Walk {
  static constexpr int kVecs = static_cast<int>(sizeof(T)) / 2;  // 16-byte vectors of eight values
  static constexpr uint32_t kStep = (kGrad ? 4 : 2) * kVecs * 16 * kThreads;  // bytes of a step, all threads
  static_assert((kDepth & (kDepth - 1)) == 0, "the ring wraps by masking");
  const Side<T>& side;
  const Shape& sh;
  int team_log2, per_warp, slot, a, b, H, iters;
  bool live, turned;
  // Where an item lies: its piece of the position's heads, and the position
  // (place in the sequence, batch entry); kept by additions, since a division
  // an item cost more than its heads' arithmetic.
  struct At {
    unsigned item, c, s, b;
  };
  At at, by, ahead;  // of the current item, of a stride, of the item to copy next
  unsigned items, chunks, S;
  int f_left, f_h;
  const T *xp, *gp;  // heads of the position to copy next, at this lane's place
  long long xh, gh;
  uint32_t ring, f_off, r_off;
  const uint8_t* ring_p;

  __device__ __forceinline__ Walk(const Side<T>& side_, const Shape& sh_, unsigned block, uint8_t* smem)
      : side(side_), sh(sh_) {
    const int lane = threadIdx.x & 31;
    team_log2 = kTeam >= 0 ? kTeam : sh.team_log2;
    per_warp = 32 >> team_log2;
    slot = lane >> team_log2;
    const int i = lane & ((1 << team_log2) - 1);
    live = 16 * i < sh.D;
    turned = 16 * i < sh.R;
    a = turned ? 8 * i : live ? 16 * i : 0;
    b = turned ? sh.R / 2 + 8 * i : a + 8;
    H = side.H;
    iters = side.iters;
    xh = side.xh;
    gh = side.gh;
    S = sh.S;
    chunks = static_cast<unsigned>(side.chunks);
    items = sh.positions * chunks;
    by = place(static_cast<unsigned>(side.blocks) * kWarps);
    // one value a warp, in the open, lets the compiler branch on it without masks
    at = place(block * kWarps + __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0));
    ahead = at;
    ring_p = smem + 16 * threadIdx.x;
    ring = smem_u32(ring_p);
    f_off = r_off = 0;
    f_left = 0;
    if (at.item < items) aim();
#pragma unroll
    for (int s = 0; s < kDepth - 1; ++s) copy_step();
  }

  __device__ __forceinline__ At place(unsigned item) const {
    At p;
    p.item = item;
    const unsigned pos = chunks > 1 ? item / chunks : item;
    p.c = item - pos * chunks;
    p.b = pos / S;
    p.s = pos - p.b * S;
    return p;
  }
  // Moves an item on by the stride; false at the end.
  __device__ __forceinline__ bool next(At& p) const {
    if (items - p.item <= by.item) return false;
    p.item += by.item;
    p.c += by.c;
    p.s += by.s;
    p.b += by.b;
    if (p.c >= chunks) {
      p.c -= chunks;
      ++p.s;
    }
    if (p.s >= S) {
      p.s -= S;
      ++p.b;
    }
    return true;
  }
  __device__ __forceinline__ int first_head(const At& p) const { return static_cast<int>(p.c) * iters * per_warp + slot; }

  __device__ __forceinline__ void aim() {
    f_h = first_head(ahead);
    xp = side.x + ahead.b * side.xb + ahead.s * side.xs + a;
    if (kGrad) gp = side.g + ahead.b * side.gb + ahead.s * side.gs + a;
    f_left = iters;
  }

  __device__ __forceinline__ void copy8(int part, const T* p) {
    const uint32_t d = ring + f_off + part * (16 * kThreads);
    async_copy16(d, p);
    if (kVecs == 2) async_copy16(d + 16 * kThreads, p + 4);
  }

  // Starts the copies of the next step, if there is one; a group either way.
  __device__ __forceinline__ void copy_step() {
    if (f_left > 0) {
      const int h = min(f_h, H - 1);
      const T* p = xp + h * xh;
      copy8(0, p);
      copy8(kVecs, p + (b - a));
      if (kGrad) {
        const T* e = gp + h * gh;
        copy8(2 * kVecs, e);
        copy8(3 * kVecs, e + (b - a));
      }
      f_h += per_warp;
      if (--f_left == 0 && next(ahead)) aim();
    }
    async_commit();
    f_off = (f_off + kStep) & (kDepth * kStep - 1);
  }

  __device__ __forceinline__ F8 read8(int part) const {
    const uint8_t* p = ring_p + r_off + part * (16 * kThreads);
    Raw8<T> r;
    if constexpr (kVecs == 2) {
      r.a = *reinterpret_cast<const float4*>(p);
      r.b = *reinterpret_cast<const float4*>(p + 16 * kThreads);
    } else {
      r.q = *reinterpret_cast<const uint4*>(p);
    }
    return widen(r);
  }

  // Makes the current step's values readable (read8) after starting those of a later one.
  __device__ __forceinline__ void arrive() {
    copy_step();
    async_wait<kDepth - 1>();
  }
  __device__ __forceinline__ void leave() { r_off = (r_off + kStep) & (kDepth * kStep - 1); }
};

// Forward.  With A = (offset + w) cos and B = the partner's (offset + w) sin,
// held for all heads of a position, a pair is r (x1 A1 - x2 B1),
// r (x2 A2 + x1 B2).  One warp per item, grid-stride within a side; the first
// q.blocks blocks serve the queries, the rest the keys.  TC: type of the tables.
template <typename T, typename TC, int kTeam>
__global__ void __launch_bounds__(kThreads, sizeof(TC) == 4 ? kFwdBlocksWide : kFwdBlocks)
    qk_norm_rope_fwd_kernel(const __grid_constant__ Side<T> q, const __grid_constant__ Side<T> k,
                            const __grid_constant__ Shape sh) {
  extern __shared__ __align__(16) uint8_t qsmem[];
  const bool is_q = blockIdx.x < static_cast<unsigned>(q.blocks);
  const Side<T>& side = is_q ? q : k;
  Walk<T, false, kTeam> w(side, sh, is_q ? blockIdx.x : blockIdx.x - q.blocks, qsmem);
  const float inv_d = 1.f / static_cast<float>(sh.D), eps = sh.eps;
  const long long ostep = static_cast<long long>(w.per_warp) * sh.D;
  bool more = w.at.item < w.items;
  while (more) {
    const unsigned bi = w.at.b, si = w.at.s;
    int h = w.first_head(w.at);
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
    T* op = side.out + ((static_cast<long long>(bi) * sh.S + si) * w.H + h) * sh.D + w.a;
    more = w.next(w.at);
#pragma unroll 1
    for (int it = w.iters; it > 0; --it) {
      w.arrive();
      const F8 x1 = w.read8(0), x2 = w.read8(w.kVecs);
      w.leave();
      const float ss = w.live ? sum_squares(x1, x2) : 0.f;
      const float r = rsqrtf(fmaf(team_sum<kTeam>(ss, w.team_log2), inv_d, eps));
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
      if (w.live && h < w.H) {
        store8<T>(op, o1);
        store8<T>(op + (w.b - w.a), o2);
      }
      h += w.per_warp;
      op += ostep;
    }
  }
}

// Backward, on the same items.  kWeights: also leave this block's sum of
// g * n, of its side's weight gradient, in partials[blockIdx.x][D].  A lane
// adds at most kFlushSteps - 1 and one item's steps in 32 bits.
template <typename T, typename TC, bool kWeights, int kTeam>
__global__ void __launch_bounds__(kThreads, sizeof(TC) == 4 ? kBwdBlocksWide : kBwdBlocks)
    qk_norm_rope_bwd_kernel(const __grid_constant__ Side<T> q, const __grid_constant__ Side<T> k,
                            const __grid_constant__ Shape sh, float* __restrict__ partials) {
  extern __shared__ __align__(16) uint8_t qsmem[];
  const bool is_q = blockIdx.x < static_cast<unsigned>(q.blocks);
  const Side<T>& side = is_q ? q : k;
  Walk<T, true, kTeam> w(side, sh, is_q ? blockIdx.x : blockIdx.x - q.blocks, qsmem);
  const float inv_d = 1.f / static_cast<float>(sh.D), eps = sh.eps;
  const long long ostep = static_cast<long long>(w.per_warp) * sh.D;
  F8 w1, w2, dw1, dw2;
#pragma unroll
  for (int j = 0; j < 4; ++j) w1.v[j] = w2.v[j] = dw1.v[j] = dw2.v[j] = both(0.f);
  if (w.live) {
    w1 = weights<T>(side.w, sh.w_f32, w.a, sh.offset);
    w2 = weights<T>(side.w, sh.w_f32, w.b, sh.offset);
  }
  // this warp's sums; a column is the first team's lane's that holds it
  double* sums = reinterpret_cast<double*>(qsmem + kRingBytes<T, true>) + (threadIdx.x >> 5) * sh.D;
  const bool keeps = w.slot == 0 && w.live;
  if (kWeights && keeps) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[w.a + j] = sums[w.b + j] = 0.0;
  }
  auto flush = [&] {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      for (int o = 1 << w.team_log2; o < 32; o <<= 1) {
        dw1.v[j].x += __shfl_xor_sync(0xffffffffu, dw1.v[j].x, o);
        dw1.v[j].y += __shfl_xor_sync(0xffffffffu, dw1.v[j].y, o);
        dw2.v[j].x += __shfl_xor_sync(0xffffffffu, dw2.v[j].x, o);
        dw2.v[j].y += __shfl_xor_sync(0xffffffffu, dw2.v[j].y, o);
      }
      if (keeps) {
        sums[w.a + 2 * j] += dw1.v[j].x, sums[w.a + 2 * j + 1] += dw1.v[j].y;
        sums[w.b + 2 * j] += dw2.v[j].x, sums[w.b + 2 * j + 1] += dw2.v[j].y;
      }
      dw1.v[j] = dw2.v[j] = both(0.f);
    }
  };
  int steps = 0;
  bool more = w.at.item < w.items;
  while (more) {
    const unsigned bi = w.at.b, si = w.at.s;
    int h = w.first_head(w.at);
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
    T* op = side.out + ((static_cast<long long>(bi) * sh.S + si) * w.H + h) * sh.D + w.a;
    more = w.next(w.at);
#pragma unroll 1
    for (int it = w.iters; it > 0; --it) {
      w.arrive();
      F8 n1 = w.read8(0), n2 = w.read8(w.kVecs), g1 = w.read8(2 * w.kVecs), g2 = w.read8(3 * w.kVecs);
      w.leave();
      const float ss = w.live ? sum_squares(n1, n2) : 0.f;
      const float r = rsqrtf(fmaf(team_sum<kTeam>(ss, w.team_log2), inv_d, eps));
      const bool counts = h < w.H;  // a team past the last head adds nothing to the weights' sum, not even inf * 0
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
        if (kWeights && counts) {
          dw1.v[j] = __ffma2_rn(g1.v[j], n1.v[j], dw1.v[j]);
          dw2.v[j] = __ffma2_rn(g2.v[j], n2.v[j], dw2.v[j]);
        }
        g1.v[j] = __fmul2_rn(g1.v[j], w1.v[j]);
        g2.v[j] = __fmul2_rn(g2.v[j], w2.v[j]);
        dot = __ffma2_rn(g1.v[j], n1.v[j], dot);
        dot = __ffma2_rn(g2.v[j], n2.v[j], dot);
      }
      const float m = -team_sum<kTeam>(w.live ? dot.x + dot.y : 0.f, w.team_log2) * inv_d;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        n1.v[j] = __fmul2_rn(both(r), __ffma2_rn(n1.v[j], both(m), g1.v[j]));
        n2.v[j] = __fmul2_rn(both(r), __ffma2_rn(n2.v[j], both(m), g2.v[j]));
      }
      if (w.live && h < w.H) {
        store8<T>(op, n1);
        store8<T>(op + (w.b - w.a), n2);
      }
      h += w.per_warp;
      op += ostep;
    }
    if (kWeights && (steps += w.iters) >= kFlushSteps) {
      flush();
      steps = 0;
    }
  }
  if (kWeights) {
    flush();
    __syncthreads();
    const double* all = reinterpret_cast<const double*>(qsmem + kRingBytes<T, true>);
    for (int c = threadIdx.x; c < sh.D; c += kThreads) {
      double t = 0.0;
#pragma unroll
      for (int v = 0; v < kWarps; ++v) t += all[v * sh.D + c];
      partials[static_cast<long long>(blockIdx.x) * sh.D + c] = static_cast<float>(t);
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
