// Global norm of many gradients and their clipping in place (HBM-bandwidth
// bound; for a few hundred tensors of a few values, launch bound).
//
//   norm = sqrt(sum over tensors of sum g^2)  or  max |g|
//   g   *= min(1, max_norm / (norm + 1e-6))
//
// Pass 1 leaves one 64-bit partial per block; pass 2 joins the partials in
// every block in the same order, so the result does not depend on which
// block ends first, and scales.  The tensors come as kernel parameters: no
// copy of a descriptor table to the device, and a captured graph holds its
// own.  A tensor is walked in chunks of 32 KB of the address range, so vector
// loads are aligned whatever the tensor's first address is; a chunk that lies
// in its tensor as a whole takes a path without any check of its own.
#pragma once

#include "common.cuh"

namespace vq {
namespace clip {

constexpr int kThreads = 256;
constexpr int kChunkBytes = 32768;  // 8 vectors of 16 bytes per thread
constexpr int kVecs = kChunkBytes / (16 * kThreads);
// Resident blocks per SM of the two passes.  0.59 G bf16 values: the norm takes
// 167 us with 4, 171 with 3, 204 with 6, and behind a pass that scaled, whose
// last writes are still on their way to memory, 195, 188 and 211; the scaling
// 382 us with 3, 388 with 4, 371 with 2, 462 with 1.
constexpr int kBlocksPerSm = 4, kScaleBlocksPerSm = 3;
constexpr int kSmallThreads = 1024;
constexpr int kSmallChunkBytes = 512;
constexpr int kMaxBlocks = 1024;  // of one launch: the partials it leaves

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// The parameter space of a launch is 32764 bytes; the short table serves the
// usual few hundred tensors without copying all of it on every launch (226 of
// six values: 4.9 us on the device, with the long table 5.1).
constexpr int kShortTable = 240;
constexpr int kLongTable = 1536;

template <int N>
struct Table {
  uintptr_t ptr[N];    // first byte
  long long bytes[N];  // of the tensor
  int first_chunk[N];  // chunks of the tensors before it
  uint8_t dtype[N / 8 * 8 + 8];
  int n;
  int chunks;  // in all
};

__device__ __forceinline__ int esize(int dtype) { return dtype == kF32 ? 4 : 2; }

// Values of a 16-byte vector (8 of 16 bits; 4 of 32).
template <int kType>
struct Values {
  static constexpr int kCount = kType == kF32 ? 4 : 8;
  float f[kCount];
  __device__ __forceinline__ explicit Values(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kType == kF32) {
        f[i] = __uint_as_float(w[i]);
      } else if constexpr (kType == kBF16) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
  __device__ __forceinline__ uint4 scaled(float s) const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kType == kF32) {
        w[i] = __float_as_uint(f[i] * s);
      } else if constexpr (kType == kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i] * s, f[2 * i + 1] * s);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(f[2 * i] * s, f[2 * i + 1] * s);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ float load_one(uintptr_t p, int dtype) {
  if (dtype == kF32) return *reinterpret_cast<const float*>(p);
  if (dtype == kBF16) return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
  return __half2float(*reinterpret_cast<const __half*>(p));
}

__device__ __forceinline__ void store_one(uintptr_t p, int dtype, float v) {
  if (dtype == kF32)
    *reinterpret_cast<float*>(p) = v;
  else if (dtype == kBF16)
    *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(v);
  else
    *reinterpret_cast<__half*>(p) = __float2half_rn(v);
}

// Joins one value into a partial: the sum of squares, or the largest
// magnitude with a NaN kept.
template <bool kMax>
__device__ __forceinline__ double join(double acc, double v) {
  if (!kMax) return acc + v;
  return (acc > v || acc != acc) ? acc : v;
}

template <bool kMax>
__device__ __forceinline__ double one(float f) {
  return kMax ? static_cast<double>(fabsf(f)) : static_cast<double>(f) * static_cast<double>(f);
}

// A vector's share.  The squares of a vector are summed in fp32, which holds
// them to 2^-21 (eight sums, each rounded by 2^-24 at most), and joined in 64
// bits; where that sum leaves the range that
// fp32 squares keep their precision in, it is taken in 64 bits instead.
template <bool kMax, int kType>
__device__ __forceinline__ double of_vec(const uint4& v) {
  const Values<kType> x(v);
  if (kMax) {
    float m = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < x.kCount; ++i) {
      m = fmaxf(m, fabsf(x.f[i]));
      nan |= x.f[i] != x.f[i];
    }
    return static_cast<double>(nan ? __int_as_float(0x7fffffff) : m);
  }
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < x.kCount; ++i) s = fmaf(x.f[i], x.f[i], s);
  if (s > 1e-26f && s < 1e37f) return static_cast<double>(s);
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < x.kCount; ++i) d += static_cast<double>(x.f[i]) * static_cast<double>(x.f[i]);
  return d;
}

// Sum (or maximum) over the block in a fixed order; every thread gets it.
template <bool kMax>
__device__ __forceinline__ double block_join(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join<kMax>(v, __shfl_down_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x) / 32; ++w) t = join<kMax>(t, red[w]);
  return t;
}

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& tab, int chunk) {
  int lo = 0, hi = tab.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first_chunk[mid] <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// Address range [b, e) of a chunk, its tensor's type, and the vectors' base.
struct Chunk {
  uintptr_t base, b, e;
  int dtype;
  __device__ __forceinline__ bool whole() const { return b == base && e == base + kChunkBytes; }
};

template <int N>
__device__ __forceinline__ Chunk chunk_at(const Table<N>& tab, int chunk) {
  const int t = tensor_of(tab, chunk);
  const uintptr_t p = tab.ptr[t], end = p + static_cast<uintptr_t>(tab.bytes[t]);
  Chunk c;
  c.base = (p & ~uintptr_t(15)) + static_cast<uintptr_t>(chunk - tab.first_chunk[t]) * kChunkBytes;
  c.b = c.base > p ? c.base : p;
  c.e = c.base + kChunkBytes < end ? c.base + kChunkBytes : end;
  c.dtype = tab.dtype[t];
  return c;
}

__device__ __forceinline__ float clip_scale(double total, bool is_max, float max_norm, float* norm) {
  const float nf = static_cast<float>(is_max ? total : sqrt(total));
  *norm = nf;
  const float s = max_norm / (nf + 1e-6f);
  return s < 1.f || s != s ? s : 1.f;
}

// The share of this thread's vectors of a chunk.
template <bool kMax, int kType>
__device__ __forceinline__ double norm_of_chunk(const Chunk& c) {
  const uint4* p = reinterpret_cast<const uint4*>(c.base) + threadIdx.x;
  double acc = 0.0;
  if (c.whole()) {
    uint4 v[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) v[j] = __ldg(p + j * kThreads);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) acc = join<kMax>(acc, of_vec<kMax, kType>(v[j]));
    return acc;
  }
  constexpr int kSize = kType == kF32 ? 4 : 2;
  for (int j = 0; j < kVecs; ++j) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p + j * kThreads);
    if (a >= c.b && a + 16 <= c.e) {
      acc = join<kMax>(acc, of_vec<kMax, kType>(*reinterpret_cast<const uint4*>(a)));
    } else {  // a vector that the tensor shares with a neighbour
      for (uintptr_t e = a; e < a + 16; e += kSize)
        if (e >= c.b && e + kSize <= c.e) acc = join<kMax>(acc, one<kMax>(load_one(e, kType)));
    }
  }
  return acc;
}

template <int kType>
__device__ __forceinline__ void scale_chunk(const Chunk& c, float s) {
  uint4* p = reinterpret_cast<uint4*>(c.base) + threadIdx.x;
  if (c.whole()) {
    uint4 v[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) v[j] = p[j * kThreads];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const uint4 w = Values<kType>(v[j]).scaled(s);
      // Not written where no value changed, as for 16-bit values and a factor within about 2^-9 of 1 (0.59 G bf16
      // values, both passes: 577 us for 0.9 either way; a factor that changes no value 330, not 577)
      if (((w.x ^ v[j].x) | (w.y ^ v[j].y) | (w.z ^ v[j].z) | (w.w ^ v[j].w)) != 0) p[j * kThreads] = w;
    }
    return;
  }
  constexpr int kSize = kType == kF32 ? 4 : 2;
  for (int j = 0; j < kVecs; ++j) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p + j * kThreads);
    if (a >= c.b && a + 16 <= c.e) {
      uint4* q = reinterpret_cast<uint4*>(a);
      *q = Values<kType>(*q).scaled(s);
    } else {
      for (uintptr_t e = a; e < a + 16; e += kSize)
        if (e >= c.b && e + kSize <= c.e) store_one(e, kType, load_one(e, kType) * s);
    }
  }
}

template <int N, bool kMax>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) norm_kernel(const __grid_constant__ Table<N> tab,
                                                                      double* __restrict__ partials) {
  __shared__ double red[kThreads / 32];
  double acc = 0.0;
  for (int chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
    const Chunk c = chunk_at(tab, chunk);
    acc = join<kMax>(acc, c.dtype == kF32    ? norm_of_chunk<kMax, kF32>(c)
                          : c.dtype == kBF16 ? norm_of_chunk<kMax, kBF16>(c)
                                             : norm_of_chunk<kMax, kF16>(c));
  }
  acc = block_join<kMax>(acc, red);
  if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// Walks the chunks from the last to the first: what pass 1 read last is
// still in L2.
template <int N, bool kMax>
__global__ void __launch_bounds__(kThreads, kScaleBlocksPerSm)
    scale_kernel(const __grid_constant__ Table<N> tab, const double* __restrict__ partials, int num_partials,
                 float max_norm, bool scale, float* __restrict__ norm_out) {
  __shared__ double red[kThreads / 32];
  double acc = 0.0;
  for (int i = threadIdx.x; i < num_partials; i += kThreads) acc = join<kMax>(acc, partials[i]);
  float norm;
  const float s = clip_scale(block_join<kMax>(acc, red), kMax, max_norm, &norm);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) *norm_out = norm;
  if (!scale || s == 1.f) return;  // nothing changes
  for (int chunk = tab.chunks - 1 - static_cast<int>(blockIdx.x); chunk >= 0; chunk -= gridDim.x) {
    const Chunk c = chunk_at(tab, chunk);
    if (c.dtype == kF32)
      scale_chunk<kF32>(c, s);
    else if (c.dtype == kBF16)
      scale_chunk<kBF16>(c, s);
    else
      scale_chunk<kF16>(c, s);
  }
}

// Few values in all: one block takes the norm and scales, in one launch.  A
// warp per piece of kSmallChunkBytes of a tensor: tensors of a few values (a
// layer's gates) take a warp each, one of some thousand is spread over all.
template <int N, class Op>
__device__ __forceinline__ void small_pieces(const Table<N>& tab, Op op) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int c = warp; c < tab.chunks; c += kSmallThreads / 32) {
    const int t = tab.chunks == tab.n ? c : tensor_of(tab, c);
    const int dt = tab.dtype[t], es = esize(dt);
    const long long at = static_cast<long long>(c - tab.first_chunk[t]) * kSmallChunkBytes;
    const long long left = tab.bytes[t] - at;
    const uintptr_t b = tab.ptr[t] + static_cast<uintptr_t>(at);
    const uintptr_t e = b + static_cast<uintptr_t>(left < kSmallChunkBytes ? left : kSmallChunkBytes);
#pragma unroll 4
    for (uintptr_t a = b + lane * es; a < e; a += 32 * es) op(a, dt);
  }
}

template <int N, bool kMax>
__global__ void __launch_bounds__(kSmallThreads) small_kernel(const __grid_constant__ Table<N> tab, float max_norm,
                                                              bool scale, float* __restrict__ norm_out) {
  __shared__ double red[kSmallThreads / 32];
  double acc = 0.0;
  small_pieces(tab, [&](uintptr_t a, int dt) { acc = join<kMax>(acc, one<kMax>(load_one(a, dt))); });
  float norm;
  const float s = clip_scale(block_join<kMax>(acc, red), kMax, max_norm, &norm);
  if (threadIdx.x == 0 && norm_out != nullptr) *norm_out = norm;
  if (!scale || s == 1.f) return;
  small_pieces(tab, [&](uintptr_t a, int dt) { store_one(a, dt, load_one(a, dt) * s); });
}

}  // namespace clip
}  // namespace vq
