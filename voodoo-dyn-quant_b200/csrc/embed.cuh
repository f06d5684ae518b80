// Lookup of token rows in a gated embedding (the mixture of K packed
// candidates), and the gradient of the mixture's probabilities.
//
//   out[t]  = scale * sum_k p_k W_k[id_t]
//   dL/dp_k = scale * sum_t <dy_t, W_k[id_t]>
//           = scale * sum over runs of equal id of <sum of the run's dy, W_k[id]>
//
// Neither writes a decoded row of a candidate: the lookup decodes and mixes a
// token's packed rows in registers, the gradient sums the rows of dy of equal
// tokens first (token_plan_kernel brings them together) and multiplies the
// decoded weights into that sum as it decodes them.  Both are bound by HBM
// (packed rows, and T x D of out or dy), closely followed by the decoding.
//
// Eight lanes hold a unit (256 weights) of a row, a lane 32 consecutive
// weights.  The lanes of a unit copy its packed bytes of every candidate into
// their own slots of shared memory (16-byte asynchronous copies), so that no
// block-wide barrier is needed; the SM's other warps decode meanwhile.
#pragma once

#include <type_traits>

#include "decode_mix.cuh"

namespace vq {
namespace embed {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnits = 4;   // units of a warp
#ifndef VQ_EMBED_MIX_BLOCKS
#define VQ_EMBED_MIX_BLOCKS 3
#endif
#ifndef VQ_EMBED_GRAD_BLOCKS
#define VQ_EMBED_GRAD_BLOCKS 3
#endif
constexpr int kMixBlocks = VQ_EMBED_MIX_BLOCKS, kGradBlocks = VQ_EMBED_GRAD_BLOCKS;  // resident per SM
constexpr int kMaxBlocks = 1184;  // of a gradient launch: the partials it leaves

// A unit's slot: the 16-byte aligned span of a 2-byte aligned unit, and a
// word more for the field reads that join two words.
__host__ __device__ inline int slot_bytes(int ub) { return ((ub + 14 + 15) & ~15) + 16; }
__host__ __device__ inline int warp_bytes(const CandSet& cs) {
  int s = 0;
  for (int k = 0; k < cs.K; ++k) s += kUnits * slot_bytes(cs.ubytes[k]);
  return s;
}

__device__ __forceinline__ void async_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Copies unit `unit` (of the whole table) of every candidate into slot `lu`
// of the warp's buffer; lane c of the unit's eight takes every eighth vector
// (18 at most: a Q8_0 unit that starts inside a vector).
__device__ __forceinline__ void stage_unit(const CandSet& cs, uint32_t buf, int lu, int c, long long unit) {
  for (int k = 0; k < cs.K; ++k) {
    const int ub = cs.ubytes[k], slot = slot_bytes(ub);
    const uint8_t* a = cs.ptr[k] + unit * ub;
    const int rel = static_cast<int>(reinterpret_cast<uintptr_t>(a) & 15u);
    const uint8_t* src = a - rel + 16 * c;
    const uint32_t dst = buf + lu * slot + 16 * c;
    const int left = rel + ub - 16 * c;  // bytes from this lane's first vector on
    if (left > 0) async_copy16(dst, src);
    if (left > 128) async_copy16(dst + 128, src + 128);
    if (left > 256) async_copy16(dst + 256, src + 256);
    buf += kUnits * slot;
  }
}

// The staged unit of candidate k, whose slots start at `region`; `unit` modulo 2^32.
__device__ __forceinline__ URef staged(const CandSet& cs, const uint8_t* region, int k, int lu, uint32_t unit) {
  const int ub = cs.ubytes[k];
  const uint32_t rel = (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(cs.ptr[k])) + unit * ub) & 15u;
  return URef{reinterpret_cast<const uint32_t*>(region + lu * slot_bytes(ub) + (rel & ~3u)), static_cast<int>(rel & 3u),
              8u * (rel & 3u)};
}

struct Ids {
  const void* p;
  bool i32;
  __device__ __forceinline__ long long at(long long i) const {
    return i32 ? static_cast<long long>(static_cast<const int*>(p)[i]) : static_cast<const long long*>(p)[i];
  }
};

// Row of this table that token id names, or -1.
__device__ __forceinline__ long long local_row(long long id, long long vocab_start, long long rows) {
  const long long r = id - vocab_start;
  return r >= 0 && r < rows ? r : -1;
}

// The tokens of a call in the order of their rows, cut into pieces of equal
// rows (token_plan_kernel): piece i holds the tokens order[start[i]] to
// order[start[i + 1] - 1], all naming row key[i].
struct Plan {
  int *order, *start, *key, *count;
};

// Most tokens of a piece: a token that fills much of a batch is then worked
// on by many warps, each decoding its row again.
constexpr int kPieceTokens = 16;

// The units that eight lanes work on one after the other: unit u of piece
// (kRuns) or token i, i * units_per_row + u ascending by a fixed stride.
template <bool kRuns>
struct UnitWalk {
  Plan plan;
  Ids ids;
  int count;  // pieces, or tokens
  long long vocab_start;
  int rows, units_per_row;
  int i, di, u, du;

  __device__ __forceinline__ void start_at(long long first, long long stride) {
    i = static_cast<int>(first / units_per_row);
    u = static_cast<int>(first - static_cast<long long>(i) * units_per_row);
    di = static_cast<int>(stride / units_per_row);
    du = static_cast<int>(stride - static_cast<long long>(di) * units_per_row);
  }
  __device__ __forceinline__ bool on() const { return i < count; }
  __device__ __forceinline__ void step() {
    i += di;
    u += du;
    if (u >= units_per_row) {
      u -= units_per_row;
      ++i;
    }
  }
  // Row of the table, or -1 for a token of another one.
  __device__ __forceinline__ int row() const {
    if (!on()) return -1;
    if (!kRuns) return static_cast<int>(local_row(ids.at(i), vocab_start, rows));
    const int key = plan.key[i];
    return key < rows ? key : -1;
  }
};

// ---------------------------------------------------------------- lookup
// Rows of ids outside [vocab_start, vocab_start + rows) are written as zeros
// (another shard's tokens); `strict` also reports them.  The mixture is
// mix_units_kernel's, in the same order, so for scale 1 the rows are those of
// W_mix bit for bit; the scaled row is rounded to bf16 once.  kRuns: each row
// is decoded once per piece of the plan and written to all its tokens;
// otherwise once per token, with no plan to wait for.
template <bool kRuns>
__global__ void __launch_bounds__(kThreads, kMixBlocks)
    embed_mix_kernel(const __grid_constant__ CandSet cs, const float* __restrict__ probs, Ids ids, int T, Plan plan,
                     long long vocab_start, int rows, int units_per_row, int cols, float scale, bool strict, bool vec,
                     __nv_bfloat16* __restrict__ out, long long ldo, int* err) {
  extern __shared__ __align__(16) uint8_t esmem[];
  __shared__ float pk_s[kMaxCandidates];
  if (threadIdx.x < cs.K) pk_s[threadIdx.x] = probs[threadIdx.x];
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lu = lane >> 3, c = lane & 7;
  uint8_t* buf = esmem + warp * warp_bytes(cs);
  UnitWalk<kRuns> w{plan, ids, kRuns ? *plan.count : T, vocab_start, rows, units_per_row};
  w.start_at((static_cast<long long>(blockIdx.x) * kWarps + warp) * kUnits + lu,
             static_cast<long long>(gridDim.x) * kWarps * kUnits);
  bool bad = false, fmt_ok = true;
  for (; __any_sync(0xffffffffu, w.on()); w.step()) {
    const int row = w.row();
    const long long unit = static_cast<long long>(row) * units_per_row + w.u;
    if (row >= 0) stage_unit(cs, smem_u32(buf), lu, c, unit);
    async_commit();
    float2 acc[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = make_float2(0.f, 0.f);
    float cst[2] = {0.f, 0.f};
    const int col = 256 * w.u + 32 * c;
    async_wait<0>();
    __syncwarp();
    if (row >= 0 && col < cols) {
      const uint8_t* region = buf;
      for (int k = 0; k < cs.K; ++k) {
        const URef ur = staged(cs, region, k, lu, static_cast<uint32_t>(unit));
        const float pk = pk_s[k];
        switch (cs.fmt[k]) {
          case kQ8_0: mix_chunk<kQ8_0>(ur, c, pk, acc, cst); break;
          case kQ2_K: mix_chunk<kQ2_K>(ur, c, pk, acc, cst); break;
          case kQ3_K: mix_chunk<kQ3_K>(ur, c, pk, acc, cst); break;
          case kQ4_K: mix_chunk<kQ4_K>(ur, c, pk, acc, cst); break;
          case kQ5_K: mix_chunk<kQ5_K>(ur, c, pk, acc, cst); break;
          case kQ6_K: mix_chunk<kQ6_K>(ur, c, pk, acc, cst); break;
          case kIQ4_XS: mix_chunk<kIQ4_XS>(ur, c, pk, acc, cst); break;
          default: fmt_ok = false;
        }
        region += kUnits * slot_bytes(cs.ubytes[k]);
      }
    }
    if (w.on()) {
      bad |= row < 0;
      if (col < cols) {
        __align__(16) __nv_bfloat162 hv[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float cs0 = cst[j >> 3];
          hv[j] = __floats2bfloat162_rn((acc[j].x + cs0) * scale, (acc[j].y + cs0) * scale);
        }
        const int begin = kRuns ? plan.start[w.i] : w.i, end = kRuns ? plan.start[w.i + 1] : w.i + 1;
        for (int i = begin; i < end; ++i) {
          __nv_bfloat16* dst = out + static_cast<long long>(kRuns ? plan.order[i] : i) * ldo + col;
          if (vec && col + 32 <= cols) {
#pragma unroll
            for (int v = 0; v < 4; ++v) reinterpret_cast<uint4*>(dst)[v] = reinterpret_cast<const uint4*>(hv)[v];
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (col + 2 * j < cols) dst[2 * j] = hv[j].x;
              if (col + 2 * j + 1 < cols) dst[2 * j + 1] = hv[j].y;
            }
          }
        }
      }
    }
    __syncwarp();  // the slots are filled again
  }
  if (bad && strict) report_error(err, kDevBadIndex, 30);
  if (!fmt_ok) report_error(err, kDevBadFormat, 3);
}

// ---------------------------------------------------------------- plan
// Stable radix sort of the tokens' local rows by one cluster, nine bits a
// pass, and the pieces of equal rows.  Tokens of other shards get the key
// `rows` and so end up last.  Each CTA owns a contiguous slice of a pass's
// input and ranks it a tile of 1024 tokens at a time: within a warp by
// matching digits, over the warps and tiles by counts; the slices' counts
// meet through distributed shared memory.  Latency bound: a dozen barriers
// and the round trips between them.
constexpr int kSortThreads = 1024;
constexpr int kSortCtas = 8;  // largest portable cluster
constexpr int kDigitBits = 9;
constexpr int kBins = 1 << kDigitBits;
constexpr int kSortSmem = 32 * kBins * 2;
constexpr int kKeepTiles = 2;  // tiles whose keys and ranks stay in registers between the two halves of a pass

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__global__ void __launch_bounds__(kSortThreads) token_plan_kernel(Ids ids, int T, long long vocab_start, int rows,
                                                                  int passes, Plan plan, int* keys, int* keys_tmp,
                                                                  int* order_tmp) {
  extern __shared__ __align__(16) uint8_t ssmem[];
  uint16_t* wcount = reinterpret_cast<uint16_t*>(ssmem);  // [32 warps][kBins]
  __shared__ int count[kBins];                            // this slice's tokens of each digit, so far
  __shared__ int base[kBins];
  __shared__ int wsum[32];
  __shared__ int pieces;
  int* order = plan.order;
  int* ranks = plan.start;  // free until the pieces are written
  uint32_t nctas;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(nctas));
  const int rank = static_cast<int>(cluster_ctarank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slice = (T + static_cast<int>(nctas) - 1) / static_cast<int>(nctas);
  const int b = min(T, rank * slice), e = min(T, b + slice);
  for (int p = 0; p < passes; ++p) {
    const bool to_tmp = ((passes - 1 - p) & 1) != 0;
    const int* ksrc = to_tmp ? keys : keys_tmp;
    const int* osrc = to_tmp ? order : order_tmp;
    int* kdst = to_tmp ? keys_tmp : keys;
    int* odst = to_tmp ? order_tmp : order;
    const int shift = p * kDigitBits;
    auto key_at = [&](int i) -> int {
      if (p > 0) return __ldcg(ksrc + i);  // another CTA wrote it: from L2
      const long long r = local_row(ids.at(i), vocab_start, rows);
      return r < 0 ? rows : static_cast<int>(r);
    };
    auto digit = [&](int key) { return (key >> shift) & (kBins - 1); };
    // place of token i among this slice's tokens of the same digit
    auto rank_of = [&](bool in, int key) -> int {
      const int d = in ? digit(key) : kBins;  // no digit
      uint4* mine = reinterpret_cast<uint4*>(wcount + warp * kBins);
      for (int v = lane; v < kBins / 8; v += 32) mine[v] = make_uint4(0, 0, 0, 0);
      __syncwarp();
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      const int ahead = __popc(same & ((1u << lane) - 1u));
      if (in && ahead == 0) wcount[warp * kBins + d] = static_cast<uint16_t>(__popc(same));
      __syncthreads();
      int run = 0;
      if (tid < kBins) {
#pragma unroll 8
        for (int w = 0; w < 32; ++w) {
          const int n = wcount[w * kBins + tid];
          wcount[w * kBins + tid] = static_cast<uint16_t>(run);
          run += n;
        }
      }
      __syncthreads();
      const int r = in ? count[d] + wcount[warp * kBins + d] + ahead : 0;
      __syncthreads();
      if (tid < kBins) count[tid] += run;
      return r;
    };
    for (int d = tid; d < kBins; d += kSortThreads) count[d] = 0;
    int kept_key[kKeepTiles], kept_rank[kKeepTiles];
#pragma unroll
    for (int t = 0; t < kKeepTiles; ++t) {
      const int i0 = b + t * kSortThreads;
      if (i0 >= e) break;
      const bool in = i0 + tid < e;
      kept_key[t] = in ? key_at(i0 + tid) : 0;
      kept_rank[t] = rank_of(in, kept_key[t]);
    }
    for (int i0 = b + kKeepTiles * kSortThreads; i0 < e; i0 += kSortThreads) {
      const bool in = i0 + tid < e;
      const int r = rank_of(in, in ? key_at(i0 + tid) : 0);
      if (in) ranks[i0 + tid] = r;
    }
    cluster_sync();
    // first place of each digit of this slice: smaller digits, then the same digit in earlier slices
    int total = 0, before = 0;
    if (tid < kBins) {
      for (int r = 0; r < static_cast<int>(nctas); ++r) {
        const int h = ld_cluster_s32(map_to_rank(smem_u32(&count[tid]), r));
        before += r < rank ? h : 0;
        total += h;
      }
    }
    int x = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    if (tid < kBins) {
      int ahead = 0;
      for (int w = 0; w < warp; ++w) ahead += wsum[w];
      base[tid] = ahead + x - total + before;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kKeepTiles; ++t) {
      const int i = b + t * kSortThreads + tid;
      if (i < e) {
        const int at = base[digit(kept_key[t])] + kept_rank[t];
        kdst[at] = kept_key[t];
        odst[at] = p > 0 ? __ldcg(osrc + i) : i;
      }
    }
    for (int i = b + kKeepTiles * kSortThreads + tid; i < e; i += kSortThreads) {
      const int key = key_at(i);
      const int at = base[digit(key)] + ranks[i];
      kdst[at] = key;
      odst[at] = p > 0 ? __ldcg(osrc + i) : i;
    }
    cluster_sync();  // this pass's keys are written, and nobody reads the counts any more
  }
  // pieces: where a row begins, and every kPieceTokens-th place of the order
  auto begins = [&](int i) -> bool {
    return i < e && (i % kPieceTokens == 0 || __ldcg(keys + i) != __ldcg(keys + i - 1));
  };
  int mine = 0;
  for (int i0 = b; i0 < e; i0 += kSortThreads) mine += __syncthreads_count(begins(i0 + tid));
  if (tid == 0) pieces = mine;
  cluster_sync();
  int at = 0, all = 0;
  for (int r = 0; r < static_cast<int>(nctas); ++r) {
    const int n = ld_cluster_s32(map_to_rank(smem_u32(&pieces), r));
    at += r < rank ? n : 0;
    all += n;
  }
  for (int i0 = b; i0 < e; i0 += kSortThreads) {
    const int i = i0 + tid;
    const bool f = begins(i);
    const uint32_t m = __ballot_sync(0xffffffffu, f);
    if (lane == 0) wsum[warp] = __popc(m);
    __syncthreads();
    int ahead = __popc(m & ((1u << lane) - 1u)), sum = 0;
    for (int w = 0; w < 32; ++w) {
      ahead += w < warp ? wsum[w] : 0;
      sum += wsum[w];
    }
    if (f) {
      plan.start[at + ahead] = i;
      plan.key[at + ahead] = __ldcg(keys + i);
    }
    at += sum;
    __syncthreads();
  }
  if (rank == 0 && tid == 0) {
    plan.start[all] = T;
    *plan.count = all;
  }
  cluster_sync();  // nobody reads this CTA's shared memory any more
}

// ---------------------------------------------------------------- gradient
template <int F>
__device__ __forceinline__ float dot_chunk(const URef& u, int c, const float2 (&g)[16], const float (&gs)[2]) {
  float a[2], b[2];
  uint32_t qb[8];
  MixChunk<F>::get(u, c, a, b, qb);
  const float2 nsub = make_float2(-MixChunk<F>::kSub, -MixChunk<F>::kSub);
  float2 s[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 q01 = __fadd2_rn(make_float2(magic_byte(qb[j], 0), magic_byte(qb[j], 1)), nsub);
    const float2 q23 = __fadd2_rn(make_float2(magic_byte(qb[j], 2), magic_byte(qb[j], 3)), nsub);
    s[j >> 2] = __ffma2_rn(g[2 * j], q01, s[j >> 2]);
    s[j >> 2] = __ffma2_rn(g[2 * j + 1], q23, s[j >> 2]);
  }
  float d = a[0] * (s[0].x + s[0].y) + a[1] * (s[1].x + s[1].y);
  if (MixChunk<F>::kMin) d = fmaf(b[0], gs[0], fmaf(b[1], gs[1], d));
  return d;
}

// Adds 32 values of a row of dy at column col (zeros past cols); vec: the rows
// are 16-byte aligned.
template <typename T>
__device__ __forceinline__ void add_row(const T* row, int col, int cols, bool vec, float2 (&g)[16]) {
  constexpr int kPer = 16 / sizeof(T);
  if (vec && col + 32 <= cols) {
    uint4 v[32 / kPer];
#pragma unroll
    for (int j = 0; j < 32 / kPer; ++j) v[j] = __ldg(reinterpret_cast<const uint4*>(row + col) + j);
#pragma unroll
    for (int j = 0; j < 32 / kPer; ++j) {
      const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          float2& d = g[2 * j + (i >> 1)];
          (i & 1 ? d.y : d.x) += __uint_as_float(w[i]);
        } else {
          const float2 f = [&] {
            if constexpr (std::is_same<T, __half>::value)
              return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            else
              return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
          }();
          g[4 * j + i].x += f.x;
          g[4 * j + i].y += f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (col + 2 * j < cols) g[j].x += static_cast<float>(row[col + 2 * j]);
      if (col + 2 * j + 1 < cols) g[j].y += static_cast<float>(row[col + 2 * j + 1]);
    }
  }
}

// Eight lanes take a unit of a piece of the plan: they sum the unit's columns
// of the rows of dy of the piece's tokens in registers, then multiply every
// candidate's decoded weights into the sum; a run of equal tokens that is cut
// into several pieces is finished in each, the products being linear.  Sums
// over pieces are held in 64 bits, in the thread's own place of shared memory
// (an index that varies would put a register array into local memory), and
// the block's are left in partials[blockIdx.x][K].
template <typename T>
__global__ void __launch_bounds__(kThreads, kGradBlocks)
    embed_gategrad_kernel(const __grid_constant__ CandSet cs, Plan plan, int rows, int units_per_row, int cols,
                          const T* __restrict__ dy, long long lddy, bool vec, double* __restrict__ partials, int* err) {
  extern __shared__ __align__(16) uint8_t esmem[];
  double* acc = reinterpret_cast<double*>(esmem);  // [K][kThreads]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lu = lane >> 3, c = lane & 7;
  uint8_t* buf = esmem + cs.K * kThreads * sizeof(double) + warp * warp_bytes(cs);
  for (int k = 0; k < cs.K; ++k) acc[k * kThreads + threadIdx.x] = 0.0;
  UnitWalk<true> w{plan, Ids{nullptr, false}, *plan.count, 0, rows, units_per_row};
  w.start_at((static_cast<long long>(blockIdx.x) * kWarps + warp) * kUnits + lu,
             static_cast<long long>(gridDim.x) * kWarps * kUnits);
  bool fmt_ok = true;
  for (;; w.step()) {
    const int row = w.row();
    if (!__any_sync(0xffffffffu, row >= 0)) break;  // other shards' pieces come last
    const long long unit = static_cast<long long>(row) * units_per_row + w.u;
    if (row >= 0) stage_unit(cs, smem_u32(buf), lu, c, unit);
    async_commit();
    const int col = 256 * w.u + 32 * c;
    const bool on = row >= 0 && col < cols;
    float2 g[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) g[j] = make_float2(0.f, 0.f);
    if (on) {
      const int end = plan.start[w.i + 1];
      for (int i = plan.start[w.i]; i < end; ++i)
        add_row<T>(dy + static_cast<long long>(plan.order[i]) * lddy, col, cols, vec, g);
    }
    float gs[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 16; ++j) gs[j >> 3] += g[j].x + g[j].y;
    async_wait<0>();
    __syncwarp();
    if (on) {
      const uint8_t* region = buf;
      for (int k = 0; k < cs.K; ++k) {
        const URef ur = staged(cs, region, k, lu, static_cast<uint32_t>(unit));
        float d = 0.f;
        switch (cs.fmt[k]) {
          case kQ8_0: d = dot_chunk<kQ8_0>(ur, c, g, gs); break;
          case kQ2_K: d = dot_chunk<kQ2_K>(ur, c, g, gs); break;
          case kQ3_K: d = dot_chunk<kQ3_K>(ur, c, g, gs); break;
          case kQ4_K: d = dot_chunk<kQ4_K>(ur, c, g, gs); break;
          case kQ5_K: d = dot_chunk<kQ5_K>(ur, c, g, gs); break;
          case kQ6_K: d = dot_chunk<kQ6_K>(ur, c, g, gs); break;
          case kIQ4_XS: d = dot_chunk<kIQ4_XS>(ur, c, g, gs); break;
          default: fmt_ok = false;
        }
        acc[k * kThreads + threadIdx.x] += static_cast<double>(d);
        region += kUnits * slot_bytes(cs.ubytes[k]);
      }
    }
    __syncwarp();  // the slots are filled again
  }
  if (!fmt_ok) report_error(err, kDevBadFormat, 4);
  __syncthreads();
  for (int k = warp; k < cs.K; k += kWarps) {
    double t = 0.0;
    for (int i = lane; i < kThreads; i += 32) t += acc[k * kThreads + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_down_sync(0xffffffffu, t, o);
    if (lane == 0) partials[static_cast<long long>(blockIdx.x) * cs.K + k] = t;
  }
}

// grad[k] = scale * the blocks' partials, joined in a fixed order; one warp per candidate.
__global__ void __launch_bounds__(32 * kMaxCandidates) embed_gategrad_join_kernel(const double* __restrict__ partials,
                                                                                  int blocks, int K, float scale,
                                                                                  float* __restrict__ grad) {
  const int k = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (k >= K) return;
  double t = 0.0;
  for (int b = lane; b < blocks; b += 32) t += partials[static_cast<long long>(b) * K + k];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_down_sync(0xffffffffu, t, o);
  if (lane == 0) grad[k] = static_cast<float>(t * static_cast<double>(scale));
}

}  // namespace embed
}  // namespace vq
