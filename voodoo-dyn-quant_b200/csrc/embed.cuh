// Lookup of token rows in a gated embedding (the mixture of K packed
// candidates), and the gradient of the mixture's probabilities.
//
//   out[t]  = scale * sum_k p_k W_k[id_t]
//   dL/dp_k = scale * sum_t <dy_t, W_k[id_t]>
//           = scale * sum over runs of equal id of <sum of the run's dy, W_k[id]>
//
// Neither writes a decoded row of a candidate: the lookup decodes and mixes a
// packed row in registers and writes it to all tokens of a piece, the gradient
// sums a piece's rows of dy first and multiplies the decoded weights into that
// sum as it decodes them.  What they cannot do without is the packed rows and
// T x D of out or dy (16384 x 4096 of text, six candidates: 35 us of HBM each);
// the decoding bounds them, 220 to 330 instructions for 32 weights of a
// candidate (63 us the lookup, 75 us the gradient).
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

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kUnits = 4;  // units of a warp
// Resident blocks per SM, and so 72 registers a thread: decoding waits for its
// own results, so warps count, until they spill (16384 x 4096 text, six
// candidates, lookup and gradient: 63 and 75 us with 7, 63 and 77 with 6, 65
// and 84 with 8).
constexpr int kBlocksPerSm = 7;
constexpr int kMaxBlocks = 1184;  // of a launch: the partials that the gradient leaves

// A unit's slot: the 16-byte aligned span of a 2-byte aligned unit, and a
// word more for the field reads that join two words.
inline int slot_bytes(int ub) { return ((ub + 14 + 15) & ~15) + 16; }

// The candidates of a launch.  In a warp's buffer the four slots of candidate
// k start at byte `region`.
struct Cands {
  struct Info {
    int decode, ubytes, slot, region;
  };
  const uint8_t* ptr[kMaxCandidates];
  Info info[kMaxCandidates];
  int K, warp_bytes;
};

// The 16 bytes at kAbove, where a > kAbove.
template <int kAbove>
__device__ __forceinline__ void async_copy16(uint32_t dst, const void* src, int a) {
  asm volatile(
      "{ .reg .pred p; setp.gt.s32 p, %2, %3;\n"
      "  @p cp.async.cg.shared.global [%0 + %3], [%1 + %3], 16; }" ::"r"(dst),
      "l"(src), "r"(a), "n"(kAbove)
      : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Copies unit `unit` (of the whole table) of every candidate into slot `lu`
// of the warp's buffer; lane c of the unit's eight takes every eighth vector
// (18 at most: a Q8_0 unit that starts inside a vector).
__device__ __forceinline__ void stage_unit(const Cands& cs, uint32_t buf, int lu, int c, long long unit) {
  for (int k = 0; k < cs.K; ++k) {
    const Cands::Info f = cs.info[k];
    const uint8_t* a = cs.ptr[k] + unit * f.ubytes;
    const int rel = static_cast<int>(reinterpret_cast<uintptr_t>(a) & 15u);
    const uint8_t* src = a - rel + 16 * c;
    const uint32_t dst = buf + f.region + lu * f.slot + 16 * c;
    const int left = rel + f.ubytes - 16 * c;  // bytes from this lane's first vector on
    async_copy16<0>(dst, src, left);
    async_copy16<128>(dst, src, left);
    async_copy16<256>(dst, src, left);
  }
}

// How a candidate's units are decoded: its format, and whether they start at
// words or 16-byte vectors, so that its fields can be read whole.  Dense
// numbers, for a jump table.
enum Decode : int { kDQ8, kDQ3, kDQ6, kDQ2, kDIQ4, kDQ4, kDQ5, kDQ2Words, kDIQ4Words, kDQ4Vectors, kDQ5Vectors };

inline int decode_code(int fmt, const uint8_t* p) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  switch (fmt) {
    case kQ8_0: return kDQ8;
    case kQ3_K: return kDQ3;
    case kQ6_K: return kDQ6;
    case kQ2_K: return a % 4 == 0 ? kDQ2Words : kDQ2;      // 84 bytes a unit
    case kIQ4_XS: return a % 4 == 0 ? kDIQ4Words : kDIQ4;  // 136
    case kQ4_K: return a % 16 == 0 ? kDQ4Vectors : kDQ4;   // 144
    default: return a % 16 == 0 ? kDQ5Vectors : kDQ5;      // Q5_K: 176
  }
}

template <int F>
using Format = std::integral_constant<int, F>;

// Calls op(format, unit) for the staged unit of candidate k; `unit` counts
// modulo 2^32.
template <class Op>
__device__ __forceinline__ void with_unit(const Cands& cs, const uint8_t* buf, int k, int lu, uint32_t unit,
                                          const Op& op) {
  const Cands::Info f = cs.info[k];
  const uint32_t rel = (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(cs.ptr[k])) + unit * f.ubytes) & 15u;
  const uint32_t* s = reinterpret_cast<const uint32_t*>(buf + f.region + lu * f.slot + (rel & ~3u));
  const URefHalf any{s, static_cast<int>(rel & 2u)};
  const URefAligned<false> words{s};
  const URefAligned<true> vectors{s};
  switch (f.decode) {
    case kDQ8: op(Format<kQ8_0>{}, any); break;
    case kDQ3: op(Format<kQ3_K>{}, any); break;
    case kDQ6: op(Format<kQ6_K>{}, any); break;
    case kDQ2: op(Format<kQ2_K>{}, any); break;
    case kDIQ4: op(Format<kIQ4_XS>{}, any); break;
    case kDQ4: op(Format<kQ4_K>{}, any); break;
    case kDQ5: op(Format<kQ5_K>{}, any); break;
    case kDQ2Words: op(Format<kQ2_K>{}, words); break;
    case kDIQ4Words: op(Format<kIQ4_XS>{}, words); break;
    case kDQ4Vectors: op(Format<kQ4_K>{}, vectors); break;
    case kDQ5Vectors: op(Format<kQ5_K>{}, vectors); break;
    default: break;
  }
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
// rows: piece i holds the tokens order[start[i]] to order[start[i + 1] - 1],
// all naming row key[i].  A piece begins where a row does, at every 1024th
// place of the order (a tile of the sort, which then needs no carry from the
// one before) and kPieceTokens after the piece before it.
struct Plan {
  int *order, *start, *key, *count;  // count[1], count[2]: the tokens and rows that the plan was made for

  __device__ __forceinline__ void finish(int pieces, int tokens, int rows) const {
    start[pieces] = tokens;
    *reinterpret_cast<int4*>(count) = make_int4(pieces, tokens, rows, 0);
  }
  // Pieces to walk; none where the plan is not one of these tokens and rows.
  __device__ __forceinline__ int pieces(int tokens, int rows, int* err) const {
    const int4 h = *reinterpret_cast<const int4*>(count);
    if (h.y == tokens && h.z == rows) return h.x;  // its places and keys lie in what this call reads and writes
    report_error(err, kDevBadPlan, 31);
    return 0;
  }
};

// Most tokens of a piece: a token that fills much of a batch is then worked
// on by many warps, each decoding its row again.  8 is what a unit's lanes
// read in one load (16384 tokens of text, six candidates, 6600 rows: 7500
// pieces, lookup and gradient 63 and 75 us; pieces of 4: 8600, 70 and 76).
// Longer ones decode less, but the warps that get them end last: when the
// lookup took 88 us, pieces of 16 and 32 took 91 and 95.
constexpr int kPieceTokens = 8;

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
  // Row of the table (-1: a token of another one), unit, and the tokens: places in the order from begin to end.
  struct At {
    int row, u, begin, end;
  };
  __device__ __forceinline__ At get() const {
    At a{-1, u, 0, 0};
    if (!on()) return a;
    if (kRuns) {
      const int key = plan.key[i];
      a.begin = plan.start[i];
      a.end = plan.start[i + 1];
      a.row = key < rows ? key : -1;
    } else {
      a.row = static_cast<int>(local_row(ids.at(i), vocab_start, rows));
      a.begin = i;
      a.end = i + 1;
    }
    return a;
  }
};

// ---------------------------------------------------------------- lookup
// mix_chunk on any reference of a unit: the same operations in the same order.
template <int F, class U>
__device__ __forceinline__ void mix_unit(const U& u, int c, float pk, float (&acc)[32], float (&cst)[2]) {
  float a[2], b[2];
  uint32_t qb[8];
  MixChunk<F>::get(u, c, a, b, qb);
  const float pa[2] = {pk * a[0], pk * a[1]};
  if (MixChunk<F>::kMin) {
    cst[0] = fmaf(pk, b[0], cst[0]);
    cst[1] = fmaf(pk, b[1], cst[1]);
  }
  const float2 nsub = make_float2(-MixChunk<F>::kSub, -MixChunk<F>::kSub);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int i = 2 * (j & 1);
    const float2 q = __fadd2_rn(make_float2(magic_byte(qb[j >> 1], i), magic_byte(qb[j >> 1], i + 1)), nsub);
    const float2 r = __ffma2_rn(make_float2(pa[j >> 3], pa[j >> 3]), q, make_float2(acc[2 * j], acc[2 * j + 1]));
    acc[2 * j] = r.x, acc[2 * j + 1] = r.y;
  }
}

// Rows of ids outside [vocab_start, vocab_start + rows) are written as zeros
// (another shard's tokens); `strict` also reports them.  The mixture is
// mix_units_kernel's, in the same order, so for scale 1 the rows are those of
// W_mix bit for bit; the scaled row is rounded to bf16 once.  kRuns: each row
// is decoded once per piece of the plan and written to all its tokens;
// otherwise once per token, with no plan to wait for.
template <bool kRuns>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    embed_mix_kernel(const __grid_constant__ Cands cs, const float* __restrict__ probs, Ids ids, int T, Plan plan,
                     long long vocab_start, int rows, int units_per_row, int cols, float scale, bool strict, bool vec,
                     __nv_bfloat16* __restrict__ out, long long ldo, int* err) {
  extern __shared__ __align__(16) uint8_t esmem[];
  __shared__ float pk_s[kMaxCandidates];
  if (threadIdx.x < cs.K) pk_s[threadIdx.x] = probs[threadIdx.x];
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lu = lane >> 3, c = lane & 7;
  uint8_t* buf = esmem + kWarps * kUnits * 512 + warp * cs.warp_bytes;
  uint4* rows_s = reinterpret_cast<uint4*>(esmem + (warp * kUnits + lu) * 512);
  const int count = kRuns ? plan.pieces(T, rows, err) : T;
  if (kRuns && count == 0) {  // another call's plan (T > 0 tokens have a piece): zeros, not what the memory held
    for (int t = blockIdx.x; t < T; t += gridDim.x)
      for (int j = threadIdx.x; j < cols; j += kThreads) out[t * ldo + j] = __float2bfloat16_rn(0.f);
    return;
  }
  UnitWalk<kRuns> w{plan, ids, count, vocab_start, rows, units_per_row};
  w.start_at((static_cast<long long>(blockIdx.x) * kWarps + warp) * kUnits + lu,
             static_cast<long long>(gridDim.x) * kWarps * kUnits);
  bool bad = false;
  for (;; w.step()) {
    const auto now = w.get();
    if (!__any_sync(0xffffffffu, now.begin < now.end)) break;
    const long long unit = static_cast<long long>(now.row) * units_per_row + now.u;
    if (now.row >= 0) stage_unit(cs, smem_u32(buf), lu, c, unit);
    async_commit();
    const int len = now.end - now.begin;
    // lane c holds the unit's c-th token
    const int mine = kRuns ? (c < len ? plan.order[now.begin + c] : 0) : now.begin;
    float acc[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] = 0.f;
    float cst[2] = {0.f, 0.f};
    const int col = 256 * now.u + 32 * c;
    async_wait<0>();
    __syncwarp();
    if (now.row >= 0 && col < cols) {
      for (int k = 0; k < cs.K; ++k) {
        const float pk = pk_s[k];
        with_unit(cs, buf, k, lu, static_cast<uint32_t>(unit), [&](auto f, const auto& u) {
          mix_unit<decltype(f)::value>(u, c, pk, acc, cst);
        });
      }
    }
    bad |= now.row < 0 && len > 0;
    // Lane c holds columns 32 c to 32 c + 31 of the unit; written like that a
    // store would touch half of each 32-byte sector.  By way of shared memory
    // it gets columns 64 v + 8 c for v = 0..3, 128 bytes of the row a store.
    uint4 hv[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      __align__(16) __nv_bfloat162 h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 x = __fadd2_rn(make_float2(acc[8 * v + 2 * j], acc[8 * v + 2 * j + 1]), make_float2(cst[v >> 1], cst[v >> 1]));
        x = __fmul2_rn(x, make_float2(scale, scale));  // exact for scale 1
        h[j] = __floats2bfloat162_rn(x.x, x.y);
      }
      rows_s[c * 4 + (v ^ (c >> 1))] = *reinterpret_cast<const uint4*>(h);
    }
    __syncwarp();
#pragma unroll
    for (int v = 0; v < 4; ++v) hv[v] = rows_s[v * 8 + (c & 4) + ((c & 3) ^ v)];
    const int most = kRuns ? __reduce_max_sync(0xffffffffu, len) : 1;
    const int col0 = 256 * now.u + 8 * c;
    for (int i = 0; i < most; ++i) {
      const int tok = kRuns ? __shfl_sync(0xffffffffu, mine, (lane & 24) + i) : mine;
      if (i >= len) continue;
      __nv_bfloat16* dst = out + static_cast<long long>(tok) * ldo + col0;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int left = cols - col0 - 64 * v;
        if (vec && left >= 8) {
          *reinterpret_cast<uint4*>(dst + 64 * v) = hv[v];
        } else if (left > 0) {
          const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&hv[v]);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < left) dst[64 * v + j] = h[j];
        }
      }
    }
    __syncwarp();  // the slots are filled again
  }
  if (bad && strict) report_error(err, kDevBadIndex, 30);
}

// ---------------------------------------------------------------- plan
// Stable radix sort of the tokens' local rows, nine bits a pass, and the
// pieces.  Tokens of other shards get the key `rows` and so end up last.
// Latency bound: barriers and the round trips between them.
constexpr int kSortThreads = 1024;
constexpr int kSortCtas = 16;  // the largest cluster (the portable 8 take 25 us for 16384 tokens, these 21)
constexpr int kDigitBits = 9;
constexpr int kBins = 1 << kDigitBits;
constexpr int kSortSmem = 32 * kBins * 2;
constexpr int kKeepTiles = 2;  // tiles whose keys and ranks stay in registers between the two halves of a pass

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// Exclusive scan over the digits of a block (thread d < kBins holds digit d's
// total; wsum: 32 ints of scratch).  One barrier inside.
__device__ __forceinline__ int digit_scan(int total, int* wsum) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int x = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) wsum[warp] = x;
  __syncthreads();
  int ahead = 0;
#pragma unroll
  for (int w = 0; w < kBins / 32; ++w) ahead += w < warp ? wsum[w] : 0;
  return ahead + x - total;
}

// Turns each digit's counts by warp into the sums over the warps before, and
// returns the digit's total (threads < kBins).
__device__ __forceinline__ int warp_prefix(uint16_t* wcount) {
  int run = 0;
  if (threadIdx.x < kBins) {
#pragma unroll 16
    for (int w = 0; w < 32; ++w) {
      const int n = wcount[w * kBins + threadIdx.x];
      wcount[w * kBins + threadIdx.x] = static_cast<uint16_t>(run);
      run += n;
    }
  }
  return run;
}

// Up to 1024 * kItems tokens: one block sorts in shared memory, a warp holding
// 32 * kItems consecutive places, without the cluster's barriers.
template <int kItems>
__global__ void __launch_bounds__(kSortThreads) token_plan_block_kernel(Ids ids, int T, long long vocab_start, int rows,
                                                                        int passes, Plan plan) {
  extern __shared__ __align__(16) uint8_t ssmem[];
  uint16_t* wcount = reinterpret_cast<uint16_t*>(ssmem);              // [32 warps][kBins]
  int* skey = reinterpret_cast<int*>(ssmem + kSortSmem);              // [1024 * kItems]
  uint16_t* sidx = reinterpret_cast<uint16_t*>(skey + kSortThreads * kItems);
  __shared__ int base[kBins];
  __shared__ int wsum[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int first = warp * 32 * kItems + lane;  // this lane's places: first + 32 r
  int key[kItems], idx[kItems], rank[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const int i = first + 32 * r;
    idx[r] = i;
    const long long row = i < T ? local_row(ids.at(i), vocab_start, rows) : -1;
    // places past the end sort behind everything (the sort is stable): all bits of the passes set
    key[r] = i >= T ? 0x7fffffff : row < 0 ? rows : static_cast<int>(row);
  }
  for (int p = 0; p < passes; ++p) {
    const int shift = p * kDigitBits;
    uint4* z = reinterpret_cast<uint4*>(wcount);
    for (int v = tid; v < kSortSmem / 16; v += kSortThreads) z[v] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint16_t* mine = wcount + warp * kBins;
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const int d = (key[r] >> shift) & (kBins - 1);
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      const int before = mine[d];
      __syncwarp();
      const int ahead = __popc(same & ((1u << lane) - 1u));
      if (ahead == 0) mine[d] = static_cast<uint16_t>(before + __popc(same));
      __syncwarp();
      rank[r] = before + ahead;
    }
    __syncthreads();
    const int total = warp_prefix(wcount);
    const int at0 = digit_scan(total, wsum);
    if (tid < kBins) base[tid] = at0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const int d = (key[r] >> shift) & (kBins - 1);
      const int at = base[d] + mine[d] + rank[r];
      skey[at] = key[r];
      sidx[at] = static_cast<uint16_t>(idx[r]);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      key[r] = skey[first + 32 * r];
      idx[r] = sidx[first + 32 * r];
    }
  }
  // pieces: the last place before each warp's where a row or a tile begins ...
  uint32_t heads[kItems];
  int last = -1;
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const int i = first + 32 * r;
    if (i < T) plan.order[i] = idx[r];
    heads[r] = __ballot_sync(0xffffffffu, i % kSortThreads == 0 || skey[i] != skey[i - 1]);
    if (heads[r]) last = i - lane + 31 - __clz(heads[r]);
  }
  if (lane == 0) wsum[warp] = last;
  __syncthreads();
  int from = -1;
#pragma unroll
  for (int w = 0; w < 32; ++w) from = w < warp ? max(from, wsum[w]) : from;
  // ... every kPieceTokens places from which a piece begins
  uint32_t starts[kItems];
  int n = 0;
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const int i = first + 32 * r;
    const uint32_t upto = heads[r] & (0xffffffffu >> (31 - lane));
    const int begin = upto ? i - lane + 31 - __clz(upto) : from;
    starts[r] = __ballot_sync(0xffffffffu, i < T && (i - begin) % kPieceTokens == 0);
    n += __popc(starts[r]);
    if (heads[r]) from = i - lane + 31 - __clz(heads[r]);
  }
  __syncthreads();
  if (lane == 0) wsum[warp] = n;
  __syncthreads();
  int at = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 32; ++w) {
    at += w < warp ? wsum[w] : 0;
    all += wsum[w];
  }
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    if ((starts[r] >> lane) & 1u) {
      const int q = at + __popc(starts[r] & ((1u << lane) - 1u));
      plan.start[q] = first + 32 * r;
      plan.key[q] = key[r];
    }
    at += __popc(starts[r]);
  }
  if (tid == 0) {
    plan.finish(all, T, rows);
  }
}

// More tokens: one cluster.  Each CTA owns a contiguous slice (of whole
// tiles) of a pass's input and ranks it a tile of 1024 tokens at a time:
// within a warp by matching digits, over the warps and tiles by counts; the
// slices' counts meet through distributed shared memory.
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
  const int tiles = (T + kSortThreads - 1) / kSortThreads;
  const int slice = (tiles + static_cast<int>(nctas) - 1) / static_cast<int>(nctas) * kSortThreads;
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
      const int run = warp_prefix(wcount);
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
#pragma unroll
      for (int r = 0; r < kSortCtas; ++r) {  // in flight together
        const int h = r < static_cast<int>(nctas) ? ld_cluster_s32(map_to_rank(smem_u32(&count[tid]), r)) : 0;
        before += r < rank ? h : 0;
        total += h;
      }
    }
    const int at0 = digit_scan(total, wsum);
    if (tid < kBins) base[tid] = at0 + before;
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
  // pieces, a tile at a time; first their number
  auto starts_of = [&](int i) -> uint32_t {
    const bool in = i < e;
    const uint32_t heads =
        __ballot_sync(0xffffffffu, in && (i % kSortThreads == 0 || __ldcg(keys + i) != __ldcg(keys + i - 1)));
    if (lane == 0) wsum[warp] = heads ? i + 31 - __clz(heads) : -1;
    __syncthreads();
    int from = -1;
#pragma unroll
    for (int w = 0; w < 32; ++w) from = w < warp ? max(from, wsum[w]) : from;
    __syncthreads();
    const uint32_t upto = heads & (0xffffffffu >> (31 - lane));
    const int begin = upto ? i - lane + 31 - __clz(upto) : from;
    return __ballot_sync(0xffffffffu, in && (i - begin) % kPieceTokens == 0);
  };
  int mine = 0;
  uint32_t kept[kKeepTiles];
#pragma unroll
  for (int t = 0; t < kKeepTiles; ++t) {
    kept[t] = b + t * kSortThreads < e ? starts_of(b + t * kSortThreads + tid) : 0;
    mine += __popc(kept[t]);
  }
  for (int i0 = b + kKeepTiles * kSortThreads; i0 < e; i0 += kSortThreads) mine += __popc(starts_of(i0 + tid));
  __syncthreads();
  if (lane == 0) wsum[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < 32; ++w) n += wsum[w];
    pieces = n;
  }
  cluster_sync();
  int at = 0, all = 0;
#pragma unroll
  for (int r = 0; r < kSortCtas; ++r) {
    const int n = r < static_cast<int>(nctas) ? ld_cluster_s32(map_to_rank(smem_u32(&pieces), r)) : 0;
    at += r < rank ? n : 0;
    all += n;
  }
  auto write_starts = [&](int i, uint32_t m) {
    if (lane == 0) wsum[warp] = __popc(m);
    __syncthreads();
    int ahead = __popc(m & ((1u << lane) - 1u)), sum = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      ahead += w < warp ? wsum[w] : 0;
      sum += wsum[w];
    }
    if ((m >> lane) & 1u) {
      plan.start[at + ahead] = i;
      plan.key[at + ahead] = __ldcg(keys + i);
    }
    at += sum;
    __syncthreads();
  };
#pragma unroll
  for (int t = 0; t < kKeepTiles; ++t)
    if (b + t * kSortThreads < e) write_starts(b + t * kSortThreads + tid, kept[t]);
  for (int i0 = b + kKeepTiles * kSortThreads; i0 < e; i0 += kSortThreads) write_starts(i0 + tid, starts_of(i0 + tid));
  if (rank == 0 && tid == 0) {
    plan.finish(all, T, rows);
  }
  cluster_sync();  // nobody reads this CTA's shared memory any more
}

// ---------------------------------------------------------------- gradient
template <int F, class U>
__device__ __forceinline__ float dot_unit(const U& u, int c, const float (&g)[32], const float (&gs)[2]) {
  float a[2], b[2];
  uint32_t qb[8];
  MixChunk<F>::get(u, c, a, b, qb);
  float2 s[2];
  const float2 nsub = make_float2(-MixChunk<F>::kSub, -MixChunk<F>::kSub);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s[h] = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 8 * h; j < 8 * h + 8; ++j) {
      const int i = 2 * (j & 1);
      const float2 q = __fadd2_rn(make_float2(magic_byte(qb[j >> 1], i), magic_byte(qb[j >> 1], i + 1)), nsub);
      s[h] = __ffma2_rn(make_float2(g[2 * j], g[2 * j + 1]), q, s[h]);
    }
  }
  float d = a[0] * (s[0].x + s[0].y) + a[1] * (s[1].x + s[1].y);
  if (MixChunk<F>::kMin) d = fmaf(b[0], gs[0], fmaf(b[1], gs[1], d));
  return d;
}

// Adds 32 values of a row of dy at column col (zeros past cols); vec: the rows
// are 16-byte aligned.
template <typename T>
__device__ __forceinline__ void add_row(const T* row, int col, int cols, bool vec, float (&g)[32]) {
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
          g[4 * j + i] += __uint_as_float(w[i]);
        } else {
          float2 f;
          if constexpr (std::is_same<T, __half>::value)
            f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          else
            f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
          f = __fadd2_rn(make_float2(g[8 * j + 2 * i], g[8 * j + 2 * i + 1]), f);
          g[8 * j + 2 * i] = f.x, g[8 * j + 2 * i + 1] = f.y;
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (col + j < cols) g[j] += static_cast<float>(row[col + j]);
  }
}

// Eight lanes take a unit of a piece of the plan: they sum the unit's columns
// of the rows of dy of the piece's tokens in registers, then multiply every
// candidate's decoded weights into the sum; a run of equal tokens that is cut
// into several pieces is finished in each, the products being linear.  Sums
// over pieces are held in 64 bits, in the thread's own place of shared memory
// (an index that varies would put a register array into local memory), and
// the block's are left in partials[K][gridDim.x].
template <typename T>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    embed_gategrad_kernel(const __grid_constant__ Cands cs, Plan plan, int tokens, int rows, int units_per_row,
                          int cols, const T* __restrict__ dy, long long lddy, bool vec, double* __restrict__ partials,
                          int* err) {
  extern __shared__ __align__(16) uint8_t esmem[];
  double* acc = reinterpret_cast<double*>(esmem);  // [K][kThreads]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lu = lane >> 3, c = lane & 7;
  uint8_t* buf = esmem + cs.K * kThreads * sizeof(double) + warp * cs.warp_bytes;
  for (int k = 0; k < cs.K; ++k) acc[k * kThreads + threadIdx.x] = 0.0;
  UnitWalk<true> w{plan, Ids{nullptr, false}, plan.pieces(tokens, rows, err), 0, rows, units_per_row};
  w.start_at((static_cast<long long>(blockIdx.x) * kWarps + warp) * kUnits + lu,
             static_cast<long long>(gridDim.x) * kWarps * kUnits);
  for (;; w.step()) {
    const auto now = w.get();
    if (!__any_sync(0xffffffffu, now.row >= 0)) break;  // other shards' pieces come last
    const long long unit = static_cast<long long>(now.row) * units_per_row + now.u;
    if (now.row >= 0) stage_unit(cs, smem_u32(buf), lu, c, unit);
    async_commit();
    const int col = 256 * now.u + 32 * c;
    const bool on = now.row >= 0 && col < cols;
    const int len = now.row >= 0 ? now.end - now.begin : 0;
    const int mine = c < len ? plan.order[now.begin + c] : 0;  // lane c holds the unit's c-th token
    float g[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) g[j] = 0.f;
    const int most = __reduce_max_sync(0xffffffffu, len);
    for (int i = 0; i < most; ++i) {
      const int tok = __shfl_sync(0xffffffffu, mine, (lane & 24) + i);
      if (i < len && on) add_row<T>(dy + static_cast<long long>(tok) * lddy, col, cols, vec, g);
    }
    float gs[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float2 t = make_float2(g[16 * h], g[16 * h + 1]);
#pragma unroll
      for (int j = 2; j < 16; j += 2) t = __fadd2_rn(t, make_float2(g[16 * h + j], g[16 * h + j + 1]));
      gs[h] = t.x + t.y;
    }
    async_wait<0>();
    __syncwarp();
    if (on) {
      for (int k = 0; k < cs.K; ++k) {
        float d = 0.f;
        with_unit(cs, buf, k, lu, static_cast<uint32_t>(unit), [&](auto f, const auto& u) {
          d = dot_unit<decltype(f)::value>(u, c, g, gs);
        });
        acc[k * kThreads + threadIdx.x] += static_cast<double>(d);
      }
    }
    __syncwarp();  // the slots are filled again
  }
  __syncthreads();
  for (int k = warp; k < cs.K; k += kWarps) {
    double t = 0.0;
    for (int i = lane; i < kThreads; i += 32) t += acc[k * kThreads + i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_down_sync(0xffffffffu, t, o);
    if (lane == 0) partials[k * gridDim.x + blockIdx.x] = t;
  }
}

// grad[k] = scale * the blocks' partials, joined in a fixed order; one warp per candidate.
__global__ void __launch_bounds__(32 * kMaxCandidates) embed_gategrad_join_kernel(const double* __restrict__ partials,
                                                                                  int blocks, int K, float scale,
                                                                                  float* __restrict__ grad) {
  const int k = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (k >= K) return;
  double t = 0.0;
#pragma unroll 8
  for (int b = lane; b < blocks; b += 32) t += partials[k * blocks + b];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_down_sync(0xffffffffu, t, o);
  if (lane == 0) grad[k] = static_cast<float>(t * static_cast<double>(scale));
}

}  // namespace embed
}  // namespace vq
