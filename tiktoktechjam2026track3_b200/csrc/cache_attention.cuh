// Attention of the newest tokens of each sequence over its paged cache (cache_append.cuh): a single token, or a
// token and the few drafts behind it. Query row t of sequence b, of q_len, stands at p = kv_len[b] - q_len + t and
// sees the keys j <= p with (window == 0 or p - j < window or j < sinks):
//   out = sum_j w_j v_j,  w_j = exp(scale q.k_j) / sum of them;  0 where no key is visible.
//
// The work is a stream of keys and values read once (bound by HBM; 2 operations per byte and query head).
// The rows that share a key head, q_len x (query heads per key head), form the 8-column operand of
// mma.m16n8k16, with 16 tokens as its rows:
//   S^T[token][row] = K Q^T,   O^T[dim][row] += V^T P^T.
// tcgen05 would need 128 rows of queries (or of keys brought through shared memory and, in 8 bits, queries in 8
// bits too); here the tensor work is a few percent of the time and the registers it wants are the
// ones the loads arrive in:
//   - K: thread (g, t) of the warp (g = lane / 4, t = lane % 4) holds 16-byte pieces of tokens g and g + 8. Which
//     dims a k-step takes is free as long as Q is laid out alike, so the pieces are the fragments as loaded.
//   - V: it holds 16-byte pieces of tokens 2t, 2t+1, 2t+8, 2t+9, for its own dims; byte permutes pair the tokens,
//     and which dims an m-tile takes is free as well.
//   - 8-bit codes become fp16 (exactly), bf16 stays. Scores come out as [token][row] and are wanted as [row][token]
//     pairs: one movmatrix per 8 tokens.
// 8-bit pages: the scale of K, a power of two, multiplies the scores; that of V, 2^ev, goes into the exponent of the
// weights, w = 2^(s + ev - m), with m the running maximum of s + ev, so that the weights stay within fp16
// whatever the scales; the sum takes w 2^-ev. Q is turned into fp16 after a power of two per row that brings its
// largest element to [2^14, 2^15): bf16's 8 bits then fit exactly down to 2^-28 of the largest.
// The maximum moves only when a score exceeds it by 2^8 (the weights keep 2^7 of headroom below fp16's
// subnormals); sums, maxima and outputs are fp32.
// Roundings to fewer bits, for the products' sake: weights to the type of the values they meet, fp16 over 8 bits (11
// bits, far below the codes' own 4) and bf16 over bf16 (one mma takes one type); the sums take them unrounded. Measured
// over whole outputs against 64 bits, with the output's own rounding to bf16 in it: 0.0015 to 0.0017 of the norm over 8
// bits, as with weights of 32 bits, and 0.0023 over bf16 (0.0017). fp16 bounds the range, too: a weight times its
// page's scale of V loses bits from 2^21 below the largest on and is dropped from 2^32 on, even in dims where the page with the
// large scale holds zeros.
//
// Split: a (sequence, key head) is cut into units of 16 tokens per warp. Calls of moderate length give each to one CTA,
// or to a cluster of CTAs that share its units and join their maxima, sums and outputs through shared memory. Else all
// units of the call are laid on one line and the CTAs take equal stretches of it, so that one long sequence among short
// ones, and few sequences on 148 SMs, fill the machine alike. A CTA whose stretch holds only part of a (sequence, head)
// leaves its results in the workspace; the last one to arrive (a counter) joins them, in the order of the stretches.
//
// What bounds a warp is the chain of one tile (loads, 8 dependent products, maximum, exponentials, products: about
// 1500 cycles besides the loads), so the loads' latency is kept out of it: the lanes hold the page numbers of the
// next 32 tiles, and each lane prefetches one line of a tile two or three units ahead into L2, at no cost in registers
// or shared memory. Heads of 64 and 32 take 2 and 4 tiles of 16 tokens at a time, interleaved.
// Measured on one B200 (us a call back to back, floor at the measured copy rate in brackets; first form, which read each
// page number in the loop and joined element by element): 8 x 131072 8-bit tokens, 8 key heads of 128, 4 query heads
// each: 331 (328; 355); 64 sequences of up to 8192: 115 (100; 129); one of 131072: 59 (41; 111), one of 8192: 12 (2.6; 22);
// bf16, 32 x 8192: 165 (164; 181); 32 windows of 4096 bf16 tokens, 10 rows: 52 (41; 104); 16 key heads of 64: 180 (165;
// 265), of 32: 109 (82; 226); 12 heads of 1001 tokens: 6.8 (0.2; 12.6). At the 1000 W limit the clock drops and the
// first two take 378 and 127. A short call is 5 us of dependent steps (lengths, page numbers, keys, join of the warps),
// a join of CTAs 3 to 5 more.
#pragma once
#include <algorithm>

#include <cuda_fp16.h>

#include "b2_common.cuh"
#include "cache_append.cuh"

namespace b2 {

struct CacheAttnParams {
  CachePages c;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  int64_t ld_q, ld_out;
  const int32_t* page_table;
  int64_t ld_table;
  int table_pages;
  const int32_t* kv_len;
  int batch, q_len, group, window, sinks;
  int block0;  // first row block of this launch
  float scale_log2;
  int* counters;        // [row blocks][CTAs]: of the head that begins in a CTA's stretch and goes on; zero between calls
  int* group_counters;  // [row blocks][groups of CTAs][2], likewise
  float* partials;      // [row blocks][CTAs][2][rows][head_dim + 2]
};

constexpr int kCacheMaxBatch = 4096;
constexpr int kCacheAtOnce = 40;  // parts of a (sequence, head) that one CTA joins in one go;
constexpr int kCacheGroup = 16;   // of more, so many in a first go
constexpr int kCacheCluster = 16;  // CTAs of a cluster, at most (a power of two)
// Row blocks that one launch of the line form takes: more take turns over the same partial results, so that the workspace
// does not grow with them (160 MB at most; 512 blocks of 16 rows would be 2.5 GB). A turn costs the end of one launch and the
// start of the next, about 30 us: 1024 rows over 100000 bf16 tokens 925 us in one launch, 988 in two, 1346 in sixteen.
constexpr int kCacheBlocksAtOnce = 32;
constexpr float kCacheRescale = 8.f;   // log2: the maximum moves when a score exceeds it by more
constexpr float kCacheHeadroom = 7.f;  // log2: weights are at most 2^(8 + 7), below fp16's largest

// What a sequence's tokens come to in tiles of 16: those of the sinks that lie before the window, then the window's.
struct SeqTiles {
  int len, sink_tiles, first_win, count;
};

__device__ __forceinline__ SeqTiles seq_tiles(const CacheAttnParams& p, int len) {
  SeqTiles s;
  s.len = len;
  s.sink_tiles = 0;
  s.first_win = 0;
  if (p.window > 0) {
    const int lo = max(0, len - p.q_len - p.window + 1);
    s.first_win = lo >> 4;
    s.sink_tiles = min((p.sinks + 15) >> 4, s.first_win);
  }
  s.count = s.sink_tiles + ((len + 15) >> 4) - s.first_win;
  return s;
}

__device__ __forceinline__ int seq_length(const CacheAttnParams& p, int b) {
  const int len = p.kv_len[b];
  const int most = p.table_pages << p.c.page_shift;
  if (len < 0 || len > most) record_status(kKernelCacheAttention, 1, kReasonBadIndex);
  return min(max(len, 0), most);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool kFp8>
__device__ __forceinline__ void cache_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if (kFp8)
    mma_f16(d, a0, a1, a2, a3, b0, b1);
  else
    mma_bf16(d, a0, a1, a2, a3, b0, b1);
}

// Transpose of an 8 x 8 matrix of 16-bit values spread over the warp as an mma fragment.
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t w) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(w)));
  return h;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Pages and scales may be written by the launch before this one, which is still running when this grid's first CTAs are
// resident: they are not constant for the grid's time, as the read-only path asks, so they come by coherent loads. These
// leave no line in L1, where nothing would read it again, and are not volatile, so that the compiler may place them
// freely (their addresses come from loads behind the wait for the grid before). Against plain loads: 64 query heads on 4
// key heads, 32 x 8192 8-bit tokens, 78.8 -> 74.5 us; 64 x 8192 of 16 heads of 64, 187.6 -> 179.5.
__device__ __forceinline__ uint4 load_once4(const void* p) {
  uint4 u;
  asm("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
}
__device__ __forceinline__ uint2 load_once2(const void* p) {
  uint2 u;
  asm("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p));
  return u;
}
__device__ __forceinline__ uint32_t load_once(const void* p) {
  uint32_t u;
  asm("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(u) : "l"(p));
  return u;
}

// 32-bit words of a token that one thread holds, and where they lie: vectors of up to 4 words; a thread's vectors are
// `lanes` vectors apart, so that each load of the warp covers consecutive bytes of a row.
template <int kWords, int kLanes>
struct RowPieces {
  static constexpr int kVec = kWords < 4 ? kWords : 4;
  static constexpr int kVectors = kWords / kVec;
  // Byte offset of word i of the thread at place `at` of kLanes.
  __device__ static __forceinline__ int offset(int i, int at) {
    return (i / kVec) * (4 * kVec * kLanes) + at * 4 * kVec + (i % kVec) * 4;
  }
  __device__ static __forceinline__ void load(const uint8_t* row, int at, uint32_t (&w)[kWords]) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      const uint8_t* src = row + v * (4 * kVec * kLanes) + at * 4 * kVec;
      if constexpr (kVec == 4) {
        const uint4 u = load_once4(src);
        w[4 * v] = u.x;
        w[4 * v + 1] = u.y;
        w[4 * v + 2] = u.z;
        w[4 * v + 3] = u.w;
      } else if constexpr (kVec == 2) {
        const uint2 u = load_once2(src);
        w[2 * v] = u.x;
        w[2 * v + 1] = u.y;
      } else {
        w[v] = load_once(src);
      }
    }
  }
};

__device__ __forceinline__ int cluster_nctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return static_cast<int>(r);
}
// From a shared::cluster address.
__device__ __forceinline__ float cluster_load(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

template <int HD, bool kFp8, int NT, int kShare>
struct CacheAttnCfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kBytes = kFp8 ? 1 : 2;
  static constexpr int kKWords = HD * kBytes / 16;  // of one token, per thread: 4 threads share a row of K,
  static constexpr int kVWords = HD * kBytes / 32;  // 8 a row of V
  static constexpr int kSteps = HD / 16;
  // A warp takes kSub tiles of 16 tokens at a time, interleaved: 4 KB of keys and values on their way per warp.
  static constexpr int kSub = 128 / (HD * kBytes * NT) > 1 ? 128 / (HD * kBytes * NT) : 1;
  // Registers decide the warps: the loads' (32, or 64 for 256-byte rows), O's and Q's (6 per row block and 16 dims). 16
  // warps an SM at 128 registers, 12 at 168, 8 at 255; in CTAs of 4, so that one that joins does not idle many (64
  // sequences of up to 8192 tokens: 116 us, 122 in CTAs of 8), or of 6 where 12 is the number.
  static constexpr bool kWide = HD == 128 && (!kFp8 || NT == 2);
  static constexpr bool kSharedQ = NT == 2 || (HD == 128 && kFp8);
  // kShare 1 or 4: a CTA takes a whole (sequence, head) with all the warps of an SM, or a quarter; kCacheCluster: a
  // cluster does, each CTA with those of an SM; 0: a stretch of the line.
  static constexpr int kWarpsPerSm = !kWide ? 16 : kFp8 || NT == 1 ? 12 : 8;
  static constexpr int kWarps = kShare > 0 ? kWarpsPerSm / (kShare == 4 ? 4 : 1) : kWarpsPerSm == 12 ? 6 : 4;
  static constexpr int kCtasPerSm = kWarpsPerSm / kWarps;
  static constexpr int kThreads = 32 * kWarps;
  // Units of a CTA's stretch at least (not of a head's): shorter ones cost more in the join than they save.
  static constexpr int kLeast = 16 / kWarps;
  static constexpr int kUnitTiles = kWarps * kSub;  // of 16 tokens: what a CTA takes at a time
  // Twelve warps with 8 KB on their way each need no prefetch (183 us with it, 168 without: 32 x 8192 tokens, 8 heads).
  static constexpr bool kPrefetch = !(kWide && !kFp8 && NT == 1);
  static constexpr int kLines = kSub * 2 * 16 * HD * kBytes / 128;  // 128-byte lines of a warp's part of a unit
  static constexpr int kPartial = kRows * (HD + 2);  // floats of one partial result: outputs, then maxima, then sums
  // Shared memory: the join of the warps' results, or the factors of the join of CTAs; then (batch + 1) first units.
  static constexpr int kSmemBytes = kWarps * kPartial * 4 > 24576 ? kWarps * kPartial * 4 : 24576;
};

// A stretch's part of one (sequence, head): units [u0, u1) of its `units`, the first of which is head_begin on the line.
struct Part {
  int b, h, head_begin, u0, u1, units;
  SeqTiles seq;
};

template <class Cfg>
__device__ __forceinline__ int seq_units(const CacheAttnParams& p, int b) {
  return max(1, (seq_tiles(p, seq_length(p, b)).count + Cfg::kUnitTiles - 1) / Cfg::kUnitTiles);
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <int HD, bool kFp8, int NT, int kShare>
__global__ void __launch_bounds__(CacheAttnCfg<HD, kFp8, NT, kShare>::kThreads,
                                  CacheAttnCfg<HD, kFp8, NT, kShare>::kCtasPerSm)
    cache_attention_kernel(const CacheAttnParams p) {
  using Cfg = CacheAttnCfg<HD, kFp8, NT, kShare>;
  constexpr bool kWhole = kShare > 0;
  constexpr bool kCluster = kShare == kCacheCluster;
  using KPieces = RowPieces<Cfg::kKWords, 4>;
  using VPieces = RowPieces<Cfg::kVWords, 8>;
  constexpr int R = Cfg::kRows;
  constexpr int kSub = Cfg::kSub;
  constexpr int kWarps = Cfg::kWarps;
  extern __shared__ __align__(16) uint8_t s_dyn[];
  float* s_merge = reinterpret_cast<float*>(s_dyn);
  int* s_first = reinterpret_cast<int*>(s_dyn + Cfg::kSmemBytes);  // [batch + 1] first unit of each sequence
  __shared__ uint2 s_q[Cfg::kSharedQ ? NT * Cfg::kSteps * 32 : 1];
  __shared__ int s_scan[kWarps];
  __shared__ Part s_part;  // what the join needs of `now`, out of the registers of the loop
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int kv_heads = p.c.kv_heads;
  const int rows_total = p.q_len * p.group;
  const int row_block = (p.block0 + static_cast<int>(blockIdx.y)) * R;

  pdl_wait_previous_grid();
  pdl_allow_next_grid();

  const int64_t cta = blockIdx.x;
  int64_t total = 0, ctas = 0;    // of units; of the CTAs that take some
  int w_begin = 0, w_end = 0;  // this one's stretch
  if constexpr (!kWhole) {
    // First unit of each sequence on the line of all units.
    int base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += Cfg::kThreads) {
      const int b = b0 + tid;
      int v = b < p.batch ? seq_units<Cfg>(p, b) * kv_heads : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) s_scan[warp] = v;
      __syncthreads();
      int before = base;
      int all = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += s_scan[i];
        all += s_scan[i];
      }
      if (b < p.batch) s_first[b + 1] = before + v;
      base += all;
      __syncthreads();
    }
    if (tid == 0) s_first[0] = 0;
    __syncthreads();
    total = base;
    ctas = min(static_cast<int64_t>(gridDim.x),
               max(static_cast<int64_t>(p.batch) * kv_heads, (total + Cfg::kLeast - 1) / Cfg::kLeast));
    if (cta >= ctas) return;
    w_begin = static_cast<int>(cta * total / ctas);
    w_end = static_cast<int>((cta + 1) * total / ctas);
  }

  constexpr int kNoTile = 1 << 30;         // a first token that no row sees
  constexpr int kIds = 32 / kSub;          // units whose page numbers the lanes hold
  constexpr int kAhead = kIds > 4 ? 3 : 2;  // units that the prefetch into L2 runs ahead
  const int page_bytes = static_cast<int>(p.c.page_stride) * Cfg::kBytes;  // below 2^31 (checked by the host)
  const int slot_mask = (1 << p.c.page_shift) - 1;

  auto part_from = [&](int w, int b) {
    Part x;
    while (s_first[b + 1] <= w) ++b;
    x.b = b;
    x.seq = seq_tiles(p, seq_length(p, b));
    x.units = (s_first[b + 1] - s_first[b]) / kv_heads;
    x.h = (w - s_first[b]) / x.units;
    x.head_begin = s_first[b] + x.h * x.units;
    x.u0 = w - x.head_begin;
    x.u1 = min(x.units, w_end - x.head_begin);
    return x;
  };
  // Lane l: the first token (kNoTile: none) and the page of this warp's tile l % kSub in unit ids_from + l / kSub.
  int my_tok = kNoTile, my_page = 0, ids_from = 0;
  auto read_ids = [&](const Part& x, int u) {
    ids_from = u;
    const int i = ((u + lane / kSub) * kWarps + warp) * kSub + lane % kSub;
    my_tok = kNoTile;
    my_page = 0;
    if (i < x.seq.count) {
      my_tok = 16 * (i < x.seq.sink_tiles ? i : i - x.seq.sink_tiles + x.seq.first_win);
      my_page = p.page_table[x.b * p.ld_table + (my_tok >> p.c.page_shift)];
      if (my_page < 0 || my_page >= p.c.pages) {
        record_status(kKernelCacheAttention, 2, kReasonBadIndex);
        my_tok = kNoTile;
        my_page = 0;
      }
    }
  };
  // The lines of the warp's part of unit u into L2, a lane each.
  auto prefetch = [&](const Part& x, int u) {
    constexpr int kTileLines = Cfg::kLines / kSub;  // K's, then V's
#pragma unroll
    for (int line0 = 0; line0 < Cfg::kLines; line0 += 32) {
      const int line = line0 + lane;
      const int src = min((u - ids_from) * kSub + line / kTileLines, 31);
      const int tok = __shfl_sync(0xffffffffu, my_tok, src);
      const int page = __shfl_sync(0xffffffffu, my_page, src);
      const int in = line % kTileLines;
      const bool keys = in < kTileLines / 2;
      if (u < x.u1 && (Cfg::kLines % 32 == 0 || line < Cfg::kLines) && tok != kNoTile)
        prefetch_l2((keys ? p.c.k : p.c.v) + static_cast<int64_t>(page) * page_bytes + x.h * p.c.head_stride * Cfg::kBytes +
                    (tok & slot_mask) * (HD * Cfg::kBytes) + (keys ? in : in - kTileLines / 2) * 128);
    }
  };
  Part now;
  const int rank = kCluster ? static_cast<int>(cluster_ctarank()) : 0;
  const int ranks = kCluster ? cluster_nctarank() : 1;  // a power of two
  const int ranks_shift = __ffs(ranks) - 1;
  if constexpr (kWhole) {
    const int head = static_cast<int>(blockIdx.x) >> ranks_shift;
    now.b = head / kv_heads;
    now.h = head - now.b * kv_heads;
    now.seq = seq_tiles(p, seq_length(p, now.b));
    now.units = max(1, (now.seq.count + Cfg::kUnitTiles - 1) / Cfg::kUnitTiles);
    now.head_begin = 0;
    now.u0 = static_cast<int>(static_cast<int64_t>(rank) * now.units >> ranks_shift);
    now.u1 = static_cast<int>(static_cast<int64_t>(rank + 1) * now.units >> ranks_shift);
  } else {
    int lo = 0, hi = p.batch;  // s_first[lo] <= w_begin < s_first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_first[mid] <= w_begin) lo = mid; else hi = mid;
    }
    now = part_from(w_begin, lo);
  }
  while (true) {
    read_ids(now, now.u0);
    if (tid == 0) s_part = now;
    const SeqTiles seq = now.seq;
    const int64_t head_bytes = now.h * p.c.head_stride * Cfg::kBytes;

    // Q: fragments of the 8-row operand(s), and the factor of its rows' scores.
    uint32_t qf[NT][Cfg::kSteps][2];  // (in shared memory where registers are short: it is alike for every warp)
    float row_scale[NT][2];
    int limit[NT][2];  // position of the rows 2t, 2t + 1 of each operand, -1: no such row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row_block + 8 * nt + g;
      const bool real = row < rows_total;
      const __nv_bfloat16* src =
          p.q + (static_cast<int64_t>(now.b) * p.q_len + (real ? row / p.group : 0)) * p.ld_q +
          (now.h * p.group + (real ? row % p.group : 0)) * HD;
      if constexpr (kFp8) {
        float f[Cfg::kSteps][4];
        float amax = 0.f;
#pragma unroll
        for (int s = 0; s < Cfg::kSteps; ++s) {
          const uint2 u = real ? *reinterpret_cast<const uint2*>(src + KPieces::offset(s, t)) : make_uint2(0, 0);
          f[s][0] = __uint_as_float(u.x << 16);
          f[s][1] = __uint_as_float(u.x & 0xffff0000u);
          f[s][2] = __uint_as_float(u.y << 16);
          f[s][3] = __uint_as_float(u.y & 0xffff0000u);
#pragma unroll
          for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(f[s][i]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^(14 - e) for the largest element's exponent e, both factors kept normal.
        const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100), 127);
        const float up = exp2_int(14 - e);
#pragma unroll
        for (int s = 0; s < Cfg::kSteps; ++s) {
          qf[nt][s][0] = pack_f16x2(f[s][0] * up, f[s][1] * up);
          qf[nt][s][1] = pack_f16x2(f[s][2] * up, f[s][3] * up);
        }
        const float down = exp2_int(e - 14) * p.scale_log2;
        row_scale[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t);      // the thread that holds row 2t
        row_scale[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);  // row 2t + 1
      } else {
#pragma unroll
        for (int s = 0; s < Cfg::kSteps; ++s) {
          qf[nt][s][0] = real ? *reinterpret_cast<const uint32_t*>(src + KPieces::offset(2 * s, t) / 2) : 0u;
          qf[nt][s][1] = real ? *reinterpret_cast<const uint32_t*>(src + KPieces::offset(2 * s + 1, t) / 2) : 0u;
        }
        row_scale[nt][0] = row_scale[nt][1] = p.scale_log2;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = row_block + 8 * nt + 2 * t + i;
        limit[nt][i] = r < rows_total ? seq.len - p.q_len + r / p.group : -1;
      }
    }

    if constexpr (Cfg::kSharedQ) {
      if (warp == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int st = 0; st < Cfg::kSteps; ++st)
            s_q[(nt * Cfg::kSteps + st) * 32 + lane] = make_uint2(qf[nt][st][0], qf[nt][st][1]);
      }
      __syncthreads();
    }

    float o[NT][Cfg::kSteps][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < Cfg::kSteps; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][j][i] = 0.f;
    }

    // (behind Q's loads, which need not wait for the page numbers; the first unit's own loads come next)
    if (Cfg::kPrefetch) {
#pragma unroll
      for (int d = 1; d < kAhead; ++d) prefetch(now, now.u0 + d);
    }

    // Tokens that every row sees lie below `all_see`, and (with a window) from `all_from` on or below the sinks.
    const int all_see = seq.len - p.q_len + 1;
    const int all_from = p.window > 0 ? max(0, seq.len - p.window) : 0;

#pragma unroll 1
    for (int u = now.u0; u < now.u1; ++u) {
      if ((u * kWarps + warp) * kSub >= seq.count) break;
      if (u + kAhead >= ids_from + kIds && ids_from + kIds < now.u1) read_ids(now, u);
      uint32_t kr[kSub][2][Cfg::kKWords], vr[kSub][4][Cfg::kVWords];
      float ks[kSub], vs[kSub];
      int tok[kSub];
#pragma unroll
      for (int c = 0; c < kSub; ++c) {
        const int src = (u - ids_from) * kSub + c;
        tok[c] = __shfl_sync(0xffffffffu, my_tok, src);
        const int page = __shfl_sync(0xffffffffu, my_page, src);
        // (a tile that is missing reads page 0, slot 0, whosever it is, and is masked)
        const int64_t at = static_cast<int64_t>(page) * page_bytes + head_bytes + (tok[c] & slot_mask) * (HD * Cfg::kBytes);
#pragma unroll
        for (int x = 0; x < 2; ++x) KPieces::load(p.c.k + at + (g + 8 * x) * (HD * Cfg::kBytes), t, kr[c][x]);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          VPieces::load(p.c.v + at + (2 * t + (x & 1) + 4 * (x & 2)) * (HD * Cfg::kBytes), g, vr[c][x]);
        ks[c] = vs[c] = 1.f;
        if (kFp8) {
          ks[c] = p.c.k_scale[static_cast<int64_t>(page) * kv_heads + now.h];
          vs[c] = p.c.v_scale[static_cast<int64_t>(page) * kv_heads + now.h];
        }
      }
      if (Cfg::kPrefetch) prefetch(now, u + kAhead);

      float s[kSub][NT][4];
#pragma unroll
      for (int c = 0; c < kSub; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[c][nt][0] = s[c][nt][1] = s[c][nt][2] = s[c][nt][3] = 0.f;
#pragma unroll
      for (int st = 0; st < Cfg::kSteps; ++st)
#pragma unroll
        for (int c = 0; c < kSub; ++c) {
          uint32_t a0, a1, a2, a3;
          if constexpr (kFp8) {
            a0 = e4m3x2_to_f16x2(kr[c][0][st]);
            a1 = e4m3x2_to_f16x2(kr[c][1][st]);
            a2 = e4m3x2_to_f16x2(kr[c][0][st] >> 16);
            a3 = e4m3x2_to_f16x2(kr[c][1][st] >> 16);
          } else {
            a0 = kr[c][0][2 * st];
            a1 = kr[c][1][2 * st];
            a2 = kr[c][0][2 * st + 1];
            a3 = kr[c][1][2 * st + 1];
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint2 q2 = make_uint2(qf[nt][st][0], qf[nt][st][1]);
            if constexpr (Cfg::kSharedQ) q2 = s_q[(nt * Cfg::kSteps + st) * 32 + lane];
            cache_mma<kFp8>(s[c][nt], a0, a1, a2, a3, q2.x, q2.y);
          }
        }

      // Tokens g and g + 8 of rows 2t and 2t + 1, in exponents of 2 with V's scale in.
      float inv_v[kSub];
      bool edge = false;
#pragma unroll
      for (int c = 0; c < kSub; ++c) {
        float ev = 0.f;
        inv_v[c] = 1.f;
        if (kFp8) {
          const int e = static_cast<int>(__float_as_uint(vs[c]) >> 23) - 127;
          ev = static_cast<float>(e);
          inv_v[c] = exp2_int(-e);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[c][nt][x] = fmaf(s[c][nt][x], row_scale[nt][x & 1] * ks[c], ev);
        edge |= tok[c] + 16 > all_see || (tok[c] < all_from && tok[c] + 16 > p.sinks);
      }
      if (edge) {
        const int from = max(0, seq.len - p.q_len - p.window + 1);
#pragma unroll
        for (int c = 0; c < kSub; ++c) {
          if (tok[c] == kNoTile) inv_v[c] = 1.f;  // of a scale that may be anything: its weights are 0, but 0 times a NaN is a NaN
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int j = tok[c] + g + 8 * (x >> 1);
              const int pos = limit[nt][x & 1];
              if (j > pos || (p.window > 0 && pos - j >= p.window && j >= p.sinks)) s[c][nt][x] = -INFINITY;
            }
          // Values of tokens that no row sees may be anything (0 times a NaN is a NaN).
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = tok[c] + 2 * t + (x & 1) + 4 * (x & 2);
            if (j >= seq.len || (p.window > 0 && j < from && j >= p.sinks)) {
#pragma unroll
              for (int i2 = 0; i2 < Cfg::kVWords; ++i2) vr[c][x][i2] = 0u;
            }
          }
        }
      }

      bool grew = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[nt][x] = fmaxf(s[0][nt][x], s[0][nt][x + 2]);
#pragma unroll
          for (int c = 1; c < kSub; ++c) top[nt][x] = max3f(top[nt][x], s[c][nt][x], s[c][nt][x + 2]);
          grew |= top[nt][x] > m[nt][x] + kCacheRescale;
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float best = top[nt][x];
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 4));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 8));
            best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 16));
            if (best > m[nt][x]) {
              const float alpha = fast_exp2(m[nt][x] - best);  // 0 the first time
              m[nt][x] = best;
              l[nt][x] *= alpha;
#pragma unroll
              for (int j = 0; j < Cfg::kSteps; ++j) {
                o[nt][j][x] *= alpha;
                o[nt][j][x + 2] *= alpha;
              }
            }
          }
      }

      uint32_t pf[kSub][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float ref0 = m[nt][0] == -INFINITY ? -kCacheHeadroom : m[nt][0] - kCacheHeadroom;
        const float ref1 = m[nt][1] == -INFINITY ? -kCacheHeadroom : m[nt][1] - kCacheHeadroom;
#pragma unroll
        for (int c = 0; c < kSub; ++c) {
          const float w0 = fast_exp2(s[c][nt][0] - ref0), w1 = fast_exp2(s[c][nt][1] - ref1);
          const float w2 = fast_exp2(s[c][nt][2] - ref0), w3 = fast_exp2(s[c][nt][3] - ref1);
          l[nt][0] = fmaf(w0 + w2, inv_v[c], l[nt][0]);
          l[nt][1] = fmaf(w1 + w3, inv_v[c], l[nt][1]);
          pf[c][nt][0] = movmatrix_trans(kFp8 ? pack_f16x2(w0, w1) : pack_bf16x2(w0, w1));
          pf[c][nt][1] = movmatrix_trans(kFp8 ? pack_f16x2(w2, w3) : pack_bf16x2(w2, w3));
        }
      }

#pragma unroll
      for (int c = 0; c < kSub; ++c) {
        if constexpr (kFp8) {
#pragma unroll
          for (int i2 = 0; i2 < Cfg::kVWords; ++i2) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t sel = half ? 0x7362u : 0x5140u;
              const uint32_t lo = __byte_perm(vr[c][0][i2], vr[c][1][i2], sel);  // tokens 2t, 2t+1 of two dims
              const uint32_t hi = __byte_perm(vr[c][2][i2], vr[c][3][i2], sel);  // tokens 2t+8, 2t+9
              const uint32_t a0 = e4m3x2_to_f16x2(lo), a1 = e4m3x2_to_f16x2(lo >> 16);
              const uint32_t a2 = e4m3x2_to_f16x2(hi), a3 = e4m3x2_to_f16x2(hi >> 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                cache_mma<kFp8>(o[nt][2 * i2 + half], a0, a1, a2, a3, pf[c][nt][0], pf[c][nt][1]);
            }
          }
        } else {
#pragma unroll
          for (int i2 = 0; i2 < Cfg::kVWords; ++i2) {
            const uint32_t a0 = __byte_perm(vr[c][0][i2], vr[c][1][i2], 0x5410u);
            const uint32_t a1 = __byte_perm(vr[c][0][i2], vr[c][1][i2], 0x7632u);
            const uint32_t a2 = __byte_perm(vr[c][2][i2], vr[c][3][i2], 0x5410u);
            const uint32_t a3 = __byte_perm(vr[c][2][i2], vr[c][3][i2], 0x7632u);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) cache_mma<kFp8>(o[nt][i2], a0, a1, a2, a3, pf[c][nt][0], pf[c][nt][1]);
          }
        }
      }
    }

    // The warps' results into shared memory, each [row][dim], maxima, sums.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 4);
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 8);
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 16);
        const int r = 8 * nt + 2 * t + x;
        float* dst = s_merge + warp * Cfg::kPartial;
#pragma unroll
        for (int j = 0; j < Cfg::kSteps; ++j) {
          const int d = kFp8 ? VPieces::offset(j / 2, g) + 2 * (j & 1) : VPieces::offset(j, g) / 2;
          *reinterpret_cast<float2*>(dst + r * HD + d) = make_float2(o[nt][j][x], o[nt][j][x + 2]);
        }
        if (g == 0) {
          dst[R * HD + r] = m[nt][x];
          dst[R * HD + R + r] = l[nt][x];
        }
      }
    __syncthreads();

    const volatile Part& part_now = s_part;
    const int b = part_now.b, h = part_now.h, head_begin = part_now.head_begin, units = part_now.units;
    const int u0 = part_now.u0, u1 = part_now.u1;
    // One row's output, joined: into `out` as bf16, or with its maximum and sum into a partial result.
    const int rows = min(R, rows_total - row_block);
    auto finish = [&](int r, int d, float2 acc, float sum) {
      const int row = row_block + r;
      // sum is 0 only where nothing is visible; a NaN stays one.
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (sum == 0.f) acc = make_float2(0.f, 0.f);
      *reinterpret_cast<uint32_t*>(
          p.out + (static_cast<int64_t>(b) * p.q_len + row / p.group) * p.ld_out + (h * p.group + row % p.group) * HD + d) =
          pack_bf16x2(acc.x * inv, acc.y * inv);
    };
    const bool whole = kWhole ? !kCluster : u1 - u0 == units;
    const int64_t mine = static_cast<int64_t>(blockIdx.y) * gridDim.x * 2;
    // Slot 0 of a CTA: the part of a head that began before its stretch (or with it); slot 1: of one that begins inside.
    // (Of a cluster: in shared memory.)
    float* const s_partial = reinterpret_cast<float*>(s_dyn + Cfg::kSmemBytes);
    float* partial = kWhole ? s_partial : p.partials + (mine + cta * 2 + (w_begin >= head_begin ? 0 : 1)) * Cfg::kPartial;
    for (int i = tid; i < rows * (HD / 2); i += Cfg::kThreads) {
      const int r = i / (HD / 2), d = 2 * (i - r * (HD / 2));
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) top = fmaxf(top, s_merge[k * Cfg::kPartial + R * HD + r]);
      const float ref = top == -INFINITY ? 0.f : top;
      float2 acc = make_float2(0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float* one = s_merge + k * Cfg::kPartial;
        const float f = fast_exp2(one[R * HD + r] - ref);
        const float2 v = *reinterpret_cast<const float2*>(one + r * HD + d);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        sum = fmaf(one[R * HD + R + r], f, sum);
      }
      if (whole) {
        finish(r, d, acc, sum);
      } else {
        *reinterpret_cast<float2*>(partial + r * HD + d) = acc;
        if (d == 0) {
          partial[R * HD + r] = top;
          partial[R * HD + R + r] = sum;
        }
      }
    }
    if constexpr (kCluster) {
      // The cluster's partial results, in the order of its CTAs, each of which joins a share of the outputs.
      cluster_sync_all();
      for (int i = rank * Cfg::kThreads + tid; i < rows * (HD / 2); i += ranks * Cfg::kThreads) {
        const int r = i / (HD / 2), d = 2 * (i - r * (HD / 2));
        float top = -INFINITY, sum = 0.f;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int k0 = 0; k0 < ranks; k0 += 8) {
          float m_of[8], l_of[8];
          float2 v_of[8];
          const float before = top;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            m_of[k] = -INFINITY;
            l_of[k] = 0.f;
            v_of[k] = make_float2(0.f, 0.f);
            if (k0 + k < ranks) {
              const uint32_t at = cluster_map_to_rank(s_partial, k0 + k);
              m_of[k] = cluster_load(at + 4 * (R * HD + r));
              l_of[k] = cluster_load(at + 4 * (R * HD + R + r));
              v_of[k] = cluster_load2(at + 4 * (r * HD + d));
            }
            top = fmaxf(top, m_of[k]);
          }
          const float ref = top == -INFINITY ? 0.f : top;
          const float old = fast_exp2(before - ref);
          acc = make_float2(acc.x * old, acc.y * old);
          sum *= old;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float f = fast_exp2(m_of[k] - ref);
            acc.x = fmaf(v_of[k].x, f, acc.x);
            acc.y = fmaf(v_of[k].y, f, acc.y);
            sum = fmaf(l_of[k], f, sum);
          }
        }
        finish(r, d, acc, sum);
      }
      cluster_sync_all();  // nobody leaves while others read from it
    }
    if constexpr (!kWhole) if (!whole) {
      // Joins of CTAs' parts, in their order on the line. Up to kCacheAtOnce parts in one go; more (few sequences with few
      // key heads) first in groups of kCacheGroup CTAs, whose result takes the place of its first part.
      const int64_t c_first = ((static_cast<int64_t>(head_begin) + 1) * ctas - 1) / total;
      const int64_t c_last = (static_cast<int64_t>(head_begin + units) * ctas - 1) / total;
      auto part = [&](int64_t c) {
        return p.partials + (mine + c * 2 + (c * total / ctas >= head_begin ? 0 : 1)) * Cfg::kPartial;
      };
      // True (in every thread) for the last of n arrivals; all their writes are then visible past this SM's L1.
      auto last_of = [&](int* counter, int n) {
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          const int last = atomicAdd(counter, 1) == n - 1;
          if (last) *counter = 0;
          s_last = last;
        }
        __syncthreads();
        const bool last = s_last != 0;
        if (last) __threadfence();
        return last;
      };
      // Parts of the CTAs c_from(k), k < n.
      auto join = [&](auto c_from, int n, float* into) {
        const float** s_at = reinterpret_cast<const float**>(s_merge);  // [n]
        float* s_f = reinterpret_cast<float*>(s_at + n);                // [n][R] maxima, then factors
        float* s_l = s_f + n * R;                                       // [n][R] sums
        float* s_row = s_l + n * R;                                     // [2][R] joined sums and maxima
        if (tid < n) s_at[tid] = part(c_from(tid));
        __syncthreads();
        for (int i = tid; i < n * 2 * R; i += Cfg::kThreads) {
          const int k = i / (2 * R), x = i - k * 2 * R;
          (x < R ? s_f + k * R + x : s_l + k * R + x - R)[0] = __ldcg(s_at[k] + R * HD + x);
        }
        __syncthreads();
        if (tid < rows) {
          float top = -INFINITY;
          for (int k = 0; k < n; ++k) top = fmaxf(top, s_f[k * R + tid]);
          const float ref = top == -INFINITY ? 0.f : top;
          float sum = 0.f;
          for (int k = 0; k < n; ++k) {
            const float f = fast_exp2(s_f[k * R + tid] - ref);
            s_f[k * R + tid] = f;
            sum = fmaf(s_l[k * R + tid], f, sum);
          }
          s_row[tid] = sum;
          s_row[R + tid] = top;
        }
        __syncthreads();
        // Four dims to a thread; where that leaves threads over, they share the parts.
        const int quads = rows * (HD / 4);
        const int shares = max(1, Cfg::kThreads / quads);
        float4* s_acc = reinterpret_cast<float4*>(s_merge + (n * (2 * R + 2) + 2 * R + 3) / 4 * 4);  // [shares][quads]
        for (int i0 = 0; i0 < quads; i0 += Cfg::kThreads) {
          const int share = shares > 1 ? tid / quads : 0;
          const int i = shares > 1 ? tid - share * quads : i0 + tid;
          const int r = i / (HD / 4), d = 4 * (i - r * (HD / 4));
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i < quads && share < shares) {
#pragma unroll 8
            for (int k = share; k < n; k += shares) {
              const float4 v = __ldcg(reinterpret_cast<const float4*>(s_at[k] + r * HD + d));
              const float f = s_f[k * R + r];
              acc.x = fmaf(v.x, f, acc.x);
              acc.y = fmaf(v.y, f, acc.y);
              acc.z = fmaf(v.z, f, acc.z);
              acc.w = fmaf(v.w, f, acc.w);
            }
          }
          if (shares > 1) {
            if (share < shares) s_acc[share * quads + i] = acc;
            __syncthreads();
            if (share == 0) {
              for (int x = 1; x < shares; ++x) {
                const float4 v = s_acc[x * quads + i];
                acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
              }
            }
          }
          if (i < quads && share == 0) {
            if (into == nullptr) {
              finish(r, d, make_float2(acc.x, acc.y), s_row[r]);
              finish(r, d + 2, make_float2(acc.z, acc.w), s_row[r]);
            } else {
              *reinterpret_cast<float4*>(into + r * HD + d) = acc;
              if (d == 0) {
                into[R * HD + r] = s_row[R + r];
                into[R * HD + R + r] = s_row[r];
              }
            }
          }
        }
        __syncthreads();
      };
      const int n = static_cast<int>(c_last - c_first) + 1;
      // Of the heads that a stretch holds, only its last one can go on behind it: one counter a CTA is enough.
      int* head_counter = p.counters + static_cast<int64_t>(blockIdx.y) * gridDim.x + c_first;
      if (n <= kCacheAtOnce) {
        if (last_of(head_counter, n)) join([&](int k) { return c_first + k; }, n, nullptr);
      } else {
        const int64_t group = cta / kCacheGroup;
        const int64_t g_first = max(c_first, group * kCacheGroup), g_last = min(c_last, group * kCacheGroup + kCacheGroup - 1);
        // Of the heads that cross a border of the group, one crosses its first (or both), one only its last.
        int* group_counter = p.group_counters + ((static_cast<int64_t>(blockIdx.y) * gridDim.x / kCacheGroup + blockIdx.y + group) * 2 +
                                                 (c_first < group * kCacheGroup ? 0 : 1));
        const int members = static_cast<int>(g_last - g_first) + 1;
        const int64_t groups_from = c_first / kCacheGroup;
        const int groups = static_cast<int>(c_last / kCacheGroup - groups_from) + 1;
        if (last_of(group_counter, members)) {
          join([&](int k) { return g_first + k; }, members, part(g_first));
          if (last_of(head_counter, groups))
            join([&](int k) { return max(c_first, (groups_from + k) * kCacheGroup); }, groups, nullptr);
        }
      }
    }
    if (kWhole || head_begin + u1 >= w_end) break;
    __syncthreads();
    now = part_from(head_begin + u1, b);
  }
}

// CTAs of a launch of the line form, at most (CacheAttnCfg::kCtasPerSm of both types), and the bytes of its workspace.
static int cache_attention_ctas(int64_t head_dim, int nt, int sm_count) {
  return (head_dim == 128 && nt == 2 ? 2 : 4) * sm_count;
}

// Rows of a block: 8, or 16 where there are more than 8 rows (a block reads the keys and values anew).
static int64_t cache_attention_row_blocks(int64_t rows, int* nt) {
  *nt = rows <= 8 ? 1 : 2;
  return (rows + 8 * *nt - 1) / (8 * *nt);
}

// Counters of the heads, then of the groups, at the start of a workspace: as many for every call, so that no call's
// partial results lie where another's counters do, whatever their sizes and in whatever order they come.
static int64_t cache_attention_head_counters(int sm_count) { return kCacheBlocksAtOnce * 4 * static_cast<int64_t>(sm_count); }

static int64_t cache_attention_counter_bytes(int sm_count) {
  const int64_t groups = kCacheBlocksAtOnce * (4 * static_cast<int64_t>(sm_count) / kCacheGroup + 1) * 2;
  return ((cache_attention_head_counters(sm_count) + groups) * 4 + 255) / 256 * 256;
}

static int64_t cache_attention_partial_bytes(int64_t head_dim, int64_t rows, int sm_count) {
  int nt = 1;
  const int64_t blocks = std::min<int64_t>(cache_attention_row_blocks(rows, &nt), kCacheBlocksAtOnce);
  return (blocks * cache_attention_ctas(head_dim, nt, sm_count) * 2 * (8 * nt) * (head_dim + 2) * 4 + 255) / 256 * 256;
}

static int64_t cache_attention_workspace_bytes(int64_t head_dim, int64_t rows, int sm_count) {
  return cache_attention_counter_bytes(sm_count) + cache_attention_partial_bytes(head_dim, rows, sm_count);
}

// A launch with programmatic dependence in clusters of `cluster` CTAs along x.
struct CacheClusterLaunch {
  cudaLaunchConfig_t config = {};
  cudaLaunchAttribute attr[2];
  CacheClusterLaunch(dim3 grid, int threads, int cluster, size_t smem, cudaStream_t stream) {
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 2;
  }
};

// How many clusters of `cluster` CTAs run side by side on the current device. (It depends on which SMs a GPU has in each
// of its parts: 16 SMs next to each other were found for 6 clusters, not for 8.)
template <int HD, bool kFp8, int NT>
static cudaError_t cache_attention_clusters(int cluster, int* side_by_side) {
  using Cfg = CacheAttnCfg<HD, kFp8, NT, kCacheCluster>;
  const auto kernel = cache_attention_kernel<HD, kFp8, NT, kCacheCluster>;
  constexpr int kSmem = Cfg::kSmemBytes + Cfg::kPartial * 4;
  static std::once_flag once[64];
  static int fit[64][kCacheCluster + 1];
  static cudaError_t result[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  dev &= 63;
  std::call_once(once[dev], [&] {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    for (int c = 2; e == cudaSuccess && c <= kCacheCluster; c *= 2) {
      const CacheClusterLaunch launch(dim3(c), Cfg::kThreads, c, kSmem, nullptr);
      e = cudaOccupancyMaxActiveClusters(&fit[dev][c], kernel, &launch.config);
    }
    result[dev] = e;
  });
  *side_by_side = fit[dev][cluster];
  return result[dev];
}

template <int HD, bool kFp8, int NT>
static cudaError_t launch_cache_attention_cluster(const CacheAttnParams& p, int64_t row_blocks, int cluster,
                                                  cudaStream_t stream) {
  using Cfg = CacheAttnCfg<HD, kFp8, NT, kCacheCluster>;
  const CacheClusterLaunch launch(dim3(p.batch * p.c.kv_heads * cluster, static_cast<unsigned>(row_blocks)), Cfg::kThreads,
                                  cluster, Cfg::kSmemBytes + Cfg::kPartial * 4, stream);
  return cudaLaunchKernelEx(&launch.config, cache_attention_kernel<HD, kFp8, NT, kCacheCluster>, p);
}

template <int HD, bool kFp8, int NT, int kShare>
static cudaError_t launch_cache_attention_t(const CacheAttnParams& p, int64_t row_blocks, int sm_count, cudaStream_t stream) {
  using Cfg = CacheAttnCfg<HD, kFp8, NT, kShare>;
  const size_t smem = Cfg::kSmemBytes + (kShare > 0 ? 0 : (static_cast<size_t>(p.batch) + 1) * 4);
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(cache_attention_kernel<HD, kFp8, NT, kShare>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Cfg::kSmemBytes + (kShare > 0 ? 0 : 4 * (kCacheMaxBatch + 1)));
  });
  if (e != cudaSuccess) return e;
  if constexpr (kShare > 0) {
    return launch_pdl(cache_attention_kernel<HD, kFp8, NT, kShare>,
                      dim3(p.batch * p.c.kv_heads, static_cast<unsigned>(row_blocks)), dim3(Cfg::kThreads), smem, stream, p);
  } else {
    static_assert(Cfg::kCtasPerSm <= (HD == 128 && NT == 2 ? 2 : 4), "as cache_attention_ctas says");
    CacheAttnParams turn = p;
    for (int64_t block = 0; block < row_blocks && e == cudaSuccess; block += kCacheBlocksAtOnce) {
      turn.block0 = static_cast<int>(block);
      const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(row_blocks - block, kCacheBlocksAtOnce));
      e = launch_pdl(cache_attention_kernel<HD, kFp8, NT, kShare>, dim3(sm_count * Cfg::kCtasPerSm, blocks),
                     dim3(Cfg::kThreads), smem, stream, turn);
    }
    return e;
  }
}

template <int HD, bool kFp8, int NT>
static cudaError_t launch_cache_attention_nt(const CacheAttnParams& p, int64_t row_blocks, int sm_count, cudaStream_t stream) {
  // The most tokens that a sequence can see; the host does not know their lengths.
  const int64_t room = static_cast<int64_t>(p.table_pages) << p.c.page_shift;
  const int64_t band = static_cast<int64_t>(p.window) + p.sinks + p.q_len + 32;
  const bool windowed = p.window > 0 && band < room;
  const int64_t tokens = windowed ? band : room;
  // A head to itself saves the line's sums, the start of a second part and the joins through global memory, 5 to 15 us;
  // a stretch saves what long or unlike heads leave idle. Up to as many heads as SMs, each gets an SM; of more than two
  // rounds of its warps, a cluster of 2, 4, 8 or 16 SMs, up to one a round (8 heads of 1000 tokens: 8.3 us, 10.0 on one SM
  // each; 4 of 16000 12.9 in sixteens, 16.4 in eights), as far as all heads' clusters run side by side (16 heads in eights
  // took two turns, 15.5 us, 9.9 in fours). More heads get a quarter of an SM each. How many rounds are taken
  // so depends on the share of the places, SMs or quarters, that the heads fill in their last turn.
  // Measured, us, heads / stretches, 8-bit heads of 128 unless said:
  //   two thirds, up to 32 rounds: 32 heads of 2000 tokens 10.2 / 14.7, of 16000 31.0 / 39.1, of up to 32000 48 / 47; 128 heads
  //     of 4096 28.9 / 39.4, of up to 8192 46.0 / 42.5, of up to 16384 83 / 73; 512 heads of 2000 47.8 / 57.2;
  //   two thirds behind a window, which makes lengths alike, up to 72: windows of 4096 of 100 heads 29.0 / 35.7, of 512
  //     heads 90.9 / 99.3 (of 8192 165.5 / 164.3), of 128 bf16 heads with 10 rows 51.6 / 64.0;
  //   a third, or in quarters, up to 20: 8 heads of 8000 12.5 / 19.5, of 32000 28.2 / 29.4, of 64000 47 / 39; 256 heads
  //     of 1000 20.8 / 28.0, of 4000 62.6 / 58.7;
  //   else up to 8: 4 heads of 8000 10.4 / 18.0, of 32000 17.4 / 20.2; 1 of 8000 9.9 / 13.5, of 32000 16.7 / 17.1.
  const int64_t heads = static_cast<int64_t>(p.batch) * p.c.kv_heads * row_blocks;
  const bool sm_each = heads <= sm_count;
  const int64_t round = 16 * (sm_each ? CacheAttnCfg<HD, kFp8, NT, 1>::kUnitTiles : CacheAttnCfg<HD, kFp8, NT, 4>::kUnitTiles);
  int cluster = 1;
  if (sm_each && tokens > 2 * round) {
    while (cluster < kCacheCluster && tokens > cluster * round) {
      int side_by_side = 0;
      const cudaError_t e = cache_attention_clusters<HD, kFp8, NT>(2 * cluster, &side_by_side);
      if (e != cudaSuccess) return e;
      if (heads > side_by_side) break;
      cluster *= 2;
    }
  }
  const int64_t places = sm_each ? sm_count : 4 * static_cast<int64_t>(sm_count);
  const int64_t ctas = heads * cluster;
  const int64_t thirds = 3 * ctas / ((ctas + places - 1) / places * places);
  const int64_t most = thirds >= 2 ? (windowed ? 72 : 32) : thirds == 1 || !sm_each ? 20 : 8;
  if (tokens <= most * cluster * round) {
    if (cluster > 1)
      return launch_cache_attention_cluster<HD, kFp8, NT>(p, row_blocks, cluster, stream);
    if (sm_each) return launch_cache_attention_t<HD, kFp8, NT, 1>(p, row_blocks, sm_count, stream);
    return launch_cache_attention_t<HD, kFp8, NT, 4>(p, row_blocks, sm_count, stream);
  }
  return launch_cache_attention_t<HD, kFp8, NT, 0>(p, row_blocks, sm_count, stream);
}

template <int HD>
static cudaError_t launch_cache_attention_hd(const CacheAttnParams& p, bool fp8, int nt, int64_t row_blocks, int sm_count,
                                             cudaStream_t stream) {
  if (fp8)
    return nt == 1 ? launch_cache_attention_nt<HD, true, 1>(p, row_blocks, sm_count, stream)
                   : launch_cache_attention_nt<HD, true, 2>(p, row_blocks, sm_count, stream);
  return nt == 1 ? launch_cache_attention_nt<HD, false, 1>(p, row_blocks, sm_count, stream)
                 : launch_cache_attention_nt<HD, false, 2>(p, row_blocks, sm_count, stream);
}

static cudaError_t launch_cache_attention(CacheAttnParams p, void* workspace, bool fp8, int sm_count, cudaStream_t stream) {
  int nt = 1;
  const int64_t rows = static_cast<int64_t>(p.q_len) * p.group;
  const int64_t blocks = cache_attention_row_blocks(rows, &nt);
  p.counters = static_cast<int*>(workspace);
  p.group_counters = p.counters + cache_attention_head_counters(sm_count);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + cache_attention_counter_bytes(sm_count));
  switch (p.c.head_dim) {
    case 32:
      return launch_cache_attention_hd<32>(p, fp8, nt, blocks, sm_count, stream);
    case 64:
      return launch_cache_attention_hd<64>(p, fp8, nt, blocks, sm_count, stream);
    case 128:
      return launch_cache_attention_hd<128>(p, fp8, nt, blocks, sm_count, stream);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace b2
