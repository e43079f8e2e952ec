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
//
// Split: every (sequence, key head) is cut into units of 16 tokens per warp, all units of the call are laid on one line
// and the CTAs take equal stretches of it, so that one long sequence among short ones, and few sequences on 148 SMs, fill the
// machine alike. A CTA whose stretch holds only part of a (sequence, head) leaves its maximum, sum and
// output in the workspace; the last one to arrive (a counter) joins them, in the order of the stretches.
#pragma once
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
  float scale_log2;
  int* counters;    // [row blocks][batch * kv_heads], zero between calls
  float* partials;  // [row blocks][CTAs][2][rows][head_dim + 2]
};

constexpr int kCacheWarps = 8;
constexpr int kCacheThreads = 32 * kCacheWarps;
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

__device__ __forceinline__ int seq_units(const CacheAttnParams& p, int b) {
  return max(1, (seq_tiles(p, seq_length(p, b)).count + kCacheWarps - 1) / kCacheWarps);
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
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(src));
        w[4 * v] = u.x;
        w[4 * v + 1] = u.y;
        w[4 * v + 2] = u.z;
        w[4 * v + 3] = u.w;
      } else if constexpr (kVec == 2) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(src));
        w[2 * v] = u.x;
        w[2 * v + 1] = u.y;
      } else {
        w[v] = __ldg(reinterpret_cast<const uint32_t*>(src));
      }
    }
  }
};

template <int HD, bool kFp8, int NT>
struct CacheAttnCfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kBytes = kFp8 ? 1 : 2;
  static constexpr int kKWords = HD * kBytes / 16;  // of one token, per thread: 4 threads share a row of K,
  static constexpr int kVWords = HD * kBytes / 32;  // 8 a row of V
  static constexpr int kSteps = HD / 16;
  static constexpr int kPartial = kRows * (HD + 2);  // floats of one partial result
  static constexpr int kMergeFloats = kCacheWarps * kPartial;
};

template <int HD, bool kFp8, int NT>
__global__ void __launch_bounds__(kCacheThreads, NT == 1 ? 2 : 1) cache_attention_kernel(const CacheAttnParams p) {
  using Cfg = CacheAttnCfg<HD, kFp8, NT>;
  using KPieces = RowPieces<Cfg::kKWords, 4>;
  using VPieces = RowPieces<Cfg::kVWords, 8>;
  constexpr int R = Cfg::kRows;
  extern __shared__ float s_dyn[];
  float* s_merge = s_dyn;                                            // [warps][R][HD + 2]
  int* s_first = reinterpret_cast<int*>(s_dyn + Cfg::kMergeFloats);  // [batch + 1] first unit of each sequence
  __shared__ int s_scan[kCacheWarps];
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int g = lane >> 2;
  const int t = lane & 3;
  const int kv_heads = p.c.kv_heads;
  const int rows_total = p.q_len * p.group;
  const int row_block = blockIdx.y * R;

  pdl_wait_previous_grid();
  pdl_allow_next_grid();

  // First unit of each sequence on the line of all units.
  int base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kCacheThreads) {
    const int b = b0 + tid;
    int v = b < p.batch ? seq_units(p, b) * kv_heads : 0;
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
    for (int i = 0; i < kCacheWarps; ++i) {
      if (i < warp) before += s_scan[i];
      all += s_scan[i];
    }
    if (b < p.batch) s_first[b + 1] = before + v;
    base += all;
    __syncthreads();
  }
  if (tid == 0) s_first[0] = 0;
  __syncthreads();
  const int64_t total = base;
  const int64_t ctas = min(static_cast<int64_t>(gridDim.x), total);
  const int64_t cta = blockIdx.x;
  if (cta >= ctas) return;
  const int w_begin = static_cast<int>(cta * total / ctas);
  const int w_end = static_cast<int>((cta + 1) * total / ctas);

  int b = 0;
  {
    int hi = p.batch;  // s_first[b] <= w_begin < s_first[hi]
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if (s_first[mid] <= w_begin) b = mid; else hi = mid;
    }
  }

  for (int w = w_begin; w < w_end;) {
    while (s_first[b + 1] <= w) ++b;
    const SeqTiles seq = seq_tiles(p, seq_length(p, b));
    const int units = (s_first[b + 1] - s_first[b]) / kv_heads;
    const int h = (w - s_first[b]) / units;
    const int head_begin = s_first[b] + h * units;  // of the line
    const int u0 = w - head_begin;
    const int u1 = min(units, w_end - head_begin);

    // Q: fragments of the 8-row operand(s), and the factor of its rows' scores.
    uint32_t qf[NT][Cfg::kSteps][2];
    float row_scale[NT][2];
    int limit[NT][2];  // position of the rows 2t, 2t + 1 of each operand, -1: no such row
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row_block + 8 * nt + g;
      const bool real = row < rows_total;
      const __nv_bfloat16* src =
          p.q + (static_cast<int64_t>(b) * p.q_len + (real ? row / p.group : 0)) * p.ld_q +
          (h * p.group + (real ? row % p.group : 0)) * HD;
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

    const uint8_t* k_head = p.c.k + h * p.c.head_stride * Cfg::kBytes;
    const uint8_t* v_head = p.c.v + h * p.c.head_stride * Cfg::kBytes;
    const int32_t* pages = p.page_table + b * p.ld_table;
    // Tokens that every row sees lie below `all_see`, and (with a window) from `all_from` on or below the sinks.
    const int all_see = seq.len - p.q_len + 1;
    const int all_from = p.window > 0 ? max(0, seq.len - p.window) : 0;

    for (int u = u0; u < u1; ++u) {
      const int i = u * kCacheWarps + warp;
      if (i >= seq.count) break;
      const int tok0 = 16 * (i < seq.sink_tiles ? i : i - seq.sink_tiles + seq.first_win);
      const int page = pages[tok0 >> p.c.page_shift];
      if (page < 0 || page >= p.c.pages) {
        record_status(kKernelCacheAttention, 2, kReasonBadIndex);
        continue;
      }
      const int slot0 = tok0 & ((1 << p.c.page_shift) - 1);
      const int64_t at = (page * p.c.page_stride + slot0 * HD) * Cfg::kBytes;
      uint32_t kr[2][Cfg::kKWords], vr[4][Cfg::kVWords];
#pragma unroll
      for (int x = 0; x < 2; ++x) KPieces::load(k_head + at + (g + 8 * x) * (HD * Cfg::kBytes), t, kr[x]);
#pragma unroll
      for (int x = 0; x < 4; ++x)
        VPieces::load(v_head + at + (2 * t + (x & 1) + 4 * (x & 2)) * (HD * Cfg::kBytes), g, vr[x]);
      float k_scale = 1.f, ev = 0.f, inv_v = 1.f;
      if (kFp8) {
        k_scale = __ldg(p.c.k_scale + static_cast<int64_t>(page) * kv_heads + h);
        const float vs = __ldg(p.c.v_scale + static_cast<int64_t>(page) * kv_heads + h);
        ev = static_cast<float>(static_cast<int>(__float_as_uint(vs) >> 23) - 127);
        inv_v = exp2_int(-static_cast<int>(ev));
      }

      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int st = 0; st < Cfg::kSteps; ++st) {
        uint32_t a0, a1, a2, a3;
        if constexpr (kFp8) {
          a0 = e4m3x2_to_f16x2(kr[0][st]);
          a1 = e4m3x2_to_f16x2(kr[1][st]);
          a2 = e4m3x2_to_f16x2(kr[0][st] >> 16);
          a3 = e4m3x2_to_f16x2(kr[1][st] >> 16);
        } else {
          a0 = kr[0][2 * st];
          a1 = kr[1][2 * st];
          a2 = kr[0][2 * st + 1];
          a3 = kr[1][2 * st + 1];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) cache_mma<kFp8>(s[nt], a0, a1, a2, a3, qf[nt][st][0], qf[nt][st][1]);
      }

      // Tokens g and g + 8 of rows 2t and 2t + 1, in exponents of 2 with V's scale in.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[nt][x] = fmaf(s[nt][x], row_scale[nt][x & 1] * k_scale, ev);
      const bool edge = tok0 + 16 > all_see || (tok0 < all_from && tok0 + 16 > p.sinks);
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = tok0 + g + 8 * (x >> 1);
            const int pos = limit[nt][x & 1];
            if (j > pos || (p.window > 0 && pos - j >= p.window && j >= p.sinks)) s[nt][x] = -INFINITY;
          }
        // Values of tokens that no row sees may be anything (0 times a NaN is a NaN).
        const int see = seq.len;
        const int from = max(0, seq.len - p.q_len - p.window + 1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int j = tok0 + 2 * t + (x & 1) + 4 * (x & 2);
          if (j >= see || (p.window > 0 && j < from && j >= p.sinks)) {
#pragma unroll
            for (int i2 = 0; i2 < Cfg::kVWords; ++i2) vr[x][i2] = 0u;
          }
        }
      }

      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) grew |= fmaxf(s[nt][x], s[nt][x + 2]) > m[nt][x] + kCacheRescale;
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = fmaxf(s[nt][x], s[nt][x + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            if (top > m[nt][x]) {
              const float alpha = fast_exp2(m[nt][x] - top);  // 0 the first time
              m[nt][x] = top;
              l[nt][x] *= alpha;
#pragma unroll
              for (int j = 0; j < Cfg::kSteps; ++j) {
                o[nt][j][x] *= alpha;
                o[nt][j][x + 2] *= alpha;
              }
            }
          }
      }

      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w4[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float ref = m[nt][x & 1] == -INFINITY ? 0.f : m[nt][x & 1];
          w4[x] = fast_exp2(s[nt][x] - ref + kCacheHeadroom);
        }
        l[nt][0] = fmaf(w4[0] + w4[2], inv_v, l[nt][0]);
        l[nt][1] = fmaf(w4[1] + w4[3], inv_v, l[nt][1]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          pf[nt][x] = movmatrix_trans(kFp8 ? pack_f16x2(w4[2 * x], w4[2 * x + 1])
                                           : pack_bf16x2(w4[2 * x], w4[2 * x + 1]));
      }

      if constexpr (kFp8) {
#pragma unroll
        for (int i2 = 0; i2 < Cfg::kVWords; ++i2) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362u : 0x5140u;
            const uint32_t lo = __byte_perm(vr[0][i2], vr[1][i2], sel);  // tokens 2t, 2t+1 of two dims
            const uint32_t hi = __byte_perm(vr[2][i2], vr[3][i2], sel);  // tokens 2t+8, 2t+9
            const uint32_t a0 = e4m3x2_to_f16x2(lo), a1 = e4m3x2_to_f16x2(lo >> 16);
            const uint32_t a2 = e4m3x2_to_f16x2(hi), a3 = e4m3x2_to_f16x2(hi >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              cache_mma<kFp8>(o[nt][2 * i2 + half], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
          }
        }
      } else {
#pragma unroll
        for (int i2 = 0; i2 < Cfg::kVWords; ++i2) {
          const uint32_t a0 = __byte_perm(vr[0][i2], vr[1][i2], 0x5410u);
          const uint32_t a1 = __byte_perm(vr[0][i2], vr[1][i2], 0x7632u);
          const uint32_t a2 = __byte_perm(vr[2][i2], vr[3][i2], 0x5410u);
          const uint32_t a3 = __byte_perm(vr[2][i2], vr[3][i2], 0x7632u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) cache_mma<kFp8>(o[nt][i2], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
        }
      }
    }

    // The warps' results into shared memory, [warp][row][dims, maximum, sum].
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 4);
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 8);
        l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 16);
        float* dst = s_merge + (warp * R + 8 * nt + 2 * t + x) * (HD + 2);
#pragma unroll
        for (int j = 0; j < Cfg::kSteps; ++j)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const int d = kFp8 ? VPieces::offset(j / 2, g) + 2 * (j & 1) + hi : VPieces::offset(j, g) / 2 + hi;
            dst[d] = o[nt][j][x + 2 * hi];
          }
        if (g == 0) {
          dst[HD] = m[nt][x];
          dst[HD + 1] = l[nt][x];
        }
      }
    __syncthreads();

    // Join `count` results of the rows, in order; into the output or a partial result.
    const int rows = min(R, rows_total - row_block);
    auto join = [&](const float* from, auto read, int64_t count, auto slot_of, float* partial) {
      for (int i = tid; i < rows * HD; i += kCacheThreads) {
        const int r = i / HD, d = i - r * HD;
        float top = -INFINITY;
        for (int64_t k = 0; k < count; ++k) top = fmaxf(top, read(from + slot_of(k) * Cfg::kPartial + r * (HD + 2) + HD));
        const float ref = top == -INFINITY ? 0.f : top;
        float acc = 0.f, sum = 0.f;
        for (int64_t k = 0; k < count; ++k) {
          const float* one = from + slot_of(k) * Cfg::kPartial + r * (HD + 2);
          const float f = fast_exp2(read(one + HD) - ref);
          acc = fmaf(read(one + d), f, acc);
          sum = fmaf(read(one + HD + 1), f, sum);
        }
        if (partial != nullptr) {
          partial[r * (HD + 2) + d] = acc;
          if (d == 0) {
            partial[r * (HD + 2) + HD] = top;
            partial[r * (HD + 2) + HD + 1] = sum;
          }
        } else {
          const int row = row_block + r;
          // sum is 0 only where nothing is visible; a NaN stays one.
          p.out[(static_cast<int64_t>(b) * p.q_len + row / p.group) * p.ld_out + (h * p.group + row % p.group) * HD + d] =
              __float2bfloat16_rn(sum == 0.f ? 0.f : acc / sum);
        }
      }
    };
    auto same = [](int64_t k) { return k; };
    auto shared = [](const float* x) { return *x; };
    auto other = [](const float* x) { return __ldcg(x); };  // another SM's: not from this one's L1
    if (u1 - u0 == units) {
      join(s_merge, shared, kCacheWarps, same, nullptr);
    } else {
      float* mine = p.partials + static_cast<int64_t>(blockIdx.y) * gridDim.x * 2 * Cfg::kPartial;
      const int64_t c_first = ((head_begin + 1) * ctas - 1) / total;
      const int64_t c_last = (static_cast<int64_t>(head_begin + units) * ctas - 1) / total;
      // Slot 0 of a CTA: the stretch's part of a head that began before it (or with it); slot 1: of one that begins inside.
      join(s_merge, shared, kCacheWarps, same,
           mine + (cta * 2 + (w_begin >= head_begin ? 0 : 1)) * Cfg::kPartial);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        int* counter = p.counters + static_cast<int64_t>(blockIdx.y) * p.batch * kv_heads + b * kv_heads + h;
        const int last = atomicAdd(counter, 1) == static_cast<int>(c_last - c_first);
        if (last) *counter = 0;
        s_last = last;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        auto slot = [&](int64_t k) {
          const int64_t c = c_first + k;
          return c * 2 + (c * total / ctas >= head_begin ? 0 : 1);
        };
        join(mine, other, c_last - c_first + 1, slot, nullptr);
      }
    }
    __syncthreads();
    w = head_begin + u1;
  }
}

// CTAs of a launch, and the bytes of its workspace.
static int cache_attention_ctas(int sm_count) { return 2 * sm_count; }

// Rows of a block: 8, or 16 where there are more than 8 rows (a block reads the keys and values anew).
static int64_t cache_attention_row_blocks(int64_t rows, int* nt) {
  *nt = rows <= 8 ? 1 : 2;
  return (rows + 8 * *nt - 1) / (8 * *nt);
}

static int64_t cache_attention_counter_bytes(int64_t batch, int64_t kv_heads, int64_t row_blocks) {
  return (batch * kv_heads * row_blocks * 4 + 255) / 256 * 256;
}

static int64_t cache_attention_partial_bytes(int64_t head_dim, int64_t rows, int sm_count) {
  int nt = 1;
  const int64_t blocks = cache_attention_row_blocks(rows, &nt);
  return (blocks * cache_attention_ctas(sm_count) * 2 * (8 * nt) * (head_dim + 2) * 4 + 255) / 256 * 256;
}

static int64_t cache_attention_workspace_bytes(int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t rows,
                                               int sm_count) {
  int nt = 1;
  return cache_attention_counter_bytes(batch, kv_heads, cache_attention_row_blocks(rows, &nt)) +
         cache_attention_partial_bytes(head_dim, rows, sm_count);
}

template <int HD, bool kFp8, int NT>
static cudaError_t launch_cache_attention_t(const CacheAttnParams& p, dim3 grid, cudaStream_t stream) {
  using Cfg = CacheAttnCfg<HD, kFp8, NT>;
  const size_t smem = Cfg::kMergeFloats * 4 + (static_cast<size_t>(p.batch) + 1) * 4;
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(cache_attention_kernel<HD, kFp8, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
  });
  if (e != cudaSuccess) return e;
  return launch_pdl(cache_attention_kernel<HD, kFp8, NT>, grid, dim3(kCacheThreads), smem, stream, p);
}

template <int HD>
static cudaError_t launch_cache_attention_hd(const CacheAttnParams& p, bool fp8, int nt, dim3 grid, cudaStream_t stream) {
  if (fp8)
    return nt == 1 ? launch_cache_attention_t<HD, true, 1>(p, grid, stream)
                   : launch_cache_attention_t<HD, true, 2>(p, grid, stream);
  return nt == 1 ? launch_cache_attention_t<HD, false, 1>(p, grid, stream)
                 : launch_cache_attention_t<HD, false, 2>(p, grid, stream);
}

// Counters from the start of the workspace, partial results up to its end: a workspace made for the largest batch and
// the most rows then serves smaller calls in turn, whose partial results never lie over a larger call's counters.
static cudaError_t launch_cache_attention(CacheAttnParams p, void* workspace, int64_t workspace_bytes, bool fp8,
                                          int sm_count, cudaStream_t stream) {
  int nt = 1;
  const int64_t rows = static_cast<int64_t>(p.q_len) * p.group;
  const int64_t blocks = cache_attention_row_blocks(rows, &nt);
  p.counters = static_cast<int*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + workspace_bytes / 256 * 256 -
                                        cache_attention_partial_bytes(p.c.head_dim, rows, sm_count));
  const dim3 grid(static_cast<unsigned>(cache_attention_ctas(sm_count)), static_cast<unsigned>(blocks));
  switch (p.c.head_dim) {
    case 32:
      return launch_cache_attention_hd<32>(p, fp8, nt, grid, stream);
    case 64:
      return launch_cache_attention_hd<64>(p, fp8, nt, grid, stream);
    case 128:
      return launch_cache_attention_hd<128>(p, fp8, nt, grid, stream);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace b2
