// Keys and values of new tokens into a paged cache, with the rotation of their positions applied on the
// way (the formulas of rotary.cuh), and the rotated queries written next to it. The reference computes
// every token's keys and values anew (models.py:51-75); it has no cache.
//
// A page holds page_size consecutive tokens of one sequence for every key head,
// [kv_heads][page_size][head_dim], as bf16 or as e4m3 codes with one scale per page and head. The scale
// is a power of two, 2^e: dividing by it is exact, so a code's only rounding is that to 3 mantissa bits
// (which does not depend on e), and raising a page's e later re-rounds only what falls below e4m3's normal
// range. e is the least with max|x| <= 448 * 2^e over the page's finite new values, within [-40, 40],
// and at least the e the page had if it holds earlier tokens of its sequence; those tokens' codes are
// then multiplied by 2^(e_old - e). The bounds on e keep the attention's sums of 2^e-weighted terms
// inside fp32; magnitudes above 448 * 2^40 saturate, and values that are not finite become the NaN code.
//
// Bound by HBM (the projection's rows in, codes or bf16 and rotated queries out), and nearly as much by the number of
// instructions per element, so each is kept short: a thread holds up to two chunks of 16 elements, whose place in the
// page is worked out once. A team of 1 to 16 warps, as many as hold the page's new tokens, takes one head of K or of
// V (in 8 bits the page's maximum is then known before the first code is written, without reading twice; pages with
// more than 1024 chunks are read twice), or the query heads of one key head, whose rows of the table stay in registers.
// Measured on one B200 (us a call, floor in brackets): ragged prompts of 16 sequences of up to 2048 tokens, 16 heads of
// 64, 8-bit pages of 32: 71 (43; 94 with a CTA of 128 threads per head that read its rows twice); 32768 tokens of 16
// query and 4 key heads of 128: 82 (64; 92); bf16 chunks of three documents 30 (20); one token in each of 64 sequences
// 3.9, a launch. Issue slots are 55 % busy and the L1 data pipe (the table, 64 bytes a thread) 54 %: more warps do not
// fit their registers, and going through several heads with the table in registers cost more instructions than it saved.
#pragma once
#include <cuda_fp16.h>

#include "b2_common.cuh"
#include "rotary.cuh"

namespace b2 {

constexpr int kScaleExpMin = -40;
constexpr int kScaleExpMax = 40;
constexpr float kE4m3Max = 448.f;

struct CachePages {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;  // [pages][kv_heads]
  float* v_scale;
  int64_t pages, page_stride, head_stride;  // strides in elements
  int kv_heads, head_dim, page_shift;
};

struct AppendParams {
  CachePages c;
  const __nv_bfloat16* qkv;
  int64_t ld, tokens;
  int q_col, k_col, v_col;
  int batch, group;  // query heads per key head
  int64_t max_new;
  const int32_t* new_start;
  const int32_t* new_len;
  const int32_t* past_len;
  const int32_t* page_table;
  int64_t ld_table;
  int table_pages;
  int rotary_dim;  // 0: none
  const float2* table;
  int64_t max_positions;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_out;
  int64_t ld_q_out, ld_k_out;
};

// Least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), from amax's exponent and mantissa fields.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleExpMin), kScaleExpMax);
}

__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// 8 values as codes of the scale whose inverse is `inv`; a NaN becomes the NaN code, and with `check` an infinity
// does too (it would saturate).
__device__ __forceinline__ uint2 e4m3x8(const float (&f)[8], float inv, bool check) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = f[4 * i + k] * inv;
    if (check) {
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = is_finite(f[4 * i + k]) ? y[k] : __uint_as_float(0x7fffffffu);
    }
    w[i] = static_cast<uint32_t>(e4m3x2(y[0], y[1])) | (static_cast<uint32_t>(e4m3x2(y[2], y[3])) << 16);
  }
  return make_uint2(w[0], w[1]);
}

// 4 codes times `f` (a power of two), rounded again.
__device__ __forceinline__ uint32_t e4m3x4_scale(uint32_t w, float f) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(w >> (16 * i))));
    const __half2 h2 = *reinterpret_cast<__half2*>(&h);
    out |= static_cast<uint32_t>(e4m3x2(__low2float(h2) * f, __high2float(h2) * f)) << (16 * i);
  }
  return out;
}

constexpr int kAppendMaxThreads = 512;
constexpr int kAppendItems = 2;  // chunks that a thread holds

template <bool kFp8, bool kInterleaved>
__global__ void __launch_bounds__(kAppendMaxThreads, 2)
    cache_append_kernel(const AppendParams p, const int team_shift, const unsigned role_blocks) {
  __shared__ float s_red[kAppendMaxThreads / 32];
  const unsigned block_page = blockIdx.x / role_blocks;
  const unsigned team_threads = 32u << team_shift;
  const unsigned tt = threadIdx.x & (team_threads - 1);
  const unsigned team = threadIdx.x >> (5 + team_shift);
  const int kv_heads = p.c.kv_heads;
  const int role = static_cast<int>((blockIdx.x - block_page * role_blocks) * (blockDim.x >> (5 + team_shift)) + team);
  if (role >= kv_heads * (p.rotary_dim > 0 ? 3 : 2)) return;  // the whole team: its barrier is its own
  pdl_wait_previous_grid();
  pdl_allow_next_grid();
  const int b = blockIdx.z;
  const int past = p.past_len[b];
  const int count = p.new_len[b];
  const int first = p.new_start[b];
  if (count <= 0) return;
  const int shift = p.c.page_shift;
  // Every index comes from device memory: one that does not fit is recorded and nothing is written.
  if (past < 0 || first < 0 || count > p.max_new || static_cast<int64_t>(first) + count > p.tokens ||
      static_cast<int64_t>(past) + count > (static_cast<int64_t>(p.table_pages) << shift) ||
      (p.rotary_dim > 0 && static_cast<int64_t>(past) + count > p.max_positions)) {
    record_status(kKernelCacheAppend, 1, kReasonBadIndex);
    return;
  }
  const int page_index = (past >> shift) + static_cast<int>(block_page);
  const int page0 = page_index << shift;  // first position of the page
  const int t0 = max(past, page0);
  const int t1 = min(past + count, page0 + (1 << shift));
  if (t0 >= t1) return;
  const int held = t0 - page0;  // earlier tokens of the sequence in this page
  const int hd = p.c.head_dim;
  const unsigned chunks = static_cast<unsigned>(hd) >> 4;
  const unsigned items = (t1 - t0) * chunks;
  const int64_t row0 = static_cast<int64_t>(first) + (t0 - past);
  const int ld = static_cast<int>(p.ld);
  const bool is_v = role >= kv_heads && role < 2 * kv_heads;
  const int rotary_dim = is_v ? 0 : p.rotary_dim;
  auto angles_of = [&](unsigned token, int pair0, float (&c)[8], float (&s)[8]) {
    rotary_load_table(p.table + static_cast<int64_t>(t0 + static_cast<int>(token)) * (rotary_dim >> 1) + pair0, c, s);
  };

  if (role >= 2 * kv_heads) {
    // The query heads of one key head.
    const int h0 = (role - 2 * kv_heads) * p.group;
    const __nv_bfloat16* rows = p.qkv + row0 * p.ld + p.q_col + h0 * hd;
    __nv_bfloat16* out = p.q_out + row0 * p.ld_q_out + h0 * hd;
    for (unsigned i = tt; i < items; i += team_threads) {
      const unsigned token = i / chunks;
      const RotaryChunk ch = rotary_chunk<kInterleaved>(i - token * chunks, rotary_dim);
      float c[8], s[8];
      if (ch.pair0 >= 0) angles_of(token, ch.pair0, c, s);
      const __nv_bfloat16* x = rows + token * static_cast<int64_t>(ld);
      __nv_bfloat16* y = out + token * p.ld_q_out;
#pragma unroll 2
      for (int g = 0; g < p.group; ++g, x += hd, y += hd) {
        uint4 ua = *reinterpret_cast<const uint4*>(x + ch.off0);
        uint4 ub = *reinterpret_cast<const uint4*>(x + ch.off1);
        if (ch.pair0 >= 0) {
          float a[8], bb[8];
          unpack_bf16x8(ua, a);
          unpack_bf16x8(ub, bb);
          rotary_apply<kInterleaved>(a, bb, c, s);
          ua = pack_bf16x8(a);
          ub = pack_bf16x8(bb);
        }
        *reinterpret_cast<uint4*>(y + ch.off0) = ua;
        *reinterpret_cast<uint4*>(y + ch.off1) = ub;
      }
    }
    return;
  }

  const int h = is_v ? role - kv_heads : role;
  // Looked at once the rows' loads are on their way; a page that does not exist is not written.
  int64_t page = p.page_table[b * p.ld_table + page_index];
  const __nv_bfloat16* rows = p.qkv + row0 * p.ld + (is_v ? p.v_col : p.k_col) + h * hd;
  // The page, and where K goes besides.
  uint8_t* dst = nullptr;
  float* scale = nullptr;
  auto find_page = [&]() {
    if (page < 0 || page >= p.c.pages) {
      record_status(kKernelCacheAppend, 2, kReasonBadIndex);
      return false;
    }
    dst = (is_v ? p.c.v : p.c.k) + (page * p.c.page_stride + h * p.c.head_stride) * (kFp8 ? 1 : 2);
    if (kFp8) scale = (is_v ? p.c.v_scale : p.c.k_scale) + page * kv_heads + h;
    return true;
  };
  __nv_bfloat16* copy = !is_v && p.k_out != nullptr ? p.k_out + row0 * p.ld_k_out + h * hd : nullptr;
  auto team_sync = [&]() {
    if (team_shift > 0)
      named_barrier_sync(1 + team, team_threads);
    else
      __syncwarp();
  };
  auto load = [&](unsigned token, const RotaryChunk& ch, float (&a)[8], float (&bb)[8]) {
    const __nv_bfloat16* x = rows + token * static_cast<int64_t>(ld);
    const uint4 ua = *reinterpret_cast<const uint4*>(x + ch.off0);
    const uint4 ub = *reinterpret_cast<const uint4*>(x + ch.off1);
    if (ch.pair0 >= 0) {
      float c[8], s[8];
      angles_of(token, ch.pair0, c, s);
      unpack_bf16x8(ua, a);
      unpack_bf16x8(ub, bb);
      rotary_apply<kInterleaved>(a, bb, c, s);
    } else {
      unpack_bf16x8(ua, a);
      unpack_bf16x8(ub, bb);
    }
  };
  auto write = [&](unsigned token, const RotaryChunk& ch, const float (&a)[8], const float (&bb)[8], float inv, bool check) {
    uint8_t* at = dst + (held + static_cast<int>(token)) * hd * (kFp8 ? 1 : 2);
    if (kFp8) {
      *reinterpret_cast<uint2*>(at + ch.off0) = e4m3x8(a, inv, check);
      *reinterpret_cast<uint2*>(at + ch.off1) = e4m3x8(bb, inv, check);
    } else {
      *reinterpret_cast<uint4*>(at + 2 * ch.off0) = pack_bf16x8(a);
      *reinterpret_cast<uint4*>(at + 2 * ch.off1) = pack_bf16x8(bb);
    }
    if (copy != nullptr) {
      __nv_bfloat16* y = copy + token * p.ld_k_out;
      *reinterpret_cast<uint4*>(y + ch.off0) = pack_bf16x8(a);
      *reinterpret_cast<uint4*>(y + ch.off1) = pack_bf16x8(bb);
    }
  };
  // Largest magnitude (infinity if there is one; a NaN is passed over), and with `check` that of the finite values.
  auto largest = [&](float amax, const float (&a)[8], const float (&bb)[8], bool check) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (check)
        amax = fmaxf(amax, fmaxf(is_finite(a[k]) ? fabsf(a[k]) : 0.f, is_finite(bb[k]) ? fabsf(bb[k]) : 0.f));
      else
        amax = max3f(amax, fabsf(a[k]), fabsf(bb[k]));
    }
    return amax;
  };
  auto team_max = [&](float amax) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (team_shift > 0) {
      if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = amax;
      team_sync();
      const int warp0 = static_cast<int>(team) << team_shift;
      for (int i = 0; i < (1 << team_shift); ++i) amax = fmaxf(amax, s_red[warp0 + i]);
    }
    return amax;
  };
  // The page's scale from the team's largest value; earlier codes are rounded again if it grew. Returns its inverse.
  auto settle_scale = [&](float amax) {
    int e = scale_exponent(amax);
    if (held > 0) {
      const int e_old = min(static_cast<int>((__float_as_uint(*scale) >> 23) & 0xffu) - 127, kScaleExpMax);
      if (e > e_old) {
        const float f = exp2_int(max(e_old - e, -126));
        uint32_t* w = reinterpret_cast<uint32_t*>(dst);
        for (int i = tt; i < held * hd / 4; i += team_threads) w[i] = e4m3x4_scale(w[i], f);
      } else {
        e = e_old;
      }
      team_sync();  // every thread of the team has read the old scale
    }
    if (tt == 0) *scale = exp2_int(e);
    return exp2_int(-e);
  };

  if (items <= kAppendItems * team_threads) {
    float a[kAppendItems][8], bb[kAppendItems][8];
    RotaryChunk ch[kAppendItems];
    unsigned token[kAppendItems];
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < kAppendItems; ++k) {
      const unsigned i = tt + k * team_threads;
      token[k] = i / chunks;
      ch[k] = rotary_chunk<kInterleaved>(i - token[k] * chunks, rotary_dim);
      if (i < items) load(token[k], ch[k], a[k], bb[k]);
    }
    if (!find_page()) return;  // the whole team
    float inv = 1.f;
    bool check = false;
    if (kFp8) {
#pragma unroll
      for (int k = 0; k < kAppendItems; ++k)
        if (tt + k * team_threads < items) amax = largest(amax, a[k], bb[k], false);
      amax = team_max(amax);
      if (!is_finite(amax)) {  // an infinity among them: the scale goes by the finite values
        check = true;
        amax = 0.f;
#pragma unroll
        for (int k = 0; k < kAppendItems; ++k)
          if (tt + k * team_threads < items) amax = largest(amax, a[k], bb[k], true);
        team_sync();  // the first maxima have been read
        amax = team_max(amax);
      }
      inv = settle_scale(amax);
    }
#pragma unroll
    for (int k = 0; k < kAppendItems; ++k)
      if (tt + k * team_threads < items) write(token[k], ch[k], a[k], bb[k], inv, check);
  } else {
    if (!find_page()) return;
    auto each = [&](auto f) {
      for (unsigned i = tt; i < items; i += team_threads) {
        const unsigned token = i / chunks;
        const RotaryChunk ch = rotary_chunk<kInterleaved>(i - token * chunks, rotary_dim);
        float a[8], bb[8];
        load(token, ch, a, bb);
        f(token, ch, a, bb);
      }
    };
    float inv = 1.f;
    if (kFp8) {
      float amax = 0.f;
      each([&](unsigned, const RotaryChunk&, const float(&a)[8], const float(&bb)[8]) { amax = largest(amax, a, bb, true); });
      inv = settle_scale(team_max(amax));  // between reading and writing: k_out may be the projection's own columns
    }
    each([&](unsigned token, const RotaryChunk& ch, const float(&a)[8], const float(&bb)[8]) {
      write(token, ch, a, bb, inv, true);
    });
  }
}

static cudaError_t launch_cache_append(const AppendParams& p, int64_t max_new, bool fp8, int interleaved,
                                       cudaStream_t stream) {
  // max_new tokens touch at most this many pages, wherever in a page they begin. 256 threads a CTA (ragged prompts as
  // above: 71 us, 78 with 512, 106 with 128), 512 where one team needs them.
  const int64_t page_size = int64_t{1} << p.c.page_shift;
  const int64_t pages = (max_new + page_size - 2) / page_size + 1;
  const int64_t chunks = (max_new < page_size ? max_new : page_size) * (p.c.head_dim / 16);
  int team_shift = 0;
  while (team_shift < 4 && chunks > (int64_t{32 * kAppendItems} << team_shift)) ++team_shift;
  const int threads = team_shift == 4 ? kAppendMaxThreads : 256;
  const int64_t roles = static_cast<int64_t>(p.c.kv_heads) * (p.rotary_dim > 0 ? 3 : 2);
  const int64_t teams = (threads / 32) >> team_shift;
  const int64_t role_blocks = (roles + teams - 1) / teams;
  if (role_blocks * pages > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(role_blocks * pages), 1, static_cast<unsigned>(p.batch));
  const unsigned rb = static_cast<unsigned>(role_blocks);
  if (fp8)
    return interleaved ? launch_pdl(cache_append_kernel<true, true>, grid, dim3(threads), 0, stream, p, team_shift, rb)
                       : launch_pdl(cache_append_kernel<true, false>, grid, dim3(threads), 0, stream, p, team_shift, rb);
  return interleaved ? launch_pdl(cache_append_kernel<false, true>, grid, dim3(threads), 0, stream, p, team_shift, rb)
                     : launch_pdl(cache_append_kernel<false, false>, grid, dim3(threads), 0, stream, p, team_shift, rb);
}

}  // namespace b2
