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
// One CTA takes one page of one sequence and one head of K, of V, or (with a rotation) the query heads
// of one key head for the page's tokens. Two passes over the new tokens of K and V in 8 bits: the page's
// maximum has to be known before the first code is written.
#pragma once
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

// 8 values as codes of the scale whose inverse is `inv`; a value that is not finite becomes NaN.
__device__ __forceinline__ uint2 e4m3x8(const float (&f)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = f[4 * i + k];
      y[k] = is_finite(x) ? x * inv : __uint_as_float(0x7fffffffu);
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

constexpr int kAppendThreads = 128;

__device__ __forceinline__ float append_block_max(float v, float* s_red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
  __syncthreads();
  float m = s_red[0];
#pragma unroll
  for (int i = 1; i < kAppendThreads / 32; ++i) m = fmaxf(m, s_red[i]);
  return m;
}

template <bool kFp8, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads) cache_append_kernel(const AppendParams p) {
  __shared__ float s_red[kAppendThreads / 32];
  pdl_wait_previous_grid();
  pdl_allow_next_grid();
  const int b = blockIdx.z;
  const int past = p.past_len[b];
  const int count = p.new_len[b];
  if (count <= 0) return;
  const int shift = p.c.page_shift;
  const int page_size = 1 << shift;
  const int first = p.new_start[b];
  // Every index comes from device memory: one that does not fit is recorded and nothing is written.
  if (past < 0 || first < 0 || count > p.max_new || static_cast<int64_t>(first) + count > p.tokens ||
      static_cast<int64_t>(past) + count > (static_cast<int64_t>(p.table_pages) << shift) ||
      (p.rotary_dim > 0 && static_cast<int64_t>(past) + count > p.max_positions)) {
    record_status(kKernelCacheAppend, 1, kReasonBadIndex);
    return;
  }
  const int page_index = (past >> shift) + static_cast<int>(blockIdx.x);
  const int page0 = page_index << shift;  // first position of the page
  const int t0 = max(past, page0);
  const int t1 = min(past + count, page0 + page_size);
  if (t0 >= t1) return;
  const int n = t1 - t0;
  const int64_t row0 = static_cast<int64_t>(first) + (t0 - past);
  const unsigned chunks = static_cast<unsigned>(p.c.head_dim) >> 4;
  const unsigned items = n * chunks;
  const int kv_heads = p.c.kv_heads;
  const int role = blockIdx.y;

  auto load_table = [&](int token, int pair0, float (&c)[8], float (&s)[8]) {
    rotary_load_table(p.table + static_cast<int64_t>(t0 + token) * (p.rotary_dim >> 1) + pair0, c, s);
  };

  if (role >= 2 * kv_heads) {
    // Query heads of one key head.
    const int h0 = (role - 2 * kv_heads) * p.group;
    for (unsigned i = threadIdx.x; i < items; i += kAppendThreads) {
      const unsigned token = i / chunks;
      const RotaryChunk ch = rotary_chunk<kInterleaved>(i - token * chunks, p.rotary_dim);
      float c[8], s[8];
      if (ch.pair0 >= 0) load_table(token, ch.pair0, c, s);
      const __nv_bfloat16* x = p.qkv + (row0 + token) * p.ld + p.q_col + h0 * p.c.head_dim;
      __nv_bfloat16* y = p.q_out + (row0 + token) * p.ld_q_out + h0 * p.c.head_dim;
      for (int g = 0; g < p.group; ++g, x += p.c.head_dim, y += p.c.head_dim) {
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

  const bool is_v = role >= kv_heads;
  const int h = is_v ? role - kv_heads : role;
  const int64_t page = p.page_table[b * p.ld_table + page_index];
  if (page < 0 || page >= p.c.pages) {
    record_status(kKernelCacheAppend, 2, kReasonBadIndex);
    return;
  }
  const int rotary_dim = is_v ? 0 : p.rotary_dim;
  const __nv_bfloat16* src = p.qkv + row0 * p.ld + (is_v ? p.v_col : p.k_col) + h * p.c.head_dim;
  uint8_t* dst = (is_v ? p.c.v : p.c.k) + (page * p.c.page_stride + h * p.c.head_stride) * (kFp8 ? 1 : 2);

  auto load = [&](unsigned i, unsigned& token, RotaryChunk& ch, float (&a)[8], float (&bb)[8]) {
    token = i / chunks;
    ch = rotary_chunk<kInterleaved>(i - token * chunks, rotary_dim);
    const __nv_bfloat16* x = src + token * p.ld;
    unpack_bf16x8(*reinterpret_cast<const uint4*>(x + ch.off0), a);
    unpack_bf16x8(*reinterpret_cast<const uint4*>(x + ch.off1), bb);
    if (ch.pair0 >= 0) {
      float c[8], s[8];
      load_table(token, ch.pair0, c, s);
      rotary_apply<kInterleaved>(a, bb, c, s);
    }
  };

  float inv = 1.f;
  if (kFp8) {
    float amax = 0.f;
    for (unsigned i = threadIdx.x; i < items; i += kAppendThreads) {
      unsigned token;
      RotaryChunk ch;
      float a[8], bb[8];
      load(i, token, ch, a, bb);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (is_finite(a[k])) amax = fmaxf(amax, fabsf(a[k]));
        if (is_finite(bb[k])) amax = fmaxf(amax, fabsf(bb[k]));
      }
    }
    int e = scale_exponent(append_block_max(amax, s_red));
    float* scale = (is_v ? p.c.v_scale : p.c.k_scale) + page * kv_heads + h;
    const int held = t0 - page0;  // earlier tokens of the sequence in this page
    if (held > 0) {
      const float old = *scale;
      const int e_old = min(static_cast<int>((__float_as_uint(old) >> 23) & 0xffu) - 127, kScaleExpMax);
      if (e > e_old) {
        const float f = exp2_int(max(e_old - e, -126));
        uint32_t* w = reinterpret_cast<uint32_t*>(dst);
        for (int i = threadIdx.x; i < held * p.c.head_dim / 4; i += kAppendThreads) w[i] = e4m3x4_scale(w[i], f);
      } else {
        e = e_old;
      }
    }
    __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) *scale = exp2_int(e);
    inv = exp2_int(-e);
  }
  for (unsigned i = threadIdx.x; i < items; i += kAppendThreads) {
    unsigned token;
    RotaryChunk ch;
    float a[8], bb[8];
    load(i, token, ch, a, bb);
    const int64_t at = static_cast<int64_t>(t0 - page0 + token) * p.c.head_dim;
    if (kFp8) {
      *reinterpret_cast<uint2*>(dst + at + ch.off0) = e4m3x8(a, inv);
      *reinterpret_cast<uint2*>(dst + at + ch.off1) = e4m3x8(bb, inv);
    } else {
      *reinterpret_cast<uint4*>(dst + 2 * (at + ch.off0)) = pack_bf16x8(a);
      *reinterpret_cast<uint4*>(dst + 2 * (at + ch.off1)) = pack_bf16x8(bb);
    }
    if (!is_v && p.k_out != nullptr) {
      __nv_bfloat16* y = p.k_out + (row0 + token) * p.ld_k_out + h * p.c.head_dim;
      *reinterpret_cast<uint4*>(y + ch.off0) = pack_bf16x8(a);
      *reinterpret_cast<uint4*>(y + ch.off1) = pack_bf16x8(bb);
    }
  }
}

static cudaError_t launch_cache_append(const AppendParams& p, int64_t max_new, bool fp8, int interleaved,
                                       cudaStream_t stream) {
  // max_new tokens touch at most this many pages, wherever in a page they begin.
  const int64_t page_size = int64_t{1} << p.c.page_shift;
  const unsigned pages = static_cast<unsigned>((max_new + page_size - 2) / page_size + 1);
  const unsigned roles = static_cast<unsigned>(p.c.kv_heads * (p.rotary_dim > 0 ? 3 : 2));
  const dim3 grid(pages, roles, static_cast<unsigned>(p.batch));
  const dim3 block(kAppendThreads);
  if (fp8)
    return interleaved ? launch_pdl(cache_append_kernel<true, true>, grid, block, 0, stream, p)
                       : launch_pdl(cache_append_kernel<true, false>, grid, block, 0, stream, p);
  return interleaved ? launch_pdl(cache_append_kernel<false, true>, grid, block, 0, stream, p)
                     : launch_pdl(cache_append_kernel<false, false>, grid, block, 0, stream, p);
}

}  // namespace b2
