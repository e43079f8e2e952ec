// Keys and values of new tokens into a paged cache of 4-bit codes, with the rotation of their positions applied on the way,
// and a cache's tokens, of any type, back as bf16 rows. The reference has no cache (models.py:51-75 computes keys and values
// anew for every token).
//
// 32 neighbouring elements of a head of one token are a group with a step and a middle, both bf16; code c of 0 ... 15 stands
// for mid + (c - 8) step. Of the group's values
//   step = bf16((most - least) / 15), 0 where that is below 2^-100;  mid = bf16(least + 8 step);  r = bf16(1 / step)
//   c = clamp(nearest even of (x - mid) r, -8, 7) + 8
// with each operation rounded to fp32 by itself. A token is quantised by itself, so that what a page held before never
// changes and a code does not depend on the order in which tokens came. bf16 holds a step and a middle to 2^-9 of
// themselves: the codes are made for the rounded ones, so that a step's rounding costs a value at most 8 * 2^-9 of a step, and the
// middle's is no more than what a bf16 value of its size loses. r has 8 bits too: with x and mid in bf16 the product is then
// exact, and a value halfway between two codes goes to the even one in whatever form the formula is computed. A group with a
// value that is not finite, or whose range is not, has NaN for its step and middle: all 32 read as NaN.
//
// A token's row is head_dim / 2 bytes: for g = 0 ... 7 and each group, two bytes with the codes of elements 4 g ... 4 g + 3
// of the group, the first in the lowest bits. That is how the attention's threads want them (cache_attention.cuh): a
// quarter of a row of K, or an eighth of a row of V, of all groups, is one load. Its parameters are [2][groups] bf16, steps then
// middles.
//
// Both kernels are bound by HBM, the append by the projection's rows in and the rotated queries out, and nearly as much by
// their instructions. A warp takes a tile of tokens of one head (of K, of V, or the query heads of one key head), four lanes
// to a token: a lane holds 8 elements of every group, so that two exchanges find a group's least and most value, the codes
// and parameters are whole vectors of a lane's own, and where the whole head is turned in halves a pair's elements lie in one
// lane. (A lane to 8 elements, with exchanges to put words together: prompts' append 138 us, 458 to read 4 x 65536 tokens.)
// Measured on one B200 (us a call, floor at the measured copy rate in brackets): append of ragged prompts of 16 sequences of up to
// 2048 tokens, 16 heads of 64, rotated queries and keys kept: 69 (40); chunks of three documents, 16 query and 4 key heads of
// 128, a quarter turned: 18 (8); one token in each of 64 sequences 4, a launch. Reading 4 x 65536 tokens of 8 heads of 128 in 4
// bits: 221 (218); 16 sequences of up to 4096 tokens of 16 heads of 64 in 8 bits: 50 (43). The append's issue slots are 57 %
// busy (20 instructions an element for ranges and codes), its warps wait for their rows the rest of the time.
#pragma once
#include "b2_common.cuh"
#include "cache_append.cuh"
#include "cache_attention.cuh"
#include "rotary.cuh"

namespace b2 {

constexpr int kInt4Group = 32;
constexpr float kInt4LeastStep = 7.888609052210118e-31f;  // 2^-100
constexpr int kInt4Threads = 256;
constexpr int kInt4Tile = 32;  // tokens of a warp, at most

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint32_t bf16x2_less_136(uint32_t a) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), __float2bfloat162_rn(136.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bf16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b),
                                   *reinterpret_cast<__nv_bfloat162*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// x / 15, rounded to nearest: the quotient by the rounded 1 / 15, and what it leaves, once more. Equal to the division for
// every x whose remainder does not fall below fp32's normal range (checked over all mantissas; test_more_serving_host.py).
__device__ __forceinline__ float divide_by_15(float x) {
  constexpr float k = 1.f / 15.f;
  const float q = x * k;
  return fmaf(fmaf(-q, 15.f, x), k, q);
}

// 8 values of a group, whose other 24 are in the lanes that differ in bits 0 and 1, as codes in 4 bits each; `params`: the
// group's step and middle as bf16 bits, the step in the lower half.
__device__ __forceinline__ uint32_t int4_codes(const float (&x)[8], uint32_t& params) {
  float lo = min3_nan(min3_nan(x[0], x[1], x[2]), x[3], x[4]);
  float hi = max3_nan(max3_nan(x[0], x[1], x[2]), x[3], x[4]);
  lo = min_nan(min3_nan(x[5], x[6], x[7]), lo);
  hi = max_nan(max3_nan(x[5], x[6], x[7]), hi);
  lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
  hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
  lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, 2));
  hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, 2));
  const float range = __fsub_rn(hi, lo);  // not finite where a value is not
  float step = bf16_round(divide_by_15(range));
  if (step < kInt4LeastStep) step = 0.f;
  float mid = bf16_round(__fadd_rn(lo, 8.f * step));
  if (!is_finite(range)) step = mid = __uint_as_float(0x7fc00000u);
  // (1 / step is never within 2^-17 of the middle between two bf16 values, so that an approximate one rounds alike)
  const float r = step > 0.f ? bf16_round(fast_rcp(step)) : 0.f;
  params = pack_bf16x2(step, mid);
  // Adding 1.5 * 2^23 rounds to a whole number (to the even one at a half), 8 more makes it the code in the lowest bits; the
  // words' sum in 16ths, less the constant's, has the codes side by side.
  constexpr float kMagic = 12582912.f + 8.f;
  constexpr uint32_t kOver = 0x4b400000u;
  uint32_t w = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    const float t = fmaxf(fminf(__fmul_rn(__fsub_rn(x[i], mid), r), 7.f), -8.f);
    w = w * 16u + (__float_as_uint(__fadd_rn(t, kMagic)) - kOver);
  }
  return w;
}

// G words of a lane's own, 4 G bytes apart from its neighbours'. Loads are coherent: see load_once4.
template <int G>
__device__ __forceinline__ void load_words(const void* from, uint32_t (&w)[G]) {
  const uint8_t* p = static_cast<const uint8_t*>(from);
#pragma unroll
  for (int i = 0; i < G;) {
    if constexpr (G % 4 == 0) {
      const uint4 u = load_once4(p + 4 * i);
      w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
      i += 4;
    } else if constexpr (G % 2 == 0) {
      const uint2 u = load_once2(p + 4 * i);
      w[i] = u.x, w[i + 1] = u.y;
      i += 2;
    } else {
      w[i] = load_once(p + 4 * i);
      ++i;
    }
  }
}
template <int G>
__device__ __forceinline__ void store_words(void* to, const uint32_t (&w)[G]) {
  uint8_t* p = static_cast<uint8_t*>(to);
#pragma unroll
  for (int i = 0; i < G;) {
    if constexpr (G % 4 == 0) {
      *reinterpret_cast<uint4*>(p + 4 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      i += 4;
    } else if constexpr (G % 2 == 0) {
      *reinterpret_cast<uint2*>(p + 4 * i) = make_uint2(w[i], w[i + 1]);
      i += 2;
    } else {
      *reinterpret_cast<uint32_t*>(p + 4 * i) = w[i];
      ++i;
    }
  }
}

// The lower halves of all groups' words, then the upper ones (a lane's codes, or a token's parameters, as they are stored),
// and back.
template <int G>
__device__ __forceinline__ void halves_apart(const uint32_t (&x)[G], uint32_t (&w)[G]) {
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int a = 2 * i, b = 2 * i + 1;
    w[i] = __byte_perm(a < G ? x[a] : x[a - G], b < G ? x[b] : x[b - G], (a < G ? 0x10u : 0x32u) | (b < G ? 0x5400u : 0x7600u));
  }
}
template <int G>
__device__ __forceinline__ uint32_t halves_together(const uint32_t (&w)[G], int y) {
  return __byte_perm(w[y / 2], w[(G + y) / 2], (y % 2 ? 0x32u : 0x10u) | ((G + y) % 2 ? 0x7600u : 0x5400u));
}

// (64 registers, four CTAs an SM, up to 4 groups: ragged prompts of 16 heads of 64 69 us, 78 with three.)
template <int G, bool kInterleaved>
__global__ void __launch_bounds__(kInt4Threads, G <= 4 ? 4 : 2) cache_append_int4_kernel(const AppendParams p, const int tile_tokens,
                                                                         const unsigned role_blocks) {
  const unsigned tile = blockIdx.x / role_blocks;
  const unsigned lane = threadIdx.x & 31;
  const int kv_heads = p.c.kv_heads;
  const int role = static_cast<int>((blockIdx.x - tile * role_blocks) * (kInt4Threads / 32) + (threadIdx.x >> 5));
  if (role >= kv_heads * (p.rotary_dim > 0 ? 3 : 2)) return;  // the whole warp
  pdl_wait_previous_grid();
  pdl_allow_next_grid();
  const int b = blockIdx.z;
  const int past = p.past_len[b];
  const int count = p.new_len[b];
  const int first = p.new_start[b];
  if (count <= 0) return;
  const int shift = p.c.page_shift;
  if (append_bad_index(p, past, count, first)) {
    record_status(kKernelCacheAppend, 1, kReasonBadIndex);
    return;
  }
  if (static_cast<int64_t>(tile) * tile_tokens >= count) return;
  const int from = static_cast<int>(tile) * tile_tokens;  // of the sequence's new tokens
  const int tokens = min(tile_tokens, count - from);
  const int64_t row0 = static_cast<int64_t>(first) + from;
  const int pos0 = past + from;
  constexpr int hd = 32 * G;
  if (role >= 2 * kv_heads) {
    append_queries<kInterleaved>(p, role - 2 * kv_heads, row0, pos0, static_cast<unsigned>(tokens), lane, 32u);
    return;
  }
  const bool is_v = role >= kv_heads;
  const int h = is_v ? role - kv_heads : role;
  const int t = static_cast<int>(lane) & 3;
  const int half = (is_v ? 0 : p.rotary_dim) >> 1;
  const bool whole = G % 2 == 0 && !kInterleaved && half == hd / 2;  // pairs lie in one lane
  const __nv_bfloat16* x = p.qkv + row0 * p.ld + (is_v ? p.v_col : p.k_col) + h * hd + 8 * t;
  __nv_bfloat16* copy = !is_v && p.k_out != nullptr ? p.k_out + row0 * p.ld_k_out + h * hd + 8 * t : nullptr;
  uint8_t* const codes = (is_v ? p.c.v : p.c.k) + h * p.c.head_stride / 2 + 4 * G * t;
  uint16_t* const prms = is_v ? p.c.v_group : p.c.k_group;

  for (int token0 = 0; token0 < tokens; token0 += 8) {
    const int token = token0 + static_cast<int>(lane >> 2);
    const bool real = token < tokens;
    const __nv_bfloat16* src = x + token * p.ld;
    const float2* row = p.table + static_cast<int64_t>(pos0 + token) * half;
    int64_t page = -2;
    uint4 u[G];
    if (real) {
      page = p.page_table[b * p.ld_table + ((pos0 + token) >> shift)];
#pragma unroll
      for (int y = 0; y < G; ++y) u[y] = *reinterpret_cast<const uint4*>(src + 32 * y);
    } else {
#pragma unroll
      for (int y = 0; y < G; ++y) u[y] = make_uint4(0, 0, 0, 0);
    }
    float f[G][8];
#pragma unroll
    for (int y = 0; y < G; ++y) unpack_bf16x8(u[y], f[y]);
    if (real && whole) {
#pragma unroll
      for (int y = 0; y < G / 2; ++y) {
        float c[8], s[8];
        rotary_load_table(row + 32 * y + 8 * t, c, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) rotary_turn(f[y][i], f[G / 2 + y][i], c[i], s[i]);
      }
    } else if (real && half > 0) {
#pragma unroll
      for (int y = 0; y < G; ++y) {
        const int at = 32 * y + 8 * t;
        if (at >= 2 * half) continue;
        if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float4 cs = __ldg(reinterpret_cast<const float4*>(row + at / 2) + i);  // as rotary_load_table says
            rotary_turn(f[y][4 * i], f[y][4 * i + 1], cs.x, cs.y);
            rotary_turn(f[y][4 * i + 2], f[y][4 * i + 3], cs.z, cs.w);
          }
        } else {
          // The piece is its pairs' second half, or the first: one of rotary_turn's two sums.
          const bool second = at >= half;
          float o[8], c[8], s[8];
          unpack_bf16x8(*reinterpret_cast<const uint4*>(src + 32 * y + (second ? -half : half)), o);
          rotary_load_table(row + (second ? at - half : at), c, s);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = __fmul_rn(f[y][i], c[i]), d = __fmul_rn(o[i], s[i]);
            f[y][i] = second ? __fadd_rn(a, d) : __fsub_rn(a, d);
          }
        }
      }
    }
    __syncwarp();  // every lane has read its pieces: k_out may be the projection's own columns
    uint32_t w[G], params[G], out[G];
#pragma unroll
    for (int y = 0; y < G; ++y) w[y] = int4_codes(f[y], params[y]);
    if (!real) continue;
    if (page < 0 || page >= p.c.pages) {
      record_status(kKernelCacheAppend, 2, kReasonBadIndex);
      continue;
    }
    if (copy != nullptr) {
#pragma unroll
      for (int y = 0; y < G; ++y) *reinterpret_cast<uint4*>(copy + token * p.ld_k_out + 32 * y) = pack_bf16x8(f[y]);
    }
    const int slot = (pos0 + token) & ((1 << shift) - 1);
    halves_apart(w, out);
    store_words(codes + page * p.c.page_stride / 2 + slot * (hd / 2), out);
    if (t == 0) {
      halves_apart(params, out);
      store_words(prms + (((page * kv_heads + h) << shift) + slot) * (2 * G), out);
    }
  }
}

// Tokens of a warp: as many as keep the call's warps at least four times the machine's, so that a short call has all its
// loads under way at once.
static int int4_tile_tokens(int64_t tokens, int64_t roles, int64_t batch, int sm_count) {
  int tile = kInt4Tile;
  while (tile > 1 && (tokens + tile - 1) / tile * roles * batch < int64_t{64} * sm_count) tile /= 2;
  return tile;
}

template <int G>
static cudaError_t launch_cache_append_int4_g(const AppendParams& p, dim3 grid, int interleaved, int tile, unsigned role_blocks,
                                              cudaStream_t stream) {
  return interleaved
             ? launch_pdl(cache_append_int4_kernel<G, true>, grid, dim3(kInt4Threads), 0, stream, p, tile, role_blocks)
             : launch_pdl(cache_append_int4_kernel<G, false>, grid, dim3(kInt4Threads), 0, stream, p, tile, role_blocks);
}

static cudaError_t launch_cache_append_int4(const AppendParams& p, int64_t max_new, int interleaved, int sm_count,
                                            cudaStream_t stream) {
  const int64_t roles = static_cast<int64_t>(p.c.kv_heads) * (p.rotary_dim > 0 ? 3 : 2);
  const int tile = int4_tile_tokens(max_new, roles, p.batch, sm_count);
  const int64_t role_blocks = (roles + kInt4Threads / 32 - 1) / (kInt4Threads / 32);
  const int64_t blocks = (max_new + tile - 1) / tile * role_blocks;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks), 1, static_cast<unsigned>(p.batch));
  const unsigned rb = static_cast<unsigned>(role_blocks);
  switch (p.c.head_dim / kInt4Group) {
    case 1: return launch_cache_append_int4_g<1>(p, grid, interleaved, tile, rb, stream);
    case 2: return launch_cache_append_int4_g<2>(p, grid, interleaved, tile, rb, stream);
    case 3: return launch_cache_append_int4_g<3>(p, grid, interleaved, tile, rb, stream);
    case 4: return launch_cache_append_int4_g<4>(p, grid, interleaved, tile, rb, stream);
    case 5: return launch_cache_append_int4_g<5>(p, grid, interleaved, tile, rb, stream);
    case 6: return launch_cache_append_int4_g<6>(p, grid, interleaved, tile, rb, stream);
    case 7: return launch_cache_append_int4_g<7>(p, grid, interleaved, tile, rb, stream);
    case 8: return launch_cache_append_int4_g<8>(p, grid, interleaved, tile, rb, stream);
    default: return cudaErrorInvalidValue;
  }
}

// ---------------------------------------------------------------------------------------------
// A cache's tokens as rows
// ---------------------------------------------------------------------------------------------
struct ReadParams {
  CachePages c;
  int batch;
  int64_t rows;  // of k_out and v_out
  int64_t max_len;
  const int32_t* out_start;
  const int32_t* length;
  const int32_t* start;
  const int32_t* page_table;
  int64_t ld_table;
  int table_pages;
  __nv_bfloat16* k_out;  // [rows][ld], or null
  __nv_bfloat16* v_out;
  int64_t ld_k_out, ld_v_out;
};

// 8 neighbours' codes as values in bf16: a code in the lowest bits of a half is 128 + code there, and the sum with the
// middle is rounded once, as from 32 bits (a product of a code and a step has 12 bits: no sum of it and a middle is next to
// the border between two bf16 values without being exact in fp32).
__device__ __forceinline__ uint4 int4_values(uint32_t w, uint32_t params) {
  const uint32_t step = __byte_perm(params, params, 0x1010u), mid = __byte_perm(params, params, 0x3232u);
  const uint32_t high = w >> 4;
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = __byte_perm(w, high, i | (4 + i) << 8);  // byte i in each half, of w and of its upper codes
    const uint32_t c = (pair & 0x000f000fu) | 0x43004300u;
    v[i] = bf16x2_fma(bf16x2_less_136(c), step, mid);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// What is read comes by coherent loads: the launch before this one may be the append that wrote it. G: groups of 4-bit
// codes; other types take 16 elements to a lane, 8 in each half of the head.
template <int kType, int G>
__global__ void __launch_bounds__(kInt4Threads, G <= 4 ? 4 : 2) cache_read_kernel(const ReadParams p, const int tile_tokens,
                                                                  const unsigned role_blocks) {
  constexpr int kAtOnce = G <= 4 ? 4 : 2;  // turns in flight together
  const unsigned tile = blockIdx.x / role_blocks;
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int kv_heads = p.c.kv_heads;
  const int role = static_cast<int>((blockIdx.x - tile * role_blocks) * (kInt4Threads / 32) + (threadIdx.x >> 5));
  if (role >= kv_heads * (p.k_out != nullptr && p.v_out != nullptr ? 2 : 1)) return;
  pdl_wait_previous_grid();
  pdl_allow_next_grid();
  const int b = blockIdx.z;
  const int count = p.length[b];
  const int from0 = p.start[b];
  const int first = p.out_start[b];
  if (count <= 0) return;
  const int shift = p.c.page_shift;
  if (from0 < 0 || first < 0 || count > p.max_len || static_cast<int64_t>(first) + count > p.rows ||
      static_cast<int64_t>(from0) + count > (static_cast<int64_t>(p.table_pages) << shift)) {
    record_status(kKernelCacheRead, 1, kReasonBadIndex);
    return;
  }
  if (static_cast<int64_t>(tile) * tile_tokens >= count) return;
  const int from = static_cast<int>(tile) * tile_tokens;
  const int tokens = min(tile_tokens, count - from);
  const int pos0 = from0 + from;
  const bool is_v = p.k_out == nullptr || role >= kv_heads;
  const int h = role >= kv_heads ? role - kv_heads : role;
  const int hd = kType == kCacheInt4 ? 32 * G : p.c.head_dim;
  const int lanes = kType == kCacheInt4 ? 4 : hd >> 4;  // of a token
  const int per_turn = 32 / lanes;
  const int mine = lane / lanes;
  const int t = lane - mine * lanes;
  const int64_t ld = is_v ? p.ld_v_out : p.ld_k_out;
  __nv_bfloat16* out = (is_v ? p.v_out : p.k_out) + (static_cast<int64_t>(first) + from) * ld + h * hd + 8 * t;
  const uint8_t* const data = is_v ? p.c.v : p.c.k;
  const uint16_t* const prms = is_v ? p.c.v_group : p.c.k_group;
  const float* const scales = is_v ? p.c.v_scale : p.c.k_scale;
  const int32_t* const table = p.page_table + b * p.ld_table;
  if (mine >= per_turn) return;

  for (int token0 = mine; token0 < tokens; token0 += kAtOnce * per_turn) {
    int page[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int token = token0 + k * per_turn;
      page[k] = -1;  // no token
      if (token < tokens) {
        page[k] = table[(pos0 + token) >> shift];
        if (page[k] < 0 || page[k] >= p.c.pages) {
          record_status(kKernelCacheRead, 2, kReasonBadIndex);
          page[k] = -1;
        }
      }
    }
    if constexpr (kType == kCacheInt4) {
      uint32_t w[kAtOnce][G], prm[kAtOnce][G];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        if (page[k] < 0) continue;
        const int slot = (pos0 + token0 + k * per_turn) & ((1 << shift) - 1);
        load_words(data + (page[k] * p.c.page_stride + h * p.c.head_stride) / 2 + slot * (hd / 2) + 4 * G * t, w[k]);
        load_words(prms + (((static_cast<int64_t>(page[k]) * kv_heads + h) << shift) + slot) * (2 * G), prm[k]);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        if (page[k] < 0) continue;
        __nv_bfloat16* y_out = out + (token0 + k * per_turn) * ld;
#pragma unroll
        for (int y = 0; y < G; ++y)
          __stcs(reinterpret_cast<uint4*>(y_out + 32 * y), int4_values(halves_together(w[k], y), halves_together(prm[k], y)));
      }
    } else {
      uint4 u[kAtOnce][2];
      float scale[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        if (page[k] < 0) continue;
        const int slot = (pos0 + token0 + k * per_turn) & ((1 << shift) - 1);
        const int64_t element = page[k] * p.c.page_stride + h * p.c.head_stride + slot * hd + 8 * t;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (kType == kCacheE4m3) {
            const uint2 codes = load_once2(data + element + i * (hd / 2));
            u[k][i].x = codes.x;
            u[k][i].y = codes.y;
          } else {
            u[k][i] = load_once4(data + 2 * (element + i * (hd / 2)));
          }
        }
        if constexpr (kType == kCacheE4m3) scale[k] = __uint_as_float(load_once(scales + static_cast<int64_t>(page[k]) * kv_heads + h));
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        if (page[k] < 0) continue;
        __nv_bfloat16* y_out = out + (token0 + k * per_turn) * ld;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if constexpr (kType == kCacheE4m3) {
            const uint32_t two[4] = {u[k][i].x, u[k][i].x >> 16, u[k][i].y, u[k][i].y >> 16};
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 v = f16x2_values(e4m3x2_to_f16x2(two[j]));
              o[j] = pack_bf16x2(v.x * scale[k], v.y * scale[k]);
            }
            u[k][i] = make_uint4(o[0], o[1], o[2], o[3]);
          }
          __stcs(reinterpret_cast<uint4*>(y_out + i * (hd / 2)), u[k][i]);
        }
      }
    }
  }
}

static cudaError_t launch_cache_read(const ReadParams& p, int type, int sm_count, cudaStream_t stream) {
  const int64_t roles = static_cast<int64_t>(p.c.kv_heads) * (p.k_out != nullptr && p.v_out != nullptr ? 2 : 1);
  const int tile = int4_tile_tokens(p.max_len, roles, p.batch, sm_count);
  const int64_t role_blocks = (roles + kInt4Threads / 32 - 1) / (kInt4Threads / 32);
  const int64_t blocks = (p.max_len + tile - 1) / tile * role_blocks;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks), 1, static_cast<unsigned>(p.batch)), threads(kInt4Threads);
  const unsigned rb = static_cast<unsigned>(role_blocks);
  if (type == kCacheE4m3) return launch_pdl(cache_read_kernel<kCacheE4m3, 0>, grid, threads, 0, stream, p, tile, rb);
  if (type == kCacheBf16) return launch_pdl(cache_read_kernel<kCacheBf16, 0>, grid, threads, 0, stream, p, tile, rb);
  switch (p.c.head_dim / kInt4Group) {
    case 1: return launch_pdl(cache_read_kernel<kCacheInt4, 1>, grid, threads, 0, stream, p, tile, rb);
    case 2: return launch_pdl(cache_read_kernel<kCacheInt4, 2>, grid, threads, 0, stream, p, tile, rb);
    case 3: return launch_pdl(cache_read_kernel<kCacheInt4, 3>, grid, threads, 0, stream, p, tile, rb);
    case 4: return launch_pdl(cache_read_kernel<kCacheInt4, 4>, grid, threads, 0, stream, p, tile, rb);
    case 5: return launch_pdl(cache_read_kernel<kCacheInt4, 5>, grid, threads, 0, stream, p, tile, rb);
    case 6: return launch_pdl(cache_read_kernel<kCacheInt4, 6>, grid, threads, 0, stream, p, tile, rb);
    case 7: return launch_pdl(cache_read_kernel<kCacheInt4, 7>, grid, threads, 0, stream, p, tile, rb);
    case 8: return launch_pdl(cache_read_kernel<kCacheInt4, 8>, grid, threads, 0, stream, p, tile, rb);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace b2
