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
// A token's parameters are worked out by one lane a group (for 2 and 4 groups) and handed round, the codes of two elements
// come from one packed instruction each where there is one (69 -> 62 us with the next rows' loads ahead).
// Measured on one B200 (us a call, floor at the measured copy rate in brackets): append of ragged prompts of 16 sequences of up to
// 2048 tokens, 16 heads of 64, rotated queries and keys kept: 60 (40); chunks of three documents, 16 query and 4 key heads of
// 128, a quarter turned: 15 (8); one token in each of 64 sequences 4, a launch. Reading 4 x 65536 tokens of 8 heads of 128 in 4
// bits: 221 (218); 16 sequences of up to 4096 tokens of 16 heads of 64 in 8 bits: 51 (43); in bf16 4 x 65536 tokens of 8 heads of
// 128 328 (332), 16 x 4096 of 16 heads of 64 88 (83). The append's issue slots are 62 % busy and its ALU 56 (some 18
// instructions an element for ranges and codes).
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

// The least and the most value of each group, of 8 values in each of the four lanes that share a token: after it lane t (of
// the four) holds those of group t (of t % 2 for two groups), or of all groups (`lo`, `hi` per group) otherwise.
template <int G>
__device__ __forceinline__ void int4_ranges(const float (&x)[G][8], int t, float (&lo)[G], float (&hi)[G]) {
#pragma unroll
  for (int y = 0; y < G; ++y) {
    lo[y] = min_nan(min3_nan(x[y][5], x[y][6], x[y][7]), min3_nan(min3_nan(x[y][0], x[y][1], x[y][2]), x[y][3], x[y][4]));
    hi[y] = max_nan(max3_nan(x[y][5], x[y][6], x[y][7]), max3_nan(max3_nan(x[y][0], x[y][1], x[y][2]), x[y][3], x[y][4]));
  }
  if constexpr (G == 2 || G == 4) {
    // Each exchange leaves a lane half of the groups, those whose number agrees with its own in that bit.
    const bool odd = t & 1;
#pragma unroll
    for (int y = 0; y < G; y += 2) {
      const float lo_mine = odd ? lo[y + 1] : lo[y], hi_mine = odd ? hi[y + 1] : hi[y];
      lo[y] = min_nan(lo_mine, __shfl_xor_sync(0xffffffffu, odd ? lo[y] : lo[y + 1], 1));
      hi[y] = max_nan(hi_mine, __shfl_xor_sync(0xffffffffu, odd ? hi[y] : hi[y + 1], 1));
    }
    const bool high = G == 4 && (t & 2);
    const float lo_mine = high ? lo[G - 2] : lo[0], hi_mine = high ? hi[G - 2] : hi[0];
    lo[0] = min_nan(lo_mine, __shfl_xor_sync(0xffffffffu, high ? lo[0] : lo[G - 2], 2));
    hi[0] = max_nan(hi_mine, __shfl_xor_sync(0xffffffffu, high ? hi[0] : hi[G - 2], 2));
  } else {
#pragma unroll
    for (int i = 1; i < 4; i *= 2)
#pragma unroll
      for (int y = 0; y < G; ++y) {
        lo[y] = min_nan(lo[y], __shfl_xor_sync(0xffffffffu, lo[y], i));
        hi[y] = max_nan(hi[y], __shfl_xor_sync(0xffffffffu, hi[y], i));
      }
  }
}

// A group's step and middle as bf16 bits, the step in the lower half; `clamp`: whether a code may need it.
struct Int4Group {
  float mid, r;
  uint32_t params;
  bool clamp;
};
__device__ __forceinline__ Int4Group int4_group(float lo, float hi) {
  const float range = __fsub_rn(hi, lo);  // not finite where a value is not
  float step = bf16_round(divide_by_15(range));
  if (step < kInt4LeastStep) step = 0.f;
  Int4Group q;
  q.mid = bf16_round(__fadd_rn(lo, 8.f * step));
  if (!is_finite(range)) step = q.mid = __uint_as_float(0x7fc00000u);
  // (1 / step is never within 2^-17 of the middle between two bf16 values, so that an approximate one rounds alike)
  q.r = step > 0.f ? bf16_round(fast_rcp(step)) : 0.f;
  q.params = pack_bf16x2(step, q.mid);
  // (Rounded to the nearest whole number they lie in [-8, 7] unless the middle's own rounding is half a step or more: the
  // products grow with x, so the least and the most value tell.)
  q.clamp = !(__fmul_rn(__fsub_rn(lo, q.mid), q.r) >= -8.5f && __fmul_rn(__fsub_rn(hi, q.mid), q.r) < 7.5f);
  return q;
}

// 8 values of a group as codes in 4 bits each.
__device__ __forceinline__ uint32_t int4_codes(const float (&x)[8], float mid, float r, bool clamp) {
  float q[8];  // (each operation rounded by itself, two at a time)
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    asm("{.reg .b64 a, m, s;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 m, {%4, %4};\n\tmov.b64 s, {%5, %5};\n\t"
        "add.rn.f32x2 a, a, m;\n\tmul.rn.f32x2 a, a, s;\n\tmov.b64 {%0, %1}, a;}"
        : "=f"(q[i]), "=f"(q[i + 1]) : "f"(x[i]), "f"(x[i + 1]), "f"(-mid), "f"(r));
  }
  if (clamp) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = fmaxf(fminf(q[i], 7.f), -8.f);
  }
  // Adding 1.5 * 2^23 rounds to a whole number (to the even one at a half), 8 more makes it the code in the lowest bits; the
  // words' sum in 16ths, less the constant's, has the codes side by side.
  constexpr float kMagic = 12582912.f + 8.f;
  constexpr uint32_t kOver = 0x4b400000u;
  uint32_t w = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) w = w * 16u + __float_as_uint(__fadd_rn(q[i], kMagic));
  w -= kOver * 0x11111111u;
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

// (64 registers, four CTAs an SM, up to 4 groups: ragged prompts of 16 heads of 64 63 us, 70 with three or with five. They are a few
// too few: 4 to 12 bytes of spills for 2 groups, 24 for 3, 32 to 84 for 4; of 6 and 8 groups, with 128, 16 and 52 to 68.)
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

  // Up to 2 groups the next tokens' rows are under way while these are coded (ragged prompts of 16 heads of 64 69 -> 64 us; of 4
  // groups the registers do not hold both: 16 query and 4 key heads of 128 17.6 -> 18.7).
  uint4 u[G];
  int64_t page = -2;
  auto fetch = [&](int token) {
    page = -2;
    if (token < tokens) {
      page = p.page_table[b * p.ld_table + ((pos0 + token) >> shift)];
#pragma unroll
      for (int y = 0; y < G; ++y) u[y] = *reinterpret_cast<const uint4*>(x + token * p.ld + 32 * y);
    } else {
#pragma unroll
      for (int y = 0; y < G; ++y) u[y] = make_uint4(0, 0, 0, 0);
    }
  };
  if constexpr (G <= 2) fetch(static_cast<int>(lane >> 2));
  for (int token0 = 0; token0 < tokens; token0 += 8) {
    const int token = token0 + static_cast<int>(lane >> 2);
    if constexpr (G > 2) fetch(token);
    const bool real = token < tokens;
    const __nv_bfloat16* src = x + token * p.ld;
    const float2* row = p.table + static_cast<int64_t>(pos0 + token) * half;
    const int64_t my_page = page;
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
    if constexpr (G <= 2) fetch(token + 8);
    __syncwarp();  // every lane has read its pieces: k_out may be the projection's own columns
    uint32_t w[G], params[G], out[G];
    float lo[G], hi[G];
    int4_ranges<G>(f, t, lo, hi);
    if constexpr (G == 2 || G == 4) {
      const Int4Group mine = int4_group(lo[0], hi[0]);
      const bool clamp = __any_sync(0xffffffffu, mine.clamp);
#pragma unroll
      for (int y = 0; y < G; ++y) {
        const int from = (lane & 28) + y;
        params[y] = __shfl_sync(0xffffffffu, mine.params, from);
        const float r = __shfl_sync(0xffffffffu, mine.r, from);
        w[y] = int4_codes(f[y], __uint_as_float(params[y] & 0xffff0000u), r, clamp);
      }
    } else {
#pragma unroll
      for (int y = 0; y < G; ++y) {
        const Int4Group group = int4_group(lo[y], hi[y]);
        params[y] = group.params;
        w[y] = int4_codes(f[y], group.mid, group.r, __any_sync(0xffffffffu, group.clamp));
      }
    }
    if (!real) continue;
    if (my_page < 0 || my_page >= p.c.pages) {
      record_status(kKernelCacheAppend, 2, kReasonBadIndex);
      continue;
    }
    if (copy != nullptr) {
#pragma unroll
      for (int y = 0; y < G; ++y) *reinterpret_cast<uint4*>(copy + token * p.ld_k_out + 32 * y) = pack_bf16x8(f[y]);
    }
    const int slot = (pos0 + token) & ((1 << shift) - 1);
    halves_apart(w, out);
    store_words(codes + my_page * p.c.page_stride / 2 + slot * (hd / 2), out);
    if (t == 0) {
      halves_apart(params, out);
      store_words(prms + (((my_page * kv_heads + h) << shift) + slot) * (2 * G), out);
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
