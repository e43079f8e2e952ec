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
// Both kernels are bound by HBM, the append by the projection's rows in and the rotated queries out. A warp takes a tile of
// tokens of one head (of K, of V, or the query heads of one key head); 8 neighbouring elements are a thread's piece, so that
// 4 lanes share a group and two exchanges find its least and most value, and lanes of neighbouring groups exchange halves so
// that each stores (or loads) a whole word. A thread rotates only its own piece and reads the pair's other half beside it.
#pragma once
#include "b2_common.cuh"
#include "cache_append.cuh"
#include "cache_attention.cuh"
#include "rotary.cuh"

namespace b2 {

constexpr int kInt4Group = 32;
constexpr float kInt4LeastStep = 7.888609052210118e-31f;  // 2^-100
constexpr int kInt4Threads = 256;
constexpr int kInt4Tile = 16;   // tokens of a warp, at most
constexpr int kInt4Unroll = 2;  // turns of a warp that are in flight together

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
  float step = bf16_round(__fdiv_rn(range, 15.f));
  if (step < kInt4LeastStep) step = 0.f;
  float mid = bf16_round(__fadd_rn(lo, 8.f * step));
  if (!is_finite(range)) step = mid = __uint_as_float(0x7fc00000u);
  const float r = step > 0.f ? bf16_round(__frcp_rn(step)) : 0.f;
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

// Where a thread's piece of 8 elements (number `piece` of a row) lies, and who holds what: pieces 4 group + j.
struct Int4Piece {
  int group, j;
  bool odd;
};
__device__ __forceinline__ Int4Piece int4_piece(int piece) { return {piece >> 2, piece & 3, ((piece >> 2) & 1) != 0}; }

// Stores a piece's codes, and its group's parameters, of the token whose row and parameters begin at `row` and `prm`. `partner`s:
// the same of the neighbouring group's lane (4 lanes away), used where the number of groups is even.
__device__ __forceinline__ void int4_store(uint8_t* row, uint16_t* prm, int groups, const Int4Piece& at, uint32_t w,
                                           uint32_t params, uint32_t w_partner, uint32_t params_partner) {
  const int first = 2 * (2 * at.j * groups + at.group);  // bytes to the piece's first half
  if ((groups & 1) == 0) {
    if (at.odd)
      *reinterpret_cast<uint32_t*>(row + first + 2 * groups - 2) = __byte_perm(w_partner, w, 0x7632u);
    else
      *reinterpret_cast<uint32_t*>(row + first) = __byte_perm(w, w_partner, 0x5410u);
    if (!at.odd && at.j == 0) *reinterpret_cast<uint32_t*>(prm + at.group) = __byte_perm(params, params_partner, 0x5410u);
    if (!at.odd && at.j == 1)
      *reinterpret_cast<uint32_t*>(prm + groups + at.group) = __byte_perm(params, params_partner, 0x7632u);
  } else {
    *reinterpret_cast<uint16_t*>(row + first) = static_cast<uint16_t>(w);
    *reinterpret_cast<uint16_t*>(row + first + 2 * groups) = static_cast<uint16_t>(w >> 16);
    if (at.j == 0) prm[at.group] = static_cast<uint16_t>(params);
    if (at.j == 1) prm[groups + at.group] = static_cast<uint16_t>(params >> 16);
  }
}

template <bool kInterleaved>
__global__ void __launch_bounds__(kInt4Threads) cache_append_int4_kernel(const AppendParams p, const int tile_tokens,
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
  const int hd = p.c.head_dim;
  if (role >= 2 * kv_heads) {
    append_queries<kInterleaved>(p, role - 2 * kv_heads, row0, pos0, static_cast<unsigned>(tokens), lane, 32u);
    return;
  }
  const bool is_v = role >= kv_heads;
  const int h = is_v ? role - kv_heads : role;
  const int pieces = hd >> 3;
  const int groups = hd >> 5;
  const int per_turn = 32 / pieces;  // whole tokens: a token's pieces are read before one of them is written (k_out may be x)
  const int half = (is_v ? 0 : p.rotary_dim) >> 1;
  const int mine = static_cast<int>(lane) / pieces;
  const int piece = static_cast<int>(lane) - mine * pieces;
  const Int4Piece at = int4_piece(piece);
  const bool turned = 8 * piece < 2 * half;
  const bool second = turned && !kInterleaved && 8 * piece >= half;
  const int pair0 = kInterleaved ? 4 * piece : second ? 8 * piece - half : 8 * piece;
  const int partner = second ? 8 * piece - half : 8 * piece + half;
  const __nv_bfloat16* x = p.qkv + row0 * p.ld + (is_v ? p.v_col : p.k_col) + h * hd;
  __nv_bfloat16* copy = !is_v && p.k_out != nullptr ? p.k_out + row0 * p.ld_k_out + h * hd : nullptr;
  uint8_t* const codes = is_v ? p.c.v : p.c.k;
  uint16_t* const prms = is_v ? p.c.v_group : p.c.k_group;

  for (int token0 = mine; __any_sync(0xffffffffu, token0 < tokens && mine < per_turn); token0 += kInt4Unroll * per_turn) {
    uint4 own[kInt4Unroll], other[kInt4Unroll];
    float cs[kInt4Unroll][16];
    int64_t page[kInt4Unroll];
#pragma unroll
    for (int k = 0; k < kInt4Unroll; ++k) {
      const int token = token0 + k * per_turn;
      const bool real = mine < per_turn && token < tokens;
      own[k] = other[k] = make_uint4(0, 0, 0, 0);
      page[k] = -2;
      if (!real) continue;
      const __nv_bfloat16* src = x + token * p.ld;
      own[k] = *reinterpret_cast<const uint4*>(src + 8 * piece);
      page[k] = p.page_table[b * p.ld_table + ((pos0 + token) >> shift)];
      if (turned) {
        const float2* row = p.table + static_cast<int64_t>(pos0 + token) * half + pair0;
        if (!kInterleaved) other[k] = *reinterpret_cast<const uint4*>(src + partner);
#pragma unroll
        for (int i = 0; i < (kInterleaved ? 2 : 4); ++i) {
          const float4 t = __ldg(reinterpret_cast<const float4*>(row) + i);  // as rotary_load_table says
          cs[k][4 * i] = t.x;
          cs[k][4 * i + 1] = t.y;
          cs[k][4 * i + 2] = t.z;
          cs[k][4 * i + 3] = t.w;
        }
      }
    }
    __syncwarp();  // every lane has read its pieces
#pragma unroll
    for (int k = 0; k < kInt4Unroll; ++k) {
      const int token = token0 + k * per_turn;
      float f[8];
      unpack_bf16x8(own[k], f);
      if (turned) {
        if constexpr (kInterleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) rotary_turn(f[2 * i], f[2 * i + 1], cs[k][2 * i], cs[k][2 * i + 1]);
        } else {
          float o[8];
          unpack_bf16x8(other[k], o);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            // The piece is its pairs' second half, or the first: one of rotary_turn's two sums.
            const float a = __fmul_rn(f[i], cs[k][2 * i]);
            const float c = __fmul_rn(o[i], cs[k][2 * i + 1]);
            f[i] = second ? __fadd_rn(a, c) : __fsub_rn(a, c);
          }
        }
      }
      uint32_t params;
      const uint32_t w = int4_codes(f, params);
      const uint32_t w_partner = __shfl_xor_sync(0xffffffffu, w, 4);
      const uint32_t params_partner = __shfl_xor_sync(0xffffffffu, params, 4);
      if (mine >= per_turn || token >= tokens) continue;
      if (page[k] < 0 || page[k] >= p.c.pages) {
        record_status(kKernelCacheAppend, 2, kReasonBadIndex);
        continue;
      }
      if (copy != nullptr) *reinterpret_cast<uint4*>(copy + token * p.ld_k_out + 8 * piece) = pack_bf16x8(f);
      const int slot = (pos0 + token) & ((1 << shift) - 1);
      uint8_t* row = codes + (page[k] * p.c.page_stride + h * p.c.head_stride) / 2 + slot * (hd / 2);
      uint16_t* prm = prms + (((page[k] * kv_heads + h) << shift) + slot) * (2 * groups);
      int4_store(row, prm, groups, at, w, params, w_partner, params_partner);
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

static cudaError_t launch_cache_append_int4(const AppendParams& p, int64_t max_new, int interleaved, int sm_count,
                                            cudaStream_t stream) {
  const int64_t roles = static_cast<int64_t>(p.c.kv_heads) * (p.rotary_dim > 0 ? 3 : 2);
  const int tile = int4_tile_tokens(max_new, roles, p.batch, sm_count);
  const int64_t role_blocks = (roles + kInt4Threads / 32 - 1) / (kInt4Threads / 32);
  const int64_t blocks = (max_new + tile - 1) / tile * role_blocks;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks), 1, static_cast<unsigned>(p.batch));
  const unsigned rb = static_cast<unsigned>(role_blocks);
  return interleaved ? launch_pdl(cache_append_int4_kernel<true>, grid, dim3(kInt4Threads), 0, stream, p, tile, rb)
                     : launch_pdl(cache_append_int4_kernel<false>, grid, dim3(kInt4Threads), 0, stream, p, tile, rb);
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

// 8 codes as values.
__device__ __forceinline__ uint4 int4_values(uint32_t w, float step, float mid) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = __uint_as_float(((w >> (4 * i)) & 15u) | 0x4b000000u) - (8388608.f + 8.f);
    f[i] = __fadd_rn(__fmul_rn(c, step), mid);  // (the product is exact)
  }
  return pack_bf16x8(f);
}

// The codes and values that are read come by coherent loads: the launch before this one may be the append that wrote them.
template <int kType>
__global__ void __launch_bounds__(kInt4Threads) cache_read_kernel(const ReadParams p, const int tile_tokens,
                                                                  const unsigned role_blocks) {
  constexpr int kAtOnce = 4;  // turns in flight together
  const unsigned tile = blockIdx.x / role_blocks;
  const unsigned lane = threadIdx.x & 31;
  const int kv_heads = p.c.kv_heads;
  int role = static_cast<int>((blockIdx.x - tile * role_blocks) * (kInt4Threads / 32) + (threadIdx.x >> 5));
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
  const int hd = p.c.head_dim;
  const int pieces = hd >> 3;
  const int groups = hd >> 5;
  const int per_turn = 32 / pieces;
  const int mine = static_cast<int>(lane) / pieces;
  const int piece = static_cast<int>(lane) - mine * pieces;
  const Int4Piece at = int4_piece(piece);
  const int64_t ld = is_v ? p.ld_v_out : p.ld_k_out;
  __nv_bfloat16* out = (is_v ? p.v_out : p.k_out) + (static_cast<int64_t>(first) + from) * ld + h * hd + 8 * piece;
  const uint8_t* const codes = is_v ? p.c.v : p.c.k;
  const uint16_t* const prms = is_v ? p.c.v_group : p.c.k_group;
  const float* const scales = is_v ? p.c.v_scale : p.c.k_scale;
  const int even_at = 2 * (2 * at.j * groups + at.group) + (at.odd ? 2 * groups - 2 : 0);

  for (int token0 = mine; __any_sync(0xffffffffu, token0 < tokens && mine < per_turn); token0 += kAtOnce * per_turn) {
    int64_t page[kAtOnce];
    uint4 u[kAtOnce];
    uint32_t prm[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int token = token0 + k * per_turn;
      page[k] = -2;  // no token
      if (mine < per_turn && token < tokens) {
        page[k] = p.page_table[b * p.ld_table + ((pos0 + token) >> shift)];
        if (page[k] < 0 || page[k] >= p.c.pages) {
          record_status(kKernelCacheRead, 2, kReasonBadIndex);
          page[k] = -2;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int slot = (pos0 + token0 + k * per_turn) & ((1 << shift) - 1);
      u[k] = make_uint4(0, 0, 0, 0);
      prm[k] = 0;
      if (page[k] < 0) continue;
      const int64_t element = page[k] * p.c.page_stride + h * p.c.head_stride + static_cast<int64_t>(slot) * hd;
      if constexpr (kType == kCacheInt4) {
        const uint8_t* row = codes + element / 2;
        const uint16_t* q = prms + (((page[k] * kv_heads + h) << shift) + slot) * (2 * groups);
        if ((groups & 1) == 0) {
          u[k].x = load_once(row + even_at);
        } else {
          u[k].x = load_once_u16(row + 2 * (2 * at.j * groups + at.group)) |
                   static_cast<uint32_t>(load_once_u16(row + 2 * ((2 * at.j + 1) * groups + at.group))) << 16;
        }
        prm[k] = load_once_u16(q + at.group) | static_cast<uint32_t>(load_once_u16(q + groups + at.group)) << 16;
      } else if constexpr (kType == kCacheE4m3) {
        const uint2 w = load_once2(codes + element + 8 * piece);
        u[k].x = w.x;
        u[k].y = w.y;
        prm[k] = load_once(scales + page[k] * kv_heads + h);
      } else {
        u[k] = load_once4(codes + 2 * (element + 8 * piece));
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if constexpr (kType == kCacheInt4) {
        uint32_t w = u[k].x;
        if ((groups & 1) == 0) {
          const uint32_t partner = __shfl_xor_sync(0xffffffffu, w, 4);
          w = at.odd ? __byte_perm(partner, w, 0x7632u) : __byte_perm(w, partner, 0x5410u);
        }
        u[k] = int4_values(w, __uint_as_float(prm[k] << 16), __uint_as_float(prm[k] & 0xffff0000u));
      } else if constexpr (kType == kCacheE4m3) {
        const float scale = __uint_as_float(prm[k]);
        const uint32_t w[4] = {u[k].x, u[k].x >> 16, u[k].y, u[k].y >> 16};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t two = e4m3x2_to_f16x2(w[i]);
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&two));
          o[i] = pack_bf16x2(v.x * scale, v.y * scale);
        }
        u[k] = make_uint4(o[0], o[1], o[2], o[3]);
      }
      if (page[k] >= 0) __stcs(reinterpret_cast<uint4*>(out + (token0 + k * per_turn) * ld), u[k]);
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
  switch (type) {
    case kCacheInt4:
      return launch_pdl(cache_read_kernel<kCacheInt4>, grid, threads, 0, stream, p, tile, rb);
    case kCacheE4m3:
      return launch_pdl(cache_read_kernel<kCacheE4m3>, grid, threads, 0, stream, p, tile, rb);
    default:
      return launch_pdl(cache_read_kernel<kCacheBf16>, grid, threads, 0, stream, p, tile, rb);
  }
}

}  // namespace b2
