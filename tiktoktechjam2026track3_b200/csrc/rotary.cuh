// Rotary positions: pairs (x1, x2) of a head turned by the angle of their token's position,
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s,   (c, s) = table[position][pair],
// with the transpose (s -> -s), which is the gradient. Half layout: pair i is (x[i], x[i + r/2]) of the
// head's first r = rotary_dim elements; interleaved: (x[2i], x[2i + 1]). Elements past r are copied.
// The reference has no positions; the projections whose rows are turned are models.py:51-53.
//
// Bound by HBM: two bytes in and two out per element, and one table row (4 r bytes) per token, which its
// heads share. The work is cut into chunks of 16 elements (8 pairs): two 16-byte loads, which are
// neighbours in the interleaved layout and r/2 elements apart in the half layout, where eight
// neighbouring threads still cover whole 128-byte lines. Rows are read and written once, so both go past the caches
// (streaming loads and stores), and a CTA is small, so that its slot is free again soon.
// Measured on one B200 (us a call, floor at the measured copy rate in brackets): 32768 rows of 32 heads of 128, half
// layout, 108 (85; 132 with cached accesses and 256 threads a CTA); the gradient over half of each head, neighbouring
// pairs, 94 (83; 113); 16384 x 32 heads of 64: 26 (21). What is left is the table: 64 bytes a thread and chunk, from
// L1 (its data pipe is 52 % busy) for each of the heads or, four heads to a thread, once for four.
#pragma once
#include "b2_common.cuh"

namespace b2 {

struct RotaryParams {
  const __nv_bfloat16* x;  // may be `out`: a pair is read and written by one thread
  __nv_bfloat16* out;
  int64_t ld_x, ld_out;
  const int32_t* positions;
  const float2* table;  // [max_positions][rotary_dim / 2] (cos, sin)
  int64_t max_positions;
  int tokens, heads, head_dim, rotary_dim;
  int inverse;
  int head_splits;     // threads that share one (token, chunk): each takes heads hs, hs + head_splits, ...
  int tokens_per_cta;
};

// Both products and the sum are rounded one by one (no fused multiply-add): the value of a turned key
// is then the same in whatever form it is computed, and the 8-bit codes made from it are too.
__device__ __forceinline__ void rotary_turn(float& x1, float& x2, float c, float s) {
  const float y1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  const float y2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
  x1 = y1;
  x2 = y2;
}

__device__ __forceinline__ void unpack_bf16x8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack_bf16x8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}

// The 16 elements of one chunk of a head and where its two 8-element pieces start.
struct RotaryChunk {
  int off0, off1;  // element offsets of the two pieces within the head
  int pair0;       // first of the chunk's 8 pairs, or -1: past rotary_dim, copied
};

template <bool kInterleaved>
__device__ __forceinline__ RotaryChunk rotary_chunk(int chunk, int rotary_dim) {
  RotaryChunk c;
  if (16 * chunk >= rotary_dim) {
    c.off0 = 16 * chunk;
    c.off1 = c.off0 + 8;
    c.pair0 = -1;
  } else if (kInterleaved) {
    c.off0 = 16 * chunk;
    c.off1 = c.off0 + 8;
    c.pair0 = 8 * chunk;
  } else {
    c.off0 = 8 * chunk;
    c.off1 = c.off0 + (rotary_dim >> 1);
    c.pair0 = 8 * chunk;
  }
  return c;
}

// (The read-only path: no kernel of this library writes a table, and a grid that lets its successor start early is one
// of them, so a table is constant for as long as any CTA of its reader runs.)
__device__ __forceinline__ void rotary_load_table(const float2* row, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 t = __ldg(reinterpret_cast<const float4*>(row) + i);
    c[2 * i] = t.x;
    s[2 * i] = t.y;
    c[2 * i + 1] = t.z;
    s[2 * i + 1] = t.w;
  }
}

// a: elements off0..off0+7, b: off1..off1+7.
template <bool kInterleaved>
__device__ __forceinline__ void rotary_apply(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8]) {
  if (kInterleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      rotary_turn(a[2 * i], a[2 * i + 1], c[i], s[i]);
      rotary_turn(b[2 * i], b[2 * i + 1], c[4 + i], s[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) rotary_turn(a[i], b[i], c[i], s[i]);
  }
}

constexpr int kRotaryThreads = 128;

template <bool kInterleaved, int kHeads>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
  const unsigned chunks = static_cast<unsigned>(p.head_dim) >> 4;
  const unsigned columns = chunks * p.head_splits;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.tokens_per_cta;
  pdl_wait_previous_grid();
  pdl_allow_next_grid();
  for (unsigned i = threadIdx.x; i < columns * p.tokens_per_cta; i += kRotaryThreads) {
    const unsigned local = i / columns;
    const unsigned col = i - local * columns;
    const int64_t token = token0 + local;
    if (token >= p.tokens) break;
    const unsigned hs = col / chunks;
    const RotaryChunk ch = rotary_chunk<kInterleaved>(col - hs * chunks, p.rotary_dim);
    const int pos = p.positions[token];
    if (pos < 0) continue;  // no token: the row is left as it is
    if (pos >= p.max_positions) {
      record_status(kKernelRotary, 1, kReasonBadIndex);
      continue;
    }
    float c[8], s[8];
    if (ch.pair0 >= 0) {
      rotary_load_table(p.table + static_cast<int64_t>(pos) * (p.rotary_dim >> 1) + ch.pair0, c, s);
      if (p.inverse) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] = -s[k];
      }
    }
    const __nv_bfloat16* x = p.x + token * p.ld_x;
    __nv_bfloat16* y = p.out + token * p.ld_out;
    // kHeads heads at a time: all their loads, then all their stores (out may be x, so the compiler cannot move them).
    for (int h0 = hs; h0 < p.heads; h0 += kHeads * p.head_splits) {
      uint4 ua[kHeads], ub[kHeads];
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + k * p.head_splits;
        if (h < p.heads) {
          ua[k] = __ldcs(reinterpret_cast<const uint4*>(x + h * p.head_dim + ch.off0));
          ub[k] = __ldcs(reinterpret_cast<const uint4*>(x + h * p.head_dim + ch.off1));
        }
      }
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int h = h0 + k * p.head_splits;
        if (h < p.heads) {
          if (ch.pair0 >= 0) {
            float a[8], b[8];
            unpack_bf16x8(ua[k], a);
            unpack_bf16x8(ub[k], b);
            rotary_apply<kInterleaved>(a, b, c, s);
            ua[k] = pack_bf16x8(a);
            ub[k] = pack_bf16x8(b);
          }
          __stcs(reinterpret_cast<uint4*>(y + h * p.head_dim + ch.off0), ua[k]);
          __stcs(reinterpret_cast<uint4*>(y + h * p.head_dim + ch.off1), ub[k]);
        }
      }
    }
  }
}

static cudaError_t launch_rotary(RotaryParams p, int interleaved, int sm_count, cudaStream_t stream) {
  const int chunks = p.head_dim / 16;
  // Four heads to a thread, which then loads its part of the table once for the four, where that still leaves each SM
  // 2048 threads eight times over; else one, so that a small call has all its loads in flight at once.
  const int64_t work = static_cast<int64_t>(p.tokens) * p.heads * chunks;
  const bool four = p.heads >= 4 && work >= int64_t{4 * 8 * 2048} * sm_count;
  p.head_splits = four ? (p.heads + 3) / 4 : p.heads;
  const int columns = chunks * p.head_splits;
  p.tokens_per_cta = columns >= kRotaryThreads ? 1 : kRotaryThreads / columns;
  const unsigned blocks = static_cast<unsigned>((static_cast<int64_t>(p.tokens) + p.tokens_per_cta - 1) / p.tokens_per_cta);
  const dim3 grid(blocks), block(kRotaryThreads);
  if (four)
    return interleaved ? launch_pdl(rotary_kernel<true, 4>, grid, block, 0, stream, p)
                       : launch_pdl(rotary_kernel<false, 4>, grid, block, 0, stream, p);
  return interleaved ? launch_pdl(rotary_kernel<true, 1>, grid, block, 0, stream, p)
                     : launch_pdl(rotary_kernel<false, 1>, grid, block, 0, stream, p);
}

}  // namespace b2
