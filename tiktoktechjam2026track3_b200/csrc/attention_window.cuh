// Causal prompt attention with a sliding window and first tokens that stay visible (sinks): query i of a sequence of
// n tokens sees key j <= i iff window == 0 or i - j < window or j < sinks;
//   out_i = softmax(scale q_i k_j) v_j over the keys it sees,  0 for the rows i >= n of a padded batch.
// The reference's attention (models.py:55-75) is the case window == 0.
//
// Bound by the tensor cores and the exponential unit like attention_solo.cuh (head_dim 32, 64) and
// attention_wide.cuh (head_dim 128), whose pipelines these kernels keep: one tile of 128 query rows per CTA, scores and
// weights in tensor memory, keys and values by TMA. What differs is which keys a CTA goes through:
//   - The query heads of one key head share a tile: with a group of 2^k heads it holds 128 / 2^k tokens x 2^k heads
//     (a group that is not a power of two takes its largest power-of-two divisor). The band of keys that any row of the tile
//     sees is window + tokens - 1 long, so fewer tokens waste fewer masked scores, and each key is read once for 2^k heads.
//   - The tile's keys are a list of its own: the sinks (rounded up to 16), then the band from its first key on, cut
//     into tiles of 128 wherever that falls. The keys of a tile are rows [128 t, 128 t + 128) of the list; a tile
//     across the seam is loaded in boxes of 16 rows. A window thus costs ceil((sinks + window + tokens) / 128) tiles,
//     not one tile for the sinks and up to one more for the band's alignment. The last tile's products and
//     exponentials stop at its last key.
//   - In list places v, row i sees v <= d and (v >= c or v < a), with a = sinks, d the place of key i and c that of key
//     i - window + 1; only tiles where these cut are masked.
//   - Weights are rounded to bf16, the type of the values (one tcgen05.mma takes one type), sums and maxima are fp32 and take
//     them unrounded; at head_dim 128 one pair of exponentials in four is the polynomial of attention_wide.cuh. Measured over
//     whole outputs against 64 bits: 0.0019 to 0.0022 of the norm, 0.0016 of which is the output's own rounding.
//   - Values behind the band's last key are cleared in shared memory: a weight of zero does not remove a NaN there. Those
//     between the last sink and the next multiple of 16 come from a map that ends with the sinks: its rows behind read as zeros.
// Measured on one B200 (us a call back to back; floor, the larger of products at the measured GEMM rate and bytes at the copy
// rate, in brackets): 32768 tokens, 16 heads of 128 on 4 key heads, window 4096: 1000 to 1150 as the 1000 W limit lets it
// (627); 16 ragged sequences of up to 2048, 16 heads of 64, window 512: 153 (28); the same on 4 key heads, not ragged: 156
// (37); causal without a window, 16 x 2048 x 16 heads of 64: 248 (83; attention_solo_kernel 229), 8192 x 16 heads
// of 128: 270 (167; attention_wide_kernel 260). Per tile of 128 x 128 the exponential unit needs 1024 cycles at head_dim
// 64 and the issue of twelve products as many; a masked tile costs about half as much again as an open one,
// and of the six tiles of a window of 512 four are masked. The sinks' own maps cost 1 us of the 153, and 0.8 of 36 for
// 4 x 1000 tokens of 16 heads of 128.
#pragma once
#include <mutex>
#include <type_traits>

#include "b2_common.cuh"
#include "attention.cuh"

namespace b2 {

struct WindowParams {
  __nv_bfloat16* ctx;
  int64_t ld_ctx;
  const int32_t* kv_len;
  int B, S, heads, kv_heads;
  int group_shift;  // log2 of the query heads in a tile
  int tiles;        // query tiles of a sequence
  int window, sinks;  // window <= 0: none
  float scale_log2;
  int head_major;  // as in AttnParams
};

// Keys and values [B][S][kv_heads][head_dim] in boxes of 64 columns and 128 or 16 rows; Q in boxes of a query tile.
struct WindowMaps {
  CUtensorMap q, k, v, k16, v16;
  CUtensorMap v_sinks, v16_sinks;  // the sequence's first `sinks` rows only
};

// The list of keys of one query tile.
struct KeyList {
  int i0, i1;      // its tokens
  int lo;          // first key of the band
  int sink_rows;   // rows of the list in front of the band
  int rows, tiles;
};

__device__ __forceinline__ KeyList window_keys(const WindowParams& p, int tile, int len) {
  KeyList l;
  const int tokens = 128 >> p.group_shift;
  l.i0 = tile * tokens;
  l.i1 = min(l.i0 + tokens, len);
  l.lo = p.window > 0 ? max(0, l.i0 - p.window + 1) : 0;
  if (p.sinks >= l.lo) {
    l.lo = 0;  // the sinks reach the band: one piece
    l.sink_rows = 0;
  } else {
    l.sink_rows = (p.sinks + 15) & ~15;
  }
  l.rows = l.sink_rows + l.i1 - l.lo;
  l.tiles = (l.rows + 127) >> 7;
  return l;
}

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x, int32_t y,
                                            int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Tile t of the list, 64 columns from `col` on: one box, or eight across the seam. Every box counts its full bytes.
// `sinks`, `sinks16`: the maps for the part in front of the band.
__device__ __forceinline__ void window_load_tile(uint8_t* dst, const CUtensorMap* map, const CUtensorMap* map16,
                                                 const CUtensorMap* sinks, const CUtensorMap* sinks16, uint64_t* bar,
                                                 const KeyList& l, int t, int col, int head, int b) {
  const int v0 = 128 * t;
  if (v0 >= l.sink_rows) {
    tma_load_4d(dst, map, bar, col, head, l.lo + v0 - l.sink_rows, b);
    return;
  }
  if (v0 + 128 <= l.sink_rows) {
    tma_load_4d(dst, sinks, bar, col, head, v0, b);
    return;
  }
#pragma unroll 1
  for (int r = 0; r < 128; r += 16) {
    const int v = v0 + r;
    const bool sink = v < l.sink_rows;
    tma_load_4d(dst + r * 128, sink ? sinks16 : map16, bar, col, head, sink ? v : l.lo + v - l.sink_rows, b);
  }
}

// Which places of the list a row sees: v <= d and (v >= c or v < a).
struct RowKeys {
  int a, c, d;
};

__device__ __forceinline__ RowKeys window_row(const WindowParams& p, int lo, int sink_rows, int i) {
  RowKeys r;
  r.a = p.sinks;
  r.c = (p.window > 0 ? max(i - p.window + 1 - lo, 0) : 0) + sink_rows;
  r.d = i - lo + sink_rows;
  return r;
}

// What the softmax threads need to know of the list, kept in shared memory: their registers are all in use on the tiles
// that hide nothing.
struct WindowTiles {
  int i0, lo, sink_rows, rows, count;
  int open_a, open_c, open_d;  // tiles below open_d that lie from open_c on or below open_a hide no key from these rows
  __device__ __forceinline__ bool open(int t) const { return t < open_d && (t >= open_c || t < open_a); }
  __device__ __forceinline__ RowKeys row(const WindowParams& p, int i) const { return window_row(p, lo, sink_rows, i); }
};

// For the rows of tokens first ... last of the query tile.
__device__ __forceinline__ WindowTiles window_tiles(const WindowParams& p, const KeyList& l, int first, int last) {
  WindowTiles t;
  t.i0 = l.i0;
  t.count = l.tiles;
  t.lo = l.lo;
  t.sink_rows = l.sink_rows;
  t.rows = l.rows;
  t.open_a = p.sinks >> 7;
  t.open_c = (window_row(p, l.lo, l.sink_rows, last).c + 127) >> 7;
  t.open_d = min(window_row(p, l.lo, l.sink_rows, first).d + 1, l.rows) >> 7;
  return t;
}

// Bit k: whether a row sees place v0 + k.
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t window_bits(const RowKeys& r, int v0) {
  return low_bits(r.d + 1 - v0) & (~low_bits(r.c - v0) | low_bits(r.a - v0));
}
__device__ __forceinline__ void window_hide(float* v, uint32_t bits) {
#pragma unroll
  for (int k = 0; k < 32; ++k) v[k] = (bits >> k) & 1u ? v[k] : -INFINITY;
}

// Zeros for the rows of a query tile that lie behind the sequence's end.
template <int HD>
__device__ __forceinline__ void window_zero_rows(const WindowParams& p, int b, int head0, int i0) {
  const int group = 1 << p.group_shift;
  const int tokens = min(128 >> p.group_shift, p.S - i0);
  constexpr int kPieces = HD / 8;
  for (int i = threadIdx.x; i < tokens * group * kPieces; i += blockDim.x) {
    const int token = i / (group * kPieces);
    const int rest = i - token * (group * kPieces);
    uint4* dst = reinterpret_cast<uint4*>(p.ctx + (static_cast<int64_t>(b) * p.S + i0 + token) * p.ld_ctx + head0 * HD);
    dst[rest] = make_uint4(0, 0, 0, 0);
  }
}

// Clears rows [from, 128) of a value tile (128-byte rows, `boxes` boxes of 64 columns) and makes that visible to the
// tensor core; the threads of `warps` warps share it.
template <int kBoxes>
__device__ __forceinline__ void window_clear_values(uint8_t* tile, int from, int thread, int threads) {
  for (int i = from * 8 + thread; i < 128 * 8; i += threads) {
#pragma unroll
    for (int box = 0; box < kBoxes; ++box) reinterpret_cast<uint4*>(tile + box * 128 * 128)[i] = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void window_cta(const WindowParams& p, int& b, int& head0, int& tile) {
  const int bh = static_cast<int>(p.head_major ? blockIdx.y : blockIdx.x);
  const int row = static_cast<int>(p.head_major ? blockIdx.x : blockIdx.y);
  const int groups = p.heads >> p.group_shift;
  b = bh / groups;
  head0 = (bh - b * groups) << p.group_shift;
  tile = p.tiles - 1 - row;  // the longest lists first
}

// ---------------------------------------------------------------------------------------------
// head_dim 32 and 64: the pipeline of attention_solo_kernel (two CTAs per SM). head_dim 32 is loaded in 64-column boxes
// whose second half lies outside the head and reads as zeros.
// ---------------------------------------------------------------------------------------------
template <int HD>
__global__ void __launch_bounds__(192, 2)
    window_solo_kernel(const __grid_constant__ WindowMaps maps, const WindowParams p) {
  static_assert(HD == 32 || HD == 64, "head_dim 32 or 64");
  constexpr int kTileBytes = 128 * 128;
  constexpr int kStages = 2;
  constexpr int kON = 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  uint8_t* s_k = s_q + kTileBytes;
  uint8_t* s_v = s_k + kStages * kTileBytes;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_v + kStages * kTileBytes);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;
  uint64_t* p_full = s_full + 1;
  uint64_t* o_full = p_full + 1;
  uint64_t* s_free = o_full + 1;
  uint64_t* drain = s_free + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  WindowTiles* s_tiles = reinterpret_cast<WindowTiles*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int b, head0, tile;
  window_cta(p, b, head0, tile);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(p_full, 4);
    mbar_init(o_full, 1);
    mbar_init(s_free, 4);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  pdl_wait_previous_grid();
  pdl_allow_next_grid();
  const int len = p.kv_len != nullptr ? min(max(p.kv_len[b], 0), p.S) : p.S;
  const KeyList keys = window_keys(p, tile, len);
  if (keys.i0 >= len) {  // uniform for the CTA; no tensor memory allocated yet
    window_zero_rows<HD>(p, b, head0, keys.i0);
    return;
  }
  const int n = keys.tiles;
  const int last_rows = keys.rows - 128 * (n - 1);  // of the last tile
  if (warp >= 2 && lane == 0) {
    const int r0 = (warp & 3) * 32;
    s_tiles[warp & 3] = window_tiles(p, keys, keys.i0 + (r0 >> p.group_shift), keys.i0 + ((r0 + 31) >> p.group_shift));
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      const int kv_head = head0 / (p.heads / p.kv_heads);
      mbar_arrive_expect_tx(q_full, kTileBytes);
      tma_load_4d(s_q, &maps.q, q_full, 0, head0, keys.i0, b);
      int k_next = 0, v_next = 0;
      bool ok = true;
      PollTimeout poll;
      poll.reset();
      while (k_next < n || v_next < n) {
        bool progress = false;
        if (k_next < n && mbar_test_wait(&k_empty[k_next % kStages], ((k_next / kStages) & 1) ^ 1u)) {
          const int st = k_next % kStages;
          mbar_arrive_expect_tx(&k_full[st], kTileBytes);
          window_load_tile(s_k + st * kTileBytes, &maps.k, &maps.k16, &maps.k, &maps.k16, &k_full[st], keys, k_next, 0, kv_head, b);
          ++k_next;
          progress = true;
        }
        if (v_next < n && mbar_test_wait(&v_empty[v_next % kStages], ((v_next / kStages) & 1) ^ 1u)) {
          const int st = v_next % kStages;
          mbar_arrive_expect_tx(&v_full[st], kTileBytes);
          window_load_tile(s_v + st * kTileBytes, &maps.v, &maps.v16, &maps.v_sinks, &maps.v16_sinks, &v_full[st], keys, v_next, 0, kv_head, b);
          ++v_next;
          progress = true;
        }
        if (progress) {
          poll.reset();
        } else if (*abort_flag) {
          ok = false;
          break;
        } else if (poll.expired()) {
          record_status(kKernelAttention, 101, kReasonTimeout);
          *abort_flag = 1;
          ok = false;
          break;
        }
      }
      if (!ok) {
        // Let copies in flight land: Q and the last (up to kStages) K and V tiles.
        const uint64_t t0 = global_timer_ns();
        const uint64_t lim = wait_limit_ns();
        auto drain_wait = [&](uint64_t* bar, uint32_t par) {
          while (!mbar_try_wait(bar, par) && global_timer_ns() - t0 < lim) {
          }
        };
        drain_wait(q_full, 0);
        for (int j = k_next - 1; j >= 0 && j >= k_next - kStages; --j)
          drain_wait(&k_full[j % kStages], (j / kStages) & 1);
        for (int j = v_next - 1; j >= 0 && j >= v_next - kStages; --j)
          drain_wait(&v_full[j % kStages], (j / kStages) & 1);
      }
    }
  } else if (warp == 1) {
    // ---------------- UMMA issuer ----------------
    if (lane == 0) {
      const uint32_t idesc_last = make_idesc_bf16_f32(128, static_cast<uint32_t>((last_rows + 15) & ~15), 0, 0);
      constexpr uint32_t idesc_s = make_idesc_bf16_f32(128, 128, 0, 0);
      constexpr uint32_t idesc_o = make_idesc_bf16_f32(128, kON, 0, 1);
      const uint32_t q_addr = smem_u32(s_q);
      const uint32_t d_s = tmem_base;
      const uint32_t a_p = tmem_base + 128;
      const uint32_t d_o = tmem_base + 192;
      auto issue_s = [&](int j) {
        const uint32_t k_addr = smem_u32(s_k + (j % kStages) * kTileBytes);
        const uint32_t idesc = j == n - 1 ? idesc_last : idesc_s;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          umma_bf16_ss(d_s, make_sdesc_sw128(q_addr + kk * 32, 16, 1024), make_sdesc_sw128(k_addr + kk * 32, 16, 1024),
                       idesc, kk > 0 ? 1u : 0u);
        umma_commit(s_full);
        umma_commit(&k_empty[j % kStages]);
      };
      auto issue_o = [&](int j) {
        const int vst = j % kStages;
        const uint32_t v_addr = smem_u32(s_v + vst * kTileBytes);
        const int steps = j == n - 1 ? (last_rows + 15) >> 4 : 8;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          if (kk < steps)
            umma_bf16_ts(d_o, a_p + kk * 8, make_sdesc_sw128(v_addr + kk * 2048, kTileBytes, 1024), idesc_o,
                         (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(o_full);
        umma_commit(&v_empty[vst]);
      };
      auto wait_pv = [&](int j) {
        return mbar_wait(p_full, j & 1, abort_flag, kKernelAttention, 106) &&
               mbar_wait(&v_full[j % kStages], (j / kStages) & 1, abort_flag, kKernelAttention, 107);
      };
      bool ok = mbar_wait(q_full, 0, abort_flag, kKernelAttention, 103);
      for (int j = 0; j < n && ok; ++j) {
        if (!mbar_wait(&k_full[j % kStages], (j / kStages) & 1, abort_flag, kKernelAttention, 104) ||
            (j > 0 && !mbar_wait(s_free, (j - 1) & 1, abort_flag, kKernelAttention, 105))) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        issue_s(j);
        if (j > 0) {
          if (!wait_pv(j - 1)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          issue_o(j - 1);
        }
      }
      if (ok && wait_pv(n - 1)) {
        tc_fence_after_sync();
        issue_o(n - 1);
      }
      umma_commit(drain);
      const uint64_t t0 = global_timer_ns();
      const uint64_t lim = wait_limit_ns();
      while (!mbar_try_wait(drain, 0) && global_timer_ns() - t0 < lim) {
      }
    }
  } else {
    // ---------------- softmax: one row per thread ----------------
    s_tiles += warp & 3;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane;
    const uint32_t t_p = t_lane + 128;
    const uint32_t t_o = t_lane + 192;
    const float c = p.scale_log2;
    constexpr float kRescaleThreshold = 8.0f;

    float m_ref = -INFINITY;  // reference maximum, -inf until the row has seen a key
    float l_sum = 0.f;
    bool alive = true;

#pragma unroll 1
    for (int j = 0; j < s_tiles->count; ++j) {
      float alpha = 1.f;
      softmax_wait(s_full, j & 1, 108, alive, abort_flag);
      tc_fence_after_sync();
      auto new_reference = [&](float rmax) {
        if (m_ref == -INFINITY) {
          m_ref = rmax;  // nothing accumulated so far: nothing to rescale
        } else if ((rmax - m_ref) * c > kRescaleThreshold) {
          alpha = fast_exp2((m_ref - rmax) * c);
          m_ref = rmax;
        }
      };
      auto whole_tile = [&](auto hide) {
        // The scores once into registers, S free for the next product meanwhile.
        float v[128];
        tmem_load_128cols(t_s, v);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        if constexpr (decltype(hide)::value) {
          const RowKeys row = s_tiles->row(p, s_tiles->i0 + (r >> p.group_shift));
#pragma unroll
          for (int g = 0; g < 4; ++g) window_hide(v + 32 * g, window_bits(row, 128 * j + 32 * g));
        }
        new_reference(fmaxf(fmaxf(max32(v), max32(v + 32)), fmaxf(max32(v + 64), max32(v + 96))));
        const uint64_t c2 = splat2(c);
        const uint64_t neg_mc2 = splat2(decltype(hide)::value && m_ref == -INFINITY ? 0.f : -m_ref * c);
        uint64_t sum2 = 0;
        uint32_t w[64];
#pragma unroll
        for (int k = 0; k < 64; ++k) {
          float x0 = v[2 * k], x1 = v[2 * k + 1];
          fma2_inplace(x0, x1, c2, neg_mc2);
          const float e0 = fast_exp2(x0);
          const float e1 = fast_exp2(x1);
          sum2 = add2f(sum2, pack2f(e0, e1));
          w[k] = pack_bf16x2(e0, e1);
        }
        float sum0, sum1;
        unpack2f(sum2, sum0, sum1);
        l_sum = l_sum * alpha + (sum0 + sum1);
        if (j > 0) {
          softmax_wait(o_full, (j - 1) & 1, 109, alive, abort_flag);
          tc_fence_after_sync();
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) tmem_store_16cols_async(t_p + 16 * g, w + 16 * g);
      };
      if (s_tiles->open(j)) {
        whole_tile(std::false_type{});
      } else if (s_tiles->rows - 128 * j > 96) {
        whole_tile(std::true_type{});
      } else {
        // Some row does not see some place: 32 places at a time, as far as there are keys, the scores read twice (maximum,
        // then weights), so that the masks cost no registers that the other path needs.
        const RowKeys row = s_tiles->row(p, s_tiles->i0 + (r >> p.group_shift));
        const int groups = (min(128, s_tiles->rows - 128 * j) + 31) >> 5;
        float rmax = -INFINITY;
#pragma unroll 1
        for (int g = 0; g < groups; ++g) {
          float v[32];
          tmem_load_32cols(t_s + 32 * g, v);
          window_hide(v, window_bits(row, 128 * j + 32 * g));
          rmax = fmaxf(rmax, max32(v));
        }
        new_reference(rmax);
        if (j > 0) {
          softmax_wait(o_full, (j - 1) & 1, 109, alive, abort_flag);
          tc_fence_after_sync();
        }
        const uint64_t c2 = splat2(c);
        const uint64_t neg_mc2 = splat2(m_ref == -INFINITY ? 0.f : -m_ref * c);
        uint64_t sum2 = 0;
#pragma unroll 1
        for (int g = 0; g < groups; ++g) {
          float v[32];
          uint32_t w[16];
          tmem_load_32cols(t_s + 32 * g, v);
          window_hide(v, window_bits(row, 128 * j + 32 * g));
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float x0 = v[2 * k], x1 = v[2 * k + 1];
            fma2_inplace(x0, x1, c2, neg_mc2);
            const float e0 = fast_exp2(x0);
            const float e1 = fast_exp2(x1);
            sum2 = add2f(sum2, pack2f(e0, e1));
            w[k] = pack_bf16x2(e0, e1);
          }
          tmem_store_16cols_async(t_p + 16 * g, w);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        float sum0, sum1;
        unpack2f(sum2, sum0, sum1);
        l_sum = l_sum * alpha + (sum0 + sum1);
      }
      tmem_wait_st();
      if (__any_sync(0xffffffffu, alpha < 1.f)) {
#pragma unroll 1
        for (int cc = 0; cc < kON / 32; ++cc) {
          float o[32];
          tmem_load_32cols(t_o + cc * 32, o);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] *= alpha;
          tmem_store_32cols(t_o + cc * 32, o);
        }
      }
      // Products stop at the next multiple of 16 rows. (O += P(j-1) V has completed, so the stage's barrier is in this
      // tile's phase.)
      if (const int last_rows = s_tiles->rows - 128 * j; last_rows < 128 && (last_rows & 15) != 0) {
        softmax_wait(&v_full[j % kStages], (j / kStages) & 1, 111, alive, abort_flag);
        window_clear_values<1>(s_v + (j % kStages) * kTileBytes, last_rows, threadIdx.x - 64, 128);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }

    softmax_wait(o_full, (s_tiles->count - 1) & 1, 110, alive, abort_flag);
    tc_fence_after_sync();
    const int token = s_tiles->i0 + (r >> p.group_shift);
    const float inv = token < len && l_sum != 0.f ? 1.0f / l_sum : 0.f;
    const int head = head0 + (r & ((1 << p.group_shift) - 1));
    uint4* dst = reinterpret_cast<uint4*>(p.ctx + (static_cast<int64_t>(b) * p.S + token) * p.ld_ctx + head * HD);
#pragma unroll
    for (int cc = 0; cc < HD / 32; ++cc) {
      float o[32];
      tmem_load_32cols(t_o + 32 * cc, o);
      if (token < p.S) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = token < len ? o[k] * inv : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          dst[4 * cc + k] = make_uint4(pack_bf16x2(o[8 * k], o[8 * k + 1]), pack_bf16x2(o[8 * k + 2], o[8 * k + 3]),
                                       pack_bf16x2(o[8 * k + 4], o[8 * k + 5]), pack_bf16x2(o[8 * k + 6], o[8 * k + 7]));
      }
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 256);
  }
}

// ---------------------------------------------------------------------------------------------
// head_dim 128: the pipeline of attention_wide_kernel (one CTA per SM, three score buffers, two issuers).
// ---------------------------------------------------------------------------------------------
struct WindowWideCfg {
  static constexpr int kSoftmaxWarps = 8;
  static constexpr int kPvWarp = 2 + kSoftmaxWarps;
  static constexpr int kThreads = 32 * (kPvWarp + 1);
  static constexpr int kBoxBytes = 128 * 128;
  static constexpr int kTileBytes = 2 * kBoxBytes;
  static constexpr int kStages = 3;
  static constexpr int kVStages = 2;
  static constexpr int kBufs = 3;
  static constexpr int kOffK = kTileBytes;
  static constexpr int kOffV = kOffK + kStages * kTileBytes;
  static constexpr int kOffRed = kOffV + kVStages * kTileBytes;
  static constexpr int kOffBar = kOffRed + 3 * 2 * 128 * 4;
  static constexpr int kSmemBytes = kOffBar + 256 + 1024;
  static constexpr int kOCol = kBufs * 128;
  static constexpr int kPolyPairs = 0x1;  // as in AttnWideCfg
};

__global__ void __launch_bounds__(WindowWideCfg::kThreads, 1)
    window_wide_kernel(const __grid_constant__ WindowMaps maps, const WindowParams p) {
  using Cfg = WindowWideCfg;
  constexpr int HD = 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  uint8_t* s_k = smem + Cfg::kOffK;
  uint8_t* s_v = smem + Cfg::kOffV;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + Cfg::kStages;
  uint64_t* v_full = k_empty + Cfg::kStages;
  uint64_t* v_empty = v_full + Cfg::kVStages;
  uint64_t* s_full = v_empty + Cfg::kVStages;
  uint64_t* p_full = s_full + Cfg::kBufs;
  uint64_t* o_done = p_full + Cfg::kBufs;
  uint64_t* drain = o_done + Cfg::kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  int b, head0, tile;
  window_cta(p, b, head0, tile);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < Cfg::kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < Cfg::kVStages; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < Cfg::kBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], Cfg::kSoftmaxWarps);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 2);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  pdl_wait_previous_grid();
  pdl_allow_next_grid();
  const int len = p.kv_len != nullptr ? min(max(p.kv_len[b], 0), p.S) : p.S;
  const KeyList keys = window_keys(p, tile, len);
  if (keys.i0 >= len) {  // uniform for the CTA; no tensor memory allocated yet
    window_zero_rows<HD>(p, b, head0, keys.i0);
    return;
  }
  const int n = keys.tiles;
  const int last_rows = keys.rows - 128 * (n - 1);
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      const int kv_head = head0 / (p.heads / p.kv_heads);
      mbar_arrive_expect_tx(q_full, Cfg::kTileBytes);
      tma_load_4d(s_q, &maps.q, q_full, 0, head0, keys.i0, b);
      tma_load_4d(s_q + Cfg::kBoxBytes, &maps.q, q_full, 64, head0, keys.i0, b);
      int k_next = 0, v_next = 0;
      bool ok = true;
      PollTimeout poll;
      poll.reset();
      while (k_next < n || v_next < n) {
        bool progress = false;
        if (k_next < n && mbar_test_wait(&k_empty[k_next % Cfg::kStages], ((k_next / Cfg::kStages) & 1) ^ 1u)) {
          const int st = k_next % Cfg::kStages;
          uint8_t* dst = s_k + st * Cfg::kTileBytes;
          mbar_arrive_expect_tx(&k_full[st], Cfg::kTileBytes);
          window_load_tile(dst, &maps.k, &maps.k16, &maps.k, &maps.k16, &k_full[st], keys, k_next, 0, kv_head, b);
          window_load_tile(dst + Cfg::kBoxBytes, &maps.k, &maps.k16, &maps.k, &maps.k16, &k_full[st], keys, k_next, 64, kv_head, b);
          ++k_next;
          progress = true;
        }
        if (v_next < n && mbar_test_wait(&v_empty[v_next % Cfg::kVStages], ((v_next / Cfg::kVStages) & 1) ^ 1u)) {
          const int st = v_next % Cfg::kVStages;
          uint8_t* dst = s_v + st * Cfg::kTileBytes;
          mbar_arrive_expect_tx(&v_full[st], Cfg::kTileBytes);
          window_load_tile(dst, &maps.v, &maps.v16, &maps.v_sinks, &maps.v16_sinks, &v_full[st], keys, v_next, 0, kv_head, b);
          window_load_tile(dst + Cfg::kBoxBytes, &maps.v, &maps.v16, &maps.v_sinks, &maps.v16_sinks, &v_full[st], keys, v_next, 64, kv_head, b);
          ++v_next;
          progress = true;
        }
        if (progress) {
          poll.reset();
        } else if (*abort_flag) {
          ok = false;
          break;
        } else if (poll.expired()) {
          record_status(kKernelAttention, 121, kReasonTimeout);
          *abort_flag = 1;
          ok = false;
          break;
        }
      }
      if (!ok) {
        // Let copies in flight land: Q and the last K and V tiles of the rings.
        const uint64_t t0 = global_timer_ns();
        const uint64_t lim = wait_limit_ns();
        auto drain_wait = [&](uint64_t* bar, uint32_t par) {
          while (!mbar_try_wait(bar, par) && global_timer_ns() - t0 < lim) {
          }
        };
        drain_wait(q_full, 0);
        for (int j = k_next - 1; j >= 0 && j >= k_next - Cfg::kStages; --j)
          drain_wait(&k_full[j % Cfg::kStages], (j / Cfg::kStages) & 1);
        for (int j = v_next - 1; j >= 0 && j >= v_next - Cfg::kVStages; --j)
          drain_wait(&v_full[j % Cfg::kVStages], (j / Cfg::kVStages) & 1);
      }
    }
  } else if (warp == 1 || warp == Cfg::kPvWarp) {
    // ---------------- UMMA issuers: warp 1 S = Q K^T, warp kPvWarp O += P V ----------------
    if (lane == 0) {
      bool ok = true;
      if (warp == 1) {
        const uint32_t idesc_last = make_idesc_bf16_f32(128, static_cast<uint32_t>((last_rows + 15) & ~15), 0, 0);
        constexpr uint32_t idesc_s = make_idesc_bf16_f32(128, 128, 0, 0);
        const uint32_t q_addr = smem_u32(s_q);
        ok = mbar_wait(q_full, 0, abort_flag, kKernelAttention, 125);
        for (int j = 0; j < n && ok; ++j) {
          const int st = j % Cfg::kStages;
          // The buffer's last reader, O += P(j-3) V, must have completed.
          if (j >= Cfg::kBufs)
            ok = mbar_wait(&o_done[j % Cfg::kBufs], ((j / Cfg::kBufs) - 1) & 1, abort_flag, kKernelAttention, 129);
          if (!ok || !mbar_wait(&k_full[st], (j / Cfg::kStages) & 1, abort_flag, kKernelAttention, 122)) break;
          tc_fence_after_sync();
          const uint32_t k_addr = smem_u32(s_k + st * Cfg::kTileBytes);
          const uint32_t d_s = tmem_base + (j % Cfg::kBufs) * 128;
          const uint32_t idesc = j == n - 1 ? idesc_last : idesc_s;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t off = (kk >> 2) * Cfg::kBoxBytes + (kk & 3) * 32;
            umma_bf16_ss(d_s, make_sdesc_sw128(q_addr + off, 16, 1024), make_sdesc_sw128(k_addr + off, 16, 1024), idesc,
                         kk > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[j % Cfg::kBufs]);
          umma_commit(&k_empty[st]);
        }
      } else {
        constexpr uint32_t idesc_o = make_idesc_bf16_f32(128, HD, 0, 1);
        const uint32_t d_o = tmem_base + Cfg::kOCol;
        for (int j = 0; j < n && ok; ++j) {
          const int st = j % Cfg::kVStages;
          const int buf = j % Cfg::kBufs;
          if (!mbar_wait(&p_full[buf], (j / Cfg::kBufs) & 1, abort_flag, kKernelAttention, 123) ||
              !mbar_wait(&v_full[st], (j / Cfg::kVStages) & 1, abort_flag, kKernelAttention, 124)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t v_addr = smem_u32(s_v + st * Cfg::kTileBytes);
          const uint32_t a_p = tmem_base + buf * 128;
          const int steps = j == n - 1 ? (last_rows + 15) >> 4 : 8;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            if (kk < steps)
              umma_bf16_ts(d_o, a_p + kk * 8, make_sdesc_sw128(v_addr + kk * 2048, Cfg::kBoxBytes, 1024), idesc_o,
                           (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&o_done[buf]);
          umma_commit(&v_empty[st]);
        }
      }
      umma_commit(drain);
      const uint64_t t0 = global_timer_ns();
      const uint64_t lim = wait_limit_ns();
      while (!mbar_try_wait(drain, 0) && global_timer_ns() - t0 < lim) {
      }
    }
  } else {
    // ---------------- softmax: two warps per row quadrant, 64 keys of a tile each ----------------
    const int quad = warp & 3;
    const int half = (warp - 2) >> 2;
    const int r = quad * 32 + lane;
    const int token = keys.i0 + (r >> p.group_shift);
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t t_o = t_lane + Cfg::kOCol + 64 * half;
    float* red = reinterpret_cast<float*>(smem + Cfg::kOffRed);
    const uint32_t pair_bar = 1 + quad;
    const float c = p.scale_log2;
    const WindowTiles tiles = window_tiles(p, keys, keys.i0 + ((quad * 32) >> p.group_shift),
                                           keys.i0 + ((quad * 32 + 31) >> p.group_shift));
    constexpr float kRescaleThreshold = 8.0f;

    float m_ref = -INFINITY;
    float l_sum = 0.f;
    bool alive = true;

    // One tile; `hide`: some row does not see some place of it.
    auto softmax_tile = [&](int j, auto hide) {
      const int buf = j % Cfg::kBufs;
      const uint32_t t_s = t_lane + buf * 128;
      float alpha = 1.f;
      softmax_wait(&s_full[buf], (j / Cfg::kBufs) & 1, 126, alive, abort_flag);
      tc_fence_after_sync();
      float v[64];
      tmem_load_64cols(t_s + 64 * half, v);
      if constexpr (decltype(hide)::value) {
        const RowKeys row = tiles.row(p, token);
#pragma unroll
        for (int g = 0; g < 2; ++g) window_hide(v + 32 * g, window_bits(row, 128 * j + 64 * half + 32 * g));
      }
      // Row maximum over both halves; after the barrier both warps have loaded their scores, so P may be written over
      // the buffer's first 64 columns (slots alternate by tile).
      float* slot = red + (j & 1) * 256;
      slot[half * 128 + r] = fmaxf(max32(v), max32(v + 32));
      named_barrier_sync(pair_bar, 64);
      const float rmax = fmaxf(slot[r], slot[128 + r]);
      if (m_ref == -INFINITY) {
        m_ref = rmax;  // nothing accumulated so far: nothing to rescale
      } else if ((rmax - m_ref) * c > kRescaleThreshold) {
        alpha = fast_exp2((m_ref - rmax) * c);
        m_ref = rmax;
      }
      const uint64_t c2 = splat2(c);
      const uint64_t neg_mc2 = splat2(m_ref == -INFINITY ? 0.f : -m_ref * c);
      uint64_t sum2 = 0;
      uint32_t w[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        float x0 = v[2 * k], x1 = v[2 * k + 1];
        fma2_inplace(x0, x1, c2, neg_mc2);
        float e0, e1;
        if ((Cfg::kPolyPairs >> (k & 3)) & 1) {
          exp2_poly_x2(x0, x1, e0, e1);
        } else {
          e0 = fast_exp2(x0);
          e1 = fast_exp2(x1);
        }
        sum2 = add2f(sum2, pack2f(e0, e1));
        w[k] = pack_bf16x2(e0, e1);
      }
      float sum0, sum1;
      unpack2f(sum2, sum0, sum1);
      l_sum = l_sum * alpha + (sum0 + sum1);
#pragma unroll
      for (int g = 0; g < 2; ++g) tmem_store_16cols_async(t_s + 32 * half + 16 * g, w + 16 * g);
      tmem_wait_st();
      if (__any_sync(0xffffffffu, alpha < 1.f)) {
        const int jp = j - 1;
        softmax_wait(&o_done[jp % Cfg::kBufs], (jp / Cfg::kBufs) & 1, 127, alive, abort_flag);
        tc_fence_after_sync();
#pragma unroll 1
        for (int cc = 0; cc < 2; ++cc) {
          float o[32];
          tmem_load_32cols(t_o + cc * 32, o);
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] *= alpha;
          tmem_store_32cols(t_o + cc * 32, o);
        }
      }
      if constexpr (decltype(hide)::value) {
        if (j == n - 1 && (last_rows & 15) != 0) {
          const int st = j % Cfg::kVStages;
          // First O += P(j-2) V, the stage's last reader: its barrier is then in this tile's phase.
          const int jv = j - Cfg::kVStages;
          if (jv >= 0) softmax_wait(&o_done[jv % Cfg::kBufs], (jv / Cfg::kBufs) & 1, 132, alive, abort_flag);
          softmax_wait(&v_full[st], (j / Cfg::kVStages) & 1, 131, alive, abort_flag);
          window_clear_values<2>(s_v + st * Cfg::kTileBytes, last_rows, threadIdx.x - 64, 256);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf]);
    };
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      if (tiles.open(j))
        softmax_tile(j, std::false_type{});
      else
        softmax_tile(j, std::true_type{});
    }

    red[2 * 256 + half * 128 + r] = l_sum;
    named_barrier_sync(pair_bar, 64);
    const float l_row = l_sum + red[2 * 256 + (1 - half) * 128 + r];
    softmax_wait(&o_done[(n - 1) % Cfg::kBufs], ((n - 1) / Cfg::kBufs) & 1, 128, alive, abort_flag);
    tc_fence_after_sync();
    const float inv = l_row != 0.f ? 1.0f / l_row : 0.f;
    const int head = head0 + (r & ((1 << p.group_shift) - 1));
    uint4* dst =
        reinterpret_cast<uint4*>(p.ctx + (static_cast<int64_t>(b) * p.S + token) * p.ld_ctx + head * HD + 64 * half);
#pragma unroll
    for (int cc = 0; cc < 2; ++cc) {
      float o[32];
      tmem_load_32cols(t_o + 32 * cc, o);
      if (token < p.S) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = token < len ? o[k] * inv : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          dst[4 * cc + k] = make_uint4(pack_bf16x2(o[8 * k], o[8 * k + 1]), pack_bf16x2(o[8 * k + 2], o[8 * k + 3]),
                                       pack_bf16x2(o[8 * k + 4], o[8 * k + 5]), pack_bf16x2(o[8 * k + 6], o[8 * k + 7]));
      }
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
cudaError_t make_tmap_bf16_4d(CUtensorMap* map, const void* base, const uint64_t (&dims)[4], const uint64_t (&strides)[3],
                              const uint32_t (&box)[4]);

template <typename Kernel>
static cudaError_t launch_window(Kernel kernel, int threads, int smem, std::once_flag (&once)[64], const WindowMaps& maps,
                                 const WindowParams& p, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63],
                 [&] { e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (e != cudaSuccess) return e;
  const unsigned bh = static_cast<unsigned>(p.B) * static_cast<unsigned>(p.heads >> p.group_shift);
  const unsigned rows = static_cast<unsigned>(p.tiles);
  return launch_pdl(kernel, p.head_major ? dim3(rows, bh) : dim3(bh, rows), dim3(threads), smem, stream, maps, p);
}

static cudaError_t launch_window_attention(const __nv_bfloat16* q, int64_t ld_q, const __nv_bfloat16* k, int64_t ld_k,
                                           const __nv_bfloat16* v, int64_t ld_v, int64_t hd, WindowParams p,
                                           cudaStream_t stream) {
  const int group = p.heads / p.kv_heads;
  p.group_shift = 0;
  while (p.group_shift < 4 && group % (2 << p.group_shift) == 0) ++p.group_shift;
  const uint32_t tokens = 128u >> p.group_shift;
  p.tiles = static_cast<int>((p.S + tokens - 1) / tokens);
  const int64_t bh = static_cast<int64_t>(p.B) * (p.heads >> p.group_shift);
  p.head_major = (p.S >= 16384 && bh <= 65535) || p.tiles > 65535;
  if (p.head_major && bh > 65535) return cudaErrorInvalidConfiguration;
  WindowMaps maps;
  const uint64_t h = static_cast<uint64_t>(hd), S = static_cast<uint64_t>(p.S), B = static_cast<uint64_t>(p.B);
  auto make = [&](CUtensorMap* m, const __nv_bfloat16* base, int64_t ld, int heads, uint32_t box_heads, uint32_t box_rows,
                  uint64_t rows) {
    const uint64_t row = static_cast<uint64_t>(ld) * 2;
    const uint64_t dims[4] = {h, static_cast<uint64_t>(heads), rows, B};
    const uint64_t strides[3] = {h * 2, row, row * S};
    const uint32_t box[4] = {64, box_heads, box_rows, 1};
    return make_tmap_bf16_4d(m, base, dims, strides, box);
  };
  const uint64_t sinks = p.sinks > 0 ? static_cast<uint64_t>(p.sinks) : 1;
  cudaError_t e = make(&maps.q, q, ld_q, p.heads, 1u << p.group_shift, tokens, S);
  if (e == cudaSuccess) e = make(&maps.k, k, ld_k, p.kv_heads, 1, 128, S);
  if (e == cudaSuccess) e = make(&maps.v, v, ld_v, p.kv_heads, 1, 128, S);
  if (e == cudaSuccess) e = make(&maps.k16, k, ld_k, p.kv_heads, 1, 16, S);
  if (e == cudaSuccess) e = make(&maps.v16, v, ld_v, p.kv_heads, 1, 16, S);
  if (e == cudaSuccess) e = make(&maps.v_sinks, v, ld_v, p.kv_heads, 1, 128, sinks);
  if (e == cudaSuccess) e = make(&maps.v16_sinks, v, ld_v, p.kv_heads, 1, 16, sinks);
  if (e != cudaSuccess) return e;
  static std::once_flag once32[64], once64[64], once128[64];
  constexpr int kSoloSmem = 5 * 128 * 128 + 256 + 1024;
  switch (hd) {
    case 32:
      return launch_window(window_solo_kernel<32>, 192, kSoloSmem, once32, maps, p, stream);
    case 64:
      return launch_window(window_solo_kernel<64>, 192, kSoloSmem, once64, maps, p, stream);
    case 128:
      return launch_window(window_wide_kernel, WindowWideCfg::kThreads, WindowWideCfg::kSmemBytes, once128, maps, p, stream);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace b2
