// C-ABI entry points of libb200tx.so (declared in include/b200tx.h).
//
// Conventions (the same ones the reference's ctypes cuBLASLt binding and its torch-extension
// kernels follow: transformer_benchmark/cublaslt_linear.py:63-145 maps an integer status to an
// exception; case6_exact_attention.cu:324-379 checks preconditions, launches on the caller's
// stream and checks the launch):
//   * every entry point returns int (B2_OK = 0) and takes the cudaStream_t last, as void*;
//   * pointers are device pointers the caller owns; the library allocates no device memory and
//     never synchronises the stream;
//   * on failure, b2_last_error() returns a message for the calling thread.
#include <cudaTypedefs.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <string>

#include "../../include/b200tx.h"
#include "b2_common.cuh"
#include "layernorm.cuh"
#include "gemm.cuh"
#include "attention.cuh"
#include "attention_solo.cuh"
#include "attention_wide.cuh"
#include "attention_simt.cuh"
#include "peer.cuh"
#include "mask.cuh"
#include "rotary.cuh"
#include "cache_append.cuh"
#include "cache_attention.cuh"
#include "cache_int4.cuh"
#include "attention_window.cuh"

#define B2_API extern "C" __attribute__((visibility("default")))

namespace b2 {


static thread_local char g_last_error[512] = "";

static int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

static int check_launch(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return 0;
  return fail(3, "%s: CUDA error %d (%s)", what, static_cast<int>(e), cudaGetErrorString(e));
}

static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

cudaError_t make_tmap_bf16_2d(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer,
                              uint64_t row_stride_bytes, uint32_t box_inner, uint32_t box_outer) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return cudaErrorNotSupported;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {row_stride_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t make_tmap_bf16_4d(CUtensorMap* map, const void* base, const uint64_t (&dims)[4], const uint64_t (&strides)[3],
                              const uint32_t (&box)[4]) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return cudaErrorNotSupported;
  cuuint64_t d[4], s[3];
  cuuint32_t x[4], one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 4; ++i) {
    d[i] = dims[i];
    x[i] = box[i];
    if (i < 3) s[i] = strides[i];
  }
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), d, s, x, one,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

int device_sm_count(int device) {
  static int cache[64] = {0};
  int& c = cache[device & 63];
  if (c == 0) {
    int v = 0;
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, device);
    c = v > 0 ? v : 148;
  }
  return c;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static bool is_sm100(int* major_out) {
  static int cache[64] = {0};  // 10 * major + minor by device, as device_sm_count keeps its answer
  int dev = 0, major = 0, minor = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  int& c = cache[dev & 63];
  if (c == 0) {
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    c = major * 10 + minor;
  }
  if (major_out) *major_out = c;
  return c == 100;
}

}  // namespace b2

using namespace b2;

B2_API int b2_abi_version(void) { return 1; }

B2_API const char* b2_last_error(void) { return g_last_error; }

B2_API int b2_device_status(uint32_t* out_status, int clear) {
  if (out_status == nullptr) return fail(1, "b2_device_status: out_status is null");
  uint32_t v = 0, index = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_device_status, sizeof(v));
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&index, g_index_status, sizeof(index));
  if (e != cudaSuccess) return check_launch(e, "b2_device_status");
  if (clear) {
    const uint32_t zero = 0;
    if (v != 0) e = cudaMemcpyToSymbol(g_device_status, &zero, sizeof(zero));
    if (e == cudaSuccess && index != 0) e = cudaMemcpyToSymbol(g_index_status, &zero, sizeof(zero));
    if (e != cudaSuccess) return check_launch(e, "b2_device_status(clear)");
  }
  *out_status = v != 0 ? v : index;
  return 0;
}

B2_API int b2_device_status_async(uint32_t* host_dst, void* stream) {
  if (host_dst == nullptr) return fail(1, "b2_device_status_async: host_dst is null");
  return check_launch(cudaMemcpyFromSymbolAsync(host_dst, g_device_status, sizeof(uint32_t), 0,
                                                cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream)),
                      "b2_device_status_async");
}

B2_API int b2_index_status_async(uint32_t* host_dst, void* stream) {
  if (host_dst == nullptr) return fail(1, "b2_index_status_async: host_dst is null");
  return check_launch(cudaMemcpyFromSymbolAsync(host_dst, g_index_status, sizeof(uint32_t), 0, cudaMemcpyDeviceToHost,
                                                static_cast<cudaStream_t>(stream)),
                      "b2_index_status_async");
}

B2_API int b2_set_wait_limit(uint64_t limit_ns) {
  const uint64_t v = limit_ns == 0 ? kWaitTimeoutNs : limit_ns;
  if (v < 1000000ull) return fail(1, "b2_set_wait_limit: limit below 1 ms");
  return check_launch(cudaMemcpyToSymbol(g_wait_limit_ns, &v, sizeof(v)), "b2_set_wait_limit");
}

B2_API int b2_test_set_fault(int fault) {
  if (fault < 0 || fault > static_cast<int>(kFaultGemmWithholdStage))
    return fail(1, "b2_test_set_fault: unknown fault %d", fault);
  const uint32_t v = static_cast<uint32_t>(fault);
  return check_launch(cudaMemcpyToSymbol(g_test_fault, &v, sizeof(v)), "b2_test_set_fault");
}

B2_API int b2_mask_lengths(const uint8_t* mask, int64_t batch, int64_t seq_len, int32_t* kv_len, uint8_t* row_mask_out,
                           uint8_t* not_prefix, void* stream) {
  if (mask == nullptr || kv_len == nullptr || not_prefix == nullptr)
    return fail(1, "b2_mask_lengths: null pointer argument");
  if (batch < 0 || seq_len <= 0) return fail(1, "b2_mask_lengths: invalid shape batch=%lld seq_len=%lld",
                                             (long long)batch, (long long)seq_len);
  if (batch > 0x7fffffffLL || seq_len > 0x7fffffffLL) return fail(2, "b2_mask_lengths: dimension exceeds 2^31");
  if (batch == 0) return 0;
  return check_launch(launch_mask_lengths(mask, batch, seq_len, kv_len, row_mask_out, not_prefix,
                                          static_cast<cudaStream_t>(stream)),
                      "b2_mask_lengths");
}

B2_API int b2_layernorm_fwd(const void* x, int x_is_bf16, const void* gamma, const void* beta, float eps, void* y,
                            float* resid_out, const uint8_t* row_mask, int64_t rows, int64_t d_model, void* stream) {
  if (x == nullptr || gamma == nullptr || beta == nullptr || y == nullptr)
    return fail(1, "b2_layernorm_fwd: null pointer argument");
  if (rows < 0 || d_model <= 0) return fail(1, "b2_layernorm_fwd: invalid shape rows=%lld d_model=%lld", (long long)rows,
                                            (long long)d_model);
  if (!(eps > 0.f)) return fail(1, "b2_layernorm_fwd: eps must be positive");
  if (rows == 0) return 0;
  if (rows > (int64_t)0x7fffffff * 8) return fail(2, "b2_layernorm_fwd: too many rows");
  return check_launch(launch_layernorm(x, x_is_bf16, static_cast<const __nv_bfloat16*>(gamma),
                                       static_cast<const __nv_bfloat16*>(beta), eps, static_cast<__nv_bfloat16*>(y),
                                       x_is_bf16 ? resid_out : nullptr, row_mask, rows, d_model,
                                       static_cast<cudaStream_t>(stream)),
                      "b2_layernorm_fwd");
}

B2_API int b2_linear_fwd(const void* a, const void* w, const void* bias, int64_t m, int64_t n, int64_t k, int epilogue,
                         void* out, int64_t ldo, const uint8_t* row_mask, int tile_n, void* stream) {
  if (a == nullptr || w == nullptr || out == nullptr) return fail(1, "b2_linear_fwd: null pointer argument");
  if (m < 0 || n <= 0 || k <= 0) return fail(1, "b2_linear_fwd: invalid shape m=%lld n=%lld k=%lld", (long long)m,
                                             (long long)n, (long long)k);
  if (epilogue < 0 || epilogue > 4)
    return fail(1, "b2_linear_fwd: unknown epilogue %d (reduce-scatter epilogues go through b2_linear_rs_fwd)",
                epilogue);
  if (n % 32 != 0) return fail(2, "b2_linear_fwd: n=%lld must be a multiple of 32", (long long)n);
  if (k % 8 != 0) return fail(2, "b2_linear_fwd: k=%lld must be a multiple of 8", (long long)k);
  if (ldo < n || ldo % 8 != 0) return fail(2, "b2_linear_fwd: ldo=%lld must be >= n and a multiple of 8", (long long)ldo);
  {
    const int bn = tile_n & 0xFFFF;
    const bool pair = (tile_n & kTilePair) != 0;
    if ((tile_n & ~(kTilePair | 0xFFFF)) != 0 || (tile_n != 0 && bn != 128 && bn != 192 && bn != 256) ||
        (pair && bn == 128))
      return fail(1, "b2_linear_fwd: tile_n must be 0, 128, 192, 256, or B2_TILE_PAIR | 192 / 256");
    if ((bn == 256 || bn == 192) && n % bn != 0)
      return fail(2, "b2_linear_fwd: an N tile of %d needs n %% %d == 0", bn, bn);
  }
  if (!aligned16(a) || !aligned16(w) || !aligned16(out) || (bias && !aligned16(bias)))
    return fail(2, "b2_linear_fwd: pointers must be 16-byte aligned");
  if (m > 0x7fffff00LL || n > 0x7fffff00LL) return fail(2, "b2_linear_fwd: dimension exceeds 2^31");
  if (m == 0) return 0;
  if (!is_sm100(nullptr)) return fail(2, "b2_linear_fwd: needs an sm_100 (B200) device");
  return check_launch(launch_gemm(static_cast<const __nv_bfloat16*>(a), static_cast<const __nv_bfloat16*>(w),
                                  static_cast<const __nv_bfloat16*>(bias), m, n, k, epilogue, out, ldo, row_mask, tile_n,
                                  static_cast<cudaStream_t>(stream)),
                      "b2_linear_fwd");
}

B2_API int b2_linear_ln_plan(int64_t m, int64_t n, int64_t k, int sm_count, int* tile_n, int* cluster,
                             int* recommended) {
  if (m <= 0 || n <= 0 || k <= 0) return fail(1, "b2_linear_ln_plan: invalid shape");
  int sms = sm_count;
  if (sms <= 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(2, "b2_linear_ln_plan: no CUDA device and no sm_count");
    sms = device_sm_count(dev);
  }
  if (m > 0x7fffff00LL || n > 0x7fffff00LL) return fail(2, "b2_linear_ln_plan: dimension exceeds 2^31");
  if (!gemm_ln_plan(m, n, k, sms, tile_n, cluster, recommended))
    return fail(2, "b2_linear_ln_plan: n=%lld has no fused plan (n %% 32 == 0 and n <= 256 or n = {128,192,256} x c, "
                "c <= 8)", (long long)n);
  return 0;
}

B2_API int b2_linear_ln_fwd(const void* a, const void* w, const void* bias, int64_t m, int64_t n, int64_t k,
                            int zero_masked_rows, float* resid, const uint8_t* row_mask, const void* gamma,
                            const void* beta, float eps, void* ln_out, void* stream) {
  if (a == nullptr || w == nullptr || resid == nullptr || gamma == nullptr || beta == nullptr || ln_out == nullptr)
    return fail(1, "b2_linear_ln_fwd: null pointer argument");
  if (m < 0 || n <= 0 || k <= 0) return fail(1, "b2_linear_ln_fwd: invalid shape m=%lld n=%lld k=%lld", (long long)m,
                                             (long long)n, (long long)k);
  if (!(eps > 0.f)) return fail(1, "b2_linear_ln_fwd: eps must be positive");
  if (k % 8 != 0) return fail(2, "b2_linear_ln_fwd: k=%lld must be a multiple of 8", (long long)k);
  if (m > 0x7fffff00LL || n > 0x7fffff00LL) return fail(2, "b2_linear_ln_fwd: dimension exceeds 2^31");
  if (!gemm_ln_plan(m > 0 ? m : 1, n, k, 0, nullptr, nullptr, nullptr))
    return fail(2, "b2_linear_ln_fwd: n=%lld has no fused plan (see b2_linear_ln_plan)", (long long)n);
  if (!aligned16(a) || !aligned16(w) || !aligned16(resid) || !aligned16(ln_out) || !aligned16(gamma) ||
      !aligned16(beta) || (bias && !aligned16(bias)))
    return fail(2, "b2_linear_ln_fwd: pointers must be 16-byte aligned");
  if (m == 0) return 0;
  if (!is_sm100(nullptr)) return fail(2, "b2_linear_ln_fwd: needs an sm_100 (B200) device");
  return check_launch(launch_gemm_ln(static_cast<const __nv_bfloat16*>(a), static_cast<const __nv_bfloat16*>(w),
                                     static_cast<const __nv_bfloat16*>(bias), m, n, k, zero_masked_rows != 0, resid,
                                     row_mask, static_cast<const __nv_bfloat16*>(gamma),
                                     static_cast<const __nv_bfloat16*>(beta), eps, static_cast<__nv_bfloat16*>(ln_out),
                                     static_cast<cudaStream_t>(stream)),
                      "b2_linear_ln_fwd");
}

B2_API int b2_attention_rows_fwd(const void* qkv, int64_t ld_qkv, int64_t q_col, int64_t k_col, int64_t v_col,
                                 int64_t batch, int64_t seq_len, int64_t num_heads, int64_t head_dim,
                                 const int32_t* kv_len, int causal, float scale, const int64_t* q_ranges,
                                 int n_ranges, void* ctx, int64_t ld_ctx, void* stream) {
  if (qkv == nullptr || ctx == nullptr) return fail(1, "b2_attention_rows_fwd: null pointer argument");
  if (batch < 0 || seq_len < 0 || num_heads <= 0) return fail(1, "b2_attention_rows_fwd: invalid shape");
  const bool tensor_core = head_dim == 64 || head_dim == 128;
  if (!tensor_core && head_dim != 8 && head_dim != 16 && head_dim != 32 && head_dim != 256)
    return fail(2, "b2_attention_rows_fwd: head_dim=%lld not supported (8, 16, 32, 64, 128, 256)", (long long)head_dim);
  // 64 / 128: 64-column TMA boxes per head; 32 (also tensor cores, 64-column boxes starting at the
  // head's 32-column offset) and the CUDA-core head dims: 16-byte aligned column offsets.
  const int64_t col_align = tensor_core ? 64 : 8;
  if (q_col % col_align || k_col % col_align || v_col % col_align || q_col < 0 || k_col < 0 || v_col < 0)
    return fail(2, "b2_attention_rows_fwd: q/k/v column offsets must be non-negative multiples of %lld",
                (long long)col_align);
  const int64_t width = num_heads * head_dim;
  if (q_col + width > ld_qkv || k_col + width > ld_qkv || v_col + width > ld_qkv)
    return fail(1, "b2_attention_rows_fwd: q/k/v columns exceed ld_qkv");
  if (ld_qkv % 8 != 0 || ld_ctx % 8 != 0 || ld_ctx < width) return fail(2, "b2_attention_rows_fwd: bad leading dimensions");
  if (!aligned16(qkv) || !aligned16(ctx)) return fail(2, "b2_attention_rows_fwd: pointers must be 16-byte aligned");
  if (batch * seq_len > 0x7fffff00LL || batch * num_heads > 0x7fffffffLL || (seq_len + 127) / 128 > 65535)
    return fail(2, "b2_attention_rows_fwd: problem too large");
  if (!(scale > 0.f)) return fail(1, "b2_attention_rows_fwd: scale must be positive");
  if (q_ranges == nullptr || n_ranges < 1 || n_ranges > 2)
    return fail(1, "b2_attention_rows_fwd: 1 or 2 query ranges are required");
  int64_t rows = 0;
  for (int r = 0; r < n_ranges; ++r) {
    const int64_t q_begin = q_ranges[2 * r], q_count = q_ranges[2 * r + 1];
    if (q_begin < 0 || q_count <= 0 || q_begin + q_count > seq_len || q_begin % 128 != 0 ||
        (q_count % 128 != 0 && q_begin + q_count != seq_len))
      return fail(1, "b2_attention_rows_fwd: query rows [%lld, +%lld) must be non-empty, start on a multiple of 128 "
                  "and end on one or at seq_len", (long long)q_begin, (long long)q_count);
    if (r == 1 && q_begin < q_ranges[0] + q_ranges[1])
      return fail(1, "b2_attention_rows_fwd: the second query range must start after the first one ends");
    rows += q_count;
  }
  if (batch == 0 || seq_len == 0 || rows == 0) return 0;
  if (!is_sm100(nullptr)) return fail(2, "b2_attention_rows_fwd: needs an sm_100 (B200) device");
  return check_launch(launch_attention(static_cast<const __nv_bfloat16*>(qkv), ld_qkv, q_col, k_col, v_col, batch,
                                       seq_len, num_heads, head_dim, kv_len, causal, scale,
                                       static_cast<__nv_bfloat16*>(ctx), ld_ctx, static_cast<cudaStream_t>(stream), q_ranges,
                                       n_ranges),
                      "b2_attention_rows_fwd");
}

B2_API int b2_attention_fwd(const void* qkv, int64_t ld_qkv, int64_t q_col, int64_t k_col, int64_t v_col,
                            int64_t batch, int64_t seq_len, int64_t num_heads, int64_t head_dim, const int32_t* kv_len,
                            int causal, float scale, void* ctx, int64_t ld_ctx, void* stream) {
  const int64_t whole[2] = {0, seq_len};
  if (seq_len == 0 && batch >= 0 && num_heads > 0) return 0;
  const int rc = b2_attention_rows_fwd(qkv, ld_qkv, q_col, k_col, v_col, batch, seq_len, num_heads, head_dim, kv_len,
                                       causal, scale, whole, 1, ctx, ld_ctx, stream);
  if (rc != 0) {
    std::string msg = g_last_error;
    const std::string from = "b2_attention_rows_fwd";
    if (msg.compare(0, from.size(), from) == 0) msg = "b2_attention_fwd" + msg.substr(from.size());
    snprintf(g_last_error, sizeof(g_last_error), "%s", msg.c_str());
  }
  return rc;
}

B2_API int b2_add_layernorm_fwd(float* resid, const float* delta, const void* bias, const uint8_t* row_mask,
                                int flags, const void* gamma, const void* beta, float eps, void* y, int64_t rows,
                                int64_t d_model, void* stream) {
  if (resid == nullptr || delta == nullptr || gamma == nullptr || beta == nullptr || y == nullptr)
    return fail(1, "b2_add_layernorm_fwd: null pointer argument");
  if (rows < 0 || d_model <= 0) return fail(1, "b2_add_layernorm_fwd: invalid shape");
  if (!(eps > 0.f)) return fail(1, "b2_add_layernorm_fwd: eps must be positive");
  if (flags & ~3) return fail(1, "b2_add_layernorm_fwd: unknown flags %d", flags);
  if (!add_layernorm_supported(d_model))
    return fail(2, "b2_add_layernorm_fwd: d_model=%lld not supported (128 * {1,2,4,6,8,16,32})", (long long)d_model);
  if (!aligned16(resid) || !aligned16(delta) || !aligned16(y) || (bias && !aligned16(bias)) || !aligned16(gamma) ||
      !aligned16(beta))
    return fail(2, "b2_add_layernorm_fwd: pointers must be 16-byte aligned");
  if (rows == 0) return 0;
  return check_launch(launch_add_layernorm(resid, delta, static_cast<const __nv_bfloat16*>(bias), row_mask, flags & 1,
                                           (flags >> 1) & 1, static_cast<const __nv_bfloat16*>(gamma),
                                           static_cast<const __nv_bfloat16*>(beta), eps,
                                           static_cast<__nv_bfloat16*>(y), rows, d_model,
                                           static_cast<cudaStream_t>(stream)),
                      "b2_add_layernorm_fwd");
}

B2_API int b2_peer_barrier(void* const* pads, int world, int rank, int channel, void* stream) {
  if (pads == nullptr) return fail(1, "b2_peer_barrier: pads is null");
  if (world < 1 || world > kMaxPeers) return fail(2, "b2_peer_barrier: world=%d not in [1, %d]", world, kMaxPeers);
  if (rank < 0 || rank >= world) return fail(1, "b2_peer_barrier: rank %d outside world %d", rank, world);
  if (channel < 0 || channel >= kPadChannels)
    return fail(1, "b2_peer_barrier: channel %d not in [0, %d)", channel, kPadChannels);
  PeerPads p{};
  for (int r = 0; r < world; ++r) {
    if (pads[r] == nullptr || (reinterpret_cast<uintptr_t>(pads[r]) & 3u))
      return fail(1, "b2_peer_barrier: pad of rank %d is null or misaligned", r);
    p.pad[r] = static_cast<uint32_t*>(pads[r]);
  }
  if (world == 1) return 0;
  return check_launch(launch_peer_barrier(p, world, rank, channel, static_cast<cudaStream_t>(stream)),
                      "b2_peer_barrier");
}

B2_API int b2_linear_rs_fwd(const void* a, const void* w, const void* bias, int64_t m, int64_t n, int64_t k,
                            int zero_masked_rows, void* const* peer_resid, int world, int rank, int64_t rows_per_rank,
                            int64_t ldo, const uint8_t* row_mask, int tile_n, void* stream) {
  if (a == nullptr || w == nullptr || peer_resid == nullptr) return fail(1, "b2_linear_rs_fwd: null pointer argument");
  if (m < 0 || n <= 0 || k <= 0) return fail(1, "b2_linear_rs_fwd: invalid shape");
  if (world < 1 || world > kGemmMaxPeers || rank < 0 || rank >= world)
    return fail(1, "b2_linear_rs_fwd: rank %d / world %d invalid (world <= %d)", rank, world, kGemmMaxPeers);
  if (rows_per_rank <= 0 || rows_per_rank * world < m) return fail(1, "b2_linear_rs_fwd: rows_per_rank too small");
  if (n % 32 != 0 || k % 8 != 0 || ldo < n || ldo % 8 != 0)
    return fail(2, "b2_linear_rs_fwd: n %% 32, k %% 8, ldo >= n and ldo %% 8 are required");
  if ((tile_n & ~(kTilePair | 0xFFFF)) != 0) return fail(1, "b2_linear_rs_fwd: bad tile_n");
  void* peers[kGemmMaxPeers] = {};
  for (int r = 0; r < world; ++r) {
    if (peer_resid[r] == nullptr || !aligned16(peer_resid[r]))
      return fail(2, "b2_linear_rs_fwd: residual of rank %d is null or not 16-byte aligned", r);
    peers[r] = peer_resid[r];
  }
  if (!aligned16(a) || !aligned16(w) || (bias && !aligned16(bias)))
    return fail(2, "b2_linear_rs_fwd: pointers must be 16-byte aligned");
  if (m == 0) return 0;
  if (!is_sm100(nullptr)) return fail(2, "b2_linear_rs_fwd: needs an sm_100 (B200) device");
  return check_launch(launch_gemm(static_cast<const __nv_bfloat16*>(a), static_cast<const __nv_bfloat16*>(w),
                                  static_cast<const __nv_bfloat16*>(bias), m, n, k,
                                  zero_masked_rows ? kEpiRsResidualZero : kEpiRsResidual, peers[rank], ldo, row_mask,
                                  tile_n, static_cast<cudaStream_t>(stream), peers, world, rank, rows_per_rank),
                      "b2_linear_rs_fwd");
}

B2_API int b2_layernorm_gather_fwd(const float* x, const void* gamma, const void* beta, float eps,
                                   void* const* y_ranks, int world, const uint8_t* row_mask, int64_t rows,
                                   int64_t d_model, void* stream) {
  if (x == nullptr || gamma == nullptr || beta == nullptr || y_ranks == nullptr)
    return fail(1, "b2_layernorm_gather_fwd: null pointer argument");
  if (rows < 0 || d_model <= 0 || !(eps > 0.f)) return fail(1, "b2_layernorm_gather_fwd: invalid arguments");
  if (world < 1 || world > kGatherMaxRanks) return fail(1, "b2_layernorm_gather_fwd: world %d not in [1, 8]", world);
  if (!layernorm_gather_supported(d_model))
    return fail(2, "b2_layernorm_gather_fwd: d_model=%lld not supported (256 * {1,2,3,4,8,16})", (long long)d_model);
  GatherDst dst{};
  for (int r = 0; r < world; ++r) {
    if (y_ranks[r] == nullptr || !aligned16(y_ranks[r]))
      return fail(2, "b2_layernorm_gather_fwd: destination of rank %d is null or not 16-byte aligned", r);
    dst.rank_rows[r] = static_cast<__nv_bfloat16*>(y_ranks[r]);
  }
  if (!aligned16(x) || !aligned16(gamma) || !aligned16(beta))
    return fail(2, "b2_layernorm_gather_fwd: pointers must be 16-byte aligned");
  if (rows == 0) return 0;
  return check_launch(launch_layernorm_gather(x, static_cast<const __nv_bfloat16*>(gamma),
                                              static_cast<const __nv_bfloat16*>(beta), eps, dst, world, row_mask, rows,
                                              d_model, static_cast<cudaStream_t>(stream)),
                      "b2_layernorm_gather_fwd");
}

B2_API int b2_linear_bcast_fwd(const void* a, const void* w, const void* bias, int64_t m, int64_t n, int64_t k,
                               void* const* peer_out, int world, int rank, int64_t col_begin, int64_t ldo, int tile_n,
                               void* stream) {
  if (a == nullptr || w == nullptr || peer_out == nullptr) return fail(1, "b2_linear_bcast_fwd: null pointer argument");
  if (m < 0 || n <= 0 || k <= 0) return fail(1, "b2_linear_bcast_fwd: invalid shape");
  if (world < 1 || world > kGemmMaxPeers || rank < 0 || rank >= world)
    return fail(1, "b2_linear_bcast_fwd: rank %d / world %d invalid (world <= %d)", rank, world, kGemmMaxPeers);
  if (n % 32 != 0 || k % 8 != 0 || ldo < n || ldo % 8 != 0)
    return fail(2, "b2_linear_bcast_fwd: n %% 32, k %% 8, ldo >= n and ldo %% 8 are required");
  if (col_begin < 0 || col_begin > n || col_begin % 32 != 0)
    return fail(1, "b2_linear_bcast_fwd: col_begin must be a multiple of 32 in [0, n]");
  if ((tile_n & ~(kTilePair | 0xFFFF)) != 0) return fail(1, "b2_linear_bcast_fwd: bad tile_n");
  void* peers[kGemmMaxPeers] = {};
  for (int r = 0; r < world; ++r) {
    if (peer_out[r] == nullptr || !aligned16(peer_out[r]))
      return fail(2, "b2_linear_bcast_fwd: output of rank %d is null or not 16-byte aligned", r);
    peers[r] = peer_out[r];
  }
  if (!aligned16(a) || !aligned16(w) || (bias && !aligned16(bias)))
    return fail(2, "b2_linear_bcast_fwd: pointers must be 16-byte aligned");
  if (m == 0) return 0;
  if (!is_sm100(nullptr)) return fail(2, "b2_linear_bcast_fwd: needs an sm_100 (B200) device");
  return check_launch(launch_gemm(static_cast<const __nv_bfloat16*>(a), static_cast<const __nv_bfloat16*>(w),
                                  static_cast<const __nv_bfloat16*>(bias), m, n, k, kEpiBiasPeers, peers[rank], ldo,
                                  nullptr, tile_n, static_cast<cudaStream_t>(stream), peers, world, rank, 0, col_begin),
                      "b2_linear_bcast_fwd");
}

B2_API int b2_rotary_fwd(const b2_rotary_args* args, void* stream) {
  if (args == nullptr) return fail(1, "b2_rotary_fwd: null pointer argument");
  const auto [x, ld_x, tokens, heads, head_dim, rotary_dim, interleaved, inverse, positions, table, max_positions, out,
              ld_out] = *args;
  if (tokens < 0 || heads <= 0 || max_positions <= 0)
    return fail(1, "b2_rotary_fwd: invalid shape tokens=%lld heads=%lld max_positions=%lld", (long long)tokens,
                (long long)heads, (long long)max_positions);
  if (head_dim % 16 != 0 || head_dim < 16 || head_dim > 256)
    return fail(2, "b2_rotary_fwd: head_dim=%lld must be a multiple of 16 up to 256", (long long)head_dim);
  if (rotary_dim % 16 != 0 || rotary_dim < 16 || rotary_dim > head_dim)
    return fail(2, "b2_rotary_fwd: rotary_dim=%lld must be a multiple of 16 up to head_dim", (long long)rotary_dim);
  if (heads > 65536 || tokens > 0x7fffffffLL) return fail(2, "b2_rotary_fwd: problem too large");
  if (ld_x < heads * head_dim || ld_out < heads * head_dim || ld_x % 8 != 0 || ld_out % 8 != 0)
    return fail(2, "b2_rotary_fwd: row strides must be multiples of 8 and at least heads * head_dim");
  if (tokens == 0) return 0;
  if (x == nullptr || positions == nullptr || table == nullptr || out == nullptr)
    return fail(1, "b2_rotary_fwd: null pointer argument");
  if (!aligned16(x) || !aligned16(out) || !aligned16(table))
    return fail(2, "b2_rotary_fwd: pointers must be 16-byte aligned");
  RotaryParams p{};
  p.x = static_cast<const __nv_bfloat16*>(x);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ld_x = ld_x;
  p.ld_out = ld_out;
  p.positions = positions;
  p.table = reinterpret_cast<const float2*>(table);
  p.max_positions = max_positions;
  p.tokens = static_cast<int>(tokens);
  p.heads = static_cast<int>(heads);
  p.head_dim = static_cast<int>(head_dim);
  p.rotary_dim = static_cast<int>(rotary_dim);
  p.inverse = inverse != 0;
  int dev = 0;
  cudaGetDevice(&dev);
  return check_launch(launch_rotary(p, interleaved != 0, device_sm_count(dev), static_cast<cudaStream_t>(stream)),
                      "b2_rotary_fwd");
}

// The pages of a cache as the kernels take them, or a status.
static int cache_pages(const b2_kv_cache* c, const char* what, CachePages* out, int* type) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr) return fail(1, "%s: null pointer argument", what);
  static_assert(B2_CACHE_BF16 == kCacheBf16 && B2_CACHE_E4M3 == kCacheE4m3 && B2_CACHE_INT4 == kCacheInt4, "one numbering");
  if (c->dtype != B2_CACHE_E4M3 && c->dtype != B2_CACHE_BF16 && c->dtype != B2_CACHE_INT4)
    return fail(1, "%s: unknown cache dtype %d", what, c->dtype);
  const bool int4 = c->dtype == B2_CACHE_INT4;
  *type = c->dtype;
  if (c->dtype == B2_CACHE_E4M3 && (c->k_scale == nullptr || c->v_scale == nullptr))
    return fail(1, "%s: an e4m3 cache needs k_scale and v_scale", what);
  if (int4 && (c->k_group == nullptr || c->v_group == nullptr))
    return fail(1, "%s: a 4-bit cache needs k_group and v_group", what);
  if (c->pages <= 0 || c->kv_heads <= 0) return fail(1, "%s: invalid cache shape", what);
  int shift = 0;
  while (shift < 8 && (int64_t{1} << shift) < c->page_size) ++shift;
  if (c->page_size < 16 || (int64_t{1} << shift) != c->page_size)
    return fail(2, "%s: page_size=%lld must be 16, 32, 64, 128 or 256", what, (long long)c->page_size);
  if (c->head_dim % 16 != 0 || c->head_dim < 16 || c->head_dim > 256)
    return fail(2, "%s: head_dim=%lld must be a multiple of 16 up to 256", what, (long long)c->head_dim);
  if (int4 && c->head_dim % 32 != 0)
    return fail(2, "%s: head_dim=%lld of a 4-bit cache must be a multiple of 32", what, (long long)c->head_dim);
  if (c->kv_heads > 16384 || c->pages > 0x7fffffffLL || c->page_stride > (0x7fffffffLL >> 1))
    return fail(2, "%s: cache too large", what);
  const int64_t head = c->page_size * c->head_dim;
  if (c->head_stride < head || (c->kv_heads > 1 && c->head_stride > c->page_stride) || c->page_stride < c->head_stride * (c->kv_heads - 1) + head)
    return fail(1, "%s: page_stride or head_stride too small", what);
  if (c->head_stride % 16 != 0 || c->page_stride % 16 != 0 || !aligned16(c->k) || !aligned16(c->v))
    return fail(2, "%s: cache pointers must be 16-byte aligned, strides multiples of 16 elements", what);
  if (int4 && (c->head_stride % 32 != 0 || c->page_stride % 32 != 0 || !aligned16(c->k_group) || !aligned16(c->v_group)))
    return fail(2, "%s: strides of a 4-bit cache must be multiples of 32 elements, k_group and v_group 16-byte aligned", what);
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->k_group = int4 ? static_cast<uint16_t*>(c->k_group) : nullptr;  // (a cache of another type may be an older, shorter struct)
  out->v_group = int4 ? static_cast<uint16_t*>(c->v_group) : nullptr;
  out->pages = c->pages;
  out->page_stride = c->page_stride;
  out->head_stride = c->head_stride;
  out->kv_heads = static_cast<int>(c->kv_heads);
  out->head_dim = static_cast<int>(c->head_dim);
  out->page_shift = shift;
  return 0;
}

B2_API int b2_cache_append_fwd(const b2_cache_append_args* args, void* stream) {
  if (args == nullptr) return fail(1, "b2_cache_append_fwd: null pointer argument");
  const auto [cache, qkv, ld_qkv, q_col, k_col, v_col, tokens, num_heads, batch, new_start, new_len, past_len, page_table,
              table_pages, max_new, table, max_positions, rotary_dim, interleaved, q_out, ld_q_out, k_out, ld_k_out] = *args;
  AppendParams p{};
  int type = 0;
  if (const int rc = cache_pages(cache, "b2_cache_append_fwd", &p.c, &type)) return rc;
  const int64_t hd = cache->head_dim, hk = cache->kv_heads;
  if (tokens < 0 || batch < 0 || max_new < 0 || num_heads <= 0 || table_pages <= 0)
    return fail(1, "b2_cache_append_fwd: invalid shape");
  if (num_heads % hk != 0)
    return fail(1, "b2_cache_append_fwd: num_heads=%lld must be a multiple of the cache's kv_heads=%lld",
                (long long)num_heads, (long long)hk);
  if (batch > 65535 || tokens > 0x7fffffffLL || max_new > 0x7fffffffLL || num_heads > 65536 ||
      table_pages > (0x7fffffffLL >> p.c.page_shift) || ld_qkv > 0x7fffffffLL)
    return fail(2, "b2_cache_append_fwd: problem too large");
  if (rotary_dim < 0 || rotary_dim > hd || rotary_dim % 16 != 0)
    return fail(2, "b2_cache_append_fwd: rotary_dim=%lld must be 0 or a multiple of 16 up to head_dim", (long long)rotary_dim);
  if (ld_qkv < 0 || q_col < 0 || k_col < 0 || v_col < 0 || q_col % 8 != 0 || k_col % 8 != 0 || v_col % 8 != 0 || ld_qkv % 8 != 0)
    return fail(2, "b2_cache_append_fwd: q/k/v columns and ld_qkv must be non-negative multiples of 8");
  if (k_col > ld_qkv - hk * hd || v_col > ld_qkv - hk * hd || (rotary_dim > 0 && q_col > ld_qkv - num_heads * hd))
    return fail(1, "b2_cache_append_fwd: q/k/v columns exceed ld_qkv");
  if (rotary_dim > 0 && max_positions <= 0) return fail(1, "b2_cache_append_fwd: max_positions must be positive");
  if (rotary_dim > 0 && (ld_q_out < num_heads * hd || ld_q_out % 8 != 0))
    return fail(2, "b2_cache_append_fwd: ld_q_out must be a multiple of 8 and at least num_heads * head_dim");
  if (k_out != nullptr && (ld_k_out < hk * hd || ld_k_out % 8 != 0))
    return fail(2, "b2_cache_append_fwd: ld_k_out must be a multiple of 8 and at least kv_heads * head_dim");
  if (tokens == 0 || batch == 0 || max_new == 0) return 0;
  if (qkv == nullptr || new_start == nullptr || new_len == nullptr || past_len == nullptr || page_table == nullptr ||
      (rotary_dim > 0 && (table == nullptr || q_out == nullptr)))
    return fail(1, "b2_cache_append_fwd: null pointer argument");
  if (!aligned16(qkv) || !aligned16(table) || !aligned16(q_out) || !aligned16(k_out))
    return fail(2, "b2_cache_append_fwd: pointers must be 16-byte aligned");
  if (!is_sm100(nullptr)) return fail(2, "b2_cache_append_fwd: needs an sm_100 (B200) device");
  p.qkv = static_cast<const __nv_bfloat16*>(qkv);
  p.ld = ld_qkv;
  p.tokens = tokens;
  p.q_col = static_cast<int>(q_col);
  p.k_col = static_cast<int>(k_col);
  p.v_col = static_cast<int>(v_col);
  p.batch = static_cast<int>(batch);
  p.group = static_cast<int>(num_heads / hk);
  p.max_new = max_new;
  p.new_start = new_start;
  p.new_len = new_len;
  p.past_len = past_len;
  p.page_table = page_table;
  p.ld_table = table_pages;
  p.table_pages = static_cast<int>(table_pages);
  p.rotary_dim = static_cast<int>(rotary_dim);
  p.table = reinterpret_cast<const float2*>(table);
  p.max_positions = max_positions;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.ld_q_out = ld_q_out;
  p.ld_k_out = ld_k_out;
  if (type == kCacheInt4) {
    int dev = 0;
    cudaGetDevice(&dev);
    return check_launch(launch_cache_append_int4(p, max_new, interleaved != 0, device_sm_count(dev), static_cast<cudaStream_t>(stream)),
                        "b2_cache_append_fwd");
  }
  return check_launch(launch_cache_append(p, max_new, type == kCacheE4m3, interleaved != 0, static_cast<cudaStream_t>(stream)),
                      "b2_cache_append_fwd");
}

B2_API int b2_cache_read_fwd(const b2_cache_read_args* args, void* stream) {
  if (args == nullptr) return fail(1, "b2_cache_read_fwd: null pointer argument");
  const auto [cache, out_start, length, start, batch, page_table, table_pages, max_len, rows, k_out, ld_k_out, v_out,
              ld_v_out] = *args;
  ReadParams p{};
  int type = 0;
  if (const int rc = cache_pages(cache, "b2_cache_read_fwd", &p.c, &type)) return rc;
  const int64_t width = cache->head_dim * cache->kv_heads;
  if (batch < 0 || rows < 0 || max_len < 0 || table_pages <= 0) return fail(1, "b2_cache_read_fwd: invalid shape");
  if (batch > 65535 || rows > 0x7fffffffLL || max_len > 0x7fffffffLL || table_pages > (0x7fffffffLL >> p.c.page_shift))
    return fail(2, "b2_cache_read_fwd: problem too large");
  if (k_out == nullptr && v_out == nullptr && rows > 0) return fail(1, "b2_cache_read_fwd: k_out and v_out are both null");
  if ((k_out != nullptr && (ld_k_out < width || ld_k_out % 8 != 0)) || (v_out != nullptr && (ld_v_out < width || ld_v_out % 8 != 0)))
    return fail(2, "b2_cache_read_fwd: row strides must be multiples of 8 and at least kv_heads * head_dim");
  if (batch == 0 || rows == 0 || max_len == 0) return 0;
  if (out_start == nullptr || length == nullptr || start == nullptr || page_table == nullptr)
    return fail(1, "b2_cache_read_fwd: null pointer argument");
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(2, "b2_cache_read_fwd: pointers must be 16-byte aligned");
  if (!is_sm100(nullptr)) return fail(2, "b2_cache_read_fwd: needs an sm_100 (B200) device");
  p.batch = static_cast<int>(batch);
  p.rows = rows;
  p.max_len = max_len;
  p.out_start = out_start;
  p.length = length;
  p.start = start;
  p.page_table = page_table;
  p.ld_table = table_pages;
  p.table_pages = static_cast<int>(table_pages);
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.ld_k_out = ld_k_out;
  p.ld_v_out = ld_v_out;
  int dev = 0;
  cudaGetDevice(&dev);
  return check_launch(launch_cache_read(p, type, device_sm_count(dev), static_cast<cudaStream_t>(stream)), "b2_cache_read_fwd");
}

B2_API int b2_cache_attention_workspace(int64_t batch, int64_t q_len, int64_t num_heads, int64_t kv_heads,
                                        int64_t head_dim, int sm_count, int64_t* bytes) {
  if (bytes == nullptr) return fail(1, "b2_cache_attention_workspace: null pointer argument");
  if (batch < 0 || q_len <= 0 || num_heads <= 0 || kv_heads <= 0 || num_heads % kv_heads != 0)
    return fail(1, "b2_cache_attention_workspace: invalid shape");
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(2, "b2_cache_attention_workspace: head_dim=%lld not supported (32, 64, 128)", (long long)head_dim);
  if (q_len > 1024 || num_heads > 65536 || sm_count > 65536)
    return fail(2, "b2_cache_attention_workspace: problem too large");
  int sms = sm_count;
  if (sms <= 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(2, "b2_cache_attention_workspace: no CUDA device and no sm_count");
    sms = device_sm_count(dev);
  }
  *bytes = cache_attention_workspace_bytes(head_dim, q_len * (num_heads / kv_heads), sms);
  return 0;
}

B2_API int b2_cache_attention_fwd(const b2_cache_attention_args* args, void* stream) {
  if (args == nullptr) return fail(1, "b2_cache_attention_fwd: null pointer argument");
  const auto [cache, q, ld_q, batch, q_len, num_heads, page_table, table_pages, kv_len, window, sinks, scale64, out, ld_out,
              workspace, workspace_bytes] = *args;
  const float scale = static_cast<float>(scale64);
  CacheAttnParams p{};
  int type = 0;
  if (const int rc = cache_pages(cache, "b2_cache_attention_fwd", &p.c, &type)) return rc;
  const int64_t hd = cache->head_dim, hk = cache->kv_heads;
  if (hd != 32 && hd != 64 && hd != 128)
    return fail(2, "b2_cache_attention_fwd: head_dim=%lld not supported (32, 64, 128)", (long long)hd);
  if (batch < 0 || q_len <= 0 || num_heads <= 0 || table_pages <= 0) return fail(1, "b2_cache_attention_fwd: invalid shape");
  if (num_heads % hk != 0)
    return fail(1, "b2_cache_attention_fwd: num_heads=%lld must be a multiple of the cache's kv_heads=%lld",
                (long long)num_heads, (long long)hk);
  if (window < 0 || sinks < 0 || (window == 0 && sinks != 0))
    return fail(1, "b2_cache_attention_fwd: window and sinks must not be negative, and sinks need a window");
  if (!(scale > 0.f) || std::isinf(scale)) return fail(1, "b2_cache_attention_fwd: scale must be positive and finite");
  // Token positions stay below 2^30, so that sums of a position and a window do not leave 32 bits.
  if (batch > kCacheMaxBatch || q_len > 1024 || num_heads > 65536 || table_pages > ((int64_t{1} << 30) >> p.c.page_shift))
    return fail(2, "b2_cache_attention_fwd: problem too large");
  const int64_t units = (table_pages << p.c.page_shift) / 64 + 1;  // at most one for 64 tokens
  const int64_t rows = q_len * (num_heads / hk);
  if (batch * hk > 0x7fffffffLL / units || rows > 16 * 65535)
    return fail(2, "b2_cache_attention_fwd: problem too large");
  if (ld_q < num_heads * hd || ld_out < num_heads * hd || ld_q % 8 != 0 || ld_out % 8 != 0)
    return fail(2, "b2_cache_attention_fwd: row strides must be multiples of 8 and at least num_heads * head_dim");
  if (batch == 0) return 0;
  if (q == nullptr || page_table == nullptr || kv_len == nullptr || out == nullptr || workspace == nullptr)
    return fail(1, "b2_cache_attention_fwd: null pointer argument");
  if (!aligned16(q) || !aligned16(out) || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0)
    return fail(2, "b2_cache_attention_fwd: pointers must be 16-byte aligned, the workspace 256-byte aligned");
  if (!is_sm100(nullptr)) return fail(2, "b2_cache_attention_fwd: needs an sm_100 (B200) device");
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = device_sm_count(dev);
  if (workspace_bytes < cache_attention_workspace_bytes(hd, rows, sms))
    return fail(1, "b2_cache_attention_fwd: the workspace is smaller than b2_cache_attention_workspace says");
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ld_q = ld_q;
  p.ld_out = ld_out;
  p.page_table = page_table;
  p.ld_table = table_pages;
  p.table_pages = static_cast<int>(table_pages);
  p.kv_len = kv_len;
  p.batch = static_cast<int>(batch);
  p.q_len = static_cast<int>(q_len);
  p.group = static_cast<int>(num_heads / hk);
  p.window = static_cast<int>(window < (int64_t{1} << 30) ? window : 0);  // beyond every position: none
  p.sinks = static_cast<int>(sinks < (int64_t{1} << 30) ? sinks : (int64_t{1} << 30));
  p.scale_log2 = scale * 1.4426950408889634f;
  return check_launch(launch_cache_attention(p, workspace, type, sms, static_cast<cudaStream_t>(stream)),
                      "b2_cache_attention_fwd");
}

B2_API int b2_window_attention_fwd(const b2_window_attention_args* args, void* stream) {
  if (args == nullptr) return fail(1, "b2_window_attention_fwd: null pointer argument");
  const auto [q, ld_q, k, ld_k, v, ld_v, batch, seq_len, num_heads, kv_heads, head_dim, kv_len, window, sinks, scale64, out,
              ld_out] = *args;
  const float scale = static_cast<float>(scale64);
  if (batch < 0 || seq_len < 0 || num_heads <= 0 || kv_heads <= 0) return fail(1, "b2_window_attention_fwd: invalid shape");
  if (num_heads % kv_heads != 0)
    return fail(1, "b2_window_attention_fwd: num_heads=%lld must be a multiple of kv_heads=%lld", (long long)num_heads,
                (long long)kv_heads);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(2, "b2_window_attention_fwd: head_dim=%lld not supported (32, 64, 128)", (long long)head_dim);
  if (window < 0 || sinks < 0 || (window == 0 && sinks != 0))
    return fail(1, "b2_window_attention_fwd: window and sinks must not be negative, and sinks need a window");
  if (!(scale > 0.f) || std::isinf(scale)) return fail(1, "b2_window_attention_fwd: scale must be positive and finite");
  if (num_heads > 65535) return fail(2, "b2_window_attention_fwd: problem too large");
  const int64_t kv_width = kv_heads * head_dim;
  if (ld_q < num_heads * head_dim || ld_out < num_heads * head_dim || ld_k < kv_width || ld_v < kv_width)
    return fail(1, "b2_window_attention_fwd: row strides must be at least heads * head_dim");
  if (ld_q % 8 != 0 || ld_k % 8 != 0 || ld_v % 8 != 0 || ld_out % 8 != 0)
    return fail(2, "b2_window_attention_fwd: row strides must be multiples of 8");
  // List places (sinks + window + tokens) stay below 2^31; the tensor maps' strides below 2^40 bytes.
  if (seq_len > (int64_t{1} << 28) || batch > 65535 || batch * num_heads > 0x7fffffffLL ||
      ((seq_len > 0) && (ld_q | ld_k | ld_v) > ((int64_t{1} << 38) / seq_len)) ||
      (batch * num_heads > 65535 && seq_len >= (int64_t{1} << 18)))
    return fail(2, "b2_window_attention_fwd: problem too large");
  if (batch == 0 || seq_len == 0) return 0;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr)
    return fail(1, "b2_window_attention_fwd: null pointer argument");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(2, "b2_window_attention_fwd: pointers must be 16-byte aligned");
  if (!is_sm100(nullptr)) return fail(2, "b2_window_attention_fwd: needs an sm_100 (B200) device");
  WindowParams p{};
  p.ctx = static_cast<__nv_bfloat16*>(out);
  p.ld_ctx = ld_out;
  p.kv_len = kv_len;
  p.B = static_cast<int>(batch);
  p.S = static_cast<int>(seq_len);
  p.heads = static_cast<int>(num_heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.window = window < seq_len ? static_cast<int>(window) : 0;  // a window of the whole sequence hides nothing
  p.sinks = p.window > 0 ? static_cast<int>(sinks < seq_len ? sinks : seq_len) : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  return check_launch(launch_window_attention<false>(static_cast<const __nv_bfloat16*>(q), ld_q,
                                                     static_cast<const __nv_bfloat16*>(k), ld_k,
                                                     static_cast<const __nv_bfloat16*>(v), ld_v, head_dim, p,
                                                     static_cast<cudaStream_t>(stream)),
                      "b2_window_attention_fwd");
}

B2_API int b2_packed_attention_fwd(const b2_packed_attention_args* args, void* stream) {
  if (args == nullptr) return fail(1, "b2_packed_attention_fwd: null pointer argument");
  const auto [q, ld_q, q_rows, k, ld_k, v, ld_v, kv_rows, q_start, kv_start, batch, num_heads, kv_heads, head_dim, window,
              sinks, scale64, out, ld_out] = *args;
  const float scale = static_cast<float>(scale64);
  if (batch < 0 || q_rows < 0 || kv_rows < 0 || num_heads <= 0 || kv_heads <= 0)
    return fail(1, "b2_packed_attention_fwd: invalid shape");
  if (num_heads > 65535) return fail(2, "b2_packed_attention_fwd: problem too large");
  if (num_heads % kv_heads != 0)
    return fail(1, "b2_packed_attention_fwd: num_heads=%lld must be a multiple of kv_heads=%lld", (long long)num_heads,
                (long long)kv_heads);
  if (head_dim != 32 && head_dim != 64 && head_dim != 128)
    return fail(2, "b2_packed_attention_fwd: head_dim=%lld not supported (32, 64, 128)", (long long)head_dim);
  if (window < 0 || sinks < 0 || (window == 0 && sinks != 0))
    return fail(1, "b2_packed_attention_fwd: window and sinks must not be negative, and sinks need a window");
  if (!(scale > 0.f) || std::isinf(scale)) return fail(1, "b2_packed_attention_fwd: scale must be positive and finite");
  const int64_t kv_width = kv_heads * head_dim;
  if (ld_q < num_heads * head_dim || ld_out < num_heads * head_dim || ld_k < kv_width || ld_v < kv_width)
    return fail(1, "b2_packed_attention_fwd: row strides must be at least heads * head_dim");
  if (ld_q % 8 != 0 || ld_k % 8 != 0 || ld_v % 8 != 0 || ld_out % 8 != 0)
    return fail(2, "b2_packed_attention_fwd: row strides must be multiples of 8");
  // List places (sinks + window + tokens) stay below 2^31; the tensor maps' strides below 2^40 bytes.
  const int64_t most = q_rows > kv_rows ? q_rows : kv_rows;
  if (most > (int64_t{1} << 28) || batch > (int64_t{1} << 20) || (most > 0 && (ld_q | ld_k | ld_v) > ((int64_t{1} << 38) / most)))
    return fail(2, "b2_packed_attention_fwd: problem too large");
  if (batch == 0 || q_rows == 0) return 0;
  if (q == nullptr || (kv_rows > 0 && (k == nullptr || v == nullptr)) || q_start == nullptr || kv_start == nullptr || out == nullptr)
    return fail(1, "b2_packed_attention_fwd: null pointer argument");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(2, "b2_packed_attention_fwd: pointers must be 16-byte aligned");
  if (!is_sm100(nullptr)) return fail(2, "b2_packed_attention_fwd: needs an sm_100 (B200) device");
  WindowParams p{};
  p.ctx = static_cast<__nv_bfloat16*>(out);
  p.ld_ctx = ld_out;
  p.heads = static_cast<int>(num_heads);
  p.kv_heads = static_cast<int>(kv_heads);
  p.window = window < kv_rows ? static_cast<int>(window) : 0;  // a window of all keys hides nothing
  p.sinks = p.window > 0 ? static_cast<int>(sinks < kv_rows ? sinks : kv_rows) : 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.q_start = q_start;
  p.kv_start = kv_start;
  p.batch = static_cast<int>(batch);
  p.q_rows = static_cast<int>(q_rows);
  p.kv_rows = static_cast<int>(kv_rows);
  const bool keys = kv_rows > 0;  // without any, the queries' memory stands in for theirs: no row of it is read
  return check_launch(launch_window_attention<true>(static_cast<const __nv_bfloat16*>(q), ld_q,
                                                    static_cast<const __nv_bfloat16*>(keys ? k : q), keys ? ld_k : ld_q,
                                                    static_cast<const __nv_bfloat16*>(keys ? v : q), keys ? ld_v : ld_q, head_dim,
                                                    p, static_cast<cudaStream_t>(stream)),
                      "b2_packed_attention_fwd");
}
