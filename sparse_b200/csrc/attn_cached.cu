// Decode attention (one query per sequence) over a quantised cache, and over a cache whose
// first `shared_len` positions are the same for the whole batch and lie in sequence 0's
// rows only.  out[b, h] = sum_j p_j v_j,  p = softmax_j(scale * q[b, h] . k_j), over the
// positions j < seq_lens[b]; a sequence without positions gives zeros.
#include <math.h>

#include "kv_fp8.cuh"

namespace sb {
namespace {

constexpr int kWarps = 4;

struct Cache {                        // bf16: [B, s_max, n_kv, d]; quantised: codes [B, n_kv, s_max, d], scales [B, n_kv, s_max]
  const void *k, *v;
  const uint8_t *ks, *vs;
};

// One CTA per (sequence, query head), one key per warp at a time.
template <int DK, int DV, bool FP8>
__global__ void __launch_bounds__(kWarps * 32)
attn_cached_kernel(const __nv_bfloat16 *__restrict__ q, int64_t q_stride, Cache cache, const int32_t *__restrict__ seq_lens,
                   int n_q, int n_kv, int s_max, int shared_len, float scale, __nv_bfloat16 *__restrict__ out) {
  constexpr int NK = DK / 32, NV = DV / 32;
  __shared__ float sm[kWarps], sl[kWarps], sacc[kWarps][DV];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x / n_q, h = blockIdx.x - b * n_q, hk = h / (n_q / n_kv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int len = min(max(seq_lens[b], 0), s_max);
  float qv[NK], acc[NV], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < NK; ++i) qv[i] = __bfloat162float(q[b * q_stride + h * DK + lane + 32 * i]) * scale;
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
  for (int j = warp; j < len; j += kWarps) {
    const int bb = j < shared_len ? 0 : b;
    float kv[NK], vv[NV], s = 0.f;
    if constexpr (FP8) {
      const size_t row = ((size_t)bb * n_kv + hk) * s_max + j;
      const uint8_t *kp = static_cast<const uint8_t *>(cache.k) + row * DK, *vp = static_cast<const uint8_t *>(cache.v) + row * DV;
      const float ks = e8m0_value(cache.ks[row]), vs = e8m0_value(cache.vs[row]);
#pragma unroll
      for (int i = 0; i < NK; ++i) kv[i] = f16x2_to_float2(e4m3x2_to_f16x2(kp[lane + 32 * i])).x * ks;
#pragma unroll
      for (int i = 0; i < NV; ++i) vv[i] = f16x2_to_float2(e4m3x2_to_f16x2(vp[lane + 32 * i])).x * vs;
    } else {
      const size_t row = ((size_t)bb * s_max + j) * n_kv + hk;
      const __nv_bfloat16 *kp = static_cast<const __nv_bfloat16 *>(cache.k) + row * DK;
      const __nv_bfloat16 *vp = static_cast<const __nv_bfloat16 *>(cache.v) + row * DV;
#pragma unroll
      for (int i = 0; i < NK; ++i) kv[i] = __bfloat162float(kp[lane + 32 * i]);
#pragma unroll
      for (int i = 0; i < NV; ++i) vv[i] = __bfloat162float(vp[lane + 32 * i]);
    }
#pragma unroll
    for (int i = 0; i < NK; ++i) s += qv[i] * kv[i];
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    // a score of -inf weighs nothing, also where no other has been seen
    const float m_new = fmaxf(m, s), ref = m_new == -INFINITY ? 0.f : m_new;
    const float corr = __expf(m - ref), p = s != s ? s : __expf(s - ref);
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = acc[i] * corr + p * vv[i];
    m = m_new;
  }
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
  for (int i = 0; i < NV; ++i) sacc[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
  float c[kWarps], total = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) { c[w] = sm[w] == -INFINITY ? (sl[w] == 0.f ? 0.f : 1.f) : __expf(sm[w] - top); total += sl[w] * c[w]; }
  for (int i = threadIdx.x; i < DV; i += kWarps * 32) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) o += sacc[w][i] * c[w];
    out[(size_t)blockIdx.x * DV + i] = __float2bfloat16_rn(total == 0.f ? 0.f : o / total);
  }
}

template <bool FP8>
int32_t attend(const char *name, const void *q, int64_t q_stride, Cache cache, const int32_t *seq_lens, int B, int n_q,
               int n_kv, int dk, int dv, int s_max, int shared_len, float scale, void *ws, size_t ws_bytes, void *out,
               void *stream) {
  if (B < 0 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || s_max < 1 || shared_len < 0 || shared_len > s_max ||
      (int64_t)B * n_q > (1 << 24))
    return fail(SB_E_INVALID_ARG, "%s: bad shape (B=%d heads %d/%d s_max=%d shared %d)", name, B, n_q, n_kv, s_max, shared_len);
  if (q_stride == 0) q_stride = (int64_t)n_q * dk;
  if (q_stride < (int64_t)n_q * dk) return fail(SB_E_INVALID_ARG, "%s: q_stride smaller than a token's heads", name);
  if (!((dk == 128 && dv == 128) || (dk == 192 && dv == 128) || (dk == 64 && dv == 64)))
    return fail(SB_E_UNSUPPORTED, "%s: head dims (%d,%d) not built (128/128, 192/128, 64/64)", name, dk, dv);
  if (B == 0) return SB_OK;
  if (!q || !cache.k || !cache.v || (FP8 && (!cache.ks || !cache.vs)) || !seq_lens || !ws || !out)
    return fail(SB_E_INVALID_ARG, "%s: null pointer", name);
  if (!aligned(cache.k, 16) || !aligned(cache.v, 16) || !aligned(ws, 16))
    return fail(SB_E_INVALID_ARG, "%s: cache and workspace must be 16-byte aligned", name);
  if (ws_bytes < sb_attn_cached_workspace_bytes(B, n_q, n_kv, dv, s_max, shared_len))
    return fail(SB_E_WORKSPACE, "%s: workspace too small", name);
  auto kern = dk == 128 ? attn_cached_kernel<128, 128, FP8> : dk == 192 ? attn_cached_kernel<192, 128, FP8>
                                                                        : attn_cached_kernel<64, 64, FP8>;
  SB_CUDA_CHECK(launch_pdl(kern, dim3(B * n_q), dim3(kWarps * 32), 0, static_cast<cudaStream_t>(stream),
                           static_cast<const __nv_bfloat16 *>(q), q_stride, cache, seq_lens, n_q, n_kv, s_max, shared_len,
                           scale, static_cast<__nv_bfloat16 *>(out)));
  SB_LAUNCH_CHECK();
  return SB_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" {

size_t sb_attn_cached_workspace_bytes(int32_t B, int32_t n_q, int32_t n_kv, int32_t dv, int32_t s_max, int32_t shared_len) {
  if (B < 0 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || dv < 1 || s_max < 1 || shared_len < 0) return 0;
  return 16;
}

int32_t sb_attn_decode_shared(const void *q, int64_t q_stride, const void *cache_k, const void *cache_v,
                              const int32_t *seq_lens, int32_t B, int32_t n_q, int32_t n_kv, int32_t dk, int32_t dv,
                              int32_t s_max, int32_t shared_len, float scale, void *ws, size_t ws_bytes, void *out,
                              int32_t *status, void *stream) {
  (void)status;
  return attend<false>("sb_attn_decode_shared", q, q_stride, Cache{cache_k, cache_v, nullptr, nullptr}, seq_lens, B, n_q,
                       n_kv, dk, dv, s_max, shared_len, scale, ws, ws_bytes, out, stream);
}

int32_t sb_attn_decode_fp8(const void *q, int64_t q_stride, const void *codes_k, const void *scale_k, const void *codes_v,
                           const void *scale_v, const int32_t *seq_lens, int32_t B, int32_t n_q, int32_t n_kv, int32_t dk,
                           int32_t dv, int32_t s_max, int32_t shared_len, float scale, void *ws, size_t ws_bytes, void *out,
                           int32_t *status, void *stream) {
  (void)status;
  return attend<true>("sb_attn_decode_fp8", q, q_stride,
                      Cache{codes_k, codes_v, static_cast<const uint8_t *>(scale_k), static_cast<const uint8_t *>(scale_v)},
                      seq_lens, B, n_q, n_kv, dk, dv, s_max, shared_len, scale, ws, ws_bytes, out, stream);
}

}  // extern "C"
