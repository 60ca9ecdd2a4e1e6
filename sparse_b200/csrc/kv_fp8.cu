// The quantised key/value cache: rotary embedding with the rows quantised as they are
// written, and reading positions back as bf16.  Row format: kv_fp8.cuh.
//
// Both kernels move bytes.  The append reads q, k and v once (bf16) and writes q once
// (bf16) and half the bytes of k and v; the read-back reads one byte and writes two per
// value.  Measured: 8 x 512 tokens of 16 heads of 128 (84 MB) 16.3 us, 5.2 TB/s, an instruction
// issued in two of three clocks; one token of eight sequences 2.1 us, the launch and two round
// trips; 8 x 4096 positions read back (345 MB) 57 us, 6.0 TB/s.
//
// The bf16 cache's append (model_ops.cu) rounds cos, sin and both products to bf16, as
// the model classes it stands for do.  Here angles and products stay in fp32 and a value is
// rounded once, to its code or to the bf16 query: an 8-bit code has no bits to spare for
// three earlier roundings.
#include <math.h>

#include "kv_fp8.cuh"

namespace sb {
namespace {

constexpr int kAppendThreads = 128;
constexpr int kAppendCtas = 10;                  // an SM holds at once, 48 registers a thread
constexpr int kMaxHead = 256;                    // angles are kept for one CTA's threads
constexpr int kMaxHalf = kMaxHead / 2;

// theta^(-2j / rope_dim) / (2 pi), turns per position, as the sum of two floats
struct RopeFreq { float2 turns[kMaxHalf]; };

// rows of token t, head h at base + t * token + h * head
struct RowSource {
  const __nv_bfloat16 *base;
  int64_t token, head;
  __device__ __forceinline__ const __nv_bfloat16 *at(int t, int h) const { return base + t * token + h * head; }
};

template <bool VEC>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16 *p) {
  if constexpr (VEC) return __ldg(reinterpret_cast<const uint4 *>(p));
  const unsigned short *e = reinterpret_cast<const unsigned short *>(p);
  return make_uint4(e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16), e[4] | ((uint32_t)e[5] << 16),
                    e[6] | ((uint32_t)e[7] << 16));
}
__device__ __forceinline__ void unpack8(const uint4 &v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = bf16_lo(w[i]); x[2 * i + 1] = bf16_hi(w[i]); }
}

// A row is held by L lanes, two vectors of eight values each: a lane of the rotated part has
// the two that are turned into one another, so both are loaded once and share their angles.
struct RowPlace {
  int e0, e1;                         // first elements of the two vectors
  bool turned;
};
__device__ __forceinline__ RowPlace row_place(int lane, int half) {
  const int pairs = half >> 3;
  if (lane < pairs) return RowPlace{8 * lane, half + 8 * lane, true};
  return RowPlace{16 * lane, 16 * lane + 8, false};
}

__device__ __forceinline__ void turn(float (&x)[8], float (&y)[8], const float2 *table, int pairs, int lane) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 cs = table[i * pairs + lane];        // neighbouring lanes on neighbouring banks
    const float a = x[i], b = y[i];
    x[i] = a * cs.x - b * cs.y;
    y[i] = b * cs.x + a * cs.y;
  }
}

__device__ __forceinline__ uint2 codes8(float (&x)[8], uint32_t byte, float inv) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= inv;
  if (byte == kScaleTop) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i], -kCodeTop), kCodeTop);
  }
  return make_uint2(e4m3x4(x[0], x[1], x[2], x[3]), e4m3x4(x[4], x[5], x[6], x[7]));
}

// max(a, |b|), NaN where one is
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// a + b as the rounded sum and what the rounding leaves
__device__ __forceinline__ float2 two_sum(float a, float b) {
  const float s = __fadd_rn(a, b), b_part = __fsub_rn(s, a);
  return make_float2(s, __fadd_rn(__fsub_rn(a, __fsub_rn(s, b_part)), __fsub_rn(b, b_part)));
}

// Codes and scale byte of the row that L lanes hold (`mask`: those lanes), `in`: the lane has values of it.
template <int L>
__device__ __forceinline__ void store_codes(float (&x)[8], float (&y)[8], RowPlace at, bool in, int lane, uint32_t mask,
                                            uint8_t *codes, uint8_t *scale) {
  float top = 0.f;
  if (in) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_abs(max_abs(top, x[i]), y[i]);
  }
#pragma unroll
  for (int off = L / 2; off >= 1; off >>= 1) top = max_abs(top, __shfl_xor_sync(mask, top, off));
  if (!in) return;
  const uint32_t byte = e8m0_of_amax(__float_as_uint(top) & 0x7fffffffu);
  const float inv = e8m0_inverse(byte);
  uint2 c0 = codes8(x, byte, inv), c1 = codes8(y, byte, inv);
  if (byte == kScaleNan) c0 = c1 = make_uint2(0, 0);
  *reinterpret_cast<uint2 *>(codes + at.e0) = c0;
  *reinterpret_cast<uint2 *>(codes + at.e1) = c1;
  if (lane == 0) *scale = (uint8_t)byte;
}

__device__ __forceinline__ void store_bf16(__nv_bfloat16 *p, const float (&x)[8]) {
  *reinterpret_cast<uint4 *>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                             pack_bf16x2(x[6], x[7]));
}

// grid = (tokens, shares of a token's rows).  A token's angles are worked out once per CTA:
// turns = pos * frequency, both as sums of two floats, the large product without error in its
// fraction and what a float leaves of the turns put behind the sine and cosine, so that these are
// the 64-bit formula's to fp32's last bits, far into a long context too (to 2^-14 at the last
// positions that 32 bits have): codes differ from the 64-bit rows' as often as those of rows turned
// by correctly rounded cosines do (148 each of 132 million values, positions up to 30 thousand).
template <int L, bool VEC>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas)
rope_append_fp8_kernel(RowSource q, RowSource k_rot, RowSource k_rest, RowSource v, __nv_bfloat16 *__restrict__ q_out,
                       const int32_t *__restrict__ seq_of_token, const int32_t *__restrict__ pos_of_token, int B,
                       int n_q, int n_kv, int dk, int dv, int rope, int s_max, uint8_t *__restrict__ codes_k,
                       uint8_t *__restrict__ scale_k, uint8_t *__restrict__ codes_v, uint8_t *__restrict__ scale_v,
                       const __grid_constant__ RopeFreq freq) {
  __shared__ float2 table[kMaxHalf];
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x;
  const int half = rope >> 1, pairs = half >> 3;
  const int lane = threadIdx.x % L;
  const RowPlace key_at = row_place(lane, half), value_at = row_place(lane, 0);
  const bool in_key = lane * 16 < dk, in_value = lane * 16 < dv;
  constexpr int kRows = kAppendThreads / L;              // rows of a CTA in one turn
  // a lane's two vectors of row r: queries, then keys, then values
  const auto fetch = [&](int r, uint4 &a, uint4 &b) {
    const bool value = r >= n_q + n_kv;
    if (r >= n_q + 2 * n_kv || !(value ? in_value : in_key)) return;
    // (an unrotated vector of a key stands in k_rest, rope elements further on than there)
    const __nv_bfloat16 *src = r < n_q ? q.at(t, r) : value ? v.at(t, r - n_q - n_kv)
                               : key_at.turned ? k_rot.at(t, r - n_q) : k_rest.at(t, r - n_q) - rope;
    a = load8<VEC>(src + (value ? value_at.e0 : key_at.e0));
    b = load8<VEC>(src + (value ? value_at.e1 : key_at.e1));
  };
  // the first turn's rows are on their way while the position is read and its angles are worked out,
  // a later turn's during the one before it
  int r = blockIdx.y * kRows + threadIdx.x / L;
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  fetch(r, a, b);
  const int pos = pos_of_token[t], seq = seq_of_token[t];
  if (threadIdx.x < half) {
    // (pos = p + what a float's 24 bits leave of it, none below 2^24)
    const float p = __int2float_rz(pos), rest = (float)(pos - (int)p);
    const float hi = freq.turns[threadIdx.x].x, lo = freq.turns[threadIdx.x].y;
    const float f = p * hi;
    const float2 whole = two_sum(f - rintf(f), fmaf(p, hi, -f));
    const float2 turns = two_sum(whole.x, p * lo + rest * hi);
    float sn, cs;
    sincospif(2.f * turns.x, &sn, &cs);
    const float tiny = 6.2831853f * (whole.y + turns.y);       // radians that a float of the turns leaves
    const float sn0 = sn;
    sn = fmaf(tiny, cs, sn);
    cs = fmaf(-tiny, sn0, cs);
    table[(threadIdx.x & 7) * pairs + (threadIdx.x >> 3)] = make_float2(cs, sn);
  }
  __syncthreads();
  const bool cached = pos >= 0 && pos < s_max && seq >= 0 && seq < B;
  const int rows = n_q + (cached ? 2 * n_kv : 0);
  const uint32_t mask = ((1u << L) - 1u) << (threadIdx.x & 31 & ~(L - 1));
  const size_t row0 = (size_t)(cached ? seq : 0) * n_kv * s_max + (cached ? pos : 0);      // of head 0 in the cache
  while (r < rows) {
    const int next = r + gridDim.y * kRows;
    float x[8], y[8];
    unpack8(a, x);
    unpack8(b, y);
    fetch(next, a, b);
    if (r < n_q) {
      if (in_key) {
        if (key_at.turned) turn(x, y, table, pairs, lane);
        __nv_bfloat16 *dst = q_out + ((size_t)t * n_q + r) * dk;
        store_bf16(dst + key_at.e0, x);
        store_bf16(dst + key_at.e1, y);
      }
    } else if (r < n_q + n_kv) {
      const size_t row = row0 + (size_t)(r - n_q) * s_max;
      if (in_key && key_at.turned) turn(x, y, table, pairs, lane);
      store_codes<L>(x, y, key_at, in_key, lane, mask, codes_k + row * dk, scale_k + row);
    } else {
      const size_t row = row0 + (size_t)(r - n_q - n_kv) * s_max;
      store_codes<L>(x, y, value_at, in_value, lane, mask, codes_v + row * dv, scale_v + row);
    }
    r = next;
  }
}

template <int L>
int32_t launch_append(bool vec, dim3 grid, cudaStream_t st, RowSource q, RowSource k_rot, RowSource k_rest, RowSource v,
                      void *q_out, const int32_t *seq, const int32_t *pos, int B, int n_q, int n_kv, int dk, int dv,
                      int rope, int s_max, void *ck, void *sk, void *cv, void *sv, const RopeFreq &freq) {
  auto kern = vec ? rope_append_fp8_kernel<L, true> : rope_append_fp8_kernel<L, false>;
  SB_CUDA_CHECK(launch_pdl(kern, grid, dim3(kAppendThreads), 0, st, q, k_rot, k_rest, v,
                           static_cast<__nv_bfloat16 *>(q_out), seq, pos, B, n_q, n_kv, dk, dv, rope, s_max,
                           static_cast<uint8_t *>(ck), static_cast<uint8_t *>(sk), static_cast<uint8_t *>(cv),
                           static_cast<uint8_t *>(sv), freq));
  SB_LAUNCH_CHECK();
  return SB_OK;
}

// grid = (shares of the positions, heads, sequences).  A position of a head is dk/8 + dv/8 vectors of
// eight codes; a thread keeps its place in the row and walks over positions, kReadAhead of them
// in flight.  Eight codes a thread, so that a warp's 16-byte stores are one run of bytes.
constexpr int kReadThreads = 256, kReadAhead = 4;
__global__ void __launch_bounds__(kReadThreads)
cache_read_fp8_kernel(const uint8_t *__restrict__ codes_k, const uint8_t *__restrict__ scale_k,
                      const uint8_t *__restrict__ codes_v, const uint8_t *__restrict__ scale_v, int n_kv, int dk, int dv,
                      int s_max, int begin, int count, int shared_len, __nv_bfloat16 *__restrict__ out_k,
                      __nv_bfloat16 *__restrict__ out_v) {
  pdl_launch_dependents();
  pdl_wait();
  const int per_row = (dk + dv) >> 3;
  const int lane = threadIdx.x % per_row, step = kReadThreads / per_row;
  const int first = threadIdx.x / per_row;
  if (first >= step) return;                              // (threads left over where per_row does not divide the CTA)
  const int h = blockIdx.y, b = blockIdx.z;
  const bool key = lane < (dk >> 3);
  const int d = key ? dk : dv, e = (key ? lane : lane - (dk >> 3)) * 8;
  const uint8_t *codes = key ? codes_k : codes_v, *scales = key ? scale_k : scale_v;
  // rows of this head in sequence 0's cache and in the sequence's own, from position `begin` on
  const size_t row_shared = (size_t)h * s_max + begin, row_own = row_shared + (size_t)b * n_kv * s_max;
  const int shared = shared_len - begin;
  __nv_bfloat16 *dst = (key ? out_k : out_v) + ((size_t)b * n_kv + h) * count * d + e;
  for (int i0 = blockIdx.x * step * kReadAhead + first; i0 < count; i0 += gridDim.x * step * kReadAhead) {
    uint2 c[kReadAhead];
    uint32_t byte[kReadAhead];
#pragma unroll
    for (int a = 0; a < kReadAhead; ++a) {
      const int i = i0 + a * step;
      if (i < count) {
        const size_t row = (i < shared ? row_shared : row_own) + i;
        c[a] = __ldg(reinterpret_cast<const uint2 *>(codes + row * d + e));
        byte[a] = __ldg(scales + row);
      }
    }
#pragma unroll
    for (int a = 0; a < kReadAhead; ++a) {
      const int i = i0 + a * step;
      if (i >= count) break;
      const float scale = e8m0_value(byte[a]);
      const float2 v0 = f16x2_to_float2(e4m3x2_to_f16x2(c[a].x)), v1 = f16x2_to_float2(e4m3x2_to_f16x2(c[a].x >> 16));
      const float2 v2 = f16x2_to_float2(e4m3x2_to_f16x2(c[a].y)), v3 = f16x2_to_float2(e4m3x2_to_f16x2(c[a].y >> 16));
      __stcs(reinterpret_cast<uint4 *>(dst + (size_t)i * d),
             make_uint4(pack_bf16x2(v0.x * scale, v0.y * scale), pack_bf16x2(v1.x * scale, v1.y * scale),
                        pack_bf16x2(v2.x * scale, v2.y * scale), pack_bf16x2(v3.x * scale, v3.y * scale)));
    }
  }
}

// The frequencies of a model are the same in every call: a thread keeps the last table.
const RopeFreq &rope_freq(double theta, int rope_dim) {
  static thread_local RopeFreq kept;
  static thread_local double kept_theta = 0.0;
  static thread_local int kept_dim = -1;
  if (kept_theta != theta || kept_dim != rope_dim) {
    const double log_theta = log(theta);
    for (int j = 0; j < rope_dim / 2; ++j) {
      const double turns = exp(-2.0 * j / rope_dim * log_theta) / (2.0 * M_PI);
      kept.turns[j].x = (float)turns;
      kept.turns[j].y = (float)(turns - (double)kept.turns[j].x);
    }
    kept_theta = theta;
    kept_dim = rope_dim;
  }
  return kept;
}

bool head_ok(int d) { return d >= 16 && d <= kMaxHead && d % 16 == 0; }

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" {

int32_t sb_rope_append_fp8(const sb_rope_append_args *args, void *stream) {
  if (!args) return fail(SB_E_INVALID_ARG, "sb_rope_append_fp8: null pointer");
  const sb_rope_append_args &a = *args;
  const int T = a.T, B = a.B, n_q = a.n_q, n_kv = a.n_kv, dk = a.dk, dv = a.dv, rope_dim = a.rope_dim, s_max = a.s_max;
  const double theta = (double)a.theta + (double)a.theta_rest;
  if (T < 0 || B < 1 || n_q < 1 || n_kv < 1 || n_q > 65536 || n_kv > 65536 || s_max < 1 || !head_ok(dk) || !head_ok(dv) ||
      rope_dim < 0 || rope_dim > dk || rope_dim % 16 != 0 || !(theta > 0.0) || !isfinite(theta))
    return fail(SB_E_INVALID_ARG, "sb_rope_append_fp8: bad shape (T=%d B=%d heads %d/%d widths %d/%d rope %d s_max=%d)", T,
                B, n_q, n_kv, dk, dv, rope_dim, s_max);
  if (T == 0) return SB_OK;
  if (!a.q || (rope_dim > 0 && !a.k_rot) || (rope_dim < dk && !a.k_rest) || !a.v || !a.seq_of_token || !a.pos_of_token ||
      !a.q_out || !a.codes_k || !a.scale_k || !a.codes_v || !a.scale_v)
    return fail(SB_E_INVALID_ARG, "sb_rope_append_fp8: null pointer");
  if (!aligned(a.q_out, 16) || !aligned(a.codes_k, 16) || !aligned(a.codes_v, 16))
    return fail(SB_E_INVALID_ARG, "sb_rope_append_fp8: q_out and the codes must be 16-byte aligned");
  const void *base[4] = {a.q, a.k_rot, a.k_rest, a.v};
  RowSource src[4];
  bool vec = true;
  for (int i = 0; i < 4; ++i) {
    src[i] = RowSource{static_cast<const __nv_bfloat16 *>(base[i]), a.stride[2 * i], a.stride[2 * i + 1]};
    vec = vec && aligned(base[i], 16) && a.stride[2 * i] % 8 == 0 && a.stride[2 * i + 1] % 8 == 0;
  }
  const RopeFreq &freq = rope_freq(theta, rope_dim);
  const int widest = dk > dv ? dk : dv;
  const int lanes = widest <= 64 ? 4 : widest <= 128 ? 8 : 16;
  // As many CTAs as the SMs hold at once, so that a CTA has few turns: a turn is a load round trip.
  // 1003 tokens of 16 heads of 192/128: one CTA a token (six turns) 10.9 us, two 8.2 us; 8 x 512 tokens
  // of 16 heads of 128, one CTA a token in either case, 16.3 us.  At 61 registers, eight CTAs an SM:
  // 8.8 and 17.3 us; at 40, twelve: 8.7 and 16.1 us.
  const int sms = sb_device_sm_count() > 0 ? sb_device_sm_count() : 148;
  const int wanted = ((n_q + 2 * n_kv) * lanes + kAppendThreads - 1) / kAppendThreads;
  const int room = (int)(((int64_t)kAppendCtas * sms + T - 1) / T);
  const dim3 grid(T, wanted < room ? wanted : room);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto launch = lanes == 4 ? launch_append<4> : lanes == 8 ? launch_append<8> : launch_append<16>;
  return launch(vec, grid, st, src[0], src[1], src[2], src[3], a.q_out, a.seq_of_token, a.pos_of_token, B, n_q, n_kv, dk, dv,
                rope_dim, s_max, a.codes_k, a.scale_k, a.codes_v, a.scale_v, freq);
}

int32_t sb_cache_read_fp8(const sb_cache_read_args *args, void *stream) {
  if (!args) return fail(SB_E_INVALID_ARG, "sb_cache_read_fp8: null pointer");
  const sb_cache_read_args &a = *args;
  const int B = a.B, n_kv = a.n_kv, dk = a.dk, dv = a.dv, s_max = a.s_max, begin = a.begin, count = a.count, shared_len = a.shared_len;
  if (B < 0 || B > 65535 || n_kv < 1 || n_kv > 65535 || !head_ok(dk) || !head_ok(dv) || s_max < 1 || begin < 0 ||
      count < 0 || count > s_max - begin || shared_len < 0 || shared_len > s_max)
    return fail(SB_E_INVALID_ARG, "sb_cache_read_fp8: bad shape (B=%d n_kv=%d widths %d/%d positions %d+%d of %d, shared %d)",
                B, n_kv, dk, dv, begin, count, s_max, shared_len);
  if (B == 0 || count == 0) return SB_OK;
  if (!a.codes_k || !a.scale_k || !a.codes_v || !a.scale_v || !a.out_k || !a.out_v)
    return fail(SB_E_INVALID_ARG, "sb_cache_read_fp8: null pointer");
  if (!aligned(a.codes_k, 16) || !aligned(a.codes_v, 16) || !aligned(a.out_k, 16) || !aligned(a.out_v, 16))
    return fail(SB_E_INVALID_ARG, "sb_cache_read_fp8: codes and outputs must be 16-byte aligned");
  const int step = kReadThreads / ((dk + dv) >> 3) * kReadAhead;
  const int wanted = (count + step - 1) / step;
  const int sms = sb_device_sm_count() > 0 ? sb_device_sm_count() : 148;
  const long long heads = (long long)B * n_kv;
  const long long room = (32ll * sms + heads - 1) / heads;
  const dim3 grid((unsigned)(wanted < room ? wanted : room), n_kv, B);
  SB_CUDA_CHECK(launch_pdl(cache_read_fp8_kernel, grid, dim3(kReadThreads), 0, static_cast<cudaStream_t>(stream),
                           static_cast<const uint8_t *>(a.codes_k), static_cast<const uint8_t *>(a.scale_k),
                           static_cast<const uint8_t *>(a.codes_v), static_cast<const uint8_t *>(a.scale_v), n_kv, dk, dv,
                           s_max, begin, count, shared_len, static_cast<__nv_bfloat16 *>(a.out_k),
                           static_cast<__nv_bfloat16 *>(a.out_v)));
  SB_LAUNCH_CHECK();
  return SB_OK;
}

size_t sb_cache_struct_bytes(int32_t which) {
  return which == 0 ? sizeof(sb_rope_append_args) : which == 1 ? sizeof(sb_cache_read_args) : which == 2 ? sizeof(sb_attn_cached_args) : 0;
}

}  // extern "C"
