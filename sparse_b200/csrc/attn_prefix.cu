// Attention of a whole batch's queries over the positions that its sequences share: for
// every key head one matrix product of the batch's rows (sequences x query heads of the
// group, tiles of 128) with the shared keys, a softmax along the keys, and a second product
// with the values, on the tensor cores.
//
// Bound by the bytes of the prefix while the rows fit one tile (bf16, heads of 128: 64 KB
// per 128 positions are 2.8 K clocks of an SM's share of HBM, the two products 1 K, the
// exponentials 1 K).  For 256 rows by the products: 128 positions take 3.6 K clocks, of which the 48
// products issued for them take 3.1 K (one of 64 score columns takes as long as one of 128, but
// leaves room in TMEM for a second score buffer, without which the products wait for the
// exponentials: 52 instead of 50 us).  With codes and few rows by the conversion, some 2.9 K clocks.  One CTA
// per SM.  The positions are cut into 148 / (key heads x row tiles) runs, rounded down, at least one:
// between 75 and 147 such pairs the other SMs have nothing to do.
//
// Measured (alone, cold, ncu): 8192 positions of a bf16 cache of 16 heads for 32 sequences 20.4 us
// (67 MB, 3.3 TB/s); 16384 quantised positions of 4 heads for 512 rows each 33.6 us (17 GFLOP, 0.51
// PF/s; 34 M exponentials).
//
// Roles: warp 0 loads tiles of 128 keys and values (TMA: bf16 boxes into the swizzled operand
// layout; codes as one run of bytes each), warp 1 issues the products, two groups of four
// warps do the softmax of 64-position blocks, one thread per row.  Up to 128 rows the groups
// take one half of every tile each, above (heads of 128 and less) one of two row tiles each, so
// that a tile is loaded and converted once for 256 rows.  A group has its own running maximum,
// its own output accumulator and two score buffers in TMEM (2 x 2 x 64 + 2 x DV columns): the
// groups exchange nothing until the end, and a block's products run under the exponentials of
// the block before it.  Probabilities go back into TMEM (bf16, over their scores), where the
// second product takes its left operand from.  Quantised: four warps turn the keys' codes into
// bf16 operands and four the values', scale applied (as exact as reading the row back
// is, kv_fp8.cuh), so the products are the bf16 ones.  (The fp8 products would round the queries and
// probabilities to codes.)
//
// Probabilities are rounded to bf16 (2^-8), the type of the values that they are multiplied
// with, and their sum is taken over the rounded ones; scores, sums and accumulators are fp32.  Against
// probabilities in fp32 (attn_decode_kernel) that shows where values average out: 8192 positions of
// independent values 2.3e-3 from 64 bits in norm, of which the rounding of the output makes 1.65e-3.
//
// All mbarrier waits are bounded; when one runs out the CTA raises its abort flag, reports
// through `status`, makes its partial result NaN, waits for its copies and frees its TMEM.
#include <math.h>

#include <atomic>

#include "attn_cached.cuh"
#include "sb_tc.cuh"

namespace sb {
namespace {

constexpr int kKeys = 128;                       // positions of a tile
constexpr uint32_t kBox = kKeys * 128;           // 64 bf16 columns of 128 rows: 16 KB
constexpr int kBlock = 64;                        // positions of a block: what a group works on at a time
constexpr int kSoftmaxWarp = 4, kConvertWarp = 12;

// TWO: two row tiles of 128 rows, one for each group
template <int DK, int DV, bool FP8, bool TWO>
struct Layout {
  static constexpr uint32_t kQ = DK / 64 * kBox, kK = DK / 64 * kBox, kV = DV / 64 * kBox;
  static constexpr uint32_t kAllQ = (TWO ? 2 : 1) * kQ;
  // operand buffers: filled by TMA (bf16), or by the converting warps from stages of codes
  static constexpr int kStages = FP8 ? (DK > 128 ? 1 : 2) : (TWO || DK > 128 ? 2 : DK > 64 ? 3 : 4);
  // stages of codes: half a tile each, so that one is loaded while another is converted
  static constexpr int kRaw = FP8 ? (TWO && DK > 64 ? 2 : 4) : 0;
  static constexpr uint32_t kRawK = kBlock * DK, kRawV = kBlock * DV;
  static constexpr uint32_t kBytes = kAllQ + kStages * (kK + kV) + kRaw * (kRawK + kRawV);
  // One CTA per SM, whatever its registers are: a CTA takes all of the tensor memory, and a second one on the SM
  // would stand there until the first is through.
  static constexpr uint32_t kAlone = 117 * 1024;
  static constexpr uint32_t kSmem = kBytes + 1024 + 384 > kAlone ? kBytes + 1024 + 384 : kAlone;
  static_assert(2 * (kSmem + 1024) > 228 * 1024, "room for one CTA only");
  static constexpr int kThreads = FP8 ? 640 : 384;
  static_assert(kSmem <= 232448, "shared memory of a CTA");
  static_assert(!TWO || DK <= 128, "two row tiles of wider heads leave no room for the keys");
};

// one lane of a warp that runs together
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(tm), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D (TMEM) = or += A (shared memory) * B (shared memory)
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// D (TMEM) = or += A (TMEM, two bf16 a column) * B (shared memory)
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// fp32 accumulator, bf16 operands, M = 128; b_mn: B lies along N instead of along K
constexpr uint32_t idesc_m128(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// The values as the right operand of the second product: a row per position (the product's
// K), 64-column boxes of 128-byte rows under the 128-byte swizzle; 16 KB from box to box along
// N, 1 KB from eight rows to the next eight along K.
__device__ __forceinline__ uint64_t desc_values(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(kBox >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// byte offset of 16-byte chunk `chunk` of row `row` in 64-column boxes under the 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
  return (uint32_t)(chunk >> 3) * kBox + (uint32_t)row * 128 + (uint32_t)(((chunk & 7) ^ (row & 7)) << 4);
}

// Codes -> bf16 operands.  An e4m3 byte s eeee mmm put at bit 4 of a bf16 (s 0000eeee mmm0000) is
// the code's value times 2^-120 (subnormal codes included: both types have the same step there), so
// one packed multiplication by 2^(e + 120) makes two operands; powers above bf16's largest, 2^127,
// in two steps.
struct RowScale { uint32_t first, second; };           // bf16 pairs; second: 1 unless e > 7
__device__ __forceinline__ RowScale row_scale(uint32_t byte) {
  if (byte == kScaleNan) return RowScale{0x7fc07fc0u, 0x3f803f80u};
  const uint32_t first = min(byte + 120u, 254u), second = 127u + (byte + 120u - first);
  return RowScale{(first << 7) * 0x10001u, (second << 7) * 0x10001u};
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// sixteen codes (one 16-byte chunk) -> two chunks; `top`: the largest magnitudes so far, of both halves of a pair
constexpr uint32_t kNanSize = 0x07f0u;                 // e4m3's own NaN, 0x7f or 0xff: it becomes 480 here
__device__ __forceinline__ void convert16(const uint4 &c, RowScale scale, bool twice, uint4 &lo, uint4 &hi, uint32_t &top) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t0 = __byte_perm(w[i], 0, 0x1404), t1 = __byte_perm(w[i], 0, 0x3424);     // two codes, each in the high byte of a half
    const uint32_t size0 = (t0 >> 4) & 0x07f007f0u, size1 = (t1 >> 4) & 0x07f007f0u;
    top = __vimax3_u16x2(top, size0, size1);
    o[2 * i] = mul_bf16x2(size0 | (t0 & 0x80008000u), scale.first);
    o[2 * i + 1] = mul_bf16x2(size1 | (t1 & 0x80008000u), scale.first);
  }
  if (twice) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = mul_bf16x2(o[i], scale.second);
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

// Four warps turn the codes of `n` tiles, one side's (keys or values, D bytes a row), into operands: half
// a tile at a time, half a row of it per thread.  A thread's chunks are every second one from a place
// that moves with the row: eight neighbouring rows are on different banks, in the codes and in
// the swizzled operand.  The next half's codes are fetched as soon as this one's are stored.  A stage
// is given back behind those stores, which cannot be made before its codes are in registers (given
// back right behind the loads, it was refilled under them).  The loop is short on purpose: one code for
// both sides and all scales takes 0.93 of the time of one for each (16384 positions, 24 rows a head:
// 44.6 and 48.0 us), unrolled over both halves with the next one's codes fetched ahead 62 us.
// Returns whether one of the thread's codes is e4m3's own NaN.
template <int D, int NS, int RAW>
__device__ __forceinline__ bool convert_tiles(const unsigned char *raw, uint32_t raw_stage, unsigned char *op, uint32_t raw_full,
                                              uint32_t raw_empty, uint32_t full, uint32_t empty, const uint8_t *scales, int first,
                                              int end, int n, volatile int *abort_flag) {
  constexpr int kChunks = D / 16, kMine = kChunks / 2;
  const int row = threadIdx.x & 63, part = (threadIdx.x >> 6) & 1, lane = threadIdx.x & 31;
  uint32_t from[kMine], to[kMine];
#pragma unroll
  for (int x = 0; x < kMine; ++x) {
    const int chunk = (row + part + 2 * x) % kChunks;
    from[x] = row * D + chunk * 16;
    to[x] = swizzled(row, 2 * chunk);                     // (the second one's is the same but for bit 4)
  }
  const auto key_of = [&](int i) { return first + i * kBlock + row; };
  const auto scale_at = [&](int i) { return i < 2 * n && key_of(i) < end ? (uint32_t)__ldg(scales + key_of(i)) : 0u; };
  const auto fetch = [&](int i, uint4 (&c)[kMine]) {
    const unsigned char *src = raw + i % RAW * raw_stage;
    const bool in = key_of(i) < end;                      // (behind the end stands whatever was there before)
#pragma unroll
    for (int x = 0; x < kMine; ++x) c[x] = in ? *reinterpret_cast<const uint4 *>(src + from[x]) : make_uint4(0, 0, 0, 0);
  };
  const auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
  uint4 c[kMine];
  uint32_t byte = scale_at(0);
  uint32_t top = 0;
  const auto nan_seen = [&] { return (top & 0xffffu) == kNanSize || (top >> 16) == kNanSize; };
  if (!wait(raw_full, 0)) return false;
  fetch(0, c);
#pragma unroll 1
  for (int i = 0; i < 2 * n; ++i) {
    const int st = (i >> 1) % NS;
    const bool more = i + 1 < 2 * n;
    const uint32_t next_byte = scale_at(i + 1);
    if (!(i & 1) && !wait(empty + 8 * st, (((i >> 1) / NS) & 1) ^ 1u)) return nan_seen();
    const bool in = key_of(i) < end;
    const RowScale scale = in ? row_scale(byte) : RowScale{0u, 0u};
    const bool twice = __any_sync(0xffffffffu, in && scale.second != 0x3f803f80u);
    unsigned char *dst = op + st * (uint32_t)(D / 64 * kBox) + (i & 1) * (kBlock * 128);
#pragma unroll
    for (int x = 0; x < kMine; ++x) {
      uint4 lo, hi;
      convert16(c[x], scale, twice, lo, hi, top);
      *reinterpret_cast<uint4 *>(dst + to[x]) = lo;
      *reinterpret_cast<uint4 *>(dst + (to[x] ^ 16u)) = hi;
    }
    if (i & 1) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(raw_empty + 8 * (i % RAW));
      if (i & 1) mbar_arrive(full + 8 * st);
    }
    if (more) {
      if (!wait(raw_full + 8 * ((i + 1) % RAW), ((i + 1) / RAW) & 1)) return nan_seen();
      fetch(i + 1, c);
    }
    byte = next_byte;
  }
  return nan_seen();
}

// A cache that somebody filled by a cast of their own may hold e4m3's NaN, and the conversion makes 480
// of it.  What such a code does is the same for every query row: with one in a key all scores are NaN, with one
// in a value its column.  So the conversion only notes that there was one, and at the end all threads of the CTA
// look through its run of codes once more and put NaN where it belongs in the partial result: cold, out of
// line.  (16384 positions, 24 and 512 rows a head: without the note 43.8 and 48.1 us, with it 44.8 and 48.6, with
// NaN put into the operands as they are made 45.5 and 48.6, with the note made by the two warps without a
// role 44.5 and 49.1.)
__device__ __noinline__ void mark_nan_codes(const uint8_t *k, int64_t k_bytes, const uint8_t *v, int64_t v_bytes, int dv, int rows,
                                            float *part, float *lse, uint32_t *found) {
  const float nan = __uint_as_float(0x7fc00000u);
  for (int64_t i = threadIdx.x; i < k_bytes; i += blockDim.x)
    if ((k[i] & 0x7f) == 0x7f) atomicOr(found, 1u);
  for (int64_t i = threadIdx.x; i < v_bytes; i += blockDim.x)
    if ((v[i] & 0x7f) == 0x7f) atomicOr(found + 1 + i % dv / 32, 1u << (i % 32));
  __syncthreads();
  if (found[0] != 0)
    for (int i = threadIdx.x; i < rows; i += blockDim.x) lse[i] = nan;
  for (int i = threadIdx.x; i < rows * dv; i += blockDim.x)
    if ((found[1 + i % dv / 32] >> (i % 32)) & 1) part[i] = nan;
}

// two fp32 operations at once
__device__ __forceinline__ unsigned long long pack_f32x2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack_f32x2(unsigned long long v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ unsigned long long fma_f32x2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add_f32x2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

constexpr float kNone = -3.0e38f;                // the maximum of no score, or of scores of -inf alone

// The largest score of a row, kNone at least.  In the last blocks (TAIL) only the first `keys`
// positions count.
template <bool TAIL>
__device__ __forceinline__ float row_top(uint32_t st_at, int keys) {
  float top[4] = {kNone, kNone, kNone, kNone};
#pragma unroll
  for (int x = 0; x < kBlock; x += 32) {
    uint32_t r[32];
    tc_ld32(st_at + x, r);
    tc_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float a = TAIL && x + 2 * e >= keys ? kNone : __uint_as_float(r[2 * e]);
      const float b = TAIL && x + 2 * e + 1 >= keys ? kNone : __uint_as_float(r[2 * e + 1]);
      top[e & 3] = fmaxf(top[e & 3], fmaxf(a, b));
    }
  }
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

// A row's exponentials against the maximum `m` into TMEM, bf16 pairs over the scores (a pair is
// stored behind the scores it replaces); returns the sum of the pairs as stored, so that the weights
// of a row add up to one (0 to 0.9 % of a call's time; summed before they are rounded, equal values of 1
// came out as 0.996 where most probabilities round the same way).
template <bool TAIL>
__device__ __forceinline__ float exponentials(uint32_t st_at, int keys, float scale_log2, float m) {
  unsigned long long sum[2] = {0ull, 0ull};
  const unsigned long long scale2 = pack_f32x2(scale_log2, scale_log2), m2 = pack_f32x2(-m, -m);
#pragma unroll
  for (int x = 0; x < kBlock; x += 32) {
    uint32_t r[32], p[16];
    tc_ld32(st_at + x, r);
    tc_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float2 t = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), scale2, m2));
      float a = exp2_approx(t.x), b = exp2_approx(t.y);
      if constexpr (TAIL) {
        a = x + 2 * e < keys ? a : 0.f;
        b = x + 2 * e + 1 < keys ? b : 0.f;
      }
      p[e] = pack_bf16x2(a, b);
      sum[e & 1] = add_f32x2(sum[e & 1], pack_f32x2(bf16_lo(p[e]), bf16_hi(p[e])));
    }
    tc_st16(st_at + x / 2, p);
  }
  const float2 s = unpack_f32x2(add_f32x2(sum[0], sum[1]));
  return s.x + s.y;
}

// Warps of a group that have one of its `rows` rows (one at least: a barrier counts them).  What
// the products hold in the other warps' rows is never read.
__device__ __forceinline__ int busy_warps(int rows) { return max(1, min(4, (rows + 31) / 32)); }

// grid = (runs of positions, row tiles, key heads)
template <int DK, int DV, bool FP8, bool TWO>
__global__ void __launch_bounds__(Layout<DK, DV, FP8, TWO>::kThreads, 1)
attn_prefix_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __nv_bfloat16 *__restrict__ q, Cache cache, Shape s, float *__restrict__ part,
                   float *__restrict__ part_lse, int32_t *__restrict__ status) {
  using L = Layout<DK, DV, FP8, TWO>;
  constexpr int NS = L::kStages, kRows = TWO ? 2 * kPrefixRows : kPrefixRows;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *aligned_base = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_smem = base, k_smem = q_smem + L::kAllQ, v_smem = k_smem + NS * L::kK, raw_smem = v_smem + NS * L::kV;
  const uint32_t bars = base + L::kBytes;
  const uint32_t k_full = bars, k_empty = k_full + 8 * 4, v_full = k_empty + 8 * 4, v_empty = v_full + 8 * 4;
  const uint32_t s_full = v_empty + 8 * 4, p_full = s_full + 8 * 4;                            // [group][buffer]
  // [group][buffer]; waited for at need only, so the two buffers' barriers are apart: a phase that
  // is waited for ends before the barrier's next one can, whenever the waiting warp comes by
  const uint32_t pv_done = p_full + 8 * 4;
  const uint32_t rk_full = pv_done + 8 * 4, rv_full = rk_full + 8 * 4, r_empty = rv_full + 8 * 4;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(aligned_base + L::kBytes + 8 * (10 * 4));
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  uint32_t *nan_found = tmem_slot + 2;                  // a NaN among the codes: at all; among the keys', in a column (four words)

  // (the warp's number and the TMEM address as values that are the same for the whole warp: the
  // instructions that issue products and copies take uniform registers)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int hk = blockIdx.z, rt = blockIdx.y;
  const int all_tiles = (s.shared_len + kKeys - 1) / kKeys;
  const int least = all_tiles / (int)gridDim.x, longer = all_tiles - least * (int)gridDim.x;      // (the first runs are one tile longer)
  const int tile0 = (int)blockIdx.x * least + min((int)blockIdx.x, longer), tile1 = tile0 + least + ((int)blockIdx.x < longer ? 1 : 0);
  const int n = tile1 - tile0;                          // tiles of this run, at least one
  const int blocks = TWO ? 2 * n : n;                   // of each group
  const int rows = min(kRows, s.B * s.group - rt * kRows);
  const int busy_of[2] = {busy_warps(rows), busy_warps(TWO ? rows - kPrefixRows : rows)};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(k_full + 8 * i, FP8 ? 4 : 1); mbar_init(k_empty + 8 * i, 1);
      mbar_init(v_full + 8 * i, FP8 ? 4 : 1); mbar_init(v_empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1); mbar_init(p_full + 8 * i, busy_of[i >> 1]);
      mbar_init(pv_done + 8 * i, 1);
      mbar_init(rk_full + 8 * i, 1); mbar_init(rv_full + 8 * i, 1); mbar_init(r_empty + 8 * i, 8);
    }
    *abort_flag = 0;
    for (int i = 0; i < 6; ++i) nan_found[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait();
  // (behind the wait: a CTA that started early would hold the tensor memory that one of a launch before this
  // one, a library's too, may still have to get; 0.1 us of the calls that are measured)
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Loads of a tile of bf16 keys or values; positions behind the last shared one lie outside the
  // tensor map: zeros.
  const auto load_keys = [&](int i) {
    const int st = i % NS;
    mbar_expect_tx(k_full + 8 * st, L::kK);
#pragma unroll
    for (int x = 0; x < DK / 64; ++x) tma_load_3d(k_smem + st * L::kK + x * kBox, &tm_k, k_full + 8 * st, x * 64, hk, (tile0 + i) * kKeys);
  };
  const auto load_values = [&](int i) {
    const int st = i % NS;
    mbar_expect_tx(v_full + 8 * st, L::kV);
#pragma unroll
    for (int x = 0; x < DV / 64; ++x) tma_load_3d(v_smem + st * L::kV + x * kBox, &tm_v, v_full + 8 * st, x * 64, hk, (tile0 + i) * kKeys);
  };
  // The first ones by the thread that made the barriers, so that they are on their way while the queries
  // are fetched (32 sequences, 8192 positions: 0.7 us less; codes, whose loads are smaller and
  // wait for their conversion, gained nothing).
  if (!FP8 && threadIdx.x == 0)
    for (int i = 0; i < NS && i < n; ++i) { load_keys(i); load_values(i); }
  // the tile's query rows, zeros behind the last one
  const bool q_vec = s.q_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  for (int i = threadIdx.x; i < kRows * (DK / 8); i += L::kThreads) {
    const int row = i / (DK / 8), chunk = i - row * (DK / 8);
    const uint32_t at = row / kPrefixRows * L::kQ + swizzled(row % kPrefixRows, chunk);
    const int r = min(rt * kRows + row, s.B * s.group - 1), b = r / s.group, h = hk * s.group + r - b * s.group;
    const __nv_bfloat16 *src = q + b * s.q_stride + (size_t)h * DK + chunk * 8;
    if (q_vec) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + at), "l"(src), "r"(row < rows ? 16 : 0) : "memory");
    } else {
      const unsigned short *e = reinterpret_cast<const unsigned short *>(src);
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row < rows)
        x = make_uint4(e[0] | ((uint32_t)e[1] << 16), e[2] | ((uint32_t)e[3] << 16), e[4] | ((uint32_t)e[5] << 16),
                       e[6] | ((uint32_t)e[7] << 16));
      *reinterpret_cast<uint4 *>(aligned_base + at) = x;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  // group w: score buffers at s_tmem + (2 w + 0, 1) * 64, accumulator at o_tmem + w * DV
  const uint32_t s_tmem = tmem, o_tmem = tmem + 4 * kBlock;

  if (warp == 0) {
    if constexpr (FP8) {
      const size_t row0 = (size_t)hk * s.s_max;
      for (int i = 0; i < 2 * n; ++i) {
        const int st = i % L::kRaw, key = tile0 * kKeys + i * kBlock;
        const uint32_t keys = max(0, min(kBlock, s.shared_len - key)), dst = raw_smem + st * (L::kRawK + L::kRawV);
        if (!__all_sync(0xffffffffu, mbar_wait(r_empty + 8 * st, ((i / L::kRaw) & 1) ^ 1u, abort_flag))) break;
        if (elect_one()) {
          mbar_expect_tx(rk_full + 8 * st, keys * DK);             // (no position: the barrier completes at once)
          if (keys > 0) bulk_load(dst, static_cast<const uint8_t *>(cache.k) + (row0 + key) * DK, keys * DK, rk_full + 8 * st);
          mbar_expect_tx(rv_full + 8 * st, keys * DV);
          if (keys > 0)
            bulk_load(dst + L::kRawK, static_cast<const uint8_t *>(cache.v) + (row0 + key) * DV, keys * DV, rv_full + 8 * st);
        }
      }
    } else {
      for (int i = NS; i < n; ++i) {
        const uint32_t ph = ((i / NS) & 1) ^ 1u;
        if (!__all_sync(0xffffffffu, mbar_wait(k_empty + 8 * (i % NS), ph, abort_flag))) break;
        if (elect_one()) load_keys(i);
        if (!__all_sync(0xffffffffu, mbar_wait(v_empty + 8 * (i % NS), ph, abort_flag))) break;
        if (elect_one()) load_values(i);
      }
    }
  } else if (warp == 1) {
    // (one and the same lane issues everything: completion is tracked per thread)
    const bool leader = elect_one();
    constexpr uint32_t id_s = idesc_m128(kBlock, false), id_o = idesc_m128(DV, true);
    constexpr uint32_t half_rows = kBlock * 128 >> 4;         // a tile's second half, in descriptor units
    const uint64_t q_desc = umma_desc_sw128(q_smem), k_desc = umma_desc_sw128(k_smem), v_desc = desc_values(v_smem);
    // block j of a group: tile, and which half of it
    const auto tile_of = [](int j) { return TWO ? j >> 1 : j; };
    const auto half_of = [](int j, int w) { return TWO ? j & 1 : w; };
    const auto wait = [&](uint32_t bar, uint32_t parity) {
      const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
      tc_fence_after();
      return ok;
    };
    // scores of block j of group w
    const auto scores = [&](int j, int w) {
      const int i = tile_of(j), st = i % NS;
      if (w == 0 && (!TWO || !(j & 1)) && !wait(k_full + 8 * st, (i / NS) & 1)) return false;
      if (leader) {
        const uint64_t a = q_desc + (TWO ? w * (L::kQ >> 4) : 0), b = k_desc + (uint64_t)(st * (L::kK >> 4) + half_of(j, w) * half_rows);
#pragma unroll
        for (int x = 0; x < DK / 16; ++x) {
          const uint64_t off = (uint64_t)((x >> 2) * (kBox >> 4) + (x & 3) * 2);
          tc_mma_ss(s_tmem + (2 * w + (j & 1)) * kBlock, a + off, b + off, id_s, x > 0);
        }
        tc_commit(s_full + 8 * (2 * w + (j & 1)));
        if (w == 1 && (!TWO || (j & 1))) tc_commit(k_empty + 8 * st);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    for (int j = 0; j < 2 && j < blocks; ++j) ok = ok && scores(j, 0) && scores(j, 1);
    for (int j = 0; ok && j < blocks; ++j) {
      const int i = tile_of(j), st = i % NS;
      if ((!TWO || !(j & 1)) && !wait(v_full + 8 * st, (i / NS) & 1)) break;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        ok = ok && wait(p_full + 8 * (2 * w + (j & 1)), (j >> 1) & 1);
        if (ok && leader) {
          const uint64_t b = v_desc + (uint64_t)(st * (L::kV >> 4) + half_of(j, w) * half_rows);
#pragma unroll
          for (int x = 0; x < kBlock / 16; ++x)
            tc_mma_ts(o_tmem + w * DV, s_tmem + (2 * w + (j & 1)) * kBlock + x * 8, b + (uint64_t)(x * (2048 >> 4)), id_o, j > 0 || x > 0);
          tc_commit(pv_done + 8 * (2 * w + (j & 1)));
          if (w == 1 && (!TWO || (j & 1))) tc_commit(v_empty + 8 * st);
        }
        __syncwarp();
        // (block j + 2's scores go where this block's probabilities are: products run in the order of their issue)
        if (ok && j + 2 < blocks) ok = scores(j + 2, w);
      }
    }
  } else if (warp >= kSoftmaxWarp && warp < kConvertWarp) {
    const int w = (warp - kSoftmaxWarp) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_at = (uint32_t)(warp & 3) * 32u << 16;
    const uint32_t ot_at = o_tmem + w * DV + lane_at;
    float m = kNone, l = 0.f;
    bool ok = true;
    const bool busy = (warp & 3) < busy_of[w];
    for (int j = 0; busy && j < blocks; ++j) {
      const uint32_t st_at = s_tmem + (2 * w + (j & 1)) * kBlock + lane_at;
      ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * (2 * w + (j & 1)), (j >> 1) & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      const int keys = s.shared_len - tile0 * kKeys - (TWO ? j * kBlock : j * kKeys + w * kBlock);
      const bool whole = keys >= kBlock;
      const float top = (whole ? row_top<false>(st_at, keys) : row_top<true>(st_at, keys)) * s.scale_log2;
      if (__any_sync(0xffffffffu, top > m + kLazy)) {
        const float up = fmaxf(m, top), f = exp2_approx(m - up);
        l *= f;
        m = up;
        if (j > 0) {
          // (block j - 2's product into the accumulator is behind these scores; block j - 1's may be under way)
          ok = __all_sync(0xffffffffu, mbar_wait(pv_done + 8 * (2 * w + ((j - 1) & 1)), ((j - 1) >> 1) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int x = 0; x < DV; x += 32) {
            uint32_t r[32], h[16];
            tc_ld32(ot_at + x, r);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) h[e] = __float_as_uint(__uint_as_float(r[e]) * f);
            tc_st16(ot_at + x, h);
#pragma unroll
            for (int e = 0; e < 16; ++e) h[e] = __float_as_uint(__uint_as_float(r[16 + e]) * f);
            tc_st16(ot_at + x + 16, h);
          }
        }
      }
      l += whole ? exponentials<false>(st_at, keys, s.scale_log2, m) : exponentials<true>(st_at, keys, s.scale_log2, m);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 8 * (2 * w + (j & 1)));
    }
    // A row's result: its accumulator over its sum.  Groups on the two halves of one row tile
    // first agree on the weights of their sums.  Rows go through shared memory (every product is
    // done, so the operands' place is free) to be written whole.
    const auto groups_sync = [&] {
      if (TWO) asm volatile("bar.sync %0, 128;" ::"r"(2 + w) : "memory");
      else asm volatile("bar.sync 1, 256;" ::: "memory");
    };
    // (completion is in order: the last block's product is behind all others)
    if (ok) ok = __all_sync(0xffffffffu, mbar_wait(pv_done + 8 * (2 * w + ((blocks - 1) & 1)), ((blocks - 1) >> 1) & 1, abort_flag));
    tc_fence_after();
    asm volatile("bar.sync 1, 256;" ::: "memory");                                       // both groups' products
    constexpr int kPitch = DV + 4;
    float2 *sums = reinterpret_cast<float2 *>(aligned_base);                             // [2][128]
    float *rows_at = reinterpret_cast<float *>(aligned_base + 4096);                     // [2][128][kPitch]
    static_assert(4096 + 2 * kPrefixRows * kPitch * 4 <= L::kBytes, "room for the accumulators");
    float most = m, sum = l, f = l == 0.f ? 0.f : 1.f / l;
    if constexpr (!TWO) {
      sums[w * kPrefixRows + row] = make_float2(m, l);
      groups_sync();
      const float2 other = sums[(w ^ 1) * kPrefixRows + row];
      most = fmaxf(m, other.x);
      const float mine = exp2_approx(m - most);
      sum = l * mine + other.y * exp2_approx(other.x - most);
      f = sum == 0.f ? 0.f : mine / sum;
    }
    float4 *row_at = reinterpret_cast<float4 *>(rows_at + (w * kPrefixRows + row) * kPitch);
#pragma unroll 1
    for (int x = 0; busy && x < DV; x += 32) {
      uint32_t r[32];
      tc_ld32(ot_at + x, r);
      tc_wait_ld();
#pragma unroll
      for (int e = 0; e < 32; e += 4)
        row_at[(x + e) / 4] = sum == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                         : make_float4(__uint_as_float(r[e]) * f, __uint_as_float(r[e + 1]) * f,
                                                       __uint_as_float(r[e + 2]) * f, __uint_as_float(r[e + 3]) * f);
    }
    groups_sync();
    if (ok) {
      const size_t slot_row = (((size_t)hk * gridDim.y + rt) * gridDim.x + blockIdx.x) * s.pre_rows;
      const int r0 = TWO ? w * kPrefixRows : 0, here = min(kPrefixRows, rows - r0), threads = TWO ? 128 : 256;
#pragma unroll 4
      for (int i = threadIdx.x - kSoftmaxWarp * 32 - r0; i < here * (DV / 4); i += threads) {
        const int r = i / (DV / 4), col = i - r * (DV / 4);
        float4 o = *reinterpret_cast<const float4 *>(rows_at + (r0 + r) * kPitch + col * 4);
        if constexpr (!TWO) {
          const float4 t = *reinterpret_cast<const float4 *>(rows_at + (kPrefixRows + r) * kPitch + col * 4);
          o = make_float4(o.x + t.x, o.y + t.y, o.z + t.z, o.w + t.w);
        }
        *reinterpret_cast<float4 *>(part + (slot_row + r0 + r) * DV + col * 4) = o;
      }
      if ((TWO || w == 0) && r0 + row < rows) part_lse[slot_row + r0 + row] = sum == 0.f ? -INFINITY : most + log2f(sum);
    }
    tc_fence_before();
  } else if (FP8 && warp >= kConvertWarp) {
    const size_t row0 = (size_t)hk * s.s_max;
    const int first = tile0 * kKeys, end = s.shared_len;
    const bool keys_side = warp < kConvertWarp + 4;
    const unsigned char *raw = aligned_base + (raw_smem - base) + (keys_side ? 0 : L::kRawK);
    unsigned char *op = aligned_base + ((keys_side ? k_smem : v_smem) - base);
    const uint8_t *scales = (keys_side ? cache.ks : cache.vs) + row0;
    const uint32_t raw_full = keys_side ? rk_full : rv_full, full = keys_side ? k_full : v_full, empty = keys_side ? k_empty : v_empty;
    bool nan;
    if (DK == DV || keys_side)
      nan = convert_tiles<DK, NS, L::kRaw>(raw, L::kRawK + L::kRawV, op, raw_full, r_empty, full, empty, scales, first, end, n, abort_flag);
    else
      nan = convert_tiles<DV, NS, L::kRaw>(raw, L::kRawK + L::kRawV, op, raw_full, r_empty, full, empty, scales, first, end, n, abort_flag);
    if (nan) atomicOr(nan_found, 1u);
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && status) atomicExch(status, 1);
    // what this CTA should have found is not known: NaN, for every output that is joined from it
    const size_t slot_row = (((size_t)hk * gridDim.y + rt) * gridDim.x + blockIdx.x) * s.pre_rows;
    for (int i = threadIdx.x; i < rows; i += L::kThreads) part_lse[slot_row + i] = __uint_as_float(0x7fc00000u);
    const unsigned long long t0 = gtime_ns();
    while (gtime_ns() - t0 < 2000000ull) __nanosleep(1000);       // copies in flight
    __syncthreads();
  }
  if (FP8 && nan_found[0] != 0) {
    const int64_t slot_row = (((int64_t)hk * gridDim.y + rt) * gridDim.x + blockIdx.x) * s.pre_rows;
    const int64_t row0 = (int64_t)hk * s.s_max + (int64_t)tile0 * kKeys, keys = min((int64_t)n * kKeys, s.shared_len - (int64_t)tile0 * kKeys);
    mark_nan_codes(static_cast<const uint8_t *>(cache.k) + row0 * DK, keys * DK, static_cast<const uint8_t *>(cache.v) + row0 * DV,
                   keys * DV, DV, rows, part + slot_row * DV, part_lse + slot_row, nan_found + 1);
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// The shared rows of a bf16 cache as [shared_len][n_kv][d], boxes of 64 columns, one head, 128 positions.
int32_t encode_rows(CUtensorMap *tm, const void *base, int d, int n_kv, int shared_len) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(SB_E_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)n_kv, (cuuint64_t)shared_len};
  cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)d * n_kv * 2};
  cuuint32_t box[3] = {64, 1, kKeys}, step[3] = {1, 1, 1};
  const CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SB_E_CUDA, "cuTensorMapEncodeTiled of the shared rows failed with CUresult %d", (int)r);
  return SB_OK;
}

template <int DK, int DV, bool FP8, bool TWO>
int32_t launch(const __nv_bfloat16 *q, const Cache &cache, const Shape &s, float *part, float *lse, int32_t *status,
               cudaStream_t stream) {
  using L = Layout<DK, DV, FP8, TWO>;
  CUtensorMap tm_k = {}, tm_v = {};
  if (!FP8) {
    int32_t rc = encode_rows(&tm_k, cache.k, DK, s.n_kv, s.shared_len);
    if (rc == SB_OK) rc = encode_rows(&tm_v, cache.v, DV, s.n_kv, s.shared_len);
    if (rc != SB_OK) return rc;
  }
  auto kern = attn_prefix_kernel<DK, DV, FP8, TWO>;
  // once per device and instance (setting it twice does no harm)
  static std::atomic<uint64_t> opted_in{0};
  int dev = 0;
  SB_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (!(opted_in.load(std::memory_order_relaxed) & bit)) {
    SB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem));
    opted_in.fetch_or(bit, std::memory_order_relaxed);
  }
  const dim3 grid(s.pre_splits, s.pre_tiles, s.n_kv);
  SB_CUDA_CHECK(launch_pdl(kern, grid, dim3(L::kThreads), L::kSmem, stream, tm_k, tm_v, q, cache, s, part, lse, status));
  SB_LAUNCH_CHECK();
  return SB_OK;
}

}  // namespace

void plan_prefix(Shape &s, int dk) {
  const int rows = s.B * s.group;                       // (at most 2^22)
  s.pre_tile_rows = rows > kPrefixRows && dk <= 128 ? 2 * kPrefixRows : kPrefixRows;
  s.pre_tiles = (rows + s.pre_tile_rows - 1) / s.pre_tile_rows;
  s.pre_rows = rows < s.pre_tile_rows ? rows : s.pre_tile_rows;
  const int64_t tiles = (s.shared_len + kKeys - 1) / kKeys, heads = (int64_t)s.n_kv * s.pre_tiles;
  const int64_t fit = 148 / heads;
  s.pre_splits = (int)(fit < 1 ? 1 : fit < tiles ? fit : tiles);
}

int32_t launch_attn_prefix(bool fp8, int dk, int dv, const __nv_bfloat16 *q, const Cache &cache, const Shape &s, float *part,
                           float *lse, int32_t *status, cudaStream_t stream) {
  const bool two = s.pre_tile_rows > kPrefixRows;
  if (dk == 192) return (fp8 ? launch<192, 128, true, false> : launch<192, 128, false, false>)(q, cache, s, part, lse, status, stream);
  if (dk == 128)
    return (fp8 ? two ? launch<128, 128, true, true> : launch<128, 128, true, false>
                : two ? launch<128, 128, false, true> : launch<128, 128, false, false>)(q, cache, s, part, lse, status, stream);
  return (fp8 ? two ? launch<64, 64, true, true> : launch<64, 64, true, false>
              : two ? launch<64, 64, false, true> : launch<64, 64, false, false>)(q, cache, s, part, lse, status, stream);
}

}  // namespace sb
