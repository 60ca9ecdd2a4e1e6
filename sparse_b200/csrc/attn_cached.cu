// Decode attention (one query per sequence) over a quantised cache, and over a cache whose
// first `shared_len` positions are the same for the whole batch and lie in sequence 0's
// rows only.  out[b, h] = sum_j p_j v_j,  p = softmax_j(scale * q[b, h] . k_j), over the
// positions j < seq_lens[b]; a sequence without positions gives zeros.
//
// Bound by the bytes of the cache, each of which should be read once: up to sixteen query heads
// that share a key head (and, over the shared positions, the sequences) are rows of one small
// matrix product.  More query heads than that are row tiles of sixteen, and each asks for the keys
// and values again (20 heads over one key head, 64 sequences of up to 16384 positions: 67 us for a
// cache of 136 MB, of which DRAM gives 179 MB and L2 the rest of twice 136). attn_stream_kernel
// turns it round, S^T = K Q^T and O^T = V^T P^T, so that the keys fill the 16-row side of the
// warp-level MMA and up to eight query rows its 8-column side.  Keys and values then go from global
// memory straight into the fragments of the instruction (which positions of a row a lane holds is
// free, as long as both operands agree), without shared memory: what counts is bytes in flight, and
// each warp has the keys and values of its next step (16 positions of bf16, 32 quantised: 8 KB) on
// the way while it works on the present ones.  The tensor core's own rate is no concern here (13 %
// busy), which is why the warp-level instruction does: an accumulator in tensor memory would need
// the keys in shared memory first.
//
// The work, all tiles (64 positions of bf16, 128 quantised) of all sequences and heads in one
// line, is cut into equal runs, one per CTA, whatever the lengths are; a head that ends in the
// middle of a run or reaches over several leaves a partial result for each, and
// attn_join_kernel joins those.
//
// Measured (repeated in a graph, inputs larger than L2 in turn): 64 sequences of 0 to 16384
// quantised positions, 32 query and 8 key heads of 128: 171 us, 6.3 TB/s, in the first ten
// milliseconds of a loop and 189 us, 5.7 TB/s, when it goes on; 8 x 2048, 16 heads: 20 us for 68
// MB, of which 3 to 4.5 us pass before the first scores (1 us to read the lengths and find the run,
// a load from DRAM), a tile takes 1.3 us, the end of a piece 1.2 us, so that CTAs of four tiles are
// through at 10.5 to 13 us, those of five at 12.5 to 14.5, those of five in two pieces at 14 to 16,
// and the second kernel is at 19; one sequence of 1000: 7.2 us, all of it round trips.  A join
// inside this kernel (marks in memory, the last CTA joins) has one launch less but five round trips
// to L2 behind one another instead of three: 9.6 us for the sequence of 1000, 23.7 us for 8 x 2048.
#include <math.h>

#include <type_traits>

#include "attn_cached.cuh"

namespace sb {
namespace {

constexpr int kThreads = 128;                 // four warps, a quarter of a tile's positions each
// Positions of a tile: a step of a warp is 32 quantised or 16 bf16 positions, 8 KB of heads of 128 either way.
template <bool FP8> constexpr int kTile = FP8 ? 128 : 64;
constexpr int kLeastTile = 64;
constexpr int kMaxCtas = 444;                 // 148 SMs, three CTAs each

// The line of tiles: first the shared positions (per key head and row tile), then
// sequence by sequence, key head by key head, row tile by row tile.
__device__ __forceinline__ int seq_len(const Shape &s, const int32_t *seq_lens, int b) { return min(max(__ldg(seq_lens + b), 0), s.s_max); }
// A sequence that ends inside the shared positions does not take part in their common pass:
// its own tiles are those positions, up to its end.
__device__ __forceinline__ int own_begin(const Shape &s, int len) { return len >= s.shared_len ? s.shared_len : 0; }
template <bool FP8> __device__ __forceinline__ int own_tiles(const Shape &s, int len) {
  return (len - own_begin(s, len) + kTile<FP8> - 1) / kTile<FP8>;
}
template <bool FP8> __device__ __forceinline__ int pre_tiles(const Shape &s) {
  return s.pre_row_tiles > 0 ? (s.shared_len + kTile<FP8> - 1) / kTile<FP8> : 0;
}

// The line in equal runs: the first `longer` CTAs have one tile more than the others.
struct Runs {
  int least, longer;
  __device__ __forceinline__ int first(int cta) const { return cta * least + min(cta, longer); }
  __device__ __forceinline__ int cta_of(int tile) const {
    const int head = longer * (least + 1);
    return tile < head ? tile / (least + 1) : longer + (tile - head) / least;
  }
};

__device__ __forceinline__ int warp_sum_int(int v) { return __reduce_add_sync(0xffffffffu, v); }

// ---- loads and fragments --------------------------------------------------------------------

__device__ __forceinline__ uint4 ldg_stream(const void *p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 ldg_stream8(const void *p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&v);
}

// The state of one warp over a run of positions, NT * 8 query rows (row 8 nt + 2c + r in
// registers [nt][r] of lanes with lane % 4 == c), U * 16 positions a step.
//
// Quantised: the keys' codes become fp16 (exact) and so do the queries, each row scaled by a
// power of two to a largest value in [1, 2) (bf16's eight bits fit; a value below 2^-14 of the
// row's largest is rounded to 2^-25 of that).  The row's and the key's powers of two
// multiply the fp32 score.  The weight of a value is its probability times the value's power of
// two, rounded to fp16 (2^-11) relative to a maximum of its own: powers of two that differ by
// more than fp16's range do not push a small value with all the probability out of it.  The sum is
// of the unrounded probabilities: 2^-11 is a quarter of what the output's own rounding may leave.
// bf16: probabilities are rounded to bf16 (2^-8, the type of the values they are multiplied
// with), and their sum is taken over the rounded ones.
template <int DK, int DV, bool FP8, int NT>
struct Stream {
  static constexpr int kBytes = FP8 ? 1 : 2;
  static constexpr int U = FP8 ? 2 : 1;
  static constexpr int KP = DK * kBytes / 64;          // 16-byte pieces a lane holds of a key
  static constexpr int CPL = DV / 8;                   // value columns of a lane
  static constexpr int VW = CPL * kBytes / 4;          // 4-byte words a lane holds of a value
  static constexpr int MT = DV / 16;
  static constexpr float kNone = -3.0e38f;             // the maximum of no score, or of scores of -inf alone

  uint4 k[U][2][KP];
  uint32_t v[U][4][VW];
  uint32_t k_scale, v_scale;                           // bytes of position `lane` of the step
  uint32_t q[NT][DK / 16][2];
  float q_factor[NT][2];
  float m[NT][2], l[NT][2];                            // running maximum (log2 units) and sum
  float mv[NT][2], r_v[NT][2];                         // quantised: maximum of the weights, 2^(m - mv): up to 2^127, for byte 0
  float acc[MT][NT][4];

  // the value columns of a lane: column(e), e < CPL
  static __device__ __forceinline__ int column(int g, int e) { return FP8 ? g * CPL + e : (e >> 3) * 64 + g * 8 + (e & 7); }

  // Where a lane reads: `kp` the first piece of its key of the step, `vp` the first word of its value.
  struct Place {
    const unsigned char *kp, *vp;
    const uint8_t *ks, *vs;
    size_t k_step, v_step;                             // bytes from a position to the next
    int left;                                          // positions from the step's first one to the segment's end
  };
  __device__ __forceinline__ void load_k(const Place &at, int g, int c, int lane) {
    if (at.left >= 16 * U) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < KP; ++i) k[u][r][i] = ldg_stream(at.kp + (16 * u + 8 * r) * at.k_step + i * 64);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < KP; ++i)
            k[u][r][i] = 16 * u + 8 * r + g < at.left ? ldg_stream(at.kp + (16 * u + 8 * r) * at.k_step + i * 64)
                                                      : make_uint4(0, 0, 0, 0);
    }
    if constexpr (FP8) {
      const bool in = lane < at.left;
      k_scale = in ? __ldg(at.ks + lane) : 0u;
      v_scale = in ? __ldg(at.vs + lane) : 0u;
    }
  }
  __device__ __forceinline__ void load_v_row(const unsigned char *p, uint32_t (&x)[VW]) {
    if constexpr (VW == 2) {
      const uint2 y = ldg_stream8(p);
      x[0] = y.x; x[1] = y.y;
    } else {
#pragma unroll
      for (int i = 0; i < VW / 4; ++i) {
        const uint4 y = ldg_stream(p + i * 128);
        x[4 * i] = y.x; x[4 * i + 1] = y.y; x[4 * i + 2] = y.z; x[4 * i + 3] = y.w;
      }
    }
  }
  // positions behind the end give zeros, whatever stands there
  __device__ __forceinline__ void load_v(const Place &at, int c) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * u + (r & 1) + 8 * (r >> 1);
        if (at.left >= 16 * U || j + 2 * c < at.left) {
          load_v_row(at.vp + j * at.v_step, v[u][r]);
        } else {
#pragma unroll
          for (int i = 0; i < VW; ++i) v[u][r][i] = 0;
        }
      }
  }

  // Query rows g (+ 8) of `rows` from shared memory ([row][DK]).  MMA step i takes four elements of a
  // lane, those of its word(s) of the key's piece, so a lane's elements of a 64-byte key piece
  // stand side by side in the query too.
  __device__ __forceinline__ void fetch(const __nv_bfloat16 *staged, int rows, int g, int c) {
    constexpr int kPerPiece = 16 / kBytes;             // elements of a 16-byte piece of a key
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < DK / 16; i += 2) {
        // eight elements: the words of MMA steps i and i + 1
        const int first = (i * 4 / kPerPiece) * (4 * kPerPiece) + c * kPerPiece + (i * 4) % kPerPiece;
        const uint4 x = nt * 8 + g < rows ? *reinterpret_cast<const uint4 *>(staged + (nt * 8 + g) * DK + first)
                                          : make_uint4(0, 0, 0, 0);
        q[nt][i][0] = x.x; q[nt][i][1] = x.y; q[nt][i + 1][0] = x.z; q[nt][i + 1][1] = x.w;
      }
  }
  // The rows just fetched, with nothing summed yet.
  __device__ __forceinline__ void begin(float scale_log2, int c) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < DK / 16; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          top = max(top, max(q[nt][s][half] & 0x7fffu, (q[nt][s][half] >> 16) & 0x7fffu));
      float factor = 1.f;
      if constexpr (FP8) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int x = top >= 0x7f80u ? 127 : max((int)(top >> 7), 1);       // the largest value's exponent byte
        const float down = x == 254 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)(254 - x) << 23);
        factor = __uint_as_float((uint32_t)x << 23);
#pragma unroll
        for (int s = 0; s < DK / 16; ++s)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            q[nt][s][half] = pack_f16x2(bf16_lo(q[nt][s][half]) * down, bf16_hi(q[nt][s][half]) * down);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // (row 2c + r is held by lanes of group 2c + r)
        q_factor[nt][r] = __shfl_sync(0xffffffffu, factor, (2 * c + r) * 4) * scale_log2;
        m[nt][r] = mv[nt][r] = kNone;
        r_v[nt][r] = 1.f;
        l[nt][r] = 0.f;
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][nt][i] = 0.f;
  }

  // s[u][nt]: scores of keys 16u + g (elements 0, 1: rows 2c, 2c + 1) and 16u + g + 8 (2, 3)
  __device__ __forceinline__ void scores(float (&s)[U][NT][4]) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][nt][i] = 0.f;
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const uint32_t a[4] = {k[u][0][i].x, k[u][0][i].y, k[u][0][i].z, k[u][0][i].w};
        const uint32_t b[4] = {k[u][1][i].x, k[u][1][i].y, k[u][1][i].z, k[u][1][i].w};
        if constexpr (FP8) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = e4m3x2_to_f16x2(a[w]), a2 = e4m3x2_to_f16x2(a[w] >> 16);
            const uint32_t a1 = e4m3x2_to_f16x2(b[w]), a3 = e4m3x2_to_f16x2(b[w] >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<true>(s[u][nt], a0, a1, a2, a3, q[nt][i * 4 + w][0], q[nt][i * 4 + w][1]);
          }
        } else {
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<false>(s[u][nt], a[2 * w], b[2 * w], a[2 * w + 1], b[2 * w + 1], q[nt][i * 2 + w][0], q[nt][i * 2 + w][1]);
        }
      }
    }
  }

  // Scores -> weights as the right-hand operand of the second product.  `left`: positions of
  // the step that count.  Weights are worked out against the maxima as they stand; where one
  // comes out above 2^kLazy (and in the first step) the maxima move and they are worked out again.
  __device__ __forceinline__ void weights(float (&s)[U][NT][4], uint32_t k_byte, uint32_t v_byte, int left, int g,
                                          uint32_t (&w)[U][NT][2]) {
    float vs[U][2];
    if constexpr (FP8) {
      const float mine_k = e8m0_value(k_byte), mine_v = e8m0_value(v_byte);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float ks = __shfl_sync(0xffffffffu, mine_k, 16 * u + 8 * h + g);
          vs[u][h] = __shfl_sync(0xffffffffu, mine_v, 16 * u + 8 * h + g);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) { s[u][nt][2 * h] *= ks; s[u][nt][2 * h + 1] *= ks; }
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u][nt][i] *= q_factor[nt][i & 1];
    if (left < 16 * U) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * u + 8 * (i >> 1) + g >= left) s[u][nt][i] = -INFINITY;
    }
    float p[U][NT][4], x[U][NT][4];
    const auto exponentials = [&] {
      bool over = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[u][nt][i] = exp2_approx(s[u][nt][i] - m[nt][i & 1]);
            top[i & 1] = fmaxf(top[i & 1], p[u][nt][i]);
            if constexpr (FP8) {
              x[u][nt][i] = p[u][nt][i] * vs[u][i >> 1] * r_v[nt][i & 1];
              top[i & 1] = fmaxf(top[i & 1], x[u][nt][i]);
            }
          }
        over |= fmaxf(top[0], top[1]) > (float)(1 << (int)kLazy);
      }
      return over;
    };
    if (__any_sync(0xffffffffu, exponentials())) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = kNone, topv = kNone;
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              top = fmaxf(top, s[u][nt][2 * h + r]);
              if constexpr (FP8) topv = fmaxf(topv, s[u][nt][2 * h + r] + log2f(vs[u][h]));
            }
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            if constexpr (FP8) topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, off));
          }
          top = fmaxf(top, m[nt][r]);
          float f = exp2_approx(m[nt][r] - top);
          l[nt][r] *= f;
          m[nt][r] = top;
          if constexpr (FP8) {
            topv = fmaxf(topv, mv[nt][r]);
            f = exp2_approx(mv[nt][r] - topv);
            mv[nt][r] = topv;
            r_v[nt][r] = exp2_approx(fminf(top - topv, 127.f));
          }
#pragma unroll
          for (int t = 0; t < MT; ++t) { acc[t][nt][r] *= f; acc[t][nt][2 + r] *= f; }
        }
      exponentials();
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pair;
          if constexpr (FP8) {
            pair = pack_f16x2(x[u][nt][2 * h], x[u][nt][2 * h + 1]);
            l[nt][0] += p[u][nt][2 * h];
            l[nt][1] += p[u][nt][2 * h + 1];
          } else {
            pair = pack_bf16x2(p[u][nt][2 * h], p[u][nt][2 * h + 1]);
            l[nt][0] += bf16_lo(pair);
            l[nt][1] += bf16_hi(pair);
          }
          w[u][nt][h] = transpose8x8(pair);
        }
  }

  __device__ __forceinline__ void values(const uint32_t (&w)[U][NT][2]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        if constexpr (FP8) {
          // bytes of two neighbouring positions side by side, then both to fp16 at once
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362u : 0x5140u;
            const uint32_t lo = __byte_perm(v[u][0][i], v[u][1][i], sel), hi = __byte_perm(v[u][2][i], v[u][3][i], sel);
            const uint32_t a0 = e4m3x2_to_f16x2(lo), a1 = e4m3x2_to_f16x2(lo >> 16);
            const uint32_t a2 = e4m3x2_to_f16x2(hi), a3 = e4m3x2_to_f16x2(hi >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<true>(acc[2 * i + half][nt], a0, a1, a2, a3, w[u][nt][0], w[u][nt][1]);
          }
        } else {
          const uint32_t a0 = __byte_perm(v[u][0][i], v[u][1][i], 0x5410), a1 = __byte_perm(v[u][0][i], v[u][1][i], 0x7632);
          const uint32_t a2 = __byte_perm(v[u][2][i], v[u][3][i], 0x5410), a3 = __byte_perm(v[u][2][i], v[u][3][i], 0x7632);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<false>(acc[i][nt], a0, a1, a2, a3, w[u][nt][0], w[u][nt][1]);
        }
      }
  }
};

// A piece's place in the line of tiles.
template <bool FP8>
struct Cursor {
  int b;                              // sequence, -1: the shared positions
  int w;                              // key head * row tiles + row tile
  int tile, tiles;                    // first tile of the piece in its segment, tiles of the segment
  int begin, end;                     // positions of the segment
  int row_tiles;

  __device__ __forceinline__ void enter(const Shape &s, const int32_t *seq_lens, int b_) {
    b = b_;
    w = tile = 0;
    row_tiles = b < 0 ? s.pre_row_tiles : s.row_tiles;
    const int len = b < 0 ? s.shared_len : seq_len(s, seq_lens, b);
    begin = b < 0 ? 0 : own_begin(s, len);
    end = len;
    tiles = b < 0 ? pre_tiles<FP8>(s) : own_tiles<FP8>(s, len);
  }
  __device__ __forceinline__ void next_segment(const Shape &s, const int32_t *seq_lens) {
    tile = 0;
    if (++w == s.n_kv * row_tiles) {
      int n = b;
      do { enter(s, seq_lens, ++n); } while (tiles == 0 && n < s.B - 1);
    }
  }
  __device__ __forceinline__ int segment(const Shape &s) const {
    return b < 0 ? w : s.n_kv * (s.pre_row_tiles + b * s.row_tiles) + w;
  }
  // whose rows hold the segment's positions
  __device__ __forceinline__ int home(const Shape &s) const { return b < 0 || end < s.shared_len ? 0 : b; }
};

// Partial results: slot = CTA + segment (from one piece of the line to the next at least one
// of the two grows), `rows` rows each: the row's attention over the piece, and the logarithm
// (base 2) of its sum of exponentials.
template <int DK, int DV, bool FP8, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 && DK <= 128 ? 3 : 2)
attn_stream_kernel(const __nv_bfloat16 *__restrict__ q, Cache cache, const int32_t *__restrict__ seq_lens, Shape s,
                   float *__restrict__ part, float *__restrict__ part_lse, int2 *__restrict__ pieces) {
  using St = Stream<DK, DV, FP8, NT>;
  constexpr int kStep = 16 * St::U;
  static_assert(4 * kStep == kTile<FP8>, "four warps cover a tile");
  __shared__ __align__(16) float s_out[4][NT * 8][DV];
  __shared__ float s_lse[4][NT * 8];
  __shared__ __align__(16) __nv_bfloat16 s_q[2][NT * 8 * DK];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  // this CTA's run: tiles first .. last-1 of the line
  const int own_heads = s.n_kv * s.row_tiles, pre_line = s.n_kv * s.pre_row_tiles * pre_tiles<FP8>(s);
  int sum = 0;
  for (int b = lane; b < s.B; b += 32) sum += own_tiles<FP8>(s, seq_len(s, seq_lens, b));
  const int total = pre_line + own_heads * warp_sum_int(sum);
  const Runs runs{total / (int)gridDim.x, total % (int)gridDim.x};
  const int first = runs.first(blockIdx.x), last = runs.first(blockIdx.x + 1);
  if (first >= last) return;
  Cursor<FP8> at;
  if (first < pre_line) {
    at.enter(s, seq_lens, -1);
    at.w = first / at.tiles;
    at.tile = first - at.w * at.tiles;
  } else {
    // the sequence among whose tiles the first one is: 32 sequences' tiles summed at a time
    int before = pre_line, b0 = 0;
    for (;; b0 += 32) {
      const int mine = b0 + lane < s.B ? own_heads * own_tiles<FP8>(s, seq_len(s, seq_lens, b0 + lane)) : 0;
      int upto = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += x;
      }
      const uint32_t beyond = __ballot_sync(0xffffffffu, before + upto > first);
      if (beyond != 0 || b0 + 32 >= s.B) {
        const int at_lane = beyond != 0 ? __ffs(beyond) - 1 : 0;
        before += __shfl_sync(0xffffffffu, upto - mine, at_lane);
        b0 += at_lane;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    at.enter(s, seq_lens, b0);
    at.w = (first - before) / at.tiles;
    at.tile = first - before - at.w * at.tiles;
  }

  St st;
  typename St::Place place;
  place.k_step = (FP8 ? 1 : (size_t)s.n_kv) * (DK * St::kBytes);
  place.v_step = (FP8 ? 1 : (size_t)s.n_kv) * (DV * St::kBytes);
  const auto enter = [&](const Cursor<FP8> &a) {
    const int hk = a.w / a.row_tiles, home = a.home(s), key = a.begin + a.tile * kTile<FP8> + warp * kStep;
    // row of the step's first position in the cache
    const size_t row = FP8 ? ((size_t)home * s.n_kv + hk) * s.s_max + key : ((size_t)home * s.s_max + key) * s.n_kv + hk;
    place.kp = static_cast<const unsigned char *>(cache.k) + row * (DK * St::kBytes) + g * place.k_step + c * 16;
    place.vp = static_cast<const unsigned char *>(cache.v) + row * (DV * St::kBytes) + 2 * c * place.v_step + g * (St::VW <= 4 ? St::VW * 4 : 16);
    if constexpr (FP8) { place.ks = cache.ks + row; place.vs = cache.vs + row; }
    place.left = a.end - key;
  };
  // The rows of a segment's queries on their way into shared memory, ahead of the piece.  Two
  // buffers: a warp that runs ahead writes the next piece's while another reads this one's.
  const bool q_vec = s.q_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  const auto rows_of = [&](const Cursor<FP8> &a) {
    return min(s.rows, (a.b < 0 ? s.B * s.group : s.group) - a.w % a.row_tiles * s.rows);
  };
  const auto stage = [&](const Cursor<FP8> &a, __nv_bfloat16 *dst) {
    const int hk = a.w / a.row_tiles, r0 = (a.w - hk * a.row_tiles) * s.rows, rows = rows_of(a);
    for (int i = threadIdx.x; i < rows * (DK / 8); i += kThreads) {
      const int row = i / (DK / 8), e = (i - row * (DK / 8)) * 8, r = r0 + row;
      const int b = a.b < 0 ? r / s.group : a.b, h = a.b < 0 ? r - b * s.group : r;
      const __nv_bfloat16 *src = q + b * s.q_stride + (size_t)(hk * s.group + h) * DK + e;
      if (q_vec) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                     ::"r"((uint32_t)__cvta_generic_to_shared(dst + row * DK + e)), "l"(src) : "memory");
      } else {
        for (int x = 0; x < 8; ++x) dst[row * DK + e + x] = src[x];
      }
    }
  };
  int buffer = 0;
  stage(at, s_q[0]);
  enter(at);
  st.load_k(place, g, c, lane);
  st.load_v(place, c);
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  for (int t = first; t < last;) {
    // one piece: tiles of one segment
    const Cursor<FP8> now = at;
    const int piece_end = min(last, t + now.tiles - now.tile);
    // the segment's slots follow one another: its first one, and how many, for attn_join_kernel
    if (now.tile == 0 && threadIdx.x == 0)
      pieces[now.segment(s)] = make_int2(blockIdx.x + now.segment(s), runs.cta_of(t + now.tiles - 1) - (int)blockIdx.x + 1);
    st.fetch(s_q[buffer], rows_of(now), g, c);
    buffer ^= 1;
    st.begin(s.scale_log2, c);
    for (; t < piece_end; ++t) {
      float sc[St::U][NT][4];
      uint32_t w[St::U][NT][2];
      st.scores(sc);
      const uint32_t k_byte = st.k_scale, v_byte = st.v_scale;
      const int left = place.left;
      // the next step's keys are on their way during the rest of this one, its values during the next's first half
      if (t + 1 < piece_end) {
        place.kp += kTile<FP8> * place.k_step;
        place.vp += kTile<FP8> * place.v_step;
        if constexpr (FP8) { place.ks += kTile<FP8>; place.vs += kTile<FP8>; }
        place.left -= kTile<FP8>;
      } else if (t + 1 < last) {
        at.next_segment(s, seq_lens);
        enter(at);
        stage(at, s_q[buffer]);
      }
      if (t + 1 < last) st.load_k(place, g, c, lane);
      st.weights(sc, k_byte, v_byte, left, g, w);
      st.values(w);
      if (t + 1 < last) st.load_v(place, c);
    }
    // the end of a piece: the four warps' results joined, one partial result
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float l = st.l[nt][r];
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        const int row = nt * 8 + 2 * c + r;
        const float f = l == 0.f ? 0.f : 1.f / l;
        // back from weights against mv: the inverse of r_v, which may be 2^-127, as a factor of its own
        // (with 1 / l in one number it would have few bits left, or none)
        const float back = FP8 ? exp2f(fmaxf(st.mv[nt][r] - st.m[nt][r], -127.f)) : 1.f;
        if (g == 0) s_lse[warp][row] = l == 0.f ? -INFINITY : st.m[nt][r] + log2f(l);
        // (four columns at a time; the four rows that a warp writes together go to different banks)
        float4 *dst = reinterpret_cast<float4 *>(s_out[warp][row]);
#pragma unroll
        for (int e = 0; e < DV / 8; e += 4)
          dst[(st.column(g, e) >> 2) ^ ((row >> 1) & 3)] =
              make_float4(st.acc[e >> 1][nt][r] * f * back, st.acc[e >> 1][nt][2 + r] * f * back,
                          st.acc[(e >> 1) + 1][nt][r] * f * back, st.acc[(e >> 1) + 1][nt][2 + r] * f * back);
      }
    asm volatile("cp.async.wait_all;" ::: "memory");     // the next piece's queries
    __syncthreads();
    const int rows = rows_of(now);
    const size_t slot_row = ((size_t)blockIdx.x + now.segment(s)) * s.rows;
    constexpr int kCols = DV / 32;                       // columns of a lane
    for (int row = warp; row < rows; row += 4) {
      float lse[4], top = -INFINITY, total_w = 0.f, o[kCols];
#pragma unroll
      for (int x = 0; x < 4; ++x) { lse[x] = s_lse[x][row]; top = fmaxf(top, lse[x]); }
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int e = 0; e < kCols; ++e) o[e] = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float f = exp2_approx(lse[x] - ref);
        total_w += f;
#pragma unroll
        for (int e = 0; e < kCols; ++e)
          o[e] += f * s_out[x][row][(((lane * kCols) >> 2) ^ ((row >> 1) & 3)) * 4 + ((lane * kCols + e) & 3)];
      }
      const float f = total_w == 0.f ? 0.f : 1.f / total_w;
      float *dst = part + (slot_row + row) * DV + lane * kCols;
      if constexpr (kCols == 4) *reinterpret_cast<float4 *>(dst) = make_float4(o[0] * f, o[1] * f, o[2] * f, o[3] * f);
      else *reinterpret_cast<float2 *>(dst) = make_float2(o[0] * f, o[1] * f);
      if (lane == 0) part_lse[slot_row + row] = total_w == 0.f ? -INFINITY : top + log2f(total_w);
    }
    __syncthreads();
  }
}

// One CTA per (sequence, key head, up to eight of its rows): each row's pieces of the shared
// positions and of its own, weighted by their sums of exponentials.  SHARE warps take a row (four
// where a key head has one row, two where it has two).  Bound by round trips to L2, so there are
// two behind one another: the length and the place of the pieces, then their rows and, at the same
// time, their logarithms (lane i looks after the weight of piece i of a round).
constexpr int kJoinRows = 8;
template <int DV, int SHARE>
__global__ void __launch_bounds__(kJoinRows * 32)
attn_join_kernel(const int32_t *__restrict__ seq_lens, Shape s, const int2 *__restrict__ pieces,
                 const float *__restrict__ part, const float *__restrict__ part_lse, const float *__restrict__ pre_part,
                 const float *__restrict__ pre_lse, __nv_bfloat16 *__restrict__ out) {
  constexpr int kCols = DV / 32, kAhead = SHARE == 1 ? 16 : 8, kRound = kAhead * SHARE;       // at most a warp's lanes
  using Vec = typename std::conditional<kCols == 4, float4, float2>::type;
  __shared__ __align__(16) float s_acc[kJoinRows][DV];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = min(s.group, kJoinRows), groups = (s.group + rows - 1) / rows;
  const int head = blockIdx.x / groups, b = head / s.n_kv, hk = head - b * s.n_kv;
  const int hg = (blockIdx.x - head * groups) * rows + warp / SHARE, mine_of = warp % SHARE;
  const bool row_ok = warp / SHARE < rows && hg < s.group;
  const int rt = min(hg, s.group - 1) / s.rows, r = b * s.group + hg;
  const int len = seq_len(s, seq_lens, b);
  const int2 own_at = __ldg(pieces + s.n_kv * (s.pre_row_tiles + b * s.row_tiles) + hk * s.row_tiles + rt);
  const int2 pre_at = s.pre_row_tiles > 0 ? __ldg(pieces + hk) : make_int2(0, 0);
  // pieces: of the shared positions, then of the sequence's own (whose place stands only where there are any)
  const float *pre = part, *pre_l = part_lse;
  size_t pre_first = (size_t)pre_at.x * s.rows + r, pre_step = s.rows;
  int n_pre = pre_at.y;
  if (s.pre_splits > 0) {
    const int tile = r / s.pre_tile_rows;
    pre = pre_part;
    pre_l = pre_lse;
    pre_step = s.pre_rows;
    pre_first = ((size_t)hk * s.pre_tiles + tile) * s.pre_splits * pre_step + r - tile * s.pre_tile_rows;
    n_pre = s.pre_splits;
  }
  if (s.shared_len == 0 || len < s.shared_len) n_pre = 0;
  const size_t own_first = (size_t)own_at.x * s.rows + hg - rt * s.rows;
  const int n = row_ok ? n_pre + (len > own_begin(s, len) ? own_at.y : 0) : 0;
  const auto row_of = [&](int i) { return i < n_pre ? pre_first + i * pre_step : own_first + (size_t)(i - n_pre) * s.rows; };
  float top = -INFINITY, sum = 0.f;
  __align__(16) float acc[kCols];
#pragma unroll
  for (int e = 0; e < kCols; ++e) acc[e] = 0.f;
  for (int i0 = 0; i0 < n; i0 += kRound) {
    Vec v[kAhead];
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const int i = i0 + y * SHARE + mine_of;
      v[y] = Vec{};
      if (i < n) v[y] = __ldg(reinterpret_cast<const Vec *>((i < n_pre ? pre : part) + row_of(i) * DV) + lane);
    }
    const int mine = i0 + lane;
    const bool ok = lane < kRound && mine < n;
    const float lse = ok ? __ldg((mine < n_pre ? pre_l : part_lse) + row_of(mine)) : -INFINITY;
    float most = lse;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
    most = fmaxf(most, top);
    const float ref = most == -INFINITY ? 0.f : most, f = exp2_approx(top - ref), w = exp2_approx(lse - ref);
    float weights = w;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) weights += __shfl_xor_sync(0xffffffffu, weights, off);
    sum = sum * f + weights;
#pragma unroll
    for (int e = 0; e < kCols; ++e) acc[e] *= f;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const float wy = __shfl_sync(0xffffffffu, w, y * SHARE + mine_of);
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] += wy * reinterpret_cast<const float *>(&v[y])[e];
    }
    top = most;
  }
  if (SHARE > 1) {
    *(reinterpret_cast<Vec *>(s_acc[warp]) + lane) = *reinterpret_cast<const Vec *>(acc);
    __syncthreads();
    if (mine_of != 0) return;
#pragma unroll
    for (int y = 1; y < SHARE; ++y)
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] += s_acc[warp + y][lane * kCols + e];
  }
  if (!row_ok) return;
  // no piece, or only such without weight: zeros
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t *dst = reinterpret_cast<uint32_t *>(out + ((size_t)b * s.n_q + hk * s.group + hg) * DV + lane * kCols);
#pragma unroll
  for (int e = 0; e < kCols; e += 2) dst[e / 2] = sum == 0.f ? 0u : pack_bf16x2(acc[e] * f, acc[e + 1] * f);
}

constexpr int kMaxRows = 16;

// How a call is cut; the rest of the shape is the caller's.  Up to sixteen rows share one
// pass of the streamed line over the prefix, more go through the tensor-core tiles.
void plan(Shape &s, int dk) {
  const int64_t pre_rows = s.shared_len > 0 ? (int64_t)s.B * s.group : 0;
  s.pre_splits = 0;
  s.pre_tile_rows = s.pre_tiles = s.pre_rows = 0;
  if (pre_rows > kMaxRows) plan_prefix(s, dk);
  s.rows = s.group > kMaxRows ? kMaxRows : s.group;
  if (pre_rows > s.rows && s.pre_splits == 0) s.rows = (int)pre_rows;
  s.row_tiles = (s.group + s.rows - 1) / s.rows;
  s.pre_row_tiles = pre_rows > 0 && s.pre_splits == 0 ? 1 : 0;
}
// Workspace: partial results of the streamed line and of the shared positions' tiles, then their
// logarithms, then the place of each segment's pieces.
int64_t segments(const Shape &s) { return (int64_t)s.n_kv * (s.pre_row_tiles + (int64_t)s.B * s.row_tiles); }
int64_t slot_rows(const Shape &s) { return (kMaxCtas + segments(s)) * s.rows; }
int64_t pre_slot_rows(const Shape &s) { return s.pre_splits > 0 ? prefix_slots(s) * s.pre_rows : 0; }

// A dependent launch of the stream kernel that asks for 100 of the SM's 228 KB as shared memory, which
// two or three of its CTAs take (two of 44.25 KB and 1 KB for the system each at most).  Its loads in flight live in what is left as L1:
// behind a kernel that used all of the shared memory the SM would stay as it is otherwise, and 64
// sequences of up to 16384 positions take 249 us with all of it against 171 with 66 to 148 KB.
template <typename... KArgs, typename... Args>
cudaError_t launch_stream(void (*kernel)(KArgs...), int ctas, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributePreferredSharedMemoryCarveout;
  attr[1].val.sharedMemCarveout = 44;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

template <int DK, int DV, bool FP8>
int32_t launch(const __nv_bfloat16 *q, const Cache &cache, const int32_t *seq_lens, const Shape &s, float *part,
               __nv_bfloat16 *out, int32_t *status, cudaStream_t st) {
  float *pre_part = part + slot_rows(s) * DV, *lse = pre_part + pre_slot_rows(s) * DV, *pre_lse = lse + slot_rows(s);
  int2 *pieces = reinterpret_cast<int2 *>((reinterpret_cast<uintptr_t>(pre_lse + pre_slot_rows(s)) + 7) & ~(uintptr_t)7);
  if (s.pre_splits > 0) {
    const int32_t rc = launch_attn_prefix(FP8, DK, DV, q, cache, s, pre_part, pre_lse, status, st);
    if (rc != SB_OK) return rc;
  }
  const int sms = sb_device_sm_count() > 0 ? sb_device_sm_count() : 148;
  // a CTA for every tile there can be, up to what the SMs hold at once
  const int64_t tiles = (int64_t)s.n_kv * ((int64_t)s.pre_row_tiles * ((s.shared_len + kTile<FP8> - 1) / kTile<FP8>) +
                                           (int64_t)s.B * s.row_tiles * ((s.s_max + kTile<FP8> - 1) / kTile<FP8>));
  const int per_sm = s.rows <= 8 && DK <= 128 ? 3 : 2, most = per_sm * sms < kMaxCtas ? per_sm * sms : kMaxCtas;
  const int ctas = tiles < most ? (int)tiles : most;
  auto kern = s.rows <= 8 ? attn_stream_kernel<DK, DV, FP8, 1> : attn_stream_kernel<DK, DV, FP8, 2>;
  SB_CUDA_CHECK(launch_stream(kern, ctas, st, q, cache, seq_lens, s, part, lse, pieces));
  SB_LAUNCH_CHECK();
  const int rows = s.group < kJoinRows ? s.group : kJoinRows, warps = rows < 4 ? 4 : rows;
  auto join = rows == 1 ? attn_join_kernel<DV, 4> : rows == 2 ? attn_join_kernel<DV, 2> : attn_join_kernel<DV, 1>;
  SB_CUDA_CHECK(launch_pdl(join, dim3(s.B * s.n_kv * ((s.group + rows - 1) / rows)), dim3(warps * 32), 0, st,
                           seq_lens, s, static_cast<const int2 *>(pieces), static_cast<const float *>(part),
                           static_cast<const float *>(lse), static_cast<const float *>(pre_part),
                           static_cast<const float *>(pre_lse), out));
  SB_LAUNCH_CHECK();
  return SB_OK;
}

template <bool FP8>
int32_t attend(const char *name, const sb_attn_cached_args *args, void *stream) {
  if (!args) return fail(SB_E_INVALID_ARG, "%s: null pointer", name);
  const sb_attn_cached_args &a = *args;
  const int B = a.B, n_q = a.n_q, n_kv = a.n_kv, dk = a.dk, dv = a.dv, s_max = a.s_max, shared_len = a.shared_len;
  const float scale = a.scale;
  int64_t q_stride = a.q_stride;
  const Cache cache = {a.k, a.v, static_cast<const uint8_t *>(a.scale_k), static_cast<const uint8_t *>(a.scale_v)};
  // (the line's tiles are counted in 32 bits)
  if (B < 0 || n_q < 1 || n_kv < 1 || n_kv > 65535 || n_q % n_kv != 0 || s_max < 1 || shared_len < 0 || shared_len > s_max ||
      (int64_t)B * n_q > (1 << 22) || (int64_t)B * n_q * (s_max / kLeastTile + 2) > (1ll << 30))
    return fail(SB_E_INVALID_ARG, "%s: bad shape (B=%d heads %d/%d s_max=%d shared %d)", name, B, n_q, n_kv, s_max, shared_len);
  if (!(scale >= 0.f) || !isfinite(scale)) return fail(SB_E_INVALID_ARG, "%s: scale must be finite and not negative", name);
  if (q_stride == 0) q_stride = (int64_t)n_q * dk;
  if (q_stride < (int64_t)n_q * dk) return fail(SB_E_INVALID_ARG, "%s: q_stride smaller than a token's heads", name);
  if (!((dk == 128 && dv == 128) || (dk == 192 && dv == 128) || (dk == 64 && dv == 64)))
    return fail(SB_E_UNSUPPORTED, "%s: head dims (%d,%d) not built (128/128, 192/128, 64/64)", name, dk, dv);
  if (B == 0) return SB_OK;
  if (!a.q || !cache.k || !cache.v || (FP8 && (!cache.ks || !cache.vs)) || !a.seq_lens || !a.ws || !a.out)
    return fail(SB_E_INVALID_ARG, "%s: null pointer", name);
  if (!aligned(cache.k, 16) || !aligned(cache.v, 16) || !aligned(a.ws, 16) || !aligned(a.out, 4))
    return fail(SB_E_INVALID_ARG, "%s: cache and workspace must be 16-byte aligned, out 4-byte", name);
  if (a.ws_bytes < sb_attn_cached_workspace_bytes(B, n_q, n_kv, dk, dv, s_max, shared_len))
    return fail(SB_E_WORKSPACE, "%s: workspace too small", name);
  Shape s = {B, n_q, n_kv, n_q / n_kv, s_max, shared_len, 0, 0, 0, 0, 0, 0, 0, q_stride, scale * 1.4426950408889634f};
  plan(s, dk);
  const __nv_bfloat16 *qq = static_cast<const __nv_bfloat16 *>(a.q);
  float *part = static_cast<float *>(a.ws);
  __nv_bfloat16 *oo = static_cast<__nv_bfloat16 *>(a.out);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dk == 128 ? launch<128, 128, FP8>(qq, cache, a.seq_lens, s, part, oo, a.status, st)
         : dk == 192 ? launch<192, 128, FP8>(qq, cache, a.seq_lens, s, part, oo, a.status, st)
                     : launch<64, 64, FP8>(qq, cache, a.seq_lens, s, part, oo, a.status, st);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" {

size_t sb_attn_cached_workspace_bytes(int32_t B, int32_t n_q, int32_t n_kv, int32_t dk, int32_t dv, int32_t s_max,
                                      int32_t shared_len) {
  if (B < 0 || dk < 1 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || dv < 1 || s_max < 1 || shared_len < 0 || (int64_t)B * n_q > (1 << 22))
    return 0;
  Shape s = {B, n_q, n_kv, n_q / n_kv, s_max, shared_len, 0, 0, 0, 0, 0, 0, 0, 0, 0.f};
  plan(s, dk);
  return (size_t)(slot_rows(s) + pre_slot_rows(s)) * (dv + 1) * sizeof(float) + (size_t)(segments(s) + 1) * sizeof(int2);
}

int32_t sb_attn_decode_shared(const sb_attn_cached_args *args, void *stream) {
  return attend<false>("sb_attn_decode_shared", args, stream);
}

int32_t sb_attn_decode_fp8(const sb_attn_cached_args *args, void *stream) {
  return attend<true>("sb_attn_decode_fp8", args, stream);
}

}  // extern "C"
