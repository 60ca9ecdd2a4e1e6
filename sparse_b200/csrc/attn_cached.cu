// Decode attention (one query per sequence) over a quantised cache, and over a cache whose
// first `shared_len` positions are the same for the whole batch and lie in sequence 0's
// rows only.  out[b, h] = sum_j p_j v_j,  p = softmax_j(scale * q[b, h] . k_j), over the
// positions j < seq_lens[b]; a sequence without positions gives zeros.
//
// Bound by the bytes of the cache, each of which should be read once: the query heads that
// share a key head (and, over the shared positions, the sequences) are rows of one small
// matrix product.  attn_stream_kernel turns it round, S^T = K Q^T and O^T = V^T P^T, so
// that the keys fill the 16-row side of the warp-level MMA and up to eight query rows its
// 8-column side.  Keys and values then go from global memory straight into the fragments of
// the instruction (which positions of a row a lane holds is free, as long as both operands
// agree), without shared memory: what counts is bytes in flight, and each warp has the 16
// keys and 16 values of its next step on the way while it works on the present ones.
//
// The work, all 64-position tiles of all sequences and heads in one line, is cut into
// equal runs, one per CTA, whatever the lengths are; a head that ends in the middle of a run
// or reaches over several leaves a partial result for each, and attn_join_kernel joins those.
#include <math.h>

#include "attn_cached.cuh"

namespace sb {
namespace {

constexpr int kThreads = 128;                 // four warps, 16 positions of a tile each
constexpr int kTile = 64;
constexpr int kMaxCtas = 592;                 // 148 SMs, four CTAs each

// The line of tiles: first the shared positions (per key head and row tile), then
// sequence by sequence, key head by key head, row tile by row tile.
__device__ __forceinline__ int seq_len(const Shape &s, const int32_t *seq_lens, int b) { return min(max(__ldg(seq_lens + b), 0), s.s_max); }
// A sequence that ends inside the shared positions does not take part in their common pass:
// its own tiles are those positions, up to its end.
__device__ __forceinline__ int own_begin(const Shape &s, int len) { return len >= s.shared_len ? s.shared_len : 0; }
__device__ __forceinline__ int own_tiles(const Shape &s, int len) { return (len - own_begin(s, len) + kTile - 1) / kTile; }
__device__ __forceinline__ int pre_tiles(const Shape &s) { return s.pre_row_tiles > 0 ? (s.shared_len + kTile - 1) / kTile : 0; }

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
// registers [nt][.][r] of lanes with lane % 4 == c).
//
// Quantised: the keys' codes become fp16 (exact) and so do the queries, each row scaled by a
// power of two to a largest value in [1, 2) (bf16's eight bits fit; what falls below 2^-24 of the
// row's largest is below the rounding of the fp32 sum).  The row's and the key's powers of two
// multiply the fp32 score.  The weight of a value is its probability times the value's power of
// two, rounded to fp16 (2^-11) relative to a maximum of its own: powers of two that differ by
// more than fp16's range do not push a small value with all the probability out of it.
// bf16: probabilities are rounded to bf16 (2^-8, the type of the values they are multiplied
// with), and their sum is taken over the rounded ones.
template <int DK, int DV, bool FP8, int NT>
struct Stream {
  static constexpr int kBytes = FP8 ? 1 : 2;
  static constexpr int KP = DK * kBytes / 64;          // 16-byte pieces a lane holds of a key
  static constexpr int CPL = DV / 8;                   // value columns of a lane
  static constexpr int VW = CPL * kBytes / 4;          // 4-byte words a lane holds of a value
  static constexpr int MT = DV / 16;

  uint4 k[2][KP];
  uint32_t v[4][VW];
  uint32_t scale_bytes[4];                             // of keys g, g + 8, of values g, g + 8
  uint32_t q[NT][DK / 16][2];
  float q_factor[NT][2];
  float m[NT][2], mv[NT][2], l[NT][2];
  float acc[MT][NT][4];

  // the value columns of a lane: column(e), e < CPL
  static __device__ __forceinline__ int column(int g, int e) { return FP8 ? g * CPL + e : (e >> 3) * 64 + g * 8 + (e & 7); }

  __device__ __forceinline__ void load_k(const Cache &cache, size_t row0, size_t row_step, int key, int end, int g, int c) {
    const unsigned char *base = static_cast<const unsigned char *>(cache.k);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int j = key + g + 8 * r;
      const unsigned char *p = base + (row0 + (size_t)j * row_step) * (DK * kBytes) + c * 16;
#pragma unroll
      for (int i = 0; i < KP; ++i) k[r][i] = j < end ? ldg_stream(p + i * 64) : make_uint4(0, 0, 0, 0);
      if constexpr (FP8) {
        scale_bytes[r] = j < end ? __ldg(cache.ks + row0 + j) : 0u;
        scale_bytes[2 + r] = j < end ? __ldg(cache.vs + row0 + j) : 0u;
      }
    }
  }
  // positions behind the end give zeros, whatever stands there
  __device__ __forceinline__ void load_v(const Cache &cache, size_t row0, size_t row_step, int key, int end, int g, int c) {
    const unsigned char *base = static_cast<const unsigned char *>(cache.v);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = key + 2 * c + (r & 1) + 8 * (r >> 1);
      const unsigned char *p = base + (row0 + (size_t)j * row_step) * (DV * kBytes) + g * (VW <= 4 ? VW * 4 : 16);
      if constexpr (VW == 2) {
        const uint2 x = j < end ? ldg_stream8(p) : make_uint2(0, 0);
        v[r][0] = x.x; v[r][1] = x.y;
      } else {
#pragma unroll
        for (int i = 0; i < VW / 4; ++i) {
          const uint4 x = j < end ? ldg_stream(p + i * 128) : make_uint4(0, 0, 0, 0);
          v[r][4 * i] = x.x; v[r][4 * i + 1] = x.y; v[r][4 * i + 2] = x.z; v[r][4 * i + 3] = x.w;
        }
      }
    }
  }

  // Query rows g (+ 8) of a segment: `row(r)` is the address of row r, or null.
  template <typename Row>
  __device__ __forceinline__ void begin(const Row &row, float scale_log2, int g, int c) {
    constexpr int kPerPiece = 16 / kBytes;             // elements of a 16-byte piece of a key
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const __nv_bfloat16 *src = row(nt * 8 + g);
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < DK / 16; ++s) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // MMA step s takes four elements of a lane: those of its word(s) of the key's piece
          const int first = (s * 4 / kPerPiece) * (4 * kPerPiece) + c * kPerPiece + (s * 4) % kPerPiece + 2 * half;
          const uint32_t lo = src ? __bfloat16_as_ushort(src[first]) : 0, hi = src ? __bfloat16_as_ushort(src[first + 1]) : 0;
          q[nt][s][half] = lo | (hi << 16);
          top = max(top, max(lo & 0x7fffu, hi & 0x7fffu));
        }
      }
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
        m[nt][r] = mv[nt][r] = -INFINITY;
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

  __device__ __forceinline__ void scores(float (&s)[NT][4]) const {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const uint32_t a[4] = {k[0][i].x, k[0][i].y, k[0][i].z, k[0][i].w}, b[4] = {k[1][i].x, k[1][i].y, k[1][i].z, k[1][i].w};
      if constexpr (FP8) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = e4m3x2_to_f16x2(a[w]), a2 = e4m3x2_to_f16x2(a[w] >> 16);
          const uint32_t a1 = e4m3x2_to_f16x2(b[w]), a3 = e4m3x2_to_f16x2(b[w] >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<true>(s[nt], a0, a1, a2, a3, q[nt][i * 4 + w][0], q[nt][i * 4 + w][1]);
        }
      } else {
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<false>(s[nt], a[2 * w], b[2 * w], a[2 * w + 1], b[2 * w + 1], q[nt][i * 2 + w][0], q[nt][i * 2 + w][1]);
      }
    }
  }

  // s: scores of keys g (elements 0, 1: rows 2c, 2c + 1) and g + 8 (2, 3) -> weights as the
  // right-hand operand of the second product
  __device__ __forceinline__ void weights(float (&s)[NT][4], const uint32_t (&bytes)[4], bool in0, bool in1, uint32_t (&w)[NT][2]) {
    float u[NT][4];
    bool over = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = i < 2 ? in0 : in1;
        float t = s[nt][i];
        if constexpr (FP8) t *= e8m0_value(bytes[i >> 1]);
        t *= q_factor[nt][i & 1];
        s[nt][i] = in ? t : -INFINITY;
        over |= s[nt][i] > m[nt][i & 1] + kLazy;
        if constexpr (FP8) {
          u[nt][i] = s[nt][i] + (bytes[2 + (i >> 1)] == kScaleNan ? NAN : (float)((int)bytes[2 + (i >> 1)] - 127));
          if (!in) u[nt][i] = -INFINITY;
          over |= u[nt][i] > mv[nt][i & 1] + kLazy;
        }
      }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = fmaxf(s[nt][r], s[nt][2 + r]), topv = FP8 ? fmaxf(u[nt][r], u[nt][2 + r]) : 0.f;
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            if constexpr (FP8) topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, off));
          }
          top = fmaxf(top, m[nt][r]);
          const float fl = m[nt][r] == -INFINITY ? 0.f : exp2_approx(m[nt][r] - top);
          l[nt][r] *= fl;
          m[nt][r] = top;
          float fa = fl;
          if constexpr (FP8) {
            topv = fmaxf(topv, mv[nt][r]);
            fa = mv[nt][r] == -INFINITY ? 0.f : exp2_approx(mv[nt][r] - topv);
            mv[nt][r] = topv;
          }
#pragma unroll
          for (int t = 0; t < MT; ++t) { acc[t][nt][r] *= fa; acc[t][nt][2 + r] *= fa; }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // only scores of -inf so far: they weigh exp(-inf - 0) = 0
        const float ref = m[nt][i & 1] == -INFINITY ? 0.f : m[nt][i & 1];
        p[i] = exp2_approx(s[nt][i] - ref);
        if constexpr (FP8) {
          l[nt][i & 1] += p[i];
          p[i] = exp2_approx(u[nt][i] - (mv[nt][i & 1] == -INFINITY ? 0.f : mv[nt][i & 1]));
        }
      }
      uint32_t w0, w1;
      if constexpr (FP8) {
        w0 = pack_f16x2(p[0], p[1]);
        w1 = pack_f16x2(p[2], p[3]);
      } else {
        w0 = pack_bf16x2(p[0], p[1]);
        w1 = pack_bf16x2(p[2], p[3]);
        l[nt][0] += bf16_lo(w0) + bf16_lo(w1);
        l[nt][1] += bf16_hi(w0) + bf16_hi(w1);
      }
      w[nt][0] = transpose8x8(w0);
      w[nt][1] = transpose8x8(w1);
    }
  }

  __device__ __forceinline__ void values(const uint32_t (&w)[NT][2]) {
#pragma unroll
    for (int i = 0; i < VW; ++i) {
      if constexpr (FP8) {
        // bytes of two neighbouring positions side by side, then both to fp16 at once
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x7362u : 0x5140u;
          const uint32_t lo = __byte_perm(v[0][i], v[1][i], sel), hi = __byte_perm(v[2][i], v[3][i], sel);
          const uint32_t a0 = e4m3x2_to_f16x2(lo), a1 = e4m3x2_to_f16x2(lo >> 16);
          const uint32_t a2 = e4m3x2_to_f16x2(hi), a3 = e4m3x2_to_f16x2(hi >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<true>(acc[2 * i + half][nt], a0, a1, a2, a3, w[nt][0], w[nt][1]);
        }
      } else {
        const uint32_t a0 = __byte_perm(v[0][i], v[1][i], 0x5410), a1 = __byte_perm(v[0][i], v[1][i], 0x7632);
        const uint32_t a2 = __byte_perm(v[2][i], v[3][i], 0x5410), a3 = __byte_perm(v[2][i], v[3][i], 0x7632);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<false>(acc[i][nt], a0, a1, a2, a3, w[nt][0], w[nt][1]);
      }
    }
  }
};

// A run's place in the line of tiles.
struct Cursor {
  int b;                              // sequence, -1: the shared positions
  int w;                              // key head * row tiles + row tile
  int tile, tiles;                    // tile of the segment
  int begin, end;                     // positions of the segment
  int row_tiles;

  __device__ __forceinline__ void enter(const Shape &s, const int32_t *seq_lens, int b_) {
    b = b_;
    w = tile = 0;
    row_tiles = b < 0 ? s.pre_row_tiles : s.row_tiles;
    const int len = b < 0 ? s.shared_len : seq_len(s, seq_lens, b);
    begin = b < 0 ? 0 : own_begin(s, len);
    end = len;
    tiles = b < 0 ? pre_tiles(s) : own_tiles(s, len);
  }
  // false: the next tile belongs to another segment
  __device__ __forceinline__ bool next(const Shape &s, const int32_t *seq_lens) {
    if (++tile < tiles) return true;
    tile = 0;
    if (++w == s.n_kv * row_tiles) {
      int n = b;
      do { enter(s, seq_lens, ++n); } while (tiles == 0 && n < s.B - 1);
    }
    return false;
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
__global__ void __launch_bounds__(kThreads, NT == 1 ? (FP8 ? 4 : 3) : (FP8 ? 3 : 2))
attn_stream_kernel(const __nv_bfloat16 *__restrict__ q, Cache cache, const int32_t *__restrict__ seq_lens, Shape s,
                   float *__restrict__ part, float *__restrict__ part_lse) {
  __shared__ float s_out[4][NT * 8][DV];
  __shared__ float s_lse[4][NT * 8];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  // this CTA's run: tiles first .. last-1 of the line
  const int own_heads = s.n_kv * s.row_tiles, pre_line = s.n_kv * s.pre_row_tiles * pre_tiles(s);
  int sum = 0;
  for (int b = lane; b < s.B; b += 32) sum += own_tiles(s, seq_len(s, seq_lens, b));
  const int total = pre_line + own_heads * warp_sum_int(sum);
  const int share = (total + gridDim.x - 1) / gridDim.x;
  const int first = blockIdx.x * share, last = min(total, first + share);
  if (first >= last) return;
  Cursor at;
  if (first < pre_line) {
    at.enter(s, seq_lens, -1);
    at.w = first / at.tiles;
    at.tile = first - at.w * at.tiles;
  } else {
    int before = pre_line, b0 = 0;
    for (; b0 + 32 < s.B; b0 += 32) {               // the 32 sequences among whose tiles the first one is
      const int n = own_heads * warp_sum_int(b0 + lane < s.B ? own_tiles(s, seq_len(s, seq_lens, b0 + lane)) : 0);
      if (before + n > first) break;
      before += n;
    }
    for (; b0 + 1 < s.B; ++b0) {
      const int n = own_heads * own_tiles(s, seq_len(s, seq_lens, b0));
      if (before + n > first) break;
      before += n;
    }
    at.enter(s, seq_lens, b0);
    at.w = (first - before) / at.tiles;
    at.tile = first - before - at.w * at.tiles;
  }

  Stream<DK, DV, FP8, NT> st;
  // row of position j in the cache: row0 + j * row_step
  const size_t row_step = FP8 ? 1 : (size_t)s.n_kv;
  const auto row0_of = [&](const Cursor &a) {
    const int hk = a.w / a.row_tiles, home = a.home(s);
    return FP8 ? ((size_t)home * s.n_kv + hk) * s.s_max : (size_t)home * s.s_max * s.n_kv + hk;
  };
  // query row r of the segment
  const auto begin = [&](const Cursor &a) {
    const int hk = a.w / a.row_tiles, rt = a.w - hk * a.row_tiles;
    const int rows = a.b < 0 ? s.B * s.group : s.group;
    st.begin([&](int r) -> const __nv_bfloat16 * {
      r += rt * s.rows;
      if (r >= rows || r >= (rt + 1) * s.rows) return nullptr;
      const int b = a.b < 0 ? r / s.group : a.b, h = a.b < 0 ? r - b * s.group : r;
      return q + b * s.q_stride + (size_t)(hk * s.group + h) * DK;
    }, s.scale_log2, g, c);
  };
  size_t row0 = row0_of(at);
  int key = at.begin + at.tile * kTile + warp * 16;
  st.load_k(cache, row0, row_step, key, at.end, g, c);
  st.load_v(cache, row0, row_step, key, at.end, g, c);
  begin(at);
  for (int t = first; t < last; ++t) {
    float sc[NT][4];
    uint32_t w[NT][2];
    st.scores(sc);
    const uint32_t bytes[4] = {st.scale_bytes[0], st.scale_bytes[1], st.scale_bytes[2], st.scale_bytes[3]};
    const bool in0 = key + g < at.end, in1 = key + g + 8 < at.end;
    const Cursor now = at;
    const bool more = t + 1 < last;
    bool same = false;
    if (more) {
      same = at.next(s, seq_lens);
      if (!same) row0 = row0_of(at);
      key = at.begin + at.tile * kTile + warp * 16;
      st.load_k(cache, row0, row_step, key, at.end, g, c);
    }
    st.weights(sc, bytes, in0, in1, w);
    st.values(w);
    if (more) st.load_v(cache, row0, row_step, key, at.end, g, c);
    if (same) continue;
    // the end of a piece: the four warps' results joined, one partial result
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float l = st.l[nt][r];
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        const int row = nt * 8 + 2 * c + r;
        float f = 1.f / l;
        if constexpr (FP8) f *= exp2_approx(st.mv[nt][r] - st.m[nt][r]);
        if (l == 0.f) f = 0.f;
        if (g == 0) s_lse[warp][row] = l == 0.f ? -INFINITY : st.m[nt][r] + log2f(l);
#pragma unroll
        for (int e = 0; e < DV / 8; ++e) s_out[warp][row][st.column(g, e)] = st.acc[e >> 1][nt][2 * (e & 1) + r] * f;
      }
    __syncthreads();
    const int hk = now.w / now.row_tiles, rt = now.w - hk * now.row_tiles;
    const int rows = min(s.rows, (now.b < 0 ? s.B * s.group : s.group) - rt * s.rows);
    const size_t slot = (size_t)blockIdx.x + now.segment(s);
    for (int i = threadIdx.x; i < rows * DV; i += kThreads) {
      const int row = i / DV, col = i - row * DV;
      float top = -INFINITY, sum_w = 0.f, o = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) top = fmaxf(top, s_lse[x][row]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float lse = s_lse[x][row], f = lse == -INFINITY ? 0.f : exp2_approx(lse - top);
        sum_w += f;
        o += f * s_out[x][row][col];
      }
      part[(slot * s.rows + row) * DV + col] = sum_w == 0.f ? 0.f : o / sum_w;
      if (col == 0) part_lse[slot * s.rows + row] = sum_w == 0.f ? -INFINITY : top + log2f(sum_w);
    }
    __syncthreads();
    if (more) begin(at);
  }
}

// One CTA per (sequence, query head): its pieces of the shared positions and of its own,
// weighted by their sums of exponentials.
template <int DV>
__global__ void __launch_bounds__(DV)
attn_join_kernel(const int32_t *__restrict__ seq_lens, Shape s, int n_ctas, const float *__restrict__ part,
                 const float *__restrict__ part_lse, const float *__restrict__ pre_part, const float *__restrict__ pre_lse,
                 __nv_bfloat16 *__restrict__ out) {
  __shared__ int s_sum[2][DV / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x / s.n_q, h = blockIdx.x - b * s.n_q, hk = h / s.group, hg = h - hk * s.group;
  int before = 0, all = 0;
  for (int i = threadIdx.x; i < s.B; i += DV) {
    const int n = own_tiles(s, seq_len(s, seq_lens, i));
    all += n;
    if (i < b) before += n;
  }
  before = warp_sum_int(before);
  all = warp_sum_int(all);
  if ((threadIdx.x & 31) == 0) { s_sum[0][threadIdx.x >> 5] = before; s_sum[1][threadIdx.x >> 5] = all; }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < DV / 32; ++w) { before += s_sum[0][w]; all += s_sum[1][w]; }
  const int own_heads = s.n_kv * s.row_tiles, pre_line = s.n_kv * s.pre_row_tiles * pre_tiles(s);
  const int total = pre_line + own_heads * all, share = (total + n_ctas - 1) / n_ctas;
  const int len = seq_len(s, seq_lens, b);
  float top = -INFINITY, sum = 0.f, acc = 0.f;
  const auto take = [&](const float *from, const float *from_lse, size_t slot_row) {
    const float lse = from_lse[slot_row], o = from[slot_row * DV + threadIdx.x];
    const float m = fmaxf(top, lse), ref = m == -INFINITY ? 0.f : m;
    const float f = exp2_approx(top - ref), w = exp2_approx(lse - ref);
    sum = sum * f + w;
    acc = acc * f + w * o;
    top = m;
  };
  const auto pieces = [&](int first, int tiles, int segment, int row) {
    for (int cta = first / share; cta <= (first + tiles - 1) / share; ++cta) take(part, part_lse, ((size_t)cta + segment) * s.rows + row);
  };
  if (s.pre_splits > 0 && len >= s.shared_len) {
    const int r = b * s.group + hg, rt = r / kPrefixRows, rows = prefix_rows(s);
    const size_t slot = ((size_t)hk * prefix_row_tiles(s) + rt) * s.pre_splits * 2;
    for (int i = 0; i < 2 * s.pre_splits; ++i) take(pre_part, pre_lse, (slot + i) * rows + r - rt * kPrefixRows);
  } else if (pre_line > 0 && len >= s.shared_len) {
    const int r = b * s.group + hg, rt = r / s.rows, n = pre_tiles(s);
    const int seg = hk * s.pre_row_tiles + rt;
    pieces(seg * n, n, seg, r - rt * s.rows);
  }
  const int n = own_tiles(s, len);
  if (n > 0) {
    const int rt = hg / s.rows, w = hk * s.row_tiles + rt;
    pieces(pre_line + own_heads * before + w * n, n, s.n_kv * (s.pre_row_tiles + b * s.row_tiles) + w, hg - rt * s.rows);
  }
  out[(size_t)blockIdx.x * DV + threadIdx.x] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc / sum);
}

constexpr int kMaxRows = 16;

// How a call is cut; the rest of the shape is the caller's.  Up to sixteen rows share one
// pass of the streamed line over the prefix, more go through the tensor-core tiles.
void plan(Shape &s) {
  const int64_t pre_rows = s.shared_len > 0 ? (int64_t)s.B * s.group : 0;
  s.pre_splits = pre_rows > kMaxRows ? prefix_splits(s) : 0;
  s.rows = s.group > kMaxRows ? kMaxRows : s.group;
  if (pre_rows > s.rows && s.pre_splits == 0) s.rows = (int)pre_rows;
  s.row_tiles = (s.group + s.rows - 1) / s.rows;
  s.pre_row_tiles = pre_rows > 0 && s.pre_splits == 0 ? 1 : 0;
}
// Partial results: of the streamed line, then of the shared positions' tiles; outputs first,
// then logarithms.
int64_t slot_rows(const Shape &s) { return (kMaxCtas + (int64_t)s.n_kv * (s.pre_row_tiles + (int64_t)s.B * s.row_tiles)) * s.rows; }
int64_t pre_slot_rows(const Shape &s) { return prefix_slots(s) * prefix_rows(s); }

template <int DK, int DV, bool FP8>
int32_t launch(const __nv_bfloat16 *q, const Cache &cache, const int32_t *seq_lens, const Shape &s, float *part,
               __nv_bfloat16 *out, int32_t *status, cudaStream_t st) {
  float *pre_part = part + slot_rows(s) * DV, *lse = pre_part + pre_slot_rows(s) * DV, *pre_lse = lse + slot_rows(s);
  if (s.pre_splits > 0) {
    const int32_t rc = launch_attn_prefix(FP8, DK, DV, q, cache, s, pre_part, pre_lse, status, st);
    if (rc != SB_OK) return rc;
  }
  const int sms = sb_device_sm_count() > 0 ? sb_device_sm_count() : 148;
  // a CTA for every tile there can be, up to four per SM
  const int64_t tiles = (int64_t)s.n_kv * ((int64_t)s.pre_row_tiles * ((s.shared_len + kTile - 1) / kTile) +
                                           (int64_t)s.B * s.row_tiles * ((s.s_max + kTile - 1) / kTile));
  const int most = 4 * sms < kMaxCtas ? 4 * sms : kMaxCtas;
  const int ctas = tiles < most ? (int)tiles : most;
  auto kern = s.rows <= 8 ? attn_stream_kernel<DK, DV, FP8, 1> : attn_stream_kernel<DK, DV, FP8, 2>;
  SB_CUDA_CHECK(launch_pdl(kern, dim3(ctas), dim3(kThreads), 0, st, q, cache, seq_lens, s, part, lse));
  SB_LAUNCH_CHECK();
  SB_CUDA_CHECK(launch_pdl(attn_join_kernel<DV>, dim3(s.B * s.n_q), dim3(DV), 0, st, seq_lens, s, ctas,
                           static_cast<const float *>(part), static_cast<const float *>(lse),
                           static_cast<const float *>(pre_part), static_cast<const float *>(pre_lse), out));
  SB_LAUNCH_CHECK();
  return SB_OK;
}

template <bool FP8>
int32_t attend(const char *name, const void *q, int64_t q_stride, Cache cache, const int32_t *seq_lens, int B, int n_q,
               int n_kv, int dk, int dv, int s_max, int shared_len, float scale, void *ws, size_t ws_bytes, void *out,
               int32_t *status, void *stream) {
  // (the line's tiles are counted in 32 bits)
  if (B < 0 || n_q < 1 || n_kv < 1 || n_kv > 65535 || n_q % n_kv != 0 || s_max < 1 || shared_len < 0 || shared_len > s_max ||
      (int64_t)B * n_q > (1 << 22) || (int64_t)B * n_q * (s_max / kTile + 2) > (1ll << 30))
    return fail(SB_E_INVALID_ARG, "%s: bad shape (B=%d heads %d/%d s_max=%d shared %d)", name, B, n_q, n_kv, s_max, shared_len);
  if (!(scale >= 0.f) || !isfinite(scale)) return fail(SB_E_INVALID_ARG, "%s: scale must be finite and not negative", name);
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
  Shape s = {B, n_q, n_kv, n_q / n_kv, s_max, shared_len, 0, 0, 0, 0, q_stride, scale * 1.4426950408889634f};
  plan(s);
  const __nv_bfloat16 *qq = static_cast<const __nv_bfloat16 *>(q);
  float *part = static_cast<float *>(ws);
  __nv_bfloat16 *oo = static_cast<__nv_bfloat16 *>(out);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dk == 128 ? launch<128, 128, FP8>(qq, cache, seq_lens, s, part, oo, status, st)
         : dk == 192 ? launch<192, 128, FP8>(qq, cache, seq_lens, s, part, oo, status, st)
                     : launch<64, 64, FP8>(qq, cache, seq_lens, s, part, oo, status, st);
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" {

size_t sb_attn_cached_workspace_bytes(int32_t B, int32_t n_q, int32_t n_kv, int32_t dv, int32_t s_max, int32_t shared_len) {
  if (B < 0 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || dv < 1 || s_max < 1 || shared_len < 0 || (int64_t)B * n_q > (1 << 22))
    return 0;
  Shape s = {B, n_q, n_kv, n_q / n_kv, s_max, shared_len, 0, 0, 0, 0, 0, 0.f};
  plan(s);
  return (size_t)(slot_rows(s) + pre_slot_rows(s)) * (dv + 1) * sizeof(float);
}

int32_t sb_attn_decode_shared(const void *q, int64_t q_stride, const void *cache_k, const void *cache_v,
                              const int32_t *seq_lens, int32_t B, int32_t n_q, int32_t n_kv, int32_t dk, int32_t dv,
                              int32_t s_max, int32_t shared_len, float scale, void *ws, size_t ws_bytes, void *out,
                              int32_t *status, void *stream) {
  return attend<false>("sb_attn_decode_shared", q, q_stride, Cache{cache_k, cache_v, nullptr, nullptr}, seq_lens, B, n_q,
                       n_kv, dk, dv, s_max, shared_len, scale, ws, ws_bytes, out, status, stream);
}

int32_t sb_attn_decode_fp8(const void *q, int64_t q_stride, const void *codes_k, const void *scale_k, const void *codes_v,
                           const void *scale_v, const int32_t *seq_lens, int32_t B, int32_t n_q, int32_t n_kv, int32_t dk,
                           int32_t dv, int32_t s_max, int32_t shared_len, float scale, void *ws, size_t ws_bytes, void *out,
                           int32_t *status, void *stream) {
  return attend<true>("sb_attn_decode_fp8", q, q_stride,
                      Cache{codes_k, codes_v, static_cast<const uint8_t *>(scale_k), static_cast<const uint8_t *>(scale_v)},
                      seq_lens, B, n_q, n_kv, dk, dv, s_max, shared_len, scale, ws, ws_bytes, out, status, stream);
}

}  // extern "C"
