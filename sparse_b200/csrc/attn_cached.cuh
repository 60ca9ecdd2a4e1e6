// Decode attention over cached positions: what its kernels share.
#pragma once

#include "kv_fp8.cuh"

namespace sb {

struct Cache {                        // bf16: [B, s_max, n_kv, d]; quantised: codes [B, n_kv, s_max, d], scales [B, n_kv, s_max]
  const void *k, *v;
  const uint8_t *ks, *vs;
};

struct Shape {
  int B, n_q, n_kv, group;            // group = query heads per key head
  int s_max, shared_len;
  int rows;                           // query rows of a segment of the streamed line (at most 16)
  int row_tiles, pre_row_tiles;       // its segments per key head: of a sequence, and of the shared positions
  int pre_splits;                     // > 0: the shared positions go through attn_prefix_kernel, cut in so many
  int pre_tile_rows, pre_tiles, pre_rows;    // its rows per tile, row tiles of a key head, rows of a partial result
  int64_t q_stride;
  float scale_log2;                   // scale * log2(e), >= 0
};

// attn_prefix_kernel takes the rows of a key head, numbered sequence by sequence (row = b * group
// + h), in tiles of 128, or of two times 128.
constexpr int kPrefixRows = 128;
// Partial results of that kernel: one per CTA, of `pre_rows` rows.
inline int64_t prefix_slots(const Shape &s) { return (int64_t)s.n_kv * s.pre_tiles * s.pre_splits; }

// Sets the pre_* fields of a call whose shared positions go through attn_prefix_kernel.
void plan_prefix(Shape &s, int dk);

// softmax(q k) v of every row of the batch over the shared positions, as partial results:
// part [slot][row][dv] attention over the slot's positions, lse [slot][row] log2 of their sum of exponentials.
int32_t launch_attn_prefix(bool fp8, int dk, int dv, const __nv_bfloat16 *q, const Cache &cache, const Shape &s, float *part,
                           float *lse, int32_t *status, cudaStream_t stream);

// 2^x; results below 2^-126 are zero
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A weight below this power of two of the running maximum's does not move the maximum: sums
// and weights stay below 2^8 times their usual size, and most steps have nothing to rescale.
constexpr float kLazy = 8.f;

}  // namespace sb
