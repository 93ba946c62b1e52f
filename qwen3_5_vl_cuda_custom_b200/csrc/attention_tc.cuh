// The fp16-operand form of the tensor-memory attention kernels (attention_tc.cu),
// which attention over rows read back from a 4-bit cache runs on.
#pragma once

#include "common.cuh"

namespace q35 {

// Partial sums are stored times this: they are up to 2^53 (weights to 2^15, values to 2^14,
// 2^24 keys) times an output factor of up to 2^114, which fp32 does not hold.
constexpr float kPartScale = 0x1p-40f;

struct F16Extra {
  const float2 *scales; // [B * Hkv]: the scale in log2 units, what the output is multiplied by
  const int *nan;       // [B * Hkv][4]: first key that makes 32 output channels NaN each
  float *part;          // fp32 partials [rows, splits, D], then (m, l) [rows, splits]; or null
  int64_t rows;         // B * Hq * Sq
  int splits, tiles_per_split, D;
};

// CTAs of one pass over all key tiles, and the rows of a query or key tile.
int attn_tc_ctas(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t *tile_rows);

// q [B,Hq,Sq,128], k / v [B,Hkv,kv_cap,128] fp16 (channels behind D zero, rows behind
// Skv finite), out token-major bf16 [B,Sq,Hq*D] unless x.part takes partials.
int attn_tc_f16(const void *q, const void *k, const void *v, void *out, int64_t B, int Hq, int Hkv,
                int64_t Sq, int64_t Skv, int64_t kv_cap, int causal, const F16Extra &x,
                q35_stream_t stream);

}  // namespace q35
