// Attention over a 4-bit KV cache (layout: kv_q4.cuh).
//
// out[b, s, h D + d] = sum_k p_k V[k, d] / sum_k p_k, p_k = exp(scale q . K[k] - max),
// over the keys k < kv_len_b, with a causal mask aligned to the last key
// (query s of Sq sees k <= s + kv_len_b - Sq).  A row that sees no key is zero.
#include "kv_q4.cuh"

namespace q35 {
namespace {

constexpr int kWarps = 4;

struct Shape {
  int Hq, Hkv, D, group;
  int64_t Sq, kv_len, cap;
  float scale_log2;
  int causal;
};

// One warp per (b, head, query) row; a lane scores one key of 32 at a time and
// owns D/32 channels of the output.
__global__ void __launch_bounds__(kWarps * 32) attn_q4_rows_kernel(
    const uint16_t *__restrict__ q, q4::Cache c, uint16_t *__restrict__ out, Shape p,
    const int32_t *__restrict__ kv_lens, int64_t rows, int *err) {
  __shared__ float sq[kWarps][128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (row >= rows) return;
  const int64_t s = row % p.Sq, bh = row / p.Sq;
  const int64_t b = bh / p.Hq;
  const int h = static_cast<int>(bh - b * p.Hq);
  const int D = p.D, W = D / 8, J = D / 32, NS = D / p.group, GT = p.group / 8;
  const int64_t base = (b * p.Hkv + h / (p.Hq / p.Hkv)) * p.cap;
  int64_t len = p.kv_len;
  if (kv_lens) {
    len = kv_lens[b];
    if (len < 0 || len > p.kv_len) {
      if (lane == 0) report_error(err, DEV_ERR_INDEX, 311, static_cast<int>(b), static_cast<int>(len));
      len = len < 0 ? 0 : p.kv_len;
    }
  }
  const int64_t end = p.causal ? min(len, len - p.Sq + s + 1) : len;
  for (int d = lane; d < D; d += 32) sq[warp][d] = bf2f(q[row * D + d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t k0 = 0; k0 < end; k0 += 32) {
    float dot = -INFINITY;
    if (k0 + lane < end) {
      const int64_t at = base + k0 + lane;
      dot = 0.f;
      for (int ch = 0; ch < W; ++ch) {
        const uint32_t word = c.k_codes[at * W + (ch & 3) * J + (ch >> 2)];
        const uint32_t pair = c.k_scales[at * NS + ch / GT];
        for (int e = 0; e < 8; ++e)
          dot = fmaf(sq[warp][8 * ch + e], q4::value(q4::code_of(word, e), pair), dot);
      }
    }
    const float mx = fmaxf(m, warp_max(dot));
    const float mu = mx == -INFINITY ? 0.f : mx;
    const float alpha = exp2f((m - mu) * p.scale_log2);
    const float pk = exp2f((dot - mu) * p.scale_log2);
    m = mx;
    l = l * alpha + warp_sum(pk);
    for (int e = 0; e < J; ++e) acc[e] *= alpha;
    const int n = static_cast<int>(min(static_cast<int64_t>(32), end - k0));
    for (int kk = 0; kk < n; ++kk) {
      const float w = __shfl_sync(0xffffffffu, pk, kk);
      const int64_t at = base + k0 + kk;
      for (int e = 0; e < J; ++e) {
        const int d = lane * J + e, ch = d / 8;
        const uint32_t word = c.v_codes[at * W + (ch & 3) * J + (ch >> 2)];
        acc[e] = fmaf(w, q4::value(q4::code_of(word, d & 7), c.v_scales[at * NS + ch / GT]), acc[e]);
      }
    }
  }
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  for (int e = 0; e < J; ++e)
    out[((b * p.Sq + s) * p.Hq + h) * D + lane * J + e] = f2bf(acc[e] * inv);
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int64_t q35_attn_q4_workspace(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len,
                                         int D) {
  return 0;
}

extern "C" int q35_attn_q4_fwd(const void *q, const void *k_codes, const void *k_scales,
                               const void *v_codes, const void *v_scales, void *out, int64_t B,
                               int Hq, int Hkv, int64_t Sq, int64_t kv_len, const int32_t *kv_lens,
                               int64_t cap, int D, int group, float scale, int causal,
                               float *workspace, q35_stream_t stream) {
  const int st = q4::check_cache("attn_q4", k_codes, k_scales, v_codes, v_scales, B, Hkv, D, group,
                                 cap);
  if (st) return st;
  if (Sq < 0 || kv_len < 0 || Hq <= 0 || Hq % Hkv != 0)
    return fail(Q35_ERR_SHAPE, "attn_q4: Sq %lld, kv_len %lld, Hq %d, Hkv %d", (long long)Sq,
                (long long)kv_len, Hq, Hkv);
  if (kv_len > cap)
    return fail(Q35_ERR_SHAPE, "attn_q4: %lld rows exceed the capacity %lld", (long long)kv_len,
                (long long)cap);
  if (B * Sq == 0) return Q35_OK;
  if (!q || !out) return fail(Q35_ERR_INVALID, "attn_q4: null");
  if (!aligned16(q) || !aligned16(out))
    return fail(Q35_ERR_ALIGN, "attn_q4: q, out not 16-byte aligned");
  int *err = device_error_word();
  if (!err) return fail(Q35_ERR_CUDA, "attn_q4: no device error word");
  const q4::Cache c{static_cast<uint32_t *>(const_cast<void *>(k_codes)),
                    static_cast<uint32_t *>(const_cast<void *>(k_scales)),
                    static_cast<uint32_t *>(const_cast<void *>(v_codes)),
                    static_cast<uint32_t *>(const_cast<void *>(v_scales))};
  const Shape p{Hq, Hkv, D, group, Sq, kv_len, cap, scale * 1.4426950408889634f, causal ? 1 : 0};
  const int64_t rows = B * Hq * Sq;
  const int64_t blocks = (rows + kWarps - 1) / kWarps;
  if (blocks >= (int64_t(1) << 31)) return fail(Q35_ERR_SHAPE, "attn_q4: too many rows");
  attn_q4_rows_kernel<<<static_cast<unsigned>(blocks), kWarps * 32, 0,
                        reinterpret_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint16_t *>(q), c, static_cast<uint16_t *>(out), p, kv_lens, rows, err);
  Q35_LAUNCH_CHECK("attn_q4 launch");
  return Q35_OK;
}
