// Attention of a chunk of a prompt over a 4-bit KV cache: many query rows per kv head.
//
// With hundreds of rows per key the products belong on the tensor-memory attention
// kernels, which want dense operands; reading the rows back once costs 5 % of the
// attention of a 512-token chunk (32 heads, 8704 keys).  But rounding the keys to
// bf16 on the way shows: a score moves by 2^-9 of its terms, 3 times the error of all
// other roundings together.  So the operands are fp16, whose 11 bits make it vanish,
// scaled per sequence and kv head by powers of two to a largest value in
// [2^13, 2^14): the range that bf16 has and fp16 has not.
//
//   1. attn_q4_absmax_kernel: largest |q|, |k|, |v| of each kv head (k, v from the
//      scales alone, a fifth of the cache's bytes).
//   2. attn_q4_operands_kernel: q, k, v as scaled fp16 [.., 128].
//   3. attn_tc_f16: the attention.  A short chunk has fewer query blocks than the GPU
//      has SMs (512 tokens x 32 heads: 64 CTAs), so the key tiles are cut into as many
//      splits as fill it, which leave fp32 partials ...
//   4. attn_q4_splits_kernel: ... joined here.
#include <cuda_fp16.h>
#include <float.h>

#include "attention_tc.cuh"
#include "kv_q4.cuh"

namespace q35 {
namespace {

using q4::Cache;

constexpr int kThreads = 256;
constexpr int kSlices = 16;  // CTAs per kv head of the largest values
constexpr int kPad = 128;    // rows of a key tile, channels of an operand row

struct Chunk {
  const uint16_t *q;
  Cache c;
  float4 *maxima;  // [kSlices][B * Hkv] (|q|, |k|, |v|)
  float2 *fac;     // [B * Hkv]
  __half *qo, *ko, *vo;
  int D, group, q_rows;  // q_rows = Hq / Hkv * Sq
  int64_t cap;
  int len, pad;          // keys, and their rows in ko / vo
};

__device__ __forceinline__ float largest(float a, float x) {
  x = fabsf(x);
  return x < INFINITY ? fmaxf(a, x) : a;
}

__global__ void __launch_bounds__(kThreads) attn_q4_absmax_kernel(Chunk p) {
  const int64_t bh = blockIdx.y;
  const int ns = p.D / p.group, tid = blockIdx.x * kThreads + threadIdx.x;
  constexpr int step = kSlices * kThreads;
  float m[3] = {0.f, 0.f, 0.f};
  const uint4 *q = reinterpret_cast<const uint4 *>(p.q + bh * p.q_rows * p.D);
  const int64_t nq = int64_t(p.q_rows) * p.D / 8;
  for (int64_t i = tid; i < nq; i += step) {
    const uint4 x = q[i];
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a, b;
      unpack_bf2(w[k], a, b);
      m[0] = largest(largest(m[0], a), b);
    }
  }
  const int64_t base = bh * p.cap * ns, n = int64_t(p.len) * ns;
  for (int64_t i = tid; i < n; i += step) {
    const uint32_t k = p.c.k_scales[base + i], v = p.c.v_scales[base + i];
    m[1] = largest(largest(m[1], q4::value(0.f, k)), q4::value(15.f, k));
    m[2] = largest(largest(m[2], q4::value(0.f, v)), q4::value(15.f, v));
  }
  __shared__ float part[3][kThreads / 32];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    m[i] = warp_max(m[i]);
    if ((threadIdx.x & 31) == 0) part[i][threadIdx.x >> 5] = m[i];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      for (int w = 0; w < kThreads / 32; ++w) m[i] = fmaxf(m[i], part[i][w]);
    p.maxima[int64_t(blockIdx.x) * gridDim.y + bh] = make_float4(m[0], m[1], m[2], 0.f);
  }
}

// e with 2^-e * a in [2^13, 2^14); 0 for a = 0.
__device__ __forceinline__ int exponent(float a) {
  if (a == 0.f) return 0;
  int e;
  frexpf(a, &e);  // a = f 2^e, f in [0.5, 1)
  return max(-100, min(e - 14, 126));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// A thread writes 8 of the 128 channels of an operand row; rows: keys, values, queries.
__global__ void __launch_bounds__(kThreads) attn_q4_operands_kernel(Chunk p) {
  const int64_t bh = blockIdx.y;
  __shared__ float scale[3];
  if (threadIdx.x < 32) {
    float m[3] = {0.f, 0.f, 0.f};
    if (threadIdx.x < kSlices) {
      const float4 x = p.maxima[int64_t(threadIdx.x) * gridDim.y + bh];
      m[0] = x.x, m[1] = x.y, m[2] = x.z;
    }
    int e[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) e[i] = exponent(warp_max(m[i]));
    if (threadIdx.x == 0) {
#pragma unroll
      for (int i = 0; i < 3; ++i) scale[i] = pow2(-e[i]);
      if (blockIdx.x == 0) p.fac[bh] = make_float2(ldexpf(1.f, e[0] + e[1]), pow2(e[2]));
    }
  }
  __syncthreads();
  const int ch = threadIdx.x & 15, W = p.D / 8;
  const int64_t r = int64_t(blockIdx.x) * (kThreads / 16) + threadIdx.x / 16;
  const int which = r < p.pad ? 1 : r < 2 * int64_t(p.pad) ? 2 : 0;
  const int64_t row = which == 1 ? r : which == 2 ? r - p.pad : r - 2 * int64_t(p.pad);
  if (which == 0 && row >= p.q_rows) return;
  const float f = scale[which];
  uint32_t o[4] = {0u, 0u, 0u, 0u};
  if (ch < W) {
    if (which == 0) {
      const uint4 x = *reinterpret_cast<const uint4 *>(p.q + (bh * p.q_rows + row) * p.D + 8 * ch);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack_bf2(w[i], a, b);
        o[i] = pack_h2(a * f, b * f);
      }
    } else if (row < p.len) {
      const int64_t at = bh * p.cap + row;
      const uint32_t word = (which == 2 ? p.c.v_codes : p.c.k_codes)[at * W + (ch & 3) * (p.D / 32) + (ch >> 2)];
      const uint32_t pair = (which == 2 ? p.c.v_scales : p.c.k_scales)[at * (p.D / p.group) + 8 * ch / p.group];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = pack_h2(q4::value(q4::code_of(word, 2 * i), pair) * f,
                       q4::value(q4::code_of(word, 2 * i + 1), pair) * f);
    }
  }
  __half *dst = which == 0 ? p.qo + (bh * p.q_rows + row) * kPad
                           : (which == 2 ? p.vo : p.ko) + (bh * p.pad + row) * kPad;
  reinterpret_cast<uint4 *>(dst)[ch] = make_uint4(o[0], o[1], o[2], o[3]);
}

// One warp per query row: joins the splits.
__global__ void __launch_bounds__(kThreads) attn_q4_splits_kernel(F16Extra x, uint16_t *out, int Hq,
                                                                  int64_t Sq) {
  const int lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= x.rows) return;
  const float2 *ml = reinterpret_cast<const float2 *>(x.part + x.rows * x.splits * x.D) + row * x.splits;
  const float *part = x.part + row * x.splits * x.D;
  float top = -FLT_MAX, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < x.splits; ++s) top = fmaxf(top, ml[s].x);
  for (int s = 0; s < x.splits; ++s) {
    const float2 w = ml[s];
    const float f = exp2f(w.x - top);
    l = fmaf(w.y, f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (32 * e < x.D) v[e] = fmaf(part[int64_t(s) * x.D + 32 * e + lane], f, v[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t b = row / (Hq * Sq), h = row / Sq % Hq, s = row % Sq;
  uint16_t *dst = out + ((b * Sq + s) * Hq + h) * x.D + lane;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (32 * e < x.D) dst[32 * e] = f2bf(v[e] * inv);
}

// Splits of the key tiles and the workspace's parts, in bytes.
struct Plan {
  int splits, tiles_per_split, pad;
  int64_t fac, ko, vo, qo, part, bytes;
};
Plan plan(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len, int D) {
  Plan pl{};
  int64_t tile;
  const int ctas = attn_tc_ctas(B, Hq, Hkv, Sq, &tile);
  const int tiles = static_cast<int>((kv_len + tile - 1) / tile);
  // Splits that fill the SMs once; a split of fewer than 4 tiles costs more to begin
  // and join than it saves.
  int n = ctas > 0 ? num_sms() / ctas : 1;
  if (n > tiles / 4) n = tiles / 4;
  if (n < 1) n = 1;
  pl.tiles_per_split = (tiles + n - 1) / n;
  pl.splits = (tiles + pl.tiles_per_split - 1) / pl.tiles_per_split;
  pl.pad = static_cast<int>(tiles * tile);
  const int64_t bh = B * Hkv, rows = B * Hq * Sq;
  pl.fac = kSlices * bh * int64_t(sizeof(float4));
  pl.ko = pl.fac + (bh * int64_t(sizeof(float2)) + 15) / 16 * 16;
  pl.vo = pl.ko + bh * pl.pad * kPad * 2;
  pl.qo = pl.vo + bh * pl.pad * kPad * 2;
  pl.part = pl.qo + rows * kPad * 2;
  pl.bytes = pl.part + (pl.splits > 1 ? rows * pl.splits * (D + 2) * 4 : 0);
  return pl;
}

bool plannable(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len) {
  const int64_t lim = int64_t(1) << 31;
  return B > 0 && Hq > 0 && Hkv > 0 && Sq > 0 && kv_len > 0 && kv_len < lim - 256 && B < lim / Hq &&
         Sq < lim / (B * Hq) && kv_len + 128 < lim / (B * Hkv);
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int64_t q35_attn_q4_chunk_workspace(int64_t B, int Hq, int Hkv, int64_t Sq,
                                               int64_t kv_len, int D) {
  if (!plannable(B, Hq, Hkv, Sq, kv_len) || Hq % Hkv != 0) return 0;
  return plan(B, Hq, Hkv, Sq, kv_len, D).bytes;
}

extern "C" int q35_attn_q4_chunk_fwd(const void *q, const void *k_codes, const void *k_scales,
                                     const void *v_codes, const void *v_scales, void *out,
                                     int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len,
                                     int64_t cap, int D, int group, float scale, int causal,
                                     void *workspace, q35_stream_t stream) {
  int st = q4::check_cache("attn_q4_chunk", k_codes, k_scales, v_codes, v_scales, B, Hkv, D, group,
                           cap);
  if (st) return st;
  if (Sq < 0 || kv_len < 1 || Hq <= 0 || Hq % Hkv != 0)
    return fail(Q35_ERR_SHAPE, "attn_q4_chunk: Sq %lld, kv_len %lld, Hq %d, Hkv %d", (long long)Sq,
                (long long)kv_len, Hq, Hkv);
  if (kv_len > cap)
    return fail(Q35_ERR_SHAPE, "attn_q4_chunk: %lld rows exceed the capacity %lld",
                (long long)kv_len, (long long)cap);
  if (B * Sq == 0) return Q35_OK;
  if (!q || !out || !workspace) return fail(Q35_ERR_INVALID, "attn_q4_chunk: null");
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace))
    return fail(Q35_ERR_ALIGN, "attn_q4_chunk: q, out or workspace not 16-byte aligned");
  if (!plannable(B, Hq, Hkv, Sq, kv_len) || B * Hq > 65535)
    return fail(Q35_ERR_SHAPE, "attn_q4_chunk: too many heads, query rows or keys");
  const Plan pl = plan(B, Hq, Hkv, Sq, kv_len, D);
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  Chunk c{};
  c.q = static_cast<const uint16_t *>(q);
  c.c = Cache{static_cast<uint32_t *>(const_cast<void *>(k_codes)),
              static_cast<uint32_t *>(const_cast<void *>(k_scales)),
              static_cast<uint32_t *>(const_cast<void *>(v_codes)),
              static_cast<uint32_t *>(const_cast<void *>(v_scales))};
  c.maxima = reinterpret_cast<float4 *>(ws);
  c.fac = reinterpret_cast<float2 *>(ws + pl.fac);
  c.ko = reinterpret_cast<__half *>(ws + pl.ko);
  c.vo = reinterpret_cast<__half *>(ws + pl.vo);
  c.qo = reinterpret_cast<__half *>(ws + pl.qo);
  c.D = D;
  c.group = group;
  c.q_rows = static_cast<int>(Hq / Hkv * Sq);
  c.cap = cap;
  c.len = static_cast<int>(kv_len);
  c.pad = pl.pad;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned bh = static_cast<unsigned>(B * Hkv);
  attn_q4_absmax_kernel<<<dim3(kSlices, bh), kThreads, 0, s>>>(c);
  Q35_LAUNCH_CHECK("attn_q4 absmax launch");
  const int64_t rows = 2 * int64_t(c.pad) + c.q_rows;
  attn_q4_operands_kernel<<<dim3(static_cast<unsigned>((rows + 15) / 16), bh), kThreads, 0, s>>>(c);
  Q35_LAUNCH_CHECK("attn_q4 operands launch");
  F16Extra x{};
  x.fac = c.fac;
  x.rows = B * Hq * Sq;
  x.splits = pl.splits;
  x.tiles_per_split = pl.tiles_per_split;
  x.D = D;
  x.part = pl.splits > 1 ? reinterpret_cast<float *>(ws + pl.part) : nullptr;
  st = attn_tc_f16(c.qo, c.ko, c.vo, out, B, Hq, Hkv, Sq, kv_len, c.pad, scale, causal, x, stream);
  if (st) return st;
  if (pl.splits > 1) {
    attn_q4_splits_kernel<<<static_cast<unsigned>((x.rows + 7) / 8), kThreads, 0, s>>>(
        x, static_cast<uint16_t *>(out), Hq, Sq);
    Q35_LAUNCH_CHECK("attn_q4 splits launch");
  }
  return Q35_OK;
}
