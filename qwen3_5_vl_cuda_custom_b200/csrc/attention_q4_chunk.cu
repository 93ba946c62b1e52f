// Attention of a chunk of a prompt over a 4-bit KV cache: many query rows per kv head.
//
// With hundreds of rows per key the products belong on the tensor-memory attention
// kernels, which want dense operands; reading the rows back once costs 5 % of the
// attention of a 512-token chunk (32 heads, 8704 keys).  But rounding the keys to
// bf16 on the way shows: a score moves by up to 2^-8 of its terms and the output by
// 0.0048 (relative, normal data), against 0.0017 from its own rounding to bf16.  So
// the operands are fp16, whose 11 bits make it vanish, scaled per sequence and kv head
// by powers of two, for the range that bf16 has and fp16 has not: q, k and v to largest
// values in [2^13, 2^14) each.  The attention kernels multiply the scores by what q and
// k were divided by, and the output by v's.
//
//   1. attn_q4_absmax_kernel: largest |q|, |k|, |v| of each kv head (k, v from the
//      scales alone, a fifth of the cache's bytes).
//   2. attn_q4_operands_kernel: q, k, v as scaled fp16 [.., 128].  A NaN among the
//      values would reach rows that do not see it (0 * NaN), and one among the keys is
//      lost in 3., whose polynomial exponential clamps its argument; both become 0 and 3.
//      puts the NaN into the rows that see it, from the first such key of every 32
//      channels (of all channels for a key).
//   3. attn_tc_f16: the attention.  A short chunk has fewer query blocks than the GPU
//      has SMs (512 tokens x 32 heads: 64 CTAs), so the key tiles are cut into as many
//      splits as fill it, which leave fp32 partials ...
//   4. attn_q4_splits_kernel: ... joined here.
//
// Measured, that chunk: 104 us in a captured graph, 0.41 of the measured matrix peak (one
// by one under ncu: largest values 5.9, operands 15.1, attention 89.9, join 10.4 us);
// relative error 0.0017.
#include <cuda_fp16.h>
#include <float.h>
#include <limits.h>

#include "attention_tc.cuh"
#include "kv_q4.cuh"

namespace q35 {
namespace {

using q4::Cache;

constexpr int kThreads = 256;
constexpr int kMaxSlices = 64;  // CTAs per kv head of the largest values, at most
constexpr int kPad = 128;       // rows of a key tile, channels of an operand row
constexpr int kRows = 4;        // operand rows of a thread

struct Chunk {
  const uint16_t *q;
  Cache c;
  float4 *maxima;  // [slices][B * Hkv] (|q|, |k|, |v|)
  float2 *scales;  // [B * Hkv] factors of the scores and of the output
  int *nan;        // [B * Hkv][4] first key that makes 32 output channels NaN
  __half *qo, *ko, *vo;
  int D, group, q_rows;  // q_rows = Hq / Hkv * Sq
  int64_t cap;
  int len, pad;          // keys, and their rows in ko / vo
  int slices;
  float scale;
};

__device__ __forceinline__ bool nonfinite(uint32_t pair) {
  return (((pair & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
}
__device__ __forceinline__ float largest(float a, float x) {
  x = fabsf(x);
  return x < INFINITY ? fmaxf(a, x) : a;
}
// The largest magnitude that a (scale, minimum) pair's codes can stand for.
__device__ __forceinline__ float largest_of(float a, uint32_t pair) {
  if (nonfinite(pair)) return a;  // its values count as NaN
  return fminf(fmaxf(a, fmaxf(fabsf(q4::value(0.f, pair)), fabsf(q4::value(15.f, pair)))), FLT_MAX);
}

__global__ void __launch_bounds__(kThreads) attn_q4_absmax_kernel(Chunk p) {
  const int64_t bh = blockIdx.y;
  const int ns = p.D / p.group, tid = blockIdx.x * kThreads + threadIdx.x;
  const int step = p.slices * kThreads;
  float m[3] = {0.f, 0.f, 0.f};
  const uint4 *q = reinterpret_cast<const uint4 *>(p.q + bh * p.q_rows * p.D);
  const int64_t nq = int64_t(p.q_rows) * p.D / 8;
#pragma unroll 4
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
#pragma unroll 4
  for (int64_t i = tid; i < n; i += step) {
    const uint32_t k = p.c.k_scales[base + i], v = p.c.v_scales[base + i];
    m[1] = largest_of(m[1], k);
    m[2] = largest_of(m[2], v);
  }
  __shared__ float part[3][kThreads / 32];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    m[i] = warp_max(m[i]);
    if ((threadIdx.x & 31) == 0) part[i][threadIdx.x >> 5] = m[i];
  }
  let_next_launch();
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x < 4) p.nan[bh * 4 + threadIdx.x] = INT_MAX;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      for (int w = 0; w < kThreads / 32; ++w) m[i] = fmaxf(m[i], part[i][w]);
    p.maxima[int64_t(blockIdx.x) * gridDim.y + bh] = make_float4(m[0], m[1], m[2], 0.f);
  }
}

// Exponent of a > 0: a = f 2^e, f in [0.5, 1); 0 for a = 0.
__device__ __forceinline__ int exponent(float a) {
  int e = 0;
  if (a > 0.f) frexpf(a, &e);
  return e;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// fp16's finite range: a value that fp32 cannot hold (finite scale and minimum, infinite
// together) must not become 0 * infinity in a row that does not see it.
__device__ __forceinline__ float saturate(float x) { return fminf(fmaxf(x, -65504.f), 65504.f); }

// A thread writes 8 of the 128 channels of kRows operand rows; rows: keys, values,
// queries.  What it reads is on its way before the scales are known.
__global__ void __launch_bounds__(kThreads) attn_q4_operands_kernel(Chunk p) {
  const int64_t bh = blockIdx.y;
  __shared__ float scale[3];
  const int ch = threadIdx.x & 15, W = p.D / 8;
  const int64_t r0 = int64_t(blockIdx.x) * (kRows * kThreads / 16) + threadIdx.x / 16;
  uint4 x[kRows];  // 8 channels of q, or (code word, scale pair)
  int which[kRows];
  int64_t row[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t r = r0 + i * (kThreads / 16);
    which[i] = r < p.pad ? 1 : r < 2 * int64_t(p.pad) ? 2 : 0;
    row[i] = which[i] == 1 ? r : which[i] == 2 ? r - p.pad : r - 2 * int64_t(p.pad);
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (ch >= W) continue;
    if (which[i] == 0) {
      if (row[i] < p.q_rows)
        x[i] = *reinterpret_cast<const uint4 *>(p.q + (bh * p.q_rows + row[i]) * p.D + 8 * ch);
    } else if (row[i] < p.len) {
      const int64_t at = bh * p.cap + row[i];
      const bool v = which[i] == 2;
      x[i].x = (v ? p.c.v_codes : p.c.k_codes)[at * W + (ch & 3) * (p.D / 32) + (ch >> 2)];
      x[i].y = (v ? p.c.v_scales : p.c.k_scales)[at * (p.D / p.group) + 8 * ch / p.group];
    }
  }
  // (the kernel in front was launched behind all that wrote q and the cache)
  wait_for_earlier();
  let_next_launch();
  if (threadIdx.x < 32) {
    float m[3] = {0.f, 0.f, 0.f};
    for (int s = threadIdx.x; s < p.slices; s += 32) {
      const float4 y = p.maxima[int64_t(s) * gridDim.y + bh];
      m[0] = fmaxf(m[0], y.x), m[1] = fmaxf(m[1], y.y), m[2] = fmaxf(m[2], y.z);
    }
    int e[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) e[i] = exponent(warp_max(m[i]));
    if (threadIdx.x == 0) {
#pragma unroll
      for (int i = 0; i < 3; ++i) e[i] = max(-100, e[i] - 14);  // (at most 114)
      scale[0] = p.scale < 0.f ? -pow2(-e[0]) : pow2(-e[0]);  // (the scores' factor is positive)
      scale[1] = pow2(-e[1]);
      scale[2] = pow2(-e[2]);
      if (blockIdx.x == 0) {
        // In log2 units.  Not 0, which would turn masked scores into 0 * inf, and finite:
        // scores reach 2^35.
        const float s = scalbnf(fabsf(p.scale) * 1.4426950408889634f, e[0] + e[1]);
        p.scales[bh] = make_float2(fminf(fmaxf(s, 0x1p-120f), 0x1p90f), pow2(e[2]));
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (which[i] == 0 && row[i] >= p.q_rows) continue;
    const float f = scale[which[i]];
    uint32_t o[4];
    if (which[i] == 0) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        unpack_bf2(w[k], a, b);
        // (an infinity makes NaN of a row's scores sooner or later)
        o[k] = nonfinite(w[k]) ? 0x7fff7fffu : pack_h2(a * f, b * f);
      }
    } else {
      if (nonfinite(x[i].y)) {
        // a value's group covers its own channels; a key's score is NaN, and so are all
        for (int c = which[i] == 2 ? ch / 4 : 0; c < (which[i] == 2 ? ch / 4 + 1 : 4); ++c)
          atomicMin(&p.nan[bh * 4 + c], static_cast<int>(row[i]));
        x[i].x = x[i].y = 0u;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        o[k] = pack_h2(saturate(q4::value(q4::code_of(x[i].x, 2 * k), x[i].y) * f),
                       saturate(q4::value(q4::code_of(x[i].x, 2 * k + 1), x[i].y) * f));
    }
    __half *dst = which[i] == 0 ? p.qo + (bh * p.q_rows + row[i]) * kPad
                                : (which[i] == 2 ? p.vo : p.ko) + (bh * p.pad + row[i]) * kPad;
    reinterpret_cast<uint4 *>(dst)[ch] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

// Joins the splits; a thread owns 4 channels of a query row.
__global__ void __launch_bounds__(kThreads) attn_q4_splits_kernel(F16Extra x, uint16_t *out, int Hq,
                                                                  int64_t Sq) {
  wait_for_earlier();
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t row = i / (x.D / 4);
  const int ch = static_cast<int>(i - row * (x.D / 4)) * 4;
  if (row >= x.rows) return;
  const float2 *ml = reinterpret_cast<const float2 *>(x.part + x.rows * x.splits * x.D) + row * x.splits;
  const float *part = x.part + row * x.splits * x.D + ch;
  float top = -FLT_MAX, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < x.splits; ++s) top = fmaxf(top, ml[s].x);
#pragma unroll 2
  for (int s = 0; s < x.splits; ++s) {
    const float2 w = ml[s];
    const float4 o = *reinterpret_cast<const float4 *>(part + int64_t(s) * x.D);
    const float f = exp2f(w.x - top);
    l = fmaf(w.y, f, l);
    v.x = fmaf(o.x, f, v.x);
    v.y = fmaf(o.y, f, v.y);
    v.z = fmaf(o.z, f, v.z);
    v.w = fmaf(o.w, f, v.w);
  }
  const float inv = l == 0.f ? 0.f : (1.f / kPartScale) / l;
  const int64_t bh = row / Sq, sq = row - bh * Sq, b = bh / Hq, h = bh - b * Hq;
  *reinterpret_cast<uint2 *>(out + ((b * Sq + sq) * Hq + h) * x.D + ch) =
      make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
}

// Splits of the key tiles and the workspace's parts, in bytes (by the device's SMs, not
// by a thread's limit: the launch takes what was asked for).
struct Plan {
  int splits, tiles_per_split, pad, slices;
  int64_t scales, nan, ko, vo, qo, part, bytes;
};
Plan plan(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len, int D) {
  Plan pl{};
  int64_t tile;
  const int ctas = attn_tc_ctas(B, Hq, Hkv, Sq, &tile);
  const int tiles = static_cast<int>((kv_len + tile - 1) / tile);
  // Splits that fill the SMs once; a split of fewer than 4 tiles costs more to begin
  // and join than it saves.
  int n = ctas > 0 ? device_sms() / ctas : 1;
  if (n > tiles / 4) n = tiles / 4;
  if (n < 1) n = 1;
  pl.tiles_per_split = (tiles + n - 1) / n;
  pl.splits = (tiles + pl.tiles_per_split - 1) / pl.tiles_per_split;
  pl.pad = static_cast<int>(tiles * tile);
  const int64_t bh = B * Hkv, rows = B * Hq * Sq;
  // about four CTAs per SM read for the largest values
  const int64_t slices = 4 * int64_t(device_sms()) / bh;
  pl.slices = static_cast<int>(slices < 2 ? 2 : slices > kMaxSlices ? kMaxSlices : slices);
  pl.scales = pl.slices * bh * int64_t(sizeof(float4));
  pl.nan = pl.scales + (bh * int64_t(sizeof(float2)) + 15) / 16 * 16;
  pl.ko = pl.nan + bh * int64_t(sizeof(int4));
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

// Fitted to 972 shapes (head_dim 32, 64 and 128, 8 to 32 heads on 1 to 8, 1 to 16
// sequences, 4 to 512 queries, 512 to 32768 keys); its choice costs 0.6 % on average
// over the better of the two measured times, a fixed limit of 256 rows 7 %.  In
// microseconds: on the codes 16 query rows pass over all keys at a time; in chunks
// a 128-key tile takes 2 in each of the CTAs the GPU holds, and the operands move at
// 5 TB/s.  (32 heads on 4, 8192 keys: 512 queries 355 on the codes, 100 in chunks; 64
// queries 68 and 46; 16 queries 25 and 44.)
extern "C" int q35_attn_q4_prefers_chunk(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len,
                                         int D) {
  if (!plannable(B, Hq, Hkv, Sq, kv_len) || Hq % Hkv != 0 || B * Hq > 65535) return 0;
  const Plan pl = plan(B, Hq, Hkv, Sq, kv_len, D);
  int64_t tile;
  const double ctas = static_cast<double>(attn_tc_ctas(B, Hq, Hkv, Sq, &tile)) * pl.splits;
  const double waves = static_cast<double>((static_cast<int64_t>(ctas) + device_sms() - 1) / device_sms());
  const double passes = static_cast<double>((Hq / Hkv * Sq + 15) / 16);
  const double keys = static_cast<double>(B) * Hkv * kv_len;
  const double bytes = keys * (1.25 * D + 1024) + static_cast<double>(B) * Hq * Sq * 768;
  const double chunk = 14 + 2 * waves * pl.tiles_per_split + bytes * 0.2e-6;
  const double codes = 12 + keys * passes * (D + 96) * 0.16e-6;
  return chunk < codes ? 1 : 0;
}

extern "C" int q35_attn_q4_chunk_fwd(const void *q, const void *k_codes, const void *k_scales,
                                     const void *v_codes, const void *v_scales, void *out,
                                     int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len,
                                     int64_t cap, int D, int group, float scale, int causal,
                                     void *workspace, q35_stream_t stream) {
  int st = q4::check_cache("attn_q4_chunk", k_codes, k_scales, v_codes, v_scales, B, Hkv, D, group,
                           cap);
  if (st) return st;
  if (Sq < 0 || Sq >= int64_t(1) << 31 || kv_len < 1 || Hq <= 0 || Hq % Hkv != 0)
    return fail(Q35_ERR_SHAPE, "attn_q4_chunk: Sq %lld, kv_len %lld, Hq %d, Hkv %d", (long long)Sq,
                (long long)kv_len, Hq, Hkv);
  if (kv_len > cap)
    return fail(Q35_ERR_SHAPE, "attn_q4_chunk: %lld rows exceed the capacity %lld",
                (long long)kv_len, (long long)cap);
  if (const int bad = q4::check_scale("attn_q4_chunk", scale)) return bad;
  if (B == 0 || Sq == 0) return Q35_OK;
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
  c.scales = reinterpret_cast<float2 *>(ws + pl.scales);
  c.nan = reinterpret_cast<int *>(ws + pl.nan);
  c.ko = reinterpret_cast<__half *>(ws + pl.ko);
  c.vo = reinterpret_cast<__half *>(ws + pl.vo);
  c.qo = reinterpret_cast<__half *>(ws + pl.qo);
  c.D = D;
  c.group = group;
  c.q_rows = static_cast<int>(Hq / Hkv * Sq);
  c.cap = cap;
  c.len = static_cast<int>(kv_len);
  c.pad = pl.pad;
  c.slices = pl.slices;
  c.scale = scale;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const unsigned bh = static_cast<unsigned>(B * Hkv);
  attn_q4_absmax_kernel<<<dim3(pl.slices, bh), kThreads, 0, s>>>(c);
  Q35_LAUNCH_CHECK("attn_q4 absmax launch");
  const int64_t rows = 2 * int64_t(c.pad) + c.q_rows, step = kRows * kThreads / 16;
  Q35_CHECK_CUDA(launch_early(attn_q4_operands_kernel,
                              dim3(static_cast<unsigned>((rows + step - 1) / step), bh), dim3(kThreads),
                              0, s, c));
  Q35_LAUNCH_CHECK("attn_q4 operands launch");
  F16Extra x{};
  x.scales = c.scales;
  x.nan = c.nan;
  x.rows = B * Hq * Sq;
  x.splits = pl.splits;
  x.tiles_per_split = pl.tiles_per_split;
  x.D = D;
  x.part = pl.splits > 1 ? reinterpret_cast<float *>(ws + pl.part) : nullptr;
  st = attn_tc_f16(c.qo, c.ko, c.vo, out, B, Hq, Hkv, Sq, kv_len, c.pad, causal, x, stream);
  if (st) return st;
  if (pl.splits > 1) {
    Q35_CHECK_CUDA(launch_early(
        attn_q4_splits_kernel, dim3(static_cast<unsigned>((x.rows * (D / 4) + kThreads - 1) / kThreads)),
        dim3(kThreads), 0, s, x, static_cast<uint16_t *>(out), Hq, Sq));
    Q35_LAUNCH_CHECK("attn_q4 splits launch");
  }
  return Q35_OK;
}
