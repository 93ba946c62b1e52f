// Attention over a 4-bit KV cache (layout: kv_q4.cuh).
//
// out[b, s, h D + d] = sum_k p_k V[k, d] / sum_k p_k, p_k = exp(scale q . K[k] - max),
// over the keys k < len_b, with a causal mask aligned to the last key (query s
// of Sq sees k <= s + len_b - Sq).  A row that sees no key is zero.
//
// What bounds it: a key and its value are 160 bytes at D = 128 (groups of 32),
// read once, so a long cache should run at memory speed; but each of those bytes
// is two codes to unpack, so the instructions per code decide.  Per SM and clock
// HBM delivers about 24 bytes = 48 codes against 128 lanes of issue.
//
// Codes as bf16.  The bits c << 4 (c = 0..15) read as bf16 are c * 2^-129 and the
// bits c are c * 2^-133: bf16's subnormals and its first binade are evenly
// spaced.  The matrix units and fma.bf16x2 take subnormals at full precision, so
// `w & 0x000f000f` and `w & 0x00f000f0` are pairs of codes as they stand, without
// a conversion or an offset to take out again; one shift by 8 gives the other
// four codes of a word.  The powers of two go into the other operand.
//
// Scores.  With K = m + s c per group j, q . K = sum_j s_j (Q_j . c_j) + m_j sum(Q_j).
// Q is scaled by 2^52 (codes at bit 0) or 2^48 (at bit 4), so a product is
// 2^-81 Q . c; the minima go through one more matrix instruction whose other
// operand is 2^-81 sum(Q_j) split into three bf16 parts (24 bits).  So K is never
// rounded, and the scale costs one fp32 operation per key, query and group.
// |Q| must stay below 2^75.
//
// Keys are the 16 rows of the instruction and queries its 8 columns (S^T = K Q^T,
// O^T = V^T P^T): a decode step has G = Hq/Hkv queries per kv head, often 8, and
// no half of the tile is idle.  P moves from accumulator to operand layout by an
// 8x8 transpose between the lanes (movmatrix).  P is rounded to bf16 (as in the
// bf16 attention kernels), V is dequantised to bf16 in registers, one rounding of
// m + s c: what a read back gives, as (2^-129 c) (2^69 s) + 2^-60 m, or 2^-64 of the
// value for codes at bit 0 (exact scales: |V| between 2^-60 and 2^58).
//
// Each warp walks its own 32-key tiles with a private ring of bulk copies (four
// per tile: K codes, K scales, V codes, V scales, all contiguous in memory), so
// no warp waits for another before the end.  Within a block of 8 keys, row r of
// the instruction is key pi(r) = 0,3,1,2,6,5,7,4: the four keys a V load touches
// are then on both sides of the 128-byte bank window at every head size.
#include "kv_q4.cuh"
#include "sm100.cuh"

#include <float.h>

#include <type_traits>

namespace q35 {
namespace {

using q4::Cache;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 32;    // keys per tile
constexpr int kStages = 3;   // tiles in flight per warp

struct Params {
  const uint16_t *q;
  Cache c;
  uint16_t *out;
  float *ws;
  const int32_t *kv_lens;
  int *err;
  int Hq, Hkv, G, Sq, R, n_rg, n_splits, causal;
  int64_t kv_len, cap;
  float scale_log2;
};

template <int D, int GS>
struct Layout {
  static constexpr int J = D / 32;       // code words per lane and key
  static constexpr int NS = D / GS;      // scale words per key
  static constexpr int kCodes = kTile * D / 2, kScales = kTile * NS * 4;
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kRing = kStages * kStage;
  static constexpr int kRowF = D + 4;    // floats per row of the warps' merge
  static constexpr int smem(int nt) {
    const int merge = kWarps * 8 * nt * kRowF * 4;
    return kWarps * kRing > merge ? kWarps * kRing : merge;
  }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
      : "memory");
}
// D = A(16x16 bf16) * B(16x8 bf16) + C, fp32.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1,
                                    float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The codes of fields 0..3 and 4..7 of a word as bf16 pairs (field i, field i + 4):
// c * 2^-133 for i = 0, 2 and c * 2^-129 for i = 1, 3.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t (&c)[4]) {
  const uint32_t h = w >> 8;
  c[0] = w & 0x000f000fu;
  c[1] = w & 0x00f000f0u;
  c[2] = h & 0x000f000fu;
  c[3] = h & 0x00f000f0u;
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// Powers of two as bf16 bits.
constexpr uint32_t pow2_bf16(int e) { return static_cast<uint32_t>(127 + e) << 7; }
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t addr) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ bool nonfinite(uint32_t pair) {
  return (((pair & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
}

// One CTA = (sequence, kv head, group of 8 NT query rows, split of the keys).
template <int D, int GS, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2) attn_q4_kernel(Params p) {
  using L = Layout<D, GS>;
  constexpr int J = L::J, NS = L::NS, BPG = GS / 32;
  constexpr int WV = D >= 64 ? D / 64 : 1;      // V words per lane and key
  constexpr int MT = D / 16;                    // 16-channel tiles of O^T
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWarps][kStages];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  int64_t id = blockIdx.x;
  const int split = static_cast<int>(id % p.n_splits);
  id /= p.n_splits;
  const int rg = static_cast<int>(id % p.n_rg);
  const int64_t bh = id / p.n_rg;
  const int b = static_cast<int>(bh / p.Hkv), hk = static_cast<int>(bh - int64_t(b) * p.Hkv);

  int len = static_cast<int>(p.kv_len);
  if (p.kv_lens) {
    const int n = p.kv_lens[b];
    if (n < 0 || n > len) {
      if (tid == 0) report_error(p.err, DEV_ERR_INDEX, 311, b, n);
      len = n < 0 ? 0 : len;
    } else {
      len = n;
    }
  }
  const int n_tiles_all = (len + kTile - 1) / kTile;
  const int per = (n_tiles_all + p.n_splits - 1) / p.n_splits;  // tiles of a split
  const int tile0 = min(split * per, n_tiles_all), tile1 = min(tile0 + per, n_tiles_all);

  const int64_t row0 = bh * p.cap;
  const uint8_t *kc = reinterpret_cast<const uint8_t *>(p.c.k_codes) + row0 * (D / 2);
  const uint8_t *vc = reinterpret_cast<const uint8_t *>(p.c.v_codes) + row0 * (D / 2);
  const uint8_t *ks = reinterpret_cast<const uint8_t *>(p.c.k_scales) + row0 * (NS * 4);
  const uint8_t *vs = reinterpret_cast<const uint8_t *>(p.c.v_scales) + row0 * (NS * 4);
  const uint32_t ring = sm100::smem_u32(smem) + warp * L::kRing;

  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(&bars[warp][i], 1);
    sm100::fence_mbar_init();
  }
  __syncwarp();
  // Copies tile `tl` into a stage (lane 0).  The last tile copies whole groups of
  // 4 rows: 16-byte sizes at every scale width, inside the capacity (a multiple of 16).
  auto issue = [&](int tl, int stage) {
    const int r0 = tl * kTile;
    const uint32_t n = static_cast<uint32_t>(min(kTile, (len - r0 + 3) & ~3));
    const uint32_t dst = ring + stage * L::kStage;
    uint64_t *bar = &bars[warp][stage];
    sm100::mbar_arrive_expect_tx(bar, n * (D + 8 * NS));
    bulk_load(dst, kc + int64_t(r0) * (D / 2), n * (D / 2), bar);
    bulk_load(dst + L::kCodes, ks + int64_t(r0) * (NS * 4), n * (NS * 4), bar);
    bulk_load(dst + L::kCodes + L::kScales, vc + int64_t(r0) * (D / 2), n * (D / 2), bar);
    bulk_load(dst + 2 * L::kCodes + L::kScales, vs + int64_t(r0) * (NS * 4), n * (NS * 4), bar);
  };
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i)
      if (tile0 + warp + i * kWarps < tile1) issue(tile0 + warp + i * kWarps, i);
  }

  // Query rows: row r -> head hk G + r / Sq, position r % Sq.  Column g of an
  // operand tile holds 8 channels of every 32; accumulator columns are 2t, 2t + 1.
  uint32_t qf[NT][J][4];
  uint32_t qm[NT][2];  // 2^-81 sum(Q_t) of group t in three bf16 parts
  int lim[NT][2];      // keys the column's query sees
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = (rg * NT + nt) * 8 + g;
    const uint16_t *src = nullptr;
    if (r < p.R) {
      const int h = r / p.Sq, s = r - h * p.Sq;
      src = p.q + ((int64_t(b) * p.Hq + hk * p.G + h) * p.Sq + s) * D;
    }
    float sum[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) sum[j] = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint4 x = src ? *reinterpret_cast<const uint4 *>(src + 32 * j + 8 * t)
                          : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float lo, hi;
        unpack_bf2(xs[i], lo, hi);
        sum[j / BPG] += lo + hi;
        const float up = i % 2 == 0 ? 0x1p52f : 0x1p48f;
        qf[nt][j][i] = pack_bf2(lo * up, hi * up);
      }
    }
    float mine = 0.f;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      float v = sum[j];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (j == t) mine = v * 0x1p-81f;
    }
    const float h0 = bf2f(f2bf(mine)), h1 = bf2f(f2bf(mine - h0));
    qm[nt][0] = pack_bf2(h0, h1);
    qm[nt][1] = pack_bf2(mine - h0 - h1, 0.f);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int rc = (rg * NT + nt) * 8 + 2 * t + c;
      lim[nt][c] = p.causal ? min(len, len - p.Sq + rc % p.Sq + 1) : len;
    }
  }
  const int lim_all = p.causal ? min(len, len - p.Sq + 1) : len;  // keys every query sees

  float o[MT][NT][4];
  float row_m[NT][2], row_l[NT][2];  // in units of log2; l of this lane's keys only
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    row_m[nt][0] = row_m[nt][1] = -FLT_MAX;
    row_l[nt][0] = row_l[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
  }

  const int pig = ((g >> 1) + (g >= 4 ? 4 : 0)) ^ ((g & 1) * 3);  // pi(g)
  const int pit = t + (t >= 2 ? 4 : 0);                           // pi(2t); pi(2t + 1) = pit ^ 3
  const int jv = D == 128 ? 2 * (g & 1) : (D == 64 ? (g & 1) : 0);  // 32-channel block of V word 0

  constexpr uint32_t kUpS = pow2_bf16(69) * 0x10001u, kDownM0 = pow2_bf16(-64) * 0x10001u,
                     kDownM1 = pow2_bf16(-60) * 0x10001u;
  const float scale_up = p.scale_log2 * 0x1p81f;
  bool ok = true;
  int stage = 0, phase = 0;
  int tl = tile0 + warp;
  for (; tl < tile1; tl += kWarps) {
    if (!sm100::mbar_wait(&bars[warp][stage], phase)) {
      report_error(p.err, DEV_ERR_WAIT_TIMEOUT, 312, static_cast<int>(bh), tl);
      ok = false;
      break;
    }
    const uint32_t sk = ring + stage * L::kStage;
    const uint32_t sks = sk + L::kCodes, sv = sks + L::kScales, svs = sv + L::kCodes;
    const int key0 = tl * kTile;
    const bool masked = key0 + kTile > lim_all;

    // ---- S^T = K Q^T (two blocks of 16 keys), in units of log2
    float s[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t wl[J], wh[J], pl[NS], ph[NS], ml[1], mh[1];
      const int kl = 16 * mt + pig;
      lds_words<J>(wl, sk + kl * (D / 2) + t * (4 * J));
      lds_words<J>(wh, sk + (kl + 8) * (D / 2) + t * (4 * J));
      lds_words<NS>(pl, sks + kl * (NS * 4));
      lds_words<NS>(ph, sks + (kl + 8) * (NS * 4));
      lds_words<1>(ml, sks + (kl * NS + t % NS) * 4);
      lds_words<1>(mh, sks + ((kl + 8) * NS + t % NS) * 4);
      // minima: (m, m, m) of group t times the parts of its sum(Q)
      const uint32_t m0 = __byte_perm(ml[0], 0u, 0x3232), m1 = __byte_perm(mh[0], 0u, 0x3232);
      float part[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        mma(s[mt][nt], m0, m1, m0, m1, qm[nt][0], qm[nt][1], 0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t a[4], c[4];
        codes4(wl[j], a);
        codes4(wh[j], c);
        const int sg = j / BPG;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (j % BPG == 0)
            mma(part[nt], a[0], c[0], a[1], c[1], qf[nt][j][0], qf[nt][j][1], 0.f, 0.f, 0.f, 0.f);
          else
            mma(part[nt], a[0], c[0], a[1], c[1], qf[nt][j][0], qf[nt][j][1], part[nt][0],
                part[nt][1], part[nt][2], part[nt][3]);
          mma(part[nt], a[2], c[2], a[3], c[3], qf[nt][j][2], qf[nt][j][3], part[nt][0],
              part[nt][1], part[nt][2], part[nt][3]);
        }
        if (j % BPG == BPG - 1) {
          const float s0 = __uint_as_float(pl[sg] << 16), s1 = __uint_as_float(ph[sg] << 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            s[mt][nt][0] = fmaf(s0, part[nt][0], s[mt][nt][0]);
            s[mt][nt][1] = fmaf(s0, part[nt][1], s[mt][nt][1]);
            s[mt][nt][2] = fmaf(s1, part[nt][2], s[mt][nt][2]);
            s[mt][nt][3] = fmaf(s1, part[nt][3], s[mt][nt][3]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][nt][e] *= scale_up;
    }

    if (masked) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + 16 * mt + pig + 8 * (e >> 1) >= lim[nt][e & 1]) s[mt][nt][e] = -INFINITY;
      // A weight of 0 does not silence a NaN or an infinity in V: rows behind the
      // length are cleared, and a non-finite group that some query must not see is
      // cleared too and put into the outputs of the queries that do see it.
      const bool behind = key0 + lane >= len;
      uint32_t clear = behind ? (1u << NS) - 1u : 0u;  // groups of key row `lane`
      if (!behind) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          uint32_t w[1];
          lds_words<1>(w, svs + (lane * NS + i) * 4);
          if (nonfinite(w[0])) clear |= 1u << i;
        }
      }
      uint32_t todo = __ballot_sync(0xffffffffu, clear != 0 && !behind);
      while (todo) {
        const int kk = __ffs(todo) - 1;
        todo &= todo - 1;
#pragma unroll
        for (int w = 0; w < WV; ++w) {
          uint32_t pr[1];
          lds_words<1>(pr, svs + (kk * NS + (jv + w) / BPG) * 4);
          if (nonfinite(pr[0])) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int i = 0; i < MT / WV; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (key0 + kk < lim[nt][e & 1]) o[w * (MT / WV) + i][nt][e] = NAN;
          }
        }
      }
      __syncwarp();
      if (clear) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (clear >> i & 1u)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(svs + (lane * NS + i) * 4), "r"(0u) : "memory");
      }
      __syncwarp();
    }

    // ---- softmax: the maximum is raised (and O rescaled) only when some key exceeds it
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx0 = fmaxf(fmaxf(s[0][nt][0], s[0][nt][2]), fmaxf(s[1][nt][0], s[1][nt][2]));
      float mx1 = fmaxf(fmaxf(s[0][nt][1], s[0][nt][3]), fmaxf(s[1][nt][1], s[1][nt][3]));
      if (__any_sync(0xffffffffu, mx0 > row_m[nt][0] || mx1 > row_m[nt][1])) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
        }
        mx0 = fmaxf(mx0, row_m[nt][0]);
        mx1 = fmaxf(mx1, row_m[nt][1]);
        const float a0 = exp2_fast(row_m[nt][0] - mx0), a1 = exp2_fast(row_m[nt][1] - mx1);
        row_m[nt][0] = mx0;
        row_m[nt][1] = mx1;
        row_l[nt][0] *= a0;
        row_l[nt][1] *= a1;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          o[i][nt][0] *= a0;
          o[i][nt][1] *= a1;
          o[i][nt][2] *= a0;
          o[i][nt][3] *= a1;
        }
      }
      const float mu0 = row_m[nt][0], mu1 = row_m[nt][1];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float p0 = exp2_fast(s[mt][nt][0] - mu0), p1 = exp2_fast(s[mt][nt][1] - mu1);
        const float p2 = exp2_fast(s[mt][nt][2] - mu0), p3 = exp2_fast(s[mt][nt][3] - mu1);
        row_l[nt][0] += p0 + p2;
        row_l[nt][1] += p1 + p3;
        pb[mt][nt][0] = transpose8x8(pack_bf2(p0, p1));
        pb[mt][nt][1] = transpose8x8(pack_bf2(p2, p3));
      }
    }

    // ---- O^T += V^T P^T
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const int ka = 16 * mt + pit, kb = 16 * mt + (pit ^ 3);
      uint32_t wa[WV], wb[WV], wa8[WV], wb8[WV];
      if constexpr (D == 32) {
        wa[0] = lds_u16(sv + ka * 16 + g * 2);
        wb[0] = lds_u16(sv + kb * 16 + g * 2);
        wa8[0] = lds_u16(sv + (ka + 8) * 16 + g * 2);
        wb8[0] = lds_u16(sv + (kb + 8) * 16 + g * 2);
      } else {
        lds_words<WV>(wa, sv + ka * (D / 2) + g * (4 * WV));
        lds_words<WV>(wb, sv + kb * (D / 2) + g * (4 * WV));
        lds_words<WV>(wa8, sv + (ka + 8) * (D / 2) + g * (4 * WV));
        lds_words<WV>(wb8, sv + (kb + 8) * (D / 2) + g * (4 * WV));
      }
      constexpr int PS = WV > BPG ? WV / BPG : 1;  // scale words per lane and key
      uint32_t pa[PS], pbb[PS], pa8[PS], pb8[PS];
      lds_words<PS>(pa, svs + (ka * NS + jv / BPG) * 4);
      lds_words<PS>(pbb, svs + (kb * NS + jv / BPG) * 4);
      lds_words<PS>(pa8, svs + ((ka + 8) * NS + jv / BPG) * 4);
      lds_words<PS>(pb8, svs + ((kb + 8) * NS + jv / BPG) * 4);
#pragma unroll
      for (int w = 0; w < WV; ++w) {
        const int sw = w * PS / WV;
        // (key a, key b) pairs of scales and minima, with their powers of two, and of codes
        const uint32_t s2 = mul2(__byte_perm(pa[sw], pbb[sw], 0x5410), kUpS);
        const uint32_t m2[2] = {mul2(__byte_perm(pa[sw], pbb[sw], 0x7632), kDownM0),
                                mul2(__byte_perm(pa[sw], pbb[sw], 0x7632), kDownM1)};
        const uint32_t s28 = mul2(__byte_perm(pa8[sw], pb8[sw], 0x5410), kUpS);
        const uint32_t m28[2] = {mul2(__byte_perm(pa8[sw], pb8[sw], 0x7632), kDownM0),
                                 mul2(__byte_perm(pa8[sw], pb8[sw], 0x7632), kDownM1)};
        uint32_t x[4], x8[4], y[4], y8[4];
        codes4(__byte_perm(wa[w], wb[w], 0x5410), x);
        codes4(__byte_perm(wa8[w], wb8[w], 0x5410), x8);
        if constexpr (D > 32) {
          codes4(__byte_perm(wa[w], wb[w], 0x7632), y);
          codes4(__byte_perm(wa8[w], wb8[w], 0x7632), y8);
        }
#pragma unroll
        for (int i = 0; i < MT / WV; ++i) {
          // channels of rows g and g + 8: fields i, i + 4 (D = 32: i, i + 2 of a half word)
          const uint32_t a0 = fma2(x[i], s2, m2[i % 2]);
          const uint32_t a1 = fma2(D == 32 ? x[i + 2] : y[i], s2, m2[i % 2]);
          const uint32_t a2 = fma2(x8[i], s28, m28[i % 2]);
          const uint32_t a3 = fma2(D == 32 ? x8[i + 2] : y8[i], s28, m28[i % 2]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float(&acc)[4] = o[w * (MT / WV) + i][nt];
            mma(acc, a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1], acc[0], acc[1], acc[2], acc[3]);
          }
        }
      }
    }
    // cleared scales (ordinary stores) before the next bulk copy into this stage
    if (masked) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0 && tl + kStages * kWarps < tile1) issue(tl + kStages * kWarps, stage);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  if (!ok) {
    // give up: let the copies still in flight land (bounded) before the block ends
    for (int i = 1; i < kStages; ++i) {
      tl += kWarps;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
      if (tl < tile1) sm100::mbar_wait(&bars[warp][stage], phase);
    }
  }

  // ---- join the warps: [warp][row][D channels, m, l]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][nt][e] *= i % 2 == 0 ? 0x1p64f : 0x1p60f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1)
        row_l[nt][c] += __shfl_xor_sync(0xffffffffu, row_l[nt][c], d);
  __syncthreads();
  float *sm = reinterpret_cast<float *>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float *row = sm + (warp * 8 * NT + nt * 8 + 2 * t + c) * L::kRowF;
      if constexpr (D == 32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          row[8 * (g >> 1) + 2 * i + (g & 1)] = o[i][nt][c];
          row[8 * (g >> 1) + 2 * (i + 2) + (g & 1)] = o[i][nt][c + 2];
        }
      } else {
#pragma unroll
        for (int w = 0; w < WV; ++w) {
          float4 *dst = reinterpret_cast<float4 *>(row + 32 * (jv + w) + 8 * (g >> 1));
          const int i0 = w * (MT / WV);
          dst[0] = make_float4(o[i0][nt][c], o[i0][nt][c + 2], o[i0 + 1][nt][c], o[i0 + 1][nt][c + 2]);
          dst[1] = make_float4(o[i0 + 2][nt][c], o[i0 + 2][nt][c + 2], o[i0 + 3][nt][c],
                               o[i0 + 3][nt][c + 2]);
        }
      }
      if (g == 0) {
        row[D] = row_m[nt][c];
        row[D + 1] = row_l[nt][c];
      }
    }
  __syncthreads();
  for (int it = tid; it < 8 * NT * (D / 4); it += kThreads) {
    const int lr = it / (D / 4), ch = (it - lr * (D / 4)) * 4;
    const int r = rg * 8 * NT + lr;
    if (r >= p.R) continue;
    float M = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[(w * 8 * NT + lr) * L::kRowF + D]);
    float l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float *row = sm + (w * 8 * NT + lr) * L::kRowF;
      const float f = exp2_fast(row[D] - M);
      l += row[D + 1] * f;
      const float4 x = *reinterpret_cast<const float4 *>(row + ch);
      acc.x += x.x * f;
      acc.y += x.y * f;
      acc.z += x.z * f;
      acc.w += x.w * f;
    }
    if (p.n_splits == 1) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const int h = r / p.Sq, sq = r - h * p.Sq;
      uint2 v = make_uint2(pack_bf2(acc.x * inv, acc.y * inv), pack_bf2(acc.z * inv, acc.w * inv));
      *reinterpret_cast<uint2 *>(p.out + ((int64_t(b) * p.Sq + sq) * p.Hq + hk * p.G + h) * D + ch) = v;
    } else {
      const int64_t rows = int64_t(gridDim.x) / (int64_t(p.n_splits) * p.n_rg) * p.R * p.n_splits;
      const int64_t at = (bh * p.R + r) * p.n_splits + split;
      *reinterpret_cast<float4 *>(p.ws + at * D + ch) = acc;
      if (ch == 0) *reinterpret_cast<float2 *>(p.ws + rows * D + at * 2) = make_float2(M, l);
    }
  }
}

// One warp per query row: joins the splits.
template <int D>
__global__ void __launch_bounds__(128) attn_q4_join_kernel(Params p, int64_t rows) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t gr = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (gr >= rows) return;
  const float2 *ml = reinterpret_cast<const float2 *>(p.ws + rows * p.n_splits * D) + gr * p.n_splits;
  const float *acc = p.ws + gr * p.n_splits * D + lane * E;
  float M = -FLT_MAX;
  for (int s = lane; s < p.n_splits; s += 32) M = fmaxf(M, ml[s].x);
  M = warp_max(M);
  float l = 0.f, v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.n_splits; ++s) {
    const float2 x = ml[s];
    const float f = exp2_fast(x.x - M);
    l += x.y * f;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] += acc[int64_t(s) * D + e] * f;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int64_t bh = gr / p.R;
  const int r = static_cast<int>(gr - bh * p.R);
  const int64_t b = bh / p.Hkv;
  const int hk = static_cast<int>(bh - b * p.Hkv), h = r / p.Sq, sq = r - h * p.Sq;
  uint16_t *dst = p.out + ((b * p.Sq + sq) * p.Hq + hk * p.G + h) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = f2bf(v[e] * inv);
}

// Rows per CTA and splits of the keys.
struct Plan {
  int nt, n_rg, n_splits;
};
Plan plan(int64_t B, int Hkv, int64_t R, int64_t kv_len) {
  Plan pl;
  pl.nt = R > 8 ? 2 : 1;
  pl.n_rg = static_cast<int>((R + 8 * pl.nt - 1) / (8 * pl.nt));
  const int64_t groups = B * Hkv * pl.n_rg;
  const int64_t want = (2LL * 148 * 3) / (groups > 0 ? groups : 1);
  const int64_t most = (kv_len + 4 * kTile - 1) / (4 * kTile);
  int64_t n = want < most ? want : most;
  pl.n_splits = static_cast<int>(n < 1 ? 1 : n);
  return pl;
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int64_t q35_attn_q4_workspace(int64_t B, int Hq, int Hkv, int64_t Sq, int64_t kv_len,
                                         int D) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || Sq <= 0 || D <= 0) return 0;
  const Plan pl = plan(B, Hkv, Hq / Hkv * Sq, kv_len);
  if (pl.n_splits == 1) return 0;
  return B * Hq * Sq * pl.n_splits * (static_cast<int64_t>(D) + 2);
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
  const int64_t R = Hq / Hkv * Sq;
  if (R >= (int64_t(1) << 30)) return fail(Q35_ERR_SHAPE, "attn_q4: %lld query rows", (long long)R);
  const Plan pl = plan(B, Hkv, R, kv_len);
  if (pl.n_splits > 1 && !workspace) return fail(Q35_ERR_INVALID, "attn_q4: no workspace");
  if (pl.n_splits > 1 && !aligned16(workspace))
    return fail(Q35_ERR_ALIGN, "attn_q4: workspace not 16-byte aligned");
  int *err = device_error_word();
  if (!err) return fail(Q35_ERR_CUDA, "attn_q4: no device error word");
  Params p{};
  p.q = static_cast<const uint16_t *>(q);
  p.c = Cache{static_cast<uint32_t *>(const_cast<void *>(k_codes)),
              static_cast<uint32_t *>(const_cast<void *>(k_scales)),
              static_cast<uint32_t *>(const_cast<void *>(v_codes)),
              static_cast<uint32_t *>(const_cast<void *>(v_scales))};
  p.out = static_cast<uint16_t *>(out);
  p.ws = workspace;
  p.kv_lens = kv_lens;
  p.err = err;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  p.Sq = static_cast<int>(Sq);
  p.R = static_cast<int>(R);
  p.n_rg = pl.n_rg;
  p.n_splits = pl.n_splits;
  p.causal = causal ? 1 : 0;
  p.kv_len = kv_len;
  p.cap = cap;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int64_t blocks = B * Hkv * pl.n_rg * pl.n_splits, rows = B * Hkv * R;
  if (blocks >= (int64_t(1) << 31) || rows >= (int64_t(1) << 32))
    return fail(Q35_ERR_SHAPE, "attn_q4: too many rows");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto d, auto gs, auto nt) -> int {
    auto *kern = &attn_q4_kernel<d(), gs(), nt()>;
    constexpr int smem = Layout<d(), gs()>::smem(nt());
    const int e = ensure_smem_attr(reinterpret_cast<const void *>(kern), smem);
    if (e) return e;
    kern<<<static_cast<unsigned>(blocks), kThreads, smem, s>>>(p);
    Q35_LAUNCH_CHECK("attn_q4 launch");
    if (pl.n_splits > 1) {
      attn_q4_join_kernel<d()><<<static_cast<unsigned>((rows + 3) / 4), 128, 0, s>>>(p, rows);
      Q35_LAUNCH_CHECK("attn_q4 join launch");
    }
    return Q35_OK;
  };
  using std::integral_constant;
  auto by_nt = [&](auto d, auto gs) {
    return pl.nt == 2 ? go(d, gs, integral_constant<int, 2>{}) : go(d, gs, integral_constant<int, 1>{});
  };
  integral_constant<int, 128> c128;
  integral_constant<int, 64> c64;
  integral_constant<int, 32> c32;
  if (D == 128) return group == 128 ? by_nt(c128, c128) : group == 64 ? by_nt(c128, c64) : by_nt(c128, c32);
  if (D == 64) return group == 64 ? by_nt(c64, c64) : by_nt(c64, c32);
  return by_nt(c32, c32);
}
