// Writing rows into a 4-bit KV cache and reading them back (layout: kv_q4.cuh).
//
// For a group of `group` channels with minimum m and maximum M:
//   s = bf16((M - m) / 15), c = min(15, rint((x - m) / s)), value = m + c s.
// m is a bf16 input and is stored exactly; s is rounded to nearest once and the
// codes are taken with the rounded s, so a value is off by at most s/2, and by
// 15 * 2^-8 s more at the top of its group.  s = 0 (all equal, or (M - m) / 15 below
// the smallest bf16) stores codes of 0.  A group that holds a NaN or an infinity
// stores s = m = NaN and reads back as NaN.
//
// Both kernels move bytes.  A thread writes two code words of a row (16 channels),
// or reads one in each of two or four rows; group statistics go over the group/16
// neighbouring threads by shuffles, K and V share one launch.  At 20 bytes per word
// HBM feeds about 1.2 words per SM and clock, so about 100 instructions are what a
// word may cost: hence paired fp32 arithmetic, one shuffle a step for minimum and
// maximum together, and no division by S or Hkv: rows are found by multiplication, and
// in the append kernel the next one by adding up.
//
// Both are launched ahead of the kernel in front (4096 rows appended: 3.7, not 4.1 us).
//
// Measured (4 kv heads x 128): 8 x 8192 rows appended in 39.9 us with groups of 32 or 64,
// 39.2 with 128, 4.4 TB/s (223 instructions per warp and 512 channels, 40 of them paired
// fp32 at half rate; issue slots 68 % busy), 4096 rows 3.7 us, 64 sequences x 1 row 1.8 us;
// 16 x 8192 rows read in 59.0 us, 5.9 TB/s.
#include <type_traits>

#include "kv_q4.cuh"

namespace q35 {
namespace {

using q4::Cache;

constexpr int kThreads = 256;
// A CTA prefetches its next rows while it quantises: 7 CTAs of 128 threads per SM hold
// in registers (6, 7 and 8 CTAs: 8 x 8192 rows 39.8, 39.1 and 38.6 us, 4096 rows 4.0,
// 4.1 and 4.4), but for 8 bytes of spills at head_dim 128 with groups of 32 and 64, and 64
// with 32.
constexpr int kAppendThreads = 128, kAppendCtas = 7;

struct Rows {
  int64_t sb, sh, ss;  // element strides of batch, head, position
};

// What the append kernel needs of K (0) and V (1), and how far a thread's rows are apart:
// the digits of the stride in (sequence, head, position), what they and their carries
// add to the address.
struct Append {
  const uint16_t *src[2];
  uint32_t *codes[2], *scales[2];
  Rows at[2];
  uint32_t ds, dh, db, S, Hkv;
  int64_t add[2], carry_s[2], carry_h[2];
};

// n / d for 0 <= n < 2^31 by multiplication (Granlund and Montgomery): with
// L = ceil(log2 d) and m = floor(2^32 (2^L - d) / d) + 1, n / d = (mulhi(m, n) + n) >> L.
struct Divisor {
  uint32_t d, m, shift;
};
Divisor divisor(uint32_t d) {
  uint32_t l = 0;
  while ((uint64_t(1) << l) < d) ++l;
  const uint64_t m = ((uint64_t(1) << 32) * ((uint64_t(1) << l) - d)) / d + 1;
  return {d, static_cast<uint32_t>(m), l};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor &v, uint32_t &rest) {
  const uint32_t q = (__umulhi(v.m, n) + n) >> v.shift;
  rest = n - q * v.d;
  return q;
}

// Minimum and maximum of bf16 pairs; a NaN stays.
__device__ __forceinline__ uint32_t bf2_min(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t bf2_max(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// bf16((M - m) / 15) in one rounding, from 64 bits: a quotient that fp32 rounds
// onto a border between two bf16 numbers is put back on its own side.
__device__ __forceinline__ uint16_t scale_exact(float lo, float hi) {
  const double s = (static_cast<double>(hi) - static_cast<double>(lo)) / 15.0;
  float f = static_cast<float>(s);
  uint32_t u = __float_as_uint(f);
  if ((u & 0xffffu) == 0x8000u) {
    if (static_cast<double>(f) < s) u += 1;
    else if (static_cast<double>(f) > s) u -= 1;
  }
  return f2bf(__uint_as_float(u));
}
// The rounding of a quotient s32 next to a border, in fp32: 15 times the border has
// at most 13 significant bits, M - m = d + err exactly (Knuth's two-sum), and 15
// borders lie next to d.
__device__ __forceinline__ uint16_t scale_at_border(float lo, float hi, float s32) {
  const uint32_t below = __float_as_uint(s32) >> 16;
  const float border = __uint_as_float(below << 16 | 0x8000u);
  const float d = hi - lo, z = d - hi;
  const float err = (hi - (d - z)) + (-lo - z);
  const float u = fmaf(border, -15.f, d) + err;
  return static_cast<uint16_t>(below + ((u > 0.f || (u == 0.f && (below & 1u))) ? 1u : 0u));
}
__device__ __forceinline__ float code_exact(float x, float lo, float s) {
  const double y = (static_cast<double>(x) - static_cast<double>(lo)) / static_cast<double>(s);
  return static_cast<float>(fmin(rint(y), 15.0));
}

// 16 channels w (bf16 pairs) of a group -> their code words; `pair` receives the
// group's (scale, minimum).  The threads of a group are neighbours.
//
// The codes are the 64-bit rule's, halves included (x - m and s have few bits: one
// channel in 500 lies exactly on a half).  The quotient is a reciprocal's, one Newton step
// and a correction by its exact remainder (Markstein, Computation of elementary functions
// on the IBM RISC System/6000 processor, 1990): with d = x - m, r within 2^-24 of 1/s and
// y0 = d r, the rest d - y0 s is exact in one fma (it has at most 10 bits), so
// y = y0 + rest r is d / s rounded to fp32, but for 2^-23 of a step.  If d is exact, it
// is either (n + 1/2) s, then y = n + 1/2, or off by a step of d at least, which is more
// than 0.502 steps of y: then y lies on the side of d / s.  d is not exact only where
//   |m| < 2^-16 d, not 0: then |m / s| < 2^-12;
//   |x| < 2^-16 |m|, not 0: such an x can only matter where -m / s is within 2^-12 of a
//   half itself.
// Groups of the first kind (one in some thousands, if their values have one sign) and
// the tiny channels of groups of the second are decided in 64 bits one by one, and so
// are groups outside the range in which 1/s and M - m are normal numbers.  A scale
// within 4 fp32 steps of a bf16 border is decided in exact fp32 steps.
template <int GT>  // threads per group: 2, 4 or 8
__device__ __forceinline__ void quantise16(const uint32_t (&w)[8], uint32_t (&word)[2],
                                           uint32_t &pair) {
  uint32_t mn = w[0], mx = w[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    mn = bf2_min(mn, w[i]);
    mx = bf2_max(mx, w[i]);
  }
  // (minimum, -maximum) as a pair: one minimum per step serves both
  uint32_t ext = __byte_perm(mn, mx ^ 0x80008000u, 0x5410);
  ext = bf2_min(ext, __byte_perm(mn, mx ^ 0x80008000u, 0x7632));
#pragma unroll
  for (int o = 1; o < GT; o <<= 1) ext = bf2_min(ext, __shfl_xor_sync(0xffffffffu, ext, o));
  float lo, hi;
  unpack_bf2(ext, lo, hi);
  hi = -hi;
  word[0] = word[1] = 0u;
  if (((ext & 0x7f807f80u) + 0x00800080u) & 0x80008000u) {  // an infinity or a NaN
    pair = 0x7fc07fc0u;
    return;
  }
  const float d = hi - lo;
  const float s32 = d * (1.0f / 15.0f);
  const uint32_t su = __float_as_uint(s32);
  // 2^-100 <= s32 <= 2^120: 1/s and x - m stay normal numbers
  const bool plain = s32 >= 7.8886091e-31f && s32 <= 1.3292280e36f;
  const uint32_t low = (su & 0xffffu) - (0x8000u - 4u);
  uint16_t sb = f2bf(s32);
  if (!plain) sb = d == 0.f ? uint16_t(0) : scale_exact(lo, hi);
  else if (low <= 8u) sb = scale_at_border(lo, hi, s32);
  const float s = bf2f(sb);
  pair = static_cast<uint32_t>(sb) | ext << 16;
  if (s == 0.f) return;
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(s));
  r = fmaf(r, fmaf(-s, r, 1.f), r);
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer
  const float2 r2 = make_float2(r, r), m2 = make_float2(-lo, -lo), s2 = make_float2(-s, -s),
               up = make_float2(kRound, kRound);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v;
      unpack_bf2(w[4 * h + i], v.x, v.y);
      const float2 d = __fadd2_rn(v, m2), y0 = __fmul2_rn(d, r2);
      const float2 y = __ffma2_rn(__ffma2_rn(y0, s2, d), r2, y0);
      // the codes in the low 16 bits of two sums: (even channel, odd channel)
      const float2 z = __fadd2_rn(y, up);
      q[i] = __byte_perm(__float_as_uint(z.x), __float_as_uint(z.y), 0x5410);
    }
    word[h] = (q[3] * 16u + q[2]) * 256u + (q[1] * 16u + q[0]);
  }
  const float c = -lo * r;
  uint32_t todo = 0;  // channels to decide in 64 bits
  if (!plain || (lo != 0.f && fabsf(c) < 0x1p-11f)) {
    todo = 0xffffu;
  } else if (c < 16.f && fabsf(c - floorf(c) - 0.5f) < 0x1p-11f) {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const uint32_t two = w[k >> 1] & 0x7fff7fffu;
      const float x = __uint_as_float(k & 1 ? two & 0xffff0000u : two << 16) * r;
      if (x > 0.f && x < 0x1p-11f) todo |= 1u << k;
    }
  }
#pragma unroll 1
  while (todo) {
    const int k = __ffs(todo) - 1, i = k >> 1;  // channel k of the 16
    todo &= todo - 1;
    const uint32_t a0 = i & 1 ? w[1] : w[0], a1 = i & 1 ? w[3] : w[2], a2 = i & 1 ? w[5] : w[4],
                   a3 = i & 1 ? w[7] : w[6];
    const uint32_t b0 = i & 2 ? a1 : a0, b1 = i & 2 ? a3 : a2, two = i & 4 ? b1 : b0;
    const float x = __uint_as_float(k & 1 ? two & 0xffff0000u : two << 16);
    const uint32_t code = static_cast<uint32_t>(code_exact(x, lo, s));
    const int at = 4 * ((i & 3) + 4 * (k & 1));
    const uint32_t keep = ~(15u << at), put = code << at;
    if (k < 8) word[0] = (word[0] & keep) | put;
    else word[1] = (word[1] & keep) | put;
  }
}

// blockIdx.y picks K or V.
template <int D, int GROUP>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) kv_append_q4_kernel(
    const __grid_constant__ Append p, uint32_t rows, Divisor by_s, Divisor by_h, uint32_t cap,
    int64_t offset, const int32_t *__restrict__ offsets, int *err) {
  constexpr int W = D / 8, J = D / 32, GT = GROUP / 16, NS = D / GROUP;
  constexpr int T = D / 16;  // threads per row
  const int kv = blockIdx.y;
  const Rows rs = p.at[kv];
  const int ch = threadIdx.x & (T - 1);  // channels 16 ch ..
  // words 2 ch and 2 ch + 1 in channel order: (t, j) = (2 ch % 4, ch / 2) and the next t
  uint32_t *codes = p.codes[kv] + (2 * ch & 3) * J + (ch >> 1);
  uint32_t *scales = p.scales[kv] + ch / GT;
  constexpr uint32_t kStep = kAppendThreads / T;  // rows of a CTA's step
  const uint32_t stride = gridDim.x * kStep;
  uint32_t row = blockIdx.x * kStep + threadIdx.x / T, b, h, s;
  b = divide(divide(row, by_s, s), by_h, h);
  const uint16_t *src = p.src[kv] + 16 * ch + b * rs.sb + h * rs.sh + s * rs.ss;
  wait_for_earlier();
  let_next_launch();
  uint32_t w[8] = {};
  auto load = [&]() {  // the row's channels, ahead of their use
    const uint4 *at = reinterpret_cast<const uint4 *>(src);
    const uint4 x = at[0], y = at[1];
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
  };
  if (row < rows) load();
  // every thread of a warp takes the same number of steps: the shuffles need them all
  for (uint32_t base = blockIdx.x * kStep; base < rows; base += stride, row += stride) {
    uint32_t now[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) now[i] = w[i];
    const uint32_t bh0 = b * p.Hkv + h, b0 = b, s0 = s;
    if (row + stride < rows) {
      s += p.ds, h += p.dh, b += p.db, src += p.add[kv];
      if (s >= p.S) s -= p.S, ++h, src += p.carry_s[kv];
      if (h >= p.Hkv) h -= p.Hkv, ++b, src += p.carry_h[kv];
      load();
    }
    uint32_t word[2], pair;
    quantise16<GT>(now, word, pair);
    if (row >= rows) continue;
    const int64_t dst = (offsets ? static_cast<int64_t>(offsets[b0]) : offset) + s0;
    if (dst < 0 || dst >= cap) {
      report_error(err, DEV_ERR_INDEX, 105, static_cast<int>(b0), static_cast<int>(dst));
      continue;
    }
    const int64_t out = static_cast<uint64_t>(bh0) * cap + dst;
    codes[out * W] = word[0];
    codes[out * W + J] = word[1];
    if (ch % GT == 0) scales[out * NS] = pair;
  }
}

// Rows [start, start + n) as bf16 [B, Hkv, out_cap, D]; rows n .. out_cap are zeros.
// kWords code words per thread: 4 when that still gives every SM eight CTAs (16 x 8192
// rows: 58.7 us, 92 % of the copy rate; 63.7 with 2), else 2 (4096 rows: 3.4, not 3.7).
template <int D, int GROUP, int kWords>
__global__ void __launch_bounds__(kThreads) kv_read_q4_kernel(
    Cache c, uint16_t *__restrict__ k, uint16_t *__restrict__ v, uint32_t rows, Divisor by_out,
    Divisor by_h, uint32_t n, int64_t cap, int64_t start, const int32_t *__restrict__ starts,
    int *err) {
  constexpr int W = D / 8, J = D / 32, GT = GROUP / 8, NS = D / GROUP;
  constexpr int kRows = kThreads / W;
  const bool is_v = blockIdx.y != 0;
  const uint32_t *codes = is_v ? c.v_codes : c.k_codes, *scales = is_v ? c.v_scales : c.k_scales;
  const int ch = threadIdx.x & (W - 1);
  uint32_t word[kWords], pair[kWords], row[kWords];
  bool live[kWords];
  wait_for_earlier();
  let_next_launch();
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    row[i] = (blockIdx.x * kWords + i) * kRows + threadIdx.x / W;
    uint32_t r, h;
    const uint32_t bh = divide(row[i] < rows ? row[i] : 0u, by_out, r);
    live[i] = row[i] < rows && r < n;
    word[i] = pair[i] = 0u;  // a scale and a minimum of 0: the value 0
    if (live[i]) {
      const int64_t src =
          (starts ? static_cast<int64_t>(starts[divide(bh, by_h, h)]) : start) + r;
      if (src < 0 || src >= cap) {
        report_error(err, DEV_ERR_INDEX, 106, static_cast<int>(bh / by_h.d), static_cast<int>(src));
      } else {
        const int64_t at = bh * cap + src;
        word[i] = codes[at * W + (ch & 3) * J + (ch >> 2)];
        pair[i] = scales[at * NS + ch / GT];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if (row[i] >= rows) continue;
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = pack_bf2(q4::value(q4::code_of(word[i], 2 * e), pair[i]),
                      q4::value(q4::code_of(word[i], 2 * e + 1), pair[i]));
    *reinterpret_cast<uint4 *>((is_v ? v : k) + int64_t(row[i]) * D + 8 * ch) =
        make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <typename F>
cudaError_t by_shape(int D, int group, F &&f) {
  using std::integral_constant;
  auto go = [&](auto d, auto g) { return f(d, g); };
  if (D == 128 && group == 32) return go(integral_constant<int, 128>{}, integral_constant<int, 32>{});
  if (D == 128 && group == 64) return go(integral_constant<int, 128>{}, integral_constant<int, 64>{});
  if (D == 128) return go(integral_constant<int, 128>{}, integral_constant<int, 128>{});
  if (D == 64 && group == 32) return go(integral_constant<int, 64>{}, integral_constant<int, 32>{});
  if (D == 64) return go(integral_constant<int, 64>{}, integral_constant<int, 64>{});
  return go(integral_constant<int, 32>{}, integral_constant<int, 32>{});
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int q35_kv_append_q4(const void *k_new, const void *v_new, const int64_t *k_strides,
                                const int64_t *v_strides, void *k_codes, void *k_scales,
                                void *v_codes, void *v_scales, int64_t B, int Hkv, int64_t S, int D,
                                int group, int64_t cap, int64_t offset, const int32_t *offsets,
                                q35_stream_t stream) {
  const int st = q4::check_cache("kv_append_q4", k_codes, k_scales, v_codes, v_scales, B, Hkv, D,
                                 group, cap);
  if (st) return st;
  if (S < 0) return fail(Q35_ERR_SHAPE, "kv_append_q4: %lld rows", (long long)S);
  if (S > cap || (!offsets && (offset < 0 || offset > cap - S)))
    return fail(Q35_ERR_SHAPE, "kv_append_q4: offset %lld + %lld rows exceed capacity %lld",
                (long long)(offsets ? 0 : offset), (long long)S, (long long)cap);
  if (B == 0 || S == 0) return Q35_OK;
  if (!k_new || !v_new || !k_strides || !v_strides)
    return fail(Q35_ERR_INVALID, "kv_append_q4: null");
  if (!aligned16(k_new) || !aligned16(v_new))
    return fail(Q35_ERR_ALIGN, "kv_append_q4: k, v not 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
      return fail(Q35_ERR_ALIGN, "kv_append_q4: strides not multiples of 8 elements");
  int *err = device_error_word();
  if (!err) return fail(Q35_ERR_CUDA, "kv_append_q4: no device error word");
  const int64_t rows = B * Hkv * S, step = kAppendThreads / (D / 16);
  if (rows >= (int64_t(1) << 30))
    return fail(Q35_ERR_SHAPE, "kv_append_q4: too many rows");
  int64_t ctas = (rows + step - 1) / step;  // per K and V; at most the resident ones
  const int64_t most = (int64_t(num_sms()) * kAppendCtas + 1) / 2;
  if (ctas > most) ctas = most;
  const int64_t stride = ctas * step;
  const uint32_t bh = static_cast<uint32_t>(stride / S);
  Append p{};
  p.ds = static_cast<uint32_t>(stride % S), p.dh = bh % Hkv, p.db = bh / Hkv;
  p.S = static_cast<uint32_t>(S), p.Hkv = Hkv;
  for (int i = 0; i < 2; ++i) {
    p.src[i] = static_cast<const uint16_t *>(i ? v_new : k_new);
    p.codes[i] = static_cast<uint32_t *>(i ? v_codes : k_codes);
    p.scales[i] = static_cast<uint32_t *>(i ? v_scales : k_scales);
    const int64_t *by = i ? v_strides : k_strides;
    p.at[i] = Rows{by[0], by[1], by[2]};
    p.add[i] = p.db * by[0] + p.dh * by[1] + p.ds * by[2];
    p.carry_s[i] = by[1] - S * by[2];
    p.carry_h[i] = by[0] - Hkv * by[1];
  }
  Q35_CHECK_CUDA(by_shape(D, group, [&](auto d, auto g) {
    return launch_early(&kv_append_q4_kernel<d(), g()>, dim3(static_cast<unsigned>(ctas), 2),
                        dim3(kAppendThreads), 0, reinterpret_cast<cudaStream_t>(stream), p,
                        static_cast<uint32_t>(rows), divisor(static_cast<uint32_t>(S)), divisor(Hkv),
                        static_cast<uint32_t>(cap), offset, offsets, err);
  }));
  Q35_LAUNCH_CHECK("kv_append_q4 launch");
  return Q35_OK;
}

extern "C" int q35_kv_read_q4(const void *k_codes, const void *k_scales, const void *v_codes,
                              const void *v_scales, void *k_out, void *v_out, int64_t B, int Hkv,
                              int64_t n, int64_t out_cap, int D, int group, int64_t cap,
                              int64_t start, const int32_t *starts, q35_stream_t stream) {
  const int st = q4::check_cache("kv_read_q4", k_codes, k_scales, v_codes, v_scales, B, Hkv, D,
                                 group, cap);
  if (st) return st;
  if (n < 0 || out_cap < n || out_cap >= (int64_t(1) << 31))
    return fail(Q35_ERR_SHAPE, "kv_read_q4: %lld rows into %lld", (long long)n, (long long)out_cap);
  if (n > cap || (!starts && (start < 0 || start > cap - n)))
    return fail(Q35_ERR_SHAPE, "kv_read_q4: rows %lld + %lld exceed capacity %lld",
                (long long)(starts ? 0 : start), (long long)n, (long long)cap);
  if (B == 0 || out_cap == 0) return Q35_OK;
  if (!k_out || !v_out) return fail(Q35_ERR_INVALID, "kv_read_q4: null");
  if (!aligned16(k_out) || !aligned16(v_out))
    return fail(Q35_ERR_ALIGN, "kv_read_q4: outputs not 16-byte aligned");
  int *err = device_error_word();
  if (!err) return fail(Q35_ERR_CUDA, "kv_read_q4: no device error word");
  const int64_t rows = B * Hkv * out_cap, step = kThreads / (D / 8);
  if (rows >= (int64_t(1) << 31) - 4 * step)
    return fail(Q35_ERR_SHAPE, "kv_read_q4: too many rows");
  const Cache c{static_cast<uint32_t *>(const_cast<void *>(k_codes)),
                static_cast<uint32_t *>(const_cast<void *>(k_scales)),
                static_cast<uint32_t *>(const_cast<void *>(v_codes)),
                static_cast<uint32_t *>(const_cast<void *>(v_scales))};
  const int words = rows >= 4 * step * 4 * num_sms() ? 4 : 2;
  Q35_CHECK_CUDA(by_shape(D, group, [&](auto d, auto g) {
    auto *kern = words == 4 ? &kv_read_q4_kernel<d(), g(), 4> : &kv_read_q4_kernel<d(), g(), 2>;
    return launch_early(
        kern, dim3(static_cast<unsigned>((rows + words * step - 1) / (words * step)), 2),
        dim3(kThreads), 0, reinterpret_cast<cudaStream_t>(stream), c, static_cast<uint16_t *>(k_out),
        static_cast<uint16_t *>(v_out), static_cast<uint32_t>(rows),
        divisor(static_cast<uint32_t>(out_cap)), divisor(Hkv), static_cast<uint32_t>(n), cap, start,
        starts, err);
  }));
  Q35_LAUNCH_CHECK("kv_read_q4 launch");
  return Q35_OK;
}
