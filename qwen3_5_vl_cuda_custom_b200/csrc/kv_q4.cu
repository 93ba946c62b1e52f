// Writing rows into a 4-bit KV cache and reading them back (layout: kv_q4.cuh).
//
// For a group of `group` channels with minimum m and maximum M:
//   s = bf16((M - m) / 15), c = min(15, rint((x - m) / s)), value = m + c s.
// m is a bf16 input and is stored exactly; s is rounded to nearest once and the
// codes are taken with the rounded s, so a value is off by s/2 plus at most
// 15 * 2^-9 s at the top of its group.  s = 0 (all equal, or (M - m) / 15 below
// the smallest bf16) stores codes of 0.  A group that holds a NaN or an infinity
// stores s = m = NaN and reads back as NaN.
//
// Both kernels move bytes: a thread owns the eight channels of one 32-bit code
// word (16 bytes of bf16), group statistics go over the group/8 neighbouring
// threads by shuffles, K and V share one launch.
#include <type_traits>

#include "kv_q4.cuh"

namespace q35 {
namespace {

using q4::Cache;

constexpr int kThreads = 256;

struct Rows {
  int64_t sb, sh, ss;  // element strides of batch, head, position
};

__device__ __forceinline__ uint32_t bf2_min(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmin2(*reinterpret_cast<__nv_bfloat162 *>(&a),
                             *reinterpret_cast<__nv_bfloat162 *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t bf2_max(uint32_t a, uint32_t b) {
  __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162 *>(&a),
                             *reinterpret_cast<__nv_bfloat162 *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}

// bf16((M - m) / 15) in one rounding, from 64 bits: a quotient that fp32 rounds
// onto a border between two bf16 numbers is put back on its own side.
__device__ __noinline__ uint16_t scale_exact(float lo, float hi) {
  const double s = (static_cast<double>(hi) - static_cast<double>(lo)) / 15.0;
  float f = static_cast<float>(s);
  uint32_t u = __float_as_uint(f);
  if ((u & 0xffffu) == 0x8000u) {
    if (static_cast<double>(f) < s) u += 1;
    else if (static_cast<double>(f) > s) u -= 1;
  }
  return f2bf(__uint_as_float(u));
}
__device__ __noinline__ uint32_t code_exact(float x, float lo, float s) {
  const double y = (static_cast<double>(x) - static_cast<double>(lo)) / static_cast<double>(s);
  return static_cast<uint32_t>(fmin(rint(y), 15.0));
}

// Eight channels x (bf16 pairs) of a group -> their code word; `pair` receives
// the group's (scale, minimum).  The threads of a group are neighbours.
//
// The fp32 quotient (x - m) * (1/s) is off by less than 3 * 2^-24 * 15 = 2.7e-6,
// so a code can only differ from the 64-bit rule when the quotient lies within
// 1e-5 of a half; those (about one in 10^5) are decided in 64 bits, as are
// scales within 4 fp32 steps of a bf16 border and groups outside the range in
// which 1/s and M - m are finite.
template <int GT>  // threads per group: 4, 8 or 16
__device__ __forceinline__ uint32_t quantise8(uint4 x, uint32_t &pair) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t mn = bf2_min(bf2_min(w[0], w[1]), bf2_min(w[2], w[3]));
  uint32_t mx = bf2_max(bf2_max(w[0], w[1]), bf2_max(w[2], w[3]));
  uint32_t bad = 0;  // an exponent of all ones carries into bit 15 / 31
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f807f80u) + 0x00800080u;
  bad &= 0x80008000u;
#pragma unroll
  for (int o = 1; o < GT; o <<= 1) {
    mn = bf2_min(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = bf2_max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    bad |= __shfl_xor_sync(0xffffffffu, bad, o);
  }
  float a, b, lo, hi;
  unpack_bf2(mn, a, b);
  lo = fminf(a, b);
  unpack_bf2(mx, a, b);
  hi = fmaxf(a, b);
  if (bad) {
    pair = 0x7fc07fc0u;
    return 0u;
  }
  const float d = hi - lo;
  const float s32 = d * (1.0f / 15.0f);
  const uint32_t su = __float_as_uint(s32);
  // 2^-100 <= s32 <= 2^120: 1/s and x - m stay normal numbers
  const bool plain = s32 >= 7.8886091e-31f && s32 <= 1.3292280e36f;
  const uint32_t low = (su & 0xffffu) - (0x8000u - 4u);
  const uint16_t sb = (d == 0.f) ? uint16_t(0)
                      : (plain && low > 8u) ? f2bf(s32)
                                            : scale_exact(lo, hi);
  const float s = bf2f(sb);
  pair = static_cast<uint32_t>(sb) | (__float_as_uint(lo) & 0xffff0000u);
  if (s == 0.f) return 0u;
  const float r = 1.0f / s;
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer
  uint32_t word = 0;
  bool border = !plain;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float v[2];
    unpack_bf2(w[i], v[0], v[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float y = (v[h] - lo) * r;
      const float t = y + kRound;
      border |= fabsf(y - (t - kRound)) > 0.49999f;
      const uint32_t c = min(__float_as_uint(t) - __float_as_uint(kRound), 15u);
      word |= c << (4 * (i + 4 * h));
    }
  }
  if (border) {
    word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v0, v1;
      unpack_bf2(w[i], v0, v1);
      word |= code_exact(v0, lo, s) << (4 * i);
      word |= code_exact(v1, lo, s) << (4 * (i + 4));
    }
  }
  return word;
}

// One thread per code word; blockIdx.y picks K or V.
template <int D, int GROUP>
__global__ void __launch_bounds__(kThreads) kv_append_q4_kernel(
    const uint16_t *__restrict__ k, const uint16_t *__restrict__ v, Rows rk, Rows rv, Cache c,
    int64_t words, int Hkv, int64_t S, int64_t cap, int64_t offset,
    const int32_t *__restrict__ offsets, int *err) {
  constexpr int W = D / 8, J = D / 32, GT = GROUP / 8, NS = D / GROUP;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const bool is_v = blockIdx.y != 0;
  const uint16_t *src = is_v ? v : k;
  const Rows rs = is_v ? rv : rk;
  const bool live = i < words;
  const int64_t row = live ? i / W : 0;
  const int ch = static_cast<int>(i & (W - 1));  // channels 8 ch ..
  const int64_t bh = row / S, s = row - bh * S;
  const int64_t b = bh / Hkv, h = bh - b * Hkv;
  uint4 x = make_uint4(0u, 0u, 0u, 0u);
  if (live)
    x = *reinterpret_cast<const uint4 *>(src + b * rs.sb + h * rs.sh + s * rs.ss + 8 * ch);
  uint32_t pair;
  const uint32_t word = quantise8<GT>(x, pair);
  if (!live) return;
  const int64_t dst = (offsets ? static_cast<int64_t>(offsets[b]) : offset) + s;
  if (dst < 0 || dst >= cap) {
    report_error(err, DEV_ERR_INDEX, 105, static_cast<int>(b), static_cast<int>(dst));
    return;
  }
  const int64_t out = bh * cap + dst;
  (is_v ? c.v_codes : c.k_codes)[out * W + (ch & 3) * J + (ch >> 2)] = word;
  if (ch % GT == 0) (is_v ? c.v_scales : c.k_scales)[out * NS + ch / GT] = pair;
}

// Rows [start, start + n) as bf16 [B, Hkv, out_cap, D]; rows n .. out_cap are
// zeros.  One thread per code word.
template <int D, int GROUP>
__global__ void __launch_bounds__(kThreads) kv_read_q4_kernel(
    Cache c, uint16_t *__restrict__ k, uint16_t *__restrict__ v, int64_t words, int Hkv, int64_t n,
    int64_t out_cap, int64_t cap, int64_t start, const int32_t *__restrict__ starts, int *err) {
  constexpr int W = D / 8, J = D / 32, GT = GROUP / 8, NS = D / GROUP;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= words) return;
  const bool is_v = blockIdx.y != 0;
  const int64_t row = i / W;
  const int ch = static_cast<int>(i & (W - 1));
  const int64_t bh = row / out_cap, r = row - bh * out_cap;
  uint4 x = make_uint4(0u, 0u, 0u, 0u);
  if (r < n) {
    const int64_t b = bh / Hkv;
    const int64_t src = (starts ? static_cast<int64_t>(starts[b]) : start) + r;
    if (src < 0 || src >= cap) {
      report_error(err, DEV_ERR_INDEX, 106, static_cast<int>(b), static_cast<int>(src));
    } else {
      const int64_t at = bh * cap + src;
      const uint32_t word = (is_v ? c.v_codes : c.k_codes)[at * W + (ch & 3) * J + (ch >> 2)];
      const uint32_t pair = (is_v ? c.v_scales : c.k_scales)[at * NS + ch / GT];
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = pack_bf2(q4::value(q4::code_of(word, 2 * e), pair),
                        q4::value(q4::code_of(word, 2 * e + 1), pair));
      x = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
  *reinterpret_cast<uint4 *>((is_v ? v : k) + row * D + 8 * ch) = x;
}

template <typename F>
int by_shape(int D, int group, F &&f) {
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
  if (offsets ? S > cap : (offset < 0 || offset + S > cap))
    return fail(Q35_ERR_SHAPE, "kv_append_q4: offset %lld + %lld rows exceed capacity %lld",
                (long long)(offsets ? 0 : offset), (long long)S, (long long)cap);
  if (B * S == 0) return Q35_OK;
  if (!k_new || !v_new || !k_strides || !v_strides)
    return fail(Q35_ERR_INVALID, "kv_append_q4: null");
  if (!aligned16(k_new) || !aligned16(v_new))
    return fail(Q35_ERR_ALIGN, "kv_append_q4: k, v not 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
      return fail(Q35_ERR_ALIGN, "kv_append_q4: strides not multiples of 8 elements");
  int *err = device_error_word();
  if (!err) return fail(Q35_ERR_CUDA, "kv_append_q4: no device error word");
  const int64_t words = B * Hkv * S * (D / 8);
  const int64_t blocks = (words + kThreads - 1) / kThreads;
  if (blocks >= (int64_t(1) << 31)) return fail(Q35_ERR_SHAPE, "kv_append_q4: too many rows");
  const Cache c{static_cast<uint32_t *>(k_codes), static_cast<uint32_t *>(k_scales),
                static_cast<uint32_t *>(v_codes), static_cast<uint32_t *>(v_scales)};
  const Rows rk{k_strides[0], k_strides[1], k_strides[2]};
  const Rows rv{v_strides[0], v_strides[1], v_strides[2]};
  by_shape(D, group, [&](auto d, auto g) {
    kv_append_q4_kernel<d(), g()><<<dim3(static_cast<unsigned>(blocks), 2), kThreads, 0,
                                    reinterpret_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint16_t *>(k_new), static_cast<const uint16_t *>(v_new), rk, rv, c,
        words, Hkv, S, cap, offset, offsets, err);
    return 0;
  });
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
  if (n < 0 || out_cap < n)
    return fail(Q35_ERR_SHAPE, "kv_read_q4: %lld rows into %lld", (long long)n, (long long)out_cap);
  if (starts ? n > cap : (start < 0 || start + n > cap))
    return fail(Q35_ERR_SHAPE, "kv_read_q4: rows %lld + %lld exceed capacity %lld",
                (long long)(starts ? 0 : start), (long long)n, (long long)cap);
  if (B * out_cap == 0) return Q35_OK;
  if (!k_out || !v_out) return fail(Q35_ERR_INVALID, "kv_read_q4: null");
  if (!aligned16(k_out) || !aligned16(v_out))
    return fail(Q35_ERR_ALIGN, "kv_read_q4: outputs not 16-byte aligned");
  int *err = device_error_word();
  if (!err) return fail(Q35_ERR_CUDA, "kv_read_q4: no device error word");
  const int64_t words = B * Hkv * out_cap * (D / 8);
  const int64_t blocks = (words + kThreads - 1) / kThreads;
  if (blocks >= (int64_t(1) << 31)) return fail(Q35_ERR_SHAPE, "kv_read_q4: too many rows");
  const Cache c{static_cast<uint32_t *>(const_cast<void *>(k_codes)),
                static_cast<uint32_t *>(const_cast<void *>(k_scales)),
                static_cast<uint32_t *>(const_cast<void *>(v_codes)),
                static_cast<uint32_t *>(const_cast<void *>(v_scales))};
  by_shape(D, group, [&](auto d, auto g) {
    kv_read_q4_kernel<d(), g()><<<dim3(static_cast<unsigned>(blocks), 2), kThreads, 0,
                                  reinterpret_cast<cudaStream_t>(stream)>>>(
        c, static_cast<uint16_t *>(k_out), static_cast<uint16_t *>(v_out), words, Hkv, n, out_cap,
        cap, start, starts, err);
    return 0;
  });
  Q35_LAUNCH_CHECK("kv_read_q4 launch");
  return Q35_OK;
}
