// The stored form of a 4-bit KV cache, shared by the kernels that write it,
// read it back and attend over it.
//
// A row of D channels (D = 32, 64 or 128) is D/8 32-bit words of eight 4-bit
// codes and D/group (scale, minimum) pairs of bf16, the scale in the low half
// of a 32-bit word.  Word t * (D/32) + j (t = 0..3) holds channels
// 32 j + 8 t + e, e = 0..7, channel e in field e/2 + 4 * (e & 1).
//
// Why this order: a matrix instruction wants its operands as pairs of
// neighbouring values along the summed axis.  With channel 2i in field i and
// channel 2i + 1 in field i + 4, `w & 0x000f000f` and `w & 0x00f000f0` (and the same
// of w >> 8) are such pairs, c * 2^-133 and c * 2^-129 as they stand: bf16's smallest
// numbers are evenly spaced.  The words of a thread quarter t are contiguous, so the
// four threads that share a key read 16 bytes each (D = 128).
#pragma once

#include "common.cuh"

namespace q35 {
namespace q4 {

// Device arrays of one layer's cache: codes [B, Hkv, cap, D/2] bytes, scales
// [B, Hkv, cap, D/group] (scale, minimum) words.
struct Cache {
  uint32_t *k_codes, *k_scales, *v_codes, *v_scales;
};

// Host-side checks that every entry point over a cache shares.
inline int check_cache(const char *what, const void *kc, const void *ks, const void *vc,
                       const void *vs, int64_t B, int Hkv, int D, int group, int64_t cap) {
  if (D != 32 && D != 64 && D != 128)
    return fail(Q35_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64 or 128)", what, D);
  if ((group != 32 && group != 64 && group != 128) || group > D)
    return fail(Q35_ERR_UNSUPPORTED, "%s: group %d (32, 64 or 128, at most head_dim %d)", what,
                group, D);
  if (B < 0 || Hkv <= 0 || cap < 0 || cap % 16 != 0)
    return fail(Q35_ERR_SHAPE, "%s: B %lld, Hkv %d, capacity %lld (a multiple of 16)", what,
                (long long)B, Hkv, (long long)cap);
  if (cap >= (int64_t(1) << 31) - 256)
    return fail(Q35_ERR_SHAPE, "%s: capacity %lld does not fit 31 bits", what, (long long)cap);
  if (B >= (int64_t(1) << 31) / Hkv)
    return fail(Q35_ERR_SHAPE, "%s: %lld sequences x %d heads", what, (long long)B, Hkv);
  if (B == 0 || cap == 0) return Q35_OK;
  if (!kc || !ks || !vc || !vs) return fail(Q35_ERR_INVALID, "%s: null cache pointer", what);
  if (!aligned16(kc) || !aligned16(ks) || !aligned16(vc) || !aligned16(vs))
    return fail(Q35_ERR_ALIGN, "%s: cache pointers not 16-byte aligned", what);
  return Q35_OK;
}

// The factor of the scores, for both forms of attention: beyond 2^100 (or NaN) one would
// give NaN and the other finite numbers.
inline int check_scale(const char *what, float scale) {
  if (scale >= -0x1p100f && scale <= 0x1p100f) return Q35_OK;
  return fail(Q35_ERR_INVALID, "%s: scale %g", what, static_cast<double>(scale));
}

// value = minimum + code * scale, rounded once to fp32 (code * scale is exact:
// 4 x 8 significant bits).
__device__ __forceinline__ float value(float code, uint32_t pair) {
  return fmaf(code, __uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
}
// Code of channel e of a word: the field under 2^23's exponent, less 2^23 (an
// integer conversion runs at an eighth of this rate).
__device__ __forceinline__ float code_of(uint32_t word, int e) {
  const int field = (e >> 1) + 4 * (e & 1);
  return __uint_as_float((word >> (4 * field) & 15u) | 0x4b000000u) - 8388608.f;
}

}  // namespace q4
}  // namespace q35
