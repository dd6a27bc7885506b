// Quantised cache rows, shared by the kernels that write and read them.
//
// A group is one (token, kv head) row of head_dim values. With a = the largest
// finite magnitude of the group and M the largest value of the format (448 for
// e4m3, 127 for int8), e is the smallest integer with a <= M * 2^e, and the
// codes are x * 2^-e rounded to nearest even. The scale is a power of two, so
// x * 2^-e and code * 2^e are exact and the one rounding is the code's own:
// at most half a step of the format. The group keeps the byte e + 127, i.e.
// the exponent field of 2^e as a float; byte 0 (a slot never written) reads as
// scale zero. e is clamped to [-100, e_max]: the lower end keeps every
// nonzero dequantised value a normal bf16 number, the upper end keeps it
// finite (the codes saturate there). Byte 255 marks a group with a NaN: all of
// it reads as NaN.
#pragma once

#include "common.cuh"

namespace dllm {

constexpr int kFmtBf16 = 0;
constexpr int kFmtE4m3 = 1;
constexpr int kFmtInt8 = 2;

template <int kFmt>
struct KvFormat;
template <>
struct KvFormat<kFmtE4m3> {
  // 448 = 1.75 * 2^8: mantissa bits of a bf16 number up to 1.75, and its exponent
  static constexpr uint32_t kTopMant = 0x60;
  static constexpr int kTopExp = 8;
  static constexpr int kMaxByte = 119 + 127;
};
template <>
struct KvFormat<kFmtInt8> {
  // 127 = 1.984375 * 2^6
  static constexpr uint32_t kTopMant = 0x7e;
  static constexpr int kTopExp = 6;
  static constexpr int kMaxByte = 121 + 127;
};
constexpr int kMinExpByte = -100 + 127;

// Exponent byte of a group whose largest finite magnitude has the bf16 bits
// `amax` (sign clear): exponent field - kTopExp, one more if the mantissa is
// above the format's largest.
template <int kFmt>
DLLM_DEVICE uint32_t exp_byte(uint32_t amax) {
  const int b = (int)(amax >> 7) - KvFormat<kFmt>::kTopExp + ((amax & 0x7f) > KvFormat<kFmt>::kTopMant ? 1 : 0);
  return (uint32_t)min(max(b, kMinExpByte), KvFormat<kFmt>::kMaxByte);
}

constexpr uint32_t kNanByte = 255;

// 2^(byte - 127), 0 for byte 0, NaN for kNanByte.
DLLM_DEVICE float exp_scale(uint32_t byte) {
  return byte == kNanByte ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

// Four codes (in memory order) of y = x * 2^-e.
template <int kFmt>
DLLM_DEVICE uint32_t encode4(float y0, float y1, float y2, float y3) {
  if constexpr (kFmt == kFmtE4m3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y1), "f"(y0));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y3), "f"(y2));
    return (uint32_t)lo | ((uint32_t)hi << 16);
  } else {
    // infinities saturate
    const int c0 = min(max(__float2int_rn(y0), -127), 127), c1 = min(max(__float2int_rn(y1), -127), 127);
    const int c2 = min(max(__float2int_rn(y2), -127), 127), c3 = min(max(__float2int_rn(y3), -127), 127);
    const uint32_t lo = __byte_perm((uint32_t)c0, (uint32_t)c1, 0x0040);
    const uint32_t hi = __byte_perm((uint32_t)c2, (uint32_t)c3, 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
}

// Largest finite bf16 magnitude of kWords words (pairs of bf16). bad: 1 if any
// value is infinite, 2 if any is NaN.
template <int kWords>
DLLM_DEVICE uint32_t finite_max(const uint32_t (&w)[kWords], uint32_t& bad) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kWords; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  m = max(m & 0xffffu, m >> 16);
  bad = m > 0x7f80u ? 2 : m == 0x7f80u ? 1 : 0;
  if (bad) {
    m = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
      if (lo < 0x7f80u) m = max(m, lo);
      if (hi < 0x7f80u) m = max(m, hi);
    }
  }
  return m;
}

// Quantises kWords words of bf16 pairs with the group's exponent byte.
template <int kFmt, int kWords>
DLLM_DEVICE void quantise(const uint32_t (&w)[kWords], uint32_t byte, uint32_t (&c)[kWords / 2]) {
  if (byte == kNanByte) {
#pragma unroll
    for (int i = 0; i < kWords / 2; ++i) c[i] = 0;
    return;
  }
  const float inv = __uint_as_float((254u - byte) << 23);  // 2^-e
#pragma unroll
  for (int i = 0; i < kWords / 2; ++i) {
    const uint32_t a = w[2 * i], b = w[2 * i + 1];
    c[i] = encode4<kFmt>(__uint_as_float(a << 16) * inv, __uint_as_float(a & 0xffff0000u) * inv,
                         __uint_as_float(b << 16) * inv, __uint_as_float(b & 0xffff0000u) * inv);
  }
}

// Exponent bytes of a K and a V group spread over kLanes lanes (kWords words
// each; every lane of `mask` takes part). Infinities and NaN set *err.
template <int kFmt, int kLanes, int kWords>
DLLM_DEVICE void group_bytes(const uint32_t (&k)[kWords], const uint32_t (&v)[kWords], uint32_t mask, int32_t* err,
                             uint32_t& ek, uint32_t& ev) {
  uint32_t bad_k, bad_v;
  const uint32_t mk = finite_max(k, bad_k), mv = finite_max(v, bad_v);
  uint32_t both = mk | (mv << 16);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) both = __vmaxu2(both, __shfl_xor_sync(mask, both, o));
  ek = exp_byte<kFmt>(both & 0xffffu);
  ev = exp_byte<kFmt>(both >> 16);
  if (__any_sync(mask, (bad_k | bad_v) != 0)) {
    uint32_t nan = (bad_k >> 1) | (bad_v & 2);  // bit 0: a NaN in the K row, bit 1: in the V row
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) nan |= __shfl_xor_sync(mask, nan, o);
    if (nan & 1) ek = kNanByte;
    if (nan & 2) ev = kNanByte;
    if (bad_k | bad_v) set_error(err, kDevNonFinite);
  }
}

// Expansion of codes to bf16, exact. No conversion instruction: e4m3
// conversions run at 16 per cycle and SM, the exponentials' rate, which the
// attention kernels need for those.
//
// e4m3: the code s eeee mmm, put into a bf16 as s 0000eeee mmm0000, is the
// value times 2^-120 (subnormal codes included, as subnormal bf16); one
// product by 2^(120 + e) follows, or two where that is no bf16 (e > 7).
// int8: the code + 128 in the low mantissa bits of 2^23 is 2^23 + 128 + code;
// one fma by 2^e takes the bias off, or a subtraction and a product where
// 2^(23 + e) is no float (e > 100).
// Groups that need the second form are rare: `exp_is_big`.
template <int kFmt>
DLLM_DEVICE bool exp_is_big(uint32_t byte) {
  return kFmt == kFmtE4m3 ? byte > 7 + 127 : byte > 100 + 127;  // (a NaN's byte too)
}

// What a group's codes are multiplied by (not for big exponents).
template <int kFmt>
DLLM_DEVICE float2 code_scale(uint32_t byte) {
  if constexpr (kFmt == kFmtE4m3) {
    const uint32_t s = byte == 0 ? 0u : (byte + 120) << 7;
    return make_float2(__uint_as_float(s | (s << 16)), 0.f);  // a bf16 pair
  } else {
    const float s = exp_scale(byte);
    return make_float2(s, -8388736.f * s);
  }
}

// e4m3 codes of a word as four bf16, times 2^-120.
DLLM_DEVICE void e4m3_bits(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t h = ((w >> 4) & 0x07070707u) | (w & 0x80808080u);  // upper bytes
  const uint32_t l = (w & 0x0f0f0f0fu) * 16u;                       // lower bytes (the FMA pipe: the others are busier)
  lo = __byte_perm(l, h, 0x5140);
  hi = __byte_perm(l, h, 0x7362);
}

DLLM_DEVICE uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 z = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&z);
}

// 16 codes -> 16 bf16 values (eight words), with code_scale() of the group.
template <int kFmt>
DLLM_DEVICE void expand16(uint4 c, float2 scale, uint32_t (&w)[8]) {
  const uint32_t cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kFmt == kFmtE4m3) {
      uint32_t lo, hi;
      e4m3_bits(cs[i], lo, hi);
      w[2 * i] = mul_bf16x2(lo, __float_as_uint(scale.x));
      w[2 * i + 1] = mul_bf16x2(hi, __float_as_uint(scale.x));
    } else {
      const uint32_t u = cs[i] ^ 0x80808080u;
      float y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = fmaf(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + k)), scale.x, scale.y);
      w[2 * i] = pack_bf16x2(y[0], y[1]);
      w[2 * i + 1] = pack_bf16x2(y[2], y[3]);
    }
  }
}

// The same for any exponent byte.
template <int kFmt>
DLLM_DEVICE void dequantise16(uint4 c, uint32_t byte, uint32_t (&w)[8]) {
  if (!exp_is_big<kFmt>(byte)) {
    expand16<kFmt>(c, code_scale<kFmt>(byte), w);
    return;
  }
  const uint32_t cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kFmt == kFmtE4m3) {
      const uint32_t s = byte == kNanByte ? 0x7fc0u : (byte + 6) << 7;  // 2^114, then 2^(e + 6)
      uint32_t lo, hi;
      e4m3_bits(cs[i], lo, hi);
      w[2 * i] = mul_bf16x2(mul_bf16x2(lo, 0x78807880u), s | (s << 16));
      w[2 * i + 1] = mul_bf16x2(mul_bf16x2(hi, 0x78807880u), s | (s << 16));
    } else {
      const float s = exp_scale(byte);
      const uint32_t u = cs[i] ^ 0x80808080u;
      float y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + k)) - 8388736.f) * s;
      w[2 * i] = pack_bf16x2(y[0], y[1]);
      w[2 * i + 1] = pack_bf16x2(y[2], y[3]);
    }
  }
}

}  // namespace dllm
