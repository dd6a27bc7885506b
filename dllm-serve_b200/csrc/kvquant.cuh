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
// finite (the codes saturate there).
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

// 2^(byte - 127), 0 for byte 0.
DLLM_DEVICE float exp_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Four codes (in memory order) of y = x * 2^-e.
template <int kFmt>
DLLM_DEVICE uint32_t encode4(float y0, float y1, float y2, float y3) {
  if constexpr (kFmt == kFmtE4m3) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y1), "f"(y0));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y3), "f"(y2));
    return (uint32_t)lo | ((uint32_t)hi << 16);
  } else {
    // NaN converts to 0, infinities saturate
    const int c0 = min(max(__float2int_rn(y0), -127), 127), c1 = min(max(__float2int_rn(y1), -127), 127);
    const int c2 = min(max(__float2int_rn(y2), -127), 127), c3 = min(max(__float2int_rn(y3), -127), 127);
    const uint32_t lo = __byte_perm((uint32_t)c0, (uint32_t)c1, 0x0040);
    const uint32_t hi = __byte_perm((uint32_t)c2, (uint32_t)c3, 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  }
}

// Four codes -> values times `scale`, float32 (exact: scale is a power of two).
template <int kFmt>
DLLM_DEVICE void decode4(uint32_t w, float scale, float (&y)[4]) {
  if constexpr (kFmt == kFmtE4m3) {
    uint32_t h0, h1;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h0) : "h"((uint16_t)(w & 0xffffu)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h1) : "h"((uint16_t)(w >> 16)));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
    y[0] = a.x * scale;
    y[1] = a.y * scale;
    y[2] = b.x * scale;
    y[3] = b.y * scale;
  } else {
    // byte + 128 into the low mantissa bits of 2^23, then subtract 2^23 + 128
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      y[i] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)) - 8388736.f) * scale;
  }
}

// Largest finite bf16 magnitude of eight words (pairs of bf16), and whether any
// value is not finite.
DLLM_DEVICE uint32_t finite_max16(const uint32_t (&w)[8], bool& bad) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  m = max(m & 0xffffu, m >> 16);
  bad = m >= 0x7f80u;
  if (bad) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
      if (lo < 0x7f80u) m = max(m, lo);
      if (hi < 0x7f80u) m = max(m, hi);
    }
  }
  return m;
}

// Quantises 16 bf16 values (eight words) with the group's exponent byte.
template <int kFmt>
DLLM_DEVICE uint4 quantise16(const uint32_t (&w)[8], uint32_t byte) {
  const float inv = __uint_as_float((254u - byte) << 23);  // 2^-e
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = w[2 * i], b = w[2 * i + 1];
    c[i] = encode4<kFmt>(__uint_as_float(a << 16) * inv, __uint_as_float(a & 0xffff0000u) * inv,
                         __uint_as_float(b << 16) * inv, __uint_as_float(b & 0xffff0000u) * inv);
  }
  return make_uint4(c[0], c[1], c[2], c[3]);
}

// 16 codes -> 16 bf16 values (eight words), exact.
template <int kFmt>
DLLM_DEVICE void dequantise16(uint4 c, float scale, uint32_t (&w)[8]) {
  const uint32_t cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float y[4];
    decode4<kFmt>(cs[i], scale, y);
    w[2 * i] = pack_bf16x2(y[0], y[1]);
    w[2 * i + 1] = pack_bf16x2(y[2], y[3]);
  }
}

}  // namespace dllm
