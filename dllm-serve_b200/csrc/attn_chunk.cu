// Attention of a chunk of new tokens over a paged KV cache, for launches bound
// by the cache's bytes: few query rows per KV head, long contexts (sm_100a).
//
// The keys of sequence b are [its cached rows, found by block table or slot
// list ; its fresh rows]. Query row i of the chunk sees the first
// L - Lq + i + 1 of the L keys (causal) or all of them. Softmax is online: a
// running maximum m and sum l per row, O rescaled when m grows.
//
// With a quantised cache the matrix products run on the codes themselves: the
// scores are multiplied by the key's 2^e after their product, the
// probabilities by the value's 2^e before theirs. Codes expand to f16 in one
// conversion per pair (to bf16 it takes four), so both products use f16
// operands, and powers of two keep that as exact as bf16:
//   Q: each row is scaled so that its largest element lies in [2^14, 2^15).
//      bf16 values fit f16's 11 bits; elements below 2^-31 of the row's largest
//      lose some, an error of at most 2^-39 of that largest.
//   P: p * 2^(e_v - E + 15), E the largest value exponent this warp has met
//      (O is in units of 2^(E - 15) and is rescaled when E grows). p <= 1, so
//      nothing overflows; down to 2^-14 these keep 11 bits, and below that the
//      rounding is at most 2^-25, i.e. 2^-39 of the largest |v| met once
//      multiplied by the code and the unit. bf16 probabilities (2^-8 of p)
//      would be further off wherever p |v| is above 2^-31 of the largest |v|.
//
// A CTA takes one tile of packed rows (row r of the chunk for query head g of
// the KV head's group is packed row r * group + g) and one split of the keys;
// its four warps take the split's key chunks in turn, each with a private
// ring of stages filled by cp.async, so the main loop has no CTA barrier. The
// warps' partial results are merged in shared memory in a fixed order; splits
// are merged by their cluster, or by a second kernel, also in a fixed order.
// Products are
// mma.sync m16n8k16: at up to 16 rows per KV head (32 with a quantised cache) a
// launch reads 512 (256) bytes per key for at most 16 x 512 (32 x 512)
// operations, below what this instruction sustains, and its operands go
// straight from shared memory to registers, where codes are expanded; the
// tcgen05 kernel writes them to shared memory first.
//
// Measured, decode (one row, 32 heads): 8 contexts of 4,096-32,768 rows bf16 350
// us, 6.6 TB/s, e4m3 202 us, 5.8 TB/s (of 16,384 rows each 170 us, 6.4 TB/s):
// the cache's bytes, where lengths are even. 32 contexts of 128-1,024 bf16 rows,
// 28/4 heads: 14.7 us, 2.6 TB/s: a launch, one split's chunks and the merge one
// after another. 8 x 32 rows over 1,144 e4m3 rows: 42.5 us: with eight warps an SM
// the latencies of conversions and products, one launch not filling the last
// seventh of the SMs' places.
//
// Operand layout: keys (scores) and dimensions (outputs) take the products' 16
// rows and the packed query rows their 8 columns, so eight rows leave nothing
// idle and need half the accumulators of the other way round. The reduction
// order over head dimensions and over keys is free as long as both operands
// agree, and so is the order of the outputs' dimensions. Thread (g, t) of a
// warp (g = lane / 4, t = lane % 4) takes dimensions 16t .. 16t+15 and
// 64+16t .. 64+16t+15 of keys g and g + 8 for the scores (two 16-byte reads of
// codes a key), and dimensions 16g .. 16g+15 of keys 2t, 2t+1, 2t+8, 2t+9 for
// the outputs: rows g and g + 8 of output tile j are dimensions 16g + 2j and
// 16g + 2j + 1. Probabilities get from the scores' layout to the second
// operand's by an 8x8 transpose across the warp.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "common.cuh"
#include "kvquant.cuh"
#include "attn_chunk.cuh"

namespace dllm {
namespace chunk {

namespace {

constexpr int kD = 128;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr uint32_t kStageBytes = 8192;  // K half then V half
constexpr int kFreshKeys = 16;          // keys of a bf16 chunk
constexpr uint32_t kScaleBytes = 34 * 8;  // of a stage: 32 (K, V) scales, the largest exponent
constexpr int kNoExp = -(1 << 30);        // no value exponent met
constexpr int kClusterSplits = 8;         // splits that merge within a cluster
// A scaled Q (below 2^15) times codes (at most 448) over 128 dimensions is below 2^31; with keys'
// 2^e (e <= 121) lowered by 2^-kKeyDown the products stay finite, whatever the cache holds. The row's
// factor makes up for it (fit_row_factors() where that is no float).
constexpr int kKeyDown = 24;

template <int kFmt>
constexpr int chunk_keys() { return kFmt == kFmtBf16 ? 16 : 32; }

// A quantised chunk is bound by the latency of its conversions and products
// (issue slots 36 % used with eight warps an SM), a bf16 chunk by bytes in
// flight. Eight e4m3 contexts of 16,384 rows, 32 heads: two CTAs of three
// stages 195 us, three CTAs of two 184 us; bf16 contexts of 4,096 rows, 28/4
// heads: 54 and 66 us. Four 8-row groups take the registers of two CTAs.
template <int kFmt, int kN>
struct Cfg {
  static constexpr int kCtas = kFmt == kFmtBf16 || kN > 2 ? 2 : 3;  // per SM
  static constexpr int kStages = kCtas == 2 ? 3 : 2;
  static constexpr uint32_t kOffStages = 0;
  static constexpr uint32_t kOffScales = kOffStages + kWarps * kStages * kStageBytes;
  static constexpr uint32_t kOffRowFactor = kOffScales + kWarps * kStages * kScaleBytes;  // float per packed row
  static constexpr uint32_t kOffBlind = kOffRowFactor + kN * 8 * 4;  // how many rows of the chunk see no key
  static constexpr uint32_t kOffDown = kOffBlind + 4;                 // float: what the keys' 2^e are lowered by
  static constexpr uint32_t kOffQ = kOffBlind + 16;
  static constexpr uint32_t kSmemBytes = kOffQ + kN * 8 * kD * 2;
  static_assert(kCtas * (kSmemBytes + 1024) <= 233472, "the CTAs do not fit an SM");
  // the merge buffers (per warp: rows x 128 floats, then rows float2) reuse the stages
  // (and one more float2 per row)
  static_assert(kN * 8 * (kWarps * (kD * 4 + 8) + 8) <= kWarps * kStages * kStageBytes, "merge buffers exceed the stages");
};

DLLM_DEVICE void cp_async16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;  // 0: the 16 bytes are filled with zeros, nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
DLLM_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
DLLM_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory"); }

DLLM_DEVICE uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}

DLLM_DEVICE void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

DLLM_DEVICE void mma16816_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Every thread of the cluster's CTAs that have not ended.
DLLM_DEVICE void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared memory of the cluster's CTA `rank`, at this CTA's address `a`.
DLLM_DEVICE uint32_t cluster_addr(uint32_t a, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
DLLM_DEVICE float2 cluster_ld2(uint32_t a, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_addr(a, rank)));
  return v;
}
DLLM_DEVICE float4 cluster_ld4(uint32_t a, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr(a, rank)));
  return v;
}

// 2^e, 0 below the normal range.
DLLM_DEVICE float pow2(int e) { return __int_as_float(max(e + 127, 0) << 23); }

// Four codes -> two words of f16 pairs, unscaled (exact).
template <int kFmt>
DLLM_DEVICE void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kFmt == kFmtE4m3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // byte + 128 into the low mantissa bits of 1024, then subtract 1024 + 128
    const uint32_t u = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
    __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), bias), q = __hsub2(*reinterpret_cast<__half2*>(&y), bias);
    lo = *reinterpret_cast<uint32_t*>(&p);
    hi = *reinterpret_cast<uint32_t*>(&q);
  }
}
DLLM_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// f16 pair times `f`, as a bf16 pair.
DLLM_DEVICE uint32_t f16_to_bf16(uint32_t w, float f) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pack_bf16x2(x.x * f, x.y * f);
}

// Shared-memory swizzles (16-byte units of a row) that make the reads of the
// header comment free of bank conflicts: eight lanes read two K rows x four
// units, or four V rows x two units.
template <int kFmt>
DLLM_DEVICE uint32_t k_unit(uint32_t unit, uint32_t key) {
  return kFmt == kFmtBf16 ? unit ^ (key & 1) : unit ^ ((key & 1) << 2);
}
template <int kFmt>
DLLM_DEVICE uint32_t v_unit(uint32_t unit, uint32_t key) {
  return kFmt == kFmtBf16 ? unit ^ (((key >> 1) & 1) | (key & 4)) : unit ^ (key & 6);
}

}  // namespace

// Running state of a warp: thread (g, t) holds packed rows 8n + 2t and 8n + 2t + 1,
// n < kN (all eight lanes of equal t hold the same m).
template <int kN>
struct Rows {
  float m[kN][2];        // running maximum, log2 units
  float l[kN][2];        // sum over this thread's keys
  float rf[kN][2];       // score of a product: times this (log2 units)
  int seen[kN][2];       // keys the row sees, from the sequence's first
  float o[8][kN][4];     // dimensions 16g + 2j, 16g + 2j + 1 of both rows
  int e;                 // O is in units of 2^(e - 15) (quantised caches)
};

// Q stays in registers for up to 16 rows, else it is read from shared memory chunk by chunk.
template <int kN>
constexpr bool kQInRegs = kN <= 2;

// The 8x8 matrix of 16-bit values whose row g the lanes 4g .. 4g+3 hold, transposed.
DLLM_DEVICE uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Products, softmax and products of one chunk of KB keys in shared memory. A
// row sees the chunk's first min(seen, end) - pos keys; `whole`: all of them,
// for every row. kQuant: the kernel's cache is quantised (Q is f16 with a
// factor `back` for row 8n + g, O scaled), kFmt: the format of this chunk (its
// fresh chunks are bf16).
template <bool kQuant, int kFmt, int kN>
DLLM_DEVICE void chunk_step(uint32_t ks, uint32_t vs, uint32_t scales, uint32_t qs, const uint32_t (&qf)[kN][16],
                            const float (&back)[kN], int lane, float sl2, bool whole, int pos, int end, Rows<kN>& w) {
  constexpr int KB = chunk_keys<kFmt>();
  constexpr int KT = KB / 16;  // 16-key tiles
  constexpr bool kCodes = kFmt != kFmtBf16;
  constexpr uint32_t kRow = kCodes ? 128 : 256;  // bytes of a key's row
  const int g = lane >> 2, t = lane & 3;
  float s[KT][kN][4];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[kt][n][e] = 0.f;
  // scores: half h covers dimensions 64h + 16t .. + 15 of this thread
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t ka[KT][2][8];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t key = 16 * kt + 8 * e + g;
        uint32_t(&k)[8] = ka[kt][e];
        if constexpr (!kCodes) {
          const uint4 x = lds128(ks + key * kRow + (k_unit<kFmt>(8 * h + 2 * t, key) << 4));
          const uint4 y = lds128(ks + key * kRow + (k_unit<kFmt>(8 * h + 2 * t + 1, key) << 4));
          k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w;
          k[4] = y.x, k[5] = y.y, k[6] = y.z, k[7] = y.w;
        } else {
          const uint4 x = lds128(ks + key * kRow + (k_unit<kFmt>(4 * h + t, key) << 4));
          codes_to_f16<kFmt>(x.x, k[0], k[1]);
          codes_to_f16<kFmt>(x.y, k[2], k[3]);
          codes_to_f16<kFmt>(x.z, k[4], k[5]);
          codes_to_f16<kFmt>(x.w, k[6], k[7]);
        }
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t q[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if constexpr (kQInRegs<kN>) {
#pragma unroll
          for (int i = 0; i < 4; ++i) q[n][i] = qf[n][8 * h + 4 * c + i];
        } else {
          const int row = 8 * n + g;
          const uint4 x = lds128(qs + row * 256 + (((8 * h + 2 * t + c) ^ (row & 1)) << 4));
          q[n][0] = x.x, q[n][1] = x.y, q[n][2] = x.z, q[n][3] = x.w;
        }
        if constexpr (kQuant && !kCodes) {
#pragma unroll
          for (int i = 0; i < 4; ++i) q[n][i] = f16_to_bf16(q[n][i], back[n]);
        }
      }
      // (a product waits for the one before it into the same scores: kN * KT products apart)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const uint32_t(&k0)[8] = ka[kt][0];
            const uint32_t(&k1)[8] = ka[kt][1];
            const int x = 4 * c + 2 * i;
            if constexpr (kCodes)
              mma16816_f16(s[kt][n], k0[x], k1[x], k0[x + 1], k1[x + 1], q[n][2 * i], q[n][2 * i + 1]);
            else
              mma16816(s[kt][n], k0[x], k1[x], k0[x + 1], k1[x + 1], q[n][2 * i], q[n][2 * i + 1]);
          }
    }
  }
  // the value exponents of the chunk against the unit of O
  float ufac = 1.f, grow = 1.f;  // P times this; O times this
  if constexpr (kQuant && kCodes) {
    int ev;  // largest value exponent of the chunk (kNoExp: no live value)
    asm volatile("ld.shared.s32 %0, [%1];" : "=r"(ev) : "r"(scales + 32 * 8));
    if (ev != kNoExp) {
      if (ev > w.e) {
        grow = w.e == kNoExp ? 1.f : pow2(w.e - ev);
        w.e = ev;
      }
      ufac = pow2(ev - w.e);
    }
  } else if constexpr (kQuant) {
    // fresh values may be of any size: their P must not exceed 1
    if (w.e < 15) {
      grow = w.e == kNoExp ? 1.f : pow2(w.e - 15);
      w.e = 15;
    }
    ufac = pow2(15 - w.e);
  }
  // masks and key factors: keys 16kt + g, 16kt + 8 + g
  float vsc[KT][2];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float k0 = 1.f;
      vsc[kt][e] = ufac;
      if constexpr (kCodes) {
        float v0;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(k0), "=f"(v0) : "r"(scales + (16 * kt + 8 * e + g) * 8));
        vsc[kt][e] *= v0;
      }
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (kCodes) s[kt][n][2 * e + r] *= k0;
          if (!whole && 16 * kt + 8 * e + g >= min(w.seen[n][r], end) - pos) s[kt][n][2 * e + r] = -INFINITY;
        }
    }
  float alpha[kN][2];
  bool moved = grow != 1.f;
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float rf = kQuant && !kCodes ? sl2 : w.rf[n][r];
      float mx = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) mx = max3f(mx, s[kt][n][r], s[kt][n][2 + r]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      const float mn = fmaxf(w.m[n][r], mx * rf);
      const float base = mn == -INFINITY ? 0.f : mn;  // a row that has seen no key yet
      moved |= mn > w.m[n][r];
      alpha[n][r] = ex2_approx(w.m[n][r] - base);
      w.m[n][r] = mn;
      float sum = 0.f;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = ex2_approx(fmaf(s[kt][n][2 * e + r], rf, -base));
          sum += p;
          s[kt][n][2 * e + r] = kQuant ? p * vsc[kt][e] : p;
        }
      w.l[n][r] = fmaf(w.l[n][r], alpha[n][r], sum);
    }
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = alpha[n][r] * grow;
#pragma unroll
        for (int j = 0; j < 8; ++j) w.o[j][n][r] *= f, w.o[j][n][2 + r] *= f;
      }
  }
  // outputs: probabilities are rounded to f16 (see above) or bf16 (2^-8 of their value)
  auto pack = [](float lo, float hi) { return kCodes ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi); };
#pragma unroll
  for (int u = 0; u < KT; ++u) {
    uint32_t pb[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) pb[n][e] = transpose8(pack(s[u][n][2 * e], s[u][n][2 * e + 1]));
    const uint32_t k0 = 16 * u + 2 * t;
    auto product = [&](int j, const uint32_t (&x)[2], const uint32_t (&y)[2]) {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if constexpr (kCodes)
          mma16816_f16(w.o[j][n], x[0], y[0], x[1], y[1], pb[n][0], pb[n][1]);
        else
          mma16816(w.o[j][n], x[0], y[0], x[1], y[1], pb[n][0], pb[n][1]);
      }
    };
    if constexpr (!kCodes) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // eight dimensions of this thread at a time
        uint32_t vb[8][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t ka = k0 + 8 * e, kb = ka + 1;
          const uint4 x = lds128(vs + ka * kRow + (v_unit<kFmt>(2 * g + c, ka) << 4));
          const uint4 y = lds128(vs + kb * kRow + (v_unit<kFmt>(2 * g + c, kb) << 4));
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vb[2 * i][e] = __byte_perm(xs[i], ys[i], 0x5410);
            vb[2 * i + 1][e] = __byte_perm(xs[i], ys[i], 0x7632);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) product(4 * c + j, vb[2 * j], vb[2 * j + 1]);
      }
    } else {
      uint32_t x[4][4];  // codes of keys 2t, 2t + 1, 2t + 8, 2t + 9: 16 dimensions each
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t key = k0 + (i >> 1) * 8 + (i & 1);
        const uint4 y = lds128(vs + key * kRow + (v_unit<kFmt>(g, key) << 4));
        x[i][0] = y.x, x[i][1] = y.y, x[i][2] = y.z, x[i][3] = y.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t vb[4][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          codes_to_f16<kFmt>(__byte_perm(x[2 * e][i], x[2 * e + 1][i], 0x5140), vb[0][e], vb[1][e]);
          codes_to_f16<kFmt>(__byte_perm(x[2 * e][i], x[2 * e + 1][i], 0x7362), vb[2][e], vb[3][e]);
        }
        product(2 * i, vb[0], vb[1]);
        product(2 * i + 1, vb[2], vb[3]);
      }
    }
  }
}

// A row's scores are its products (2^kKeyDown too small) times scale_log2 2^kKeyDown 2^-up, Q having been
// scaled by 2^up. For |q| from 2^121 on, at a scale of 128^-0.5, that factor is no float. The tile's keys are
// then lowered by x powers of two less, x what its largest factor needs: that row's products can only
// overflow where its scores do. The other rows' Q is lowered by 2^-x instead, so their products and
// factors stay as they are (bits are lost from 2^-(31 - x) of the largest element on). Every thread of the
// CTA calls this, with row factors and Q in shared memory; returns x. (Two factors per score in the main
// loop instead took 184 us for 178: eight int8 contexts of 16,384 rows, 32 heads; this form 179.)
template <int kRows>
DLLM_DEVICE int fit_row_factors(float* factor, uint32_t qs, float scale_log2, int lane) {
  const float all = scale_log2 * pow2(kKeyDown);
  float top = 0.f;
  for (int p = lane; p < kRows; p += 32) top = fmaxf(top, factor[p]);
  if (!__any_sync(0xffffffffu, all * top == INFINITY)) return 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int x = min((__float_as_int(all) >> 23) + (__float_as_int(top) >> 23) - 2 * 127 - 126, kKeyDown);
  __half2 f = __float2half2_rn(pow2(-x));
  for (int i = threadIdx.x; i < kRows * 64; i += kThreads) {
    if (all * factor[i >> 6] == INFINITY) continue;
    uint32_t w;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(qs + i * 4));
    const __half2 y = __hmul2(*reinterpret_cast<__half2*>(&w), f);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(qs + i * 4), "r"(*reinterpret_cast<const uint32_t*>(&y)) : "memory");
  }
  __syncthreads();  // every thread has read the factors
  for (int p = threadIdx.x; p < kRows; p += kThreads)
    if (all * factor[p] != INFINITY) factor[p] *= pow2(x);
  __syncthreads();
  return x;
}

template <int kFmt, int kN>
__global__ void __launch_bounds__(kThreads, Cfg<kFmt, kN>::kCtas) attn_chunk_kernel(const __grid_constant__ ChunkArgs a) {
  constexpr int KB = chunk_keys<kFmt>();
  using C = Cfg<kFmt, kN>;
  constexpr int kStages = C::kStages;
  constexpr int kRows = 8 * kN;  // packed rows of a tile
  constexpr bool kQuant = kFmt != kFmtBf16;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % a.splits;
  const int item = blockIdx.x / a.splits;
  const int mtile = item % a.mtiles;
  const int bh = item / a.mtiles;
  const int hkv = bh % a.Hkv, b = bh / a.Hkv;
  griddep_wait();
  griddep_launch_dependents();
  const Seq sq = load_seq(a, b, hkv == 0 && mtile == 0 && split == 0 && threadIdx.x == 0);
  const int row0 = mtile * kRows;           // first packed row
  const int rows = sq.Lq * a.group - row0;  // packed rows left
  if (rows <= 0) return;
  const Span sp = tile_span<KB, kFreshKeys>(a, sq, (row0 + min(rows, kRows) - 1) / a.group);
  const int c_begin = split * a.split_chunks;
  const int c_end = min(sp.total, c_begin + a.split_chunks);
  if (split > 0 && c_begin >= c_end) return;  // this split has no keys (split 0 writes empty rows)

  // ------------------------------------------------------------ key chunks
  const uint32_t stage0 = base + C::kOffStages + warp * (kStages * kStageBytes);
  const uint32_t scale0 = base + C::kOffScales + warp * (kStages * kScaleBytes);
  const int n_mine = c_begin + warp < c_end ? (c_end - c_begin - warp + kWarps - 1) / kWarps : 0;
  const int64_t row_bytes = (int64_t)a.Hkv * (kQuant ? kD : 2 * kD);  // a cache slot
  const uint8_t* kc = a.kc + (int64_t)hkv * (kQuant ? kD : 2 * kD);
  const uint8_t* vc = a.vc + (int64_t)hkv * (kQuant ? kD : 2 * kD);
  const int32_t* table = a.tables != nullptr ? a.tables + (int64_t)b * a.table_stride : nullptr;

  // Table or slot-list entry of this lane's key in its warp's i-th chunk (-1: no such key).
  auto lookup = [&](int i) -> int {
    const int c = c_begin + warp + i * kWarps;
    if (i >= n_mine || c >= sp.cached) return -1;
    const int pos = c * KB + lane;
    if (lane >= KB || pos >= sp.nc) return -1;
    if (table != nullptr) {
      const int blk = a.block_shift >= 0 ? pos >> a.block_shift : pos / a.block_size;
      return blk < a.max_blocks ? table[blk] : -1;
    }
    return a.slots[sq.s_begin + pos];
  };
  uint32_t pend_k = 0, pend_v = 0;  // exponent bytes of this lane's key in the chunk issued last (0: none)
  auto issue = [&](int i, int raw) {
    if (i < n_mine) {
      const int c = c_begin + warp + i * kWarps;
      const uint32_t st = stage0 + (i % kStages) * kStageBytes;
      if (c < sp.cached) {
        const int pos = c * KB + lane;
        int64_t slot = raw;
        if (table != nullptr && raw >= 0) {
          const int off = a.block_shift >= 0 ? pos & (a.block_size - 1) : pos % a.block_size;
          slot = (int64_t)raw * a.block_size + off;
        }
        if (slot < 0 || slot >= a.num_slots) {  // reads as a zero row
          if (lane < KB && pos < sp.nc) set_error(a.err, kDevSlotOutOfRange);
          slot = -1;
        }
        const int row = (int)slot;  // num_slots < 2^31
        if constexpr (kQuant) {
          pend_k = pend_v = 0;
          if (row >= 0) {
            pend_k = a.k_exp[slot * a.Hkv + hkv];
            pend_v = a.v_exp[slot * a.Hkv + hkv];
          }
        }
        constexpr int kUnits = kQuant ? 8 : 16;  // 16-byte units of a row
        constexpr int kStep = 32 / kUnits;       // rows of one warp-wide copy
        const int u = lane % kUnits;
#pragma unroll
        for (int it = 0; it < KB / kStep; ++it) {
          const int key = it * kStep + lane / kUnits;
          const int r = __shfl_sync(0xffffffffu, row, key);
          const int64_t off = (int64_t)max(r, 0) * row_bytes + u * 16;
          cp_async16(st + key * (kUnits * 16) + (k_unit<kFmt>(u, key) << 4), kc + off, r >= 0);
          cp_async16(st + kStageBytes / 2 + key * (kUnits * 16) + (v_unit<kFmt>(u, key) << 4), vc + off, r >= 0);
        }
      } else {
        const int first = (c - sp.cached) * kFreshKeys;
        const int u = lane & 15;
#pragma unroll
        for (int it = 0; it < kFreshKeys / 2; ++it) {
          const int key = it * 2 + (lane >> 4);
          const bool live = first + key < sp.nk;
          const int64_t r = live ? sq.k_begin + first + key : 0;
          const int64_t col = (int64_t)hkv * kD + u * 8;
          cp_async16(st + key * 256 + (k_unit<kFmtBf16>(u, key) << 4), a.k + r * a.k_stride + col, live);
          cp_async16(st + kStageBytes / 2 + key * 256 + (v_unit<kFmtBf16>(u, key) << 4), a.v + r * a.v_stride + col, live);
        }
      }
    }
    cp_async_commit();
  };
  // Scales of chunk i, issued by the last issue(): 2^e of each key times `down`, 2^(e - e_max + 15) of
  // each value, then the values' largest exponent.
  auto put_scales = [&](int i, float down) {
    if constexpr (kQuant) {
      if (i < n_mine && c_begin + warp + i * kWarps < sp.cached) {
        const uint32_t at = scale0 + (i % kStages) * kScaleBytes;
        const int ev = (int)pend_v - 127;
        const bool live = pend_v != 0 && pend_v != kNanByte;
        const int hi = __reduce_max_sync(0xffffffffu, live ? ev : kNoExp);
        const float2 x = make_float2(exp_scale(pend_k) * down, live ? pow2(ev - hi + 15) : exp_scale(pend_v));
        asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(at + lane * 8), "f"(x.x), "f"(x.y) : "memory");
        if (lane == 0) asm volatile("st.shared.s32 [%0], %1;" ::"r"(at + 32 * 8), "r"(hi) : "memory");
      }
    }
  };

  // The first chunks' copies start before Q is staged.
  int raw = lookup(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    issue(i, raw);
    raw = lookup(i + 1);
    if (i + 1 < kStages - 1) put_scales(i, pow2(-kKeyDown));
  }

  if (threadIdx.x == 0) {  // (in shared memory: fewer registers in the main loop)
    asm volatile("st.shared.s32 [%0], %1;" ::"r"(base + C::kOffBlind), "r"(blind_rows(a, sq)) : "memory");
    if constexpr (kQuant) asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + C::kOffDown), "f"(pow2(-kKeyDown)) : "memory");
  }
  // Q rows, packed and swizzled (zero past the tile's rows); f16 with a row factor if the cache is quantised
  for (int i = threadIdx.x; i < kRows * 16; i += kThreads) {
    const int p = i >> 4, u = i & 15;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (p < rows) {
      const int r = (row0 + p) / a.group, h = hkv * a.group + (row0 + p) - r * a.group;
      x = __ldg(reinterpret_cast<const uint4*>(a.q + (sq.q_begin + r) * a.q_stride + (int64_t)h * kD) + u);
    }
    if constexpr (kQuant) {
      uint32_t mx = __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
      mx = max(mx & 0xffffu, mx >> 16);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      // exponent field E -> factor 2^(14 - (E - 127)); zero and non-finite rows keep factor 1
      const int ex = (int)(mx >> 7);
      const int up = mx == 0 || ex == 255 ? 0 : min(141 - ex, 126);
      const float f = pow2(up);
      float y[8];
      bf16x8_to_f32(x, y);
      x = make_uint4(pack_f16x2(y[0] * f, y[1] * f), pack_f16x2(y[2] * f, y[3] * f), pack_f16x2(y[4] * f, y[5] * f),
                     pack_f16x2(y[6] * f, y[7] * f));
      if (u == 0)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + C::kOffRowFactor + p * 4), "f"(pow2(-up)) : "memory");
    }
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(base + C::kOffQ + p * 256 + ((u ^ (p & 1)) << 4)),
                 "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                 : "memory");
  }
  __syncthreads();
  float* factor = reinterpret_cast<float*>(smem + C::kOffRowFactor);
  int less = 0;
  if constexpr (kQuant) {
    less = fit_row_factors<kRows>(factor, base + C::kOffQ, a.scale_log2, lane);
    if (less > 0) {
      if (threadIdx.x == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + C::kOffDown), "f"(pow2(less - kKeyDown)) : "memory");
#pragma unroll
      for (int i = 0; i + 1 < kStages - 1; ++i)  // scales that are there already
        *reinterpret_cast<float*>(smem + (scale0 - base) + i * kScaleBytes + lane * 8) *= pow2(less);
      __syncthreads();
    }
  }
  uint32_t qf[kN][16] = {};
  float back[kN];
  const int64_t L = (int64_t)sq.nc + sq.nk;
  Rows<kN> w;
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const int row = 8 * n + g;
#pragma unroll
    for (int hc = 0; hc < 4 && kQInRegs<kN>; ++hc) {
      const uint4 x = lds128(base + C::kOffQ + row * 256 + (((8 * (hc >> 1) + 2 * t + (hc & 1)) ^ (row & 1)) << 4));
      qf[n][4 * hc] = x.x, qf[n][4 * hc + 1] = x.y, qf[n][4 * hc + 2] = x.z, qf[n][4 * hc + 3] = x.w;
    }
    back[n] = kQuant ? factor[row] : 1.f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int p = 8 * n + 2 * t + r;
      const int i = (row0 + p) / a.group;
      w.m[n][r] = -INFINITY;
      w.l[n][r] = 0.f;
      w.seen[n][r] = (int)(a.causal ? min(L, max((int64_t)0, L - sq.Lq + i + 1)) : L);
      w.rf[n][r] = kQuant ? a.scale_log2 * pow2(kKeyDown - less) * factor[p] : a.scale_log2;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) w.o[j][n][e] = 0.f;
  }
  w.e = kNoExp;
  const int seen_by_all = (int)(a.causal ? min(L, max((int64_t)0, L - sq.Lq + row0 / a.group + 1)) : L);

  for (int i = 0; i < n_mine; ++i) {
    float down = 0.f;
    if constexpr (kQuant) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(down) : "r"(base + C::kOffDown));
    put_scales(i + kStages - 2, down);
    cp_async_wait<kStages - 2>();
    __syncwarp();  // chunk i has arrived for every lane, and no lane still reads chunk i - 1
    issue(i + kStages - 1, raw);
    raw = lookup(i + kStages);
    const int c = c_begin + warp + i * kWarps;
    const uint32_t st = stage0 + (i % kStages) * kStageBytes;
    const uint32_t sc = scale0 + (i % kStages) * kScaleBytes;
    if (c < sp.cached) {
      const int pos = c * KB;
      chunk_step<kQuant, kFmt, kN>(st, st + kStageBytes / 2, sc, base + C::kOffQ, qf, back, lane, a.scale_log2,
                                        min(seen_by_all, sq.nc) - pos >= KB, pos, sq.nc, w);
    } else {
      const int pos = sq.nc + (c - sp.cached) * kFreshKeys;
      chunk_step<kQuant, kFmtBf16, kN>(st, st + kStageBytes / 2, sc, base + C::kOffQ, qf, back, lane, a.scale_log2,
                                            seen_by_all - pos >= kFreshKeys, pos, (int)L, w);
    }
  }
  cp_async_wait<0>();

  // ---------------------------------------------------- merge of the warps
  __syncthreads();  // every warp is done with its stages
  float* mo = reinterpret_cast<float*>(smem);                              // [warp][row][128]
  float2* ml = reinterpret_cast<float2*>(smem + kWarps * kRows * kD * 4);  // [warp][row]
  const float unit = !kQuant ? 1.f : w.e == kNoExp ? 0.f : pow2(w.e - 15);
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = 8 * n + 2 * t + r;
      float sum = w.l[n][r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0) ml[warp * kRows + row] = make_float2(w.m[n][r], sum);
      float* dst = mo + ((size_t)warp * kRows + row) * kD + 16 * g;
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        *reinterpret_cast<float4*>(dst + 2 * j) = make_float4(w.o[j][n][r] * unit, w.o[j][n][2 + r] * unit,
                                                              w.o[j + 1][n][r] * unit, w.o[j + 1][n][2 + r] * unit);
    }
  __syncthreads();
  const bool alone = sp.total <= a.split_chunks;  // no other split has keys of this tile
  int blind;
  asm volatile("ld.shared.s32 %0, [%1];" : "=r"(blind) : "r"(base + C::kOffBlind));
  for (int i = threadIdx.x; i < kRows * (kD / 4); i += kThreads) {
    const int row = i / (kD / 4), d = (i % (kD / 4)) * 4;
    if (row >= rows) break;
    float mm = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) mm = fmaxf(mm, ml[x * kRows + row].x);
    const float least = mm == -INFINITY ? 0.f : mm;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float2 s = ml[x * kRows + row];
      const float f = ex2_approx(s.x - least);
      const float4 y = *reinterpret_cast<const float4*>(mo + ((size_t)x * kRows + row) * kD + d);
      sum = fmaf(s.y, f, sum);  // (a NaN sum stays, whatever its maximum)
      acc.x = fmaf(y.x, f, acc.x), acc.y = fmaf(y.y, f, acc.y);
      acc.z = fmaf(y.z, f, acc.z), acc.w = fmaf(y.w, f, acc.w);
    }
    if (mm == -INFINITY) acc = make_float4(0.f, 0.f, 0.f, 0.f);  // no visible key here, or scores that leave no maximum
    if (alone) {
      const int r = (row0 + row) / a.group, h = hkv * a.group + (row0 + row) - r * a.group;
      const float inv = r >= blind ? 1.f / sum : 0.f;
      uint2 x;
      x.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      x.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(a.o + (sq.q_begin + r) * a.o_stride + (int64_t)h * kD + d) = x;
    } else if (a.cluster) {  // over warp 0's partial, which only this thread reads
      *reinterpret_cast<float4*>(mo + (size_t)row * kD + d) = acc;
      if (d == 0) ml[kWarps * kRows + row] = make_float2(mm, sum);
    } else {
      const int64_t at = ((int64_t)item * a.splits + split) * kRows + row;
      *reinterpret_cast<float4*>(a.part_o + at * kD + d) = acc;
      if (d == 0) a.part_ml[at] = make_float2(mm, sum);
    }
  }
  if (alone || !a.cluster) return;
  // ----------------------------- merge of the cluster's splits, in split order
  const int n = (sp.total + a.split_chunks - 1) / a.split_chunks;  // splits with keys (the others have left)
  cluster_barrier();
  for (int i = split * kThreads + threadIdx.x; i < min(rows, kRows) * (kD / 4); i += n * kThreads) {
    const int row = i / (kD / 4), d = (i % (kD / 4)) * 4;
    const uint32_t from = base + (row * kD + d) * 4, from_ml = base + kWarps * kRows * (kD * 4 + 8) + row * 8;
    float2 x[kClusterSplits];
    float mm = -INFINITY;
#pragma unroll
    for (int s = 0; s < kClusterSplits; ++s) {
      x[s] = make_float2(-INFINITY, 0.f);
      if (s < n) x[s] = cluster_ld2(from_ml, s);
      mm = fmaxf(mm, x[s].x);
    }
    const float least = mm == -INFINITY ? 0.f : mm;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < kClusterSplits; ++s) {
      if (s >= n) break;
      const float f = ex2_approx(x[s].x - least);
      const float4 y = cluster_ld4(from, s);
      sum = fmaf(x[s].y, f, sum);
      acc.x = fmaf(y.x, f, acc.x), acc.y = fmaf(y.y, f, acc.y);
      acc.z = fmaf(y.z, f, acc.z), acc.w = fmaf(y.w, f, acc.w);
    }
    const int r = (row0 + row) / a.group, h = hkv * a.group + (row0 + row) - r * a.group;
    const float inv = r >= blind ? 1.f / sum : 0.f;
    uint2 out;
    out.x = pack_bf16x2(acc.x * inv, acc.y * inv);
    out.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(a.o + (sq.q_begin + r) * a.o_stride + (int64_t)h * kD + d) = out;
  }
  cluster_barrier();  // no CTA leaves while another reads its shared memory
}

// Merges the splits of each row in split order; one warp per packed row, each
// lane four dimensions. The splits' maxima and sums are read 32 at a time, one
// per lane, and their outputs eight at a time, so that no load waits for
// another.
template <int KB, int FB, int kRows>
__global__ void __launch_bounds__(256) attn_chunk_merge_kernel(const __grid_constant__ ChunkArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t item = w / kRows;
  const int row = (int)(w % kRows);
  if (item >= (int64_t)a.B * a.Hkv * a.mtiles) return;
  const int mtile = (int)(item % a.mtiles);
  const int hkv = (int)(item / a.mtiles % a.Hkv), b = (int)(item / a.mtiles / a.Hkv);
  const Seq sq = load_seq(a, b, false);
  const int row0 = mtile * a.tile_rows;
  const int rows = min(sq.Lq * a.group - row0, a.tile_rows);
  if (row >= rows) return;
  const Span sp = tile_span<KB, FB>(a, sq, (row0 + rows - 1) / a.group);
  if (sp.total <= a.split_chunks) return;  // written by its only split
  const int n = (sp.total + a.split_chunks - 1) / a.split_chunks;
  const int64_t at = item * a.splits * kRows + row;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float mm = -INFINITY, sum = 0.f;
  for (int s0 = 0; s0 < n; s0 += 32) {
    float2 x = make_float2(-INFINITY, 0.f);
    if (s0 + lane < n) x = a.part_ml[at + (int64_t)(s0 + lane) * kRows];
    float mx = x.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(mm, mx);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float alpha = ex2_approx(mm - base), f = ex2_approx(x.x - base);
    mm = mn;
    float part = x.y * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    sum = fmaf(sum, alpha, part);
    acc.x *= alpha, acc.y *= alpha, acc.z *= alpha, acc.w *= alpha;
    const int cnt = min(32, n - s0);
    const float* src = a.part_o + (at + (int64_t)s0 * kRows) * kD + lane * 4;
    for (int s = 0; s < cnt; s += 8) {
      float4 y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        y[i] = s + i < cnt ? *reinterpret_cast<const float4*>(src + (int64_t)(s + i) * kRows * kD) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, (s + i) & 31);  // 0 past the last split
        acc.x = fmaf(y[i].x, fi, acc.x), acc.y = fmaf(y[i].y, fi, acc.y);
        acc.z = fmaf(y[i].z, fi, acc.z), acc.w = fmaf(y[i].w, fi, acc.w);
      }
    }
  }
  const int r = (row0 + row) / a.group, h = hkv * a.group + (row0 + row) - r * a.group;
  const float inv = r >= blind_rows(a, sq) ? 1.f / sum : 0.f;
  uint2 out;
  out.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  out.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.o + (sq.q_begin + r) * a.o_stride + (int64_t)h * kD + lane * 4) = out;
}

// The cached rows of every sequence as bf16 rows, one after another: 16 codes
// of K and of V per thread, items (position, head, unit) of a sequence in
// order along x, sequences along y.
template <int kFmt>
__global__ void __launch_bounds__(256) expand_rows_kernel(const __grid_constant__ ChunkArgs a, uint4* k_out, uint4* v_out) {
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.y;
  const Seq sq = load_seq(a, b, false);
  const int per_row = a.Hkv * 8;
  const int64_t first = (int64_t)blockIdx.x * 256;
  const int p0 = (int)(first / per_row);
  const uint32_t at = (uint32_t)(first - (int64_t)p0 * per_row) + threadIdx.x;
  const int pos = p0 + (int)(at / (uint32_t)per_row);
  if (pos >= sq.nc) return;
  const int item = (int)(at % (uint32_t)per_row);
  int64_t slot;
  if (a.tables != nullptr) {
    const int blk = a.block_shift >= 0 ? pos >> a.block_shift : pos / a.block_size;
    const int e = blk < a.max_blocks ? a.tables[b * a.table_stride + blk] : -1;
    slot = e < 0 ? -1 : (int64_t)e * a.block_size + (pos - blk * a.block_size);
  } else {
    slot = a.slots[sq.s_begin + pos];
  }
  uint32_t k[8] = {}, v[8] = {};
  if (slot >= 0 && slot < a.num_slots) {
    const int64_t code = slot * per_row + item, ex = slot * a.Hkv + (item >> 3);
    dequantise16<kFmt>(__ldg(reinterpret_cast<const uint4*>(a.kc) + code), a.k_exp[ex], k);
    dequantise16<kFmt>(__ldg(reinterpret_cast<const uint4*>(a.vc) + code), a.v_exp[ex], v);
  } else if (item == 0) {
    set_error(a.err, kDevSlotOutOfRange);
  }
  const int64_t o = (((int64_t)b * a.dense + pos) * per_row + item) * 2;
  k_out[o] = make_uint4(k[0], k[1], k[2], k[3]);
  k_out[o + 1] = make_uint4(k[4], k[5], k[6], k[7]);
  v_out[o] = make_uint4(v[0], v[1], v[2], v[3]);
  v_out[o + 1] = make_uint4(v[4], v[5], v[6], v[7]);
}

template <int kFmt, int kN>
cudaError_t launch(const ChunkArgs& a, cudaStream_t stream) {
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(attn_chunk_kernel<kFmt, kN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)Cfg<kFmt, kN>::kSmemBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t items = (int64_t)a.B * a.Hkv * a.mtiles;
  if (items * a.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
  e = launch_pdl_cluster(attn_chunk_kernel<kFmt, kN>, dim3((unsigned)(items * a.splits)), dim3(kThreads),
                         Cfg<kFmt, kN>::kSmemBytes, stream, a.cluster ? a.splits : 1, a);
  if (e != cudaSuccess || a.splits == 1 || a.cluster) return e;
  return launch_pdl(attn_chunk_merge_kernel<chunk_keys<kFmt>(), kFreshKeys, 8 * kN>,
                    dim3((unsigned)(items * kN)), dim3(256), 0, stream, a);
}

template <int kFmt>
cudaError_t launch_rows(const ChunkArgs& a, int rows, cudaStream_t stream) {
  if (rows == 8) return launch<kFmt, 1>(a, stream);
  if (rows == 16) return launch<kFmt, 2>(a, stream);
  if constexpr (kFmt != kFmtBf16) return launch<kFmt, 4>(a, stream);
  return cudaErrorInvalidValue;
}

}  // namespace chunk

ChunkPlan plan_attn_chunk(int format, int B, int Hkv, int group, int max_q, int64_t total_q, int max_context,
                          int max_fresh, int num_sms) {
  constexpr int kDenseTiles = 8;
  ChunkPlan p = {};
  const int64_t rows = (int64_t)max_q * group;
  // Which kernel (8 sequences of 32 heads over 1,144 rows in slot lists): 32 rows, e4m3, 42.5 us in
  // attn_chunk.cu, 36 rows 52.6 in the 128-row kernel (from block tables 41.4 and 41.1); 64 rows, e4m3,
  // 79 and 52.7; 32 rows, bf16, 47 in attn_chunk.cu, 34 in the 128-row kernel (block tables).
  p.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 && format != kFmtBf16 ? 32 : kChunkMmaRows;
  if (p.rows == kChunkMmaRows) {
    // One CTA per SM. Splits only while SMs would have nothing to do, and four
    // tiles of keys at least for each.
    p.tile_rows = p.unit_rows = kChunkMmaRows / group * group;  // whole chunk rows
    p.mtiles = (int)((rows + p.tile_rows - 1) / p.tile_rows);
    const int64_t tiles = ((int64_t)max_context + 127) / 128 + ((int64_t)max_fresh + 127) / 128;
    int64_t units = (int64_t)B * Hkv * p.mtiles;
    const int64_t splits = std::max<int64_t>(1, std::min(units > 0 ? num_sms / units : 1, tiles / 4));
    p.split_chunks = (int)std::max<int64_t>(1, (tiles + splits - 1) / splits);
    p.splits = (int)std::max<int64_t>(1, (tiles + p.split_chunks - 1) / p.split_chunks);
    p.workspace_bytes = p.splits > 1 ? units * p.splits * p.rows * (chunk::kD * 4 + 8) : 0;
    // Every work unit expands the quantised rows it reads. From eight row tiles on they are expanded
    // once instead, into bf16 rows that all units read, unless that copy would be larger than 1 GiB
    // (e4m3, 32 heads, 8 sequences over 2,000 rows, in the units, two tiles each, and once: 4 tiles 230
    // and 256 us, 6 tiles 337 and 344, 8 tiles 452 and 435, 16 tiles 1,004 and 896).
    const int64_t cap = ((int64_t)max_context + 127) / 128 * 128;
    const int64_t bytes = 2 * (int64_t)B * cap * Hkv * chunk::kD * 2;
    if (format != kFmtBf16 && p.mtiles >= kDenseTiles && bytes > 0 && bytes <= ((int64_t)1 << 30) &&
        (int64_t)B * cap < ((int64_t)1 << 31) && B < 65536) {
      p.dense = (int)cap;
      p.dense_bytes = bytes;
      p.workspace_bytes += bytes;
    }
    // One or two row tiles per unit: a KV tile takes a unit of two 1.83 times as long (bf16, 2 x 1,024
    // rows over 2,000, 32 heads: 107 us, one tile 117) or 1.45 to 1.8 times (quantised, where one
    // expansion serves both; the less, the more units have one tile only: 32 x 48 rows, 28/4 heads,
    // int8: 41 us, one tile 47; 8 x 256 rows over 2,000 e4m3 rows, 32 heads: 109 and 135; 8 x 384: 212
    // and 194), but fewer, larger units fill the SMs less evenly (bf16, 4 chunks of 300-512 rows, 28/4
    // heads: 131 us, one tile 113). The better estimate of rounds x time decides; half the sequences are
    // taken to end inside a tile, none to be longer than max_q.
    if (p.mtiles >= 2 && p.splits == 1) {
      auto rounds = [&](int64_t unit_rows) {
        const double most = (double)((rows + unit_rows - 1) / unit_rows) * B;
        const double n = Hkv * std::min(most, (double)total_q * group / (double)unit_rows + 0.5 * B) / num_sms;
        return n > 3 ? n + 0.5 : std::ceil(n);
      };
      const double pair = format == kFmtBf16 || p.dense > 0 ? 1.83 : 1.45;
      if (pair * rounds(2 * p.tile_rows) < rounds(p.tile_rows)) {
        p.unit_rows = 2 * p.tile_rows;
        p.mtiles = (int)((rows + p.unit_rows - 1) / p.unit_rows);
      }
    }
    return p;
  }
  p.tile_rows = p.unit_rows = p.rows;
  p.mtiles = (int)((rows + p.rows - 1) / p.rows);
  const int kb = format == kFmtBf16 ? 16 : 32;
  const int64_t chunks = ((int64_t)max_context + kb - 1) / kb + ((int64_t)max_fresh + 15) / 16;
  const int64_t items = (int64_t)B * Hkv * p.mtiles;
  // Splits: the count with the least estimated time, in chunks of a warp. A CTA
  // of c chunks a warp takes c + 3; the launch takes whole waves of CTAs if all
  // contexts are as long as the bound, and if they are 60 % of it on average
  // its mean load and the last CTA's tail: the sum of both estimates decides.
  // A second kernel that merges costs eight chunks and one for 8 splits. Up to 8 splits of a launch that
  // fits the SMs at once are clusters that merge their own (32 contexts of 128-1,024 bf16 rows, 28/4
  // heads, two splits: 15.1 us with the second kernel, 13.5 as clusters; 16 x 2 rows over 8,192 e4m3
  // rows, 32/4 heads: 53 and 44). In larger launches a cluster waits for as many free places (8 contexts
  // of 16,384 e4m3 rows, 32 heads, five splits: 170 us and 200).
  const int64_t slots = (int64_t)(format == kFmtBf16 || p.rows > 16 ? 2 : 3) * num_sms;  // Cfg::kCtas
  auto in_cluster = [&](int64_t s) { return s > 1 && s <= chunk::kClusterSplits && items * s <= slots; };
  int64_t splits = 1;
  double best = 0;
  for (int64_t s = 1; items > 0 && s <= std::max<int64_t>(1, chunks / chunk::kWarps) && s <= 1024; s += std::max<int64_t>(1, s / 8)) {
    const int64_t per = (chunks + s - 1) / s;
    const double cta = (double)((per + chunk::kWarps - 1) / chunk::kWarps) + 3;
    const double waves = (double)(items * s) / (double)slots;
    const double cost = cta * (double)((items * s + slots - 1) / slots) + cta * (0.6 * waves + 1) + (in_cluster(s) ? 4 : s > 1 ? 8 + (double)s / 8 : 0);
    if (s == 1 || cost < best) {
      best = cost;
      splits = s;
    }
  }
  p.split_chunks = (int)std::max<int64_t>(1, (chunks + splits - 1) / splits);
  p.splits = (int)std::max<int64_t>(1, (chunks + p.split_chunks - 1) / p.split_chunks);
  p.cluster = in_cluster(p.splits);
  p.workspace_bytes = p.splits > 1 && !p.cluster ? items * p.splits * p.rows * (chunk::kD * 4 + 8) : 0;
  return p;
}

cudaError_t launch_expand_rows(const ChunkArgs& a, int format, void* k_out, void* v_out, cudaStream_t stream) {
  const int64_t items = (int64_t)a.max_context * a.Hkv * 8;
  const dim3 grid((unsigned)((items + 255) / 256), (unsigned)a.B);
  return format == kFmtE4m3
             ? launch_pdl(chunk::expand_rows_kernel<kFmtE4m3>, grid, dim3(256), 0, stream, a, (uint4*)k_out, (uint4*)v_out)
             : launch_pdl(chunk::expand_rows_kernel<kFmtInt8>, grid, dim3(256), 0, stream, a, (uint4*)k_out, (uint4*)v_out);
}

cudaError_t launch_attn_chunk(ChunkArgs a, int format, const ChunkPlan& plan, const ChunkMaps& maps, void* workspace,
                              int num_sms, cudaStream_t stream) {
  a.tile_rows = plan.tile_rows;
  a.unit_rows = plan.unit_rows;
  a.mtiles = plan.mtiles;
  a.splits = plan.splits;
  a.split_chunks = plan.split_chunks;
  a.cluster = plan.cluster;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.mtiles * a.splits * plan.rows;
  a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.dense_bytes);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * chunk::kD);
  if (plan.rows == kChunkMmaRows) {
    const int64_t items = (int64_t)a.B * a.Hkv * a.mtiles;
    if (items * a.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
    a.total_units = (int)(items * a.splits);
    a.dense = plan.dense;
    cudaError_t e = cudaSuccess;
    if (plan.dense > 0) {
      e = launch_expand_rows(a, format, workspace, static_cast<uint8_t*>(workspace) + plan.dense_bytes / 2, stream);
      if (e != cudaSuccess) return e;
      a.num_slots = (int64_t)a.B * plan.dense;
      format = kFmtBf16;
    }
    e = launch_attn_chunk_mma(maps, a, format, num_sms, stream);
    if (e != cudaSuccess || a.splits == 1) return e;
    return launch_pdl(chunk::attn_chunk_merge_kernel<128, 128, kChunkMmaRows>,
                      dim3((unsigned)(items * (kChunkMmaRows / 8))), dim3(256), 0, stream, a);
  }
  switch (format) {
    case kFmtBf16: return chunk::launch_rows<kFmtBf16>(a, plan.rows, stream);
    case kFmtE4m3: return chunk::launch_rows<kFmtE4m3>(a, plan.rows, stream);
    default: return chunk::launch_rows<kFmtInt8>(a, plan.rows, stream);
  }
}

}  // namespace dllm
