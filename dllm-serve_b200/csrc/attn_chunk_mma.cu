// Attention of a chunk of new tokens over a paged KV cache, for launches with
// more query rows per KV head than attn_chunk.cu takes (diffusion blocks,
// prefill chunks): tcgen05 + TMEM + TMA, sm_100a.
//
// A work unit is (sequence b, KV head, one or two tiles of packed rows, split
// of the keys); packed row p of a (sequence, KV head) is row p / group of the
// chunk for head p % group of the KV head's group, so grouped heads share every
// key tile they read. A row tile holds as many whole chunk rows as fit 128
// packed rows (all 128 where the group divides them). Keys come in tiles of
// 128: the sequence's cached rows, then its fresh rows, cut at the last key
// that a row of the unit sees. Softmax is online (a running maximum and sum per
// row, the accumulator rescaled when the maximum has grown by 2^8).
// Probabilities are rounded to bf16 (2^-8 of their value, up to 256).
//
// One row tile ("single"): each KV tile's 128 columns are split between two
// softmax warpgroups, each with its own running maximum, sum and accumulator,
// merged once per unit (exact: softmax of a union). Two row tiles ("pair",
// where such units fill the SMs evenly enough): a warpgroup per row tile, and
// every key tile that is read, and expanded, serves both: the single form
// needs 64 KB per 2,290 cycles and SM, close to what L2 delivers, and expands a
// quantised tile in about as long.
//
// Quantised caches: 8-bit rows are brought into shared memory as they are
// (TMA boxes, or four rows at a time where the slots are scattered) and two more
// warpgroups expand them into the bf16 stages that the matrix instructions
// read. Every value a code stands for is a bf16 number, so this rounds
// nothing, and the rest of the kernel is the same for every format. HBM and
// L2 carry one byte per element.
//
// Measured: 4 chunks of 300-512 rows over 2,000-4,600 bf16 rows, 28/4 heads: 116
// us, 785 TFLOP/s; 4 prefill chunks of 1,024-2,048 rows over 1,024-6,144, 32
// heads: 544 us, 882 TFLOP/s (bf16), 609 us (e4m3, expanded once by a kernel of
// its own). Between a tile's first product and its second stands one
// warpgroup's softmax, about 1,500 cycles in which that row tile's products
// wait; the tensor pipe is busy half of the time, the exponentials' half. 32
// blocks of 32 rows over 176-496 int8 rows, 28/4 heads: 21 us, where a unit's
// first loads and its epilogue are as long as its four tiles.
//
// Roles (12 warps, 20 with a quantised cache):
//   warps 0-3, 4-7  softmax warpgroups
//   warp 8          loader of K: bf16 stages, or the raw K ring of a quantised cache
//   warp 9          issues the MMAs, owns TMEM
//   warp 10         loader of V
//   warp 11         loader of Q
//   warps 12-15     quantised: fill the K ring (expand cached tiles, load fresh ones)
//   warps 16-19     quantised: fill the V ring
// (Single, e4m3:) one warpgroup for both rings was the bottleneck: 1,560 cycles
// to expand a tile of K or V, 4,270 per KV tile against 2,290 of the bf16
// kernel. With this many roles instruction fetches count: loops that are not
// unrolled took 126 us to 114 (8 x 128 rows over 4,000 e4m3 rows, 32 heads).
// TMEM (512 columns): S buffers [0,128) [128,256), accumulators at 256 and 384;
// P (bf16) over the first columns of S (pair) or of each half of it (single).
// MMA order per KV tile j: single PV(j) of both halves, then QK(j+2); pair, for
// each row tile, PV(j), then QK(j+1).
#include <algorithm>
#include <atomic>
#include <cuda.h>

#include "attn_chunk.cuh"
#include "kvquant.cuh"

namespace dllm {
namespace chunk128 {

namespace {

using chunk::load_seq;
using chunk::Seq;
using chunk::Span;
using chunk::tile_span;

constexpr int kD = 128;
constexpr int kTileM = kChunkMmaRows;
constexpr int kTileN = 128;
constexpr int kHalfN = 64;
constexpr uint32_t kTileBytes = 128 * kD * 2;  // bf16 tile
constexpr uint32_t kChunkBytes = 128 * 128;    // its 64-column half; also an 8-bit tile

template <int kFmt, bool kPair>
struct Layout {
  static constexpr bool kQuant = kFmt != kFmtBf16;
  // Registers: the softmax warpgroups take those that the other roles do not need.
  // bf16: 384 x 168 = 256 x 208 + 128 x 88; quantised: 640 x 96 = 256 x 144 + 384 x 64.
  static constexpr int kThreads = kQuant ? 640 : 384;
  static constexpr int kRegsSoftmax = kQuant ? 144 : 208;
  static constexpr int kRegsOther = kQuant ? 64 : 88;
  static constexpr int kTilesQ = kPair ? 2 : 1;
  static constexpr int kRaw = kPair ? 1 : 2;  // stages of each raw ring (the second Q tile takes one's place)
  static constexpr int kStagesK = kQuant ? 2 : 3;
  static constexpr int kStagesV = kQuant || kPair ? 2 : 3;
  // arrivals that complete a bf16 stage: the four expanding warps, or the loader's
  static constexpr int kFull = kQuant ? 4 : 1;
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffK = kOffQ + kTilesQ * kTileBytes;
  static constexpr uint32_t kOffV = kOffK + kStagesK * kTileBytes;
  static constexpr uint32_t kOffRaw = kOffV + kStagesV * kTileBytes;  // K ring, V ring
  static constexpr uint32_t kOffExp = kOffRaw + (kQuant ? 2 * kRaw * kChunkBytes : 0);  // exponent bytes of each raw stage
  static constexpr uint32_t kOffBar = kOffExp + (kQuant ? 2 * kRaw * 128 : 0);
  static constexpr int BAR_QFULL = 0;
  static constexpr int BAR_QEMPTY = 1;
  static constexpr int BAR_KFULL = 2;
  static constexpr int BAR_KEMPTY = BAR_KFULL + kStagesK;
  static constexpr int BAR_VFULL = BAR_KEMPTY + kStagesK;
  static constexpr int BAR_VEMPTY = BAR_VFULL + kStagesV;
  static constexpr int BAR_SFULL = BAR_VEMPTY + kStagesV;  // 2: S buffer holds QK of a tile
  static constexpr int BAR_PFULL = BAR_SFULL + 2;          // 2: both P halves written
  static constexpr int BAR_OREADY = BAR_PFULL + 2;         // single: PVs of one more tile completed
  static constexpr int BAR_OFULL = BAR_OREADY + 1;         // 2: a unit's last PVs (of a row tile) completed
  static constexpr int BAR_XML = BAR_OFULL + 2;            // warpgroup 1's (max, sum) published
  static constexpr int BAR_XF = BAR_XML + 1;               // the merge factors published
  static constexpr int BAR_DRAIN = BAR_XF + 1;
  static constexpr int BAR_VLAND = BAR_DRAIN + 1;          // a partial V tile landed
  static constexpr int BAR_RFULL = BAR_VLAND + 1;          // 2 rings x kRaw: raw tile and exponents landed
  static constexpr int BAR_REMPTY = BAR_RFULL + 2 * kRaw;  // 2 rings x kRaw
  static constexpr int kNumBars = BAR_REMPTY + 2 * kRaw;
  static constexpr uint32_t kOffMisc = kOffBar + kNumBars * 8;  // abort flag, TMEM address
  static constexpr uint32_t kOffXch = (kOffMisc + 64 + 15) & ~15u;
  static constexpr uint32_t kSmemBytes = kOffXch + kTileM * 8 + 1024;  // + alignment slack
  static_assert(kSmemBytes <= 232448, "over the sm_100a per-CTA shared-memory limit");
};

struct Unit {
  bool valid;
  int b, hkv, item, split;
  int row0, rows;      // first packed row, number of packed rows (at most a.unit_rows)
  Seq sq;
  Span sp;             // tiles of the whole row tile
  int t0, nkv;         // this split's tiles
  int64_t L;
};

// Units are numbered ((b * Hkv + hkv) * mtiles + (last tile first)) * splits +
// split: neighbours read the same keys (L2), and a causal chunk's longest
// tiles come first.
DLLM_DEVICE Unit decode_unit(int u, const ChunkArgs& a, bool report) {
  Unit r;
  r.split = u % a.splits;
  const int v = u / a.splits;
  const int mt = a.mtiles - 1 - v % a.mtiles;
  const int bh = v / a.mtiles;
  r.b = bh / a.Hkv;
  r.hkv = bh - r.b * a.Hkv;
  r.item = bh * a.mtiles + mt;
  r.row0 = mt * a.unit_rows;
  r.sq = load_seq(a, r.b, report && r.hkv == 0 && mt == 0 && r.split == 0);
  r.rows = min(r.sq.Lq * a.group - r.row0, a.unit_rows);
  r.L = (int64_t)r.sq.nc + r.sq.nk;
  r.valid = r.rows > 0;
  r.t0 = r.nkv = 0;
  r.sp = Span{};
  if (!r.valid) return r;
  r.sp = tile_span<kTileN, kTileN>(a, r.sq, (r.row0 + r.rows - 1) / a.group);
  r.t0 = r.split * a.split_chunks;
  r.nkv = min(r.sp.total, r.t0 + a.split_chunks) - r.t0;
  if (r.split > 0 && r.nkv <= 0) r.valid = false;  // split 0 writes rows without keys
  r.nkv = max(r.nkv, 0);
  return r;
}

struct KvTile {
  bool fresh;
  int pos;      // first key's position in the sequence
  int valid;    // live keys (1..128)
  int64_t row;  // fresh tiles: first row of k / v
};
DLLM_DEVICE KvTile kv_tile(const Unit& u, int j) {
  const int t = u.t0 + j;
  KvTile r;
  r.fresh = t >= u.sp.cached;
  if (!r.fresh) {
    r.pos = t * kTileN;
    r.valid = min(kTileN, u.sp.nc - r.pos);
    r.row = 0;
  } else {
    const int at = (t - u.sp.cached) * kTileN;
    r.pos = u.sq.nc + at;
    r.valid = min(kTileN, u.sp.nk - at);
    r.row = u.sq.k_begin + at;
  }
  return r;
}

// Keys past a partial tile's end must not reach the second product as NaN: V
// rows up to the next multiple of 16 (the product's step) are cleared, by one
// warp, once the tile has landed.
DLLM_DEVICE void clear_tail(uint8_t* tile, int valid, int lane) {
  const int n = ((valid + 15) & ~15) - valid;
  for (int i = lane; i < n * 16; i += 32)
    *reinterpret_cast<uint4*>(tile + ((i >> 3) & 1) * kChunkBytes + (valid + (i >> 4)) * 128 + ((i & 7) << 4)) =
        make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();  // generic-proxy writes -> tensor-core reads
  __syncwarp();
}

// Four rows (any order) of a 2-D tensor map whose box is one row: they land one
// after another. A row index past the map's end gives zeros.
DLLM_DEVICE void tma_gather4(uint32_t dst, const void* tmap, uint32_t bar, int x, const int (&r)[4]) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
      : "memory");
}

template <int kRegs, bool kMore>
DLLM_DEVICE void set_max_registers() {
  if constexpr (kMore)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// The matrix instructions with descriptors given as their low words: the high
// word (stride 1024, 128-byte swizzle) is the same for every tile here, and
// one 32-bit word per operand keeps the issuing thread's registers few.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
DLLM_DEVICE uint32_t desc_lo(uint32_t saddr, uint32_t lbo_bytes) {
  return ((saddr >> 4) & 0x3fffu) | ((lbo_bytes >> 4) << 16);
}
DLLM_DEVICE void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}
DLLM_DEVICE void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(acc), "n"(kDescHi)
      : "memory");
}

// P = 2^(S*scale_log2 - m) for 32 kChunks columns of one row, packed to bf16
// pairs and stored to TMEM at tP; returns the row sum of P (fp32).
template <int kChunks>
DLLM_DEVICE float exp_store(const uint32_t (&s)[kChunks][32], float sl2, float m, uint32_t tP) {
  const float neg_m = -m;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    uint32_t pk[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p0 = ex2_approx(fmaf(__uint_as_float(s[c][2 * e]), sl2, neg_m));
      const float p1 = ex2_approx(fmaf(__uint_as_float(s[c][2 * e + 1]), sl2, neg_m));
      acc[(2 * e) & 3] += p0;
      acc[(2 * e + 1) & 3] += p1;
      pk[e] = pack_bf16x2(p0, p1);
    }
    tmem_st16(tP + c * 16, pk);
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

}  // namespace

// Softmax warpgroup w of a pair launch: row tile w of every unit, KV tile by KV
// tile. PV(j-1) was issued before QK(j), so when S(j) is there the accumulator
// holds every earlier tile and may be rescaled.
template <typename S>
DLLM_DEVICE void softmax_pair(const ChunkArgs& a, uint32_t tmem, uint32_t bar0, volatile int* abort_flag) {
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * (uint32_t)i; };
  const int lane = threadIdx.x & 31;
  const int wg = threadIdx.x >> 7, wq = (threadIdx.x >> 5) & 3;
  const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
  const uint32_t tS = tmem + lane_base + wg * 128;
  const uint32_t tO = tmem + lane_base + 256 + wg * 128;
  const float sl2 = a.scale_log2;
  uint32_t s_it = 0, o_it = 0;
  for (int u = blockIdx.x; u < a.total_units; u += gridDim.x) {
    const Unit t = decode_unit(u, a, false);
    if (!t.valid || t.rows <= wg * a.tile_rows) continue;
    const int rows = min(t.rows - wg * a.tile_rows, a.tile_rows);  // of this tile
    const int p = t.row0 + wg * a.tile_rows + (threadIdx.x & 127);
    const int qr = p / a.group;  // row of the chunk
    const int seen = (int)(a.causal ? min(t.L, max((int64_t)0, t.L - t.sq.Lq + qr + 1)) : t.L);
    const bool row_ok = (int)(threadIdx.x & 127) < rows;
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < t.nkv; ++j) {
      const KvTile kt = kv_tile(t, j);
      if (!mbar_wait_warp(bar(S::BAR_SFULL + wg), s_it & 1, abort_flag)) return;
      ++s_it;
      tc_fence_after();
      const int nv = min(kt.valid, seen - kt.pos);  // this row's visible columns
      // bf16 caches: the row's 128 scores at once. Quantised ones leave registers for 64: the upper
      // half is read for its maximum, and again once the lower half's P is written.
      constexpr int kHalves = S::kQuant ? 2 : 1, kChunks = 4 / kHalves;
      uint32_t s[kChunks][32];
      auto load = [&](int col) {  // from column `col` on, hidden ones as -inf
#pragma unroll
        for (int c = 0; c < kChunks; ++c) tmem_ld32(tS + col + c * 32, s[c]);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, nv < col + kChunks * 32)) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (col + c * 32 + e >= nv) s[c][e] = __float_as_uint(-INFINITY);
        }
      };
      auto largest = [&]() -> float {
        float mq[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          float x = __uint_as_float(s[c][0]);
#pragma unroll
          for (int e = 1; e < 31; e += 2) x = max3f(x, __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
          mq[c] = fmaxf(x, __uint_as_float(s[c][31]));
        }
        return kChunks == 4 ? max3f(mq[0], mq[1], fmaxf(mq[kChunks - 2], mq[kChunks - 1])) : fmaxf(mq[0], mq[1]);
      };
      float mxs = -INFINITY;
      const int last = kHalves > 1 && kt.valid > kHalfN ? 1 : 0;
#pragma unroll 1
      for (int h = last; h >= 0; --h) {
        load(h * kHalfN);
        mxs = fmaxf(mxs, largest());
      }
      mxs *= sl2;
      // Lazy rescaling: a stale maximum stays while the new one exceeds it by at most 8 (log2
      // units), so P stays <= 256; a row's first visible key sets it (its accumulator holds zeros).
      const bool first = m == -INFINITY;
      // (rows past the tile's last hold another sequence's queries: they decide nothing)
      const bool rescale = __any_sync(0xffffffffu, row_ok && !first && mxs > m + 8.f);
      float alpha = 1.f;
      if (first) {
        m = mxs;
      } else if (rescale) {
        const float mn = fmaxf(m, mxs);
        alpha = ex2_approx(m - mn);
        m = mn;
        l *= alpha;
      }
      const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 1
      for (int h = 0; h <= last; ++h) {
        if (h > 0) load(h * kHalfN);
        l += exp_store<kChunks>(s, sl2, base, tS + h * (kHalfN / 2));  // hidden columns give exact zeros
      }
      if (rescale) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(tO + c * 32, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(S::BAR_PFULL + wg));
    }
    // Epilogue: O / l -> bf16. A 4x4 transpose of 16-byte vectors inside each lane quad lets every
    // store write 8 rows x 64 contiguous bytes instead of 32 rows x 16.
    const int h = t.hkv * a.group + p - qr * a.group;
    __nv_bfloat16* orow = a.o + (t.sq.q_begin + qr) * a.o_stride + (int64_t)h * kD;
    if (t.nkv > 0) {
      if (!mbar_wait_warp(bar(S::BAR_OFULL + wg), o_it & 1, abort_flag)) return;
      ++o_it;
      tc_fence_after();
      const float inv = 1.f / l;
      const bool none = seen <= 0;  // no visible key: zero row
      const int qj = lane & 3;
      __nv_bfloat16* quad[4];
      bool live[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        quad[r] = reinterpret_cast<__nv_bfloat16*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(orow), (lane & ~3) + r));
        live[r] = __shfl_sync(0xffffffffu, row_ok ? 1 : 0, (lane & ~3) + r) != 0;
      }
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
        uint4 v[4];
        auto val = [&](int e) { return none ? 0.f : __uint_as_float(o[e]) * inv; };
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = make_uint4(pack_bf16x2(val(8 * e), val(8 * e + 1)), pack_bf16x2(val(8 * e + 2), val(8 * e + 3)),
                            pack_bf16x2(val(8 * e + 4), val(8 * e + 5)), pack_bf16x2(val(8 * e + 6), val(8 * e + 7)));
        quad_transpose16(v, qj);  // v[r] = vector qj of the quad's row r
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (live[r]) reinterpret_cast<uint4*>(quad[r] + c * 32)[qj] = v[r];
      }
      // O is read out; the next unit's first PV may overwrite it once this
      // warpgroup arrives on its first P barrier (program order + fence).
      tc_fence_before();
    } else if (row_ok) {
      uint4* dst = reinterpret_cast<uint4*>(orow);
      for (int v = 0; v < kD / 8; ++v) dst[v] = make_uint4(0, 0, 0, 0);
    }
  }
}

template <int kFmt, bool kPair>
__global__ void __launch_bounds__(Layout<kFmt, kPair>::kThreads, 1)
    attn_chunk_mma_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmKc, const __grid_constant__ CUtensorMap tmVc,
                          const __grid_constant__ CUtensorMap tmKg, const __grid_constant__ CUtensorMap tmVg,
                          const __grid_constant__ ChunkArgs a) {
  using S = Layout<kFmt, kPair>;
  constexpr bool kQuant = S::kQuant;
  constexpr int kStagesK = S::kStagesK, kStagesV = S::kStagesV, kRaw = S::kRaw;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t base = (raw_base + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_base);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int total_units = a.total_units;
  const uint32_t bar0 = base + S::kOffBar;
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * (uint32_t)i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kOffMisc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::kOffMisc + 16);

  if (threadIdx.x == 0) {
    mbar_init(bar(S::BAR_QFULL), 1);
    mbar_init(bar(S::BAR_QEMPTY), 1);
    for (int s = 0; s < kStagesK; ++s) {
      mbar_init(bar(S::BAR_KFULL + s), S::kFull);
      mbar_init(bar(S::BAR_KEMPTY + s), 1);
    }
    for (int s = 0; s < kStagesV; ++s) {
      mbar_init(bar(S::BAR_VFULL + s), S::kFull);
      mbar_init(bar(S::BAR_VEMPTY + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(S::BAR_SFULL + i), 1);
      mbar_init(bar(S::BAR_PFULL + i), kPair ? 4 : 8);  // one arrival per warp that writes this P
      mbar_init(bar(S::BAR_OFULL + i), 1);
    }
    mbar_init(bar(S::BAR_OREADY), 1);
    mbar_init(bar(S::BAR_XML), 128);  // every thread of warpgroup 1
    mbar_init(bar(S::BAR_XF), 128);   // every thread of warpgroup 0
    mbar_init(bar(S::BAR_DRAIN), 1);
    mbar_init(bar(S::BAR_VLAND), 1);
    for (int s = 0; s < 2 * kRaw; ++s) {
      mbar_init(bar(S::BAR_RFULL + s), 2);   // the copies' bytes, the exponents
      mbar_init(bar(S::BAR_REMPTY + s), 4);  // the expanding warps
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  // Register counts are stated inside each role's branch, where the compiler
  // takes them into account.
  if (warp >= 8 && warp < 12) {
    set_max_registers<S::kRegsOther, false>();
    if (warp == 8 || warp == 10) {
      // ---------------------------------------------------------------- loaders
      const bool is_k = warp == 8;
      const uint64_t pol = policy_evict_last();
      const int nst = is_k ? kStagesK : kStagesV;
      const int bfull = is_k ? S::BAR_KFULL : S::BAR_VFULL;
      const int bempty = is_k ? S::BAR_KEMPTY : S::BAR_VEMPTY;
      const uint32_t ring = base + (is_k ? S::kOffK : S::kOffV);
      const int rfull = S::BAR_RFULL + (is_k ? 0 : kRaw), rempty = S::BAR_REMPTY + (is_k ? 0 : kRaw);
      const uint32_t raw_ring = base + S::kOffRaw + (is_k ? 0 : kRaw * kChunkBytes);
      const uint32_t exp_ring = base + S::kOffExp + (is_k ? 0 : kRaw * 128);
      const uint8_t* exps = is_k ? a.k_exp : a.v_exp;
      const CUtensorMap* mfresh = is_k ? &tmK : &tmV;
      const CUtensorMap* mcache = is_k ? &tmKc : &tmVc;
      const CUtensorMap* mgather = is_k ? &tmKg : &tmVg;
      uint32_t done = 0;                           // tiles passed in the bf16 ring
      uint32_t raw_done = 0;                       // tiles issued into the raw ring
      uint32_t land = 0;                           // partial V tiles landed
      bool ok = true;
      for (int u = blockIdx.x; u < total_units && ok; u += gridDim.x) {
        const Unit t = decode_unit(u, a, is_k && lane == 0);
        if (!t.valid) continue;
        const int32_t* table = a.tables != nullptr ? a.tables + (int64_t)t.b * a.table_stride : nullptr;
        for (int j = 0; j < t.nkv && ok; ++j, ++done) {
          const KvTile kt = kv_tile(t, j);
          if (kQuant && kt.fresh) break;  // the expanding warps load fresh tiles, which come last
          const int st = done % nst;
          // cached tiles: this lane's four rows 4 * lane + i, and whether the tile is one run of slots
          int sl[4], s0 = 0;
          bool contig = true;
          if (!kt.fresh) {
            if (!kQuant && a.dense > 0) {
              s0 = t.b * a.dense + kt.pos;
#pragma unroll
              for (int i = 0; i < 4; ++i) sl[i] = s0 + 4 * lane + i;
            } else if (table != nullptr && a.block_size % kTileN == 0) {
              // the tile lies inside one block
              const int blk = kt.pos / a.block_size;
              const int e = blk < a.max_blocks ? table[blk] : -1;
              const int64_t at = e < 0 ? -1 : (int64_t)e * a.block_size + kt.pos % a.block_size;
              const bool in = at >= 0 && at < a.num_slots;
              s0 = in ? (int)at : (int)a.num_slots;  // past the cache: the copy brings zeros
#pragma unroll
              for (int i = 0; i < 4; ++i) sl[i] = in ? s0 + 4 * lane + i : -1;
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = 4 * lane + i, pos = kt.pos + r;
                sl[i] = -1;
                if (r < kt.valid) {
                  if (table != nullptr) {
                    const int blk = pos / a.block_size;
                    const int e = blk < a.max_blocks ? table[blk] : -1;
                    const int64_t at = e < 0 ? -1 : (int64_t)e * a.block_size + pos % a.block_size;
                    sl[i] = at < a.num_slots ? (int)at : -1;
                  } else {
                    sl[i] = a.slots[t.sq.s_begin + pos];
                  }
                }
              }
              s0 = __shfl_sync(0xffffffffu, sl[0], 0);
              contig = s0 >= 0 && (int64_t)s0 + kt.valid <= a.num_slots;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (4 * lane + i < kt.valid && sl[i] != s0 + 4 * lane + i) contig = false;
              contig = __all_sync(0xffffffffu, contig);
            }
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool live = 4 * lane + i < kt.valid;
              if (live && (sl[i] < 0 || sl[i] >= a.num_slots)) bad = true;
              if (!live || sl[i] >= a.num_slots) sl[i] = -1;  // -1: reads as a zero row
            }
            if (bad) set_error(a.err, kDevSlotOutOfRange);
          }
          if constexpr (kQuant) {
            // ---- raw ring
            const int rs = raw_done % kRaw;
            if (raw_done >= (uint32_t)kRaw)
              ok = mbar_wait_warp(bar(rempty + rs), (raw_done / kRaw - 1) & 1, abort_flag);
            if (!ok) break;
            const uint32_t dst = raw_ring + rs * kChunkBytes, fb = bar(rfull + rs);
            if (contig) {
              if (lane == 0) {
                mbar_arrive_expect_tx(fb, kChunkBytes);
                tma_load_3d(dst, mcache, fb, 0, t.hkv, s0, pol);
              }
            } else {
              if (lane == 0) mbar_arrive_expect_tx(fb, kChunkBytes);
              __syncwarp();
              int r[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) r[i] = sl[i] >= 0 ? sl[i] : (int)a.num_slots;
              tma_gather4(dst + 4 * lane * kD, mgather, fb, t.hkv * kD, r);
            }
            uint32_t e4 = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (sl[i] >= 0) e4 |= (uint32_t)exps[(int64_t)sl[i] * a.Hkv + t.hkv] << (8 * i);
            *reinterpret_cast<uint32_t*>(smem + (exp_ring - base) + rs * 128 + 4 * lane) = e4;
            __syncwarp();
            if (lane == 0) mbar_arrive(fb);
            ++raw_done;
          } else {
            // ---- a bf16 stage
            if (done >= (uint32_t)nst) ok = mbar_wait_warp(bar(bempty + st), (done / nst - 1) & 1, abort_flag);
            if (!ok) break;
            const uint32_t dst = ring + st * kTileBytes;
            uint8_t* tile = smem + (dst - base);
            const bool clear = !is_k && (kt.valid & 15) != 0;
            const uint32_t fb = bar(clear ? S::BAR_VLAND : bfull + st);
            if (lane == 0) mbar_arrive_expect_tx(fb, kTileBytes);
            __syncwarp();
            if (kt.fresh || contig) {
              if (lane == 0) {
                const CUtensorMap* mp = kt.fresh ? mfresh : mcache;
                const int row = kt.fresh ? (int)kt.row : s0;
                tma_load_3d(dst, mp, fb, 0, t.hkv, row, pol);
                tma_load_3d(dst + kChunkBytes, mp, fb, 64, t.hkv, row, pol);
              }
            } else {
              int r[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) r[i] = sl[i] >= 0 ? sl[i] : (int)a.num_slots;
              tma_gather4(dst + 4 * lane * 128, mgather, fb, t.hkv * kD, r);
              tma_gather4(dst + kChunkBytes + 4 * lane * 128, mgather, fb, t.hkv * kD + 64, r);
            }
            if (clear) {
              ok = mbar_wait_warp(fb, land & 1, abort_flag);
              if (!ok) break;
              ++land;
              clear_tail(tile, kt.valid, lane);
              if (lane == 0) mbar_arrive(bar(bfull + st));
            }
          }
        }
      }
      if (lane == 0 && *abort_flag) {
        // Drain: wait (bounded) for the loads that may still be in flight.
        if (!kQuant)
          for (uint32_t n = (done > (uint32_t)nst ? done - nst : 0); n < done; ++n)
            mbar_wait_drain(bar(bfull + n % nst), (n / nst) & 1, 100000000ull);
        if (kQuant)
          for (uint32_t n = (raw_done > (uint32_t)kRaw ? raw_done - kRaw : 0); n < raw_done; ++n)
            mbar_wait_drain(bar(rfull + n % kRaw), (n / kRaw) & 1, 100000000ull);
        if (!kQuant && !is_k) mbar_wait_drain(bar(S::BAR_VLAND), land & 1, 100000000ull);
      }
      __syncwarp();
    } else if (warp == 9) {
      // -------------------------------------------------------------------- MMA
      if (lane == 0) {
        const uint32_t idesc_pv = make_idesc_bf16(128, 128, true);
        const uint32_t idesc_qk_full = make_idesc_bf16(128, 128, false);
        const uint32_t dq = desc_lo(base + S::kOffQ, 16);
        const uint32_t dk0 = desc_lo(base + S::kOffK, 16);
        const uint32_t dv0 = desc_lo(base + S::kOffV, kChunkBytes);
        constexpr uint32_t kStageStep = kTileBytes >> 4;  // (all offsets stay inside the address field)
        // S(sb) = Q K(kst)^T over n_rows keys
        auto qk = [&](int kst, int n_rows, uint32_t sb) {
          const uint32_t idesc =
              n_rows == kTileN ? idesc_qk_full : make_idesc_bf16(128, (n_rows + 15) & ~15, false);
          const uint32_t b = dk0 + kst * kStageStep;
          const uint32_t d = tmem + sb * 128;
#pragma unroll
          for (int s = 0; s < kD / 16; ++s) {
            const uint32_t off = ((s >> 2) * kChunkBytes + (s & 3) * 32) >> 4;
            mma_ss(d, dq + off, b + off, idesc, s > 0 ? 1u : 0u);
          }
        };
        // O_h (+)= P_h V[64h .. 64h + 16 ksteps)
        auto pv_half = [&](int vst, uint32_t sb, int h, int ksteps, bool acc) {
          const uint32_t b = dv0 + vst * kStageStep;
          const uint32_t d = tmem + 256 + h * 128;
          const uint32_t p = tmem + sb * 128 + h * kHalfN;
          if (ksteps == 4) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
              mma_ts(d, p + s * 8, b + (4 * h + s) * (2048 >> 4), idesc_pv, (acc || s > 0) ? 1u : 0u);
          } else {
            for (int s = 0; s < ksteps; ++s)
              mma_ts(d, p + s * 8, b + (4 * h + s) * (2048 >> 4), idesc_pv, (acc || s > 0) ? 1u : 0u);
          }
        };
        // pair: row tile i against KV tiles: S(i) = Q(i) K^T, O(i) (+)= P(i) V
        auto qk_tile = [&](int i, int kst, int n_rows) {
          const uint32_t idesc = n_rows == kTileN ? idesc_qk_full : make_idesc_bf16(128, (n_rows + 15) & ~15, false);
          const uint32_t x = dq + i * kStageStep, b = dk0 + kst * kStageStep;
#pragma unroll
          for (int s = 0; s < kD / 16; ++s) {
            const uint32_t off = ((s >> 2) * kChunkBytes + (s & 3) * 32) >> 4;
            mma_ss(tmem + i * 128, x + off, b + off, idesc, s > 0 ? 1u : 0u);
          }
        };
        auto pv_tile = [&](int i, int vst, int ksteps, bool acc) {
          const uint32_t b = dv0 + vst * kStageStep;
          const uint32_t d = tmem + 256 + i * 128, p = tmem + i * 128;
          if (ksteps == 8) {
#pragma unroll
            for (int s = 0; s < 8; ++s) mma_ts(d, p + s * 8, b + s * (2048 >> 4), idesc_pv, (acc || s > 0) ? 1u : 0u);
          } else {
            for (int s = 0; s < ksteps; ++s) mma_ts(d, p + s * 8, b + s * (2048 >> 4), idesc_pv, (acc || s > 0) ? 1u : 0u);
          }
        };
        uint32_t q_it = 0, k_it = 0, v_it = 0;
        uint32_t p_it[2] = {0, 0};
        bool ok = true;
        for (int u = blockIdx.x; kPair && u < total_units && ok; u += gridDim.x) {
          const Unit t = decode_unit(u, a, false);
          if (!t.valid || t.nkv == 0) continue;
          const int nt = t.rows > a.tile_rows ? 2 : 1;
          ok = mbar_wait(bar(S::BAR_QFULL), q_it & 1, abort_flag);
          if (!ok) break;
          ++q_it;
          {
            const int kst = k_it % kStagesK;
            ok = mbar_wait(bar(S::BAR_KFULL + kst), (k_it / kStagesK) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const int valid = kv_tile(t, 0).valid;
            for (int i = 0; i < nt; ++i) {
              qk_tile(i, kst, valid);
              umma_commit(bar(S::BAR_SFULL + i));
            }
            umma_commit(bar(S::BAR_KEMPTY + kst));
            ++k_it;
            if (t.nkv == 1) umma_commit(bar(S::BAR_QEMPTY));
          }
          for (int j = 0; j < t.nkv && ok; ++j) {
            const int ks = (kv_tile(t, j).valid + 15) >> 4;  // 1..8 K-steps
            const int vst = v_it % kStagesV, kst = k_it % kStagesK;
            ok = mbar_wait(bar(S::BAR_VFULL + vst), (v_it / kStagesV) & 1, abort_flag);
            if (!ok) break;
            const bool more = j + 1 < t.nkv;
            const int next = more ? kv_tile(t, j + 1).valid : 0;
            for (int i = 0; i < nt && ok; ++i) {
              ok = mbar_wait(bar(S::BAR_PFULL + i), p_it[i] & 1, abort_flag);
              if (!ok) break;
              ++p_it[i];
              tc_fence_after();
              pv_tile(i, vst, ks, j > 0);
              if (more) {
                if (i == 0) {
                  ok = mbar_wait(bar(S::BAR_KFULL + kst), (k_it / kStagesK) & 1, abort_flag);
                  if (!ok) break;
                  tc_fence_after();
                }
                qk_tile(i, kst, next);
                umma_commit(bar(S::BAR_SFULL + i));
              } else {
                umma_commit(bar(S::BAR_OFULL + i));
              }
            }
            if (!ok) break;
            umma_commit(bar(S::BAR_VEMPTY + vst));
            ++v_it;
            if (more) {
              umma_commit(bar(S::BAR_KEMPTY + kst));
              ++k_it;
              if (j + 2 == t.nkv) umma_commit(bar(S::BAR_QEMPTY));  // last QK issued
            }
          }
        }
        uint32_t g = 0;  // KV tiles whose PVs were issued (all units), = S tile index
        for (int u = blockIdx.x; !kPair && u < total_units && ok; u += gridDim.x) {
          const Unit t = decode_unit(u, a, false);
          if (!t.valid || t.nkv == 0) continue;
          ok = mbar_wait(bar(S::BAR_QFULL), q_it & 1, abort_flag);
          if (!ok) break;
          ++q_it;
          const int npro = t.nkv < 2 ? t.nkv : 2;
          for (int j = 0; j < npro && ok; ++j) {
            const KvTile kt = kv_tile(t, j);
            const int kst = k_it % kStagesK;
            ok = mbar_wait(bar(S::BAR_KFULL + kst), (k_it / kStagesK) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            qk(kst, kt.valid, (g + j) & 1);
            umma_commit(bar(S::BAR_SFULL + ((g + j) & 1)));
            umma_commit(bar(S::BAR_KEMPTY + kst));
            ++k_it;
          }
          if (!ok) break;
          if (t.nkv <= 2) umma_commit(bar(S::BAR_QEMPTY));  // every QK of the unit issued
          bool b_started = false;  // O_b written in this unit
          for (int j = 0; j < t.nkv && ok; ++j, ++g) {
            const KvTile kt = kv_tile(t, j);
            const uint32_t sb = g & 1;
            const int vst = v_it % kStagesV;
            ok = mbar_wait(bar(S::BAR_VFULL + vst), (v_it / kStagesV) & 1, abort_flag);
            if (!ok) break;
            ok = mbar_wait(bar(S::BAR_PFULL + sb), (g >> 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const int ks = (kt.valid + 15) >> 4;  // 1..8 K-steps
            pv_half(vst, sb, 0, ks < 4 ? ks : 4, j > 0);
            if (ks > 4) {
              pv_half(vst, sb, 1, ks - 4, b_started);
              b_started = true;
            }
            umma_commit(bar(S::BAR_VEMPTY + vst));
            umma_commit(bar(S::BAR_OREADY));
            ++v_it;
            if (j + 2 < t.nkv) {
              const KvTile kn = kv_tile(t, j + 2);
              const int kst = k_it % kStagesK;
              ok = mbar_wait(bar(S::BAR_KFULL + kst), (k_it / kStagesK) & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
              qk(kst, kn.valid, sb);  // tile g + 2 uses the same S buffer
              umma_commit(bar(S::BAR_SFULL + sb));
              umma_commit(bar(S::BAR_KEMPTY + kst));
              ++k_it;
              if (j + 3 == t.nkv) umma_commit(bar(S::BAR_QEMPTY));  // last QK issued
            }
          }
          if (!ok) break;
          umma_commit(bar(S::BAR_OFULL));
        }
        // Make sure every issued MMA has finished before TMEM is released.
        umma_commit(bar(S::BAR_DRAIN));
        mbar_wait_drain(bar(S::BAR_DRAIN), 0, 100000000ull);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------- loader of Q
      // The box brings all heads of the KV head's group for a tile's chunk rows: packed order.
      const uint64_t pol = policy_evict_first();
      const uint32_t half_bytes = a.tile_rows * 128;
      uint32_t q_it = 0;  // units whose Q was loaded
      bool ok = true;
      for (int u = blockIdx.x; u < total_units && ok; u += gridDim.x) {
        const Unit t = decode_unit(u, a, false);
        if (!t.valid || t.nkv == 0) continue;
        if (q_it > 0) ok = mbar_wait_warp(bar(S::BAR_QEMPTY), (q_it - 1) & 1, abort_flag);
        if (!ok) break;
        ++q_it;
        if (lane == 0) {
          const int nt = t.rows > a.tile_rows ? 2 : 1;
          mbar_arrive_expect_tx(bar(S::BAR_QFULL), nt * 2 * half_bytes);
          for (int i = 0; i < nt; ++i) {
            const uint32_t dst = base + S::kOffQ + i * kTileBytes;
            const int row = (int)t.sq.q_begin + (t.row0 + i * a.tile_rows) / a.group;
            tma_load_3d(dst, &tmQ, bar(S::BAR_QFULL), 0, t.hkv * a.group, row, pol);
            tma_load_3d(dst + kChunkBytes, &tmQ, bar(S::BAR_QFULL), 64, t.hkv * a.group, row, pol);
          }
        }
        __syncwarp();
      }
      if (lane == 0 && *abort_flag && q_it > 0) mbar_wait_drain(bar(S::BAR_QFULL), (q_it - 1) & 1, 100000000ull);
      __syncwarp();
    }
  } else if (kQuant && warp >= 12) {
    set_max_registers<S::kRegsOther, false>();
    // ------------------------------------------------------------- expansion
    // Warps 12-15 fill the K ring, warps 16-19 the V ring.
    const bool is_k = warp < 16;
    const int lead = is_k ? 12 : 16;  // this warpgroup's first warp
    const int tid = threadIdx.x - lead * 32;
    const int nst = is_k ? kStagesK : kStagesV;
    const int bfull = is_k ? S::BAR_KFULL : S::BAR_VFULL, bempty = is_k ? S::BAR_KEMPTY : S::BAR_VEMPTY;
    const int rfull = S::BAR_RFULL + (is_k ? 0 : kRaw), rempty = S::BAR_REMPTY + (is_k ? 0 : kRaw);
    const uint32_t ring = is_k ? S::kOffK : S::kOffV;
    uint32_t n = 0;     // ring positions filled; every position is filled by this warpgroup, in order, so each
                        // wait below is for the phase right before (a wait by parity cannot tell phases two apart)
    uint32_t raw_it = 0, land = 0;
    bool ok = true;
    // expands the raw tile `raw_it` into ring position n
    auto expand = [&]() -> bool {
      const int st = n % nst, rs = raw_it % kRaw;
      if (!mbar_wait_warp(bar(rfull + rs), (raw_it / kRaw) & 1, abort_flag)) return false;
      if (n >= (uint32_t)nst && !mbar_wait_warp(bar(bempty + st), (n / nst - 1) & 1, abort_flag)) return false;
      const int rb = (is_k ? 0 : kRaw) + rs;
      const uint8_t* src = smem + S::kOffRaw + rb * kChunkBytes;
      const uint8_t* ex = smem + S::kOffExp + rb * 128;
      uint8_t* dst = smem + ring + st * kTileBytes;
      // This thread's 16 codes are unit `un` of rows r0 + 16 i; their bf16 form is 16-byte units
      // 2 un, 2 un + 1 of the row (half un / 4 of the tile). Neighbouring rows change places for the
      // upper units: eight lanes then read eight different units and write eight different banks.
      const int un = tid & 7;
      const int r0 = (tid >> 3) ^ (un >> 2);
      const int x = (2 * un) & 7;
      uint8_t* d0 = dst + (un >> 2) * kChunkBytes + r0 * 128 + ((x ^ (r0 & 7)) << 4);
      uint8_t* d1 = dst + (un >> 2) * kChunkBytes + r0 * 128 + (((x + 1) ^ (r0 & 7)) << 4);
      auto put = [&](int i, const uint32_t (&w)[8]) {
        *reinterpret_cast<uint4*>(d0 + i * 2048) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4*>(d1 + i * 2048) = make_uint4(w[4], w[5], w[6], w[7]);
      };
      src += r0 * kD + un * 16;
#pragma unroll 1
      for (int i0 = 0; i0 < 8; i0 += 2) {  // (unrolled, the loop costs every role instruction fetches)
        uint4 c[2];
        uint32_t e[2];
        bool big = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          c[i] = *reinterpret_cast<const uint4*>(src + (i0 + i) * 16 * kD);
          e[i] = ex[(i0 + i) * 16 + r0];
          big |= exp_is_big<kFmt>(e[i]);
        }
        if (!__any_sync(0xffffffffu, big)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t w[8];
            expand16<kFmt>(c[i], code_scale<kFmt>(e[i]), w);
            put(i0 + i, w);
          }
        } else {
#pragma unroll 1
          for (int i = i0; i < i0 + 2; ++i) {
            uint32_t w[8];
            dequantise16<kFmt>(*reinterpret_cast<const uint4*>(src + i * 16 * kD), ex[i * 16 + r0], w);
            put(i, w);
          }
        }
      }
      fence_proxy_async_smem();  // generic-proxy writes -> tensor-core reads
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(bfull + st));
        mbar_arrive(bar(rempty + rs));
      }
      return true;
    };
    // loads a fresh tile into ring position n by TMA: the first warp issues it, the others arrive
    auto direct = [&](int hkv, const KvTile& kt) -> bool {
      const int st = n % nst;
      if (n >= (uint32_t)nst && !mbar_wait_warp(bar(bempty + st), (n / nst - 1) & 1, abort_flag)) return false;
      const uint32_t full = bar(bfull + st);
      if (warp != lead) {
        if (lane == 0) mbar_arrive(full);
        return true;
      }
      const bool clear = !is_k && (kt.valid & 15) != 0;
      const uint32_t fb = clear ? bar(S::BAR_VLAND) : full;
      const uint32_t dst = ring + st * kTileBytes;
      if (lane == 0) {
        const uint64_t pol = policy_evict_last();
        const CUtensorMap* mp = is_k ? &tmK : &tmV;
        mbar_arrive_expect_tx(fb, kTileBytes);
        tma_load_3d(base + dst, mp, fb, 0, hkv, (int)kt.row, pol);
        tma_load_3d(base + dst + kChunkBytes, mp, fb, 64, hkv, (int)kt.row, pol);
      }
      if (clear) {
        if (!mbar_wait_warp(fb, land & 1, abort_flag)) return false;
        ++land;
        clear_tail(smem + dst, kt.valid, lane);
        if (lane == 0) mbar_arrive(full);
      }
      return true;
    };
    for (int u = blockIdx.x; u < total_units && ok; u += gridDim.x) {
      const Unit t = decode_unit(u, a, false);
      if (!t.valid || t.nkv == 0) continue;
      for (int j = 0; j < t.nkv && ok; ++j, ++n) {
        if (t.t0 + j < t.sp.cached) {
          ok = expand();
          ++raw_it;
        } else {
          ok = direct(t.hkv, kv_tile(t, j));
        }
      }
    }
    if (warp == lead && lane == 0 && *abort_flag) {
      // Drain: fresh tiles' copies that may still be in flight.
      for (uint32_t i = (n > (uint32_t)nst ? n - nst : 0); i < n; ++i)
        mbar_wait_drain(bar(bfull + i % nst), (i / nst) & 1, 100000000ull);
      if (!is_k) mbar_wait_drain(bar(S::BAR_VLAND), land & 1, 100000000ull);
    }
    __syncwarp();
  } else {
    set_max_registers<S::kRegsSoftmax, true>();
    // ---------------------------------------------------------------- softmax
    if constexpr (kPair) {
      softmax_pair<S>(a, tmem, bar0, abort_flag);
    } else {
      const int wg = warp >> 2;           // 0: keys 0-63 of a tile, 1: keys 64-127
      const int wq = warp & 3;
      const int row_in_tile = threadIdx.x & 127;
      const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
      const uint32_t tOwn = tmem + lane_base + 256 + wg * 128;  // this warpgroup's accumulator
      const uint32_t tOa = tmem + lane_base + 256;
      const uint32_t tOb = tmem + lane_base + 384;
      float2* xch = reinterpret_cast<float2*>(smem + S::kOffXch);
      const float sl2 = a.scale_log2;
      uint32_t g = 0, o_it = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < total_units && ok; u += gridDim.x) {
        const Unit t = decode_unit(u, a, false);
        if (!t.valid) continue;
        const int qr = (t.row0 + row_in_tile) / a.group;  // row of the chunk
        const int seen = (int)(a.causal ? min(t.L, max((int64_t)0, t.L - t.sq.Lq + qr + 1)) : t.L);
        // A warp whose 32 rows lie past the unit's last one only keeps the barriers going (its rows
        // of P hold anything: rows of a product do not mix).
        const bool idle = wq * 32 >= t.rows;
        const bool row_ok = row_in_tile < t.rows;
        float m = -INFINITY;  // running max (log2 units), -inf until a visible key
        float l = 0.f;
        for (int j = 0; j < t.nkv; ++j, ++g) {
          const KvTile kt = kv_tile(t, j);
          const uint32_t sb = g & 1;
          ok = mbar_wait_warp(bar(S::BAR_SFULL + sb), (g >> 1) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t tS = tmem + lane_base + sb * 128 + wg * kHalfN;
          if (!idle && kt.valid > wg * kHalfN) {
            uint32_t s[2][32];
            tmem_ld32(tS, s[0]);
            tmem_ld32(tS + 32, s[1]);
            tmem_wait_ld();
            const int nv = min(kt.valid, seen - kt.pos) - wg * kHalfN;  // this row's visible columns
            if (__any_sync(0xffffffffu, nv < kHalfN)) {
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (c * 32 + e >= nv) s[c][e] = __float_as_uint(-INFINITY);
            }
            float mq[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = __uint_as_float(s[c][0]);
#pragma unroll
              for (int e = 1; e < 31; e += 2)
                x = max3f(x, __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
              mq[c] = fmaxf(x, __uint_as_float(s[c][31]));
            }
            const float mxs = fmaxf(mq[0], mq[1]) * sl2;
            // Lazy rescaling: a stale maximum stays while the new one exceeds it
            // by at most 8 (log2 units), so P stays <= 256. A row's first visible
            // key sets it (its accumulator holds zeros or is not written yet).
            const bool first = m == -INFINITY;
            const bool need = row_ok && !first && mxs > m + 8.f;  // (rows past the tile's last are another sequence's)
            if (first) m = mxs;
            if (__any_sync(0xffffffffu, need)) {
              const float mn = first ? m : fmaxf(m, mxs);
              const float alpha = first ? 1.f : ex2_approx(m - mn);
              m = mn;
              l *= alpha;
              // The accumulator must hold every PV up to tile g-1: PV(g-2)
              // completed before S(g) did, so one more completion of OREADY
              // (parity of tile g-1) is all there is to wait for.
              ok = mbar_wait_warp(bar(S::BAR_OREADY), (g - 1) & 1, abort_flag);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld32(tOwn + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st32(tOwn + c * 32, o);
              }
            }
            l += exp_store<2>(s, sl2, m == -INFINITY ? 0.f : m, tS);  // hidden columns give exact zeros
            tmem_wait_st();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(S::BAR_PFULL + sb));
        }
        if (!ok) break;
        // Epilogue: merge the two halves, then O / l -> bf16 (the row's only split)
        // or O, (m, l) -> fp32 partials. Warpgroup w writes output columns [64w, 64w + 64).
        const bool alone = t.sp.total <= a.split_chunks;
        const int h = t.hkv * a.group + (t.row0 + row_in_tile) - qr * a.group;
        __nv_bfloat16* orow = a.o + (t.sq.q_begin + qr) * a.o_stride + (int64_t)h * kD + wg * kHalfN;
        const int64_t prow = ((int64_t)t.item * a.splits + t.split) * kTileM + row_in_tile;
        if (t.nkv > 0) {
          ok = mbar_wait_warp(bar(S::BAR_OFULL), o_it & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          // O = ca * O_a + cb * O_b. A half without a visible key (m = -inf) counts nothing: factor
          // -1, its accumulator is not read (O_b may not have been written at all). Where both
          // have none above -inf, but the row sees keys, the factors come out as NaN.
          float ca, cb;
          if (wg == 1) {
            xch[row_in_tile] = make_float2(m, l);
            mbar_arrive(bar(S::BAR_XML));
            ok = mbar_wait_warp(bar(S::BAR_XF), o_it & 1, abort_flag);
            if (!ok) break;
            const float2 f = xch[row_in_tile];
            ca = f.x;
            cb = f.y;
          } else {
            ok = mbar_wait_warp(bar(S::BAR_XML), o_it & 1, abort_flag);
            if (!ok) break;
            const float2 o1 = xch[row_in_tile];
            const float mm = fmaxf(m, o1.x);
            const float fa = m == -INFINITY ? 0.f : ex2_approx(m - mm);
            const float fb = o1.x == -INFINITY ? 0.f : ex2_approx(o1.x - mm);
            const float sum = l * fa + o1.y * fb;
            const float inv = !alone ? 1.f : seen <= 0 ? 0.f : 1.f / sum;  // no visible key: zero row
            const bool none = !alone || seen <= 0 || mm > -INFINITY;
            ca = none && m == -INFINITY ? -1.f : fa * inv;
            cb = none && o1.x == -INFINITY ? -1.f : fb * inv;
            xch[row_in_tile] = make_float2(ca, cb);
            mbar_arrive(bar(S::BAR_XF));
            if (!alone && row_ok) a.part_ml[prow] = make_float2(mm, sum);
          }
          ++o_it;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            if (idle) break;
            uint32_t oa[32], ob[32];
            tmem_ld32(tOa + wg * kHalfN + c * 32, oa);
            tmem_ld32(tOb + wg * kHalfN + c * 32, ob);
            tmem_wait_ld();
            if (row_ok) {
              float v[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                v[e] = ca == -1.f ? 0.f : __uint_as_float(oa[e]) * ca;
                if (cb != -1.f) v[e] = fmaf(__uint_as_float(ob[e]), cb, v[e]);
              }
              if (alone) {
                uint4* dst = reinterpret_cast<uint4*>(orow + c * 32);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  dst[q] = make_uint4(pack_bf16x2(v[8 * q + 0], v[8 * q + 1]), pack_bf16x2(v[8 * q + 2], v[8 * q + 3]),
                                      pack_bf16x2(v[8 * q + 4], v[8 * q + 5]), pack_bf16x2(v[8 * q + 6], v[8 * q + 7]));
              } else {
                float4* dst = reinterpret_cast<float4*>(a.part_o + prow * kD + wg * kHalfN + c * 32);
#pragma unroll
                for (int q = 0; q < 8; ++q) dst[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
              }
            }
          }
          // O is read out; the next unit's first PV may overwrite it once every
          // softmax warp arrives on its first P barrier (program order + fence).
          tc_fence_before();
        } else if (row_ok) {
          // No keys at all: the output row is zero.
          uint4* dst = reinterpret_cast<uint4*>(orow);
          for (int v = 0; v < kHalfN / 8; ++v) dst[v] = make_uint4(0, 0, 0, 0);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) set_error(a.err, kDevWaitTimeout);
}

template <int kFmt, bool kPair>
cudaError_t launch(const ChunkMaps& m, const ChunkArgs& a, int num_sms, cudaStream_t stream) {
  using S = Layout<kFmt, kPair>;
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(attn_chunk_mma_kernel<kFmt, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)S::kSmemBytes);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return launch_pdl(attn_chunk_mma_kernel<kFmt, kPair>, dim3(std::min(a.total_units, num_sms)), dim3(S::kThreads),
                    S::kSmemBytes, stream, m.q, m.k, m.v, m.kc, m.vc, m.kg, m.vg, a);
}

}  // namespace chunk128

cudaError_t launch_attn_chunk_mma(const ChunkMaps& maps, const ChunkArgs& a, int format, int num_sms,
                                  cudaStream_t stream) {
  const bool pair = a.unit_rows > a.tile_rows;
  switch (format) {
    case kFmtBf16:
      return pair ? chunk128::launch<kFmtBf16, true>(maps, a, num_sms, stream)
                  : chunk128::launch<kFmtBf16, false>(maps, a, num_sms, stream);
    case kFmtE4m3:
      return pair ? chunk128::launch<kFmtE4m3, true>(maps, a, num_sms, stream)
                  : chunk128::launch<kFmtE4m3, false>(maps, a, num_sms, stream);
    default:
      return pair ? chunk128::launch<kFmtInt8, true>(maps, a, num_sms, stream)
                  : chunk128::launch<kFmtInt8, false>(maps, a, num_sms, stream);
  }
}

}  // namespace dllm
