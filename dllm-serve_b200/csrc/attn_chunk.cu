// Attention of a chunk of new tokens over a paged KV cache, for launches bound
// by the cache's bytes: few query rows per KV head, long contexts (sm_100a).
//
// The keys of sequence b are [its cached rows, found by block table or slot
// list ; its fresh rows]. Query row i of the chunk sees the first
// L - Lq + i + 1 of the L keys (causal) or all of them. Softmax is online: a
// running maximum m and sum l per row, O rescaled when m grows; with a
// quantised cache the scores are multiplied by the key's 2^e after the product
// and the probabilities by the value's 2^e before theirs, so the matrix
// products run on the codes themselves, which bf16 holds exactly.
//
// A CTA takes one tile of packed rows (row r of the chunk for query head g of
// the KV head's group is packed row r * group + g) and one split of the keys;
// its four warps take the split's key chunks in turn, each with a private
// ring of stages filled by cp.async, so the main loop has no CTA barrier. The
// warps' partial results are merged in shared memory in a fixed order; splits
// are merged by a second kernel, also in a fixed order. Products are
// mma.sync m16n8k16: at one to 32 rows per KV head a launch reads
// 256 (K) + 256 (V) bytes per bf16 key for at most 32 x 512 operations, below
// what this instruction sustains, and its operands go straight from
// shared memory to registers, where codes are expanded.
//
// Operand layout: the reduction order over head dimensions and over keys is
// free as long as both operands agree, and so is the order of output columns.
// Thread (g, t) of a warp (g = lane / 4, t = lane % 4) takes dimensions
// 16t .. 16t+15 and 64+16t .. 64+16t+15 of key g for the scores (two 16-byte
// reads of codes), and dimensions 16g .. 16g+15 of keys 2t, 2t+1, 2t+8, 2t+9
// for the outputs, whose column n of tile j is then dimension 16n + j.
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "kvquant.cuh"
#include "attn_chunk.h"

namespace dllm {
namespace chunk {

namespace {

constexpr int kD = 128;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 3;
constexpr uint32_t kStageBytes = 8192;  // K half then V half
constexpr int kFreshKeys = 16;          // keys of a bf16 chunk

template <int kFmt>
constexpr int chunk_keys() { return kFmt == kFmtBf16 ? 16 : 32; }

constexpr uint32_t kOffStages = 0;
constexpr uint32_t kOffScales = kOffStages + kWarps * kStages * kStageBytes;  // float2 per (warp, stage, key)
constexpr uint32_t kOffQ = kOffScales + kWarps * kStages * 32 * 8;

template <int kMT>
constexpr uint32_t smem_bytes() { return kOffQ + kMT * 16 * kD * 2; }
// the merge buffers (per warp: rows x 128 floats, then rows float2) reuse the stages
static_assert(kWarps * (32 * kD * 4 + 32 * 8) <= kWarps * kStages * kStageBytes, "merge buffers exceed the stages");

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

// Four codes -> two words of bf16 pairs, unscaled (exact).
template <int kFmt>
DLLM_DEVICE void codes_to_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  float y[4];
  decode4<kFmt>(w, 1.f, y);
  lo = pack_bf16x2(y[0], y[1]);
  hi = pack_bf16x2(y[2], y[3]);
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

// Sizes of one sequence, every value checked against the buffers it indexes.
struct Seq {
  int64_t q_begin, s_begin, k_begin;
  int Lq, nc, nk;
};

DLLM_DEVICE Seq load_seq(const ChunkArgs& a, int b, bool report) {
  Seq s;
  bool bad = false;
  auto range = [&](const int32_t* cu, int64_t total, int64_t& begin, int& n, int most) {
    const int64_t lo = cu[b], hi = cu[b + 1];
    begin = min(max(lo, (int64_t)0), total);
    const int64_t end = min(max(hi, begin), total);
    n = (int)min(end - begin, (int64_t)most);
    bad |= lo != begin || hi != begin + n;
  };
  range(a.cu_q, a.total_q, s.q_begin, s.Lq, a.max_q);
  s.k_begin = 0;
  s.nk = 0;
  if (a.cu_k != nullptr) range(a.cu_k, a.total_k, s.k_begin, s.nk, a.max_fresh);
  s.s_begin = 0;
  if (a.tables != nullptr) {
    const int c = a.ctx[b];
    s.nc = min(max(c, 0), a.max_context);
    bad |= c != s.nc;
  } else if (a.slots != nullptr) {
    range(a.cu_s, a.total_slots, s.s_begin, s.nc, a.max_context);
  } else {
    s.nc = 0;
  }
  if (bad && report) set_error(a.err, kDevBadSequence);
  return s;
}

// Key chunks of a row tile: the cached rows in chunks of KB keys, then the
// fresh rows in chunks of kFreshKeys, both cut at the last key any row of the
// tile sees.
struct Span {
  int nc, nk;      // keys to walk in each segment
  int cached;      // chunks of the cached segment
  int total;       // all chunks
};

template <int kFmt>
DLLM_DEVICE Span tile_span(const ChunkArgs& a, const Seq& s, int last_row) {
  constexpr int KB = chunk_keys<kFmt>();
  int64_t seen = (int64_t)s.nc + s.nk;
  if (a.causal) seen = min(seen, max((int64_t)0, seen - s.Lq + last_row + 1));
  Span r;
  r.nc = (int)min(seen, (int64_t)s.nc);
  r.nk = (int)(seen - r.nc);
  r.cached = (r.nc + KB - 1) / KB;
  r.total = r.cached + (r.nk + kFreshKeys - 1) / kFreshKeys;
  return r;
}

// Products, softmax and products of one chunk of KB keys in shared memory.
// lim[r]: keys this thread's row r (of 2 * MT) sees, counted from the chunk's
// first key; `whole`: every row sees all KB keys.
template <int kFmt, int kMT>
DLLM_DEVICE void chunk_step(uint32_t ks, uint32_t vs, uint32_t scales, uint32_t qs, const uint32_t (&qf)[8][4],
                            int lane, float sl2, bool whole, const int (&lim)[2 * kMT], float (&m)[2 * kMT],
                            float (&l)[2 * kMT], float (&o)[kMT][16][4]) {
  constexpr int KB = chunk_keys<kFmt>();
  constexpr int NT = KB / 8;
  constexpr uint32_t kRow = kFmt == kFmtBf16 ? 256 : 128;  // bytes of a key's row
  const int g = lane >> 2, t = lane & 3;
  float s[kMT][NT][4];
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.f;
  // scores: half h covers dimensions 64h + 16t .. + 15 of this thread
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t qa[kMT][4][4];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      if constexpr (kMT == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) qa[mt][i][e] = qf[4 * h + i][e];
      } else {
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int row = mt * 16 + rr * 8 + g;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint4 w = lds128(qs + row * 256 + (((8 * h + 2 * t + c) ^ (row & 1)) << 4));
            qa[mt][2 * c][rr] = w.x, qa[mt][2 * c][2 + rr] = w.y;
            qa[mt][2 * c + 1][rr] = w.z, qa[mt][2 * c + 1][2 + rr] = w.w;
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint32_t key = 8 * n + g;
      uint32_t kb[8];
      if constexpr (kFmt == kFmtBf16) {
        const uint4 x = lds128(ks + key * kRow + (k_unit<kFmt>(8 * h + 2 * t, key) << 4));
        const uint4 y = lds128(ks + key * kRow + (k_unit<kFmt>(8 * h + 2 * t + 1, key) << 4));
        kb[0] = x.x, kb[1] = x.y, kb[2] = x.z, kb[3] = x.w;
        kb[4] = y.x, kb[5] = y.y, kb[6] = y.z, kb[7] = y.w;
      } else {
        const uint4 x = lds128(ks + key * kRow + (k_unit<kFmt>(4 * h + t, key) << 4));
        codes_to_bf16<kFmt>(x.x, kb[0], kb[1]);
        codes_to_bf16<kFmt>(x.y, kb[2], kb[3]);
        codes_to_bf16<kFmt>(x.z, kb[4], kb[5]);
        codes_to_bf16<kFmt>(x.w, kb[6], kb[7]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
          mma16816(s[mt][n], qa[mt][i][0], qa[mt][i][1], qa[mt][i][2], qa[mt][i][3], kb[2 * i], kb[2 * i + 1]);
    }
  }
  // scores in log2 units, masked
  float vsc[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float ks0 = sl2, ks1 = sl2;
    if constexpr (kFmt != kFmtBf16) {
      const uint4 w = lds128(scales + (8 * n + 2 * t) * 8);  // (K, V) scales of two keys
      ks0 *= __uint_as_float(w.x), ks1 *= __uint_as_float(w.z);
      vsc[n][0] = __uint_as_float(w.y), vsc[n][1] = __uint_as_float(w.w);
    }
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
      s[mt][n][0] *= ks0, s[mt][n][1] *= ks1, s[mt][n][2] *= ks0, s[mt][n][3] *= ks1;
      if (!whole) {
        const int c = 8 * n + 2 * t;
        if (c >= lim[2 * mt]) s[mt][n][0] = -INFINITY;
        if (c + 1 >= lim[2 * mt]) s[mt][n][1] = -INFINITY;
        if (c >= lim[2 * mt + 1]) s[mt][n][2] = -INFINITY;
        if (c + 1 >= lim[2 * mt + 1]) s[mt][n][3] = -INFINITY;
      }
    }
  }
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) mx = max3f(mx, s[mt][n][2 * r], s[mt][n][2 * r + 1]);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int i = 2 * mt + r;
      const float mn = fmaxf(m[i], mx);
      const float base = mn == -INFINITY ? 0.f : mn;  // a row that has seen no key yet
      const float alpha = ex2_approx(m[i] - base);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float p0 = ex2_approx(s[mt][n][2 * r] - base), p1 = ex2_approx(s[mt][n][2 * r + 1] - base);
        sum += p0 + p1;
        s[mt][n][2 * r] = p0;
        s[mt][n][2 * r + 1] = p1;
      }
      l[i] = l[i] * alpha + sum;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        o[mt][j][2 * r] *= alpha;
        o[mt][j][2 * r + 1] *= alpha;
      }
    }
  }
  // outputs: probabilities are rounded to bf16 (at most 2^-8 of their value), after the value's scale
#pragma unroll
  for (int u = 0; u < NT / 2; ++u) {
    uint32_t pa[kMT][4];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* x = s[mt][2 * u + e];
        if constexpr (kFmt != kFmtBf16) {
          x[0] *= vsc[2 * u + e][0], x[1] *= vsc[2 * u + e][1];
          x[2] *= vsc[2 * u + e][0], x[3] *= vsc[2 * u + e][1];
        }
        pa[mt][2 * e] = pack_bf16x2(x[0], x[1]);
        pa[mt][2 * e + 1] = pack_bf16x2(x[2], x[3]);
      }
    const uint32_t k0 = 16 * u + 2 * t;
#pragma unroll
    for (int c = 0; c < 2; ++c) {  // eight output columns of this thread at a time
      uint32_t vb[8][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t ka = k0 + 8 * e, kb = ka + 1;
        if constexpr (kFmt == kFmtBf16) {
          const uint4 x = lds128(vs + ka * kRow + (v_unit<kFmt>(2 * g + c, ka) << 4));
          const uint4 y = lds128(vs + kb * kRow + (v_unit<kFmt>(2 * g + c, kb) << 4));
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vb[2 * i][e] = __byte_perm(xs[i], ys[i], 0x5410);
            vb[2 * i + 1][e] = __byte_perm(xs[i], ys[i], 0x7632);
          }
        } else {
          uint2 x, y;
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                       : "=r"(x.x), "=r"(x.y)
                       : "r"(vs + ka * kRow + (v_unit<kFmt>(g, ka) << 4) + 8 * c));
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                       : "=r"(y.x), "=r"(y.y)
                       : "r"(vs + kb * kRow + (v_unit<kFmt>(g, kb) << 4) + 8 * c));
          codes_to_bf16<kFmt>(__byte_perm(x.x, y.x, 0x5140), vb[0][e], vb[1][e]);
          codes_to_bf16<kFmt>(__byte_perm(x.x, y.x, 0x7362), vb[2][e], vb[3][e]);
          codes_to_bf16<kFmt>(__byte_perm(x.y, y.y, 0x5140), vb[4][e], vb[5][e]);
          codes_to_bf16<kFmt>(__byte_perm(x.y, y.y, 0x7362), vb[6][e], vb[7][e]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
          mma16816(o[mt][8 * c + j], pa[mt][0], pa[mt][1], pa[mt][2], pa[mt][3], vb[j][0], vb[j][1]);
    }
  }
}

template <int kFmt, int kMT>
__global__ void __launch_bounds__(kThreads, 2) attn_chunk_kernel(const __grid_constant__ ChunkArgs a) {
  constexpr int KB = chunk_keys<kFmt>();
  constexpr int kRows = 16 * kMT;
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
  const Span sp = tile_span<kFmt>(a, sq, (row0 + min(rows, kRows) - 1) / a.group);
  const int c_begin = split * a.split_chunks;
  const int c_end = min(sp.total, c_begin + a.split_chunks);
  if (split > 0 && c_begin >= c_end) return;  // this split has no keys (split 0 writes empty rows)

  // Q rows, packed and swizzled (zero past the tile's rows)
  for (int i = threadIdx.x; i < kRows * 16; i += kThreads) {
    const int p = i >> 4, u = i & 15;
    const bool live = p < rows;
    const int r = (row0 + p) / a.group, h = hkv * a.group + (row0 + p) - r * a.group;
    const __nv_bfloat16* src = a.q + (live ? (sq.q_begin + r) * a.q_stride + (int64_t)h * kD + u * 8 : 0);
    cp_async16(base + kOffQ + p * 256 + ((u ^ (p & 1)) << 4), src, live);
  }
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();
  uint32_t qf[8][4];
  if constexpr (kMT == 1) {
#pragma unroll
    for (int rr = 0; rr < 2; ++rr)
#pragma unroll
      for (int hc = 0; hc < 4; ++hc) {
        const int row = rr * 8 + g, unit = 8 * (hc >> 1) + 2 * t + (hc & 1);
        const uint4 w = lds128(base + kOffQ + row * 256 + ((unit ^ (row & 1)) << 4));
        qf[2 * hc][rr] = w.x, qf[2 * hc][2 + rr] = w.y;
        qf[2 * hc + 1][rr] = w.z, qf[2 * hc + 1][2 + rr] = w.w;
      }
  }

  // keys each of this thread's rows sees (from the sequence's first key)
  int seen[2 * kMT];
  const int64_t L = (int64_t)sq.nc + sq.nk;
#pragma unroll
  for (int i = 0; i < 2 * kMT; ++i) {
    const int r = (row0 + (i >> 1) * 16 + (i & 1) * 8 + g) / a.group;
    seen[i] = (int)(a.causal ? min(L, max((int64_t)0, L - sq.Lq + r + 1)) : L);
  }
  const int seen_by_all = (int)(a.causal ? min(L, max((int64_t)0, L - sq.Lq + row0 / a.group + 1)) : L);

  float m[2 * kMT], l[2 * kMT], o[kMT][16][4];
#pragma unroll
  for (int i = 0; i < 2 * kMT; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.f;

  // ------------------------------------------------------------ key chunks
  const uint32_t stage0 = base + kOffStages + warp * (kStages * kStageBytes);
  const uint32_t scale0 = base + kOffScales + warp * (kStages * 32 * 8);
  const int n_mine = c_begin + warp < c_end ? (c_end - c_begin - warp + kWarps - 1) / kWarps : 0;
  const int64_t row_bytes = (int64_t)a.Hkv * (kFmt == kFmtBf16 ? 2 * kD : kD);  // a cache slot
  const uint8_t* kc = a.kc + (int64_t)hkv * (kFmt == kFmtBf16 ? 2 * kD : kD);
  const uint8_t* vc = a.vc + (int64_t)hkv * (kFmt == kFmtBf16 ? 2 * kD : kD);
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
  float2 pend = make_float2(0.f, 0.f);  // (K, V) scales of this lane's key in the chunk issued last
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
        if constexpr (kFmt != kFmtBf16) {
          pend = make_float2(0.f, 0.f);
          if (row >= 0) {
            pend.x = exp_scale(a.k_exp[slot * a.Hkv + hkv]);
            pend.y = exp_scale(a.v_exp[slot * a.Hkv + hkv]);
          }
        }
        constexpr int kUnits = kFmt == kFmtBf16 ? 16 : 8;  // 16-byte units of a row
        constexpr int kStep = 32 / kUnits;                 // rows of one warp-wide copy
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
  auto put_scales = [&](int i) {  // scales of chunk i, issued by the last issue()
    if constexpr (kFmt != kFmtBf16) {
      if (i < n_mine)
        asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(scale0 + ((i % kStages) * 32 + lane) * 8), "f"(pend.x),
                     "f"(pend.y)
                     : "memory");
    }
  };

  int raw = lookup(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    issue(i, raw);
    raw = lookup(i + 1);
    if (i + 1 < kStages - 1) put_scales(i);
  }
  for (int i = 0; i < n_mine; ++i) {
    put_scales(i + kStages - 2);
    cp_async_wait<kStages - 2>();
    __syncwarp();  // chunk i has arrived for every lane, and no lane still reads chunk i - 1
    issue(i + kStages - 1, raw);
    raw = lookup(i + kStages);
    const int c = c_begin + warp + i * kWarps;
    const uint32_t st = stage0 + (i % kStages) * kStageBytes;
    const uint32_t sc = scale0 + (i % kStages) * 32 * 8;
    int lim[2 * kMT];
    if (c < sp.cached) {
      const int pos = c * KB;
#pragma unroll
      for (int r = 0; r < 2 * kMT; ++r) lim[r] = min(seen[r], sq.nc) - pos;
      const bool whole = min(seen_by_all, sq.nc) - pos >= KB;
      chunk_step<kFmt, kMT>(st, st + kStageBytes / 2, sc, base + kOffQ, qf, lane, a.scale_log2, whole, lim, m, l, o);
    } else {
      const int pos = sq.nc + (c - sp.cached) * kFreshKeys;
#pragma unroll
      for (int r = 0; r < 2 * kMT; ++r) lim[r] = seen[r] - pos;
      const bool whole = seen_by_all - pos >= kFreshKeys;
      chunk_step<kFmtBf16, kMT>(st, st + kStageBytes / 2, sc, base + kOffQ, qf, lane, a.scale_log2, whole, lim, m, l, o);
    }
  }
  cp_async_wait<0>();

  // ---------------------------------------------------- merge of the warps
  __syncthreads();  // every warp is done with its stages
  float* mo = reinterpret_cast<float*>(smem);                                      // [warp][row][128]
  float2* ml = reinterpret_cast<float2*>(smem + kWarps * kRows * kD * 4);          // [warp][row]
#pragma unroll
  for (int i = 0; i < 2 * kMT; ++i) {
    const int row = (i >> 1) * 16 + (i & 1) * 8 + g;
    float sum = l[i];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (t == 0) ml[warp * kRows + row] = make_float2(m[i], sum);
    // column n of tile j is dimension 16n + j: this thread's n are 2t, 2t + 1
    float* dst = mo + ((size_t)warp * kRows + row) * kD;
#pragma unroll
    for (int j = 0; j < 16; j += 4)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<float4*>(dst + 32 * t + 16 * e + j) =
            make_float4(o[i >> 1][j][2 * (i & 1) + e], o[i >> 1][j + 1][2 * (i & 1) + e],
                        o[i >> 1][j + 2][2 * (i & 1) + e], o[i >> 1][j + 3][2 * (i & 1) + e]);
  }
  __syncthreads();
  const bool alone = sp.total <= a.split_chunks;  // no other split has keys of this tile
  for (int i = threadIdx.x; i < kRows * (kD / 4); i += kThreads) {
    const int row = i / (kD / 4), d = (i % (kD / 4)) * 4;
    if (row >= rows) break;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml[w * kRows + row].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (mm != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 x = ml[w * kRows + row];
        const float f = ex2_approx(x.x - mm);
        const float4 y = *reinterpret_cast<const float4*>(mo + ((size_t)w * kRows + row) * kD + d);
        sum = fmaf(x.y, f, sum);
        acc.x = fmaf(y.x, f, acc.x), acc.y = fmaf(y.y, f, acc.y);
        acc.z = fmaf(y.z, f, acc.z), acc.w = fmaf(y.w, f, acc.w);
      }
    }
    if (alone) {
      const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;  // a row without keys is zero
      const int r = (row0 + row) / a.group, h = hkv * a.group + (row0 + row) - r * a.group;
      uint2 w;
      w.x = pack_bf16x2(acc.x * inv, acc.y * inv);
      w.y = pack_bf16x2(acc.z * inv, acc.w * inv);
      *reinterpret_cast<uint2*>(a.o + (sq.q_begin + r) * a.o_stride + (int64_t)h * kD + d) = w;
    } else {
      const int64_t at = ((int64_t)item * a.splits + split) * kRows + row;
      *reinterpret_cast<float4*>(a.part_o + at * kD + d) = acc;
      if (d == 0) a.part_ml[at] = make_float2(mm, sum);
    }
  }
}

// Merges the splits of each row in split order; one warp per packed row.
template <int kFmt, int kMT>
__global__ void __launch_bounds__(256) attn_chunk_merge_kernel(const __grid_constant__ ChunkArgs a) {
  constexpr int kRows = 16 * kMT;
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
  const int row0 = mtile * kRows;
  const int rows = sq.Lq * a.group - row0;
  if (row >= rows) return;
  const Span sp = tile_span<kFmt>(a, sq, (row0 + min(rows, kRows) - 1) / a.group);
  if (sp.total <= a.split_chunks) return;  // written by its only split
  const int n = (sp.total + a.split_chunks - 1) / a.split_chunks;
  const int64_t at = item * a.splits * kRows + row;
  float mm = -INFINITY;
  for (int s = 0; s < n; ++s) mm = fmaxf(mm, a.part_ml[at + (int64_t)s * kRows].x);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  if (mm != -INFINITY) {
    for (int s = 0; s < n; ++s) {
      const float2 x = a.part_ml[at + (int64_t)s * kRows];
      const float f = ex2_approx(x.x - mm);
      const float4 y = *reinterpret_cast<const float4*>(a.part_o + (at + (int64_t)s * kRows) * kD + lane * 4);
      sum = fmaf(x.y, f, sum);
      acc.x = fmaf(y.x, f, acc.x), acc.y = fmaf(y.y, f, acc.y);
      acc.z = fmaf(y.z, f, acc.z), acc.w = fmaf(y.w, f, acc.w);
    }
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const int r = (row0 + row) / a.group, h = hkv * a.group + (row0 + row) - r * a.group;
  uint2 out;
  out.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  out.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(a.o + (sq.q_begin + r) * a.o_stride + (int64_t)h * kD + lane * 4) = out;
}

template <int kFmt, int kMT>
cudaError_t launch(const ChunkArgs& a, cudaStream_t stream) {
  static std::atomic<bool> attr_set[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    e = cudaFuncSetAttribute(attn_chunk_kernel<kFmt, kMT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem_bytes<kMT>());
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const int64_t items = (int64_t)a.B * a.Hkv * a.mtiles;
  if (items * a.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
  e = launch_pdl(attn_chunk_kernel<kFmt, kMT>, dim3((unsigned)(items * a.splits)), dim3(kThreads), smem_bytes<kMT>(),
                 stream, a);
  if (e != cudaSuccess || a.splits == 1) return e;
  const int64_t rows = items * 16 * kMT;
  return launch_pdl(attn_chunk_merge_kernel<kFmt, kMT>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream, a);
}

}  // namespace chunk

ChunkPlan plan_attn_chunk(int format, int B, int Hkv, int group, int max_q, int max_context, int max_fresh,
                          int num_sms) {
  ChunkPlan p;
  const int64_t rows = (int64_t)max_q * group;
  p.mt = rows <= 16 ? 1 : 2;
  p.mtiles = (int)((rows + 16 * p.mt - 1) / (16 * p.mt));
  const int kb = format == kFmtBf16 ? 16 : 32;
  const int64_t chunks = ((int64_t)max_context + kb - 1) / kb + ((int64_t)max_fresh + 15) / 16;
  const int64_t items = (int64_t)B * Hkv * p.mtiles;
  // Two CTAs fit an SM. Split the keys until every SM has its two, but leave
  // each split four chunks per warp.
  int64_t splits = items > 0 ? (2 * (int64_t)num_sms + items - 1) / items : 1;
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, chunks / (4 * chunk::kWarps)));
  p.split_chunks = (int)std::max<int64_t>(1, (chunks + splits - 1) / splits);
  p.splits = (int)std::max<int64_t>(1, (chunks + p.split_chunks - 1) / p.split_chunks);
  p.workspace_bytes = p.splits > 1 ? items * p.splits * 16 * p.mt * (chunk::kD * 4 + 8) : 0;
  return p;
}

cudaError_t launch_attn_chunk(ChunkArgs a, int format, const ChunkPlan& plan, void* workspace, cudaStream_t stream) {
  a.mtiles = plan.mtiles;
  a.splits = plan.splits;
  a.split_chunks = plan.split_chunks;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.mtiles * a.splits * 16 * plan.mt;
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * chunk::kD);
  switch (format * 2 + plan.mt - 1) {
    case kFmtBf16 * 2: return chunk::launch<kFmtBf16, 1>(a, stream);
    case kFmtBf16 * 2 + 1: return chunk::launch<kFmtBf16, 2>(a, stream);
    case kFmtE4m3 * 2: return chunk::launch<kFmtE4m3, 1>(a, stream);
    case kFmtE4m3 * 2 + 1: return chunk::launch<kFmtE4m3, 2>(a, stream);
    case kFmtInt8 * 2: return chunk::launch<kFmtInt8, 1>(a, stream);
    default: return chunk::launch<kFmtInt8, 2>(a, stream);
  }
}

}  // namespace dllm
