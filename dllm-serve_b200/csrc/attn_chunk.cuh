// Device helpers shared by the chunk-attention kernels.
#pragma once

#include "common.cuh"
#include "attn_chunk.h"

namespace dllm {
namespace chunk {

// Sizes of one sequence, every value checked against the buffers it indexes.
struct Seq {
  int64_t q_begin, s_begin, k_begin;
  int Lq, nc, nk;
};

DLLM_DEVICE Seq load_seq(const ChunkArgs& a, int b, bool report) {
  Seq s;
  bool bad = false;
  auto range = [&](const int32_t* cu, int64_t total, int64_t& begin, int& n, int most) {
    // (without offsets, as q's may be: one row per sequence)
    const int64_t lo = cu != nullptr ? cu[b] : b, hi = cu != nullptr ? cu[b + 1] : b + 1;
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
    // a length, or the difference of two sums; without a branch, which cost the kernel for few rows
    // eight registers and 13 % (e4m3 contexts of 4,096-32,768 rows: 198 us, 223 with it)
    const int c = a.ctx[b] - (a.ctx_base[b] & a.ctx_mask);
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

// How many of the chunk's first rows see no key; those are zero. (A maximum of
// -infinity does not tell: the maxima drop NaN scores, and a row that has met
// nothing else is NaN.)
DLLM_DEVICE int blind_rows(const ChunkArgs& a, const Seq& s) {
  const int L = s.nc + s.nk;  // at most 2^30
  return a.causal ? s.Lq - L : L > 0 ? 0 : s.Lq;
}

// Key chunks of a row tile: the cached rows in chunks of KB keys, then the
// fresh rows in chunks of FB, both cut at the last key any row of the tile
// sees.
struct Span {
  int nc, nk;      // keys to walk in each segment
  int cached;      // chunks of the cached segment
  int total;       // all chunks
};

template <int KB, int FB>
DLLM_DEVICE Span tile_span(const ChunkArgs& a, const Seq& s, int last_row) {
  int64_t seen = (int64_t)s.nc + s.nk;
  if (a.causal) seen = min(seen, max((int64_t)0, seen - s.Lq + last_row + 1));
  Span r;
  r.nc = (int)min(seen, (int64_t)s.nc);
  r.nk = (int)(seen - r.nc);
  r.cached = (r.nc + KB - 1) / KB;
  r.total = r.cached + (r.nk + FB - 1) / FB;
  return r;
}

}  // namespace chunk
}  // namespace dllm
