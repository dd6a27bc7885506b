// Internal launch interface of chunk attention over a paged, possibly
// quantised KV cache (not part of the public C ABI; see include/dllm_attn.h).
#pragma once

#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_bf16.h>

namespace dllm {

struct ChunkArgs {
  const __nv_bfloat16* q;  // [total_q, Hq, 128]
  int64_t q_stride;        // elements between token rows
  const __nv_bfloat16* k;  // fresh rows [total_k, Hkv, 128], or null
  int64_t k_stride;
  const __nv_bfloat16* v;
  int64_t v_stride;
  const uint8_t* kc;       // cache: slot rows of Hkv * 128 elements (bf16) or codes
  const uint8_t* vc;
  const uint8_t* k_exp;    // exponent bytes of a quantised cache: slot rows of Hkv bytes
  const uint8_t* v_exp;
  int64_t num_slots;
  const int32_t* slots;    // slot list (cached rows of sequence b: slots[cu_s[b] .. cu_s[b+1])) or null
  const int32_t* cu_s;
  int64_t total_slots;
  const int32_t* tables;   // block tables [B, table_stride], or null
  int64_t table_stride;
  int max_blocks;          // entries of a table row
  int block_size;          // slots of a block
  int block_shift;         // log2(block_size), or -1
  const int32_t* ctx;      // with tables: sequence b has ctx[b] - (ctx_base[b] & ctx_mask) cached rows
  const int32_t* ctx_base;
  int ctx_mask;            // 0 (lengths) or -1 (running sums)
  int max_context;         // no sequence has more cached rows
  const int32_t* cu_q;
  const int32_t* cu_k;     // fresh rows per sequence, or null
  int64_t total_q;
  int64_t total_k;
  int max_q;
  int max_fresh;           // no sequence has more fresh rows
  int B;
  int Hkv;
  int group;               // Hq / Hkv (Hq query heads)
  float scale_log2;        // softmax_scale * log2(e)
  int causal;
  __nv_bfloat16* o;
  int64_t o_stride;
  int32_t* err;
  // Dense cached rows (128-row launches): the cached rows of sequence b are rows b * dense +
  // position of kc / vc (bf16), as expand_rows() laid them out. 0: by table or slot list.
  int dense;
  // set by the launcher
  int tile_rows;           // packed rows of a tile that are used
  int unit_rows;           // packed rows of a work unit: one or two (128-row launches) tiles
  int mtiles;              // work units per (sequence, KV head)
  int splits;              // key splits per row tile
  int split_chunks;        // key chunks of a split
  bool cluster;            // the splits of a row tile are a cluster, which merges them (kernel for few rows)
  int total_units;         // items * splits
  float* part_o;           // [items * splits, rows, 128] partial outputs (splits > 1)
  float2* part_ml;         // [items * splits, rows] (maximum, sum)
};

constexpr int kChunkMmaRows = 128;  // packed rows of a tile of the tcgen05 kernel

// How a launch is laid out, from sizes the host knows.
struct ChunkPlan {
  int rows;                // packed rows of a tile: 8, 16 or 32 (attn_chunk.cu), 128 (attn_chunk_mma.cu)
  int tile_rows, unit_rows;
  int mtiles;
  int splits;
  int split_chunks;
  bool cluster;            // the splits merge within a cluster (no workspace)
  int dense;               // rows per sequence of the expanded copy of a quantised cache's rows, 0: none
  int64_t dense_bytes;     // its bytes (K, then V), at the workspace's start
  int64_t workspace_bytes;
};

// (total_q decides only how row tiles are grouped, not the workspace)
ChunkPlan plan_attn_chunk(int format, int B, int Hkv, int group, int max_q, int64_t total_q, int max_context,
                          int max_fresh, int num_sms);

// Tensor maps of a 128-row launch: q (boxes of 64 dimensions, a KV head's group of heads, as
// many rows as fit 128); fresh k / v (bf16 boxes of 64 x 1 x 128, 128-byte
// swizzle); caches (the same, or 8-bit boxes of 128 x 1 x 128, no swizzle); caches as
// [slots, Hkv * 128] matrices with boxes of one 128-byte row, for scattered slots.
struct ChunkMaps {
  CUtensorMap q, k, v, kc, vc, kg, vg;
};

// maps: read only by 128-row launches.
cudaError_t launch_attn_chunk(ChunkArgs a, int format, const ChunkPlan& plan, const ChunkMaps& maps, void* workspace,
                              int num_sms, cudaStream_t stream);

// Expands the cached rows of every sequence to bf16: rows b * dense + position of
// k_out, v_out [B * dense, Hkv, 128].
cudaError_t launch_expand_rows(const ChunkArgs& a, int format, void* k_out, void* v_out, cudaStream_t stream);

cudaError_t launch_attn_chunk_mma(const ChunkMaps& maps, const ChunkArgs& a, int format, int num_sms,
                                  cudaStream_t stream);

}  // namespace dllm
