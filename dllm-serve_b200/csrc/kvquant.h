// Internal launch interface of the quantised KV-cache copy kernels.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace dllm {

struct KvQuantArgs {
  void* key;                  // bf16 token rows (source for store, destination for load)
  void* value;
  int64_t key_stride;         // elements between token rows
  int64_t value_stride;
  uint8_t* k_cache;           // codes: slot rows of heads * head_dim bytes
  uint8_t* v_cache;
  uint8_t* k_exp;             // exponent bytes: slot rows of `heads` bytes
  uint8_t* v_exp;
  const int32_t* slots;
  int64_t n_tokens;
  int64_t num_slots;
  int heads;
  int32_t* err;
};

// format: DLLM_KV_E4M3 or DLLM_KV_INT8. head_dim: 64, 128 or 256. wide: every
// key/value row starts on a 32-byte boundary (else 16).
cudaError_t launch_kv_quant(const KvQuantArgs& a, bool store, int format, int head_dim, bool wide,
                            cudaStream_t stream);

}  // namespace dllm
