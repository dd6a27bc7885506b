// Quantised paged KV-cache store / load (slot-mapped rows), sm_100a.
//
// store: codes, exponent <- quantise(key[i]) at slot[i], and the same for value
// load:  key[i], value[i] <- code * 2^e of slot[i]
// (the bf16 forms are store_kvcache / load_kvcache, dllmserve/layers/attention.py:11-92;
// the group format is described in kvquant.cuh)
//
// Bound by HBM: 2 bytes in and 1 out per element (store), 1 in and 2 out
// (load). One lane owns 16 elements of a row of K and of V (a 32-byte and a
// 16-byte access each), so a 128-element group is 8 lanes: three shuffles give
// its maximum. A thread does one such item; a block covers 256 consecutive
// items of the [tokens, heads, head_dim / 16] space.
// Measured, kernels back to back (32 heads of 128): storing 36,864 rows in e4m3
// 139 us, 6.5 TB/s; 11,902 rows in int8 52 us, 5.7 TB/s; loading 9,152 e4m3 rows
// 36.4 us, 6.2 TB/s (a plain copy: 6.5).
#include "common.cuh"
#include "kvquant.cuh"
#include "kvquant.h"

namespace dllm {

namespace {

constexpr int kThreads = 256;

template <bool kWide>
DLLM_DEVICE void load32(const void* p, uint32_t (&w)[8]) {
  if constexpr (kWide) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
  }
}

template <bool kWide>
DLLM_DEVICE void store32(void* p, const uint32_t (&w)[8]) {
  if constexpr (kWide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

template <int kFmt, int kD, bool kWide, bool kStore>
__global__ void __launch_bounds__(kThreads) kv_quant_kernel(KvQuantArgs a) {
  constexpr int kLanes = kD / 16;  // lanes of a group
  const int per_row = a.heads * kLanes;
  griddep_wait();  // inputs are read only after the previous grid in the stream finished
  griddep_launch_dependents();
  // (token, item of the row) of this thread: one 64-bit division for the block
  const int64_t first = (int64_t)blockIdx.x * kThreads;
  const int64_t tok0 = first / per_row;
  const uint32_t at = (uint32_t)(first - tok0 * per_row) + threadIdx.x;
  const int64_t tok = tok0 + at / (uint32_t)per_row;
  const int item = (int)(at % (uint32_t)per_row);
  const int head = item / kLanes, part = item % kLanes;
  const bool live = tok < a.n_tokens;
  const int64_t slot = live ? a.slots[tok] : -1;
  const bool ok = slot >= 0 && slot < a.num_slots;
  if (slot >= a.num_slots && item == 0) set_error(a.err, kDevSlotOutOfRange);
  const int64_t src = tok, col = (int64_t)head * kD + part * 16;
  __nv_bfloat16* key = reinterpret_cast<__nv_bfloat16*>(a.key) + src * a.key_stride + col;
  __nv_bfloat16* value = reinterpret_cast<__nv_bfloat16*>(a.value) + src * a.value_stride + col;
  const int64_t code = slot * ((int64_t)a.heads * kD) + col, ex = slot * a.heads + head;
  if constexpr (kStore) {
    uint32_t k[8] = {}, v[8] = {};
    if (ok) {
      load32<kWide>(key, k);
      load32<kWide>(value, v);
    }
    // the lanes of a group are one token's, so they are all live or all idle
    uint32_t ek, ev, ck[4], cv[4];
    group_bytes<kFmt, kLanes>(k, v, 0xffffffffu, a.err, ek, ev);
    if (!ok) return;
    quantise<kFmt>(k, ek, ck);
    quantise<kFmt>(v, ev, cv);
    *reinterpret_cast<uint4*>(a.k_cache + code) = make_uint4(ck[0], ck[1], ck[2], ck[3]);
    *reinterpret_cast<uint4*>(a.v_cache + code) = make_uint4(cv[0], cv[1], cv[2], cv[3]);
    if (part == 0) {
      a.k_exp[ex] = (uint8_t)ek;
      a.v_exp[ex] = (uint8_t)ev;
    }
  } else {
    if (!live) return;
    uint32_t k[8] = {}, v[8] = {};
    if (ok) {
      const uint4 ck = __ldg(reinterpret_cast<const uint4*>(a.k_cache + code));
      const uint4 cv = __ldg(reinterpret_cast<const uint4*>(a.v_cache + code));
      const uint32_t ek = a.k_exp[ex], ev = a.v_exp[ex];
      dequantise16<kFmt>(ck, ek, k);
      dequantise16<kFmt>(cv, ev, v);
    }
    store32<kWide>(key, k);
    store32<kWide>(value, v);
  }
}

template <int kFmt, int kD, bool kWide>
cudaError_t launch_typed(const KvQuantArgs& a, bool store, cudaStream_t stream) {
  const int64_t items = a.n_tokens * a.heads * (kD / 16);
  const int64_t blocks = (items + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  return store ? launch_pdl(kv_quant_kernel<kFmt, kD, kWide, true>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, a)
               : launch_pdl(kv_quant_kernel<kFmt, kD, kWide, false>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
}

template <int kFmt>
cudaError_t launch_fmt(const KvQuantArgs& a, bool store, int head_dim, bool wide, cudaStream_t stream) {
  switch (head_dim) {
    case 64:
      return wide ? launch_typed<kFmt, 64, true>(a, store, stream) : launch_typed<kFmt, 64, false>(a, store, stream);
    case 128:
      return wide ? launch_typed<kFmt, 128, true>(a, store, stream) : launch_typed<kFmt, 128, false>(a, store, stream);
    default:
      return wide ? launch_typed<kFmt, 256, true>(a, store, stream) : launch_typed<kFmt, 256, false>(a, store, stream);
  }
}

}  // namespace

cudaError_t launch_kv_quant(const KvQuantArgs& a, bool store, int format, int head_dim, bool wide,
                            cudaStream_t stream) {
  if (a.n_tokens == 0) return cudaSuccess;
  return format == kFmtE4m3 ? launch_fmt<kFmtE4m3>(a, store, head_dim, wide, stream)
                            : launch_fmt<kFmtInt8>(a, store, head_dim, wide, stream);
}

}  // namespace dllm
