// The key/value cache in 4 bits: its layout and what the kernels that use it share.
//
// An entry of one key/value head is two rows of d codes of 4 bits, K and V, and four numbers of the model's 16-bit type: scale and
// minimum of K, scale and minimum of V.  A code c stands for minimum + scale * c.
//
//   k_codes [B, KV, capacity, d/2] bytes: byte i holds channels 2i (low half) and 2i + 1
//   v_codes [B, KV, capacity/2, d] bytes: the rows (bytes as for K) of entries 2p and 2p + 1, in turns of two bytes
//   params  [B, KV, capacity, 4]
//
// K is summed over channels and V over entries, and the matrix instructions take their operands as 32-bit words of two
// neighbours along the summed axis.  A word of a K row holds eight channels, a word of a V pair four channels of two entries: masked
// with 0x000F000F (or 0x00F000F0, 4 bits up), each is such an operand as it stands.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "../../include/matgptq_b200.h"
#include "async.cuh"

namespace mg {

struct Kv4Cache {
  uint8_t *k;
  uint8_t *v;
  uint16_t *params;
  int batch, kv_heads, dim, capacity;
};

// kv4.cu, host side: the checks every entry point makes of a cache (MG_OK or an error), and the cache as the kernels take it
int kv4_check_cache(const matgptq_b200_kv4_cache *cache);
Kv4Cache kv4_cache(const matgptq_b200_kv4_cache *cache);

// a length, a position or an entry outside the cache or its tables was asked for; nothing outside was read or written
constexpr int kStatusCacheRange = 106;

// Entries of sequence b.  The including file reports (report_status of async.cuh) what is past the capacity.
__device__ __forceinline__ int kv4_length(const int *lengths, int b, int capacity) {
  const int n = lengths[b];
  if (n > capacity) report_status(kStatusCacheRange);
  return min(max(n, 0), capacity);
}

template <typename T> __device__ __forceinline__ float kv4_to_f(uint16_t v);
template <> __device__ __forceinline__ float kv4_to_f<__half>(uint16_t v) { return __half2float(__ushort_as_half(v)); }
template <> __device__ __forceinline__ float kv4_to_f<__nv_bfloat16>(uint16_t v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
template <typename T> __device__ __forceinline__ uint16_t kv4_bits(float v);
template <> __device__ __forceinline__ uint16_t kv4_bits<__half>(float v) { return __half_as_ushort(__float2half_rn(v)); }
template <> __device__ __forceinline__ uint16_t kv4_bits<__nv_bfloat16>(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
// two of them, the first in the low half, in one instruction
template <typename T> __device__ __forceinline__ uint32_t kv4_two_bits(float a, float b);
template <> __device__ __forceinline__ uint32_t kv4_two_bits<__half>(float a, float b) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&r);
}
template <> __device__ __forceinline__ uint32_t kv4_two_bits<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&r);
}

}  // namespace mg
