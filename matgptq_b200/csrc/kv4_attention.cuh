// What the attention kernels over the 4-bit cache share (kv4_attention.cu: few rows; kv4_prompt.cu: many).
#pragma once
#include "kv4.cuh"

namespace mg {

struct Kv4AttentionParams {
  Kv4Cache cache;
  const uint16_t *q;   // [B, S, H, D]
  uint16_t *out;       // [B, S, H, D]
  const int *lengths;  // [B]
  float *weights;      // [B, KV, capacity] or null
  float *lse;          // few rows: [B, KV, rows] or null: log2 of the sum of exp2(score), scores in units of log 2
  uint8_t *row_tiles;  // many rows: [B, KV, tiles of 128 rows, kv4_row_tile_bytes] or null
  int seq, heads, group;
  int window, sinks;   // window 0: none
  float scale_log2;    // softmax scale * log2(e)
};

// The blocks of N entries that rows of positions lo .. hi see: those that hold first entries, then those of the window.
struct Kv4Range {
  int first_blocks, window_block, blocks;
  __device__ __forceinline__ int block(int i) const { return i < first_blocks ? i : window_block + (i - first_blocks); }
};

template <int N> __device__ __forceinline__ Kv4Range kv4_range(int lo, int hi, int window, int sinks, int capacity) {
  Kv4Range r;
  const int end = min(hi + 1, capacity);  // entries 0 .. end - 1 at most
  if (end <= 0) {
    r.first_blocks = r.window_block = r.blocks = 0;
    return r;
  }
  const int start = window > 0 ? max(0, lo - window + 1) : 0;
  r.first_blocks = start > 0 ? (min(sinks, end) + N - 1) / N : 0;
  r.window_block = max(start / N, r.first_blocks);
  r.blocks = r.first_blocks + max(0, (end + N - 1) / N - r.window_block);
  return r;
}

__device__ __forceinline__ bool kv4_sees(int p, int j, int window, int sinks) {
  return j <= p && (window == 0 || j > p - window || j < sinks);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Codes of two neighbours less 8, exact: 1024 + c and 1024 + 16 c are fp16 numbers with the code in their last bits.
__device__ __forceinline__ uint32_t centred_low(uint32_t w) {
  uint32_t r = (w & 0x000F000Fu) | 0x64006400u;
  asm("add.rn.f16x2 %0, %0, %1;" : "+r"(r) : "r"(0xE408E408u));  // - 1032
  return r;
}
__device__ __forceinline__ uint32_t centred_high(uint32_t w) {
  uint32_t r = (w & 0x00F000F0u) | 0x64006400u;
  asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(r) : "r"(0x2C002C00u), "r"(0xD480D480u));  // / 16 - 72
  return r;
}

constexpr int kKv4FewRows = 32;  // of a key/value head, for kv4_attention.cu; more go to kv4_prompt.cu

// What the second pass over many rows, for the weights, reads of 128 rows: q as the operand it is in shared memory, then three
// numbers for each row: log2 of a weight per score, per minimum of K, and the log2 of the row's sum.
__host__ __device__ constexpr int kv4_row_tile_bytes(int dim) { return 128 * dim * 2 + 3 * 128 * 4; }

// kv4_prompt.cu
int kv4_prompt_launch(const Kv4AttentionParams &p, bool bf16, bool pdl, cudaStream_t stream);

}  // namespace mg
