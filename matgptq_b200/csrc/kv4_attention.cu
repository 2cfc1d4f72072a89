// Attention over the key/value cache in 4 bits (layout: kv4.cuh), with a sliding window and first entries that stay visible.
//
// Row r of a key/value head is query i = r / G, head r % G of the group of G heads that share it; its position is
// p = length - seq + i, and it sees entry j when j <= p and (no window, or j > p - window, or j < sinks).  With codes c, d channels:
//
//   score(r, j) = scale * q_r . (k_min_j + k_scale_j c_j)  =  scale * (k_scale_j (q_r . c_j)  +  k_min_j sum(q_r))
//   out(r)      = sum_j p_rj (v_min_j + v_scale_j c_j)     =  sum_j (p_rj v_scale_j) (c_j - 8)  +  sum_j p_rj (v_min_j + 8 v_scale_j)
//
// so the tensor cores multiply the codes themselves.  Masked out of a word, a code of K is a fp16 subnormal (c 2^-24, or c 2^-20 for
// the masks 4 bits up) and the products are exact; neither K nor V is ever rounded.  q is scaled by a power of two per row so that its
// largest value lies in [1, 2): as fp16 it then keeps all of fp16's and bf16's bits down to 2^-25 of the largest value.
// What is rounded is p v_scale, to fp16 (2^-11), as the operand of the second product, in units of a power of two near the largest
// v_scale.  The codes of V are centred first: their mean would multiply that rounding, and the tensor cores would sum up numbers of
// one sign, which over 131072 entries cost three bits of the result.  Row maximum and sums are fp32.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>

#include "../../include/matgptq_b200.h"
#include "async.cuh"
#include "gemv_common.cuh"
#include "helper_kernels.cuh"
#include "host_util.h"
#include "kernels.h"
#include "kv4_attention.cuh"
#include "tc_common.cuh"

namespace mg {

MG_DEFINE_STATUS_ACCESSOR(kv4_attention_device_status)

// Rows r0 .. r0 + 7 of a key/value head as operands: lane (g, t) holds of row g the channels that lane t of a K row's words has,
// in the order in which the masks take them out of a word; and the constants of the rows that its results are for, 2t and 2t + 1.
template <int D> struct Kv4Rows {
  uint32_t q[D / 32][4];
  float unit[2];  // score per k_scale * (q . c 2^-24)
  float sum[2];   // score per k_min
  int pos[2];     // position; before every entry where there is no such row
};

template <typename T, int D>
__device__ __forceinline__ void kv4_load_rows(Kv4Rows<D> &rows, const Kv4AttentionParams &p, int b, int h, int r0, int total, int length) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int W = D / 32;
  float v[W][8], top = 0.f;
  const int r = r0 + g;
  const bool live = r < total;
  const int i = r / p.group;
  const uint16_t *src =
      p.q + ((static_cast<size_t>(b) * p.seq + (live ? i : 0)) * p.heads + static_cast<size_t>(h) * p.group + (live ? r - i * p.group : 0)) * D +
      t * (D / 4);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) raw = *reinterpret_cast<const uint4 *>(src + 8 * w);
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[w][2 * c] = kv4_to_f<T>(static_cast<uint16_t>(u[c]));
      v[w][2 * c + 1] = kv4_to_f<T>(static_cast<uint16_t>(u[c] >> 16));
      top = fmaxf(top, fmaxf(fabsf(v[w][2 * c]), fabsf(v[w][2 * c + 1])));
    }
  }
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  // 2^-e with 2^e <= top < 2^(e+1), exact; a row of zeros stays as it is, one with an infinity keeps it
  const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 1), 253);
  const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(e) << 23);
  float sum = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    uint32_t h2[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const __half x = __float2half_rn(v[w][c] * down);
      sum += __half2float(x);
      h2[c] = __half_as_ushort(x);
    }
    rows.q[w][0] = h2[0] | h2[4] << 16;
    rows.q[w][1] = h2[2] | h2[6] << 16;
    rows.q[w][2] = h2[1] | h2[5] << 16;
    rows.q[w][3] = h2[3] | h2[7] << 16;
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 1);
  sum += __shfl_xor_sync(0xffffffffu, sum, 2);
  const float per = up * p.scale_log2;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float f = __shfl_sync(0xffffffffu, per, (2 * t + k) * 4);
    rows.unit[k] = f * 16777216.f;
    rows.sum[k] = f * __shfl_sync(0xffffffffu, sum, (2 * t + k) * 4);
    const int row = r0 + 2 * t + k;
    rows.pos[k] = row < total ? length - p.seq + row / p.group : -1;
  }
}

// What a lane (g, t) loads of a block of 16 entries: K words of entries g and g + 8, V words of the pairs t and t + 4, the params
// of entries g and g + 8.
template <int D> struct Kv4Block {
  uint32_t k[2][D / 32], v[2][D / 32];
  uint2 param[2];
};

template <int W> __device__ __forceinline__ void kv4_load_words(uint32_t (&dst)[W], const uint8_t *src) {
  if constexpr (W == 4) {
    const uint4 x = *reinterpret_cast<const uint4 *>(src);
    dst[0] = x.x, dst[1] = x.y, dst[2] = x.z, dst[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2 *>(src);
    dst[0] = x.x, dst[1] = x.y;
  }
}

template <int D, bool WITH_V = true>
__device__ __forceinline__ void kv4_load_block(Kv4Block<D> &blk, const Kv4Cache &c, size_t first, int block) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const size_t e = first + static_cast<size_t>(block) * 16;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    kv4_load_words(blk.k[i], c.k + (e + g + 8 * i) * (D / 2) + t * (D / 8));
    blk.param[i] = *reinterpret_cast<const uint2 *>(c.params + (e + g + 8 * i) * 4);
    if constexpr (WITH_V) kv4_load_words(blk.v[i], c.v + ((e >> 1) + t + 4 * i) * D + g * (D / 8));
  }
}

// Scores of 16 entries x 8 rows in units of log 2: s[0], s[1] entry g, rows 2t and 2t + 1; s[2], s[3] entry g + 8.
template <typename T, int D>
__device__ __forceinline__ void kv4_scores(float (&s)[4], const Kv4Block<D> &blk, const Kv4Rows<D> &rows) {
  float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    const uint32_t x = blk.k[0][w], y = blk.k[1][w], xs = x >> 8, ys = y >> 8;
    const uint32_t a[4] = {x & 0x000F000Fu, y & 0x000F000Fu, xs & 0x000F000Fu, ys & 0x000F000Fu};
    const uint32_t c[4] = {x & 0x00F000F0u, y & 0x00F000F0u, xs & 0x00F000F0u, ys & 0x00F000F0u};
    mma16816<false>(lo, a, rows.q[w][0], rows.q[w][1]);
    mma16816<false>(hi, c, rows.q[w][2], rows.q[w][3]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float ks = kv4_to_f<T>(static_cast<uint16_t>(blk.param[i].x)), kl = kv4_to_f<T>(static_cast<uint16_t>(blk.param[i].x >> 16));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float dot = fmaf(hi[2 * i + k], 0.0625f, lo[2 * i + k]) * rows.unit[k];
      s[2 * i + k] = fmaf(ks, dot, kl * rows.sum[k]);
    }
  }
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

constexpr int kKv4Warps = 8;

// Up to 8 NT rows of one key/value head and sequence per cluster; its warps share out the blocks of 16 entries, one range each.
// Every warp keeps its own running maximum; they are joined in shared memory, then over the cluster's CTAs through distributed
// shared memory, in a fixed order.  blockIdx.x: the CTA of the cluster, y: tile of rows, z: sequence and head.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kKv4Warps * 32) kv4_attention_kernel(const Kv4AttentionParams p) {
  pdl_prologue();
  constexpr int R = 8 * NT, W = D / 32;
  extern __shared__ float smem[];
  float *part = smem;                                  // [warps][R][D]
  float *part_m = smem + kKv4Warps * R * D;            // [warps][R]
  float *part_l = part_m + kKv4Warps * R;              // [warps][R]
  float *cta_m = part_l + kKv4Warps * R;               // [R]
  float *cta_l = cta_m + R;                            // [R]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x, ctas = gridDim.x;
  const int b = blockIdx.z / p.cache.kv_heads, h = blockIdx.z - b * p.cache.kv_heads;
  const int total = p.seq * p.group, r0 = blockIdx.y * R;
  const int length = kv4_length(p.lengths, b, p.cache.capacity);
  const size_t first = static_cast<size_t>(blockIdx.z) * p.cache.capacity;
  const int pos_lo = length - p.seq + r0 / p.group, pos_hi = length - p.seq + (min(r0 + R, total) - 1) / p.group;
  const Kv4Range range = kv4_range<16>(pos_lo, pos_hi, p.window, p.sinks, p.cache.capacity);
  const int units = ctas * kKv4Warps, unit = cta * kKv4Warps + warp;
  const int from = static_cast<int>(static_cast<long long>(range.blocks) * unit / units);
  const int to = static_cast<int>(static_cast<long long>(range.blocks) * (unit + 1) / units);

  Kv4Rows<D> rows[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) kv4_load_rows<T, D>(rows[n], p, b, h, r0 + 8 * n, total, length);

  float o[NT][2 * W][4], m[NT][2], l[NT][2], fix[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 2 * W; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) m[n][k] = -INFINITY, l[n][k] = 0.f, fix[n][k] = 0.f;
  }
  float v_unit = 0x1p-100f, v_per = 0x1p100f;  // p v_scale is rounded in these units, a power of two; the warp's largest v_scale sets it

  Kv4Block<D> cur, nxt;
  if (from < to) kv4_load_block<D>(cur, p.cache, first, range.block(from));
  for (int i = from; i < to; ++i) {
    if (i + 1 < to) kv4_load_block<D>(nxt, p.cache, first, range.block(i + 1));
    const int j0 = range.block(i) * 16;
    const bool whole = j0 + 15 <= pos_lo && r0 + R <= total && (p.window == 0 || j0 > pos_hi - p.window || j0 + 16 <= p.sinks);
    float s[NT][4];
    float vs[2], vl[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      vs[e] = kv4_to_f<T>(static_cast<uint16_t>(cur.param[e].y));
      vl[e] = kv4_to_f<T>(static_cast<uint16_t>(cur.param[e].y >> 16));
    }
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      kv4_scores<T, D>(s[n], cur, rows[n]);
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!kv4_sees(rows[n].pos[e & 1], j0 + g + 8 * (e >> 1), p.window, p.sinks)) s[n][e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) grow |= !(s[n][e] <= m[n][e & 1] + 4.f);
    }
    // entries that no row of the warp's tile sees may hold anything
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (j0 + g + 8 * e > pos_hi) vs[e] = vl[e] = 0.f;
    }
    grow |= fmaxf(fabsf(vs[0]), fabsf(vs[1])) > 16.f * v_unit;
    // Maximum and unit may lag by a factor of 16: both cancel in the end, and fp16 has the room.
    if (__any_sync(0xffffffffu, grow)) {
      float top = fmaxf(fabsf(vs[0]), fabsf(vs[1]));
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
      float rescale = 1.f;
      if (top > v_unit && top <= FLT_MAX) {
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23), 27), 250);
        const float unit_new = __uint_as_float(static_cast<uint32_t>(e) << 23);
        rescale = v_unit * __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        v_unit = unit_new;
        v_per = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          // a NaN counts as an infinity here: the row's results are NaN then
          float x = s[n][k] == s[n][k] && s[n][2 + k] == s[n][2 + k] ? fmaxf(s[n][k], s[n][2 + k]) : INFINITY;
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float m_new = fmaxf(m[n][k], x);
          const float f = m[n][k] == -INFINITY ? 0.f : exp2_approx(m[n][k] - m_new);
          m[n][k] = m_new;
          l[n][k] *= f;
          fix[n][k] *= f;
#pragma unroll
          for (int w = 0; w < 2 * W; ++w) {
            o[n][w][k] *= f * rescale;
            o[n][w][2 + k] *= f * rescale;
          }
        }
    }
    const float mid[2] = {fmaf(8.f, vs[0], vl[0]), fmaf(8.f, vs[1], vl[1])}, per[2] = {vs[0] * v_per, vs[1] * v_per};
    uint32_t pv[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // hidden entries may hold a NaN: nothing of theirs is multiplied
        const bool hidden = s[n][e] == -INFINITY;
        const float pe = hidden ? 0.f : exp2_approx(s[n][e] - m[n][e & 1]);
        l[n][e & 1] += pe;
        fix[n][e & 1] = fmaf(pe, hidden ? 0.f : mid[e >> 1], fix[n][e & 1]);
        x[e] = hidden ? 0.f : pe * per[e >> 1];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const __half2 r = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
        pv[n][e] = transpose_8x8(*reinterpret_cast<const uint32_t *>(&r));
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t x = cur.v[0][w], y = cur.v[1][w], xs = x >> 8, ys = y >> 8;
      const uint32_t a[4] = {centred_low(x), centred_high(x), centred_low(y), centred_high(y)};
      const uint32_t c[4] = {centred_low(xs), centred_high(xs), centred_low(ys), centred_high(ys)};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma16816<false>(o[n][2 * w], a, pv[n][0], pv[n][1]);
        mma16816<false>(o[n][2 * w + 1], c, pv[n][0], pv[n][1]);
      }
    }
    cur = nxt;
  }

  // the warp's sums: lanes of equal t hold parts of the same rows' l and fix
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) {
        l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], off);
        fix[n][k] += __shfl_xor_sync(0xffffffffu, fix[n][k], off);
      }
      const int row = 8 * n + 2 * t + k;
      if (g == 0) {
        part_m[warp * R + row] = m[n][k];
        part_l[warp * R + row] = l[n][k];
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        float4 x;  // channels D/8 g + 4 w + 0 .. 3
        x.x = fmaf(o[n][2 * w][k], v_unit, fix[n][k]);
        x.y = fmaf(o[n][2 * w][2 + k], v_unit, fix[n][k]);
        x.z = fmaf(o[n][2 * w + 1][k], v_unit, fix[n][k]);
        x.w = fmaf(o[n][2 * w + 1][2 + k], v_unit, fix[n][k]);
        *reinterpret_cast<float4 *>(part + (warp * R + row) * D + (D / 8) * g + 4 * w) = x;
      }
    }
  __syncthreads();
  for (int r = threadIdx.x; r < R; r += kKv4Warps * 32) {
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kKv4Warps; ++w) top = fmaxf(top, part_m[w * R + r]);
    for (int w = 0; w < kKv4Warps; ++w) {
      const float f = part_m[w * R + r] == -INFINITY ? 0.f : exp2_approx(part_m[w * R + r] - top);
      sum = fmaf(part_l[w * R + r], f, sum);
      part_m[w * R + r] = f;
    }
    cta_m[r] = top;
    cta_l[r] = sum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * D; i += kKv4Warps * 32) {
    const int r = i / D;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) {
      const float f = part_m[w * R + r];
      if (f != 0.f) sum = fmaf(part[w * R * D + i], f, sum);
    }
    part[i] = sum;
  }
  cluster_sync_all();
  const uint32_t part_u32 = smem_u32(part), m_u32 = smem_u32(cta_m), l_u32 = smem_u32(cta_l);
  auto remote = [](uint32_t addr, int c) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(addr, c)) : "memory");
    return v;
  };
  for (int i = cta * kKv4Warps * 32 + threadIdx.x; i < R * D; i += ctas * kKv4Warps * 32) {
    const int r = i / D, row = r0 + r;
    float top = -INFINITY;
    for (int c = 0; c < ctas; ++c) top = fmaxf(top, remote(m_u32 + 4 * r, c));
    float sum = 0.f, norm = 0.f;
    for (int c = 0; c < ctas; ++c) {
      const float mc = remote(m_u32 + 4 * r, c);
      if (mc == -INFINITY) continue;
      const float f = exp2_approx(mc - top);
      norm = fmaf(remote(l_u32 + 4 * r, c), f, norm);
      sum = fmaf(remote(part_u32 + 4 * i, c), f, sum);
    }
    if (row < total) {
      const int q = row / p.group;
      const size_t at = ((static_cast<size_t>(b) * p.seq + q) * p.heads + static_cast<size_t>(h) * p.group + (row - q * p.group)) * D + (i - r * D);
      p.out[at] = kv4_bits<T>(top == -INFINITY ? 0.f : sum / norm);  // a row that sees nothing: zeros
      if (p.lse != nullptr && i % D == 0) p.lse[static_cast<size_t>(blockIdx.z) * total + row] = top == -INFINITY ? INFINITY : top + log2f(norm);
    }
  }
  cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// weights[j] += sum over all rows of exp2(score - lse): a warp per block of 16 entries goes over the rows that see it, so that the
// sum has one order and needs no atomics.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_weights_kernel(const Kv4AttentionParams p) {
  pdl_prologue();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.y / p.cache.kv_heads, h = blockIdx.y - b * p.cache.kv_heads;
  const int total = p.seq * p.group, length = kv4_length(p.lengths, b, p.cache.capacity);
  const size_t first = static_cast<size_t>(blockIdx.y) * p.cache.capacity;
  const int block = blockIdx.x * 8 + warp, j0 = block * 16;
  if (j0 >= length) return;
  // rows whose query is at j0 or behind; with a window, and past the first entries, only those it reaches
  int lo = max(0, j0 - (length - p.seq)), hi = p.seq;
  if (p.window > 0 && j0 >= p.sinks) hi = static_cast<int>(min(static_cast<long long>(hi), static_cast<long long>(j0) + 15 + p.window - (length - p.seq)));
  if (lo >= hi) return;
  Kv4Block<D> blk;
  kv4_load_block<D, false>(blk, p.cache, first, block);
  float sum[2] = {0.f, 0.f};
  const float *lse = p.lse + static_cast<size_t>(blockIdx.y) * total;
  for (int r0 = lo * p.group; r0 < hi * p.group; r0 += 8) {
    Kv4Rows<D> rows;
    kv4_load_rows<T, D>(rows, p, b, h, r0, total, length);
    float s[4];
    kv4_scores<T, D>(s, blk, rows);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = r0 + 2 * t + (e & 1);
      if (row < total && kv4_sees(rows.pos[e & 1], j0 + g + 8 * (e >> 1), p.window, p.sinks)) sum[e >> 1] += exp2_approx(s[e] - lse[row]);
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
    sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
    const int j = j0 + g + 8 * e;
    if (t == 0 && j < length) p.weights[first + j] += sum[e];
  }
}

namespace {

template <typename T, int D, int NT> int kv4_attention_launch(const Kv4AttentionParams &p, cudaStream_t stream, bool pdl) {
  constexpr int R = 8 * NT;
  constexpr int smem = (kKv4Warps * R * (D + 2) + 2 * R) * 4;
  static SharedMemoryOptIn opt_in;
  int st = opt_in.ensure(kv4_attention_kernel<T, D, NT>, smem);
  if (st != MG_OK) return st;
  int sms = 0;
  st = current_device_sm_count(&sms);
  if (st != MG_OK) return st;
  const int tiles = (p.seq * p.group + R - 1) / R, bh = p.cache.batch * p.cache.kv_heads;
  if (tiles > 65535) return MG_ERR_UNSUPPORTED;
  const long long most = p.window > 0 ? static_cast<long long>(p.window) + p.sinks + p.seq + 32 : p.cache.capacity;
  const long long blocks = (std::min<long long>(most, p.cache.capacity) + 15) / 16;
  int ctas = 1;
  while (ctas < 8 && static_cast<long long>(tiles) * bh * ctas < 2 * sms && ctas * kKv4Warps < blocks) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, tiles, bh);
  cfg.blockDim = dim3(kKv4Warps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kv4_attention_kernel<T, D, NT>, p) == cudaSuccess ? MG_OK : MG_ERR_CUDA;
}

template <typename T, int D> int kv4_attention_dispatch(const Kv4AttentionParams &p, cudaStream_t stream, bool pdl) {
  const int st = p.seq * p.group <= 8 ? kv4_attention_launch<T, D, 1>(p, stream, pdl) : kv4_attention_launch<T, D, 2>(p, stream, pdl);
  if (st != MG_OK || p.weights == nullptr) return st;
  const dim3 grid((p.cache.capacity + 127) / 128, p.cache.batch * p.cache.kv_heads);
  return launch_helper(kv4_weights_kernel<T, D>, grid, 256, stream, true, p);
}

}  // namespace

int kv4_attention(const Kv4AttentionParams &p, bool bf16, bool pdl, cudaStream_t stream) {
  if (p.seq * p.group > kKv4FewRows) return kv4_prompt_launch(p, bf16, pdl, stream);
  if (p.cache.dim == 64)
    return bf16 ? kv4_attention_dispatch<__nv_bfloat16, 64>(p, stream, pdl) : kv4_attention_dispatch<__half, 64>(p, stream, pdl);
  return bf16 ? kv4_attention_dispatch<__nv_bfloat16, 128>(p, stream, pdl) : kv4_attention_dispatch<__half, 128>(p, stream, pdl);
}

}  // namespace mg

extern "C" {

int64_t matgptq_b200_attention_kv4_workspace_bytes(const matgptq_b200_kv4_cache *cache, int64_t seq, int64_t n_heads, int with_weights) {
  if (!cache || !with_weights || cache->batch <= 0 || cache->n_kv_heads <= 0 || seq <= 0 || n_heads < cache->n_kv_heads) return 0;
  const int64_t rows = seq * (n_heads / cache->n_kv_heads), heads = cache->batch * cache->n_kv_heads;
  return rows <= mg::kKv4FewRows ? heads * rows * 4 : heads * ((rows + 127) / 128) * mg::kv4_row_tile_bytes(static_cast<int>(cache->head_dim));
}

int matgptq_b200_attention_kv4(const matgptq_b200_kv4_cache *cache, const void *q, int64_t seq, int64_t n_heads, const int32_t *lengths,
                               int64_t window, int64_t sinks, float scale, float *weights, void *out, void *workspace,
                               int64_t workspace_bytes, uint32_t flags, void *stream) {
  const int st = mg::kv4_check_cache(cache);
  if (st != MG_OK) return st;
  if (!q || !lengths || !out) return MG_ERR_BAD_ARG;
  if (seq < 0 || n_heads <= 0 || n_heads % cache->n_kv_heads != 0 || window < 0 || sinks < 0) return MG_ERR_BAD_ARG;
  if (seq > (1 << 24) || n_heads > (1 << 16) || seq * (n_heads / cache->n_kv_heads) > (1 << 24)) return MG_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 != 0) return MG_ERR_ALIGNMENT;
  if (cache->batch == 0 || seq == 0) return MG_OK;
  if (weights && (!workspace || workspace_bytes < matgptq_b200_attention_kv4_workspace_bytes(cache, seq, n_heads, 1))) return MG_ERR_BAD_ARG;
  if (weights && reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return MG_ERR_ALIGNMENT;
  mg::Kv4AttentionParams p = {};
  p.cache = mg::kv4_cache(cache);
  p.q = static_cast<const uint16_t *>(q);
  p.out = static_cast<uint16_t *>(out);
  p.lengths = lengths;
  p.weights = weights;
  const bool few = seq * (n_heads / cache->n_kv_heads) <= mg::kKv4FewRows;
  p.lse = weights && few ? static_cast<float *>(workspace) : nullptr;
  p.row_tiles = weights && !few ? static_cast<uint8_t *>(workspace) : nullptr;
  p.seq = static_cast<int>(seq);
  p.heads = static_cast<int>(n_heads);
  p.group = static_cast<int>(n_heads / cache->n_kv_heads);
  // a window or first entries past the capacity reach everything; kept small so that positions +- window stay in 32 bits
  p.window = static_cast<int>(window > cache->capacity ? 0 : window);
  p.sinks = static_cast<int>(sinks > cache->capacity ? cache->capacity : sinks);
  p.scale_log2 = scale * 1.44269504088896340736f;
  return mg::kv4_attention(p, (flags & MATGPTQ_B200_FLAG_BF16) != 0, (flags & MATGPTQ_B200_FLAG_PDL) != 0, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
