// Page scores: for every (sequence, kv head, page) an upper bound of the logits that the query rows
// of the kv head can have with the page's keys, from the smallest and largest key code of each head
// dim in the page (kept up to date by the cache's append).
//
//   score = key_scale[page, head] * max_r  f_r * sum_d max(q_rd * min_d, q_rd * max_d)
//         = key_scale[page, head] * max_r  f_r * ( q_r^+ . max  +  q_r^- . min )
//
// with q^+ = max(q, 0), q^- = min(q, 0) and f_r the row's softmax (and query) scale: the
// bound of an interval product is a plain dot product of length 2 * 128, so it runs on tensor
// cores: pages are the 16 rows of a tile, query rows its columns.
//
// What bounds it: 256 bytes of bounds per (page, kv head), read once, against 2 * 256 * rows
// operations: HBM for the query groups of a decode step.  The bounds go straight from global memory
// to registers (16 bytes per thread and load, 128 bytes per thread in flight): the tile's k order is
// free, so each thread takes 16 consecutive bytes of a page and the query is laid out to match;
// nothing is staged.  e4m3 becomes f16 with shifts and masks -- the exponent field moves by one
// place, value * 2^-8, exact and subnormals included -- because the convert instructions run at a
// fraction of the ALUs' rate.  The query is multiplied by a power of two per row so that its
// largest element is near 2^15: f16 then holds every bf16 element exactly that is not 2^-22 below
// the row's largest.
#pragma once

#include "../../include/pa_decode_sm100.h"
#include "pa_common.cuh"
#include "pa_params.cuh"

namespace pa {

constexpr int kScoreWarps = 8;
constexpr int kScoreTilePages = 16;
constexpr int kScoreRowBytes = kD * 2 + 16;    // one query row as f16; the padding spreads the rows over the banks
constexpr int kScoreMaxRows = 128;             // query rows (padded to 8 per kv head) that a CTA holds

struct BlockScoreParams {
  const uint8_t* q;            // [S, Hkv * rows, 128] bf16 or e4m3
  const uint8_t* bounds;       // [NB, Hkv, 2, 128] e4m3: smallest, then largest
  const int32_t* block_tables; // [S, width]
  const int32_t* context_lens; // [S]
  const float* q_scale;
  const float* k_scale;        // per block (strides) or one value (strides 0) or null
  float* scores;               // [S, Hkv, width]
  int32_t* status;
  int32_t S, Hkv, rows, block_size, num_blocks, width;
  int32_t q_is_fp8, q_quant_mode;
  int32_t heads_per_cta, tiles_per_cta;
  int64_t q_stride_seq;        // bytes
  int64_t bounds_stride_block, bounds_stride_head;   // bytes
  int64_t bt_stride_seq;
  int64_t q_scale_stride_seq;
  int64_t ks_stride_block, ks_stride_head;
  int64_t out_stride_seq, out_stride_head;
  float softmax_scale;
};

// Bytes 1 and 3, and bytes 0 and 2, of four e4m3 as two f16 (times 2^-8).
__device__ __forceinline__ uint32_t e4m3_odd_to_f16(uint32_t w) {
  return (w & 0x80008000u) | ((w >> 1) & 0x3f803f80u);
}
__device__ __forceinline__ uint32_t e4m3_even_to_f16(uint32_t w) {
  return e4m3_odd_to_f16(w << 8);
}
__device__ __forceinline__ uint32_t f16x2_max0(uint32_t v) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0u));
  return r;
}
__device__ __forceinline__ uint32_t f16x2_min0(uint32_t v) {
  uint32_t r;
  asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0u));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ldg_stream128(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// NB8: blocks of eight query rows per kv head.
template <int NB8>
__global__ void __launch_bounds__(kScoreWarps * 32)
pa_block_score_kernel(const __grid_constant__ BlockScoreParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  float* factor = reinterpret_cast<float*>(smem + (size_t)p.heads_per_cta * NB8 * 8 * kScoreRowBytes);   // [heads][NB8 * 8]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int groups = (p.Hkv + p.heads_per_cta - 1) / p.heads_per_cta;
  const int seq = (int)blockIdx.x / groups, head0 = ((int)blockIdx.x - seq * groups) * p.heads_per_cta;
  const int heads = min(p.heads_per_cta, p.Hkv - head0);
  grid_dependency_wait();
  grid_launch_dependents();   // (the dependent waits for this grid's end before it reads the scores)
  const int ctx = p.context_lens[seq];
  const int64_t cap = (int64_t)p.width * p.block_size;
  if (ctx > cap && p.status && tid == 0) atomicOr(p.status, PA_DEV_CTX_TOO_LONG);
  const int pages = ctx <= 0 ? 0 : (int)min((int64_t)p.width, ((int64_t)ctx + p.block_size - 1) / p.block_size);
  const int page0 = (int)blockIdx.y * p.tiles_per_cta * kScoreTilePages;
  const int page1 = min(p.width, page0 + p.tiles_per_cta * kScoreTilePages);
  // pages without tokens: nothing to choose
  for (int h = 0; h < heads; ++h) {
    float* out = p.scores + (int64_t)seq * p.out_stride_seq + (int64_t)(head0 + h) * p.out_stride_head;
    for (int i = max(page0, pages) + tid; i < page1; i += kScoreWarps * 32) out[i] = -INFINITY;
  }
  if (page0 >= pages) return;

  // ---- the CTA's query rows: a quad of lanes per row, lane t the 32 dims of its quarter.  Padding rows
  // repeat row 0, which changes no maximum.  Within each group of four dims the order is 0, 2, 1, 3
  // (what the e4m3 unpacking below yields).
  constexpr int kRows = NB8 * 8;
  for (int r0 = warp * 8; r0 < heads * kRows; r0 += kScoreWarps * 8) {
    const int r = r0 + g, h = r / kRows;
    int row = r - h * kRows;
    if (row >= p.rows) row = 0;
    const int64_t grow = (int64_t)(head0 + h) * p.rows + row;
    float x[32];
    if (p.q_is_fp8) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)seq * p.q_stride_seq + grow * kD + t * 32);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 v = __ldg(src + e);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t ev = e4m3_even_to_f16(w[k]), od = e4m3_odd_to_f16(w[k]);
          float f0, f1, f2, f3;   // times 2^-8, taken back by the factor below
          asm("{.reg .f16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(f0), "=f"(f2) : "r"(ev));
          asm("{.reg .f16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(f1), "=f"(f3) : "r"(od));
          x[e * 16 + k * 4] = f0 * 256.f, x[e * 16 + k * 4 + 1] = f1 * 256.f;
          x[e * 16 + k * 4 + 2] = f2 * 256.f, x[e * 16 + k * 4 + 3] = f3 * 256.f;
        }
      }
    } else {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (int64_t)seq * p.q_stride_seq + grow * (kD * 2) + t * 64);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint4 v = __ldg(src + e);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) x[e * 8 + k * 2] = bf16_lo_to_f32(w[k]), x[e * 8 + k * 2 + 1] = bf16_hi_to_f32(w[k]);
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 32; ++e) amax = fmaxf(amax, fabsf(x[e]));
    amax = quad_max(amax);
    // power of two that brings the row's largest element into [2^14, 2^15)
    const int be = (int)((__float_as_uint(amax) >> 23) & 0xff);
    float pre = 1.0f, back = 1.0f;
    if (be > 0 && be < 255) {
      pre = __uint_as_float((uint32_t)min(253, 254 + 14 - be) << 23);
      back = 1.0f / pre;   // a power of two
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint4 v;
      v.x = pack_f16x2(x[e * 8] * pre, x[e * 8 + 2] * pre);
      v.y = pack_f16x2(x[e * 8 + 1] * pre, x[e * 8 + 3] * pre);
      v.z = pack_f16x2(x[e * 8 + 4] * pre, x[e * 8 + 6] * pre);
      v.w = pack_f16x2(x[e * 8 + 5] * pre, x[e * 8 + 7] * pre);
      *reinterpret_cast<uint4*>(smem + (size_t)r * kScoreRowBytes + t * 64 + e * 16) = v;
    }
    if (t == 0) {
      float qs = 1.0f;
      if (p.q_quant_mode == PA_QUANT_PER_TENSOR) qs = __ldg(p.q_scale);
      if (p.q_quant_mode == PA_QUANT_PER_TOKEN) qs = __ldg(p.q_scale + (int64_t)seq * p.q_scale_stride_seq + grow);
      factor[r] = back * 256.0f * qs * p.softmax_scale;   // 2^8: the bounds' f16 values are the codes times 2^-8
    }
  }
  __syncthreads();

  // ---- tiles of 16 pages of one kv head, dealt to the warps with the head fastest (neighbouring
  // warps read neighbouring heads of the same pages)
  const int tiles = (min(pages, page1) - page0 + kScoreTilePages - 1) / kScoreTilePages;
  const int32_t* table = p.block_tables + (int64_t)seq * p.bt_stride_seq;
  for (int task = warp; task < tiles * heads; task += kScoreWarps) {
    const int tile = task / heads, h = task - tile * heads;
    const int pg[2] = {page0 + tile * kScoreTilePages + g, page0 + tile * kScoreTilePages + g + 8};
    int id[2];
    uint4 raw[2][2][2];   // [row half][min, max][16-byte chunk]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      id[i] = pg[i] < pages ? __ldg(table + pg[i]) : 0;
      if ((unsigned)id[i] >= (unsigned)p.num_blocks) {
        id[i] = 0;
        if (p.status) atomicOr(p.status, PA_DEV_BAD_PAGE_ID);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint8_t* src = p.bounds + (int64_t)id[i] * p.bounds_stride_block + (int64_t)(head0 + h) * p.bounds_stride_head + t * 16;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int c = 0; c < 2; ++c) raw[i][m][c] = ldg_stream128(src + m * kD + c * 64);
      }
    }
    float acc[NB8][4];
#pragma unroll
    for (int n = 0; n < NB8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    const uint8_t* qrow = smem + (size_t)(h * kRows + g) * kScoreRowBytes + t * 32;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint4 qv[NB8][2];   // this thread's 16 dims of the chunk: four k-steps of (b0, b1)
#pragma unroll
      for (int n = 0; n < NB8; ++n) {
        qv[n][0] = *reinterpret_cast<const uint4*>(qrow + n * 8 * kScoreRowBytes + c * 128);
        qv[n][1] = *reinterpret_cast<const uint4*>(qrow + n * 8 * kScoreRowBytes + c * 128 + 16);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t w0[4] = {raw[0][m][c].x, raw[0][m][c].y, raw[0][m][c].z, raw[0][m][c].w};
        const uint32_t w1[4] = {raw[1][m][c].x, raw[1][m][c].y, raw[1][m][c].z, raw[1][m][c].w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t a0 = e4m3_even_to_f16(w0[u]), a1 = e4m3_even_to_f16(w1[u]);
          const uint32_t a2 = e4m3_odd_to_f16(w0[u]), a3 = e4m3_odd_to_f16(w1[u]);
#pragma unroll
          for (int n = 0; n < NB8; ++n) {
            const uint4 v = qv[n][u >> 1];
            const uint32_t b0 = (u & 1) ? v.z : v.x, b1 = (u & 1) ? v.w : v.y;
            // against the largest code the positive part of the query, against the smallest the negative
            mma_f16(acc[n], a0, a1, a2, a3, m ? f16x2_max0(b0) : f16x2_min0(b0), m ? f16x2_max0(b1) : f16x2_min0(b1));
          }
        }
      }
    }
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < NB8; ++n) {
      const float2 f = *reinterpret_cast<const float2*>(factor + h * kRows + n * 8 + 2 * t);
      best[0] = fmaxf(best[0], fmaxf(acc[n][0] * f.x, acc[n][1] * f.y));
      best[1] = fmaxf(best[1], fmaxf(acc[n][2] * f.x, acc[n][3] * f.y));
    }
    best[0] = quad_max(best[0]);
    best[1] = quad_max(best[1]);
    if (t < 2) {
      const int i = t;
      const int page = i ? pg[1] : pg[0];
      if (page < pages) {
        float ks = 1.0f;
        if (p.k_scale) ks = __ldg(p.k_scale + (int64_t)(i ? id[1] : id[0]) * p.ks_stride_block + (int64_t)(head0 + h) * p.ks_stride_head);
        p.scores[(int64_t)seq * p.out_stride_seq + (int64_t)(head0 + h) * p.out_stride_head + page] = (i ? best[1] : best[0]) * ks;
      }
    }
  }
}

}  // namespace pa
