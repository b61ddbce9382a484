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
// operations: HBM for the query groups of a decode step.  One CTA per SM takes an equal share of all
// tiles (16 pages of up to eight kv heads) of the batch, whatever the sequences' lengths; a
// pair of producer warps runs through them with bulk copies -- a page's heads are one run of up to 2 KB -- into
// a ring of about 170 KB, and eight or sixteen warps multiply, one kv head (or every so many tiles) each.
// (With a CTA per (sequence, 128 pages) the chain length -> page ids -> query -> bounds was paid by four or
// five waves of CTAs: 54 us for 32 sequences of 16 K to 64 K tokens whose bounds take 27; with 16-byte
// copies by the multiplying warps themselves their load units were the limit: 47-50 us.)
// The tile's k order is free, so each thread takes 16 consecutive bytes of a page and the query is laid
// out to match.  e4m3 becomes f16 with shifts and masks -- the exponent field moves by one place,
// value * 2^-8, exact and subnormals included -- for one half of a page's bounds and with convert
// instructions, whose pipe is slower but otherwise idle, for the other.  The query is multiplied by a
// power of two per row so that its largest element is near 2^15: f16 then holds every bf16
// element exactly that is not 2^-22 below the row's largest.
#pragma once

#include "../../include/pa_decode_sm100.h"
#include "pa_common.cuh"
#include "pa_params.cuh"
#include "pa_tcgen05.cuh"

namespace pa {

// Warps that multiply, by the blocks of eight query rows: with one block its operand stays in registers and eight
// warps keep up with HBM; two blocks take sixteen; with more of them the accumulators leave room for eight.
__host__ __device__ constexpr int score_warps(int nb8) { return nb8 == 2 ? 16 : 8; }
constexpr int kScoreTilePages = 16;
// Warps that request tiles.  Two are enough for tiles of eight heads (31.8 us against 47.3 with one, whose bulk copies
// go out 75-90 cycles apart, and 32.5 with four); smaller tiles are more of them (one kv head: 16.9 us with
// two, 11.8 with four, 11.3 with eight; sixteen rows, four heads: 54, 41 and 43).
__host__ __device__ constexpr int score_producers(int heads_per_cta) { return heads_per_cta == 8 ? 2 : 4; }
constexpr int kScoreMaxSlots = 40;
constexpr int kScoreRingBytes = 176 * 1024;
constexpr int kScoreRowBytes = kD * 2 + 16;    // one query row as f16; the padding spreads the rows over the banks
constexpr int kScoreMaxRows = 64;              // query rows (padded to 8 per kv head) that a CTA holds
// A tile in the ring: [16 pages][heads][256 bytes], 64 bytes between pages so that neighbouring pages of
// one head lie in different banks, then its key scales [16 pages][heads].
__host__ __device__ constexpr int score_page_pitch(int heads) { return heads * 2 * kD + 64; }
__host__ __device__ constexpr int score_slot_bytes(int heads) { return kScoreTilePages * (score_page_pitch(heads) + heads * 4); }

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
  int32_t heads_per_cta;       // a power of two that divides the warps
  // Ring depth in tiles, a multiple of warps / heads_per_cta: a slot then holds tiles of the same warps
  // every time, and not less than the producers.  So nobody waits for a phase of its barriers that is not the
  // next one: a warp has waited for the slot's tile before itself, and a producer that comes to a slot has
  // filled it the last time, or has since filled a slot that was free only after this one was.
  int32_t slots;
  int32_t off_index, off_ring; // shared-memory carve: query rows and factors, index of the sequences, ring
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
// The same by the convert instruction, whose halves are bytes 0, 1 and bytes 2, 3 (true values).
__device__ __forceinline__ void e4m3_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
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
// The larger of two, NaN if one is: a query row that is no number has no bound, and its pages' scores say so.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float quad_max_or_nan(float v) {
  v = max_or_nan(v, __shfl_xor_sync(kFullMask, v, 1));
  return max_or_nan(v, __shfl_xor_sync(kFullMask, v, 2));
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
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// NB8: blocks of eight query rows per kv head.  PRODUCERS: warps that request tiles.
template <int NB8, int PRODUCERS>
__global__ void __launch_bounds__((score_warps(NB8) + PRODUCERS) * 32, 1)
pa_block_score_kernel(const __grid_constant__ BlockScoreParams p) {
  constexpr int kRows = NB8 * 8, kScoreWarps = score_warps(NB8);
  constexpr int threads = (kScoreWarps + PRODUCERS) * 32, producers = PRODUCERS;
  constexpr bool kKeep = NB8 == 1;   // the query operand of a warp's head stays in registers (32 of them)
  extern __shared__ __align__(128) uint8_t smem[];
  float* factor = reinterpret_cast<float*>(smem + p.heads_per_cta * kRows * kScoreRowBytes);   // [heads][kRows]
  int* tile_off = reinterpret_cast<int*>(smem + p.off_index);   // [S + 1] tiles before each sequence
  int* seq_pages = tile_off + p.S + 1;                          // [S]
  __shared__ int scan[32];
  __shared__ __align__(8) uint64_t bar_full[kScoreMaxSlots], bar_empty[kScoreMaxSlots];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hpc = p.heads_per_cta;
  const uint32_t ring = smem_addr(smem) + p.off_ring;
  const int slot_bytes = score_slot_bytes(hpc), pitch = score_page_pitch(hpc);
  if (tid < p.slots) {
    mbar_init(smem_addr(&bar_full[tid]), 33);     // the producer's arrival, and its lanes' key scale copies
    mbar_init(smem_addr(&bar_empty[tid]), hpc);   // the warps that multiply the tile
    // (a fence orders what its own thread has done: every thread that has initialised a barrier, not one for all)
    mbar_fence_init();
    fence_proxy_async();
  }
  grid_dependency_wait();
  grid_launch_dependents();   // (the dependent waits for this grid's end before it reads the scores)

  // ---- pages of every sequence, and tiles of 16 pages summed over the sequences (every CTA for itself).  The
  // lengths are read side by side before anything is summed: 1 024 sequences of 128 to 512 tokens take 22 us, and
  // took 34 when a thread read its four one after the other and CTAs, not warps, went over the rows for -inf.
  const int64_t cap = (int64_t)p.width * p.block_size;
  {
    bool too_long = false;
#pragma unroll 4
    for (int s = tid; s < p.S; s += threads) {
      const int ctx = __ldg(p.context_lens + s);
      too_long = too_long || ctx > cap;
      const uint32_t len = ctx <= 0 ? 0u : (uint32_t)ctx;
      const uint32_t pages = len / (uint32_t)p.block_size + (len % (uint32_t)p.block_size ? 1u : 0u);
      seq_pages[s] = (int)min((uint32_t)p.width, pages);
    }
    if (too_long && blockIdx.x == 0 && p.status) atomicOr(p.status, PA_DEV_CTX_TOO_LONG);
    const int chunk = (p.S + threads - 1) / threads;
    if (chunk > 1) __syncthreads();   // (else each thread has written what it reads)
    const int beg = min(tid * chunk, p.S), end = min(beg + chunk, p.S);
    int sum = 0;
    for (int s = beg; s < end; ++s) {
      tile_off[s + 1] = (seq_pages[s] + kScoreTilePages - 1) / kScoreTilePages;
      sum += tile_off[s + 1];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFullMask, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    if (tid == 0) tile_off[0] = 0;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < warp; ++w) run += scan[w];
    for (int s = beg; s < end; ++s) {
      run += tile_off[s + 1];
      tile_off[s + 1] = run;
    }
    __syncthreads();
  }
  const int total = tile_off[p.S];

  // ---- this CTA's share of the (head group, tile) units, the group slowest
  const int groups = (p.Hkv + hpc - 1) / hpc;
  const int64_t units = (int64_t)total * groups;
  const int64_t u_beg = units * blockIdx.x / gridDim.x, u_end = units * (blockIdx.x + 1) / gridDim.x;
  const int n_tiles = (int)(u_end - u_beg);
  struct Place { int group, seq, tile; } at0{0, 0, 0};
  if (n_tiles > 0) {
    at0.group = (int)(u_beg / total);
    const int at = (int)(u_beg - (int64_t)at0.group * total);
    int lo = 0, hi = p.S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tile_off[mid] <= at) lo = mid; else hi = mid;
    }
    at0.seq = lo;
    at0.tile = at - tile_off[lo];
  }
  auto next_seq = [&](Place& a) {   // the next sequence that has tiles (past the last unit nobody looks)
    a.tile = 0;
    do {
      if (++a.seq == p.S) a.seq = 0, ++a.group;
    } while (tile_off[a.seq + 1] == tile_off[a.seq] && a.group < groups);
  };

  if (warp >= kScoreWarps) {
    // ------------------------------------------------------------------ producers, a tile in turn: lane = page of the tile
    const int first = warp - kScoreWarps;
    Place a = at0;
    auto skip = [&](int n) {
      for (; n > 0; --n)
        if (++a.tile >= tile_off[a.seq + 1] - tile_off[a.seq]) next_seq(a);
    };
    if (n_tiles > 0) skip(first);
    const uint64_t pol = l2_policy_evict_first();
    // A page's heads are one run of up to 2 KB, brought by a bulk copy.  An SM gets through one every 75-90
    // cycles, so runs of one or two heads, and heads that lie apart, come in 16-byte pieces instead, two
    // pages' worth with every instruction (32 contexts of 16 K to 64 K tokens, one kv head: 17 us against 23).
    const bool whole = p.bounds_stride_head == 2 * kD && hpc > 2;
    // the page ids of two tiles ahead are on their way while a tile is requested
    auto fetch = [&](int k, int& group, int& valid, int& id) {
      valid = 0;
      id = 0;
      group = a.group;
      if (k < n_tiles) {
        valid = min(kScoreTilePages, seq_pages[a.seq] - a.tile * kScoreTilePages);
        if (lane < valid) id = __ldg(p.block_tables + (int64_t)a.seq * p.bt_stride_seq + a.tile * kScoreTilePages + lane);
        skip(producers);
      }
    };
    int g0, v0, id0, g1, v1, id1;
    fetch(first, g0, v0, id0);
    fetch(first + producers, g1, v1, id1);
    int slot = first, k = first;
    uint32_t phase = 1;
    for (; k < n_tiles; k += producers) {
      const int group = g0, valid = v0;
      int id = id0;
      g0 = g1, v0 = v1, id0 = id1;
      fetch(k + 2 * producers, g1, v1, id1);
      const uint32_t full = smem_addr(&bar_full[slot]);
      if (!__all_sync(kFullMask, mbar_wait(smem_addr(&bar_empty[slot]), phase))) {
        if (lane == 0 && p.status) atomicOr(p.status, PA_DEV_WAIT_TIMEOUT);
        break;
      }
      if ((unsigned)id >= (unsigned)p.num_blocks) {
        id = 0;
        if (p.status) atomicOr(p.status, PA_DEV_BAD_PAGE_ID);
      }
      const int head0 = group * hpc, heads = min(hpc, p.Hkv - head0);
      const uint32_t at = ring + slot * slot_bytes;
      const uint8_t* src = p.bounds + (int64_t)id * p.bounds_stride_block + (int64_t)head0 * p.bounds_stride_head;
      if (whole) {
        if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(valid * heads * 2 * kD));
        __syncwarp();
        if (lane < valid) bulk_g2s(at + lane * pitch, src, (uint32_t)(heads * 2 * kD), full, pol);
      } else {
        // lane = (page of a pair, piece of its 256 bytes)
        const uint64_t mine = reinterpret_cast<uint64_t>(src);
        for (int h = 0; h < heads; ++h) {
#pragma unroll
          for (int j = 0; j < kScoreTilePages / 2; ++j) {
            const int page = 2 * j + (lane >> 4);
            const uint64_t from = __shfl_sync(kFullMask, mine, page) + (uint64_t)((int64_t)h * p.bounds_stride_head) + (lane & 15) * 16;
            if (page < valid) cp_async16(at + page * pitch + h * 2 * kD + (lane & 15) * 16, reinterpret_cast<const void*>(from));
          }
        }
        if (lane == 0) tc::mbar_arrive(full);
      }
      if (lane < valid) {
        if (p.k_scale) {
          const float* ks = p.k_scale + (int64_t)id * p.ks_stride_block + (int64_t)head0 * p.ks_stride_head;
          for (int h = 0; h < heads; ++h) cp_async4(at + kScoreTilePages * pitch + (lane * hpc + h) * 4, ks + (int64_t)h * p.ks_stride_head);
        }
      }
      cp_async_arrive(full);
      slot += producers;
      if (slot >= p.slots) slot -= p.slots, phase ^= 1;
    }
    // Nobody leaves with a copy in flight.  The multiplying warps wait for every tile, but not after a wait of theirs
    // has run out; so each producer waits, bounded again, for its tiles that are the last in their slots (k: the
    // first one that it has not requested).
    for (int last = k - producers; last >= first && last + p.slots >= min(k, n_tiles); last -= producers) {
      if (!__all_sync(kFullMask, mbar_wait(smem_addr(&bar_full[last % p.slots]), (uint32_t)(last / p.slots) & 1))) {
        if (lane == 0 && p.status) atomicOr(p.status, PA_DEV_WAIT_TIMEOUT);
        break;
      }
    }
    return;
  }

  // -------------------------------------------------------------------- the multiplying warps
  // ---- pages without tokens: nothing to choose ((sequence, kv head, 1024 pages) after the other over the warps)
  const int parts = (p.width + 1023) >> 10;
  for (int64_t r = (int64_t)blockIdx.x * kScoreWarps + warp; r < (int64_t)p.S * parts * p.Hkv; r += (int64_t)gridDim.x * kScoreWarps) {
    const int sp = (int)(r / p.Hkv), h = (int)(r - (int64_t)sp * p.Hkv), s = sp / parts, beg = (sp - s * parts) << 10;
    float* out = p.scores + (int64_t)s * p.out_stride_seq + (int64_t)h * p.out_stride_head;
    for (int i = max(seq_pages[s], beg) + lane; i < min(p.width, beg + 1024); i += 32) out[i] = -INFINITY;
  }
  // A warp works for one kv head of the group and takes the tiles k with k % step == sub.
  const int g = lane >> 2, t = lane & 3;
  const int my_head = warp & (hpc - 1), sub = warp / hpc, step = kScoreWarps / hpc;
  Place a = at0;
  int k = 0;                          // tiles of the CTA before the segment
  int mine = sub, slot = sub;         // this warp's next tile and its slot
  uint32_t phase = 0;
  bool dead = false;                  // a wait ran out: go through the barriers, touch nothing
  // A segment's query rows, eight a warp (there are at most 64): a quad of lanes per row, lane t the 32 dims of its
  // quarter.  Padding rows repeat row 0, which changes no maximum.  They are requested a segment ahead:
  // 32 long sequences take 31.8 us so and 33.1 without, 256 of 1 024 to 4 096 tokens 23.4 and 24.5.
  static_assert(kScoreWarps * 8 >= kScoreMaxRows, "a warp's rows of the query are one group of eight");
  uint4 raw[4];
  float raw_scale = 1.0f;
  auto fetch_query = [&](const Place& at) {
    const int head0 = at.group * hpc, heads = min(hpc, p.Hkv - head0);
    const int r = warp * 8 + g, h = r / kRows;
    if (warp * 8 >= heads * kRows) return;
    int row = r - h * kRows;
    if (row >= p.rows) row = 0;
    const int64_t grow = (int64_t)(head0 + h) * p.rows + row;
    const uint8_t* src = p.q + (int64_t)at.seq * p.q_stride_seq;
    if (p.q_is_fp8) {
#pragma unroll
      for (int e = 0; e < 2; ++e) raw[e] = __ldg(reinterpret_cast<const uint4*>(src + grow * kD + t * 32) + e);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[e] = __ldg(reinterpret_cast<const uint4*>(src + grow * (kD * 2) + t * 64) + e);
    }
    if (p.q_quant_mode == PA_QUANT_PER_TENSOR) raw_scale = __ldg(p.q_scale);
    if (p.q_quant_mode == PA_QUANT_PER_TOKEN) raw_scale = __ldg(p.q_scale + (int64_t)at.seq * p.q_scale_stride_seq + grow);
  };
  constexpr bool kAhead = NB8 <= 4;   // (64 rows need the registers)
  if (kAhead && n_tiles > 0) fetch_query(a);
  while (k < n_tiles) {
    // a segment: tiles of one sequence and head group
    const int seq = a.seq, tile_a = a.tile;
    const int count = min(tile_off[seq + 1] - tile_off[seq] - tile_a, n_tiles - k);
    const int head0 = a.group * hpc, heads = min(hpc, p.Hkv - head0);
    const int pages = seq_pages[seq];

    // ---- the group's query rows.  Within each group of four dims the order is 0, 2, 1, 3 (what the e4m3
    // unpacking below yields).
    if (!kAhead) fetch_query(a);
    if (k > 0) tc::named_barrier_sync(1, kScoreWarps * 32);   // the rows of the segment before are no longer read
    if (warp * 8 < heads * kRows) {
      const int r = warp * 8 + g;
      float x[32];
      if (p.q_is_fp8) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t lo, hi;
            e4m3_to_f16(w[j], lo, hi);
            asm("{.reg .f16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}"
                : "=f"(x[e * 16 + j * 4]), "=f"(x[e * 16 + j * 4 + 1]) : "r"(lo));
            asm("{.reg .f16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}"
                : "=f"(x[e * 16 + j * 4 + 2]), "=f"(x[e * 16 + j * 4 + 3]) : "r"(hi));
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t w[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) x[e * 8 + j * 2] = bf16_lo_to_f32(w[j]), x[e * 8 + j * 2 + 1] = bf16_hi_to_f32(w[j]);
        }
      }
      float amax = 0.f;
      // An infinite element leaves the scale to the finite ones, which keep their digits.  Up to 32 rows a rare branch
      // looks for those (without it 23.2 us against 22.3 for 1 024 sequences of 128 to 512 tokens); with 64 rows that
      // branch makes the kernel spill (94.3 us against 88.0 for 32 sequences of 16 K to 64 K), so every element is asked.
      constexpr bool kAsk = NB8 > 4;
#pragma unroll
      for (int e = 0; e < 32; ++e) amax = max_or_nan(amax, kAsk && fabsf(x[e]) == INFINITY ? 0.f : fabsf(x[e]));
      amax = quad_max_or_nan(amax);
      if (!kAsk && __any_sync(kFullMask, amax == INFINITY)) {
        float finite = 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) finite = fmaxf(finite, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
        finite = quad_max_or_nan(finite);
        if (amax == INFINITY) amax = finite;
      }
      // power of two that brings the row's largest element into [2^14, 2^15)
      const int be = (int)((__float_as_uint(amax) >> 23) & 0xff);
      float pre = 1.0f, back = 1.0f;
      if (be < 255) {        // (zeros and subnormal rows: the largest power there is room for)
        pre = __uint_as_float((uint32_t)min(253, 254 + 14 - be) << 23);
        back = 1.0f / pre;   // a power of two
      } else if (amax != amax) {
        back = amax;         // (the halves of the operand below are zero for NaN)
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint4 v;
        v.x = pack_f16x2(x[e * 8] * pre, x[e * 8 + 2] * pre);
        v.y = pack_f16x2(x[e * 8 + 1] * pre, x[e * 8 + 3] * pre);
        v.z = pack_f16x2(x[e * 8 + 4] * pre, x[e * 8 + 6] * pre);
        v.w = pack_f16x2(x[e * 8 + 5] * pre, x[e * 8 + 7] * pre);
        *reinterpret_cast<uint4*>(smem + r * kScoreRowBytes + t * 64 + e * 16) = v;
      }
      if (t == 0) factor[r] = back * 256.0f * raw_scale * p.softmax_scale;   // 2^8: the bounds' f16 values are the codes times 2^-8
    }
    tc::named_barrier_sync(1, kScoreWarps * 32);

    // operand fragment of (row block n, smallest / largest m, chunk c): this thread's 16 dims, four k-steps
    // of (b0, b1); against the smallest codes the negative part of the query, against the largest the positive
    const uint8_t* qrow = smem + (my_head * kRows + g) * kScoreRowBytes + t * 32;
    auto load_q = [&](int n, int m, int c, uint4 (&v)[2]) {
      const uint4* src = reinterpret_cast<const uint4*>(qrow + n * 8 * kScoreRowBytes + c * 128);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 q = src[e];
        v[e] = m ? make_uint4(f16x2_max0(q.x), f16x2_max0(q.y), f16x2_max0(q.z), f16x2_max0(q.w))
                 : make_uint4(f16x2_min0(q.x), f16x2_min0(q.y), f16x2_min0(q.z), f16x2_min0(q.w));
      }
    };
    uint4 held[2][2][2];
    if (kKeep) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          load_q(0, m, c, held[m][c]);
          if (m == 0) {   // dims 0, 1 and 2, 3, as the convert instruction yields them
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 v = held[0][c][e];
              held[0][c][e] = make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632),
                                         __byte_perm(v.z, v.w, 0x5410), __byte_perm(v.z, v.w, 0x7632));
            }
          }
        }
      }
    }
    float* out = p.scores + (int64_t)seq * p.out_stride_seq + (int64_t)(head0 + my_head) * p.out_stride_head;
    a.tile += count;
    if (a.tile >= tile_off[seq + 1] - tile_off[seq]) next_seq(a);
    if (kAhead && k + count < n_tiles) fetch_query(a);
#pragma unroll 1
    while (mine < k + count) {
      if (!dead && !__all_sync(kFullMask, mbar_wait(smem_addr(&bar_full[slot]), phase))) {
        if (lane == 0 && p.status) atomicOr(p.status, PA_DEV_WAIT_TIMEOUT);
        dead = true;
      }
      if (my_head < heads && !dead) {
        const uint32_t tile = ring + slot * slot_bytes;
        const uint32_t row0 = tile + g * pitch + my_head * 2 * kD + t * 16, row1 = row0 + 8 * pitch;
        float acc[2][NB8][4];   // the two halves of the bound: two chains of products
#pragma unroll
        for (int n = 0; n < NB8; ++n)
#pragma unroll
          for (int m = 0; m < 2; ++m) acc[m][n][0] = acc[m][n][1] = acc[m][n][2] = acc[m][n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            uint4 qv[NB8][2];
#pragma unroll
            for (int n = 0; n < NB8; ++n) {
              if (kKeep) qv[n][0] = held[m][c][0], qv[n][1] = held[m][c][1];
              else load_q(n, m, c, qv[n]);
            }
            const uint4 r0 = lds128(row0 + m * kD + c * 64), r1 = lds128(row1 + m * kD + c * 64);
            const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              // (with one row block the unpacking, not the products, is the work: half of it goes to the
              // convert instructions, which run beside the ALUs)
              uint32_t a0, a1, a2, a3;
              if (kKeep && m == 0) {
                e4m3_to_f16(w0[e], a0, a2);
                e4m3_to_f16(w1[e], a1, a3);
              } else {
                a0 = e4m3_even_to_f16(w0[e]), a1 = e4m3_even_to_f16(w1[e]);
                a2 = e4m3_odd_to_f16(w0[e]), a3 = e4m3_odd_to_f16(w1[e]);
              }
#pragma unroll
              for (int n = 0; n < NB8; ++n) {
                const uint4 v = qv[n][e >> 1];
                mma_f16(acc[m][n], a0, a1, a2, a3, (e & 1) ? v.z : v.x, (e & 1) ? v.w : v.y);
              }
            }
          }
        }
        float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NB8; ++n) {
          const float2 f = *reinterpret_cast<const float2*>(factor + my_head * kRows + n * 8 + 2 * t);
          constexpr float kLow = kKeep ? 0x1p-8f : 1.0f;   // converted codes carry their true value
#pragma unroll
          for (int i = 0; i < 2; ++i)
            best[i] = max_or_nan(best[i], max_or_nan(fmaf(acc[0][n][2 * i], kLow, acc[1][n][2 * i]) * f.x,
                                                     fmaf(acc[0][n][2 * i + 1], kLow, acc[1][n][2 * i + 1]) * f.y));
        }
        best[0] = quad_max_or_nan(best[0]);
        best[1] = quad_max_or_nan(best[1]);
        const int in_tile = g + 8 * t, page = (tile_a + mine - k) * kScoreTilePages + in_tile;   // what lanes t = 0, 1 store
        if (t < 2 && page < pages) {
          const float ks = p.k_scale ? __uint_as_float(lds32(tile + kScoreTilePages * pitch + (in_tile * hpc + my_head) * 4)) : 1.0f;
          out[page] = (t ? best[1] : best[0]) * ks;
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(smem_addr(&bar_empty[slot]));
      mine += step;
      slot += step;
      if (slot >= p.slots) slot -= p.slots, phase ^= 1;
    }
    k += count;
  }
}

}  // namespace pa
