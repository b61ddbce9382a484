// Page selection: for every (sequence, kv head) the pages that its attention will read -- the first
// `keep_first` and the last `keep_last` pages of the context and, of the others, those with the
// highest scores, ties to the lower page, top_k pages in all -- written as a block table of its own
// in the order of the context, with the number of tokens those pages hold.
//
// One CTA per (sequence, kv head).  Scores become unsigned keys of the same order (NaN
// as -inf).  The key of rank top_k is found by narrowing a key range: a histogram of equal bins over
// [smallest, largest] key, then the bin in which the rank falls.  Bins over the ACTUAL range spread the
// shared-memory counters, where a fixed digit would count most pages of a head in two or three of
// them (their scores share sign and exponent), and leave few keys in the rank's bin: up to 32 of them
// are ranked outright by a warp, more make the next range.  Then one ordered pass writes the pages above
// the threshold and the first of those on it.  Nothing here is a sum of floating-point numbers and
// counters are only added to: the same scores give the same table whatever the order of the threads.
//
// What bounds it: 4 bytes per page and kv head, a few MB at most; it is the latency of one CTA's chain
// (lengths and scores, range, histogram, rank, ordered pass: six block barriers), and in wide tables the warps that
// hold the context: a warp owns neighbouring rows of the table's width, so those past a shorter context have none.  So keys stay in
// registers, a warp's pages are rows of 32 (coalesced loads, ballots give a page's place among
// the warp's), every warp combines the block's partial results for itself instead of waiting for
// one that does, and the CTA is as large as the table is wide.
#pragma once

#include "../../include/pa_decode_sm100.h"
#include "pa_common.cuh"
#include "pa_params.cuh"

namespace pa {

// Threads and pages per thread by the width of the table: a CTA holds THREADS * ITEMS pages at a time and
// sweeps over more than that.
constexpr int kSelectSmall = 128 * 4, kSelectMedium = 256 * 8, kSelectLarge = 256 * 32;

struct BlockSelectParams {
  const float* scores;         // [S, Hkv, >= pages]
  const int32_t* block_tables; // [S, width]
  const int32_t* context_lens; // [S]
  int32_t* tables;             // [S, Hkv, top_k]
  int32_t* lengths;            // [S]
  int32_t* status;
  int32_t S, Hkv, block_size, width, top_k, keep_first, keep_last;
  int64_t sc_stride_seq, sc_stride_head;
  int64_t bt_stride_seq;
  int64_t out_stride_seq, out_stride_head;
};

// Unsigned key with the order of the floats, NaN as -inf.  Two keys no score has mark the pages that do
// not compete: kKeyNone for places past the context, kKeyKept for the kept pages.
constexpr uint32_t kKeyNone = 0u, kKeyLowest = 0x007fffffu, kKeyKept = 0xffffffffu;
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);   // (the two zeros are one value)
  if ((u & 0x7fffffffu) > 0x7f800000u) return kKeyLowest;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS, ITEMS > 8 ? 4 : 1)
pa_block_select_kernel(const __grid_constant__ BlockSelectParams p) {
  constexpr int kWarps = THREADS / 32, kSweep = THREADS * ITEMS, kPer = 4, kBins = kPer * THREADS;
  __shared__ __align__(16) int bins[kBins];
  __shared__ uint32_t part_lo[32], part_hi[32];
  __shared__ int part_sum[32];
  __shared__ uint32_t part_pair[32];
  __shared__ uint32_t cand[32];
  __shared__ int found[4];   // bin, keys above it, keys in it; candidates stored
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = (int)blockIdx.x / p.Hkv, head = (int)blockIdx.x - seq * p.Hkv;
#pragma unroll
  for (int i = 0; i < kPer; ++i) bins[i * THREADS + tid] = 0;
  grid_dependency_wait();
  grid_launch_dependents();

  const float* scores = p.scores + (int64_t)seq * p.sc_stride_seq + (int64_t)head * p.sc_stride_head;
  uint32_t keys[ITEMS];
  // a warp's pages are ITEMS rows of 32: page of item j
  auto page_of = [&](int sweep, int j) -> int { return sweep + (warp * ITEMS + j) * 32 + lane; };
  // (the scores of a narrow table are requested before the length is known: the buffer has its full width)
  constexpr bool kEarly = ITEMS <= 8;
  const bool one_sweep = p.width <= kSweep;
  float early[kEarly ? ITEMS : 1];
  if (kEarly) {
#pragma unroll
    for (int j = 0; j < (kEarly ? ITEMS : 1); ++j) {
      const int i = page_of(0, j);
      early[j] = i < p.width ? scores[i] : 0.f;
    }
  }

  const int ctx = p.context_lens[seq];
  const int64_t cap = (int64_t)p.width * p.block_size;
  const int64_t tokens = ctx <= 0 ? 0 : min(cap, (int64_t)ctx);
  if (ctx > cap && p.status && tid == 0) atomicOr(p.status, PA_DEV_CTX_TOO_LONG);
  const int pages = (int)((tokens + p.block_size - 1) / p.block_size);
  const int held = min(pages, p.top_k);
  if (head == 0 && tid == 0)   // every page but the last is full
    p.lengths[seq] = held == 0 ? 0 : (int)min((int64_t)0x7fffffff, (int64_t)held * p.block_size - ((int64_t)pages * p.block_size - tokens));
  const int32_t* table = p.block_tables + (int64_t)seq * p.bt_stride_seq;
  int32_t* out = p.tables + (int64_t)seq * p.out_stride_seq + (int64_t)head * p.out_stride_head;
  for (int i = held + tid; i < p.top_k; i += THREADS) out[i] = 0;
  if (pages <= p.top_k) {
    for (int i = tid; i < pages; i += THREADS) out[i] = __ldg(table + i);
    return;
  }

  // keep_first + keep_last <= top_k < pages, so the two ends do not meet
  const int first = p.keep_first, last = pages - p.keep_last;   // pages [first, last) compete
  int need = p.top_k - p.keep_first - p.keep_last;              // for these places
  uint32_t lo = 0xffffffffu, hi = 0u;                           // range of the competing keys
  auto load = [&](int sweep) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int i = page_of(sweep, j);
      if (i >= first && i < last) {
        keys[j] = score_key(kEarly && one_sweep ? early[kEarly ? j : 0] : scores[i]);
        lo = min(lo, keys[j]), hi = max(hi, keys[j]);
      } else {
        keys[j] = i < pages ? kKeyKept : kKeyNone;
      }
    }
  };
  for (int sweep = 0; sweep < pages; sweep += kSweep) load(sweep);
  auto reload = [&](int sweep) {     // the same keys, the range as it has become
    const uint32_t keep_lo = lo, keep_hi = hi;
    load(sweep);
    lo = keep_lo, hi = keep_hi;
  };

  // keys above the threshold are taken, and the first `ties` of those equal to it (kept pages are above
  // any; with no place to compete for, they alone)
  uint32_t threshold = kKeyKept - 1u;
  int ties = 0;
  if (need > 0) {
    lo = __reduce_min_sync(kFullMask, lo);
    hi = __reduce_max_sync(kFullMask, hi);
    if (lane == 0) part_lo[warp] = lo, part_hi[warp] = hi;
    if (tid == 0) found[3] = 0;
    __syncthreads();
    lo = __reduce_min_sync(kFullMask, lane < kWarps ? part_lo[lane] : 0xffffffffu);
    hi = __reduce_max_sync(kFullMask, lane < kWarps ? part_hi[lane] : 0u);

    while (true) {
      if (lo == hi) {        // what is left is one key
        threshold = lo;
        ties = need;
        break;
      }
      // the smallest shift that maps the range into the bins
      const int width_bits = 32 - __clz((int)(hi - lo));
      constexpr int kBinBits = 31 - __builtin_clz(kBins);
      const int shift = max(width_bits - kBinBits, 0);
      for (int sweep = 0; sweep < pages; sweep += kSweep) {
        if (!one_sweep) reload(sweep);
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
          if (keys[j] >= lo && keys[j] <= hi) atomicAdd(&bins[(keys[j] - lo) >> shift], 1);
        }
      }
      __syncthreads();
      // the bin that holds rank `need`, counted from the top: thread tid has four bins from kBins - 1 - 4 tid down
      const int4 own = *reinterpret_cast<const int4*>(&bins[kBins - 4 - tid * kPer]);
      const int sum = own.x + own.y + own.z + own.w;
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFullMask, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) part_sum[warp] = incl;
      __syncthreads();
      const int before = incl - sum + (int)__reduce_add_sync(kFullMask, lane < warp ? (unsigned)part_sum[lane] : 0u);
      *reinterpret_cast<int4*>(&bins[kBins - 4 - tid * kPer]) = make_int4(0, 0, 0, 0);   // for the next round
      if (before < need && before + sum >= need) {
        const int top[4] = {own.w, own.z, own.y, own.x};
        int above = before;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (above < need && above + top[j] >= need) {
            found[0] = kBins - 1 - tid * kPer - j;
            found[1] = above;
            found[2] = top[j];
          }
          above += top[j];
        }
      }
      __syncthreads();
      const uint32_t bin_lo = lo + ((uint32_t)found[0] << shift);
      const uint32_t bin_hi = min(hi, bin_lo + ((1u << shift) - 1u));
      const int inside = found[2];
      need -= found[1];
      if (need == inside) {   // the whole bin is taken: everything from bin_lo up
        threshold = bin_lo;
        ties = 0x7fffffff;
        break;
      }
      lo = bin_lo;
      hi = bin_hi;
      if (inside > 32 || lo == hi) continue;
      // few are left: gather them, and every warp finds the need-th for itself (ties share a key, so
      // the order in which they were gathered does not matter)
      for (int sweep = 0; sweep < pages; sweep += kSweep) {
        if (!one_sweep) reload(sweep);
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
          if (keys[j] >= lo && keys[j] <= hi) cand[atomicAdd(&found[3], 1) & 31] = keys[j];
        }
      }
      __syncthreads();
      const uint32_t mine = lane < inside ? cand[lane] : 0u;
      int above = 0, equal = 0;
      for (int l = 0; l < inside; ++l) {
        const uint32_t other = __shfl_sync(kFullMask, mine, l);
        above += other > mine;
        equal += other == mine;
      }
      const unsigned hit = __ballot_sync(kFullMask, lane < inside && above < need && above + equal >= need);
      const int src = __ffs((int)hit) - 1;
      threshold = __shfl_sync(kFullMask, mine, src);
      ties = need - __shfl_sync(kFullMask, above, src);
      break;
    }
  }
  // ---- ordered pass: a taken page goes to the place that the taken pages before it leave
  // (places first get the number of their page, in shared memory if top_k of them fit, and the page ids are
  // looked up for all together: a look-up per row would wait for memory row after row)
  int* list = p.top_k <= kBins ? bins : out;
  const unsigned below = (1u << lane) - 1u;
  int placed = 0, tied = 0;     // over the sweeps so far: pages above the threshold (or kept), pages on it
  for (int sweep = 0; sweep < pages; sweep += kSweep) {
    if (!one_sweep) reload(sweep);
    int n_above = 0, n_equal = 0;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) n_above += keys[j] > threshold, n_equal += keys[j] == threshold;
    const uint32_t sums = __reduce_add_sync(kFullMask, (uint32_t)n_above | ((uint32_t)n_equal << 16));   // at most kSweep <= 8192 each
    if (sweep > 0) __syncthreads();
    if (lane == 0) part_pair[warp] = sums;
    __syncthreads();
    const uint32_t pair = lane < kWarps ? part_pair[lane] : 0u;
    const uint32_t mine = __reduce_add_sync(kFullMask, lane < warp ? pair : 0u), all = __reduce_add_sync(kFullMask, pair);
    int before = placed + (int)(mine & 0xffffu), ties_before = tied + (int)(mine >> 16);
    placed += (int)(all & 0xffffu);
    tied += (int)(all >> 16);
    if (sums == 0) continue;   // nothing of this warp's
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const unsigned any = __ballot_sync(kFullMask, keys[j] >= threshold);
      if (any == 0) continue;
      const unsigned is_above = __ballot_sync(kFullMask, keys[j] > threshold), is_equal = any & ~is_above;
      const int rank_equal = ties_before + __popc(is_equal & below);
      if (((is_above >> lane) & 1u) || (((is_equal >> lane) & 1u) && rank_equal < ties)) {
        const int place = before + __popc(is_above & below) + min(rank_equal, ties);
        if (place < p.top_k) list[place] = page_of(sweep, j);
      }
      before += __popc(is_above);
      ties_before += __popc(is_equal);
    }
  }
  __syncthreads();
  for (int i = tid; i < p.top_k; i += THREADS) out[i] = __ldg(table + list[i]);
}

}  // namespace pa
