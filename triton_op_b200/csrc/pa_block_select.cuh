// Page selection: for every (sequence, kv head) the pages that its attention will read -- the first
// `keep_first` and the last `keep_last` pages of the context and, of the others, those with the
// highest scores, ties to the lower page, top_k pages in all -- written as a block table of its own
// in the order of the context, with the number of tokens those pages hold.
//
// One CTA per (sequence, kv head).  Scores become unsigned keys of the same order (NaN below
// everything).  The key of rank top_k is found by narrowing a key range: a histogram of 2048 equal
// bins over [smallest, largest] key, the bin in which the rank falls becomes the next range.  Bins
// over the ACTUAL range spread the shared-memory counters, where a fixed digit would count most
// pages of a head in two or three of them (their scores share sign and exponent); a 32-bit range is down
// to single keys after three rounds at most, and as a rule the search ends after two, as soon as the
// bin is taken whole.  Then one ordered pass writes the pages above the threshold and the first of those on it.
// Nothing here is a sum of floating-point numbers and counters are only added to: the same
// scores give the same table whatever the order of the threads.
#pragma once

#include "../../include/pa_decode_sm100.h"
#include "pa_common.cuh"
#include "pa_params.cuh"

namespace pa {

constexpr int kSelectThreads = 512;
constexpr int kSelectItems = 16;     // pages per thread and sweep
constexpr int kSelectSweep = kSelectThreads * kSelectItems;
constexpr int kSelectBins = 2048;

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

// Unsigned key with the order of the floats; NaN is below -inf.
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kSelectThreads)
pa_block_select_kernel(const __grid_constant__ BlockSelectParams p) {
  __shared__ int bins[kSelectBins];
  __shared__ int warp_sums[kSelectThreads / 32], warp_sums2[kSelectThreads / 32];
  __shared__ uint32_t warp_lo[kSelectThreads / 32], warp_hi[kSelectThreads / 32];
  __shared__ int found_bin, found_above, found_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = (int)blockIdx.x / p.Hkv, head = (int)blockIdx.x - seq * p.Hkv;
  grid_dependency_wait();
  grid_launch_dependents();
  const int ctx = p.context_lens[seq];
  const int64_t cap = (int64_t)p.width * p.block_size;
  const int tokens = ctx <= 0 ? 0 : (int)min(cap, (int64_t)ctx);
  if (ctx > cap && p.status && tid == 0) atomicOr(p.status, PA_DEV_CTX_TOO_LONG);
  const int pages = (int)(((int64_t)tokens + p.block_size - 1) / p.block_size);
  const int held = min(pages, p.top_k);
  if (head == 0 && tid == 0)   // every page but the last is full
    p.lengths[seq] = held == 0 ? 0 : (int)min((int64_t)0x7fffffff, (int64_t)held * p.block_size - ((int64_t)pages * p.block_size - tokens));
  const int32_t* table = p.block_tables + (int64_t)seq * p.bt_stride_seq;
  int32_t* out = p.tables + (int64_t)seq * p.out_stride_seq + (int64_t)head * p.out_stride_head;
  for (int i = held + tid; i < p.top_k; i += kSelectThreads) out[i] = 0;
  if (pages <= p.top_k) {
    for (int i = tid; i < pages; i += kSelectThreads) out[i] = __ldg(table + i);
    return;
  }

  // keep_first + keep_last <= top_k < pages, so the two ends do not meet
  const float* scores = p.scores + (int64_t)seq * p.sc_stride_seq + (int64_t)head * p.sc_stride_head;
  const int first = p.keep_first, last = pages - p.keep_last;   // pages [first, last) compete
  int need = p.top_k - p.keep_first - p.keep_last;              // for this many places
  const bool one_sweep = pages <= kSelectSweep;
  uint32_t keys[kSelectItems];
  // thread tid holds pages sweep + tid * kSelectItems + [0, kSelectItems)
  auto load = [&](int sweep) {
    const int at = sweep + tid * kSelectItems;
#pragma unroll
    for (int j = 0; j < kSelectItems; ++j) keys[j] = (at + j >= first && at + j < last) ? score_key(scores[at + j]) : 0u;
  };
  if (one_sweep) load(0);

  uint32_t lo = 0xffffffffu, hi = 0u;   // range of the competing keys
  for (int sweep = 0; sweep < pages; sweep += kSelectSweep) {
    if (!one_sweep) load(sweep);
    const int at = sweep + tid * kSelectItems;
#pragma unroll
    for (int j = 0; j < kSelectItems; ++j) {
      if (at + j >= first && at + j < last) lo = min(lo, keys[j]), hi = max(hi, keys[j]);
    }
  }
  lo = __reduce_min_sync(kFullMask, lo);
  hi = __reduce_max_sync(kFullMask, hi);
  if (lane == 0) warp_lo[warp] = lo, warp_hi[warp] = hi;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) lo = min(lo, warp_lo[w]), hi = max(hi, warp_hi[w]);

  // The `need` best of the keys in [lo, hi]; all keys above hi are taken already.  Ends with
  // threshold: keys > threshold are taken, and `ties` of those equal to it.
  uint32_t threshold = hi;
  int ties = 0;
  while (need > 0) {
    if (lo == hi) {        // what is left is one key
      threshold = lo;
      ties = need;
      break;
    }
    int shift = 0;
    while (((hi - lo) >> shift) >= (uint32_t)kSelectBins) ++shift;
    for (int i = tid; i < kSelectBins; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (int sweep = 0; sweep < pages; sweep += kSelectSweep) {
      if (!one_sweep) load(sweep);
      const int at = sweep + tid * kSelectItems;
#pragma unroll
      for (int j = 0; j < kSelectItems; ++j) {
        if (at + j >= first && at + j < last && keys[j] >= lo && keys[j] <= hi) atomicAdd(&bins[(keys[j] - lo) >> shift], 1);
      }
    }
    __syncthreads();
    // the bin that holds rank `need`, counted from the top: thread tid has the bins top - 4 tid - {0..3}
    constexpr int kPer = kSelectBins / kSelectThreads;
    int own[kPer], sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) own[j] = bins[kSelectBins - 1 - tid * kPer - j], sum += own[j];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFullMask, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < warp; ++w) before += warp_sums[w];
    if (before < need && before + sum >= need) {
      int above = before;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (above < need && above + own[j] >= need) {
          found_bin = kSelectBins - 1 - tid * kPer - j;
          found_above = above;
          found_count = own[j];
        }
        above += own[j];
      }
    }
    __syncthreads();
    const uint32_t bin_lo = lo + ((uint32_t)found_bin << shift);
    const uint32_t bin_hi = min(hi, bin_lo + ((1u << shift) - 1u));
    need -= found_above;
    if (need == found_count) {   // the whole bin is taken: everything from bin_lo up
      threshold = bin_lo;
      ties = 0x7fffffff;
      break;
    }
    lo = bin_lo;
    hi = bin_hi;
  }

  // ---- ordered pass: page i goes to place (taken pages before it)
  int placed = 0, tied = 0;     // over the sweeps so far
  for (int sweep = 0; sweep < pages; sweep += kSelectSweep) {
    if (!one_sweep) load(sweep);
    const int at = sweep + tid * kSelectItems;
    int above = 0, equal = 0;
    const bool any = p.top_k > p.keep_first + p.keep_last;
#pragma unroll
    for (int j = 0; j < kSelectItems; ++j) {
      const int i = at + j;
      if (i < pages && (i < first || i >= last)) ++above;
      else if (i < pages && any) above += keys[j] > threshold, equal += keys[j] == threshold;
    }
    int sum = above, sum2 = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFullMask, sum, o), v2 = __shfl_up_sync(kFullMask, sum2, o);
      if (lane >= o) sum += v, sum2 += v2;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = sum, warp_sums2[warp] = sum2;
    __syncthreads();
    int before = placed + sum - above, ties_before = tied + sum2 - equal;
    for (int w = 0; w < kSelectThreads / 32; ++w) {
      if (w < warp) before += warp_sums[w], ties_before += warp_sums2[w];
      placed += warp_sums[w], tied += warp_sums2[w];
    }
#pragma unroll
    for (int j = 0; j < kSelectItems; ++j) {
      const int i = at + j;
      bool take = false;
      if (i < pages && (i < first || i >= last)) take = true;
      else if (i < pages && any && keys[j] > threshold) take = true;
      else if (i < pages && any && keys[j] == threshold) {
        if (ties_before < ties) {
          const int place = before + min(ties_before, ties);
          if (place < p.top_k) out[place] = __ldg(table + i);
        }
        ++ties_before;
        continue;
      }
      if (take) {
        const int place = before + min(ties_before, ties);
        if (place < p.top_k) out[place] = __ldg(table + i);
        ++before;
      }
    }
  }
}

}  // namespace pa
