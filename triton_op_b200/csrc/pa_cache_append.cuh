// Append to a cache with one scale for each (page, kv head): the new tokens of every sequence are
// quantised to e4m3 and stored behind the tokens that its pages hold already.
//
// For a page and kv head that receives the rows x_i (keys and values separately):
//   want  = the smallest power of two >= max|x| / 448 (finite elements; at least 2^-40)
//   scale = want                        where the rows begin the page
//         = max(old scale, want)        where the page holds tokens already (an old scale that is no
//                                       power of two counts as the next one)
//   codes of the page := e4m3(code * (old scale / scale))   where the scale grew
//   code_i = e4m3(x_i / scale), saturating
// A scale that is a power of two costs no precision (e4m3 keeps its four significant bits wherever
// the value lies), and it makes growing a page a shift of exponents: only codes that become
// subnormal are rounded again, however often a page grows.  With a per-tensor scale (read, never
// written) only the last line applies.  Optionally the smallest and largest key code of each head
// dim are kept per (page, kv head), as the page scores need them; rounding is monotone, so they
// are found on the bf16 inputs and rounded once.
//
// A unit of work is (page, kv head, key or value), and all of it belongs to one group of warps: the
// scale is a maximum over every row the page gets, and two writers of one page would race on it.
// Each warp takes 16 consecutive slots of the page, whose rows stay in registers between the
// maximum and the store.  A page of 1024 tokens is 64 such runs.  Eight warps take eight each and read
// the rows twice; where there are fewer pages than could keep the GPU busy that way, a page is shared by
// a cluster of eight CTAs that find the maximum through each other's shared memory (9 us against 17 for
// two prompts of 2 200 and 3 300 tokens, one kv head, when that was chosen, 5.9 since; for many pages the clusters'
// barriers cost more than they save); with a few rows per sequence, where most warps would have nothing to do, four
// warps take the runs in turn.  A page of 64 has four warps, or one where each gets a few rows.  Keys are
// stored as 16-byte chunks [d/16][token][16], values as 16 tokens of a head dim, 16 bytes too;
// values of a run that is not whole are merged with the bytes that are there.
// What bounds it: 512 bytes read and 256 written per (token, kv head).  A prompt in pages of 16 fills nothing alone:
// 59 % of the issue slots, 56 % of the ALU pipe, 71 % of the copy bandwidth, its warps waiting for their loads more than
// for anything else.  16 000 tokens of eight kv heads take 22 us in pages of 16, 25 in pages of 64 and 33 in
// pages of 1024 (15 at the copy bandwidth).  A row for each of 64 sequences takes 4.3, 5.1 and 9.1 us: launch
// latency and one chain of loads, which is why whatever a page holds already is asked for at once.
#pragma once

#include <cooperative_groups.h>

#include "../../include/pa_decode_sm100.h"
#include "pa_common.cuh"
#include "pa_params.cuh"

namespace pa {

constexpr float kAppendMinScale = 0x1p-40f;
constexpr int kAppendMaxSeqs = 8192;     // sequences whose index a CTA holds (one int each)

struct CacheAppendParams {
  const uint8_t* key;          // [T, Hkv, 128] bf16
  const uint8_t* value;
  uint8_t* key_cache;
  uint8_t* value_cache;
  float* k_scale;              // [NB, Hkv] by strides (written), or one value (read)
  float* v_scale;
  uint8_t* bounds;             // [NB, Hkv, 2, 128] e4m3, or null
  const int32_t* block_tables; // [S, width]
  const int32_t* context_lens; // [S]: lengths with the new tokens
  const int32_t* row_start;    // [S + 1]: the sequence's first row in key / value
  int32_t* status;
  int32_t T, S, Hkv, num_blocks, width, v_trans;
  int64_t key_stride_tok, key_stride_head;       // elements
  int64_t value_stride_tok, value_stride_head;
  int64_t kc_stride_block, kc_stride_head;       // bytes
  int64_t vc_stride_block, vc_stride_head;
  int64_t ks_stride_block, ks_stride_head;       // elements
  int64_t b_stride_block, b_stride_head;         // bytes
  int64_t bt_stride_seq;
};

// Four e4m3 codes times a factor, rounded to e4m3 again.
__device__ __forceinline__ uint32_t rescale_e4m3x4(uint32_t w, float f) {
  uint32_t lo, hi;
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
  float x0, x1, x2, x3;
  asm("{.reg .f16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(x0), "=f"(x1) : "r"(lo));
  asm("{.reg .f16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(x2), "=f"(x3) : "r"(hi));
  return pack_e4m3x4(x0 * f, x1 * f, x2 * f, x3 * f);
}
__device__ __forceinline__ uint4 rescale_e4m3x16(uint4 v, float f) {
  return make_uint4(rescale_e4m3x4(v.x, f), rescale_e4m3x4(v.y, f), rescale_e4m3x4(v.z, f), rescale_e4m3x4(v.w, f));
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
  uint32_t h;
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %1; cvt.rn.f16x2.e4m3x2 %0, a;}" : "=r"(h) : "r"(byte & 0xffu));
  float x;
  asm("{.reg .f16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, a;}" : "=f"(x) : "r"(h));
  return x;
}
// Largest |x| of two packed bf16 as a bf16 bit pattern per half; NaN and infinity count as zero.
__device__ __forceinline__ uint32_t finite_abs2(uint32_t w) {
  const uint32_t a = w & 0x7fff7fffu;
  uint32_t lo = a & 0xffffu, hi = a >> 16;
  lo = lo >= 0x7f80u ? 0u : lo;
  hi = hi >= 0x7f80u ? 0u : hi;
  return lo | (hi << 16);
}
// The smallest power of two s with amax <= 448 s, at least 2^-40.  amax is a finite bf16 value.
__device__ __forceinline__ float page_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) + ((u & 0x7fffffu) > 0x600000u ? 1 : 0) - 8;   // 448 = 1.75 * 2^8
  return __uint_as_float((uint32_t)max(e, 127 - 40) << 23);
}
__device__ __forceinline__ uint32_t bf16x2_min(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t bf16x2_max(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The larger magnitude of two, per half (the sign is of no use); passes over NaN.
__device__ __forceinline__ uint32_t bf16x2_max_abs(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t bf16x2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two words of bf16 pairs -> four e4m3 codes of x / scale.  A page's scale is a power of two, so its
// reciprocal and the product are exact, in bf16 too (what underflows there is far below e4m3's
// smallest code); a per-tensor scale may be anything and is divided by.
template <bool DIVIDE>
__device__ __forceinline__ uint32_t quantise_four(uint32_t w0, uint32_t w1, float scale, float inv) {
  if (DIVIDE)
    return pack_e4m3x4(__fdiv_rn(bf16_lo_to_f32(w0), scale), __fdiv_rn(bf16_hi_to_f32(w0), scale),
                       __fdiv_rn(bf16_lo_to_f32(w1), scale), __fdiv_rn(bf16_hi_to_f32(w1), scale));
  const uint32_t inv2 = (__float_as_uint(inv) >> 16) | (__float_as_uint(inv) & 0xffff0000u);
  const uint32_t s0 = bf16x2_mul(w0, inv2), s1 = bf16x2_mul(w1, inv2);
  return pack_e4m3x4(bf16_lo_to_f32(s0), bf16_hi_to_f32(s0), bf16_lo_to_f32(s1), bf16_hi_to_f32(s1));
}
// The smallest power of two >= s, for a positive s (what a page's scale becomes if it came as none).
__device__ __forceinline__ float up_to_power(float s) {
  const uint32_t u = __float_as_uint(s);
  return (u & 0x7fffffu) == 0u ? s : __uint_as_float(min((u >> 23) + 1u, 254u) << 23);
}

// Brings a page's codes to a larger scale: runs first, first + WPU, ... of 16 slots.  A rare path, out
// of line so that the common one keeps its registers, but one that a step over many pages nearly always
// takes somewhere: a run's four pieces (two where a page is one run) are read before the first is written, so that
// their latencies overlap; more at a time cost the kernel registers, and a prompt 1 to 5 % of its time.
// Each thread touches the 16-byte pieces that it writes in the kernel below, so nothing has to be
// waited for in between.
template <int BS, int WPU>
static __device__ __noinline__ void rescale_runs(uint8_t* cache, bool is_v, bool v_trans, int first, float ratio, int lane) {
  constexpr int kAtOnce = BS == 16 ? 2 : 4;
  auto piece = [&](int run, int e) -> uint4* {
    const int d = 4 * lane + e;
    return reinterpret_cast<uint4*>(
        is_v ? (v_trans ? cache + ((int64_t)run * kD + d) * 16 : cache + (int64_t)d * BS + run * 16)
             : cache + ((int64_t)(lane >> 2) * BS + run * 16 + 4 * e + (lane & 3)) * 16);
  };
#pragma unroll 1
  for (int run = first; run < BS / 16; run += WPU) {
#pragma unroll
    for (int at = 0; at < 4; at += kAtOnce) {
      uint4 was[kAtOnce];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) was[e] = *piece(run, at + e);
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) *piece(run, at + e) = rescale_e4m3x16(was[e], ratio);
    }
  }
}

// BS: tokens per page.  WPU: warps per unit.  PER_BLOCK: scales per (page, kv head), else per tensor.
// CLUSTER: CTAs that share a unit.
template <int BS, int WPU, bool PER_BLOCK, int CLUSTER = 1>
__global__ void __launch_bounds__(WPU / CLUSTER > 4 ? WPU / CLUSTER * 32 : 128, WPU > 4 ? 2 : 5)
pa_cache_append_kernel(const __grid_constant__ CacheAppendParams p) {
  constexpr int kCtaWarps = WPU / CLUSTER;                          // warps of a unit in one CTA
  constexpr int kThreads = kCtaWarps > 4 ? kCtaWarps * 32 : 128;
  constexpr int kUnits = CLUSTER > 1 ? 1 : kThreads / 32 / WPU;     // units a CTA (or cluster) works on at a time
  constexpr int kRuns = BS / 16;                                    // 16-slot runs of a page
  constexpr int kPerWarp = (kRuns + WPU - 1) / WPU;                 // ... that a warp takes
  extern __shared__ int index_smem[];
  int* unit_off = index_smem;          // [S + 1] pages touched before each sequence
  __shared__ int scan[32];
  __shared__ uint32_t red_max[kThreads / 32];
  __shared__ uint4 red_bounds[kCtaWarps][32];
  __shared__ uint32_t cta_max;                                      // CLUSTER: this CTA's share
  __shared__ uint4 cta_bounds[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int team = (int)blockIdx.x / CLUSTER, teams = (int)gridDim.x / CLUSTER, rank = (int)blockIdx.x - team * CLUSTER;
  const int sub = CLUSTER > 1 ? rank * kCtaWarps + warp : warp % WPU;   // warp inside its unit

  grid_dependency_wait();
  // rows of a sequence: [first row, count), and its first new token's position
  auto rows_of = [&](int s, int& row, int& count, int& pos, bool report) {
    const int a = p.row_start[s], b = p.row_start[s + 1], len = p.context_lens[s];
    row = min(max(a, 0), p.T);
    const int end = min(max(b, row), p.T);
    count = end - row;
    bool bad = a < 0 || b > p.T || b < a;
    if (count > len) {       // more rows than tokens: the first ones have no place
      bad = bad || count > 0;
      row += count - max(len, 0);
      count = max(len, 0);
    }
    pos = max(len, 0) - count;
    const int64_t cap = (int64_t)p.width * BS;
    if (pos + (int64_t)count > cap) {   // tokens past the table have no page
      count = (int)max((int64_t)0, cap - pos);
      if (report && p.status) atomicOr(p.status, PA_DEV_CTX_TOO_LONG);
    }
    if (bad && report && p.status) atomicOr(p.status, PA_DEV_BAD_RANGE);
  };
  // ---- pages touched, summed over the sequences (every CTA for itself: S is small)
  {
    const int chunk = (p.S + kThreads - 1) / kThreads;
    const int beg = min(tid * chunk, p.S), end = min(beg + chunk, p.S);
    int sum = 0;
    for (int s = beg; s < end; ++s) {
      int row, count, pos;
      rows_of(s, row, count, pos, blockIdx.x == 0);
      const int n = count > 0 ? (pos + count - 1) / BS - pos / BS + 1 : 0;
      unit_off[s + 1] = n;
      sum += n;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFullMask, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    if (tid == 0) unit_off[0] = 0;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < warp; ++w) run += scan[w];
    for (int s = beg; s < end; ++s) {
      run += unit_off[s + 1];
      unit_off[s + 1] = run;
    }
    __syncthreads();
  }
  // (32-bit unit numbers: the host refuses batches that could have more than 2^30 units)
  const uint32_t units = (uint32_t)min((int64_t)unit_off[p.S] * p.Hkv * 2, (int64_t)1 << 30);

  // A unit, decoded: ((page of the sequence, sequence), head, key or value), the last fastest.  The next
  // unit is decoded, and its block-table entry requested, while the rows of the current one are on
  // their way: of the chain sequence -> page id -> rows only the rows are waited for.
  struct Unit {
    bool live, is_v;
    int head, o0, o1;      // slots [o0, o1) of the page receive rows row0 ..
    int row0, blk;
  };
  auto decode = [&](uint32_t u) -> Unit {
    Unit n;
    n.live = u < units;
    n.is_v = (u & 1u) != 0;
    const uint32_t ph = n.live ? u >> 1 : 0u;
    const int touched = (int)(ph / (uint32_t)p.Hkv);
    n.head = (int)(ph - (uint32_t)touched * p.Hkv);
    n.o0 = n.o1 = n.row0 = n.blk = 0;
    if (!n.live) return n;
    int lo = 0, hi = p.S;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (unit_off[mid] <= touched) lo = mid; else hi = mid;
    }
    int row, count, pos;
    rows_of(lo, row, count, pos, false);
    const int page = pos / BS + (touched - unit_off[lo]);
    n.blk = p.block_tables[(int64_t)lo * p.bt_stride_seq + page];
    n.o0 = max(pos - page * BS, 0);
    n.o1 = min(BS, pos + count - page * BS);
    n.row0 = row + (page * BS + n.o0 - pos);
    return n;
  };
  const uint32_t in_team = CLUSTER > 1 ? 0u : (uint32_t)(warp / WPU);
  Unit next = decode(team * kUnits + in_team);
  for (uint32_t u0 = team * kUnits; u0 < units; u0 += teams * kUnits) {
    const Unit cur = next;
    bool live = cur.live;
    const bool is_v = cur.is_v;
    const int head = cur.head, o0 = cur.o0, o1 = cur.o1, row0 = cur.row0;
    const uint8_t* src = (is_v ? p.value : p.key) +
                         2 * ((int64_t)row0 * (is_v ? p.value_stride_tok : p.key_stride_tok) +
                              (int64_t)head * (is_v ? p.value_stride_head : p.key_stride_head));
    const int64_t tok_bytes = 2 * (is_v ? p.value_stride_tok : p.key_stride_tok);
    // keys: lane = (chunk c of 16 dims, phase f), slots f, f + 4, f + 8, f + 12 of a run, 32 bytes each
    // values: lane = head dims 4 lane .. 4 lane + 3 of every slot of a run, 8 bytes each
    const int c = lane >> 2, f = lane & 3;
    uint32_t raw[32];     // the warp's (last) run: keys [slot f + 4 m][8 words], values [slot][2 words]
    auto load_run = [&](int run) {
      if (is_v) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int o = run * 16 + i;
          const uint2 v = (o >= o0 && o < o1) ? __ldg(reinterpret_cast<const uint2*>(src + (int64_t)(o - o0) * tok_bytes) + lane) : make_uint2(0u, 0u);
          raw[2 * i] = v.x, raw[2 * i + 1] = v.y;
        }
      } else {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int o = run * 16 + 4 * m + f;
          const bool in = o >= o0 && o < o1;
          const uint4* at = reinterpret_cast<const uint4*>(src + (int64_t)(o - o0) * tok_bytes + c * 32);
          const uint4 a = in ? __ldg(at) : make_uint4(0u, 0u, 0u, 0u), b = in ? __ldg(at + 1) : make_uint4(0u, 0u, 0u, 0u);
          raw[8 * m] = a.x, raw[8 * m + 1] = a.y, raw[8 * m + 2] = a.z, raw[8 * m + 3] = a.w;
          raw[8 * m + 4] = b.x, raw[8 * m + 5] = b.y, raw[8 * m + 6] = b.z, raw[8 * m + 7] = b.w;
        }
      }
    };
    // runs of the page that receive rows: [run0, run1); this warp takes sub, sub + WPU, ... of all runs
    const int run0 = o0 >> 4, run1 = o1 > o0 ? ((o1 - 1) >> 4) + 1 : run0;
    auto mine = [&](int k) -> int { return sub + k * WPU; };
    int loaded = -1;
    const int first = mine(kPerWarp > 1 && run0 > sub ? (run0 - sub + WPU - 1) / WPU : 0);   // the warp's first run with rows
    if (first >= run0 && first < run1) {
      loaded = first;
      load_run(loaded);
    }
    next = decode(u0 + teams * kUnits + in_team);
    int blk = cur.blk;
    if ((unsigned)blk >= (unsigned)p.num_blocks) {
      if (live && lane == 0 && p.status) atomicOr(p.status, PA_DEV_BAD_PAGE_ID);
      live = false;
      blk = 0;
    }
    uint8_t* cache = is_v ? p.value_cache + (int64_t)blk * p.vc_stride_block + (int64_t)head * p.vc_stride_head
                          : p.key_cache + (int64_t)blk * p.kc_stride_block + (int64_t)head * p.kc_stride_head;
    float* scale_at = (is_v ? p.v_scale : p.k_scale) + (PER_BLOCK ? (int64_t)blk * p.ks_stride_block + (int64_t)head * p.ks_stride_head : 0);
    const float old_scale = live ? *scale_at : 1.0f;
    const bool want_bounds = p.bounds != nullptr && !is_v;
    const bool fresh = o0 == 0;
    // the page's bounds of head dims 4 lane .. 4 lane + 3, asked for with its scale
    uint32_t* bounds_at = want_bounds ? reinterpret_cast<uint32_t*>(p.bounds + (int64_t)blk * p.b_stride_block + (int64_t)head * p.b_stride_head) + lane : nullptr;
    uint32_t old_lo = 0, old_hi = 0;
    if (want_bounds && live && !fresh && sub == 0) old_lo = bounds_at[0], old_hi = bounds_at[kD / 4];

    auto v_piece = [&](int run, int e) -> uint4* {      // where the codes of head dim 4 lane + e, slots of a run, are
      const int d = 4 * lane + e;
      return reinterpret_cast<uint4*>(p.v_trans ? cache + ((int64_t)run * kD + d) * 16 : cache + (int64_t)d * BS + run * 16);
    };
    auto partial = [&](int run) -> bool { return run * 16 < o0 || run * 16 + 16 > o1; };
    // Registers that keys use for the smallest (0 .. 7) and largest (8 .. 15) of a lane's head dims, and
    // values for the codes that share a run with new ones.  Those are asked for here, with the scale: after
    // the barrier below they would be read from sectors that another warp has just written half of, which took
    // 67 us where this takes 49 (64 sequences of 448 rows into pages of 64, the first page begun inside a run; 73 and 49 for 1 to 900 rows)
    uint32_t ext[16];
    // (A page of 16 belongs to one warp, which reads its codes when it needs them: the registers are worth more.)
    constexpr bool kEarly = BS > 16;
    int held = -1;                                      // the run whose codes are in ext
    if (!is_v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) ext[e] = 0x7f807f80u, ext[8 + e] = 0xff80ff80u;   // +inf, -inf
    } else if (kEarly && live && run1 > run0) {
      if (partial(run0) && run0 % WPU == sub) held = run0;
      else if (partial(run1 - 1) && (run1 - 1) % WPU == sub) held = run1 - 1;
      if (held >= 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint4 was = *v_piece(held, e);
          ext[4 * e] = was.x, ext[4 * e + 1] = was.y, ext[4 * e + 2] = was.z, ext[4 * e + 3] = was.w;
        }
      }
    }

    // ---- the largest finite |x|, and the smallest and largest key of every head dim
    uint32_t top = 0;
#pragma unroll 1
    for (int k = 0; k < kPerWarp; ++k) {
      const int run = mine(k);
      if (run < run0 || run >= run1) continue;
      if (run != loaded) {
        load_run(run);
        loaded = run;
      }
      // non-negative bf16 bit patterns order like integers; infinity and NaN lie above all others.  A key's
      // largest magnitude is that of its bounds (which pass over NaN).
      uint32_t any = 0;
      if (is_v) {
#pragma unroll
        for (int e = 0; e < 32; ++e) any = bf16x2_max_abs(any, raw[e]);
        any &= 0x7fff7fffu;
      } else {
        uint32_t lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] = 0x7f807f80u, hi[e] = 0xff80ff80u;   // +inf, -inf
        bool some = run * 16 >= o0 && run * 16 + 16 <= o1;   // a whole run
        if (some) {
#pragma unroll
          for (int e = 0; e < 32; ++e) lo[e & 7] = bf16x2_min(lo[e & 7], raw[e]), hi[e & 7] = bf16x2_max(hi[e & 7], raw[e]);
        } else {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const int o = run * 16 + 4 * m + f;
            if (o >= o0 && o < o1) {
              some = true;
#pragma unroll
              for (int e = 0; e < 8; ++e) lo[e] = bf16x2_min(lo[e], raw[8 * m + e]), hi[e] = bf16x2_max(hi[e], raw[8 * m + e]);
            }
          }
        }
        if (some) {
#pragma unroll
          for (int e = 0; e < 8; ++e) any = __vmaxu2(any, __vmaxu2(lo[e] & 0x7fff7fffu, hi[e] & 0x7fff7fffu));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ext[e] = bf16x2_min(ext[e], lo[e]), ext[8 + e] = bf16x2_max(ext[8 + e], hi[e]);
      }
      if ((any & 0xffffu) >= 0x7f80u || (any >> 16) >= 0x7f80u) {
        any = 0;
#pragma unroll
        for (int e = 0; e < 32; ++e) any = __vmaxu2(any, finite_abs2(raw[e]));
      }
      top = __vmaxu2(top, any);
    }
    uint32_t top1 = __reduce_max_sync(kFullMask, max(top & 0xffffu, top >> 16));
    // The bounds over the four lanes of a chunk, halved at each step: lane f keeps words 2 f, 2 f + 1 of
    // the chunk's eight, which are head dims 4 lane .. 4 lane + 3 (12 exchanges; 32 if all lanes kept all).
    uint4 bound = make_uint4(0x7f807f80u, 0x7f807f80u, 0xff80ff80u, 0xff80ff80u);   // min, min, max, max
    auto join = [](const uint4& a, const uint4& b) -> uint4 {
      return make_uint4(bf16x2_min(a.x, b.x), bf16x2_min(a.y, b.y), bf16x2_max(a.z, b.z), bf16x2_max(a.w, b.w));
    };
    if (want_bounds) {
      const bool up2 = (f & 2) != 0, up1 = (f & 1) != 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t l = __shfl_xor_sync(kFullMask, up2 ? ext[e] : ext[e + 4], 2);
        const uint32_t h = __shfl_xor_sync(kFullMask, up2 ? ext[e + 8] : ext[e + 12], 2);
        ext[e] = bf16x2_min(up2 ? ext[e + 4] : ext[e], l);
        ext[e + 8] = bf16x2_max(up2 ? ext[e + 12] : ext[e + 8], h);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t l = __shfl_xor_sync(kFullMask, up1 ? ext[e] : ext[e + 2], 1);
        const uint32_t h = __shfl_xor_sync(kFullMask, up1 ? ext[e + 8] : ext[e + 10], 1);
        ext[e] = bf16x2_min(up1 ? ext[e + 2] : ext[e], l);
        ext[e + 8] = bf16x2_max(up1 ? ext[e + 10] : ext[e + 8], h);
      }
      bound = make_uint4(ext[0], ext[1], ext[8], ext[9]);
    }
    if (WPU > 1) {   // over the warps of the unit (a CTA, or a cluster, then has one unit)
      if (lane == 0) red_max[warp] = top1;
      if (want_bounds) red_bounds[warp % kCtaWarps][lane] = bound;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kCtaWarps; ++w) top1 = max(top1, red_max[w]);
      if (want_bounds && warp == 0) {
#pragma unroll 4
        for (int w = 1; w < kCtaWarps; ++w) bound = join(bound, red_bounds[w][lane]);
      }
      if constexpr (CLUSTER > 1) {
        namespace cg = cooperative_groups;
        const cg::cluster_group cluster = cg::this_cluster();
        if (warp == 0) {
          if (lane == 0) cta_max = top1;
          if (want_bounds) cta_bounds[lane] = bound;
        }
        cluster.sync();
        const uint32_t theirs = lane < CLUSTER ? *cluster.map_shared_rank(&cta_max, lane) : 0u;
        top1 = __reduce_max_sync(kFullMask, theirs);
        if (want_bounds && sub == 0) {
#pragma unroll
          for (int r = 1; r < CLUSTER; ++r) bound = join(bound, *cluster.map_shared_rank(&cta_bounds[lane], r));
        }
      }
    }
    float scale = old_scale, ratio = 1.0f;
    bool grew = false;
    if (PER_BLOCK) {
      const float want = page_scale(__uint_as_float(top1 << 16));
      scale = fresh ? want : fmaxf(up_to_power(old_scale), want);
      grew = !fresh && scale != old_scale;
      if (grew) ratio = __fdiv_rn(old_scale, scale);
    }
    if (live && o1 > o0) {
      const float inv = 1.0f / scale;
      if (PER_BLOCK && grew) rescale_runs<BS, WPU>(cache, is_v, p.v_trans != 0, sub, ratio, lane);
      auto four = [&](uint32_t w0, uint32_t w1) -> uint32_t { return quantise_four<!PER_BLOCK>(w0, w1, scale, inv); };
#pragma unroll 1
      for (int k = kPerWarp - 1; k >= 0; --k) {   // backwards: the last run's rows are still here
        const int run = mine(k);
        if (run < run0 || run >= run1) continue;
        if (run != loaded) {
          load_run(run);
          loaded = run;
        }
        if (!is_v) {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const int o = run * 16 + 4 * m + f;
            uint4* dst = reinterpret_cast<uint4*>(cache + ((int64_t)c * BS + o) * 16);
            if (o >= o0 && o < o1) {
              *dst = make_uint4(four(raw[8 * m], raw[8 * m + 1]), four(raw[8 * m + 2], raw[8 * m + 3]),
                                four(raw[8 * m + 4], raw[8 * m + 5]), four(raw[8 * m + 6], raw[8 * m + 7]));
            }
          }
        } else {
          const int a = max(o0 - run * 16, 0), b = min(o1 - run * 16, 16);   // slots [a, b) of the run are new
          uint32_t qv[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) qv[i] = four(raw[2 * i], raw[2 * i + 1]);
          auto word = [&](int e, int j) -> uint32_t {       // the new codes of head dim 4 lane + e, slots 4 j ..
            const uint32_t lo = __byte_perm(qv[4 * j], qv[4 * j + 1], 0x0040 + 0x0011 * e);
            const uint32_t hi = __byte_perm(qv[4 * j + 2], qv[4 * j + 3], 0x0040 + 0x0011 * e);
            return __byte_perm(lo, hi, 0x5410);
          };
          if (!partial(run)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *v_piece(run, e) = make_uint4(word(e, 0), word(e, 1), word(e, 2), word(e, 3));
          } else {
            if (!kEarly || grew || (kPerWarp > 1 && run != held)) {   // all four before the first is written
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint4 was = *v_piece(run, e);
                ext[4 * e] = was.x, ext[4 * e + 1] = was.y, ext[4 * e + 2] = was.z, ext[4 * e + 3] = was.w;
              }
              held = -1;
            }
            uint32_t fresh_bytes[4];                        // bytes of word j that are new: slots 4 j .. 4 j + 3 inside [a, b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int from = min(max(a - 4 * j, 0), 4), to = min(max(b - 4 * j, 0), 4);
              const uint32_t below_to = to >= 4 ? 0xffffffffu : (1u << (8 * to)) - 1u;
              const uint32_t below_from = from >= 4 ? 0xffffffffu : (1u << (8 * from)) - 1u;
              fresh_bytes[j] = below_to & ~below_from;
            }
            auto mix = [&](uint32_t now, uint32_t then, int j) -> uint32_t { return (now & fresh_bytes[j]) | (then & ~fresh_bytes[j]); };
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *v_piece(run, e) = make_uint4(mix(word(e, 0), ext[4 * e], 0), mix(word(e, 1), ext[4 * e + 1], 1),
                                            mix(word(e, 2), ext[4 * e + 2], 2), mix(word(e, 3), ext[4 * e + 3], 3));
          }
        }
      }
      if (want_bounds && sub == 0) {
        uint32_t l4 = four(bound.x, bound.y), h4 = four(bound.z, bound.w);
        if (!fresh) {
          if (grew) old_lo = rescale_e4m3x4(old_lo, ratio), old_hi = rescale_e4m3x4(old_hi, ratio);
          float a[4], b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] = fminf(e4m3_to_f32(l4 >> (8 * e)), e4m3_to_f32(old_lo >> (8 * e)));
            b[e] = fmaxf(e4m3_to_f32(h4 >> (8 * e)), e4m3_to_f32(old_hi >> (8 * e)));
          }
          l4 = pack_e4m3x4(a[0], a[1], a[2], a[3]);
          h4 = pack_e4m3x4(b[0], b[1], b[2], b[3]);
        }
        bounds_at[0] = l4;
        bounds_at[kD / 4] = h4;
      }
    }
    // every warp of the unit has read the old scale (before the barrier of the maximum, or, with one
    // warp, by the lanes above): the new one may go there
    __syncwarp();
    if (PER_BLOCK && live && o1 > o0 && sub == 0 && lane == 0) *scale_at = scale;
    // the reduction buffers are free for the next unit (and nobody leaves while they may be read)
    if constexpr (CLUSTER > 1) cooperative_groups::this_cluster().sync();
    else if (WPU > 1) __syncthreads();
  }
}

}  // namespace pa
