// Host side of the C ABI's operators around a cache with scales per (page, kv head): the append, the
// page scores and the page selection.  Argument checks, launch shapes and the launches; nothing here
// allocates, synchronises or touches any stream but the caller's.
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/pa_decode_sm100.h"
#include "pa_host.h"
#include "pa_places.h"
#include "pa_block_score.cuh"
#include "pa_block_select.cuh"
#include "pa_cache_append.cuh"

namespace {

using pa_host::cuda_fail;
using pa_host::device_info;
using pa_host::DeviceInfo;

inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Launch as a programmatic dependent of the kernel before it in the stream; the kernels here wait
// (griddepcontrol.wait) before they touch global memory.
template <typename P>
int launch(void (*kernel)(P), dim3 grid, int threads, size_t smem, cudaStream_t stream, const P& params, int cluster = 1) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, params);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? PA_OK : cuda_fail(e);
}

}  // namespace

extern "C" {

int pa_cache_append_sm100(const PaCacheAppendParams* p, void* stream) {
  if (!p) return PA_ERR_NULL_POINTER;
  if (p->struct_size != sizeof(*p) || p->abi_version != PA_ABI_VERSION) return PA_ERR_ABI;
  if (p->num_tokens < 0 || p->num_seqs < 0 || p->num_kv_heads <= 0 || p->num_blocks <= 0 || p->max_blocks_per_seq <= 0)
    return PA_ERR_BAD_SHAPE;
  if (p->head_size != pa::kD) return PA_ERR_UNSUPPORTED;
  if (p->block_size != 16 && p->block_size != 64 && p->block_size != 1024) return PA_ERR_UNSUPPORTED;
  if (p->kv_quant_mode != PA_QUANT_PER_BLOCK && p->kv_quant_mode != PA_QUANT_PER_TENSOR) return PA_ERR_UNSUPPORTED;
  if (p->v_layout != PA_V_NORMAL && p->v_layout != PA_V_TRANSPOSED) return PA_ERR_UNSUPPORTED;
  if (p->num_seqs > pa::kAppendMaxSeqs) return PA_ERR_TOO_LARGE;
  if (p->num_seqs == 0 || p->num_tokens == 0) return PA_OK;
  if (!p->key || !p->value || !p->key_cache || !p->value_cache || !p->key_scale || !p->value_scale || !p->block_tables ||
      !p->context_lens || !p->row_start)
    return PA_ERR_NULL_POINTER;
  if (!aligned(p->key, 16) || !aligned(p->value, 16) || !aligned(p->key_cache, 16) || !aligned(p->value_cache, 16) ||
      !aligned(p->key_bounds, 16))
    return PA_ERR_ALIGNMENT;
  if ((p->key_stride_token & 7) || (p->key_stride_head & 7) || (p->value_stride_token & 7) || (p->value_stride_head & 7) ||
      (p->k_stride_block & 15) || (p->k_stride_head & 15) || (p->v_stride_block & 15) || (p->v_stride_head & 15) ||
      (p->bounds_stride_block & 15) || (p->bounds_stride_head & 15))
    return PA_ERR_ALIGNMENT;
  // what is written by units that know nothing of each other: every page and kv head needs a place of its own
  if (!pa_places::distinct(p->num_blocks, p->num_kv_heads, p->k_stride_block, p->k_stride_head) ||
      !pa_places::distinct(p->num_blocks, p->num_kv_heads, p->v_stride_block, p->v_stride_head) ||
      (p->key_bounds && !pa_places::distinct(p->num_blocks, p->num_kv_heads, p->bounds_stride_block, p->bounds_stride_head)))
    return PA_ERR_BAD_SHAPE;
  if (p->kv_quant_mode == PA_QUANT_PER_BLOCK &&
      (!pa_places::distinct(p->num_blocks, p->num_kv_heads, p->kv_scale_stride_block, p->kv_scale_stride_head) ||
       pa_places::meet(p->value_scale - p->key_scale, p->num_blocks, p->num_kv_heads, p->kv_scale_stride_block, p->kv_scale_stride_head)))
    return PA_ERR_BAD_SHAPE;
  DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != PA_OK) return rc;
  pa::CacheAppendParams k;
  memset(&k, 0, sizeof(k));
  k.key = static_cast<const uint8_t*>(p->key);
  k.value = static_cast<const uint8_t*>(p->value);
  k.key_cache = static_cast<uint8_t*>(p->key_cache);
  k.value_cache = static_cast<uint8_t*>(p->value_cache);
  k.k_scale = p->key_scale;
  k.v_scale = p->value_scale;
  k.bounds = static_cast<uint8_t*>(p->key_bounds);
  k.block_tables = p->block_tables;
  k.context_lens = p->context_lens;
  k.row_start = p->row_start;
  k.status = p->status;
  k.T = p->num_tokens;
  k.S = p->num_seqs;
  k.Hkv = p->num_kv_heads;
  k.num_blocks = p->num_blocks;
  k.width = p->max_blocks_per_seq;
  k.v_trans = p->v_layout == PA_V_TRANSPOSED;
  const bool blk = p->kv_quant_mode == PA_QUANT_PER_BLOCK;
  k.key_stride_tok = p->key_stride_token;
  k.key_stride_head = p->key_stride_head;
  k.value_stride_tok = p->value_stride_token;
  k.value_stride_head = p->value_stride_head;
  k.kc_stride_block = p->k_stride_block;
  k.kc_stride_head = p->k_stride_head;
  k.vc_stride_block = p->v_stride_block;
  k.vc_stride_head = p->v_stride_head;
  k.ks_stride_block = p->kv_scale_stride_block;
  k.ks_stride_head = p->kv_scale_stride_head;
  k.b_stride_block = p->bounds_stride_block;
  k.b_stride_head = p->bounds_stride_head;
  k.bt_stride_seq = p->bt_stride_seq;
  // pages touched: one for every bs rows, and up to two more per sequence (its ends); never more than rows
  int64_t pages = (int64_t)p->num_tokens / p->block_size + 2 * (int64_t)p->num_seqs;
  if (pages > p->num_tokens) pages = p->num_tokens;
  const int64_t units = pages * p->num_kv_heads * 2;
  if (units > (1 << 30)) return PA_ERR_TOO_LARGE;
  const size_t smem = (size_t)(p->num_seqs + 1) * 4;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t cap = (int64_t)dev->sm_count * 5;   // CTAs of four warps that are resident at a time
  // The form goes by the mean number of rows a sequence brings: the lengths are on the device.  It was measured with
  // sequences alike; a prompt chunk beside single rows is judged by a mean that describes neither (8 000 rows and 600
  // single ones, eight kv heads, pages of 64: 39 us; 3 000 rows and 60 single ones, one head, pages of 1024: 22 us).
  // Pages of 1024 tokens.  Four warps a page where a sequence brings a few rows (fewer than 64 on average), and up to
  // 256 where there are more pages than such CTAs at a time (40 sequences of 100 rows, eight kv heads: 11.5 us against
  // 13.8 with eight warps and 20.5 with sixteen; of 400 rows 36, 41 and 41, but lengths from 1 to 900 want more:
  // 84, 78 and 75).  For more rows eight warps (of 1 000 rows: 46 us, with sixteen 49), or, while all pages find
  // room at once that way, a cluster of eight CTAs.
  const int64_t few = units > cap ? 256 : 64;
  if (p->block_size == 1024 && p->num_tokens >= few * p->num_seqs) {
    constexpr int kCluster = 8;
    if (units <= 2 * dev->sm_count / kCluster)   // (two of its CTAs fit an SM)
      return launch(blk ? pa::pa_cache_append_kernel<1024, 64, true, kCluster> : pa::pa_cache_append_kernel<1024, 64, false, kCluster>,
                    dim3((unsigned)(units * kCluster)), 256, smem, st, k, kCluster);
    const int64_t grid = units < 2 * dev->sm_count ? units : 2 * dev->sm_count;
    return launch(blk ? pa::pa_cache_append_kernel<1024, 8, true> : pa::pa_cache_append_kernel<1024, 8, false>, dim3((unsigned)grid), 256, smem, st, k);
  }
  // Pages of 64 tokens that get a few rows each (fewer than a run of 16 per sequence, on average), more of them
  // than four warps apiece could take at once: a warp each (5.1 us against 7.5 for a row of 64 sequences with
  // eight kv heads; prompts, whose pages have four full runs, would lose: 31 us against 25 for 16 000 rows).
  const bool lone = p->block_size == 64 && p->num_tokens < 16 * (int64_t)p->num_seqs && units > cap;
  const int per_cta = p->block_size == 16 || lone ? 4 : 1;
  int64_t grid = (units + per_cta - 1) / per_cta;
  if (grid > cap) grid = cap;
  switch (p->block_size) {
    case 16: return launch(blk ? pa::pa_cache_append_kernel<16, 1, true> : pa::pa_cache_append_kernel<16, 1, false>, dim3((unsigned)grid), 128, smem, st, k);
    case 64:
      if (lone) return launch(blk ? pa::pa_cache_append_kernel<64, 1, true> : pa::pa_cache_append_kernel<64, 1, false>, dim3((unsigned)grid), 128, smem, st, k);
      return launch(blk ? pa::pa_cache_append_kernel<64, 4, true> : pa::pa_cache_append_kernel<64, 4, false>, dim3((unsigned)grid), 128, smem, st, k);
    default: return launch(blk ? pa::pa_cache_append_kernel<1024, 4, true> : pa::pa_cache_append_kernel<1024, 4, false>, dim3((unsigned)grid), 128, smem, st, k);
  }
}

int pa_block_scores_sm100(const PaBlockScoreParams* p, void* stream) {
  if (!p) return PA_ERR_NULL_POINTER;
  if (p->struct_size != sizeof(*p) || p->abi_version != PA_ABI_VERSION) return PA_ERR_ABI;
  if (p->num_seqs < 0 || p->num_kv_heads <= 0 || p->rows <= 0 || p->block_size <= 0 || p->num_blocks <= 0 ||
      p->max_blocks_per_seq <= 0)
    return PA_ERR_BAD_SHAPE;
  if (p->head_size != pa::kD || p->rows > 64) return PA_ERR_UNSUPPORTED;
  if (p->q_dtype != PA_DT_BF16 && p->q_dtype != PA_DT_E4M3FN) return PA_ERR_UNSUPPORTED;
  if (p->q_quant_mode < PA_QUANT_NONE || p->q_quant_mode > PA_QUANT_PER_TOKEN) return PA_ERR_UNSUPPORTED;
  if (p->kv_quant_mode != PA_QUANT_NONE && p->kv_quant_mode != PA_QUANT_PER_TENSOR && p->kv_quant_mode != PA_QUANT_PER_BLOCK)
    return PA_ERR_UNSUPPORTED;
  if (!(p->softmax_scale > 0.f)) return PA_ERR_UNSUPPORTED;   // the largest product would not be the largest logit
  if (p->num_seqs == 0) return PA_OK;
  if (!p->query || !p->key_bounds || !p->block_tables || !p->context_lens || !p->scores ||
      (p->q_quant_mode != PA_QUANT_NONE && !p->query_scale) || (p->kv_quant_mode != PA_QUANT_NONE && !p->key_scale))
    return PA_ERR_NULL_POINTER;
  const int item = p->q_dtype == PA_DT_BF16 ? 2 : 1;
  if (!aligned(p->query, 16) || ((p->q_stride_seq * item) & 15) || !aligned(p->key_bounds, 16) || (p->bounds_stride_block & 15) ||
      (p->bounds_stride_head & 15))
    return PA_ERR_ALIGNMENT;
  DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc != PA_OK) return rc;
  pa::BlockScoreParams k;
  memset(&k, 0, sizeof(k));
  k.q = static_cast<const uint8_t*>(p->query);
  k.bounds = static_cast<const uint8_t*>(p->key_bounds);
  k.block_tables = p->block_tables;
  k.context_lens = p->context_lens;
  k.q_scale = p->query_scale;
  k.k_scale = p->kv_quant_mode == PA_QUANT_NONE ? nullptr : p->key_scale;
  k.scores = p->scores;
  k.status = p->status;
  k.S = p->num_seqs;
  k.Hkv = p->num_kv_heads;
  k.rows = p->rows;
  k.block_size = p->block_size;
  k.num_blocks = p->num_blocks;
  k.width = p->max_blocks_per_seq;
  k.q_is_fp8 = item == 1;
  k.q_quant_mode = p->q_quant_mode;
  k.q_stride_seq = p->q_stride_seq * item;
  k.bounds_stride_block = p->bounds_stride_block;
  k.bounds_stride_head = p->bounds_stride_head;
  k.bt_stride_seq = p->bt_stride_seq;
  k.q_scale_stride_seq = p->q_scale_stride_seq;
  if (p->kv_quant_mode == PA_QUANT_PER_BLOCK) {
    k.ks_stride_block = p->kv_scale_stride_block;
    k.ks_stride_head = p->kv_scale_stride_head;
  }
  k.out_stride_seq = p->scores_stride_seq;
  k.out_stride_head = p->scores_stride_head;
  k.softmax_scale = p->softmax_scale;
  const int nb8 = p->rows <= 8 ? 1 : (p->rows <= 16 ? 2 : (p->rows <= 32 ? 4 : 8));
  // kv heads per CTA: neighbouring heads of a page are neighbours in memory; as many as their query
  // rows fit, a power of two that divides the CTA's warps (three heads take the places of four)
  int heads = pa::kScoreMaxRows / (nb8 * 8);
  while (heads / 2 >= p->num_kv_heads) heads >>= 1;
  k.heads_per_cta = heads;
  const int64_t tiles = ((int64_t)p->max_blocks_per_seq + pa::kScoreTilePages - 1) / pa::kScoreTilePages;
  const int64_t most = (int64_t)p->num_seqs * tiles * ((p->num_kv_heads + heads - 1) / heads);   // units of work, at most
  if ((int64_t)p->num_seqs * tiles > 0x7fffffff) return PA_ERR_TOO_LARGE;
  const int64_t grid = most < dev->sm_count ? most : dev->sm_count;
  k.off_index = (heads * nb8 * 8 * (pa::kScoreRowBytes + 4) + 15) & ~15;
  const int64_t off_ring = (k.off_index + ((int64_t)2 * p->num_seqs + 1) * 4 + 127) & ~(int64_t)127;
  const int slot = pa::score_slot_bytes(heads);
  constexpr int kDeclared = 1024;   // the kernel's barriers and scan buffer
  int64_t slots = ((int64_t)dev->max_smem_optin - kDeclared - off_ring) / slot;
  if (slots > pa::kScoreRingBytes / slot) slots = pa::kScoreRingBytes / slot;
  if (slots > pa::kScoreMaxSlots) slots = pa::kScoreMaxSlots;
  const int warps = pa::score_warps(nb8), step = warps / heads;
  slots -= slots % step;
  const int producers = pa::score_producers(heads);
  if (slots < step || slots < producers) return PA_ERR_TOO_LARGE;   // the index of the sequences leaves no room
  k.off_ring = (int)off_ring;
  k.slots = (int)slots;
  const int64_t smem = off_ring + slots * slot;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void (*kernel)(pa::BlockScoreParams) = nb8 == 1   ? (heads == 8 ? pa::pa_block_score_kernel<1, 2> : pa::pa_block_score_kernel<1, 4>)
                                         : nb8 == 2 ? pa::pa_block_score_kernel<2, 4>
                                         : nb8 == 4 ? pa::pa_block_score_kernel<4, 4>
                                                    : pa::pa_block_score_kernel<8, 4>;
  const cudaError_t e = pa_host::raise_dynamic_smem(kernel, *dev, kDeclared);
  if (e != cudaSuccess) return cuda_fail(e);
  return launch(kernel, dim3((unsigned)grid), (warps + producers) * 32, (size_t)smem, st, k);
}

int pa_block_select_sm100(const PaBlockSelectParams* p, void* stream) {
  if (!p) return PA_ERR_NULL_POINTER;
  if (p->struct_size != sizeof(*p) || p->abi_version != PA_ABI_VERSION) return PA_ERR_ABI;
  if (p->num_seqs < 0 || p->num_kv_heads <= 0 || p->block_size <= 0 || p->max_blocks_per_seq <= 0 || p->top_k <= 0 ||
      p->keep_first < 0 || p->keep_last < 1 || (int64_t)p->keep_first + p->keep_last > p->top_k)
    return PA_ERR_BAD_SHAPE;
  if (p->num_seqs == 0) return PA_OK;
  if (!p->scores || !p->block_tables || !p->context_lens || !p->tables || !p->lengths) return PA_ERR_NULL_POINTER;
  // outputs that other CTAs still read
  if (p->lengths == p->context_lens || p->tables == p->block_tables) return PA_ERR_BAD_SHAPE;
  const int64_t grid = (int64_t)p->num_seqs * p->num_kv_heads;
  if (grid > 0x7fffffff || (int64_t)p->max_blocks_per_seq > 0x7fffffff - pa::kSelectLarge) return PA_ERR_TOO_LARGE;
  pa::BlockSelectParams k;
  memset(&k, 0, sizeof(k));
  k.scores = p->scores;
  k.block_tables = p->block_tables;
  k.context_lens = p->context_lens;
  k.tables = p->tables;
  k.lengths = p->lengths;
  k.status = p->status;
  k.S = p->num_seqs;
  k.Hkv = p->num_kv_heads;
  k.block_size = p->block_size;
  k.width = p->max_blocks_per_seq;
  k.top_k = p->top_k;
  k.keep_first = p->keep_first;
  k.keep_last = p->keep_last;
  k.sc_stride_seq = p->scores_stride_seq;
  k.sc_stride_head = p->scores_stride_head;
  k.bt_stride_seq = p->bt_stride_seq;
  k.out_stride_seq = p->tables_stride_seq;
  k.out_stride_head = p->tables_stride_head;
  const dim3 ctas((unsigned)grid);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p->max_blocks_per_seq <= pa::kSelectSmall) return launch(pa::pa_block_select_kernel<128, 4>, ctas, 128, 0, st, k);
  if (p->max_blocks_per_seq <= pa::kSelectMedium) return launch(pa::pa_block_select_kernel<256, 8>, ctas, 256, 0, st, k);
  return launch(pa::pa_block_select_kernel<256, 32>, ctas, 256, 0, st, k);
}

}  // extern "C"
