"""Decode attention over the pages that a cheap score picks, for long contexts.

A decode step over a long context reads the whole cache although few pages hold weight.  Here each
kv head reads a fixed number of pages instead:

1. :func:`score_blocks` -- for every page an upper bound of the logits that the head's query rows can
   have with the page's keys, from the smallest and largest key code of each head dim
   (``key_bounds``, 256 bytes per page and kv head, kept by
   :func:`triton_op_b200.cache_write.append_kv_cache`);
2. :func:`select_blocks` -- the best pages, with the first and the last ones of the context kept, as a
   block table per kv head;
3. :func:`triton_op_b200.paged_attention_decode` on those tables.

:func:`sparse_attention_decode` is the three in a row.  All run on torch's current stream, on
tensors only; nothing is copied to the host, nothing is kept from one call for the next.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from .pa_decode import (FP8_DTYPE, SUPPORTED_BLOCK_SIZES, PaArgumentError, _dtype_code, _kv_scale, paged_attention_decode)

__all__ = ["score_blocks", "select_blocks", "sparse_attention_decode"]

_SCORE = struct.Struct("=2I8Q10i9qfi")
_SELECT = struct.Struct("=2I6Q8i5q")
assert _SCORE.size == C.sizeof(_lib.PaBlockScoreParams) and _SELECT.size == C.sizeof(_lib.PaBlockSelectParams)


def _fail(msg: str) -> None:
    raise PaArgumentError(msg)


def _tables_and_lengths(sequence_lengths, block_tables, on: int):
    """(sequence_lengths, block_tables, rows, columns, row stride) after the checks."""
    if not (sequence_lengths.dtype == torch.int32 and block_tables.dtype == torch.int32):
        _fail("sequence_lengths and block_tables must be int32")
    shape = block_tables.shape
    if not (len(shape) == 2 and sequence_lengths.numel() == shape[0]):
        _fail("block_tables must be [num_seqs, max_blocks] and sequence_lengths [num_seqs]")
    if shape[1] < 1:
        _fail("block_tables must have at least one column")
    if not (sequence_lengths.get_device() == on and block_tables.get_device() == on):
        _fail("sequence_lengths and block_tables must live on the device of the other tensors")
    if not sequence_lengths.is_contiguous():
        sequence_lengths = sequence_lengths.contiguous()
    stride = block_tables.stride()
    if stride[1] != 1:
        block_tables = block_tables.contiguous()
        stride = block_tables.stride()
    return sequence_lengths, block_tables, shape[0], shape[1], stride[0]


def _own_rows(t: torch.Tensor, name: str) -> None:
    """Refuses an output [num_seqs, num_kv_heads, ..] whose rows share memory by a stride of zero."""
    if any(n > 1 and s == 0 for n, s in zip(t.shape[:2], t.stride()[:2])):
        _fail(f"{name} is written: every sequence and kv head needs a row of its own")


def _status_ptr(status, dev) -> int:
    if status is None:
        return 0
    if not (status.dtype == torch.int32 and status.device == dev):
        _fail(f"status must be an int32 tensor on {dev}")
    return status.data_ptr()


def score_blocks(query: torch.Tensor, key_bounds: torch.Tensor, sequence_lengths: torch.Tensor,
                 block_tables: torch.Tensor, softmax_scale: float, query_sequence_length: int, block_size: int, *,
                 query_scale=None, key_scale=None, scores: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Upper bounds of the logits in every page: fp32 ``[num_seqs, num_kv_heads, max_blocks]``.

    ``scores[s, h, i] = key_scale * max_r softmax_scale * query_scale_r * sum_d max(q_rd lo_d, q_rd hi_d)``
    over the query rows ``r`` of kv head ``h`` (all query tokens), ``lo`` and ``hi`` the page's key
    bounds (sums in 32 bits, rounded to nearest or truncated: a bound to choose pages by, not a proof); ``-inf`` for entries past the sequence's last page, NaN where a query row holds one (an infinite
    element gives infinity, or NaN where it meets a bound of zero).  ``query`` as in
    ``paged_attention_decode`` (bf16, or e4m3fn with ``query_scale``); ``key_bounds`` e4m3fn
    ``[num_blocks, num_kv_heads, 2, head_size]``; ``key_scale`` ``None``, per tensor or
    ``[num_blocks, num_kv_heads, 1, 1]``; ``scores``: an output tensor to use.  At most 17 800 sequences.
    """
    if query_scale is None and scores is None:
        done = _lib.calls().scores(query, key_bounds, sequence_lengths, block_tables, softmax_scale, query_sequence_length,
                                   block_size, key_scale, status)
        if type(done) is tuple:
            return done[0]
        if done is not None:
            raise _lib.PaError(done, "pa_block_scores_sm100")
    dev, on = query.device, query.get_device()
    q_shape, b_shape = query.shape, key_bounds.shape
    if len(q_shape) != 3:
        _fail(f"Expected 3D query tensor, but got shape {tuple(q_shape)}")
    q_dtype = _lib.PA_DT_BF16 if query.dtype == torch.bfloat16 else _dtype_code(query.dtype, "query")
    if not (len(b_shape) == 4 and key_bounds.dtype == FP8_DTYPE and key_bounds.get_device() == on):
        _fail(f"key_bounds must be a 4D {FP8_DTYPE} tensor on {dev}")
    num_blocks, num_kv_heads, two, head_size = b_shape
    num_seqs, q_heads, q_size = q_shape
    if not (two == 2 and head_size == 128 and q_size == 128):
        _fail("key_bounds must be [num_blocks, num_kv_heads, 2, 128] and query [num_seqs, heads, 128]")
    b_stride = key_bounds.stride()
    if b_stride[3] != 1 or b_stride[2] != head_size:
        _fail("the last two dims of key_bounds must be contiguous")
    if block_size not in SUPPORTED_BLOCK_SIZES:
        _fail(f"block_size == {block_size} not in {list(SUPPORTED_BLOCK_SIZES)}")
    if not 1 <= query_sequence_length <= 4:
        _fail(f"QUERY_SEQ_LEN={query_sequence_length}, only 1 to 4 are supported")
    rows = q_heads // num_kv_heads if num_kv_heads else 0
    if rows < 1 or rows * num_kv_heads != q_heads or rows % query_sequence_length:
        _fail("query heads must be num_kv_heads * query_sequence_length * group_size")
    if rows > 64:
        _fail(f"equivalent query group size {rows} exceeds maximum of 64")
    if not softmax_scale > 0:
        _fail(f"softmax_scale must be positive, but got {softmax_scale}")
    sequence_lengths, block_tables, table_rows, width, t_stride = _tables_and_lengths(sequence_lengths, block_tables, on)
    if table_rows != num_seqs:
        _fail("block_tables must be [num_seqs, max_blocks] and sequence_lengths [num_seqs]")
    stride = query.stride()
    if stride[2] != 1 or stride[1] != head_size or (stride[0] * query.element_size()) % 16 or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)
        stride = query.stride()
    q_mode, q_ptr, q_stride = _lib.PA_QUANT_NONE, 0, 0
    if query_scale is not None:
        if isinstance(query_scale, (int, float)):
            query_scale = torch.full((), float(query_scale), dtype=torch.float32, device=dev)
        if not (query_scale.dtype == torch.float32 and query_scale.device == dev):
            _fail(f"query_scale must be a float32 tensor on {dev}")
        if query_scale.dim() == 0:
            q_mode = _lib.PA_QUANT_PER_TENSOR
        else:
            if query_scale.shape != (num_seqs, q_heads, 1):
                _fail(f"Expected query_scale [num_seqs, heads, 1], but got shape {tuple(query_scale.shape)}")
            if query_scale.stride(1) != 1:
                query_scale = query_scale.contiguous()
            q_mode, q_stride = _lib.PA_QUANT_PER_TOKEN, query_scale.stride(0)
        q_ptr = query_scale.data_ptr()
    kv_mode, ks_ptr, s_block, s_head = _lib.PA_QUANT_NONE, 0, 0, 0
    if key_scale is not None:
        if isinstance(key_scale, (int, float)):
            key_scale = torch.full((), float(key_scale), dtype=torch.float32, device=dev)
        key_scale, kv_mode = _kv_scale(key_scale, None, "key_scale", dev)
        if key_scale.get_device() != on:
            _fail(f"key_scale must live on {dev}")
        if kv_mode == _lib.PA_QUANT_PER_TOKEN:
            _fail("key bounds go with a key scale per tensor or per (block, head), not per token")
        if kv_mode == _lib.PA_QUANT_PER_BLOCK:
            if key_scale.shape != (num_blocks, num_kv_heads, 1, 1):
                _fail(f"key_scale must be [num_blocks, num_kv_heads, 1, 1] = {(num_blocks, num_kv_heads, 1, 1)}")
            ks_stride = key_scale.stride()
            s_block, s_head = ks_stride[0], ks_stride[1]
        ks_ptr = key_scale.data_ptr()
    if scores is None:
        scores = torch.empty_strided((num_seqs, num_kv_heads, width), (num_kv_heads * width, width, 1), dtype=torch.float32, device=dev)
    elif not (scores.dtype == torch.float32 and scores.device == dev and scores.shape == (num_seqs, num_kv_heads, width)
              and scores.stride(2) == 1):
        _fail(f"scores must be fp32 {(num_seqs, num_kv_heads, width)} on {dev}, its last dim contiguous")
    else:
        _own_rows(scores, "scores")
    s_stride = scores.stride()
    status_ptr = _status_ptr(status, dev)
    if on < 0:
        raise RuntimeError("score_blocks runs on CUDA tensors only; there is no CPU fallback")
    p = _lib.PaBlockScoreParams.from_buffer_copy(_SCORE.pack(
        _SCORE.size, _lib.PA_ABI_VERSION,
        query.data_ptr(), key_bounds.data_ptr(), block_tables.data_ptr(), sequence_lengths.data_ptr(), q_ptr, ks_ptr,
        scores.data_ptr(), status_ptr,
        num_seqs, num_kv_heads, rows, head_size, block_size, num_blocks, width, q_dtype, q_mode, kv_mode,
        stride[0], b_stride[0], b_stride[1], t_stride, q_stride, s_block, s_head,
        s_stride[0], s_stride[1], float(softmax_scale), 0))
    _lib.launch(on, _lib.lib().pa_block_scores_sm100, "pa_block_scores_sm100", C.byref(p))
    return scores


def select_blocks(scores: torch.Tensor, sequence_lengths: torch.Tensor, block_tables: torch.Tensor, block_size: int,
                  top_k: int, *, keep_first: int = 1, keep_last: int = 1, tables: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The best ``top_k`` pages of each (sequence, kv head) as block tables of their own.

    Returns ``(tables, lengths)``: int32 ``[num_seqs, num_kv_heads, top_k]`` page ids in the order of
    the context (0 where a sequence has fewer pages) and int32 ``[num_seqs]``, the tokens in one
    such table -- what ``paged_attention_decode`` takes as ``block_tables`` and ``sequence_lengths``.
    The first ``keep_first`` and the last ``keep_last`` pages are always among them; the others go by
    ``scores`` (fp32 ``[num_seqs, num_kv_heads, max_blocks]``), NaN as -inf, ties to the lower place.
    With several query tokens ``keep_last`` has to cover the last ``query_len`` tokens: 2.  ``tables`` and
    ``lengths``: output tensors to use, not the ones that are read.
    """
    if tables is None and lengths is None:
        done = _lib.calls().select(scores, sequence_lengths, block_tables, block_size, top_k, keep_first, keep_last, status)
        if type(done) is tuple:
            return done
        if done is not None:
            raise _lib.PaError(done, "pa_block_select_sm100")
    dev, on = scores.device, scores.get_device()
    sc_shape = scores.shape
    if not (len(sc_shape) == 3 and scores.dtype == torch.float32):
        _fail(f"scores must be a 3D float32 tensor, but got {scores.dtype} of shape {tuple(sc_shape)}")
    if block_size not in SUPPORTED_BLOCK_SIZES:
        _fail(f"block_size == {block_size} not in {list(SUPPORTED_BLOCK_SIZES)}")
    num_seqs, num_kv_heads, columns = sc_shape
    sequence_lengths, block_tables, table_rows, width, bt_stride = _tables_and_lengths(sequence_lengths, block_tables, on)
    if table_rows != num_seqs or columns < width or num_kv_heads < 1:
        _fail("scores must be [num_seqs, num_kv_heads, >= max_blocks]")
    if keep_first < 0 or keep_last < 1 or top_k < keep_first + keep_last:
        _fail(f"top_k must hold keep_first >= 0 and keep_last >= 1 pages, but got {top_k}, {keep_first}, {keep_last}")
    sc_stride = scores.stride()
    if sc_stride[2] != 1:
        scores = scores.contiguous()
        sc_stride = scores.stride()
    if tables is None:
        tables = torch.empty_strided((num_seqs, num_kv_heads, top_k), (num_kv_heads * top_k, top_k, 1), dtype=torch.int32, device=dev)
    elif not (tables.dtype == torch.int32 and tables.device == dev and tables.shape == (num_seqs, num_kv_heads, top_k)
              and tables.stride(2) == 1):
        _fail(f"tables must be int32 {(num_seqs, num_kv_heads, top_k)} on {dev}, its last dim contiguous")
    else:
        _own_rows(tables, "tables")
        if tables.numel() > 0 and tables.data_ptr() == block_tables.data_ptr():
            _fail("tables must not be block_tables, which are read")
    if lengths is None:
        lengths = torch.empty_strided((num_seqs,), (1,), dtype=torch.int32, device=dev)
    elif not (lengths.dtype == torch.int32 and lengths.device == dev and lengths.shape == (num_seqs,) and lengths.is_contiguous()):
        _fail(f"lengths must be a contiguous int32 tensor of {num_seqs} on {dev}")
    elif num_seqs > 0 and abs(lengths.data_ptr() - sequence_lengths.data_ptr()) < 4 * num_seqs:
        _fail("lengths must not be sequence_lengths, which every kv head reads")
    t_stride = tables.stride()
    status_ptr = _status_ptr(status, dev)
    if on < 0:
        raise RuntimeError("select_blocks runs on CUDA tensors only; there is no CPU fallback")
    p = _lib.PaBlockSelectParams.from_buffer_copy(_SELECT.pack(
        _SELECT.size, _lib.PA_ABI_VERSION,
        scores.data_ptr(), block_tables.data_ptr(), sequence_lengths.data_ptr(), tables.data_ptr(), lengths.data_ptr(), status_ptr,
        num_seqs, num_kv_heads, block_size, width, int(top_k), int(keep_first), int(keep_last), 0,
        sc_stride[0], sc_stride[1], bt_stride, t_stride[0], t_stride[1]))
    _lib.launch(on, _lib.lib().pa_block_select_sm100, "pa_block_select_sm100", C.byref(p))
    return tables, lengths


def sparse_attention_decode(output: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor,
                            value_cache: torch.Tensor, key_bounds: torch.Tensor, sequence_lengths: torch.Tensor,
                            block_tables: torch.Tensor, softmax_scale: float, query_sequence_length: int, top_k: int,
                            query_scale=None, key_scale=None, value_scale=None, *, keep_first: int = 1,
                            keep_last: Optional[int] = None, sink_tokens: Optional[torch.Tensor] = None,
                            status: Optional[torch.Tensor] = None) -> Dict:
    """Decode attention of every kv head over its best ``top_k`` pages: :func:`score_blocks`,
    :func:`select_blocks` and ``paged_attention_decode``.  Arguments as there (e4m3fn caches; scales
    ``None``, per tensor or ``[num_blocks, num_kv_heads, 1, 1]``); ``keep_last`` defaults to 1, or 2 with
    several query tokens; at most 5 199 sequences (2 639 with more than eight query rows a kv head).  A sequence of at most ``top_k`` pages gets its full attention.  Returns
    ``paged_attention_decode``'s dictionary with the ``block_tables`` and ``sequence_lengths`` that were read.
    """
    if key_cache.dim() != 5:
        _fail(f"Expected 5D key_cache tensor, but got shape {tuple(key_cache.shape)}")
    if key_bounds.shape[:2] != key_cache.shape[:2]:
        _fail("key_bounds and key_cache must have the same num_blocks and num_kv_heads")
    block_size = key_cache.shape[3]
    least = 1 if query_sequence_length == 1 else 2
    keep_last = least if keep_last is None else keep_last
    if keep_last < least:
        _fail(f"keep_last must be at least {least} with {query_sequence_length} query tokens, but got {keep_last}")
    scores = score_blocks(query, key_bounds, sequence_lengths, block_tables, softmax_scale, query_sequence_length,
                          block_size, query_scale=query_scale, key_scale=key_scale, status=status)
    tables, lengths = select_blocks(scores, sequence_lengths, block_tables, block_size, top_k, keep_first=keep_first,
                                    keep_last=keep_last, status=status)
    res = paged_attention_decode(output, query, key_cache, value_cache, lengths, tables, softmax_scale,
                                 query_sequence_length, min(top_k, block_tables.shape[1]) * block_size, torch.bfloat16, query_scale, key_scale,
                                 value_scale, sink_tokens=sink_tokens, status=status)
    res["block_tables"], res["sequence_lengths"] = tables, lengths
    return res
