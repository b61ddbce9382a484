"""KV-cache write side: new key / value tokens into the paged caches the decode operator reads.

The reference prepares its caches offline (layouts: test_pa_mtp.py:109-172; per-token e4m3
quantisation ``quantize_kv_cache_symmetric``: :294-369).  A serving loop does the same for the
tokens of every step; :func:`write_kv_cache` is that step as one CUDA kernel
(``pa_cache_write_sm100``): quantise and scatter, no intermediate tensors.  :func:`append_kv_cache` is
the same step for caches with one scale per (page, kv head) (``pa_cache_append_sm100``).
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

import torch

from . import _lib
from .pa_decode import FP8_DTYPE, SUPPORTED_BLOCK_SIZES, PaArgumentError, _check_block_scales, _inner_contiguous

__all__ = ["write_kv_cache", "append_kv_cache", "slots_for"]


def slots_for(block_tables: torch.Tensor, positions: torch.Tensor, seq_ids: torch.Tensor, block_size: int) -> torch.Tensor:
    """Slot (``block * block_size + offset``) of token ``positions[i]`` of sequence ``seq_ids[i]``."""
    blocks = block_tables[seq_ids.long(), (positions // block_size).long()].long()
    return blocks * block_size + (positions % block_size).long()


def write_kv_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                   slot_mapping: torch.Tensor, key_scale: Optional[torch.Tensor] = None,
                   value_scale: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """Writes ``key`` / ``value`` ``[T, Hkv, D]`` bf16 into the paged caches at ``slot_mapping [T]`` (int64).

    Caches: keys ``[NB, Hkv, D/x, bs, x]``, values ``[NB, Hkv, D, bs]`` or transposed
    ``[NB, Hkv, bs/16, D, 16]``; bf16 (bits copied, no scales) or e4m3fn.  For e4m3fn caches the
    scales select the mode: 0-dim fp32 tensors are per-tensor scales that are READ
    (``q = x / scale``); ``[NB, Hkv, bs, 1]`` fp32 tensors receive the per-token scales
    ``max(amax / 448, 1e-12)`` of the written tokens; ``None`` stores ``x`` unscaled.
    Negative slots are skipped.  Runs on the current stream; there is no CPU fallback.
    """
    if not (key.is_cuda and value.is_cuda and key_cache.is_cuda and value_cache.is_cuda):
        raise RuntimeError("write_kv_cache runs on CUDA tensors only; there is no CPU fallback")
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16 or key.shape != value.shape or key.dim() != 3:
        raise PaArgumentError("key and value must be bf16 [num_tokens, num_kv_heads, head_size] of one shape")
    if key_cache.dim() != 5 or value_cache.dim() not in (4, 5) or value_cache.dtype != key_cache.dtype:
        raise PaArgumentError("key_cache must be 5-D, value_cache 4-D or 5-D, of one dtype")
    T, hkv, d = key.shape
    nb, bs = key_cache.shape[0], key_cache.shape[3]
    x = 16 // key_cache.element_size()
    if tuple(key_cache.shape) != (nb, hkv, d // x, bs, x):
        raise PaArgumentError(f"key_cache must be [num_blocks, {hkv}, {d // x}, block_size, {x}]")
    trans = value_cache.dim() == 5
    want_v = (nb, hkv, bs // x, d, x) if trans else (nb, hkv, d, bs)
    if tuple(value_cache.shape) != want_v:
        raise PaArgumentError(f"value_cache must be {want_v}")
    if key_cache.dtype == torch.bfloat16:
        kv_dtype, mode = _lib.PA_DT_BF16, _lib.PA_QUANT_NONE
        if key_scale is not None or value_scale is not None:
            raise PaArgumentError("bf16 caches take no scales")
    elif key_cache.dtype == FP8_DTYPE:
        kv_dtype = _lib.PA_DT_E4M3FN
        if (key_scale is None) != (value_scale is None):
            raise PaArgumentError("key_scale and value_scale go together")
        if key_scale is None:
            mode = _lib.PA_QUANT_NONE
        elif key_scale.dim() == 0 and value_scale.dim() == 0:
            mode = _lib.PA_QUANT_PER_TENSOR
        elif tuple(key_scale.shape) == (nb, hkv, bs, 1) and tuple(value_scale.shape) == (nb, hkv, bs, 1):
            mode = _lib.PA_QUANT_PER_TOKEN
            if key_scale.stride(2) != 1 or value_scale.stride() != key_scale.stride():
                raise PaArgumentError("per-token scales must be contiguous along block_size and share strides")
        else:
            raise PaArgumentError("scales must be 0-dim (per tensor) or [num_blocks, num_kv_heads, block_size, 1]")
        for s in (key_scale, value_scale):
            if s is not None and (s.dtype != torch.float32 or not s.is_cuda):
                raise PaArgumentError("scales must be fp32 CUDA tensors")
    else:
        raise PaArgumentError(f"unsupported cache dtype {key_cache.dtype}")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != T or not slot_mapping.is_cuda:
        raise PaArgumentError("slot_mapping must be an int64 CUDA tensor with one entry per token")
    if key.stride(2) != 1:
        key = key.contiguous()
    if value.stride(2) != 1:
        value = value.contiguous()
    slot_mapping = slot_mapping.contiguous()

    p = _lib.PaCacheWriteParams()
    p.struct_size = C.sizeof(_lib.PaCacheWriteParams)
    p.abi_version = _lib.PA_ABI_VERSION
    p.key, p.value, p.slot_mapping = key.data_ptr(), value.data_ptr(), slot_mapping.data_ptr()
    p.key_cache, p.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    p.key_scale = key_scale.data_ptr() if key_scale is not None else None
    p.value_scale = value_scale.data_ptr() if value_scale is not None else None
    p.status = status.data_ptr() if status is not None else None
    p.num_tokens, p.num_kv_heads, p.head_size, p.block_size, p.num_blocks = T, hkv, d, bs, nb
    p.kv_dtype, p.kv_quant_mode = kv_dtype, mode
    p.v_layout = _lib.PA_V_TRANSPOSED if trans else _lib.PA_V_NORMAL
    p.key_stride_token, p.key_stride_head = key.stride(0), key.stride(1)
    p.value_stride_token, p.value_stride_head = value.stride(0), value.stride(1)
    p.k_stride_block, p.k_stride_head = key_cache.stride(0), key_cache.stride(1)
    p.v_stride_block, p.v_stride_head = value_cache.stride(0), value_cache.stride(1)
    if mode == _lib.PA_QUANT_PER_TOKEN:
        p.kv_scale_stride_block, p.kv_scale_stride_head = key_scale.stride(0), key_scale.stride(1)
    with torch.cuda.device(key.device):
        _lib.check(_lib.lib().pa_cache_write_sm100(C.byref(p), torch.cuda.current_stream().cuda_stream),
                   "pa_cache_write_sm100")


_APPEND = struct.Struct("=2I11Q10i13q")
assert _APPEND.size == C.sizeof(_lib.PaCacheAppendParams)


def _rows(t: torch.Tensor):
    """``t`` [T, Hkv, D] bf16 with 16-byte aligned rows (a copy where it has none), and its strides."""
    stride = t.stride()
    if stride[2] != 1 or stride[0] % 8 or stride[1] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        stride = t.stride()
    return t, stride


def _distinct(stride, shape) -> bool:
    """Every page and kv head has a place of its own (no stride of zero)."""
    return not ((shape[0] > 1 and stride[0] == 0) or (shape[1] > 1 and stride[1] == 0))


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """An entry [page, kv head] of one is an entry of the other (both with the same strides)."""
    (n0, n1), (s0, s1) = a.shape[:2], a.stride()[:2]
    apart, left = divmod(b.data_ptr() - a.data_ptr(), 4)
    if left or abs(apart) > (n0 - 1) * s0 + (n1 - 1) * s1:
        return False
    rests = (apart - j * s1 for j in range(1 - n1, n1))
    return any(r == 0 if s0 == 0 else r % s0 == 0 and abs(r // s0) < n0 for r in rests)


def append_kv_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                    key_scale: torch.Tensor, value_scale: torch.Tensor, block_tables: torch.Tensor,
                    sequence_lengths: torch.Tensor, query_start_loc: torch.Tensor, *,
                    key_bounds: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """Appends every sequence's new tokens to an e4m3fn cache with one scale per (page, kv head).

    Rows ``query_start_loc[s] .. query_start_loc[s + 1] - 1`` of ``key`` / ``value`` (bf16
    ``[T, num_kv_heads, head_size]``) become the last tokens of sequence ``s``, whose length with them
    is ``sequence_lengths[s]`` -- the tensors the decode call after it takes.  ``key_scale`` /
    ``value_scale`` fp32 ``[num_blocks, num_kv_heads, 1, 1]`` are read and written: a page that begins with
    this call gets the smallest power of two that brings its largest value to 448 at most (2**-40 at
    least); in a page with tokens the scale grows if it has to (or to the next power of two if it is none),
    and the page's codes are brought to the new scale.  Nothing else of the cache changes.  0-dim scales (per tensor) are read only.

    ``key_bounds``: e4m3fn ``[num_blocks, num_kv_heads, 2, head_size]``, the smallest and largest key
    code of every head dim over the page's tokens, kept up to date for
    :func:`triton_op_b200.score_blocks`.  ``status`` (int32 scalar) receives ``PA_DEV_*`` bits for rows
    that have no place; they are skipped.  No page may get rows of two sequences in a call; what is
    written (scales, codes and bounds of each page and kv head) may not share memory.  At most 8 192
    sequences.  Runs on the current stream; there is no CPU fallback.
    """
    done = _lib.calls().append(key, value, key_cache, value_cache, key_scale, value_scale, block_tables, sequence_lengths,
                               query_start_loc, key_bounds, status)
    if type(done) is tuple:
        return
    if done is not None:
        raise _lib.PaError(done, "pa_cache_append_sm100")
    on, dev = key.get_device(), key.device
    k_shape, c_shape = key.shape, key_cache.shape
    if not (key.dtype == torch.bfloat16 and value.dtype == torch.bfloat16 and k_shape == value.shape and len(k_shape) == 3):
        raise PaArgumentError("key and value must be bf16 [num_tokens, num_kv_heads, head_size] of one shape")
    if not (len(c_shape) == 5 and key_cache.dtype == FP8_DTYPE and value_cache.dtype == FP8_DTYPE):
        raise PaArgumentError(f"append_kv_cache needs {FP8_DTYPE} caches, a 5-D key_cache and a 4-D or 5-D value_cache")
    num_tokens, num_kv_heads, head_size = k_shape
    num_blocks, bs = c_shape[0], c_shape[3]
    if head_size != 128 or bs not in SUPPORTED_BLOCK_SIZES:
        raise PaArgumentError(f"head_size must be 128 and block_size in {list(SUPPORTED_BLOCK_SIZES)}, but got {head_size} and {bs}")
    if c_shape != (num_blocks, num_kv_heads, head_size // 16, bs, 16):
        raise PaArgumentError(f"key_cache must be [num_blocks, {num_kv_heads}, {head_size // 16}, block_size, 16]")
    v_shape = value_cache.shape
    trans = len(v_shape) == 5
    want_v = (num_blocks, num_kv_heads, bs // 16, head_size, 16) if trans else (num_blocks, num_kv_heads, head_size, bs)
    if v_shape != want_v:
        raise PaArgumentError(f"value_cache must be {want_v}")
    kc_stride, vc_stride = key_cache.stride(), value_cache.stride()
    if not ((kc_stride[4] == 1 and kc_stride[3] == 16 and kc_stride[2] == 16 * bs) or _inner_contiguous(key_cache, 2)) or not (
            (not trans and vc_stride[3] == 1 and vc_stride[2] == bs) or _inner_contiguous(value_cache, 2)):
        raise PaArgumentError("the per-(block, head) slabs of the KV caches must be contiguous")
    if not (_distinct(kc_stride, c_shape) and _distinct(vc_stride, c_shape)):
        raise PaArgumentError("the caches are written: every page and kv head needs a place of its own")
    if not (isinstance(key_scale, torch.Tensor) and isinstance(value_scale, torch.Tensor)
            and key_scale.dtype == torch.float32 and value_scale.dtype == torch.float32):
        raise PaArgumentError("key_scale and value_scale must be float32 tensors")
    if key_scale.dim() == 0 and value_scale.dim() == 0:
        mode, s_block, s_head = _lib.PA_QUANT_PER_TENSOR, 0, 0
    else:
        s_block, s_head = _check_block_scales(key_scale, value_scale, key_cache)
        if not _distinct((s_block, s_head), c_shape) or _meet(key_scale, value_scale):
            raise PaArgumentError("block kv scales are written: every page and kv head needs a place of its own, for its keys and for its values")
        mode = _lib.PA_QUANT_PER_BLOCK
    b_block = b_head = b_ptr = st_ptr = 0
    if key_bounds is not None:
        b_stride = key_bounds.stride()
        if not (key_bounds.dtype == FP8_DTYPE and key_bounds.shape == (num_blocks, num_kv_heads, 2, head_size)
                and b_stride[3] == 1 and b_stride[2] == head_size and key_bounds.get_device() == on):
            raise PaArgumentError(f"key_bounds must be {FP8_DTYPE} {(num_blocks, num_kv_heads, 2, head_size)} on {dev}, its last two dims contiguous")
        if not _distinct(b_stride, c_shape):
            raise PaArgumentError("key_bounds are written: every page and kv head needs a place of its own")
        b_block, b_head, b_ptr = b_stride[0], b_stride[1], key_bounds.data_ptr()
    t_shape = block_tables.shape
    num_seqs = t_shape[0]
    if not (block_tables.dtype == torch.int32 and sequence_lengths.dtype == torch.int32 and query_start_loc.dtype == torch.int32):
        raise PaArgumentError("block_tables, sequence_lengths and query_start_loc must be int32")
    if not (len(t_shape) == 2 and t_shape[1] >= 1 and sequence_lengths.numel() == num_seqs
            and query_start_loc.numel() == num_seqs + 1):
        raise PaArgumentError("block_tables must be [num_seqs, max_blocks], sequence_lengths [num_seqs] and query_start_loc [num_seqs + 1]")
    if not (value.get_device() == on and key_cache.get_device() == on and value_cache.get_device() == on
            and key_scale.get_device() == on and value_scale.get_device() == on and block_tables.get_device() == on
            and sequence_lengths.get_device() == on and query_start_loc.get_device() == on):
        raise PaArgumentError(f"all tensors must live on {dev}, the key's device")
    if status is not None:
        if not (status.dtype == torch.int32 and status.device == dev):
            raise PaArgumentError(f"status must be an int32 tensor on {dev}")
        st_ptr = status.data_ptr()
    if on < 0:
        raise RuntimeError("append_kv_cache runs on CUDA tensors only; there is no CPU fallback")
    key, key_stride = _rows(key)
    value, value_stride = _rows(value)
    if block_tables.stride(1) != 1:
        block_tables = block_tables.contiguous()
    if not sequence_lengths.is_contiguous():
        sequence_lengths = sequence_lengths.contiguous()
    if not query_start_loc.is_contiguous():
        query_start_loc = query_start_loc.contiguous()
    p = _lib.PaCacheAppendParams.from_buffer_copy(_APPEND.pack(
        _APPEND.size, _lib.PA_ABI_VERSION,
        key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_scale.data_ptr(),
        value_scale.data_ptr(), b_ptr, block_tables.data_ptr(), sequence_lengths.data_ptr(), query_start_loc.data_ptr(), st_ptr,
        num_tokens, num_seqs, num_kv_heads, head_size, bs, num_blocks, t_shape[1], mode,
        _lib.PA_V_TRANSPOSED if trans else _lib.PA_V_NORMAL, 0,
        key_stride[0], key_stride[1], value_stride[0], value_stride[1], kc_stride[0], kc_stride[1],
        vc_stride[0], vc_stride[1], s_block, s_head, b_block, b_head, block_tables.stride(0)))
    _lib.launch(on, _lib.lib().pa_cache_append_sm100, "pa_cache_append_sm100", C.byref(p))
