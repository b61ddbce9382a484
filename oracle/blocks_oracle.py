"""The operators around a cache with scales per (page, kv head), from their definitions in 64 bits.

Loops over sequences, heads and pages, torch CPU tensors, no code shared with the package.  Test
infrastructure only.  Layouts: keys ``[NB, Hkv, D/16, bs, 16]``, values ``[NB, Hkv, D, bs]`` or
``[NB, Hkv, bs/16, D, 16]``, scales ``[NB, Hkv, 1, 1]``, key bounds ``[NB, Hkv, 2, D]``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
MIN_SCALE = 2.0 ** -40


def codes(t: torch.Tensor) -> torch.Tensor:
    """An e4m3fn tensor's values in 64 bits."""
    return t.float().double()


def to_fp8(x: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3fn value (ties to even), saturating; NaN stays NaN."""
    return x.clamp(-FP8_MAX, FP8_MAX).float().to(FP8)


def key_page(key_cache: torch.Tensor, page: int, head: int) -> torch.Tensor:
    """Codes [bs, D] of a page's keys."""
    p = codes(key_cache[page, head])                     # [D/16, bs, 16]
    return p.permute(1, 0, 2).reshape(p.shape[1], -1)


def value_page(value_cache: torch.Tensor, page: int, head: int) -> torch.Tensor:
    """Codes [bs, D] of a page's values."""
    p = codes(value_cache[page, head])
    if p.dim() == 2:                                     # [D, bs]
        return p.T
    return p.permute(0, 2, 1).reshape(-1, p.shape[1])    # [bs/16, D, 16]


def power_scale(amax: float) -> float:
    """The smallest power of two s with amax <= 448 s, at least 2^-40."""
    s = MIN_SCALE
    while s * FP8_MAX < amax:
        s *= 2.0
    return s


def append(key, value, key_cache, value_cache, key_scale, value_scale, block_tables, lengths, start, key_bounds=None):
    """In place on CPU tensors.  Per-tensor scales (0-dim) are read only."""
    bs = key_cache.shape[3]
    per_block = key_scale.dim() == 4
    for s in range(len(lengths)):
        n, first_row = int(lengths[s]), int(start[s])
        count = int(start[s + 1]) - first_row
        pos = n - count
        while pos < n:
            page, slot = int(block_tables[s, pos // bs]), pos % bs
            rows = min(bs - slot, n - pos)
            for h in range(key.shape[1]):
                for x, cache, scale in ((key, key_cache, key_scale), (value, value_cache, value_scale)):
                    new = x[first_row:first_row + rows, h].double()              # [rows, D]
                    is_key = cache is key_cache
                    old_page = key_page(cache, page, h) if is_key else value_page(cache, page, h)
                    bounds = codes(key_bounds[page, h]) if is_key and key_bounds is not None else None
                    if per_block:
                        finite = new[torch.isfinite(new)]
                        want = power_scale(float(finite.abs().max()) if finite.numel() else 0.0)
                        old = float(scale[page, h, 0, 0])
                        use = want if slot == 0 else max(2.0 ** math.ceil(math.log2(old)), want)
                        if slot > 0 and use != old:
                            ratio = torch.tensor(old / use, dtype=torch.float32).double()
                            old_page = codes(to_fp8((old_page * ratio).float()))
                            if bounds is not None:
                                bounds = codes(to_fp8((bounds * ratio).float()))
                        scale[page, h, 0, 0] = use
                    else:
                        use = float(scale)
                    # one rounding to 32 bits (the quotient), then one to 8
                    q = codes(to_fp8((new.float() / torch.tensor(use, dtype=torch.float32))))
                    page_codes = old_page.clone()
                    page_codes[slot:slot + rows] = q
                    packed = page_codes.float().to(FP8)
                    if is_key:
                        cache[page, h] = packed.view(bs, -1, 16).permute(1, 0, 2)
                        if bounds is not None:
                            seen = q.clone()
                            lo = torch.where(seen.isnan(), math.inf, seen).amin(0)
                            hi = torch.where(seen.isnan(), -math.inf, seen).amax(0)
                            if slot > 0:
                                lo, hi = torch.minimum(lo, bounds[0]), torch.maximum(hi, bounds[1])
                            key_bounds[page, h] = to_fp8(torch.stack((lo, hi)))
                    elif cache.dim() == 4:
                        cache[page, h] = packed.T
                    else:
                        cache[page, h] = packed.view(bs // 16, 16, -1).permute(0, 2, 1)
            pos += rows
            first_row += rows


def attention(query, key_cache, value_cache, key_scale, value_scale, block_tables, lengths, softmax_scale: float,
              query_len: int, alibi_slopes=None, sink_tokens=None, query_scale=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(output, sum_j w_j |v_j|, max_j(w_j sV_j) sum_j |code_j|) in 64 bits, all [S, Hkv*rows, D]; w the softmax.

    ``block_tables`` [S, pages] or [S, Hkv, pages]; scales [NB, Hkv, 1, 1], 0-dim or None.
    """
    num_seqs, q_heads, d = query.shape
    hkv, bs = key_cache.shape[1], key_cache.shape[3]
    rows = q_heads // hkv
    group = rows // query_len
    out = torch.zeros(query.shape, dtype=torch.float64)
    mass, floor = torch.zeros_like(out), torch.zeros_like(out)

    def scale_of(scale, page, head) -> float:
        if scale is None:
            return 1.0
        return float(scale) if scale.dim() == 0 else float(scale[page, head, 0, 0])

    for s in range(num_seqs):
        n = int(lengths[s])
        if n == 0:
            continue
        for h in range(hkv):
            table = block_tables[s, h] if block_tables.dim() == 3 else block_tables[s]
            ids = [int(table[i]) for i in range((n + bs - 1) // bs)]
            k = torch.cat([key_page(key_cache, i, h) * scale_of(key_scale, i, h) for i in ids])[:n]
            vc = torch.cat([value_page(value_cache, i, h) for i in ids])[:n]
            vs = torch.cat([torch.full((bs, 1), scale_of(value_scale, i, h), dtype=torch.float64) for i in ids])[:n]
            for r in range(rows):
                t, g = divmod(r, group)
                visible = n - (query_len - 1 - t)
                if visible <= 0:
                    continue
                row = h * rows + r
                q = query[s, row].float().double()
                if query_scale is not None:
                    q = q * (float(query_scale) if query_scale.dim() == 0 else float(query_scale[s, row, 0]))
                logits = (k[:visible] @ q) * softmax_scale
                if alibi_slopes is not None:
                    logits = logits + float(alibi_slopes[h * group + g]) * (torch.arange(visible) - (n - 1)).double()
                top = logits.max()
                w = torch.exp(logits - top)
                total = w.sum()
                if sink_tokens is not None:
                    total = total + math.exp(float(sink_tokens[h * group + g]) - float(top))
                w = (w / total)[:, None]
                v = vc[:visible] * vs[:visible]
                out[s, row] = (w * v).sum(0)
                mass[s, row] = (w * v.abs()).sum(0)
                floor[s, row] = (w * vs[:visible]).max() * vc[:visible].abs().sum(0)
    return out, mass, floor


def attention_tolerance(out, mass, floor) -> torch.Tensor:
    """What the kernel's roundings can add up to: probabilities as two e4m3 numbers (2^-7 of each, and 2^-18
    of the largest weighted value scale below the subnormals), bf16 partial outputs (2^-8 of each; only where a
    caller's workspaces hold them so) and the bf16 result (2^-8), with 2^-12 for everything that is held in 32 bits."""
    return (2.0 ** -7 + 2.0 ** -8 + 2.0 ** -12) * mass + 2.0 ** -8 * out.abs() + 2.0 ** -18 * floor


def scores(query, key_bounds, lengths, block_tables, softmax_scale: float, bs: int, key_scale=None, query_scale=None
           ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(scores, the largest sum of absolute terms behind each) [S, Hkv, pages]; -inf past the context."""
    num_seqs, q_heads, d = query.shape
    hkv = key_bounds.shape[1]
    rows = q_heads // hkv
    width = block_tables.shape[1]
    out = torch.full((num_seqs, hkv, width), -math.inf, dtype=torch.float64)
    terms = torch.zeros_like(out)
    for s in range(num_seqs):
        pages = min(width, (max(int(lengths[s]), 0) + bs - 1) // bs)
        for h in range(hkv):
            q = query[s, h * rows:(h + 1) * rows].float().double()
            if query_scale is not None:
                q = q * (query_scale.double() if query_scale.dim() == 0 else query_scale[s, h * rows:(h + 1) * rows].double())
            for i in range(pages):
                page = int(block_tables[s, i])
                lo, hi = codes(key_bounds[page, h])
                factor = softmax_scale
                if key_scale is not None:
                    factor *= float(key_scale) if key_scale.dim() == 0 else float(key_scale[page, h, 0, 0])
                term = torch.maximum(q * lo, q * hi)
                out[s, h, i] = factor * term.sum(-1).max()
                terms[s, h, i] = factor * term.abs().sum(-1).max()
    return out, terms


def select(score, lengths, block_tables, bs: int, top_k: int, keep_first: int = 1, keep_last: int = 1
           ) -> Tuple[torch.Tensor, torch.Tensor]:
    num_seqs, hkv, _ = score.shape
    width = block_tables.shape[1]
    tables = torch.zeros(num_seqs, hkv, top_k, dtype=torch.int32)
    tokens = torch.zeros(num_seqs, dtype=torch.int32)
    for s in range(num_seqs):
        n = min(max(int(lengths[s]), 0), width * bs)
        pages = (n + bs - 1) // bs
        held = min(pages, top_k)
        tokens[s] = held * bs - (pages * bs - n)
        for h in range(hkv):
            def rank(i: int):
                if i < keep_first or i >= pages - keep_last:
                    return (0, 0.0, i)
                x = float(score[s, h, i])
                return (1, math.inf if math.isnan(x) else -x, i)      # NaN as -inf
            best = sorted(sorted(range(pages), key=rank)[:held])
            for place, i in enumerate(best):
                tables[s, h, place] = block_tables[s, i]
    return tables, tokens
