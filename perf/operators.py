"""Cases and plain forms of the operators around the block-scaled 8-bit cache.

The cache: e4m3fn pages of ``block`` tokens with one fp32 scale for each (page, kv head), keys
``[NB, Hkv, D/16, bs, 16]``, values ``[NB, Hkv, D, bs]``, scales ``[NB, Hkv, 1, 1]``, and for each
(page, kv head) the smallest and the largest key code of every head dim, ``[NB, Hkv, 2, D]``.

Operators:
  append    a step's keys and values quantised into the cache, scales and key bounds kept up to date
  attend    decode attention over all pages of each sequence
  score     an upper bound of the logits in each page, from the key bounds
  select    the best pages of each (sequence, kv head)
  picked    decode attention over a list of pages of each (sequence, kv head)

Each case runs in its plain form (``own`` false: elementary torch operations in 32 bits) or through
the package (``own`` true).  Lengths follow from the case alone, values and page order from the seed.
"""
import math

import torch

own = False

D = 128
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -40
OPS = ("append", "attend", "score", "select", "picked")


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one user's chat: a context just past one partition, latency is all that counts
        dict(name="attend_one_short", op="attend", seqs=1, kv_heads=8, group=4, query_len=1, block=16, lo=257, hi=257),
        # the benchmark's decode shape (64 sequences of 4096 tokens, 8 kv heads of 4 query heads)
        dict(name="attend_batch", op="attend", seqs=64, kv_heads=8, group=4, query_len=1, block=16, lo=4096, hi=4096),
        # two tokens a step (speculative), 8 query heads per kv head, long pages, ragged lengths
        dict(name="attend_two_tokens", op="attend", seqs=48, kv_heads=8, group=8, query_len=2, block=64, lo=1023, hi=8191),
        # page scores for one user's medium context
        dict(name="score_one", op="score", seqs=1, kv_heads=8, group=4, query_len=1, block=16, lo=4097, hi=4097),
        # page scores for a batch of long, ragged contexts
        dict(name="score_batch_long", op="score", seqs=32, kv_heads=8, group=4, query_len=1, block=16, lo=16385, hi=65536),
        # the best 32 pages of a medium context, one user
        dict(name="select_one", op="select", seqs=1, kv_heads=8, block=16, lo=4097, hi=4097, top_k=32),
        # the best 128 pages of long contexts, a batch
        dict(name="select_batch_long", op="select", seqs=64, kv_heads=8, block=16, lo=16385, hi=131072, top_k=128),
        # attention over the chosen 512 tokens of two users
        dict(name="picked_two_users", op="picked", seqs=2, kv_heads=8, group=4, query_len=1, block=16, lo=8001, hi=8192, top_k=32),
        # 2048 of up to 16384 tokens for a batch of 64
        dict(name="picked_batch", op="picked", seqs=64, kv_heads=8, group=4, query_len=1, block=16, lo=4001, hi=16384, top_k=128),
        # two tokens a step over 33 pages of 64 tokens, 8 query heads per kv head
        dict(name="picked_two_tokens", op="picked", seqs=24, kv_heads=8, group=8, query_len=2, block=64, lo=2049, hi=16000, top_k=33),
        # a decode step's one token per sequence
        dict(name="append_step", op="append", seqs=64, kv_heads=8, block=16, before=1000, lo=1, hi=1),
        # ragged prompt chunks that begin inside a page
        dict(name="append_prompts", op="append", seqs=8, kv_heads=8, block=16, before=517, lo=513, hi=4001),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(OPS)
    c = dict(op=op, seqs=_log_int(rng, 1, 64), kv_heads=rng.choice((1, 2, 4, 8)), block=rng.choice((16, 16, 64, 1024)))
    if op == "append":
        c["seqs"] = _log_int(rng, 1, 64)
        c["before"] = rng.randrange(0, 2000)
        c["hi"] = _log_int(rng, 1, max(1, 14000 // c["seqs"]))
        c["lo"] = rng.randint(1, c["hi"])
        return c
    if op in ("score", "select", "picked"):
        c["block"] = rng.choice((16, 16, 64))
    budget = {"attend": 262144, "score": 1048576, "select": 4194304, "picked": 524288}[op] // c["seqs"]
    c["hi"] = _log_int(rng, min(17, budget), min(131072, budget))
    c["lo"] = rng.randint(1, c["hi"])
    if op != "select":
        c["group"], c["query_len"] = rng.choice(((1, 1), (2, 1), (4, 1), (5, 1), (8, 1), (4, 2), (8, 2), (3, 3), (2, 4), (16, 1)))
    if op in ("select", "picked"):
        c["top_k"] = _log_int(rng, 3, 128 if c["block"] == 16 else 32)
    return c


def _lengths(c):
    """Ragged lengths between lo and hi that depend on the case only (golden-ratio steps)."""
    n, lo, hi = c["seqs"], c["lo"], c["hi"]
    return [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _pages(tokens, block):
    return (tokens + block - 1) // block


def _listed_pages(c):
    """(pages, tokens) that each head's list holds, for every sequence of a "picked" case."""
    got = []
    for n in _lengths(c):
        pages = _pages(n, c["block"])
        k = min(pages, c["top_k"])
        got.append((k, k * c["block"] - (pages * c["block"] - n)))
    return got


def work(c):
    """Bytes read once and written once, and operations of products (two for each multiply-add)."""
    lens, h, bs = _lengths(c), c["kv_heads"], c["block"]
    pages = sum(_pages(n, bs) for n in lens)
    rows = c.get("group", 0) * c.get("query_len", 0)
    q_bytes = len(lens) * h * rows * D * 2
    if c["op"] == "append":
        tokens = sum(lens)
        touched = sum(_pages(c["before"] + n, bs) - c["before"] // bs for n in lens)
        return {"bytes": tokens * h * D * (2 * 2 + 2) + touched * h * (8 + 2 * D) + len(lens) * 8, "flops": 0}
    if c["op"] == "attend":
        return {"bytes": sum(lens) * h * 2 * D + pages * (8 * h + 4) + 2 * q_bytes, "flops": sum(lens) * h * rows * 4 * D}
    if c["op"] == "score":
        return {"bytes": pages * h * (2 * D + 4 + 4) + pages * 4 + q_bytes, "flops": pages * h * rows * 4 * D}
    if c["op"] == "select":
        k = sum(min(_pages(n, bs), c["top_k"]) for n in lens)
        return {"bytes": pages * h * 4 + k * h * 8 + len(lens) * 8, "flops": 0}
    got = _listed_pages(c)
    tokens = sum(t for _, t in got)
    return {"bytes": tokens * h * 2 * D + sum(k for k, _ in got) * h * 12 + 2 * q_bytes, "flops": tokens * h * rows * 4 * D}


# ----------------------------------------------------------------------------- inputs
def _codes(shape, g, spread=90.0):
    """e4m3 codes as a page holds them: about normal, the largest near the end of the type's range."""
    x = torch.empty(shape, dtype=FP8, device="cuda")
    flat = x.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        part = torch.randn(n, generator=g, device="cuda", dtype=torch.bfloat16)
        flat[i:i + n] = part.mul_(spread).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
    return x


def _scales(nb, h, g, octaves=2):
    """Powers of two around 1/64, as appending to the cache makes them."""
    e = torch.randint(-6 - octaves // 2, -6 + octaves, (nb, h, 1, 1), generator=g, device="cuda")
    return torch.exp2(e.float())


def _tables(c, lens, nb, g):
    """Every sequence's pages, scattered over the pool."""
    per = [_pages(n, c["block"]) for n in lens]
    width = max(1, max(per))
    perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    t = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        t[i, :n] = perm[at:at + n]
        at += n
    return t


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 17)
    lens, h, bs = _lengths(c), c["kv_heads"], c["block"]
    s = dict(case=dict(c), block=bs)
    if c["op"] == "append":
        after = [c["before"] + n for n in lens]
        nb = sum(_pages(n, bs) for n in after) + 3
        s["block_tables"] = _tables(c, after, nb, g)
        s["lengths"] = torch.tensor(after, dtype=torch.int32, device="cuda")
        start = [0]
        for n in lens:
            start.append(start[-1] + n)
        s["start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        s["key_cache"] = _codes((nb, h, D // 16, bs, 16), g)
        s["value_cache"] = _codes((nb, h, D, bs), g)
        s["key_scale"], s["value_scale"] = _scales(nb, h, g), _scales(nb, h, g)
        k = s["key_cache"].float().permute(0, 1, 2, 4, 3).reshape(nb, h, D, bs)
        s["bounds"] = torch.stack((k.amin(-1), k.amax(-1)), 2).to(FP8)
        # tokens of very different sizes, so that some pages' scales grow and some stay
        size = torch.exp2(torch.randint(-1, 3, (start[-1], 1, 1), generator=g, device="cuda").float())
        s["key"] = (torch.randn(start[-1], h, D, generator=g, device="cuda") * size).bfloat16()
        s["value"] = (torch.randn(start[-1], h, D, generator=g, device="cuda") * size).bfloat16()
        return s
    nb = sum(_pages(n, bs) for n in lens) + 3
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["block_tables"] = _tables(c, lens, nb, g)
    if c["op"] == "select":
        width = s["block_tables"].shape[1]
        sc = torch.randn(len(lens), h, width, generator=g, device="cuda") * 4.0 + 9.0
        past = torch.arange(width, device="cuda")[None, None] * bs >= s["lengths"][:, None, None]
        s["scores"] = sc.masked_fill(past, -math.inf)
        return s
    rows = c["group"] * c["query_len"]
    s["query"] = torch.randn(len(lens), h * rows, D, generator=g, device="cuda").bfloat16()
    s["key_scale"] = _scales(nb, h, g)
    if c["op"] == "score":
        mid = torch.randn(1, h, 1, D, generator=g, device="cuda") * 60.0
        half = torch.rand(nb, h, 1, D, generator=g, device="cuda") * 90.0 + 60.0
        mid = mid + torch.randn(nb, h, 1, D, generator=g, device="cuda") * 30.0
        s["bounds"] = torch.cat((mid - half, mid + half), 2).clamp_(-FP8_MAX, FP8_MAX).to(FP8)
        return s
    s["key_cache"] = _codes((nb, h, D // 16, bs, 16), g)
    s["value_cache"] = _codes((nb, h, D, bs), g)
    s["value_scale"] = _scales(nb, h, g)
    s["longest"] = max(lens)
    if c["op"] == "picked":
        # any pages of the context and its last one, in order: what a selection hands over
        width = s["block_tables"].shape[1]
        pages = ((s["lengths"] + bs - 1) // bs).long()
        r = torch.rand(len(lens), h, width, generator=g, device="cuda")
        at = torch.arange(width, device="cuda")[None, None]
        r = r.masked_fill(at >= pages[:, None, None] - (1 if c["query_len"] == 1 else 2), 2.0)
        r = r.masked_fill(at >= pages[:, None, None], -1.0)
        k = min(c["top_k"], width)
        picked = r.topk(k, dim=-1).indices
        live = picked < pages[:, None, None]
        picked = picked.masked_fill(~live, width).sort(-1).values
        live = picked < width
        tables = torch.gather(s["block_tables"][:, None].expand(-1, h, -1), 2, picked.clamp_max(width - 1))
        s["tables"] = tables.masked_fill(~live, 0).contiguous()
        s["picked_lengths"] = torch.tensor([t for _, t in _listed_pages(c)], dtype=torch.int32, device="cuda")
        s["longest"] = k * bs
    s["out"] = torch.empty_like(s["query"])
    return s


# ----------------------------------------------------------------------------- one pass
SCALE = D ** -0.5


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(op, s)
    return {"append": _append, "attend": _attend, "score": _score, "select": _select, "picked": _picked}[op](s)


def _own(op, s):
    import triton_op_b200 as pa
    if op == "append":
        pa.append_kv_cache(s["key"], s["value"], s["key_cache"], s["value_cache"], s["key_scale"], s["value_scale"],
                           s["block_tables"], s["lengths"], s["start"], key_bounds=s["bounds"])
        return _cache(s)
    if op == "score":
        return pa.score_blocks(s["query"], s["bounds"], s["lengths"], s["block_tables"], SCALE, s["case"]["query_len"],
                               s["block"], key_scale=s["key_scale"])
    if op == "select":
        return pa.select_blocks(s["scores"], s["lengths"], s["block_tables"], s["block"], s["case"]["top_k"],
                                keep_first=1, keep_last=1)
    lengths, tables = (s["lengths"], s["block_tables"]) if op == "attend" else (s["picked_lengths"], s["tables"])
    pa.paged_attention_decode(s["out"], s["query"], s["key_cache"], s["value_cache"], lengths, tables, SCALE,
                              s["case"]["query_len"], s["longest"], torch.bfloat16, None, s["key_scale"], s["value_scale"])
    return s["out"]


def _cache(s):
    return {k: s[k] for k in ("key_cache", "value_cache", "key_scale", "value_scale", "bounds")}


def _rows_of(x, ids):
    """x[ids] along the first dim for 8-bit floats."""
    return x.view(torch.uint8)[ids].view(FP8)


def _place(t, start, lengths, tables, bs):
    """(sequence, page id, offset inside the page) of every token row of an append."""
    row = torch.arange(t, device=start.device)
    seq = torch.searchsorted(start[1:].long(), row, right=True)
    pos = lengths.long()[seq] - (start.long()[seq + 1] - row)
    return tables.long()[seq, pos // bs], pos % bs


def _grown(x, old, page, first, fp):
    """The pages' scales after rows x [T, Hkv, D] joined them: (scales [NB, Hkv], touched [NB], begun [NB])."""
    nb, h = old.shape[:2]
    top = torch.zeros(nb, h, dtype=fp, device=x.device)
    top.scatter_reduce_(0, page[:, None].expand(-1, h), x.to(fp).abs().amax(-1), "amax")
    # the smallest power of two that brings the largest value to 448 at most
    m, e = torch.frexp(top / FP8_MAX)
    want = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e)).clamp_min(SMALLEST_SCALE)
    want = torch.where(top > 0, want, torch.full_like(want, SMALLEST_SCALE))
    touched = torch.zeros(nb, dtype=torch.bool, device=x.device).index_fill_(0, page, True)
    begun = torch.zeros(nb, dtype=torch.bool, device=x.device).index_fill_(0, page[first], True)
    kept = torch.maximum(old[:, :, 0, 0].to(fp), want)
    new = torch.where(begun[:, None], want, kept)
    return torch.where(touched[:, None], new, old[:, :, 0, 0].to(fp)), touched, begun


def _append(s):
    page, off = _place(s["key"].shape[0], s["start"], s["lengths"], s["block_tables"], s["block"])
    begun, ids, ratio, q = _joined(s, "key", page, off)
    lo, hi = s["bounds"].float().unbind(2)
    lo, hi = lo.clone(), hi.clone()
    lo[ids], hi[ids] = (lo[ids] * ratio[..., None]).to(FP8).float(), (hi[ids] * ratio[..., None]).to(FP8).float()
    lo.masked_fill_(begun[:, None, None], math.inf)
    hi.masked_fill_(begun[:, None, None], -math.inf)
    at = page[:, None, None].expand(-1, q.shape[1], D)
    lo.scatter_reduce_(0, at, q.float(), "amin")
    hi.scatter_reduce_(0, at, q.float(), "amax")
    s["bounds"].copy_(torch.stack((lo, hi), 2).to(FP8))
    s["key_cache"].view(torch.uint8)[page, :, :, off] = q.view(torch.uint8).view(q.shape[0], q.shape[1], D // 16, 16)
    q = _joined(s, "value", page, off)[-1]
    s["value_cache"].view(torch.uint8)[page, :, :, off] = q.view(torch.uint8)
    return _cache(s)


def _joined(s, name, page, off):
    """Brings the touched pages of one cache to their new scales; (begun, grown pages, their ratios, the rows' codes)."""
    x, cache, scale = s[name].float(), s[name + "_cache"], s[name + "_scale"]
    new, touched, begun = _grown(x, scale, page, off == 0, torch.float32)
    ids = (touched & ~begun).nonzero()[:, 0]
    ratio = scale[ids, :, 0, 0] / new[ids]
    codes = _rows_of(cache, ids).float()
    codes = (codes * ratio.view(ratio.shape + (1,) * (codes.dim() - 2))).to(FP8)
    cache.view(torch.uint8)[ids] = codes.view(torch.uint8)
    scale.copy_(new[:, :, None, None])
    return begun, ids, ratio, (x / new[page][:, :, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8)


def _attention(s, tables, lengths):
    """Attention of every query row over the pages of tables [S, Hkv, K]."""
    n, h, k = tables.shape
    bs, ql, heads = s["block"], s["case"]["query_len"], torch.arange(h, device=tables.device)[None, :, None]
    ids = tables.long()
    keys = s["key_cache"].view(torch.uint8)[ids, heads].view(FP8).float()              # [S, H, K, D/16, bs, 16]
    keys = keys * s["key_scale"][ids, heads].unsqueeze(-1)
    keys = keys.permute(0, 1, 2, 4, 3, 5).reshape(n, h, k * bs, D)
    q = s["query"].float().view(n, h, -1, D)
    logits = torch.matmul(q, keys.transpose(-1, -2)) * SCALE
    del keys
    rows = q.shape[2]
    ahead = ql - 1 - torch.arange(rows, device=q.device) // (rows // ql)                # row t*G + g holds token t
    seen = torch.arange(k * bs, device=q.device)[None, None, None] + ahead[None, None, :, None] < lengths[:, None, None, None]
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top.isinf(), torch.zeros_like(top), top))
    del logits, seen
    total = p.sum(-1, keepdim=True)
    values = s["value_cache"].view(torch.uint8)[ids, heads].view(FP8).float()          # [S, H, K, D, bs]
    values = values * s["value_scale"][ids, heads]
    values = values.permute(0, 1, 2, 4, 3).reshape(n, h, k * bs, D)
    o = torch.matmul(p, values) / torch.where(total > 0, total, torch.ones_like(total))
    return o.reshape(n, h * rows, D).bfloat16()


def _attend(s):
    h = s["key_cache"].shape[1]
    return _attention(s, s["block_tables"][:, None].expand(-1, h, -1), s["lengths"])


def _picked(s):
    return _attention(s, s["tables"], s["picked_lengths"])


def _score(s):
    ids, bs = s["block_tables"].long(), s["block"]
    n, width = ids.shape
    h = s["bounds"].shape[1]
    lo, hi = _rows_of(s["bounds"], ids).float().permute(0, 2, 3, 1, 4).unbind(2)       # [S, H, P, D]
    q = s["query"].float().view(n, h, -1, D)
    u = torch.matmul(q.clamp_min(0), hi.transpose(-1, -2)) + torch.matmul(q.clamp_max(0), lo.transpose(-1, -2))
    u = (u * SCALE).amax(2) * s["key_scale"][ids][..., 0, 0].transpose(1, 2)
    past = torch.arange(width, device=q.device)[None, None] * bs >= s["lengths"][:, None, None]
    return u.masked_fill(past, -math.inf)


def _select(s):
    c, bs = s["case"], s["block"]
    scores, lengths = s["scores"], s["lengths"].long()
    n, h, width = scores.shape
    pages = (lengths + bs - 1) // bs
    at = torch.arange(width, device=scores.device)[None, None]
    key = scores.masked_fill(scores.isnan(), -math.inf)
    key = key.masked_fill((at < 1) | (at >= pages[:, None, None] - 1), math.inf)
    key = key.masked_fill(at >= pages[:, None, None], -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    k = c["top_k"]
    if width < k:
        order = torch.cat((order, torch.full((n, h, k - width), width, device=order.device)), -1)
    best = order[..., :k]
    best = best.masked_fill(torch.arange(k, device=order.device)[None, None] >= pages[:, None, None], width).sort(-1).values
    tables = torch.gather(s["block_tables"][:, None].expand(-1, h, -1), 2, best.clamp_max(width - 1))
    tables = tables.masked_fill(best >= width, 0)
    held = pages.clamp_max(k)
    tokens = held * bs - (pages * bs - lengths)
    return tables, tokens.to(torch.int32)


# ----------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(c, seed):
    def append(s):
        """Token by token would be the same: a page's rows share one scale, fixed by the page's old one and the rows' largest value."""
        bs = s["block"]
        lens, start = s["lengths"].tolist(), s["start"].tolist()
        tables = s["block_tables"].tolist()
        out = {k: s[k].double() for k in ("key_cache", "value_cache", "key_scale", "value_scale", "bounds")}

        def rounded(x):
            return x.clamp(-FP8_MAX, FP8_MAX).float().to(FP8).double()

        for i, n in enumerate(lens):
            at = n - (start[i + 1] - start[i])
            row = start[i]
            while at < n:
                page, first = tables[i][at // bs], at % bs
                count = min(bs - first, n - at)
                for name in ("key", "value"):
                    x = s[name][row:row + count].double()                                  # [count, Hkv, D]
                    top = x.abs().amax((0, 2))
                    near = torch.log2(top.clamp_min(1e-30) / FP8_MAX).round()                # the power is this, or one off
                    want = torch.where(FP8_MAX * torch.exp2(near - 1) >= top, torch.exp2(near - 1),
                                       torch.where(FP8_MAX * torch.exp2(near) >= top, torch.exp2(near), torch.exp2(near + 1)))
                    want = want.clamp_min(SMALLEST_SCALE)
                    old = out[name + "_scale"][page, :, 0, 0]
                    scale = want if first == 0 else torch.maximum(old, want)
                    pages = out[name + "_cache"][page]                                     # [Hkv, ...]
                    if first:
                        pages = rounded(pages * (old / scale).view(-1, 1, *[1] * (pages.dim() - 2)))
                    codes = rounded(x / scale[None, :, None])
                    if name == "key":
                        pages[:, :, first:first + count] = codes.view(count, -1, D // 16, 16).permute(1, 2, 0, 3)
                        lo, hi = codes.amin(0), codes.amax(0)
                        if first:
                            was = rounded(out["bounds"][page] * (old / scale)[:, None, None])
                            lo, hi = torch.minimum(lo, was[:, 0]), torch.maximum(hi, was[:, 1])
                        out["bounds"][page] = torch.stack((lo, hi), 1)
                    else:
                        pages[:, :, first:first + count] = codes.permute(1, 2, 0)
                    out[name + "_cache"][page] = pages
                    out[name + "_scale"][page, :, 0, 0] = scale
                at += count
                row += count
        return out

    def attention(s):
        picked = s["case"]["op"] == "picked"
        lengths = (s["picked_lengths"] if picked else s["lengths"]).tolist()
        bs, ql = s["block"], s["case"]["query_len"]
        h = s["key_cache"].shape[1]
        out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
        for i, n in enumerate(lengths):
            if n == 0:
                continue
            pages = _pages(n, bs)
            for j in range(h):
                ids = (s["tables"][i, j, :pages] if picked else s["block_tables"][i, :pages]).long()
                k = s["key_cache"][:, j].view(torch.uint8)[ids].view(FP8).double() * s["key_scale"][ids, j].double()[..., None]
                v = s["value_cache"][:, j].view(torch.uint8)[ids].view(FP8).double() * s["value_scale"][ids, j].double()
                k = k.transpose(1, 2).reshape(pages * bs, D)[:n]
                v = v.transpose(1, 2).reshape(pages * bs, D)[:n]
                rows = s["query"].shape[1] // h
                q = s["query"][i, j * rows:(j + 1) * rows].double()
                l = q @ k.T / math.sqrt(D)
                for r in range(rows):
                    visible = n - (ql - 1 - r // (rows // ql))
                    if visible > 0:
                        out[i, j * rows + r] = torch.softmax(l[r, :visible], 0) @ v[:visible]
        return out

    def score(s):
        bs = s["block"]
        n, width = s["block_tables"].shape
        h = s["bounds"].shape[1]
        out = torch.full((n, h, width), -math.inf, dtype=torch.float64, device="cuda")
        for i, tokens in enumerate(s["lengths"].tolist()):
            pages = _pages(tokens, bs)
            ids = s["block_tables"][i, :pages].long()
            b = s["bounds"].view(torch.uint8)[ids].view(FP8).double()                       # [P, H, 2, D]
            q = s["query"][i].double().view(h, -1, D)
            best = None
            for r in range(q.shape[1]):
                u = torch.maximum(q[:, r] * b[:, :, 0], q[:, r] * b[:, :, 1]).sum(-1) / math.sqrt(D)
                best = u if best is None else torch.maximum(best, u)
            out[i, :, :pages] = (best * s["key_scale"][ids, :, 0, 0].double()).T
        return out

    if c["op"] == "select":
        return None
    return {"append": append, "attend": attention, "picked": attention, "score": score}[c["op"]](prepare(c, seed))
