"""Calls around a cache with scales per (page, kv head) that are easy to get wrong: where a rounding hides, where
two writers meet, what the host path refuses, host threads, far pages."""
import ctypes as C
import math

import pytest
import torch

import triton_op_b200 as pa
from oracle import blocks_oracle as bo
from test_block_cache import D, FP8, SCALE, Cache, assert_attention, assert_same, cuda, decode, serve, transposed
from triton_op_b200 import PaArgumentError, _lib
from triton_op_b200.pa_decode import build_params
from triton_op_b200.sharding import KvShardedDecoder, decode_kv_shard, local_block_table, merge_triples_cuda, plan_kv_shards


# ----------------------------------------------------------------------------- attention: what is rounded, and when
def cancelling(c):
    """Values whose means are large in every partition of 256 tokens and cancel between them."""
    for s, n in enumerate(c.lengths.tolist()):
        for i in range(-(-n // c.bs)):
            page = int(c.tables[s, i])
            v = c.value[page].float().abs() + 64.0                       # [Hkv, D, bs]
            sign = 1.0 - 2.0 * ((torch.arange(c.bs) + i * c.bs) // 256 % 2)
            c.value[page] = (v * sign).clamp(-448, 448).to(FP8)


def assert_rounded_once(got, want):
    """Equal logits are exact probabilities (one e4m3 number each, no remainder), so what is left are sums in
    32 bits -- 256 products a partition, which the tensor core may truncate (2^-23 each), and 16 partitions at most -- and the
    bf16 result, half a step of its own value."""
    out, mass, _ = want
    err = (got.double() - out).abs()
    assert bool((err <= 2.0 ** -8 * out.abs() + 2.0 ** -14 * mass).all()), float((err / mass).max())


@pytest.mark.gpu
@pytest.mark.parametrize("bs,group,query_len", [(16, 4, 1), (16, 8, 1), (16, 8, 2), (64, 2, 1), (64, 16, 1), (1024, 6, 1), (1024, 16, 4)])
def test_partial_outputs_are_not_rounded(bs, group, query_len):
    c = Cache([2000, 257, 512, 3900], 2, bs, seed=bs + group)
    cancelling(c)
    c.vs[:] = 2.0 ** -3
    q = torch.zeros_like(c.query(group, query_len))
    got = decode(c, q, query_len=query_len)
    assert_rounded_once(got, bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, query_len))


@pytest.mark.gpu
@pytest.mark.parametrize("scales", ["none", "one value", "per page"])
@pytest.mark.parametrize("hkv", [1, 3])
def test_partial_outputs_are_not_rounded_with_a_table_per_head(hkv, scales):
    c = Cache([2000, 600], hkv, 16, seed=hkv)
    cancelling(c)
    c.vs[:] = 0.25
    q = torch.zeros_like(c.query(4))
    ks, vs = dict([("none", (None, None)), ("one value", (torch.tensor(0.5), torch.tensor(0.25))), ("per page", (c.ks, c.vs))])[scales]
    tables = c.tables[:, None].expand(-1, hkv, -1).contiguous()
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    res = pa.paged_attention_decode(out, *cuda(q, c.key, c.value, c.lengths, tables), SCALE, 1, 2000, torch.bfloat16, None, *cuda(ks, vs))
    assert res["temporary_output"].dtype == torch.float32
    assert_rounded_once(out.cpu(), bo.attention(q, c.key, c.value, ks, vs, tables, c.lengths, SCALE, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("parts", [40, 140])
@pytest.mark.parametrize("seqs", [1, 40])
def test_many_partitions_are_merged_from_whole_outputs(parts, seqs):
    """Each way of merging: a warp, eight warps or sixteen warps a row."""
    c = Cache([parts * 256 - 9] + [700] * (seqs - 1), 2, 64, seed=parts)
    cancelling(c)
    c.vs[:] = 0.5
    q = torch.zeros_like(c.query(8))
    got = decode(c, q)
    out, mass, _ = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 1)
    err = (got.double() - out).abs()
    assert bool((err <= 2.0 ** -8 * out.abs() + 2.0 ** -14 * mass).all()), float((err / mass).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_workspaces_of_the_caller(dtype):
    """A workspace in 32 bits rounds nothing; one in the output's type rounds each partition (2^-8 of it) as it says."""
    c = Cache([2000, 300], 2, 16, seed=4)
    cancelling(c)
    c.vs[:] = 0.5
    q = torch.zeros_like(c.query(4))
    shape = (2, 2, 8, 4)
    kw = dict(exp_sums=torch.empty(shape, device="cuda"), max_logits=torch.empty(shape, device="cuda"),
              tmp_output=torch.empty(*shape, D, dtype=dtype, device="cuda"))
    got = decode(c, q, **kw)
    out, mass, _ = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 1)
    slack = 2.0 ** -14 if dtype == torch.float32 else 2.0 ** -14 + 2.0 ** -8
    assert bool(((got.double() - out).abs() <= 2.0 ** -8 * out.abs() + slack * mass).all())
    with pytest.raises(PaArgumentError):
        decode(c, q, **{**kw, "tmp_output": torch.empty(*shape, D, dtype=torch.float16, device="cuda")})


@pytest.mark.parametrize("given", [(), ("exp_sums", "max_logits"), ("tmp_output",)])
def test_block_scales_never_share_workspaces(given):
    """Two calls of one shape, as two streams or two captured graphs make them, whatever their options."""
    c = Cache([600, 40], 2, 16)
    q = c.query(3)
    shape = (2, 2, 3, 3)
    mine = dict(exp_sums=torch.empty(shape), max_logits=torch.empty(shape), tmp_output=torch.empty(*shape, D))
    blocks = [build_params(torch.empty_like(q), q, c.key, c.value, c.lengths, c.tables, SCALE, 1, 600, None, None, c.ks, c.vs, None, 256,
                           *(mine[n] if n in given else None for n in mine), None, dict(fuse=1)) for _ in range(2)]
    for name, field in (("exp_sums", "exp_sums"), ("max_logits", "max_logits"), ("tmp_output", "tmp_out")):
        a, b = (getattr(p, field) for p, _ in blocks)
        assert (a == b == mine[name].data_ptr()) if name in given else (a != b), name


@pytest.mark.gpu
def test_timed_calls_keep_their_workspaces():
    c = Cache([600, 40], 2, 16, seed=8)
    q = cuda(c.query(3))
    res = [pa.paged_attention_decode(torch.empty_like(q), q * k, *cuda(c.key, c.value, c.lengths, c.tables), SCALE, 1, 600, torch.bfloat16, None,
                                     *cuda(c.ks, c.vs), time_kernels=True) for k in (1, 3)]
    assert not torch.equal(res[0]["maximum_logits"], res[1]["maximum_logits"])
    plain = pa.paged_attention_decode(torch.empty_like(q), q, *cuda(c.key, c.value, c.lengths, c.tables), SCALE, 1, 600, torch.bfloat16, None, *cuda(c.ks, c.vs))
    assert torch.equal(plain["final_output"], res[0]["final_output"])
    assert torch.equal(plain["maximum_logits"][0], res[0]["maximum_logits"][0])


def at_token(c, cache, seq, token, head):
    """(page, slot) of a token, and a writable uint8 view of its page and kv head."""
    page, slot = int(c.tables[seq, token // c.bs]), token % c.bs
    return cache.view(torch.uint8)[page, head], slot


def assert_attention_but(got, want, nan):
    """The attention wherever `nan` [S, heads, D] is false, NaN wherever it is true."""
    assert torch.equal(got.isnan(), nan), (int(got.isnan().sum()), int(nan.sum()), int((got.isnan() & nan).sum()))
    out, mass, floor = want
    err = (got.double() - out).abs()
    assert bool((err <= bo.attention_tolerance(out, mass, floor))[~nan].all())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [200, 2000, 9000, 36000])
@pytest.mark.parametrize("bs,group,query_len", [(16, 4, 1), (64, 8, 1), (1024, 4, 4)])
def test_what_is_no_number_stays_none(bs, group, query_len, tokens):
    """A NaN that a row attends to reaches that row, whichever partition it lies in, and no other row; so does an infinite
    query element, whose logits have no softmax."""
    c = Cache([tokens, 700, 300, 500, 40], 2, bs, seed=tokens + bs)
    q = c.query(group, query_len)
    want = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, query_len)
    rows = group * query_len
    nan = torch.zeros(q.shape, dtype=torch.bool)
    q[0, 1, 17], nan[0, 1] = math.nan, True                             # a query row of head 0
    q[1, rows, 3], nan[1, rows] = math.inf, True                        # one of head 1
    page, slot = at_token(c, c.key, 0, tokens // 2, 1)                  # a key element: every row of the head
    page[3, slot, 5], nan[0, rows:] = 0x7f, True
    page, slot = at_token(c, c.value, 1, 650, 0)                        # a value element: its head dim
    page[77, slot], nan[1, :rows, 77] = 0xff, True
    c.ks[int(c.tables[2, 0]), 0], nan[2, :rows] = math.nan, True        # scales of pages in use
    c.vs[int(c.tables[3, 0]), 1], nan[3, rows:] = math.nan, True
    assert_attention_but(decode(c, q, query_len=query_len), want, nan)
    if query_len == 1:                                                   # tables per head, and the pieces of a sharded call
        heads = c.tables[:, None].expand(-1, 2, -1).contiguous()
        assert_attention_but(decode(c, q, tables=heads), want, nan)
        kc, vc, ks, vs, tables, dq = cuda(c.key, c.value, c.ks, c.vs, c.tables, q)
        plan = plan_kv_shards(c.lengths.tolist(), 2, max(256, bs), 1)
        triples = [decode_kv_shard(dq, kc, vc, plan[r], local_block_table(tables, plan[r], bs), SCALE, ks, vs) for r in range(2)]
        got = merge_triples_cuda(*(torch.stack([t[i] for t in triples]) for i in range(3)))
        assert_attention_but(got.view(q.shape).cpu(), want, nan)


@pytest.mark.gpu
def test_what_is_no_number_stays_none_among_many_rows():
    """Rows of 33 to 128 partitions among many short ones, which eight warps share: a NaN in a later chunk of 32, and
    rows that are NaN throughout."""
    c = Cache([9000, 20000] + [300] * 40, 2, 16, seed=77)
    q = c.query(8)
    want = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 1)
    nan = torch.zeros(q.shape, dtype=torch.bool)
    page, slot = at_token(c, c.key, 0, 8700, 1)
    page[0, slot, 0], nan[0, 8:] = 0x7f, True
    for row in (0, 5):
        q[1, row, 100], nan[1, row] = math.nan, True
    q[7, 3, 1], nan[7, 3] = -math.inf, True
    assert_attention_but(decode(c, q), want, nan)


@pytest.mark.gpu
def test_what_is_no_number_stays_none_in_the_callers_workspaces():
    c = Cache([900, 40], 2, 16, seed=6)
    q = c.query(4)
    want = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 1)
    nan = torch.zeros(q.shape, dtype=torch.bool)
    q[0, 2, 0], nan[0, 2] = math.nan, True
    for dtype in (torch.float32, torch.bfloat16):
        shape = (2, 2, 4, 4)
        got = decode(c, q, exp_sums=torch.empty(shape, device="cuda"), max_logits=torch.empty(shape, device="cuda"),
                     tmp_output=torch.empty(*shape, D, dtype=dtype, device="cuda"))
        assert_attention_but(got, want, nan)


# ----------------------------------------------------------------------------- scores
def scores_of(q, bounds, lengths, tables, bs, ks, query_len=1, **kw):
    return pa.score_blocks(*cuda(q, bounds, lengths, tables), SCALE, query_len, bs, key_scale=cuda(ks), **kw).cpu()


def assert_scores(got, want, terms):
    """256 products added in 32 bits, whose additions may truncate (2^-23 each), and three more roundings."""
    live = want > -math.inf
    assert torch.equal(got > -math.inf, live)
    assert bool(((got.double() - want).abs()[live] <= (260 * 2.0 ** -23) * terms[live]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,group", [(1, 2), (2, 3), (8, 1), (2, 12), (1, 40)])
def test_scores_through_every_slot_of_the_ring(hkv, group):
    """Launches that each set the ring's barriers up anew and use all of them at once, with other inputs every time."""
    c = Cache([16 * 16 * 148 * 3 + 5, 90], hkv, 16, seed=hkv + group, spare=1)
    for _ in range(3):
        q = c.query(group)
        got = scores_of(q, c.bounds(), c.lengths, c.tables, 16, c.ks)
        ids = c.tables[0].long()
        lo, hi = bo.codes(c.bounds()[ids]).permute(2, 1, 0, 3)                 # [Hkv, pages, D]
        rows = q[0].double().view(hkv, group, D)
        terms = rows.clamp_min(0) @ hi.abs().transpose(1, 2) + (-rows.clamp_max(0)) @ lo.abs().transpose(1, 2)
        want = rows.clamp_min(0) @ hi.transpose(1, 2) + rows.clamp_max(0) @ lo.transpose(1, 2)
        factor = SCALE * c.ks[ids, :, 0, 0].double().T
        assert_scores(got[0], want.amax(1) * factor, terms.amax(1) * factor)
        assert bool((got[1, :, 6:] == -math.inf).all()) and not bool((got[1, :, :6] == -math.inf).any())


def split_scores(q, c, bounds, group):
    """q+ . hi + q- . lo in 64 bits, and the finite terms' absolute sum: [Hkv, group, pages] of sequence 0 each, unscaled by head."""
    ids = c.tables[0, :-(-int(c.lengths[0]) // c.bs)].long()
    lo, hi = bo.codes(bounds[ids]).permute(2, 1, 0, 3)
    rows = q[0].double().view(c.hkv, group, D)
    up, down = rows.clamp_min(0), rows.clamp_max(0)
    terms = (up.nan_to_num(posinf=0) @ hi.abs().transpose(1, 2)) + (-down.nan_to_num(neginf=0)) @ lo.abs().transpose(1, 2)
    return up @ hi.transpose(1, 2) + down @ lo.transpose(1, 2), terms, c.ks[ids, :, 0, 0].double().T


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 3, 12, 20, 50])
def test_scores_of_infinite_query_elements(group):
    c = Cache([400], 2, 16, seed=group)
    bounds = c.bounds()
    bounds.view(torch.uint8)[c.tables[0, 2].long(), :, 1, 9] = 0           # one page's largest code of dim 9 is zero
    for dim in (6, 10, 11):                     # pages on which large finite elements give zero, or less
        bounds.view(torch.uint8)[c.tables[0, 4].long(), :, :, dim] = 0
        bounds[c.tables[0, 3].long(), :, :, dim] = torch.tensor([-20.0, -5.0]).to(FP8)
    q = c.query(group)
    q[0, 0, 9] = math.inf                       # head 0: one infinity beside elements far below and above f16's largest
    q[0, 0, 10], q[0, 0, 11] = 2.0 ** 70, 2.0 ** 55
    q[0, group, 5], q[0, group, 6] = -math.inf, 2.0 ** 100                  # head 1
    got = scores_of(q, bounds, c.lengths, c.tables, 16, c.ks)[0]
    sums, terms, ks = split_scores(q, c, bounds, group)
    nan = sums.isnan().any(1)
    want = sums.nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf).amax(1) * SCALE * ks
    assert bool(nan.any()) and bool((want == math.inf).any())
    assert torch.equal(got.isnan(), nan)
    fine = ~nan
    assert torch.equal(got.isinf() & fine, want.isinf() & fine)
    assert torch.equal(got[want.isinf() & fine].double(), want[want.isinf() & fine])
    fine &= ~want.isinf()
    slack = 260 * 2.0 ** -23 * terms.amax(1) * SCALE * ks
    assert bool(((got.double() - want).abs()[fine] <= slack[fine]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("group", [2, 12])
def test_scores_of_subnormal_query_rows(group):
    """Rows whose largest element is below bf16's smallest normal number (2^-126) beside rows that are not."""
    c = Cache([400], 2, 16, seed=group)
    bounds = c.bounds()
    q = c.query(group)
    steps = torch.randint(-127, 128, (2, D), generator=c.g).float()
    q[0, 0], q[0, group] = (steps * 2.0 ** -133).bfloat16()
    q[0, 1:group] = 0                                   # head 0 has nothing larger
    got = scores_of(q, bounds, c.lengths, c.tables, 16, c.ks)[0]
    sums, terms, ks = split_scores(q, c, bounds, group)
    # (no product, sum or factor of head 0 is subnormal in 32 bits: terms of 2^-133 * SCALE * 2^-8 at least are summed scaled up)
    assert bool(((got.double() - sums.amax(1) * SCALE * ks).abs() <= 260 * 2.0 ** -23 * terms.amax(1) * SCALE * ks).all())


# ----------------------------------------------------------------------------- append: two writers of one place
def append_args(device="cpu"):
    c = Cache([40, 7], 2, 16)
    kv = torch.randn(5, 2, D, generator=c.g).bfloat16()
    args = dict(key=kv, value=kv, key_cache=c.key, value_cache=c.value, key_scale=c.ks, value_scale=c.vs, block_tables=c.tables,
                sequence_lengths=c.lengths, query_start_loc=torch.tensor([0, 3, 5], dtype=torch.int32), key_bounds=c.bounds())
    return {k: v.to(device) for k, v in args.items()}


def shared_places(a):
    """Changes of append_args whose pages, heads or scales share memory, and ones that only look so."""
    nb, dev = a["key_scale"].shape[0], a["key_scale"].device
    pool = torch.ones(2 * nb + 1, 2, 1, 1, device=dev)
    side = torch.ones(nb, 2, 2, 1, device=dev)
    bad = [dict(value_scale=a["key_scale"]),
           dict(key_scale=pool[:nb], value_scale=pool[nb - 1:2 * nb - 1]),                    # one page of both
           dict(key_scale=pool[1:nb + 1], value_scale=pool[:nb]),
           dict(key_scale=pool.view(-1)[:2 * nb].view(nb, 2, 1, 1), value_scale=pool.view(-1)[1:2 * nb + 1].view(nb, 2, 1, 1)),
           dict(key_bounds=a["key_bounds"][:1].expand(nb, -1, -1, -1)),
           dict(key_bounds=a["key_bounds"][:, :1].expand(-1, 2, -1, -1)),
           dict(key_cache=a["key_cache"][:1].expand(nb, -1, -1, -1, -1)),
           dict(value_cache=a["value_cache"][:, :1].expand(-1, 2, -1, -1))]
    good = [dict(key_scale=pool[:nb], value_scale=pool[nb:2 * nb]),
            dict(key_scale=side[:, :, :1], value_scale=side[:, :, 1:]),                       # side by side, never met
            dict(key_scale=pool[:2 * nb:2], value_scale=pool[1:2 * nb:2])]
    return bad, good


def test_append_refuses_places_that_are_shared():
    a = append_args()
    bad, good = shared_places(a)
    for over in bad:
        with pytest.raises(PaArgumentError, match="place of its own"):
            pa.append_kv_cache(**{**a, **over})
    for over in good:
        with pytest.raises(RuntimeError, match="CUDA"):            # refused for being on the CPU only
            pa.append_kv_cache(**{**a, **over})
    one = torch.tensor(0.5)
    with pytest.raises(RuntimeError, match="CUDA"):                # read only: the same value twice is fine
        pa.append_kv_cache(**{**a, "key_scale": one, "value_scale": one})


def test_the_library_refuses_places_that_are_shared():
    lib = _lib.lib()
    p = _lib.PaCacheAppendParams()
    p.struct_size, p.abi_version = C.sizeof(p), _lib.PA_ABI_VERSION
    room = (C.c_float * 64)()
    at = (C.addressof(room) + 15) & ~15
    p.num_tokens, p.num_seqs, p.num_kv_heads, p.head_size, p.block_size, p.num_blocks, p.max_blocks_per_seq = 1, 1, 2, D, 16, 4, 1
    p.kv_quant_mode, p.v_layout = _lib.PA_QUANT_PER_BLOCK, _lib.PA_V_NORMAL
    for name in ("key", "value", "key_cache", "value_cache", "block_tables", "context_lens", "row_start", "key_bounds"):
        setattr(p, name, at)                                       # (nothing is read before the refusal)
    p.key_stride_token = p.value_stride_token = 2 * D
    p.key_stride_head = p.value_stride_head = D
    p.k_stride_block = p.v_stride_block = 2 * 16 * D
    p.k_stride_head = p.v_stride_head = 16 * D
    p.bounds_stride_block, p.bounds_stride_head = 4 * D, 2 * D
    p.kv_scale_stride_block, p.kv_scale_stride_head = 2, 1
    for apart in (0, 1, -1, 6, 7, -7):
        p.key_scale, p.value_scale = at + 64, at + 64 + 4 * apart
        assert lib.pa_cache_append_sm100(C.byref(p), None) == -2, apart
    p.key_scale, p.value_scale = at, at + 4 * 16
    for name in ("k_stride_block", "v_stride_head", "bounds_stride_block", "bounds_stride_head", "kv_scale_stride_block"):
        was = getattr(p, name)
        setattr(p, name, 0)
        assert lib.pa_cache_append_sm100(C.byref(p), None) == -2, name
        setattr(p, name, was)


@pytest.mark.gpu
def test_append_refuses_shared_places_on_the_gpu_and_takes_neighbours():
    a = append_args("cuda")
    bad, good = shared_places(a)
    before = {k: v.clone() for k, v in a.items()}
    for over in bad:
        with pytest.raises(PaArgumentError, match="place of its own"):
            pa.append_kv_cache(**{**a, **over})
    torch.cuda.synchronize()
    assert all(torch.equal(a[k].view(torch.uint8), before[k].view(torch.uint8)) for k in a if a[k].dtype == FP8)
    state = ("key_cache", "value_cache", "key_scale", "value_scale", "key_bounds")
    for over in good:
        mine = {k: v.clone() for k, v in a.items()}
        views = {k: v.copy_(a[k]) for k, v in over.items()}
        pa.append_kv_cache(**{**mine, **views})
        ref = {k: v.cpu().clone() for k, v in a.items()}
        bo.append(ref["key"], ref["value"], ref["key_cache"], ref["value_cache"], ref["key_scale"], ref["value_scale"],
                  ref["block_tables"], ref["sequence_lengths"], ref["query_start_loc"], ref["key_bounds"])
        got = {**mine, **views}
        assert_same([got[k].cpu() for k in state], [ref[k] for k in state])


# ----------------------------------------------------------------------------- outputs that are read, or shared
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_outputs_need_places_of_their_own(device):
    c = Cache([40, 7], 2, 16)
    lengths, tables = c.lengths.to(device), c.tables.to(device)
    score = torch.zeros(2, 2, 3, device=device)
    one = torch.zeros(2, 1, 3, dtype=torch.int32, device=device)
    for over in (dict(lengths=lengths), dict(tables=one.expand(-1, 2, -1)[:, :, :2]), dict(tables=one[:1].expand(2, 2, -1)[:, :, :2])):
        with pytest.raises(PaArgumentError):
            pa.select_blocks(score, lengths, tables, 16, 2, **over)
    with pytest.raises(PaArgumentError):                               # one kv head: its tables could be the sequences'
        pa.select_blocks(score[:, :1], lengths, tables, 16, 3, tables=tables[:, None])
    for out in (score[:, :1].expand(-1, 2, -1), score[:1].expand(2, -1, -1)):
        with pytest.raises(PaArgumentError):
            pa.score_blocks(c.query(3).to(device), c.bounds().to(device), lengths, tables, SCALE, 1, 16, scores=out)


# ----------------------------------------------------------------------------- refusals, whichever way a call takes
def calls_and_mistakes(device):
    """(function, an ordinary call, changes that make it a mistake) of each operator."""
    c = Cache([40, 7], 2, 16)
    t = {k: v.to(device) for k, v in dict(kc=c.key, vc=c.value, ks=c.ks, vs=c.vs, bt=c.tables, len=c.lengths, b=c.bounds(), q=c.query(3),
                                          wide=c.query(65)).items()}
    nb, ones = c.nb, lambda *shape, **kw: torch.ones(*shape, device=device, **kw)
    kv = torch.zeros(5, 2, D, dtype=torch.bfloat16, device=device)
    start = torch.tensor([0, 3, 5], dtype=torch.int32, device=device)
    heads = t["bt"][:, None].expand(-1, 2, -1).contiguous()
    half_pages = t["kc"].view(torch.uint8)[:, :, :, ::2].view(FP8)
    yield pa.append_kv_cache, dict(
        key=kv, value=kv, key_cache=t["kc"], value_cache=t["vc"], key_scale=t["ks"], value_scale=t["vs"], block_tables=t["bt"],
        sequence_lengths=t["len"], query_start_loc=start), [
        dict(key=kv.float()), dict(value=kv[:4]), dict(key=kv[0]), dict(key_cache=t["kc"].float().bfloat16()), dict(key_cache=t["kc"][:, :1]),
        dict(value_cache=t["vc"][:, :, :, :8]), dict(key_scale=ones(())), dict(key_scale=1.0), dict(value_scale=t["vs"].double()),
        dict(key_bounds=t["b"].float()), dict(key_bounds=t["b"][..., :64]), dict(key_bounds=t["b"][:1]), dict(block_tables=t["bt"].long()),
        dict(block_tables=t["bt"][:, :0]), dict(sequence_lengths=t["len"][:1]), dict(query_start_loc=start[:2]), dict(query_start_loc=start.long()),
        dict(status=ones(())), dict(key_cache=half_pages), dict(key_scale=ones(nb + 1, 2, 1, 1), value_scale=ones(nb + 1, 2, 1, 1))]
    yield pa.paged_attention_decode, dict(
        output=torch.empty_like(t["q"]), query=t["q"], key_cache=t["kc"], value_cache=t["vc"], sequence_lengths=t["len"], block_tables=t["bt"],
        softmax_scale=SCALE, query_sequence_length=1, max_sequence_length=40, compute_type=torch.bfloat16, query_scale=None,
        key_scale=t["ks"], value_scale=t["vs"]), [
        dict(value_scale=ones(())), dict(value_scale=None), dict(key_scale=ones(nb, 1, 1, 1), value_scale=ones(nb, 1, 1, 1)),
        dict(key_scale=ones(nb + 1, 2, 1, 1), value_scale=ones(nb + 1, 2, 1, 1)), dict(key_scale=t["ks"].double(), value_scale=t["vs"].double()),
        dict(key_scale=ones(2, nb, 1, 1).transpose(0, 1)), dict(block_tables=heads[:, :1]), dict(block_tables=heads.long()), dict(block_tables=heads[:1]),
        dict(block_tables=heads, key_scale=ones(nb, 2, 16, 1), value_scale=ones(nb, 2, 16, 1)), dict(query_sequence_length=5),
        dict(query_sequence_length=2), dict(query_sequence_length=0), dict(output=torch.empty(2, 6, D, device=device)),
        dict(output=torch.empty_like(t["q"])[:1]), dict(query=t["q"].half()), dict(key_cache=t["kc"].float().bfloat16()), dict(key_cache=half_pages),
        dict(value_cache=t["vc"][:, :, :64]), dict(sequence_lengths=t["len"].long()), dict(sequence_lengths=t["len"][:1]),
        dict(status=torch.zeros((), dtype=torch.int64, device=device)), dict(query=t["wide"], output=torch.empty_like(t["wide"]))]
    yield pa.score_blocks, dict(
        query=t["q"], key_bounds=t["b"], sequence_lengths=t["len"], block_tables=t["bt"], softmax_scale=SCALE, query_sequence_length=1,
        block_size=16, key_scale=t["ks"]), [
        dict(query=t["q"].half()), dict(query=t["q"][0]), dict(query=t["q"][..., :64]), dict(query=t["wide"]), dict(key_bounds=t["b"].float()),
        dict(key_bounds=t["b"][..., :64]), dict(key_bounds=t["b"][:, :, :1]), dict(softmax_scale=0.0), dict(softmax_scale=-1.0),
        dict(softmax_scale=math.nan), dict(query_sequence_length=2), dict(query_sequence_length=0), dict(query_sequence_length=5), dict(block_size=32),
        dict(key_scale=ones(nb, 2, 16, 1)), dict(key_scale=ones(nb, 1, 1, 1)), dict(key_scale=ones(nb + 1, 2, 1, 1)), dict(block_tables=t["bt"][:1]),
        dict(block_tables=t["bt"].long()), dict(sequence_lengths=t["len"].long()), dict(sequence_lengths=t["len"][:1]), dict(status=ones(()))]
    score = torch.zeros(2, 2, 3, device=device)
    yield pa.select_blocks, dict(scores=score, sequence_lengths=t["len"], block_tables=t["bt"], block_size=16, top_k=2), [
        dict(scores=score[:, :, :2]), dict(scores=score.double()), dict(scores=score[0]), dict(scores=score[:1]), dict(top_k=1), dict(top_k=0),
        dict(keep_first=-1), dict(keep_last=0), dict(keep_first=2), dict(block_size=48), dict(block_tables=t["bt"].long()),
        dict(sequence_lengths=t["len"].long()), dict(sequence_lengths=t["len"][:1]), dict(status=ones(()))]


@pytest.mark.gpu
def test_mistakes_on_the_gpu_are_refused(monkeypatch):
    """The host calls check for themselves what the Python functions check: nothing that those refuse is taken."""
    taken = []

    class Watched:
        def __getattr__(self, name):
            def call(*args):
                done = getattr(real, name)(*args)
                taken.append(done is not None)
                return done
            return call
    real = _lib.calls()
    monkeypatch.setattr(_lib, "_CALLS", Watched())
    for fn, good, mistakes in calls_and_mistakes("cuda"):
        taken.clear()
        fn(**good)
        assert taken == [True], fn                                     # the ordinary call goes that way
        names = [k for k, v in good.items() if isinstance(v, torch.Tensor)]
        for over in mistakes + [{k: good[k].cpu()} for k in names]:
            taken.clear()
            with pytest.raises(PaArgumentError):
                fn(**{**good, **over})
            assert not any(taken), (fn, over.keys())
    torch.cuda.synchronize()


# ----------------------------------------------------------------------------- the operators in a row
@pytest.mark.gpu
@pytest.mark.parametrize("bs,query_len,group", [(16, 1, 4), (16, 2, 8), (64, 1, 1), (64, 3, 2)])
def test_served_selections_are_those_of_the_scores(bs, query_len, group):
    """The tables of a served step are the exact selection of the kernel's scores, and that of the oracle's wherever
    the last page taken and the first one left are further apart than the scores may be off."""
    sure = 0
    for c, q, out, res, (kc, vc, ks, vs, bounds, lengths) in serve(4, bs, 6, group, query_len):
        keep = 1 if query_len == 1 else 2
        score = scores_of(q, bounds, lengths, c.tables, bs, ks, query_len)
        want, terms = bo.scores(q, bounds, lengths, c.tables, SCALE, bs, ks)
        assert_scores(score, want, terms)
        got = res["block_tables"].cpu()
        tables, tokens = bo.select(score, lengths, c.tables, bs, 6, 1, keep)
        assert torch.equal(got, tables) and torch.equal(res["sequence_lengths"].cpu(), tokens)
        tables, _ = bo.select(want, lengths, c.tables, bs, 6, 1, keep)
        for s in range(3):
            pages = -(-int(lengths[s]) // bs)
            for h in range(c.hkv):
                if pages > 6:
                    rest, order = want[s, h, 1:pages - keep].sort(descending=True)
                    slack = 2 * 260 * 2.0 ** -23 * float(terms[s, h, :pages].max())
                    if float(rest[6 - 1 - keep - 1] - rest[6 - 1 - keep]) <= slack:
                        continue
                sure += 1
                assert torch.equal(got[s, h], tables[s, h])
    assert sure >= 12                                                  # of 24 selections: the comparison is not an empty one


def strided_pool(c):
    """The same pool as views of one allocation: a page's keys, values and scales side by side, heads apart."""
    room = torch.zeros(c.nb, c.hkv, 2, D * c.bs + 32, dtype=torch.uint8, device="cuda")
    key = room[:, :, 0, :D * c.bs].unflatten(2, (D // 16, c.bs, 16)).view(FP8)
    value = room[:, :, 1, 16:D * c.bs + 16].unflatten(2, (D, c.bs)).view(FP8)
    key.view(torch.uint8).copy_(c.key.view(torch.uint8))
    value.view(torch.uint8).copy_(c.value.view(torch.uint8))
    scales = torch.stack((c.ks, c.vs), 2).cuda()
    return key, value, scales[:, :, 0], scales[:, :, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64, 1024])
@pytest.mark.parametrize("form", ["plain", "one pool", "transposed", "no scales", "one value", "fp8 query", "fp8 query rows", "sinks", "64 rows", "keeps"])
def test_sparse_decode_in_every_form(form, bs):
    """What paged_attention_decode takes, sparse_attention_decode takes: the exact selection of the kernel's scores, and
    the attention over it."""
    query_len, group = (4, 16) if form == "64 rows" else (1, 4)
    c = Cache([9 * bs + 5, 40, 3 * bs, 0, 7 * bs + bs // 2 + 1], 2, bs, seed=bs + len(form))
    q, bounds = c.query(group, query_len), c.bounds()
    kc, vc, ks, vs = cuda(c.key, transposed(c.value) if form == "transposed" else c.value, c.ks, c.vs)
    kw, ref, scale, top_k, first, last = {}, {}, {}, 5, 1, 1 if query_len == 1 else 2
    oks, ovs = c.ks, c.vs
    if form == "one pool":
        kc, vc, ks, vs = strided_pool(c)
    elif form == "no scales":
        ks = vs = oks = ovs = None
    elif form == "one value":
        ks, vs, oks, ovs = 0.02, 0.03, torch.tensor(0.02), torch.tensor(0.03)
    elif form.startswith("fp8"):
        q = (q.float() * 40).to(FP8)
        scale = dict(query_scale=torch.tensor(1 / 40) if form == "fp8 query" else torch.rand(5, 8, 1, generator=c.g) / 20 + 0.01)
    elif form == "sinks":
        ref["sink_tokens"] = torch.linspace(-2, 3, 8)
        kw["sink_tokens"] = ref["sink_tokens"].cuda()
    elif form == "keeps":
        first, last = 0, 4
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    dq, db, dl, dt = cuda(q, bounds, c.lengths, c.tables)
    dscale = {k: v.cuda() for k, v in scale.items()}
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    res = pa.sparse_attention_decode(out, dq, kc, vc, db, dl, dt, SCALE, query_len, top_k, dscale.get("query_scale"), ks, vs,
                                     keep_first=first, keep_last=last, status=status, **kw)
    assert int(status) == 0 and res["final_output"] is out
    score = pa.score_blocks(dq, db, dl, dt, SCALE, query_len, bs, key_scale=ks, **dscale).cpu()
    assert_scores(score, *bo.scores(q, bounds, c.lengths, c.tables, SCALE, bs, oks, **scale))
    tables, tokens = bo.select(score, c.lengths, c.tables, bs, top_k, first, last)
    assert torch.equal(res["block_tables"].cpu(), tables) and torch.equal(res["sequence_lengths"].cpu(), tokens)
    assert_attention(out.cpu(), bo.attention(q, c.key, c.value, oks, ovs, tables, tokens, SCALE, query_len, **ref, **scale), form)
    again = torch.empty_like(out)
    for _ in range(5):
        pa.sparse_attention_decode(again, dq, kc, vc, db, dl, dt, SCALE, query_len, top_k, dscale.get("query_scale"), ks, vs,
                                   keep_first=first, keep_last=last, **kw)
        assert torch.equal(again, out)


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64, 1024])
def test_append_to_a_pool_of_views(bs):
    counts, before = [5, 33, 1], [13, 20, 0]
    c = Cache([18, 53, 1], 2, bs, seed=11)
    start = torch.tensor([0, 5, 38, 39], dtype=torch.int32)
    key, value = torch.randn(39, 2, D, generator=c.g).bfloat16(), torch.randn(39, 2, D, generator=c.g).bfloat16()
    views = strided_pool(c)
    bounds = c.bounds().cuda()
    pa.append_kv_cache(*cuda(key, value), *views, *cuda(c.tables, c.lengths, start), key_bounds=bounds)
    want = [c.key.clone(), c.value.clone(), c.ks.clone(), c.vs.clone(), c.bounds()]
    bo.append(key, value, *want[:4], c.tables, c.lengths, start, want[4])
    assert_same([t.cpu() for t in (*views, bounds)], want)


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 1024])
def test_decode_without_allocation_with_block_scales(bs):
    """The library's own array holds bf16 partial outputs, whatever the parameter block says of its workspaces."""
    c = Cache([700, 40, 0], 2, bs, seed=19)
    q = c.query(4)
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    dev = cuda(q, c.key, c.value, c.lengths, c.tables, c.ks, c.vs)
    p, keep = build_params(out, *dev[:5], SCALE, 1, 700, None, None, *dev[5:], None, 256, None, None, None, None, None)
    assert p.tmp_dtype == _lib.PA_DT_F32
    p.exp_sums = p.max_logits = p.tmp_out = None
    _lib.check(_lib.lib().pa_decode_noalloc_sm100(C.byref(p), torch.cuda.current_stream().cuda_stream), "pa_decode_noalloc_sm100")
    assert_attention(out.cpu(), bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 1))
    del keep


@pytest.mark.gpu
def test_bounds_beyond_32_bits():
    """Key bounds more than 4 GB into their tensor: appended, scored and selected by."""
    hkv, bs, n = 8, 16, 200
    nb = (1 << 32) // (hkv * 16 * D) + 40
    kc = torch.empty(nb, hkv, 8, bs, 16, dtype=torch.uint8, device="cuda").view(FP8)
    vc = torch.empty(nb, hkv, D, bs, dtype=torch.uint8, device="cuda").view(FP8)
    ks, vs = torch.ones(nb, hkv, 1, 1, device="cuda"), torch.ones(nb, hkv, 1, 1, device="cuda")
    bounds = torch.empty(nb, hkv, 16, D, dtype=torch.uint8, device="cuda").view(FP8)[:, :, :2]
    assert bounds.stride(0) * (nb - 13) > 1 << 32
    g = torch.Generator().manual_seed(1)
    tables = torch.arange(nb - 13, nb).int()[None]
    near = torch.arange(13).int()[None]
    key, value = torch.randn(n, hkv, D, generator=g).bfloat16(), torch.randn(n, hkv, D, generator=g).bfloat16()
    lengths, start = torch.tensor([n], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32)
    pa.append_kv_cache(*cuda(key, value), kc, vc, ks, vs, *cuda(tables, lengths, start), key_bounds=bounds)
    far = slice(nb - 13, nb)
    ref = [torch.zeros(13, hkv, 8, bs, 16).to(FP8), torch.zeros(13, hkv, D, bs).to(FP8), torch.ones(13, hkv, 1, 1), torch.ones(13, hkv, 1, 1),
           torch.zeros(13, hkv, 2, D).to(FP8)]
    bo.append(key, value, *ref[:4], near, lengths, start, ref[4])
    assert_same([ks[far].cpu(), vs[far].cpu(), bounds[far].cpu()], ref[2:])
    q = torch.randn(1, hkv * 4, D, generator=g).bfloat16()
    score = pa.score_blocks(q.cuda(), bounds, *cuda(lengths, tables), SCALE, 1, bs, key_scale=ks).cpu()
    assert_scores(score, *bo.scores(q, ref[4], lengths, near, SCALE, bs, ref[2]))
    got = pa.select_blocks(*cuda(score, lengths, tables), bs, 5)
    assert torch.equal(got[0].cpu() - (nb - 13), bo.select(score, lengths, near, bs, 5)[0])


# ----------------------------------------------------------------------------- KV-partition sharding
@pytest.mark.gpu
@pytest.mark.parametrize("world", [1, 2, 4])
@pytest.mark.parametrize("bs,query_len", [(16, 1), (64, 2), (1024, 1)])
def test_sharded_decode_with_block_scales(bs, query_len, world):
    """Each rank's maxima are those of logit + log(value scale): ranks whose pages have scales far apart merge all the same."""
    c = Cache([3000, 257, 1100, 60], 2, bs, seed=world)
    for s, n in enumerate(c.lengths.tolist()):      # the pages of the context's second half: values a thousand times smaller
        late = c.tables[s, -(-n // bs) // 2:-(-n // bs)].long()
        c.vs[late] *= 2.0 ** -10
    q = c.query(4, query_len)
    kc, vc, ks, vs, tables, dq = cuda(c.key, c.value, c.ks, c.vs, c.tables, q)
    plan = plan_kv_shards(c.lengths.tolist(), world, max(256, bs), query_len)
    triples = [decode_kv_shard(dq, kc, vc, plan[r], local_block_table(tables, plan[r], bs), SCALE, ks, vs) for r in range(world)]
    got = merge_triples_cuda(*(torch.stack([t[i] for t in triples]) for i in range(3)))
    want = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, query_len)
    assert_attention(got.view(q.shape).cpu(), want)
    if world == 1:
        dec = KvShardedDecoder(dq, kc, vc, plan[0], tables, SCALE, ks, vs)
        assert_attention(dec.step().cpu(), want)
        assert dec.params.tmp_dtype == _lib.PA_DT_F32


# ----------------------------------------------------------------------------- host threads
def launches_of(monkeypatch, call):
    """The library calls that `call` makes, as functions that make them again on a stream: () -> status."""
    made = []

    def record(index, fn, where, *args):
        made.append((fn, args))
    with monkeypatch.context() as m:
        m.setattr(_lib, "launch", record)
        call()
    stream = torch.cuda.Stream()
    return [lambda fn=fn, args=args: fn(*args, stream.cuda_stream) for fn, args in made]


def in_two_threads(a, b, rounds):
    """Library calls a and b over and over, each from a thread of its own (a call into the library leaves the other
    thread its turn): the statuses that are not 0."""
    import threading
    bad = []
    go = threading.Barrier(2)

    def run(call):
        go.wait()
        for _ in range(rounds):
            status = call()
            if status:
                bad.append(status)
            if bad:
                return

    threads = [threading.Thread(target=run, args=(call,)) for call in (a, b)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return bad


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["scores", "attention", "attention, scales per token"])
def test_two_threads_call_with_batches_of_different_sizes(monkeypatch, what):
    """The index of a large batch lies in shared memory: its launch asks for more of it than a small one's."""
    calls, outs, kept = [], [], []
    for seqs in (4000, 3):
        c = Cache([5] * seqs, 2, 16, seed=seqs)
        q, bounds, lengths, tables, ks, vs, kc, vc = cuda(c.query(1), c.bounds(), c.lengths, c.tables, c.ks, c.vs, c.key, c.value)
        if what == "scores":
            out = torch.full((seqs, 2, 1), math.nan, device="cuda")
            made = launches_of(monkeypatch, lambda: pa.score_blocks(q, bounds, lengths, tables, SCALE, 1, 16, key_scale=ks, scores=out))
        elif what == "attention":
            out = torch.full_like(q, math.nan)
            sink = torch.zeros(2, device="cuda")
            def call():
                kept.append(pa.paged_attention_decode(out, q, kc, vc, lengths, tables, SCALE, 1, 5, torch.bfloat16, None, ks, vs, sink_tokens=sink))
            made = launches_of(monkeypatch, call)
            kept.append(sink)
        else:
            out = torch.full_like(q, math.nan)
            tok = ks.expand(-1, -1, 16, -1).contiguous()
            p, keep = build_params(out, q, kc, vc, lengths, tables, SCALE, 1, 5, None, None, tok, tok, None, 256, None, None, None, None, None)
            stream = torch.cuda.Stream()
            made = [lambda p=p, stream=stream: _lib.lib().pa_decode_sm100(C.byref(p), stream.cuda_stream)]
            kept.append((keep, tok))
        assert len(made) == 1
        torch.cuda.synchronize()
        assert made[0]() == 0
        torch.cuda.synchronize()
        calls.append(made[0])
        outs.append((out, out.clone()))
        kept.append((q, bounds, lengths, tables, ks, vs, kc, vc))
    assert in_two_threads(*calls, 10000) == []
    for out, want in outs:
        assert not want.isnan().any() and torch.equal(out, want)
