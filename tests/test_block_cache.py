"""The operators around a cache with scales per (page, kv head): refusals and host logic on the CPU, the
kernels against the 64-bit oracle on the GPU."""
import ctypes as C
import math
import os
import re

import pytest
import torch

import triton_op_b200 as pa
from oracle import blocks_oracle as bo
from triton_op_b200 import PaArgumentError, _lib
from triton_op_b200 import build as pa_build
from triton_op_b200.pa_decode import build_params

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FP8 = torch.float8_e4m3fn
D = 128
SCALE = D ** -0.5


# ----------------------------------------------------------------------------- inputs
def random_codes(shape, g, spread=90.0):
    return (torch.randn(shape, generator=g) * spread).clamp(-448, 448).to(FP8)


def transposed(value_cache):
    nb, h, d, bs = value_cache.shape
    return value_cache.view(torch.uint8).view(nb, h, d, bs // 16, 16).permute(0, 1, 3, 2, 4).contiguous().view(FP8)


class Cache:
    """A pool of pages with random codes, scales and bounds, and scattered block tables (CPU)."""

    def __init__(self, lengths, hkv, bs, seed=0, spare=2, octaves=4, width=None):
        g = torch.Generator().manual_seed(seed)
        self.lengths = torch.tensor(lengths, dtype=torch.int32)
        self.bs, self.hkv = bs, hkv
        pages = [-(-n // bs) for n in lengths]
        self.nb = sum(pages) + spare
        self.width = width or max(1, max(pages, default=1))
        perm = torch.randperm(self.nb, generator=g)
        self.tables = torch.full((len(lengths), self.width), -7, dtype=torch.int32)   # ids past the context are no pages
        at = 0
        for s, n in enumerate(pages):
            self.tables[s, :n] = perm[at:at + n].int()
            at += n
        self.free = perm[at:]
        self.key = random_codes((self.nb, hkv, D // 16, bs, 16), g)
        self.value = random_codes((self.nb, hkv, D, bs), g)
        self.ks = torch.exp2(torch.randint(-8, -8 + octaves, (self.nb, hkv, 1, 1), generator=g).float())
        self.vs = torch.exp2(torch.randint(-8, -8 + octaves, (self.nb, hkv, 1, 1), generator=g).float())
        self.g = g

    def bounds(self):
        k = self.key.float().permute(0, 1, 2, 4, 3).reshape(self.nb, self.hkv, D, self.bs)
        return torch.stack((k.amin(-1), k.amax(-1)), 2).to(FP8)

    def query(self, group, query_len=1):
        return torch.randn(len(self.lengths), self.hkv * group * query_len, D, generator=self.g).bfloat16()


def cuda(*tensors):
    got = tuple(None if t is None else t.cuda() for t in tensors)
    return got if len(got) > 1 else got[0]


def decode(c, q, tables=None, lengths=None, query_len=1, ks=None, vs=None, value=None, longest=None, status=None, **kw):
    """paged_attention_decode on the GPU; returns the output on the CPU."""
    tables = c.tables if tables is None else tables
    lengths = c.lengths if lengths is None else lengths
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    kv = cuda(c.key, c.value if value is None else value)
    pa.paged_attention_decode(out, q.cuda(), *kv, lengths.cuda(), tables.cuda(), SCALE, query_len,
                              longest or max(1, int(lengths.max())), torch.bfloat16, kw.pop("query_scale", None),
                              *cuda(c.ks if ks is None else ks, c.vs if vs is None else vs), status=status, **kw)
    return out.cpu()


def assert_attention(got, want, what=""):
    out, mass, floor = want
    err = (got.double() - out).abs()
    over = err - bo.attention_tolerance(out, mass, floor)
    assert not got.isnan().any(), what
    assert float(over.max()) <= 0, f"{what}: {float(err.max())} off, {float(over.max())} over its tolerance"


# ----------------------------------------------------------------------------- CPU: host logic and refusals
@pytest.fixture(scope="module")
def lib():
    pa_build.build()
    return _lib.lib()


@pytest.mark.parametrize("name", ["PaCacheAppendParams", "PaBlockScoreParams", "PaBlockSelectParams"])
def test_struct_mirrors_match_the_header(lib, name):
    header = open(os.path.join(ROOT, "include", "pa_decode_sm100.h")).read()
    start = header.index(f"typedef struct {name} {{") + len(f"typedef struct {name} {{")
    body = re.sub(r"/\*.*?\*/", "", header[start:header.index(f"}} {name};")], flags=re.S)
    names = []
    for decl in body.split(";"):
        decl = re.sub(r"^(const\s+)?(void|float|int32_t|uint32_t|int64_t|uint64_t)\s*\*?\s*", "", decl.strip())
        names += [n.strip().lstrip("*") for n in decl.split(",") if n.strip()]
    assert names == [f[0] for f in getattr(_lib, name)._fields_]


def test_c_abi_refuses_before_any_cuda_call(lib):
    for fn, struct in ((lib.pa_cache_append_sm100, _lib.PaCacheAppendParams),
                       (lib.pa_block_scores_sm100, _lib.PaBlockScoreParams),
                       (lib.pa_block_select_sm100, _lib.PaBlockSelectParams)):
        p = struct()
        assert fn(None, None) == -1
        assert fn(C.byref(p), None) == -6                      # struct_size 0
        p.struct_size, p.abi_version = C.sizeof(struct), _lib.PA_ABI_VERSION
        assert fn(C.byref(p), None) in (-2, -3)                # sizes of zero
    p = _lib.PaBlockSelectParams()
    p.struct_size, p.abi_version = C.sizeof(p), _lib.PA_ABI_VERSION
    p.num_seqs, p.num_kv_heads, p.block_size, p.max_blocks_per_seq = 1, 1, 16, 4
    for top_k, first, last in ((0, 0, 0), (1, 1, 1), (4, -1, 1), (4, 1, 0), (2147483647, 2147483647, 1)):
        p.top_k, p.keep_first, p.keep_last = top_k, first, last
        assert lib.pa_block_select_sm100(C.byref(p), None) == -2
    p.top_k, p.keep_first, p.keep_last = 4, 1, 1
    assert lib.pa_block_select_sm100(C.byref(p), None) == -1   # no pointers
    p.num_seqs = 0
    assert lib.pa_block_select_sm100(C.byref(p), None) == 0    # nothing to do
    d = _lib.PaDecodeParams()
    assert lib.pa_decode_tables_sm100(C.byref(d), -1, None) == -2
    assert lib.pa_decode_tables_sm100(C.byref(d), 0, None) == -6


def small_decode_args(**over):
    c = Cache([40, 7], 2, 16)
    q = c.query(3)
    a = dict(output=torch.empty_like(q), query=q, key_cache=c.key, value_cache=c.value, sequence_lengths=c.lengths,
             block_tables=c.tables, softmax_scale=SCALE, query_sequence_length=1, max_sequence_length=40,
             compute_type=torch.bfloat16, query_scale=None, key_scale=c.ks, value_scale=c.vs)
    a.update(over)
    return a


def test_decode_refusals():
    c = Cache([40, 7], 2, 16)
    per_head = c.tables[:, None].expand(-1, 2, -1).contiguous()
    tok = torch.ones(c.nb, 2, 16, 1)
    bad = [
        dict(key_scale=torch.ones(c.nb, 2, 1, 1), value_scale=torch.ones(())),
        dict(key_scale=torch.ones(c.nb, 1, 1, 1), value_scale=torch.ones(c.nb, 1, 1, 1)),
        dict(key_scale=torch.ones(c.nb + 1, 2, 1, 1), value_scale=torch.ones(c.nb + 1, 2, 1, 1)),
        dict(value_scale=None),
        dict(key_scale=torch.ones(c.nb, 2, 1, 1).double(), value_scale=torch.ones(c.nb, 2, 1, 1).double()),
        dict(key_scale=torch.ones(2, c.nb, 1, 1).transpose(0, 1)),
        dict(block_tables=per_head[:, :1]),
        dict(block_tables=per_head.long()),
        dict(block_tables=per_head, key_scale=tok, value_scale=tok),
        dict(block_tables=per_head, alibi_slopes=torch.ones(6)),
        dict(block_tables=per_head, time_kernels=True),
        dict(block_tables=per_head, tune={"stages": 3}),
        dict(block_tables=per_head[:1]),
        dict(partition_size=128),
        dict(query_sequence_length=5),
        dict(query_sequence_length=2),
        dict(output=torch.empty(2, 6, D)),
        dict(query=torch.empty(2, 6, D, dtype=torch.float16)),
        dict(key_cache=c.key.float().bfloat16()),
        dict(value_cache=c.value[:, :, :64]),
        dict(sequence_lengths=c.lengths.long()),
        dict(sink_tokens=torch.ones(5)),
        dict(status=torch.zeros((), dtype=torch.int64)),
        dict(query_scale=torch.ones(2, 5, 1)),
    ]
    for over in bad:
        with pytest.raises((PaArgumentError, RuntimeError)) as e:
            pa.paged_attention_decode(**small_decode_args(**over))
        assert isinstance(e.value, PaArgumentError), (over.keys(), e.value)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa.paged_attention_decode(**small_decode_args())


def test_block_scales_reach_the_parameter_block():
    a = small_decode_args()
    order = ("output", "query", "key_cache", "value_cache", "sequence_lengths", "block_tables", "softmax_scale",
             "query_sequence_length", "max_sequence_length", "compute_type", "query_scale", "key_scale", "value_scale")
    p, _ = build_params(*(a[k] for k in order), None, 256, None, None, None, None, None)
    assert p.kv_quant_mode == _lib.PA_QUANT_PER_BLOCK
    assert (p.kv_scale_stride_block, p.kv_scale_stride_head) == a["key_scale"].stride()[:2]
    a["block_tables"] = a["block_tables"][:, None].expand(-1, 2, -1)
    with pytest.raises(PaArgumentError):       # the other entry points know one table per sequence only
        build_params(*(a[k] for k in order), None, 256, None, None, None, None, None)


def test_append_refusals():
    c = Cache([40, 7], 2, 16)
    kv = torch.zeros(5, 2, D, dtype=torch.bfloat16)
    good = dict(key=kv, value=kv, key_cache=c.key, value_cache=c.value, key_scale=c.ks, value_scale=c.vs,
                block_tables=c.tables, sequence_lengths=c.lengths, query_start_loc=torch.tensor([0, 3, 5], dtype=torch.int32))
    bad = [dict(key=kv.float()), dict(value=kv[:4]), dict(key=kv[0]), dict(key_cache=c.key.float().bfloat16()),
           dict(key_cache=c.key[:, :1]), dict(value_cache=c.value[:, :, :, :8]), dict(key_scale=torch.ones(())),
           dict(key_scale=c.ks[:1].expand(c.nb, -1, -1, -1), value_scale=c.vs[:1].expand(c.nb, -1, -1, -1)),
           dict(key_scale=1.0), dict(value_scale=c.vs.double()), dict(key_bounds=torch.zeros(c.nb, 2, 2, D)),
           dict(key_bounds=torch.zeros(c.nb, 2, 2, 64).to(FP8)), dict(block_tables=c.tables.long()),
           dict(sequence_lengths=c.lengths[:1]), dict(query_start_loc=torch.tensor([0, 3], dtype=torch.int32)),
           dict(query_start_loc=torch.tensor([0, 3, 5])), dict(status=torch.zeros(())),
           dict(key_cache=c.key.view(torch.uint8)[:, :, :, ::2].view(FP8)), dict(block_tables=c.tables[:, :0])]
    for over in bad:
        with pytest.raises((PaArgumentError, RuntimeError)) as e:
            pa.append_kv_cache(**{**good, **over})
        assert isinstance(e.value, PaArgumentError), (over.keys(), e.value)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa.append_kv_cache(**good)


def test_score_and_select_refusals():
    c = Cache([40, 7], 2, 16)
    good = dict(query=c.query(3), key_bounds=c.bounds(), sequence_lengths=c.lengths, block_tables=c.tables,
                softmax_scale=SCALE, query_sequence_length=1, block_size=16, key_scale=c.ks)
    bad = [dict(query=c.query(3).half()), dict(query=c.query(3)[0]), dict(key_bounds=c.bounds().float()),
           dict(key_bounds=c.bounds()[..., :64]), dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=math.nan),
           dict(query_sequence_length=2), dict(query_sequence_length=0), dict(block_size=32), dict(query=c.query(65)),
           dict(key_scale=torch.ones(c.nb, 2, 16, 1)), dict(key_scale=torch.ones(c.nb, 1, 1, 1)), dict(block_tables=c.tables[:1]),
           dict(sequence_lengths=c.lengths.long()), dict(scores=torch.empty(2, 2, 1)), dict(query_scale=torch.ones(2, 5, 1)),
           dict(status=torch.zeros(()))]
    for over in bad:
        with pytest.raises((PaArgumentError, RuntimeError)) as e:
            pa.score_blocks(**{**good, **over})
        assert isinstance(e.value, PaArgumentError), (over.keys(), e.value)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa.score_blocks(**good)
    good = dict(scores=torch.zeros(2, 2, 3), sequence_lengths=c.lengths, block_tables=c.tables, block_size=16, top_k=2)
    bad = [dict(scores=torch.zeros(2, 2, 2)), dict(scores=torch.zeros(2, 2, 3).double()), dict(scores=torch.zeros(2, 3)),
           dict(top_k=1), dict(top_k=0), dict(keep_first=-1), dict(keep_last=0), dict(keep_first=2), dict(block_size=48),
           dict(tables=torch.zeros(2, 2, 3, dtype=torch.int32)), dict(lengths=torch.zeros(3, dtype=torch.int32)),
           dict(scores=torch.zeros(1, 2, 3)), dict(block_tables=c.tables.long())]
    for over in bad:
        with pytest.raises((PaArgumentError, RuntimeError)) as e:
            pa.select_blocks(**{**good, **over})
        assert isinstance(e.value, PaArgumentError), (over.keys(), e.value)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa.select_blocks(**good)
    q = c.query(2, 2)
    with pytest.raises(PaArgumentError):       # two query tokens need the last two pages
        pa.sparse_attention_decode(torch.empty_like(q), q, c.key, c.value, c.bounds(), c.lengths, c.tables, SCALE, 2, 4,
                                   None, c.ks, c.vs, keep_last=1)
    with pytest.raises(PaArgumentError):
        pa.sparse_attention_decode(torch.empty_like(q), q, c.key, c.value, c.bounds()[:1], c.lengths, c.tables, SCALE, 2, 4,
                                   None, c.ks, c.vs)


# ----------------------------------------------------------------------------- GPU: attention with block scales
LENGTHS = [0, 1, 15, 255, 256, 257, 700, 2, 1025]


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["normal", "transposed"])
@pytest.mark.parametrize("bs", [16, 64, 1024])
@pytest.mark.parametrize("group,query_len", [(1, 1), (3, 1), (4, 1), (8, 1), (5, 3), (16, 1), (8, 2), (2, 4), (16, 4)])
def test_attention_with_block_scales(bs, group, query_len, layout):
    c = Cache(LENGTHS, 2, bs, seed=bs + group)
    q = c.query(group, query_len)
    value = transposed(c.value) if layout == "transposed" else c.value
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = decode(c, q, query_len=query_len, value=value, status=status)
    assert int(status) == 0
    want = bo.attention(q, c.key, value, c.ks, c.vs, c.tables, c.lengths, SCALE, query_len)
    assert_attention(got, want, f"bs {bs} group {group}")
    assert not got[0].any()                     # no token, nothing to attend to


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64])
def test_value_scales_far_apart_keep_their_digits(bs):
    """The token that holds the weight may lie in a page whose values are a million times smaller."""
    c = Cache([200, 530], 2, bs, seed=5)
    q = c.query(4) * 4
    for s in range(2):
        page = int(c.tables[s, 2])
        c.vs[page] = 2.0 ** -30
        # keys of that page along each head's first query row: their logits exceed the others by far
        for h in range(2):
            row = q[s, h * 4].float()
            want = (row / row.abs().max() * 300).to(FP8)
            c.key[page, h] = want.view(8, 1, 16).expand(8, bs, 16)
            c.ks[page, h] = 2.0 ** -2
    got = decode(c, q)
    out, mass, floor = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 1)
    assert_attention(got, (out, mass, floor))
    row = got[:, 0].double()
    assert float(row.abs().max()) < 1e-3        # the small page's values: no other page's weight shows
    assert float((row - out[:, 0]).norm() / out[:, 0].norm()) < 2.0 ** -6


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["alibi", "sink", "fp8 query", "fp8 query rows", "one value"])
def test_attention_options(form):
    c = Cache([300, 17, 0, 600], 2, 16, seed=9)
    q = c.query(4)
    kw, ref = {}, {}
    if form == "alibi":
        slopes = torch.linspace(0.02, 0.3, 8)
        kw["alibi_slopes"], ref["alibi_slopes"] = slopes.cuda(), slopes
    elif form == "sink":
        sink = torch.linspace(-2, 3, 8)
        kw["sink_tokens"], ref["sink_tokens"] = sink.cuda(), sink
    elif form == "fp8 query":
        q = (q.float() * 40).to(FP8)
        kw["query_scale"], ref["query_scale"] = torch.tensor(1 / 40, device="cuda"), torch.tensor(1 / 40)
    elif form == "fp8 query rows":
        q = (q.float() * 40).to(FP8)
        scale = torch.rand(4, 8, 1) / 20 + 0.01
        kw["query_scale"], ref["query_scale"] = scale.cuda(), scale
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    ks, vs = (torch.tensor(0.03), torch.tensor(0.02)) if form == "one value" else (c.ks, c.vs)
    tables = c.tables
    if form == "one value":                     # per-tensor scales go with tables per kv head too
        tables = c.tables[:, None].expand(-1, 2, -1).contiguous()
    pa.paged_attention_decode(out, *cuda(q, c.key, c.value, c.lengths, tables), SCALE, 1, 600, torch.bfloat16,
                              kw.pop("query_scale", None), *cuda(ks, vs), **kw)
    assert_attention(out.cpu(), bo.attention(q, c.key, c.value, ks, vs, tables, c.lengths, SCALE, 1, **ref), form)


@pytest.mark.gpu
def test_masked_places_may_hold_anything():
    """NaN codes behind the last token, NaN and infinite scales of unused pages, ids that are no pages."""
    c = Cache([37, 250, 513], 2, 16, seed=3, spare=4)
    q = c.query(8, 2)
    want = bo.attention(q, c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 2)
    nan = torch.tensor(0x7f, dtype=torch.uint8)
    for s, n in enumerate([37, 250, 513]):
        page, used = int(c.tables[s, (n - 1) // 16]), (n - 1) % 16 + 1
        c.key.view(torch.uint8)[page, :, :, used:] = nan
        c.value.view(torch.uint8)[page, :, :, used:] = nan
    for page in c.free:
        c.ks[page], c.vs[page] = math.nan, math.inf
        c.key.view(torch.uint8)[page] = nan
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = decode(c, q, query_len=2, status=status)
    assert int(status) == 0
    assert_attention(got, want)


@pytest.mark.gpu
def test_bad_tables_and_lengths_are_reported():
    c = Cache([300, 40], 2, 16, seed=2)
    q = c.query(2)
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    tables = c.tables.clone()
    tables[1, 0] = c.nb                         # no page of the pool: read as page 0
    lengths = torch.tensor([c.width * 16 + 5, 40], dtype=torch.int32)
    got = decode(c, q, tables=tables, lengths=lengths, status=status, longest=c.width * 16)
    assert int(status) == _lib.PA_DEV_BAD_PAGE_ID | _lib.PA_DEV_CTX_TOO_LONG
    tables[1, 0] = 0
    want = bo.attention(q, c.key, c.value, c.ks, c.vs, tables, torch.tensor([c.width * 16, 40]), SCALE, 1)
    assert_attention(got[1:], tuple(t[1:] for t in want))


@pytest.mark.gpu
def test_a_single_value_is_a_scale_per_tensor():
    """Scales of shape [1, 1, 1, 1] mean what they always did, for every cache the operator takes."""
    g = torch.Generator().manual_seed(3)
    kc, vc = torch.randn(9, 2, 16, 16, 8, generator=g).bfloat16().cuda(), torch.randn(9, 2, D, 16, generator=g).bfloat16().cuda()
    q = torch.randn(1, 8, D, generator=g).bfloat16().cuda()
    tables, lengths = torch.arange(9).int()[None].cuda(), torch.tensor([140], dtype=torch.int32).cuda()
    outs = []
    for shape in ((), (1, 1, 1, 1)):
        out = torch.empty_like(q)
        ks, vs = torch.full(shape, 0.5, device="cuda"), torch.full(shape, 2.0, device="cuda")
        pa.paged_attention_decode(out, q, kc, vc, lengths, tables, SCALE, 1, 144, torch.bfloat16, None, ks, vs)
        outs.append(out)
    assert torch.equal(*outs)


@pytest.mark.gpu
def test_nothing_to_do():
    """No sequences, no tokens: nothing happens and nothing is refused."""
    c = Cache([40], 2, 16)
    empty = torch.zeros(0, c.width, dtype=torch.int32).cuda()
    none = torch.zeros(0, dtype=torch.int32).cuda()
    kc, vc, ks, vs, bounds = cuda(c.key, c.value, c.ks, c.vs, c.bounds())
    q = torch.zeros(0, 8, D, dtype=torch.bfloat16, device="cuda")
    res = pa.sparse_attention_decode(torch.empty_like(q), q, kc, vc, bounds, none, empty, SCALE, 1, 4, None, ks, vs)
    assert res["block_tables"].shape == (0, 2, 4) and res["sequence_lengths"].shape == (0,)
    pa.paged_attention_decode(torch.empty_like(q), q, kc, vc, none, empty, SCALE, 1, 16, torch.bfloat16, None, ks, vs)
    rows = torch.zeros(0, 2, D, dtype=torch.bfloat16, device="cuda")
    pa.append_kv_cache(rows, rows, kc, vc, ks, vs, empty, none, torch.zeros(1, dtype=torch.int32).cuda(), key_bounds=bounds)
    pa.append_kv_cache(rows, rows, kc, vc, ks, vs, c.tables.cuda(), c.lengths.cuda(), torch.zeros(2, dtype=torch.int32).cuda())
    assert_same([t.cpu() for t in (kc, vc, ks, vs, bounds)], [c.key, c.value, c.ks, c.vs, c.bounds()])


@pytest.mark.gpu
def test_query_and_output_views():
    """Rows that begin anywhere, sequences further apart than their rows are long."""
    c = Cache([300, 40], 2, 16, seed=17)
    wide = torch.randn(2, 13, D + 3, generator=c.g).bfloat16()
    dev = wide.cuda()
    room = torch.full((2, 11, D), 7.0, dtype=torch.bfloat16, device="cuda")
    pa.paged_attention_decode(room[:, 2:10], dev[:, 1:9, 3:], *cuda(c.key, c.value, c.lengths, c.tables), SCALE, 1, 300,
                              torch.bfloat16, None, *cuda(c.ks, c.vs))
    want = bo.attention(wide[:, 1:9, 3:], c.key, c.value, c.ks, c.vs, c.tables, c.lengths, SCALE, 1)
    assert_attention(room[:, 2:10].cpu(), want)
    assert bool((room[:, :2] == 7).all()) and bool((room[:, 10:] == 7).all())


# ----------------------------------------------------------------------------- GPU: tables per kv head
@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("group,query_len", [(1, 1), (4, 1), (8, 1), (8, 2), (16, 4)])
def test_attention_with_a_table_per_head(bs, group, query_len):
    c = Cache([3000, 70, 1, 0, 900], 3, bs, seed=group)
    q = c.query(group, query_len)
    k = 9
    pages = [-(-int(n) // bs) for n in c.lengths]
    tables = torch.full((5, 3, k + 4), 2 ** 30, dtype=torch.int32)[:, :, :k]        # rows further apart than they are long
    lengths = torch.zeros(5, dtype=torch.int32)
    for s, n in enumerate(pages):
        held = min(n, k)
        lengths[s] = held * bs - (n * bs - int(c.lengths[s]))
        for h in range(3):
            keep = 2 if query_len > 1 else 1
            picked = torch.cat((torch.randperm(max(n - keep, 0), generator=c.g)[:held - min(keep, held)].sort().values,
                                torch.arange(max(n - keep, 0), n)))[-held:] if held else torch.empty(0).long()
            tables[s, h, :held] = c.tables[s, picked.long()]
    got = decode(c, q, tables=tables, lengths=lengths, query_len=query_len, longest=k * bs)
    want = bo.attention(q, c.key, c.value, c.ks, c.vs, tables, lengths, SCALE, query_len)
    assert_attention(got, want)


@pytest.mark.gpu
def test_equal_tables_per_head_change_nothing():
    c = Cache([300, 17, 1200], 4, 16, seed=1)
    q = c.query(4)
    a = decode(c, q)
    b = decode(c, q, tables=c.tables[:, None].expand(-1, 4, -1).contiguous())
    assert torch.equal(a, b)
    d = decode(c, q, tables=c.tables[:, None].expand(-1, 4, -1))     # heads that share a table by a stride of zero
    assert torch.equal(a, d)


# ----------------------------------------------------------------------------- GPU: scores
@pytest.mark.gpu
@pytest.mark.parametrize("hkv,group,query_len", [(1, 1, 1), (2, 4, 1), (3, 5, 1), (8, 4, 1), (5, 3, 3), (2, 16, 1), (3, 8, 4), (2, 16, 4), (9, 2, 1)])
@pytest.mark.parametrize("bs", [16, 64])
def test_scores(hkv, group, query_len, bs):
    lengths = [0, 1, 16, 17, 255, 256, 257, 3000, 5]
    c = Cache(lengths, hkv, bs, seed=hkv, width=-(-3000 // bs) + 5)
    q = c.query(group, query_len)
    q[1] *= 2.0 ** 60                           # rows of any size
    q[2, :, 3] = 1000.0
    q[5] = 0
    bounds = c.bounds()
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = pa.score_blocks(*cuda(q, bounds, c.lengths, c.tables), SCALE, query_len, bs, key_scale=c.ks.cuda(), status=status).cpu()
    assert int(status) == 0
    want, terms = bo.scores(q, bounds, c.lengths, c.tables, SCALE, bs, c.ks)
    live = want > -math.inf
    assert torch.equal(got > -math.inf, live)
    # 256 products added in 32 bits, whose additions may truncate (2^-23 each), and three more roundings
    assert ((got.double() - want).abs()[live] <= (260 * 2.0 ** -23) * terms[live]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["no scale", "one scale", "float", "fp8 query", "fp8 query rows", "strided"])
def test_score_options(form):
    c = Cache([300, 17, 0, 600], 4, 16, seed=4)
    q = c.query(4)
    bounds = c.bounds()
    kw, ref = dict(key_scale=c.ks), dict(key_scale=c.ks)
    if form == "no scale":
        kw, ref = {}, {}
    elif form in ("one scale", "float"):
        kw = dict(key_scale=torch.tensor(0.25) if form == "one scale" else 0.25)
        ref = dict(key_scale=torch.tensor(0.25))
    elif form == "fp8 query":
        q = (q.float() * 40).to(FP8)
        kw["query_scale"] = ref["query_scale"] = torch.tensor(1 / 40)
    elif form == "fp8 query rows":
        q = (q.float() * 40).to(FP8)
        kw["query_scale"] = ref["query_scale"] = torch.rand(4, 16, 1) / 20 + 0.01
    kw = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    dq, db, dl, dt = cuda(q, bounds, c.lengths, c.tables)
    if form == "strided":                       # every operand a view, pages of the bounds apart, heads not adjacent
        wide = torch.zeros(4, 16, 2 * D, dtype=torch.bfloat16, device="cuda")
        wide[:, :, :D] = dq
        dq = wide[:, :, :D]
        room = torch.zeros(c.nb, 4, 3, 2, D, dtype=torch.uint8, device="cuda").view(FP8)
        room.view(torch.uint8)[:, :, 1] = db.view(torch.uint8)
        db = room[:, :, 1]
        table = torch.zeros(4, c.width * 2, dtype=torch.int32, device="cuda")
        table[:, ::2] = dt
        dt = table[:, ::2]
        ks = torch.zeros(4, c.nb, 1, 1, device="cuda")
        ks.copy_(c.ks.transpose(0, 1))
        kw["key_scale"] = ks.transpose(0, 1)
        kw["scores"] = torch.zeros(4, 4, c.width + 3, device="cuda")[:, :, :c.width]
    got = pa.score_blocks(dq, db, dl, dt, SCALE, 1, 16, **kw).cpu()
    want, terms = bo.scores(q, bounds, c.lengths, c.tables, SCALE, 16, **ref)
    live = want > -math.inf
    assert torch.equal(got > -math.inf, live)
    assert ((got.double() - want).abs()[live] <= (260 * 2.0 ** -23) * terms[live]).all()


@pytest.mark.gpu
def test_no_logit_exceeds_its_page_score():
    c = Cache([700], 2, 16, seed=8)
    q = c.query(4)
    got = pa.score_blocks(*cuda(q, c.bounds(), c.lengths, c.tables), SCALE, 1, 16, key_scale=c.ks.cuda()).cpu()
    for h in range(2):
        for i in range(c.width):
            page = int(c.tables[0, i])
            k = bo.key_page(c.key, page, h)[:min(16, 700 - 16 * i)] * float(c.ks[page, h])
            logits = q[0, 4 * h:4 * h + 4].double() @ k.T * SCALE
            assert float(logits.max()) <= float(got[0, h, i]) * (1 + 1e-6) + 1e-6


@pytest.mark.gpu
def test_scores_report_bad_tables():
    c = Cache([300, 40], 2, 16, seed=2)
    q = c.query(2)
    tables = c.tables.clone()
    tables[0, 3] = -1
    lengths = torch.tensor([2 ** 31 - 1, 40], dtype=torch.int32)
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = pa.score_blocks(*cuda(q, c.bounds(), lengths, tables), SCALE, 1, 16, key_scale=c.ks.cuda(), status=status).cpu()
    assert int(status) == _lib.PA_DEV_BAD_PAGE_ID | _lib.PA_DEV_CTX_TOO_LONG
    tables[0, 3] = 0
    want, terms = bo.scores(q, c.bounds(), torch.tensor([c.width * 16, 40]), tables, SCALE, 16, c.ks)
    live = want > -math.inf
    assert torch.equal(got > -math.inf, live)
    assert ((got.double() - want).abs()[live] <= (260 * 2.0 ** -23) * terms[live]).all()


@pytest.mark.gpu
def test_scores_of_many_short_sequences():
    lengths = [(7 * i) % 90 for i in range(700)]
    c = Cache(lengths, 2, 16, seed=6)
    q = c.query(2)
    got = pa.score_blocks(*cuda(q, c.bounds(), c.lengths, c.tables), SCALE, 1, 16, key_scale=c.ks.cuda()).cpu()
    want, terms = bo.scores(q, c.bounds(), c.lengths, c.tables, SCALE, 16, c.ks)
    live = want > -math.inf
    assert torch.equal(got > -math.inf, live)
    assert ((got.double() - want).abs()[live] <= (260 * 2.0 ** -23) * terms[live]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["bf16", "fp8", "fp8, a scale a row"])
@pytest.mark.parametrize("hkv,group", [(8, 4), (3, 2), (2, 16), (1, 30), (2, 40)])
def test_scores_of_many_sequences_and_queries(hkv, group, rows):
    """A CTA goes from one sequence's query (and its scales) to the next; what lies past a short context is -inf."""
    lengths = [(41 * i) % 700 if i % 5 else 0 for i in range(500)]
    c = Cache(lengths, hkv, 16, seed=hkv, width=1500)
    q = c.query(group) * torch.exp2(torch.randint(-4, 5, (500, hkv * group, 1), generator=c.g).float()).bfloat16()
    scale = None
    if rows != "bf16":
        q = (q.float() * 8).to(FP8)
        scale = torch.rand(500, hkv * group, 1, generator=c.g) + 0.1 if rows == "fp8, a scale a row" else torch.tensor(0.125)
    out = torch.full((500, hkv, 1500), 7.0, device="cuda")
    kw = dict(key_scale=c.ks.cuda(), scores=out, query_scale=None if scale is None else scale.cuda())
    got = pa.score_blocks(*cuda(q, c.bounds(), c.lengths, c.tables), SCALE, 1, 16, **kw).cpu()
    want, terms = bo.scores(q, c.bounds(), c.lengths, c.tables, SCALE, 16, c.ks, **({} if scale is None else dict(query_scale=scale)))
    live = want > -math.inf
    assert torch.equal(got > -math.inf, live)
    assert ((got.double() - want).abs()[live] <= (260 * 2.0 ** -23) * terms[live]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,group", [(1, 4), (2, 4), (3, 20), (1, 64), (8, 4)])
def test_scores_of_long_contexts_are_the_same_every_time(hkv, group):
    """Many tiles for every SM, few kv heads: rings whose slots pass between warps."""
    g = torch.Generator().manual_seed(hkv)
    lengths = torch.tensor([60000, 31, 45001, 70000], dtype=torch.int32)
    width, nb = 4375, 11000
    tables = torch.randint(0, nb, (4, width), generator=g, dtype=torch.int32)
    bounds = random_codes((nb, hkv, 2, D), g).float().sort(2).values.to(FP8)
    ks = torch.exp2(torch.randint(-6, -2, (nb, hkv, 1, 1), generator=g).float())
    q = torch.randn(4, hkv * group, D, generator=g).bfloat16()
    dev = cuda(q, bounds, lengths, tables)
    first = pa.score_blocks(*dev, SCALE, 1, 16, key_scale=ks.cuda())
    for _ in range(20):
        assert torch.equal(pa.score_blocks(*dev, SCALE, 1, 16, key_scale=ks.cuda()), first)
    # against 64 bits on the GPU, sequence by sequence
    for s in range(4):
        pages = -(-int(lengths[s]) // 16)
        ids = tables[s, :pages].long().cuda()
        b, k = dev[1].float().double()[ids], ks.cuda().double()[ids, :, 0, 0].T
        for h in range(hkv):
            rows = q[s, h * group:(h + 1) * group].cuda().double()
            lo, hi = b[:, h, 0], b[:, h, 1]
            u = rows.clamp_min(0) @ hi.T + rows.clamp_max(0) @ lo.T
            terms = rows.clamp_min(0) @ hi.abs().T + rows.clamp_max(0).abs() @ lo.abs().T
            want, slack = u.amax(0) * SCALE * k[h], terms.amax(0) * SCALE * k[h] * 260 * 2.0 ** -23
            assert bool(((first[s, h, :pages].double() - want).abs() <= slack).all())


# ----------------------------------------------------------------------------- GPU: selection
def run_select(score, lengths, tables, bs, k, **kw):
    got = pa.select_blocks(*cuda(score, lengths, tables), bs, k, **kw)
    return tuple(t.cpu() for t in got)


@pytest.mark.gpu
@pytest.mark.parametrize("values", ["normal", "ties", "one value", "nan", "infinite", "tiny", "wide"])
@pytest.mark.parametrize("width,top_k", [(3, 2), (5, 40), (40, 7), (300, 64), (600, 2), (2100, 700), (9000, 33), (9000, 3000)])
def test_selection(width, top_k, values):
    g = torch.Generator().manual_seed(width)
    pages = [width, max(1, width // 2), 1, 0, min(top_k, width), min(top_k + 1, width)]
    lengths = torch.tensor([max(0, n * 16 - (5 * i) % 16) for i, n in enumerate(pages)], dtype=torch.int32)
    score = torch.randn(6, 2, width, generator=g)
    if values == "ties":
        score = (score * 2).round()
    elif values == "one value":
        score = torch.full_like(score, -3.5)
    elif values == "nan":
        score[torch.rand(score.shape, generator=g) < 0.7] = math.nan
    elif values == "infinite":
        score[torch.rand(score.shape, generator=g) < 0.3] = math.inf
        score[torch.rand(score.shape, generator=g) < 0.5] = -math.inf
    elif values == "tiny":
        score = score * 1e-42 * (torch.rand(score.shape, generator=g) < 0.5)
    elif values == "wide":
        score = score * torch.exp2(torch.randint(-120, 120, score.shape, generator=g).float())
    tables = torch.randint(0, 2 ** 30, (6, width), generator=g, dtype=torch.int32)
    want = bo.select(score, lengths, tables, 16, top_k)
    got = run_select(score, lengths, tables, 16, top_k)
    assert torch.equal(got[1], want[1])
    assert torch.equal(got[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("first,last", [(0, 1), (3, 2), (1, 6), (4, 4)])
def test_selection_keeps_the_ends(first, last):
    g = torch.Generator().manual_seed(3)
    score = torch.randn(3, 2, 100, generator=g)
    lengths = torch.tensor([100 * 64, 9 * 64 - 1, 8 * 64], dtype=torch.int32)
    tables = torch.randint(0, 1000, (3, 100), generator=g, dtype=torch.int32)
    want = bo.select(score, lengths, tables, 64, 8, first, last)
    got = run_select(score, lengths, tables, 64, 8, keep_first=first, keep_last=last)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_selection_on_views():
    g = torch.Generator().manual_seed(4)
    score = torch.randn(2, 3, 50, generator=g)
    lengths = torch.tensor([800, 333], dtype=torch.int32)
    tables = torch.randint(0, 1000, (2, 50), generator=g, dtype=torch.int32)
    want = bo.select(score, lengths, tables, 16, 9)
    wide = torch.full((3, 2, 64), math.nan, device="cuda")
    wide[:, :, :50] = score.transpose(0, 1)
    room = torch.full((2, 3, 12), -5, dtype=torch.int32, device="cuda")
    out = torch.full((2,), -5, dtype=torch.int32, device="cuda")
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    got = pa.select_blocks(wide.transpose(0, 1), lengths.cuda(), tables.cuda(), 16, 9, tables=room[:, :, :9], lengths=out, status=status)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(out.cpu(), want[1]) and int(status) == 0
    assert bool((room[:, :, 9:] == -5).all())
    got = pa.select_blocks(wide.transpose(0, 1), torch.tensor([801, 333], dtype=torch.int32).cuda(), tables.cuda(), 16, 9, status=status)
    assert int(status) == _lib.PA_DEV_CTX_TOO_LONG and torch.equal(got[0].cpu(), want[0])


# ----------------------------------------------------------------------------- GPU: append
def append_both(c, key, value, lengths, start, bounds, value_cache=None, per_tensor=None, **kw):
    """One append on the GPU and one by the oracle; returns both sides' state."""
    vc = c.value if value_cache is None else value_cache
    state = [c.key.clone(), vc.clone(), c.ks.clone(), c.vs.clone(), None if bounds is None else bounds.clone()]
    if per_tensor is not None:
        state[2], state[3] = torch.tensor(per_tensor), torch.tensor(per_tensor * 0.7)
    dev = [None if t is None else t.cuda() for t in state]
    status = torch.zeros((), dtype=torch.int32, device="cuda")
    pa.append_kv_cache(*cuda(key, value), dev[0], dev[1], dev[2], dev[3], *cuda(c.tables, lengths, start), key_bounds=dev[4],
                       status=status, **kw)
    bo.append(key, value, state[0], state[1], state[2], state[3], c.tables, lengths, start, state[4])
    return [None if t is None else t.cpu() for t in dev], state, int(status)


def assert_same(got, want):
    for name, a, b in zip(("keys", "values", "key scales", "value scales", "bounds"), got, want):
        if a is None:
            continue
        a, b = a.float(), b.float()
        same = (a == b) | (a.isnan() & b.isnan())
        assert bool(same.all()), f"{name}: {int((~same).sum())} of {same.numel()} differ"


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["normal", "transposed"])
@pytest.mark.parametrize("bs", [16, 64, 1024])
@pytest.mark.parametrize("counts,before", [([1, 1, 1, 1], [0, 15, 16, 40]), ([3, 0, 40, 17], [14, 9, 0, 63]),
                                           ([200, 1, 90, 130], [5, 1100, 64, 1000])])
def test_append(bs, counts, before, layout):
    after = [a + b for a, b in zip(before, counts)]
    c = Cache(after, 2, bs, seed=sum(counts))
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    n = sum(counts)
    size = torch.exp2(torch.randint(-3, 6, (n, 1, 1), generator=c.g).float())
    key = (torch.randn(n, 2, D, generator=c.g) * size).bfloat16()
    value = (torch.randn(n, 2, D, generator=c.g) * size).bfloat16()
    vc = transposed(c.value) if layout == "transposed" else None
    got, want, status = append_both(c, key, value, c.lengths, start, c.bounds(), value_cache=vc)
    assert status == 0
    assert_same(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64, 1024])
@pytest.mark.parametrize("hkv,counts,before", [(1, [1500, 700], [900, 0]), (2, [64] * 40, [1000] * 40), (4, [3000], [5]), (1, [300, 0, 2], [1020, 8, 5])])
def test_append_of_prompts(bs, hkv, counts, before):
    """Many rows for few pages, and for many: each way of dividing a page's rows over warps and CTAs."""
    c = Cache([a + b for a, b in zip(before, counts)], hkv, bs, seed=len(counts))
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    n = sum(counts)
    key, value = torch.randn(n, hkv, D, generator=c.g).bfloat16() * 3, torch.randn(n, hkv, D, generator=c.g).bfloat16()
    key[n // 2, 0, 17] = 4000.0                  # one page that has to grow far
    got, want, status = append_both(c, key, value, c.lengths, start, c.bounds())
    assert status == 0
    assert_same(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["normal", "transposed"])
@pytest.mark.parametrize("bs", [16, 64, 1024])
@pytest.mark.parametrize("per_tensor", [None, 0.013])
def test_append_of_a_few_rows_to_many_pages(bs, layout, per_tensor):
    """More (page, head) pairs than are worked on at once, a few rows each; pages that grow and pages that stay."""
    counts = [(7 * i) % 25 if i % 9 else 0 for i in range(60)]
    before = [(37 * i) % 150 for i in range(60)]
    c = Cache([a + b for a, b in zip(before, counts)], 7, bs, seed=5)
    start = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    n = sum(counts)
    size = torch.exp2(torch.randint(-7, 3, (n, 1, 1), generator=c.g).float())      # some pages' scales stay, some grow
    key = (torch.randn(n, 7, D, generator=c.g) * size).bfloat16()
    value = (torch.randn(n, 7, D, generator=c.g) * size).bfloat16()
    vc = transposed(c.value) if layout == "transposed" else None
    got, want, status = append_both(c, key, value, c.lengths, start, c.bounds(), value_cache=vc, per_tensor=per_tensor)
    assert status == 0
    assert_same(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("per_tensor", [None, 0.013])
@pytest.mark.parametrize("bs,count,seqs", [(64, 15, 40), (64, 30, 3), (1024, 60, 10), (1024, 260, 10), (1024, 260, 2), (1024, 1030, 6)])
def test_append_begins_and_ends_inside_runs(bs, count, seqs, per_tensor):
    """Values that share a 16-token run with older ones at the first row and with none at the last, on scales that stay."""
    c = Cache([8 + count] * seqs, 11, bs, seed=count)
    start = torch.arange(seqs + 1, dtype=torch.int32) * count
    key = torch.randn(seqs * count, 11, D, generator=c.g).bfloat16() * 0.05
    value = torch.randn(seqs * count, 11, D, generator=c.g).bfloat16() * 0.05
    got, want, status = append_both(c, key, value, c.lengths, start, c.bounds(), per_tensor=per_tensor)
    assert status == 0
    assert_same(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("bs", [16, 64])
def test_append_token_by_token_grows_pages(bs):
    """Tokens that get larger and larger: each page's scale grows again and again."""
    steps = 70
    c = Cache([steps, steps + 3], 1, bs, seed=1)
    state = [c.key.cuda(), c.value.cuda(), torch.full_like(c.ks, math.nan).cuda(), torch.full_like(c.vs, math.nan).cuda(), c.bounds().cuda()]
    ref = [c.key.clone(), c.value.clone(), torch.full_like(c.ks, math.nan), torch.full_like(c.vs, math.nan), c.bounds()]
    for i in range(steps):
        lengths = torch.tensor([i + 1, i + 1], dtype=torch.int32)
        start = torch.tensor([0, 1, 2], dtype=torch.int32)
        key = (torch.randn(2, 1, D, generator=c.g) * 1.3 ** (i % 40)).bfloat16()
        value = (torch.randn(2, 1, D, generator=c.g) * 0.9 ** i).bfloat16()
        pa.append_kv_cache(*cuda(key, value), *state[:4], *cuda(c.tables, lengths, start), key_bounds=state[4])
        bo.append(key, value, *ref[:4], c.tables, lengths, start, ref[4])
    got = [t.cpu() for t in state]
    used = c.tables[c.tables >= 0].unique().long()
    assert_same([t[used] for t in got], [t[used] for t in ref])


@pytest.mark.gpu
def test_append_of_anything():
    """Infinities saturate and do not set the scale, NaN stays, zeros get the smallest scale."""
    counts = [16, 16, 5, 20]
    c = Cache([16, 16, 12, 40], 2, 16, seed=7)
    start = torch.tensor([0, 16, 32, 37, 57], dtype=torch.int32)
    key = torch.randn(57, 2, D, generator=c.g).bfloat16()
    value = torch.randn(57, 2, D, generator=c.g).bfloat16()
    key[0, 0, 5], key[3, 0, 5], value[2, 1, 9] = math.inf, -math.inf, -math.inf
    key[1, 1, 7], value[4, 0, 3] = math.nan, math.nan
    key[16:32], value[16:32] = 0, 0
    value[40, 0, 0] = 3e38
    key[38, 1] = 1e-38
    got, want, status = append_both(c, key, value, c.lengths, start, c.bounds())
    assert status == 0
    assert_same(got, want)
    assert float(got[2][int(c.tables[1, 0]), 0]) == 2.0 ** -40


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["no bounds", "per tensor", "odd scales", "views", "misaligned"])
def test_append_options(form):
    counts, before = [5, 33, 1], [13, 20, 0]
    c = Cache([18, 53, 1], 2, 16, seed=11)
    start = torch.tensor([0, 5, 38, 39], dtype=torch.int32)
    rows = torch.randn(39, 3, 2, D + 8, generator=c.g).bfloat16()
    key, value = rows[:, 0, :, :D].contiguous(), rows[:, 2, :, :D].contiguous()
    bounds = None if form == "no bounds" else c.bounds()
    kw = {}
    if form == "odd scales":                    # a cache that came with scales that are no powers of two
        c.ks, c.vs = c.ks * 1.37, c.vs * 1.9
    if form == "per tensor":
        kw["per_tensor"] = 0.013
    if form in ("views", "misaligned"):
        dev = [t.cuda() for t in (c.key, c.value, c.ks, c.vs, bounds)]
        drows = rows.cuda()
        dk, dv = (drows[:, 0, :, :D], drows[:, 2, :, :D]) if form == "views" else (drows[:, 0, :, 3:D + 3], drows[:, 2, :, 3:D + 3])
        pa.append_kv_cache(dk, dv, *dev[:4], *cuda(c.tables, c.lengths, start), key_bounds=dev[4])
        want = [c.key.clone(), c.value.clone(), c.ks.clone(), c.vs.clone(), bounds.clone()]
        bo.append(dk.cpu(), dv.cpu(), *want[:4], c.tables, c.lengths, start, want[4])
        assert_same([t.cpu() for t in dev], want)
        return
    got, want, status = append_both(c, key, value, c.lengths, start, bounds, **kw)
    assert status == 0
    assert_same(got, want)


@pytest.mark.gpu
def test_append_skips_rows_without_a_place():
    c = Cache([20, 20, 20], 2, 16, seed=13)
    kv = torch.randn(12, 2, D, generator=c.g).bfloat16()

    def call(tables, lengths, start):
        status = torch.zeros((), dtype=torch.int32, device="cuda")
        state = [t.cuda() for t in (c.key, c.value, c.ks, c.vs)]
        pa.append_kv_cache(*cuda(kv, kv), *state, *cuda(tables, torch.tensor(lengths, dtype=torch.int32), torch.tensor(start, dtype=torch.int32)),
                           status=status)
        return [t.cpu() for t in state], int(status)

    def oracle(*parts):
        """parts: (sequence, its length, first row, rows) that do get a place"""
        want = [t.clone() for t in (c.key, c.value, c.ks, c.vs)]
        for s, length, row, rows in parts:
            bo.append(kv[row:], kv[row:], *want, c.tables[s:s + 1], [length], [0, rows])
        return want

    everything = [(0, 20, 0, 4), (1, 20, 4, 4), (2, 20, 8, 4)]
    got, status = call(c.tables, [20, 20, 20], [0, 4, 8, 12])
    assert status == 0
    assert_same(got, oracle(*everything))
    tables = c.tables.clone()
    tables[1, 1] = c.nb                          # no page of the pool
    got, status = call(tables, [20, 20, 20], [0, 4, 8, 12])
    assert status == _lib.PA_DEV_BAD_PAGE_ID
    assert_same(got, oracle(everything[0], everything[2]))
    got, status = call(c.tables, [20, 40, 20], [0, 4, 8, 12])                # past the table
    assert status == _lib.PA_DEV_CTX_TOO_LONG
    assert_same(got, oracle(everything[0], everything[2]))
    got, status = call(c.tables, [20, 34, 20], [0, 4, 8, 12])                # the last two of four past the table
    assert status == _lib.PA_DEV_CTX_TOO_LONG
    assert_same(got, oracle(everything[0], (1, 32, 4, 2), everything[2]))
    got, status = call(c.tables, [20, 20, 3], [0, 4, 8, 12])                 # more rows than tokens
    assert status == _lib.PA_DEV_BAD_RANGE
    assert_same(got, oracle(everything[0], everything[1], (2, 3, 9, 3)))
    got, status = call(c.tables, [20, 20, 20], [0, 4, 2, 6])                 # a start that runs backwards: no rows
    assert status == _lib.PA_DEV_BAD_RANGE
    assert_same(got, oracle(everything[0], (2, 20, 2, 4)))
    got, status = call(c.tables, [20, 20, 20], [-3, 4, 8, 2 ** 30])          # ranges cut to the rows there are
    assert status == _lib.PA_DEV_BAD_RANGE
    assert_same(got, oracle(*everything))
    got, status = call(c.tables, [0, 0, -5], [0, 0, 0, 0])
    assert status == 0
    assert_same(got, oracle())


# ----------------------------------------------------------------------------- GPU: together
def serve(steps, bs, top_k, group=4, query_len=1, hkv=2, graph=False):
    """A prompt, then decode steps: append, then attention over selected pages, against the oracle."""
    prompts = [700, 90, 333]
    total = [n + steps * query_len for n in prompts]
    c = Cache(total, hkv, bs, seed=bs)
    ks, vs = torch.zeros_like(c.ks).cuda(), torch.zeros_like(c.vs).cuda()
    kc, vc = torch.zeros_like(c.key.view(torch.uint8)).view(FP8).cuda(), torch.zeros_like(c.value.view(torch.uint8)).view(FP8).cuda()
    bounds = torch.zeros(c.nb, hkv, 2, D, dtype=torch.uint8).view(FP8).cuda()
    tables = c.tables.cuda()
    g = c.g

    def rows(n):
        return torch.randn(n, hkv, D, generator=g).bfloat16(), torch.randn(n, hkv, D, generator=g).bfloat16()

    start = torch.tensor([0] + torch.tensor(prompts).cumsum(0).tolist(), dtype=torch.int32).cuda()
    lengths = torch.tensor(prompts, dtype=torch.int32).cuda()
    k, v = rows(sum(prompts))
    pa.append_kv_cache(*cuda(k, v), kc, vc, ks, vs, tables, lengths, start, key_bounds=bounds)
    start = (torch.arange(4) * query_len).int().cuda()
    for _ in range(steps):
        lengths = lengths + query_len
        k, v = rows(3 * query_len)
        pa.append_kv_cache(*cuda(k, v), kc, vc, ks, vs, tables, lengths, start, key_bounds=bounds)
        q = torch.randn(3, hkv * group * query_len, D, generator=g).bfloat16()
        out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
        status = torch.zeros((), dtype=torch.int32, device="cuda")
        res = pa.sparse_attention_decode(out, q.cuda(), kc, vc, bounds, lengths, tables, SCALE, query_len, top_k, None, ks, vs, status=status)
        assert int(status) == 0
        yield c, q, out.cpu(), res, [t.cpu() for t in (kc, vc, ks, vs, bounds, lengths)]


@pytest.mark.gpu
@pytest.mark.parametrize("bs,query_len,group", [(16, 1, 4), (16, 2, 8), (64, 1, 1), (64, 3, 2)])
def test_serving_steps(bs, query_len, group):
    for c, q, out, res, (kc, vc, ks, vs, bounds, lengths) in serve(3, bs, 6, group, query_len):
        # the bounds are those of the codes in the cache
        for s in range(3):
            for i in range(-(-int(lengths[s]) // bs)):
                page, n = int(c.tables[s, i]), min(bs, int(lengths[s]) - i * bs)
                k = bo.key_page(kc, page, 0)[:n]
                assert torch.equal(bo.codes(bounds[page, 0]), torch.stack((k.amin(0), k.amax(0))))
        # the selection is that of the oracle wherever its scores leave no doubt
        want, terms = bo.scores(q, bounds, lengths, c.tables, SCALE, bs, ks)
        keep = 1 if query_len == 1 else 2
        tables, tokens = bo.select(want.float(), lengths, c.tables, bs, 6, 1, keep)
        got = res["block_tables"].cpu()
        assert torch.equal(res["sequence_lengths"].cpu(), tokens)
        assert float((got != tables).any(-1).double().mean()) < 0.2
        assert_attention(out, bo.attention(q, kc, vc, ks, vs, got, tokens, SCALE, query_len))


class NotTaken:
    """Host calls that take nothing: every call goes through the Python functions."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["plain", "transposed", "status", "per tensor", "two tokens"])
def test_both_ways_to_the_library_give_the_same_bits(monkeypatch, form):
    """Ordinary calls go from the tensors to the library in C++, the others through Python."""
    lib_calls = _lib.calls()
    query_len = 2 if form == "two tokens" else 1
    c = Cache([300, 17, 700], 2, 64 if form == "transposed" else 16, seed=23)
    value = transposed(c.value) if form == "transposed" else c.value
    q = c.query(4, query_len).cuda()
    rows = torch.randn(9, 2, D, generator=c.g).bfloat16().cuda()
    start = torch.tensor([0, 4, 4, 9], dtype=torch.int32).cuda()
    tables, lengths = cuda(c.tables, c.lengths)
    got = []
    for calls in (lib_calls, NotTaken()):
        monkeypatch.setattr(_lib, "_CALLS", calls)
        kc, vc, ks, vs, bounds = cuda(c.key.clone(), value.clone(), c.ks.clone(), c.vs.clone(), c.bounds())
        if form == "per tensor":
            ks, vs = torch.tensor(0.02, device="cuda"), torch.tensor(0.03, device="cuda")
        status = torch.zeros((), dtype=torch.int32, device="cuda") if form == "status" else None
        pa.append_kv_cache(rows, rows, kc, vc, ks, vs, tables, lengths, start, key_bounds=bounds, status=status)
        out = torch.full_like(q, math.nan)
        res = pa.sparse_attention_decode(out, q, kc, vc, bounds, lengths, tables, SCALE, query_len, 5, None, ks, vs, status=status)
        score = pa.score_blocks(q, bounds, lengths, tables, SCALE, query_len, c.bs, key_scale=ks, status=status)
        full = torch.full_like(q, math.nan)
        if form != "per tensor":
            pa.paged_attention_decode(full, q, kc, vc, lengths, tables, SCALE, query_len, 700, torch.bfloat16, None, ks, vs, status=status)
        got.append([kc, vc, ks, vs, bounds, out, res["block_tables"], res["sequence_lengths"], res["exponential_sums"].shape, score, full])
    for a, b in zip(*got):
        if isinstance(a, torch.Tensor):
            assert torch.equal(a.view(torch.uint8) if a.dim() else a, b.view(torch.uint8) if b.dim() else b)
        else:
            assert a == b


@pytest.mark.gpu
def test_errors_of_the_library_are_raised_either_way(monkeypatch):
    c = Cache([300], 2, 16)
    room = torch.zeros(c.nb * 2 * 2 * D + 8, dtype=torch.uint8, device="cuda")
    bounds = room[8:].view(FP8).view(c.nb, 2, 2, D)              # not on a 16-byte boundary
    q = c.query(2).cuda()
    for calls in (_lib.calls(), NotTaken()):
        monkeypatch.setattr(_lib, "_CALLS", calls)
        with pytest.raises(_lib.PaError, match="16-byte|align"):
            pa.score_blocks(q, bounds, *cuda(c.lengths, c.tables), SCALE, 1, 16, key_scale=c.ks.cuda())


@pytest.mark.gpu
def test_few_pages_are_all_read():
    """top_k at least the number of pages: the full attention, bit for bit."""
    for c, q, out, res, (kc, vc, ks, vs, bounds, lengths) in serve(1, 16, 64):
        full = torch.empty_like(out).cuda()
        pa.paged_attention_decode(full, *cuda(q, kc, vc, lengths, c.tables), SCALE, 1, 64 * 16, torch.bfloat16, None, *cuda(ks, vs))
        assert torch.equal(out, full.cpu())


@pytest.mark.gpu
def test_captured_steps_and_streams():
    """The whole step in CUDA graphs; two graphs of one shape replayed side by side, and eager calls on a
    third stream between them."""
    c = Cache([900, 200, 33, 512], 2, 16, seed=21)
    kv = [t.cuda() for t in (c.key, c.value, c.ks, c.vs, c.bounds(), c.tables)]
    lengths = c.lengths.cuda()
    qs = [c.query(4).cuda() for _ in range(3)]
    outs = [torch.full_like(q, math.nan) for q in qs]

    def step(i):
        pa.sparse_attention_decode(outs[i], qs[i], kv[0], kv[1], kv[4], lengths, kv[5], SCALE, 1, 8, None, kv[2], kv[3])

    step(0)
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            step(i)
        graphs.append(g)
    want = []
    for i in range(3):
        step(i)
        want.append(outs[i].clone())
        outs[i].fill_(math.nan)
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        with torch.cuda.stream(streams[2]):
            step(2)
    torch.cuda.synchronize()
    for i in range(3):
        assert torch.equal(outs[i], want[i]), i
    # lengths and query change under the graph
    lengths.copy_(torch.tensor([100, 0, 1, 300], dtype=torch.int32))
    qs[0].copy_(qs[1])
    graphs[0].replay()
    torch.cuda.synchronize()
    again = outs[0].clone()
    step(0)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], again)
    assert not outs[0][1].any()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A pool of more than 4 GB a side, pages at its far end."""
    hkv, bs = 8, 16
    nb = (1 << 32) // (hkv * bs * D) + 300
    kc = torch.empty(nb, hkv, 8, bs, 16, dtype=torch.uint8, device="cuda").view(FP8)
    vc = torch.empty(nb, hkv, D, bs, dtype=torch.uint8, device="cuda").view(FP8)
    ks, vs = torch.ones(nb, hkv, 1, 1, device="cuda"), torch.ones(nb, hkv, 1, 1, device="cuda")
    bounds = torch.zeros(nb, hkv, 2, D, dtype=torch.uint8, device="cuda").view(FP8)
    g = torch.Generator().manual_seed(0)
    n = 200
    tables = torch.full((1, 13), -1, dtype=torch.int32)
    tables[0] = torch.arange(nb - 13, nb).int()
    key, value = torch.randn(n, hkv, D, generator=g).bfloat16(), torch.randn(n, hkv, D, generator=g).bfloat16()
    lengths, start = torch.tensor([n], dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32)
    pa.append_kv_cache(*cuda(key, value), kc, vc, ks, vs, *cuda(tables, lengths, start), key_bounds=bounds)
    q = torch.randn(1, hkv * 4, D, generator=g).bfloat16()
    out = torch.empty_like(q).cuda()
    res = pa.sparse_attention_decode(out, q.cuda(), kc, vc, bounds, *cuda(lengths, tables), SCALE, 1, 5, None, ks, vs)
    far = slice(nb - 13, nb)
    small = [t[far].cpu() for t in (kc, vc, ks, vs)]
    want_state = [torch.zeros_like(t.view(torch.uint8)).view(FP8) if t.dtype == FP8 else torch.ones_like(t) for t in small]
    bo.append(key, value, *want_state, torch.arange(13)[None].int(), lengths, start)
    assert_same([small[2], small[3]], want_state[2:])
    for page in range(13):
        held = min(bs, n - page * bs)
        assert torch.equal(bo.key_page(small[0], page, 7)[:held], bo.key_page(want_state[0], page, 7)[:held])
        assert torch.equal(bo.value_page(small[1], page, 7)[:held], bo.value_page(want_state[1], page, 7)[:held])
    picked = res["block_tables"].cpu() - (nb - 13)
    assert_attention(out.cpu(), bo.attention(q, *small, picked, res["sequence_lengths"].cpu(), SCALE, 1))
