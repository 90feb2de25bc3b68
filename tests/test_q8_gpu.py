"""The operators over a cache in 8 bits, alone and one after the other, against tests/q8_refs.py."""
import math

import numpy as np
import pytest
import torch

import q8_refs as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
KINDS = [E4M3, INT8]


def ops():
    from neurogrid_b200.csrc import ops as o
    return o


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def codes(shape, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    return (x * 90).clamp(-448, 448).to(E4M3) if kind == E4M3 else (x * 36).round().clamp(-127, 127).to(INT8)


def scales(shape, seed, lo=-9, hi=-4):
    return torch.pow(2.0, torch.randint(lo, hi + 1, shape, generator=torch.Generator().manual_seed(seed)).float())


class Cache:
    """Pages of a few entries in random order, with pages over; every place that belongs to no entry holds the worst: NaN (e4m3) or
    the largest integer, scales of NaN."""

    def __init__(self, q_lens, ctx, n_kv, hd, page, block, kind, seed=0, extra=3, stride=None, dirty=True):
        self.q_lens, self.ctx, self.block, self.kind, self.page = list(q_lens), list(ctx), block, kind, page
        held = [-(-(n + c) // page) for n, c in zip(q_lens, ctx)]
        pages = sum(held) + extra
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((len(q_lens), stride or max(held + [1])), -1, dtype=torch.int32)
        for i, n in enumerate(held):
            table[i, :n] = torch.tensor(perm[sum(held[:i]):sum(held[:i]) + n], dtype=torch.int32)
        self.k, self.v = (codes((pages, n_kv, page, hd), kind, seed + 1 + i) for i in range(2))
        self.ks, self.vs = (scales((pages, n_kv, page // block), seed + 3 + i) for i in range(2))
        if dirty:
            live = torch.zeros(pages, page, dtype=torch.bool)
            for i, n in enumerate(held):
                for j in range(n):
                    live[int(table[i, j]), :max(0, min(page, q_lens[i] + ctx[i] - j * page))] = True
            bad = 0x7f
            for t in (self.k, self.v):
                t.view(torch.uint8).masked_fill_(~live[:, None, :, None], bad)
            used = live.view(pages, page // block, block).any(-1)
            for t in (self.ks, self.vs):
                t.masked_fill_(~used[:, None], math.nan)
        self.table_host = table
        self.cu_host = [0] + np.cumsum(q_lens).tolist()
        self.cu, self.ctx_d, self.table = i32(self.cu_host), i32(self.ctx), table.to(DEV)
        self.rows = self.cu_host[-1]
        self.row_entry = i32([e for e, n in enumerate(q_lens) for _ in range(n)])
        self.dev = [t.to(DEV) for t in (self.k, self.v, self.ks, self.vs)]

    def args(self):
        return (*self.dev, self.table)


def rnd(*shape, dtype=torch.bfloat16, seed=0, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def same_codes(got, values):
    """Codes equal to the oracle's values (a zero's sign may differ; NaN is NaN)."""
    got = got.cpu().to(torch.float64)
    return bool(((got == values) | (got.isnan() & values.isnan())).all())


# ------------------------------------------------------------------------------------------------ write
def check_write(c, k, v):
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = [t.clone() for t in c.dev]
    ops().cache_write_q8(k, v, *c.args(), c.row_entry, c.cu, c.ctx_d, st)
    for x, pages, sc, p0, s0 in ((k, c.dev[0], c.dev[2], before[0], before[2]), (v, c.dev[1], c.dev[3], before[1], before[3])):
        values, factors = ref.write(x.cpu(), p0.cpu(), s0.cpu(), c.table_host, c.cu_host, c.ctx)
        assert same_codes(pages, values)
        f = sc.cpu().double()
        assert bool(((f == factors) | (f.isnan() & factors.isnan())).all())
    return int(st)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_kv,hd,page,block,q_lens,ctx", [
    (8, 64, 16, 16, [1] * 7, [0, 1, 15, 16, 17, 100, 31]),            # decode: begun blocks, a block's first token
    (3, 80, 32, 8, [1, 40, 0, 7, 33], [5, 3, 9, 0, 31]),              # ragged, one entry brings nothing
    (1, 16, 8, 8, [130], [2]),
    (2, 256, 64, 64, [65, 1], [63, 64]),                              # more values than a warp keeps
    (4, 128, 64, 16, [600], [11]),                                    # many rows: eight a block
])
def test_write(kind, dtype, n_kv, hd, page, block, q_lens, ctx):
    c = Cache(q_lens, ctx, n_kv, hd, page, block, kind, seed=hd)
    k, v = (rnd(c.rows, n_kv * hd, dtype=dtype, seed=s, std=2.0) for s in (5, 6))
    k[:, ::hd // 16] *= 37.0
    assert check_write(c, k, v) == 0


@pytest.mark.parametrize("kind", KINDS)
def test_write_grows_and_keeps_scales(kind):
    """Tokens one by one, each twice as large as the one before, then smaller again: the block's scale only grows."""
    c = Cache([1], [0], 2, 16, 16, 16, kind, extra=0)
    for t in range(16):
        size = 2.0 ** (t if t < 9 else 18 - t) * 0.01
        c.ctx, c.ctx_d = [t], i32([t])
        assert check_write(c, rnd(1, 32, seed=t, std=size), rnd(1, 32, seed=t + 50, std=size)) == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_write_extremes(kind, dtype):
    """Zeros, the type's largest and smallest values, infinities and NaN: each in heads of its own, and beside ordinary values."""
    c = Cache([20], [4], 10, 16, 32, 16, kind, seed=1)
    k, v = (rnd(c.rows, 160, dtype=dtype, seed=s) for s in (1, 2))
    big = torch.finfo(dtype).max
    x = k.view(c.rows, 10, 16)
    x[:, 0] = 0.0
    x[:, 1] = big
    x[:, 2] = torch.finfo(dtype).tiny
    x[3, 3, 5], x[4, 3, 6], x[5, 3, 7] = math.inf, -math.inf, math.nan
    x[:, 4] = math.inf
    x[:, 5] = math.nan
    x[:, 6] *= 1e-38
    x[:, 7] = torch.linspace(-448, 448, 16, device=DEV).to(dtype)
    x[:, 8] = (torch.arange(16, device=DEV) + 0.5).to(dtype)               # ties
    x[0, 8, 0] = 127.0
    x[:, 9] *= 1e30
    v.view(c.rows, 10, 16)[:, 0] = 448.0 if kind == E4M3 else 127.0
    v.view(c.rows, 10, 16)[:, 1] = 448.5 if dtype == torch.float32 else 450.0
    assert check_write(c, k, v) == 0


def test_write_takes_columns_of_a_wider_buffer_and_odd_addresses():
    c = Cache([1, 9], [3, 20], 2, 32, 16, 8, E4M3)
    for offset in (0, 64, 8, 1, 3):
        wide = rnd(c.rows, 300, seed=offset)
        assert check_write(c, wide[:, offset:offset + 64], wide[:, offset + 128:offset + 192]) == 0
    assert check_write(c, *(rnd(c.rows * 64 + 5, seed=s)[5:].view(c.rows, 64) for s in (1, 2))) == 0


def test_write_passes_over_padding_and_pages_that_are_not_there():
    c = Cache([3, 2], [14, 0], 2, 16, 16, 16, INT8, extra=1)
    k, v = (rnd(8, 32, seed=s) for s in (1, 2))
    row_entry = i32([0, 0, 0, 1, 1, -1, -1, 7])                              # padding rows; an entry that is not there
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = [t.clone() for t in c.dev]
    ops().cache_write_q8(k, v, *c.args(), row_entry, c.cu, c.ctx_d, st)
    values, _ = ref.write(k.cpu(), before[0].cpu(), before[2].cpu(), c.table_host, c.cu_host, c.ctx)
    assert same_codes(c.dev[0], values) and int(st) == 0
    # the second page of entry 0 is missing, entry 1 names a page beyond the pool: a status bit, the rest is written
    c.table_host[0, 1] = -1
    table = c.table_host.to(DEV)
    table[1, 0] = 1000
    c.table_host[1, 0] = -1
    before = [t.clone() for t in c.dev]
    ops().cache_write_q8(k, v, *c.dev, table, row_entry, c.cu, c.ctx_d, st)
    values, _ = ref.write(k.cpu(), before[0].cpu(), before[2].cpu(), c.table_host, c.cu_host, c.ctx)
    assert same_codes(c.dev[0], values) and int(st) == 2


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nH,nKV,hd,page,block,norm,turn,half", [(4, 2, 64, 16, 16, True, True, True), (3, 1, 16, 8, 8, False, True, False),
                                                                (6, 2, 128, 32, 16, True, False, True), (2, 2, 80, 16, 8, True, True, False),
                                                                (2, 1, 256, 64, 64, False, False, True)])
@pytest.mark.parametrize("parts", [0, 1, 3])
def test_rope_and_write_in_one_launch(kind, nH, nKV, hd, page, block, norm, turn, half, parts):
    """Bit for bit what rope_cache and cache_write_q8 give one after the other; padding rows; a page that is not there."""
    c = Cache([1] * 6, [0, 1, block - 1, block, 3 * block + 5, 70], nKV, hd, page, block, kind, seed=hd)
    n, width = 8, (nH + 2 * nKV) * hd
    qkv = rnd(n, width, seed=1, std=2.0) if parts == 0 else rnd(parts, n, width, dtype=torch.float32, seed=1)
    w = [1 + 0.1 * rnd(hd, dtype=torch.float32, seed=s) if norm else None for s in (2, 3)]
    inv = 10000.0 ** (-torch.arange(hd // 2, device=DEV).float() / (hd // 2)) if turn else None
    row_entry, positions = i32([0, 1, 2, -1, 3, 4, 5, -1]), i32([0, 1, block - 1, 0, block, 3 * block + 5, 70, 0])
    cu, st = i32([0, 1, 2, 4, 5, 6, 8]), torch.zeros(1, dtype=torch.int32, device=DEV)
    q1, q2 = (torch.full((n, nH * hd), 9.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k, v = (torch.zeros(n, nKV, 1, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    twin = [t.clone() for t in c.dev]
    # (rope_cache takes a stack of one part for a bfloat16 tensor: it is given that part, rounded as the stack would be)
    ops().rope_cache(qkv[0].bfloat16() if parts == 1 else qkv, q1, *w, inv, half, 1.0, k, v, None, positions, row_entry, nH, nKV, hd, 1e-5, st)
    for r, e in enumerate(row_entry.tolist()):                               # (row by row: the entries' rows do not follow one another here)
        if e >= 0:
            ops().cache_write_q8(k[r:r + 1].view(1, -1), v[r:r + 1].view(1, -1), *twin, c.table[e:e + 1].contiguous(), i32([0]), i32([0, 1]),
                                 c.ctx_d[e:e + 1].contiguous(), st)
    ops().rope_cache_q8(qkv, q2, *w, inv, half, 1.0, *c.args(), positions, row_entry, nH, 1e-5, st)
    assert torch.equal(q1, q2) and int(st) == 0
    for a, b in zip(c.dev, twin):
        raw = torch.uint8 if a.element_size() == 1 else torch.int32
        assert torch.equal(a.view(raw), b.view(raw))
    row_entry[6] = len(c.q_lens)                                             # (an entry that the table has no row for counts as padding)
    twin = [t.clone() for t in c.dev]
    ops().rope_cache_q8(qkv, q2, *w, inv, half, 1.0, *c.args(), positions, row_entry, nH, 1e-5, st)
    assert bool((q2[6] == 0).all()) and torch.equal(q1[:6], q2[:6]) and int(st) == 0
    for t, b in zip(twin, c.dev):
        page = int(c.table_host[5, 70 // c.page])
        assert torch.equal(t.view(torch.uint8)[page], b.view(torch.uint8)[page])
    c.table[1, 0] = -1
    before = [t.clone() for t in c.dev]
    ops().rope_cache_q8(qkv, q2, *w, inv, half, 1.0, *c.args(), positions, row_entry, nH, 1e-5, st)
    page = int(c.table_host[1, 0])
    assert int(st) == 2 and all(torch.equal(a.view(torch.uint8)[page], b.view(torch.uint8)[page]) for a, b in zip(c.dev, before))


# ------------------------------------------------------------------------------------------------ attention
def check_rows(got, want, bound, rows=None):
    err = (got.cpu().double() - want).abs()
    ok = err <= bound
    if rows is not None:
        ok, err = ok[rows], err[rows]
    if ok.numel() == 0:
        return
    assert bool(ok.all()), f"worst {float(err.max()):.3e}, over the bound at {int((~ok).sum())} of {ok.numel()}"


def run_decode(c, q, nH, window, scale, splits, slopes=None, max_ctx=None):
    out = torch.full_like(q, 7.0)
    n = ops().attn_q8_scratch_floats(len(c.q_lens), nH, c.dev[0].shape[3], splits)
    scratch = torch.full((n,), math.nan, device=DEV) if n else None
    longest = max(a + b for a, b in zip(c.q_lens, c.ctx)) if max_ctx is None else max_ctx
    ops().attn_decode_q8(q, *c.args(), c.cu, c.ctx_d, out, scratch, len(c.q_lens), nH, window, scale, splits, longest, slopes)
    return out


def run_prefill(c, q, nH, window, scale, splits=1, skip_single=False, slopes=None):
    out = torch.full_like(q, 7.0)
    n = ops().attn_q8_scratch_floats(q.shape[0], nH, c.dev[0].shape[3], splits)
    scratch = torch.full((n,), math.nan, device=DEV) if n else None
    ops().attn_prefill_q8(q, *c.args(), c.cu, c.ctx_d, out, len(c.q_lens), max(c.q_lens), nH, window, scale, skip_single, slopes, scratch, splits)
    return out


SHAPES = [
    # heads, KV heads, head size, page, block
    (16, 8, 64, 16, 16), (32, 8, 64, 64, 32), (6, 2, 64, 8, 8), (12, 4, 128, 32, 16), (16, 1, 80, 16, 8), (20, 1, 32, 16, 16),
    (4, 4, 16, 8, 8), (8, 2, 256, 64, 64), (3, 1, 48, 32, 32), (40, 2, 96, 16, 16),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nH,nKV,hd,page,block", SHAPES)
@pytest.mark.parametrize("window,splits,bias", [(None, 1, False), (None, 5, True), (37, 2, False)])
def test_decode(kind, nH, nKV, hd, page, block, window, splits, bias):
    c = Cache([1, 1, 1, 3, 0, 1, 1], [0, 1, 7, 4, 9, 130, 517], nKV, hd, page, block, kind, seed=nH)
    q = rnd(c.rows, nH * hd, seed=9, std=1.5)
    slopes = torch.pow(2.0, -torch.arange(1, nH + 1).float() / nH).to(DEV) if bias else None
    scale = hd ** -0.5
    got = run_decode(c, q, nH, window, scale, splits, slopes)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, nH, window, scale, slopes)
    single = [r for e, n in enumerate(c.q_lens) for r in range(c.cu_host[e], c.cu_host[e + 1]) if n == 1]
    check_rows(got, want, bound, single)
    others = [r for r in range(c.rows) if r not in single]
    assert bool((got[others] == 7.0).all())                                 # rows of portions: left as they were


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nH,nKV,hd,page,block", SHAPES)
@pytest.mark.parametrize("window,splits,bias", [(None, 1, False), (None, 3, True), (50, 1, False)])
def test_prefill(kind, nH, nKV, hd, page, block, window, splits, bias):
    c = Cache([1, 70, 0, 5, 1, 33], [0, 0, 3, 260, 64, 90], nKV, hd, page, block, kind, seed=nH + 1)
    q = rnd(c.rows, nH * hd, seed=4, std=1.5)
    slopes = torch.pow(2.0, -torch.arange(1, nH + 1).float() / nH).to(DEV) if bias else None
    scale = hd ** -0.5
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, nH, window, scale, slopes)
    check_rows(run_prefill(c, q, nH, window, scale, splits, False, slopes), want, bound)
    got = run_prefill(c, q, nH, window, scale, splits, True, slopes)
    many = [r for e, n in enumerate(c.q_lens) for r in range(c.cu_host[e], c.cu_host[e + 1]) if n > 1]
    check_rows(got, want, bound, many)
    assert bool((got[[r for r in range(c.rows) if r not in many]] == 7.0).all())


@pytest.mark.parametrize("portion", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_over_scales_far_apart(kind, portion):
    """Blocks whose values are 2^40 apart, among them blocks of zeros at the least scale, and scores that favour the small ones."""
    c = Cache([2 if portion else 1] * 3, [300, 64, 511], 2, 64, 16, 16, kind, seed=3)
    g = torch.Generator().manual_seed(8)
    vs = torch.pow(2.0, torch.randint(-30, 11, c.vs.shape, generator=g).float())
    zero = torch.rand(c.vs.shape, generator=g) < 0.2
    vs[zero] = 2.0 ** -100
    v = c.v.view(c.v.shape[0], 2, 1, 16, 64)
    v.view(torch.uint8).masked_fill_(zero[..., None, None], 0)
    c.dev[3], c.dev[1] = vs.to(DEV), c.v.to(DEV)
    c.dev[2] = torch.pow(2.0, torch.randint(-12, -5, c.ks.shape, generator=g).float()).to(DEV)
    q = rnd(c.rows, 4 * 64, seed=1, std=2.0)
    q[0] *= 1e-4
    run = (lambda s: run_prefill(c, q, 4, None, 0.125, s)) if portion else (lambda s: run_decode(c, q, 4, None, 0.125, s))
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 4, None, 0.125)
    for s in (1, 4):
        check_rows(run(s), want, bound)


@pytest.mark.parametrize("portion", [False, True])
def test_rows_of_q_at_the_ends_of_the_type(portion):
    c = Cache([4] if portion else [1, 1, 1, 1], [40] if portion else [40] * 4, 1, 64, 16, 16, E4M3, seed=5)
    q = rnd(4, 2 * 64, seed=2)
    q[0] *= 1e-37                                                            # scores of nothing: the mean of the values
    q[1] = 0.0
    q[2, :64] *= 1e10                                                        # one key takes all
    q[3, 0] = math.nan
    got = run_prefill(c, q, 2, None, 0.125) if portion else run_decode(c, q, 2, None, 0.125, 1)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 2, None, 0.125)
    check_rows(got[:2], want[:2], bound[:2])
    assert torch.isfinite(got[2]).all()
    assert torch.isnan(got[3, :64]).all() and not torch.isnan(got[3, 64:]).any()


def test_decode_many_splits_and_a_bound_on_the_context_that_is_too_low():
    c = Cache([1], [1500], 2, 64, 16, 16, E4M3)
    q = rnd(1, 8 * 64, seed=1)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 8, None, 0.125)
    for splits in (1, 2, 7, 40):
        check_rows(run_decode(c, q, 8, None, 0.125, splits), want, bound)
        check_rows(run_decode(c, q, 8, None, 0.125, splits, max_ctx=100), want, bound)


def test_pages_that_a_window_has_given_back_are_not_needed():
    c = Cache([1, 20], [400, 300], 2, 64, 16, 16, INT8)
    q = rnd(c.rows, 4 * 64, seed=1)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 4, 64, 0.125)
    c.table[0, :(400 - 63) // 16] = -1
    c.table[1, :(300 - 63) // 16] = -1
    check_rows(run_decode(c, q, 4, 64, 0.125, 2), want, bound, [0])
    check_rows(run_prefill(c, q, 4, 64, 0.125, 2), want, bound)


def test_attention_and_write_beyond_32_bit_offsets():
    """Keys whose codes lie more than 2^32 bytes into their pool."""
    n_kv, hd, page = 8, 256, 64
    pages = (1 << 32) // (n_kv * hd * page) + 8
    c = Cache([1], [120], n_kv, hd, page, 16, E4M3, dirty=False)
    big = [torch.zeros((pages,) + t.shape[1:], dtype=t.dtype, device=DEV) for t in c.dev]
    for e, p in enumerate(c.table_host[0].tolist()):
        for b, t in zip(big, c.dev):
            b.view(torch.uint8 if b.element_size() == 1 else b.dtype)[pages - 1 - e].copy_(t.view(torch.uint8 if b.element_size() == 1 else b.dtype)[p])
    c.table_host[0] = torch.arange(pages - 1, pages - 1 - c.table_host.shape[1], -1)
    c.table, c.dev = c.table_host.to(DEV), big
    k, v = (rnd(1, n_kv * hd, seed=s) for s in (1, 2))
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops().cache_write_q8(k, v, *c.args(), c.row_entry, c.cu, c.ctx_d, st)
    q = rnd(1, 8 * hd, seed=3)
    tail = [t[pages - 8:].contiguous() for t in (b.view(torch.uint8) if b.element_size() == 1 else b for b in big)]
    tail = [t.view(E4M3) if t.dtype == torch.uint8 else t for t in tail]
    want, bound = ref.attention(q, *tail, c.table_host - (pages - 8), c.cu_host, c.ctx, 8, None, 1 / 16)
    check_rows(run_decode(c, q, 8, None, 1 / 16, 1), want, bound)
    check_rows(run_prefill(c, q, 8, None, 1 / 16), want, bound)
    ops().copy_pages([t[None] for t in big], [pages - 1], [pages - 5])
    for b in big:
        raw = b.view(torch.uint8) if b.element_size() == 1 else b
        assert torch.equal(raw[pages - 5], raw[pages - 1])


def test_a_captured_run_of_write_and_both_attentions_replays_with_new_data():
    """One graph over the batch's buffers; between replays the contexts grow and the tokens change.  The same calls made
    outside the graph, on another stream, give the same bits."""
    nH, nKV, hd, page, block = 8, 2, 64, 16, 16
    total = 64
    c = Cache([1, 6], [20, 9], nKV, hd, page, block, E4M3, stride=total // page, extra=16, dirty=False)
    for e, held in enumerate((2, 1)):
        free = [p for p in range(c.k.shape[0]) if p not in c.table_host.flatten().tolist()]
        c.table_host[e, held:] = torch.tensor(free[:total // page - held], dtype=torch.int32)
    c.table.copy_(c.table_host)
    k, v, q = rnd(7, nKV * hd, seed=1), rnd(7, nKV * hd, seed=2), rnd(7, nH * hd, seed=3)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    scratch = torch.empty(ops().attn_q8_scratch_floats(7, nH, hd, 3), device=DEV)

    def calls(dev, out):
        ops().cache_write_q8(k, v, *dev, c.table, c.row_entry, c.cu, c.ctx_d, st)
        ops().attn_prefill_q8(q, *dev, c.table, c.cu, c.ctx_d, out, 2, 6, nH, None, 0.125, True, None, scratch, 3)
        ops().attn_decode_q8(q, *dev, c.table, c.cu, c.ctx_d, out, scratch, 2, nH, None, 0.125, 3, total, None)

    out, other = torch.empty_like(q), torch.empty_like(q)
    twin = [t.clone() for t in c.dev]
    calls(twin, other)
    twin = [t.clone() for t in c.dev]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(c.dev, out)
    side = torch.cuda.Stream()
    for step in range(5):
        for t, s in ((k, 10), (v, 20), (q, 30)):
            t.copy_(rnd(*t.shape, seed=s + step))
        c.ctx = [20 + step, 9 + 6 * step]
        c.ctx_d.copy_(i32(c.ctx))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            calls(twin, other)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, other)
        for a, b in zip(c.dev, twin):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, nH, None, 0.125)
        check_rows(out, want, bound)
    assert int(st) == 0


def test_no_rows_and_no_entries():
    c = Cache([0, 0], [3, 0], 2, 16, 8, 8, INT8)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    before = [t.clone() for t in c.dev]
    none = torch.empty(0, 32, dtype=torch.bfloat16, device=DEV)
    ops().cache_write_q8(none, none, *c.args(), c.row_entry, c.cu, c.ctx_d, st)
    q = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    ops().attn_decode_q8(q, *c.args(), c.cu, c.ctx_d, q, None, 2, 4, None, 0.25, 1, 4)
    ops().attn_prefill_q8(q, *c.args(), c.cu, c.ctx_d, q, 2, 0, 4, None, 0.25, False)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c.dev, before))


def test_many_entries_and_longer_portions():
    """Sizes at which a launch has many blocks: 40 entries, one portion of 300 rows."""
    lens = [1] * 37 + [300, 2, 129]
    ctx = [(37 * i) % 200 for i in range(40)]
    c = Cache(lens, ctx, 4, 64, 16, 16, INT8, seed=2)
    q = rnd(c.rows, 16 * 64, seed=7)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 16, None, 0.125)
    out = run_prefill(c, q, 16, None, 0.125, 1, True)
    got = run_decode(c, q, 16, None, 0.125, 1)
    check_rows(got, want, bound, list(range(37)))
    check_rows(out, want, bound, list(range(37, c.rows)))


@pytest.mark.parametrize("hd", [48, 64])
@pytest.mark.parametrize("splits", [1, 3])
def test_entries_behind_their_table_or_in_front_of_it_are_left_alone(hd, splits):
    """A context that no row of the table holds, or of less than nothing: the rows stay as they were, the others are right."""
    q = rnd(5, 4 * hd, seed=6)
    c = Cache([1, 1, 1, 1, 1], [40, 9, 70, 0, 100], 2, hd, 16, 16, E4M3, seed=4)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 4, None, 0.125)
    c.ctx_d = i32([40, -1, 70, 2 ** 31 - 1, c.table.shape[1] * 16])
    got = run_decode(c, q, 4, None, 0.125, splits)
    check_rows(got, want, bound, [0, 2])
    assert bool((got[[1, 3, 4]] == 7.0).all())
    q = rnd(60, 4 * hd, seed=6)
    c = Cache([20, 7, 30, 3], [40, 9, 70, 5], 2, hd, 16, 16, E4M3, seed=4)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 4, None, 0.125)
    c.ctx_d = i32([40, -1, 70, c.table.shape[1] * 16])
    got = run_prefill(c, q, 4, None, 0.125, splits)
    check_rows(got, want, bound, [*range(20), *range(27, 57)])
    assert bool((got[[*range(20, 27), *range(57, 60)]] == 7.0).all())


@pytest.mark.parametrize("splits", [2, 9])
def test_decode_shares_of_many_entries(splits):
    """More entries than a warp looks over at once, of very different lengths, some with no single token."""
    lens = [1 if i % 7 else (0, 2)[i % 2] for i in range(100)]
    ctx = [(i * i * 13) % 900 if i % 5 else 0 for i in range(100)]
    c = Cache(lens, ctx, 2, 64, 16, 16, E4M3, seed=8)
    q = rnd(c.rows, 8 * 64, seed=3)
    single = [c.cu_host[e] for e, n in enumerate(lens) if n == 1]
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 8, None, 0.125)
    got = run_decode(c, q, 8, None, 0.125, splits)
    check_rows(got, want, bound, single)
    assert bool((got[[r for r in range(c.rows) if r not in single]] == 7.0).all())


@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("lens", [[1] * 70 + [90] + [0, 1, 2] * 20 + [65], [1], [3, 1], [1] * 40 + [0] * 40, [0, 0, 5, 0]])
def test_portions_beside_many_single_tokens(hd, splits, lens):
    """Row tiles are counted over the entries that have any, wherever they lie."""
    ctx = [(37 * i) % 150 for i in range(len(lens))]
    c = Cache(lens, ctx, 2, hd, 16, 16, INT8, seed=3)
    q = rnd(c.rows, 6 * hd, seed=7)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 6, None, 0.125)
    many = [r for e, n in enumerate(lens) for r in range(c.cu_host[e], c.cu_host[e + 1]) if n > 1]
    got = run_prefill(c, q, 6, None, 0.125, splits, True)
    check_rows(got[many], want[many], bound[many])
    assert bool((got[[r for r in range(c.rows) if r not in many]] == 7.0).all())
    check_rows(run_prefill(c, q, 6, None, 0.125, splits, False), want, bound)


def test_the_integer_that_the_writer_never_stores():
    """-128 stands for -128 times the scale."""
    c = Cache([1, 5], [60, 30], 2, 64, 16, 16, INT8, seed=6)
    for x in (c.k, c.v):
        x[torch.rand(x.shape, generator=torch.Generator().manual_seed(1)) < 0.1] = -128
    c.dev[0], c.dev[1] = c.k.to(DEV), c.v.to(DEV)
    q = rnd(c.rows, 4 * 64, seed=3)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 4, None, 0.125)
    check_rows(run_decode(c, q, 4, None, 0.125, 1), want, bound, [0])
    check_rows(run_prefill(c, q, 4, None, 0.125), want, bound)


def test_calls_on_two_streams_at_once():
    """Each with outputs and scratch of its own: nothing of a call is kept anywhere else."""
    c = Cache([1] * 8 + [200], [700 + 40 * i for i in range(8)] + [300], 2, 64, 16, 16, E4M3, seed=6)
    qs = [rnd(c.rows, 8 * 64, seed=10 + i) for i in range(2)]
    wants = [ref.attention(q, *c.args(), c.cu_host, c.ctx, 8, None, 0.125) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, (s, q) in enumerate(zip(streams, qs)):
            with torch.cuda.stream(s):
                got[i].append((run_decode(c, q, 8, None, 0.125, 6), run_prefill(c, q, 8, None, 0.125, 2, True)))
    torch.cuda.synchronize()
    for i, (want, bound) in enumerate(wants):
        for single, portion in got[i]:
            check_rows(single, want, bound, list(range(8)))
            check_rows(portion, want, bound, list(range(8, c.rows)))


# ------------------------------------------------------------------------------------------------ copies
@pytest.mark.parametrize("dtype", [E4M3, INT8, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,pages,tail,n", [(1, 5, (2, 8, 16), 1), (3, 40, (4, 16, 64), 15), (2, 3000, (1, 8, 16), 1300), (2, 70, (3, 8, 80), 33),
                                                (2, 9, (1, 1, 3), 4)])
def test_copy_pages(dtype, layers, pages, tail, n):
    g = torch.Generator().manual_seed(n)
    pools = [torch.randint(0, 256, (layers, pages) + tail + (torch.empty((), dtype=dtype).element_size(),), generator=g, dtype=torch.uint8)
             .to(DEV).view(dtype).squeeze(-1) for _ in range(2)]
    pools += [torch.rand(layers, pages, 3, 2, generator=g).to(DEV), None]
    order = torch.randperm(pages, generator=g)[:2 * n].to(torch.int32)
    src, dst = order[:n].clone(), order[n:2 * n]
    src[-1] = src[0]                                                          # one page to two
    raw = [p.view(torch.uint8).clone() for p in pools if p is not None]
    for r in raw:
        r[:, dst.long()] = r[:, src.long()].clone()
    for how in (lambda t: t, lambda t: t.numpy(), lambda t: t.tolist(), lambda t: t.long()):
        ops().copy_pages(pools, how(src), how(dst))
    for p, r in zip(pools, raw):
        assert torch.equal(p.view(torch.uint8), r)


def test_copy_pages_from_an_odd_address_and_in_a_graph():
    store = torch.arange(2 * 6 * 33 + 1, device=DEV).to(torch.uint8)
    pool = store[1:].view(2, 6, 33)
    want = pool.clone()
    want[:, [4, 5]] = want[:, [0, 3]]
    graph = torch.cuda.CUDAGraph()
    ops().copy_pages([pool], [], [])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops().copy_pages([pool], [0, 3], [4, 5])
    graph.replay()
    assert torch.equal(pool, want)
    pool[:, 0] += 1
    want[:, 0] += 1
    want[:, 4] += 1
    graph.replay()
    assert torch.equal(pool, want)


def test_copy_pages_refuses_what_has_no_one_result():
    pool = torch.zeros(2, 40, 8, device=DEV)
    pool += torch.arange(40, device=DEV)[None, :, None]
    want = pool.clone()
    many = list(range(18))
    for src, dst in (([0], [0]), ([0, 1], [5, 5]), ([0, 1], [1, 2]), ([40], [1]), ([-1], [1]), ([1], [40]), (many, many[::-1]),
                     (many, list(range(17, 35))), (many, [20] * 18), ([2 ** 40], [1])):
        with pytest.raises(ops().KernelError):
            ops().copy_pages([pool], src, dst)
    with pytest.raises(ops().KernelError):
        ops().copy_pages([pool], torch.zeros(1, dtype=torch.int32, device=DEV), [1])
    assert torch.equal(pool, want)
