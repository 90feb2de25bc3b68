"""Corners of the operators over a cache in 8 bits: neighbours on the stream, heads of NaN, scales far apart, tables with holes."""
import math

import pytest
import torch

import q8_refs as ref
from test_q8_gpu import DEV, E4M3, INT8, KINDS, Cache, check_rows, ops, rnd, run_decode, run_prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,hd", [(3, 64), (9, 64), (16, 64), (40, 64), (9, 128)])
def test_portions_between_products_that_use_tensor_memory(rows, hd):
    """A short portion between two tcgen05 products of as many rows, the three on one stream with nothing between them, many times: what each
    gives when the device is waited for after it."""
    nH, nKV, H = 32, 8, 512
    c = Cache([rows], [70], nKV, hd, 16, 16, E4M3, seed=rows)
    x, w1, w2 = rnd(rows, H, seed=1), rnd(nH * hd, H, seed=2, std=0.05), rnd(H, nH * hd, seed=3, std=0.05)
    q, a, y = (torch.empty(rows, n, dtype=torch.bfloat16, device=DEV) for n in (nH * hd, nH * hd, H))

    def step(between=lambda: None):
        ops().gemm_sm100(x, w1, None, q)
        between()
        ops().attn_prefill_q8(q, *c.args(), c.cu, c.ctx_d, a, 1, rows, nH, None, hd ** -0.5, False)
        between()
        ops().gemm_sm100(a, w2, None, y)
        between()

    step(torch.cuda.synchronize)
    want = y.clone()
    check_rows(a, *ref.attention(q, *c.args(), c.cu_host, c.ctx, nH, None, hd ** -0.5))
    for _ in range(200):
        step()
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(20):
            step()
    for _ in range(10):
        y.zero_()
        graph.replay()
        assert torch.equal(y, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nH,nKV,hd", [(8, 1, 64), (7, 1, 64), (16, 1, 64), (16, 2, 128), (15, 1, 32), (8, 1, 48), (24, 3, 256)])
@pytest.mark.parametrize("splits", [1, 5])
def test_heads_of_nan_leave_the_other_heads_of_their_tile_alone(kind, nH, nKV, hd, splits):
    """NaN in one head of every pair that a lane looks after, over many groups of keys."""
    c = Cache([1, 1, 1], [700, 3, 1500], nKV, hd, 16, 16, kind, seed=nH)
    q = rnd(3, nH * hd, seed=9, std=1.5)
    sick = torch.zeros(nH, dtype=torch.bool)
    sick[0::2] = True
    q.view(3, nH, hd)[:2, sick.to(DEV), hd // 2] = math.nan
    q.view(3, nH, hd)[2, (~sick).to(DEV), 0] = math.nan
    got = run_decode(c, q, nH, None, hd ** -0.5, splits)
    want, bound = ref.attention(torch.nan_to_num(q), *c.args(), c.cu_host, c.ctx, nH, None, hd ** -0.5)
    for r in range(3):
        ill = sick if r < 2 else ~sick
        of_row = [t[r].view(nH, hd) for t in (got, want, bound)]
        assert bool(torch.isnan(of_row[0][ill.to(DEV)]).all())
        check_rows(of_row[0][(~ill).to(DEV)], of_row[1][~ill], of_row[2][~ill])


def attention_with_holes(q, c, n_heads, window, scale, slopes, hidden):
    """ref.attention's 64-bit values where keys in ``hidden`` [entry][key] are not there, and sum_j weight_j |v_j|."""
    k_pages, v_pages, ks, vs = (t.cpu() for t in c.dev)
    n_kv, hd = k_pages.shape[1], k_pages.shape[3]
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    for e in range(len(c.ctx)):
        ctx, q0, n = c.ctx[e], c.cu_host[e], c.q_lens[e]
        j = torch.arange(ctx + n)
        p, at = c.table_host[e][j // c.page].long(), j % c.page
        pos = torch.arange(ctx, ctx + n)[:, None]
        for h in range(n_heads):
            g = h // (n_heads // n_kv)
            k, v = ((t[:, g].view(torch.uint8)[p, at].view(t.dtype).double() * s[p, g, at // c.block].double()[:, None])
                    for t, s in ((k_pages, ks), (v_pages, vs)))
            k[hidden[e][:ctx + n]], v[hidden[e][:ctx + n]] = 0.0, 0.0
            s = q[q0:q0 + n, h * hd:(h + 1) * hd].cpu().double() @ k.T * scale
            if slopes is not None:
                s = s - float(slopes[h]) * (pos - j).double()
            seen = (j <= pos) & ~hidden[e][:ctx + n]
            if window:
                seen = seen & (j > pos - window)
            w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            w = torch.where(seen.any(-1, keepdim=True), w, 0.0)
            out[q0:q0 + n, h * hd:(h + 1) * hd] = w @ v
            size[q0:q0 + n, h * hd:(h + 1) * hd] = w @ v.abs()
    return out, size


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("page,block", [(8, 8), (32, 16), (64, 64)])
@pytest.mark.parametrize("window,bias", [(None, False), (None, True), (150, False)])
@pytest.mark.parametrize("splits", [1, 3])
def test_keys_without_a_page_are_hidden_from_portions_and_single_tokens_alike(kind, hd, page, block, window, bias, splits):
    """A table with holes, of no page and of a page beyond the pool, behind the tokens and among them; an entry none of whose pages is there."""
    lens, ctx = [40, 1, 70, 1, 9], [300, 300, 5, 200, 30]
    c = Cache(lens, ctx, 2, hd, page, block, kind, seed=hd + page)
    q = rnd(c.rows, 8 * hd, seed=3, std=1.5)
    slopes = torch.pow(2.0, -torch.arange(1, 9).float() / 2).to(DEV) if bias else None
    hidden = [torch.zeros(400, dtype=torch.bool) for _ in lens]
    table = c.table_host.clone()
    for e in range(len(lens)):
        held = -(-(lens[e] + ctx[e]) // page)
        for i in (range(held) if e == 4 else {1, held // 2, held - 2} - {held - 1}):
            if 0 <= i < held:
                table[e, i] = -1 if (i + e) % 2 else c.k.shape[0] + 1000 * i
                hidden[e][i * page:(i + 1) * page] = True
    c.table = table.to(DEV)
    want, size = attention_with_holes(q, c, 8, window, hd ** -0.5, slopes, hidden)
    # q8_refs' terms: the output's rounding, weights in float16 and their smallest step, the scores' roundings (together below 2^-12 here)
    largest = ref.LARGEST[kind] * 2.0 ** -4
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -12) * size + 2.0 ** -25 * 400 * largest
    single = [c.cu_host[e] for e, n in enumerate(lens) if n == 1]
    many = [r for r in range(c.rows) if r not in single]
    portions = run_prefill(c, q, 8, window, hd ** -0.5, splits, False, slopes)
    check_rows(portions, want, bound)
    check_rows(run_decode(c, q, 8, window, hd ** -0.5, splits, slopes), want, bound, single)
    check_rows(run_prefill(c, q, 8, window, hd ** -0.5, splits, True, slopes), want, bound, many)
    none = list(range(c.cu_host[4], c.cu_host[5]))
    assert bool((portions[none] == 0).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("how", ["zeros", "any", "rising", "falling"])
@pytest.mark.parametrize("portion", [False, True])
def test_every_key_counts_whatever_the_scale_of_its_values(kind, hd, how, portion):
    """Scales of values over their whole range, 2^-100 to 2^100: a key's weight in the denominator has nothing to do with them.  Rows of q of zero (all
    keys alike) and others; the far scales in one warp's keys, in different ones, in different runs."""
    c = Cache([5, 3, 2] if portion else [1, 1, 1], [30, 700, 1500], 2, hd, 16, 16, kind, seed=hd)
    g = torch.Generator().manual_seed(8)
    shape = c.vs.shape
    if how == "zeros":                                       # blocks of zeros, at the least scale, beside blocks of large values
        zero = torch.rand(shape, generator=g) < 0.5
        exps = torch.full(shape, 27.0).masked_fill(zero, -100.0)
        c.v.view(shape + (16, hd)).view(torch.uint8).masked_fill_(zero[..., None, None], 0)
    elif how == "any":
        exps = torch.randint(-100, 101, shape, generator=g).float()
    else:                                                    # along each entry's keys, in a few steps
        exps = torch.zeros(shape)
        for e in range(3):
            held = [p for p in c.table_host[e].tolist() if p >= 0]
            for i, p in enumerate(held):
                x = -100 + 50 * (4 * i // max(1, len(held) - 1))
                exps[p] = x if how == "rising" else -x
    c.dev[1], c.dev[3] = c.v.to(DEV), torch.pow(2.0, exps).to(DEV)
    q = rnd(c.rows, 8 * hd, seed=1, std=1.5)
    q.view(c.rows, 8, hd)[:, ::2] = 0.0
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 8, None, hd ** -0.5)
    assert bool(torch.isfinite(want).all())
    for splits in (1, 2, 7):
        got = (run_prefill if portion else run_decode)(c, q, 8, None, hd ** -0.5, splits)
        check_rows(got, want, bound)


def test_decode_planned_for_short_contexts_serves_long_ones():
    """The number of runs comes from a plan for 1,400 tokens, and stays in a captured graph, while contexts grow to more than four times that."""
    nH, nKV, hd, page, n = 8, 2, 64, 16, 3
    splits = ops().attn_decode_q8_splits(n, nH, nKV, hd, 1400, None, torch.device(DEV, 0))
    assert splits > 1
    c = Cache([1] * n, [6399, 4000, 1], nKV, hd, page, 16, INT8, stride=400, dirty=False)
    q = rnd(n, nH * hd, seed=1)
    out = torch.empty_like(q)
    scratch = torch.full((ops().attn_q8_scratch_floats(n, nH, hd, splits),), math.nan, device=DEV)

    def call():
        ops().attn_decode_q8(q, *c.args(), c.cu, c.ctx_d, out, scratch, n, nH, None, 0.125, splits, 1400)

    call()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    for ctx in ([899, 20, 1], [2000, 899, 0], [6399, 4000, 1]):
        c.ctx = ctx
        c.ctx_d.copy_(torch.tensor(ctx, dtype=torch.int32))
        graph.replay()
        check_rows(out, *ref.attention(q, *c.args(), c.cu_host, ctx, nH, None, 0.125))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens,ctx,window,splits", [([256], [0], None, 2), ([256], [70], None, 5), ([200, 256], [40, 130], None, 6), ([256], [600], 100, 3),
                                                   ([129], [60], None, 4), ([300], [1], None, 7), ([200], [120], None, 2), ([256], [100], None, 3)])
def test_runs_of_keys_that_only_the_second_row_tile_sees(hd, lens, ctx, window, splits):
    """One query head a KV head: a block's first 128 tokens end two key tiles before its last 128 do, so runs begin behind what they see."""
    c = Cache(lens, ctx, 2, hd, 16, 16, E4M3, seed=hd)
    q = rnd(c.rows, 2 * hd, seed=4, std=1.5)
    want, bound = ref.attention(q, *c.args(), c.cu_host, c.ctx, 2, window, hd ** -0.5)
    check_rows(run_prefill(c, q, 2, window, hd ** -0.5, splits), want, bound)
