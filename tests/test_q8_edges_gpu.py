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
