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
