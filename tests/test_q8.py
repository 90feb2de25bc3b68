"""What the operators over a cache in 8 bits refuse, and their arithmetic's plain statement (no GPU)."""
import ctypes
import struct

import numpy as np
import pytest
import torch

import q8_refs as ref
from neurogrid_b200.csrc import build, ops

E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def cache(pages=4, n_kv=2, page=16, hd=32, block=8, kind=E4M3):
    return [torch.zeros(pages, n_kv, page, hd, dtype=kind), torch.zeros(pages, n_kv, page, hd, dtype=kind),
            torch.ones(pages, n_kv, page // block), torch.ones(pages, n_kv, page // block), torch.zeros(2, 3, dtype=torch.int32)]


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def write(k=None, v=None, c=None, row_entry=None, cu=None, ctx=None, status=None):
    k = torch.zeros(3, 64, dtype=torch.bfloat16) if k is None else k
    ops.cache_write_q8(k, torch.zeros_like(k) if v is None else v, *(c or cache()), i32(0, 0, 1) if row_entry is None else row_entry,
                       i32(0, 2, 3) if cu is None else cu, i32(0, 5) if ctx is None else ctx, i32(0) if status is None else status)


@pytest.mark.parametrize("kw,why", [
    (dict(), "CUDA"),                                                         # nothing wrong but the place
    (dict(k=torch.zeros(3, 63, dtype=torch.bfloat16)), "do not fit the pages"),
    (dict(k=torch.zeros(3, 64, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(v=torch.zeros(3, 64)), "do not fit the pages"),
    (dict(c=cache(kind=torch.bfloat16)), "8 bits"),
    (dict(c=cache(kind=torch.uint8)), "8 bits"),
    (dict(c=cache(block=4)), "at least 8"),
    (dict(c=cache(page=24, block=8)), "powers of two"),
    (dict(c=cache(hd=24)), "multiples of 16"),
    (dict(c=cache()[:3] + cache(block=16)[3:]), "scales"),
    (dict(c=cache()[:2] + [torch.ones(4, 2, 2, dtype=torch.float64)] * 2 + cache()[4:]), "float32"),
    (dict(c=cache()[:4] + [torch.zeros(2, 3, dtype=torch.int64)]), "int32"),
    (dict(c=cache()[:4] + [torch.zeros(1, 3, dtype=torch.int32)]), "batch description"),
    (dict(row_entry=i32(0, 0)), "batch description"),
    (dict(cu=i32(0, 3)), "batch description"),
    (dict(status=torch.zeros(1)), "int32"),
])
def test_write_refuses(kw, why):
    with pytest.raises(ops.KernelError, match=why):
        write(**kw)


@pytest.mark.parametrize("kw,why", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros(3, 64)), "bfloat16"),
    (dict(q=torch.zeros(3, 65, dtype=torch.bfloat16)), "q is bfloat16"),
    (dict(qkv=torch.zeros(3, 128, dtype=torch.bfloat16)), "expected"),
    (dict(qkv=torch.zeros(2, 3, 192, dtype=torch.bfloat16)), "float32"),
    (dict(positions=i32(0, 0)), "do not fit"),
    (dict(inv_freq=torch.ones(8)), "do not fit"),
    (dict(weight=torch.ones(31)), "do not fit"),
    (dict(weight=torch.ones(32, dtype=torch.float64)), "float32"),
    (dict(c=cache(kind=torch.bfloat16)), "8 bits"),
])
def test_rope_and_write_refuses(kw, why):
    with pytest.raises(ops.KernelError, match=why):
        ops.rope_cache_q8(kw.get("qkv", torch.zeros(3, 192, dtype=torch.bfloat16)), kw.get("q", torch.zeros(3, 64, dtype=torch.bfloat16)),
                          kw.get("weight"), None, kw.get("inv_freq"), True, 1.0, *kw.get("c", cache()), kw.get("positions", i32(0, 5, 9)),
                          i32(0, 1, 1), 2, 1e-5, i32(0))


def attend(fn, q=None, out=None, c=None, heads=4, splits=1, scratch=None, n=2, cu=None, **kw):
    q = torch.zeros(3, 128, dtype=torch.bfloat16) if q is None else q
    out = torch.zeros_like(q) if out is None else out
    args = (q, *(c or cache()), i32(0, 2, 3) if cu is None else cu, i32(0, 5), out)
    if fn == "decode":
        ops.attn_decode_q8(*args, scratch, n, heads, None, 1.0, splits, 16, kw.get("slopes"))
    else:
        ops.attn_prefill_q8(*args, n, 2, heads, None, 1.0, False, kw.get("slopes"), scratch, splits)


@pytest.mark.parametrize("fn", ["decode", "portion"])
@pytest.mark.parametrize("kw,why", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros(3, 128)), "bfloat16"),
    (dict(out=torch.zeros(3, 128)), "bfloat16"),
    (dict(q=torch.zeros(3, 96, dtype=torch.bfloat16)), "shapes"),
    (dict(heads=3, q=torch.zeros(3, 96, dtype=torch.bfloat16)), "shapes"),
    (dict(c=cache(hd=272), q=torch.zeros(3, 4 * 272, dtype=torch.bfloat16)), "above 256"),
    (dict(splits=2), "scratch"),
    (dict(splits=2, scratch=torch.zeros(2 * 4 * 2 * 36 - 1)), "scratch"),
    (dict(splits=2, scratch=torch.zeros(10000, dtype=torch.float64)), "scratch"),
    (dict(splits=0), "runs"),
    (dict(n=3), "batch description"),
    (dict(cu=i32(0, 2)), "batch description"),
    (dict(c=cache(kind=torch.bfloat16)), "8 bits"),
])
def test_attention_refuses(fn, kw, why):
    with pytest.raises(ops.KernelError, match=why):
        attend(fn, **kw)


def test_copy_refuses():
    pool = torch.zeros(2, 9, 4)
    for pools, src, dst, why in (([pool], [0], [1], "CUDA"), ([pool], [0, 1], [2], "as many"), ([pool], [0.5], [1.5], "whole"),
                                 ([pool], [[0]], [[1]], "whole"), ([pool, torch.zeros(2, 8, 4)], [0], [1], "CUDA|same pages"),
                                 ([torch.zeros(9)], [0], [1], "same pages"), ([pool], [2 ** 40], [1], "page number"), ([pool], [-(2 ** 40)], [1], "page number")):
        with pytest.raises(ops.KernelError, match=why):
            ops.copy_pages(pools, src, dst)


def test_the_copy_launcher_checks_every_page_number_before_it_launches():
    """The library's own answer for lists that it must not launch (there is no GPU here to launch on)."""
    f = build.load("cache_q8").ng_copy_pages
    f.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_char_p, ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p]

    def call(src, dst, pages=(50, 40)):
        pools = b"".join(struct.pack("@Pq2i", 4096, 64, 2, p) for p in pages)
        a, b = np.asarray(src, dtype=np.int32), np.asarray(dst, dtype=np.int32)
        return f(pools, len(pages), a.tobytes(), b.tobytes(), len(a), None)

    assert call([], []) == 0
    many = list(range(20))
    for src, dst in (([0], [0]), ([0], [40]), ([45], [1]), ([-1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), (many, many[::-1]),
                     (many, list(range(19, 39))), (many, [25] * 20), (many, [39] * 19 + [40])):
        assert call(src, dst) == 6, (src, dst)


@pytest.mark.parametrize("kind", [E4M3, INT8])
def test_the_plain_write(kind):
    """The statement that the kernel is held to: nearest codes at the least scale, old codes carried along."""
    top = ref.LARGEST[kind]
    for x, e in ((top, 0), (top * 2, 1), (top * 1.001, 1), (0.0, -100), (1e-40, -100), (3e38, 120 if kind == E4M3 else 100)):
        assert ref.exponent(x, kind) == min(e, 100)
    x = torch.randn(4, 32, generator=torch.Generator().manual_seed(1))
    values, factors = ref.write(x, torch.zeros(2, 1, 8, 32, dtype=kind), torch.ones(2, 1, 1), torch.tensor([[1]]), [0, 4], [0])
    back = values[1, 0, :4] * factors[1, 0, 0]
    step = 2.0 ** -4 * x.abs().double() + 2.0 ** -10 * factors[1, 0, 0] if kind == E4M3 else 0.5 * factors[1, 0, 0]
    assert bool(((back - x.double()).abs() <= step).all()) and float(values[0].abs().max()) == 0.0
    assert float(values.abs().max()) * 2 > top and float(values.abs().max()) <= top
