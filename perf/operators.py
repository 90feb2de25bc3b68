"""The operators of a cache that holds keys and values in 8 bits, case by case: its writer, the attention that reads it
(single tokens, prompt portions), and the copying of pages.

The cache.  ``k_pages`` and ``v_pages`` [pages, KV heads, page, head] hold codes, e4m3 or int8; ``k_scales`` and ``v_scales``
[pages, KV heads, page / block] hold a power of two for each block of tokens and head, and a code c stands for c * scale.  A
request's token t lies in page ``table[request, t // page]`` at place ``t % page``.

``write``: new keys and values (rows, in request order) join what their requests hold.  A block's scale is the least power of
two (2^-100 .. 2^100) with which its largest finite value fits the type (448, 127); a block that already holds tokens of its request
keeps its scale if that is the larger one, otherwise those tokens' codes are rounded to the new scale.  Codes are rounded to
nearest, ties to even.
``decode`` / ``portion``: softmax(q k^T * scale - slope * distance) v over the keys at or before a row's position, within a window if
there is one; query head h reads KV head h // (heads / KV heads).
``copy``: pages of every layer of a cache, codes and scales, to other pages.

A case's fields: ``op``; ``requests``; ``tokens`` (new tokens of a request) and ``context`` (tokens before them), each that of the longest
request (``ragged``: the others have a quarter of it and more); ``heads`` (query heads), ``kv``, ``dim``; ``page``, ``block``; ``cache``
(type of the codes), ``dtype`` (type of q, or of the keys and values written); ``window`` (0: none), ``slopes``; for copies
``layers``, ``pool`` (pages of a layer) and ``pages`` (those copied).
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"
_TYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8, "bfloat16": torch.bfloat16, "float32": torch.float32}
_LARGEST = {"e4m3": 448.0, "int8": 127.0}
_LOWEST_EXP, _HIGHEST_EXP = -100, 100


# ------------------------------------------------------------------------------------------------ cases
def _case(op, name=None, **kw):
    base = dict(op=op, requests=1, tokens=1, context=0, ragged=False, heads=32, kv=8, dim=64, page=16, block=16, cache="e4m3",
                dtype="bfloat16", window=0, slopes=False, layers=1, pool=0, pages=0)
    base.update(kw)
    return dict(base, name=name) if name else base


def listed():
    return [
        # a decode step of a full server: one key and value of each of 64 requests, most of them into begun blocks
        _case("write", "write-step", requests=64, context=4000, ragged=True),
        # a prompt of 2,048 tokens, read in one step
        _case("write", "write-prompt", tokens=2048),
        # portions of odd lengths behind begun blocks, from a 32-bit model with wide heads into 8-bit integers
        _case("write", "write-ragged", requests=5, tokens=611, context=1001, ragged=True, kv=4, dim=128, page=32, block=16, cache="int8",
              dtype="float32"),
        # the next token behind a short question: latency
        _case("decode", "decode-one", context=299, heads=16),
        # the headline: a batch of 8 behind prompts of 2,048 tokens
        _case("decode", "decode-8", requests=8, context=2100),
        # a full server: 64 requests of differing lengths up to 4,096 tokens, codes in integers
        _case("decode", "decode-64", requests=64, context=4095, ragged=True, cache="int8"),
        # documents: two requests behind 131,072 tokens, wide heads, large pages
        _case("decode", "decode-long", requests=2, context=131071, dim=128, page=64),
        # time to the first token of one ordinary long prompt
        _case("portion", "portion-2048", tokens=2048),
        # portions of odd lengths behind contexts of odd lengths, a window, a distance bias, wide heads, integers
        _case("portion", "portion-ragged", requests=6, tokens=611, context=1500, ragged=True, heads=16, kv=4, dim=128, page=32,
              block=32, cache="int8", window=1024, slopes=True),
        # a document's later portion: 512 tokens behind 32,768
        _case("portion", "portion-long", tokens=512, context=32768, heads=24),
        # a prompt's samples begin: the last, partly filled page of four requests, every layer, codes and scales
        _case("copy", "copy-fork", layers=6, pool=1024, pages=4),
        # a pool is packed: 4,096 of its pages move into gaps
        _case("copy", "copy-compact", layers=6, pool=10240, pages=4096),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: an operator with sizes of its own."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    while True:
        op = rng.choice(("write", "decode", "decode", "portion", "portion", "copy"))
        kv = rng.choice((1, 2, 4, 8))
        page = rng.choice((8, 16, 16, 32, 64))
        kw = dict(kv=kv, heads=kv * rng.choice((1, 2, 3, 4, 4, 8)), dim=rng.choice((64, 64, 128, 80, 256)), page=page,
                  block=rng.choice([b for b in (8, 16, 32, 64) if b <= page]), cache=rng.choice(("e4m3", "int8")),
                  ragged=rng.random() < 0.6)
        if op == "copy":
            pool = _log(rng, 64, 10240)
            kw.update(layers=rng.choice((1, 2, 6, 8)), pool=pool, pages=_log(rng, 1, pool * 2 // 5),
                      cache=rng.choice(("e4m3", "int8", "bfloat16", "float32")), heads=kv, ragged=False)
        elif op == "write":
            kw.update(dtype=rng.choice(("bfloat16", "float32")), requests=_log(rng, 1, 64), context=_log(rng, 1, 4096) - 1,
                      tokens=1 if rng.random() < 0.5 else _log(rng, 2, 2048))
        else:
            kw.update(requests=_log(rng, 1, 64) if op == "decode" else _log(rng, 1, 8),
                      tokens=1 if op == "decode" else _log(rng, 2, 2048), context=_log(rng, 1, 131072 if op == "decode" else 32768) - 1,
                      window=rng.choice((0, 0, 0, 128, 1024, 4096)), slopes=rng.random() < 0.3)
        c = _case(op, **kw)
        if _cost(c) <= most[op] and _held(c) <= 4 << 30 and c not in [{k: v for k, v in x.items() if k != "name"} for x in listed()]:
            return c


def _lengths(case):
    """[(new tokens, tokens before them)] of the requests."""
    n = case["requests"]
    if not case["ragged"]:
        return [(case["tokens"], case["context"])] * n
    share = [1.0 if i == 0 else 0.25 + 0.75 * (i * 0.6180339887 % 1.0) for i in range(n)]
    other = [1.0 if i == 0 else 0.25 + 0.75 * (i * 0.7548776662 % 1.0) for i in range(n)]
    return [(max(1, round(case["tokens"] * a)), round(case["context"] * b)) for a, b in zip(share, other)]


def _pool_pages(case):
    if case["op"] == "copy":
        return case["pool"]
    return sum(-(-(t + c) // case["page"]) for t, c in _lengths(case)) + 3


def _held(case):
    """Bytes of the cache."""
    esz = torch.empty((), dtype=_TYPES[case["cache"]]).element_size()
    return 2 * case["layers"] * _pool_pages(case) * case["kv"] * (case["page"] * case["dim"] * esz + 4 * case["page"] // case["block"])


def _pairs_seen(case):
    """(row, key) pairs a query head computes, and the keys of the cache that at least one row sees."""
    w, pairs, keys = case["window"], 0, 0
    for n, c in _lengths(case):
        if not w:
            pairs += n * c + n * (n + 1) // 2
            keys += n + c
        else:
            pairs += sum(min(w, c + i + 1) for i in range(n))
            keys += n + min(c, w - 1)
    return pairs, keys


def work(case):
    """Bytes: each input read once, each output written once.  Flops: two products over the visible pairs."""
    kv, dim, page, block = case["kv"], case["dim"], case["page"], case["block"]
    if case["op"] == "copy":
        quant = case["cache"] in _LARGEST
        esz = torch.empty((), dtype=_TYPES[case["cache"]]).element_size()
        of_page = 2 * kv * (page * dim * esz + (4 * page // block if quant else 0))
        return {"bytes": 2 * case["layers"] * case["pages"] * of_page, "flops": 0}
    esz = torch.empty((), dtype=_TYPES[case["dtype"]]).element_size()
    rows = sum(n for n, _ in _lengths(case))
    if case["op"] == "write":
        blocks = sum((c + n - 1) // block - c // block + 1 for n, c in _lengths(case))
        return {"bytes": 2 * kv * (rows * dim * (esz + 1) + 4 * blocks), "flops": 0}
    pairs, keys = _pairs_seen(case)
    return {"bytes": 2 * kv * (keys * dim + 4 * (keys / block)) + 2 * rows * case["heads"] * dim * esz,
            "flops": 4 * case["heads"] * dim * pairs}


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 200


# ------------------------------------------------------------------------------------------------ inputs
def _codes(shape, kind, gen):
    x = torch.randn(shape, generator=gen, device=DEVICE)
    if kind == "e4m3":
        return (x * 90.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    if kind == "int8":
        return (x * 36.0).round_().clamp_(-127.0, 127.0).to(torch.int8)
    return x.to(_TYPES[kind])


def _scales(shape, kind, gen):
    at = -7 if kind == "e4m3" else -6
    return torch.pow(2.0, torch.randint(at - 1, at + 2, shape, generator=gen, device=DEVICE).float())


def _inputs(case, seed):
    """What a user's program holds before the call, without its plan."""
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed) * 7919 + 11)
    host = torch.Generator().manual_seed(int(seed) * 104729 + 5)
    kv, dim, page, block, kind = case["kv"], case["dim"], case["page"], case["block"], case["cache"]
    layers, pages = case["layers"], _pool_pages(case)
    s = {"case": case}
    if case["op"] == "copy":
        lead = (layers, pages, kv)
        s["pools"] = [_codes(lead + (page, dim), kind, gen) for _ in range(2)]
        if kind in _LARGEST:
            s["pools"] += [_scales(lead + (page // block,), kind, gen) for _ in range(2)]
        order = torch.randperm(pages, generator=host)[:2 * case["pages"]].to(torch.int32)
        s["src"], s["dst"] = order[:case["pages"]].numpy().copy(), order[case["pages"]:].numpy().copy()
        return s
    lengths = _lengths(case)
    held = [-(-(n + c) // page) for n, c in lengths]
    order = torch.randperm(pages, generator=host).tolist()
    table = torch.full((len(lengths), max(held)), -1, dtype=torch.int32)
    for i, n in enumerate(held):
        table[i, :n] = torch.tensor(order[sum(held[:i]):sum(held[:i + 1])], dtype=torch.int32)
    news = [n for n, _ in lengths]
    rows = sum(news)
    s["lengths"] = lengths
    s["pages_of"] = [table[i, :n].long().to(DEVICE) for i, n in enumerate(held)]
    s["table"] = table.to(DEVICE)
    s["cu_q"] = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32).to(DEVICE)
    s["ctx_before"] = torch.tensor([c for _, c in lengths], dtype=torch.int32).to(DEVICE)
    s["row_entry"] = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(news)).to(torch.int32).to(DEVICE)
    s["status"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    s["k_pages"], s["v_pages"] = (_codes((pages, kv, page, dim), kind, gen) for _ in range(2))
    s["k_scales"], s["v_scales"] = (_scales((pages, kv, page // block), kind, gen) for _ in range(2))
    dtype = _TYPES[case["dtype"]]
    if case["op"] == "write":
        # keys with a few large channels and heads of differing sizes, as projections leave them
        size = torch.exp(0.8 * torch.randn(1, kv, 1, generator=gen, device=DEVICE))
        channel = torch.ones(1, 1, dim, device=DEVICE)
        channel[..., ::17] = 6.0
        s["k"] = (torch.randn(rows, kv, dim, generator=gen, device=DEVICE) * size * channel).to(dtype).view(rows, kv * dim)
        s["v"] = (torch.randn(rows, kv, dim, generator=gen, device=DEVICE) * size).to(dtype).view(rows, kv * dim)
        return s
    s["q"] = (1.5 * torch.randn(rows, case["heads"] * dim, generator=gen, device=DEVICE)).to(dtype)
    s["scale"] = dim ** -0.5
    s["slopes"] = (torch.pow(2.0, -8.0 * torch.arange(1, case["heads"] + 1, device=DEVICE).float() / case["heads"])
                   if case["slopes"] else None)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] in ("decode", "portion"):
        s["out"] = torch.empty_like(s["q"])
        if own:
            from neurogrid_b200.csrc import ops
            heads, kv, dim, window = case["heads"], case["kv"], case["dim"], case["window"] or None
            s["longest"] = max(n + c for n, c in s["lengths"])
            if case["op"] == "decode":
                s["splits"] = ops.attn_decode_q8_splits(len(s["lengths"]), heads, kv, dim, s["longest"], window, DEVICE)
            else:
                s["splits"] = ops.attn_prefill_q8_splits([n for n, _ in s["lengths"]], heads, kv, dim, s["longest"], window, DEVICE)
            floats = ops.attn_q8_scratch_floats(s["q"].shape[0], heads, dim, s["splits"])
            s["scratch"] = torch.empty(floats, dtype=torch.float32, device=DEVICE) if floats else None
    return s


# ------------------------------------------------------------------------------------------------ the passes
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from neurogrid_b200.csrc import ops
    c = s["case"]
    if c["op"] == "copy":
        ops.copy_pages(s["pools"], s["src"], s["dst"])
        return s["pools"]
    cache = (s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"])
    if c["op"] == "write":
        ops.cache_write_q8(s["k"], s["v"], *cache, s["row_entry"], s["cu_q"], s["ctx_before"], s["status"])
        return list(cache[:4])
    n, window = len(s["lengths"]), c["window"] or None
    if c["op"] == "decode":
        ops.attn_decode_q8(s["q"], *cache, s["cu_q"], s["ctx_before"], s["out"], s["scratch"], n, c["heads"], window, s["scale"],
                           s["splits"], s["longest"], s["slopes"])
    else:
        ops.attn_prefill_q8(s["q"], *cache, s["cu_q"], s["ctx_before"], s["out"], n, max(t for t, _ in s["lengths"]), c["heads"], window,
                            s["scale"], False, s["slopes"], s["scratch"], s["splits"])
    return s["out"]


def _run_plain(s):
    c = s["case"]
    if c["op"] == "copy":
        src, dst = (torch.from_numpy(s[x]).long().to(DEVICE) for x in ("src", "dst"))
        for pool in s["pools"]:
            raw = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
            raw[:, dst] = raw[:, src]
        return s["pools"]
    if c["op"] == "write":
        for x, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
            row = 0
            for i, (n, ctx) in enumerate(s["lengths"]):
                _write_plain(x[row:row + n].float(), pages, scales, s["pages_of"][i], ctx, c)
                row += n
        return [s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]]
    row, dim, kv, group = 0, c["dim"], c["kv"], c["heads"] // c["kv"]
    for i, (n, ctx) in enumerate(s["lengths"]):
        first = max(0, ctx - c["window"] + 1) if c["window"] else 0        # the first key that a row of the request sees
        p0 = first // c["page"]
        keys = [(p[s["pages_of"][i][p0:]].float().unflatten(2, (-1, c["block"])) * f[s["pages_of"][i][p0:]][..., None, None])
                .flatten(2, 3).transpose(0, 1).flatten(1, 2) for p, f in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"]))]
        k, v = (t[:, :n + ctx - p0 * c["page"]] for t in keys)
        at_k = torch.arange(p0 * c["page"], n + ctx, device=DEVICE)
        for a in range(0, n, 256):
            b = min(n, a + 256)
            q = s["q"][row + a:row + b].float().view(b - a, kv, group, dim).permute(1, 2, 0, 3)
            score = torch.matmul(q, k[:, None].transpose(2, 3)) * s["scale"]
            gap = torch.arange(ctx + a, ctx + b, device=DEVICE)[:, None] - at_k[None]
            if s["slopes"] is not None:
                score -= s["slopes"].view(kv, group, 1, 1) * gap.float()
            seen = (gap >= 0) & ((gap < c["window"]) if c["window"] else True)
            score.masked_fill_(~seen, float("-inf"))
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.matmul(p, v[:, None]) / p.sum(-1, keepdim=True)
            s["out"][row + a:row + b] = o.permute(2, 0, 1, 3).reshape(b - a, -1).to(s["out"].dtype)
        row += n
    return s["out"]


def _write_plain(x, pages, scales, table, ctx, c):
    """One request's new keys (or values) x [n, KV heads * dim] behind ``ctx`` tokens."""
    page, block, kv, dim, kind = c["page"], c["block"], c["kv"], c["dim"], c["cache"]
    n, b0 = x.shape[0], ctx // block
    blocks = (ctx + n - 1) // block - b0 + 1
    lead = ctx - b0 * block                                                # tokens of the first block that are already there
    new = torch.zeros(blocks * block, kv, dim, device=DEVICE)
    new[lead:lead + n] = x.view(n, kv, dim)
    new = new.view(blocks, block, kv, dim)
    at = torch.arange(b0, b0 + blocks, device=DEVICE) * block
    ids, place = table[at // page], at % page
    top = torch.where(torch.isfinite(new), new.abs(), torch.zeros_like(new)).amax((1, 3))          # [blocks, KV heads]
    m, e = torch.frexp(top)
    fits = 0.875 if kind == "e4m3" else 127.0 / 128.0                      # 448 = 0.875 * 2^9, 127 = (127 / 128) * 2^7
    e = torch.where(m <= fits, e, e + 1) - (9 if kind == "e4m3" else 7)
    e = torch.where(top > 0, e, torch.full_like(e, _LOWEST_EXP)).clamp(_LOWEST_EXP, _HIGHEST_EXP)
    old = torch.frexp(scales[ids, :, place // block])[1] - 1
    if lead:
        e[0] = torch.maximum(e[0], old[0])
    codes = _to_codes(torch.ldexp(new.double(), -e[:, None, :, None]), kind)
    slots = place[:, None] + torch.arange(block, device=DEVICE)
    held = pages[ids[:, None], :, slots] if kind == "int8" else pages.view(torch.uint8)[ids[:, None], :, slots].view(pages.dtype)
    flat = held.view(torch.uint8).clone().view(blocks * block, kv, dim)
    if lead:
        was = held[0, :lead].double()
        flat[:lead] = _to_codes(torch.ldexp(was, (old[0] - e[0])[None, :, None]), kind).view(torch.uint8)
    flat[lead:lead + n] = codes.view(torch.uint8).view(blocks * block, kv, dim)[lead:lead + n]
    pages.view(torch.uint8)[ids[:, None], :, slots] = flat.view(blocks, block, kv, dim)
    scales[ids, :, place // block] = torch.ldexp(torch.ones_like(top), e)


def _to_codes(x, kind):
    if kind == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127.0, 127.0).to(torch.int8)
    # a value of at most 448 in 64 bits has at most the bits of the 32-bit input behind its leading one: .float() is exact here
    return x.clamp(-448.0, 448.0).float().to(torch.float8_e4m3fn)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    """The same outputs by the definition, one head (or one block) at a time, in 64 bits."""
    s = _inputs(case, seed)
    c = case
    if c["op"] == "copy":
        for pool in s["pools"]:
            raw = pool.view(torch.uint8) if pool.element_size() == 1 else pool
            taken = {int(d): int(f) for f, d in zip(s["src"], s["dst"])}
            for layer in raw:
                was = layer.clone()
                layer.copy_(torch.index_select(was, 0, torch.tensor([taken.get(i, i) for i in range(layer.shape[0])], device=DEVICE)))
        return s["pools"]
    if c["op"] == "write":
        return _exact_write(s)
    if _pairs_seen(c)[0] * c["heads"] * c["dim"] > 4e11:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    group, dim, row = c["heads"] // c["kv"], c["dim"], 0
    for i, (n, ctx) in enumerate(s["lengths"]):
        total = n + ctx
        token = torch.arange(total, device=DEVICE)
        page_of, place = s["pages_of"][i][token // c["page"]], token % c["page"]
        for g in range(c["kv"]):
            k, v = (p[:, g].view(torch.uint8)[page_of, place].view(p.dtype).double() * f[page_of, g, place // c["block"]].double()[:, None]
                    for p, f in ((s["k_pages"], s["k_scales"]), (s["v_pages"], s["v_scales"])))
            for h in range(g * group, (g + 1) * group):
                for a in range(0, n, 1024):
                    b = min(n, a + 1024)
                    q = s["q"][row + a:row + b, h * dim:(h + 1) * dim].double()
                    away = torch.arange(ctx + a, ctx + b, device=DEVICE)[:, None] - token[None, :]
                    z = q @ k.t() * s["scale"]
                    if s["slopes"] is not None:
                        z = z - float(s["slopes"][h]) * away.double()
                    hidden = away < 0
                    if c["window"]:
                        hidden |= away >= c["window"]
                    z[hidden] = -math.inf
                    out[row + a:row + b, h * dim:(h + 1) * dim] = torch.softmax(z, -1) @ v
        row += n
    return out


def _grid(kind):
    """The values of the codes, ascending, and which of them are even (the side that a tie goes to)."""
    if kind == "int8":
        v = torch.arange(-127, 128, dtype=torch.float64)
        return v.to(DEVICE), (v % 2 == 0).to(DEVICE)
    half = [((8 if e else 0) + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127]
    v = [-x for x in reversed(half[1:])] + half
    even = [i % 2 == 0 for i in reversed(range(1, 127))] + [i % 2 == 0 for i in range(127)]
    return torch.tensor(v, dtype=torch.float64, device=DEVICE), torch.tensor(even, device=DEVICE)


def _nearest(x, grid, even):
    """Values of the grid that are nearest to x (within its ends)."""
    x = x.clamp(float(grid[0]), float(grid[-1]))
    hi = torch.searchsorted(grid, x.contiguous()).clamp(1, grid.numel() - 1)
    lo = hi - 1
    below, above = x - grid[lo], grid[hi] - x
    return torch.where((below < above) | ((below == above) & even[lo]), grid[lo], grid[hi])


def _exact_write(s):
    c = s["case"]
    page, block, kv, dim, kind = c["page"], c["block"], c["kv"], c["dim"], c["cache"]
    grid, even = _grid(kind)
    done = []
    for x, pages, scales in ((s["k"], s["k_pages"], s["k_scales"]), (s["v"], s["v_pages"], s["v_scales"])):
        value, factor = pages.double(), scales.double()
        row = 0
        for i, (n, ctx) in enumerate(s["lengths"]):
            x64 = x[row:row + n].double().view(n, kv, dim)
            row += n
            for b in range(ctx // block, (ctx + n - 1) // block + 1):
                lo, hi = max(ctx, b * block), min(ctx + n, (b + 1) * block)
                p, at = int(s["pages_of"][i][b * block // page]), b * block % page
                part = x64[lo - ctx:hi - ctx]                              # [tokens, KV heads, dim]
                top = part.abs().amax((0, 2))
                e = torch.ceil(torch.log2(top / _LARGEST[kind]))
                e = torch.where(torch.exp2(e - 1) * _LARGEST[kind] >= top, e - 1, e)          # log2 may be off by its last place
                e = torch.where(torch.exp2(e) * _LARGEST[kind] < top, e + 1, e).clamp(_LOWEST_EXP, _HIGHEST_EXP)
                f = torch.exp2(e)
                if lo > b * block:                                         # begun: tokens of the request lie in front
                    f = torch.maximum(f, factor[p, :, at // block])
                    ratio = factor[p, :, at // block] / f
                    front = value[p, :, at:at + lo - b * block]
                    value[p, :, at:at + lo - b * block] = _nearest(front * ratio[:, None, None], grid, even)
                value[p, :, at + lo - b * block:at + hi - b * block] = _nearest((part / f[:, None]).transpose(0, 1), grid, even)
                factor[p, :, at // block] = f
        done.append((value if kind == "e4m3" else value.to(torch.int64), factor))
    return [done[0][0], done[1][0], done[0][1], done[1][1]]
