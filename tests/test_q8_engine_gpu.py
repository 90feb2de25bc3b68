"""The engine over a cache in 8 bits, and forked requests: one attention layer against what its cache holds, a model against the plain
one with its keys and values rounded the same way, graphs, samples, compaction, the command line."""
import json
import math
import os
import subprocess
import sys

import pytest
import torch

import plain_lfm2
import q8_refs as ref
from helpers import make_ctx, make_runner, rel_err
from neurogrid_b200.cache.storage import EIGHT_BIT_DTYPES
from neurogrid_b200.config.specs import AttentionSpec, DistanceBiasSpec, RopeSpec
from neurogrid_b200.engine import ModelRunner, StepEntry
from neurogrid_b200.engine.loading import model_from_dir
from neurogrid_b200.parts import PagedView
from neurogrid_b200.parts.registry import build
from neurogrid_b200.sampling import SamplingParams
from tiny_configs import PAGE_SIZE

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tokens(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("nH,nKV,hd,window,bias", [(6, 2, 64, None, False), (4, 4, 32, 13, False), (8, 2, 128, None, True)])
def test_attention_part_reads_what_it_wrote(kind, nH, nKV, hd, window, bias):
    """Portions and single tokens through the mixer: its output is the attention of the rotated queries over what the cache holds
    after the step, and the cache holds the rotated keys and the values, off by a code's half step."""
    H, ps, block = 96, 16, 16
    position = DistanceBiasSpec(nH) if bias else RopeSpec(hd, 5000.0, "half")
    part = build("mixer", AttentionSpec(H, nH, nKV, hd, position, qk_norm=not bias, qk_norm_eps=2e-6, window=window),
                 dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(hd)
    w = {n: (torch.randn(d.shape, generator=g) / math.sqrt(d.shape[-1]) if len(d.shape) == 2 else 1 + 0.1 * torch.randn(d.shape, generator=g))
         for n, d in part.tensors().items()}
    part.bind(w)
    dtype = EIGHT_BIT_DTYPES[kind]
    pages, T = 12, 100
    view = PagedView(torch.full((pages, nKV, ps, hd), 0x7f, dtype=torch.uint8, device=DEV).view(dtype),
                     torch.full((pages, nKV, ps, hd), 0x7f, dtype=torch.uint8, device=DEV).view(dtype),
                     torch.randperm(pages, generator=g)[None, :-(-T // ps)].to(torch.int32).to(DEV),
                     k_scales=torch.full((pages, nKV, ps // block), math.nan, device=DEV),
                     v_scales=torch.full((pages, nKV, ps // block), math.nan, device=DEV))
    x = torch.randn(T, H, generator=g).bfloat16().to(DEV)
    xs = x.double().cpu()
    wr = {n: t.bfloat16().double() if t.dim() == 2 else t.double() for n, t in w.items()}
    r = lambda t: t.bfloat16().double()
    q, k, v = (r(xs @ wr[f"{n}_proj.weight"].T).view(T, -1, hd) for n in "qkv")
    if not bias:
        pos = torch.arange(T)
        q, k = plain_lfm2.rmsnorm(q, wr["q_norm.weight"], 2e-6), plain_lfm2.rmsnorm(k, wr["k_norm.weight"], 2e-6)
        q, k = (r(plain_lfm2.rope(t, pos, 5000.0, "half")) for t in (q, k))
    slopes = torch.pow(2.0, -float(position.exponent) * torch.arange(1, nH + 1).double() / nH) if bias else None
    at = 0
    for n in (33, 1, 1, 7, 1, 40, 1, 2, 13, 1):
        ctx = make_ctx([n], [at], [0], dtype=torch.bfloat16)
        y = part.forward(x[at:at + n].contiguous(), ctx, view)
        y = (y.sum(0) if y.dim() == 3 else y).double().cpu()
        at += n
        a, _ = ref.attention(q[at - n:at].reshape(n, -1).bfloat16(), view.k_pages, view.v_pages, view.k_scales, view.v_scales, view.table,
                             [0, n], [at - n], nH, window, hd ** -0.5, slopes)
        want = r(a) @ wr["o_proj.weight"].T
        assert float((y - want).abs().max() / want.abs().max()) < 1.2e-2           # as for the other bfloat16 parts
        assert int(ctx.status) == 0
    assert at == T
    i = torch.arange(T)
    p, s = view.table.cpu()[0].long()[i // ps], i % ps
    for pages_, scales_, true in ((view.k_pages, view.k_scales, k), (view.v_pages, view.v_scales, v)):
        f = scales_.cpu().double()[p, :, s // block][..., None]
        got = pages_.cpu().double()[p, :, s] * f
        # half a code's step (int8: of the block's scale, twice that where a block has grown; e4m3: of the value or of its smallest step),
        # and the bfloat16 roundings of the product in front
        step = f if kind == "int8" else true.abs() * 2.0 ** -4 * 1.02 + 2.0 ** -10 * f
        assert bool(((got - true).abs() <= step + 1.2e-2 * true.abs().max()).all())


def _q8_attention(kind, block, ps):
    """plain_lfm2.attention with keys and values as a cache in 8 bits holds them when the sequence was written at once."""
    def attention(n, wq, wk, wv, wo, q_norm_w, k_norm_w, *, n_heads, n_kv, hd, eps, theta, pairing, positions=None, window=None, rb=False):
        T, r = n.shape[0], plain_lfm2._r
        pos = torch.arange(T)
        q, k, v = (r(n @ m.T, rb).reshape(T, -1, hd) for m in (wq, wk, wv))
        q, k = plain_lfm2.rmsnorm(q, q_norm_w, eps), plain_lfm2.rmsnorm(k, k_norm_w, eps)
        q, k = (r(plain_lfm2.rope(t, pos, theta, pairing), rb) for t in (q, k))
        pages = -(-T // ps)
        held = []
        for t in (k, v):
            codes, f = ref.write(t.reshape(T, -1), torch.zeros(pages, n_kv, ps, hd, dtype=kind), torch.ones(pages, n_kv, ps // block),
                                 torch.arange(pages)[None], [0, T], [0])
            value = codes.view(pages, n_kv, ps // block, block, hd) * f[..., None, None]
            held.append(value.reshape(pages, n_kv, ps, hd).transpose(1, 2).reshape(pages * ps, n_kv, hd)[:T])
        k, v = held
        out = torch.zeros(T, n_heads, hd, dtype=torch.float64)
        for h in range(n_heads):
            s = (q[:, h] @ k[:, h // (n_heads // n_kv)].T) / math.sqrt(hd)
            out[:, h] = torch.softmax(s.masked_fill(pos[None] > pos[:, None], -math.inf), -1) @ v[:, h // (n_heads // n_kv)]
        return r(r(out.reshape(T, -1), rb) @ wo.T, rb)
    return attention


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_a_prompt_read_at_once_matches_plain_with_rounded_keys_and_values(model_dirs, monkeypatch, name, kind):
    cfg, w = plain_lfm2.load_plain(model_dirs[name])
    ps = PAGE_SIZE[name]
    monkeypatch.setattr(plain_lfm2, "attention", _q8_attention(EIGHT_BIT_DTYPES[kind], min(ps, 16), ps))
    _, model = model_from_dir(model_dirs[name], dtype="bfloat16", device=torch.device("cuda:0"))
    runner = ModelRunner(model, num_pages=40, page_size=ps, max_requests=2, max_tokens_per_step=256, cache_dtype=kind)
    for T in (1, 33, 150):
        toks = _tokens(T, cfg["vocab_size"], T)
        got = runner.step([StepEntry("r", toks, list(range(T)))]).clone()
        runner.finish("r")
        # the bound of the bfloat16 tests (2e-2), twice: activations that differ by their roundings put some elements on the other side
        # of a code's border
        assert rel_err(got, plain_lfm2.forward(cfg, w, toks, round_bf16=True)) < 4e-2
    runner.check_status()


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("name", ["B", "D"])
def test_graphs_and_eager_steps_agree(model_dirs, name, kind):
    """The same steps (portions, single tokens, mixed ones, each shape several times) with and without CUDA graphs."""
    cfg, _ = plain_lfm2.load_plain(model_dirs[name])
    logits = []
    for graphs in (True, False):
        _, model = model_from_dir(model_dirs[name], dtype="bfloat16", device=torch.device("cuda:0"))
        runner = ModelRunner(model, num_pages=120, page_size=PAGE_SIZE[name], max_requests=4, max_tokens_per_step=128, cuda_graphs=graphs,
                             max_seq_len=300, cache_dtype=kind)
        seqs = {i: _tokens(200, cfg["vocab_size"], i) for i in range(3)}
        at, got = {i: 0 for i in seqs}, []

        def step(sizes):
            out = runner.step([StepEntry(i, seqs[i][at[i]:at[i] + n], [n - 1]) for i, n in sizes])
            for i, n in sizes:
                at[i] += n
            got.append(out.float().cpu())

        for i in range(3):
            for _ in range(3):
                step([(i, 24)])
        for _ in range(6):
            step([(0, 1), (1, 1), (2, 1)])
        for _ in range(4):
            step([(0, 1), (1, 9), (2, 1)])
        for _ in range(4):
            step([(2, 1)])
        runner.check_status()
        if graphs:
            assert runner.graph_replays > 8
        logits.append(torch.cat(got))
    assert rel_err(logits[0], logits[1]) < 2e-2


def _engine(model_dir, name, **kw):
    from neurogrid_b200 import Engine
    kw.setdefault("page_size", PAGE_SIZE[name])
    kw.setdefault("max_seq_len", 256)
    return Engine(model_dir, **kw)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_engine_generates_over_a_cache_in_8_bits(model_dirs, kind):
    cfg, _ = plain_lfm2.load_plain(model_dirs["D"])
    prompts = [_tokens(n, cfg["vocab_size"], n) for n in (1, 7, 33, 100)]
    eng = _engine(model_dirs["D"], "D", dtype="bfloat16", cache_dtype=kind)
    outs = eng.generate(prompts, max_new_tokens=24)
    assert [len(o) for o in outs] == [24] * 4
    plain = _engine(model_dirs["D"], "D", dtype="bfloat16")
    assert eng.runner.storage.bytes_per_token() * 1.9 < plain.runner.storage.bytes_per_token()
    assert eng.stats()["pages_free"] == [eng.runner.cache.pools[0].num_pages]
    # a pool that preempts recomputes with portions of other sizes: it goes on and ends
    small = _engine(model_dirs["D"], "D", dtype="bfloat16", cache_dtype=kind, num_pages=14, max_tokens_per_step=40, chunk_size=16, max_requests=4)
    assert [len(o) for o in small.generate(prompts, max_new_tokens=40)] == [40] * 4 and small.stats()["preemptions"] > 0


def test_samples_of_a_prompt_equal_requests_of_their_own(model_dirs):
    """Order-fixed float32: what a forked request computes is what it would have computed alone."""
    cfg, _ = plain_lfm2.load_plain(model_dirs["B"])
    prompts = [_tokens(n, cfg["vocab_size"], n) for n in (1, 8, 45)]
    kw = dict(dtype="float32", max_requests=5, max_tokens_per_step=32)
    eng = _engine(model_dirs["B"], "B", **kw)
    got = eng.generate(prompts, max_new_tokens=12, temperature=0.8, top_p=0.9, seed=5, n=3)
    assert eng.stats()["pages_free"] == [eng.runner.cache.pools[0].num_pages]
    alone = _engine(model_dirs["B"], "B", **kw)
    for i, p in enumerate(prompts):
        for j in range(3):
            rid = alone.add_request(p, SamplingParams(temperature=0.8, top_p=0.9, max_new_tokens=12, seed=5), rng_key=3 * i + j)
            alone.run()
            assert alone._requests[rid].output == got[i][j]
    greedy = eng.generate(prompts, max_new_tokens=9, n=2)
    assert greedy == [[o, o] for o in alone.generate(prompts, max_new_tokens=9)]


def test_samples_read_their_prompt_once(model_dirs):
    cfg, _ = plain_lfm2.load_plain(model_dirs["B"])
    eng = _engine(model_dirs["B"], "B", dtype="float32", max_requests=4)
    outs = eng.generate([_tokens(45, cfg["vocab_size"], 45)], max_new_tokens=6, n=4)
    assert [len(o) for o in outs[0]] == [6] * 4
    # all but the prompt's last token once; that token and five of its own for each sample (a token more each where the next step was
    # launched before the last token was read)
    assert 44 + 4 * 6 <= eng.runner.tokens_run <= 44 + 4 * 7


def test_samples_beside_requests_with_ids_of_their_own(model_dirs):
    """An id that a caller has taken is in the way once, as it is for a single request; samples of a prompt that cannot be served all end."""
    cfg, _ = plain_lfm2.load_plain(model_dirs["B"])
    eng = _engine(model_dirs["B"], "B", dtype="float32", max_requests=4, num_pages=4)
    eng.add_request([1, 2, 3], SamplingParams(max_new_tokens=2), request_id=1)
    with pytest.raises(KeyError):
        eng.add_samples([4, 5, 6], 2)
    ids = eng.add_samples([4, 5, 6], 2, SamplingParams(max_new_tokens=2))
    assert sorted(r.id for r in eng.run()) == sorted([1] + ids)
    ids = eng.add_samples(_tokens(60, cfg["vocab_size"], 1), 3)
    done = eng.run()
    assert sorted(r.id for r in done) == ids and all(r.finish_reason == "cache_full" for r in done)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_samples_over_a_cache_in_8_bits(model_dirs, kind):
    """A fork copies codes and scales: greedy samples of one prompt are one token list."""
    cfg, _ = plain_lfm2.load_plain(model_dirs["D"])
    p = _tokens(60, cfg["vocab_size"], 2)
    eng = _engine(model_dirs["D"], "D", dtype="bfloat16", cache_dtype=kind)
    runner = eng.runner
    runner.step([StepEntry("a", p[:37])])
    runner.fork("a", "b")
    for g in range(len(runner.storage.k)):
        for t in runner.storage.pools(g):
            raw = t.view(torch.uint8) if t.element_size() == 1 else t
            ta, tb = runner.cache.table("a", g), runner.cache.table("b", g)
            assert ta[:2] == tb[:2] and ta[2] != tb[2] and torch.equal(raw[:, ta[2]], raw[:, tb[2]])
    out = runner.step([StepEntry("a", p[37:38], [0]), StepEntry("b", p[37:38], [0])]).clone()
    assert rel_err(out[0], out[1]) < 2e-2
    runner.finish("a"); runner.finish("b")
    assert [len(o) for o in eng.generate([p, p[:20]], max_new_tokens=8, temperature=0.9, n=4)[1]] == [8] * 4


def test_compaction_between_steps_changes_nothing(model_dirs):
    cfg, w = plain_lfm2.load_plain(model_dirs["B"])
    runner = make_runner(model_dirs["B"], page_size=8, max_requests=4, device=torch.device("cuda:0"), max_seq_len=120)
    seq = _tokens(60, cfg["vocab_size"], 9)
    runner.step([StepEntry("gap", _tokens(30, cfg["vocab_size"], 1))])
    got = [runner.step([StepEntry("a", seq[:41], list(range(41)))]).clone()]
    for i in range(41, 60):
        if i == 50:
            runner.finish("gap")
            assert runner.compact() > 0
            runner.cache.check()
            assert runner.cache.pools[0].held_pages() == list(range(len(runner.cache.table("a", 0))))
            assert runner.compact() == 0
        got.append(runner.step([StepEntry("a", seq[i:i + 1], [0])]).clone())
    assert rel_err(torch.cat(got), plain_lfm2.forward(cfg, w, seq)) < 2e-5


def test_command_line_takes_a_cache_type(model_dirs):
    cmd = [sys.executable, os.path.join(ROOT, "bin", "neurogrid"), "-model", model_dirs["A"], "-max-seq-len", "128", "-prompt-tokens", "5,17,3",
           "-max-new-tokens", "6", "-cache-dtype", "int8", "-log-level", "error"]
    out = subprocess.run(cmd, capture_output=True, text=True, timeout=600, check=True).stdout
    assert len(json.loads(out.splitlines()[0])["tokens"]) == 6
