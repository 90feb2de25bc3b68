"""Corners of the engine over a cache in 8 bits: what its workspaces hold, and steps whose keys are cut into runs."""
import pytest
import torch

import plain_lfm2
from neurogrid_b200 import Engine
from neurogrid_b200.engine import ModelRunner, StepEntry
from neurogrid_b200.parts.attention import Q8_SCRATCH_FLOATS
from tiny_configs import PAGE_SIZE

pytestmark = pytest.mark.gpu


def test_the_workspaces_hold_no_more_records_than_room_is_left_for(model_dirs):
    """Steps of every kind: eager, single tokens, portions, mixed ones, each from its graph."""
    cfg, _ = plain_lfm2.load_plain(model_dirs["D"])
    eng = Engine(model_dirs["D"], dtype="bfloat16", cache_dtype="e4m3", page_size=PAGE_SIZE["D"], max_seq_len=2048, max_requests=4)
    r = eng.runner
    seq = torch.randint(0, cfg["vocab_size"], (900,), generator=torch.Generator().manual_seed(1)).tolist()
    at = {i: 0 for i in range(3)}

    def step(*sizes):
        r.step([StepEntry(i, seq[at[i]:at[i] + n], [n - 1]) for i, n in sizes])
        for i, n in sizes:
            at[i] += n

    step((0, 700), (1, 20))
    for _ in range(3):
        step((2, 20))
        step((0, 1), (1, 1), (2, 1))
        step((0, 1), (1, 9))
    r.check_status()
    spaces = [w for w in (r.ws, r._graph_ws, r._portion_ws, r._mixed_ws) if w is not None]
    held = [t for w in spaces for k, t in w._bufs.items() if k[0] == "attn_q8_scratch"]
    assert len(spaces) == 4 and len(held) >= 3 and all(t.numel() <= Q8_SCRATCH_FLOATS for t in held)
    reserve = ModelRunner.workspace_reserve(eng.model, 2048, "e4m3") - ModelRunner.workspace_reserve(eng.model, 2048)
    assert sum(4 * t.numel() for t in held) <= reserve


def test_steps_behind_long_contexts_cut_their_keys_into_runs_eager_and_replayed(model_dirs, monkeypatch):
    """Single tokens behind thousands of tokens, alone and beside a portion (one scratch for both kernels), and a portion behind more than 8,192: each
    plans several runs, and gives what a runner without graphs gives."""
    from neurogrid_b200.csrc import ops
    from neurogrid_b200.engine.loading import model_from_dir
    runs = {"attn_decode_q8": set(), "attn_prefill_q8": set()}
    for name in runs:
        def call(*a, _f=getattr(ops, name), _seen=runs[name], _at=14 if name == "attn_decode_q8" else 17, **kw):
            _seen.add(a[_at])
            return _f(*a, **kw)
        monkeypatch.setattr(ops, name, call)
    cfg, _ = plain_lfm2.load_plain(model_dirs["D"])
    seqs = [torch.randint(0, cfg["vocab_size"], (9300,), generator=torch.Generator().manual_seed(i)).tolist() for i in range(2)]
    logits = []
    for graphs in (True, False):
        _, model = model_from_dir(model_dirs["D"], dtype="bfloat16", device=torch.device("cuda:0"))
        r = ModelRunner(model, num_pages=1200, page_size=16, max_requests=4, max_tokens_per_step=2048, max_seq_len=9400, cache_dtype="int8",
                        cuda_graphs=graphs)
        at, got = [0, 0], []

        def step(*sizes):
            out = r.step([StepEntry(i, seqs[i][at[i]:at[i] + n], [n - 1]) for i, n in sizes])
            for i, n in sizes:
                at[i] += n
            got.append(out.float().cpu())

        for _ in range(4):
            step((0, 2048))
        for _ in range(4):                                     # behind 8,192 and more: from the third on a replayed graph
            step((0, 40))
        step((1, 300))
        for _ in range(4):
            step((0, 1), (1, 1))
        for _ in range(4):
            step((0, 1), (1, 30))
        r.check_status()
        assert not graphs or r.graph_replays >= 6
        logits.append(torch.cat(got))
    assert max(runs["attn_decode_q8"]) > 1 and max(runs["attn_prefill_q8"]) > 1
    err = float((logits[0] - logits[1]).abs().max() / logits[1].abs().max())
    assert err < 2e-2                                          # as for the other steps of a bfloat16 model, with graphs and without
