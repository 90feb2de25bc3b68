"""What the workspaces of an engine over a cache in 8 bits hold, beside what the engine leaves for them."""
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
