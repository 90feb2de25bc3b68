"""Corners of the operators over a cache in 8 bits that need no GPU to be shown."""
import os
import re

import pytest
import torch

import q8_refs as ref
from neurogrid_b200.csrc import build


def _kernel(source, name):
    """The text of a kernel's body."""
    text = open(os.path.join(build.HERE, source)).read()
    text = re.sub(r"//[^\n]*", "", text)
    return text[text.index(f"\n{name}("):]


def test_tensor_memory_is_taken_after_the_kernels_before_and_before_the_kernels_behind():
    """A block that takes all of an SM's tensor memory must not share the SM with a block that holds some of it and waits for this kernel, or that
    this kernel waits for: its allocation stands behind the wait, and the signal that lets the next kernel in behind the allocation."""
    body = _kernel("attention_q8_sm100.cu", "attn_prefill_q8_sm100_kernel")
    alloc, signal = body.index("tcgen05.alloc"), body.index("ng_pdl_trigger()")
    assert "512" in body[alloc:alloc + 120]
    assert body.rindex("ng_pdl_wait()", 0, alloc) < alloc < body.index("__syncthreads()", alloc) < signal
    # between the last wait in front of the allocation and the allocation nothing returns
    assert "return" not in body[body.rindex("ng_pdl_wait()", 0, alloc):alloc]


def test_room_is_left_for_the_records_of_every_workspace(model_dirs):
    """The page pool is sized from what the workspaces leave: over a cache in 8 bits each of the four holds records of its own."""
    from neurogrid_b200.engine import ModelRunner
    from neurogrid_b200.engine.loading import model_from_dir
    from neurogrid_b200.parts.attention import Q8_SCRATCH_FLOATS
    _, model = model_from_dir(model_dirs["D"], dtype="bfloat16", device="cpu")
    plain = ModelRunner.workspace_reserve(model, 256)
    assert plain == 2 * 256 * model.activation_bytes_per_row() + 2 * ModelRunner.MAX_PORTION_LOGITS_BYTES
    assert ModelRunner.workspace_reserve(model, 256, "e4m3") == plain + 4 * 4 * Q8_SCRATCH_FLOATS


@pytest.mark.parametrize("kind", list(ref.LARGEST))
def test_what_a_value_is_off_by_in_a_block_written_at_once_and_in_one_that_fills_token_by_token(kind):
    """Half a step written at once.  Where the scale grows, codes are rounded again at each new scale: the errors s / 2, s / 4, ... of integers stay below a
    step of the last one, those of e4m3's subnormal codes (half a step is 2^-10 s) below 2^-9 s; some do pass what half a step allows."""
    hd, block, beyond = 32, 16, 0
    table = torch.zeros(1, 1, dtype=torch.int32)
    for seed in range(12):
        g = torch.Generator().manual_seed(seed)
        x = torch.randn(block, hd, generator=g, dtype=torch.float64) * torch.pow(2.0, torch.arange(block).double() * (0.2 + 0.1 * seed))[:, None]
        x[:4] *= torch.rand(4, hd, generator=g, dtype=torch.float64)
        for steps in ([block], [1] * block, [5, 1, 1, 9]):
            values, scale, at = torch.zeros(1, 1, block, hd, dtype=kind), torch.ones(1, 1, 1), 0
            for n in steps:
                v, f = ref.write(x[at:at + n], values, scale, table, [0, n], [at])
                values, scale, at = v.to(kind), f.float(), at + n
            s = float(scale)
            off = (values.double()[0, 0] * s - x).abs()
            if kind == torch.int8:
                once, grown = torch.full_like(off, s / 2), torch.full_like(off, s)
            else:
                once, grown = (x.abs() * 2.0 ** -4).clamp(min=2.0 ** -10 * s), x.abs() * 2.0 ** -4 + 2.0 ** -9 * s
            assert bool((off <= (once if len(steps) == 1 else grown)).all())
            beyond += int((off > once).sum())
    assert beyond > 0
