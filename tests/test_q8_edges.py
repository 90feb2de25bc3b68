"""Corners of the operators over a cache in 8 bits that need no GPU to be shown."""
import os
import re

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
