"""examples/sequence_block.py: the norm and the recurrence together, trained and served."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_block_learns_and_serves_what_it_learnt():
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "sequence_block.py")
    spec = importlib.util.spec_from_file_location("sequence_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, worst = example.main(["--steps", "100", "--channels", "64"])
    # The memory's own mean square is about 0.5: what a model without one is left with.
    assert sum(losses[-8:]) / 8 < 0.5 * sum(losses[:8]) / 8
    # Outputs of order one, through two blocks whose sums of 64 products are off by 64 x 2^-24 at
    # most each way; the orders of summation differ.
    assert worst < 1e-4


def test_block_runs_whatever_the_default_type():
    """Its values and buffers are float32 where torch makes other tensors by default."""
    import torch

    path = os.path.join(os.path.dirname(__file__), "..", "examples", "sequence_block.py")
    spec = importlib.util.spec_from_file_location("sequence_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    want, worst = example.main(["--steps", "3", "--channels", "64"])
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        losses, other = example.main(["--steps", "3", "--channels", "64"])
    finally:
        torch.set_default_dtype(before)
    # The same sums in the same types; a library product may order them anew.
    assert abs(losses[0] - want[0]) <= 1e-5 * want[0] and worst < 1e-4 and other < 1e-4
