"""examples/state_space_block.py: the norm, the convolution and the scan together, trained and served."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "state_space_block.py")
    spec = importlib.util.spec_from_file_location("state_space_block", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_block_is_trained_and_serves_what_it_learnt(example):
    losses, worst = example.main(["--steps", "20"])
    assert len(losses) == 20 and all(v == v and abs(v) < 1e6 for v in losses)
    # Outputs of order one, through two blocks whose sums of at most 128 products are off by 128 x 2^-24
    # each way; the orders of summation differ.
    assert worst < 1e-4


def test_gradients_of_the_whole_model(example):
    """The loss's gradient along random directions of each parameter against differences.  Losses of order one
    in 32 bits are off by 2^-22 or so, a step of 2^-8 makes that 2^-15 of the quotient, and its square is left of
    what is cut off; the directions' gradients are of order one."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    model = example.Model(16, 2)
    features, target = example.sample(4, 50, gen)
    lengths = torch.tensor([50, 33, 1, 0], dtype=torch.int32, device="cuda")
    valid = (torch.arange(50, device="cuda") < lengths.unsqueeze(1)).unsqueeze(2)

    def loss():
        outputs, _ = model(features, lengths)
        return torch.where(valid, outputs - target, 0.0).double().square().mean()

    loss().backward()
    for p in model.parameters():
        way = torch.randn(p.shape, generator=gen, device="cuda", dtype=torch.float32) / p.numel() ** 0.5
        along, step = float((p.grad.double() * way).sum()), 2.0 ** -8
        with torch.no_grad():
            p += step * way
            up = float(loss())
            p -= 2 * step * way
            down = float(loss())
            p += step * way
        assert abs((up - down) / (2 * step) - along) < 1e-3 + 1e-2 * abs(along), tuple(p.shape)
