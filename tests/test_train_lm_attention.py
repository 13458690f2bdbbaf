"""The sequence model of the training command: it runs, every parameter has a gradient that follows the loss, and its bits do not depend on
the device."""
import pytest
import torch

import bit_reproducible_training_amd as rg
from bit_reproducible_training_amd import train_lm

SMALL = dict(vocab=12, width=16, blocks=2, batch=40, heads=4, length=10, dropout=0.1)


def test_it_runs_and_repeats_itself():
    losses, h = train_lm.train("cpu", 3, **SMALL)
    assert len(losses) == 3 and train_lm.train("cpu", 3, **SMALL) == (losses, h)
    assert train_lm.train("cpu", 3, **{**SMALL, "sandwich": True, "kind": "rms"})[1] != h


def test_every_gradient_is_the_loss_s_slope():
    """Moving all parameters by a step along a direction changes the loss by the gradients' product with it: within a hundredth and float32's
    noise of the loss over the step."""
    torch.manual_seed(1)
    model = train_lm.SequenceModel(12, 16, 4, 2)
    rg.set_slices(3)
    symbols = torch.tensor(train_lm.text(44, 12)).view(4, 11)
    model(symbols).backward()
    for name, p in model.named_parameters():
        assert p.grad is not None, name
        direction = torch.randn(p.shape)
        slope, step = (p.grad.double() * direction).sum().item(), 2.0 ** -7
        ends = []
        with torch.no_grad():
            for sign in (1, -1):
                p.add_(direction, alpha=sign * step)
                ends.append(model(symbols).double().item())
                p.add_(direction, alpha=-sign * step)
        found = (ends[0] - ends[1]) / (2 * step)
        scale = (p.grad.double().norm() * direction.double().norm()).item()
        assert abs(found - slope) <= 0.01 * scale + 2.0 ** -19 / step + 40 * step ** 2, (name, found, slope)


@pytest.mark.gpu
def test_a_gpu_gives_the_cpu_parameters():
    for extra in ({}, dict(sandwich=True, kind="rms", state_bits=8)):
        assert train_lm.train("cuda", 3, **{**SMALL, **extra}) == train_lm.train("cpu", 3, **{**SMALL, **extra})
