"""The example's training run: it learns, and its bits are the same on every run, with any number of CPU
threads and on the GPU."""
import os
import subprocess
import sys

import pytest

from bit_reproducible_training_amd import train_lm

SMALL = dict(steps=6, vocab=24, context=3, width=32, blocks=2, batch=96)


@pytest.mark.parametrize("bits", [8, 32])
def test_runs_are_the_same_bits(bits, monkeypatch):
    first = train_lm.train("cpu", state_bits=bits, sandwich=True, **SMALL)
    monkeypatch.setenv("REPRO_CPU_THREADS", "3")
    assert train_lm.train("cpu", state_bits=bits, sandwich=True, **SMALL) == first


def test_it_learns():
    losses, _ = train_lm.train("cpu", 25, vocab=16, context=2, width=32, blocks=1, batch=128)
    assert losses[-1] < 0.75 * losses[0]  # from ln 16 = 2.77


def test_command():
    out = subprocess.run([sys.executable, "-m", "bit_reproducible_training_amd.train_lm", "--device", "cpu", "--steps", "2",
                          "--vocab", "12", "--width", "16", "--batch", "32", "--kind", "rms"], check=True,
                         capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    lines = out.stdout.split("\n")
    assert lines[0].startswith("step   0  loss ") and lines[2].startswith("parameters ")


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("kind,sandwich", [("layer", False), ("rms", True)])
def test_the_gpu_gives_the_cpu_bits(bits, kind, sandwich):
    settings = dict(SMALL, state_bits=bits, kind=kind, sandwich=sandwich)
    assert train_lm.train("cuda", **settings) == train_lm.train("cpu", **settings)
