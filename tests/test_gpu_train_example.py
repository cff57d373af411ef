"""The training example runs the chunkwise kernels, both norms and the orthogonalised update together: its loss falls
from the uniform one (log 64 = 4.16) past what the last token alone leaves (log 4 = 1.39)."""

import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_loss_falls(gpu_case):
    from train_block import train
    losses = train(steps=60, report=lambda line: print(line, flush=True))
    assert all(v == v for v in losses) and abs(losses[0] - 4.16) < 1.0
    assert losses[-1] < 1.39
