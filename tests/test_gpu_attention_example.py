"""The example that takes a ragged batch through the attention operators together."""
import importlib.util
import pathlib

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(hip, dev):
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "ragged_batch.py"
    spec = importlib.util.spec_from_file_location("ragged_batch", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_serving(example):
    """Outputs are averages of values of about unit size (the largest of some ten thousand is below 6): rounded to 8 bits, with
    weights rounded to 8 bits, they are off by at most 2 * 2^-8 of that."""
    assert example.serve() < 2 * 2.0 ** -8 * 6
    assert example.serve(prompt_lengths=(1,), decoded=1) < 2 * 2.0 ** -8 * 6


def test_training(example):
    losses = example.train()
    assert losses[-1] < 0.8 * losses[0]
    assert all(b < a for a, b in zip(losses, losses[1:]))
