"""The example that runs the fine-tuning operators together, as a program would: a head on the engine's descriptors is trained to
several datasets and served for all of them at once."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("adapted_head", os.path.join(ROOT, "examples", "adapted_head.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.gpu
@pytest.mark.parametrize("state_bits", [32, 8])
def test_the_head_learns_and_is_served(example, state_bits):
    first, last, served, (head, descriptors, dataset, system, count) = example.run(steps=150, state_bits=state_bits, quiet=True)
    # (the teacher's corrections are within reach of the adapters: nine tenths of the loss and more go)
    assert last < 0.1 * first
    # one call for the systems of all datasets gives each what a call of its own does, to the roundings of sums in another order: 64
    # terms a number, 40 atoms a system
    with torch.no_grad():
        for i in range(0, count, 5):
            mine = system == i
            alone = head(descriptors[mine], dataset[mine])
            assert abs(float(alone.double().sum()) - float(served[i])) <= 64 * 2.0 ** -24 * float(alone.abs().double().sum()) + 1e-6
