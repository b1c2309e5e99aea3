"""examples/answer_descent.py: rows and projections trained together by the losses and the
orthogonalised updates; both losses fall and the preferred answers win."""
from __future__ import annotations

import importlib.util
import math

import pytest

from tests.conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_returned():
    """What torch's allocator keeps of these tests' tensors goes back: other tests read its statistics."""
    yield
    import gc

    import torch
    gc.collect()
    torch.cuda.empty_cache()


def test_example_trains(cuda):
    spec = importlib.util.spec_from_file_location("answer_descent", ROOT / "examples" / "answer_descent.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    history = example.run(steps=6, pairs=4, seed=3)
    again = example.run(steps=6, pairs=4, seed=3)
    assert all(math.isfinite(x) for values in history.values() for x in values)
    # before the first step policy and reference agree: h = 0 up to the rounding of two sums
    assert abs(history["preference"][0] - math.log(2.0)) < 1e-3
    assert history["preference"][-1] < history["preference"][0] and history["margin"][-1] > 0.0
    assert history["policy"][-1] < history["policy"][0]
    assert history["preference"][0] == again["preference"][0]
