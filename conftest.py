"""pytest: figures of the GPU's allocator are read when the autograd engine's threads are done.

A backward pass wakes its caller before the engine's thread has dropped its own references to
the results; the last of them frees a tensor, under the interpreter's lock.  A caller
that drops the results and reads the allocator at once then counts a gradient that
nothing holds (seen in one of four runs of all GPU tests, and never in one that lets the thread run).
What is still held after a moment is counted as before."""
from __future__ import annotations

import time

import pytest


@pytest.fixture(autouse=True)
def _engine_threads_are_done(request, monkeypatch):
    if request.node.get_closest_marker("gpu") is None:
        return
    import torch

    read = torch.cuda.memory_allocated

    def memory_allocated(*args, **kwargs):
        time.sleep(0.005)  # (the lock is free meanwhile)
        return read(*args, **kwargs)

    monkeypatch.setattr(torch.cuda, "memory_allocated", memory_allocated)
