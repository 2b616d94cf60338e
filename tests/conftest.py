import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run on the GPU box with -m gpu)")


def _runs_beside(stream, a):
    """Whether work on ``stream`` leaves the current stream alone (streams share a few hardware queues)."""
    import torch
    start, there, here = (torch.cuda.Event(enable_timing=True) for _ in range(3))
    torch.cuda.synchronize()
    start.record()
    stream.wait_event(start)
    with torch.cuda.stream(stream):
        for _ in range(4):
            torch.mm(a, a)
        there.record()
    a[0, 0].clone()
    here.record()
    torch.cuda.synchronize()
    return start.elapsed_time(here) < 0.5 * start.elapsed_time(there)


@pytest.fixture(autouse=True)
def _next_stream_runs_beside(request):
    """For a test that needs its next ``torch.cuda.Stream()`` to run beside the current one (parameter ``neighbour``): streams come from a pool in turn, so
    which one is next depends on the tests before.  Goes once round the pool and on to the place before one that does."""
    if "neighbour" not in request.fixturenames or request.node.get_closest_marker("gpu") is None:
        return
    import torch
    a = torch.zeros(8192, 8192, dtype=torch.bfloat16, device="cuda")
    torch.mm(a, a)
    drawn = [torch.cuda.Stream()]
    while len(drawn) < 64:
        s = torch.cuda.Stream()
        if s.cuda_stream == drawn[0].cuda_stream:
            break
        drawn.append(s)
    else:
        return                                               # (no pool: every stream is a new one)
    # the last draw was the pool's first stream again: drawn[1] is the next
    beside = next((i for i, s in enumerate(drawn) if i > 0 and _runs_beside(s, a)), None)
    if beside is not None:
        for _ in range(beside - 1):
            torch.cuda.Stream()
