import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a HIP device (MI355X); run with -m gpu")


def gpu_available() -> bool:
    import torch

    return torch.cuda.is_available()


@pytest.fixture(scope="session")
def dev():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda", 0)


@pytest.fixture(autouse=True)
def _memory_when_autograd_has_let_go(request, monkeypatch):
    """torch.cuda.memory_allocated in tests that measure it: autograd's device thread drops its own references to a call's
    results and graph only after it has woken the caller, so a reading right behind the call may still count them (torch's
    own operations alone: 1 of 3000 readings, 69 on a busy host).  The thread takes its tasks in order: when it has done
    another small one, they are gone."""
    import inspect

    if request.node.get_closest_marker("gpu") is None or "memory_allocated" not in inspect.getsource(request.module):
        return
    import torch

    measure = torch.cuda.memory_allocated

    def settled(*args, **kw):
        t = torch.ones(1, device="cuda", requires_grad=True)
        torch.autograd.grad(t * 2, t)
        return measure(*args, **kw)

    monkeypatch.setattr(torch.cuda, "memory_allocated", settled)
