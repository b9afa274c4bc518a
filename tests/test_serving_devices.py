"""Serving operators on tensors of a device that is not the current one: every
launch is made on the tensors' device, since a default stream's handle names that
of whichever device is current. Without a GPU, by watching the launches."""
import contextlib

import pytest
import torch

from neuralzip_amd import _native
from neuralzip_amd.gpu import serving

OTHER = torch.device("cuda", 1)


@pytest.fixture
def launches(monkeypatch):
    """(function, current device) of every launch; device 0 is current."""
    seen, current, real = [], [0], _native.lib()

    class Library:
        def __getattr__(self, name):
            def launch(*args):
                seen.append((name, current[0]))
                return 0
            return launch if name in ("nz_pages_extend", "nz_pages_release", "nz_pages_trim", "nz_attention_plan", "nz_attention",
                                      "nz_shared_plan", "nz_shared_attention") else getattr(real, name)

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d.index
        yield
        current[0] = before
    monkeypatch.setattr(_native, "lib", lambda library=Library(): library)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(serving, "_stream_handle", lambda device, stream: 0)
    return seen


def test_pages_are_launched_on_their_device(launches):
    book = serving.PageTables(3, 4, 16, 8, device="cpu")
    numbers = torch.zeros(3, dtype=torch.int32)
    for device, index in ((OTHER, 1), (torch.device("cuda", 0), 0)):
        book.device, launches[:] = device, []
        step = serving.Step(3, 3, "cpu")
        book.extend(numbers, 3, out=step)
        assert launches == [("nz_pages_extend", index)]
    with pytest.raises(ValueError, match="on the GPU"):
        book.device = torch.device("cpu")
        book.extend(numbers, 3, out=step)


def plan_of(kind, rows, **more):
    plan = object.__new__(kind)
    for name, value in dict(rows=rows, heads=2, kv_heads=1, device=OTHER, _index=-1, _target=4, _parts=1, capacity=8,
                            items=torch.zeros(8, 8, dtype=torch.int32), _scratch={}, _stream=0, **more).items():
        setattr(plan, name, value)
    return plan


def test_plans_and_attention_are_launched_on_their_device(launches):
    contexts, q, caches = torch.ones(2, dtype=torch.int32), torch.zeros(2, 2, 64), [torch.zeros(3, 1, 16, 64) for _ in range(2)]
    tables, lib = torch.zeros(2, 1, dtype=torch.int32), _native.lib()
    plans = [plan_of(serving.AttentionPlan, 2, _pointers=(0, 0), _format=_native.ATTENTION, _function=lib.nz_attention),
             plan_of(serving.SharedPlan, 2, _pointers=(0, 0, 0), _groups=None, _format=_native.SHARED_ATTENTION,
                     _function=lib.nz_shared_attention)]
    for plan in plans:
        plan._partials = lambda head_dim, handle, stream: 0
        plan.update(contexts)
        serving.paged_attention(q, *caches, tables, plan)
    assert launches == [("nz_attention_plan", 1), ("nz_attention", 1), ("nz_shared_plan", 1), ("nz_shared_attention", 1)]


def test_errors_leave_the_device_as_it_was(launches):
    def refused(*args):
        return -1
    with pytest.raises(Exception):
        serving._launch(refused, OTHER, b"", 0)
    assert torch._C._cuda_getDevice() == 0
