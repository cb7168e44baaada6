"""A launch goes to the device of its tensors, whichever is current. The library
and the devices are stand-ins: this runs without a GPU."""

from __future__ import annotations

import contextlib

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import grid, linear


class Devices:
    """Device `current` of several; records where each entry point was called."""

    def __init__(self):
        self.current, self.calls = 0, []

    @contextlib.contextmanager
    def device(self, index):
        before, self.current = self.current, index
        try:
            yield
        finally:
            self.current = before

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, self.current, int(args[-1])))
            return nat.OK

        return entry


@pytest.fixture
def devices(monkeypatch):
    d = Devices()
    monkeypatch.setattr(nat, "load", lambda: d)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: d.current, raising=False)
    # every device's current stream is its default one
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: d.current)
    monkeypatch.setattr(torch.cuda, "device", d.device)
    return d


def test_a_stream_brings_its_device(devices):
    for index in (0, 1, 2):
        nat.call("mgq_entry", 5, nat.stream_of(torch.device("cuda", index)))
    nat.call("mgq_entry", 5, nat.stream_of(torch.device("cuda")))
    nat.call("mgq_entry", 5, 0)
    assert [c[1] for c in devices.calls] == [0, 1, 2, 0, 0] and devices.current == 0


def test_a_failing_launch_leaves_the_current_device(devices):
    devices.mgq_last_error = lambda: b"refused"
    devices.mgq_entry = lambda *args: nat.ERR_VALUE
    with pytest.raises(ValueError):
        nat.call("mgq_entry", nat.stream_of(torch.device("cuda", 3)))
    assert devices.current == 0


@pytest.mark.parametrize("index", [0, 1])
def test_operators_launch_on_their_tensors_device(devices, monkeypatch, index):
    # (host tensors, said to be of that device)
    dev = torch.device("cpu", index)
    monkeypatch.setattr(linear, "_device", lambda *tensors: dev)
    monkeypatch.setattr(nat, "device_for", lambda *tensors: dev)
    x, w = torch.ones(4, 32, dtype=torch.bfloat16), torch.ones(3, 32, dtype=torch.bfloat16)
    linear.grouped_linear(x, w)
    linear.grouped_linear_dgrad(torch.ones(4, 3, dtype=torch.bfloat16), w)
    q, s = linear.quantize_rows_int8(x)
    linear.int8_linear(q, s, torch.ones(3, 32, dtype=torch.int8), torch.ones(3))
    linear.mxfp_linear(x, torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, 1, dtype=torch.uint8),
                       "mxfp4")
    grid.rtn_quantize_mxfp(w, "mxfp4")
    assert len(devices.calls) == 6 and {c[1] for c in devices.calls} == {index}
    assert devices.current == 0
