"""CPU tests of the device and stream that an output-head call runs on."""
import types

import pytest

from mxs_sampler import head


def test_a_stream_of_another_device_is_refused(monkeypatch):
    """Its outputs would be allocated, and its kernels launched, on the stream's device
    and not the operands'."""
    monkeypatch.setattr(head.torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="cuda:1"):
        head._on(0, types.SimpleNamespace(device_index=1))
    with pytest.raises(ValueError, match="cuda:0"):
        head._on(1, types.SimpleNamespace(device_index=0))


def test_the_operands_stream_is_taken(monkeypatch):
    monkeypatch.setattr(head.torch.cuda, "current_device", lambda: 0)
    assert head._on(0, None) is head._HERE
    assert head._on(0, types.SimpleNamespace(device_index=0)) is not head._HERE
    assert head._on(1, None) is not head._HERE
