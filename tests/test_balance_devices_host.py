"""Balance loss of tensors that are not on the thread's current device (no GPU: the library and the device are stand-ins)."""
import contextlib
import types

import pytest
import torch


@pytest.mark.parametrize("want_grad", [False, True])
def test_workspace_size_is_asked_for_on_the_tensors_device(monkeypatch, want_grad):
    """The size depends on the current device's number of SMs, so it is asked for where the launch will be."""
    from muxi_native_layout_kernels_b200 import balance, w4
    now, asked, launched = [3], [], []

    @contextlib.contextmanager
    def device(d):
        before, now[0] = now[0], d
        yield
        now[0] = before

    def size(*a):
        asked.append(now[0])
        return 512

    def launch(*a):
        launched.append(now[0])
        return 0

    monkeypatch.setattr(torch.cuda, "device", device)
    for mod in (balance, w4):
        monkeypatch.setattr(mod, "_device_of_thread", lambda: now[0], raising=False)
    monkeypatch.setattr(w4, "_stream_of", lambda d: None)
    monkeypatch.setattr(balance, "lib", types.SimpleNamespace(mlk_router_balance_workspace_bytes=size, mlk_router_balance_loss=launch))
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)      # get_device() is -1, another than the current one
    balance._loss(x, ids, 0, 1.0, None, None, want_grad)
    assert launched == [-1] and asked == [-1] and now == [3]
    now[0] = -1                                                           # the device is current already
    balance._loss(x, ids, 0, 1.0, None, None, want_grad)
    assert launched == [-1, -1] and asked == [-1, -1]
