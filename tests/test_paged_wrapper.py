"""The Python wrappers of the paged-cache calls, without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("code,kept", [(0, True), (601, False), (602, False), (603, False), (301, False)])
@pytest.mark.parametrize("clear", [True, False])
def test_workspaces_are_dropped_after_any_status(monkeypatch, code, kept, clear):
    """A 601 may hide behind an earlier code: the status word holds the first one."""
    from yllm_b200 import attn

    def call(name, st, clear_arg):
        assert name == "yattn_device_status" and clear_arg == int(clear)
        st._obj.value = code

    ws = {(0, 0, 128): torch.zeros(1)}
    monkeypatch.setattr(attn, "call", call)
    monkeypatch.setattr(attn, "_paged_ws", ws)
    assert attn.device_status(clear=clear) == code
    assert bool(ws) == kept
