"""The stream's workspace under LoadedModule (no GPU): what it keeps as calls
grow, with buffers that count their bytes in place of device memory."""
from __future__ import annotations

import pytest

from inferrous_amd import _lib, module
from inferrous_amd.module import LoadedModule


class Counted:
    ptr = 0x10000

    def __init__(self, n, dtype):
        self.nbytes = n


@pytest.fixture
def mod(monkeypatch):
    monkeypatch.setattr(module, "DeviceBuffer", Counted)
    return LoadedModule(None)


def test_outgrown_workspaces_stay_bounded(mod):
    """A batch that creeps up one row at a time: what is held for graphs captured
    earlier never exceeds the workspace in use, and that never twice the need."""
    need = 0
    for m in range(1, 1025):
        need = max(need, _lib.lib().w8a8_experts_mlp_workspace_bytes(m, 8, 64, 4096, 1024))
        ptr, nbytes = mod._routed_workspace(None, "w8a8_experts_mlp_workspace_bytes", m, 8, 64, 4096, 1024)
        assert need <= nbytes < 2 * need + 16
        assert sum(b.nbytes for b in mod._retired) <= nbytes


def test_a_first_workspace_is_what_was_asked_for(mod):
    mod.reserve_workspace(1000)
    assert mod._gemm_ws[None].nbytes == 1008 and not mod._retired


def test_growth_without_the_memory_for_it_takes_the_need(mod, monkeypatch):
    """Where twice the last workspace cannot be had, the call's own need still can."""
    mod.reserve_workspace(1600)

    class Full(Counted):
        def __init__(self, n, dtype):
            if n > 2000:
                raise module.W8A8Error(2, "malloc")
            super().__init__(n, dtype)

    monkeypatch.setattr(module, "DeviceBuffer", Full)
    mod.reserve_workspace(1700)
    assert mod._gemm_ws[None].nbytes == 1712
