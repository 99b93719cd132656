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


SHAPES = [("experts_mlp", (8, 64, 4096, 1024)), ("experts_mlp", (2, 8, 512, 4096)), ("experts_mlp", (1, 1024, 16, 16)),
          ("linear_adapters", (4096, 4096, 16, 4)), ("linear_adapters", (6144, 4096, 32, 40)),
          ("linear_adapters", (4096, 12288, 64, 6))]


@pytest.mark.parametrize("op, shape", SHAPES)
def test_one_workspace_serves_every_batch_up_to_its_rows(mod, op, shape):
    """Sized for the largest batch, no smaller one asks for more: the need is not
    monotone in the rows."""
    rows = 2000 if shape[0] < 16 else 1100
    size = getattr(_lib.lib(), f"w8a8_{op}_workspace_bytes")
    needs = [size(m, *shape) for m in range(1, rows + 1)]
    most = getattr(LoadedModule, f"{op}_workspace_bytes")(rows, *shape)
    assert most == max(needs) > 0
    mod.reserve_workspace(most)
    for m in range(1, rows + 1):
        mod._routed_workspace(None, f"w8a8_{op}_workspace_bytes", m, *shape)
    assert not mod._retired


def test_sizes_for_no_rows_and_refused_shapes():
    assert LoadedModule.experts_mlp_workspace_bytes(0, 8, 64, 4096, 1024) == 0
    assert LoadedModule.experts_mlp_workspace_bytes(4, 8, 64, 4096, 1000) == 0
    assert LoadedModule.linear_adapters_workspace_bytes(0, 4096, 4096, 16, 4) == 0
    assert LoadedModule.linear_adapters_workspace_bytes(8, 4096, 4096, 12, 4) == 0


def test_sizes_kept_by_shape_stay_bounded(mod):
    """A server's batches have any number of rows: the sizes kept do not grow with them."""
    for m in range(1, 6000):
        ptr, nbytes = mod._routed_workspace(None, "w8a8_linear_adapters_workspace_bytes", m, 64, 64, 8, 2)
        assert nbytes >= _lib.lib().w8a8_linear_adapters_workspace_bytes(m, 64, 64, 8, 2)
    assert len(mod._routed_bytes) <= 4096
