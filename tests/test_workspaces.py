"""The workspaces that ops keeps for each stream (host logic, on CPU tensors)."""
import pytest
import torch

from anvilq_b200 import ops

CPU = torch.device("cpu")


@pytest.fixture
def kept(monkeypatch):
    """ops without workspaces of its own, its current stream called 7."""
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_outgrown", [])
    monkeypatch.setattr(ops, "_stream_ptr", lambda device: 7)
    return monkeypatch


def test_a_workspace_is_kept_and_zero(kept):
    ws = ops.workspace(CPU, 100)
    assert ws.numel() == 1 << 20 and not ws.any()
    assert ops.workspace(CPU, 1 << 20) is ws and not ops._outgrown


def test_outgrown_workspaces_stay_below_the_newest(kept):
    """Captured graphs may still use them, so they are kept; but sizes that rise step by
    step must not add up."""
    for n in range(1 << 20, 9 << 20, 100_000):
        ws = ops.workspace(CPU, n)
        assert ws.numel() >= n
        assert sum(w.numel() for w in ops._outgrown) < ws.numel()
