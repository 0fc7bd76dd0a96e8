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
    monkeypatch.setattr(ops, "_of_graphs", set(), raising=False)
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


def test_an_eager_call_does_not_use_a_graphs_workspace(kept):
    """Memory of a captured graph is zeroed by its replays alone: eager calls on the same
    stream get a workspace of their own, and captures then share that."""
    kept.setattr(ops, "_capturing", lambda device: True)
    of_graph = ops.workspace(CPU, 100)
    assert ops.workspace(CPU, 100) is of_graph
    of_graph.fill_(1)                       # as memory that no replay has zeroed
    kept.setattr(ops, "_capturing", lambda device: False)
    for call in (lambda: ops.workspace(CPU, 100), lambda: ops._call_workspace(CPU, 100, None)):
        ws = call()
        assert ws is not of_graph and not ws.any()
    assert any(w is of_graph for w in ops._outgrown), "the graph still uses it"
    assert ops.workspace(CPU, 100) is ws
    kept.setattr(ops, "_capturing", lambda device: True)
    assert ops.workspace(CPU, 100) is ws


def test_the_first_serving_call_does_not_use_a_graphs_workspace(kept):
    kept.setattr(ops, "_capturing", lambda device: True)
    of_graph = ops.workspace(CPU, 100)
    kept.setattr(ops, "_capturing", lambda device: False)
    assert ops._call_workspace(CPU, 100, None) is not of_graph
