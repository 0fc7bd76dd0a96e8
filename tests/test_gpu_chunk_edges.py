"""Chunk attention at the edges of what it accepts: outputs on any 16 bytes.

Tolerances and cases' makers: ``test_gpu_chunk``."""
import pytest
import torch

from anvilq_b200 import ops
from test_gpu_chunk import Case, dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("first", [8, 16, 24, 40])
def test_outputs_on_any_16_bytes(dev, first, D):
    """An output inside a larger buffer, of pairs that one CTA has and of shared ones; nothing beside it is written."""
    c = Case(dev, 40 + first, [20, 4000, 0], [150, 9, 300], 8, 2, D, 16, spare=2)
    want = c.run(out=torch.full((len(c.q), 8, D), 7.0, dtype=torch.float16, device=dev))
    c.check(want)
    room = torch.full((want.numel() + 64,), 5.0, dtype=torch.float16, device=dev)
    out = room[first:first + want.numel()].view(want.shape)
    out[c.starts_list[-1]:] = 7.0
    assert out.data_ptr() % 16 == 0
    c.run(out=out)
    ops.raise_device_errors(dev)
    assert torch.equal(out, want)
    assert (room[:first] == 5.0).all() and (room[first + want.numel():] == 5.0).all()
