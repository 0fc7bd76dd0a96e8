"""Beam selection at the edges of what it accepts: values that are not finite among masked ones.

Tolerances and the definition: ``test_gpu_beam``."""
import pytest
import torch

from anvilq_b200 import AnvilqError, ops
from test_gpu_beam import check, dev, inputs  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("V,at,left", [
    (1, 0, []), (2, 1, []), (7, 3, [5]), (9000, 0, []), (9001, 9000, []), (9001, 9000, [3, 17]), (9001, 4500, [9000]),
    (40000, 33333, [1, 2, 39999]), (151936, 151935, [70000])])
def test_bad_values_among_masked_ones_are_reported(dev, V, at, left, bad, half):
    """A row that a grammar leaves next to nothing of, and a logit of NaN or +inf in it: it counts as
    masked, and is reported though no finite logit lies near it."""
    x, scores, *_ = inputs(V + at, 2, 2, V, half, dev)
    keep = x[1, 0].clone()
    x[1, 0] = -float("inf")
    x[1, 0, left] = keep[left]
    clean = x.clone()
    x[1, 0, at] = bad
    got = ops.beam_select(x, scores, 6)
    with pytest.raises(AnvilqError, match="nonfinite"):
        ops.raise_device_errors(dev)
    check(clean, scores, 6, got=got)
    ops.beam_select(clean, scores, 6)
    ops.raise_device_errors(dev)             # masks alone are no error
