"""Beam selection at the edges of what it accepts: values that are not finite among masked ones,
rows of no elements, log sums of rows that do not average.

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


def test_reorder_of_empty_rows(dev):
    """A search's first step: histories of no tokens among other states, or alone, given outputs or not."""
    parents = torch.tensor([[1, 0, -1], [2, 2, 1]], dtype=torch.int32, device=dev)
    scores = torch.arange(6, device=dev).reshape(2, 3).float()
    history, wide = (torch.empty((2, 3, *rest), dtype=torch.int32, device=dev) for rest in ((0,), (4, 0)))
    a, b, c = ops.beam_reorder([history, scores, wide], parents)
    assert a.shape == (2, 3, 0) and a.dtype == torch.int32 and c.shape == (2, 3, 4, 0)
    assert b.tolist() == [[1, 0, 0], [5, 5, 4]]
    assert ops.beam_reorder([history], parents)[0].shape == (2, 3, 0)
    out = torch.empty((2, 3, 0), dtype=torch.int32, device=dev)
    assert ops.beam_reorder([history], parents, outs=[out])[0] is out
    with pytest.raises(ValueError):
        ops.beam_reorder([history, torch.zeros((2, 4), device=dev)], parents)      # another K all the same
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("kind", ["two", "three", "ten", "rising", "steep"])
def test_scores_of_rows_that_do_not_average(dev, kind, half):
    """Rows of a few live logits, and rows whose largest so far moves with every tile: the log sums are within
    3e-6 + 2^-23 d + 4e-7 V / 4096, which include/anvilq.h states, the scores within half a step more."""
    V = 151936
    g = torch.Generator(device=dev)
    g.manual_seed(len(kind))
    x = torch.full((3, 4, V), -float("inf"), device=dev)
    if kind in ("rising", "steep"):
        x[:] = torch.arange(V, device=dev) * ((1 if kind == "rising" else 30) / V)
        x += torch.rand((3, 4, 1), generator=g, device=dev)
    else:
        n = {"two": 2, "three": 3, "ten": 10}[kind]
        for b in range(3):
            for k in range(4):
                at = torch.randperm(V, generator=g, device=dev)[:n]
                x[b, k, at] = torch.randn(n, generator=g, device=dev) * 2 ** (b - 1) + 5 * k
    x = x.half() if half else x
    scores = -torch.rand((3, 4), generator=g, device=dev) * 10
    tokens, parents, new, *_ = ops.beam_select(x, scores, 8)
    ops.raise_device_errors(dev)
    y = x.double()
    top = y.amax(dim=2, keepdim=True)
    e = torch.exp(y - top)
    total = e.sum(dim=2)
    d = torch.where(e > 0, e * (top - y), 0.0).sum(dim=2) / total
    lse = top[..., 0] + torch.log(total)
    for b in range(3):
        for i in range(8):
            if int(tokens[b, i]) < 0:
                continue
            k = int(parents[b, i])
            want = float(scores[b, k].double() + y[b, k, int(tokens[b, i])] - lse[b, k])
            bound = 3e-6 + 2.0 ** -23 * float(d[b, k]) + 4e-7 * V / 4096 + 2.0 ** -24 * abs(want)
            assert abs(float(new[b, i]) - want) <= bound, (b, i, float(new[b, i]) - want, bound)
