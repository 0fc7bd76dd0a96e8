"""Frequencies of scaled rotations, and arguments that the appends with a caller's frequencies refuse (CPU)."""
import ctypes
import math

import pytest
import torch

from anvilq_b200 import _lib, ops
from test_serving_refusals import APPEND, APPEND_Q8, EALIGN, EINVAL, ESHAPE, FAKE, ODD, at

INV = at(1 << 26)


def with_rope(base):
    """The rope call's arguments in order: theta gives way to inv_freq, rotary_dim, interleaved, factor."""
    a = {}
    for key, value in base.items():
        if key == "theta":
            a.update(inv=INV, rot=64, pairs=0, factor=1.0)
        else:
            a[key] = value
    return a


ROPE, ROPE_Q8 = with_rope(APPEND), with_rope(APPEND_Q8)


@pytest.mark.parametrize("name,base", [("anvilq_paged_kv_append_rope", ROPE),
                                       ("anvilq_paged_kv_append_q8_rope", ROPE_Q8)])
@pytest.mark.parametrize("status,change", [
    *((EINVAL, c) for c in (
        dict(inv=None), dict(pairs=2), dict(pairs=-1), dict(factor=0.0), dict(factor=-1.0), dict(factor=float("nan")),
        dict(factor=float("inf")), dict(factor=65537.0), dict(qkv=None), dict(err=None), dict(flags=2), dict(Hq=9),
        dict(inv=at(1 << 24)), dict(inv=at((1 << 24) + 8184)))),      # frequencies among what is written
    *((ESHAPE, c) for c in (dict(rot=0), dict(rot=8), dict(rot=24), dict(rot=144), dict(rot=-16), dict(D=96))),
    *((EALIGN, c) for c in (dict(inv=at((1 << 26) + 4)), dict(qkv=ODD))),
])
def test_refused_before_launch(name, base, status, change):
    a = {**base, "k": at(1 << 27), "v": at(1 << 28), **change}
    if "ks" in a:
        a.update(ks=at(1 << 29), vs=at(1 << 30))
    assert getattr(_lib.load(), name)(*a.values()) == status


def test_no_tokens_is_no_work():
    assert _lib.load().anvilq_paged_kv_append_rope(*{**ROPE, "k": at(1 << 27), "v": at(1 << 28), "T": 0}.values()) == 0


@pytest.mark.parametrize("more,error", [
    (dict(inv_freq=torch.ones(32)), ValueError),                                  # fp32
    (dict(inv_freq=torch.ones(4, 8, dtype=torch.float64)), ValueError),
    (dict(inv_freq=torch.ones(64, dtype=torch.float64)[::2]), ValueError),
    (dict(inv_freq=torch.ones(12, dtype=torch.float64)), ValueError),             # 24 dims
    (dict(inv_freq=torch.ones(40, dtype=torch.float64)), ValueError),             # more than a head has
    (dict(interleaved=True), ValueError), (dict(rope_factor=1.5), ValueError),    # without frequencies
])
def test_front_end(more, error):
    qkv, ints = torch.zeros((5, 512), dtype=torch.float16), lambda *s: torch.zeros(s, dtype=torch.int32)
    pool = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    codes, scales = torch.zeros((4, 2, 16, 64), dtype=torch.int8), torch.zeros((4, 2, 1))
    with pytest.raises(error):
        ops.paged_kv_append(qkv, pool, pool.clone(), ints(2, 3), ints(2), ints(3), 4, **more)
    with pytest.raises(error):
        ops.paged_kv_append_q8(qkv, codes, codes.clone(), scales, scales.clone(), ints(2, 3), ints(2), ints(3), 4,
                               **more)


def test_frequencies():
    """The published formulas, restated one pair at a time."""
    R, theta, s, n = 64, 1e4, 8.0, 4096
    plain = [theta ** (-2.0 * i / R) for i in range(R // 2)]
    inv, factor = ops.rope_frequencies(R, theta, device="cpu")
    assert inv.tolist() == plain and factor == 1.0 and inv.dtype == torch.float64
    inv, factor = ops.rope_frequencies(R, theta, dict(kind="linear", factor=s), "cpu")
    assert inv.tolist() == [f / s for f in plain] and factor == 1.0
    inv, factor = ops.rope_frequencies(R, theta, dict(kind="ntk", factor=s), "cpu")
    assert inv[0] == 1.0 and math.isclose(inv[-1], plain[-1] / s, rel_tol=1e-12) and factor == 1.0
    inv, factor = ops.rope_frequencies(R, theta, dict(kind="yarn", factor=s, original=n), "cpu")
    assert math.isclose(factor, 0.1 * math.log(s) + 1)
    for f, g in zip(plain, inv.tolist()):
        turns = n * f / (2 * math.pi)
        assert f / s * (1 - 1e-12) <= g <= f * (1 + 1e-12)
        # the ramp runs over whole pairs: one pair beyond each limit has left it
        step = theta ** (2.0 / R)
        assert turns < 32 * step or math.isclose(f, g)
        assert turns > 1 / step or math.isclose(f / s, g)
    inv, factor = ops.rope_frequencies(R, theta, dict(kind="bands", factor=s, original=n, low=1, high=4), "cpu")
    for f, g in zip(plain, inv.tolist()):
        turns = n * f / (2 * math.pi)
        want = f if turns > 4 else f / s if turns < 1 else f / s + (f - f / s) * (turns - 1) / 3
        assert math.isclose(g, want, rel_tol=1e-12) and factor == 1.0


@pytest.mark.parametrize("a", [
    (63,), (0,), (64, 1.0), (64, float("inf")), (64, 1e4, dict(kind="cubic", factor=2)),
    (64, 1e4, dict(kind="linear", factor=0.5)), (64, 1e4, dict(kind="linear")),
    (64, 1e4, dict(kind="yarn", factor=4)), (64, 1e4, dict(kind="bands", factor=4, original=4096, low=4, high=4)),
    (64, 1e4, dict(kind="linear", factor=2, original=4096)),
])
def test_frequencies_refused(a):
    with pytest.raises(ValueError):
        ops.rope_frequencies(*a, device="cpu")
