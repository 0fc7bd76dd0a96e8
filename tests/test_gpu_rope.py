"""The appends with a caller's frequencies (part of the head, neighbouring pairs, a factor) on the GPU.

Tolerances count roundings.  Cosines and sines are good to 2 units in the last place (the
bound CUDA documents for sincosf) and rounded once more by the factor, two products and a
sum: 2^-21 factor (|a| + |b|) covers all of it.  Binary16 outputs add half a step, 2^-11
of the value (2^-25 in the subnormals).  The 8-bit forms are compared bit for bit with
calls that must do the same arithmetic on reordered dims."""
import numpy as np
import pytest
import torch

import serving_oracle as so
from anvilq_b200 import ops
from test_gpu_serving import APPENDS, append_case, code_dtype, random_codes, random_scales, rows_of, to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def turned64(x, pos, inv, pairs, factor):
    """x [T, heads, D] rotated in 64 bits, and |a| + |b| of each value's pair."""
    R = 2 * len(inv)
    angle = (np.asarray(pos, np.float64)[:, None] * inv).astype(np.float32).astype(np.float64)[:, None]
    c, s = factor * np.cos(angle), factor * np.sin(angle)
    out, size = x.astype(np.float64), np.zeros(x.shape)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if pairs else (slice(0, R // 2), slice(R // 2, R))
    xa, xb = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
    out[..., a], out[..., b] = xa * c - xb * s, xb * c + xa * s
    size[..., a] = size[..., b] = np.abs(xa) + np.abs(xb)
    return out, size


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("share,factor", [(1.0, 1.25), (0.5, 1.0), (0.25, 1.0), (0.75, 0.5)])
@pytest.mark.parametrize("before,new,Hq,Hkv,D,page", APPENDS)
def test_binary16(dev, before, new, Hq, Hkv, D, page, share, factor, pairs):
    rng = np.random.default_rng(41 + len(before))
    qkv, table, starts, lens, pages = append_case(rng, before, new, Hq, Hkv, D, page)
    R = int(D * share)
    inv, _ = ops.rope_frequencies(R, 1e4, dict(kind="bands", factor=4, original=1000), "cpu")
    pools = [rng.standard_normal((pages, page, Hkv, D)).astype(np.float16) for _ in range(2)]
    k, v = to(pools[0], dev), to(pools[1], dev)
    q_out = torch.full((len(qkv), Hq, D), 7.0, dtype=torch.float16, device=dev)
    ops.paged_kv_append(to(qkv, dev), k, v, to(table, dev), to(lens, dev), to(starts, dev), Hq, q_out=q_out,
                        inv_freq=inv.to(dev), interleaved=pairs, rope_factor=factor)
    ops.raise_device_errors(dev)
    rows = rows_of(starts, lens)
    n = len(rows)
    x = qkv[:n].reshape(n, Hq + 2 * Hkv, D)
    want, size = turned64(x[:, :Hq + Hkv], [p for _, p in rows], inv.numpy(), pairs, factor)
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -21 * factor * size + 2.0 ** -25
    tol[..., R:] = 0                     # copied
    got = q_out.cpu().numpy().astype(np.float64)
    assert (np.abs(got[:n] - want[:, :Hq]) <= tol[:, :Hq]).all()
    assert (got[n:] == 7.0).all(), "rows of no sequence are left as they were"
    gk, gv = k.cpu().numpy(), v.cpu().numpy()
    same_k, same_v = pools[0].copy(), pools[1].copy()
    for r, (b, pos) in enumerate(rows):
        at = so.physical(table[b, pos // page]), pos % page
        assert (np.abs(gk[at].astype(np.float64) - want[r, Hq:]) <= tol[r, Hq:]).all(), (b, pos)
        same_k[at], same_v[at] = gk[at], x[r, Hq + Hkv:]
    assert np.array_equal(gv, same_v) and np.array_equal(gk, same_k), "only the new rows change"


def q8_state(rng, pages, Hkv, page, D, fp8):
    return [random_codes(rng, (pages, Hkv, page, D), fp8) for _ in range(2)] + \
           [random_scales(rng, (pages, Hkv, page // 16), fp8) for _ in range(2)]


def raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("before,new,Hq,Hkv,D,page", APPENDS)
def test_8_bit_pages_by_reordered_heads(dev, before, new, Hq, Hkv, D, page, fp8):
    """theta's frequencies given by the caller are the append by theta; neighbouring pairs are split
    halves of reordered dims; a partial rotation turns the other dims by nothing."""
    rng = np.random.default_rng(43 + len(before))
    qkv, table, starts, lens, pages = append_case(rng, before, new, Hq, Hkv, D, page)
    state = q8_state(rng, pages, Hkv, page, D, fp8)
    rest = [to(a, dev) for a in (table, lens, starts)] + [Hq]
    qkv = to(qkv, dev)
    order = torch.arange(D, device=dev).reshape(2, D // 2).t().reshape(-1)     # [0, D/2, 1, D/2 + 1, ...]
    n = int(starts[-1])

    def call(x, reorder=None, **kw):
        codes = [raw(t.to(dev)) for t in state[:2]]
        if reorder is not None:
            codes = [c[..., reorder].contiguous() for c in codes]
        codes = [c.view(code_dtype(fp8)) for c in codes]
        scales = [t.to(dev) for t in state[2:]]
        q = ops.paged_kv_append_q8(x, *codes, *scales, *rest, **kw)
        ops.raise_device_errors(dev)
        return [q[:n], *map(raw, codes), *scales]

    inv, _ = ops.rope_frequencies(D, 1e6, device=dev)
    by_theta = call(qkv, theta=1e6)
    for a, b in zip(by_theta, call(qkv, inv_freq=inv)):
        assert torch.equal(a, b)
    mixed = qkv.reshape(len(qkv), -1, D)[..., order].reshape(qkv.shape).contiguous()
    for a, b in zip(by_theta, call(mixed, order, inv_freq=inv, interleaved=True)):
        assert torch.equal(a[..., order] if a.shape[-1] == D else a, b)
    few = torch.cat([inv[:D // 8], torch.zeros(D // 2 - D // 8, dtype=torch.float64, device=dev)])
    for a, b in zip(call(qkv, inv_freq=few, interleaved=True),
                    call(qkv, inv_freq=few[:D // 8].contiguous(), interleaved=True)):
        assert torch.equal(a, b)
    # the halves of a partial rotation: its dims in front, reordered into neighbouring pairs
    R = D // 4
    part = torch.cat([torch.arange(R, device=dev).reshape(2, R // 2).t().reshape(-1), torch.arange(R, D, device=dev)])
    mixed = qkv.reshape(len(qkv), -1, D)[..., part].reshape(qkv.shape).contiguous()
    for a, b in zip(call(qkv, inv_freq=inv[:R // 2].contiguous(), rope_factor=1.5),
                    call(mixed, part, inv_freq=inv[:R // 2].contiguous(), rope_factor=1.5, interleaved=True)):
        assert torch.equal(a[..., part] if a.shape[-1] == D else a, b)


def test_captured_and_replayed_with_other_frequencies(dev):
    """Frequencies are read when the call runs: a replay sees new ones."""
    rng = np.random.default_rng(7)
    qkv, table, starts, lens, pages = append_case(rng, [20, 3], [5, 1], 4, 2, 64, 16, spare_rows=0)
    args = [to(qkv, dev)] + [torch.zeros((pages, 16, 2, 64), dtype=torch.float16, device=dev) for _ in range(2)] + \
           [to(a, dev) for a in (table, lens, starts)] + [4]
    inv, _ = ops.rope_frequencies(32, 1e4, device=dev)
    other, _ = ops.rope_frequencies(32, 1e4, dict(kind="linear", factor=3.0), dev)
    want = ops.paged_kv_append(*args, inv_freq=other).clone()
    q = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_kv_append(*args, q_out=q, inv_freq=inv)
    inv.copy_(other)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(q, want)
    ops.raise_device_errors(dev)
