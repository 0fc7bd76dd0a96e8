"""Chunk attention at the edges of what it accepts: outputs on any 16 bytes, scores of any size, weights
far below a row's largest, contexts of many segments.

Tolerances and cases' makers: ``test_gpu_chunk``."""
import numpy as np
import pytest
import torch

import serving_oracle as so
from anvilq_b200 import ops
from test_gpu_chunk import Case, dev  # noqa: F401
from test_gpu_serving import to

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


def set_keys(c, b, k):
    """Other keys of sequence b, [positions, heads, D], in the pages too."""
    page = c.args[1].shape[1]
    c.k[b] = k.astype(np.float16)
    for j in range(-(-len(k) // page)):
        part = to(c.k[b][j * page:(j + 1) * page], c.dev)
        c.args[1][so.physical(c.np_table[b, j]), :len(part)] = part


@pytest.mark.parametrize("sign", [1, -1, 0])
@pytest.mark.parametrize("scale", [2.0 ** 12, 2.0 ** 19, 2.0 ** 22, 2.0 ** 25, 2.0 ** 32])
def test_scores_of_any_size(dev, scale, sign):
    """Scores are whole numbers times a large scale, all above 0, all below, or of both signs: the keys of a
    row's largest share it, the others' weights, exp(-4096) or less, are nothing.  Equal keys have equal
    probabilities, so the tolerance is their rounding, 2^-11 of sum p |v|, the output's, and 2^-20 for
    the products' and the sums' few additions."""
    c = Case(dev, 50, [300, 0, 40], [150, 77, 1], 8, 2, 64, 16, scale=scale, spare=0)
    rng = np.random.default_rng(51)
    whole = lambda *shape: rng.integers(1 if sign else -3, 4, size=shape)
    c.q[:] = whole(*c.q.shape)
    c.args[0][:] = to(c.q, dev)
    for b in range(3):
        set_keys(c, b, whole(*c.k[b].shape) * (sign or 1))
    got = c.run().cpu().numpy().astype(np.float64)
    ops.raise_device_errors(dev)
    for b, n in enumerate(c.new):
        q = c.q[c.starts_list[b]:c.starts_list[b + 1]].astype(np.float64)
        hidden = np.arange(len(c.k[b]))[None] > c.before[b] + np.arange(n)[:, None]
        for i in range(8):
            k, v = c.k[b][:, i // 4].astype(np.float64), c.v[b][:, i // 4].astype(np.float64)
            x = q[:, i] @ k.T
            x[hidden] = -np.inf
            p = (x == x.max(axis=1, keepdims=True)).astype(np.float64)
            p /= p.sum(axis=1, keepdims=True)
            want = p @ v
            tol = 2.0 ** -11 * np.abs(want) + (2.0 ** -11 + 2.0 ** -20) * (p @ np.abs(v)) + 2.0 ** -25
            assert (np.abs(got[c.starts_list[b]:c.starts_list[b + 1], i] - want) <= tol).all(), (b, i)


@pytest.mark.parametrize("below", [12, 20, 26, 28])
@pytest.mark.parametrize("D", [64, 128])
def test_many_keys_far_below_the_largest(dev, below, D):
    """One key takes most of a row, 2^17 others lie some `below` powers of two under it and have a share
    all the same.  Binary16 takes a probability to 2^-11 of it, or 2^-32 of the row's largest; a CTA has all
    keys of a pair of tokens, n / 16 accumulation steps of 2^-22; scores as in ``test_gpu_chunk``."""
    n, T, heads, page, kinds = 1 << 17, 296, 128, 256, 8
    rng = np.random.default_rng(below + D)
    q, k = rng.standard_normal((T, heads, D)) / 8, rng.standard_normal((1 + kinds, page, 1, D)) / 8
    v = 1 + rng.standard_normal(k.shape) / 4
    q[..., 0], k[..., 0] = 8, 0
    k[0], v[0] = k[1], v[1]
    k[0, 0, 0, 0], v[0, 0] = below / (8 * np.log2(np.e)) * np.sqrt(D), rng.standard_normal((1, D)) / 64
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    # page 0 first, the others in turn
    names = np.concatenate([[0], 1 + np.arange(n // page - 1) % kinds])
    table = (names.astype(np.uint32) | np.uint32(so.VALID)).view(np.int32)[None]
    lens, starts = np.array([n], np.int32), np.array([0, T], np.int32)
    out = ops.gqa_chunk_paged(*(to(a, dev) for a in (q, k, v, table, lens, starts)))
    ops.raise_device_errors(dev)
    got = out.cpu().numpy().astype(np.float64)
    keys, values = k.reshape(-1, D).astype(np.float64), v.reshape(-1, D).astype(np.float64)
    for t in (0, 1, 150, 295):
        seen = n - T + t + 1
        count = np.bincount(names[np.arange(seen) // page] * page + np.arange(seen) % page, minlength=len(keys))
        for h in (0, 77):
            x = keys @ q[t, h].astype(np.float64) / np.sqrt(D)
            p = np.exp(x - x.max())
            total = (p * count).sum()
            want, mass = p * count @ values / total, p * count @ np.abs(values) / total
            reach = np.abs(q[t, h].astype(np.float64)).sum() * np.abs(keys).max() / np.sqrt(D)
            tol = 2.0 ** -11 * np.abs(want) + mass * (2.0 ** -11 + 2.0 ** -18 * reach + n / 16 * 2.0 ** -22) + \
                2.0 ** -32 * (count @ np.abs(values)) / total + 2.0 ** -25
            off = np.abs(got[t, h] - want)
            assert (off <= tol).all(), (t, h, float(off.max()), float(tol.max()), float(want.mean()))


def long_case(dev, seed, before, new, Hq, Hkv, D, page, kinds=None):
    """(arguments, positions' page rows of every sequence) of a batch whose contexts are long; with `kinds`
    their pages are that many, named in turn."""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    need = [-(-(p + n) // page) for p, n in zip(before, new)]
    pages = kinds or sum(need)
    order = torch.randperm(pages, generator=g, device=dev).repeat(-(-sum(need) // pages))
    table = torch.zeros((len(new), max(need)), dtype=torch.int64, device=dev)
    rows, at = [], 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n] - (1 << 31)
        rows.append((order[at:at + n, None] * page + torch.arange(page, device=dev)).reshape(-1))
        at += n
    half = lambda *shape: torch.randn(shape, generator=g, device=dev).half()
    starts = np.concatenate([[0], np.cumsum(new)])
    q, k, v = half(int(starts[-1]), Hq, D), half(pages, page, Hkv, D), half(pages, page, Hkv, D)
    lens = torch.tensor([p + n for p, n in zip(before, new)], dtype=torch.int32, device=dev)
    return [q, k, v, table.to(torch.int32), lens, to(starts.astype(np.int32), dev)], rows


def exactly(args, rows, b, t, h):
    """(output, sum p |v|, scores' reach) of token t and head h of sequence b, in 64 bits."""
    q, k, v, _, lens, starts = args
    Hq, D = q.shape[1:]
    kv = h // (Hq // k.shape[2])
    seen = rows[b][:int(lens[b] - starts[b + 1] + starts[b]) + t + 1]
    query = q[int(starts[b]) + t, h].double()
    keys, values = k.flatten(0, 1)[:, kv].double(), v.flatten(0, 1)[:, kv].double()
    x = keys @ query / D ** 0.5
    p = torch.exp(x - x[seen].max()) * torch.bincount(seen, minlength=len(x))
    p /= p.sum()
    return p @ values, p @ values.abs(), query.abs().sum() * keys.abs().max() / D ** 0.5


@pytest.mark.parametrize("before,new,Hq,Hkv,D,page", [
    ([50000], [2600], 8, 8, 64, 64),                       # stretches inside pairs of several segments
    ([20000, 60000, 0], [700, 260, 5], 32, 8, 128, 16),    # and across them
    ([33000], [300], 128, 1, 64, 256),                     # whole pairs of several segments
    ([16384 - 151], [300], 128, 1, 128, 128),              # a segment's end between a pair's tiles
    ([16384, 16380, 16256], [1, 9, 3], 16, 16, 64, 32),    # a tile or a key more than a segment
])
def test_contexts_of_many_segments(dev, before, new, Hq, Hkv, D, page):
    """As ``test_gpu_chunk``, for chosen tokens and heads; a segment's products are 1024 accumulation steps of
    at most 2^-22 of sum p |v|."""
    args, rows = long_case(dev, len(before) + D, before, new, Hq, Hkv, D, page)
    out = ops.gqa_chunk_paged(*args)
    assert torch.equal(out, ops.gqa_chunk_paged(*args)), "bit-reproducible"
    ops.raise_device_errors(dev)
    for b, n in enumerate(new):
        for t in sorted({0, min(1, n - 1), n // 3, n // 2, 151 % n, max(n - 2, 0), n - 1}):
            for h in sorted({0, Hq // 2 + 1, Hq - 1}):
                want, mass, reach = exactly(args, rows, b, t, h)
                tol = 2.0 ** -11 * want.abs() + mass * (2.0 ** -11 + 2.0 ** -18 * reach + 2.0 ** -12) + 2.0 ** -25
                off = (out[int(args[5][b]) + t, h].double() - want).abs()
                assert (off <= tol).all(), (b, t, h, float(off.max()), float(tol.min()))


@pytest.mark.parametrize("D", [64, 128])
def test_long_contexts_are_not_biased(dev, D):
    """2^18 keys of nearly equal weights and values above 0, which a CTA adds up: additions that cut off,
    at most 2^-23 of the sum in each of a segment's 1024, would all err downwards.  Of the other roundings the
    mean over 100 rows of D values is far below 2^-14."""
    args, rows = long_case(dev, D, [1 << 18], [296], 128, 1, D, 256, kinds=16)
    args[0] *= 0.25
    args[2][:] = (torch.rand(args[2].shape, device=dev) * 0.5 + torch.linspace(0.3, 0.7, D, device=dev)).half()
    out = ops.gqa_chunk_paged(*args)
    ops.raise_device_errors(dev)
    off = []
    for t in range(0, 296, 30):
        for h in range(0, 128, 13):
            want, *_ = exactly(args, rows, 0, t, h)
            off.append((out[t, h].double() - want) / want)
    mean = float(torch.cat(off).mean())
    assert abs(mean) <= 2.0 ** -13 + 2.0 ** -14, mean
