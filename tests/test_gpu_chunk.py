"""Attention of a batch's new tokens over binary16 pages on the GPU, against its definition in 64 bits.

Tolerances count roundings.  The output's: 2^-11 of the value (2^-25 in the subnormals).
Probabilities enter the tensor cores in binary16, 2^-11 of each, so 2^-11 sum p |v|; below
binary16's normal range 2^-25 of the row's largest, which is at least 1: 2^-25 sum |v|.  A
score is D / 16 accumulation steps of at most 2^-22 of sum |q| |k| each, which moves a
probability by at most 2^-19 sum |q| max |k|, and the result by twice that (in the sum and
in the product).  The products' n / 16 accumulation steps add 2^-22 sum p |v| each, a
thread's sums at most 32 + n / 128 roundings of 2^-24, ex2 2^-22 twice: 2^-18 sum p |v|
covers these for n up to 2^13."""
import numpy as np
import pytest
import torch

import serving_oracle as so
from anvilq_b200 import AnvilqError, ops
from test_gpu_serving import to

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


class Case:
    """A batch over a shuffled pool whose unused rows and pages hold NaN."""

    def __init__(self, dev, seed, before, new, Hq, Hkv, D, page, spare=3, scale=0.0, size=1.0, width=None):
        rng = np.random.default_rng(seed)
        self.dev, self.before, self.new, self.D, self.Hq, self.Hkv = dev, before, new, D, Hq, Hkv
        lens = [p + n if n >= 0 else 0 for p, n in zip(before, new)]
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 2
        self.np_table = so.make_table(need, pages, rng, width)
        self.starts_list = [int(x) for x in np.concatenate([[0], np.cumsum(new)])]
        T = self.starts_list[-1]
        self.q = (rng.standard_normal((T + spare, Hq, D)) * 2 * size).astype(np.float16)
        self.k, self.v = [], []
        pools = [np.full((pages, page, Hkv, D), np.nan, np.float16) for _ in range(2)]
        for b, n in enumerate(lens):
            rows = [(rng.standard_normal((n, Hkv, D)) * (size if i == 0 else 1)).astype(np.float16) for i in range(2)]
            self.k.append(rows[0])
            self.v.append(rows[1])
            for pool, x in zip(pools, rows):
                for j in range(need[b]):
                    part = x[j * page:(j + 1) * page]
                    pool[so.physical(self.np_table[b, j]), :len(part)] = part
        self.scale = scale if scale > 0 else 1 / np.sqrt(D)
        self.args = [to(a, dev) for a in (self.q, *pools, self.np_table, np.array(lens, np.int32),
                                          np.array(self.starts_list, np.int32))]
        self.given_scale = scale

    def run(self, **kw):
        return ops.gqa_chunk_paged(*self.args, scale=self.given_scale, **kw)

    def check(self, out):
        got = out.cpu().numpy().astype(np.float64)
        g = self.Hq // self.Hkv
        for b, n in enumerate(self.new):
            if n < 1:
                continue
            q = self.q[self.starts_list[b]:self.starts_list[b + 1]].astype(np.float64)
            pos = self.before[b] + np.arange(n)
            for h in range(self.Hkv):
                k, v = self.k[b][:, h].astype(np.float64), self.v[b][:, h].astype(np.float64)
                hidden = np.arange(len(k))[None] > pos[:, None]
                for i in range(h * g, (h + 1) * g):
                    x = q[:, i] @ k.T * self.scale
                    x[hidden] = -np.inf
                    p = np.exp(x - x.max(axis=1, keepdims=True))
                    p /= p.sum(axis=1, keepdims=True)
                    want, mass = p @ v, p @ np.abs(v)
                    reach = np.abs(q[:, i]).sum(axis=1, keepdims=True) * np.abs(k).max() * self.scale
                    tol = 2.0 ** -11 * np.abs(want) + mass * (2.0 ** -11 + 2.0 ** -18 * reach + 2.0 ** -18) + \
                        2.0 ** -25 * np.abs(v).sum(axis=0) + 2.0 ** -25
                    off = np.abs(got[self.starts_list[b]:self.starts_list[b + 1], i] - want)
                    assert (off <= tol).all(), (b, i, float((off - tol).max()), float(off.max()))


CASES = [
    ([0], [1], 1, 1, 64, 16),                                     # one first token
    ([0], [1], 14, 2, 128, 32),
    ([150], [13], 14, 2, 64, 16),
    ([0], [128], 4, 4, 128, 16), ([0], [129], 4, 4, 64, 64),      # around a tile
    ([127, 128, 129, 0], [1, 1, 1, 3], 8, 2, 128, 48),
    ([0, 5, 100, 0, 63], [0, 300, 0, 64, 65], 28, 4, 128, 48),    # idle sequences between
    ([700, 3], [40, 1000], 6, 2, 64, 96),                         # tpt 42: rows of padding
    ([10, 0], [500, 200], 5, 1, 128, 128),
    ([30], [70], 128, 1, 64, 16), ([3, 200], [9, 5], 100, 1, 128, 256),   # one token a tile
    ([5000], [1], 32, 8, 128, 64),                                # few rows over a long axis
    ([6000, 17], [30, 2], 8, 1, 64, 16),
    ([3000], [1200], 8, 8, 128, 16),                              # many pairs, no groups
    ([i * 37 % 500 for i in range(70)], [1 + i * 13 % 40 if i % 9 else 0 for i in range(70)], 4, 2, 64, 32),
    ([i % 300 for i in range(300)], [1] * 300, 8, 2, 128, 16),    # a decode step
]


@pytest.mark.parametrize("before,new,Hq,Hkv,D,page", CASES)
def test_against_the_definition(dev, before, new, Hq, Hkv, D, page):
    c = Case(dev, len(before) + D + page, before, new, Hq, Hkv, D, page)
    out = torch.full((len(c.q), Hq, D), 7.0, dtype=torch.float16, device=dev)
    c.run(out=out)
    ops.raise_device_errors(dev)
    c.check(out)
    assert (out[c.starts_list[-1]:] == 7.0).all(), "rows of no sequence are left as they were"
    again = c.run()
    assert torch.equal(again[:c.starts_list[-1]], out[:c.starts_list[-1]]), "bit-reproducible"


@pytest.mark.parametrize("scale,size", [(1.0, 1.0), (0.01, 1.0), (0.0, 8.0), (2.0 ** -20, 1.0)])
def test_scales_and_large_scores(dev, scale, size):
    """Flat and peaked rows: the reference moves often, or never."""
    c = Case(dev, 5, [300, 0, 40], [150, 77, 1], 8, 2, 64, 16, scale=scale, size=size)
    c.check(c.run())
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("rising", [False, True])
def test_rows_whose_scores_rise_and_fall(dev, rising):
    """Every key tile beats the last by more than the reference's slack, or none does."""
    c = Case(dev, 6, [900], [300], 4, 1, 64, 32)
    q, k = c.args[0], c.args[1]
    n = len(c.k[0])
    slope = np.linspace(0, 1, n) if rising else np.linspace(1, 0, n)
    c.q[..., 0] = 8.0
    c.k[0][:, 0, 0] = (slope * 120).astype(np.float16)
    q[..., 0] = 8.0
    for j in range(-(-n // 32)):
        part = to(c.k[0][j * 32:(j + 1) * 32, 0, 0], dev)
        k[so.physical(c.np_table[0, j]), :len(part), 0, 0] = part
    c.check(c.run())
    ops.raise_device_errors(dev)


def test_strided_queries_and_no_tokens(dev):
    """q as the first heads of the projection's rows; no new token at all."""
    c = Case(dev, 9, [64, 9], [30, 200], 4, 2, 64, 16, spare=0)
    wide = torch.randn((230, 4 + 4, 64), device=dev).half()
    wide[:, :4] = c.args[0]
    want = c.run()
    assert torch.equal(ops.gqa_chunk_paged(wide[:, :4], *c.args[1:]), want)
    none = torch.zeros(3, dtype=torch.int32, device=dev)
    assert ops.gqa_chunk_paged(wide[:0, :4], *c.args[1:5], none).shape == (0, 4, 64)
    out = torch.full_like(want, 3.0)
    ops.gqa_chunk_paged(c.args[0], *c.args[1:5], none, out=out)
    assert (out == 3.0).all()
    ops.raise_device_errors(dev)


def test_scores_that_are_all_infinitely_low(dev):
    c = Case(dev, 10, [0], [40], 2, 1, 64, 16, spare=0)
    c.args[0][:] = 1.0
    c.args[1][torch.isfinite(c.args[1])] = -float("inf")
    assert not c.run().any()
    ops.raise_device_errors(dev)


def test_a_sequences_nan_stays_with_it(dev):
    c = Case(dev, 11, [30, 200, 10], [5, 140, 7], 4, 1, 128, 16, spare=0)
    want = c.run().clone()
    c.args[2][so.physical(c.np_table[1, 0]), 3] = float("nan")
    got = c.run()
    assert torch.equal(got[:5], want[:5]) and torch.equal(got[145:], want[145:]) and got[5:145].isnan().all()
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("what", ["short", "long", "starts", "page", "absent"])
def test_bad_contents_are_reported(dev, what):
    """Lengths and tables that no host check sees: reported; other sequences are right."""
    c = Case(dev, 12, [20, 40, 60], [30, 20, 10], 4, 2, 64, 16, spare=0)
    want = c.run().clone()
    table, lens, starts = c.args[3:6]
    if what == "short":
        lens[1] = 19                 # fewer tokens than new ones
    elif what == "long":
        lens[1] = 16 * table.shape[1] + 1
    elif what == "starts":
        starts[3] = 61               # past the last row
    else:
        table[1, 0] = 0 if what == "absent" else int(np.uint32(999 | so.VALID).view(np.int32))
    out = torch.full_like(want, 5.0)
    c.run(out=out)
    with pytest.raises(AnvilqError):
        ops.raise_device_errors(dev)
    good = slice(0, 30) if what != "starts" else slice(0, 50)
    assert torch.equal(out[good], want[good])
    if what in ("short", "long"):
        assert (out[30:50] == 5.0).all() and torch.equal(out[50:], want[50:])
    if what == "starts":
        assert (out[50:] == 5.0).all()


def test_single_tokens_agree_with_decode_attention(dev):
    """A decode step through both: within the roundings that each may make."""
    c = Case(dev, 13, [99, 0, 511, 64], [1, 1, 1, 1], 14, 2, 64, 32, spare=0)
    a = c.run()
    b = ops.gqa_decode_paged(c.args[0], c.args[1].nan_to_num(0), c.args[2].nan_to_num(0), c.args[3], c.args[4])
    c.check(a), c.check(b)
    ops.raise_device_errors(dev)


def test_captured_and_replayed_as_the_batch_changes(dev):
    """One graph over other lengths, starts and tables; two graphs side by side."""
    first = Case(dev, 20, [100, 900], [50, 3], 8, 2, 128, 16, spare=10, width=70)
    others = [Case(dev, 21 + i, b, n, 8, 2, 128, 16, spare=53 + 10 - sum(n), width=70) for i, (b, n) in enumerate((
        ([0, 0], [1, 1]), ([1000, 7], [30, 25]), ([3, 1060], [0, 60])))]
    pools = [torch.full((200, 16, 2, 128), float("nan"), dtype=torch.float16, device=dev) for _ in range(2)]
    static = [first.args[0].clone(), *pools, *(a.clone() for a in first.args[3:])]
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.gqa_chunk_paged(*static))
        graphs.append(g)
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    for c in (first, *others):
        for s, a in zip(static, c.args):
            s[:len(a)] = a
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for out in outs:
            c.check(out)
    ops.raise_device_errors(dev)


def test_a_workspace_of_the_callers_and_overlapped_launches(dev):
    c = Case(dev, 30, [2000, 10], [40, 300], 8, 2, 128, 64, spare=0)
    want = c.run()
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device=dev)
    outs = [torch.empty_like(want) for _ in range(6)]
    for o in outs:
        c.run(out=o, workspace=ws, overlap_prior=True)
    assert all(torch.equal(o, want) for o in outs)
    assert not ws[:ops.WORKSPACE_COUNTER_BYTES].any()
    with pytest.raises(ValueError):
        c.run(workspace=ws[:1 << 16])
    ops.raise_device_errors(dev)
