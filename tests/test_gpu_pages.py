"""Shared pages on the GPU against the one-entry-at-a-time forms of pages_oracle.py: all results are whole numbers
or copies, so everything is compared for equality."""
import numpy as np
import pytest
import torch

import pages_oracle as po
from anvilq_b200 import AnvilqError, ops

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def to(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Cache:
    """A table with its counts and pools, on the device and as the oracle keeps them."""

    def __init__(self, dev, rng, table, pages, width, page, kinds, Hkv=2, D=64):
        self.dev, self.page, self.width, self.pages = dev, page, width, pages
        self.table = [list(r) + [None] * (width - len(r)) for r in table]
        self.refs = po.counts(table, pages)
        self.d_table, self.d_refs = to(po.words(self.table, width), dev), ints(self.refs, dev)
        self.pools, self.d_pools = [], []
        for kind in kinds:
            if kind == "fp16":
                a, axis, unit = rng.integers(0, 1 << 15, size=(pages, page, Hkv, D)).astype(np.uint16), 1, 1
                t = to(a.view(np.float16), dev)
            elif kind in ("int8", "fp8"):
                a, axis, unit = rng.integers(0, 127, size=(pages, Hkv, page, D)).astype(np.uint8), 2, 1
                t = to(a.view(np.int8), dev)
                t = t if kind == "int8" else t.view(torch.float8_e4m3fn)
            else:
                a, axis, unit = rng.standard_normal((pages, Hkv, page // 16)).astype(np.float32), 2, 16
                t = to(a, dev)
            self.pools.append((a.copy(), axis, unit))
            self.d_pools.append(t)

    def same(self):
        ops.raise_device_errors(self.dev)
        assert po.rows(self.d_table.cpu().numpy()) == self.table
        assert self.d_refs.tolist() == self.refs
        for (a, _, _), t in zip(self.pools, self.d_pools):
            assert np.array_equal(t.view(torch.uint8).cpu().numpy().view(a.dtype).reshape(a.shape), a)

    def fork(self, parents, shape=None):
        self.d_table = ops.pages_fork(self.d_table, self.d_refs, ints(parents, self.dev) if shape is None else
                                      ints(shape, self.dev))
        self.table = po.fork(self.table, self.refs, parents, self.width)

    def reserve(self, before, after):
        got = ops.pages_reserve(self.d_table, self.d_refs, ints(before, self.dev), ints(after, self.dev), self.page,
                                self.d_pools)
        want = po.reserve(self.table, self.refs, before, after, self.page, self.pools)
        assert int(got) == want
        return want

    def release(self, keep):
        ops.pages_release(self.d_table, self.d_refs, ints(keep, self.dev), self.page)
        po.release(self.table, self.refs, keep, self.page)

    def compact(self):
        _, _, used = ops.pages_compact(self.d_table, self.d_refs, self.d_pools, self.page)
        assert int(used) == po.compact(self.table, self.refs, self.pools)


KINDS = [["fp16"] * 3, ["int8", "int8", "scale", "scale"], ["fp8", "scale", "fp16"], []]


@pytest.mark.parametrize("kinds", KINDS, ids=lambda k: "-".join(k) or "none")
@pytest.mark.parametrize("page,D,Hkv", [(16, 64, 1), (48, 128, 3), (256, 64, 2)])
def test_a_search_from_prompts_to_its_end(dev, kinds, page, D, Hkv):
    """Prompts allocated, each answered by several beams that fork, go on, die and end; then compacted."""
    rng = np.random.default_rng(page + len(kinds))
    items, beams, width = 3, 4, 6
    c = Cache(dev, rng, [[] for _ in range(items)], 90, width, page, kinds, Hkv, D)
    lens = [int(n) for n in rng.integers(1, 2 * page, size=items)]
    c.reserve([0] * items, lens)
    c.same()
    c.fork([i for i in range(items) for _ in range(beams)])       # every beam starts as its prompt
    c.same()
    lens = [n for n in lens for _ in range(beams)]
    for step in range(2 * page if page < 200 else 40):
        c.reserve(lens, [n + 1 for n in lens])
        lens = [n + 1 for n in lens]
        local = rng.integers(-1 if step % 7 == 3 else 0, beams, size=(items, beams))
        parents = [int(p) + i * beams if p >= 0 else -1 for i in range(items) for p in local[i]]
        c.fork(parents, local.tolist())
        lens = [lens[p] if p >= 0 else 0 for p in parents]
        if max(lens) + 1 > width * page:
            break
        if step % 5 == 0:
            c.same()
    c.same()
    c.release([n if i % 3 else n // 2 for i, n in enumerate(lens)])
    c.same()
    c.compact()
    c.same()
    c.compact()          # nothing is left to move
    c.same()


@pytest.mark.parametrize("seed", range(6))
def test_any_calls_in_any_order(dev, seed):
    rng = np.random.default_rng(100 + seed)
    page, width, pages, rows = 16, int(rng.integers(1, 9)), 60, int(rng.integers(1, 12))
    c = Cache(dev, rng, [[] for _ in range(rows)], pages, width, page, KINDS[seed % 3])
    short = 0
    for _ in range(30):
        n = len(c.table)
        what = rng.integers(0, 4)
        if what == 0:
            c.fork([int(p) for p in rng.integers(-1, n, size=int(rng.integers(1, 14)))])
        elif what == 1:
            c.release([int(k) for k in rng.integers(0, width * page + 1, size=n)])
        elif what == 2:
            c.compact()
        else:
            lo = rng.integers(0, width * page + 1, size=n)
            hi = np.minimum(lo + rng.integers(-3, 40, size=n), width * page)
            if c.reserve([int(x) for x in lo], [int(x) for x in hi]):
                short += 1
                with pytest.raises(AnvilqError, match="free pages"):
                    ops.raise_device_errors(dev)
        c.same()


def test_many_rows_entries_and_pages(dev):
    """More rows, entries and pages than a planning pass takes at once, with more than 128 pools."""
    rng = np.random.default_rng(3)
    rows, width, page, pages = 2500, 7, 16, 40000
    c = Cache(dev, rng, [[] for _ in range(rows)], pages, width, page, [])
    a = rng.integers(0, 1 << 15, size=(pages, page, 1, 8)).astype(np.uint16)
    lens = [int(n) for n in rng.integers(0, 100, size=rows)]
    c.reserve([0] * rows, lens)
    c.same()
    parents = [int(p) for p in rng.integers(0, rows, size=rows)]
    c.fork(parents)
    lens = [lens[p] for p in parents]
    c.pools.append((a.copy(), 1, 1))
    c.d_pools.append(to(a.view(np.float16), dev))
    c.reserve(lens, [n + 5 for n in lens])
    c.same()
    c.release([0 if rng.random() < 0.7 else n for n in lens])
    c.compact()
    c.same()
    many = [torch.arange(4 * 16 * 8, device=dev).reshape(4, 16, 1, 8).half() + i for i in range(300)]
    want = [t.clone() for t in many]
    ops.pages_copy(many, ints([0, 1, -1], dev), ints([2, 3, 0], dev), 16, rows=ints([-1, 5, 3], dev))
    for t, w in zip(many, want):
        w[2] = w[0]
        w[3, :5] = w[1, :5]
        assert torch.equal(t, w)
    ops.raise_device_errors(dev)


def test_copy_lists(dev):
    t = torch.arange(6 * 16 * 2 * 64, device=dev).reshape(6, 16, 2, 64).half()
    want = t.clone()
    want[4] = want[0]
    ops.pages_copy(ops.PagePools([t], 16), ints([0, 1, 2], dev), ints([4, 5, 3], dev), 16, count=ints([1], dev))
    ops.pages_copy([t], ints([], dev), ints([], dev), 16)
    ops.pages_copy([], ints([0], dev), ints([1], dev), 16)
    assert torch.equal(t, want)
    ops.raise_device_errors(dev)


def test_copies_of_more_rows_than_a_page_has(dev):
    """They are the whole page, also where their bytes pass 32 bits (2^24 tokens of 256 bytes)."""
    t = torch.arange(12 * 16 * 2 * 64, device=dev).reshape(12, 16, 2, 64).half()
    want = t.clone()
    src, dst, rows = [0, 1, 2, 3, 4], [6, 7, 8, 9, 10], [16, 17, 1 << 24, (1 << 24) + 3, (1 << 31) - 1]
    want[6:11] = want[:5]
    ops.pages_copy([t], ints(src, dev), ints(dst, dev), 16, rows=ints(rows, dev))
    assert torch.equal(t, want)
    ops.raise_device_errors(dev)


def test_reserve_passes_over_pages_that_more_entries_name_than_counted(dev):
    """Page 1 is named three times and counted twice: its entries and its count stay, the rest is done."""
    table = to(po.words([[0, 1], [2, 1], [3, 1]], 3), dev)
    refs = ints([1, 2, 1, 1, 0, 0, 0], dev)
    pool = torch.randn(7, 16, 1, 64, device=dev).half()
    want = pool.clone()
    lacking = ops.pages_reserve(table, refs, ints([20, 20, 20], dev), ints([40, 21, 21], dev), 16, [pool])
    assert po.rows(table.cpu().numpy()) == [[0, 1, 4], [2, 1, None], [3, 1, None]]
    assert refs.tolist() == [1, 2, 1, 1, 1, 0, 0] and int(lacking) == 0 and torch.equal(pool, want)
    with pytest.raises(AnvilqError):
        ops.raise_device_errors(dev)


def test_unaligned_pools(dev):
    """Pools that start on a 4-byte border only, and heads whose runs are odd multiples of 4 bytes."""
    rng = np.random.default_rng(9)
    flat = torch.from_numpy(rng.standard_normal(7 * 48 * 3 * 6 + 1).astype(np.float32)).to(dev).view(torch.float16)
    t = flat[2:2 + 7 * 48 * 3 * 6].view(7, 48, 3, 6)
    scales = torch.from_numpy(rng.standard_normal(7 * 3 * 3 + 1).astype(np.float32)).to(dev)[1:].view(7, 3, 3)
    want, want_s, edge = t.clone(), scales.clone(), flat[:2].clone()
    want[6, :17], want_s[6, :, :2] = want[1, :17], want_s[1, :, :2]
    ops.pages_copy([t, scales], ints([1], dev), ints([6], dev), 48, rows=ints([17], dev))
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))      # bits: some are NaN
    assert same(t, want) and torch.equal(scales, want_s) and same(flat[:2], edge)
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("what", ["fork parent", "fork page", "reserve range", "reserve page", "release keep",
                                  "release count", "copy page", "compact page"])
def test_bad_contents_are_reported(dev, what):
    """Values on the device that no host check sees: reported, passed over, the rest done."""
    bad = np.array([100 | po.VALID], np.uint32).view(np.int32)[0]
    table = to(po.words([[0, 1], [2, None]], 2), dev)
    refs = ints([1, 1, 1, 0, 0], dev)
    pool = torch.arange(5 * 16 * 64, device=dev).reshape(5, 16, 1, 64).half()
    before = pool.clone()
    if what == "fork parent":
        out = ops.pages_fork(table, refs, ints([5, 0], dev))
        assert po.rows(out.cpu().numpy()) == [[None, None], [0, 1]] and refs.tolist() == [1, 1, 0, 0, 0]
    elif what == "fork page":
        table[0, 1] = int(bad)
        out = ops.pages_fork(table, refs, ints([0, 1], dev))
        assert po.rows(out.cpu().numpy()) == [[0, None], [2, None]]
    elif what == "reserve range":
        ops.pages_reserve(table, refs, ints([-1, 16], dev), ints([5, 17], dev), 16, [pool])
        assert po.rows(table.cpu().numpy()) == [[0, 1], [2, 3]]
    elif what == "reserve page":
        table[0, 1] = int(bad)
        ops.pages_reserve(table, refs, ints([16, 16], dev), ints([17, 17], dev), 16, [pool])
        assert int(table[0, 1]) == int(bad) and po.rows(table[1:].cpu().numpy()) == [[2, 3]]
    elif what == "release keep":
        ops.pages_release(table, refs, ints([-4, 0], dev), 16)
        assert po.rows(table.cpu().numpy()) == [[0, 1], [None, None]] and refs.tolist() == [1, 1, 0, 0, 0]
    elif what == "release count":
        refs[1] = 0
        ops.pages_release(table, refs, ints([0, 5], dev), 16)
        assert refs.tolist() == [0, 0, 1, 0, 0]
    elif what == "copy page":
        ops.pages_copy([pool], ints([5, 0], dev), ints([1, 2], dev), 16)
        before[2] = before[0]
    else:
        table[0, 1] = int(bad)
        out, _, used = ops.pages_compact(table, ints([1, 0, 1, 0, 0], dev), [pool], out=torch.zeros_like(table))
        assert int(used) == 2 and int(out[0, 1]) == int(bad) and po.rows(out[1:].cpu().numpy()) == [[1, None]]
        before[1] = before[2]
    assert torch.equal(pool, before)
    with pytest.raises(AnvilqError):
        ops.raise_device_errors(dev)


def test_captured_steps_replayed(dev):
    """A search's fork and reserve captured once and replayed on what earlier replays left, each graph with
    workspaces of its own."""
    rng = np.random.default_rng(8)
    c = Cache(dev, rng, [[0, 1]] * 4, 40, 4, 16, ["fp16", "fp16"])
    parents, before, after = ints([0, 1, 2, 3], dev), ints([20] * 4, dev), ints([21] * 4, dev)
    other = torch.empty_like(c.d_table)
    graph = torch.cuda.CUDAGraph()
    ops.device_error_word(dev)
    with torch.cuda.graph(graph):
        ops.pages_fork(c.d_table, c.d_refs, parents, out=other)
        ops.pages_reserve(other, c.d_refs, before, after, 16, c.d_pools)
        c.d_table.copy_(other)
    lens = [20] * 4
    for step in range(10):
        p = [int(x) for x in rng.integers(0, 4, size=4)]
        parents.copy_(ints(p, dev)), before.copy_(ints(lens, dev)), after.copy_(ints([n + 1 for n in lens], dev))
        graph.replay()
        c.table = po.fork(c.table, c.refs, p, 4)
        assert po.reserve(c.table, c.refs, lens, [n + 1 for n in lens], 16, c.pools) == 0
        lens = [n + 1 for n in lens]
        c.same()


def test_another_stream_and_a_workspace_of_the_callers(dev):
    rng = np.random.default_rng(12)
    c = Cache(dev, rng, [[0, 1], [0, 1], [0, 2]], 30, 3, 32, ["int8", "scale"])
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device=dev)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        ops.pages_reserve(c.d_table, c.d_refs, ints([40, 41, 0], dev), ints([41, 50, 70], dev), 32, c.d_pools,
                          workspace=ws)
        ops.pages_compact(c.d_table, c.d_refs, ops.PagePools(c.d_pools, 32), workspace=ws)
    s.synchronize()
    po.reserve(c.table, c.refs, [40, 41, 0], [41, 50, 70], 32, c.pools)
    po.compact(c.table, c.refs, c.pools)
    c.same()
    assert not ws[:ops.WORKSPACE_COUNTER_BYTES].any()
