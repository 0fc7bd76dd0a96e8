"""The beam search's selection and reordering on the GPU against their definition in 64 bits.

The order within a beam is exact.  A beam's log-sum-exp is off by at most: 2^-22 for
ex2.approx's relative error, 2^-23 of the mean distance to the largest logit (the exponent's
difference and product, each rounded), and 2^-24 for each of a thread's additions, at most
32 a tile (of at least 4096 logits over 256 threads) and one for each of its tiles, of which
a span of V <= 151936 logits has at most 38: 2^-22 + 2^-23 d + 70 2^-24 in all, below
6e-6 for distances below 10.  Scores add half a step of binary32.  Ranks that differ by less than
twice that may come in either order."""
import numpy as np
import pytest
import torch

from anvilq_b200 import AnvilqError, ops

pytestmark = pytest.mark.gpu
SLACK = 6e-6


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def definition(x, scores, lengths, alpha, ended, pad, V):
    """All candidates of one item: (rank, place, parent, token, score) best first; x float64 [K, V]."""
    found = []
    for k in range(len(x)):
        n = 0 if lengths is None else max(int(lengths[k]), 0)
        if not np.isfinite(scores[k]):
            continue
        if ended is not None and ended[k]:
            found.append((scores[k] / max(n, 1) ** alpha, k * V, k, pad, scores[k]))
            continue
        row = np.where(np.isfinite(x[k]), x[k], -np.inf)
        if row.max() == -np.inf:
            continue
        top = row.max()
        s = scores[k] + (row - (top + np.log(np.exp(row - top).sum())))
        for v in np.flatnonzero(row > -np.inf):
            found.append((s[v] / (n + 1) ** alpha, k * V + v, k, v, s[v]))
    found.sort(key=lambda c: (-c[0], c[1]))
    return found


def check(x, scores, N, lengths=None, alpha=0.0, ended=None, eos=(), pad=0, got=None):
    """x: torch [B, K, V] as given to the call."""
    B, K, V = x.shape
    tokens, parents, new, new_lengths, now = [t.cpu().numpy() if t is not None else None for t in got]
    y, sc = x.double().cpu().numpy(), scores.double().cpu().numpy()
    le = None if lengths is None else lengths.cpu().numpy()
    en = None if ended is None else ended.cpu().numpy()
    for b in range(B):
        all_ = definition(y[b], sc[b], None if le is None else le[b], alpha, None if en is None else en[b], pad, V)
        ranks, where = np.array([c[0] for c in all_]), {(c[2], c[1] - c[2] * V): i for i, c in enumerate(all_)}
        n = min(N, len(all_))
        assert (tokens[b, n:] == -1).all() and (parents[b, n:] == -1).all() and (new[b, n:] == -np.inf).all()
        assert now[b, n:].all() and (le is None or (new_lengths[b, n:] == 0).all())
        picked = []
        for i in range(n):
            k = int(parents[b, i])
            over = en is not None and en[b, k]
            at = where[k, 0 if over else int(tokens[b, i])]
            if over:
                assert tokens[b, i] == pad
            want = all_[at]
            assert abs(new[b, i] - want[4]) <= SLACK + 2.0 ** -24 * abs(want[4])
            assert abs(ranks[at] - ranks[i]) <= 2 * SLACK, (b, i, ranks[at], ranks[i])
            gap = min([abs(ranks[i] - ranks[j]) for j in (i - 1, i + 1) if 0 <= j < len(ranks)] + [1.0])
            if gap > 2 * SLACK:
                assert at == i
            assert now[b, i] == (over or int(tokens[b, i]) in eos)
            if le is not None:
                assert new_lengths[b, i] == le[b, k] + (not over)
            picked.append(at)
        assert len(set(picked)) == n
        # equal ranks within a beam: the lower token first, and no lower one left out
        for k in range(K):
            mine = [a for a in picked if all_[a][2] == k]
            assert mine == sorted(mine)
            if mine and not (en is not None and en[b, k]):
                of = [i for i, c in enumerate(all_) if c[2] == k]
                assert mine == of[:len(mine)]


def inputs(seed, B, K, V, half, dev, spread=3.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = torch.randn((B, K, V), generator=g, device=dev) * spread
    scores = -torch.rand((B, K), generator=g, device=dev) * 10
    lengths = torch.randint(0, 50, (B, K), generator=g, device=dev, dtype=torch.int32)
    ended = torch.rand((B, K), generator=g, device=dev) < 0.3
    return x.half() if half else x, scores, lengths, ended


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("B,K,V,N", [
    (1, 1, 1, 1), (1, 1, 1, 8), (2, 3, 2, 5), (1, 4, 7, 4), (3, 2, 31, 4), (2, 5, 257, 10), (1, 1, 1000, 128),
    (4, 64, 100, 64), (2, 8, 4096, 16), (2, 3, 4099, 6), (5, 4, 10001, 4), (1, 2, 32002, 4), (1, 4, 151936, 8),
    (40, 6, 1003, 12)])
def test_select(dev, B, K, V, N, half):
    x, scores, lengths, ended = inputs(V + N, B, K, V, half, dev)
    check(x, scores, N, got=ops.beam_select(x, scores, N))
    eos = sorted({V // 2, V - 1})
    got = ops.beam_select(x, scores, N, lengths=lengths, length_penalty=0.75, finished=ended,
                          eos_ids=torch.tensor(eos, dtype=torch.int32, device=dev), pad_id=V // 3)
    check(x, scores, N, lengths, 0.75, ended, eos, V // 3, got)
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("V,N", [(64, 64), (128, 128), (126, 100), (256, 128), (256, 70), (384, 100), (512, 128), (768, 97)])
def test_more_candidates_than_a_warps_lanes(dev, V, N, half):
    """Rows of whole warps' units, of which a warp has to give more candidates than it has lanes."""
    x, scores, lengths, _ = inputs(V * N, 3, 2, V, half, dev)
    check(x, scores, N, got=ops.beam_select(x, scores, N))
    scores[:, 1] = -float("inf")   # the other beam gives them all
    check(x, scores, N, lengths, 1.0, got=ops.beam_select(x, scores, N, lengths=lengths, length_penalty=1.0))
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("half", [False, True])
def test_ties_go_to_the_lowest_place(dev, half):
    """Rows of few values, rows all alike, and equal beams of equal scores, at odd rows too."""
    for V in (5000, 9001):
        x = torch.zeros((2, 4, V), device=dev)
        x[0, 1] = (torch.arange(V, device=dev) * 7 % 3).float()
        x[0, 2, 17::1000] = 2.0
        x[1] = x[0, 1]
        x[1, 3] = -0.0
        x = x.half() if half else x
        scores = torch.zeros((2, 4), device=dev)
        scores[0] = torch.tensor([-1.0, -2.5, -0.25, -4.0])
        for N in (4, 40, 128):
            got = ops.beam_select(x, scores, N)
            check(x, scores, N, got=got)
            # the equal beams of item 1: beam 0's candidates first, in order of their places
            best = torch.nonzero(x[1, 0] == 2.0)[:N, 0].int()
            assert torch.equal(got[0][1], best) and not got[1][1].any()
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("order", [1, -1])
def test_sorted_rows(dev, half, order):
    """Every later logit beats all earlier ones, or none does: the list is full, or idle."""
    V = 30000
    x = (torch.arange(V, device=dev, dtype=torch.float32) * (order * 2.0 ** -9)).expand(2, 2, V).contiguous()
    x = x.half() if half else x
    scores = torch.tensor([[0.0, -3.0], [-1.0, -1.5]], device=dev)
    check(x, scores, 64, got=ops.beam_select(x, scores, 64))
    ops.raise_device_errors(dev)


def test_masks_dead_beams_and_nothing_left(dev):
    x, scores, lengths, _ = inputs(5, 4, 3, 700, False, dev)
    x[0] = -float("inf")                     # nothing is left at all
    x[1, 0] = -float("inf")
    x[1, 1, 5:] = -float("inf")              # five tokens
    x[1, 2, :] = -float("inf")
    x[1, 2, 699] = -3.4e38                   # the type's lowest value is a value
    scores[2, :2] = -float("inf")            # the item's first step: one beam
    scores[3] = -float("inf")
    check(x, scores, 9, lengths, 1.0, got=ops.beam_select(x, scores, 9, lengths=lengths, length_penalty=1.0))
    ended = torch.ones((4, 3), dtype=torch.bool, device=dev)
    got = ops.beam_select(x, scores, 9, lengths=lengths, length_penalty=-0.5, finished=ended, pad_id=-7)
    check(x, scores, 9, lengths, -0.5, ended, (), -7, got)
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_values_that_are_not_finite(dev, bad):
    """They count as masked and are reported; a row of nothing else too."""
    x, scores, *_ = inputs(6, 3, 2, 9000, False, dev)
    x[0, 0, [0, 4000, 8999]] = bad
    x[1, 1] = bad
    clean = torch.where(torch.isfinite(x), x, -float("inf"))
    got = ops.beam_select(x, scores, 8)
    with pytest.raises(AnvilqError, match="nonfinite"):
        ops.raise_device_errors(dev)
    for a, b in zip(got, ops.beam_select(clean, scores, 8)):
        assert a is None or torch.equal(a, b)
    ops.raise_device_errors(dev)
    scores[2, 0] = bad
    got = ops.beam_select(clean, scores, 8)
    assert (got[1][2] == 1).all()
    with pytest.raises(AnvilqError, match="nonfinite"):
        ops.raise_device_errors(dev)


def test_strided_rows_and_types_of_rows(dev):
    x, scores, *_ = inputs(7, 3, 4, 1001, True, dev)
    want = ops.beam_select(x, scores, 4)
    wide = torch.full((12, 1040), 9.0, dtype=torch.float16, device=dev)
    for first in (0, 1, 2, 4, 8):            # rows on every alignment
        wide[:] = 9.0
        wide[:, first:first + 1001] = x.view(12, 1001)
        for y in (wide[:, first:first + 1001], wide.view(3, 4, 1040)[:, :, first:first + 1001]):
            for a, b in zip(ops.beam_select(y, scores, 4), want):
                assert a is None or torch.equal(a, b)
    one = ops.beam_select(x[:1], scores[:1].contiguous(), 4)
    assert torch.equal(one[0], want[0][:1])
    ops.raise_device_errors(dev)


def test_captured_replayed_and_side_by_side(dev):
    """Two graphs' replays overlap on two streams, with workspaces of their own; results repeat bit for bit."""
    sets = [inputs(20 + i, 4, 5, 20000, bool(i), dev) for i in range(2)]
    want = [ops.beam_select(x, s, 10, lengths=n, length_penalty=1.0, finished=e) for x, s, n, e in sets]
    graphs, outs = [], []
    for x, s, n, e in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ops.beam_select(x, s, 10, lengths=n, length_penalty=1.0, finished=e)
            h, = ops.beam_reorder([n], o[1])
        graphs.append(g)
        outs.append((*o, h))
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w, (_, _, n, _) in zip(outs, want, sets):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert torch.equal(o[5], n.gather(1, w[1].long()))
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("B,K,N", [(1, 1, 1), (3, 4, 4), (2, 5, 11), (70, 3, 6)])
def test_reorder(dev, B, K, N):
    rng = np.random.default_rng(B)
    parents = torch.from_numpy(rng.integers(-1, K, size=(B, N)).astype(np.int32)).to(dev)
    states = [torch.from_numpy(rng.integers(0, 100, size=(B, K, *rest))).to(kind).to(dev) for kind, rest in (
        (torch.int32, (77,)), (torch.float16, (3, 8)), (torch.uint8, (13,)), (torch.float32, ()), (torch.int64, (4099,)))]
    states = states * 8                      # more than one launch takes
    outs = [torch.full((B, N, *t.shape[2:]), 3, dtype=t.dtype, device=dev) for t in states]
    for got in (ops.beam_reorder(states, parents), ops.beam_reorder(states, parents, outs=outs)):
        for t, o in zip(states, got):
            at = parents.long().clamp(min=0).reshape(B, N, *[1] * (t.dim() - 2)).expand(B, N, *t.shape[2:])
            keep = (parents >= 0).reshape(B, N, *[1] * (t.dim() - 2))
            assert torch.equal(o, torch.where(keep, t.gather(1, at), torch.zeros_like(o)))
    assert ops.beam_reorder([], parents) == []
    ops.raise_device_errors(dev)
    ops.beam_reorder([states[0]], torch.full((B, N), K, dtype=torch.int32, device=dev))
    with pytest.raises(AnvilqError):
        ops.raise_device_errors(dev)
