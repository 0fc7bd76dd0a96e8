"""The paged-cache serving operators on the GPU against their 64-bit forms
(serving_oracle.py): the append with rotation into binary16 and 8-bit pages, attention
over 8-bit pages, the logits' penalties and masks, and all of them together.

Tolerances count roundings.  Binary16 outputs: half a step, 2^-11 of the value (2^-25 in
the subnormals).  A rotated value: two products and a sum, and cosines and sines good to
2 units in the last place (the bound CUDA documents for sincosf), 2^-22 (|a| + |b|) for
all of it.  Attention: the probabilities enter the tensor cores in binary16, 2^-11 of
sum p |v|; the scores' binary32 sums of D products of at most 2 |q| max |k| each (codes
are summed with an offset that at most doubles them; 8 accumulation steps of at most
2^-22 each) move a probability by a relative 2^-18 sum |q| max |k|, at most twice (in the
sum and in the product).  What a probability times its block's scale loses below
binary16's normal range: it enters as p s / F with F at most 8 times the scale s (or the
scale is 0) and p taken against a reference at least 4 (log2) below the stretch's largest
score, so that the sum of p is at least 2^4.  Its rounding there is at most 2^-25, of the
result 2^-25 8 / 2^4 sum |v| = 2^-26 sum |v|; merging stretches averages these."""
import numpy as np
import pytest
import torch

import serving_oracle as so
from anvilq_b200 import AnvilqError, _lib, ops

pytestmark = pytest.mark.gpu
BLOCK = so.BLOCK
THETA = 1e6
HALF = 2.0 ** -11


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def to(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def code_dtype(fp8):
    return torch.float8_e4m3fn if fp8 else torch.int8


def random_codes(rng, shape, fp8):
    x = rng.standard_normal(shape).astype(np.float32)
    t = torch.from_numpy(x)
    return (t * 100).clamp(-448, 448).to(torch.float8_e4m3fn) if fp8 else (t * 45).round().clamp(-127, 127).to(torch.int8)


def random_scales(rng, shape, fp8):
    s = 2.0 ** rng.integers(-10, -4, size=shape) if fp8 else rng.uniform(0.002, 0.05, size=shape)
    return torch.from_numpy(s.astype(np.float32))


# ---- append ------------------------------------------------------------------

def append_case(rng, before, new, Hq, Hkv, D, page, extra_pages=3, spare_rows=2):
    need = [-(-(p + n) // page) if n else 0 for p, n in zip(before, new)]
    pages = sum(need) + extra_pages
    table = so.make_table(need, pages, rng)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    qkv = rng.standard_normal((starts[-1] + spare_rows, (Hq + 2 * Hkv) * D)).astype(np.float16)
    return qkv, table, starts, np.array([p + n for p, n in zip(before, new)], np.int32), pages


def rows_of(starts, lens):
    """(sequence, position) of every new row."""
    return [(b, lens[b] - (starts[b + 1] - starts[b]) + i) for b in range(len(lens))
            for i in range(starts[b + 1] - starts[b])]


APPENDS = [
    ([0], [1], 2, 1, 64, 16),                                 # one first token
    ([5, 15, 16, 31], [1, 1, 1, 1], 14, 2, 64, 16),           # a decode step around block edges
    ([0, 0, 0], [1, 17, 40], 8, 2, 128, 32),                  # prompts, blocks cut at their ends
    ([3, 100, 7, 250], [50, 0, 9, 6], 4, 4, 128, 64),         # chunks after earlier ones, an idle sequence
    ([32700, 9], [60, 300], 14, 2, 64, 48),                   # far positions, pages of three blocks
    ([0] * 70, [1] * 70, 4, 2, 128, 16),                      # more than 32 sequences
    ([i % 23 for i in range(40)], [i % 5 for i in range(40)], 2, 1, 64, 16),   # many empty ones
    ([i % 40 for i in range(150)], [1 + i % 9 for i in range(150)], 32, 8, 128, 16),   # heads in slices
    ([(7 * i) % 50 for i in range(24)], [1 + i % 3 for i in range(24)], 9, 3, 128, 32),    # a token or two, odd heads
    ([3] * 9, [2, 1, 4, 0, 1, 3, 2, 1, 2], 7, 7, 64, 16),                                  # the same over block edges
]


@pytest.mark.parametrize("before,new,Hq,Hkv,D,page", APPENDS)
def test_append_binary16(dev, before, new, Hq, Hkv, D, page):
    rng = np.random.default_rng(11 + len(before))
    qkv, table, starts, lens, pages = append_case(rng, before, new, Hq, Hkv, D, page)
    T = qkv.shape[0]
    pools = [rng.standard_normal((pages, page, Hkv, D)).astype(np.float16) for _ in range(2)]
    k, v = to(pools[0], dev), to(pools[1], dev)
    q_out = torch.full((T, Hq, D), 7.0, dtype=torch.float16, device=dev)
    ops.paged_kv_append(to(qkv, dev), k, v, to(table, dev), to(lens, dev), to(starts, dev), Hq, THETA, q_out=q_out)
    ops.raise_device_errors(dev)
    rows = rows_of(starts, lens)
    n = len(rows)
    x = qkv[:n].reshape(n, Hq + 2 * Hkv, D)
    turned = so.rotate(x[:, :Hq + Hkv], [p for _, p in rows], THETA)
    pair = np.abs(x[:, :Hq + Hkv].astype(np.float64))
    pair = pair + np.roll(pair, D // 2, axis=2)
    tol = HALF * np.abs(turned) + 2.0 ** -22 * pair + 2.0 ** -25
    got = q_out.cpu().numpy().astype(np.float64)
    assert (np.abs(got[:n] - turned[:, :Hq]) <= tol[:, :Hq]).all()
    assert (got[n:] == 7.0).all(), "rows of no sequence are left as they were"
    want_v = pools[1].copy()
    gk, gv = k.cpu().numpy(), v.cpu().numpy()
    same_k = pools[0].copy()
    for r, (b, pos) in enumerate(rows):
        at = so.physical(table[b, pos // page]), pos % page
        assert (np.abs(gk[at].astype(np.float64) - turned[r, Hq:]) <= tol[r, Hq:]).all(), (b, pos)
        same_k[at] = gk[at]
        want_v[at] = x[r, Hq + Hkv:]
    assert np.array_equal(gv, want_v) and np.array_equal(gk, same_k), "only the new rows change"


def test_append_equals_the_single_token_call(dev):
    """One token of one sequence: bit for bit anvilq_rope_kv_append, far positions included."""
    rng = np.random.default_rng(5)
    Hq, Hkv, D, page = 14, 2, 64, 16
    lib = _lib.load()
    for pos in (0, 1, 1000, 32767):
        qkv, table, starts, lens, pages = append_case(rng, [pos], [1], Hq, Hkv, D, page, spare_rows=0)
        k = torch.zeros((pages, page, Hkv, D), dtype=torch.float16, device=dev)
        v = torch.zeros_like(k)
        q = ops.paged_kv_append(to(qkv, dev), k, v, to(table, dev), to(lens, dev), to(starts, dev), Hq, THETA)
        kc = torch.zeros((pos + 1, Hkv, D), dtype=torch.float16, device=dev)
        vc, q1 = torch.zeros_like(kc), torch.zeros((Hq, D), dtype=torch.float16, device=dev)
        p = torch.tensor([pos], dtype=torch.int32, device=dev)
        x = to(qkv, dev)
        assert lib.anvilq_rope_kv_append(x.data_ptr(), p.data_ptr(), q1.data_ptr(), kc.data_ptr(), vc.data_ptr(), None,
                                         Hq, Hkv, D, pos + 1, THETA, None, 0,
                                         torch.cuda.current_stream(dev).cuda_stream) == 0
        at = so.physical(table[0, pos // page]), pos % page
        assert torch.equal(q[0], q1) and torch.equal(k[at], kc[pos]) and torch.equal(v[at], vc[pos])
    ops.raise_device_errors(dev)


def check_block(values, codes, scale, x, err, kept, old_codes, old_scale, old_err, fp8):
    """A block of one head after an append: x [n, D] the exact new rows (good to err), kept rows re-coded."""
    top = np.abs(x).max()
    want = top / 127 if not fp8 else (2.0 ** np.ceil(np.log2(top / 448)) if top > 0 else 0.0)
    if kept:
        want = max(want, old_scale)
    slack = err.max() / (448 if fp8 else 127) + 2.0 ** -23 * want
    if fp8:   # a power of two: the neighbour only where the top value sits within its error of the border
        border = top > 0 and np.abs(np.log2(top / 448) - np.round(np.log2(top / 448))) < 2.0 ** -18
        assert scale == want or (border and scale in (want / 2, want * 2)), (scale, want)
    else:
        assert abs(scale - want) <= slack, (scale, want)
    if scale == 0:
        assert not codes[kept:kept + len(x)].any()
        return
    got = codes * scale
    if fp8:   # half a step of 3 fraction bits, or of the subnormals' step 2^-9
        half = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * scale)
    else:
        half = 0.5 * scale
    assert (np.abs(got[kept:kept + len(x)] - x) <= half * (1 + 2.0 ** -14) + err + 2.0 ** -22 * np.abs(x)).all()
    if kept:
        old = old_codes * old_scale
        half = np.maximum(2.0 ** -4 * np.abs(old), 2.0 ** -10 * scale) if fp8 else 0.5 * scale
        moved = np.abs(got[:kept] - old)
        assert (moved <= (half * (1 + 2.0 ** -14) + 2.0 ** -22 * np.abs(old) if scale > old_scale else 0)).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("before,new,Hq,Hkv,D,page", APPENDS)
def test_append_q8(dev, before, new, Hq, Hkv, D, page, fp8):
    rng = np.random.default_rng(31 + len(before))
    qkv, table, starts, lens, pages = append_case(rng, before, new, Hq, Hkv, D, page)
    qkv *= (4.0 ** rng.integers(-2, 3, size=(qkv.shape[0], 1))).astype(np.float16)   # tokens of unlike sizes
    shape = (pages, Hkv, page, D)
    old = [random_codes(rng, shape, fp8) for _ in range(2)]
    old_s = [random_scales(rng, (pages, Hkv, page // BLOCK), fp8) for _ in range(2)]
    k, v, ks, vs = (t.to(dev) for t in (*old, *old_s))
    q = ops.paged_kv_append_q8(to(qkv, dev), k, v, ks, vs, to(table, dev), to(lens, dev), to(starts, dev), Hq, THETA)
    ops.raise_device_errors(dev)
    rows = rows_of(starts, lens)
    n = len(rows)
    x = qkv[:n].reshape(n, Hq + 2 * Hkv, D)
    turned = so.rotate(x[:, :Hq + Hkv], [p for _, p in rows], THETA)
    pair = np.abs(x[:, :Hq + Hkv].astype(np.float64))
    err = 2.0 ** -22 * (pair + np.roll(pair, D // 2, axis=2))
    got_q = q.cpu().numpy()[:n].astype(np.float64)
    assert (np.abs(got_q - turned[:, :Hq]) <= HALF * np.abs(turned[:, :Hq]) + err[:, :Hq] + 2.0 ** -25).all()
    at_row = {bp: r for r, bp in enumerate(rows)}
    touched = set()
    for side, (pool, scales, exact, e) in enumerate((
            (k, ks, turned[:, Hq:], err[:, Hq:]),
            (v, vs, x[:, Hq + Hkv:].astype(np.float64), np.zeros((n, Hkv, D))))):
        codes, sc = so.codes_to_values(pool.cpu()), scales.cpu().numpy().astype(np.float64)
        prev, prev_s = so.codes_to_values(old[side]), old_s[side].numpy().astype(np.float64)
        raw, raw_prev = pool.cpu().view(torch.uint8).numpy(), old[side].view(torch.uint8).numpy().copy()
        sc_prev = prev_s.copy()
        for b in range(len(lens)):
            first = lens[b] - (starts[b + 1] - starts[b])
            pos = first
            while pos < lens[b]:
                end = min(lens[b], (pos // BLOCK + 1) * BLOCK)
                pg, slot = so.physical(table[b, pos // page]), pos % page
                blk, kept = slot // BLOCK, slot % BLOCK
                r = slice(at_row[(b, pos)], at_row[(b, pos)] + end - pos)
                blk_rows = slice(blk * BLOCK, (blk + 1) * BLOCK)
                for h in range(Hkv):
                    check_block(None, codes[pg, h, blk_rows], sc[pg, h, blk], exact[r, h], e[r, h], kept,
                                prev[pg, h, blk * BLOCK:slot], prev_s[pg, h, blk], 0, fp8)
                raw_prev[pg, :, blk * BLOCK:slot + end - pos] = raw[pg, :, blk * BLOCK:slot + end - pos]
                sc_prev[pg, :, blk] = sc[pg, :, blk]
                touched.add((pg, blk))
                pos = end
        assert np.array_equal(raw, raw_prev) and np.array_equal(sc, sc_prev), "nothing else changes"
    values = ops.kv_q8_values(k, v, ks, vs)
    for got, pool, scales in zip(values, (k, v), (ks, vs)):
        exact = so.pool_values(pool.cpu(), scales.cpu())
        assert (np.abs(got.cpu().numpy() - exact) <= HALF * np.abs(exact) + 2.0 ** -24 * np.abs(exact) + 2.0 ** -25).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_append_q8_values_bit_for_bit(dev, fp8):
    """v is not rotated: its codes and scales are the formulas' in binary32, token after
    token, each one growing the block's scale or not."""
    rng = np.random.default_rng(77)
    Hq, Hkv, D, page = 2, 2, 64, 16
    dtype = code_dtype(fp8)
    k = torch.zeros((2, Hkv, page, D), device=dev).to(dtype)
    v, ks = k.clone(), torch.zeros((2, Hkv, 1), device=dev)
    vs = torch.full_like(ks, 3.0)            # a stale scale: the first row replaces it
    table = to(np.array([[so.word(1)]], np.int32), dev)
    starts = to(np.array([0, 1], np.int32), dev)
    codes, scale = torch.zeros((Hkv, page, D)).to(dtype), torch.zeros(Hkv)
    for pos in range(16):
        qkv = (rng.standard_normal((1, (Hq + 2 * Hkv) * D)) * rng.choice([0.0, 0.01, 1, 3])).astype(np.float16)
        ops.paged_kv_append_q8(to(qkv, dev), k, v, ks, vs, table, to(np.array([pos + 1], np.int32), dev), starts, Hq)
        x = torch.from_numpy(qkv.astype(np.float32)).view(Hq + 2 * Hkv, D)[Hq + Hkv:]
        top = x.abs().amax(dim=1)
        if fp8:
            want = torch.where(top > 0, 2.0 ** torch.ceil(torch.log2(top.double() / 448)), 0.0).float()
        else:
            want = top / 127
        new = torch.maximum(scale, want)
        for h in range(Hkv):
            round_ = (lambda y: y.clamp(-448, 448).to(dtype)) if fp8 else (lambda y: y.round().clamp(-127, 127).to(dtype))
            if new[h] > scale[h] and pos:
                codes[h, :pos] = round_(codes[h, :pos].float() * (scale[h] / new[h]))
            codes[h, pos] = round_(x[h] * (1 / new[h])) if new[h] > 0 else torch.zeros(D).to(dtype)
        scale = new
        assert torch.equal(vs[1, :, 0].cpu(), scale), pos
        # -0 and +0 codes stand for the same value
        assert torch.equal(v[1].cpu().float()[:, :pos + 1], codes.float()[:, :pos + 1]), pos
    ops.raise_device_errors(dev)


def test_append_strided_rows_and_errors(dev):
    rng = np.random.default_rng(9)
    Hq, Hkv, D, page = 4, 2, 64, 16
    qkv, table, starts, lens, pages = append_case(rng, [0, 20], [5, 3], Hq, Hkv, D, page, spare_rows=0)
    wide = torch.zeros((8, 2 * qkv.shape[1]), dtype=torch.float16, device=dev)
    wide[:, :qkv.shape[1]] = to(qkv, dev)
    pool = lambda: torch.zeros((pages, page, Hkv, D), dtype=torch.float16, device=dev)
    k1, v1, k2, v2 = pool(), pool(), pool(), pool()
    args = to(table, dev), to(lens, dev), to(starts, dev), Hq
    a = ops.paged_kv_append(wide[:, :qkv.shape[1]], k1, v1, *args)
    b = ops.paged_kv_append(to(qkv, dev), k2, v2, *args)
    assert torch.equal(a, b) and torch.equal(k1, k2) and torch.equal(v1, v2)
    ops.raise_device_errors(dev)

    def fails(table, lens, starts, match):
        k, v = pool(), pool()
        ops.paged_kv_append(to(qkv, dev), k, v, to(table, dev), to(np.asarray(lens, np.int32), dev),
                            to(np.asarray(starts, np.int32), dev), Hq)
        with pytest.raises(AnvilqError, match=match):
            ops.raise_device_errors(dev)
        return k

    fails(table, [5, 2], starts, "length")               # more new tokens than tokens
    fails(table, [5, 16 * table.shape[1] + 1], starts, "length")
    fails(table, lens, [0, 5, 9], "length")              # a row past the last
    bad = table.copy()
    bad[1, 1] = so.word(pages)                           # past the pool
    k = fails(bad, lens, starts, "page")
    assert k[so.physical(table[0, 0]), :5].any()         # the other sequence is stored
    bad[1, 1] = so.word(1, valid=False)
    fails(bad, lens, starts, "page")
    # entries of pages without new tokens are not read
    fine = table.copy()
    fine[1, 0] = so.word(pages + 5)
    ops.paged_kv_append(to(qkv, dev), pool(), pool(), to(fine, dev), *args[1:])
    ops.raise_device_errors(dev)


def test_append_q8_not_finite(dev):
    rng = np.random.default_rng(10)
    Hq, Hkv, D, page = 2, 1, 64, 16
    qkv, table, starts, lens, pages = append_case(rng, [0], [3], Hq, Hkv, D, page, spare_rows=0)
    qkv[1, (Hq + Hkv) * D + 5] = np.inf
    qkv[2, (Hq + Hkv) * D + 6] = np.nan
    k, v, ks, vs = (t.to(dev) for t in (random_codes(rng, (pages, Hkv, page, D), False),
                                       random_codes(rng, (pages, Hkv, page, D), False),
                                       random_scales(rng, (pages, Hkv, 1), False), random_scales(rng, (pages, Hkv, 1), False)))
    ops.paged_kv_append_q8(to(qkv, dev), k, v, ks, vs, to(table, dev), to(lens, dev), to(starts, dev), Hq)
    with pytest.raises(AnvilqError):
        ops.raise_device_errors(dev)
    pg = so.physical(table[0, 0])
    assert v[pg, 0, 1, 5] == 0 and v[pg, 0, 2, 6] == 0
    x = qkv[:, (Hq + Hkv) * D:].astype(np.float32)
    assert vs[pg, 0, 0].item() == np.abs(x[np.isfinite(x)]).max() / np.float32(127)


@pytest.mark.parametrize("fp8", [False, True])
def test_append_q8_step_not_finite(dev, fp8):
    """Of a decode step's tokens only the values that are not finite are lost."""
    rng = np.random.default_rng(22)
    B, Hq, Hkv, D, page = 4, 3, 3, 128, 16
    qkv, table, starts, lens, pages = append_case(rng, [0, 3, 15, 16], [1] * B, Hq, Hkv, D, page, spare_rows=0)
    clean = qkv.copy()
    at = (Hq + Hkv) * D + 130                                 # head 1 of V, dim 2
    for b, bad in ((1, np.inf), (2, np.nan), (3, -np.inf)):
        qkv[b, at] = bad
        clean[b, at] = 0
    ends = []
    for x in (qkv, clean):
        k = torch.zeros((pages, Hkv, page, D), device=dev).to(code_dtype(fp8))
        v, ks, vs = k.clone(), *(torch.zeros((pages, Hkv, 1), device=dev) for _ in range(2))
        q = ops.paged_kv_append_q8(to(x, dev), k, v, ks, vs, to(table, dev), to(lens, dev), to(starts, dev), Hq)
        if x is qkv:
            with pytest.raises(AnvilqError):
                ops.raise_device_errors(dev)
        ends.append([q, k.view(torch.uint8), v.view(torch.uint8), ks, vs])
    ops.raise_device_errors(dev)
    for a, b in zip(*ends):
        assert torch.equal(a, b)


# ---- attention ----------------------------------------------------------------

def attention_case(dev, rng, lens, Q, Hq, Hkv, D, page, fp8, width=None):
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    table = so.make_table(need, pages, rng, width)
    k, v = (random_codes(rng, (pages, Hkv, page, D), fp8) for _ in range(2))
    ks, vs = (random_scales(rng, (pages, Hkv, page // BLOCK), fp8) for _ in range(2))
    q = (rng.standard_normal((len(lens), Q, Hq, D)) * 2).astype(np.float16)
    return q, k, v, ks, vs, table


def check_attention(out, q, k, v, ks, vs, table, lens, scale=0.0):
    B, Q, Hq, D = q.shape
    page, Hkv = k.shape[2], k.shape[1]
    kv, vv = so.pool_values(k.cpu(), ks.cpu()), so.pool_values(v.cpu(), vs.cpu())
    scale = scale or 1 / np.sqrt(D)
    for b, n in enumerate(lens):
        at = [so.physical(e) for e in table[b, :-(-n // page)]]
        flat = lambda p: p[at].transpose(0, 2, 1, 3).reshape(-1, Hkv, D)[:n]
        ref, mass, reach, size = so.attention(q[b].astype(np.float64), flat(kv), flat(vv), n, Q, scale)
        tol = HALF * np.abs(ref) + mass * (HALF * (1 + 2.0 ** -6) + 2 * 2.0 ** -18 * reach) + 2.0 ** -24 + 2.0 ** -26 * size
        bad = np.abs(out[b].astype(np.float64) - ref) > tol
        assert not bad.any(), (b, n, np.argwhere(bad)[:4], np.abs(out[b] - ref).max())


ATTENTIONS = [
    # lens, Q, Hq, Hkv, D, page
    ([1], 1, 1, 1, 64, 16),
    ([15, 16, 17], 1, 14, 2, 64, 16),
    ([150], 1, 14, 2, 64, 48),
    ([0, 1, 33, 0, 700], 1, 32, 8, 128, 64),        # idle slots
    ([2500, 31], 1, 8, 8, 128, 256),                # no grouping, a sequence inside one page
    ([5000], 1, 16, 2, 128, 16),                    # group of 8
    ([640, 100], 1, 24, 2, 64, 32),                 # group of 12
    ([100, 0, 3, 900], 4, 8, 2, 128, 16),           # drafts; fewer tokens than queries
    ([257, 1000], 5, 14, 2, 64, 64),                # 35 query rows a head
    ([70], 64, 4, 4, 64, 16),                       # the widest chunk
    ([33] * 40, 1, 8, 8, 64, 16),                   # more than 32 sequences, many short pairs
    ([20000], 2, 4, 1, 128, 128),                   # one long pair over the whole device
    ([40000], 3, 4, 1, 64, 32),                     # the same with more than 8 rows
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lens,Q,Hq,Hkv,D,page", ATTENTIONS)
def test_attention_q8(dev, lens, Q, Hq, Hkv, D, page, fp8):
    rng = np.random.default_rng(sum(lens) + Q)
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, Q, Hq, Hkv, D, page, fp8)
    a = [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array(lens, np.int32), dev)]
    qd = to(q, dev)
    out = ops.gqa_decode_q8(qd, *a)
    again = ops.gqa_decode_q8(qd, *a, out=torch.full_like(qd, float("nan")))
    ops.raise_device_errors(dev)
    assert torch.equal(out, again), "not run-to-run deterministic"
    check_attention(out.cpu().numpy(), q, k, v, ks, vs, table, lens)
    if Q == 1:
        assert torch.equal(ops.gqa_decode_q8(qd[:, 0], *a, scale=float(1 / np.sqrt(D))), out[:, 0])


@pytest.mark.parametrize("B,top,Hq,Hkv,D", [(33, 60, 4, 2, 64), (200, 90, 16, 2, 128), (2500, 20, 2, 1, 64)])
def test_attention_q8_many_sequences(dev, B, top, Hq, Hkv, D):
    """More sequences than a warp looks over at once, idle slots and lengths out of range among them."""
    rng = np.random.default_rng(B)
    lens = rng.integers(0, top + 1, B)
    lens[rng.integers(0, B, B // 5)] = 0
    q, k, v, ks, vs, table = attention_case(dev, rng, [int(n) for n in lens], 1, Hq, Hkv, D, 16, False)
    a = [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev)]
    out = ops.gqa_decode_q8(to(q, dev), *a, to(lens.astype(np.int32), dev), out=torch.full(q.shape, float("nan"), dtype=torch.float16, device=dev))
    ops.raise_device_errors(dev)
    check_attention(out.cpu().numpy(), q, k, v, ks, vs, table, [int(n) for n in lens])
    bad = rng.choice(B, 3, replace=False)
    lens[bad] = [-7, 16 * table.shape[1] + 1, 2 ** 31 - 1]
    out = ops.gqa_decode_q8(to(q, dev), *a, to(lens.astype(np.int32), dev))
    with pytest.raises(AnvilqError, match="length"):
        ops.raise_device_errors(dev)
    lens[bad] = 0
    check_attention(out.cpu().numpy(), q, k, v, ks, vs, table, [int(n) for n in lens])


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_q8_unlike_scales(dev, fp8):
    """Blocks whose scales differ by many orders, all-zero blocks, scores far apart, another softmax scale."""
    rng = np.random.default_rng(3)
    lens = [400, 900]
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, 1, 8, 2, 128, 16, fp8)
    vs *= torch.from_numpy((2.0 ** rng.integers(-30, 12, size=vs.shape)).astype(np.float32))
    ks *= torch.from_numpy((2.0 ** rng.integers(-6, 3, size=ks.shape)).astype(np.float32))
    zero = torch.from_numpy(rng.random(vs.shape) < 0.2)
    vs[zero] = 0.0
    ks[torch.from_numpy(rng.random(ks.shape) < 0.1)] = 0.0
    a = [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array(lens, np.int32), dev)]
    out = ops.gqa_decode_q8(to(q, dev), *a, scale=0.3)
    ops.raise_device_errors(dev)
    check_attention(out.cpu().numpy(), q, k, v, ks, vs, table, lens, scale=0.3)


def test_attention_q8_ignores_what_is_not_live(dev):
    """NaN codes and scales behind a sequence's end, in its last block and in other pages, do not reach the output."""
    rng = np.random.default_rng(4)
    lens = [19, 64, 200]
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, 1, 8, 2, 64, 64, True)
    clean = [t.to(dev) for t in (k, v, ks, vs)]
    d_table, d_lens = to(table, dev), to(np.array(lens, np.int32), dev)
    ref = ops.gqa_decode_q8(to(q, dev), *clean, d_table, d_lens)
    live = np.zeros((k.shape[0], 64), bool)
    for b, n in enumerate(lens):
        for t in range(n):
            live[so.physical(table[b, t // 64]), t % 64] = True
    dead = torch.from_numpy(~live)
    for codes in (k, v):
        codes.view(torch.uint8).transpose(1, 2)[dead] = 0x7F     # e4m3's NaN
    dead_blocks = torch.from_numpy(~live.reshape(-1, 4, BLOCK).any(axis=2))
    for s in (ks, vs):
        s.transpose(1, 2)[dead_blocks] = float("nan")
    out = ops.gqa_decode_q8(to(q, dev), *(t.to(dev) for t in (k, v, ks, vs)), d_table, d_lens)
    ops.raise_device_errors(dev)
    assert torch.equal(out, ref)


def test_attention_q8_bad_pages_and_lengths(dev):
    rng = np.random.default_rng(6)
    lens = [100, 40]
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, 1, 8, 2, 64, 16, False)
    pools = [t.to(dev) for t in (k, v, ks, vs)]
    run = lambda t, n: ops.gqa_decode_q8(to(q, dev), *pools, to(t, dev), to(np.array(n, np.int32), dev))
    for word in (so.word(3, valid=False), so.word(k.shape[0]), so.word(0x7FFFFFFF)):
        bad = table.copy()
        bad[0, 2] = word
        run(bad, lens)
        with pytest.raises(AnvilqError, match="page"):
            ops.raise_device_errors(dev)
    for n in ([-1, 40], [16 * table.shape[1] + 1, 40], [2 ** 31 - 1, 40], [-2 ** 31, 40]):
        out = run(table, n)
        with pytest.raises(AnvilqError, match="length"):
            ops.raise_device_errors(dev)
        assert not out[0].any()
        check_attention(out[1:].cpu().numpy(), q[1:], k, v, ks, vs, table[1:], lens[1:])
    # entries behind the live pages are not read
    fine = table.copy()
    fine[1, 3:] = so.word(k.shape[0] + 9)
    out = run(fine, lens)
    ops.raise_device_errors(dev)
    check_attention(out.cpu().numpy(), q, k, v, ks, vs, table, lens)


# ---- logits ---------------------------------------------------------------------

def logits_case(rng, B, V, L, half, zipf=True):
    x = (rng.standard_normal((B, V)) * 3).astype(np.float16 if half else np.float32)
    history = np.minimum((rng.random((B, L)) ** (4 if zipf else 1) * V).astype(np.int32), V - 1)
    lens = np.array([L] + [int(n) for n in rng.integers(0, L + 1, size=B - 1)], np.int32)
    prompts = np.array([int(rng.integers(0, n + 1)) for n in lens], np.int32)
    f = lambda lo, hi: rng.uniform(lo, hi, B).astype(np.float32)
    return x, history, lens, prompts, f(0.8, 1.5), f(-0.5, 1.0), f(-0.2, 0.5)


def check_logits(dev, x, out, tokens, ref_args):
    ref32, token32 = so.logits(x, *ref_args, real=np.float32)
    ref64, _ = so.logits(x, *ref_args)
    got = out.cpu().numpy()
    assert np.array_equal(got, ref32, equal_nan=True)           # the formula, each operation rounded
    fine = np.isfinite(ref64)
    assert np.array_equal(fine, np.isfinite(got))
    # five roundings of values no larger than the largest that the row's formula passes through
    size = np.abs(x.astype(np.float64)) * 2 + 600 + np.abs(np.where(fine, ref64, 0))
    assert (np.abs(got[fine] - ref64[fine]) <= 5 * 2.0 ** -24 * size[fine]).all()
    assert tokens.tolist() == token32


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("B,V,L,biases,grammar", [
    (1, 1, 1, 0, False), (1, 31, 5, 2, True), (3, 1000, 50, 7, True), (2, 4097, 300, 0, True), (5, 33, 0, 3, False),
    (4, 151936, 900, 20, True), (70, 700, 40, 5, True),
])
def test_logits(dev, B, V, L, biases, grammar, half):
    rng = np.random.default_rng(B * V + L)
    x, history, lens, prompts, rep, pres, freq = logits_case(rng, B, V, L, half)
    bias = [[(int(t), float(np.float32(w))) for t, w in zip(rng.integers(0, V, n), rng.standard_normal(n) * 5)]
            for n in rng.integers(0, biases + 1, size=B)] if biases else None
    allowed = (rng.random((B, V)) < rng.choice([0.02, 0.5, 1.0], size=(B, 1))) if grammar else None
    kw = {}
    if bias is not None:
        flat = [e for row in bias for e in row]
        kw = dict(bias_starts=to(np.concatenate([[0], np.cumsum([len(r) for r in bias])]).astype(np.int32), dev),
                  bias_ids=to(np.array([t for t, _ in flat], np.int32), dev),
                  bias_values=to(np.array([w for _, w in flat], np.float32), dev))
    if grammar:
        kw["allowed"] = to(so.pack_mask(allowed), dev)
    d = lambda a: to(a, dev)
    out, tokens = ops.logits_process(d(x), history=d(history), history_lens=d(lens), prompt_lens=d(prompts),
                                     repetition=d(rep), presence=d(pres), frequency=d(freq), **kw)
    ops.raise_device_errors(dev)
    check_logits(dev, x, out, tokens, (history, lens, prompts, rep, pres, freq, bias, allowed))
    # the choice alone, and the logits alone
    only = ops.logits_process(d(x), history=d(history), history_lens=d(lens), prompt_lens=d(prompts),
                              repetition=d(rep), presence=d(pres), frequency=d(freq), write_logits=False, **kw)
    assert only[0] is None and torch.equal(only[1], tokens)
    rest = ops.logits_process(d(x), history=d(history), history_lens=d(lens), prompt_lens=d(prompts),
                              repetition=d(rep), presence=d(pres), frequency=d(freq), choose=False, **kw)
    assert rest[1] is None and torch.equal(rest[0], out)


def test_logits_long_histories(dev):
    """A row a CTA, with more special tokens than its tables hold at a time, and a
    history longer than a CTA keeps; in place and not."""
    rng = np.random.default_rng(19)
    B, V, L, n = 600, 5000, 4500, 300
    x, history, lens, prompts, rep, pres, freq = logits_case(rng, B, V, L, False, zipf=False)
    lens[:] = L - np.arange(B) % 7
    prompts = np.minimum(prompts, lens)
    d = lambda a: to(a, dev)
    ids, w = rng.integers(0, V, (B, n)).astype(np.int32), rng.standard_normal((B, n)).astype(np.float32)
    allowed = rng.random((B, V)) < 0.7
    kw = dict(history=d(history), history_lens=d(lens), prompt_lens=d(prompts), repetition=d(rep), presence=d(pres),
              frequency=d(freq), bias_starts=d(np.arange(0, B * n + 1, n, dtype=np.int32)), bias_ids=d(ids.ravel()),
              bias_values=d(w.ravel()), allowed=d(so.pack_mask(allowed)))
    out, tokens = ops.logits_process(d(x), **kw)
    ops.raise_device_errors(dev)
    bias = [[(int(t), float(v)) for t, v in zip(ids[b], w[b])] for b in range(B)]
    check_logits(dev, x, out, tokens, (history, lens, prompts, rep, pres, freq, bias, allowed))
    same = d(x)
    again, tokens2 = ops.logits_process(same, out=same, **kw)
    assert torch.equal(again, out) and torch.equal(tokens2, tokens)


@pytest.mark.parametrize("B,V,L", [(1, 33000, 9000), (3, 70001, 5000), (2, 151936, 20000)])
@pytest.mark.parametrize("bias", [False, True])
def test_logits_histories_of_several_ctas(dev, B, V, L, bias):
    """More tokens of history than a CTA keeps, most of them at one end of the vocabulary,
    over several CTAs of a row; prompts that are all of it, none, or out of range."""
    rng = np.random.default_rng(L)
    x, history, lens, prompts, rep, pres, freq = logits_case(rng, B, V, L, B == 3)
    lens[:] = [L, L - 77, 2049][:B]
    d = lambda a: to(a, dev)
    lists = [[(int(t), float(w)) for t, w in zip(rng.integers(0, V, 50), rng.standard_normal(50).astype(np.float32))]
             for _ in range(B)] if bias else None
    kw = dict(bias_starts=d(np.arange(0, 50 * B + 1, 50, dtype=np.int32)),
              bias_ids=d(np.array([t for r in lists for t, _ in r], np.int32)),
              bias_values=d(np.array([w for r in lists for _, w in r], np.float32))) if bias else {}
    for prompts in ([L, 0, 2048], [-5, 2**31 - 1, 2049], [L - 1, 3000, -2**31]):
        prompts = np.array(prompts[:B], np.int64).astype(np.int32)
        out, tokens = ops.logits_process(d(x), history=d(history), history_lens=d(lens), prompt_lens=d(prompts),
                                         repetition=d(rep), presence=d(pres), frequency=d(freq), **kw)
        ops.raise_device_errors(dev)
        check_logits(dev, x, out, tokens, (history, lens, prompts, rep, pres, freq, lists, None))
    out, tokens = ops.logits_process(d(x), history=d(history), history_lens=d(lens), repetition=d(rep), **kw)
    check_logits(dev, x, out, tokens, (history, lens, None, rep, None, None, lists, None))


def test_logits_rows_that_take_turns_or_overlap(dev):
    rng = np.random.default_rng(20)
    x = rng.standard_normal((3, 64)).astype(np.float32)
    both = torch.zeros((3, 128), device=dev)
    both[:, :64] = to(x, dev)
    out, _ = ops.logits_process(both[:, :64], out=both[:, 64:])
    assert np.array_equal(out.cpu().numpy(), x) and np.array_equal(both[:, :64].cpu().numpy(), x)
    flat = torch.zeros(300, device=dev)
    rows = flat[:192].view(3, 64)
    for logits, bad in ((rows, flat[4:196].view(3, 64)), (rows, flat[:228].view(3, 76)[:, :64]),
                        (both[:, :64], both[:, 32:96])):
        with pytest.raises(AnvilqError):
            ops.logits_process(logits, out=bad)
    with pytest.raises(AnvilqError):                       # binary16 logits under their own results
        ops.logits_process(flat[:192].view(torch.float16).view(3, 128)[:, :64], out=rows)
    ops.raise_device_errors(dev)


def test_logits_empty_history(dev):
    x = torch.ones((2, 40), device=dev)
    none = torch.zeros((2, 0), dtype=torch.int32, device=dev)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    out, _ = ops.logits_process(x, history=none, history_lens=lens, presence=torch.ones(2, device=dev))
    assert torch.equal(out, x)
    ops.raise_device_errors(dev)
    ops.logits_process(x, history=none, history_lens=lens + 1)
    with pytest.raises(AnvilqError, match="length"):
        ops.raise_device_errors(dev)


def test_append_without_tokens(dev):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    qkv = torch.zeros((0, 6 * 64), dtype=torch.float16, device=dev)
    pool = torch.zeros((2, 16, 1, 64), dtype=torch.float16, device=dev)
    table = torch.zeros((1, 1), dtype=torch.int32, device=dev)
    assert ops.paged_kv_append(qkv, pool, pool.clone(), table, i32(3), i32(0, 0), 4).shape == (0, 4, 64)
    codes, scales = torch.zeros((2, 1, 16, 64), dtype=torch.int8, device=dev), torch.zeros((2, 1, 1), device=dev)
    assert ops.paged_kv_append_q8(qkv, codes, codes.clone(), scales, scales.clone(), table, i32(3), i32(0, 0), 4).shape == (0, 4, 64)
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("given", [(), ("repetition",), ("presence",), ("frequency",), ("allowed",), ("bias",)])
def test_logits_parts_alone(dev, given):
    """Each part without the others; rows that share masks or have none; prompt lengths left out."""
    rng = np.random.default_rng(12)
    B, V, L = 4, 501, 30
    x, history, lens, _, rep, pres, freq = logits_case(rng, B, V, L, False)
    d = lambda a: to(a, dev)
    kw, ref = {}, dict(history=None, lens=None, prompts=None, rep=None, pres=None, freq=None, bias=None, allowed=None)
    if given and given[0] in ("repetition", "presence", "frequency"):
        value = dict(repetition=rep, presence=pres, frequency=freq)[given[0]]
        kw = dict(history=d(history), history_lens=d(lens), **{given[0]: d(value)})
        ref.update(history=history, lens=lens, **{given[0][:4] if given[0] != "repetition" else "rep": value})
    if "allowed" in given:
        masks = rng.random((2, V)) < 0.1
        pick = np.array([1, -1, 0, 1], np.int32)
        kw = dict(allowed=d(so.pack_mask(masks)), allowed_rows=d(pick))
        ref["allowed"] = [None if p < 0 else masks[p] for p in pick]
    if "bias" in given:
        bias = [[(5, 2.0), (7, -1.0), (5, 30.0)], [], [(0, 1.5)], [(500, 9.0), (500, -9.0)]]
        flat = [e for row in bias for e in row]
        kw = dict(bias_starts=d(np.array([0, 3, 3, 4, 6], np.int32)), bias_ids=d(np.array([t for t, _ in flat], np.int32)),
                  bias_values=d(np.array([w for _, w in flat], np.float32)))
        ref["bias"] = bias
    out, tokens = ops.logits_process(d(x), **kw)
    ops.raise_device_errors(dev)
    check_logits(dev, x, out, tokens, tuple(ref.values()))


def test_logits_odd_values(dev):
    """Infinities, NaN, ties, rows with nothing allowed, the type's lowest value, -0 against +0."""
    V = 200
    x = np.full((8, V), -1.0, np.float32)
    x[0, [17, 90]] = 5.0                        # a tie: the lower index
    x[1] = -np.inf                              # nothing to choose from
    x[2, 3] = np.nan
    x[2, 150] = np.inf
    x[3] = np.nan
    x[4] = np.finfo(np.float32).min             # still a value
    x[5] = 2.0
    x[6, :] = -0.0
    x[6, 100] = 0.0                             # equal to the -0 before it
    x[7, 199] = 8.0
    allowed = np.ones((8, V), bool)
    allowed[5] = False                          # an empty mask
    allowed[7, 199] = False
    out, tokens = ops.logits_process(to(x, dev), allowed=to(so.pack_mask(allowed), dev))
    ops.raise_device_errors(dev)
    assert tokens.tolist() == [17, -1, 150, -1, 0, -1, 0, 0]
    want = x.copy()
    want[~allowed] = -np.inf
    assert np.array_equal(out.cpu().numpy(), want, equal_nan=True)


def test_logits_in_place_strided_and_unaligned(dev):
    rng = np.random.default_rng(21)
    B, V, L = 3, 1003, 64
    x, history, lens, prompts, rep, pres, freq = logits_case(rng, B, V, L, False)
    d = lambda a: to(a, dev)
    kw = dict(history=d(history), history_lens=d(lens), prompt_lens=d(prompts), repetition=d(rep), presence=d(pres),
              frequency=d(freq))
    ref, token = ops.logits_process(d(x), **kw)
    wide = torch.full((B, V + 21), 99.0, device=dev)             # a padded vocabulary
    wide[:, 1:V + 1] = d(x)                                      # not 16-byte aligned
    view = wide[:, 1:V + 1]
    out, again = ops.logits_process(view, out=view, **kw)
    assert out is view and torch.equal(view, ref) and torch.equal(again, token)
    assert (wide[:, 0] == 99).all() and (wide[:, V + 1:] == 99).all()
    half = torch.zeros((B, V + 8), dtype=torch.float16, device=dev)[:, 3:V + 3]
    half.copy_(d(x))
    a = ops.logits_process(half, **kw)
    b = ops.logits_process(half.contiguous(), **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ops.raise_device_errors(dev)


def test_logits_bad_ids_and_ranges(dev):
    x = torch.zeros((2, 100), device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    one = torch.ones(2, device=dev)

    def fails(match, **kw):
        out, tokens = ops.logits_process(x, **kw)
        with pytest.raises(AnvilqError, match=match):
            ops.raise_device_errors(dev)
        return out, tokens

    history = torch.tensor([[1, 100], [-1, 2]], dtype=torch.int32, device=dev)
    out, tokens = fails("token", history=history, history_lens=i32(2, 2), presence=one)
    assert out[0, 1] == -1 and out[1, 2] == -1 and tokens.tolist() == [0, 0]     # the good ids count
    fails("length", history=history, history_lens=i32(1, 3), presence=one)
    fails("length", history=history, history_lens=i32(1, -1), presence=one)
    fails("token", bias_starts=i32(0, 1, 1), bias_ids=i32(100), bias_values=torch.ones(1, device=dev))
    fails("length", bias_starts=i32(0, 1, 2), bias_ids=i32(5), bias_values=torch.ones(1, device=dev))
    fails("length", allowed=torch.full((1, 4), -1, dtype=torch.int32, device=dev), allowed_rows=i32(0, 1))


# ---- together ---------------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
def test_serving_steps_together(dev, fp8):
    """Prompts, then decode steps captured once and replayed on their own stream, then a
    drafted chunk: the cache that append writes is the one that attention reads, and the
    chosen tokens are those of the formulas."""
    rng = np.random.default_rng(55)
    B, Hq, Hkv, D, page, width, V = 3, 8, 2, 64, 32, 5, 500
    pages = B * width + 1
    table = so.make_table([width] * B, pages, rng)
    shape = (pages, Hkv, page, D)
    codes = lambda: torch.zeros(shape, device=dev).to(code_dtype(fp8))
    k, v, ks, vs = codes(), codes(), *(torch.zeros((pages, Hkv, page // BLOCK), device=dev) for _ in range(2))
    t = to(table, dev)
    head = to(rng.standard_normal((Hq * D, V)).astype(np.float32) * 0.1, dev)
    lens = np.array([0, 0, 0])

    def expect(out, q, Q):
        kc, vc = k.cpu(), v.cpu()
        check_attention(out.cpu().numpy().reshape(B, Q, Hq, D), q.cpu().numpy().reshape(B, Q, Hq, D), kc, vc, ks, vs,
                        table, [int(n) for n in lens])

    def qkv_of(n):
        return to(rng.standard_normal((n, (Hq + 2 * Hkv) * D)).astype(np.float16), dev)

    new = np.array([37, 16, 50])
    lens = lens + new
    starts = to(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), dev)
    ops.paged_kv_append_q8(qkv_of(int(new.sum())), k, v, ks, vs, t, to(lens.astype(np.int32), dev), starts, Hq)
    # decode steps: one graph, replayed with new rows and lengths
    x, d_lens = qkv_of(B), to(lens.astype(np.int32), dev)
    one = to(np.arange(B + 1, dtype=np.int32), dev)
    history = torch.zeros((B, 8), dtype=torch.int32, device=dev)
    hist_lens = torch.zeros(B, dtype=torch.int32, device=dev)
    rep, pres = torch.full((B,), 1.3, device=dev), torch.full((B,), 0.5, device=dev)
    results = {}

    def step():
        q = ops.paged_kv_append_q8(x, k, v, ks, vs, t, d_lens, one, Hq)
        out = ops.gqa_decode_q8(q, k, v, ks, vs, t, d_lens)
        raw = out.float().reshape(B, -1) @ head
        results.update(q=q, out=out, raw=raw)
        results["logits"], results["tokens"] = ops.logits_process(raw, history=history, history_lens=hist_lens,
                                                                  repetition=rep, presence=pres)

    lens = lens + 1
    d_lens.copy_(to(lens.astype(np.int32), dev))
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    expect(results["out"], results["q"], 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    for i in range(1, 6):
        x.copy_(qkv_of(B))
        lens = lens + 1
        d_lens.copy_(to(lens.astype(np.int32), dev))
        graph.replay()
        torch.cuda.synchronize(dev)
        ops.raise_device_errors(dev)
        expect(results["out"], results["q"], 1)
        ref, tokens = so.logits(results["raw"].cpu().numpy(), history.cpu().numpy(), hist_lens.cpu().numpy(), None,
                                rep.cpu().numpy(), pres.cpu().numpy(), None, None, None, real=np.float32)
        assert np.array_equal(results["logits"].cpu().numpy(), ref) and results["tokens"].tolist() == tokens
        history[:, i - 1] = results["tokens"]
        hist_lens += 1
    # a drafted chunk of four tokens of each sequence
    Q = 4
    lens = lens + Q
    d_lens.copy_(to(lens.astype(np.int32), dev))
    q = ops.paged_kv_append_q8(qkv_of(B * Q), k, v, ks, vs, t, d_lens, to(np.arange(0, B * Q + 1, Q, dtype=np.int32), dev),
                               Hq)
    out = ops.gqa_decode_q8(q.view(B, Q, Hq, D), k, v, ks, vs, t, d_lens)
    ops.raise_device_errors(dev)
    expect(out, q, Q)


def test_binary16_pages_append_then_attend(dev):
    """paged_kv_append fills the pools that gqa_decode_paged reads."""
    rng = np.random.default_rng(8)
    Hq, Hkv, D, page = 8, 2, 128, 16
    new = [70, 33]
    qkv, table, starts, lens, pages = append_case(rng, [0, 0], new, Hq, Hkv, D, page, spare_rows=0)
    k = torch.zeros((pages, page, Hkv, D), dtype=torch.float16, device=dev)
    v = torch.zeros_like(k)
    q = ops.paged_kv_append(to(qkv, dev), k, v, to(table, dev), to(lens, dev), to(starts, dev), Hq, THETA)
    last = q[torch.tensor([n - 1 for n in starts[1:]], device=dev)].contiguous()
    out = ops.gqa_decode_paged(last, k, v, to(table, dev), to(lens, dev)).cpu().numpy().astype(np.float64)
    ops.raise_device_errors(dev)
    for b in range(2):
        at = [so.physical(e) for e in table[b, :-(-lens[b] // page)]]
        flat = lambda p: p.cpu().numpy()[at].reshape(-1, Hkv, D)[:lens[b]].astype(np.float64)
        ref, mass, reach, _ = so.attention(last[b:b + 1].cpu().numpy().astype(np.float64), flat(k), flat(v), int(lens[b]), 1,
                                        1 / np.sqrt(D))
        tol = HALF * np.abs(ref) + mass * (HALF * (1 + 2.0 ** -6) + 2 * 2.0 ** -18 * reach) + 2.0 ** -24
        assert (np.abs(out[b] - ref[0]) <= tol[0]).all()


def test_graphs_of_one_stream_do_not_share_a_workspace(dev):
    """Two captured calls, replayed at once on two streams."""
    rng = np.random.default_rng(14)
    lens = [4000]
    cases, graphs = [], []
    s = torch.cuda.Stream(dev)
    for seed in range(2):
        q, k, v, ks, vs, table = attention_case(dev, rng, lens, 1, 8, 2, 128, 16, False)
        a = [to(q, dev)] + [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array(lens, np.int32), dev)]
        with torch.cuda.stream(s):
            ref = ops.gqa_decode_q8(*a)
        s.synchronize()
        out = torch.empty_like(ref)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            ops.gqa_decode_q8(*a, out=out)
        cases.append((a, ref, out))
        graphs.append(g)
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    torch.cuda.synchronize(dev)
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize(dev)
    ops.raise_device_errors(dev)
    for _, ref, out in cases:
        assert torch.equal(ref, out)


def test_caller_workspace(dev):
    rng = np.random.default_rng(15)
    q, k, v, ks, vs, table = attention_case(dev, rng, [300], 1, 8, 2, 64, 16, False)
    a = [to(q, dev)] + [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array([300], np.int32), dev)]
    need = _lib.load().anvilq_gqa_decode_q8_workspace_size(1, 1, 8, 2, 64)
    ws = torch.zeros(need, dtype=torch.uint8, device=dev)
    assert torch.equal(ops.gqa_decode_q8(*a, workspace=ws), ops.gqa_decode_q8(*a))
    assert not ws[:65536].any(), "the counters are left zero"
    with pytest.raises(ValueError):
        ops.gqa_decode_q8(*a, workspace=ws[:need - 1])
    ops.raise_device_errors(dev)


def test_two_streams_at_once(dev):
    """Eager calls on two streams, each stream with its own workspace."""
    rng = np.random.default_rng(16)
    q, k, v, ks, vs, table = attention_case(dev, rng, [3000, 700], 1, 8, 2, 128, 16, True)
    a = [to(q, dev)] + [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array([3000, 700], np.int32), dev)]
    x, history, lens, prompts, rep, pres, freq = logits_case(rng, 3, 30000, 200, True)
    d = lambda t: to(t, dev)
    kw = dict(history=d(history), history_lens=d(lens), prompt_lens=d(prompts), repetition=d(rep), presence=d(pres),
              frequency=d(freq))
    logits = d(x)
    out, (log, tok) = ops.gqa_decode_q8(*a), ops.logits_process(logits, **kw)
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for _ in range(15):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((ops.gqa_decode_q8(*a), *ops.logits_process(logits, **kw)))
    torch.cuda.synchronize(dev)
    ops.raise_device_errors(dev)
    for o, l, t in got:
        assert torch.equal(o, out) and torch.equal(l, log) and torch.equal(t, tok)


@pytest.mark.parametrize("fp8", [False, True])
def test_overlapped_launches_give_the_same(dev, fp8):
    """A chain of steps under programmatic dependent launch."""
    rng = np.random.default_rng(17)
    B, Hq, Hkv, D, page, width = 5, 8, 2, 64, 16, 8
    pages = B * width
    table, one = to(so.make_table([width] * B, pages, rng), dev), to(np.arange(B + 1, dtype=np.int32), dev)
    rows = [to(rng.standard_normal((B, (Hq + 2 * Hkv) * D)).astype(np.float16), dev) for _ in range(60)]
    lens = [to(np.full(B, i + 1, np.int32), dev) for i in range(60)]
    ends = []
    for overlap in (False, True):
        k = torch.zeros((pages, Hkv, page, D), device=dev).to(code_dtype(fp8))
        v, ks, vs = k.clone(), *(torch.zeros((pages, Hkv, page // BLOCK), device=dev) for _ in range(2))
        k16, v16 = (torch.zeros((pages, page, Hkv, D), dtype=torch.float16, device=dev) for _ in range(2))
        outs = []
        for x, n in zip(rows, lens):
            q = ops.paged_kv_append_q8(x, k, v, ks, vs, table, n, one, Hq, overlap_prior=overlap)
            out = ops.gqa_decode_q8(q, k, v, ks, vs, table, n, overlap_prior=overlap)
            ops.paged_kv_append(x, k16, v16, table, n, one, Hq, overlap_prior=overlap)
            raw, token = ops.logits_process(out.view(B, -1), overlap_prior=overlap)
            outs += [out, raw, token]
        values = ops.kv_q8_values(k, v, ks, vs, overlap_prior=overlap)
        ends.append([*outs, *values, k16, v16])
    torch.cuda.synchronize(dev)
    ops.raise_device_errors(dev)
    for x, y in zip(*ends):
        assert torch.equal(x, y)


@pytest.mark.parametrize("fp8", [False, True])
def test_captured_step_replayed_as_the_sequences_grow(dev, fp8):
    """One captured step, its lengths and history counted up on the device, against eager steps."""
    rng = np.random.default_rng(21)
    B, Hq, Hkv, D, page, width, steps = 6, 14, 2, 64, 32, 5, 40
    pages = B * width
    table, one = to(so.make_table([width] * B, pages, rng), dev), to(np.arange(B + 1, dtype=np.int32), dev)
    rows = [to(rng.standard_normal((B, (Hq + 2 * Hkv) * D)).astype(np.float16), dev) for _ in range(steps)]
    start = to(rng.integers(0, 100, B).astype(np.int32), dev)
    history = to(rng.integers(0, Hq * D, (B, width * page)).astype(np.int32), dev)
    presence = torch.full((B,), 0.25, device=dev)
    ends = []
    for captured in (False, True):
        k = torch.zeros((pages, Hkv, page, D), device=dev).to(code_dtype(fp8))
        v, ks, vs = k.clone(), *(torch.zeros((pages, Hkv, page // BLOCK), device=dev) for _ in range(2))
        x, lens = rows[0].clone(), start.clone()

        def step():
            lens.add_(1)
            q = ops.paged_kv_append_q8(x, k, v, ks, vs, table, lens, one, Hq)
            out = ops.gqa_decode_q8(q, k, v, ks, vs, table, lens)
            return (out, *ops.logits_process(out.view(B, -1), history=history, history_lens=lens, presence=presence))

        if captured:
            g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream(dev)
            with torch.cuda.graph(g, stream=s):
                results = step()
        seen = []
        for row in rows:
            x.copy_(row)
            if captured:
                g.replay()
            else:
                results = step()
            seen += [t.clone() for t in results]
        ends.append([*seen, k.view(torch.uint8), v.view(torch.uint8), ks, vs, lens])
    torch.cuda.synchronize(dev)
    ops.raise_device_errors(dev)
    for a, b in zip(*ends):
        assert torch.equal(a, b)


def test_pools_beyond_31_bits(dev):
    """Codes and rows whose offsets do not fit 31 bits: the last pages of 2.2 GB pools."""
    rng = np.random.default_rng(18)
    Hq, Hkv, D, page = 4, 2, 128, 256
    pages = 2 ** 31 // (Hkv * page * D) + 1500
    k = torch.zeros((pages, Hkv, page, D), dtype=torch.int8, device=dev)
    v, ks, vs = torch.zeros_like(k), *(torch.zeros((pages, Hkv, page // BLOCK), device=dev) for _ in range(2))
    need = [2, 1]
    table = np.array([[so.word(pages - 1), so.word(pages - 3)], [so.word(pages - 2), 0]], np.int32)
    new = [300, 77]
    starts = np.array([0, 300, 377], np.int32)
    lens = np.array(new, np.int32)
    x = rng.standard_normal((377, (Hq + 2 * Hkv) * D)).astype(np.float16)
    q = ops.paged_kv_append_q8(to(x, dev), k, v, ks, vs, to(table, dev), to(lens, dev), to(starts, dev), Hq)
    last = q[torch.tensor([299, 376], device=dev)].contiguous()
    out = ops.gqa_decode_q8(last, k, v, ks, vs, to(table, dev), to(lens, dev))
    ops.raise_device_errors(dev)
    assert not k[:pages - 3].any() and not vs[:pages - 3].any()
    small = [so.word(2), so.word(0)], [so.word(1), 0]
    check_attention(out.cpu().numpy()[:, None], last.cpu().numpy()[:, None], k[pages - 3:], v[pages - 3:], ks[pages - 3:],
                    vs[pages - 3:], np.array(small, np.int32), new)
    k16 = torch.zeros((pages, page, Hkv, D), dtype=torch.float16, device=dev)
    v16 = torch.zeros_like(k16)
    assert torch.equal(ops.paged_kv_append(to(x, dev), k16, v16, to(table, dev), to(lens, dev), to(starts, dev), Hq), q)
    assert torch.equal(v16[pages - 2, :77].reshape(77, -1), to(x, dev)[300:, (Hq + Hkv) * D:])
    assert not v16[:pages - 3].any()


@pytest.mark.parametrize("lens,Q,Hq,Hkv,D,page,fp8", [
    ([80, 200], 2, 64, 1, 64, 16, False),      # 128 query rows on one kv head
    ([64], 1, 128, 128, 64, 16, True),         # many kv heads; a table without a spare place
    ([1] * 300, 1, 2, 1, 64, 16, True),        # many sequences of one token
    ([17, 0] * 40, 3, 6, 2, 128, 32, False),
])
def test_attention_q8_head_layouts(dev, lens, Q, Hq, Hkv, D, page, fp8):
    rng = np.random.default_rng(len(lens) + Hq)
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, Q, Hq, Hkv, D, page, fp8)
    out = ops.gqa_decode_q8(to(q, dev), *(t.to(dev) for t in (k, v, ks, vs)), to(table, dev),
                            to(np.array(lens, np.int32), dev))
    ops.raise_device_errors(dev)
    check_attention(out.cpu().numpy(), q, k, v, ks, vs, table, lens)


def test_logits_most_rows(dev):
    rng = np.random.default_rng(20)
    x = rng.standard_normal((4096, 70)).astype(np.float32)
    allowed = rng.random((4096, 70)) < 0.03
    out, tokens = ops.logits_process(to(x, dev), allowed=to(so.pack_mask(allowed), dev))
    ops.raise_device_errors(dev)
    want = np.where(allowed, x, -np.inf)
    assert np.array_equal(out.cpu().numpy(), want)
    assert np.array_equal(tokens.cpu().numpy(), np.where(allowed.any(axis=1), want.argmax(axis=1), -1))


# ---- waits that expire ------------------------------------------------------------

@pytest.mark.parametrize("lens,Q,Hq,Hkv,D,fp8", [
    ([5000, 0, 40, 3000], 1, 8, 2, 128, False),      # pairs over several CTAs, one inside a warp's stretch
    ([700, 650, 720], 4, 8, 2, 128, True),           # 16 rows a pair
    ([30000], 1, 14, 2, 64, False),                  # two pairs over the whole device
    ([300], 1, 14, 2, 64, True),                     # a CTA a pair
    ([1 + 7 * i % 90 for i in range(300)], 1, 8, 8, 64, False),   # many pairs a warp
])
def test_attention_q8_after_expired_waits(dev, lens, Q, Hq, Hkv, D, fp8):
    """Waits that give up, all of them or some warps': the error is reported once, the
    workspace's counters are zero behind the call, and the next call on it is right."""
    rng = np.random.default_rng(len(lens) + D)
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, Q, Hq, Hkv, D, 16, fp8)
    a = [to(q, dev)] + [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array(lens, np.int32), dev)]
    lib = _lib.load()
    ws = torch.zeros(lib.anvilq_gqa_decode_q8_workspace_size(len(lens), Q, Hq, Hkv, D), dtype=torch.uint8, device=dev)
    ref = ops.gqa_decode_q8(*a, workspace=ws)
    ops.raise_device_errors(dev)
    check_attention(ref.cpu().numpy(), q, k, v, ks, vs, table, lens)
    out, word = torch.empty_like(ref), ops.device_error_word(dev)
    for mask in (0xFFFF, 0x0001, 0x8421, 0x5555, 0x00F0, 0x0003):
        flags = mask << 16                           # ANVILQ_EXPIRE_WAITS; CTA 0's first wait is bit 0's
        ptr = lambda t: t.data_ptr()
        assert lib.anvilq_gqa_decode_q8(*map(ptr, a[:5]), int(fp8), ptr(a[5]), ptr(a[6]), ptr(out), len(lens), Q, Hq,
                                        Hkv, D, 16, table.shape[1], k.shape[0], 0.0, ptr(ws), ws.numel(), ptr(word),
                                        flags, torch.cuda.current_stream(dev).cuda_stream) == 0
        if mask & 1:
            with pytest.raises(AnvilqError, match="wait"):
                ops.raise_device_errors(dev)
        else:
            torch.cuda.synchronize(dev)
            word.zero_()
        assert not ws[:65536].any(), hex(mask)
        assert torch.equal(ops.gqa_decode_q8(*a, workspace=ws), ref), hex(mask)
    ops.raise_device_errors(dev)


# ---- blocks whose scale grows, sequences that are cut back, other rotations -----------

def step_codes(x, kept, codes, scale, dtype):
    """A block of one head after new rows x [n, D] behind `kept` ones, each operation in
    binary32: (codes [kept + n, D], scale)."""
    top = x.abs().max()
    if dtype == torch.int8:
        want, round_ = top / 127, lambda y: y.round().clamp(-127, 127).to(dtype)
    else:
        want = (2.0 ** torch.ceil(torch.log2(top.double() / 448))).float() if top > 0 else top
        round_ = lambda y: y.clamp(-448, 448).to(dtype)
    s = torch.maximum(scale, want) if kept else want
    old = codes[:kept]
    if kept and s > scale:
        old = round_(old.float() * (scale / s))
    new = round_(x * (1 / s)) if s > 0 else torch.zeros(x.shape).to(dtype)
    return torch.cat([old.float(), new.float()]).to(dtype), s


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_append_q8_growing_blocks_bit_for_bit(dev, D, fp8):
    """Blocks with 1 to 15 rows whose scale an appended run of 1 to 15 rows raises, by all
    lanes alike: kept rows, new rows and scales of V are the formulas' in binary32."""
    rng = np.random.default_rng(41)
    Hq, Hkv, page, dtype = 3, 3, 16, code_dtype(fp8)
    runs = [(kept, n) for kept in range(1, 16) for n in range(1, 17 - kept)]
    B = len(runs)
    table = to(so.make_table([1] * B, B, rng), dev)
    for group in (runs, [r for r in runs if r[1] <= 2]):        # chunks; a token or two a sequence
        kept, new = [k for k, _ in group], [n for _, n in group]
        n_seq = len(group)
        codes = random_codes(rng, (B, Hkv, page, D), fp8)
        scales = random_scales(rng, (B, Hkv, 1), fp8)
        k, v, ks, vs = codes.to(dev), codes.to(dev), scales.to(dev), scales.to(dev)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        size = 8.0 ** rng.integers(-1, 3, size=(starts[-1], 1))
        qkv = (rng.standard_normal((starts[-1], (Hq + 2 * Hkv) * D)) * size).astype(np.float16)
        lens = np.array([a + b for a, b in group], np.int32)
        ops.paged_kv_append_q8(to(qkv, dev), k, v, ks, vs, table[:n_seq].contiguous(), to(lens, dev), to(starts, dev), Hq)
        ops.raise_device_errors(dev)
        x = torch.from_numpy(qkv.astype(np.float32)).view(-1, Hq + 2 * Hkv, D)[:, Hq + Hkv:]
        got, got_s, t = v.cpu(), vs.cpu(), table.cpu().numpy()
        for b in range(n_seq):
            pg = so.physical(t[b, 0])
            for h in range(Hkv):
                want, s = step_codes(x[starts[b]:starts[b + 1], h], kept[b], codes[pg, h], scales[pg, h, 0], dtype)
                assert got_s[pg, h, 0] == s, (b, h)
                assert torch.equal(got[pg, h, :lens[b]].float(), want.float()), (group[b], h)


# ---- idle slots ---------------------------------------------------------------------

def idle_slots_case(dev, rng, B, live, tokens, Hq=8, Hkv=2, D=64, page=64):
    """B slots of which those of `live` hold `tokens` tokens, the others none."""
    lens = np.zeros(B, np.int32)
    lens[list(live)] = tokens
    q, k, v, ks, vs, table = attention_case(dev, rng, [int(n) for n in lens], 1, Hq, Hkv, D, page, False)
    a = [to(q, dev)] + [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(lens, dev)]
    return a, (q, k, v, ks, vs, table, lens)


@pytest.mark.parametrize("B,live", [
    (33, (0, 32)), (64, (31, 32)), (200, (0, 63, 64, 199)), (1024, (31, 1023)), (1025, (0, 992, 1024)),
    (3000, (5, 6, 1500, 2999)), (5000, (4999,)), (20000, (0, 31, 32, 10016, 19999)),
])
def test_attention_q8_live_slots_far_apart(dev, B, live):
    rng = np.random.default_rng(B)
    a, (q, k, v, ks, vs, table, lens) = idle_slots_case(dev, rng, B, live, 1500)
    out = ops.gqa_decode_q8(*a, out=torch.full_like(a[0].squeeze(1), float("nan")).unsqueeze(1))
    ops.raise_device_errors(dev)
    got = out.cpu().numpy()
    idle = np.ones(B, bool)
    idle[list(live)] = False
    assert not got[idle].any()
    pick = list(live)
    check_attention(got[pick], q[pick], k, v, ks, vs, table[pick], [int(n) for n in lens[pick]])


def test_attention_q8_idle_slots_cost_no_walk(dev):
    """Two sequences in the first and the last of 8192 slots take about as long as in the
    first two: no warp steps over the idle slots between them one by one (which took ten
    times as long)."""
    rng = np.random.default_rng(0)
    times = []
    for live in ((0, 1), (0, 8191)):
        a, _ = idle_slots_case(dev, rng, 8192, live, 8000)
        out = torch.empty_like(a[0])
        runs = []
        for i in range(12):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(10):
                ops.gqa_decode_q8(*a, out=out)
            end.record()
            end.synchronize()
            runs.append(begin.elapsed_time(end))
        times.append(min(runs[2:]))
    ops.raise_device_errors(dev)
    assert times[1] < 3 * times[0], times


# ---- workspaces -----------------------------------------------------------------------

def test_eager_calls_behind_a_capture_have_their_own_workspace(dev):
    """A stream whose first call was captured: its workspace is the graph's, zero only in
    replays, and eager serving calls there do not use it."""
    rng = np.random.default_rng(61)
    q, k, v, ks, vs, table = attention_case(dev, rng, [3000, 700], 1, 8, 2, 128, 16, False)
    a = [to(q, dev)] + [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array([3000, 700], np.int32), dev)]
    ref = ops.gqa_decode_q8(*a)
    kc = torch.randn((2, 900, 2, 128), device=dev).half()
    vc, q16 = torch.randn_like(kc), torch.randn((2, 8, 128), device=dev).half()
    lens = torch.tensor([900, 33], dtype=torch.int32, device=dev)
    old = ops.gqa_decode(q16, kc, vc, lens)
    torch.cuda.synchronize(dev)
    s = torch.cuda.Stream(dev)
    key = (dev.index, s.cuda_stream)
    earlier = ops._workspaces.pop(key, None)         # streams come from a pool
    ops._of_graphs.discard(key)
    g, out = torch.cuda.CUDAGraph(), torch.empty_like(old)
    with torch.cuda.graph(g, stream=s):
        out.copy_(ops.gqa_decode(q16, kc, vc, lens))
    of_graph = ops._workspaces[key]
    with torch.cuda.stream(s):
        for _ in range(3):
            assert torch.equal(ops.gqa_decode_q8(*a), ref)
            g.replay()
            assert torch.equal(out, old)
    assert ops._workspaces[key] is not of_graph
    s.synchronize()
    ops.raise_device_errors(dev)


# ---- softmax scales --------------------------------------------------------------------

@pytest.mark.parametrize("fp8", [False, True])
def test_attention_q8_largest_scale(dev, fp8):
    """Under the largest scale the softmax takes the largest score's value alone, and equal
    ones alike; zero scores (a zero query) still weigh all values the same."""
    rng = np.random.default_rng(71)
    q, k, v, ks, vs, table = attention_case(dev, rng, [100], 1, 8, 2, 64, 16, fp8)
    ks[:] = 0.5 if fp8 else 700.0
    q[0, 0, 3] = 0
    a = [to(q, dev)] + [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array([100], np.int32), dev)]
    out = ops.gqa_decode_q8(*a, scale=2.0 ** 64).cpu().numpy().astype(np.float64)
    ops.raise_device_errors(dev)
    kv, vv = so.pool_values(k, ks), so.pool_values(v, vs)
    at = [so.physical(e) for e in table[0]]
    flat = lambda p: p[at].transpose(0, 2, 1, 3).reshape(-1, 2, 64)[:100]
    kv, vv = flat(kv), flat(vv)
    for h in range(8):
        if h == 3:
            want, tol = vv[:, 0].mean(axis=0), 2 * HALF * (1 + 2.0 ** -6) * np.abs(vv[:, 0]).mean(axis=0)
        else:
            x = kv[:, h // 4] @ q[0, 0, h].astype(np.float64)
            assert np.sort(x)[-1] - np.sort(x)[-2] > 2.0 ** -18 * np.abs(kv).max() * np.abs(q[0, 0, h]).sum()
            want = vv[x.argmax(), h // 4]
            tol = 2 * HALF * (1 + 2.0 ** -6) * np.abs(want)
        assert (np.abs(out[0, 0, h] - want) <= tol + 2.0 ** -24).all(), h


@pytest.mark.parametrize("lens,Q", [([5000, 0, 40], 1), ([900, 3, 70], 4), ([33] * 40, 1)])
def test_attention_q8_in_place(dev, lens, Q):
    rng = np.random.default_rng(81)
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, Q, 8, 2, 128, 16, False)
    a = [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array(lens, np.int32), dev)]
    ref = ops.gqa_decode_q8(to(q, dev), *a)
    for _ in range(5):
        x = to(q, dev)
        assert ops.gqa_decode_q8(x, *a, out=x) is x and torch.equal(x, ref)
    ops.raise_device_errors(dev)
    both = torch.zeros((2 * x.numel(),), dtype=torch.float16, device=dev)
    with pytest.raises(AnvilqError):
        ops.gqa_decode_q8(both[:x.numel()].view_as(x), *a, out=both[64:64 + x.numel()].view_as(x))


@pytest.mark.parametrize("lens,Q,Hq,Hkv,page,fp8", [
    ([900, 40], 8, 8, 2, 16, False),           # 32 query rows a kv head: two groups
    ([300, 0, 2000], 8, 28, 4, 32, True),      # 56: four groups, the last half full
    ([700], 64, 32, 8, 64, False),             # 256
    ([5000], 16, 4, 1, 16, True),              # 64 rows of one kv head over many CTAs
])
def test_attention_q8_row_groups(dev, lens, Q, Hq, Hkv, page, fp8):
    """More query rows a kv head than one group holds, heads of 128."""
    rng = np.random.default_rng(Q + Hq)
    q, k, v, ks, vs, table = attention_case(dev, rng, lens, Q, Hq, Hkv, 128, page, fp8)
    a = [t.to(dev) for t in (k, v, ks, vs)] + [to(table, dev), to(np.array(lens, np.int32), dev)]
    qd = to(q, dev)
    out = ops.gqa_decode_q8(qd, *a)
    again = ops.gqa_decode_q8(qd, *a, out=torch.full_like(qd, float("nan")))
    ops.raise_device_errors(dev)
    assert torch.equal(out, again)
    check_attention(out.cpu().numpy(), q, k, v, ks, vs, table, lens)


def test_append_rotations_of_several_thetas(dev):
    """Calls that take turns in theta and head size, in one thread: each rotates by its own."""
    rng = np.random.default_rng(91)
    Hq, Hkv, page = 4, 2, 16
    cases = []
    for D in (64, 128):
        qkv, table, starts, lens, pages = append_case(rng, [3000, 0], [5, 20], Hq, Hkv, D, page, spare_rows=0)
        cases.append((D, qkv, to(table, dev), to(lens, dev), to(starts, dev), pages, rows_of(starts, lens)))
    for i, theta in ((0, 1e4), (0, 5e5), (0, 1e6), (1, 1e6), (1, 1e4), (0, 1e4), (0, 5e5), (1, 5e5)):   # one changes
        D, qkv, table, lens, starts, pages, rows = cases[i]
        x = qkv.reshape(len(rows), Hq + 2 * Hkv, D)[:, :Hq]
        turned = so.rotate(x, [p for _, p in rows], theta)
        pair = np.abs(x.astype(np.float64))
        tol = HALF * np.abs(turned) + 2.0 ** -22 * (pair + np.roll(pair, D // 2, axis=2)) + 2.0 ** -25
        k = torch.zeros((pages, page, Hkv, D), dtype=torch.float16, device=dev)
        q = ops.paged_kv_append(to(qkv, dev), k, torch.zeros_like(k), table, lens, starts, Hq, theta)
        assert (np.abs(q.cpu().numpy() - turned) <= tol).all(), (D, theta)
        codes, scales = torch.zeros((pages, Hkv, page, D), dtype=torch.int8, device=dev), torch.zeros((pages, Hkv, 1), device=dev)
        assert torch.equal(ops.paged_kv_append_q8(to(qkv, dev), codes, codes.clone(), scales, scales.clone(), table, lens,
                                                  starts, Hq, theta), q)
    ops.raise_device_errors(dev)


@pytest.mark.parametrize("fp8", [False, True])
def test_drafts_rejected_and_appended_over(dev, fp8):
    """Drafts of large values, cut back by seqlens and appended over: the accepted rows stay
    coded to the scale that the drafts raised, later rows of the block use it too, and a block
    that was cut back to its start takes a scale of its own."""
    rng = np.random.default_rng(95)
    Hq, Hkv, D, page, dtype = 4, 2, 64, 32, code_dtype(fp8)
    table = so.make_table([1], 2, rng)
    pg = so.physical(table[0, 0])
    k = torch.zeros((2, Hkv, page, D), device=dev).to(dtype)
    v, ks, vs = k.clone(), *(torch.zeros((2, Hkv, page // BLOCK), device=dev) for _ in range(2))
    t = to(table, dev)
    codes, scales = [torch.zeros((0, D)).to(dtype)] * Hkv, torch.zeros(Hkv)      # of the block in work
    kept = 0
    for first, n, size in ((0, 5, 1.0), (5, 4, 50.0), (6, 3, 1.0), (9, 7, 2.0),  # one draft of four accepted
                           (16, 3, 90.0), (16, 4, 0.5), (18, 2, 8.0)):           # none of three; half of four
        qkv = (rng.standard_normal((n, (Hq + 2 * Hkv) * D)) * size).astype(np.float16)
        lens = to(np.array([first + n], np.int32), dev)
        q = ops.paged_kv_append_q8(to(qkv, dev), k, v, ks, vs, t, lens, to(np.array([0, n], np.int32), dev), Hq)
        x = torch.from_numpy(qkv.astype(np.float32)).view(n, Hq + 2 * Hkv, D)[:, Hq + Hkv:]
        block, kept = first // BLOCK, first % BLOCK
        for h in range(Hkv):
            codes[h], s = step_codes(x[:, h], kept, codes[h], scales[h], dtype)
            scales[h] = s
            assert vs[pg, h, block].item() == s.item(), (first, h)
            assert torch.equal(v[pg, h, block * BLOCK:first + n].cpu().float(), codes[h].float()), (first, h)
        out = ops.gqa_decode_q8(q.view(1, n, Hq, D), k, v, ks, vs, t, lens)
        check_attention(out.cpu().numpy(), q.cpu().numpy()[None], k, v, ks, vs, table, [first + n])
    ops.raise_device_errors(dev)
