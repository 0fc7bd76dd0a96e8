"""Prompts in chunks, beams and shared pages over a paged cache, as measured cases.

Beside a decode step's operators, a serving batch needs attention of many new tokens
a sequence over the binary16 pages, rotations of other kinds than full heads in split
halves, the selection of a beam search, and pages that beams and prompts share.

A case's "op" says which: "chunk" (ops.gqa_chunk_paged), "rope" (ops.paged_kv_append
with frequencies of the caller's), "beam" (ops.beam_select, ops.beam_reorder), "fork"
(ops.pages_fork, ops.pages_reserve), "compact" (ops.pages_release, ops.pages_compact).
Cases are plain dicts; ``prepare`` makes a case's inputs on the GPU from a seed,
``run`` is one pass, in plain torch operations or (``own``) through the framework,
``work`` counts what a pass cannot do without, ``exact`` is the operator's definition
in binary64.
"""
import math
import random

import torch

own = False

THETA = 1.0e6
VALID = 1 << 31       # bit 31 of a page-table word: the entry is valid
PAGE = VALID - 1      # bits 30:0: the page


def listed():
    return [
        # a short question appended to a conversation on the 14/2 heads of 64: a first answer's latency
        dict(name="chunk one short", op="chunk", B=1, new=13, ctx=150, steps=0, Hq=14, Hkv=2, D=64, page=16),
        # a mixed batch: some sequences take a decode step, others a chunk of their prompt
        dict(name="chunk mixed batch", op="chunk", B=12, new=500, ctx=3001, steps=6, Hq=28, Hkv=4, D=128, page=48),
        # a question about one very long document: few rows over a long axis
        dict(name="chunk long document", op="chunk", B=1, new=60, ctx=60001, steps=0, Hq=32, Hkv=8, D=128, page=256),
        # the largest: one chunk of a long prompt, 4096 tokens after the first 12288
        dict(name="chunk of a long prompt", op="chunk", B=1, new=4096, ctx=12288, steps=0, Hq=32, Hkv=8, D=128,
             page=16),
        # a decode step of a batch, a quarter of each head rotated in neighbouring pairs
        dict(name="rope step", op="rope", B=64, new=1, ctx=30000, Hq=32, Hkv=8, D=128, page=16, rot=32, pairs=True,
             scale=1.0),
        # prompts of a batch at once, whole heads in split halves, frequencies scaled for 8 times the context
        dict(name="rope prompts", op="rope", B=6, new=4001, ctx=20000, Hq=14, Hkv=2, D=64, page=64, rot=64,
             pairs=False, scale=8.0),
        # one question, four beams over a large vocabulary
        dict(name="beam one item", op="beam", B=1, K=4, N=4, V=151936, half=False, masked=False, ended=False,
             alpha=0.0, L=200),
        # a batch of questions with eight beams each, a grammar's masks already in the logits
        dict(name="beam batch", op="beam", B=48, K=8, N=8, V=151936, half=True, masked=True, ended=True, alpha=0.6,
             L=700),
        # many short questions over a small vocabulary, twice as many candidates as beams
        dict(name="beam many items", op="beam", B=100, K=5, N=10, V=32000, half=False, masked=False, ended=True,
             alpha=1.0, L=60),
        # one question's four beams go on: 24 layers of the 14/2 heads of 64
        dict(name="fork one item", op="fork", items=1, beams=4, ctx=300, said=37, layers=24, Hkv=2, D=64, page=16),
        # a batch of questions with eight beams each: 32 layers of 8 heads of 128
        dict(name="fork batch", op="fork", items=8, beams=8, ctx=1800, said=100, layers=32, Hkv=8, D=128, page=64),
        # a pool after many conversations came and went, brought together again
        dict(name="compact", op="compact", rows=96, ctx=1000, left=0.4, layers=24, Hkv=2, D=64, page=32),
    ]


HEADS = [(14, 2, 64), (32, 8, 128), (32, 32, 128), (28, 4, 128), (8, 8, 64), (16, 2, 128)]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "rope", "beam", "beam", "fork", "compact"])
    Hq, Hkv, D = rng.choice(HEADS)
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if op == "chunk":
        B = _log_int(rng, 1, 32)
        new = _log_int(rng, 1, 4096)
        top = max(1, min(60000, 900_000_000 // (B * Hq * new) - new, 60_000_000 // (B * Hkv * D) - new))
        while B * Hq * new * (1 + new) > 900_000_000:
            new = max(1, new // 2)
        return dict(op=op, B=B, new=new, ctx=rng.choice([0, _log_int(rng, 1, top)]), steps=rng.choice([0, B // 2]),
                    Hq=Hq, Hkv=Hkv, D=D, page=page)
    if op == "rope":
        B = _log_int(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, 20_000_000 // (B * (Hq + 2 * Hkv) * D)))
        return dict(op=op, B=B, new=new, ctx=rng.choice([0, 15, 1000, 30000]), Hq=Hq, Hkv=Hkv, D=D, page=page,
                    rot=16 * rng.randint(1, D // 16), pairs=rng.random() < 0.5, scale=rng.choice([1.0, 4.0, 40.0]))
    if op == "beam":
        B, K = _log_int(rng, 1, 64), rng.randint(1, 16)
        V = _log_int(rng, 1000, min(151936, 50_000_000 // (B * K)))
        return dict(op=op, B=B, K=K, N=rng.choice([K, 2 * K]), V=V, half=rng.random() < 0.5,
                    masked=rng.random() < 0.5, ended=rng.random() < 0.5, alpha=rng.choice([0.0, 0.7, 1.0]),
                    L=_log_int(rng, 1, 2000))
    layers = rng.choice([4, 12, 24])
    if op == "fork":
        items, beams = _log_int(rng, 1, 16), rng.randint(2, 12)
        most = max(page, 800_000_000 // (items * 2 * layers * Hkv * D * 2) - beams * page)
        return dict(op=op, items=items, beams=beams, ctx=_log_int(rng, 1, min(3000, most)), said=rng.randint(0, page),
                    layers=layers, Hkv=Hkv, D=D, page=page)
    rows = _log_int(rng, 2, 200)
    most = max(page, 800_000_000 // (rows * 2 * layers * Hkv * D * 2))
    return dict(op=op, rows=rows, ctx=_log_int(rng, page, min(3000, most)), left=rng.uniform(0.1, 0.9), layers=layers,
                Hkv=Hkv, D=D, page=page)


# ---- a case's lengths and choices: its own, whatever the seed -----------------------

def _lens(case):
    """chunk, rope: (tokens before, new tokens) of each sequence."""
    r = random.Random("%d %d %d" % (case["B"], case["new"], case["ctx"]))
    B, new, steps = case["B"], case["new"], case.get("steps", 0)
    before = [case["ctx"]] + [r.randint(0, case["ctx"]) for _ in range(B - 1)]
    return before, [new if b == 0 else 1 if b >= B - steps else r.randint(1, new) for b in range(B)]


def _beams(case):
    """fork: (prompt length of each item, parent of each row)."""
    r = random.Random("%d %d %d" % (case["items"], case["beams"], case["ctx"]))
    prompts = [case["ctx"]] + [r.randint(1, case["ctx"]) for _ in range(case["items"] - 1)]
    n = case["beams"]
    # the better beams have more children
    parents = [i * n + int(n * r.random() ** 2) for i in range(case["items"]) for _ in range(n)]
    return prompts, parents


def _rows(case):
    """compact: (length, tokens kept) of each sequence."""
    r = random.Random("%d %d %f" % (case["rows"], case["ctx"], case["left"]))
    lens = [case["ctx"]] + [r.randint(1, case["ctx"]) for _ in range(case["rows"] - 1)]
    # most of those that end are gone, some are cut back
    return lens, [n if r.random() < case["left"] else 0 if r.random() < 0.8 else r.randint(0, n) for n in lens]


def _word(page):
    """A page-table word as the int32 that the table holds."""
    return (page | VALID) - (1 << 32)


def _frequencies(case):
    """Angles a position of a case's pairs, and the factor of the rotated values.  scale > 1 stretches
    the context from 32768 tokens by that factor (Peng et al. 2023, "YaRN"): pairs that turn less than
    once in it are slowed down, those of over 32 turns stay, a linear ramp between them."""
    R, s = case["rot"], case["scale"]
    inv = [THETA ** (-2.0 * i / R) for i in range(R // 2)]
    if s == 1.0:
        return inv, 1.0
    at = lambda turns: R * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(THETA))
    lo, hi = max(0, math.floor(at(32))), min(R // 2 - 1, math.ceil(at(1)))
    ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(R // 2)]
    return [f * (1 - w) + f / s * w for f, w in zip(inv, ramp)], 0.1 * math.log(s) + 1.0


# ---- inputs -------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    r = random.Random(int(seed))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    half = lambda *shape: torch.randn(shape, generator=g, device=dev, dtype=torch.float16)
    s = dict(case=dict(case))
    if case["op"] == "beam":
        return _prepare_beam(case, s, g, ints, dev)
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if case["op"] in ("chunk", "rope"):
        before, new = _lens(case)
        # the pages that the pass touches (a rotation writes the new tokens' only), and one more
        first = [0 if case["op"] == "chunk" else p // page for p in before]
        last = [(p + n - 1) // page for p, n in zip(before, new)]
        pages = sum(b - a + 1 for a, b in zip(first, last)) + 1
        order = list(range(pages))
        r.shuffle(order)
        table, at = [[0] * (max(last) + 1) for _ in new], 0
        for b in range(case["B"]):
            for j in range(first[b], last[b] + 1):
                table[b][j] = _word(order[at])
                at += 1
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s.update(k=half(pages, page, Hkv, D), v=half(pages, page, Hkv, D), table=ints(table), starts=ints(starts),
                 lens=ints([p + n for p, n in zip(before, new)]))
        if case["op"] == "chunk":
            s["q"] = half(starts[-1], case["Hq"], D) * 3
        else:
            s["qkv"] = half(starts[-1], (case["Hq"] + 2 * Hkv) * D)
            inv, s["factor"] = _frequencies(case)
            s["inv"] = torch.tensor(inv, dtype=torch.float64, device=dev)
        return s
    if case["op"] == "fork":
        prompts, parents = _beams(case)
        n, lens = case["beams"], [p + case["said"] for p in prompts]
        tables, refs = [], []
        for p, length in zip(prompts, lens):
            shared = p // page                 # the prompt's full pages are every beam's
            common = list(range(len(refs), len(refs) + shared))
            refs += [n] * shared
            for _ in range(n):
                private = -(-length // page) - shared
                tables.append(common + list(range(len(refs), len(refs) + private)))
                refs += [1] * private
        pages = len(refs) + len(tables) + 5
        width = max(len(t) for t in tables) + 1
        s["before"] = ints([length for length in lens for _ in range(n)])
        s["after"] = s["before"] + 1
        s["parents"] = ints(parents)
    else:
        lens, keep = _rows(case)
        tables, refs = [], []
        for n in lens:
            tables.append(list(range(len(refs), len(refs) + -(-n // page))))
            refs += [1] * len(tables[-1])
        pages, width = len(refs) + 5, max(len(t) for t in tables)
        s["keep"] = ints(keep)
    order = list(range(pages))
    r.shuffle(order)
    count = [0] * pages
    for i, c in enumerate(refs):
        count[order[i]] = c
    s["table"] = ints([[_word(order[p]) for p in t] + [0] * (width - len(t)) for t in tables])
    s["spare"] = torch.zeros_like(s["table"])
    s["refs"] = ints(count)
    s["new_refs"] = torch.zeros_like(s["refs"])
    s["k"], s["v"] = half(case["layers"], pages, page, Hkv, D), half(case["layers"], pages, page, Hkv, D)
    s["pools"] = [*s["k"].unbind(0), *s["v"].unbind(0)]
    return s


def _prepare_beam(case, s, g, ints, dev):
    B, K, V, L = case["B"], case["K"], case["V"], case["L"]
    rand = lambda *shape: torch.rand(shape, generator=g, device=dev)
    x = torch.randn((B, K, V), generator=g, device=dev, dtype=torch.float16 if case["half"] else torch.float32) * 3
    if case["masked"]:
        # a grammar that allows little in some beams, and nothing at all in one
        few = (rand(B, K, 1) < 0.3) & (rand(B, K, V) > 0.002)
        x = torch.where(few, -math.inf, x)
        x[B // 2, K - 1] = -math.inf
    scores = -rand(B, K) * 20
    scores[0, 1:] = -math.inf         # an item's first step: all its beams are the first one
    lengths = torch.randint(1, L + 1, (B, K), generator=g, device=dev, dtype=torch.int32)
    ended = (rand(B, K) < 0.15) & (scores > -math.inf) if case["ended"] else None
    s.update(x=x, scores=scores, lengths=lengths, ended=ended, eos=ints([V // 3, V - 1]),
             history=torch.randint(0, V, (B, K, L), generator=g, device=dev, dtype=torch.int32))
    return s


# ---- one pass -----------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        from anvilq_b200 import ops
        if case["op"] == "chunk":
            return ops.gqa_chunk_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"])
        if case["op"] == "rope":
            q = ops.paged_kv_append(s["qkv"], s["k"], s["v"], s["table"], s["lens"], s["starts"], case["Hq"],
                                    inv_freq=s["inv"], interleaved=case["pairs"], rope_factor=s["factor"])
            return q, s["k"], s["v"]
        if case["op"] == "beam":
            tokens, parents, scores, lengths, ended = ops.beam_select(
                s["x"], s["scores"], case["N"], lengths=s["lengths"], length_penalty=case["alpha"],
                finished=s["ended"], eos_ids=s["eos"], pad_id=0)
            history, = ops.beam_reorder([s["history"]], parents)
            return tokens, parents, scores, lengths, ended, history
        if case["op"] == "fork":
            s["table"], s["spare"] = ops.pages_fork(s["table"], s["refs"], s["parents"], out=s["spare"]), s["table"]
            ops.pages_reserve(s["table"], s["refs"], s["before"], s["after"], case["page"], s["pools"])
            return s["table"], s["refs"], s["k"], s["v"]
        ops.pages_release(s["table"], s["refs"], s["keep"], case["page"])
        ops.pages_compact(s["table"], s["refs"], s["pools"], out=s["spare"], out_refs=s["new_refs"])
        return s["spare"], s["new_refs"], s["k"], s["v"]
    return {"chunk": _chunk, "rope": _rope, "beam": _beam, "fork": _fork, "compact": _compact}[case["op"]](s)


def _place(s):
    """(sequence, position) of every new token."""
    t = torch.arange(int(s["starts"].shape[0] and s["q" if "q" in s else "qkv"].shape[0]), device=s["lens"].device)
    b = torch.searchsorted(s["starts"].long(), t, right=True) - 1
    return b, s["lens"].long()[b] - s["starts"].long()[b + 1] + t


def _chunk(s):
    q, case = s["q"], s["case"]
    T, Hq, D = q.shape
    at = (s["table"] & PAGE).long()
    B, Hkv, n, new = at.shape[0], s["k"].shape[2], at.shape[1] * case["page"], case["new"]
    # [B, heads, positions, D], the queries of a sequence from its first new one on
    k = s["k"][at].float().reshape(B, n, Hkv, D).transpose(1, 2)
    v = s["v"][at].float().reshape(B, n, Hkv, D).transpose(1, 2)
    b, pos = _place(s)
    row = torch.arange(T, device=q.device) - s["starts"].long()[b]
    rows = torch.zeros((B, new, Hq, D), device=q.device)
    rows[b, row] = q.float()
    rows = rows.reshape(B, new, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    x = torch.matmul(rows, k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).reshape(B, Hkv, Hq // Hkv, new, n)
    sees = torch.zeros((B, new), device=q.device, dtype=torch.long)
    sees[b, row] = pos + 1
    hidden = torch.arange(n, device=q.device) >= sees[:, None, None, :, None]
    x.masked_fill_(hidden, -math.inf)
    top = x.amax(dim=4, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(dim=4, keepdim=True)
    o = torch.matmul(p.reshape(B, Hkv, -1, n), v).reshape(B, Hkv, Hq // Hkv, new, D) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(B, new, Hq, D)[b, row].half()


def _rope(s):
    case = s["case"]
    Hq, Hkv, D, page, R = case["Hq"], case["Hkv"], case["D"], case["page"], case["rot"]
    T = s["qkv"].shape[0]
    b, pos = _place(s)
    # the angle is a binary64 product rounded to binary32: the operator's definition
    angle = (pos.double()[:, None] * s["inv"]).float()
    cos, sin = (torch.cos(angle) * s["factor"])[:, None], (torch.sin(angle) * s["factor"])[:, None]
    x = s["qkv"].float().reshape(T, Hq + 2 * Hkv, D)
    y = x[:, :Hq + Hkv].clone()
    if case["pairs"]:
        lo, hi = x[:, :Hq + Hkv, 0:R:2], x[:, :Hq + Hkv, 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = lo * cos - hi * sin, hi * cos + lo * sin
    else:
        lo, hi = x[:, :Hq + Hkv, :R // 2], x[:, :Hq + Hkv, R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = lo * cos - hi * sin, hi * cos + lo * sin
    at = s["table"].long()[b, pos // page] & PAGE
    s["k"][at, pos % page] = y[:, Hq:].half()
    s["v"][at, pos % page] = x[:, Hq + Hkv:].half()
    return y[:, :Hq].half(), s["k"], s["v"]


def _beam(s):
    case = s["case"]
    B, K, V, N = case["B"], case["K"], case["V"], case["N"]
    # in 64 bits: candidates of different beams may be very close
    x = s["x"].double()
    live = s["scores"].double()[..., None]
    total = torch.logsumexp(x, dim=2, keepdim=True)
    score = live + (x - torch.where(total == -math.inf, 0.0, total))
    rank = score / torch.pow((s["lengths"].double() + 1), case["alpha"])[..., None]
    ended = s["ended"] if s["ended"] is not None else torch.zeros((B, K), dtype=torch.bool, device=x.device)
    # an ended beam is one candidate, at its beam's first place
    first = torch.arange(V, device=x.device) == 0
    done = torch.where(first, live, -math.inf)
    score = torch.where(ended[..., None], done, score)
    rank = torch.where(ended[..., None], done / torch.pow(s["lengths"].double().clamp(min=1), case["alpha"])[..., None],
                       rank)
    rank, at = torch.sort(rank.reshape(B, K * V), dim=1, descending=True, stable=True)   # ties: the lowest place first
    at, some = at[:, :N], rank[:, :N] > -math.inf
    scores = torch.where(some, score.reshape(B, K * V).gather(1, at), -math.inf).float()
    beam = at // V
    was = ended.gather(1, beam)
    tokens = torch.where(some, torch.where(was, 0, at % V), -1).int()
    parents = torch.where(some, beam, -1).int()
    lengths = torch.where(some, s["lengths"].gather(1, beam) + (~was).int(), 0)
    now = was | (tokens[..., None] == s["eos"]).any(dim=2) | ~some
    history = s["history"].gather(1, beam[..., None].expand(B, N, case["L"]))
    return tokens, parents, scores, lengths, now, torch.where(some[..., None], history, 0)


def _counts(table, pages):
    """How many entries of a table name each page."""
    live = (table < 0).int().reshape(-1)
    return torch.zeros(pages, dtype=torch.int32, device=table.device).scatter_add_(
        0, (table & PAGE).long().reshape(-1) * live, live)


def _fork(s):
    case, page, refs = s["case"], s["case"]["page"], s["refs"]
    pages = refs.shape[0]
    table = s["table"][s["parents"].long()]
    refs += _counts(table, pages) - _counts(s["table"], pages)
    s["table"], s["spare"] = table, s["table"]
    # entries that the new tokens will be written to: new pages where there is none of the row's own
    B, width = table.shape
    j = torch.arange(width, device=table.device)
    need = (j >= s["before"][:, None] // page) & (j < (s["after"][:, None] + page - 1) // page)
    need &= (s["after"] > s["before"])[:, None]
    at = (table & PAGE).long()
    writes = need & (table < 0)
    flat = torch.arange(B * width, device=table.device).reshape(B, width)
    where = torch.where(writes, at, pages).reshape(-1)
    writers = torch.zeros(pages + 1, dtype=torch.int32, device=table.device).scatter_add_(
        0, where, torch.ones_like(where, dtype=torch.int32))
    last = torch.full((pages + 1,), -1, dtype=torch.long, device=table.device).scatter_reduce_(
        0, where, flat.reshape(-1), "amax")
    shared = writes & (refs[at] > 1)
    shared &= ~((refs[at] == writers[at]) & (last[at] == flat))        # the last of a page's writers keeps it
    wants = (need & (table >= 0)) | shared
    rank = torch.cumsum(wants.reshape(-1).int(), 0).reshape(B, width) - 1
    free = torch.nonzero(refs == 0)[:, 0]
    b, c = torch.nonzero(wants, as_tuple=True)
    new, old, had = free[rank[b, c]], at[b, c], shared[b, c]
    refs[new] = 1
    refs.scatter_add_(0, old[had], torch.full_like(old[had], -1).int())
    table[b, c] = (new | VALID).int()
    rows = s["before"].long()[b] - c * page             # rows of the page that were there before
    move = had & (rows > 0)
    new, old, rows = new[move], old[move], rows[move]
    i = torch.arange(page, device=table.device)
    n, i = torch.nonzero(i < rows[:, None], as_tuple=True)
    for pool in (s["k"], s["v"]):
        pool[:, new[n], i] = pool[:, old[n], i]
    return table, refs, s["k"], s["v"]


def _compact(s):
    page, refs, table = s["case"]["page"], s["refs"], s["table"]
    pages = refs.shape[0]
    drop = torch.arange(table.shape[1], device=table.device) >= ((s["keep"] + page - 1) // page)[:, None]
    refs -= _counts(torch.where(drop, table, 0), pages)
    table.masked_fill_(drop, 0)
    used = refs > 0
    n = used.sum()
    p = torch.arange(pages, device=table.device)
    src, dst = torch.nonzero(used & (p >= n))[:, 0], torch.nonzero(~used & (p < n))[:, 0]
    to = p.clone()
    to[src] = dst
    s["spare"].copy_(torch.where(table < 0, (to[(table & PAGE).long()] | VALID).int(), table))
    s["new_refs"].copy_(refs)
    s["new_refs"][dst] = refs[src]
    s["new_refs"][src] = 0
    for pool in (s["k"], s["v"]):
        pool[:, dst] = pool[:, src]
    return s["spare"], s["new_refs"], s["k"], s["v"]


# ---- what a pass cannot do without --------------------------------------------------

def work(case):
    op = case["op"]
    if op == "beam":
        B, K, V, N = case["B"], case["K"], case["V"], case["N"]
        n = B * K * V * (2 if case["half"] else 4) + B * K * 9 + B * N * 17 + 8 * B * N * case["L"]
        return dict(bytes=n, flops=4 * B * K * V)
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if op in ("chunk", "rope"):
        before, new = _lens(case)
        T, Hq = sum(new), case["Hq"]
        if op == "rope":
            return dict(bytes=2 * T * (Hq + 2 * Hkv) * D + 2 * T * Hq * D + 4 * T * Hkv * D,
                        flops=3 * T * (Hq + Hkv) * case["rot"])
        tokens = sum(before) + T
        seen = sum(n * p + n * (n + 1) // 2 for p, n in zip(before, new))
        return dict(bytes=4 * T * Hq * D + 4 * tokens * Hkv * D + 4 * tokens // page, flops=4 * seen * Hq * D)
    row = 2 * Hkv * D * 2 * case["layers"]      # bytes of a token in all layers' keys and values
    if op == "fork":
        prompts, parents = _beams(case)
        n, moved, entries = case["beams"], 0, 0
        for i, p in enumerate(prompts):
            length = p + case["said"]
            moved += (length % page) * (n - len(set(parents[i * n:(i + 1) * n])))
            entries += n * -(-length // page)
        return dict(bytes=2 * row * moved + 8 * entries + 8 * len(parents), flops=entries)
    lens, keep = _rows(case)
    total, used = sum(-(-n // page) for n in lens) + 5, sum(-(-n // page) for n in keep)
    # of the used pages, as many as lie behind the first `used` places of a shuffled pool
    moved = used * (total - used) // total
    return dict(bytes=2 * row * page * moved + 8 * total + 8 * used, flops=total)


# ---- the definitions in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"chunk": _chunk64, "rope": _rope64, "beam": _beam64, "fork": _fork64, "compact": _compact64}[case["op"]](s)


def _chunk64(s):
    q, page = s["q"], s["case"]["page"]
    Hkv, G = s["k"].shape[2], q.shape[1] // s["k"].shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    table, starts = s["table"].tolist(), s["starts"].tolist()
    for b, n in enumerate(s["lens"].tolist()):
        at = torch.tensor([w & PAGE for w in table[b][:-(-n // page)]], device=q.device)
        k = s["k"][at].flatten(0, 1)[:n].double()
        v = s["v"][at].flatten(0, 1)[:n].double()
        for t0 in range(starts[b], starts[b + 1], 256):
            t1 = min(t0 + 256, starts[b + 1])
            upto = torch.arange(n - starts[b + 1] + t0, n - starts[b + 1] + t1, device=q.device)
            for h in range(Hkv):
                rows = q[t0:t1, h * G:(h + 1) * G].double().flatten(0, 1)
                x = rows @ k[:, h].T / q.shape[2] ** 0.5
                x = x.masked_fill(torch.arange(n, device=q.device) > upto.repeat_interleave(G)[:, None], -math.inf)
                out[t0:t1, h * G:(h + 1) * G] = (torch.softmax(x, dim=1) @ v[:, h]).reshape(t1 - t0, G, -1)
    return out


def _rope64(s):
    case = s["case"]
    Hq, Hkv, D, page, R = case["Hq"], case["Hkv"], case["D"], case["page"], case["rot"]
    k, v = s["k"].double(), s["v"].double()
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist()
    q = torch.zeros((starts[-1], Hq, D), dtype=torch.float64, device=k.device)
    for b, n in enumerate(lens):
        x = s["qkv"][starts[b]:starts[b + 1]].double().reshape(-1, Hq + 2 * Hkv, D)
        first = n - x.shape[0]
        pos = torch.arange(first, n, dtype=torch.float64, device=k.device)
        angle = torch.outer(pos, s["inv"]).float().double()
        turn = torch.polar(torch.full_like(angle, s["factor"]), angle)[:, None]
        y = x[:, :Hq + Hkv, :R]
        y = y.reshape(*y.shape[:2], R // 2, 2) if case["pairs"] else y.reshape(*y.shape[:2], 2, R // 2).transpose(2, 3)
        z = torch.view_as_real(torch.complex(y[..., 0], y[..., 1]) * turn)
        x[:, :Hq + Hkv, :R] = (z if case["pairs"] else z.transpose(2, 3)).flatten(2)
        q[starts[b]:starts[b + 1]] = x[:, :Hq]
        for j in range(first // page, -(-n // page)):
            lo, hi = max(first, j * page), min(n, (j + 1) * page)
            pg = table[b][j] & PAGE
            k[pg, lo - j * page:hi - j * page] = x[lo - first:hi - first, Hq:Hq + Hkv]
            v[pg, lo - j * page:hi - j * page] = x[lo - first:hi - first, Hq + Hkv:]
    return q, k, v


def _beam64(s):
    case = s["case"]
    K, V, N, alpha = case["K"], case["V"], case["N"], case["alpha"]
    scores, lengths = s["scores"].tolist(), s["lengths"].tolist()
    ended = s["ended"].tolist() if s["ended"] is not None else [[False] * K] * case["B"]
    out = torch.full((case["B"], N), -math.inf, dtype=torch.float64, device=s["x"].device)
    for b in range(case["B"]):
        found = []                                    # (rank, score)
        for k in range(K):
            if scores[b][k] == -math.inf:
                continue
            if ended[b][k]:
                found.append((scores[b][k] / max(lengths[b][k], 1) ** alpha, scores[b][k]))
                continue
            y = torch.log_softmax(s["x"][b, k].double(), dim=0)
            for t in torch.topk(y, min(N, V)).values.tolist():
                if t > -math.inf:
                    found.append(((scores[b][k] + t) / (lengths[b][k] + 1) ** alpha, scores[b][k] + t))
        found.sort(key=lambda c: -c[0])
        for i, (_, score) in enumerate(found[:N]):
            out[b, i] = score
    return None, None, out, None, None, None


def _fork64(s):
    page, refs = s["case"]["page"], s["refs"].tolist()
    old = s["table"].tolist()
    table = [list(old[p]) for p in s["parents"].tolist()]
    for rows, by in ((table, 1), (old, -1)):
        for w in (w for row in rows for w in row if w < 0):
            refs[w & PAGE] += by
    free = [p for p, c in enumerate(refs) if c == 0]
    k, v = s["k"].double(), s["v"].double()
    for row, lo, hi in zip(table, s["before"].tolist(), s["after"].tolist()):
        for j in range(lo // page, -(-hi // page)):
            had = row[j] & PAGE if row[j] < 0 else None
            if had is not None and refs[had] == 1:
                continue
            new = free.pop(0)
            refs[new] = 1
            row[j] = _word(new)
            if had is not None:
                refs[had] -= 1
                n = max(0, lo - j * page)
                k[:, new, :n], v[:, new, :n] = s["k"][:, had, :n].double(), s["v"][:, had, :n].double()
    return None, None, k, v


def _compact64(s):
    page, refs = s["case"]["page"], s["refs"].tolist()
    for row, keep in zip(s["table"].tolist(), s["keep"].tolist()):
        for w in row[-(-keep // page):]:
            if w < 0:
                refs[w & PAGE] -= 1
    n = sum(c > 0 for c in refs)
    src = [p for p in range(n, len(refs)) if refs[p]]
    dst = [p for p in range(n) if not refs[p]]
    k, v = s["k"].double(), s["v"].double()
    for a, b in zip(src, dst):
        k[:, b], v[:, b] = s["k"][:, a].double(), s["v"][:, a].double()
    return None, None, k, v
