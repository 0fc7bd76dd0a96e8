"""The operators of one serving step over a paged cache, as measured cases.

A batch of sequences takes a step: the new tokens' rows are rotated and appended to
the paged cache (binary16 pages, or 8-bit pages with one scale for each block of 16
tokens and head), attention reads the 8-bit pages, and the logits get their
penalties, biases and grammar masks before the greedy choice.

A case's "op" says which: "attn" (ops.gqa_decode_q8), "append" (ops.paged_kv_append),
"append_q8" (ops.paged_kv_append_q8, read back by ops.kv_q8_values), "logits"
(ops.logits_process).  Cases are plain dicts; ``prepare`` makes a case's inputs on the
GPU from a seed, ``run`` is one pass, in plain torch operations or (``own``) through
the framework, ``work`` counts what a pass cannot do without, ``exact`` is the
operator's definition in binary64.
"""
import math
import random

import torch

own = False

BLOCK = 16            # tokens that share one scale of an 8-bit page
THETA = 1.0e6
VALID = 1 << 31       # bit 31 of a page-table word: the entry is valid


def listed():
    return [
        # one short sequence on the 14/2 heads of 64: the latency of a first answer's tokens
        dict(name="attn one short", op="attn", B=1, Q=1, Hq=14, Hkv=2, D=64, T=150, page=16, fp8=False, ragged=False),
        # a batch of conversations of very different lengths, one slot of it idle
        dict(name="attn ragged batch", op="attn", B=16, Q=1, Hq=32, Hkv=8, D=128, T=4096, page=64, fp8=True,
             ragged=True),
        # the largest: a full batch at the longest context of the 32/8 heads
        dict(name="attn long batch", op="attn", B=32, Q=1, Hq=32, Hkv=8, D=128, T=32768, page=16, fp8=False,
             ragged=False),
        # four drafted tokens of each sequence verified at once
        dict(name="attn verify", op="attn", B=8, Q=4, Hq=32, Hkv=8, D=128, T=8192, page=32, fp8=False, ragged=True),
        # one very long document, no grouping of heads, an odd length
        dict(name="attn one long", op="attn", B=1, Q=1, Hq=32, Hkv=32, D=128, T=30001, page=256, fp8=True,
             ragged=False),
        # a decode step of a batch: one token each, binary16 pages
        dict(name="append step", op="append", B=64, new=1, Hq=32, Hkv=8, D=128, ctx=30000, page=16, fp8=False),
        # prompts of a batch at once, binary16 pages, the 14/2 heads of 64
        dict(name="append prompts", op="append", B=6, new=4001, Hq=14, Hkv=2, D=64, ctx=0, page=64, fp8=False),
        # a decode step into 8-bit pages: the open blocks' scales may grow
        dict(name="append q8 step", op="append_q8", B=48, new=1, Hq=14, Hkv=2, D=64, ctx=4000, page=64, fp8=False),
        # chunks of prompts into 8-bit pages, continuing earlier chunks that ended inside a block
        dict(name="append q8 prompts", op="append_q8", B=5, new=2500, Hq=32, Hkv=8, D=128, ctx=5000, page=128,
             fp8=True),
        # one conversation: all penalties, a bias list and a grammar over a large vocabulary
        dict(name="logits one row", op="logits", B=1, V=151936, half=False, L=700, bias=40, grammar=True),
        # a batch of conversations with histories of up to 2048 tokens, binary16 logits
        dict(name="logits batch", op="logits", B=64, V=151936, half=True, L=2048, bias=100, grammar=True),
        # many short conversations over a small vocabulary, penalties only
        dict(name="logits many rows", op="logits", B=200, V=32000, half=False, L=300, bias=0, grammar=False),
    ]


HEADS = [(14, 2, 64), (32, 8, 128), (32, 32, 128), (28, 4, 128), (8, 8, 64), (16, 2, 128)]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "append", "append_q8", "logits"])
    if op == "logits":
        B = _log_int(rng, 1, 256)
        V = _log_int(rng, 1000, min(151936, 9_700_000 // B))
        return dict(op=op, B=B, V=V, half=rng.random() < 0.5, L=_log_int(rng, 1, 4096),
                    bias=rng.choice([0, 1, 30, 300]), grammar=rng.random() < 0.5)
    Hq, Hkv, D = rng.choice(HEADS)
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if op == "attn":
        B = _log_int(rng, 1, 64)
        Q = rng.choice([1, 1, 1, 2, 3, 5, 8])
        top = min(131072, (1 << 30) // (B * Hkv * D * (1 if Q * Hq // Hkv <= 8 else 4)))
        return dict(op=op, B=B, Q=Q, Hq=Hq, Hkv=Hkv, D=D, T=_log_int(rng, 1, top), page=page,
                    fp8=rng.random() < 0.5, ragged=rng.random() < 0.6)
    B = _log_int(rng, 1, 64)
    new = 1 if rng.random() < 0.4 else _log_int(rng, 1, max(1, 20_000_000 // (B * (Hq + 2 * Hkv) * D)))
    return dict(op=op, B=B, new=new, Hq=Hq, Hkv=Hkv, D=D, ctx=rng.choice([0, 15, 1000, 30000]), page=page,
                fp8=op == "append_q8" and rng.random() < 0.5)


# ---- a case's lengths: its own, whatever the seed ---------------------------

def _lens(case):
    """attn: the sequences' lengths; append: (tokens before, new tokens) of each."""
    r = random.Random("%d %d %d" % (case["B"], case.get("T", case.get("new")), case["page"]))
    B = case["B"]
    if case["op"] == "attn":
        T = case["T"]
        if not case["ragged"]:
            return [T] * B
        lens = [T] + [r.randint(1, T) for _ in range(B - 1)]
        if B >= 4:
            lens[1] = 0      # an idle slot of the batch
        return lens
    new = case["new"]
    before = [r.randint(0, case["ctx"]) for _ in range(B)]
    return before, [new if b == 0 or new == 1 else r.randint(1, new) for b in range(B)]


def _word(page):
    """A page-table word as the int32 that the table holds."""
    return (page | VALID) - (1 << 32)


def _history(case):
    r = random.Random("%d %d %d" % (case["B"], case["V"], case["L"]))
    lens = [case["L"]] + [r.randint(0, case["L"]) for _ in range(case["B"] - 1)]
    return lens, [r.randint(0, n) for n in lens]


# ---- inputs ------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    r = random.Random(int(seed))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    if case["op"] == "logits":
        return _prepare_logits(case, g, ints, dev)
    Hq, Hkv, D, page, B = case["Hq"], case["Hkv"], case["D"], case["page"], case["B"]
    code_type = torch.float8_e4m3fn if case["fp8"] else torch.int8

    def codes(pages):
        # what a quantised bell curve leaves: most codes well inside the range
        x = torch.randn((pages, Hkv, page, D), generator=g, device=dev, dtype=torch.float16)
        return (x * 100).clamp_(-448, 448).to(code_type) if case["fp8"] else x.mul_(40).round_().clamp_(-127, 127).to(code_type)

    def scales(pages):
        if case["fp8"]:
            return torch.randint(-8, -5, (pages, Hkv, page // BLOCK), generator=g, device=dev).float().exp2()
        return (torch.rand((pages, Hkv, page // BLOCK), generator=g, device=dev) + 0.5) * 0.025

    if case["op"] == "attn":
        lens = _lens(case)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 1
        order = torch.randperm(pages, generator=g, device=dev).tolist()
        table, at = [[0] * max(max(need), 1) for _ in lens], 0
        for b, n in enumerate(need):
            for j in range(n):
                table[b][j] = _word(order[at])
                at += 1
        q = torch.randn((B, case["Q"], Hq, D), generator=g, device=dev) * 3
        return dict(case=dict(case), q=q.half(), k=codes(pages), v=codes(pages), ks=scales(pages), vs=scales(pages),
                    table=ints(table), lens=ints(lens))
    # append: the pool holds the pages that the call touches (and some that it must
    # leave alone); a real pool's other pages are neither read nor written
    before, new = _lens(case)
    first = [p // page for p in before]
    last = [(p + n - 1) // page for p, n in zip(before, new)]
    touched = sum(b - a + 1 for a, b in zip(first, last))
    pages = touched + max(1, touched // 8)
    order = list(range(pages))
    r.shuffle(order)
    table, at = [[0] * (max(last) + 1) for _ in new], 0
    for b in range(B):
        for j in range(first[b], last[b] + 1):
            table[b][j] = _word(order[at])
            at += 1
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    qkv = torch.randn((starts[-1], (Hq + 2 * Hkv) * D), generator=g, device=dev)
    s = dict(case=dict(case), qkv=qkv.half(), table=ints(table), starts=ints(starts),
             lens=ints([p + n for p, n in zip(before, new)]))
    if case["op"] == "append":
        for name in "kv":
            s[name] = torch.randn((pages, page, Hkv, D), generator=g, device=dev).half()
    else:
        s.update(k=codes(pages), v=codes(pages), ks=scales(pages), vs=scales(pages))
    return s


def _prepare_logits(case, g, ints, dev):
    B, V, L = case["B"], case["V"], case["L"]
    lens, prompts = _history(case)
    logits = torch.randn((B, V), generator=g, device=dev) * 3
    # a few words come often, most hardly ever
    ids = (torch.rand((B, L), generator=g, device=dev).pow(4) * V).long().clamp_(0, V - 1)
    u = lambda lo, hi: torch.rand(B, generator=g, device=dev) * (hi - lo) + lo
    s = dict(case=dict(case), logits=logits.half() if case["half"] else logits, ids=ids.int(), lens=ints(lens),
             prompts=ints(prompts), rep=u(1.0, 1.3), pres=u(0.0, 0.8), freq=u(0.0, 0.4), bias_starts=None,
             bias_ids=None, bias=None, allowed=None)
    if case["bias"]:
        n = case["bias"]
        s["bias_starts"] = torch.arange(0, B * n + 1, n, device=dev, dtype=torch.int32)
        s["bias_ids"] = torch.randint(0, V, (B * n,), generator=g, device=dev, dtype=torch.int32)
        s["bias"] = torch.randn(B * n, generator=g, device=dev) * 4
    if case["grammar"]:
        words = -(-V // 32)
        bits = torch.randint(-(1 << 31), 1 << 31, (2, B, words), generator=g, device=dev, dtype=torch.int64)
        wide = (torch.rand((B, 1), generator=g, device=dev) < 0.5)
        sparse = bits[0] & bits[1] & (torch.rand((B, words), generator=g, device=dev) < 0.02)
        s["allowed"] = torch.where(wide, bits[0] | bits[1], sparse).int()
    return s


# ---- one pass ----------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        from anvilq_b200 import ops
        if case["op"] == "attn":
            return ops.gqa_decode_q8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"])
        if case["op"] == "append":
            q = ops.paged_kv_append(s["qkv"], s["k"], s["v"], s["table"], s["lens"], s["starts"], case["Hq"], THETA)
            return q, s["k"], s["v"]
        if case["op"] == "append_q8":
            q = ops.paged_kv_append_q8(s["qkv"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"],
                                       s["starts"], case["Hq"], THETA)
            k, v = ops.kv_q8_values(s["k"], s["v"], s["ks"], s["vs"])
            return q, k, v, s["ks"], s["vs"]
        return ops.logits_process(s["logits"], history=s["ids"], history_lens=s["lens"], prompt_lens=s["prompts"],
                                  repetition=s["rep"], presence=s["pres"], frequency=s["freq"],
                                  bias_starts=s["bias_starts"], bias_ids=s["bias_ids"], bias_values=s["bias"],
                                  allowed=s["allowed"])
    return {"attn": _attn, "append": _append, "append_q8": _append_q8, "logits": _logits}[case["op"]](s)


def _take(t, index):
    """t[index] for any element type (8-bit floats as bytes)."""
    return t.view(torch.uint8)[index].view(t.dtype) if t.dtype == torch.float8_e4m3fn else t[index]


def _values(codes, scales):
    """The numbers that 8-bit pages [pages, heads, tokens, D] stand for, in 32 bits."""
    return codes.float() * scales.repeat_interleave(BLOCK, dim=-1)[..., None]


def _attn(s):
    q, page = s["q"], s["case"]["page"]
    B, Q, Hq, D = q.shape
    Hkv = s["k"].shape[1]
    at = (s["table"] & 0x7FFFFFFF).long()
    T = at.shape[1] * page
    k = _values(_take(s["k"], at), s["ks"][at]).transpose(1, 2).reshape(B, Hkv, T, D)
    v = _values(_take(s["v"], at), s["vs"][at]).transpose(1, 2).reshape(B, Hkv, T, D)
    rows = q.float().reshape(B, Q, Hkv, Hq // Hkv, D).transpose(1, 2).reshape(B, Hkv, -1, D)
    x = torch.matmul(rows, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    # query i of a sequence sits at position length - Q + i and sees positions up to its own
    sees = s["lens"][:, None] - Q + 1 + torch.arange(Q, device=q.device)
    mask = torch.arange(T, device=q.device) < sees.repeat_interleave(Hq // Hkv, dim=1)[:, None, :, None]
    x = torch.where(mask, x, -math.inf)
    top = x.amax(dim=3, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(dim=3, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return o.reshape(B, Hkv, Q, Hq // Hkv, D).transpose(1, 2).reshape(B, Q, Hq, D).half()


def _rotated(s):
    """(q, k, v of every new token in 32 bits, its sequence's page, its slot in the page, its position)."""
    case = s["case"]
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    T, dev = s["qkv"].shape[0], s["qkv"].device
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(s["starts"].long(), t, right=True) - 1
    pos = s["lens"].long()[b] - s["starts"].long()[b + 1] + t
    inv = THETA ** (-2.0 * torch.arange(D // 2, device=dev, dtype=torch.float64) / D)
    # the angle is a binary64 product rounded to binary32: the operator's definition
    angle = (pos.double()[:, None] * inv).float()
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    x = s["qkv"].float().reshape(T, Hq + 2 * Hkv, D)
    lo, hi = x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:]
    turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], dim=2)
    at = (s["table"].long()[b, pos // page] & 0x7FFFFFFF)
    return turned[:, :Hq], turned[:, Hq:], x[:, Hq + Hkv:], at, pos % page, pos


def _append(s):
    q, k, v, at, slot, _ = _rotated(s)
    s["k"][at, slot] = k.half()
    s["v"][at, slot] = v.half()
    return q.half(), s["k"], s["v"]


def _scale_for(top, fp8):
    """The scale of a block whose largest magnitude is `top`."""
    if not fp8:
        return top / 127.0
    m, e = torch.frexp(top)                    # top = m 2^e, 0.5 <= m < 1; 448 = 0.875 2^9
    e = (e - torch.where(m <= 0.875, 9, 8)).clamp(min=-126)
    return torch.where(top > 0, ((e + 127) << 23).to(torch.int32).view(torch.float32), 0.0)


def _coded(x, fp8):
    return x.clamp(-448, 448).to(torch.float8_e4m3fn) if fp8 else x.round().clamp(-127, 127).to(torch.int8)


def _append_q8_one(codes, scales, x, at, slot, fp8):
    pages, Hkv, page, D = codes.shape
    T, per = x.shape[0], page // BLOCK
    blocks, mine = torch.unique(at * per + slot // BLOCK, return_inverse=True)     # the blocks that get new rows
    top = torch.zeros((blocks.numel(), Hkv), device=x.device)
    top = top.scatter_reduce(0, mine[:, None].expand(T, Hkv), x.abs().amax(dim=2), "amax")
    first = torch.full((blocks.numel(),), BLOCK, device=x.device, dtype=torch.long)
    first = first.scatter_reduce(0, mine, slot % BLOCK, "amin")                    # rows before it are kept
    pg, blk = blocks // per, blocks % per
    kept = torch.where(first[:, None] > 0, scales[pg, :, blk], 0.0)
    scale = torch.maximum(kept, _scale_for(top, fp8))
    safe = torch.where(scale > 0, scale, 1.0)
    tok = blk[:, None] * BLOCK + torch.arange(BLOCK, device=x.device)
    old = _take(codes, (pg[:, None], slice(None), tok))                            # [blocks, 16, Hkv, D]
    again = _coded(old.float() * (kept / safe)[:, None, :, None], fp8)
    again = torch.where((torch.arange(BLOCK, device=x.device) < first[:, None])[:, :, None, None],
                        again.view(torch.uint8), old.view(torch.uint8))
    raw = codes.view(torch.uint8)
    raw[pg[:, None], :, tok] = again
    new = _coded(x * (1.0 / safe)[mine][:, :, None], fp8)
    raw[at, :, slot] = new.view(torch.uint8)
    scales[pg, :, blk] = scale


def _append_q8(s):
    q, k, v, at, slot, _ = _rotated(s)
    fp8 = s["case"]["fp8"]
    _append_q8_one(s["k"], s["ks"], k, at, slot, fp8)
    _append_q8_one(s["v"], s["vs"], v, at, slot, fp8)
    return q.half(), _values(s["k"], s["ks"]).half(), _values(s["v"], s["vs"]).half(), s["ks"], s["vs"]


def _logits(s):
    x = s["logits"].float()
    B, V = x.shape
    ids, dev = s["ids"].long(), x.device
    at = torch.arange(ids.shape[1], device=dev)
    live = at < s["lens"][:, None]
    said = live & (at >= s["prompts"][:, None])
    seen = torch.zeros((B, V), device=dev).scatter_add_(1, ids, live.float())
    count = torch.zeros((B, V), device=dev).scatter_add_(1, ids, said.float())
    rep = s["rep"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, x - s["freq"][:, None] * count - s["pres"][:, None], x)
    if s["bias"] is not None:
        n = s["bias_ids"].shape[0]
        row = torch.searchsorted(s["bias_starts"].long(), torch.arange(n, device=dev), right=True) - 1
        # an id's last entry counts
        entry = torch.full((B * V,), -1, device=dev, dtype=torch.long)
        entry = entry.scatter_reduce(0, row * V + s["bias_ids"].long(), torch.arange(n, device=dev), "amax")
        entry = entry.reshape(B, V)
        x = torch.where(entry >= 0, x + s["bias"][entry.clamp(min=0)], x)
    if s["allowed"] is not None:
        t = torch.arange(V, device=dev)
        x = torch.where((s["allowed"][:, t // 32] >> (t % 32)) & 1 != 0, x, -math.inf)
    top = x.amax(dim=1, keepdim=True)
    # the lowest of the largest; none where nothing is allowed
    token = torch.where(x == top, torch.arange(V, device=dev, dtype=torch.int32), V).amin(dim=1)
    return x, torch.where(top[:, 0] == -math.inf, -1, token).int()


# ---- what a pass cannot do without --------------------------------------------

def work(case):
    if case["op"] == "logits":
        B, V = case["B"], case["V"]
        lens, _ = _history(case)
        n = B * V * (2 if case["half"] else 4) + B * V * 4 + 4 * sum(lens) + 24 * B
        n += 8 * B * case["bias"] + (B * (-(-V // 32)) * 4 if case["grammar"] else 0)
        return dict(bytes=n, flops=3 * sum(lens) + 2 * B * case["bias"] + B * V)
    Hq, Hkv, D, B = case["Hq"], case["Hkv"], case["D"], case["B"]
    if case["op"] == "attn":
        lens, Q = _lens(case), case["Q"]
        tokens = sum(lens)
        blocks = sum(-(-n // BLOCK) for n in lens)
        n = 2 * tokens * Hkv * D + 8 * blocks * Hkv + 4 * B * Q * Hq * D + 4 * sum(-(-n // case["page"]) for n in lens)
        seen = sum(max(0, n - Q + 1 + i) for n in lens for i in range(Q))
        return dict(bytes=n + 4 * B, flops=4 * seen * Hq * D)
    before, new = _lens(case)
    T = sum(new)
    n = 2 * T * (Hq + 2 * Hkv) * D + 2 * T * Hq * D + 8 * B
    flops = 3 * T * (Hq + Hkv) * D
    if case["op"] == "append":
        return dict(bytes=n + 4 * T * Hkv * D, flops=flops)
    # the codes and scales written, then all pages read back: a code, a scale's share and a binary16 value each
    page = case["page"]
    touched = sum((p + m - 1) // page - p // page + 1 for p, m in zip(before, new))
    cells = 2 * (touched + max(1, touched // 8)) * page * Hkv * D
    return dict(bytes=n + 2 * T * Hkv * D + 3 * cells + 4 * cells // (BLOCK * D), flops=flops + 3 * T * Hkv * D * 2)


# ---- the definitions in 64 bits -------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _attn64, "append": _append64, "append_q8": _append64, "logits": _logits64}[case["op"]](s)


def _pages64(codes, scales, words, heads):
    """The values of a sequence's pages, [tokens, heads, D]."""
    at = torch.tensor([w & 0x7FFFFFFF for w in words], device=codes.device, dtype=torch.long)
    c = _take(codes, at).float().double()
    n, _, page, D = c.shape
    c = c.reshape(n, heads, page // BLOCK, BLOCK, D) * scales[at].double()[..., None, None]
    return c.reshape(n, heads, page, D).permute(0, 2, 1, 3).reshape(n * page, heads, D)


def _attn64(s):
    q, page = s["q"].double(), s["case"]["page"]
    B, Q, Hq, D = q.shape
    Hkv = s["k"].shape[1]
    out = torch.zeros_like(q)
    table = s["table"].tolist()
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        words = table[b][:-(-n // page)]
        k = _pages64(s["k"], s["ks"], words, Hkv)[:n]
        v = _pages64(s["v"], s["vs"], words, Hkv)[:n]
        for i in range(Q):
            upto = n - Q + 1 + i
            if upto < 1:
                continue
            qi = q[b, i].reshape(Hkv, Hq // Hkv, D)
            w = torch.softmax(torch.einsum("hgd,thd->hgt", qi, k[:upto]) / D ** 0.5, dim=2)
            out[b, i] = torch.einsum("hgt,thd->hgd", w, v[:upto]).reshape(Hq, D)
    return out


def _round_e4m3(x):
    """x to the nearest number of 4 exponent and 3 fraction bits, ties to even."""
    e = torch.frexp(x.abs().clamp(min=2.0 ** -40))[1] - 1
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), e.clamp(min=-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _append64(s):
    case = s["case"]
    Hq, Hkv, D, page, fp8 = case["Hq"], case["Hkv"], case["D"], case["page"], case["fp8"]
    q8 = case["op"] == "append_q8"
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].tolist()
    dev = s["qkv"].device
    q_out = torch.zeros((starts[-1], Hq, D), dtype=torch.float64, device=dev)
    if q8:
        codes = [_take(s[n], slice(None)).float().double() for n in "kv"]
        scales = [s[n].double().clone() for n in ("ks", "vs")]
    else:
        pools = [s[n].double().clone() for n in "kv"]
    half = D // 2
    inv = torch.tensor([THETA ** (-2.0 * i / D) for i in range(half)], dtype=torch.float64, device=dev)
    for b, n in enumerate(lens):
        new = starts[b + 1] - starts[b]
        x = s["qkv"][starts[b]:starts[b + 1]].double().reshape(new, Hq + 2 * Hkv, D)
        pos = torch.arange(n - new, n, dtype=torch.float64, device=dev)
        angle = torch.outer(pos, inv).float().double()
        turn = torch.complex(torch.cos(angle), torch.sin(angle))[:, None]
        z = torch.complex(x[:, :Hq + Hkv, :half], x[:, :Hq + Hkv, half:]) * turn
        z = torch.cat([z.real, z.imag], dim=2)
        q_out[starts[b]:starts[b + 1]] = z[:, :Hq]
        at = n - new
        while at < n:                      # block by block
            upto = min(n, (at // BLOCK + 1) * BLOCK)
            pg, slot = table[b][at // page] & 0x7FFFFFFF, at % page
            rows = slice(at - (n - new), upto - (n - new))
            for side, y in enumerate((z[rows, Hq:], x[rows, Hq + Hkv:])):
                if not q8:
                    pools[side][pg, slot:slot + upto - at] = y
                    continue
                blk, before = slot // BLOCK, slot % BLOCK
                top = y.abs().amax(dim=(0, 2))
                if fp8:
                    want = torch.pow(2.0, torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)))
                    want = torch.where(top > 0, want, torch.zeros_like(want))
                else:
                    want = top / 127
                kept = scales[side][pg, :, blk] if before else torch.zeros_like(want)
                scale = torch.maximum(kept, want)
                code = _round_e4m3 if fp8 else (lambda a: torch.round(a).clamp(-127, 127))
                safe = torch.where(scale > 0, scale, torch.ones_like(scale))[:, None, None]
                c = codes[side]
                if before:
                    old = slice(blk * BLOCK, blk * BLOCK + before)
                    c[pg, :, old] = code(c[pg, :, old] * kept[:, None, None] / safe)
                c[pg, :, slot:slot + upto - at] = code(y.transpose(0, 1) / safe)
                scales[side][pg, :, blk] = scale
            at = upto
    if not q8:
        return q_out, pools[0], pools[1]
    values = [c * torch.repeat_interleave(w, BLOCK, dim=2)[..., None] for c, w in zip(codes, scales)]
    return q_out, values[0], values[1], scales[0], scales[1]


def _logits64(s):
    x = s["logits"].double().clone()
    lens, prompts = s["lens"].tolist(), s["prompts"].tolist()
    for b in range(x.shape[0]):
        seen = torch.unique(s["ids"][b, :lens[b]].long())
        y = x[b, seen]
        x[b, seen] = torch.where(y > 0, y / s["rep"][b].double(), y * s["rep"][b].double())
        said, count = torch.unique(s["ids"][b, prompts[b]:lens[b]].long(), return_counts=True)
        x[b, said] -= s["freq"][b].double() * count + s["pres"][b].double()
        if s["bias"] is not None:
            lo, hi = s["bias_starts"][b:b + 2].tolist()
            last = dict(zip(s["bias_ids"][lo:hi].tolist(), s["bias"][lo:hi].tolist()))
            x[b, torch.tensor(list(last), device=x.device)] += torch.tensor(list(last.values()), device=x.device,
                                                                             dtype=torch.float64)
        if s["allowed"] is not None:
            word = s["allowed"][b].long()[:, None]
            bits = ((word >> torch.arange(32, device=x.device)) & 1).reshape(-1)[:x.shape[1]]
            x[b, bits == 0] = -math.inf
    return x, None
