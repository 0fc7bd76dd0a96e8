"""Prompts, beams and shared pages together, as a serving loop uses them: prompts appended in
chunks with a scaled rotation and attended to over the pages, forked into beams, and a beam
search stepped on: pages reserved, rows appended, decode attention, penalties and masks,
selection, reordering, fork, release and compaction.  Every hypothesis' score is held to the
sum of log probabilities that its tokens have when the whole sequence is computed in 64 bits."""
import numpy as np
import pytest
import torch

import pages_oracle as po
import serving_oracle as so
from anvilq_b200 import ops

pytestmark = pytest.mark.gpu
Hq, Hkv, D, V, PAGE, R = 4, 2, 64, 50, 16, 32
ITEMS, K, STEPS, EOS = 2, 3, 40, 7


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


class Model:
    """Tokens to rows of [q | k | v], one layer of attention, and a projection to logits."""

    def __init__(self, rng, dev):
        self.rows = (rng.standard_normal((V, (Hq + 2 * Hkv) * D)) * 0.7).astype(np.float16)
        self.out = (rng.standard_normal((Hq * D, V)) * 0.25).astype(np.float32)
        self.d_rows, self.d_out = torch.from_numpy(self.rows).to(dev), torch.from_numpy(self.out).to(dev)
        self.inv, self.factor = ops.rope_frequencies(R, 1e4, dict(kind="yarn", factor=4.0, original=64), dev)
        self.turn = dict(inv_freq=self.inv, interleaved=True, rope_factor=self.factor)

    def log_probs(self, tokens, masks):
        """In 64 bits: log probabilities after every token, and how far binary16 rotated rows and
        probabilities, and the binary16 attention output, may move them: a score by 2^-10 of
        sum |q| |k| (two roundings), a probability by twice that and 2^-11 of its own, the
        logits by their weights' magnitudes, a log probability by twice the largest logit's."""
        x = self.rows[tokens].astype(np.float64).reshape(len(tokens), Hq + 2 * Hkv, D)
        angle = (np.arange(len(tokens))[:, None] * self.inv.cpu().numpy()).astype(np.float32).astype(np.float64)[:, None]
        c, s = self.factor * np.cos(angle), self.factor * np.sin(angle)
        y = x[:, :Hq + Hkv].copy()
        a, b = x[:, :Hq + Hkv, 0:R:2], x[:, :Hq + Hkv, 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
        q, k, v = y[:, :Hq], y[:, Hq:], x[:, Hq + Hkv:]
        o, off = np.zeros((len(tokens), Hq, D)), 0.0
        for h in range(Hq):
            w = q[:, h] @ k[:, h // 2].T / np.sqrt(D)
            w[np.triu_indices(len(tokens), 1)] = -np.inf
            p = np.exp(w - w.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            o[:, h] = p @ v[:, h // 2]
            reach = np.abs(q[:, h]).sum(axis=1).max() * np.abs(k[:, h // 2]).max() / np.sqrt(D)
            off = max(off, (4 * 2.0 ** -10 * reach + 2.0 ** -10) * np.abs(v[:, h // 2]).max())
        logits = o.reshape(len(tokens), -1) @ self.out.astype(np.float64)
        slack = 2 * off * np.abs(self.out).sum(axis=0).max()
        logits[:, ~masks] = -np.inf
        top = logits.max(axis=1, keepdims=True)
        return logits - top - np.log(np.exp(logits - top).sum(axis=1, keepdims=True)), slack


def test_a_beam_search(dev):
    rng = np.random.default_rng(17)
    m = Model(rng, dev)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    prompts = [[int(t) for t in rng.integers(0, V, size=n)] for n in (37, 20)]
    allowed = rng.random(V) < 0.8
    allowed[EOS] = True
    mask = torch.from_numpy(so.pack_mask(np.repeat(allowed[None], ITEMS * K, 0))).to(dev)
    pages, width = 60, 6
    k_pool, v_pool = (torch.full((pages, PAGE, Hkv, D), float("nan"), dtype=torch.float16, device=dev) for _ in range(2))
    cache = ops.PagePools([k_pool, v_pool], PAGE)
    table, refs = torch.zeros((ITEMS, width), dtype=torch.int32, device=dev), torch.zeros(pages, dtype=torch.int32,
                                                                                          device=dev)

    def consistent():
        ops.raise_device_errors(dev)
        assert refs.tolist() == po.counts(po.rows(table.cpu().numpy()), pages)

    # prompts in two chunks of unlike sizes
    done, last = [0] * ITEMS, None
    for share in (0.4, 1.0):
        upto = [max(1, int(len(p) * share)) for p in prompts]
        rows = [t for p, a, b in zip(prompts, done, upto) for t in p[a:b]]
        starts = ints(np.concatenate([[0], np.cumsum([b - a for a, b in zip(done, upto)])]).tolist())
        assert int(ops.pages_reserve(table, refs, ints(done), ints(upto), PAGE, cache)) == 0
        q = ops.paged_kv_append(m.d_rows[torch.tensor(rows, device=dev)], k_pool, v_pool, table, ints(upto), starts, Hq,
                                **m.turn)
        o = ops.gqa_chunk_paged(q, k_pool, v_pool, table, ints(upto), starts)
        last = o[(starts[1:] - 1).long()]
        done = upto
        consistent()
    logits = last.reshape(ITEMS, -1).float() @ m.d_out
    # every item's beams start as its prompt; of the first step only one counts
    table = ops.pages_fork(table, refs, ints([i for i in range(ITEMS) for _ in range(K)]))
    logits = logits.repeat_interleave(K, 0).contiguous()
    scores = torch.full((ITEMS, K), -float("inf"), device=dev)
    scores[:, 0] = 0.0
    lengths, ended = torch.zeros((ITEMS, K), dtype=torch.int32, device=dev), torch.zeros((ITEMS, K), dtype=torch.bool,
                                                                                        device=dev)
    history = torch.zeros((ITEMS, K, STEPS), dtype=torch.int32, device=dev)
    at = ints(done).repeat_interleave(K).reshape(ITEMS, K)       # tokens in the cache
    starts = torch.arange(ITEMS * K + 1, dtype=torch.int32, device=dev)
    spare = torch.empty_like(table)
    for step in range(STEPS):
        logits, _ = ops.logits_process(logits, allowed=mask, choose=True)
        tokens, parents, scores, lengths, ended = ops.beam_select(
            logits.view(ITEMS, K, V), scores, lengths=lengths, length_penalty=0.8, finished=ended, eos_ids=ints([EOS]),
            pad_id=EOS)
        history, at = ops.beam_reorder([history, at], parents)
        history.scatter_(2, (lengths.long() - 1).clamp(min=0)[..., None], torch.where(
            (lengths > 0) & (tokens >= 0), tokens, 0)[..., None])
        table, spare = ops.pages_fork(table, refs, parents, out=spare), table
        consistent()
        if step + 1 == STEPS:
            break
        flat = at.reshape(-1)
        assert int(ops.pages_reserve(table, refs, flat, flat + 1, PAGE, cache)) == 0
        consistent()
        at = at + 1
        q = ops.paged_kv_append(m.d_rows[tokens.reshape(-1).long().clamp(min=0)], k_pool, v_pool, table, at.reshape(-1),
                                starts, Hq, **m.turn)
        if step % 2:
            o = ops.gqa_decode_paged(q, k_pool, v_pool, table, at.reshape(-1))
        else:
            o = ops.gqa_chunk_paged(q, k_pool, v_pool, table, at.reshape(-1), starts)
        logits = o.reshape(ITEMS * K, -1).float() @ m.d_out
        if step % 11 == 5:      # pages brought together in the middle of it
            _, _, used = ops.pages_compact(table, refs, cache)
            assert int(used) == int((refs > 0).sum())
            consistent()
    ops.raise_device_errors(dev)
    shared = sum(c > 1 for c in refs.tolist())
    assert shared, "beams share their prompt's pages"
    seen = set()
    for i in range(ITEMS):
        assert (scores[i].isfinite()).all()
        for b in range(K):
            n = int(lengths[i, b])
            said = [int(t) for t in history[i, b, :n]]
            assert all(allowed[t] for t in said) and (EOS not in said[:-1]) and bool(ended[i, b]) == (said[-1] == EOS)
            logp, slack = m.log_probs(np.array(prompts[i] + said), allowed)
            want = sum(logp[len(prompts[i]) - 1 + j, t] for j, t in enumerate(said))
            assert abs(float(scores[i, b]) - want) <= n * slack, (i, b, float(scores[i, b]), want, slack)
            # (they are far from all alike: a wrong row in the cache moves a score by about 1)
            assert abs(float(scores[i, b]) - want) <= 0.02 * n
            seen.add((i, tuple(said)))
    assert len(seen) == ITEMS * K, "hypotheses differ"
    # all of it is given back
    ops.pages_release(table, refs, torch.zeros(ITEMS * K, dtype=torch.int32, device=dev), PAGE)
    consistent()
    assert not refs.any() and not table.any()
