"""Plain 64-bit forms of the paged-cache serving operators, and case makers (CPU)."""
from collections import Counter

import numpy as np
import torch

BLOCK = 16
VALID = np.int64(1) << 31


def word(page: int, valid: bool = True) -> int:
    """A page-table word (bit 31 valid, bits 30:0 the page) as the int32 the table tensor holds."""
    return int(np.array([(VALID if valid else 0) | page], np.int64).astype(np.uint32).view(np.int32)[0])


def make_table(need, num_pages, rng, width=None):
    """A table int32 [B, width] with need[b] pages a sequence, shuffled over the pool; the rest invalid."""
    order = rng.permutation(num_pages)
    assert sum(need) <= num_pages
    table = np.zeros((len(need), width or max(max(need), 1)), np.int32)
    at = 0
    for b, n in enumerate(need):
        for j in range(n):
            table[b, j] = word(int(order[at]))
            at += 1
    return table


def physical(entry) -> int:
    return int(entry) & 0x7FFFFFFF


def angles(pos, D, theta):
    """The rotation's angles [len(pos), D / 2]: binary64 products rounded to binary32."""
    inv = theta ** (-2.0 * np.arange(D // 2) / D)
    return (np.asarray(pos, np.float64)[:, None] * inv).astype(np.float32).astype(np.float64)


def rotate(x, pos, theta):
    """x [T, heads, D] rotated in split halves to positions pos [T], in 64 bits."""
    D = x.shape[2]
    a = angles(pos, D, theta)[:, None]
    lo, hi = x[..., :D // 2].astype(np.float64), x[..., D // 2:].astype(np.float64)
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], axis=2)


def codes_to_values(codes: torch.Tensor) -> np.ndarray:
    """The numbers of int8 or e4m3 codes, in 64 bits."""
    return codes.float().double().numpy()


def pool_values(codes: torch.Tensor, scales: torch.Tensor) -> np.ndarray:
    """Values [pages, heads, tokens, D] of an 8-bit pool, in 64 bits."""
    c = codes_to_values(codes)
    return c * np.repeat(scales.double().numpy(), BLOCK, axis=2)[..., None]


def attention(q, k, v, len_, Q, scale, ks=None):
    """One sequence: q [Q, Hq, D], k / v [len, Hkv, D] -> out [Q, Hq, D], and the sums the
    error bound needs: sum p |v|, the largest sum |q| |k| and sum |v| over what a row sees."""
    Hq, D = q.shape[1:]
    Hkv = k.shape[1] if len_ else 1
    g = Hq // Hkv
    out, mass, reach, size = np.zeros((Q, Hq, D)), np.zeros((Q, Hq, D)), np.zeros((Q, Hq, 1)), np.zeros((Q, Hq, D))
    for i in range(Q):
        n = len_ - Q + 1 + i
        if n < 1:
            continue
        for h in range(Hq):
            x = k[:n, h // g] @ q[i, h] * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h] = p @ v[:n, h // g]
            mass[i, h] = p @ np.abs(v[:n, h // g])
            reach[i, h] = (np.abs(k[:n, h // g]).max() * np.abs(q[i, h]).sum()) * scale
            size[i, h] = np.abs(v[:n, h // g]).sum(axis=0)
    return out, mass, reach, size


def logits(x, history, lens, prompts, rep, pres, freq, bias, allowed, real=np.float64):
    """Penalties, biases (a list of (id, value) a row) and masks (bool [B, V]) in `real` arithmetic."""
    y = x.astype(real).copy()
    one = lambda a, b: None if a is None else real(a[b])
    for b in range(len(y)):
        if history is not None:
            h = [int(t) for t in history[b, :lens[b]]]
            said = h[max(0, 0 if prompts is None else int(prompts[b])):]
            r, p, f = one(rep, b), one(pres, b), one(freq, b)
            count = Counter(said)
            for t in set(h):
                if r is not None:
                    y[b, t] = y[b, t] / r if y[b, t] > 0 else y[b, t] * r
                n = count[t]
                if n:
                    y[b, t] = (y[b, t] - (real(0) if f is None else f * real(n))) - (real(0) if p is None else p)
        if bias is not None:
            for t, w in dict(bias[b]).items():   # the last entry of an id
                y[b, t] = y[b, t] + real(w)
        if allowed is not None and allowed[b] is not None:
            y[b, ~allowed[b]] = -np.inf
    token = []
    for row in y:
        z = np.where(np.isnan(row), -np.inf, row)
        token.append(-1 if z.max() == -np.inf else int(np.argmax(z)))
    return y, token


def pack_mask(allowed):
    """bool [B, V] -> int32 [B, ceil(V / 32)]."""
    B, V = allowed.shape
    bits = np.zeros((B, -(-V // 32) * 32), np.uint8)
    bits[:, :V] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32)
