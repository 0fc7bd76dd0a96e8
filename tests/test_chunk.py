"""Arguments that the chunk attention refuses, on the host, before any launch."""
import ctypes

import pytest
import torch

from anvilq_b200 import _lib, ops

EINVAL, EALIGN, EWORKSPACE, ESHAPE = -1, -2, -4, -5


def at(byte):
    return ctypes.c_void_p((1 << 20) + byte)   # never dereferenced: every call here is rejected


# 4 tokens of 8 heads of 128: 8192 bytes of q and out; 8 pages x 16 x 2 x 128: 65536 bytes of a pool
CHUNK = dict(q=at(0), stride=1024, k=at(1 << 20), v=at(2 << 20), table=at(3 << 20), lens=at(4 << 20), starts=at(5 << 20),
             out=at(6 << 20), T=4, B=2, Hq=8, Hkv=2, D=128, page=16, max_pages=4, pages=8, scale=0.0, ws=at(1 << 24),
             bytes=1 << 30, err=at(-64), flags=0, stream=None)


@pytest.mark.parametrize("status,change", [
    *((EINVAL, {k: None}) for k in ("q", "k", "v", "table", "lens", "starts", "out", "err")), (EINVAL, dict(flags=2)),
    *((EINVAL, dict(scale=s)) for s in (float("nan"), float("inf"), float("-inf"), 2.0 ** 33)),
    (EINVAL, dict(T=-1)), (EINVAL, dict(stride=1016)),
    *((ESHAPE, c) for c in (dict(B=0), dict(B=65536), dict(Hq=9, stride=2048), dict(Hkv=0), dict(Hq=1032, Hkv=1032, stride=1 << 20),
                            dict(Hq=258, stride=1 << 20), dict(D=96), dict(page=8), dict(page=24), dict(max_pages=0),
                            dict(pages=0), dict(page=1 << 20, max_pages=2000), dict(pages=1 << 27, page=16))),
    (ESHAPE, dict(T=(1 << 30) + 1)),
    *((EALIGN, c) for c in (dict(q=at(8)), dict(k=at((1 << 20) + 8)), dict(v=at((2 << 20) + 2)),
                            dict(out=at((6 << 20) + 4)), dict(ws=at((1 << 24) + 8)), dict(stride=1028))),
    *((EINVAL, dict(out=at(b))) for b in (0, 16, 8176, (1 << 20) - 16, (1 << 20) + 65520, (2 << 20) + 64, (3 << 20) + 16,
                                          (4 << 20), (5 << 20) - 8176, (1 << 24) + 4096)),
])
def test_refused_before_launch(status, change):
    assert set(change) <= set(CHUNK)
    assert _lib.load().anvilq_gqa_chunk_paged(*{**CHUNK, **change}.values()) == status


def test_no_tokens_is_no_work():
    assert _lib.load().anvilq_gqa_chunk_paged(*{**CHUNK, "T": 0, "q": None, "out": None}.values()) == 0


def test_workspace_sizes_of_unsupported_shapes():
    size = _lib.load().anvilq_gqa_chunk_paged_workspace_size
    for shape in ((4, 0, 8, 2, 128, 16, 4), (4, 2, 9, 2, 128, 16, 4), (4, 2, 8, 2, 80, 16, 4), (4, 2, 8, 2, 128, 17, 4),
                  (-1, 2, 8, 2, 128, 16, 4), (4, 2, 8, 2, 128, 16, 0), (4, 2, 258, 2, 128, 16, 4)):
        assert size(*shape) == 0


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("change,error", [
    (dict(), ValueError),                                                              # CPU tensors
    (dict(q=torch.zeros(5, 4, 64)), TypeError), (dict(k=torch.zeros(4, 16, 2, 64)), TypeError),
    (dict(q=half(5, 4, 128)), ValueError), (dict(q=half(5, 256)), ValueError), (dict(v=half(4, 32, 2, 64)), ValueError),
    (dict(k=half(4, 2, 16, 64).transpose(1, 2)), ValueError), (dict(q=half(5, 64, 4).transpose(1, 2)), ValueError),
    (dict(q=half(1, 4, 64).expand(5, 4, 64)), ValueError), (dict(q=half(5, 8, 64)[:, ::2]), ValueError),
    (dict(starts=ints(2)), ValueError), (dict(starts=ints(3).long()), ValueError), (dict(lens=ints(3)), ValueError),
    (dict(table=ints(6)), ValueError), (dict(out=half(5, 4, 128)), ValueError), (dict(out=torch.zeros(5, 4, 64)), ValueError),
])
def test_front_end(change, error):
    a = dict(q=half(5, 4, 64), k=half(4, 16, 2, 64), v=half(4, 16, 2, 64), table=ints(2, 3), lens=ints(2),
             starts=ints(3), out=None)
    a.update(change)
    with pytest.raises(error):
        ops.gqa_chunk_paged(a["q"], a["k"], a["v"], a["table"], a["lens"], a["starts"], out=a["out"])
