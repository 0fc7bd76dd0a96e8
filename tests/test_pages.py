"""Arguments that the calls on shared pages refuse, on the host, before any launch."""
import ctypes

import pytest
import torch

from anvilq_b200 import AnvilqError, _lib, ops

EINVAL, EALIGN, EWORKSPACE, ESHAPE = -1, -2, -4, -5


def at(byte):
    return ctypes.c_void_p((1 << 20) + byte)   # never dereferenced: every call here is rejected


def pool(**change):
    a = (_lib.PagePool * 1)()
    for k, v in {**dict(base=(1 << 20) + (1 << 28), segments=1, segment_bytes=4096, unit_tokens=1), **change}.items():
        setattr(a[0], k, v)
    return a


TABLE, OUT, REFS, ROWS, ROWS2, WS, WORD = (at(i << 24) for i in range(7))
FORK = dict(table=TABLE, out=OUT, refs=REFS, parents=ROWS, old=4, new=4, groups=1, max_pages=8, pages=32, err=at(-64),
            flags=0, stream=None)
RESERVE = dict(table=TABLE, refs=REFS, before=ROWS, after=ROWS2, lacking=WORD, pools=pool(), n=1, rows=4, page=16,
               max_pages=8, pages=32, ws=WS, bytes=1 << 20, err=at(-64), flags=0, stream=None)
RELEASE = dict(table=TABLE, refs=REFS, keep=ROWS, rows=4, page=16, max_pages=8, pages=32, err=at(-64), flags=0,
               stream=None)
COMPACT = dict(table=TABLE, out=OUT, refs=REFS, out_refs=ROWS, used=WORD, pools=pool(), n=1, rows=4, page=16,
               max_pages=8, pages=32, ws=WS, bytes=1 << 20, err=at(-64), flags=0, stream=None)
COPY = dict(pools=pool(), n=1, src=ROWS, dst=ROWS2, rows=None, count=None, most=4, page=16, pages=32, err=at(-64),
            flags=0, stream=None)
POOL_FAULTS = [
    (EINVAL, dict(pools=None)), (EINVAL, dict(n=-1)), (EINVAL, dict(pools=pool(base=0))),
    (EINVAL, dict(pools=pool(segments=0))), (EINVAL, dict(pools=pool(segment_bytes=0))),
    (EINVAL, dict(pools=pool(unit_tokens=0))), (ESHAPE, dict(pools=pool(unit_tokens=3))),
    (ESHAPE, dict(pools=pool(segment_bytes=4100))), (EALIGN, dict(pools=pool(segment_bytes=32))),
    (ESHAPE, dict(pools=pool(segments=1 << 20))), (EALIGN, dict(pools=pool(base=(1 << 28) + 2))),
]
CASES = [
    ("anvilq_pages_fork", FORK, [
        *((EINVAL, {k: None}) for k in ("table", "out", "refs", "parents", "err")), (EINVAL, dict(flags=2)),
        (EINVAL, dict(groups=0)), (EINVAL, dict(groups=3)), (EINVAL, dict(out=TABLE)), (EINVAL, dict(out=at(124))),
        (EINVAL, dict(out=at((2 << 24) - 4))), (EINVAL, dict(refs=at(4))), (EINVAL, dict(parents=REFS)),
        (EINVAL, dict(parents=OUT)), (ESHAPE, dict(old=0)), (ESHAPE, dict(new=16385)), (ESHAPE, dict(max_pages=0)),
        (ESHAPE, dict(pages=0)), (ESHAPE, dict(max_pages=1 << 29)), (EALIGN, dict(refs=at((2 << 24) + 2)))]),
    ("anvilq_pages_reserve", RESERVE, [
        *((EINVAL, {k: None}) for k in ("table", "refs", "before", "after", "lacking", "err")), (EINVAL, dict(flags=4)),
        (EWORKSPACE, dict(ws=None)), (EWORKSPACE, dict(bytes=66047)), (ESHAPE, dict(rows=0)), (ESHAPE, dict(page=0)),
        (ESHAPE, dict(page=1 << 28)), (ESHAPE, dict(rows=16385)), (EINVAL, dict(refs=at(64))),
        (EINVAL, dict(before=at(124))), (EINVAL, dict(before=at((5 << 24) + 100))), (EINVAL, dict(lacking=REFS)),
        (EINVAL, dict(after=at((2 << 24) + 124))), (EALIGN, dict(ws=at((5 << 24) + 8))),
        (EINVAL, dict(pools=pool(base=(1 << 20) + (2 << 24) - 4096 * 31))),        # the counts inside a pool
        *POOL_FAULTS]),
    ("anvilq_pages_release", RELEASE, [
        *((EINVAL, {k: None}) for k in ("table", "refs", "keep", "err")), (EINVAL, dict(flags=8)),
        (EINVAL, dict(refs=at(100))), (EINVAL, dict(keep=at(100))), (EINVAL, dict(keep=REFS)), (ESHAPE, dict(rows=0)),
        (ESHAPE, dict(page=0)), (EALIGN, dict(keep=at(1)))]),
    ("anvilq_pages_compact", COMPACT, [
        *((EINVAL, {k: None}) for k in ("table", "out", "refs", "out_refs", "used", "err")), (EINVAL, dict(flags=2)),
        (EINVAL, dict(out=at(64))), (EINVAL, dict(out_refs=at((2 << 24) + 64))), (EINVAL, dict(out_refs=TABLE)),
        (EINVAL, dict(used=REFS)), (EWORKSPACE, dict(ws=None)), (EWORKSPACE, dict(bytes=65536)), (ESHAPE, dict(rows=0)),
        (EINVAL, dict(pools=pool(base=(1 << 20) + (1 << 24)))), *POOL_FAULTS]),
    ("anvilq_pages_copy", COPY, [
        *((EINVAL, {k: None}) for k in ("src", "dst", "err")), (EINVAL, dict(most=-1)), (EINVAL, dict(flags=2)),
        (ESHAPE, dict(pages=0)), (ESHAPE, dict(page=0)), (EALIGN, dict(src=at(2))),
        (EINVAL, dict(src=ctypes.c_void_p((1 << 20) + (1 << 28) + 64))), *POOL_FAULTS]),
]


@pytest.mark.parametrize("name,base,status,change", [(n, b, s, c) for n, b, cs in CASES for s, c in cs],
                         ids=lambda v: v if isinstance(v, str) else None)
def test_refused_before_launch(name, base, status, change):
    assert set(change) <= set(base)
    assert getattr(_lib.load(), name)(*{**base, **change}.values()) == status


def test_no_pages_is_no_work():
    assert _lib.load().anvilq_pages_copy(*{**COPY, "most": 0}.values()) == 0
    assert _lib.load().anvilq_pages_reserve_workspace_size(0, 5) == 0
    assert _lib.load().anvilq_pages_reserve_workspace_size(16385, 5) == 0
    assert _lib.load().anvilq_pages_compact_workspace_size(0) == 0


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda: ops.pages_fork(ints(4, 3), ints(9), ints(4)),                           # CPU tensors
    lambda: ops.pages_fork(ints(4, 3).long(), ints(9), ints(4)),
    lambda: ops.pages_fork(ints(4, 3), ints(9, 1), ints(4)),
    lambda: ops.pages_fork(ints(3, 4).t(), ints(9), ints(4)),
    lambda: ops.pages_reserve(ints(4, 3), ints(9), ints(3), ints(4), 16, []),
    lambda: ops.pages_release(ints(4, 3), ints(9), ints(4).long(), 16),
    lambda: ops.pages_compact(ints(4, 3), ints(9), []),
    lambda: ops.pages_copy([], ints(4), ints(4), 16),
    lambda: ops.PagePools([torch.zeros(4, 16, 2, 64, dtype=torch.float16)], 16),
])
def test_front_end(call):
    with pytest.raises(ValueError):
        call()


def test_too_few_pages_has_a_text(monkeypatch):
    word = torch.tensor([512], dtype=torch.int32)
    monkeypatch.setattr(ops, "device_error_word", lambda device: word)
    with pytest.raises(AnvilqError, match="free pages"):
        ops.raise_device_errors("cpu")


def test_more_copies_than_a_launch_numbers():
    assert _lib.load().anvilq_pages_copy(*{**COPY, "n": 128, "most": 1 << 25}.values()) == ESHAPE
