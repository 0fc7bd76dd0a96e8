"""A workspace of the chunk attention that overlaps its inputs is refused, on the host, before any launch."""
import pytest

from anvilq_b200 import _lib
from test_chunk import CHUNK, EINVAL, at


# the workspace ends in, lies in, or begins at the end of an input or the output
@pytest.mark.parametrize("ws,size", [
    (-4096, 4097), (0, 1 << 16), (8176, 1 << 16),                              # q: 8192 bytes
    ((1 << 20) - 65536, 65537), ((1 << 20) + 65520, 1 << 16),                  # the keys: 65536
    ((2 << 20) + 32768, 16), ((2 << 20) + 65520, 1 << 16),                     # the values
    ((3 << 20) - 16, 32), ((3 << 20) + 16, 1 << 16),                           # the table: 32
    (4 << 20, 1 << 16), (5 << 20, 16),                                         # lengths and starts
    ((6 << 20) + 8176, 1 << 16),                                               # the output
    (-65536, 1 << 30),                                                         # all of them
])
def test_refused_before_launch(ws, size):
    assert _lib.load().anvilq_gqa_chunk_paged(*{**CHUNK, "ws": at(ws), "bytes": size}.values()) == EINVAL
