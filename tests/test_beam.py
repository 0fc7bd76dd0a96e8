"""Arguments that the beam search's calls refuse, on the host, before any launch."""
import ctypes

import pytest
import torch

from anvilq_b200 import _lib, ops

EINVAL, EALIGN, EWORKSPACE, ESHAPE = -1, -2, -4, -5


def at(byte):
    return ctypes.c_void_p((1 << 20) + byte)   # never dereferenced: every call here is rejected


SELECT = dict(logits=at(0), half=0, stride=1000, scores=at(1 << 20), lengths=at(2 << 20), alpha=1.0, finished=at(3 << 20),
              eos=at(4 << 20), eos_count=2, pad=0, tokens=at(5 << 20), parents=at(6 << 20), new_scores=at(7 << 20),
              new_lengths=at(8 << 20), new_finished=at(9 << 20), B=2, K=4, V=1000, N=8, ws=at(16 << 20), bytes=1 << 20,
              err=at(-64), flags=0, stream=None)


def state(**change):
    a = (_lib.BeamState * 2)()
    for i in range(2):
        a[i].input, a[i].output, a[i].row_bytes = (1 << 30) + (i << 20), (1 << 31) + (i << 20), 100
    for k, v in change.items():
        setattr(a[1], k, v)
    return a


REORDER = dict(states=state(), count=2, parents=at(0), B=2, K=4, N=8, err=at(-64), flags=0, stream=None)


@pytest.mark.parametrize("status,change", [
    *((EINVAL, {k: None}) for k in ("logits", "scores", "tokens", "parents", "new_scores", "new_finished", "err",
                                    "new_lengths", "lengths", "eos")),
    (EINVAL, dict(lengths=None, new_lengths=None)),                # a penalty without lengths
    *((EINVAL, dict(alpha=a)) for a in (float("nan"), float("inf"), 17.0, -16.5)),
    (EINVAL, dict(half=2)), (EINVAL, dict(eos_count=-1)), (EINVAL, dict(flags=2)), (EINVAL, dict(stride=999)),
    *((ESHAPE, c) for c in (dict(B=0), dict(B=4097), dict(K=0), dict(K=65), dict(N=0), dict(N=129), dict(V=0),
                            dict(B=4096, K=16), dict(eos_count=1025))),
    (ESHAPE, dict(V=(1 << 30) + 1, stride=1 << 31)),
    (EALIGN, dict(logits=at(2))), (EALIGN, dict(logits=at(1), half=1)), (EALIGN, dict(scores=at((1 << 20) + 2))),
    (EALIGN, dict(tokens=at((5 << 20) + 1))), (EALIGN, dict(ws=at((16 << 20) + 8))),
    (EWORKSPACE, dict(ws=None)), (EWORKSPACE, dict(bytes=65536)),
    (EINVAL, dict(tokens=at(0))), (EINVAL, dict(tokens=at(31996))), (EINVAL, dict(parents=at((5 << 20) + 60))),
    (EINVAL, dict(new_scores=at(1 << 20))), (EINVAL, dict(new_lengths=at(2 << 20))),
    (EINVAL, dict(new_finished=at(3 << 20))), (EINVAL, dict(new_finished=at((16 << 20) + 70000))),
    (EINVAL, dict(ws=at(16000))), (EINVAL, dict(scores=at((16 << 20) + 64))),
])
def test_select_refused(status, change):
    assert set(change) <= set(SELECT)
    assert _lib.load().anvilq_beam_select(*{**SELECT, **change}.values()) == status


@pytest.mark.parametrize("status,change", [
    *((EINVAL, {k: None}) for k in ("states", "parents", "err")), (EINVAL, dict(count=-1)), (EINVAL, dict(flags=4)),
    (ESHAPE, dict(B=0)), (ESHAPE, dict(K=0)), (ESHAPE, dict(N=0)), (ESHAPE, dict(B=1 << 20, K=32)),
    (EALIGN, dict(parents=at(2))), (EINVAL, dict(states=state(input=0))), (EINVAL, dict(states=state(output=0))),
    (EINVAL, dict(states=state(row_bytes=0))), (ESHAPE, dict(states=state(row_bytes=1 << 37))),
    (EINVAL, dict(states=state(output=(1 << 30) + 799))),          # over the other state's rows
    (EINVAL, dict(states=state(output=(1 << 30) + (1 << 20)))),    # over its own
    (EINVAL, dict(states=state(output=(1 << 31) + 1599))),         # over the other's results
    (EINVAL, dict(states=state(output=(1 << 20) + 63))),           # over the parents
])
def test_reorder_refused(status, change):
    assert _lib.load().anvilq_beam_reorder(*{**REORDER, **change}.values()) == status


def test_nothing_to_reorder():
    assert _lib.load().anvilq_beam_reorder(*{**REORDER, "count": 0}.values()) == 0
    for shape in ((0, 4, 10, 4), (2, 65, 10, 4), (2, 4, 0, 4), (2, 4, 10, 129), (4096, 64, 10, 4)):
        assert _lib.load().anvilq_beam_select_workspace_size(*shape) == 0


@pytest.mark.parametrize("change", [
    dict(), dict(logits=torch.zeros(2, 4, 50, dtype=torch.float64)), dict(logits=torch.zeros(2, 3, 50)),
    dict(logits=torch.zeros(7, 50)), dict(logits=torch.zeros(50).expand(2, 4, 50)),
    dict(logits=torch.zeros(2, 50, 4).transpose(1, 2)), dict(logits=torch.zeros(2, 5, 50)[:, :4]),
    dict(scores=torch.zeros(8)), dict(scores=torch.zeros(2, 4, dtype=torch.float64)), dict(N=129), dict(N=0),
    dict(lengths=torch.zeros(2, 4)), dict(finished=torch.zeros(2, 4, dtype=torch.uint8)),
    dict(eos_ids=torch.zeros(2, dtype=torch.int64)), dict(lengths=None),
])
def test_select_front_end(change):
    a = dict(logits=torch.zeros(2, 4, 50), scores=torch.zeros(2, 4), lengths=torch.zeros((2, 4), dtype=torch.int32),
             length_penalty=1.0, finished=torch.zeros((2, 4), dtype=torch.bool),
             eos_ids=torch.zeros(1, dtype=torch.int32))
    a.update(change)
    with pytest.raises(ValueError):
        ops.beam_select(**a)


@pytest.mark.parametrize("states,outs", [
    ([torch.zeros(2, 4, 3)], None), ([torch.zeros(8, 3)], None), ([torch.zeros(2, 4, 3), torch.zeros(2, 5)], None),
    ([torch.zeros(2, 4, 3)], []), ([torch.zeros(2, 3, 4).transpose(1, 2)], None), ([torch.zeros(2, 4, 0)], None),
    ([torch.zeros(2, 4, 3)], [torch.zeros(2, 4, 3)]), ([torch.zeros(2)], None),
])
def test_reorder_front_end(states, outs):
    with pytest.raises(ValueError):
        ops.beam_reorder(states, torch.zeros((2, 8), dtype=torch.int32), outs=outs)
