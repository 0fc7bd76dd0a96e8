"""Arguments that the paged-cache serving operators refuse, on the host, before any launch."""
import ctypes

import pytest
import torch

from anvilq_b200 import _lib, ops

EINVAL, EALIGN, EWORKSPACE, ESHAPE = -1, -2, -4, -5
FAKE = ctypes.c_void_p(1 << 20)   # never dereferenced: every call here is rejected
ODD = ctypes.c_void_p((1 << 20) + 8)


def at(byte):
    return ctypes.c_void_p((1 << 20) + byte)


QKV, OUT, OUT2 = FAKE, at(1 << 24), at(1 << 25)

APPEND = dict(qkv=QKV, stride=1536, starts=FAKE, lens=FAKE, table=FAKE, q=OUT, k=FAKE, v=FAKE, T=4, B=2, Hq=8,
              Hkv=2, D=128, page=16, max_pages=4, pages=8, theta=1e6, err=FAKE, flags=0, stream=None)
APPEND_Q8 = dict(qkv=QKV, stride=1536, starts=FAKE, lens=FAKE, table=FAKE, q=OUT, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE,
                 code=0, T=4, B=2, Hq=8, Hkv=2, D=128, page=16, max_pages=4, pages=8, theta=1e6, err=FAKE, flags=0,
                 stream=None)
VALUES = dict(k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, code=0, ko=OUT, vo=OUT2, pages=4, Hkv=2, page=16, D=128, flags=0,
              stream=None)
ATTN = dict(q=FAKE, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, code=0, table=FAKE, lens=FAKE, out=FAKE, B=2, Q=1, Hq=8, Hkv=2,
            D=128, page=16, max_pages=4, pages=8, scale=0.0, ws=FAKE, bytes=1 << 30, err=FAKE, flags=0, stream=None)
LOGITS = dict(x=FAKE, half=0, stride=1000, out=FAKE, out_stride=1000, token=FAKE, B=2, V=1000, history=FAKE,
              hist_stride=10, hist_lens=FAKE, prompts=None, L=10, rep=FAKE, pres=FAKE, freq=FAKE, bias_starts=FAKE,
              bias_ids=FAKE, bias=FAKE, bias_total=5, allowed=FAKE, allowed_stride=32, allowed_rows=None, masks=2,
              ws=FAKE, bytes=65536, err=FAKE, flags=0, stream=None)

CASES = [
    ("anvilq_paged_kv_append", APPEND, EINVAL, [dict(qkv=None), dict(starts=None), dict(lens=None), dict(table=None),
     dict(q=None), dict(k=None), dict(v=None), dict(err=None), dict(T=-1), dict(B=0), dict(Hq=0), dict(Hq=9),
     dict(theta=0.0), dict(theta=float("nan")), dict(theta=float("inf")), dict(flags=2), dict(stride=1528),
     # q's rows among those that are still to be read
     dict(q=QKV), dict(q=at(6144)), dict(q=at(-8192 + 16)), dict(q=at(4 * 3088 - 32), stride=1544)]),
    ("anvilq_paged_kv_append", APPEND, ESHAPE, [dict(D=96), dict(page=8), dict(page=24), dict(page=0),
     dict(max_pages=0), dict(pages=0), dict(page=1 << 20, max_pages=1 << 20)]),
    ("anvilq_paged_kv_append", APPEND, EALIGN, [dict(qkv=ODD), dict(q=ODD), dict(k=ODD), dict(v=ODD),
     dict(stride=1540)]),
    ("anvilq_paged_kv_append_q8", APPEND_Q8, EINVAL, [dict(ks=None), dict(vs=None), dict(code=2), dict(code=-1),
     dict(k=None), dict(err=None), dict(flags=4), dict(T=-5)]),
    ("anvilq_paged_kv_append_q8", APPEND_Q8, ESHAPE, [dict(D=256), dict(page=20)]),
    ("anvilq_paged_kv_append_q8", APPEND_Q8, EALIGN, [dict(k=ODD), dict(v=ODD)]),
    ("anvilq_kv_q8_values", VALUES, EINVAL, [dict(k=None), dict(ks=None), dict(ko=None), dict(code=7), dict(pages=0),
     dict(Hkv=0), dict(flags=2), dict(ko=FAKE), dict(vo=FAKE), dict(ko=OUT2), dict(vo=at(16368)),
     dict(ko=at(-32752))]),
    ("anvilq_kv_q8_values", VALUES, ESHAPE, [dict(D=32), dict(page=17)]),
    ("anvilq_kv_q8_values", VALUES, EALIGN, [dict(ko=ODD), dict(v=ODD)]),
    ("anvilq_gqa_decode_q8", ATTN, EINVAL, [dict(q=None), dict(k=None), dict(vs=None), dict(table=None),
     dict(lens=None), dict(out=None), dict(err=None), dict(code=3), dict(flags=8),
     dict(scale=float("inf")), dict(scale=float("nan"))]),
    ("anvilq_gqa_decode_q8", ATTN, ESHAPE, [dict(B=0), dict(Q=0), dict(Q=65), dict(Hq=9), dict(Hkv=0), dict(D=80),
     dict(page=8), dict(pages=0), dict(max_pages=0), dict(page=1 << 20, max_pages=2000),
     dict(pages=1 << 26), dict(pages=2**31 - 1, page=2**31 - 16, max_pages=1),
     dict(B=65535, Hq=1024, Hkv=1024, max_pages=1 << 20)]),
    ("anvilq_gqa_decode_q8", ATTN, EALIGN, [dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(out=ODD), dict(ws=ODD)]),
    ("anvilq_logits_process", LOGITS, EINVAL, [dict(x=None), dict(out=None, token=None), dict(err=None), dict(B=0),
     dict(V=0), dict(half=2), dict(stride=999), dict(out_stride=999), dict(hist_lens=None), dict(L=-1),
     dict(hist_stride=9), dict(history=None), dict(bias_total=-1), dict(bias_ids=None), dict(bias=None),
     dict(masks=0), dict(masks=1), dict(allowed_stride=31), dict(flags=2),
     # results over logits that are still to be read
     dict(out=at(4000)), dict(out=at(-4)), dict(half=1),
     dict(out_stride=1001), dict(stride=2000, out_stride=2000, out=at(3996)),
     dict(stride=2000, out_stride=2000, out=at(-8000 + 4004))]),
    ("anvilq_logits_process", LOGITS, ESHAPE, [dict(B=4097, masks=4097), dict(V=(1 << 30) + 32, stride=1 << 40,
     out_stride=1 << 40, allowed_stride=1 << 30), dict(L=(1 << 30) + 1, hist_stride=1 << 31),
     dict(bias_total=(1 << 30) + 1)]),
    ("anvilq_logits_process", LOGITS, EWORKSPACE, [dict(ws=None), dict(bytes=65535)]),
    ("anvilq_logits_process", LOGITS, EALIGN, [dict(ws=ODD)]),
]


@pytest.mark.parametrize("name,base,status,change", [(n, b, s, c) for n, b, s, cs in CASES for c in cs],
                         ids=lambda v: v if isinstance(v, str) else None)
def test_refused_before_launch(name, base, status, change):
    assert set(change) <= set(base)
    assert getattr(_lib.load(), name)(*{**base, **change}.values()) == status


def test_workspace_sizes_of_unsupported_shapes():
    lib = _lib.load()
    assert lib.anvilq_gqa_decode_q8_workspace_size(1, 65, 8, 8, 128) == 0
    assert lib.anvilq_gqa_decode_q8_workspace_size(1, 1, 8, 3, 128) == 0
    assert lib.anvilq_logits_process_workspace_size(4097, 100) == 0
    assert lib.anvilq_logits_process_workspace_size(4096, 100) >= 65536


def test_no_tokens_is_no_work():
    assert _lib.load().anvilq_paged_kv_append(*{**APPEND, "T": 0}.values()) == 0


# ---- the Python front end: types, shapes, devices (CPU tensors never reach the library) ----

def _pools(dtype=torch.int8):
    codes = torch.zeros((4, 2, 16, 64), dtype=torch.int8).to(dtype)
    return codes, codes.clone(), torch.zeros((4, 2, 1)), torch.zeros((4, 2, 1))


def _table():
    return torch.zeros((2, 3), dtype=torch.int32), torch.ones(2, dtype=torch.int32)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 4, 64)), ValueError),                                     # fp32 q
    (dict(q=torch.zeros(2, 4, 128, dtype=torch.float16)), ValueError),               # head_dim
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), ValueError),                # batch
    (dict(k=torch.zeros((4, 2, 16, 64), dtype=torch.uint8)), TypeError),
    (dict(v=torch.zeros((4, 2, 16, 64)).to(torch.float8_e4m3fn)), TypeError),        # mixed codes
    (dict(ks=torch.zeros((4, 2, 2))), ValueError),
    (dict(vs=torch.zeros((4, 2, 1), dtype=torch.float16)), ValueError),
    (dict(table=torch.zeros((2, 3), dtype=torch.int64)), ValueError),
    (dict(lens=torch.ones(3, dtype=torch.int32)), ValueError),
    (dict(out=torch.zeros(2, 4, 64)), ValueError),
    (dict(), ValueError),                                                            # CPU tensors
])
def test_attention_front_end(change, error):
    k, v, ks, vs = _pools()
    table, lens = _table()
    a = dict(q=torch.zeros((2, 4, 64), dtype=torch.float16), k=k, v=v, ks=ks, vs=vs, table=table, lens=lens, out=None)
    a.update(change)
    with pytest.raises(error):
        ops.gqa_decode_q8(a["q"], a["k"], a["v"], a["ks"], a["vs"], a["table"], a["lens"], out=a["out"])


@pytest.mark.parametrize("change,error", [
    (dict(qkv=torch.zeros(5, 512)), ValueError),
    (dict(qkv=torch.zeros(5, 500, dtype=torch.float16)), ValueError),
    (dict(qkv=torch.zeros(512, 5, dtype=torch.float16).t()), ValueError),
    (dict(qkv=torch.zeros(512, dtype=torch.float16).expand(5, 512)), ValueError),    # overlapping rows
    (dict(starts=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(lens=torch.zeros((2, 1), dtype=torch.int32)), ValueError),
    (dict(table=torch.zeros(6, dtype=torch.int32)), ValueError),
    (dict(q_out=torch.zeros(5, 4, 64)), ValueError),
    (dict(), ValueError),
])
def test_append_front_end(change, error):
    table, lens = _table()
    a = dict(qkv=torch.zeros((5, 512), dtype=torch.float16), table=table, lens=lens,
             starts=torch.zeros(3, dtype=torch.int32), q_out=None)
    a.update(change)
    pool = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    with pytest.raises(error):
        ops.paged_kv_append(a["qkv"], pool, pool.clone(), a["table"], a["lens"], a["starts"], 4, q_out=a["q_out"])
    with pytest.raises(error):
        ops.paged_kv_append_q8(a["qkv"], *_pools(), a["table"], a["lens"], a["starts"], 4, q_out=a["q_out"])
    with pytest.raises(TypeError):
        ops.paged_kv_append(a["qkv"], pool.float(), pool.float(), a["table"], a["lens"], a["starts"], 4)


@pytest.mark.parametrize("change", [
    dict(logits=torch.zeros((2, 50), dtype=torch.float64)), dict(logits=torch.zeros(50)),
    dict(logits=torch.zeros((50, 2)).t()), dict(logits=torch.zeros(50).expand(2, 50)),
    dict(history_lens=None), dict(history=None), dict(history=torch.zeros((3, 4), dtype=torch.int32)),
    dict(repetition=torch.ones(3)), dict(presence=torch.ones(2, dtype=torch.float16)),
    dict(bias_starts=torch.zeros(2, dtype=torch.int32)), dict(bias_ids=None),
    dict(bias_starts=None), dict(bias_values=torch.zeros(2)), dict(allowed=torch.zeros((2, 1), dtype=torch.int32)),
    dict(allowed=torch.zeros((1, 2), dtype=torch.int32)), dict(out=torch.zeros((2, 49))),
    dict(write_logits=False, choose=False), dict(write_logits=False, out=torch.zeros((2, 50))), dict(),
])
def test_logits_front_end(change):
    a = dict(logits=torch.zeros((2, 50)), history=torch.zeros((2, 4), dtype=torch.int32),
             history_lens=torch.zeros(2, dtype=torch.int32), repetition=torch.ones(2),
             bias_starts=torch.zeros(3, dtype=torch.int32), bias_ids=torch.zeros(3, dtype=torch.int32),
             bias_values=torch.zeros(3), allowed=torch.zeros((2, 2), dtype=torch.int32))
    a.update(change)
    with pytest.raises(ValueError):
        ops.logits_process(**a)


@pytest.mark.parametrize("scale", [float("-inf"), 2.0 ** 64 * (1 + 2.0 ** -23), 1e35])
def test_attention_scale_refused(scale):
    """Scales that are not finite, and those whose product with an int8 block's scale is not."""
    assert _lib.load().anvilq_gqa_decode_q8(*{**ATTN, "scale": scale}.values()) == EINVAL


# 4 tokens, 12 heads of 128: 12288 bytes of qkv, 8192 of q; 8 pages x 16 x 2 x 128: 65536
# bytes of a binary16 pool, 32768 of codes, 64 of scales
APART = dict(APPEND, qkv=at(0), q=at(1 << 14), k=at(1 << 17), v=at(1 << 18))
APART_Q8 = dict(APPEND_Q8, qkv=at(0), q=at(1 << 14), k=at(1 << 17), v=at(1 << 18), ks=at(1 << 19), vs=at(1 << 20))


@pytest.mark.parametrize("name,base,change", [
    *(("anvilq_paged_kv_append", APART, c) for c in (
        dict(v=at(1 << 17)), dict(v=at((1 << 17) + 65536 - 16)), dict(v=at((1 << 17) - 65536 + 16)), dict(k=at(0)),
        dict(v=at(16)), dict(q=at((1 << 17) + 1024)), dict(k=at((1 << 14) + 8192 - 16)))),
    *(("anvilq_paged_kv_append_q8", APART_Q8, c) for c in (
        dict(v=at(1 << 17)), dict(v=at((1 << 17) + 32768 - 16)), dict(vs=at(1 << 19)), dict(vs=at((1 << 19) + 60)),
        dict(ks=at((1 << 17) + 64)), dict(vs=at((1 << 18) + 32764)), dict(ks=at(1 << 14)), dict(vs=at(12284)))),
], ids=lambda v: v if isinstance(v, str) else None)
def test_append_outputs_that_overlap_are_refused(name, base, change):
    assert getattr(_lib.load(), name)(*{**base, **change}.values()) == EINVAL


def test_append_pools_beyond_memory_are_refused():
    big = dict(pages=2**31 - 1, page=1 << 26, max_pages=1)
    assert _lib.load().anvilq_paged_kv_append(*{**APART, **big}.values()) == ESHAPE
    assert _lib.load().anvilq_paged_kv_append_q8(*{**APART_Q8, **big}.values()) == ESHAPE


# 2 queries of 8 heads of 128: 4096 bytes of q and of out
ATTN_APART = dict(ATTN, q=at(0), out=at(1 << 14), k=at(1 << 17), v=at(1 << 18), ks=at(1 << 19), vs=at(1 << 20),
                  ws=at(1 << 21))


@pytest.mark.parametrize("change", [
    dict(out=at(16)), dict(out=at(4080)), dict(out=at(-4080)), dict(out=at(1 << 17)), dict(out=at((1 << 18) + 32752)),
    dict(out=at((1 << 17) - 4080)), dict(out=at((1 << 19) + 48)), dict(out=at((1 << 20) - 16)), dict(out=at(1 << 22)),
])
def test_attention_output_over_inputs_refused(change):
    assert _lib.load().anvilq_gqa_decode_q8(*{**ATTN_APART, **change}.values()) == EINVAL
