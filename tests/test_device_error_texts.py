"""What ops.raise_device_errors says of each bit (host logic, on a CPU word)."""
import pytest
import torch

from anvilq_b200 import AnvilqError, ops


@pytest.mark.parametrize("bit,words", [
    (1, ["AWQ scale"]),
    (2, ["sequence", "history length", "bias range", "mask row"]),
    (4, ["wait expired"]),
    (8, ["token id"]),
    (16, ["nonfinite", "bias", "key or value"]),
    (32, ["page-table"]),
    (64, ["ancestor mask"]),
    (128, ["legacy cache block"]),
    (256, ["not 16-byte aligned"]),
])
def test_each_bit_has_a_text_that_names_its_causes(monkeypatch, bit, words):
    word = torch.tensor([bit], dtype=torch.int32)
    monkeypatch.setattr(ops, "device_error_word", lambda device: word)
    with pytest.raises(AnvilqError) as e:
        ops.raise_device_errors("cpu")
    assert all(w in str(e.value) for w in words), str(e.value)
    assert f"0x{bit:x}" in str(e.value) and not word.any()
    ops.raise_device_errors("cpu")          # cleared
