"""The XLA FFI handlers of the norm, of routing by groups and of the int8 experts compare their
buffers' sizes before the C entry, which sees pointers only (their text is read: JAX and its
headers are absent here)."""
import re
from pathlib import Path

import pytest

FFI_CC = Path(__file__).resolve().parents[1] / "hanuman_amd" / "xla_ffi" / "hmoe_xla_ffi.cc"
IMPLS = ["RouterGrouped", "RouterGroupedFromLogits", "AddRmsNorm", "AddRmsNormBwd", "QuantizeRowsI8", "DequantizeRowsI8",
         "DequantizeRowsFp8", "PackI8GateUp", "PackI8Down", "GroupedGateUpI8", "GroupedGateUpI8Gather", "GroupedDownI8"]


def _body(impl):
    return re.search(r"static ffi::Error %sImpl\(.*?\n}\n" % impl, FFI_CC.read_text(), flags=re.S).group(0)


@pytest.mark.parametrize("impl", IMPLS)
def test_sizes_are_compared_first(impl):
    body = _body(impl)
    assert "return BadSizes(" in body and body.index("return BadSizes(") < body.index("return Status(")


def test_routing_by_groups_compares_every_buffer():
    text = FFI_CC.read_text()
    fits = re.search(r"static bool SelectionFits\(.*?\n}\n", text, flags=re.S).group(0)
    for check in ("Rows(top_idx) == Rows(logits)", "SameRows(top_idx, gates)", "bias.element_count()) == Cols(logits)"):
        assert check in fits
    body = _body("RouterGrouped")
    for check in ("Rows(w) != Cols(x)", "Rows(*logits) != Rows(x)", "Cols(*logits) != Cols(w)",
                  "!SelectionFits(*logits, bias, mode, *top_idx, *gates)"):
        assert check in body
    assert "!SelectionFits(logits, bias, mode, *top_idx, *gates)" in _body("RouterGroupedFromLogits")
