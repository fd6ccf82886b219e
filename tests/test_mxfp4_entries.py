"""MXFP4 buffers as a layer is given them (no GPU): entries that contradict themselves, tensors that start off their place."""

import pytest
import torch

from mirai_b200 import experts as ex
from mirai_b200 import ops


def entry(E, H, I, shape_of):
    names, tensors, shapes = {}, {}, {}
    for key, (o, i) in {"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items():
        names[f"{key}_mxfp4"], names[f"{key}_mxfp4_scale"] = f"ffn.{key}", f"ffn.{key}.scale"
        tensors[f"ffn.{key}"] = torch.zeros(E, o, i // 2, dtype=torch.uint8)
        tensors[f"ffn.{key}.scale"] = torch.full((E, o, i // 32), 127, dtype=torch.uint8)
        shapes[key] = shape_of(key, [E, o, i])
    return {"kind": "grouped_experts", "quant_format": "mxfp4", "num_experts": E, "tensors": names, "shapes": shapes}, tensors


@pytest.mark.parametrize("wrong", [lambda s: [s[0], s[1], s[2] + 32], lambda s: [s[0], s[2], s[1]], lambda s: s[1:],
                                   lambda s: [s[0], s[1], s[2] + 1]])
@pytest.mark.parametrize("at", ["w1", "w2"])
def test_a_packed_entry_whose_shapes_are_not_its_codes(wrong, at):
    good = ex.B200GroupedExperts.from_packed_state(*entry(2, 64, 96, lambda k, s: s))
    assert good.is_fully_loaded()
    with pytest.raises(ValueError, match=f"{at}_mxfp4: codes of shape"):
        ex.B200GroupedExperts.from_packed_state(*entry(2, 64, 96, lambda k, s: wrong(s) if k == at else s))


def test_buffers_that_start_off_alignment_are_installed_aligned():
    """Views into a file's bytes can start anywhere. What the kernels read has to be the module's buffer itself, so that a state
    loaded into it later is seen."""
    E, o, i = 2, 96, 64
    codes = torch.arange(E * o * i // 2 + 5, dtype=torch.int32).to(torch.uint8)[5:].view(E, o, i // 2)
    tiles = torch.arange(E * 512 + 3, dtype=torch.int32).to(torch.uint8)[3:].view(E, 1, 1, 512)
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    m.load_mxfp4_weight("w1", packed=codes, scale=tiles)
    for buf, given in ((m.w1_mxfp4, codes), (m.w1_mxfp4_scale, tiles)):
        assert given.data_ptr() % 32 and buf.data_ptr() % 32 == 0 and torch.equal(buf, given)
    aligned = codes.clone()
    m.load_mxfp4_weight("w3", packed=aligned, scale=tiles.clone())
    assert m.w3_mxfp4.data_ptr() == aligned.data_ptr()  # used in place


def test_which_rows_are_quantised_inside_the_product():
    """Up to 256 rows or 16 a segment for gate/up, 1024 at most; down up to 256 rows on up to 64 segments that can have rows."""
    def of(rows, segments, width=2048):
        x = torch.empty(rows, width, dtype=torch.bfloat16, device="meta")
        return ops._few_rows(x, width, segments), ops._few_rows_down(x, width, segments)

    assert of(1, 1) == of(256, 8) == of(256, 64) == of(64, 128) == (True, True)
    assert of(257, 8) == of(1025, 1024) == of(16, 8, 4128) == (False, False)
    assert of(512, 32) == of(65, 128) == of(200, 128) == of(1024, 64) == (True, False)
