"""MXFP4 buffers as a layer is given them (no GPU): entries that contradict themselves, tensors that start off their place."""

import pytest
import torch

from mirai_b200 import _lib, ops
from mirai_b200 import experts as ex

ALIGNED = 4096  # an address for checks that end before any launch


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


def test_c_entries_refuse_types_and_addresses():
    """What the C entries see before any launch."""
    from mirai_b200.build import build
    build()
    lib = _lib.load()

    def refused(code, text, name, *args):
        assert getattr(lib, name)(*args) == code and text in lib.mirai_b200_last_error()

    A, w = ALIGNED, _lib.Mxfp4Weight(ALIGNED, ALIGNED)
    few, save = "mirai_moe_gateup_swiglu_mxfp4_few_save", "mirai_moe_gateup_swiglu_mxfp4_save"
    refused(1, b"bf16 or fp32", few, A, A, 1, 1, 8, 64, 64, w, w, A, A, 3, None)
    refused(1, b"aligned to its type", few, A, A, 1, 1, 8, 64, 64, w, w, A + 1, A, 0, None)
    refused(1, b"aligned to its type", few, A, A, 1, 1, 8, 64, 64, w, w, A, A + 2, 1, None)
    refused(1, b"aligned to its type", "mirai_moe_gateup_swiglu_mxfp4_few", A, A, 1, 1, 8, 64, 64, w, w, A, A + 1, None)
    refused(1, b"aligned to its type", "mirai_moe_down_mxfp4_few", A, A, 1, 1, 8, 64, 64, w, A + 1, None)
    refused(1, b"bf16 or fp32", save, A, A, A, 1, 1, 8, 64, 64, w, w, A, A, 3, None, None, None)
    refused(1, b"16-byte", save, A, A, A, 1, 1, 8, 64, 64, w, w, A, A + 8, 1, None, None, None)
    rows, dx = "mirai_moe_down_dx_rows_f32", "mirai_moe_gateup_dx_f32"
    refused(1, b"null rank-block", rows, A, A, A, 1, 1, 8, 64, 64, A, A, A, None, A, None)
    refused(1, b"segments", rows, A, A, A, 2, 513, 8, 64, 64, A, A, None, None, A, None)
    refused(1, b"saved gate/up", rows, A, None, A, 1, 1, 8, 64, 64, A, None, None, None, A, None)
    refused(2, b"% 64", rows, A, None, A, 1, 1, 8, 96, 64, A, A, None, None, A, None)
    refused(1, b"misaligned", dx, A, A, 1, 1, 8, 64, 64, A, A, A + 8, None)
    refused(2, b"% 64", dx, A, A, 1, 1, 8, 64, 96, A, A, A, None)
    refused(1, b"segments", dx, A, A, 0, 1, 8, 64, 64, A, A, A, None)
    refused(1, b"unknown out_dtype", "mirai_moe_combine_f32", A, A, None, 4, 2, 64, A, 2, None)
    refused(1, b"misaligned", "mirai_moe_combine_f32", A + 4, A, None, 4, 2, 64, A, 0, None)
    refused(1, b"hidden", "mirai_moe_combine_f32", A, A, None, 4, 17, 64, A, 0, None)
    back = "mirai_moe_combine_backward_rows"
    refused(1, b"null", back, A, A, A, A, 4, 2, 64, A, None, A, None)
    refused(1, b"misaligned", back, A + 2, A, A, A, 4, 2, 64, A, A, A, None)
    refused(1, b"hidden", back, A, A, A, A, 4, 2, 60, A, A, A, None)
    for name, args in ((rows, (None, None, None, 1, 1, 0, 64, 64, None, None, None, None, None, None)),
                       (dx, (None, None, 1, 1, 0, 64, 64, None, None, None, None)),
                       (back, (None, None, None, None, 0, 2, 64, None, None, None, None))):
        assert getattr(lib, name)(*args) == 0  # no rows
