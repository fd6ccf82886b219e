"""Host side of MXFP4 experts and group-limited routing (no GPU): argument checks of
the C entry points and of the Python layer, the scale layout, and ingest rules."""

import ctypes

import pytest
import torch

from mirai_b200 import _lib, block, ops
from mirai_b200 import experts as ex

ALIGNED, OFF16, OFF8 = 4096, 4096 + 16, 4096 + 8  # addresses for checks that end before any launch


@pytest.fixture(scope="module")
def lib():
    from mirai_b200.build import build
    build()
    return _lib.load()


def refused(lib, code, text, name, *args):
    assert getattr(lib, name)(*args) == code
    assert text in lib.mirai_b200_last_error()


# ----------------------------------------------------------------------------- scale layout

def test_scale_tiles_hold_each_byte_at_its_place():
    E, out, inp = 2, 150, 416
    rows = torch.randint(0, 255, (E, out, inp // 32), dtype=torch.uint8, generator=torch.Generator().manual_seed(0))
    tiles = ops.mxfp4_scale_tiles(rows)
    assert tiles.shape == (E, 2, 4, 512)
    flat = tiles.reshape(E, -1)
    for e, r, b in ((0, 0, 0), (0, 31, 3), (1, 32, 4), (1, 127, 12), (0, 128, 5), (1, 149, 7)):
        at = (r // 128 * 4 + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4
        assert flat[e, at] == rows[e, r, b]
    assert int(tiles.long().sum()) == int(rows.long().sum())  # zero bytes past the matrix
    assert torch.equal(ops.mxfp4_scale_rows(tiles, out, inp), rows)
    with pytest.raises(ValueError, match="uint8"):
        ops.mxfp4_scale_tiles(rows.int())


def test_scale_sizes(lib):
    assert lib.mirai_mxfp4_scale_bytes(2, 150, 416) == 2 * 2 * 4 * 512
    assert lib.mirai_mxfp4_scale_bytes(0, 150, 416) == 0
    for rows, segs, width in ((1, 1, 32), (300, 8, 2048), (5, 64, 160), (0, 4, 64)):
        assert lib.mirai_mxfp4_rows_scale_bytes(rows, segs, width) == ops.Mxfp4Rows.scale_bytes(rows, width, segs)
        # no split of the rows over the segments can need more
        worst = sum(-(-n // 128) for n in ([rows - min(rows, segs) + 1] + [1] * (min(rows, segs) - 1) if rows else []))
        assert ops.Mxfp4Rows.scale_bytes(rows, width, segs) >= worst * -(-width // 128) * 512


# ----------------------------------------------------------------------------- C entry points

def test_quantiser_refusals(lib):
    q = "mirai_mxfp4_quantize"
    refused(lib, 1, b"bad sizes", q, ALIGNED, 0, 0, 8, 32, ALIGNED, ALIGNED, None)
    refused(lib, 2, b"% 32", q, ALIGNED, 0, 1, 8, 48, ALIGNED, ALIGNED, None)
    refused(lib, 1, b"misaligned", q, OFF16, 0, 1, 8, 32, ALIGNED, ALIGNED, None)
    refused(lib, 1, b"misaligned", q, ALIGNED, 0, 1, 8, 32, OFF8, ALIGNED, None)
    refused(lib, 1, b"null", q, None, 0, 1, 8, 32, ALIGNED, ALIGNED, None)
    refused(lib, 1, b"unknown dtype", q, ALIGNED, 2, 1, 8, 32, ALIGNED, ALIGNED, None)
    refused(lib, 2, b"too many rows", q, ALIGNED, 0, 1 << 30, 1 << 20, 32, ALIGNED, ALIGNED, None)
    refused(lib, 2, b"2^24", q, ALIGNED, 0, 1, 8, 1 << 25, ALIGNED, ALIGNED, None)
    d = "mirai_mxfp4_dequantize"
    refused(lib, 1, b"misaligned", d, ALIGNED, ALIGNED, 1, 8, 32, OFF16, 0, None)
    refused(lib, 1, b"unknown dtype", d, ALIGNED, ALIGNED, 1, 8, 32, ALIGNED, 7, None)
    r = "mirai_mxfp4_quantize_rows"
    refused(lib, 1, b"segments", r, ALIGNED, 8, None, ALIGNED, 1025, 8, 32, ALIGNED, ALIGNED, None)
    refused(lib, 1, b"segments", r, ALIGNED, 8, None, ALIGNED, 0, 8, 32, ALIGNED, ALIGNED, None)
    refused(lib, 2, b"multiple of 32", r, ALIGNED, 8, None, ALIGNED, 1, 8, 40, ALIGNED, ALIGNED, None)
    refused(lib, 1, b"input rows", r, ALIGNED, 7, None, ALIGNED, 1, 8, 32, ALIGNED, ALIGNED, None)
    refused(lib, 2, b"2^31", r, ALIGNED, 1 << 32, None, ALIGNED, 1, 1 << 32, 32, ALIGNED, ALIGNED, None)
    assert lib.mirai_mxfp4_quantize_rows(None, 0, None, None, 1, 0, 32, None, None, None) == 0  # no rows


def test_product_refusals(lib):
    w = _lib.Mxfp4Weight(ALIGNED, ALIGNED)
    null = _lib.Mxfp4Weight(None, ALIGNED)
    g = "mirai_moe_gateup_swiglu_mxfp4"
    ok = [ALIGNED, ALIGNED, ALIGNED, 1, 4, 16, 64, 96, w, w, ALIGNED, None, None, None, None]

    def change(base, **at):
        args = list(base)
        for i, v in at.items():
            args[int(i[1:])] = v
        return args

    refused(lib, 1, b"segments", g, *change(ok, _3=300))
    refused(lib, 1, b"segments", g, *change(ok, _4=0))
    refused(lib, 2, b"% 32", g, *change(ok, _6=72))
    refused(lib, 2, b"% 32", g, *change(ok, _7=100))
    refused(lib, 1, b"bad sizes", g, *change(ok, _5=-1))
    refused(lib, 2, b"2^31", g, *change(ok, _5=1 << 31))
    refused(lib, 1, b"null operand", g, *change(ok, _0=None))
    refused(lib, 1, b"null operand", g, *change(ok, _8=null))
    refused(lib, 1, b"null operand", g, *change(ok, _9=None))
    refused(lib, 1, b"null output", g, *change(ok, _10=None))
    refused(lib, 1, b"null output", g, *change(ok, _12=ALIGNED))  # h_packed without its scales
    refused(lib, 1, b"16-byte", g, *change(ok, _10=OFF8))
    assert lib.mirai_moe_gateup_swiglu_mxfp4(*change(ok, _5=0)) == 0
    d = "mirai_moe_down_mxfp4"
    okd = [ALIGNED, ALIGNED, ALIGNED, 1, 4, 16, 64, 96, w, None, None, ALIGNED, None]
    refused(lib, 1, b"rank-block", d, *change(okd, _9=ALIGNED))
    refused(lib, 1, b"null output", d, *change(okd, _11=None))
    f = "mirai_moe_down_mxfp4_few"
    okf = [ALIGNED, ALIGNED, 1, 4, 16, 64, 96, w, ALIGNED, None]
    refused(lib, 2, b"at most 1024 rows", f, *change(okf, _4=1025))
    refused(lib, 2, b"up to 4096", f, *change(okf, _5=4128))
    refused(lib, 1, b"32-byte", f, *change(okf, _0=OFF16))
    refused(lib, 1, b"null operand", f, *change(okf, _8=None))
    x = "mirai_moe_down_dx_f32_bf16"
    refused(lib, 1, b"rank-block", x, ALIGNED, ALIGNED, 1, 4, 16, 64, 64, ALIGNED, ALIGNED, ALIGNED, None, ALIGNED, None)


def test_a_product_too_wide_for_its_tiles_is_refused(lib):
    """1023 column tiles at most: of 128 channels in gate/up, of 256 outputs in down."""
    w = _lib.Mxfp4Weight(ALIGNED, ALIGNED)
    refused(lib, 2, b"column tiles", "mirai_moe_gateup_swiglu_mxfp4", ALIGNED, ALIGNED, ALIGNED, 1, 4, 16, 64,
            1023 * 128 + 32, w, w, ALIGNED, None, None, None, None)
    refused(lib, 2, b"column tiles", "mirai_moe_down_mxfp4", ALIGNED, ALIGNED, ALIGNED, 1, 4, 16, 64, 1023 * 256 + 32, w,
            None, None, ALIGNED, None)
    refused(lib, 2, b"row tiles", "mirai_moe_down_mxfp4", ALIGNED, ALIGNED, ALIGNED, 1, 1, (1 << 31) - 257, 64,
            1023 * 256, w, None, None, ALIGNED, None)  # 2^23 x 1023 tiles


def test_route_groups_refusals(lib):
    r = "mirai_route_groups"
    ok = [ALIGNED, 1, 8, 64, 4, 8, 3, 1, 1, None, 2, 1.0, ALIGNED, ALIGNED, None]

    def but(**at):
        args = list(ok)
        for i, v in at.items():
            args[int(i[1:])] = v
        return args

    refused(lib, 1, b"experts", r, *but(_3=1025))
    refused(lib, 1, b"k <=", r, *but(_4=17))
    refused(lib, 1, b"k <=", r, *but(_4=0))
    refused(lib, 1, b"groups", r, *but(_5=7))
    refused(lib, 1, b"groups", r, *but(_5=64))
    refused(lib, 1, b"groups", r, *but(_6=0))
    refused(lib, 1, b"groups", r, *but(_6=9))
    refused(lib, 1, b"k=9", r, *but(_4=9, _6=1))
    refused(lib, 1, b"score function", r, *but(_8=2))
    refused(lib, 1, b"normalisation", r, *but(_10=4))
    refused(lib, 1, b"fp32 or bf16", r, *but(_1=3))
    refused(lib, 1, b"null", r, *but(_0=None))
    assert lib.mirai_route_groups(*but(_2=0, _0=None)) == 0
    b = "mirai_route_groups_backward"
    refused(lib, 1, b"null", b, None, ALIGNED, 1, ALIGNED, 8, 64, 4, 1, 2, 1.0, ALIGNED, None)
    refused(lib, 1, b"k <=", b, ALIGNED, ALIGNED, 1, ALIGNED, 8, 64, 65, 1, 2, 1.0, ALIGNED, None)


# ----------------------------------------------------------------------------- Python layer

def test_cpu_tensors_are_refused():
    cpu = torch.zeros(2, 8, 32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.mxfp4_quantize(cpu)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.Mxfp4Tensor(torch.zeros(2, 8, 16, dtype=torch.uint8), torch.zeros(2, 1, 1, 512, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.mxfp4_quantize_rows(torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.route_groups(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="score_func"):
        ops.route_groups(torch.zeros(4, 8), 2, score_func="relu")
    with pytest.raises(ValueError, match="norm"):
        ops.route_groups(torch.zeros(4, 8), 2, norm="max")
    with pytest.raises(ValueError, match="group_score"):
        ops.route_groups(torch.zeros(4, 8), 2, group_score="mean")
    with pytest.raises(TypeError, match="Mxfp4Tensor"):
        ops.mxfp4_dequantize(cpu)


def test_storage_table_checks_mxfp4_buffers():
    E, out, inp = 3, 96, 160
    good = {"mxfp4": torch.zeros(E, out, inp // 2, dtype=torch.uint8),
            "mxfp4_scale": torch.zeros(E, 1, 2, 512, dtype=torch.uint8)}
    assert ex.storage_problems("mxfp4", "w1", E, (E, out, inp), None, good) == []
    bad = dict(good, mxfp4=good["mxfp4"].int())
    assert any("dtype" in p for p in ex.storage_problems("mxfp4", "w1", E, (E, out, inp), None, bad))
    bad = dict(good, mxfp4_scale=torch.zeros(E, 1, 1, 512, dtype=torch.uint8))
    assert any("entries per expert" in p for p in ex.storage_problems("mxfp4", "w1", E, (E, out, inp), None, bad))
    assert any("whole blocks" in p for p in ex.storage_problems("mxfp4", "w1", E, (E, out, 80), None, good))


def test_expert_module_refuses_what_does_not_fit():
    m = ex.B200GroupedExperts.from_empty(num_experts=2, quant_format="mxfp4")
    packed = torch.zeros(2, 96, 32, dtype=torch.uint8)
    with pytest.raises(ValueError, match="rows of shape"):
        m.load_mxfp4_weight("w1", packed=packed, scale=torch.zeros(2, 96, 3, dtype=torch.uint8))
    with pytest.raises(ValueError, match="rejected"):
        m.load_mxfp4_weight("w1", packed=packed, scale=torch.zeros(2, 1, 2, 512, dtype=torch.uint8))
    with pytest.raises(ValueError, match="rejected"):
        m.load_mxfp4_weight("w1", packed=packed[:1], scale=torch.zeros(1, 96, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="weight key"):
        m.load_mxfp4_weight("w4", packed=packed, scale=torch.zeros(2, 96, 2, dtype=torch.uint8))
    m.load_mxfp4_weight("w1", packed=packed, scale=torch.zeros(2, 96, 2, dtype=torch.uint8))  # a checkpoint's rows
    assert m.w1_mxfp4_scale.shape == (2, 1, 1, 512) and m._shape_of("w1") == (2, 96, 64)
    other = ex.B200GroupedExperts.from_empty(num_experts=2, quant_format="int8")
    with pytest.raises(ValueError, match="offered to int8"):
        other.load_mxfp4_weight("w1", packed=packed, scale=torch.zeros(2, 96, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ex.GroupedExpertWeights.from_module(m)
    lacking = ex.B200GroupedExperts.from_empty(num_experts=2, quant_format="mxfp4")
    with pytest.raises(_lib.MiraiError, match="do not fit"):
        ex.GroupedExpertWeights.from_module(lacking)  # no key is loaded
    with pytest.raises(ValueError, match="quant_format"):
        ex.B200GroupedExperts.from_empty(num_experts=2, quant_format="fp8")


def test_packed_state_entry_restores_mxfp4_keys():
    E, H, I = 2, 64, 96
    g = torch.Generator().manual_seed(0)
    tensors, names, shapes = {}, {}, {}
    for key, (o, i) in {"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items():
        names[f"{key}_mxfp4"], names[f"{key}_mxfp4_scale"] = f"ffn.{key}", f"ffn.{key}.scale"
        tensors[f"ffn.{key}"] = torch.randint(0, 256, (E, o, i // 2), dtype=torch.uint8, generator=g)
        tensors[f"ffn.{key}.scale"] = torch.randint(100, 130, (E, o, i // 32), dtype=torch.uint8, generator=g)
        shapes[key] = [E, o, i]
    spec = {"kind": "grouped_experts", "quant_format": "mxfp4", "num_experts": E, "tensors": names, "shapes": shapes}
    m = ex.B200GroupedExperts.from_packed_state(spec, tensors)
    assert m.is_fully_loaded() and torch.equal(m.w2_mxfp4, tensors["ffn.w2"])
    assert torch.equal(ops.mxfp4_scale_rows(m.w1_mxfp4_scale, I, H), tensors["ffn.w1.scale"])
    del tensors["ffn.w3.scale"]
    with pytest.raises(KeyError, match="w3_mxfp4_scale"):
        ex.B200GroupedExperts.from_packed_state(spec, tensors)


def test_block_checks_its_groups():
    def make(**kw):
        return block.B200SparseMoeBlock(hidden_size=64, num_experts=8, top_k=2, experts=torch.nn.Identity(), **kw)

    assert make().num_groups == 1
    assert make(num_groups=4, top_groups=2).top_groups == 2
    for kw in ({"num_groups": 3}, {"num_groups": 4, "top_groups": 5}, {"num_groups": 4, "top_groups": 0},
               {"num_groups": 4, "group_score": "sum"}):
        with pytest.raises(ValueError, match="group"):
            make(**kw)


def test_header_names_every_argument_of_the_bindings():
    """Each new binding has as many arguments as its declaration."""
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "mirai_b200.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    for name, (_, args) in _lib.SIGNATURES.items():
        if "mxfp4" in name or "route_groups" in name or name == "mirai_moe_down_dx_f32_bf16":
            decl = re.search(rf"\b{name}\s*\((.*?)\);", text, flags=re.S).group(1)
            assert len(decl.split(",")) == len(args), name
            for a, t in zip(decl.split(","), args):
                if "int32_t " in a and "*" not in a:
                    assert t is ctypes.c_int32, (name, a)
                elif "int64_t " in a and "*" not in a:
                    assert t is ctypes.c_int64, (name, a)
                elif "float " in a and "*" not in a:
                    assert t is ctypes.c_float, (name, a)
