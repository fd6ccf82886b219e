"""MXFP4 keys as they come: padding bytes of the scale tiles, entries of a packed state, operands of the wrong shape."""

import pytest
import torch

from test_gpu_mxfp4 import _dev, rows, segments, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("K,N", [(32, 96), (96, 64), (160, 288), (224, 32), (288, 160), (1056, 64), (64, 96), (2080, 64)])
def test_padding_scales_of_a_key_do_not_count(K, N, few, monkeypatch):
    """Bytes past a key's blocks and rows are never part of a product, whatever they hold (255 stands for NaN)."""
    dev = _dev()
    from mirai_b200 import ops
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS", 1024 if few else -1)
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS_PER_SEGMENT", 0)
    counts = [5, 0, 130]
    E = len(counts)
    x, off = rows(sum(counts), K, dev), segments(counts, dev)
    clean = [ops.mxfp4_quantize(weight(E, N, K, dev, i)) for i in (1, 2)]
    dirty = []
    for w in clean:
        inside = ops.mxfp4_scale_tiles(torch.ones(E, N, K // 32, dtype=torch.uint8, device=dev)) == 1
        dirty.append(ops.Mxfp4Tensor(w.packed, torch.where(inside, w.scale, torch.full_like(w.scale, 255))))
    assert K % 128 == 0 and N % 128 == 0 or not torch.equal(dirty[0].scale, clean[0].scale)
    for make in (lambda k: ops.gateup_swiglu(x, off, *k, inter=N), lambda k: ops.down(x, off, k[0], hidden=N)):
        got, want = make(dirty), make(clean)
        ops.check_device()
        assert torch.isfinite(got.float()).all() and torch.equal(got, want)
    assert torch.equal(ops.mxfp4_dequantize(dirty[0]), ops.mxfp4_dequantize(clean[0]))


def test_down_dx_refuses_an_adapter_that_does_not_fit():
    """The rank block's operands are read by the rows and channels of the call: others are refused before the product."""
    dev = _dev()
    from mirai_b200 import ops
    E, H, I, counts = 2, 64, 128, [5, 9]
    S, off = sum(counts), segments(counts, dev)
    w2 = ops.mxfp4_quantize(weight(E, H, I, dev))
    gy, lora = rows(S, H, dev), ops.DownLoRA(weight(E, 4, I, dev), weight(E, H, 4, dev), 1.0)
    low = torch.zeros(S, 64, dtype=torch.bfloat16, device=dev)
    for dtype in (torch.bfloat16, torch.float32):
        gu = torch.randn(S, 2 * I, device=dev).to(dtype)
        ops.down_dx(gy, off, w2, gu, inter=I, lora=lora, rank_a=low)
        for bad in (low[1:], low[:, :32], low.float(), low.repeat(1, 2)[:, ::2]):
            with pytest.raises(ValueError, match="rank_a must be"):
                ops.down_dx(gy, off, w2, gu, inter=I, lora=lora, rank_a=bad)
        other = ops.DownLoRA(weight(E, 4, I // 2, dev), weight(E, H, 4, dev), 1.0)
        with pytest.raises(ValueError, match="adapter's A"):
            ops.down_dx(gy, off, w2, gu, inter=I, lora=other, rank_a=low)
    ops.check_device()
