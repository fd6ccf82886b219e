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
