"""MXFP4 keys at the expert owners of a parallel layer: what is refused before any exchange (no GPU), and the owners'
steps on source-major segments against each source by itself."""

import pytest
import torch

from mirai_b200 import expert_parallel as ep
from mirai_b200 import ops


def keys_of_shape(E, H, I):
    """Three MXFP4 keys without buffers: enough for what a call looks at before it launches anything."""
    keys = []
    for out, inp in ((I, H), (I, H), (H, I)):
        w = ops.Mxfp4Tensor.__new__(ops.Mxfp4Tensor)
        w.shape, w.device = (E, out, inp), torch.device("cpu")
        keys.append(w)
    return tuple(keys)


@pytest.mark.parametrize("H,I", [(96, 64), (64, 160)])
def test_training_widths_are_refused_before_any_exchange(H, I, monkeypatch):
    """Every rank refuses alike: none is left waiting for a peer that stopped at its owner's GEMMs, or in the backward."""
    def exchange(*a, **k):
        raise AssertionError("an exchange began")
    monkeypatch.setattr(ep.dist, "all_to_all_single", exchange)
    monkeypatch.setattr(ep.dist, "all_gather_into_tensor", exchange)
    E, T, k = 4, 6, 2
    shard = ep.ExpertShard(E, 2, 0)
    x, logits = torch.zeros(T, H, dtype=torch.bfloat16), torch.zeros(T, E)
    with pytest.raises(ValueError, match="steps of 64"):
        ep.ep_moe_forward(x, logits, keys_of_shape(2, H, I), shard=shard, top_k=k, inter=I, train=True)
    layer = ep.ExpertParallelMoE.__new__(ep.ExpertParallelMoE)
    layer.ops, layer.shard, layer.top_k, layer.inter, layer._gen = ep.CudaStepOps(), shard, k, I, 0
    with pytest.raises(ValueError, match="steps of 64"):
        layer.forward(x, logits, keys_of_shape(2, H, I), train=True)
    assert layer._gen == 0
    with pytest.raises(ValueError, match="steps of 64"):
        ep.CudaStepOps().experts_train(x, None, keys_of_shape(E, H, I), I)


def _owner_case(E, counts, H, I, seed=0):
    """(dev, keys, rows, gradient rows, per-source counts): rows source-major, counts [source][expert]."""
    from test_gpu_mxfp4 import _dev, rows, weight
    dev = _dev()
    keys = tuple(ops.mxfp4_quantize(weight(E, *shape, dev, i + 1)) for i, shape in enumerate(((I, H), (I, H), (H, I))))
    S = sum(map(sum, counts))
    g = torch.Generator().manual_seed(seed)
    return dev, keys, rows(S, H, dev), torch.randn(S, H, generator=g).bfloat16().to(dev)


def _ends(counts, dev):
    return torch.tensor(counts).flatten().cumsum(0).to(torch.int32).to(dev)


def _adapter(E, H, I, r, dev):
    from test_gpu_mxfp4 import weight
    return ops.DownLoRA(weight(E, r, I, dev, 8), weight(E, H, r, dev, 9), 2.0, compute_grads=True)


@pytest.mark.gpu
@pytest.mark.parametrize("adapter", [False, True])
@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("counts", [[[130, 0, 7], [5, 300, 0]], [[1, 2, 3], [0, 0, 1]]])
def test_owner_steps_equal_each_source_alone(counts, few, adapter, monkeypatch):
    """Two sources' rows in one call: outputs and dX are each source's own, bit for bit; factor gradients add up over
    the sources (fp32 sums in another order: 2^-20 of the sum of magnitudes, bounded by the rows' count times the largest)."""
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS", 1024 if few else -1)
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS_PER_SEGMENT", 0)
    E, H, I, r = 3, 128, 192, 8
    dev, keys, x, gy = _owner_case(E, counts, H, I)
    step = ep.CudaStepOps()
    lora = _adapter(E, H, I, r, dev) if adapter else None
    y, saved = step.experts_train(x, _ends(counts, dev), keys, I, sources=2, lora=lora)
    plain = None if adapter else step.experts(x, _ends(counts, dev), keys, I, sources=2)
    assert plain is None or torch.equal(plain, y)
    back = step.read_back(keys)
    dx = step.experts_backward(gy, _ends(counts, dev), keys, I, 2, saved, lora)
    grads = (lora.grad_a, lora.grad_b) if adapter else ()
    if adapter:
        lora.grad_a = lora.grad_b = None
    assert torch.equal(dx, step.experts_backward(gy, _ends(counts, dev), back, I, 2, saved, lora))
    if adapter:
        lora.grad_a = lora.grad_b = None
    at = 0
    for c in counts:
        n = sum(c)
        ys, ss = step.experts_train(x[at:at + n], _ends(c, dev), keys, I, lora=lora)
        ds = step.experts_backward(gy[at:at + n], _ends(c, dev), back, I, 1, ss, lora)
        assert torch.equal(y[at:at + n], ys) and torch.equal(dx[at:at + n], ds)
        at += n
    if adapter:  # (experts_backward adds up what it is called for)
        for got, want in zip(grads, (lora.grad_a, lora.grad_b)):
            assert (got - want).abs().max() <= 2.0 ** -20 * at * want.abs().max()
    # the regrouped form: the chunk's rows expert-major, one source
    order, inverse = ep.regroup_order(torch.tensor(counts, device=dev), at)
    ends = _ends([sum(c[e] for c in counts) for e in range(E)], dev)
    ye, inner = step.experts_train(x[order], ends, keys, I, lora=lora)
    assert torch.equal(ye[inverse], y)
    if adapter:
        lora.grad_a = lora.grad_b = None
    again = step.experts_backward(gy, _ends(counts, dev), back, I, 2, ("regrouped", order, inverse, ends, inner), lora)
    assert torch.equal(again, dx)
    ops.check_device()


@pytest.mark.gpu
@pytest.mark.parametrize("adapter", [False, True])
def test_one_rank_layer_in_mxfp4(adapter):
    """The parallel layer on one rank: its forward is the one-GPU layer's, its dX within the bf16 rows' roundings of it
    (gy, gate/up, dgate/dup, dx of a route and dx on one side, two of them on the other: 2^-8 sqrt(7) < 0.011 in
    the 2-norm)."""
    from test_gpu_mxfp4 import _dev, rows, weight
    dev = _dev()
    E, T, k, H, I, r = 4, 500, 2, 128, 192, 8
    keys = tuple(ops.mxfp4_quantize(weight(E, *shape, dev, i + 1)) for i, shape in enumerate(((I, H), (I, H), (H, I))))
    lora = _adapter(E, H, I, r, dev) if adapter else None
    g = torch.Generator().manual_seed(2)
    x, logits = rows(T, H, dev), torch.randn(T, E, generator=g).to(dev)
    grad = torch.randn(T, H, generator=g).bfloat16().to(dev)
    shard = ep.ExpertShard(E, 1, 0)
    out, state = ep.ep_moe_forward(x, logits, keys, shard=shard, top_k=k, inter=I, train=True, lora=lora)
    dx, dw = ep.ep_moe_backward(grad, state, keys, shard=shard, inter=I, lora=lora)
    factors = (lora.grad_a, lora.grad_b) if adapter else ()
    idx, tw = ops.route_topk(logits, k)
    want, st = ops.moe_forward_train(x, idx, tw, *keys, num_experts=E, inter=I, lora=lora)
    rx, rw = ops.moe_backward_dx(grad, st, *keys, inter=I, lora=lora)
    ops.check_device()
    assert torch.equal(out, want) and torch.equal(dw, rw)

    def rel(a, b):
        return float((a.float() - b.float()).norm() / b.float().norm())

    assert rel(dx, rx) < 0.011
    if adapter:
        assert rel(factors[0], lora.grad_a) < 0.011 and rel(factors[1], lora.grad_b) < 0.011


@pytest.mark.gpu
def test_keys_are_read_back_once_for_all_chunks(monkeypatch):
    from test_gpu_mxfp4 import _dev, rows, weight
    dev = _dev()
    E, H, I = 2, 64, 64
    keys = tuple(ops.mxfp4_quantize(weight(E, *shape, dev, i)) for i, shape in enumerate(((I, H), (I, H), (H, I))))
    calls = []
    real = ops.mxfp4_dequantize
    monkeypatch.setattr(ops, "mxfp4_dequantize", lambda w, *a, **k: calls.append(w) or real(w, *a, **k))
    step = ep.CudaStepOps()
    plan, offs = None, torch.tensor([3, 8], dtype=torch.int32, device=dev)
    chunks = []
    for c in range(3):
        y, saved = step.experts_train(rows(8, H, dev, c), offs, keys, I)
        idx = torch.tensor([[0]] * 3 + [[1]] * 5, device=dev)
        plan = ops.dispatch_plan(idx, E)
        chunks.append(dict(tw=torch.ones(8, 1, device=dev), plan=plan, y_back=y, sc=None, rc=None, offs=offs, saved=saved))
    state = ep.EPTrainState([(0, 8), (8, 16), (16, 24)], chunks, 1, H, torch.bfloat16)
    dx, _ = ep.ep_moe_backward(rows(24, H, dev, 9), state, keys, shard=ep.ExpertShard(E, 1, 0), inter=I)
    ops.check_device()
    assert torch.isfinite(dx.float()).all() and len(calls) == 3 and {id(w) for w in calls} == {id(w) for w in keys}
