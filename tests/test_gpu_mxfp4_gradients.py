"""Where the MXFP4 layer's backward rounds: the pieces that keep its intermediates in fp32, each against 64 bits,
and the layer's dx as a whole."""

import pytest
import torch

from test_gpu_mxfp4 import _dev, layer64, product64, rows, segments, step, values64, weight

pytestmark = pytest.mark.gpu


def norm_error(a, ref):
    return float((a.detach().cpu().double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("T,E,k,H,I", [(300, 6, 2, 192, 320), (1000, 3, 3, 128, 192), (1500, 2, 1, 256, 128)])
def test_layer_dx_carries_two_roundings(T, E, k, H, I):
    """dgate/dup must be bf16 (MMA operands) and dx is returned in bf16; nothing between them is rounded to 16 bits.

    Tolerance: one rounding of dx puts the 64-bit values e1 (measured on them) away, in the 2-norm.  A rounding of
    dgate/dup puts dx the same share away: the errors of its terms are independent, as relative to their terms as
    e1 is.  Two: sqrt(2) e1 = 1.414 e1; the sample (>= 38400 values, of which each error's square varies by about its
    own size) moves that by under 2%, the fp32 parts by 2^-10 of it: 1.5 e1.  (A third rounding would give 1.73 e1.)"""
    dev = _dev()
    from mirai_b200 import experts as ex
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(T)
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    for i, (key, shape) in enumerate({"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items()):
        m.load_dense_weight(key, weight(E, *shape, dev, i + 1))
    x = rows(T, H, dev).requires_grad_()
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices
    score = torch.rand(T, k, generator=g) + 0.1
    grad = torch.randn(T, H, generator=g).bfloat16()
    m.run_direct_routed(x, score.to(dev), idx.to(dev)).backward(grad.to(dev))
    ops.check_device()
    b = m.bound_weights()
    w64 = [ops.mxfp4_dequantize(t, out_dtype=torch.float32).cpu().double() for t in (b.w1, b.w3, b.w2)]
    dx = layer64(x.detach().cpu(), idx, score, w64, grad.double())[1]
    assert norm_error(x.grad, dx) <= 1.5 * norm_error(dx.bfloat16(), dx)


@pytest.mark.parametrize("k", [1, 3])
def test_rows_and_weights_of_the_combine_backward(k):
    dev = _dev()
    from mirai_b200 import ops
    T, H, E = 37, 72, 5
    g = torch.Generator().manual_seed(k)
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices
    plan = ops.dispatch_plan(idx.to(dev), E)
    w = torch.rand(T, k, generator=g)
    grad, y = torch.randn(T, H, generator=g).bfloat16(), torch.randn(T * k, H, generator=g).bfloat16()
    got, rw, gw = ops.combine_backward_rows(grad.to(dev), y.to(dev), plan.inverse_order, w.to(dev))
    same = ops.combine_backward(grad.to(dev), y.to(dev), plan.inverse_order, w.to(dev))
    ops.check_device()
    inv = plan.inverse_order.cpu().view(T, k)
    assert torch.equal(gw, same[1])
    assert torch.equal((got.float() * rw[:, None]).bfloat16(), same[0])  # its one rounding, left to the product
    for t in range(T):
        for j in range(k):
            assert torch.equal(got[inv[t, j]].cpu(), grad[t]) and rw[inv[t, j]].cpu() == w[t, j]
    with pytest.raises(ValueError, match="do not fit"):
        ops.combine_backward_rows(grad.to(dev), y[1:].to(dev), plan.inverse_order, w.to(dev))


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("T,k,H", [(1, 1, 8), (33, 2, 72), (300, 5, 264)])
def test_combine_of_fp32_rows(T, k, H, weighted):
    """k products and additions in fp32: at most 2 k roundings of 2^-24 of the sum of magnitudes, then the output's."""
    dev = _dev()
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(H)
    y = torch.randn(T * k, H, generator=g)
    inv = torch.randperm(T * k, generator=g)
    w = torch.rand(T, k, generator=g) if weighted else None
    terms = y.double()[inv].view(T, k, H) * (w.double()[..., None] if weighted else 1)
    ref, mag = terms.sum(1), terms.abs().sum(1)
    for dtype, last in ((torch.float32, 0.0), (torch.bfloat16, 2.0 ** -8)):
        out = ops.combine(y.to(dev), inv.to(dev), w.to(dev) if weighted else None, out_dtype=dtype, top_k=k)
        assert out.dtype == dtype
        assert ((out.cpu().double() - ref).abs() <= (2 * k * 2.0 ** -24) * mag + last * ref.abs() * (1 + 2.0 ** -20)).all()
    ops.check_device()
    with pytest.raises(TypeError, match="bf16_accumulate"):
        ops.combine(y.to(dev), inv.to(dev), w.to(dev) if weighted else None, top_k=k, bf16_accumulate=True)
    with pytest.raises(TypeError, match="y_sorted"):
        ops.combine(y.double().to(dev), inv.to(dev), None, top_k=k)


CASES = [([1], 64, 64), ([130, 0, 7], 192, 320), ([257, 300], 128, 448), ([5, 64, 1, 0, 40], 320, 64)]


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("counts,H,I", CASES)
def test_gate_up_saved_in_fp32(counts, H, I, few, monkeypatch):
    """The accumulators: rounded to bf16 they are what the bf16 form saves, and h does not change."""
    dev = _dev()
    from mirai_b200 import ops
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS", 1024 if few else -1)
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS_PER_SEGMENT", 0)
    E, S = len(counts), sum(counts)
    x = rows(S + 3, H, dev)
    off = segments(counts, dev)
    w1, w3 = ops.mxfp4_quantize(weight(E, I, H, dev, 1)), ops.mxfp4_quantize(weight(E, I, H, dev, 2))
    h, gu = ops.gateup_swiglu(x, off, w1, w3, inter=I, save_gate_up=True)
    h32, gu32 = ops.gateup_swiglu(x, off, w1, w3, inter=I, save_gate_up=True, gate_up_dtype=torch.float32)
    ops.check_device()
    assert gu32.dtype == torch.float32 and torch.equal(h[:S], h32[:S])
    assert torch.equal(gu32[:S].bfloat16(), gu[:S])
    for half, w in enumerate((w1, w3)):
        ref, m = product64(values64(x[:S]), counts, ops.mxfp4_dequantize(w, out_dtype=torch.float32).cpu().double())
        assert ((gu32[:S, half * I:(half + 1) * I].cpu().double() - ref).abs() <= step(H) * m).all()
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.gateup_swiglu(x, off, w1, w3, inter=I, save_gate_up=True, gate_up_dtype=torch.float16)
    dense = weight(E, I, H, dev, 1).bfloat16()
    with pytest.raises(TypeError, match="needs MXFP4"):
        ops.gateup_swiglu(x, off, dense, dense, inter=I, save_gate_up=True, gate_up_dtype=torch.float32)


@pytest.mark.parametrize("sources", [1, 2])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("counts,H,I", CASES)
def test_down_dx_from_fp32_gate_up(counts, H, I, weighted, sources):
    """dgate/dup from rows, their weights and fp32 gate/up; rows behind the last segment are left alone.

    Accumulation: K = 16 products a step, H/16 steps, each rounding (or truncating) at 2^-23 of the running magnitude, which
    sum |a b| = m bounds: dh off by (H/16 + 2) 2^-23 m, times |w|.  SwiGLU's factors are within a few units of fp32
    (2^-20 covers them and expf's), then one bf16 rounding."""
    dev = _dev()
    from mirai_b200 import ops
    counts = counts * sources
    E, S = len(counts) // sources, sum(counts)
    g = torch.Generator().manual_seed(I)
    gy = torch.randn(S + 2, H, generator=g).bfloat16()
    gu = torch.randn(S + 2, 2 * I, generator=g) * 2
    rw = torch.rand(S + 2, generator=g) + 0.1 if weighted else None
    w2 = ops.mxfp4_quantize(weight(E, H, I, dev, 3))
    w64 = ops.mxfp4_dequantize(w2, out_dtype=torch.float32).cpu().double()
    out = torch.full((S + 2, 2 * I), 7.0, dtype=torch.bfloat16, device=dev)
    off = segments(counts, dev)
    if weighted:
        ops._down_dx_mxfp4(gy.to(dev), off, w2, gu.to(dev), inter=I, out=out, lora=None, rank_a=None, sources=sources,
                           row_weights=rw.to(dev))
    else:
        ops.down_dx(gy.to(dev), off, w2, gu.to(dev), inter=I, out=out, sources=sources)
    ops.check_device()
    assert (out[S:] == 7).all()
    r = 0
    for i, n in enumerate(counts):
        a, w = gy[r:r + n].double(), w64[i % E]
        s = rw[r:r + n].double()[:, None] if weighted else torch.ones(n, 1, dtype=torch.float64)
        dh, off_by = s * (a @ w), s * (a.abs() @ w.abs()) * (H / 16 + 2) * 2.0 ** -23
        gate, up = gu[r:r + n, :I].double(), gu[r:r + n, I:].double()
        sg = torch.sigmoid(gate)
        for half, (factor, parts) in enumerate(((up * sg * (1 + gate * (1 - sg)), up.abs() * sg * (1 + gate.abs())),
                                                (gate * sg, (gate * sg).abs()))):
            # (the gate's factor 1 + g (1 - s) may cancel: the fp32 errors are of its parts)
            ref, fp32 = dh * factor, off_by * factor.abs() + 2.0 ** -20 * dh.abs() * parts
            got = out[r:r + n, half * I:(half + 1) * I].cpu().double()
            assert ((got - ref).abs() <= fp32 + 2.0 ** -8 * (ref.abs() + fp32)).all()
        r += n
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops._down_dx_mxfp4(gy.to(dev), off, w2, gu.bfloat16().to(dev), inter=I, out=None, lora=None, rank_a=None,
                           sources=sources, row_weights=torch.ones(S + 2, device=dev))
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.down_dx(gy.to(dev), off, w2, gu.half().to(dev), inter=I, sources=sources)


@pytest.mark.parametrize("sources", [1, 2])
@pytest.mark.parametrize("counts,H,I", CASES)
def test_gateup_dx_in_fp32(counts, H, I, sources):
    """dx unrounded: 2 I / 16 steps of exact products, as above.  bf16 keys and MXFP4 keys alike."""
    dev = _dev()
    from mirai_b200 import ops
    counts = counts * sources
    E, S = len(counts) // sources, sum(counts)
    g = torch.Generator().manual_seed(H)
    dgu = torch.randn(S + 2, 2 * I, generator=g).bfloat16()
    w1, w3 = ops.mxfp4_quantize(weight(E, I, H, dev, 1)), ops.mxfp4_quantize(weight(E, I, H, dev, 2))
    off = segments(counts, dev)
    out = torch.full((S + 2, H), 7.0, device=dev)
    got = ops.gateup_dx(dgu.to(dev), off, w1, w3, hidden=H, sources=sources, out=out, out_dtype=torch.float32)
    d1, d3 = ops.mxfp4_dequantize(w1), ops.mxfp4_dequantize(w3)
    assert torch.equal(ops.gateup_dx(dgu.to(dev), off, d1, d3, hidden=H, sources=sources, out_dtype=torch.float32)[:S], got[:S])
    rounded = ops.gateup_dx(dgu.to(dev), off, w1, w3, hidden=H, sources=sources)
    ops.check_device()
    assert got.dtype == torch.float32 and (got[S:] == 7).all()
    assert torch.equal(got[:S].bfloat16(), rounded[:S])
    r = 0
    for i, n in enumerate(counts):
        a = dgu[r:r + n].double()
        w = torch.cat((d1[i % E], d3[i % E])).cpu().double()
        assert ((got[r:r + n].cpu().double() - a @ w).abs() <= (2 * I / 16 + 2) * 2.0 ** -23 * (a.abs() @ w.abs())).all()
        r += n
    with pytest.raises(ValueError, match="out must be"):
        ops.gateup_dx(dgu.to(dev), off, w1, w3, hidden=H, sources=sources, out_dtype=torch.float32, out=out.bfloat16())
    with pytest.raises(ValueError, match="keys"):
        ops.gateup_dx(dgu.to(dev), off, w1, w3, hidden=H + 64, sources=sources, out_dtype=torch.float32)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.gateup_dx(dgu.to(dev), off, w1, w3, hidden=H, sources=sources, out_dtype=torch.float16)


def test_dx_beside_an_adapter():
    """With a LoRA adapter on w2: its rank block is weighted with the product, in fp32.

    dx: the roundings of dgate/dup and dx as in the layer test, and the rank block's bf16 projection (a part of dh):
    sqrt(3) e1 = 1.73 e1, 1.85 e1 with the sample's part.  Factor gradients: the projection of h or of the gradient, its weight and
    nothing else is rounded: sqrt(2) 2^-8 and h's own steps at borders, under 0.008."""
    dev = _dev()
    from mirai_b200 import experts as ex
    from mirai_b200 import ops
    E, T, k, H, I, r = 3, 700, 2, 128, 192, 8
    g = torch.Generator().manual_seed(3)
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    for i, (key, shape) in enumerate({"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items()):
        m.load_dense_weight(key, weight(E, *shape, dev, i + 1))
    m.attach_expert_lora(tensor_name="w2", rank=r, alpha=16.0)
    m.expert_lora.to(dev)
    ad = m.expert_lora["w2"]
    with torch.no_grad():
        ad.lora_a.copy_(weight(E, r, I, dev, 8))
        ad.lora_b.copy_(weight(E, H, r, dev, 9))
    x = rows(T, H, dev).requires_grad_()
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices
    score = torch.rand(T, k, generator=g) + 0.1
    grad = torch.randn(T, H, generator=g).bfloat16()
    m.run_direct_routed(x, score.to(dev), idx.to(dev)).backward(grad.to(dev))
    ops.check_device()
    b = m.bound_weights()
    w1, w3, w2 = (ops.mxfp4_dequantize(t, out_dtype=torch.float32).cpu().double() for t in (b.w1, b.w3, b.w2))
    A, B = ad.lora_a.detach().cpu().bfloat16().double(), ad.lora_b.detach().cpu().bfloat16().double()
    sc, xq = 16.0 / r, values64(x)
    dA, dB, dx = torch.zeros_like(A), torch.zeros_like(B), torch.zeros(T, H, dtype=torch.float64)
    for e in range(E):
        t, j = (idx == e).nonzero().T
        gt, u = xq[t] @ w1[e].T, xq[t] @ w3[e].T
        sg = torch.sigmoid(gt)
        h = (gt * sg * u).bfloat16().double()
        gy = score.double()[t, j][:, None] * grad.double()[t]
        dB[e] = sc * gy.T @ (h @ A[e].T)
        dA[e] = sc * (gy @ B[e]).T @ h
        dh = gy @ w2[e] + sc * (gy @ B[e]) @ A[e]
        dx.index_add_(0, t, (dh * u * sg * (1 + gt * (1 - sg))) @ w1[e] + (dh * gt * sg) @ w3[e])
    assert norm_error(x.grad, dx) <= 1.85 * norm_error(dx.bfloat16(), dx)
    assert norm_error(ad.lora_a.grad, dA) < 0.008 and norm_error(ad.lora_b.grad, dB) < 0.008


@pytest.mark.parametrize("T", [0, 1])
def test_layer_of_no_token_and_of_one(T):
    """Nothing to compute, and a token whose second weight is 0: its route adds nothing to dx."""
    dev = _dev()
    from mirai_b200 import experts as ex
    from mirai_b200 import ops
    E, H, I = 3, 64, 128
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    for i, (key, shape) in enumerate({"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items()):
        m.load_dense_weight(key, weight(E, *shape, dev, i + 1))
    x = rows(T, H, dev).requires_grad_()
    idx = torch.tensor([[2, 0]] * T, dtype=torch.int64, device=dev).view(T, 2)
    score = torch.tensor([[0.75, 0.0]] * T, device=dev).view(T, 2).requires_grad_()
    grad = torch.ones(T, H, dtype=torch.bfloat16, device=dev)
    out = m.run_direct_routed(x, score, idx)
    dx, ds = torch.autograd.grad(out, [x, score], grad)
    ops.check_device()
    assert out.shape == dx.shape == (T, H) and ds.shape == (T, 2)
    if T:
        one = x.detach().requires_grad_()
        same = m.run_direct_routed(one, score[:, :1].detach(), idx[:, :1].contiguous())
        assert torch.equal(torch.autograd.grad(same, one, grad)[0], dx) and (ds != 0).all()
