"""Group-limited routing and its gradient against a plain 64-bit statement.

Ids are exact.  Weights: a score carries at most 70 fp32 roundings (a softmax sum
of up to 1024 terms) and the renormalisation a few more, so 2^-17 of the value.
The gradient adds the cancellation g - mean: 2^-16 of scale max|g| / den * s.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mirai_b200.build import build
    build()
    return torch.device("cuda:0")


def scores64(logits, score_func):
    lg = logits.double()
    closed = torch.isnan(lg) | (lg == -float("inf"))
    if score_func == "sigmoid":
        s = torch.sigmoid(lg)
    else:
        s = torch.softmax(lg.masked_fill(closed, -float("inf")), -1)
    return s.masked_fill(closed, 0.0), closed


def normalise(s, norm, k, scale):
    total = s.sum(-1, keepdim=True)
    if norm == "clamp":
        return s / total.clamp_min(1e-20)
    if norm == "eps":
        return (s / (total + 1e-20) if k > 1 else s) * scale
    if norm == "l1":
        return s / total.clamp_min(1e-12) * scale
    return s * scale


def route64(logits, k, groups, top_groups, group_score, score_func, bias):
    """Ids [T, k], row by row with Python's sort."""
    s, closed = scores64(logits, score_func)
    T, E = s.shape
    gs = E // groups
    key = logits.double() if bias is None else s + bias.double()
    key = key.masked_fill(closed, -float("inf"))
    top = s if bias is None else key
    ids = []
    for t in range(T):
        value = []
        for g in range(groups):
            members = range(g * gs, (g + 1) * gs)
            if group_score == "max" or gs == 1:
                value.append(max(float(key[t, e]) for e in members))
            else:
                v = sorted((float(top[t, e]) for e in members if not closed[t, e]), reverse=True)
                value.append(sum(v[:2]) if v else -float("inf"))
        best = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
        members = [e for g in best for e in range(g * gs, (g + 1) * gs)]
        ids.append(sorted(members, key=lambda e: (-float(key[t, e]), e))[:k])
    return torch.tensor(ids)


SHAPES = [  # E, k, groups, top_groups
    (8, 2, 2, 1), (16, 1, 16, 4), (32, 4, 1, 1), (60, 3, 4, 2), (64, 6, 8, 3), (128, 8, 8, 4), (135, 7, 5, 3),
    (160, 6, 8, 3), (232, 2, 8, 8), (256, 8, 8, 4), (256, 16, 32, 20), (384, 8, 12, 5), (1000, 16, 4, 3), (1020, 5, 17, 9),
    (1024, 10, 1, 1), (4, 4, 2, 2), (1, 1, 1, 1),
]


@pytest.mark.parametrize("E,k,groups,top_groups", SHAPES)
@pytest.mark.parametrize("score_func,group_score,with_bias,norm", [
    ("sigmoid", "top2", True, "eps"), ("softmax", "max", False, "clamp"), ("softmax", "top2", True, "l1"),
    ("sigmoid", "max", True, "none"), ("sigmoid", "top2", False, "l1")])
def test_route_groups_matches_64_bits(E, k, groups, top_groups, score_func, group_score, with_bias, norm):
    dev = _dev()
    from mirai_b200 import ops
    T = 61
    g = torch.Generator().manual_seed(E + k)
    logits = torch.randn(T, E, generator=g) * 1.3
    logits[3] = 0.25                       # every expert ties
    logits[4, ::2] = logits[4, 0].item()   # half of them do
    logits[5] = torch.nextafter(logits[5, :1].expand(E), torch.full((E,), 9.0))
    logits[5, 0] = torch.nextafter(logits[5, 0], torch.tensor(-9.0))  # an ulp apart
    bias = torch.randn(E, generator=g) * 0.1 if with_bias else None
    for dtype in (torch.float32, torch.bfloat16):
        lg = logits.to(dtype)
        idx, w = ops.route_groups(lg.to(dev), k, num_groups=groups, top_groups=top_groups, group_score=group_score,
                                  score_func=score_func, choice_bias=None if bias is None else bias.to(dev), norm=norm,
                                  route_scale=2.5)
        ops.check_device()
        ref = route64(lg.float(), k, groups, top_groups, group_score, score_func, bias)
        assert torch.equal(idx.cpu(), ref)
        want = normalise(scores64(lg.float(), score_func)[0].gather(1, ref), norm, k, 2.5)
        assert ((w.cpu().double() - want).abs() <= 2.0 ** -17 * want.abs()).all()


def test_close_keys_are_decided_as_in_64_bits():
    """Keys that fp32 cannot tell apart: biases that undo the scores to within 1e-9."""
    dev = _dev()
    from mirai_b200 import ops
    T, E = 257, 64
    g = torch.Generator().manual_seed(0)
    row = torch.randn(E, generator=g)
    bias = (0.75 - torch.sigmoid(row.double())).float()
    logits = (row + torch.randn(T, E, generator=g) * 1e-7).float()
    for group_score in ("max", "top2"):
        idx, _ = ops.route_groups(logits.to(dev), 6, num_groups=8, top_groups=3, group_score=group_score,
                                  choice_bias=bias.to(dev))
        assert torch.equal(idx.cpu(), route64(logits, 6, 8, 3, group_score, "sigmoid", bias))


@pytest.mark.parametrize("score_func", ["sigmoid", "softmax"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("group_score", ["top2", "max"])
def test_masked_experts(score_func, with_bias, group_score):
    dev = _dev()
    from mirai_b200 import ops
    T, E, k = 40, 32, 4
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(T, E, generator=g)
    logits[torch.rand(T, E, generator=g) < 0.6] = -float("inf")
    logits[0] = -float("inf")                       # nothing left
    logits[1] = -float("inf")
    logits[1, 21] = -3.0                            # one expert left
    logits[2] = torch.finfo(torch.float32).min      # the type's lowest value is a value
    logits[3, 5] = float("nan")
    bias = torch.randn(E, generator=g) if with_bias else None
    idx, w = ops.route_groups(logits.to(dev), k, num_groups=4, top_groups=2, group_score=group_score,
                              score_func=score_func, choice_bias=None if bias is None else bias.to(dev), norm="l1")
    ops.check_device()
    ref = route64(logits, k, 4, 2, group_score, score_func, bias)
    assert torch.equal(idx.cpu(), ref)
    w = w.cpu()
    assert idx[0].tolist() == [0, 1, 2, 3] and w[0].tolist() == [0.0] * k
    assert idx[1, 0].item() == 21 and abs(w[1, 0].item() - 1) < 1e-6 and w[1, 1:].tolist() == [0.0] * 3
    assert torch.isnan(w[3]).all() and not torch.isnan(w[[r for r in range(T) if r != 3]]).any()
    want = normalise(scores64(logits, score_func)[0].gather(1, ref), "l1", k, 1.0)
    keep = torch.arange(T) != 3
    assert ((w.double() - want).abs() <= 2.0 ** -17 * want.abs())[keep].all()


@pytest.mark.parametrize("T", [0, 1, 2, 31, 33, 4097])
def test_route_groups_token_counts(T):
    dev = _dev()
    from mirai_b200 import ops
    E, k = 48, 3
    lg = torch.randn(T, E, generator=torch.Generator().manual_seed(T))
    idx, w = ops.route_groups(lg.to(dev), k, num_groups=6, top_groups=2)
    assert idx.shape == (T, k) and w.shape == (T, k)
    assert torch.equal(idx.cpu(), route64(lg, k, 6, 2, "top2", "sigmoid", None).view(T, k).long())
    gl = ops.route_groups_backward(torch.ones(T, k, device=dev), lg.to(dev), idx)
    assert gl.shape == (T, E)


GRADS = [("sigmoid", "eps"), ("softmax", "clamp"), ("softmax", "none"), ("sigmoid", "l1"), ("softmax", "eps"),
         ("sigmoid", "none")]


def grad64(gw, logits, idx, score_func, norm, scale):
    lg = logits.double().requires_grad_()
    s = torch.sigmoid(lg) if score_func == "sigmoid" else torch.softmax(lg, -1)
    w = normalise(s.gather(1, idx), norm, idx.shape[1], scale)
    return torch.autograd.grad(w, lg, gw.double())[0], s.detach()


@pytest.mark.parametrize("E,k", [(8, 2), (60, 3), (91, 9), (128, 8), (135, 7), (256, 8), (300, 1), (1023, 4), (1024, 16)])
@pytest.mark.parametrize("score_func,norm", GRADS)
def test_route_groups_gradient(E, k, score_func, norm):
    dev = _dev()
    from mirai_b200 import ops
    T = 37
    g = torch.Generator().manual_seed(E)
    gw = torch.randn(T, k, generator=g)
    for dtype in (torch.float32, torch.bfloat16):
        lg = torch.randn(T, E, generator=g).to(dtype)
        idx, _ = ops.route_groups(lg.to(dev), k, score_func=score_func, norm=norm)
        got = ops.route_groups_backward(gw.to(dev), lg.to(dev), idx, score_func=score_func, norm=norm, route_scale=1.7)
        ops.check_device()
        assert got.dtype == dtype
        ref, s = grad64(gw, lg.float(), idx.cpu(), score_func, norm, 1.7)
        den = s.gather(1, idx.cpu()).sum(-1, keepdim=True) if norm != "none" and (k > 1 or norm != "eps") else 1.0
        tol = 2.0 ** -16 * 1.7 * gw.abs().amax(-1, keepdim=True) * k / den * s + torch.finfo(dtype).eps / 2 * ref.abs()
        assert ((got.cpu().double() - ref).abs() <= tol).all()


def test_gradient_against_differences():
    dev = _dev()
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(5)
    T, E, k = 3, 16, 4
    lg = torch.randn(T, E, generator=g)
    gw = torch.randn(T, k, generator=g)
    for score_func, norm in GRADS:
        idx, _ = ops.route_groups(lg.to(dev), k, num_groups=4, top_groups=2, score_func=score_func, norm=norm)
        got = ops.route_groups_backward(gw.to(dev), lg.to(dev), idx, score_func=score_func, norm=norm).cpu().double()

        def loss(x):
            s = torch.sigmoid(x) if score_func == "sigmoid" else torch.softmax(x, -1)
            return (normalise(s.gather(1, idx.cpu()), norm, k, 1.0) * gw.double()).sum()

        for t in range(T):
            for e in range(E):
                d = torch.zeros(T, E, dtype=torch.float64)
                d[t, e] = 1e-5
                diff = (loss(lg.double() + d) - loss(lg.double() - d)) / 2e-5
                # differences are off by h^2/6 of the third derivative (<= 20 of these functions) and the kernel by 1e-5
                assert abs(float(diff - got[t, e])) < 5e-5


def test_gradient_of_masked_rows_and_repeated_ids():
    dev = _dev()
    from mirai_b200 import ops
    T, E, k = 4, 16, 3
    lg = torch.randn(T, E, generator=torch.Generator().manual_seed(2))
    lg[0] = -float("inf")
    lg[1, 2:] = -float("inf")
    gw = torch.ones(T, k)
    gw[:, 1] = -2.0
    idx = torch.tensor([[0, 1, 2], [1, 0, 2], [7, 7, 3], [5, 5, 5]])
    for score_func, norm in GRADS:
        got = ops.route_groups_backward(gw.to(dev), lg.to(dev), idx.to(dev), score_func=score_func, norm=norm).cpu()
        ops.check_device()
        assert torch.equal(got[0], torch.zeros(E))  # nothing to learn where the mask leaves nothing
        assert torch.isfinite(got).all() and (got[1, 2:] == 0).all()
        ref, s = grad64(gw[2:], lg[2:], idx[2:], score_func, norm, 1.0)
        den = s.gather(1, idx[2:]).sum(-1, keepdim=True) if norm != "none" else 1.0
        assert ((got[2:].double() - ref).abs() <= 2.0 ** -16 * 2 * k / den * s).all()
    # an id outside the experts is recorded and skipped
    idx[3, 1] = E
    got = ops.route_groups_backward(gw.to(dev), lg.to(dev), idx.to(dev))
    assert ops.device_status() == (5, 750)
    assert torch.isfinite(got).all()


def test_unaligned_rows_other_streams_and_graphs():
    """Logits and bias that start off 16 bytes, two streams at once, and a captured route replayed on new logits."""
    dev = _dev()
    from mirai_b200 import ops
    T, E, k = 300, 64, 6
    g = torch.Generator().manual_seed(9)
    xs = [torch.randn(T, E, generator=g).to(dev) for _ in range(4)]
    bias = torch.randn(E, generator=g).to(dev) * 0.1
    kw = {"num_groups": 8, "top_groups": 3, "choice_bias": bias}
    want = [ops.route_groups(x, k, **kw) for x in xs]
    grads = [ops.route_groups_backward(w, x, i) for x, (i, w) in zip(xs, want)]
    store, bstore = torch.zeros(T * E + 1, device=dev), torch.zeros(E + 1, device=dev)
    store[1:], bstore[1:] = xs[0].flatten(), bias
    off = store[1:].view(T, E)
    idx, w = ops.route_groups(off, k, **dict(kw, choice_bias=bstore[1:]))
    assert torch.equal(idx, want[0][0]) and torch.equal(w, want[0][1])
    assert torch.equal(ops.route_groups_backward(w, off, idx), grads[0])
    turned = xs[1].t().contiguous().t()
    assert torch.equal(ops.route_groups(turned, k, **kw)[0], want[1][0])
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i, x in enumerate(xs):
        streams[i % 2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.route_groups(x, k, **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) for a, b in zip(got, want))
    static, graph = xs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx, w = ops.route_groups(static, k, **kw)
        gl = ops.route_groups_backward(w, static, idx)
    for x, (i, v), d in zip(xs, want, grads):
        static.copy_(x)
        graph.replay()
        assert torch.equal(idx, i) and torch.equal(w, v) and torch.equal(gl, d)
    ops.check_device()


def test_block_routes_by_groups_with_its_gradient():
    """block.route with groups: ids and the router weight's gradient as autograd in 64 bits gives them."""
    dev = _dev()
    from mirai_b200 import block
    T, H, E, k = 33, 64, 32, 4
    g = torch.Generator().manual_seed(11)
    x = torch.randn(T, H, generator=g)
    rw = torch.randn(E, H, generator=g) * 0.2
    bias = torch.randn(E, generator=g) * 0.05
    gw = torch.randn(T, k, generator=g)
    weight = rw.to(dev).requires_grad_()
    idx, w = block.route(x.to(dev), weight, top_k=k, correction_bias=bias.to(dev), route_scale=2.0, num_groups=8,
                         top_groups=3)
    w.backward(gw.to(dev))
    wd = rw.double().requires_grad_()
    s = torch.sigmoid(x.double() @ wd.T)
    ref = route64((x.double() @ rw.double().T).float(), k, 8, 3, "top2", "sigmoid", bias)
    assert torch.equal(idx.cpu(), ref)
    want = normalise(s.gather(1, ref), "eps", k, 2.0)
    want.backward(gw.double())
    assert torch.allclose(w.detach().cpu().double(), want.detach(), rtol=1e-5, atol=0)
    # fp32 products of 64 and 33 terms: 100 roundings of 2^-24 around sums of a few units
    assert (weight.grad.cpu().double() - wd.grad).abs().max() < 1e-4
