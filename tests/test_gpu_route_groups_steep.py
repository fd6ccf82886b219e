"""Group-limited routing away from small logits and biases: gradients of sure routers, whose scores leave little of 1,
and groups whose two best keys are far larger than their sum."""

import pytest
import torch

from test_gpu_route_groups import _dev, grad64, route64

pytestmark = pytest.mark.gpu

GRADS = [("sigmoid", "eps"), ("sigmoid", "none"), ("sigmoid", "l1"), ("softmax", "eps"), ("softmax", "none"),
         ("softmax", "clamp")]


def gradient64(gw, logits, idx, score_func, norm, scale):
    """(gradient [T, E], size of the terms each entry is summed from), in 64 bits without differences of near values:
    1 - s from the other experts, g_j - mean from differences of the gradients."""
    lg = logits.double()
    T, E = lg.shape
    k = idx.shape[1]
    if score_func == "sigmoid":
        s, left = torch.sigmoid(lg), torch.sigmoid(-lg)
    else:
        p = torch.exp(lg - lg.amax(-1, keepdim=True))
        s = p / p.sum(-1, keepdim=True)
        eye = torch.eye(E, dtype=torch.bool)
        left = torch.stack([p.masked_fill(eye[e], 0.0).sum(-1) for e in range(E)], -1) / p.sum(-1, keepdim=True)
    g, sj = gw.double(), s.gather(1, idx)
    total = sj.sum(-1, keepdim=True)
    eps = 1e-20 if norm == "eps" else 0.0
    follows = norm != "none" and not (norm == "eps" and k == 1)
    den = {"none": torch.ones_like(total), "eps": total + eps if k > 1 else torch.ones_like(total),
           "clamp": total.clamp_min(1e-20), "l1": total.clamp_min(1e-12)}[norm]
    scale = 1.0 if norm == "clamp" else scale
    same = (idx[:, :, None] == idx[:, None, :]).double()  # [T, j, i]
    if follows:
        diff = (g[:, :, None] - g[:, None, :]) * (sj / den)[:, None, :]
        a, size = diff.sum(-1) + g * eps / den, diff.abs().sum(-1) + (g * eps / den).abs()
        a, size = (same * a[:, None, :]).sum(-1), (same * size[:, None, :]).sum(-1)  # an expert named twice
        dot = (g * sj).sum(-1, keepdim=True) / den * eps / den
    else:
        if score_func == "sigmoid":
            terms = same * g[:, None, :]
        else:
            terms = same * g[:, None, :] * left.gather(1, idx)[:, :, None] - (1 - same) * (g * sj)[:, None, :]
        a, size = terms.sum(-1), terms.abs().sum(-1)
        dot = (g * sj).sum(-1, keepdim=True) / den
    if score_func == "sigmoid":
        a, size, dot = a * left.gather(1, idx), size * left.gather(1, idx), dot * 0
        base = torch.zeros_like(s)
    else:
        base = -s * dot * scale
        if follows:
            a, size = a - dot * den, size + (dot * den).abs()
    grad = base.clone().scatter_(1, idx, scale * sj / den * a)
    bound = base.abs().clone().scatter_(1, idx, scale * sj / den * size)
    if score_func == "softmax":  # an unselected expert's term: the mean's parts
        mean = (g * sj).abs().sum(-1, keepdim=True) / den * (eps / den if follows else 1.0)
        bound = torch.maximum(bound, (s * mean * scale).scatter(1, idx, 0.0))
    return grad, bound


@pytest.mark.parametrize("score_func,norm", GRADS)
def test_the_64_bit_gradient_is_autograds(score_func, norm):
    """At logits where autograd loses nothing (on the CPU; no kernel runs)."""
    g = torch.Generator().manual_seed(1)
    for k in (1, 4):
        lg, gw = torch.randn(9, 12, generator=g), torch.randn(9, k, generator=g)
        idx = torch.rand(9, 12, generator=g).topk(k, dim=1).indices
        if k > 1:
            idx[3, 1] = idx[3, 0]
        ref = grad64(gw, lg, idx, score_func, norm, 1.7)[0]
        mine = gradient64(gw, lg, idx, score_func, norm, 1.7)[0]
        assert ((ref - mine).abs() <= 1e-12).all()


@pytest.mark.parametrize("E,k", [(16, 1), (16, 4), (60, 3), (128, 8), (256, 12), (1000, 16)])
@pytest.mark.parametrize("score_func,norm", GRADS)
def test_gradient_of_steep_logits(E, k, score_func, norm):
    """Logits up to +-30, one expert at +30 in a third of the rows: the gradient is right relative to its own terms.

    Tolerance, of the size of the terms.  The exponent's argument (up to 60 in fp32, times log2 e) is off by 2^-19 + 2 *
    2^-18.5 of 1, a softmax's score and what is left of it, quotients of two such sums, by twice that and a few units: under
    2^-15.5; sigmoid's by less.  share, den, a_j's sum over k <= 16 slots: 20 roundings of 2^-24, under 2^-19.  Two
    scores and a complement multiply: 3 * 2^-15.5 < 2^-13.5.  bf16 rounds the result once more.  Entries under 2^-120 may
    be flushed."""
    dev = _dev()
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(E + k)
    T = 48
    for dtype in (torch.float32, torch.bfloat16):
        lg = (torch.rand(T, E, generator=g) * 60 - 30).to(dtype)
        lg[:T // 3] = (torch.randn(T // 3, E, generator=g) * 3).to(dtype)
        lg[torch.arange(T // 3), torch.randint(E, (T // 3,), generator=g)] = 30.0
        lg[T // 3, :] = torch.linspace(8, 30, E).to(dtype)
        gw = torch.randn(T, k, generator=g)
        idx, _ = ops.route_groups(lg.to(dev), k, score_func=score_func, norm=norm)
        got = ops.route_groups_backward(gw.to(dev), lg.to(dev), idx, score_func=score_func, norm=norm, route_scale=1.7)
        ops.check_device()
        ref, size = gradient64(gw, lg, idx.cpu(), score_func, norm, 1.7)
        tol = 2.0 ** -13.5 * size + torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -10) + 2.0 ** -120
        assert ((got.cpu().double() - ref).abs() <= tol).all()


def test_gradient_of_saturated_and_repeated_experts():
    """Infinite logits, a logit whose score rounds to 1, and an expert named twice beside a sure one."""
    dev = _dev()
    from mirai_b200 import ops
    lg = torch.tensor([[20.0, -20, 0, 3, 17, 25, -1, 2], [30.0, 5, 5, 0, 1, 2, 3, 4], [40.0, 40, -3, 1, 0, 2, 3, 4]])
    idx = torch.tensor([[5, 0, 4], [0, 1, 1], [1, 0, 6]])
    gw = torch.tensor([[1.0, -2, 0.5], [3.0, 1, -0.25], [0.5, 0.25, 2]])
    for score_func, norm in GRADS:
        got = ops.route_groups_backward(gw.to(dev), lg.to(dev), idx.to(dev), score_func=score_func, norm=norm,
                                        route_scale=1.7).cpu()
        ref, size = gradient64(gw, lg, idx, score_func, norm, 1.7)
        assert ((got.double() - ref).abs() <= 2.0 ** -13.5 * size + 2.0 ** -120).all()
        if score_func == "sigmoid":  # an infinite logit: its score is 1 and has no slope
            inf = lg.clone()
            inf[0, 5] = float("inf")
            got = ops.route_groups_backward(gw.to(dev), inf.to(dev), idx.to(dev), score_func=score_func, norm=norm)
            assert torch.isfinite(got).all() and got[0, 5] == 0
    ops.check_device()


@pytest.mark.parametrize("score_func", ["sigmoid", "softmax"])
@pytest.mark.parametrize("B", [4.0, 64.0, 4096.0])
@pytest.mark.parametrize("large", ["all", "first"])
def test_groups_of_two_large_keys_with_a_small_sum(score_func, B, large):
    """Groups of two experts with biases near +B and -B: s + bias rounds at B 2^-24, the sums lie closer than that.  Groups
    are chosen as in 64 bits, whether every group has such keys or only one that is not at the border."""
    dev = _dev()
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(int(B))
    T, G, k = 400, 8, 2
    base = torch.randn(T, 1, 2, generator=g)
    near = base + (torch.rand(T, G, 2, generator=g) * 2 - 1) * 2.0 ** -22 * B  # sums apart by about their rounding
    logits = near.reshape(T, 2 * G).float()
    bias = torch.zeros(G, 2)
    if large == "all":
        bias[:, 0], bias[:, 1] = B, -B
    else:
        bias[0, 0], bias[0, 1] = B, -B
    ids, _ = ops.route_groups(logits.to(dev), k, num_groups=G, top_groups=4, group_score="top2", score_func=score_func,
                              choice_bias=bias.flatten().to(dev))
    ops.check_device()
    ref = route64(logits, k, G, 4, "top2", score_func, bias.flatten())
    assert torch.equal(ids.cpu(), ref)
    # the same with every member's logit closed but the first: its key alone counts
    logits[:, 1::2] = -float("inf")
    ids, _ = ops.route_groups(logits.to(dev), k, num_groups=G, top_groups=4, group_score="top2", score_func=score_func,
                              choice_bias=bias.flatten().to(dev))
    assert torch.equal(ids.cpu(), route64(logits, k, G, 4, "top2", score_func, bias.flatten()))


@pytest.mark.parametrize("E,G,top_groups,k", [(16, 1, 1, 4), (128, 8, 4, 8), (256, 16, 8, 8), (1000, 4, 3, 16), (1024, 1, 1, 10)])
@pytest.mark.parametrize("score_func,group_score", [("sigmoid", "max"), ("softmax", "max"), ("sigmoid", "top2")])
def test_ties_of_bf16_logits(E, G, top_groups, k, score_func, group_score):
    """Logits on bf16's grid, most rows with equal ones at the cut: ids as in 64 bits, lowest first, from bf16, from the same
    values in fp32, and from fp32 where one value of a row has low bits that the ids' would hide."""
    dev = _dev()
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(E)
    lg = (torch.randn(60, E, generator=g) * 4).round().div(8 if E < 100 else 16).bfloat16()
    lg[::7, ::3] = -float("inf")
    odd = lg.float()
    odd[torch.arange(60), torch.randint(E, (60,), generator=g)] += 2.0 ** -21
    how = {"num_groups": G, "top_groups": top_groups, "group_score": group_score, "score_func": score_func}
    for x in (lg, lg.float(), odd):
        ids, _ = ops.route_groups(x.to(dev), k, **how)
        ops.check_device()
        assert torch.equal(ids.cpu(), route64(x.float(), k, G, top_groups, group_score, score_func, None))


@pytest.mark.parametrize("k,top_groups", [(2, 1), (3, 2), (6, 3)])
def test_block_tokens_use_their_best_groups(k, top_groups):
    """The groups of a token's experts, counted token by token, and which they are, against 64 bits."""
    dev = _dev()
    from mirai_b200 import block
    T, H, E, G = 100, 64, 16, 4
    g = torch.Generator().manual_seed(k)
    # (values on a grid: the logits are the same in fp32 and in 64 bits)
    x = torch.randint(-8, 9, (T, H), generator=g) / 8
    weight = torch.randint(-8, 9, (E, H), generator=g) / 64
    bias = torch.randn(E, generator=g) * 0.05
    idx, _ = block.route(x.to(dev), weight.to(dev), top_k=k, correction_bias=bias.to(dev), num_groups=G,
                         top_groups=top_groups)
    idx = idx.cpu()
    assert torch.equal(idx, route64(x.double() @ weight.double().T, k, G, top_groups, "top2", "sigmoid", bias))
    used = [len(set((row // (E // G)).tolist())) for row in idx]
    assert max(used) <= top_groups
    free, _ = block.route(x.to(dev), weight.to(dev), top_k=k, correction_bias=bias.to(dev))
    assert max(len(set((row // (E // G)).tolist())) for row in free.cpu()) > top_groups  # the limit is what keeps them
