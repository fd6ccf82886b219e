"""The operators around microscaled 4-bit (MXFP4) experts, as cases that can be timed and compared.

* ``route``: group-limited routing to experts (scores, choice bias, best groups, top-k, renormalised
  weights) and, for training, the gradient of the weights with respect to the logits;
* ``quantise``: MXFP4 quantisation of expert weights and the read-back of the stored values;
* ``gateup`` / ``down``: the two expert products over expert-contiguous rows with both operands in MXFP4
  (the rows are quantised inside the call, the weights once when a layer is loaded);
* ``layer``: the routed expert FFN made of them, forward and backward to tokens and route weights.

MXFP4: blocks of 32 consecutive elements of a row share a power-of-two scale 2^e with
e = clamp(floor(log2 max|x|) - 2, -127, 127), stored as the byte e + 127; an element is x / 2^e rounded to the nearest
of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to the even code, saturating) with a sign bit, two elements per byte, the first
in the low half. Scale bytes are stored in tiles of 128 rows x 4 blocks (512 bytes): row r, block b of a tile
is byte (r % 32) * 16 + (r // 32) * 4 + b; rows and blocks past the matrix are zero bytes.
"""

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ----------------------------------------------------------------------------- cases

def listed():
    return [
        # a few tokens of a generation step: launch latency is all there is
        {"name": "route_few", "op": "route", "T": 4, "E": 128, "k": 8, "groups": 8, "top_groups": 4, "group_score": "top2",
         "score": "sigmoid", "bias": True, "norm": "eps", "scale": 2.5, "dtype": "fp32", "train": False},
        # a video batch (two branches of 32768 tokens) over the largest expert count of the benchmark
        {"name": "route_video", "op": "route", "T": 65536, "E": 128, "k": 8, "groups": 8, "top_groups": 4, "group_score": "top2",
         "score": "sigmoid", "bias": True, "norm": "eps", "scale": 2.5, "dtype": "fp32", "train": False},
        # a ragged training batch, softmax scores, with the gradient of the logits
        {"name": "route_train", "op": "route", "T": 21847, "E": 256, "k": 8, "groups": 8, "top_groups": 3, "group_score": "max",
         "score": "softmax", "bias": False, "norm": "clamp", "scale": 1.0, "dtype": "fp32", "train": True},
        # one expert's small projection, odd sizes, a checkpoint in fp32
        {"name": "quantise_small", "op": "quantise", "E": 1, "out": 333, "inp": 416, "dtype": "fp32"},
        # a layer's gate projections as the trainer loads them
        {"name": "quantise_layer", "op": "quantise", "E": 32, "out": 1408, "inp": 2048, "dtype": "bf16"},
        # a generation step: a handful of rows, the experts' weights are what is read
        {"name": "gateup_few", "op": "gateup", "S": 16, "E": 32, "H": 2048, "I": 1408, "spread": 0.0, "save": False},
        # the benchmark's layer: 32768 tokens, two routes each
        {"name": "gateup_layer", "op": "gateup", "S": 65536, "E": 32, "H": 2048, "I": 1408, "spread": 0.0, "save": False},
        # a training batch with uneven experts, one of them empty, that keeps gate/up for its backward pass
        {"name": "gateup_uneven", "op": "gateup", "S": 20011, "E": 64, "H": 1056, "I": 800, "spread": 0.7, "save": True},
        {"name": "down_few", "op": "down", "S": 9, "E": 16, "H": 2048, "I": 1408, "spread": 0.7},
        {"name": "down_layer", "op": "down", "S": 65536, "E": 32, "H": 2048, "I": 1408, "spread": 0.0},
        # the whole expert layer in training at a size between the two
        {"name": "layer_train", "op": "layer", "T": 8192, "E": 32, "k": 2, "H": 2048, "I": 1408},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route", "quantise", "gateup", "gateup", "down", "layer"])
    if op == "route":
        groups = rng.choice([1, 2, 4, 5, 8, 16])
        per = rng.randint(max(1, -(-16 // groups)), 256 // groups)
        top_groups = rng.randint(-(-groups // 4), groups)
        train = rng.random() < 0.5
        # (one renormalised weight is 1 whatever the logits are: it has no gradient to compare)
        k = rng.randint(2 if train else 1, max(2, min(8, top_groups * per)))
        if top_groups * per < k:
            top_groups = groups
        return {"op": op, "T": _log(rng, 1, 65536), "E": groups * per, "k": k, "groups": groups, "top_groups": top_groups,
                "group_score": rng.choice(["top2", "max"]), "score": rng.choice(["sigmoid", "softmax"]),
                "bias": rng.random() < 0.5, "norm": rng.choice(["eps", "clamp", "none", "l1"]),
                "scale": round(rng.uniform(0.5, 3.0), 2), "dtype": rng.choice(["fp32", "bf16"]), "train": train}
    if op == "quantise":
        return {"op": op, "E": _log(rng, 1, 32), "out": _log(rng, 1, 1408), "inp": 32 * _log(rng, 1, 64),
                "dtype": rng.choice(["bf16", "fp32", "fp16"])}
    E = _log(rng, 1, 64)
    if op == "layer":
        return {"op": op, "T": _log(rng, 1, 8192), "E": max(2, E // 2), "k": rng.randint(1, 2), "H": 64 * rng.randint(1, 32),
                "I": 64 * rng.randint(1, 22)}
    case = {"op": op, "S": _log(rng, 1, 32768), "E": E, "H": 32 * _log(rng, 2, 64), "I": 32 * _log(rng, 2, 44),
            "spread": rng.choice([0.0, 0.4, 0.8])}
    return case | ({"save": rng.random() < 0.5} if op == "gateup" else {})


def work(case):
    op = case["op"]
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        b = TYPES[case["dtype"]].itemsize
        # logits in; ids and weights out; for training the weights' gradient in and the logits' gradient out
        return {"bytes": T * (E * b + 12 * k) + (T * (4 * k + E * b) if case["train"] else 0),
                "flops": T * E * (6 if not case["train"] else 10)}
    if op == "quantise":
        n = case["E"] * case["out"] * case["inp"]
        # values in, codes and scales kept, stored values out
        return {"bytes": n * (2 * TYPES[case["dtype"]].itemsize + 0.5 + 1 / 32), "flops": 4 * n}
    if op == "layer":
        T, E, k, H, I = (case[x] for x in ("T", "E", "k", "H", "I"))
        S = T * k
        used = min(E, S)
        # tokens, their gradients and the outputs; every expert's codes and scales for both directions
        return {"bytes": 2 * 4 * T * H + 20 * S + 2 * used * 3 * H * I * 17 / 32, "flops": 12 * S * H * I}
    S, E, H, I = (case[x] for x in ("S", "E", "H", "I"))
    used = min(E, S)
    if op == "gateup":
        return {"bytes": S * (2 * H + 2 * I + (4 * I if case["save"] else 0)) + used * 2 * H * I * 17 / 32, "flops": 4 * S * H * I}
    return {"bytes": S * (2 * H + 2 * I) + used * H * I * 17 / 32, "flops": 2 * S * H * I}


# ----------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _counts(case, seed):
    """Rows of each expert: even up to chance, or uneven with one expert left empty."""
    g = torch.Generator().manual_seed(seed + 1)
    E = case["E"]
    p = torch.exp(case["spread"] * torch.randn(E, generator=g))
    p = p.clamp(max=float(p.mean()) * 3)
    if case["spread"] and E > 3:
        p[int(torch.randint(E, (1,), generator=g))] = 0
    return torch.bincount(torch.multinomial(p, case["S"], replacement=True, generator=g), minlength=E)


def _rows(n, width, g):
    """Hidden states: unit normal with channels of different size, and now and then a padded (zero) row."""
    x = torch.randn(n, width, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(width, device="cuda", generator=g))
    if n > 100:
        x[torch.randint(n, (n // 100,), device="cuda", generator=g)] = 0
    return x.to(torch.bfloat16)


def _weight(E, out, inp, g):
    """An expert key as a layer holds it: packed codes and tiled scales of N(0, 0.02) weights."""
    codes, scale = _quantise(torch.randn(E, out, inp, device="cuda", generator=g) * 0.02)
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    rt, kt = -(-out // 128), -(-inp // 128)
    full = torch.zeros(E, rt * 128, kt * 4, dtype=torch.uint8, device="cuda")
    full[:, :out, :inp // 32] = scale
    tiles = full.view(E, rt, 4, 32, kt, 4).permute(0, 1, 4, 3, 2, 5).contiguous().view(E, rt, kt, 512)
    return packed, tiles


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        logits = (torch.randn(T, E, device="cuda", generator=g) * 1.2).to(TYPES[case["dtype"]])
        s = {"case": case, "logits": logits, "bias": None, "grad": None}
        if case["bias"]:
            s["bias"] = torch.randn(E, device="cuda", generator=g) * 0.1
        if case["train"]:
            s["grad"] = torch.randn(T, k, device="cuda", generator=g)
        return s
    if op == "quantise":
        shape = (case["E"], case["out"], case["inp"])
        return {"case": case, "w": (torch.randn(shape, device="cuda", generator=g) * 0.02).to(TYPES[case["dtype"]])}
    E, H, I = case["E"], case["H"], case["I"]
    if op == "layer":
        T, k = case["T"], case["k"]
        idx = torch.rand(T, E, device="cuda", generator=g).topk(k, dim=1).indices
        score = torch.rand(T, k, device="cuda", generator=g) + 0.1
        return {"case": case, "x": _rows(T, H, g), "idx": idx, "score": (score / score.sum(1, keepdim=True)).to(torch.bfloat16),
                "grad": torch.randn(T, H, device="cuda", generator=g).to(torch.bfloat16),
                "most": int(torch.bincount(idx.flatten(), minlength=E).max()),
                "w": [_weight(E, I, H, g), _weight(E, I, H, g), _weight(E, H, I, g)]}
    counts = _counts(case, seed)
    s = {"case": case, "offsets": counts.cumsum(0).to(torch.int32).cuda(), "most": int(counts.max())}
    if op == "gateup":
        return s | {"x": _rows(case["S"], H, g), "w": [_weight(E, I, H, g), _weight(E, I, H, g)]}
    # rows of the intermediate: a gated product, heavier in its tails than a normal
    h = torch.nn.functional.silu(torch.randn(case["S"], I, device="cuda", generator=g))
    return s | {"x": (h * torch.randn(case["S"], I, device="cuda", generator=g)).to(torch.bfloat16), "w": [_weight(E, H, I, g)]}


# ----------------------------------------------------------------------------- plain forms

def _quantise(x):
    """(codes, scale bytes) of the last dimension's blocks of 32; a block with an infinity or a NaN has the scale byte 255."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    v = b.abs() * ((127 - e) << 23).view(torch.float32).unsqueeze(-1)  # 2^-e by its bits: a power function may be off
    c = ((v > 0.25).byte() + (v >= 0.75).byte() + (v > 1.25).byte() + (v >= 1.75).byte() + (v > 2.5).byte() + (v >= 3.5).byte()
         + (v > 5).byte())
    c = c | (torch.signbit(b).byte() << 3)
    scale = (e + 127).to(torch.uint8)
    return c.flatten(-2), torch.where(torch.isfinite(top), scale, torch.full_like(scale, 255))


def _values(codes, scale):
    """The fp32 values that codes and scale bytes stand for."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    m = table[(codes & 7).long()] * (1 - 2 * (codes >> 3).float())
    s = torch.where(scale == 0, 1 << 22, scale.int() << 23).view(torch.float32)  # 2^(byte - 127) by its bits
    s = torch.where(scale == 255, torch.full_like(s, float("nan")), s)
    return (m.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _stored(weight):
    """The fp32 [E, out, in] values of a stored key."""
    packed, tiles = weight
    E, out, half = packed.shape
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    _, rt, kt, _ = tiles.shape
    scale = tiles.view(E, rt, kt, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(E, rt * 128, kt * 4)
    return _values(codes, scale[:, :out, :half // 16])


def _slots(offsets, most):
    """Row numbers [E, most] of each expert's segment, and which of them are in it."""
    end = offsets.long()
    begin = torch.cat((end.new_zeros(1), end[:-1]))
    row = begin[:, None] + torch.arange(most, device=end.device)
    live = row < end[:, None]
    return torch.where(live, row, torch.zeros_like(row)), live


def _product(x, offsets, most, w):
    """x [S, K] times each segment's w [E, N, K] transposed, fp32 [S, N]."""
    row, live = _slots(offsets, most)
    y = torch.bmm(x[row], w.transpose(1, 2))
    out = x.new_zeros(x.shape[0], w.shape[1])
    out[row[live]] = y[live]
    return out


def _keys_and_scores(logits, case, bias):
    """Scores, what experts are ranked by, and which experts a logit leaves open, in 64 bits."""
    lg = logits.double()
    open_ = ~(torch.isnan(lg) | (lg == -math.inf))
    if case["score"] == "sigmoid":
        score = torch.sigmoid(lg)
    else:
        score = torch.softmax(lg, -1)
        score = torch.where(open_.any(-1, keepdim=True), score, torch.zeros_like(score))
    key = lg if bias is None else score + bias.double()
    return score, torch.where(open_, key, torch.full_like(key, -math.inf)), open_


def _route(state):
    """Group-limited top-k; decisions in 64 bits, since two experts can lie closer than 32 bits tell apart."""
    case, bias = state["case"], state["bias"]
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    score, key, open_ = _keys_and_scores(state["logits"], case, bias)
    if case["group_score"] == "max" or E == G:
        group = key.view(T, G, -1).amax(-1)
    else:  # the sum of a group's two best (score + bias), an expert that is not there counting nothing
        sums = torch.where(open_, score if bias is None else key, torch.full_like(score, -math.inf))
        best = sums.view(T, G, -1).topk(2, -1).values
        group = best[..., 0] + torch.where(best[..., 1] == -math.inf, torch.zeros_like(best[..., 1]), best[..., 1])
    chosen = torch.sort(group, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
    allowed = torch.zeros(T, G, dtype=torch.bool, device=key.device).scatter_(1, chosen, True).repeat_interleave(E // G, 1)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    order = order.gather(1, torch.sort(allowed.gather(1, order).byte(), dim=-1, descending=True, stable=True).indices)
    idx = order[:, :k].contiguous()
    s = score.gather(1, idx)
    s = torch.where(torch.isnan(state["logits"]).any(-1, keepdim=True), torch.full_like(s, float("nan")), s)
    den, scale = _denominator(s, case)
    w = (s / den * scale).float()
    if not case["train"]:
        return [idx, w]
    # dL/ds_j = scale (g_j / den - [den follows the sum] sum_i g_i s_i / den^2), then through the score function
    g = state["grad"].double()
    total = s.sum(-1, keepdim=True)
    follows = {"none": torch.zeros_like(total), "eps": torch.full_like(total, float(k > 1)),
               "clamp": (total >= 1e-20).double(), "l1": (total >= 1e-12).double()}[case["norm"]]
    ds = scale * (g / den - follows * (g * s).sum(-1, keepdim=True) / den ** 2)
    if case["score"] == "sigmoid":
        part = ds * s * (1 - s)
        grad = torch.zeros_like(score).scatter_add_(1, idx, part)
    else:
        grad = torch.zeros_like(score).scatter_add_(1, idx, ds * s) - score * (ds * s).sum(-1, keepdim=True)
    return [idx, w, grad.to(state["logits"].dtype)]


def _denominator(s, case):
    """What the gathered scores are divided by, and what they are then multiplied by."""
    total = s.sum(-1, keepdim=True)
    if case["norm"] == "clamp":
        return total.clamp_min(1e-20), 1.0
    if case["norm"] == "eps":
        return (total + 1e-20 if case["k"] > 1 else torch.ones_like(total)), case["scale"]
    if case["norm"] == "l1":
        return total.clamp_min(1e-12), case["scale"]
    return torch.ones_like(total), case["scale"]


def _gated(g, u):
    return g * torch.sigmoid(g) * u


def _layer(state):
    """Forward, and backward through the stored weights (a quantised activation passes its gradient on as it is)."""
    case, x, idx, score = state["case"], state["x"], state["idx"], state["score"]
    E, I, k, most = case["E"], case["I"], case["k"], state["most"]
    w1, w3, w2 = _stored(state["w"][0]), _stored(state["w"][1]), _stored(state["w"][2])
    order = torch.sort(idx.flatten(), stable=True).indices
    token = order // k
    offsets = torch.bincount(idx.flatten(), minlength=E).cumsum(0)
    xq = _values(*_quantise(x))[token]
    g, u = _product(xq, offsets, most, w1), _product(xq, offsets, most, w3)
    h = _gated(g, u).to(torch.bfloat16)  # the tensor between the two products
    y = _product(_values(*_quantise(h)), offsets, most, w2)
    route = score.flatten()[order].float()
    out = torch.zeros(x.shape, device=x.device).index_add_(0, token, y * route[:, None])
    go = state["grad"].float()[token]
    dscore = torch.zeros_like(route).scatter_(0, order, (go * y).sum(-1)).view(score.shape)
    dh = _product(go * route[:, None], offsets, most, w2.transpose(1, 2))
    sg = torch.sigmoid(g)
    dg, du = dh * u * sg * (1 + g * (1 - sg)), dh * g * sg
    dx = _product(dg, offsets, most, w1.transpose(1, 2)) + _product(du, offsets, most, w3.transpose(1, 2))
    dx = torch.zeros(x.shape, device=x.device).index_add_(0, token, dx)
    return [out.to(x.dtype), dx.to(x.dtype), dscore.to(score.dtype)]


def _keys(state):
    """The weight keys as a layer's program binds them: descriptors of the stored buffers, made once."""
    if "bound" not in state:
        from mirai_b200 import ops
        state["bound"] = [ops.Mxfp4Tensor(packed, tiles) for packed, tiles in state["w"]]
    return state["bound"]


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from mirai_b200 import experts, ops
        if op == "route":
            how = {"score_func": case["score"], "norm": case["norm"], "route_scale": case["scale"]}
            idx, w = ops.route_groups(state["logits"], case["k"], num_groups=case["groups"], top_groups=case["top_groups"],
                                      group_score=case["group_score"], choice_bias=state["bias"], **how)
            if not case["train"]:
                return [idx, w]
            return [idx, w, ops.route_groups_backward(state["grad"], state["logits"], idx, **how)]
        if op == "quantise":
            return [ops.mxfp4_dequantize(ops.mxfp4_quantize(state["w"]), out_dtype=state["w"].dtype)]
        keys = _keys(state)
        if op == "gateup":
            h = ops.gateup_swiglu(state["x"], state["offsets"], *keys, inter=case["I"], save_gate_up=case["save"])
            return list(h) if case["save"] else [h]
        if op == "down":
            return [ops.down(state["x"], state["offsets"], *keys, hidden=case["H"])]
        bound = experts.GroupedExpertWeights("mxfp4", *keys, case["E"], case["H"], case["I"])
        x, score = state["x"].detach().requires_grad_(), state["score"].detach().requires_grad_()
        out = experts.run_routed(bound, x, score, state["idx"])
        return [out.detach(), *torch.autograd.grad(out, [x, score], state["grad"])]
    if op == "route":
        return _route(state)
    if op == "quantise":
        return [_values(*_quantise(state["w"])).to(state["w"].dtype)]
    if op == "layer":
        return _layer(state)
    x = _values(*_quantise(state["x"]))
    if op == "down":
        return [_product(x, state["offsets"], state["most"], _stored(state["w"][0])).to(torch.bfloat16)]
    g = _product(x, state["offsets"], state["most"], _stored(state["w"][0]))
    u = _product(x, state["offsets"], state["most"], _stored(state["w"][1]))
    h = _gated(g, u).to(torch.bfloat16)
    return [h, torch.cat((g, u), -1).to(torch.bfloat16)] if case["save"] else [h]


# ----------------------------------------------------------------------------- 64 bits

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _rounded(x):
    """The nearest MXFP4 values of a 2-D tensor, found by comparing the distances to all eight magnitudes."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    power = torch.tensor([2.0 ** n for n in range(-149, 129)], dtype=torch.float64, device=x.device)
    floor = power[(torch.bucketize(top, power, right=True) - 1).clamp_min(0)]  # the largest power of two in it
    s = (floor / 4).clamp_min(2.0 ** -127)
    m = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    far = ((b.abs() / s).unsqueeze(-1) - m).abs()
    near = far == far.amin(-1, keepdim=True)  # two of them at a midpoint: the even code is the nearest then
    near = near & ((near.sum(-1, keepdim=True) == 1) | (torch.arange(8, device=x.device) % 2 == 0))
    return (torch.copysign((near * m).sum(-1), b) * s).reshape(x.shape)


def _expert64(weight, e):
    """Expert e's stored matrix, entry by entry from the definition of the layout."""
    packed, tiles = weight[0][e], weight[1][e].flatten(1)
    out, half = packed.shape
    col = torch.arange(2 * half, device=packed.device)
    row = torch.arange(out, device=packed.device)[:, None]
    code = (packed[:, col // 2] >> (4 * (col % 2)).to(torch.uint8)) & 15
    block = col // 32
    byte = tiles[row // 128, (block // 4) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + block % 4]
    m = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=packed.device)[code.long()]
    return m * torch.tensor([2.0 ** (n - 127) for n in range(255)], dtype=torch.float64, device=packed.device)[byte.long()]


def _exact_route(state):
    case = state["case"]
    idx = _route(state)[0]  # whole numbers, which the plain form already decides in 64 bits
    lg = state["logits"].double().requires_grad_()
    s = (torch.sigmoid(lg) if case["score"] == "sigmoid" else torch.softmax(lg, -1)).gather(1, idx)
    den, scale = _denominator(s, case)
    w = s / den * scale
    if not case["train"]:
        return [None, w.detach()]
    return [None, w.detach(), torch.autograd.grad(w, lg, state["grad"].double())[0]]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantise":
        return [torch.stack([_rounded(w) for w in state["w"]])]
    if op == "route":
        return _exact_route(state)
    if op == "layer":  # expert by expert
        x, grad, xq = state["x"].double(), state["grad"].double(), _rounded(state["x"])
        out, dx, dscore = torch.zeros_like(x), torch.zeros_like(x), state["score"].double()
        for e in range(case["E"]):
            t, j = (state["idx"] == e).nonzero().T
            w1, w3, w2 = (_expert64(w, e) for w in state["w"])
            g, u = xq[t] @ w1.T, xq[t] @ w3.T
            sg = 1 / (1 + torch.exp(-g))
            y = _rounded((g * sg * u).to(torch.bfloat16)) @ w2.T
            r = state["score"].double()[t, j][:, None]
            out.index_add_(0, t, r * y)
            dscore[t, j] = (grad[t] * y).sum(-1)
            dh = (r * grad[t]) @ w2
            dx.index_add_(0, t, (dh * u * (sg + g * sg * (1 - sg))) @ w1 + (dh * g * sg) @ w3)
        return [out, dx, dscore]
    parts, begin = [], 0
    for e, end in enumerate(state["offsets"].tolist()):
        if end > begin:
            rows = _rounded(state["x"][begin:end])
            parts.append([rows @ _expert64(w, e).T for w in state["w"]])
        begin = end
    cols = [torch.cat(c) for c in zip(*parts)]
    if op == "down":
        return cols
    h = cols[0] / (1 + torch.exp(-cols[0])) * cols[1]
    return [h, torch.cat(cols, 1)] if case["save"] else [h]
