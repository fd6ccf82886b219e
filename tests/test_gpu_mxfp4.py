"""MXFP4 experts against a plain 64-bit statement of the format and the products.

Quantised values are exact (one rounding, of exact quotients): compared for
equality.  A product accumulates exact fp4 products in fp32, one K = 64 step
at a time: each of the K/64 steps and the sum inside it may round (or truncate)
at 2^-23 of the running magnitude, which sum |a b| bounds, so
|g - g64| <= 2 (K/64 + 1) 2^-23 sum |a b|; bf16 outputs round once more (2^-8
of the value), and silu'(g) <= 1.1 carries an error of g into h.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mirai_b200.build import build
    build()
    return torch.device("cuda:0")


def values64(x):
    """The MXFP4 values of x [..., K] in 64 bits (CPU), by the definition."""
    b = x.detach().cpu().double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    m, ex = torch.frexp(top)
    e = torch.where(top > 0, ex.double() - 3, torch.full_like(top, -127.0)).clamp(-127, 127)
    s = 2.0 ** e
    v = (b.abs() / s).unsqueeze(-1)
    d = (v - VALUES).abs() + (torch.arange(8) % 2) * 2.0 ** -40  # a midpoint goes to the even code (fp32 quotients lie coarser)
    q = VALUES[d.argmin(-1)]
    out = torch.copysign(q, b) * s
    return torch.where(torch.isfinite(top), out, torch.full_like(out, float("nan"))).flatten(-2)


def segments(counts, device):
    return torch.tensor(counts).cumsum(0).to(torch.int32).to(device)


def product64(x, counts, w, sources=1):
    """(x_q W_e^T per segment, sum |a b|) of quantised rows, 64-bit."""
    E = w.shape[0]
    ys, ms, r = [], [], 0
    for g, n in enumerate(counts):
        a, b = x[r:r + n], w[g % E].T
        ys.append(a @ b)
        ms.append(a.abs() @ b.abs())
        r += n
    return torch.cat(ys), torch.cat(ms)


def step(K):
    return 2 * (K / 64 + 1) * 2.0 ** -23


def check(got, ref, tol):
    got = got.detach().cpu().double()
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got - ref).abs() / tol).max():.3g} x tolerance"


def rows(n, width, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, width, generator=g) * torch.exp(torch.randn(n, 1, generator=g))
    return x.to(torch.bfloat16).to(dev)


def weight(E, out, inp, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(E, out, inp, generator=g) * 0.05).to(dev)


# ----------------------------------------------------------------------------- format

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1, 32), (3, 5, 96), (2, 129, 160), (1, 300, 1056), (4, 128, 2048), (2, 64, 4160)])
def test_quantise_and_read_back_are_exact(shape, dtype):
    dev = _dev()
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(sum(shape))
    w = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-6, 6, (shape[0], shape[1], 1), generator=g).float())
    w[0, 0, :32] = 0
    w = w.to(dtype).to(dev)
    t = ops.mxfp4_quantize(w)
    ref = values64(w)
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = ops.mxfp4_dequantize(t, out_dtype=out_dtype)
        assert bool((got.cpu().double() == ref.to(out_dtype).double()).all())
    ops.check_device()
    # the scale tiles are the row-ordered bytes, with zero bytes past the matrix
    bytes_ = ops.mxfp4_scale_rows(t.scale, shape[1], shape[2])
    assert torch.equal(ops.mxfp4_scale_tiles(bytes_), t.scale)


def test_quantise_rounds_ties_to_even_and_saturates():
    dev = _dev()
    from mirai_b200 import ops
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.5, 7.96875]
    want = [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, 6.0]
    for sign in (1.0, -1.0):
        for scale in (2.0 ** -100, 2.0 ** -8, 1.0, 2.0 ** 90):
            row = torch.zeros(32)
            row[:len(mids)] = torch.tensor(mids) * sign * scale
            row[-1] = 4.0 * scale  # the block's exponent stays that of 4
            got = ops.mxfp4_dequantize(ops.mxfp4_quantize(row.view(1, 1, 32).to(dev)), out_dtype=torch.float32)
            assert got[0, 0, :len(mids)].cpu().tolist() == [v * sign * scale for v in want]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantise_extremes(dtype):
    dev = _dev()
    from mirai_b200 import ops
    fi = torch.finfo(dtype)
    tiny = 2.0 ** -149 if dtype == torch.float32 else 2.0 ** -133  # smallest subnormal
    w = torch.zeros(1, 7, 64, dtype=dtype)
    w[0, 0, 0] = fi.max
    w[0, 1, 0] = -fi.max
    w[0, 2, 3] = fi.tiny
    w[0, 3, :32] = tiny
    w[0, 4, 5] = float("inf")
    w[0, 5, 6] = float("nan")
    w[0, 6, 1] = float("-inf")
    w[:, 4:, 40] = 1.0  # the other block of these rows is untouched
    t = ops.mxfp4_quantize(w.to(dev))
    got = ops.mxfp4_dequantize(t, out_dtype=torch.float32).cpu().double()
    ref = values64(w)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got.nan_to_num(0.0), ref.nan_to_num(0.0))
    assert ops.mxfp4_scale_rows(t.scale, 7, 64)[0, 4:, 0].tolist() == [255] * 3


@pytest.mark.parametrize("counts,width", [([3], 32), ([0, 130, 0, 1, 257, 0], 96), ([128, 128], 256), ([1] * 40, 2048),
                                          ([0, 0], 64)])
def test_quantised_rows_match_the_matrix_quantiser(counts, width):
    """Same codes as quantising each segment as a matrix, gathered rows included."""
    dev = _dev()
    from mirai_b200 import ops
    S = sum(counts)
    x = rows(max(S, 1), width, dev)
    index = torch.randperm(max(S, 1), generator=torch.Generator().manual_seed(3)).to(dev)[:S]
    for idx in (None, index):
        q = ops.mxfp4_quantize_rows(x[:S] if idx is None else x, segments(counts, dev), row_index=idx)
        assert q.shape == (S, width)
        src = x[:S] if idx is None else x[idx]
        r = tile = 0
        for n in counts:
            if n:
                one = ops.mxfp4_quantize(src[r:r + n][None])
                assert torch.equal(q.packed[r:r + n], one.packed[0])
                nt = -(-n // 128)
                mine = ops.mxfp4_scale_rows(q.scale[tile:tile + nt][None], n, width)
                assert torch.equal(mine[0], ops.mxfp4_scale_rows(one.scale, n, width)[0])
                tile += nt
            r += n
    ops.check_device()


# ----------------------------------------------------------------------------- products

@pytest.fixture(params=["few", "general"])
def path(request, monkeypatch):
    """Both kernels of the products, whatever the rule on the rows would pick."""
    from mirai_b200 import ops
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS", 1024 if request.param == "few" else -1)
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS_PER_SEGMENT", 0)
    return request.param


CASES = [
    ([1], 32, 32), ([5], 64, 96), ([130], 96, 160), ([3, 0, 7, 0], 160, 64), ([257, 1, 0, 300], 288, 416),
    ([64, 512], 1408, 256), ([1, 1, 1, 1, 1, 1, 1, 1], 2048, 192), ([700, 0, 33], 544, 1056),
    ([0, 0, 0, 1], 256, 128), ([256, 256], 512, 512), ([2000], 320, 288),
    ([31, 32, 33, 0, 65], 4096, 96),
]


@pytest.mark.parametrize("counts,K,N", CASES)
def test_gateup_matches_64_bits(path, counts, K, N):
    dev = _dev()
    from mirai_b200 import ops
    E, S = len(counts), sum(counts)
    x, off = rows(S, K, dev), segments(counts, dev)
    w1, w3 = ops.mxfp4_quantize(weight(E, N, K, dev, 1)), ops.mxfp4_quantize(weight(E, N, K, dev, 2))
    h, gu = ops.gateup_swiglu(x, off, w1, w3, inter=N, save_gate_up=True)
    plain = ops.gateup_swiglu(x, off, w1, w3, inter=N)
    ops.check_device()
    xq = values64(x)
    g, gm = product64(xq, counts, ops.mxfp4_dequantize(w1, out_dtype=torch.float32).cpu().double())
    u, um = product64(xq, counts, ops.mxfp4_dequantize(w3, out_dtype=torch.float32).cpu().double())
    check(gu[:, :N], g, step(K) * gm + 2.0 ** -8 * g.abs())
    check(gu[:, N:], u, step(K) * um + 2.0 ** -8 * u.abs())
    sg = torch.sigmoid(g)
    ref = g * sg * u
    # expf and the fast division: 2^-20 of the value covers their few units in the last place
    check(h, ref, 1.1 * u.abs() * step(K) * gm + (g * sg).abs() * step(K) * um + (2.0 ** -8 + 2.0 ** -20) * ref.abs())
    assert torch.equal(h, plain)


@pytest.mark.parametrize("counts,K,N", CASES)
def test_down_matches_64_bits(path, counts, K, N):
    dev = _dev()
    from mirai_b200 import ops
    x, off = rows(sum(counts), K, dev), segments(counts, dev)
    w = ops.mxfp4_quantize(weight(len(counts), N, K, dev))
    y = ops.down(x, off, w, hidden=N)
    ops.check_device()
    ref, m = product64(values64(x), counts, ops.mxfp4_dequantize(w, out_dtype=torch.float32).cpu().double())
    check(y, ref, step(K) * m + 2.0 ** -8 * ref.abs())


@pytest.mark.parametrize("counts,K,N", [CASES[1], CASES[3], CASES[4], CASES[5], CASES[7]])
def test_quantised_gateup_feeds_down(counts, K, N):
    """quantize=True gives the rows that quantising the bf16 h gives."""
    dev = _dev()
    from mirai_b200 import ops
    E, off = len(counts), segments(counts, dev)
    x = ops.mxfp4_quantize_rows(rows(sum(counts), K, dev), off)
    w1, w3 = ops.mxfp4_quantize(weight(E, N, K, dev, 1)), ops.mxfp4_quantize(weight(E, N, K, dev, 2))
    w2 = ops.mxfp4_quantize(weight(E, K, N, dev, 3))
    h = ops.gateup_swiglu(x, off, w1, w3, inter=N)
    hq = ops.gateup_swiglu(x, off, w1, w3, inter=N, quantize=True)
    assert torch.equal(hq.packed, ops.mxfp4_quantize_rows(h, off).packed)
    assert torch.equal(ops.down(hq, off, w2, hidden=K), ops.down(h, off, w2, hidden=K))
    ops.check_device()


def test_source_major_segments(path):
    """Two sources' segments give what each source alone gives."""
    dev = _dev()
    from mirai_b200 import ops
    counts, E, K, N = [5, 140, 0, 3, 0, 260], 3, 160, 224
    x = rows(sum(counts), K, dev)
    w1, w3 = ops.mxfp4_quantize(weight(E, N, K, dev, 1)), ops.mxfp4_quantize(weight(E, N, K, dev, 2))
    w2 = ops.mxfp4_quantize(weight(E, K, N, dev, 3))
    off = segments(counts, dev)
    h = ops.gateup_swiglu(x, off, w1, w3, inter=N, sources=2)
    y = ops.down(h, off, w2, hidden=K, sources=2)
    cut = sum(counts[:3])
    for part, c in ((slice(0, cut), counts[:3]), (slice(cut, None), counts[3:])):
        o = segments(c, dev)
        hp = ops.gateup_swiglu(x[part], o, w1, w3, inter=N)
        assert torch.equal(h[part], hp)
        assert torch.equal(y[part], ops.down(hp, o, w2, hidden=K))
    ops.check_device()
