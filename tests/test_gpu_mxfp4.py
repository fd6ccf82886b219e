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


# ----------------------------------------------------------------------------- how the products are called

def test_empty_calls_and_rows_behind_the_last_segment(path):
    dev = _dev()
    from mirai_b200 import ops
    E, K, N = 3, 64, 96
    w1, w3 = ops.mxfp4_quantize(weight(E, N, K, dev, 1)), ops.mxfp4_quantize(weight(E, N, K, dev, 2))
    w2 = ops.mxfp4_quantize(weight(E, K, N, dev, 3))
    none = ops.gateup_swiglu(rows(0, K, dev), segments([0, 0, 0], dev), w1, w3, inter=N)
    assert none.shape == (0, N) and ops.down(none, segments([0, 0, 0], dev), w2, hidden=K).shape == (0, K)
    # 300 rows, segments that end after 170: the rest stays as it was
    x, off = rows(300, K, dev), segments([40, 0, 130], dev)
    out = torch.full((300, N), 7.0, dtype=torch.bfloat16, device=dev)
    got = ops.gateup_swiglu(x, off, w1, w3, inter=N, out=out)
    assert got.data_ptr() == out.data_ptr() and (got[170:] == 7.0).all()
    assert torch.equal(got[:170], ops.gateup_swiglu(x[:170], off, w1, w3, inter=N))
    y = torch.full((300, K), -3.0, dtype=torch.bfloat16, device=dev)
    ops.down(got, off, w2, hidden=K, out=y)
    assert (y[170:] == -3.0).all() and not (y[:170] == -3.0).all()
    zero = torch.full((300, K), -3.0, dtype=torch.bfloat16, device=dev)
    ops.down(got, segments([0, 0, 0], dev), w2, hidden=K, out=zero)
    assert (zero == -3.0).all()
    ops.check_device()


def test_a_nan_row_stays_in_its_row(path):
    dev = _dev()
    from mirai_b200 import ops
    E, K, N = 2, 320, 160
    x, off = rows(40, K, dev), segments([25, 15], dev)
    w1, w3 = ops.mxfp4_quantize(weight(E, N, K, dev, 1)), ops.mxfp4_quantize(weight(E, N, K, dev, 2))
    clean = ops.gateup_swiglu(x, off, w1, w3, inter=N)
    x[3, 100], x[30, 5] = float("nan"), float("inf")
    got = ops.gateup_swiglu(x, off, w1, w3, inter=N)
    keep = [i for i in range(40) if i not in (3, 30)]
    assert torch.isnan(got[[3, 30]]).all() and torch.equal(got[keep], clean[keep])
    # a NaN scale of the weights: the channel it belongs to, of its expert
    w = weight(E, N, K, dev, 1)
    w[1, 7, 40] = float("nan")
    y = ops.gateup_swiglu(clean.new_ones(40, K), off, ops.mxfp4_quantize(w), w3, inter=N)
    assert torch.isnan(y[25:, 7]).all() and int(torch.isnan(y).sum()) == 15


def test_large_magnitudes_and_tiny_ones(path):
    dev = _dev()
    from mirai_b200 import ops
    E, K, N = 1, 256, 64
    x = rows(20, K, dev)
    w = ops.mxfp4_quantize(weight(E, N, K, dev))
    off = segments([20], dev)
    base = ops.down(x, off, w, hidden=N).float()
    for p in (-60, 60, 100):  # powers of two move through the scales exactly
        moved = ops.down((x.float() * 2.0 ** p).to(torch.bfloat16), off, w, hidden=N).float()
        assert torch.equal(moved, base * 2.0 ** p)


def test_strided_and_offset_inputs(path):
    dev = _dev()
    from mirai_b200 import ops
    E, K, N = 2, 96, 64
    off = segments([30, 21], dev)
    w = ops.mxfp4_quantize(weight(E, N, K, dev))
    x = rows(51, K, dev)
    wide = torch.zeros(51, 2 * K, dtype=torch.bfloat16, device=dev)
    wide[:, 1::2] = x
    shifted = torch.zeros(51 * K + 3, dtype=torch.bfloat16, device=dev)
    shifted[3:] = x.flatten()
    want = ops.down(x, off, w, hidden=N)
    assert torch.equal(ops.down(wide[:, 1::2], off, w, hidden=N), want)
    assert torch.equal(ops.down(shifted[3:].view(51, K), off, w, hidden=N), want)
    turned = weight(E, N, K, dev).transpose(1, 2).contiguous().transpose(1, 2)
    again = ops.mxfp4_quantize(turned)
    assert torch.equal(again.packed, w.packed) and torch.equal(again.scale, w.scale)


def test_refused_on_the_gpu():
    dev = _dev()
    from mirai_b200 import ops
    from mirai_b200._lib import MiraiError
    E, K, N = 2, 64, 96
    x, off = rows(10, K, dev), segments([4, 6], dev)
    w1, w3 = ops.mxfp4_quantize(weight(E, N, K, dev, 1)), ops.mxfp4_quantize(weight(E, N, K, dev, 2))
    w2 = ops.mxfp4_quantize(weight(E, K, N, dev, 3))
    with pytest.raises(TypeError, match="two Mxfp4Tensor"):
        ops.gateup_swiglu(x, off, w1, weight(E, N, K, dev), inter=N)
    with pytest.raises(TypeError, match="two Mxfp4Tensor"):
        ops.gateup_swiglu(x, off, w1, w2, inter=N)
    with pytest.raises(TypeError, match="needs MXFP4"):
        ops.gateup_swiglu(x, off, weight(E, N, K, dev).bfloat16(), weight(E, N, K, dev).bfloat16(), inter=N, quantize=True)
    with pytest.raises(ValueError, match="inter"):
        ops.gateup_swiglu(x, off, w1, w3, inter=64)
    with pytest.raises(ValueError, match="segments"):
        ops.gateup_swiglu(x, segments([4, 3, 3], dev), w1, w3, inter=N)
    with pytest.raises(ValueError, match="needs"):
        ops.gateup_swiglu(rows(10, 96, dev), off, w1, w3, inter=N)
    with pytest.raises(TypeError, match="float32"):
        ops.gateup_swiglu(x.float(), off, w1, w3, inter=N)
    with pytest.raises(TypeError, match="int64"):
        ops.down(rows(10, N, dev), off.long(), w2, hidden=K)
    with pytest.raises(ValueError, match="out must be"):
        ops.down(rows(10, N, dev), off, w2, hidden=K, out=torch.empty(10, K, device=dev))
    with pytest.raises(ValueError, match="segments"):
        ops.down(ops.mxfp4_quantize_rows(rows(10, N, dev), segments([10], dev)), off, w2, hidden=K)
    with pytest.raises(ValueError, match="no bf16 out"):
        ops.gateup_swiglu(x, off, w1, w3, inter=N, quantize=True, out=torch.empty(10, N, dtype=torch.bfloat16, device=dev))
    with pytest.raises(ValueError, match="needs rank_a"):
        lora = ops.DownLoRA(torch.zeros(E, 4, N, device=dev), torch.zeros(E, K, 4, device=dev), 1.0)
        ops.down(ops.mxfp4_quantize_rows(rows(10, N, dev), off), off, w2, hidden=K, lora=lora)
    with pytest.raises(ValueError, match="scale tiles"):
        ops.Mxfp4Tensor(w1.packed, w1.scale[:, :, :0])
    with pytest.raises(ValueError, match="scale"):
        ops.Mxfp4Rows(w1.packed[0], w1.scale[:1, 0, 0, :16].contiguous(), 2)
    with pytest.raises(TypeError, match="float64"):
        ops.mxfp4_quantize(torch.zeros(1, 1, 32, dtype=torch.float64, device=dev))
    with pytest.raises(ValueError, match="in % 32"):
        ops.mxfp4_quantize(torch.zeros(1, 4, 40, device=dev))
    with pytest.raises(ValueError, match="out must be"):
        ops.mxfp4_dequantize(w1, out=torch.empty(E, N, K + 1, device=dev)[:, :, :K])
    with pytest.raises(TypeError, match="bf16 or NF4"):
        ops.gateup_ex(x, off, w1, w3, inter=N, layout="out_in", activation="swiglu")
    with pytest.raises(ValueError, match="steps of 64"):
        ops.moe_forward_train(x, torch.zeros(10, 1, dtype=torch.int64, device=dev), torch.ones(10, 1, device=dev), w1, w3, w2,
                              num_experts=E, inter=N)
    with pytest.raises(TypeError, match="all three"):
        ops.moe_forward(x, torch.zeros(10, 1, dtype=torch.int64, device=dev), torch.ones(10, 1, device=dev), w1, w3,
                        weight(E, K, N, dev).bfloat16(), num_experts=E, inter=N)
    with pytest.raises(MiraiError, match="segments"):
        ops.mxfp4_quantize_rows(x, torch.zeros(1025, dtype=torch.int32, device=dev))
    ops.check_device()


def test_bad_offsets_and_row_indices_are_recorded(path):
    """Ends that fall or pass the rows, and rows outside the input, are recorded and kept in bounds."""
    dev = _dev()
    from mirai_b200 import ops
    E, K, N = 3, 64, 64
    w = ops.mxfp4_quantize(weight(E, N, K, dev))
    for ends in ([8, 4, 20], [5, 900, 901], [-4, 3, 20]):
        y = ops.down(rows(20, K, dev), torch.tensor(ends, dtype=torch.int32, device=dev), w, hidden=N)
        assert y.shape == (20, N)
        assert ops.device_status()[0] == 5
    q = ops.mxfp4_quantize_rows(rows(20, K, dev), segments([10, 0, 10], dev),
                                row_index=torch.tensor([0, -1, 20] + [5] * 17, device=dev))
    assert ops.device_status() == (5, 701)
    assert (q.packed[1:3] == 0).all()
    ops.check_device()


def test_streams_and_graphs(path):
    """Two calls at once on two streams, and a captured call replayed on new inputs beside an eager one."""
    dev = _dev()
    from mirai_b200 import ops
    E, K, N, S = 4, 256, 160, 600
    w1, w3 = ops.mxfp4_quantize(weight(E, N, K, dev, 1)), ops.mxfp4_quantize(weight(E, N, K, dev, 2))
    w2 = ops.mxfp4_quantize(weight(E, K, N, dev, 3))
    counts = [200, 0, 150, 250]
    xs, off = [rows(S, K, dev, i) for i in range(4)], segments(counts, dev)

    def layer(x):
        return ops.down(ops.gateup_swiglu(x, off, w1, w3, inter=N), off, w2, hidden=K)

    want = [layer(x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None] * 4
    for i, x in enumerate(xs):
        streams[i % 2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i % 2]):
            got[i] = layer(x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = xs[0].clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(static)
        graphs.append((g, out))
    for i, x in enumerate(xs):
        static.copy_(x)
        graphs[i % 2][0].replay()
        eager = layer(xs[(i + 1) % 4])
        assert torch.equal(graphs[i % 2][1], want[i]) and torch.equal(eager, want[(i + 1) % 4])
    ops.check_device()


def test_many_segments():
    """1024 segments (64 sources of 16 experts), most of them empty."""
    dev = _dev()
    from mirai_b200 import ops
    E, K, N = 16, 64, 64
    g = torch.Generator().manual_seed(4)
    counts = (torch.randint(0, 40, (1024,), generator=g) * (torch.rand(1024, generator=g) < 0.1)).tolist()
    x, off = rows(sum(counts), K, dev), segments(counts, dev)
    w = ops.mxfp4_quantize(weight(E, N, K, dev))
    y = ops.down(x, off, w, hidden=N, sources=64)
    ref, m = product64(values64(x), counts, ops.mxfp4_dequantize(w, out_dtype=torch.float32).cpu().double())
    check(y, ref, step(K) * m + 2.0 ** -8 * ref.abs())
    ops.check_device()


def test_offsets_beyond_32_bits():
    """Rows and weights of more than 2^31 elements: the last ones are where they belong."""
    dev = _dev()
    from mirai_b200 import ops
    K, S = 2048, (1 << 20) + 40_000  # 2.2 G elements
    x = torch.zeros(S, K, dtype=torch.bfloat16, device=dev)
    x[-300:] = rows(300, K, dev)
    w = ops.mxfp4_quantize(weight(2, 32, K, dev))
    off = segments([S - 300, 300], dev)
    y = ops.down(x, off, w, hidden=32)
    assert torch.equal(y[-300:], ops.down(x[-300:], segments([0, 300], dev), w, hidden=32))
    assert (y[:-300] == 0).all()
    del x, y
    big = torch.zeros(600, 1800, 2048, dtype=torch.bfloat16, device=dev)
    big[-1, -1] = rows(1, 2048, dev)[0]
    t = ops.mxfp4_quantize(big)
    one = ops.mxfp4_quantize(big[-1:])
    assert torch.equal(t.packed[-1], one.packed[0]) and torch.equal(t.scale[-1], one.scale[0])
    back = ops.mxfp4_dequantize(t, out=big)
    assert torch.equal(back[-1], ops.mxfp4_dequantize(one)[0]) and not back[:-1].any()
    ops.check_device()


# ----------------------------------------------------------------------------- adapter, layer, block

@pytest.mark.parametrize("counts,I,H,r", [([130, 0, 7], 96, 160, 8), ([300, 41], 1408, 288, 32), ([3, 2], 64, 64, 1),
                                          ([600, 0, 500], 2048, 256, 16)])
def test_down_with_an_adapter(counts, I, H, r):
    dev = _dev()
    from mirai_b200 import ops
    E, S = len(counts), sum(counts)
    h, off = rows(S, I, dev), segments(counts, dev)
    w = ops.mxfp4_quantize(weight(E, H, I, dev))
    a, b = weight(E, r, I, dev, 5).bfloat16(), weight(E, H, r, dev, 6).bfloat16()
    lora = ops.DownLoRA(a, b, 0.5)
    low = ops.lora_project(h, off, lora, forward=True)
    y = ops.down(h, off, w, hidden=H, lora=lora)
    assert torch.equal(ops.down(ops.mxfp4_quantize_rows(h, off), off, w, hidden=H, lora=lora, rank_a=low), y)
    ops.check_device()
    ref, m = product64(values64(h), counts, ops.mxfp4_dequantize(w, out_dtype=torch.float32).cpu().double())
    rank = low[:, :r].cpu().double()  # the projection as the kernel is given it
    add, add_m = product64(rank, counts, b.cpu().double())
    ref, m = ref + add, m + add_m
    check(y, ref, step(I + 64) * m + 2.0 ** -8 * ref.abs())


def layer64(x, idx, score, w, grad):
    """Output and gradients of the routed MXFP4 FFN in 64 bits: h is a bf16 tensor between the products, and
    the quantisers pass gradients straight through.  w: 64-bit (w1, w3, w2)."""
    xq = values64(x)
    out = torch.zeros(x.shape, dtype=torch.float64)
    dx, ds = torch.zeros_like(out), torch.zeros(score.shape, dtype=torch.float64)
    for e in range(w[0].shape[0]):
        t, j = (idx == e).nonzero().T
        if not len(t):
            continue
        g, u = xq[t] @ w[0][e].T, xq[t] @ w[1][e].T
        sg = torch.sigmoid(g)
        y = values64((g * sg * u).to(torch.bfloat16)) @ w[2][e].T
        s = score[t, j].double()[:, None]
        out.index_add_(0, t, s * y)
        ds[t, j] = (grad[t] * y).sum(-1)
        dh = (s * grad[t]) @ w[2][e]
        dx.index_add_(0, t, (dh * u * sg * (1 + g * (1 - sg))) @ w[0][e] + (dh * g * sg) @ w[1][e])
    return out, dx, ds


@pytest.mark.parametrize("T,E,k,H,I", [(1, 2, 1, 64, 64), (37, 4, 2, 128, 64), (300, 6, 2, 192, 320), (1000, 3, 3, 128, 192)])
def test_experts_forward_and_backward(T, E, k, H, I):
    """B200GroupedExperts in MXFP4 through its public entry point, with autograd.

    Tolerance in the 2-norm: out carries the roundings of y and out (2 x 2^-8), and where h lies within 2^-20 of a
    rounding border its bf16 value, and then a code, may step (under 1 in 1000 codes, each within 1/3 of its value):
    2^-8 sqrt(2) + 0.011 < 0.02.  dx passes the bf16 tensors gy, gate/up, dgate/dup, dx of a route and the sum:
    at most 6 roundings, 2^-8 sqrt(6) < 0.01, and the same steps do not enter (gradients are straight through)."""
    dev = _dev()
    from mirai_b200 import experts as ex
    from mirai_b200 import ops
    g = torch.Generator().manual_seed(T)
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    dense = {"w1": weight(E, I, H, dev, 1), "w3": weight(E, I, H, dev, 2), "w2": weight(E, H, I, dev, 3)}
    for key, w in dense.items():
        m.load_dense_weight(key, w)
    x = rows(T, H, dev).requires_grad_()
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices
    score = (torch.rand(T, k, generator=g) + 0.1).to(dev).requires_grad_()
    grad = torch.randn(T, H, generator=g).bfloat16()
    out = m.run_direct_routed(x, score, idx.to(dev))
    out.backward(grad.to(dev))
    ops.check_device()
    with torch.no_grad():
        plain = m.run_direct_routed(x, score, idx.to(dev))
    assert torch.equal(plain, out.detach())
    w64 = [ops.mxfp4_dequantize(t, out_dtype=torch.float32).cpu().double()
           for t in (m.bound_weights().w1, m.bound_weights().w3, m.bound_weights().w2)]
    ro, rx, rs = layer64(x.detach().cpu(), idx, score.detach().cpu(), w64, grad.double())

    def rel(a, b):
        return float((a.detach().cpu().double() - b).norm() / b.norm())

    assert rel(out, ro) < 0.02 and rel(x.grad, rx) < 0.01 and rel(score.grad, rs) < 0.02


def test_a_layer_runs_either_kernel_alike(monkeypatch):
    """A generation step's rows through the few-row products and through the general ones: the same accumulations."""
    dev = _dev()
    from mirai_b200 import ops
    E, T, k, H, I = 6, 9, 2, 320, 160
    g = torch.Generator().manual_seed(2)
    w1, w3 = ops.mxfp4_quantize(weight(E, I, H, dev, 1)), ops.mxfp4_quantize(weight(E, I, H, dev, 2))
    w2 = ops.mxfp4_quantize(weight(E, H, I, dev, 3))
    x = rows(T, H, dev)
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices.to(dev)
    score = torch.rand(T, k, generator=g).to(dev)
    few = ops.moe_forward(x, idx, score, w1, w3, w2, num_experts=E, inter=I)
    before = ops.launch_count()
    ops.moe_forward(x, idx, score, w1, w3, w2, num_experts=E, inter=I)
    assert ops.launch_count() - before == 4 + 4  # the plan, then permute, two products, combine
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS", -1)
    monkeypatch.setattr(ops, "MXFP4_FEW_ROWS_PER_SEGMENT", 0)
    general = ops.moe_forward(x, idx, score, w1, w3, w2, num_experts=E, inter=I)
    ops.check_device()
    # both add the same exact products step by step in fp32: at most a rounding of y and of the sum apart
    assert ((few.float() - general.float()).abs() <= 2.0 ** -7 * general.float().abs() + 2.0 ** -8 * general.float().abs().mean()).all()


def test_layer_gradient_against_differences():
    """The gradient of the smooth part: rows the quantiser keeps as they are (values on the grid), w2 = an adapter-free
    down of one expert.  Differences of the 64-bit layer with the quantisers left out agree with the kernels'."""
    dev = _dev()
    from mirai_b200 import experts as ex
    from mirai_b200 import ops
    E, T, H, I = 1, 4, 64, 64
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    for i, key in enumerate(("w1", "w3", "w2")):
        m.load_dense_weight(key, weight(E, H if key == "w2" else I, I if key == "w2" else H, dev, i) * 4)
    grid = torch.tensor([0.5, 1, 1.5, 2, 3, 4, 6])
    g = torch.Generator().manual_seed(1)
    x = grid[torch.randint(0, 7, (T, H), generator=g)] * (torch.randint(0, 2, (T, H), generator=g) * 2 - 1) / 8
    x[:, ::32] = 0.75
    xd = x.bfloat16().to(dev).requires_grad_()
    idx = torch.zeros(T, 1, dtype=torch.int64, device=dev)
    score = torch.ones(T, 1, device=dev)
    grad = torch.randn(T, H, generator=g).bfloat16()
    m.run_direct_routed(xd, score, idx).backward(grad.to(dev))
    b = m.bound_weights()
    w1, w3, w2 = (ops.mxfp4_dequantize(t, out_dtype=torch.float32).cpu().double()[0] for t in (b.w1, b.w3, b.w2))

    def loss(v):
        a, u = v @ w1.T, v @ w3.T
        return ((a * torch.sigmoid(a) * u) @ w2.T * grad.double()).sum()

    diff = torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for c in range(H):
            d = torch.zeros(T, H, dtype=torch.float64)
            d[t, c] = 1e-4
            diff[t, c] = (loss(x.double() + d) - loss(x.double() - d)) / 2e-4
    assert float((xd.grad.cpu().double() - diff).norm() / diff.norm()) < 0.01  # six bf16 roundings, as above


def test_adapter_gradients_of_an_mxfp4_layer():
    """The adapter's factor gradients and dX with a LoRA on w2, against 64 bits."""
    dev = _dev()
    from mirai_b200 import experts as ex
    from mirai_b200 import ops
    E, T, k, H, I, r = 3, 260, 2, 128, 192, 8
    g = torch.Generator().manual_seed(3)
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    for key, (o, i) in {"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items():
        m.load_dense_weight(key, weight(E, o, i, dev, len(key) + o))
    m.attach_expert_lora(tensor_name="w2", rank=r, alpha=16.0)
    m.expert_lora.to(dev)
    ad = m.expert_lora["w2"]
    with torch.no_grad():
        ad.lora_a.copy_(weight(E, r, I, dev, 8))
        ad.lora_b.copy_(weight(E, H, r, dev, 9))
    x = rows(T, H, dev).requires_grad_()
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices
    score = (torch.rand(T, k, generator=g) + 0.1).to(dev)
    grad = torch.randn(T, H, generator=g).bfloat16()
    m.run_direct_routed(x, score, idx.to(dev)).backward(grad.to(dev))
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
        gy = score.cpu().double()[t, j][:, None] * grad.double()[t]
        dB[e] = sc * gy.T @ (h @ A[e].T)
        dA[e] = sc * (gy @ B[e]).T @ h
        dh = gy @ w2[e] + sc * (gy @ B[e]) @ A[e]
        dx.index_add_(0, t, (dh * u * sg * (1 + gt * (1 - sg))) @ w1[e] + (dh * gt * sg) @ w3[e])

    def rel(a, ref):
        return float((a.detach().cpu().double() - ref).norm() / ref.norm())

    # h, gy, the rank blocks: four bf16 roundings at most (2^-8 sqrt(4) < 0.01); dx as in the layer test
    assert rel(ad.lora_a.grad, dA) < 0.01 and rel(ad.lora_b.grad, dB) < 0.01 and rel(x.grad, dx) < 0.01


def test_block_with_groups_and_mxfp4_experts():
    """The block as it is used: grouped routing, MXFP4 experts, padding, token chunks, gradients to tokens and router."""
    dev = _dev()
    from mirai_b200 import block, ops
    from mirai_b200 import experts as ex
    B, S, H, I, E, k = 2, 60, 128, 64, 8, 2
    g = torch.Generator().manual_seed(12)
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    for key, (o, i) in {"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items():
        m.load_dense_weight(key, weight(E, o, i, dev, o + len(key)))
    kw = {"hidden_size": H, "num_experts": E, "top_k": k, "experts": m, "num_groups": 4, "top_groups": 2,
          "route_scale": 1.5}
    blk = block.B200SparseMoeBlock(**kw).to(dev)
    chunked = block.B200SparseMoeBlock(**kw, token_chunk_policy=block.TokenChunkPolicy(32)).to(dev)
    with torch.no_grad():
        blk.router_weight.copy_(torch.randn(E, H, generator=g) * 0.1)
        blk.e_score_correction_bias.copy_(torch.randn(E, generator=g) * 0.05)
        chunked.load_state_dict(blk.state_dict())
    hidden = torch.randn(B, S, H, generator=g).bfloat16().to(dev)
    mask = (torch.arange(S) < torch.tensor([[S], [41]])).reshape(-1).to(dev)
    x = hidden.clone().requires_grad_()
    out = blk(x, padding_mask=mask)
    out.float().square().sum().backward()
    x2 = hidden.clone().requires_grad_()
    out2 = chunked.train()(x2, padding_mask=mask)
    out2.float().square().sum().backward()
    ops.check_device()
    assert torch.equal(out, out2) and torch.isfinite(x.grad).all() and torch.isfinite(blk.router_weight.grad).all()
    assert (out[1, 41:] == 0).all() and not (out[1, :41] == 0).all()
    # the router's gradient does not depend on the chunks beyond fp32 sums over the tokens
    a, b = blk.router_weight.grad, chunked.router_weight.grad
    assert float((a - b).norm() / a.norm()) < 1e-2
    # tokens only see experts of their best groups
    idx, _ = block.route(hidden.reshape(-1, H), blk.router_weight, top_k=k, correction_bias=blk.e_score_correction_bias,
                         num_groups=4, top_groups=2, route_scale=1.5)
    assert ((idx // 2).sort(dim=1).values.unique(dim=1).shape[1]) <= 2
    # one token, as in generation
    with torch.no_grad():
        one = blk(hidden[:1, :1])
        assert torch.allclose(one.float(), blk(hidden)[:1, :1].float(), rtol=2 ** -6, atol=1e-2)


def test_training_step_of_the_layer_in_a_graph():
    """Forward and backward captured together replay on new inputs, with an eager step of other leaves in between."""
    dev = _dev()
    from mirai_b200 import experts as ex
    from mirai_b200 import ops
    E, T, k, H, I = 4, 200, 2, 128, 64
    m = ex.B200GroupedExperts.from_empty(num_experts=E, quant_format="mxfp4")
    for key, (o, i) in {"w1": (I, H), "w3": (I, H), "w2": (H, I)}.items():
        m.load_dense_weight(key, weight(E, o, i, dev, o + len(key)))
    g = torch.Generator().manual_seed(5)
    xs = [rows(T, H, dev, i) for i in range(3)]
    idx = torch.rand(T, E, generator=g).topk(k, dim=1).indices.to(dev)
    score = torch.rand(T, k, generator=g).to(dev)
    grad = torch.randn(T, H, generator=g).bfloat16().to(dev)

    def step_(x):
        leaf = x.detach().requires_grad_()
        out = m.run_direct_routed(leaf, score, idx)
        return out, torch.autograd.grad(out, leaf, grad)[0]

    want = [tuple(t.detach().clone() for t in step_(x)) for x in xs]
    static = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dx = step_(static)
    for i, x in enumerate(xs):
        static.copy_(x)
        graph.replay()
        eager = step_(xs[0])
        assert torch.equal(out, want[i][0]) and torch.equal(dx, want[i][1])
        assert torch.equal(eager[1], want[0][1])
    ops.check_device()
