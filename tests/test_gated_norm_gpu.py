"""The gated residual norm on the GPU against float64, and chained with the FP4 layers as a block uses them."""

import numpy as np
import pytest
import torch

from oracle import fp4 as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def generator(seed):
    return torch.Generator().manual_seed(seed)


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def h_tolerance(h, u, centre, factor, add, dtype):
    """Bound of |h_gpu - h|, in halves of a float32 step (2^-24). u takes the mean's rounding (2: the sum's and the
    division's) and the subtraction's through the root, then relative the mean square's (2, of which 1 reaches the
    root; the subtraction's once more), eps's sum, the root's and the division's: 8 in all; each affine and modulation
    step rounds what it has (4), h once to its type."""
    step = 2.0 ** -24
    du = 2 * step * centre + 8 * step * np.abs(u)
    return 1.01 * (np.abs(factor) * du + 4 * step * (np.abs(u * factor) + np.abs(add)) + HALF_STEP[dtype] * np.abs(h)) + 2.0 ** -25


CASES = [(1, 8, 1), (1, 1024, 1), (3, 1032, 3), (5, 2048, 1), (4, 2080, 2), (7, 3072, 1), (6, 4096, 3), (2, 5120, 1),
         (2, 8192, 2), (3, 16384, 1)]


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("M,K,groups", CASES)
def test_gated_norm_against_float64(kind, M, K, groups):
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    g = generator(K + M)
    mod = torch.randn(groups, 6, K, generator=g).to(DEV) * 0.3  # strided rows, as modulation.chunk(6) gives them
    gate, shift, scale = mod[:, 2], mod[:, 0], mod[:, 1]
    weight, bias = (1 + 0.1 * torch.randn(K, generator=g)).to(DEV), torch.randn(K, generator=g).to(DEV)
    rows = lambda t: np.repeat(f64(t), M // groups, axis=0)  # noqa: E731
    for tx, ty in ((torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                   (torch.bfloat16, torch.bfloat16)):
        x = (2 * torch.randn(M, K, generator=g) + 0.5).to(tx).to(DEV)
        y = torch.randn(M, K, generator=g).to(ty).to(DEV)
        for out in (torch.bfloat16, torch.float16, torch.float32):
            for full in (True, False):
                kw = dict(weight=weight, bias=bias, shift=shift, scale=scale) if full else {}
                xn, h = gated_norm(x, y, gate if full else None, kind=kind, out=out, **kw)
                assert xn.dtype == tx and h.dtype == out
                want = f64(x) + (rows(gate) if full else 1.0) * f64(y)
                # the product rounded, then the sum (2^-24 each), then the stream's type
                branch = np.abs(want - f64(x))
                assert (np.abs(f64(xn) - want) <= 1.01 * HALF_STEP[tx] * np.abs(want) + 2.0 ** -24 * (
                    np.abs(want) + 1.01 * branch)).all()
                stored = f64(xn)  # what the kernel normalizes is what it stored
                _, u = oracle.norm(stored, kind=kind)
                factor = f64(weight) * (1 + rows(scale)) if full else np.ones((M, K))
                add = f64(bias) * (1 + rows(scale)) + rows(shift) if full else np.zeros((M, K))
                err = np.abs(f64(h) - (u * factor + add))
                spread = np.sqrt(((stored - stored.mean(-1, keepdims=True)) ** 2).mean(-1, keepdims=True) + 1e-6)
                centre = np.abs(stored.mean(-1, keepdims=True)) / spread if kind == "layer" else 0.0
                loose = np.abs(f64(bias) * (1 + rows(scale))) + np.abs(rows(shift)) if full else add
                tol = h_tolerance(u * factor + add, u, centre, factor, loose, out)
                assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("out", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M,K", [(1, 32), (3, 96), (130, 288), (2, 1024), (2, 1056), (5, 3072), (2, 3104), (2, 4128), (1, 16384)])
def test_fp4_output_is_the_quantized_float32_output(out, M, K):
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    from wan_dit_lab_b200.quantization import fp4
    g = generator(K)
    x, y = torch.randn(M, K, generator=g).to(DEV), torch.randn(M, K, generator=g).to(DEV)
    t = torch.tensor([0.011], device=DEV) if out == "nvfp4" else None
    x1, h = gated_norm(x, y, scale=y[0], out=torch.float32)
    x2, rows = gated_norm(x, y, scale=y[0], out=out, tensor_scale=t)
    want = fp4.quantize_rows(h, out, t)
    assert torch.equal(x1, x2) and torch.equal(rows.codes, want.codes)
    blocks = K // fp4.BLOCK[out]
    assert torch.equal(fp4.untile_scales(rows.scales, M, blocks), fp4.untile_scales(want.scales, M, blocks))
    padded = -(-blocks // 4) * 4
    assert not fp4.untile_scales(rows.scales, M, padded)[:, blocks:].any()


def test_without_a_branch_in_place_and_strided():
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    g = generator(5)
    wide = torch.randn(9, 1100, generator=g).to(DEV)
    x = wide[:, 4:260]
    same, h = gated_norm(x, out=torch.float32)
    assert same is x
    ref = gated_norm(x.contiguous(), out=torch.float32)[1]
    assert torch.equal(h, ref)
    assert torch.equal(gated_norm(wide[:, 1:257], out=torch.float32)[1],  # misaligned rows are copied
                       gated_norm(wide[:, 1:257].contiguous(), out=torch.float32)[1])
    y = torch.randn(9, 256, generator=g).to(DEV)
    gate = torch.randn(256, generator=g).to(DEV)
    before = wide.clone()
    xn, hn = gated_norm(x, y, gate, out=torch.float32)
    x2, h2 = gated_norm(x, y, gate, out=torch.float32, inplace=True)
    assert x2 is x and torch.equal(x, xn) and torch.equal(hn, h2)
    assert torch.equal(wide[:, :4], before[:, :4]) and torch.equal(wide[:, 260:], before[:, 260:])
    for per in (1, 3):  # one modulation row beside grouped ones
        a = gated_norm(x, y, gate, shift=y[:9 // per], out=torch.float32)
        b = gated_norm(x, y, gate.expand(9 // per, 256), shift=y[:9 // per], out=torch.float32)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    empty = gated_norm(x[:0], y[:0], gate)
    assert empty[0].shape == empty[1].shape == (0, 256)


def test_a_block_of_layers_in_fp4():
    """Norm into the feed forward's operand, the feed forward onto the stream, the next norm: as a block runs them,
    captured and replayed, against the same steps in float64 from the same codes."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    from wan_dit_lab_b200.quantization import fp4
    g = generator(6)
    M, D, H = 150, 256, 544
    W1, W2 = 0.05 * torch.randn(H, D, generator=g), 0.05 * torch.randn(D, H, generator=g)
    b1, b2 = 0.1 * torch.randn(H, generator=g).to(DEV), 0.1 * torch.randn(D, generator=g).to(DEV)
    mlp = fp4.PackedFp4GeluMLP(fp4.PackedFp4Linear(**fp4.quantize(W1.to(DEV), b1)),
                               fp4.PackedFp4Linear(**fp4.quantize(W2.to(DEV), b2)))
    mod = (0.3 * torch.randn(3, 3, D, generator=g)).to(DEV)
    x, y = torch.randn(M, D, generator=g).to(DEV), torch.randn(M, D, generator=g).to(DEV)

    def block(x, y):
        x, rows = gated_norm(x, y, mod[:, 2], shift=mod[:, 0], scale=mod[:, 1], out="nvfp4")
        z = mlp(rows, residual=x, gate=mod[:, 2])
        return (x, rows, z) + gated_norm(z, kind="rms", out=torch.float32)

    first = block(x, y)
    graph = torch.cuda.CUDAGraph()
    xs, ys = x.clone(), y.clone()
    with torch.cuda.graph(graph):
        replayed = block(xs, ys)
    xs.copy_(2 * x), ys.copy_(-y)
    graph.replay()
    again = block(2 * x, -y)
    for a, b in zip(replayed, again):
        a, b = (a, b) if torch.is_tensor(a) else (a.codes, b.codes)
        assert torch.equal(a, b)
    x1, rows, z, z_again, h = first
    assert z_again is z
    rowwise = lambda t: np.repeat(f64(t), M // 3, axis=0)  # noqa: E731
    a = f64(fp4.dequantize_rows(rows, torch.float32))
    value = lambda layer: f64(fp4.dequantize_rows(layer.rows(), torch.float32))  # noqa: E731
    hid = oracle.gelu(a @ value(mlp.fc1).T + f64(b1))
    hq = oracle.rounded(hid.astype(np.float32), "nvfp4").astype(np.float64)
    want = f64(x1) + rowwise(mod[:, 2]) * (hq @ value(mlp.fc2).T + f64(b2))
    # a hidden value next to a border may take the neighbouring code: at most a whole step (a third of its magnitude)
    # of one value among a row's 544, and few rows have one
    err = np.abs(f64(z) - want)
    one = (np.abs(hq).max() / 3) * np.abs(value(mlp.fc2)).max() * np.abs(f64(mod)).max()
    assert err.max() <= 2 * one and (err > 1e-4 * np.abs(want).max()).mean() < 0.02
    _, u = oracle.norm(f64(z), kind="rms")
    assert np.abs(f64(h) - u).max() <= 2.0 ** -24 * 128 * np.abs(u).max()
    assert _native.device_error() == 0


@pytest.mark.parametrize("out", ["nvfp4", "mxfp4", torch.float32])
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_bad_and_extreme_rows_stay_their_own(kind, out):
    """Rows with a NaN, an infinity, only zeros, squares beyond float32, and subnormal values, between ordinary ones (a CTA
    takes neighbouring rows): the ordinary rows keep their bits, the bad ones are what the formula makes of them."""
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    from wan_dit_lab_b200.quantization import fp4
    g = generator(90)
    M, K = 700, 1056
    x, y = torch.randn(M, K, generator=g).to(DEV), torch.randn(M, K, generator=g).to(DEV)
    gate, shift, scale = torch.randn(3, K, generator=g).to(DEV)
    value = lambda h: h if torch.is_tensor(h) else fp4.dequantize_rows(h, torch.float32)  # noqa: E731
    want_x, h = gated_norm(x, y, gate, shift=shift, scale=scale, kind=kind, out=out)
    want = value(h)
    bad = torch.tensor([1, 2, 340, 341, 699], device=DEV)
    x[1, 7], x[2, 900] = float("nan"), float("inf")
    x[340], y[340] = 0.0, 0.0
    x[341], y[341] = 1e30, 0.0
    x[341, ::2] = -1e30
    x[699], y[699] = 1e-42, 0.0
    got_x, h = gated_norm(x, y, gate, shift=shift, scale=scale, kind=kind, out=out)
    got = value(h)
    rest = torch.ones(M, dtype=torch.bool, device=DEV)
    rest[bad] = False
    assert torch.equal(got_x[rest], want_x[rest]) and torch.equal(got[rest], want[rest])
    only_shift = value(gated_norm(torch.zeros(1, K, device=DEV), shift=shift, kind=kind, out=out)[1])[0]
    assert got[1].isnan().all()  # the row's statistics are
    if kind == "layer":
        assert got[2].isnan().all()
    else:  # an infinite root: x / inf = 0, inf / inf = NaN (in FP4 the block's scale)
        block = {"nvfp4": 16, "mxfp4": 32}.get(out, 1)
        hit = torch.arange(K, device=DEV) // block == 900 // block
        assert got[2, hit].isnan().all() and torch.equal(got[2, ~hit], only_shift[~hit])
    # zeros; 1e60 overflows to an infinite root; the subnormal row's root is sqrt(eps): 1e-42 / 1e-3 is 0 to any format here
    for row in (340, 341):
        assert torch.equal(got[row], only_shift)
    assert torch.allclose(got[699], only_shift, rtol=0, atol=0 if isinstance(out, str) else 1e-30)


@pytest.mark.parametrize("K", [12288, 16384])
def test_sums_over_long_rows_are_not_rounded_on_the_way(K):
    """Four values, each over a quarter of the row, whose float32 sums from left to right would round down three times,
    while the row's mean 1 + 2^-23 is a float32 number: the values' distances from it come out exactly, whichever columns
    they lie in."""
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    step = 2.0 ** -23
    quarter = torch.tensor([1 + step, 1.0, 1 + step, 1 + 2 * step], dtype=torch.float64)
    for x in (quarter.repeat_interleave(K // 4), quarter.repeat_interleave(8).repeat(K // 32), quarter.repeat(K // 4)):
        h = gated_norm(x.float().to(DEV)[None], eps=0.0, out=torch.float32)[1][0].double().cpu()
        want = (x - (1 + step)) / (step / 2 ** 0.5)  # the root of the mean square, (0 + 1 + 0 + 1) / 4 steps
        # the squares and their sums are exact; the root and the quotient round once each
        assert ((h - want).abs() <= 2.0 ** -24 * 2.02 * want.abs()).all()


def statistics_case(data, K, g):
    x = torch.randn(3, K, generator=g)
    if data == "offset":
        return x + 1000.0
    if data == "outliers":  # far larger values that cancel, an ordinary mean
        x[:, ::8] = 30000.0 * torch.sign(torch.randn(3, -(-K // 8), generator=g))
        return x
    return 1000.0 * x - (1000.0 * x).double().mean(-1, keepdim=True).float()  # the mean cancels to nearly nothing


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("data", ["offset", "outliers", "centred"])
@pytest.mark.parametrize("K", [1024, 3072, 4096, 5120, 8192, 16384])
def test_statistics_of_rows_far_from_standard(kind, data, K):
    """Bound, in halves of a float32 step s = 2^-24. The float32 sums of 64 columns (8 from 4097 columns on) round 6 (3)
    times, relative to the magnitudes of what they add, the sum and its division once each: the mean's error is e <= (6
    mean|x| + 2 |mean|) s. It shifts every value; of the mean square it changes e^2 alone, the values' sum being zero. The
    subtraction rounds once; the mean square takes that twice, its squares' and sums' roundings (7, or 4) and its own
    (2), eps's sum one more, half of which reach the root; the root and the quotient round once each."""
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    s, sums = 2.0 ** -24, 6 if K <= 4096 else 3
    x = statistics_case(data, K, generator(K))
    h = f64(gated_norm(x.to(DEV), kind=kind, out=torch.float32)[1])
    v = f64(x)
    _, u = oracle.norm(v, kind=kind)
    e = sub = np.zeros((3, 1))
    if kind == "layer":
        mean = v.mean(-1, keepdims=True)
        root = np.sqrt(((v - mean) ** 2).mean(-1, keepdims=True) + 1e-6)
        e, sub = (sums * np.abs(v).mean(-1, keepdims=True) + 2 * np.abs(mean)) * s / root, 1
    relative = (sub + (2 * sub + sums + 1 + 2 + 1) / 2 + 2) * s + e ** 2 / 2
    assert (np.abs(h - u) <= 1.01 * (e + relative * np.abs(u))).all(), float((np.abs(h - u) / (e + relative * np.abs(u))).max())
