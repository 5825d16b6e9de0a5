"""The FP4 operators on the GPU against the oracle: the quantizers bit for bit, the products within the bound of their
float32 accumulation, the feed forward step by step, non-finite values, strides, streams, graphs."""

import numpy as np
import pytest
import torch

from oracle import fp4 as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = ["nvfp4", "mxfp4"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def generator(seed):
    return torch.Generator().manual_seed(seed)


def activations(M, K, seed, dtype=torch.float32):
    g = generator(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(0.7 * torch.randn(K, generator=g))
    return x.to(dtype).to(DEV)


def weight_rows(N, K, fmt, seed):
    """(Rows on the GPU, its float64 values)."""
    from wan_dit_lab_b200.quantization import fp4
    W = torch.randn(N, K, generator=generator(seed)) * 0.05
    t = W.abs().max().reshape(1) / 2688 if fmt == "nvfp4" else None
    codes, byte = oracle.encode(W.numpy(), fmt, None if t is None else t.numpy()[0])
    rows = fp4.Rows(torch.from_numpy(oracle.pack(codes)).to(DEV), fp4.tile_scales(torch.from_numpy(byte)).to(DEV), fmt,
                    None if t is None else t.to(DEV))
    values = oracle.decode(codes, byte, fmt).astype(np.float64)
    return rows, values * (1.0 if t is None else float(t[0]))


def product_tolerance(a, w, y, dtype):
    """Bound of |y_gpu - y| for y = a w^T (+ bias): one truncation of the running sum, at most 2^-23 of the terms'
    magnitudes, for each of the K / 64 MMA steps and for the four K = 16 parts that a step may add one by one; the
    epilogue rounds the scaled sum, the bias sum and the two tensor scales' products (4 halves of a float32 step), and
    the result once to its type (float16 subnormals: half of 2^-24)."""
    K = a.shape[1]
    terms = np.abs(a) @ np.abs(w).T
    acc = terms * (K / 16 + 4) * 2.0 ** -23
    return acc + (np.abs(y) + acc) * (4 * 2.0 ** -24 + 1.01 * HALF_STEP[dtype]) + (2.0 ** -25 if dtype == torch.float16 else 0)


def check_rows(rows, x, fmt, t):
    from wan_dit_lab_b200.quantization import fp4
    codes, byte = oracle.encode(x, fmt, t)
    got = fp4.untile_scales(rows.scales, *byte.shape).cpu().numpy()
    np.testing.assert_array_equal(got, byte)
    np.testing.assert_array_equal(oracle.unpack(rows.codes.cpu().numpy()), codes)
    return codes, byte


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 32), (3, 96), (33, 64), (128, 256), (129, 1056), (300, 4128)])
def test_quantize_rows_equals_the_oracle(fmt, dtype, M, K):
    from wan_dit_lab_b200.quantization import fp4
    x = activations(M, K, M * K, dtype)
    for t in (None, 0.0123) if fmt == "nvfp4" else (None,):
        ts = None if t is None else torch.tensor([t], device=DEV)
        rows = fp4.quantize_rows(x, fmt, ts)
        t32 = None if t is None else np.float32(t)
        codes, byte = check_rows(rows, x.float().cpu().numpy(), fmt, t32)
        for out in DTYPES:
            want = torch.from_numpy(oracle.decode(codes, byte, fmt, t32)).to(out)
            assert torch.equal(fp4.dequantize_rows(rows, out).cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_rows_on_ties_and_extremes(fmt):
    """Every border of the codes, blocks of zeros, signed zeros, subnormals, the largest finite numbers, powers of two
    on either side of the scales' own borders, tensor scales far from 1."""
    from wan_dit_lab_b200.quantization import fp4
    borders = [0, -0.0, 0.25, -0.25, 0.5, 0.75, -0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, -2.5, 3, 3.5, -3.5, 4, 5, -5, 5.5, 6]
    base = torch.tensor((borders + [0.249, 0.251, 2.499, 2.501, 4.999, 5.001, 3.0, -6.0, 1.2, 0.1])[:32])
    near = torch.nextafter(base, torch.tensor(10.0))
    rows = [base, near, torch.nextafter(base, torch.tensor(-10.0)), torch.zeros(32), -torch.zeros(32)]
    for p in (-149, -140, -126, -125, -124, -60, -30, -10, -9, -3, 1, 7, 8, 9, 11, 12, 60, 120, 125):
        rows.append(torch.ldexp(base, torch.tensor(p)))
        rows.append(torch.ldexp(near, torch.tensor(p)))
    rows.append(torch.full((32,), torch.finfo(torch.float32).max))
    x = torch.stack(rows).float()
    x = x.clamp(-torch.finfo(torch.float32).max, torch.finfo(torch.float32).max)
    for t in (None, 1.0, 2.0 ** -70, 3e-5, 1e30) if fmt == "nvfp4" else (None,):
        ts = None if t is None else torch.tensor([t], device=DEV)
        check_rows(fp4.quantize_rows(x.to(DEV), fmt, ts), x.numpy(), fmt, None if t is None else np.float32(t))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_blocks_become_nan_and_stay_in_their_rows(fmt, bad):
    from wan_dit_lab_b200.quantization import fp4
    x = activations(5, 128, 3)
    x[2, 37] = bad
    rows = fp4.quantize_rows(x, fmt)
    check_rows(rows, x.cpu().numpy(), fmt, None)
    block = oracle.BLOCK[fmt]
    values = fp4.dequantize_rows(rows, torch.float32)
    inside = torch.zeros_like(values, dtype=torch.bool)
    inside[2, 37 // block * block:37 // block * block + block] = True
    assert torch.equal(values.isnan(), inside)
    w, _ = weight_rows(40, 128, fmt, 4)
    for M in (5, 200):  # few rows and many
        x2 = activations(M, 128, 5)
        x2[2, 37] = bad
        nan = fp4.fp4_linear(x2, w, dtype=torch.float32).isnan()
        assert nan[2].all() and not nan[torch.arange(M, device=DEV) != 2].any()
    wide = activations(40, 128, 6)
    wide[7, 100] = bad
    nan = fp4.fp4_linear(activations(9, 128, 7), fp4.quantize_rows(wide, fmt), dtype=torch.float32).isnan()
    assert nan[:, 7].all() and nan.sum() == 9


@pytest.mark.parametrize("fmt", FORMATS)
def test_strided_and_misaligned_inputs(fmt):
    from wan_dit_lab_b200.quantization import fp4
    wide = activations(20, 512, 8, torch.bfloat16)
    for x in (wide[:, 64:320], wide[:, 3:259], wide[::2, :256], wide.t()[:256, :].t(), wide.flatten()[1:1 + 15 * 512].view(15, 512)):
        check_rows(fp4.quantize_rows(x, fmt), x.float().cpu().numpy(), fmt, None)
    assert fp4.quantize_rows(wide[:0], fmt).shape == (0, 512)


SHAPES = [(1, 1, 32), (1, 130, 96), (2, 7, 64), (16, 256, 288), (17, 520, 256), (31, 64, 1056), (64, 300, 512),
          (65, 33, 2048), (127, 257, 320), (128, 128, 4128), (129, 512, 768), (300, 1000, 544), (513, 776, 1312), (300, 130, 4096),
          (70, 1030, 4160), (2100, 136, 256)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_against_float64(fmt, M, N, K):
    from wan_dit_lab_b200.quantization import fp4
    x = activations(M, K, M + N + K, torch.bfloat16)
    w, wv = weight_rows(N, K, fmt, M * 7 + N)
    bias = torch.randn(N, generator=generator(1))
    t = np.float32(0.37) if fmt == "nvfp4" and K % 64 else None
    a = oracle.rounded(x.float().cpu().numpy(), fmt, t).astype(np.float64)
    ts = None if t is None else torch.tensor([t], device=DEV)
    y = a @ wv.T + bias.double().numpy()
    for dtype in DTYPES:
        got = fp4.fp4_linear(x, w, bias.to(DEV), input_scale=ts, dtype=dtype)
        assert got.dtype == dtype and got.shape == (M, N)
        err = np.abs(got.double().cpu().numpy() - y)
        assert (err <= product_tolerance(a, wv, y, dtype)).all(), float((err / product_tolerance(a, wv, y, dtype)).max())
    # the same from an input quantized before, without a bias, and once more: every call gives the same bits
    rows = fp4.quantize_rows(x, fmt, ts)
    plain = fp4.fp4_linear(rows, w, dtype=torch.float32)
    assert (np.abs(plain.double().cpu().numpy() - a @ wv.T) <= product_tolerance(a, wv, a @ wv.T, torch.float32)).all()
    assert torch.equal(plain, fp4.fp4_linear(x, w, input_scale=ts, dtype=torch.float32))


@pytest.mark.parametrize("M,N,K,groups", [(1, 40, 64, 1), (6, 96, 128, 3), (66, 130, 256, 2), (300, 264, 512, 1), (264, 520, 96, 8),
                                            (96, 260, 4096, 3), (516, 516, 320, 2)])
def test_gated_residual(M, N, K, groups):
    from wan_dit_lab_b200.quantization import fp4
    x = activations(M, K, 9)
    w, wv = weight_rows(N, K, "nvfp4", 10)
    g = generator(11)
    residual, gate = torch.randn(M, N, generator=g).to(DEV), torch.randn(groups, N, generator=g).to(DEV)
    bias = torch.randn(N, generator=g).to(DEV)
    a = oracle.rounded(x.cpu().numpy(), "nvfp4").astype(np.float64)
    y = a @ wv.T + bias.double().cpu().numpy()
    tol = product_tolerance(a, wv, y, torch.float32)
    for gt in (None, gate, gate[0]):
        rows = np.ones((M, N)) if gt is None else np.repeat(
            gt.double().cpu().numpy().reshape(-1, N), M // (groups if gt.ndim == 2 else 1), axis=0)
        want = residual.double().cpu().numpy() + rows * y
        got = fp4.fp4_linear(x, w, bias, residual=residual, gate=gt)
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= np.abs(rows) * tol + 2.0 ** -24 * 1.01 * np.abs(want)).all()
        wide = torch.full((M, N + 6), 7.0, device=DEV)  # a strided, misaligned stream, updated in place
        stream = wide[:, 1:N + 1]
        stream.copy_(residual)
        assert fp4.fp4_linear(x, w, bias, residual=stream, gate=gt, out=stream) is stream
        assert torch.equal(stream, got)
        assert (wide[:, 0] == 7).all() and (wide[:, N + 1:] == 7).all()


def hidden_of(x, w, bias, fmt, t):
    """The hidden layer as wdl_fp4_gemm_gelu writes it."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    M, (H, K) = x.shape[0], w.shape
    rows = fp4.Rows(torch.empty(M, H // 2, dtype=torch.uint8, device=DEV),
                    torch.zeros(fp4.scale_tiles(M, H, fmt), dtype=torch.uint8, device=DEV), fmt, t)
    _native.check(_native.lib().wdl_fp4_gemm_gelu(
        x._operand, w._operand, _native.ptr(bias), M, H, K, _native.ptr(t),
        rows._codes_ptr, rows._scales_ptr, _native.stream()))
    return rows


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,H,N", [(1, 64, 96, 40), (19, 256, 544, 128), (130, 512, 288, 264), (257, 96, 1024, 33), (140, 4128, 352, 64)])
def test_gelu_mlp(fmt, M, K, H, N):
    from wan_dit_lab_b200.quantization import fp4
    x = activations(M, K, 12, torch.bfloat16)
    w1, v1 = weight_rows(H, K, fmt, 13)
    w2, _ = weight_rows(N, H, fmt, 14)
    g = generator(15)
    b1, b2 = torch.randn(H, generator=g).to(DEV), torch.randn(N, generator=g).to(DEV)
    t = torch.tensor([0.02], device=DEV) if fmt == "nvfp4" else None
    rows = fp4.quantize_rows(x, fmt)
    hidden = hidden_of(rows, w1, b1, fmt, t)
    # the hidden layer: the scale lies between the rounded scales of the largest magnitude's bounds, each code between
    # the codes of its value's bounds at that scale
    a = oracle.rounded(x.float().cpu().numpy(), fmt).astype(np.float64)
    y = a @ v1.T + b1.double().cpu().numpy()
    h = oracle.gelu(y)
    # GELU's slope is at most 1.13; its own float32 steps stay within 16 half steps of |y|
    tol = 1.13 * product_tolerance(a, v1, y, torch.float32) + 16 * 2.0 ** -24 * np.abs(y)
    block = oracle.BLOCK[fmt]
    t32 = np.float32(1) if t is None else np.float32(0.02)
    byte = fp4.untile_scales(hidden.scales, M, H // block).cpu().numpy()
    top = np.abs(h).reshape(M, -1, block).max(-1)
    slack = tol.reshape(M, -1, block).max(-1)
    low, high = (oracle.scale_bytes(np.maximum(v, 0).astype(np.float32), fmt, None if t is None else t32)
                 for v in (top - slack, top + slack))
    assert ((low <= byte) & (byte <= high)).all()
    d = np.repeat(oracle.scale_values(byte, fmt).astype(np.float64), block, axis=1) * float(t32)
    got = oracle.decode(oracle.unpack(hidden.codes.cpu().numpy()), byte, fmt).astype(np.float64) * float(t32)
    value = lambda q: np.where(q < 0, -1, 1) * oracle.E2M1[oracle._nearest(oracle.E2M1, np.abs(q))] * d  # noqa: E731
    eps = 1 + 2.0 ** -22
    assert (got >= value((h - tol) / d * np.where(h > tol, 1 / eps, eps)) - 1e-30).all()
    assert (got <= value((h + tol) / d * np.where(h > -tol, eps, 1 / eps)) + 1e-30).all()
    # and the second product of exactly those rows, into every kind of output
    for dtype in DTYPES:
        want = fp4.fp4_linear(hidden, w2, b2, dtype=dtype)
        assert torch.equal(fp4.fp4_gelu_mlp(x, w1, b1, w2, b2, hidden_scale=t, dtype=dtype), want)
    residual, gate = torch.randn(M, N, generator=g).to(DEV), torch.randn(N, generator=g).to(DEV)
    want = fp4.fp4_linear(hidden, w2, b2, residual=residual, gate=gate)
    assert torch.equal(fp4.fp4_gelu_mlp(x, w1, b1, w2, b2, hidden_scale=t, residual=residual, gate=gate), want)


def test_rows_do_not_depend_on_their_neighbours():
    """A row's result is the same bits whatever else is in the call with the same kernel, and rows of the scales' last
    tile that no row owns are left as they were."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    x = activations(150, 256, 16, torch.bfloat16)
    tiles = torch.full(fp4.scale_tiles(150, 256, "nvfp4"), 0xAB, dtype=torch.uint8, device=DEV)
    codes = torch.empty(150, 128, dtype=torch.uint8, device=DEV)
    _native.check(_native.lib().wdl_fp4_quantize_rows(x.data_ptr(), _native.BF16, 256, 150, 256, _native.NVFP4, None,
                                                      codes.data_ptr(), tiles.data_ptr(), _native.stream()))
    assert (fp4.untile_scales(tiles, 256, 16)[150:] == 0xAB).all()
    w, _ = weight_rows(512, 256, "nvfp4", 17)
    whole = fp4.fp4_linear(fp4.Rows(codes, tiles, "nvfp4"), w, dtype=torch.float32)
    assert torch.equal(whole[:140], fp4.fp4_linear(x[:140], w, dtype=torch.float32))


def test_leading_dimensions_and_modules():
    from wan_dit_lab_b200.quantization import fp4
    g = generator(18)
    W1, W2 = torch.randn(96, 64, generator=g).to(DEV), torch.randn(64, 96, generator=g).to(DEV)
    b1, b2 = torch.randn(96, generator=g).to(DEV), torch.randn(64, generator=g).to(DEV)
    x = activations(6, 64, 19).view(2, 3, 64)
    for fmt in FORMATS:
        p1, p2 = fp4.quantize(W1, b1, fmt), fp4.quantize(W2, b2, fmt)
        fc1, fc2 = fp4.PackedFp4Linear(**p1), fp4.PackedFp4Linear(**p2)
        assert fc1.fmt == fmt
        t = None if p1["tensor_scale"] is None else p1["tensor_scale"].cpu().numpy()[0]
        codes, byte = oracle.encode(W1.cpu().numpy(), fmt, t)
        np.testing.assert_array_equal(p1["scales"].cpu().numpy(), byte)
        np.testing.assert_array_equal(p1["codes"].cpu().numpy(), oracle.pack(codes))
        y = fc1(x)
        assert y.shape == (2, 3, 96) and torch.equal(y.view(6, 96), fc1(x.view(6, 64)))
        z = fp4.PackedFp4GeluMLP(fc1, fc2)(x, residual=x, gate=b2)
        assert z.shape == x.shape and torch.equal(
            z.view(6, 64), fp4.fp4_gelu_mlp(x.view(6, 64), fc1.rows(), b1, fc2.rows(), b2, residual=x.view(6, 64), gate=b2))
        zero = fp4.quantize(torch.zeros(3, 32, device=DEV), None, fmt)
        assert not fp4.dequantize_rows(fp4.PackedFp4Linear(**zero).rows()).any()


def test_other_streams_and_graphs():
    from wan_dit_lab_b200.quantization import fp4
    w1, _ = weight_rows(544, 256, "nvfp4", 20)
    w2, _ = weight_rows(256, 544, "nvfp4", 21)
    inputs = [activations(M, 256, 22 + M) for M in (3, 200)]
    want = [[fp4.fp4_gelu_mlp(x * k, w1, None, w2, None, residual=x * k) for k in (1, 2)] for x in inputs]
    side = torch.cuda.Stream()
    for x, (once, twice) in zip(inputs, want):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = fp4.fp4_gelu_mlp(x, w1, None, w2, None, residual=x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, once)
    graphs = []
    for x in inputs:  # two graphs, captured one after the other and replayed in turn
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp4.fp4_gelu_mlp(static, w1, None, w2, None, residual=static)
        graphs.append((graph, static, out))
    for k in (0, 1, 0):
        for x, (graph, static, out), w in zip(inputs, graphs, want):
            static.copy_(x * (k + 1))
            graph.replay()
            assert torch.equal(out, w[k])
    from wan_dit_lab_b200 import _native
    assert _native.device_error() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [3, 40, 150])
@pytest.mark.parametrize("N", [31, 258, 261])
def test_outputs_that_begin_anywhere(fmt, M, N):
    """Rows whose address and stride are multiples of their type's size only, against the aligned call, and nothing
    written beside them."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    K = 192
    x = fp4.quantize_rows(activations(M, K, 30), fmt)
    w, _ = weight_rows(N, K, fmt, 31)
    bias = torch.randn(N + 1, generator=generator(32)).to(DEV)[1:]
    for dtype in DTYPES:
        want = fp4.fp4_linear(x, w, bias, dtype=dtype)
        for ld, at in ((N + 1, 1), (N + 3, 2), ((N + 7) // 8 * 8, 0)):
            wide = torch.full((M + 1, ld), 5.0, dtype=dtype, device=DEV)
            out = wide.view(-1)[at:]
            _native.check(_native.lib().wdl_fp4_gemm(x._operand, w._operand, bias.data_ptr(), M, N, K, out.data_ptr(),
                                                     _native.DTYPE_CODE[dtype], ld, _native.stream()))
            rows = out[:M * ld].view(M, ld) if at + M * ld <= wide.numel() else None
            assert torch.equal(rows[:, :N], want)
            untouched = torch.ones_like(wide, dtype=torch.bool)
            untouched.view(-1)[at:][:M * ld].view(M, ld)[:, :N] = False
            assert (wide[untouched] == 5).all()


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows are quantized, restored and multiplied as the same rows alone."""
    from wan_dit_lab_b200.quantization import fp4
    M, K = 66_000, 32_768
    x = torch.empty(M, K, dtype=torch.bfloat16, device=DEV)
    tail = activations(300, K, 33, torch.bfloat16)
    x[:-300] = 1.0
    x[-300:] = tail
    rows, alone = fp4.quantize_rows(x, "nvfp4"), fp4.quantize_rows(tail, "nvfp4")
    assert torch.equal(rows.codes[-300:], alone.codes)
    end = 512 - -M % 128  # of the rows among the last four tiles'
    assert torch.equal(fp4.untile_scales(rows.scales[-4:], 512, K // 16)[end - 300:end],
                       fp4.untile_scales(alone.scales, 300, K // 16))
    del x
    values = fp4.dequantize_rows(rows)
    # a block of ones: scale E4M3(1 / 6) = 0.171875, codes E2M1(5.82) = 6, values 1.03125
    assert torch.equal(values[-300:], fp4.dequantize_rows(alone)) and (values[0] == 1.03125).all()
    del values
    w, _ = weight_rows(512, K, "nvfp4", 34)
    assert torch.equal(fp4.fp4_linear(rows, w)[-300:], fp4.fp4_linear(alone, w))
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    x = torch.empty(M, K // 2, dtype=torch.bfloat16, device=DEV)  # [M, 16384] in float32 output: 2^32 bytes
    x[:-300] = 0.5
    x[-300:] = tail[:, :K // 2]
    assert torch.equal(gated_norm(x, out=torch.float32)[1][-300:], gated_norm(tail[:, :K // 2], out=torch.float32)[1])


def test_calls_on_two_streams_at_once():
    """Nothing is shared between calls: two streams with both kernels, many times over."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    w1, _ = weight_rows(1056, 512, "mxfp4", 35)
    w2, _ = weight_rows(512, 1056, "mxfp4", 36)
    xs = [activations(M, 512, 37 + M, torch.bfloat16) for M in (5, 300)]
    want = [fp4.fp4_gelu_mlp(x, w1, None, w2, None, dtype=torch.float32) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (x, stream) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(stream):
                got[i].append(fp4.fp4_gelu_mlp(x, w1, None, w2, None, dtype=torch.float32))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)
    assert _native.device_error() == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_made_just_before(fmt):
    """A weight quantized in the launch before the product's (kernels begin before the one before them has ended)."""
    from wan_dit_lab_b200.quantization import fp4
    for M in (7, 200):
        x = activations(M, 2048, 40, torch.bfloat16)
        W = [torch.randn(1024, 2048, generator=generator(50 + i)).to(DEV) * 0.02 for i in range(4)]
        q = fp4.quantize_rows(x, fmt)
        want = [fp4.fp4_linear(q, fp4.quantize_rows(w, fmt)) for w in W]
        torch.cuda.synchronize()
        for _ in range(5):
            got = []
            for w in W:
                got.append(fp4.fp4_linear(q, fp4.quantize_rows(w, fmt)))  # straight after it
                rows = fp4.quantize_rows(w, fmt)
                got.append(fp4.fp4_linear(x, rows))  # after it and the input's quantization
            for i in range(4):
                assert torch.equal(got[2 * i], want[i]) and torch.equal(got[2 * i + 1], want[i])


def test_handles_are_copied_and_pickled():
    """A copy reads its own memory, not the original's."""
    import copy
    import io
    from wan_dit_lab_b200.quantization import fp4
    x = activations(6, 64, 60)
    w, _ = weight_rows(96, 64, "nvfp4", 61)
    want = fp4.fp4_linear(x, w)
    file = io.BytesIO()
    torch.save(w, file)
    file.seek(0)
    for other in (copy.deepcopy(w), torch.load(file, weights_only=False)):
        assert other.codes.data_ptr() != w.codes.data_ptr() and other.tensor_scale.data_ptr() != w.tensor_scale.data_ptr()
        other.codes.zero_()  # the copy's own
        assert torch.equal(fp4.fp4_linear(x, w), want) and not fp4.fp4_linear(x, other).any()
    assert copy.copy(w).codes is w.codes
    q = fp4.quantize_rows(x)  # (one buffer behind codes and scales)
    assert torch.equal(fp4.fp4_linear(copy.deepcopy(q), w), want)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_weight_with_a_bad_value_keeps_its_other_blocks(bad):
    from wan_dit_lab_b200.quantization import fp4
    W = torch.randn(8, 64, generator=generator(62)).to(DEV)
    good = fp4.quantize(W)
    W[3, 20] = bad
    parts = fp4.quantize(W)
    got = fp4.dequantize_rows(fp4.PackedFp4Linear(**parts).rows(), torch.float32)
    want = fp4.dequantize_rows(fp4.PackedFp4Linear(**good).rows(), torch.float32)
    assert got[3, 16:32].isnan().all()
    want[3, 16:32] = got[3, 16:32] = 0
    # the largest magnitude may have been the one replaced: compare where the tensor scale is the same
    assert torch.isfinite(got).all() and (parts["tensor_scale"] <= good["tensor_scale"]).all()
    if torch.equal(parts["tensor_scale"], good["tensor_scale"]):
        assert torch.equal(got, want)


def test_an_output_that_overlaps_is_refused():
    from wan_dit_lab_b200.quantization import fp4
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    x = activations(9, 64, 63)
    w, _ = weight_rows(64, 64, "mxfp4", 64)
    buffer = torch.randn(10, 128, generator=generator(65)).to(DEV)
    a, b = buffer[:9, :64], buffer[:9, 64:]
    want = fp4.fp4_linear(x, w, residual=a)
    with pytest.raises(ValueError, match="overlap"):
        fp4.fp4_linear(x, w, residual=a, out=buffer[1:, :64])
    with pytest.raises(ValueError, match="overlap"):
        fp4.fp4_gelu_mlp(x, w, None, w, None, residual=a, gate=a[0], out=a)
    assert torch.equal(fp4.fp4_linear(x, w, residual=a, out=b), want) and torch.equal(b, want)
    assert torch.equal(fp4.fp4_linear(x, w, residual=a, out=a), want) and torch.equal(a, want)
    for wrong in (dict(y=buffer[1:, :64]), dict(y=b, gate=a[0]), dict(y=b, shift=buffer[4, 32:96])):
        with pytest.raises(ValueError, match="overlap"):
            gated_norm(a, inplace=True, **wrong)
    for y in (a, b):  # the stream itself, and rows beside its own
        want = gated_norm(a, y, out=torch.float32)
        keep = a.clone()
        got = gated_norm(a, y, out=torch.float32, inplace=True)
        assert torch.equal(a, want[0]) and torch.equal(got[1], want[1])
        a.copy_(keep)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 96, 32), (1, 130, 3104), (3, 40, 96), (16, 200, 1056), (1, 40_000, 2080), (1, 20_000, 8192)])
def test_few_rows_are_quantized_by_their_product(fmt, dtype, M, N, K):
    """The same bits as from rows quantized beforehand: lengths that end inside a stage, more stages than a ring holds
    (wide N leaves K in one part), rows behind the last, non-finite values, a tensor scale, strides."""
    from wan_dit_lab_b200.quantization import fp4
    x = activations(M, K + 16, 70 + M, dtype)[:, :K]
    x[M // 2, K - 20] = 0.0
    x[M - 1, 3] = -0.0
    g = torch.Generator(device=DEV).manual_seed(71)
    w = fp4.quantize_rows(torch.randn(N, K, generator=g, device=DEV) * 0.05, fmt)
    bias = torch.randn(N, generator=g, device=DEV)
    t = (x.float().abs().max() / 2000).reshape(1) if fmt == "nvfp4" and N != 130 else None
    for options in (dict(dtype=torch.float32), dict(dtype=torch.float16), dict(residual=torch.randn(M, N, generator=g, device=DEV))):
        want = fp4.fp4_linear(fp4.quantize_rows(x, fmt, t), w, bias, **options)
        assert torch.equal(fp4.fp4_linear(x, w, bias, input_scale=t, **options), want)
    x[0, K // 2] = float("nan") if M == 16 else float("inf")
    got = fp4.fp4_linear(x, w, bias, input_scale=t)
    assert got[0].isnan().all() and torch.isfinite(got[1:]).all()
    if N % 32 == 0:
        w2 = fp4.quantize_rows(torch.randn(48, N, generator=g, device=DEV) * 0.05, fmt)
        for a in (x, activations(M, K, 72, dtype)):
            want = fp4.fp4_gelu_mlp(fp4.quantize_rows(a, fmt, t), w, bias, w2, None, dtype=torch.float32)
            got = fp4.fp4_gelu_mlp(a, w, bias, w2, None, input_scale=t, dtype=torch.float32)
            assert torch.equal(got.view(torch.int32), want.view(torch.int32))


@pytest.mark.parametrize("M", [1, 16, 17, 300])
def test_a_square_layer_onto_its_own_input(M):
    """x + W x in place: the input is the residual and the output."""
    from wan_dit_lab_b200.quantization import fp4
    x = activations(M, 512, 73)
    w, _ = weight_rows(512, 512, "nvfp4", 74)
    want = fp4.fp4_linear(x.clone(), w, residual=x)
    mlp = fp4.fp4_gelu_mlp(x.clone(), w, None, w, None, residual=x)
    for _ in range(3):
        y, z = x.clone(), x.clone()
        assert fp4.fp4_linear(y, w, residual=y, out=y) is y and torch.equal(y, want)
        assert torch.equal(fp4.fp4_gelu_mlp(z, w, None, w, None, residual=z, out=z), mlp)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_on_and_off_32_byte_boundaries(fmt, dtype):
    """Rows that begin 16 bytes off a 32-byte boundary, or every second one of them, against aligned ones; out in place."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    M, K, lib = 7, 1056, _native.lib()
    step = 16 // torch.empty(0, dtype=dtype).element_size()
    for ld, at in ((K, 0), (K, step), (K + step, 0), (K + 2 * step, step)):
        x = activations(1, M * ld + 64, 75, dtype)[0]
        view = torch.as_strided(x, (M, K), (ld, 1), at)
        rows = fp4.quantize_rows(view, fmt)
        check_rows(rows, view.float().cpu().numpy(), fmt, None)
        want = fp4.dequantize_rows(rows, dtype)
        out = torch.full((M * ld + 64,), 5.0, dtype=dtype, device=DEV)
        _native.check(lib.wdl_fp4_dequantize_rows(rows._codes_ptr, rows._scales_ptr, M, K, fp4.FORMAT_CODE[fmt], None,
                                                  out.data_ptr() + 16 * (at > 0), _native.DTYPE_CODE[dtype], ld, _native.stream()))
        got = torch.as_strided(out, (M, K), (ld, 1), at)
        assert torch.equal(got, want)
        got.fill_(5.0)
        assert (out == 5).all()


@pytest.mark.parametrize("M", [1, 3, 40, 150, 600])
@pytest.mark.parametrize("N", [31, 258, 260])
def test_gated_residual_with_rows_that_begin_anywhere(M, N):
    """residual, gate and out with odd strides and addresses, apart and in place, one gate, none, or one for groups that end
    inside a tile: the bits of the aligned call, nothing written beside the rows."""
    from wan_dit_lab_b200.quantization import fp4
    K = 192
    x = activations(M, K, 80, torch.bfloat16)
    w, _ = weight_rows(N, K, "mxfp4", 81)
    g = generator(82)
    bias = torch.randn(N, generator=g).to(DEV)
    residual = torch.randn(M, N, generator=g).to(DEV)
    gates = [None, torch.randn(N, generator=g).to(DEV), torch.randn(M // (M // 5 or 1) if M % 5 == 0 else M, N, generator=g).to(DEV)]
    for gate in gates:
        want = fp4.fp4_linear(x, w, bias, residual=residual, gate=gate)
        for extra, at in ((1, 1), (3, 0), (4, 4)):
            ld = N + extra
            off = lambda t, ld=ld, at=at: torch.zeros(t.shape[0] * ld + 8, device=DEV)[at:].as_strided(t.shape, (ld, 1), at).copy_(t)  # noqa: E731,B023,E501
            odd_gate = gate if gate is None or gate.ndim == 1 else off(gate)
            if gate is not None and gate.ndim == 1:
                odd_gate = torch.cat((gate[:at], gate))[at:]
            r = off(residual)
            assert torch.equal(fp4.fp4_linear(x, w, bias, residual=r, gate=odd_gate), want)
            wide = torch.full((M + 1, ld), 5.0, device=DEV)
            out = wide.view(-1)[at:at + M * ld].view(M, ld)[:, :N]
            assert fp4.fp4_linear(x, w, bias, residual=residual, gate=odd_gate, out=out) is out and torch.equal(out, want)
            out.fill_(5.0)
            assert (wide == 5).all()
            assert torch.equal(fp4.fp4_linear(x, w, bias, residual=r, gate=odd_gate, out=r), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [65, 127, 128, 129, 200, 513])
@pytest.mark.parametrize("N,K", [(96, 160), (300, 2080), (200, 9024)])
def test_rows_in_blocks_of_64(fmt, M, N, K):
    """More rows than one block of 64 with few features: halves of 128-row blocks, whose scales share a tile, the last one
    cut."""
    from wan_dit_lab_b200.quantization import fp4
    x = activations(M, K, 90 + M, torch.bfloat16)
    q = fp4.quantize_rows(x, fmt)
    w, W = weight_rows(N, K, fmt, 91)
    a = fp4.dequantize_rows(q, torch.float32).cpu().numpy().astype(np.float64)
    y = fp4.fp4_linear(q, w, dtype=torch.float32)
    want = a @ W.T
    assert (np.abs(y.cpu().numpy() - want) <= product_tolerance(a, W, want, torch.float32)).all()
    residual = torch.randn(M, N, generator=generator(92)).to(DEV)
    z = fp4.fp4_linear(q, w, residual=residual)
    assert (z - (residual + y)).abs().max() <= 2.0 ** -22 * (residual.abs() + y.abs()).max()  # another order of two roundings


def test_modulation_out_of_the_output_itself_is_refused():
    """gate, bias, weight, shift and scale that are the output's first rows, or a single row's own."""
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    from wan_dit_lab_b200.quantization import fp4
    w, _ = weight_rows(64, 64, "nvfp4", 140)
    for M in (1, 6):
        x = activations(M, 64, 141)
        r = torch.randn(M, 64, generator=generator(142)).to(DEV)
        keep = r.clone()
        for wrong in (dict(gate=r[:1]), dict(gate=r[0]), dict(gate=r[:M // 2 or 1]), dict(gate=r), dict(bias=r[0])):
            with pytest.raises(ValueError, match="overlap"):
                fp4.fp4_linear(x, w, residual=r, out=r, **wrong)
        for wrong in (dict(gate=r[:1]), dict(shift=r[0]), dict(scale=r[:M // 2 or 1]), dict(weight=r[0]), dict(bias=r[0]),
                      dict(gate=r)):
            with pytest.raises(ValueError, match="overlap"):
                gated_norm(r, x, inplace=True, **wrong)
        assert torch.equal(r, keep)
        # the same rows are what a call that writes elsewhere may read
        want = fp4.fp4_linear(x, w, r[0].clone(), residual=r, gate=r.clone())
        assert torch.equal(fp4.fp4_linear(x, w, r[0], residual=r, gate=r), want)
