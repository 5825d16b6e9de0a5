"""The FP4 products of many rows (gemm_pair_kernel) and of many rows over long K (the 128-row CTAs of gemm_few_kernel) against
the oracle. Every test asks the library which kernel its sizes take, so that another rule leaves no kernel untested."""

import numpy as np
import pytest
import test_fp4_gpu as small
import torch
from test_fp4_gpu import DEV, DTYPES, FORMATS, activations, generator, product_tolerance, weight_rows

from oracle import fp4 as oracle

pytestmark = pytest.mark.gpu


def takes(rows_per_cta, M, N, K):
    """The sizes take the kernel that the test is about."""
    from wan_dit_lab_b200 import _native
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _native.lib().wdl_fp4_gemm_rows_per_cta(M, N, K, sms) == rows_per_cta


# one tile a pair and several, a last tile of few rows or features, row pairs a multiple of 8 (the groups of tiles), K that
# ends inside a stage at each of its steps of 64 and inside one, one stage and more than the ring holds
MANY = [(3300, 261, 288), (3300, 258, 160), (4700, 1288, 96), (4096, 1288, 64), (520, 1416, 544), (1030, 900, 1312),
        (6500, 33, 2080), (2049, 513, 512), (1700, 512, 3808)]
LONG = [(1100, 700, 4128), (1500, 390, 9024), (1153, 704, 3872)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", MANY)
def test_linear_of_many_rows(fmt, M, N, K):
    takes(0, M, N, K)
    small.test_linear_against_float64(fmt, M, N, K)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", LONG)
def test_linear_of_many_rows_over_long_k(fmt, M, N, K):
    takes(128, M, N, K)
    small.test_linear_against_float64(fmt, M, N, K)


@pytest.mark.parametrize("kernel,M,N,K,groups", [
    (0, 3300, 264, 288, 1), (0, 3300, 261, 96, 11), (0, 4700, 1288, 64, 5), (0, 3300, 258, 160, 3300), (0, 2050, 516, 320, 2),
    (128, 1100, 700, 4128, 4), (128, 1152, 701, 3872, 9)])
def test_gated_residual_of_many_rows(kernel, M, N, K, groups):
    """Groups that are whole, that end inside a tile, and of one row; against float64, and strided in place."""
    takes(kernel, M, N, K)
    small.test_gated_residual(M, N, K, groups)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(3300, 260, 192), (4700, 1284, 192)])
def test_aligned_residual_in_place(fmt, M, N, K):
    """The stream read and written through TMA, in place, with one gate, none, and one for groups that end inside a tile."""
    from wan_dit_lab_b200.quantization import fp4
    takes(0, M, N, K)
    x = activations(M, K, 100, torch.bfloat16)
    w, wv = weight_rows(N, K, fmt, 101)
    g = generator(102)
    residual, bias = torch.randn(M, N, generator=g).to(DEV), torch.randn(N, generator=g).to(DEV)
    a = oracle.rounded(x.float().cpu().numpy(), fmt).astype(np.float64)
    y = a @ wv.T + bias.double().cpu().numpy()
    tol = product_tolerance(a, wv, y, torch.float32)
    for gate in (None, torch.randn(N, generator=g).to(DEV), torch.randn(10, N, generator=g).to(DEV)):
        rows = np.ones((1, 1)) if gate is None else np.repeat(gate.double().cpu().numpy().reshape(-1, N),
                                                               M // (1 if gate.ndim == 1 else 10), axis=0)
        stream = residual.clone()
        assert fp4.fp4_linear(x, w, bias, residual=stream, gate=gate, out=stream) is stream
        want = residual.double().cpu().numpy() + rows * y
        # the fused multiply-add rounds once
        assert (np.abs(stream.double().cpu().numpy() - want) <= np.abs(rows) * tol + 2.0 ** -24 * 1.01 * np.abs(want)).all()


@pytest.mark.parametrize("kernel,M,N", [(0, 3300, 258), (0, 4700, 1285), (0, 7000, 31)])
def test_residual_of_many_rows_that_begin_anywhere(kernel, M, N):
    takes(kernel, M, N, 192)
    small.test_gated_residual_with_rows_that_begin_anywhere(M, N)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N", [(4700, 167), (3300, 261), (4700, 1191), (4700, 1290)])
def test_outputs_of_many_rows_that_begin_anywhere(fmt, M, N):
    """Every alignment of rows; among them rows that TMA stores up to a last group of columns that ends off a 16-byte
    boundary, which the warp stores itself, in between (float32, N 167 and rows of 168)."""
    takes(0, M, N, 192)
    for _ in range(3):
        small.test_outputs_that_begin_anywhere(fmt, M, N)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("first,second,M,K,H,N", [
    (0, 0, 3300, 96, 288, 264), (0, 0, 4700, 288, 1056, 264), (0, 0, 2050, 64, 544, 513), (128, 0, 1100, 4128, 704, 800),
    (0, 128, 1100, 96, 4128, 700)])
def test_gelu_mlp_of_many_rows(fmt, first, second, M, K, H, N):
    """The hidden layer's codes and scales, the last tile's padding among them, and the second product of them."""
    takes(first, M, H, K)
    takes(second, M, N, H)
    small.test_gelu_mlp(fmt, M, K, H, N)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H", range(256 + 32, 512 + 32, 32))
def test_hidden_layers_of_many_rows_that_end_anywhere_in_a_tile(fmt, H):
    """Every width of the last tile: codes, scales, zeros in the padding of the last tile of scales, and the scales of rows
    behind the last left as they were."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    takes(0, 3300, H, 96)
    small.test_gelu_mlp(fmt, 3300, 96, H, 24)
    x = fp4.quantize_rows(activations(3300, 96, 170), fmt)
    w, _ = weight_rows(H, 96, fmt, 171)
    tiles = torch.full(fp4.scale_tiles(3300, H, fmt), 0xAB, dtype=torch.uint8, device=DEV)
    codes = torch.empty(3300, H // 2, dtype=torch.uint8, device=DEV)
    _native.check(_native.lib().wdl_fp4_gemm_gelu(x._operand, w._operand, None, 3300, H, 96, None, codes.data_ptr(),
                                                  tiles.data_ptr(), _native.stream()))
    blocks = H // fp4.BLOCK[fmt]
    by_row = fp4.untile_scales(tiles, 3328, -(-blocks // 4) * 4)
    want = small.hidden_of(x, w, None, fmt, None)
    assert torch.equal(by_row[:3300, :blocks], fp4.untile_scales(want.scales, 3300, blocks)) and torch.equal(codes, want.codes)
    assert not by_row[:3300, blocks:].any() and (by_row[3300:] == 0xAB).all()


@pytest.mark.parametrize("M", [1700, 1665])
def test_a_square_layer_of_many_rows_onto_its_own_input(M):
    takes(0, M, 512, 512)
    small.test_a_square_layer_onto_its_own_input(M)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
def test_non_finite_values_stay_in_their_rows_of_many(fmt, bad):
    from wan_dit_lab_b200.quantization import fp4
    M, N, K = 3300, 264, 288
    takes(0, M, N, K)
    x = activations(M, K, 110)
    rows = torch.tensor([0, 127, 128, 300, 3299], device=DEV)
    x[rows, torch.tensor([0, 31, 255, 256, 287], device=DEV)] = bad
    w, _ = weight_rows(N, K, fmt, 111)
    other = torch.ones(M, dtype=torch.bool, device=DEV)
    other[rows] = False
    nan = fp4.fp4_linear(x, w, dtype=torch.float32).isnan()
    assert nan[rows].all() and not nan[other].any()
    w2, _ = weight_rows(N, N + 24, fmt, 112)
    w1, _ = weight_rows(N + 24, K, fmt, 113)
    nan = fp4.fp4_gelu_mlp(x, w1, None, w2, None, residual=torch.zeros(M, N, device=DEV)).isnan()
    assert nan[rows].all() and not nan[other].any()


def test_many_rows_on_other_streams_and_in_graphs():
    """Both products of a feed forward with many rows: on a side stream, and in two graphs replayed in turn."""
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    M, D, H = 3300, 288, 1056
    takes(0, M, H, D)
    takes(0, M, D, H)
    w1, _ = weight_rows(H, D, "nvfp4", 120)
    w2, _ = weight_rows(D, H, "nvfp4", 121)
    x = activations(M, D, 122)
    want = [fp4.fp4_gelu_mlp(x * k, w1, None, w2, None, residual=x * k) for k in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [fp4.fp4_gelu_mlp(x, w1, None, w2, None, residual=x) for _ in range(10)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(y, want[0]) for y in got)
    graphs = []
    for _ in range(2):
        static = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fp4.fp4_gelu_mlp(static, w1, None, w2, None, residual=static)
        graphs.append((graph, static, out))
    for k in (1, 2, 1):
        for graph, static, out in graphs:
            static.copy_(x * k)
            graph.replay()
            assert torch.equal(out, want[k - 1])
    assert _native.device_error() == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_made_just_before_a_product_of_many_rows(fmt):
    from wan_dit_lab_b200.quantization import fp4
    M, N, K = 1700, 1024, 1056
    takes(0, M, N, K)
    x = activations(M, K, 130, torch.bfloat16)
    W = [torch.randn(N, K, generator=generator(131 + i)).to(DEV) * 0.02 for i in range(4)]
    q = fp4.quantize_rows(x, fmt)
    want = [fp4.fp4_linear(q, fp4.quantize_rows(w, fmt)) for w in W]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for w in W:
            got.append(fp4.fp4_linear(q, fp4.quantize_rows(w, fmt)))
            got.append(fp4.fp4_linear(x, fp4.quantize_rows(w, fmt)))
        for i in range(4):
            assert torch.equal(got[2 * i], want[i]) and torch.equal(got[2 * i + 1], want[i])


def test_calls_from_several_threads_at_once():
    """Threads with streams of their own, every kernel, from each kernel's first launch in a fresh process on (what is asked
    of the device once is asked by several of them)."""
    import subprocess
    import sys
    from pathlib import Path
    program = """
import sys, threading
sys.path[:0] = {paths!r}
import torch
from test_fp4_gpu import activations, weight_rows
from wan_dit_lab_b200 import _native
from wan_dit_lab_b200.kernels.gated_norm import gated_norm
from wan_dit_lab_b200.quantization import fp4
layers = [weight_rows(N, K, "nvfp4", N)[0] for N, K in ((1056, 288), (288, 1056))]
xs = [activations(M, 288, M, torch.bfloat16) for M in (1, 9, 40, 3300)]
torch.cuda.synchronize()
def call(x):
    s, rows = gated_norm(x, x, out="nvfp4")
    y = fp4.fp4_gelu_mlp(rows, layers[0], None, layers[1], None, dtype=torch.float32)
    return y, fp4.fp4_linear(x, layers[0]), fp4.dequantize_rows(fp4.quantize_rows(x, "mxfp4"))
start, got = threading.Barrier(4), {{}}
def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        got[i] = [call(x) for _ in range(20) for x in xs[i:] + xs[:i]]
        torch.cuda.current_stream().synchronize()
threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
for t in threads: t.start()
for t in threads: t.join()
for i in range(4):
    for j, out in enumerate(got[i]):
        for a, b in zip(out, call((xs[i:] + xs[:i])[j % 4])):
            assert torch.equal(a, b), (i, j)
assert _native.device_error() == 0
print("ok")
"""
    here = Path(__file__).resolve().parent
    paths = [str(here.parent / "wan-dit-lab_b200"), str(here.parent), str(here)]
    run = subprocess.run([sys.executable, "-c", program.format(paths=paths)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
