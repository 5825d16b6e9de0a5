"""The FP4 operators without a GPU: the oracle against brute force, the scale tiles, the packed argument structures against
the header, and what the entry points and the Python layer refuse before anything is launched."""

import ctypes
import itertools
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from oracle import fp4 as oracle

HEADER = Path(__file__).resolve().parents[1] / "include" / "wdl_b200.h"
FAKE = 0x10000  # a 256-byte aligned address that nothing reads: every call here is refused or has no rows


def brute(values, x):
    """Index of the nearest value, ties to the even index, by distance in exact arithmetic."""
    d = np.abs(values.astype(np.float64)[None] - x.astype(np.float64)[:, None])
    best = d == d.min(1, keepdims=True)
    return np.array([next((i for i in np.flatnonzero(row) if i % 2 == 0), np.flatnonzero(row)[0]) for row in best])


def test_oracle_rounds_to_the_nearest_with_ties_to_even():
    rng = np.random.default_rng(0)
    q = np.concatenate([np.linspace(0, 8, 1025), rng.exponential(2, 500)]).astype(np.float32)
    np.testing.assert_array_equal(oracle.e2m1(q), brute(oracle.E2M1, np.minimum(q, 6)))
    np.testing.assert_array_equal(oracle.e2m1(-q) & 7, oracle.e2m1(q))
    e4m3 = oracle.e4m3_values()
    np.testing.assert_array_equal(e4m3, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy())
    s = np.concatenate([np.exp(rng.uniform(-7, 6, 500)), e4m3, (e4m3[1:] + e4m3[:-1]) / 2]).astype(np.float32).clip(0, 448)
    np.testing.assert_array_equal(oracle._nearest(e4m3, s.astype(np.float64)), brute(e4m3, s))
    # as torch rounds to E4M3
    np.testing.assert_array_equal(oracle._nearest(e4m3, s.astype(np.float64)),
                                  torch.from_numpy(s).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_oracle_quantization_is_within_its_blocks_step(fmt):
    """Half of the largest step (2 scales) away at most, but for what the scale's own rounding cuts off above 6."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((7, 96)) * np.exp(rng.standard_normal((7, 96)))).astype(np.float32)
    x[2, :32], x[3, 5], x[4, 40] = 0, np.nan, np.inf
    v, (_, byte) = oracle.rounded(x, fmt), oracle.encode(x, fmt)
    s = np.repeat(oracle.scale_values(byte, fmt), oracle.BLOCK[fmt], axis=1)
    fine = np.isfinite(s)
    assert (~fine).sum() == 2 * oracle.BLOCK[fmt] and np.isnan(v[~fine]).all()
    cut = np.maximum(np.abs(x[fine]) - 6 * s[fine], 0)
    assert (np.abs(v[fine] - x[fine]) <= np.maximum(s[fine], cut) * (1 + 1e-6)).all()
    assert (v[2, :32] == 0).all()


def test_tiles_of_scales():
    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.quantization import fp4
    lib = _native.lib()
    for R, B in ((1, 1), (5, 6), (128, 4), (129, 5), (300, 12)):
        s = torch.randint(0, 256, (R, B), dtype=torch.uint8)
        tiles = fp4.tile_scales(s)
        assert torch.equal(fp4.untile_scales(tiles, R, B), s)
        flat, bt = tiles.flatten(), -(-B // 4)
        for r, b in itertools.product(range(0, R, 37), range(B)):
            assert flat[((r // 128) * bt + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] == s[r, b]
        assert tiles.sum() == s.sum()  # zeros elsewhere
    for fmt, code in fp4.FORMAT_CODE.items():
        for M, K in ((1, 32), (5, 96), (129, 1056), (300, 3072)):
            assert lib.wdl_fp4_scale_bytes(M, K, code) == np.prod(fp4.scale_tiles(M, K, fmt))
            first = fp4._rows_bytes(M, K, fmt) if M != 1 else 0
            assert lib.wdl_fp4_linear_workspace(M, K, code) == first
            assert lib.wdl_fp4_gelu_mlp_workspace(M, K, 544, code) == first + fp4._rows_bytes(M, 544, fmt)
    assert lib.wdl_fp4_scale_bytes(4, 48, 0) == 0 and lib.wdl_fp4_scale_bytes(4, 64, 2) == 0


def test_packed_structures_match_the_header():
    """The formats of the packed arguments are the header's fields in their order."""
    from wan_dit_lab_b200 import _native
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name, packed in (("wdl_fp4_rows", _native.FP4_ROWS), ("wdl_gated_norm_args", _native.GATED_NORM)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
        codes = ""
        for declaration in body.split(";"):
            fields = declaration.strip()
            if fields:
                code = "P" if "*" in fields else {"int64_t": "q", "int": "i", "float": "f"}[fields.split()[0]]
                codes += code * (fields.count(",") + 1)
        expanded = re.sub(r"(\d+)([a-w])", lambda m: m.group(2) * int(m.group(1)), packed.format.strip("@"))
        expanded = re.sub(r"\d*x", "", expanded)
        assert expanded == codes, (name, expanded, codes)
        types = {"P": ctypes.c_void_p, "q": ctypes.c_int64, "i": ctypes.c_int, "f": ctypes.c_float}
        plain = type(name, (ctypes.Structure,), {"_fields_": [(f"f{i}", types[c]) for i, c in enumerate(codes)]})
        assert ctypes.sizeof(plain) == packed.size, name


def rows_arg(codes=FAKE, scales=FAKE, t=0, fmt=0):
    from wan_dit_lab_b200 import _native
    return _native.FP4_ROWS.pack(codes, scales, t, fmt)


def gemm(lib, a=None, w=None, bias=None, M=4, N=64, K=64, out=FAKE, dtype=0, ld=64):
    return lib.wdl_fp4_gemm(a or rows_arg(), w or rows_arg(), bias, M, N, K, out, dtype, ld, None)


def quantize(lib, x=FAKE, dtype=0, ld=64, M=4, K=64, fmt=0, t=None, codes=FAKE, scales=FAKE):
    return lib.wdl_fp4_quantize_rows(x, dtype, ld, M, K, fmt, t, codes, scales, None)


def linear(lib, x=FAKE, dtype=0, ld=64, t=None, w=None, gate=None, groups=1, ldg=64, res=None, ldr=64, M=4, N=64, K=64,
           out=FAKE, out_dtype=0, ldo=64, work=FAKE, size=1 << 20):
    return lib.wdl_fp4_linear(x, dtype, ld, t, w or rows_arg(), None, gate, groups, ldg, res, ldr, M, N, K, out, out_dtype,
                              ldo, work, size, None)


def mlp(lib, x=FAKE, xr=None, w1=None, w2=None, M=4, H=64, N=64, K=64, res=None, gate=None, out_dtype=0, work=FAKE,
        size=1 << 20):
    return lib.wdl_fp4_gelu_mlp(x, 0, K, None, xr, w1 or rows_arg(), None, None, w2 or rows_arg(), None, gate, 1, N, res, N,
                                M, H, N, K, FAKE, out_dtype, N, work, size, None)


def residual(lib, gate=FAKE, groups=1, ldg=64, res=FAKE, ldr=64, M=4, N=64, K=64, out=FAKE, ldo=64):
    return lib.wdl_fp4_gemm_residual(rows_arg(), rows_arg(), None, gate, groups, ldg, res, ldr, M, N, K, out, ldo, None)


REFUSED = [
    (quantize, dict(K=48), b"32"), (quantize, dict(K=0), b"32"), (quantize, dict(M=-1), b"32"),
    (quantize, dict(fmt=2), b"format"), (quantize, dict(dtype=3), b"bf16"), (quantize, dict(ld=63), b"ldx"),
    (quantize, dict(ld=68), b"16-byte"), (quantize, dict(x=FAKE + 8), b"16-byte"), (quantize, dict(x=None), b"null"),
    (quantize, dict(codes=None), b"null"), (quantize, dict(scales=FAKE + 4), b"16-byte"),
    (quantize, dict(fmt=1, t=FAKE), b"tensor scale"),
    (gemm, dict(w=rows_arg(fmt=1)), b"same FP4 format"), (gemm, dict(K=40), b"32"), (gemm, dict(N=0, ld=0), b"N must"),
    (gemm, dict(ld=63), b"ldo"), (gemm, dict(ld=1 << 31), b"2^31"), (gemm, dict(dtype=5), b"bf16"),
    (gemm, dict(out=FAKE + 1), b"aligned to its type"), (gemm, dict(out=None), b"null"),
    (gemm, dict(a=rows_arg(codes=FAKE + 8)), b"16-byte"), (gemm, dict(w=rows_arg(scales=0)), b"null"),
    (gemm, dict(bias=FAKE + 2), b"4-byte"), (gemm, dict(M=-2), b"32"),
    (gemm, dict(a=rows_arg(fmt=1, t=FAKE), w=rows_arg(fmt=1)), b"tensor scale"),
    (gemm, dict(M=2 ** 31 - 1, N=2 ** 31 - 1, ld=2 ** 31 - 1), b"too many tiles"),
    (residual, dict(groups=3), b"multiple of the gate"), (residual, dict(groups=2, ldg=60), b"ld_gate"),
    (residual, dict(res=None), b"residual"), (residual, dict(ldr=1), b"ldr"), (residual, dict(out=FAKE + 2), b"4-byte"),
    (linear, dict(M=7, work=None), b"workspace"), (linear, dict(M=7, work=FAKE + 16), b"256-byte"),
    (linear, dict(M=7, size=511), b"too small"), (linear, dict(dtype=4), b"bf16"), (linear, dict(ld=62), b"ldx"),
    (linear, dict(x=FAKE + 2), b"16-byte"),
    (linear, dict(res=FAKE), b"writes f32"), (linear, dict(gate=FAKE), b"needs a residual"), (linear, dict(K=33), b"32"),
    (linear, dict(x=None), b"null"), (linear, dict(M=1, x=None), b"null"), (linear, dict(M=1, ld=62), b"ldx"),
    (linear, dict(M=1, x=FAKE + 4, work=None), b"16-byte"), (linear, dict(M=1, t=FAKE + 2), b"4-byte"), (linear, dict(w=rows_arg(fmt=1), t=FAKE), b"tensor scale"),
    (mlp, dict(H=48), b"32"), (mlp, dict(x=None), b"either"), (mlp, dict(xr=rows_arg()), b"either"),
    (mlp, dict(w2=rows_arg(fmt=1)), b"same FP4 format"), (mlp, dict(size=600), b"too small"), (mlp, dict(res=FAKE), b"f32"),
    (mlp, dict(gate=FAKE), b"needs a residual"), (mlp, dict(w1=rows_arg(codes=0)), b"null"),
    (quantize, dict(M=2 ** 31 - 1), b"rows"), (quantize, dict(K=2 ** 26 + 32, ld=2 ** 27), b"columns"),
    (gemm, dict(M=2 ** 31 - 1, N=8, ld=8), b"rows"), (gemm, dict(M=1, N=2 ** 31 - 1, ld=2 ** 31 - 1), b"2^16"),
    (linear, dict(M=2 ** 31 - 1), b"rows"), (mlp, dict(M=2 ** 31 - 1), b"rows"), (mlp, dict(H=2 ** 30), b"columns"),
]


@pytest.mark.parametrize("call,change,message", REFUSED)
def test_entry_points_refuse(call, change, message):
    from wan_dit_lab_b200 import _native
    lib = _native.lib()
    assert call(lib, **change) == _native.ERR_ARGUMENT
    assert message in lib.wdl_last_error(), lib.wdl_last_error()


def test_no_rows_is_no_work():
    from wan_dit_lab_b200 import _native
    lib = _native.lib()
    for call in (quantize, gemm, linear, mlp, residual):
        assert call(lib, M=0) == _native.OK


NORM = dict(x=FAKE, ldx=64, y=FAKE, ldy=64, gate=FAKE, ld_gate=64, weight=0, bias=0, shift=0, ld_shift=0, scale=0, ld_scale=0,
            x_out=FAKE, ldxo=64, h=FAKE, ldh=64, h_scales=FAKE, tensor_scale=0, x_dtype=2, y_dtype=2, M=4, K=64, groups=1,
            rms=0, out=3, eps=1e-6)


@pytest.mark.parametrize("change,message", [
    (dict(K=40), b"32"), (dict(K=16416), b"16384"), (dict(K=60, out=2), b"multiple of 8"), (dict(out=5), b"output type"),
    (dict(x_dtype=1), b"bf16 or f32"), (dict(y_dtype=1), b"bf16 or f32"), (dict(groups=3), b"groups"), (dict(groups=0), b"groups"),
    (dict(y=0), b"needs a branch"), (dict(y=0, gate=0), b"needs a branch"), (dict(out=4, tensor_scale=FAKE), b"tensor scale"),
    (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"), (dict(x=0), b"null"), (dict(h_scales=0), b"null"),
    (dict(x_out=0), b"null"), (dict(ldx=60), b"stride"), (dict(ldy=62), b"stride"), (dict(ldx=66), b"16-byte"),
    (dict(out=2, ldh=63), b"stride"), (dict(h=FAKE + 8), b"16-byte"), (dict(gate=FAKE + 4), b"16-byte"),
    (dict(weight=FAKE + 4), b"16-byte"), (dict(shift=FAKE, ld_shift=62), b"16-byte"),
    (dict(groups=2, ld_gate=60), b"stride"), (dict(M=-4), b"multiple"), (dict(M=2 ** 31 - 1), b"rows")])
def test_gated_norm_entry_point_refuses(change, message):
    from wan_dit_lab_b200 import _native
    lib = _native.lib()
    assert lib.wdl_gated_norm(_native.GATED_NORM.pack(*{**NORM, **change}.values()), None) == _native.ERR_ARGUMENT
    assert message in lib.wdl_last_error(), lib.wdl_last_error()
    assert lib.wdl_gated_norm(_native.GATED_NORM.pack(*{**NORM, "M": 0}.values()), None) == _native.OK
    assert lib.wdl_gated_norm(None, None) == _native.ERR_ARGUMENT


def test_rows_that_overlap():
    """out [M, K] against what a kernel reads beside it, by addresses alone."""
    from wan_dit_lab_b200._native import overlaps
    b = torch.zeros(10, 64)
    flat = b.view(-1)
    for out, t, want in [
            (b, b, False), (b[:5], b[5:], False), (b[:6], b[5:], True), (b[1:], b[:-1], True),
            (b[:, :32], b[:, 32:], False), (b[:, :33], b[:, 32:], True), (b[:, 32:], b[:, :32], False),
            (b[:, :32], b[:, 16:48], True), (b[:9, 32:], b[1:, :32], False), (b, b[3], True), (b, flat[640:], False),
            (b[:3], flat[192:256], False), (b[:3], flat[191:255], True), (b[:1], b[0], False), (b[:1], b[0, 1:], True),
            (b[::2], b[1::2], False), (b[::2], b[::2], False), (b, b.view(torch.bfloat16), True), (b[:0], b, False),
            (b, torch.zeros(10, 64), False), (b[:5], b[:10:2], True)]:
        assert overlaps(out, t) is want, (out.shape, t.shape)


def test_only_all_of_the_same_rows_are_updated_in_place():
    """A part of the rows, or what is no residual, overlaps even where it begins at the same address."""
    from wan_dit_lab_b200._native import overlaps
    b = torch.zeros(10, 64)
    for out, t, in_place, want in [
            (b, b, True, False), (b, b[:3], True, True), (b[:3], b, True, True), (b, b[0], True, True),
            (b, b[:, :32], True, True), (b[:, :32], b, True, True), (b[:1], b[0, :32], True, True), (b[:5], b[5:], False, False),
            (b, b, False, True), (b[:1], b[0], False, True), (b[:1], b[:1], False, True), (b[:, :32], b[:, 32:], False, False),
            (b[::2], b[1::2], False, False), (b[::2], b[::2], False, True), (b[:1], b[1], False, False)]:
        assert overlaps(out, t, in_place) is want, (out.shape, t.shape, in_place)


@pytest.fixture
def fake(monkeypatch):
    from wan_dit_lab_b200 import _native
    monkeypatch.setattr(_native, "elsewhere", lambda device: False)
    with FakeTensorMode():
        yield


def cuda(*shape, dtype=torch.float32, **kw):
    return torch.zeros(*shape, dtype=dtype, device="cuda", **kw)


def fake_rows(rows, columns, fmt="nvfp4"):
    """An operand without memory, for what is refused before any address is read."""
    from wan_dit_lab_b200.quantization import fp4
    r = fp4.Rows.__new__(fp4.Rows)
    r._codes = r._scales = r._buffer = None
    r._set(fmt, rows, columns, torch.device("cuda", 0), None, FAKE, FAKE)
    return r


def test_rows_refuse(fake):
    from wan_dit_lab_b200.quantization import fp4
    u8 = dict(dtype=torch.uint8)
    codes, tiles = cuda(4, 32, **u8), cuda(1, 1, 32, 4, 4, **u8)
    for args, error, message in [
            ((codes, tiles, "fp8"), ValueError, "unknown FP4 format"), ((codes.float(), tiles, "nvfp4"), TypeError, "uint8"),
            ((torch.zeros(4, 32, **u8), tiles, "nvfp4"), ValueError, "CUDA"),
            ((cuda(4, 24, **u8), tiles, "nvfp4"), ValueError, "multiple of 32"),
            ((cuda(4, 0, **u8), tiles, "nvfp4"), ValueError, "multiple of 32"),
            ((codes, cuda(1, 2, 32, 4, 4, **u8), "nvfp4"), ValueError, "tiles"),
            ((cuda(4, 64, **u8)[:, ::2], tiles, "nvfp4"), ValueError, "contiguous"),
            ((codes, tiles, "mxfp4", cuda(1)), ValueError, "tensor scale"),
            ((codes, tiles, "nvfp4", cuda(2)), TypeError, "one float32"),
            ((codes, tiles, "nvfp4", torch.zeros(1)), ValueError, "device")]:
        with pytest.raises(error, match=message):
            fp4.Rows(*args)


def test_python_operators_refuse(fake):
    from wan_dit_lab_b200.quantization import fp4
    w, x = fake_rows(96, 64), cuda(6, 64)
    q, lin, mlp_ = fp4.quantize_rows, fp4.fp4_linear, fp4.fp4_gelu_mlp
    cases = [
        (lambda: q(x, "int4"), ValueError, "unknown FP4 format"), (lambda: q(torch.zeros(6, 64)), ValueError, "CUDA"),
        (lambda: q(x.double()), TypeError, "bfloat16, float16 or float32"), (lambda: q(cuda(6, 48)), ValueError, "multiple of 32"),
        (lambda: q(cuda(6, 0)), ValueError, "multiple of 32"), (lambda: q(cuda(2, 3, 64)), ValueError, r"\[M, K\]"),
        (lambda: q(cuda(6, 64, requires_grad=True)), ValueError, "inference-only"),
        (lambda: fp4.dequantize_rows(x), TypeError, "Rows"),
        (lambda: fp4.dequantize_rows(w, torch.float64), TypeError, "dtype"),
        (lambda: lin(x, x), TypeError, "Rows"),
        (lambda: lin(fake_rows(6, 64, "mxfp4"), w), ValueError, "same FP4 format"),
        (lambda: lin(fake_rows(6, 96), w), ValueError, "64 columns"),
        (lambda: lin(fake_rows(6, 64), w, input_scale=cuda(1)), ValueError, "its own tensor scale"),
        (lambda: lin(fake_rows(6, 64), w, cuda(95)), ValueError, r"bias must be \[96\]"),
        (lambda: lin(fake_rows(6, 64), w, torch.zeros(96)), ValueError, "bias must be on"),
        (lambda: lin(fake_rows(6, 64), w, gate=cuda(96)), ValueError, "belong to a residual"),
        (lambda: lin(fake_rows(6, 64), w, out=cuda(6, 96)), ValueError, "belong to a residual"),
        (lambda: lin(fake_rows(6, 64), w, dtype=torch.float64), TypeError, "dtype"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 95)), ValueError, "residual must be float32"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96, dtype=torch.bfloat16)), ValueError, "residual must be float32"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96), gate=cuda(4, 96)), ValueError, "do not divide"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96), gate=cuda(2, 95)), ValueError, "gate must be"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96), gate=torch.zeros(96)), ValueError, "same device"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96), out=cuda(6, 97)), ValueError, "out must be float32"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96), out=cuda(96, 6).t()), ValueError, "consecutive"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96), out=cuda(1, 96).expand(6, 96)), ValueError, "apart"),
        (lambda: lin(fake_rows(6, 64), w, cuda(96, requires_grad=True)), ValueError, "inference-only"),
        (lambda: lin(fake_rows(6, 64), w, residual=cuda(6, 96), out=cuda(6, 96, requires_grad=True)), ValueError, "inference-only"),
        (lambda: q(x, "nvfp4", cuda(1, requires_grad=True)), ValueError, "inference-only"),
        (lambda: lin(x, w, input_scale=cuda(1, requires_grad=True)), ValueError, "inference-only"),
        (lambda: mlp_(fake_rows(6, 64), w, None, fake_rows(32, 96), None, hidden_scale=cuda(1, requires_grad=True)), ValueError,
         "inference-only"),
        (lambda: lin(fake_rows(6, 64, "mxfp4"), fake_rows(96, 64, "mxfp4"), input_scale=cuda(1)), ValueError, "its own"),
        (lambda: mlp_(fake_rows(6, 64), w, None, fake_rows(32, 64), None), ValueError, "96 columns"),
        (lambda: mlp_(fake_rows(6, 64), w, None, fake_rows(32, 96, "mxfp4"), None), ValueError, "format"),
        (lambda: mlp_(fake_rows(6, 64), w, cuda(4), fake_rows(32, 96), None), ValueError, "bias1"),
        (lambda: mlp_(fake_rows(6, 64), w, None, fake_rows(32, 96), cuda(96)), ValueError, "bias2"),
        (lambda: mlp_(fake_rows(6, 64), w, None, fake_rows(32, 96), None, hidden_scale=cuda(2)), TypeError, "hidden scale"),
        (lambda: mlp_(fake_rows(6, 64), w, None, fake_rows(32, 96), None, gate=cuda(32)), ValueError, "residual"),
    ]
    for call, error, message in cases:
        with pytest.raises(error, match=message):
            call()


def test_gated_norm_refuses(fake):
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    x, v = cuda(6, 64), cuda(64)
    cases = [
        (dict(kind="batch"), ValueError, "kind"), (dict(out=torch.float64), TypeError, "out must be"),
        (dict(out="fp8"), TypeError, "out must be"), (dict(tensor_scale=v[:1]), ValueError, "tensor scale"),
        (dict(out="mxfp4", tensor_scale=v[:1]), ValueError, "tensor scale"), (dict(x=torch.zeros(6, 64)), ValueError, "CUDA"),
        (dict(x=cuda(6, 60)), ValueError, "multiple of 8"), (dict(x=cuda(6, 40), out="nvfp4"), ValueError, "32 for an FP4"),
        (dict(x=cuda(1, 16392)), ValueError, "16384"), (dict(x=cuda(2, 3, 64)), ValueError, r"\[M, K\]"),
        (dict(x=x.half()), TypeError, "x must be bfloat16"), (dict(y=x.half()), TypeError, "y must be bfloat16"),
        (dict(y=cuda(5, 64)), ValueError, "y must have"), (dict(y=torch.zeros(6, 64)), ValueError, "y must have"),
        (dict(gate=v), ValueError, "belong to a branch"), (dict(inplace=True), ValueError, "belong to a branch"),
        (dict(y=x, gate=cuda(4, 64)), ValueError, "do not divide"), (dict(shift=cuda(63)), ValueError, "shift must be"),
        (dict(shift=cuda(2, 64), scale=cuda(3, 64)), ValueError, "same number of groups"),
        (dict(scale=torch.zeros(64)), ValueError, "same device"), (dict(weight=cuda(6, 64)), ValueError, "weight must be"),
        (dict(bias=torch.zeros(64)), ValueError, "bias must be"),
        (dict(x=cuda(6, 64, requires_grad=True)), ValueError, "inference-only"),
        (dict(weight=cuda(64, requires_grad=True)), ValueError, "inference-only"),
    ]
    for change, error, message in cases:
        with pytest.raises(error, match=message):
            gated_norm(**{"x": x, **change})


def test_packed_layers_refuse(fake):
    from wan_dit_lab_b200.quantization import fp4
    with pytest.raises(ValueError, match="scales must be"):
        fp4.PackedFp4Linear(cuda(8, 32, dtype=torch.uint8), cuda(8, 3, dtype=torch.uint8))
    with pytest.raises(ValueError, match="unknown FP4 format"):
        fp4.quantize(cuda(8, 64), fmt="fp6")


def test_every_product_kernel_has_its_sizes():
    """The rule by which a product's kernel is chosen, for 148 multiprocessors, on either side of its borders."""
    from wan_dit_lab_b200 import _native
    rows = _native.lib().wdl_fp4_gemm_rows_per_cta
    for sizes, want in [((1, 1 << 20, 32), 16), ((16, 64, 64), 16), ((17, 64, 64), 64), ((64, 1 << 20, 1 << 20), 64),
                        ((65, 98 * 64, 3072), 64), ((65, 99 * 64, 3072), 0), ((65, 32 * 128, 9024), 64), ((65, 33 * 128, 9024), 128),
                        ((1100, 700, 3840), 0), ((1100, 700, 3872), 128), ((128, 88 * 128, 4096), 128), ((128, 89 * 128, 4096), 0),
                        ((2 ** 31 - 2 ** 16, 2 ** 31 - 2 ** 16, 64), 0), ((0, 8, 64), -1), ((8, 0, 64), -1), ((8, 8, 0), -1)]:
        assert rows(*sizes, 148) == want, sizes
    assert rows(8, 8, 64, 0) == -1


def test_tiles_of_the_many_row_product(tmp_path):
    """Every tile is taken once, and nothing undefined is computed for the step past a pair's last tile."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    exe = tmp_path / "fp4_tiles_check"
    source = Path(__file__).resolve().parent / "native" / "fp4_tiles_check.cpp"
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(source), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stderr


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_a_cast_leaves_the_scales_and_the_bias(fmt):
    from wan_dit_lab_b200.quantization import fp4
    g = torch.Generator().manual_seed(0)
    layer = lambda N, K: fp4.PackedFp4Linear(  # noqa: E731
        torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=g),
        torch.randint(0, 127, (N, K // fp4.BLOCK[fmt]), dtype=torch.uint8, generator=g),
        torch.rand(1, generator=g) if fmt == "nvfp4" else None, torch.randn(N, generator=g), 0.1 if fmt == "nvfp4" else None)
    mlp = fp4.PackedFp4GeluMLP(layer(96, 64), layer(32, 96))
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), mlp)
    want = {name: t.clone() for name, t in mlp.state_dict().items()}
    for cast in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.bfloat16)):
        assert cast(model) is model
        now = mlp.state_dict()
        assert set(now) == set(want)
        for name, t in want.items():
            assert now[name].dtype == t.dtype and torch.equal(now[name], t), name
    assert model[0].weight.dtype == torch.bfloat16  # what is not FP4 was cast
    for t in model.to("meta")[1].state_dict().values():
        assert t.is_meta and t.dtype in (torch.uint8, torch.float32)


def test_forward_mode_tangents_are_refused(fake):
    """Dual tensors do not require a gradient; a kernel would drop their tangents. Under no_grad too, as torch has it."""
    from torch.autograd import forward_ad

    from wan_dit_lab_b200 import _native
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    from wan_dit_lab_b200.quantization import fp4
    w, rows, w2 = fake_rows(96, 64), fake_rows(6, 64), fake_rows(32, 96)
    x, y, v = cuda(6, 64), cuda(6, 96), cuda(96)
    with forward_ad.dual_level():
        d = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [
            lambda: fp4.quantize_rows(d(x)), lambda: fp4.quantize_rows(x, "nvfp4", d(cuda(1))), lambda: fp4.fp4_linear(d(x), w),
            lambda: fp4.fp4_linear(d(cuda(6, 66))[:, 1:65], w),  # (a copy is read)
            lambda: fp4.fp4_linear(rows, w, d(v)), lambda: fp4.fp4_linear(rows, w, residual=d(y)),
            lambda: fp4.fp4_linear(rows, w, residual=y, gate=d(v)), lambda: fp4.fp4_linear(rows, w, residual=y, out=d(y)),
            lambda: fp4.fp4_linear(x, w, input_scale=d(cuda(1))), lambda: fp4.fp4_gelu_mlp(d(x), w, None, w2, None),
            lambda: fp4.fp4_gelu_mlp(rows, w, d(v), w2, None), lambda: fp4.fp4_gelu_mlp(rows, w, None, w2, d(cuda(32))),
            lambda: fp4.fp4_gelu_mlp(rows, w, None, w2, None, hidden_scale=d(cuda(1))), lambda: gated_norm(d(x)),
            lambda: gated_norm(x, d(x)), lambda: gated_norm(x, x, d(cuda(64))), lambda: gated_norm(x, shift=d(cuda(64))),
            lambda: gated_norm(x, scale=d(cuda(64))), lambda: gated_norm(x, weight=d(cuda(64))),
            lambda: gated_norm(x, bias=d(cuda(64))), lambda: gated_norm(x, out="nvfp4", tensor_scale=d(cuda(1)))]
        for call in calls:
            with pytest.raises(ValueError, match="inference-only"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="inference-only"):
                call()
        _native.refuse_gradients("an ordinary tensor inside the level is not", x, None)
