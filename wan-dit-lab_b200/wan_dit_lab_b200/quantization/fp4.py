"""Linear layers in B200's own 4-bit formats, NVFP4 and MXFP4 (microscaled 4-bit floating point), beside the INT4 ones
of quantization/w4a4.py: weights and activations both in E2M1 with a scale per block of input channels, multiplied by
the tensor cores' block-scaled MMA as they lie in memory. 0.56 or 0.53 bytes a weight against the 2 of the exact INT4
operands, and four times their tensor rate; the rounding is FP4's, not INT4's, so that a layer converted for one
format does not give the other's results.

    nvfp4   blocks of 16 channels, scale s in E4M3, one float32 t per tensor (1 when absent):
            s = E4M3(max|x| / (6 t)) clamped to [2^-9, 448], code = E2M1(x / (s t))
    mxfp4   blocks of 32 channels, scale 2^e in E8M0, e = floor(log2 max|x|) - 2, code = E2M1(x / 2^e)

in float32, rounded to nearest even, magnitudes above 6 become 6. A block with an infinity or a NaN becomes NaN as a
whole. Codes are two a byte (low nibble: the even channel); scales lie in the tensor cores' tiles (tile_scales).
Inference only, like the rest of the package: inputs that require a gradient or carry a forward-mode tangent are refused.
No counterpart in the reference, whose 4-bit layers are INT4.
"""

import torch
from torch.autograd import forward_ad

from wan_dit_lab_b200 import _native

BLOCK = {"nvfp4": 16, "mxfp4": 32}  # input channels per scale
FORMAT_CODE = {"nvfp4": _native.NVFP4, "mxfp4": _native.MXFP4}
E2M1_MAX, E4M3_MAX = 6.0, 448.0


class Rows:
    """A matrix [rows, columns] in FP4: codes [rows, columns / 2] uint8, scales the uint8 tiles of tile_scales
    ([ceil(rows / 128), ceil(columns / (4 block)), 32, 4, 4]), fmt "nvfp4" or "mxfp4", tensor_scale a float32 tensor
    of one element on the same device (nvfp4) or None. Checked here, once: a handle is not changed afterwards."""

    __slots__ = ("_codes", "_scales", "_buffer", "fmt", "tensor_scale", "shape", "device", "_codes_ptr", "_scales_ptr",
                 "_packed")

    def __init__(self, codes, scales, fmt, tensor_scale=None):
        _format(fmt)
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
            raise TypeError("codes and scales must be uint8")
        device = codes.device
        if not codes.is_cuda or scales.device != device:
            raise ValueError("codes and scales must be on the same CUDA device")
        shape = codes.shape
        if len(shape) != 2 or shape[1] == 0 or shape[1] % 16:
            raise ValueError("codes must be [rows, columns / 2] with columns a positive multiple of 32")
        rows, columns = shape[0], 2 * shape[1]
        if scales.shape != scale_tiles(rows, columns, fmt):
            raise ValueError(f"scales must be the tiles {scale_tiles(rows, columns, fmt)} of tile_scales")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("codes and scales must be contiguous")
        self._codes, self._scales, self._buffer = codes, scales, None
        self._set(fmt, rows, columns, device, _tensor_scale(tensor_scale, fmt, device), codes.data_ptr(),
                  scales.data_ptr())

    def _set(self, fmt, rows, columns, device, t, codes_ptr, scales_ptr):
        self.fmt, self.tensor_scale, self.shape, self.device = fmt, t, (rows, columns), device
        self._codes_ptr, self._scales_ptr = codes_ptr, scales_ptr
        self._packed = None

    def __reduce__(self):  # copies and pickles: a new handle, of the copies' own addresses
        return Rows, (self.codes, self.scales, self.fmt, self.tensor_scale)

    @classmethod
    def _empty(cls, rows, columns, fmt, t, device):
        """Room for a matrix that a kernel is about to write: one allocation, its views made when they are asked for."""
        self = cls.__new__(cls)
        self._codes = self._scales = None
        self._buffer = torch.empty(_rows_bytes(rows, columns, fmt), dtype=torch.uint8, device=device)
        at = self._buffer.data_ptr()
        self._set(fmt, rows, columns, device, t, at, at + _codes_bytes(rows, columns))
        return self

    @property
    def _operand(self):
        """wdl_fp4_rows, packed once."""
        if self._packed is None:
            t = self.tensor_scale
            self._packed = _native.FP4_ROWS.pack(self._codes_ptr, self._scales_ptr, 0 if t is None else t.data_ptr(),
                                                 FORMAT_CODE[self.fmt])
        return self._packed

    @property
    def codes(self):
        if self._codes is None:
            rows, columns = self.shape
            self._codes = self._buffer[:rows * columns // 2].view(rows, columns // 2)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            self._scales = self._buffer[_codes_bytes(*self.shape):].view(scale_tiles(*self.shape, self.fmt))
        return self._scales


def _codes_bytes(rows, columns):
    return -(-rows * columns // 512) * 256


def _rows_bytes(rows, columns, fmt):
    """Bytes of a matrix's codes, rounded up to 256, and its tiles of scales (as wdl_fp4_linear_workspace counts them)."""
    return -(-rows * columns // 512) * 256 + -(-rows // 128) * -(-columns // (4 * BLOCK[fmt])) * 512


def _format(fmt):
    if fmt not in BLOCK:
        raise ValueError(f"unknown FP4 format {fmt!r}: nvfp4 or mxfp4")
    return FORMAT_CODE[fmt]


def _inference_only(*tensors):
    _native.refuse_gradients("the FP4 operators are", *tensors)


def _tensor_scale(t, fmt, device, name="tensor scale"):
    if t is None:
        return None
    if fmt != "nvfp4":
        raise ValueError(f"mxfp4 takes no {name}")
    if t.dtype != torch.float32 or t.numel() != 1:
        raise TypeError(f"the {name} must be one float32 number")
    if t.device != device:
        raise ValueError(f"the {name} must be on the operands' device")
    if t.requires_grad or forward_ad._current_level >= 0:
        _inference_only(t)
    return t


def _input_rows(x):
    """x [..., K] as the kernels read it: a matrix of rows of consecutive elements, 16-byte aligned."""
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if x.dtype not in _native.DTYPE_CODE:
        raise TypeError("x must be bfloat16, float16 or float32")
    shape = x.shape
    if not shape or shape[-1] == 0 or shape[-1] % 32:
        raise ValueError("x must be [..., K] with K a positive multiple of 32")
    return _native.rows16(x if len(shape) == 2 else x.reshape(-1, shape[-1]))


def _row_stride(x, columns):
    return columns if x.is_contiguous() else max(x.stride(0), columns)


def scale_tiles(rows, columns, fmt):
    """Shape of the tiled scales of a [rows, columns] matrix."""
    return -(-rows // 128), -(-columns // (4 * BLOCK[fmt])), 32, 4, 4


def tile_scales(scales):
    """Scale bytes by row [rows, blocks] (uint8, or float8_e4m3fn) in the kernels' tiles [ceil(rows / 128),
    ceil(blocks / 4), row % 32, row / 32 % 4, block % 4], padded with zeros."""
    scales = scales.view(torch.uint8)
    R, B = scales.shape
    rt, bt = -(-R // 128), -(-B // 4)
    full = torch.zeros(rt * 128, bt * 4, dtype=torch.uint8, device=scales.device)
    full[:R, :B] = scales
    return full.view(rt, 4, 32, bt, 4).permute(0, 3, 2, 1, 4).contiguous()


def untile_scales(tiles, rows, blocks):
    """The inverse of tile_scales: bytes [rows, blocks]."""
    rt, bt = tiles.shape[:2]
    return tiles.permute(0, 3, 2, 1, 4).reshape(rt * 128, bt * 4)[:rows, :blocks].contiguous()


def quantize_rows(x, fmt="nvfp4", tensor_scale=None):
    """Rows of x [M, K] (bfloat16, float16 or float32, CUDA, K a multiple of 32) in FP4: a Rows. tensor_scale (nvfp4):
    a float32 tensor of one element, read on the device."""
    code = _format(fmt)
    if x.requires_grad or forward_ad._current_level >= 0:
        _inference_only(x)
    shape = x.shape
    if len(shape) != 2:
        raise ValueError("x must be [M, K]")
    x = _input_rows(x)
    M, K = shape
    device = x.device
    if _native.elsewhere(device):
        with torch.cuda.device(device):
            return quantize_rows(x, fmt, tensor_scale)
    t = _tensor_scale(tensor_scale, fmt, device)
    rows = Rows._empty(M, K, fmt, t, device)
    status = _native.lib().wdl_fp4_quantize_rows(
        x.data_ptr(), _native.DTYPE_CODE[x.dtype], _row_stride(x, K), M, K, code, _native.ptr(t), rows._codes_ptr,
        rows._scales_ptr, _native.raw_stream(device))
    if status:
        _native.check(status)
    return rows


def dequantize_rows(rows, dtype=torch.bfloat16):
    """The values [M, K] that a Rows stands for, rounded once to dtype (bfloat16, float16 or float32)."""
    if not isinstance(rows, Rows):
        raise TypeError("rows must be fp4.Rows")
    code = _native.DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError("dtype must be bfloat16, float16 or float32")
    M, K = rows.shape
    device, t = rows.device, rows.tensor_scale
    if _native.elsewhere(device):
        with torch.cuda.device(device):
            return dequantize_rows(rows, dtype)
    out = torch.empty(M, K, dtype=dtype, device=device)
    status = _native.lib().wdl_fp4_dequantize_rows(
        rows._codes_ptr, rows._scales_ptr, M, K, FORMAT_CODE[rows.fmt], _native.ptr(t), out.data_ptr(), code, K,
        _native.raw_stream(device))
    if status:
        _native.check(status)
    return out


def _weight(w, name):
    if not isinstance(w, Rows):
        raise TypeError(f"{name} must be fp4.Rows")
    return w


def _bias(bias, N, device, name="bias"):
    if bias is None:
        return None
    if bias.ndim != 1 or bias.shape[0] != N:
        raise ValueError(f"{name} must be [{N}]")
    if bias.device != device:
        raise ValueError(f"{name} must be on the operands' device")
    return bias if bias.dtype == torch.float32 and bias.is_contiguous() else bias.float().contiguous()


def _input(x, w, input_scale):
    """(x as a Rows, or None), (x as a matrix, or None), the leading shape, nvfp4's tensor scale."""
    K = w.shape[1]
    if isinstance(x, Rows):
        if input_scale is not None:
            raise ValueError("a quantized input carries its own tensor scale")
        if x.fmt != w.fmt:
            raise ValueError("x and the weight must be in the same FP4 format")
        if x.device != w.device:
            raise ValueError("x and the weight must be on the same device")
        if x.shape[1] != K:
            raise ValueError(f"x must have {K} columns")
        return x, None, x.shape[:1], None
    t = _tensor_scale(input_scale, w.fmt, w.device, "input scale")
    rows = _input_rows(x)
    if x.device != w.device:
        raise ValueError("x and the weight must be on the same device")
    if rows.shape[1] != K:
        raise ValueError(f"x must have {K} columns")
    return None, rows, x.shape[:-1], t


_NO_UPDATE = (None, 1, 0, None, 0)


def _output(lead, M, N, device, dtype, bias, residual, gate, out):
    """Where a product goes: (the tensor to return, its address, dtype code and row stride, the entry points' gate, groups,
    ld_gate, residual and ldr, and the tensors that have to live until the launch)."""
    if residual is None:
        if gate is not None or out is not None:
            raise ValueError("gate and out belong to a residual")
        code = _native.DTYPE_CODE.get(dtype)
        if code is None:
            raise TypeError("dtype must be bfloat16, float16 or float32")
        y = torch.empty(M, N, dtype=dtype, device=device)
        return y if len(lead) == 1 else y.view(*lead, N), y.data_ptr(), code, N, _NO_UPDATE, None
    if residual.dtype is not torch.float32 or residual.shape != (*lead, N) or residual.device != device:
        raise ValueError(f"residual must be float32 {[*lead, N]} on the operands' device")
    groups, gate_ptr, ld_gate = 1, None, N
    if gate is not None:
        groups = _native.check_modulation(gate, N, device, "gate")
        if M % groups:
            raise ValueError(f"{M} rows do not divide into the gate's {groups} groups")
        gate = _native.modulation_rows(gate, N)
        gate_ptr, ld_gate = gate.data_ptr(), N if gate.ndim == 1 else max(gate.stride(0), N)
    res = _native.flat_rows(residual, N)
    ld_out = N
    if out is None:
        flat = out = torch.empty_like(residual, memory_format=torch.contiguous_format)
    else:
        if out.dtype is not torch.float32 or out.shape != residual.shape or out.device != device:
            raise ValueError("out must be float32, of the residual's shape, on the operands' device")
        flat = out if out.ndim == 2 else out.view(-1, N)
        if N > 1 and flat.stride(1) != 1 or M > 1 and flat.stride(0) < N:
            raise ValueError("out must have consecutive elements in its rows, and rows apart from one another")
        if _native.overlaps(flat, res) or any(t is not None and _native.overlaps(flat, t, False) for t in (gate, bias)):
            raise ValueError("out may be the residual itself, but must not overlap it otherwise, nor the gate or the bias")
        ld_out = _row_stride(flat, N)
    return out, flat.data_ptr(), _native.F32, ld_out, (gate_ptr, groups, ld_gate, res.data_ptr(), _row_stride(res, N)), (gate, res)


def fp4_linear(x, weight, bias=None, *, input_scale=None, dtype=torch.bfloat16, residual=None, gate=None, out=None):
    """y = x W^T + bias in FP4: x [..., K] (bfloat16, float16 or float32, quantized here to the weight's format with
    input_scale, nvfp4's tensor scale) or a Rows already; weight a Rows [N, K]; bias [N]. y [..., N] in dtype.
    With residual [..., N] float32 the gated residual update residual + gate * y instead, float32: gate [N], or [G, N]
    for G groups of consecutive rows (a modulation per frame), None for 1; out: where to write it (the residual itself
    to update it in place; nothing else that is read may overlap it). nvfp4: the two tensor scales are multiplied first, in
    float32, and their product has to be a normal number there."""
    w = _weight(weight, "weight")
    device = w.device
    if _native.elsewhere(device):
        with torch.cuda.device(device):
            return fp4_linear(x, weight, bias, input_scale=input_scale, dtype=dtype, residual=residual, gate=gate, out=out)
    rows, x2, lead, t = _input(x, w, input_scale)
    _inference_only(x2, bias, residual, gate, out)
    N, K = w.shape
    M = (rows or x2).shape[0]
    bias = _bias(bias, N, device)
    result, y, code, ldy, update, kept = _output(lead, M, N, device, dtype, bias, residual, gate, out)
    lib, stream = _native.lib(), _native.raw_stream(device)
    if out is not None and rows is None and M == 1:
        # the product would read x while it writes out: where they share memory (x + W x in place) x is quantized first
        at = x2.data_ptr()
        if at < y + N * 4 and y < at + K * x2.element_size():
            rows = quantize_rows(x2, w.fmt, t)
    if rows is None:
        need, at = 0, None
        if M != 1:  # (a single row is quantized by its product)
            need = _rows_bytes(M, K, w.fmt)
            work = torch.empty(need, dtype=torch.uint8, device=device)
            at = work.data_ptr()
        status = lib.wdl_fp4_linear(x2.data_ptr(), _native.DTYPE_CODE[x2.dtype], _row_stride(x2, K), _native.ptr(t),
                                    w._operand, _native.ptr(bias), *update, M, N, K, y, code, ldy, at, need, stream)
    elif residual is None:
        status = lib.wdl_fp4_gemm(rows._operand, w._operand, _native.ptr(bias), M, N, K, y, code, ldy, stream)
    else:
        status = lib.wdl_fp4_gemm_residual(rows._operand, w._operand, _native.ptr(bias), *update, M, N, K, y, ldy, stream)
    if status:
        _native.check(status)
    return result


def fp4_gelu_mlp(x, weight1, bias1, weight2, bias2, *, input_scale=None, hidden_scale=None, dtype=torch.bfloat16,
                 residual=None, gate=None, out=None):
    """The feed forward GELU_tanh(x W1^T + b1) W2^T + b2 in FP4 (the shape of w4a4_gelu_mlp): the first product's
    epilogue writes the hidden layer [M, H] in the weights' format, with hidden_scale its tensor scale (nvfp4). Other
    arguments as fp4_linear."""
    w1, w2 = _weight(weight1, "weight1"), _weight(weight2, "weight2")
    device = w1.device
    if _native.elsewhere(device):
        with torch.cuda.device(device):
            return fp4_gelu_mlp(x, weight1, bias1, weight2, bias2, input_scale=input_scale, hidden_scale=hidden_scale,
                                dtype=dtype, residual=residual, gate=gate, out=out)
    rows, x2, lead, t = _input(x, w1, input_scale)
    _inference_only(x2, bias1, bias2, residual, gate, out)
    (H, K), N, fmt = w1.shape, w2.shape[0], w1.fmt
    if w2.fmt != fmt or w2.device != device or w2.shape[1] != H:
        raise ValueError(f"weight2 must have {H} columns, in weight1's format and on its device")
    th = _tensor_scale(hidden_scale, fmt, device, "hidden scale")
    M = (rows or x2).shape[0]
    bias1, bias2 = _bias(bias1, H, device, "bias1"), _bias(bias2, N, device, "bias2")
    result, y, code, ldy, update, kept = _output(lead, M, N, device, dtype, bias2, residual, gate, out)
    need = _rows_bytes(M, H, fmt)
    if rows is None:
        if M != 1:  # (a single row is quantized by its product)
            need += _rows_bytes(M, K, fmt)
        source = x2.data_ptr(), _native.DTYPE_CODE[x2.dtype], _row_stride(x2, K), _native.ptr(t), None
    else:
        source = None, 0, K, None, rows._operand
    work = torch.empty(need, dtype=torch.uint8, device=device)
    status = _native.lib().wdl_fp4_gelu_mlp(
        *source, w1._operand, _native.ptr(bias1), _native.ptr(th), w2._operand, _native.ptr(bias2), *update, M, H, N, K, y,
        code, ldy, work.data_ptr(), need, _native.raw_stream(device))
    if status:
        _native.check(status)
    return result


@torch.no_grad()
def quantize(weight, bias=None, fmt="nvfp4"):
    """A float layer as its FP4 parts: codes [N, K / 2], scales by row [N, K / block], tensor_scale (nvfp4: the largest
    finite magnitude over 6 * 448, so that its block's scale is E4M3's largest; else None) and bias (float32 or None).
    weight [N, K] on a GPU."""
    _format(fmt)
    t = None
    if fmt == "nvfp4":
        top = weight.detach().nan_to_num(0.0, 0.0, 0.0).abs().max().float() / (E2M1_MAX * E4M3_MAX)
        t = torch.where(top > 0, top, torch.ones_like(top)).reshape(1)
    rows = quantize_rows(weight.detach(), fmt, t)
    N, K = rows.shape
    return dict(codes=rows.codes, scales=untile_scales(rows.scales, N, K // BLOCK[fmt]), tensor_scale=t,
                bias=None if bias is None else bias.detach().float())


def _fmt_of(codes, scales):
    for fmt, block in BLOCK.items():
        if scales.ndim == 2 and scales.shape == (codes.shape[0], codes.shape[1] * 2 // block):
            return fmt
    raise ValueError("scales must be [N, K / 16] (nvfp4) or [N, K / 32] (mxfp4)")


class PackedFp4Linear(torch.nn.Module):
    """A linear layer from the parts of quantize() (the FP4 counterpart of PackedW4A4Linear): scales are laid out in
    tiles once, here. input_scale: nvfp4's tensor scale of its input (a float32 number or tensor), None for 1."""

    def __init__(self, codes, scales, tensor_scale=None, bias=None, input_scale=None):
        super().__init__()
        self.fmt = _fmt_of(codes, scales)
        one = lambda t: None if t is None else torch.as_tensor(t, dtype=torch.float32, device=codes.device).reshape(1)  # noqa: E731
        self.register_buffer("codes", codes.contiguous())
        self.register_buffer("tiles", tile_scales(scales))
        self.register_buffer("tensor_scale", one(tensor_scale))
        self.register_buffer("bias", bias)
        self.register_buffer("input_scale", one(input_scale))

    def _apply(self, fn, recurse=True):
        """Moves as any module's; a cast of a model to another dtype leaves the scales and the bias as they are (they are
        numbers of the format and the epilogue's float32, not activations)."""
        kept = {name: getattr(self, name) for name in ("tensor_scale", "input_scale", "bias")}
        super()._apply(fn, recurse)
        for name, old in kept.items():
            new = getattr(self, name)
            if old is not None and new.dtype is not old.dtype:
                setattr(self, name, old.to(new.device))
        return self

    def rows(self):
        return Rows(self.codes, self.tiles, self.fmt, self.tensor_scale)

    def forward(self, X, **options):
        scale = None if isinstance(X, Rows) else self.input_scale  # a quantized input carries its own
        return fp4_linear(X, self.rows(), self.bias, input_scale=scale, **options)


class PackedFp4GeluMLP(torch.nn.Module):
    """The feed forward of two PackedFp4Linear layers (the FP4 counterpart of PackedW4A4GeluMLP); the second's
    input_scale is the hidden layer's tensor scale."""

    def __init__(self, fc1, fc2):
        super().__init__()
        if fc1.fmt != fc2.fmt or fc2.codes.shape[1] * 2 != fc1.codes.shape[0]:
            raise ValueError("the layers must be in one format, the second as wide as the first is high")
        self.fc1, self.fc2 = fc1, fc2

    def forward(self, X, **options):
        a, b = self.fc1, self.fc2
        scale = None if isinstance(X, Rows) else a.input_scale
        return fp4_gelu_mlp(X, a.rows(), a.bias, b.rows(), b.bias, input_scale=scale, hidden_scale=b.input_scale, **options)
