"""The gated residual update of a block and the normalization and modulation that follow it, in one kernel:

    x' = x + gate y                                   stored in x's type, and normalized as stored
    h  = (norm(x') weight + bias) (1 + scale) + shift

what a Wan block does between two of its branches (reference models/block.py:75-79: the residual updates, norm1 / norm2
with their modulation, norm3 with its affine part), h leaving in 16 or 32 bits or as the FP4 operand of the next layer
(quantization/fp4.py). Inference only.
"""

import torch

from wan_dit_lab_b200 import _native
from wan_dit_lab_b200.quantization import fp4
from wan_dit_lab_b200.quantization.fp4 import _row_stride

_OUT = {torch.bfloat16: _native.BF16, torch.float16: _native.F16, torch.float32: _native.F32,
        "nvfp4": _native.OUT_NVFP4, "mxfp4": _native.OUT_MXFP4}
_STREAM = (torch.bfloat16, torch.float32)


def _modulation(t, columns, device, name):
    """(rows, address, stride, tensor) of a modulation vector or rows, checked and as the kernel reads them; (1, 0, 0,
    None) for None."""
    if t is None:
        return 1, 0, 0, None
    count = _native.check_modulation(t, columns, device, name)
    t = _native.modulation_rows(t, columns, align=True)
    return count, t.data_ptr(), columns if count == 1 else _row_stride(t, columns), t


def _spread(t, columns, groups):
    """One modulation row for all of the groups: (address, stride, tensor)."""
    t = t.expand(groups, columns).contiguous()
    return t.data_ptr(), columns, t


def gated_norm(x, y=None, gate=None, *, weight=None, bias=None, shift=None, scale=None, eps=1e-6, kind="layer",
               out=torch.bfloat16, tensor_scale=None, inplace=False):
    """(x', h) for the stream x [M, K] (bfloat16 or float32) and the branch y [M, K] (bfloat16 or float32; None: x' is
    x). kind "layer" (LayerNorm) or "rms" (x / sqrt(mean x^2 + eps)); weight and bias [K]; gate, shift and scale [K],
    or [G, K] for G groups of consecutive rows (a modulation per frame). out: h's dtype (bfloat16, float16, float32), or
    "nvfp4" (with tensor_scale) or "mxfp4" for a fp4.Rows. inplace: x' is written over x (y may be x, but nothing else may
    overlap it). K a multiple of 8 (FP4: 32), at most 16384."""
    if kind not in ("layer", "rms"):
        raise ValueError("kind must be 'layer' or 'rms'")
    if out not in _OUT:
        raise TypeError("out must be bfloat16, float16, float32, 'nvfp4' or 'mxfp4'")
    four = isinstance(out, str)
    if tensor_scale is not None and out != "nvfp4":
        raise ValueError("only nvfp4 takes a tensor scale")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0 or shape[1] % (32 if four else 8) or shape[1] > 16384:
        raise ValueError("x must be [M, K] with K a positive multiple of 8 (32 for an FP4 output), at most 16384")
    if x.dtype not in _STREAM:
        raise TypeError("x must be bfloat16 or float32")
    M, K = shape
    dev = x.device
    if _native.elsewhere(dev):
        with torch.cuda.device(dev):
            return gated_norm(x, y, gate, weight=weight, bias=bias, shift=shift, scale=scale, eps=eps, kind=kind, out=out,
                              tensor_scale=tensor_scale, inplace=inplace)
    _native.refuse_gradients("gated_norm is", x, y, gate, weight, bias, shift, scale)
    if y is None:
        if gate is not None or inplace:
            raise ValueError("gate and inplace belong to a branch y")
    else:
        if y.shape != shape or y.device != dev:
            raise ValueError("y must have x's shape and device")
        if y.dtype not in _STREAM:
            raise TypeError("y must be bfloat16 or float32")
    # every tensor that the launch reads has a name here, so that it lives until it is enqueued
    n_g, g_ptr, g_ld, g = _modulation(gate, K, dev, "gate")
    n_h, h_ptr, h_ld, sh = _modulation(shift, K, dev, "shift")
    n_c, c_ptr, c_ld, sc = _modulation(scale, K, dev, "scale")
    groups = max(n_g, n_h, n_c)
    if groups > 1:
        if M % groups:
            raise ValueError(f"{M} rows do not divide into {groups} groups")
        if not {n_g, n_h, n_c} <= {1, groups}:
            raise ValueError("gate, shift and scale must have the same number of groups")
        if g is not None and n_g == 1:
            g_ptr, g_ld, g = _spread(g, K, groups)
        if sh is not None and n_h == 1:
            h_ptr, h_ld, sh = _spread(sh, K, groups)
        if sc is not None and n_c == 1:
            c_ptr, c_ld, sc = _spread(sc, K, groups)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (K,) or t.device != dev):
            raise ValueError(f"{name} must be [{K}] on x's device")
    source = _native.rows16(x)
    if inplace and source is not x:
        raise ValueError("an in-place stream needs consecutive elements and 16-byte aligned rows")
    w = None if weight is None else _native.modulation_rows(weight, K, align=True)
    b = None if bias is None else _native.modulation_rows(bias, K, align=True)
    t = None if tensor_scale is None else fp4._tensor_scale(tensor_scale, "nvfp4", dev)
    stored, y_ptr, ldy, y_code, out_ptr, ldo = source, 0, 0, 0, 0, 0
    if y is not None:
        y = _native.rows16(y)
        y_ptr, ldy, y_code = y.data_ptr(), _row_stride(y, K), _native.DTYPE_CODE[y.dtype]
        if inplace:
            if _native.overlaps(x, y) or any(r is not None and _native.overlaps(x, r, False) for r in (g, sh, sc, w, b)):
                raise ValueError("what the kernel reads must not overlap an in-place stream (y may be the stream itself)")
        else:
            stored = torch.empty(M, K, dtype=x.dtype, device=dev)
        out_ptr, ldo = stored.data_ptr(), _row_stride(stored, K)
    if four:
        h = fp4.Rows._empty(M, K, out, t, dev)
        codes, scales = h._codes_ptr, h._scales_ptr
    else:
        h = torch.empty(M, K, dtype=out, device=dev)
        codes, scales = h.data_ptr(), 0
    if M:
        status = _native.lib().wdl_gated_norm(_native.GATED_NORM.pack(
            source.data_ptr(), _row_stride(source, K), y_ptr, ldy, g_ptr, g_ld,
            0 if w is None else w.data_ptr(), 0 if b is None else b.data_ptr(), h_ptr, h_ld, c_ptr, c_ld,
            out_ptr, ldo, codes, K, scales, 0 if t is None else t.data_ptr(), _native.DTYPE_CODE[x.dtype], y_code, M, K,
            groups, kind == "rms", _OUT[out], eps), _native.raw_stream(dev))
        if status:
            _native.check(status)
    return (x if y is None or inplace else stored), h
