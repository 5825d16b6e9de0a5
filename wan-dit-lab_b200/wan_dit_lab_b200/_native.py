"""ctypes binding of libwdl_b200.so (include/wdl_b200.h): the only way this package reaches the GPU kernels.

The library is loaded on first use and must exist: there is no fallback to PyTorch or CPU code. A nonzero
status of an entry point becomes an exception carrying the library's message: ValueError for invalid
arguments (nothing was launched), RuntimeError otherwise.
"""

import ctypes
import struct
from pathlib import Path

import torch
from torch.autograd import forward_ad

LIBRARY = Path(__file__).resolve().parent / "libwdl_b200.so"

OK, ERR_ARGUMENT, ERR_UNSUPPORTED, ERR_CUDA, ERR_DEVICE = 0, 1, 2, 3, 4
BF16, F16, F32 = 0, 1, 2
NVFP4, MXFP4 = 0, 1
OUT_NVFP4, OUT_MXFP4 = 3, 4
CODES_INT8, CODES_E4M3, CODES_F16_FOLD, CODES_F16_PRE = 0, 1, 3, 4
DTYPE_CODE = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}

_P, _I, _I64, _SZ, _U32P = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.POINTER(ctypes.c_uint32)



class LowRank(ctypes.Structure):
    """wdl_lowrank (include/wdl_b200.h): an SVDQuant low-rank branch formed in the GEMM epilogue, act [M, ld_act]
    float32 = x proj_down, up [N, rank] float32 = proj_up, rank a multiple of 4. Whoever makes one keeps the
    tensors it points to alive until the GEMM has run (attributes set on the instance do)."""
    _fields_ = [("act", ctypes.c_void_p), ("ld_act", ctypes.c_int64), ("up", ctypes.c_void_p), ("rank", ctypes.c_int)]


_LRP = ctypes.POINTER(LowRank)


# wdl_fp4_rows and wdl_gated_norm_args (include/wdl_b200.h), packed in one call and passed as bytes: filling a
# ctypes.Structure of 26 fields takes as long as a launch. Null pointers are 0.
FP4_ROWS = struct.Struct("@PPPi4x")
GATED_NORM = struct.Struct("@PqPqPqPPPqPqPqPqPP7if")
_PACKED = ctypes.c_char_p

# name: (restype, argtypes), in the order of include/wdl_b200.h
SIGNATURES = {
    "wdl_last_error": (ctypes.c_char_p, []),
    "wdl_version": (ctypes.c_char_p, []),
    "wdl_device_error": (_I, [_P, _U32P]),
    "wdl_w4a4_quantize_rows": (_I, [_P, _I, _I64, _P, _I, _I, _I, _I, _P, _P, _P, _P]),
    "wdl_w4a4_unpack_weight": (_I, [_P, _P, _I, _I, _I, _I, _P, _P, _P]),
    "wdl_w4a4_fold_weight": (_I, [_P, _P, _I, _I, _I, _I, _P, _P, _P]),
    "wdl_w4a4_gemm": (_I, [_P, _P, _P, _P, _I, _P, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_residual": (_I, [_P, _P, _P, _P, _I, _P, _P, _P, _I64, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_group_partials": (_I, [_P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_add": (_I, [_P, _P, _P, _P, _I, _P, _P, _I64, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_residual_add": (_I, [_P, _P, _P, _P, _I, _P, _P, _I64, _P, _P, _I64, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_gelu_u4_add": (_I, [_P, _P, _P, _P, _I, _P, _P, _I64, _P, ctypes.c_float, _I, _I, _I, _I, _P,
                                       _I64, _P, _P, _I64, _P]),
    "wdl_lowrank_down": (_I, [_P, _I, _I64, _I, _I, _P, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_lowrank": (_I, [_P, _P, _P, _P, _I, _P, _LRP, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_residual_lowrank": (_I, [_P, _P, _P, _P, _I, _P, _LRP, _P, _P, _I64, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_gelu_u4_lowrank": (_I, [_P, _P, _P, _P, _I, _P, _LRP, _P, ctypes.c_float, _I, _I, _I, _I, _P,
                                           _I64, _P, _P, _I64, _P]),
    "wdl_w4a4_gemm_f32": (_I, [_P, _P, _P, _P, _I, _P, _P, _I64, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_gemm_f32_lowrank": (_I, [_P, _P, _P, _P, _I, _P, _LRP, _I, _I, _I, _P, _I64, _P]),
    "wdl_w4a4_linear_workspace": (_SZ, [_I, _I]),
    "wdl_w4a4_linear": (_I, [_P, _I64, _I, _I, _P, _I, _P, _P, _I, _P, _I, _P, _I64, _P, _SZ, _P]),
    "wdl_w4a4_linear_noalloc": (_I, [_P, _I64, _I, _I, _P, _I, _P, _P, _I, _P, _I, _P, _I64, _P]),
    "wdl_store_kv_fp8": (_I, [_P, _I, _P, _P, _I, _P, _I, _I, _I, _I, _P, _P, _P, _P, _I, _I, _P]),
    "wdl_rope_apply": (_I, [_P, _I, _P, _I, _I, _I, _I, _P, _P, _I, _P, _I, _I, _P, _I, _P]),
    "wdl_qkv_prep": (_I, [_P, _I64, _I, _I, _P, _P, ctypes.c_float, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P,
                          _I, _I, _P]),
    "wdl_qkv_prep_sharded": (_I, [_P, _I64, _I, _I, _P, _P, ctypes.c_float, _P, _I, _P, _I, _I, _I, _I, _P, _P, _P,
                                  _P, _P, _P, _I, _I, _P]),
    "wdl_w4a4_gemm_gelu_u4": (_I, [_P, _P, _P, _P, _I, _P, _P, ctypes.c_float, _I, _I, _I, _I, _P, _I64, _P, _P]),
    "wdl_ln_quant": (_I, [_P, _I, _I64, _I, _I, ctypes.c_float, _P, _P, _I, _P, _P, _P, _I, _I, _P, _P, _P]),
    "wdl_ln_quant_keep": (_I, [_P, _I, _I64, _I, _I, ctypes.c_float, _P, _P, _I, _P, _P, _P, _I, _I, _P, _P, _P,
                               _I64, _P]),
    "wdl_rms_rows": (_I, [_P, _I64, _I, _I, _P, ctypes.c_float, _P, _I64, _P]),
    "wdl_rms_rows_sharded": (_I, [_P, _I64, _I, _I, _P, ctypes.c_float, _P, _I, _P, _I64, _P]),
    "wdl_rows_sumsq": (_I, [_P, _I64, _I, _I, _I, _I64, _P, _P]),
    "wdl_residual_update": (_I, [_P, _I64, _P, _P, _P, _I64, _I, _I, _P]),
    "wdl_modulation": (_I, [_P, _P, _I, _I, _P, _P]),
    "wdl_sage_prep_kv": (_I, [_P, _P, _P, _P, _I, _P, _I, _I64, _P, _I, _I64, _I, _I, _P, _P, _P, _P, _P, _SZ, _P]),
    "wdl_sage_quant_q": (_I, [_P, _I64, _I, _I, _P, _P, _P]),
    "wdl_sage_prep_workspace": (_SZ, [_I, _I]),
    "wdl_sage_prep": (_I, [_P, _I64, _I, _P, _P, _P, _P, _I, _P, _I, _I64, _P, _I, _I64, _I, _I, _P, _P, _P, _P, _P,
                           _P, _P, _SZ, _P]),
    "wdl_sage_attention": (_I, [_P, _P, _P, _P, _P, _P, _I, _I, _I, ctypes.c_float, _P, _I64, _P]),
    "wdl_sage_attend_workspace": (_SZ, [_I, _I, _I]),
    "wdl_sage_attend": (_I, [_P, _I64, _I, _P, _P, _P, _P, _I, _P, _I, _I64, _P, _I, _I64, _I, _I, ctypes.c_float,
                             _P, _I64, _P, _SZ, _P]),
    "wdl_sage_attend_maps": (_I, [_P, _I64, _I, _P, _P, _P, _P, _I, _I, _P, _P, _I, _P, _I, _I64, _P, _I, _I64, _I,
                                  _I, ctypes.c_float, _P, _I64, _P, _SZ, _P]),
    "wdl_fp4_scale_bytes": (_SZ, [_I, _I, _I]),
    "wdl_fp4_quantize_rows": (_I, [_P, _I, _I64, _I, _I, _I, _P, _P, _P, _P]),
    "wdl_fp4_dequantize_rows": (_I, [_P, _P, _I, _I, _I, _P, _P, _I, _I64, _P]),
    "wdl_fp4_gemm": (_I, [_PACKED, _PACKED, _P, _I, _I, _I, _P, _I, _I64, _P]),
    "wdl_fp4_gemm_rows_per_cta": (_I, [_I, _I, _I, _I]),
    "wdl_fp4_gemm_residual": (_I, [_PACKED, _PACKED, _P, _P, _I, _I64, _P, _I64, _I, _I, _I, _P, _I64, _P]),
    "wdl_fp4_gemm_gelu": (_I, [_PACKED, _PACKED, _P, _I, _I, _I, _P, _P, _P, _P]),
    "wdl_fp4_linear_workspace": (_SZ, [_I, _I, _I]),
    "wdl_fp4_linear": (_I, [_P, _I, _I64, _P, _PACKED, _P, _P, _I, _I64, _P, _I64, _I, _I, _I, _P, _I, _I64, _P, _SZ, _P]),
    "wdl_fp4_gelu_mlp_workspace": (_SZ, [_I, _I, _I, _I]),
    "wdl_fp4_gelu_mlp": (_I, [_P, _I, _I64, _P, _PACKED, _PACKED, _P, _P, _PACKED, _P, _P, _I, _I64, _P, _I64, _I, _I, _I, _I,
                              _P, _I, _I64, _P, _SZ, _P]),
    "wdl_gated_norm": (_I, [_PACKED, _P]),
}

_lib = None


def lib():
    """The loaded library, with the argument types of every entry point declared."""
    global _lib
    if _lib is None:
        if not LIBRARY.exists():
            raise RuntimeError(f"{LIBRARY} is not built: run `python wan-dit-lab_b200/build.py`")
        handle = ctypes.CDLL(str(LIBRARY))
        for name, (restype, argtypes) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype, fn.argtypes = restype, argtypes
        _lib = handle
    return _lib


def check(status):
    """Raises for a nonzero status of an entry point."""
    if status == OK:
        return
    message = lib().wdl_last_error().decode()
    raise (ValueError if status == ERR_ARGUMENT else RuntimeError)(message)


def ptr(tensor):
    """Device address of a tensor (None for None)."""
    return None if tensor is None else tensor.data_ptr()


def stream(device=None):
    """The current PyTorch CUDA stream of `device`, as the library takes it."""
    return torch.cuda.current_stream(device).cuda_stream


def elsewhere(device):
    """Whether another device than the tensors' is current (switching costs microseconds: only where it must be)."""
    return device.index != torch._C._cuda_getDevice()


def raw_stream(device):
    """The current stream of a tensor's device as the library takes it, without the Stream object that stream() makes."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def refuse_gradients(what, *tensors):
    """Refuses tensors (None among them) that autograd would follow: what requires a gradient where gradients are recorded,
    and dual tensors of forward mode, whose tangents a kernel would drop (torch.no_grad does not turn these off)."""
    grad, dual = torch.is_grad_enabled(), forward_ad._current_level >= 0
    if grad or dual:
        for t in tensors:
            if t is not None and (grad and t.requires_grad or dual and forward_ad.unpack_dual(t).tangent is not None):
                raise ValueError(f"{what} inference-only")


def rows16(x):
    """A matrix [M, K], K a multiple of 8, with consecutive elements in rows that begin on 16-byte boundaries: x itself, or
    a copy."""
    if x.is_contiguous():  # rows of whole 16 bytes follow one another
        if not x.data_ptr() & 15:
            return x
    elif x.stride(1) == 1 and not x.data_ptr() & 15 and x.stride(0) >= x.shape[1] and not (
            x.stride(0) * x.element_size() & 15):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def flat_rows(x, columns):
    """x [..., columns] as a matrix with consecutive elements in its rows: a view, or a copy."""
    x = x if x.ndim == 2 else x.reshape(-1, columns)
    if x.is_contiguous() or x.stride(1) == 1 and x.stride(0) >= columns:
        return x
    return x.contiguous()


def overlaps(out, t, in_place=True):
    """Whether the rows of `t` (a matrix or a vector with consecutive elements) lie in the rows that `out` is about to be
    written to. in_place: but for the very same rows, all of them. That is right for what a kernel reads element by
    element just before it writes that one (a residual, a branch); anything else, a modulation row or a bias, is read for
    other elements too and by then may hold what was written."""
    rows, columns = out.shape
    count, width = t.shape if t.ndim == 2 else (1, t.shape[0])
    if 0 in (rows, columns, count, width):
        return False
    size, size_t = out.element_size(), t.element_size()
    step, step_t = out.stride(0) * size, t.stride(0) * size_t if t.ndim == 2 else 0
    at, at_t = out.data_ptr(), t.data_ptr()
    if at + (rows - 1) * step + columns * size <= at_t or at_t + (count - 1) * step_t + width * size_t <= at:
        return False
    same = rows == 1 == count or step == step_t
    if in_place and at == at_t and same and (rows, columns, out.dtype) == (count, width, t.dtype):
        return False
    apart = (at_t - at) % step if same and step else 0  # rows side by side in one buffer
    return not (apart >= columns * size and apart + width * size_t <= step)


def check_modulation(t, columns, device, name):
    """Refuses what is not a vector [columns] or rows [G, columns] on `device`; the number of rows."""
    if t.ndim not in (1, 2) or t.shape[-1] != columns or t.shape[0] == 0:
        raise ValueError(f"{name} must be [{columns}] or [groups, {columns}]")
    if t.device != device:
        raise ValueError(f"{name} must be on the same device as what it modulates")
    return 1 if t.ndim == 1 else t.shape[0]


def modulation_rows(t, columns, align=False):
    """A checked modulation vector or rows as float32, any stride between rows; align: rows on 16-byte boundaries."""
    if t.dtype is not torch.float32:
        t = t.float()
    if t.ndim == 1:
        if t.is_contiguous() and not (align and t.data_ptr() & 15):
            return t
        return t.clone(memory_format=torch.contiguous_format)
    return rows16(t) if align else flat_rows(t, columns)


def device_error(device=None):
    """Synchronises the current stream and reads (and clears) the device error word: 0, or raises RuntimeError
    naming the code a kernel recorded since the last check (a bounded wait given up, or an index map entry out of
    range)."""
    code = ctypes.c_uint32(0)
    check(lib().wdl_device_error(stream(device), ctypes.byref(code)))
    return code.value
