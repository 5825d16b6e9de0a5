"""The FP4 operators measured: rows quantized to microscaled 4-bit floating point (NVFP4 and MXFP4), the linear layer
and the GELU feed forward over such operands, and the gated residual update with the normalization that follows it.

`own` False runs each operator in elementary torch operations (float32, rounded once at the end); `own` True calls
the package's operators on the same state.

The two formats. A value is an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; two codes a byte, the low nibble the
even column) times its block's scale:
  nvfp4  blocks of 16 columns, scale s in E4M3, times one float32 t for the whole tensor (1 when absent):
         s = E4M3(max|x| / (6 t)), at least 2^-9 and at most 448; code = E2M1(x / (s t))
  mxfp4  blocks of 32 columns, scale 2^e in E8M0, e = floor(log2 max|x|) - 2; code = E2M1(x / 2^e)
both rounded to the nearest, ties to the even code, magnitudes above 6 to 6.
"""

import math
import sys
from pathlib import Path

import torch

own = False

F4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = {"nvfp4": 16, "mxfp4": 32}
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
DEVICE = "cuda"


def _fp4():
    _package()
    from wan_dit_lab_b200.quantization import fp4
    return fp4


def _gated_norm():
    _package()
    from wan_dit_lab_b200.kernels.gated_norm import gated_norm
    return gated_norm


def _package():
    root = str(Path.cwd() / "wan-dit-lab_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


# ---- cases

def listed():
    return [
        # one token's activations on their way into a layer: the smallest call
        dict(name="quantize token", op="quantize", fmt="nvfp4", M=1, K=3072, dtype="bfloat16", scaled=False),
        # a feed forward's hidden layer of one chunk (3 latent frames of 512 x 928, 1392 tokens) held in float32
        dict(name="quantize hidden", op="quantize", fmt="mxfp4", M=1392, K=14336, dtype="float32", scaled=False),
        # the projection of one timestep's embedding to the six modulation rows
        dict(name="linear time", op="linear", fmt="nvfp4", M=1, K=3072, N=18432, dtype="bfloat16", out="bfloat16",
             bias=True, gated=False, scaled=False),
        # a prompt of odd length through the text embedding's first layer, in float16
        dict(name="linear text", op="linear", fmt="mxfp4", M=77, K=4096, N=3072, dtype="float16", out="float16",
             bias=True, gated=False, scaled=False),
        # query, key and value of a chunk, activations with a calibrated tensor scale
        dict(name="linear qkv", op="linear", fmt="nvfp4", M=1392, K=3072, N=9216, dtype="bfloat16", out="bfloat16",
             bias=True, gated=False, scaled=True),
        # the attention's output projection onto the float32 residual stream, gated
        dict(name="linear out", op="linear", fmt="nvfp4", M=1392, K=3072, N=3072, dtype="bfloat16", out="float32",
             bias=True, gated=True, scaled=False),
        # the first feed forward layer alone on a 704 x 1280 chunk of 8 frames: the largest product
        dict(name="linear wide", op="linear", fmt="mxfp4", M=7040, K=3072, N=14336, dtype="bfloat16", out="bfloat16",
             bias=False, gated=False, scaled=False),
        # the whole feed forward of a chunk, and of a few tokens
        dict(name="mlp chunk", op="mlp", fmt="nvfp4", M=1392, K=3072, H=14336, N=3072, dtype="bfloat16", scaled=True),
        dict(name="mlp few", op="mlp", fmt="mxfp4", M=19, K=3072, H=14336, N=3072, dtype="bfloat16", scaled=False),
        # the gated residual update of a chunk, then LayerNorm and modulation straight into the next layer's operand
        dict(name="norm chunk", op="norm", M=1392, K=3072, x="float32", y="bfloat16", groups=1, kind="layer",
             affine=False, out="nvfp4"),
        # the same with a timestep per frame (8 frames of 880 tokens) on a bfloat16 stream, for a 16-bit consumer
        dict(name="norm frames", op="norm", M=7040, K=3072, x="bfloat16", y="bfloat16", groups=8, kind="layer",
             affine=False, out="bfloat16"),
        # one token, RMS normalization with a weight
        dict(name="norm token", op="norm", M=1, K=3072, x="float32", y="float32", groups=1, kind="rms", affine=True,
             out="float32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _channels(rng, low, high, step=32):
    return max(step, _log(rng, low, high) // step * step)


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "mlp", "norm"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    scaled = fmt == "nvfp4" and rng.random() < 0.5
    M = _log(rng, 1, 7040)
    if op == "quantize":
        K = _channels(rng, 64, 14336)
        return dict(op=op, fmt=fmt, M=min(M, 1392 * 14336 // K), K=K, dtype=dtype, scaled=scaled)
    if op == "linear":
        K, N = _channels(rng, 64, 14336), _log(rng, 16, 14336)
        M = min(M, 7040 * 3072 * 14336 // (K * max(N, 512)))
        gated = rng.random() < 0.3
        out = "float32" if gated else rng.choice(["bfloat16", "float16", "float32"])
        return dict(op=op, fmt=fmt, M=M, K=K, N=N, dtype=dtype, out=out, bias=rng.random() < 0.7, gated=gated,
                    scaled=scaled)
    if op == "mlp":
        K, H, N = _channels(rng, 256, 3072), _channels(rng, 512, 14336), _log(rng, 128, 3072)
        return dict(op=op, fmt=fmt, M=min(M, 1392), K=K, H=H, N=N, dtype=dtype, scaled=scaled)
    groups = rng.choice([1, 1, 3, 8])
    K = _channels(rng, 64, 8192)
    M = max(1, min(M, 7040 * 3072 // K) // groups) * groups
    x, y = rng.choice([("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16")])
    return dict(op=op, M=M, K=K, x=x, y=y, groups=groups, kind=rng.choice(["layer", "rms"]),
                affine=rng.random() < 0.5, out=rng.choice(["nvfp4", "mxfp4", "bfloat16", "float32"]))


def work(case):
    M, K, op = case["M"], case["K"], case["op"]
    size = {"bfloat16": 2, "float16": 2, "float32": 4}
    four = lambda rows, cols, fmt: rows * cols // 2 + rows * cols // BLOCK[fmt]  # noqa: E731
    if op == "quantize":  # the values in; codes and scales out and in again; the values they stand for (bfloat16) out
        return {"bytes": M * K * (size[case["dtype"]] + 2) + 2 * four(M, K, case["fmt"]), "flops": 4 * M * K}
    if op == "linear":
        N = case["N"]
        extra = 4 * N * case["bias"] + (4 * M * N + 4 * N) * case["gated"]
        return {"bytes": M * K * size[case["dtype"]] + four(N, K, case["fmt"]) + M * N * size[case["out"]] + extra,
                "flops": 2 * M * N * K}
    if op == "mlp":
        H, N = case["H"], case["N"]
        return {"bytes": M * K * size[case["dtype"]] + four(H, K, case["fmt"]) + four(N, H, case["fmt"])
                + 4 * (H + N) + 2 * M * N, "flops": 2 * M * H * (K + N)}
    out = 2 * M * K + 2 * four(M, K, case["out"]) if case["out"] in BLOCK else M * K * size[case["out"]]
    return {"bytes": M * K * (2 * size[case["x"]] + size[case["y"]]) + out + 12 * case["groups"] * K
            + 8 * K * case["affine"], "flops": 12 * M * K}


# ---- inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _activations(g, M, K, dtype):
    """Normalized activations: unit variance, channels of different size, a few channels far larger."""
    channel = torch.exp(0.5 * torch.randn(K, generator=g, device=DEVICE))
    channel[torch.randint(0, K, (max(1, K // 256),), generator=g, device=DEVICE)] *= 8.0
    return (torch.randn(M, K, generator=g, device=DEVICE) * channel).to(DTYPES[dtype])


def _tensor_scale(x, spread=0.0):
    """The largest magnitude over 6 * 448; an activation's comes from calibration data, not from these inputs."""
    return ((x.abs().max().float() / 2688.0) * (1.0 + spread)).reshape(1)


def tiled(scales):
    """Scale bytes [rows, blocks] in the layout the tensor cores read: tiles of 128 rows x 4 blocks, 512 bytes each
    and one after another along the blocks, inside a tile [row % 32, row / 32, block]; padding holds zeros."""
    R, B = scales.shape
    rt, bt = -(-R // 128), -(-B // 4)
    full = torch.zeros(rt * 128, bt * 4, dtype=torch.uint8, device=scales.device)
    full[:R, :B] = scales
    return full.view(rt, 4, 32, bt, 4).permute(0, 3, 2, 1, 4).contiguous()


def _weight(g, N, K, fmt, state, name):
    """A layer's weight as a converted checkpoint holds it: codes, scales by row and in tiles, the tensor scale."""
    W = torch.randn(N, K, generator=g, device=DEVICE) * 0.02
    t = _tensor_scale(W) if fmt == "nvfp4" else None
    codes, scales = encode(W, fmt, t)
    state[name] = dict(codes=codes, scales=scales, tiles=tiled(scales), t=t)


def prepare(case, seed):
    g = _generator(seed)
    M, K, op = case["M"], case["K"], case["op"]
    s = dict(case=case)
    if op == "norm":
        s["x"] = (_activations(g, M, K, "float32") * 2.0).to(DTYPES[case["x"]])
        s["y"] = torch.randn(M, K, generator=g, device=DEVICE).to(DTYPES[case["y"]])
        rows = torch.randn(case["groups"], 3, K, generator=g, device=DEVICE) * 0.3
        s["gate"], s["shift"], s["scale"] = rows[:, 0], rows[:, 1], rows[:, 2]
        s["weight"] = 1.0 + 0.1 * torch.randn(K, generator=g, device=DEVICE) if case["affine"] else None
        s["bias"] = (0.1 * torch.randn(K, generator=g, device=DEVICE)
                     if case["affine"] and case["kind"] == "layer" else None)
        return s
    s["x"] = _activations(g, M, K, case["dtype"])
    spread = 0.2 * torch.rand((), generator=g, device=DEVICE)
    s["t"] = _tensor_scale(s["x"], spread) if case["scaled"] else None
    if op == "quantize":
        return s
    if op == "mlp":
        _weight(g, case["H"], K, case["fmt"], s, "w1")
        _weight(g, case["N"], case["H"], case["fmt"], s, "w2")
        s["b1"] = 0.02 * torch.randn(case["H"], generator=g, device=DEVICE)
        s["b2"] = 0.02 * torch.randn(case["N"], generator=g, device=DEVICE)
        # the calibrated scale of the hidden layer: a largest magnitude of about 6 standard deviations
        s["t2"] = (10.0 * math.sqrt(K / 3072.0) / 2688.0 * (1.0 + spread)).reshape(1) if case["scaled"] else None
        return s
    N = case["N"]
    _weight(g, N, K, case["fmt"], s, "w")
    s["b"] = 0.02 * torch.randn(N, generator=g, device=DEVICE) if case["bias"] else None
    s["residual"] = 2.0 * torch.randn(M, N, generator=g, device=DEVICE) if case["gated"] else None
    s["gate"] = 0.5 * torch.randn(N, generator=g, device=DEVICE) if case["gated"] else None
    return s


# ---- the plain forms

def encode(x, fmt, t=None):
    """Codes [rows, columns / 2] and scale bytes [rows, blocks] of x in float32 arithmetic."""
    R, K = x.shape
    b = x.float().reshape(R, K // BLOCK[fmt], BLOCK[fmt])
    amax = b.abs().amax(-1)
    if fmt == "nvfp4":
        s = amax / (6.0 * t) if t is not None else amax / 6.0
        s8 = s.clamp(2.0 ** -9, 448.0).to(torch.float8_e4m3fn)
        scale = s8.float() * t if t is not None else s8.float()
        bytes_ = s8.view(torch.uint8)
    else:
        e = torch.where(amax > 0, (torch.frexp(amax).exponent - 3).clamp(min=-127), -127)
        scale = torch.ldexp(torch.ones_like(amax), e)
        bytes_ = (e + 127).to(torch.uint8)
    q = (b / scale[..., None]).reshape(R, K)
    a = q.abs()
    # ties (0.25, 0.75, ...) go to the even code: borders above an even code belong to it, those below one too
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = mag + 8 * torch.signbit(q).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), bytes_


def decode(codes, scales, fmt, t=None):
    """float32 values [rows, columns] of codes and scale bytes."""
    R = codes.shape[0]
    n = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(R, -1)
    v = torch.tensor(F4, device=codes.device)[(n & 7).long()] * (1.0 - 2.0 * (n >> 3).float())
    if fmt == "nvfp4":
        s = scales.view(torch.float8_e4m3fn).float()
    else:
        s = torch.ldexp(torch.ones(scales.shape, device=codes.device), scales.int() - 127)
    v = (v.reshape(R, -1, BLOCK[fmt]) * s[..., None]).reshape(R, -1)
    return v * t if t is not None else v


def _rounded(x, fmt, t):
    return decode(*encode(x, fmt, t), fmt, t)


def _gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))


def _values(w, fmt):
    return decode(w["codes"], w["scales"], fmt, w["t"])


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        return _rounded(s["x"], c["fmt"], s["t"]).to(torch.bfloat16)
    if c["op"] == "linear":
        y = _rounded(s["x"], c["fmt"], s["t"]) @ _values(s["w"], c["fmt"]).T
        if s["b"] is not None:
            y = y + s["b"]
        if c["gated"]:
            y = s["residual"] + s["gate"] * y
        return y.to(DTYPES[c["out"]])
    if c["op"] == "mlp":
        h = _gelu(_rounded(s["x"], c["fmt"], s["t"]) @ _values(s["w1"], c["fmt"]).T + s["b1"])
        return (_rounded(h, c["fmt"], s["t2"]) @ _values(s["w2"], c["fmt"]).T + s["b2"]).to(torch.bfloat16)
    per = c["M"] // c["groups"]
    rows = lambda v: v.repeat_interleave(per, 0)  # noqa: E731
    x = (s["x"].float() + rows(s["gate"]) * s["y"].float()).to(DTYPES[c["x"]])
    v = x.float()
    if c["kind"] == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6)
    if s["weight"] is not None:
        v = v * s["weight"]
    if s["bias"] is not None:
        v = v + s["bias"]
    v = v * (1.0 + rows(s["scale"])) + rows(s["shift"])
    if c["out"] in BLOCK:
        return x, _rounded(v, c["out"], None).to(torch.bfloat16)
    return x, v.to(DTYPES[c["out"]])


def run(state):
    if not own:
        return _plain(state)
    s, c = state, state["case"]
    if c["op"] == "norm":
        x, h = _gated_norm()(s["x"], s["y"], s["gate"], weight=s["weight"], bias=s["bias"], shift=s["shift"],
                             scale=s["scale"], eps=1e-6, kind=c["kind"],
                             out=c["out"] if c["out"] in BLOCK else DTYPES[c["out"]])
        return x, _fp4().dequantize_rows(h, torch.bfloat16) if c["out"] in BLOCK else h
    fp4 = _fp4()
    if c["op"] == "quantize":
        return fp4.dequantize_rows(fp4.quantize_rows(s["x"], c["fmt"], s["t"]), torch.bfloat16)
    weight = lambda w: fp4.Rows(w["codes"], w["tiles"], c["fmt"], w["t"])  # noqa: E731
    if c["op"] == "mlp":
        return fp4.fp4_gelu_mlp(s["x"], weight(s["w1"]), s["b1"], weight(s["w2"]), s["b2"], input_scale=s["t"],
                                hidden_scale=s["t2"])
    return fp4.fp4_linear(s["x"], weight(s["w"]), s["b"], input_scale=s["t"], dtype=DTYPES[c["out"]],
                          residual=s["residual"], gate=s["gate"])


# ---- the definition in 64 bits

def _power(x):
    """The largest power of two that is not above x."""
    return torch.ldexp(torch.full_like(x, 0.5), torch.frexp(x).exponent)


def _exact_rounded(x, fmt, t):
    x = x.double()
    t = 1.0 if t is None else t.double()
    b = x.unflatten(-1, (-1, BLOCK[fmt]))
    top = b.abs().max(-1, keepdim=True).values
    if fmt == "nvfp4":
        s = top / (6.0 * t)
        step = _power(s.clamp(min=2.0 ** -6)) / 8  # E4M3: 3 fraction bits, from 2^-6 on
        s = (torch.round(s / step) * step).clamp(2.0 ** -9, 448.0) * t
    else:
        s = _power(top.clamp(min=2.0 ** -125)) / 4
    q = b / s
    step = torch.where(q.abs() < 2, 0.5, torch.where(q.abs() < 4, 1.0, 2.0)).to(q.dtype)
    return ((torch.round(q / step) * step).clamp(-6, 6) * s).flatten(-2)


def _exact_weight(w, fmt):
    c = w["codes"].int()
    n = torch.cat(((c % 16)[..., None], (c // 16)[..., None]), -1).flatten(-2)
    m = n % 8
    mag = torch.where(m < 2, m * 0.5, torch.exp2((m // 2 - 1).double()) * (1.0 + 0.5 * (m % 2)))
    b = w["scales"].int()
    if fmt == "nvfp4":
        e, f = b // 8, b % 8
        s = torch.where(e > 0, torch.exp2((e - 7).double()) * (1 + f / 8.0), f * 2.0 ** -9)
    else:
        s = torch.exp2((b - 127).double())
    v = torch.where(n >= 8, -mag, mag).double().unflatten(-1, (-1, BLOCK[fmt])) * s[..., None]
    return v.flatten(-2) * (1.0 if w["t"] is None else w["t"].double())


def exact(case, seed):
    s, fmt = prepare(case, seed), case.get("fmt")
    if case["op"] == "quantize":
        return _exact_rounded(s["x"], fmt, s["t"])
    if case["op"] == "linear":
        y = torch.einsum("mk,nk->mn", _exact_rounded(s["x"], fmt, s["t"]), _exact_weight(s["w"], fmt))
        if case["bias"]:
            y += s["b"].double()
        return y * s["gate"].double() + s["residual"].double() if case["gated"] else y
    if case["op"] == "mlp":
        h = torch.einsum("mk,nk->mn", _exact_rounded(s["x"], fmt, s["t"]), _exact_weight(s["w1"], fmt))
        h += s["b1"].double()
        u = math.sqrt(8.0 / math.pi) * (h + 0.044715 * h ** 3)
        h = h * torch.sigmoid(u)  # (1 + tanh(u / 2)) / 2
        return torch.einsum("mk,nk->mn", _exact_rounded(h, fmt, s["t2"]), _exact_weight(s["w2"], fmt)) \
            + s["b2"].double()
    group = torch.arange(case["M"], device=DEVICE) // (case["M"] // case["groups"])
    x = s["x"].double() + s["gate"].double()[group] * s["y"].double()
    stored = x if case["x"] == "float32" else x.to(DTYPES[case["x"]]).double()  # a 16-bit stream is what the norm reads
    v = stored - stored.mean(-1, keepdim=True) if case["kind"] == "layer" else stored
    v = v * torch.rsqrt((v ** 2).mean(-1, keepdim=True) + 1e-6)
    if case["affine"]:
        v = v * s["weight"].double()
        if case["kind"] == "layer":
            v = v + s["bias"].double()
    v = v + v * s["scale"].double()[group] + s["shift"].double()[group]
    return x, _exact_rounded(v, case["out"], None) if case["out"] in BLOCK else v
