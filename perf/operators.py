"""The microscaled (MX) operators of the decoder MLP: what is measured, in which sizes, and their plain form.

An MX row is cut into blocks of 32 consecutive elements. A block's elements are codes of 8 bits (e4m3) or 4 bits
(e2m1, two to a byte, the earlier element in the low half), and one byte s stands for the block's scale 2^(s - 127)
(255: the block is NaN). The scales of a matrix lie as [ceil(k / 128), rows, 4]: a row's four blocks of 128 elements side
by side (0 behind the last block). The scale is the smallest power of two, at least 2^-126, that holds the block's largest
magnitude without saturation (448 for e4m3, 6 for e2m1); codes are rounded to nearest, ties to even.

  quantize  rows -> MX codes and scales -> the values that these stand for
  norm      x <- x + delta, then RMSNorm(x) * weight as MX e4m3
  linear    MX rows times 4-bit MX weights (+ bias) (+ residual), bf16
  gate_up   SiLU(x . Wg^T) * (x . Wu^T) of MX rows and 4-bit MX weights, as MX e4m3
  mlp       norm, gate_up and linear with the residual: a decoder layer's MLP

Sizes are those of this repository's model configurations and what lies between them.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False  # True: run() calls the framework's operators

DEV = "cuda"
BLOCK = 32
FMT = {"e4m3": (448.0, 8, 0x1FFFFF), "e2m1": (6.0, 2, 0x3FFFFF)}  # largest value, its exponent, see _quantize
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # The gate/up weight of a 7B layer taken to 4 bits, as after each weight update of a rollout's policy.
        dict(name="quantize-weight-7b", kind="quantize", rows=37888, k=3584, fmt="e2m1", dtype="bf16"),
        # The attention output of one token, ready for a product: a call of latency alone.
        dict(name="quantize-token", kind="quantize", rows=1, k=3584, fmt="e4m3", dtype="bf16"),
        # The norm before the MLP for a single token of the 1.5B model.
        dict(name="norm-token-1.5b", kind="norm", rows=1, k=1536, dtype="bf16", delta=True),
        # The same norm over a verify round's 64 x 29 tree nodes at 7B.
        dict(name="norm-verify-7b", kind="norm", rows=1856, k=3584, dtype="bf16", delta=True),
        # The norm over eight prefill chunks at 14B, from float32 rows and without an addend.
        dict(name="norm-prefill-14b", kind="norm", rows=8192, k=5120, dtype="fp32", delta=False),
        # q, k and v with their bias for one token of the 1.5B model: the smallest product.
        dict(name="linear-token-1.5b", kind="linear", rows=1, n=2048, k=1536, fmt="e4m3", bias=True, residual=False),
        # The down projection of 64 single tokens at 7B: few rows against a long reduction.
        dict(name="linear-down-64-7b", kind="linear", rows=64, n=3584, k=18944, fmt="e4m3", bias=False, residual=True),
        # The down projection of a verify round at 7B.
        dict(name="linear-down-verify-7b", kind="linear", rows=1856, n=3584, k=18944, fmt="e4m3", bias=False, residual=True),
        # Rows in 4 bits too, a ragged prompt chunk at 8B against gate and up side by side.
        dict(name="linear-4x4-8b", kind="linear", rows=777, n=28672, k=4096, fmt="e2m1", bias=False, residual=False),
        # Gate, up and SwiGLU for one token at 8B: the weights are streamed once.
        dict(name="gate-up-token-8b", kind="gate_up", rows=1, inter=14336, k=4096, fmt="e4m3"),
        # The same over a verify round at 7B: the largest product of the layer.
        dict(name="gate-up-verify-7b", kind="gate_up", rows=1856, inter=18944, k=3584, fmt="e4m3"),
        # The MLP of a 1.5B verify round of 32 x 13 nodes, norm to residual.
        dict(name="mlp-verify-1.5b", kind="mlp", rows=416, inter=8960, k=1536),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    kind = rng.choice(["quantize", "norm", "linear", "linear", "linear", "gate_up", "gate_up", "mlp"])
    fmt = rng.choice(["e4m3", "e4m3", "e2m1"])
    if kind == "quantize":
        return dict(kind=kind, rows=_log(rng, 1, 40000), k=32 * _log(rng, 1, 592), fmt=fmt, dtype=rng.choice(["bf16", "bf16", "fp32"]))
    if kind == "norm":
        return dict(kind=kind, rows=_log(rng, 1, 8192), k=32 * _log(rng, 2, 256), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    delta=rng.random() < 0.6)
    rows, k = _log(rng, 1, 4096), 32 * _log(rng, 4, 592)
    if kind == "linear":
        return dict(kind=kind, rows=rows, n=_log(rng, 64, 38000), k=k, fmt=fmt, bias=rng.random() < 0.4, residual=rng.random() < 0.4)
    if kind == "gate_up":
        return dict(kind=kind, rows=rows, inter=32 * _log(rng, 8, 592), k=k, fmt=fmt)
    return dict(kind=kind, rows=rows, inter=32 * _log(rng, 16, 592), k=32 * _log(rng, 8, 256))


_MOST = None


def draw(rng):
    global _MOST
    if _MOST is None:
        w = [work(c) for c in listed()]
        _MOST = max(x["bytes"] for x in w), max(x["flops"] for x in w)
    while True:
        c = _one(rng)
        w = work(c)
        if w["bytes"] <= _MOST[0] and w["flops"] <= _MOST[1]:
            return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _dt(case):
    return torch.float32 if case.get("dtype") == "fp32" else torch.bfloat16


def _hidden(g, rows, k, std=1.0):
    """Hidden states: normal values with a few channels far larger than the others, as a decoder's residual has."""
    ch = torch.exp(0.5 * torch.randn(k, device=DEV, generator=g))
    ch = torch.where(torch.rand(k, device=DEV, generator=g) < 0.005, 20.0 * ch, ch)
    return std * ch * torch.randn(rows, k, device=DEV, generator=g)


def _weight(g, n, k):
    """A weight in 4 bits as a user keeps it: (codes [n, k / 2], scales [ceil(k / 128), n, 4])."""
    w = torch.randn(n, k, device=DEV, generator=g) * (k ** -0.5 * torch.exp(0.3 * torch.randn(n, 1, device=DEV, generator=g)))
    return _quantize(w.to(torch.bfloat16), "e2m1")


def prepare(case, seed):
    g, kind, k = _gen(seed), case["kind"], case["k"]
    s = dict(case=dict(case), eps=1e-6)
    if kind == "quantize":
        # a weight's spread for many rows, hidden states for few
        many = case["rows"] > 8192
        s["x"] = (0.02 * torch.randn(case["rows"], k, device=DEV, generator=g) if many else _hidden(g, case["rows"], k)).to(_dt(case))
    elif kind == "norm":
        s["x"] = _hidden(g, case["rows"], k).to(_dt(case))
        s["delta"] = (0.3 * torch.randn(case["rows"], k, device=DEV, generator=g)).to(_dt(case)) if case["delta"] else None
        s["weight"] = (1.0 + 0.2 * torch.randn(k, device=DEV, generator=g)).to(_dt(case))
        s["sum"] = torch.empty_like(s["x"])
    elif kind in ("linear", "gate_up"):
        s["x"] = _quantize(_hidden(g, case["rows"], k).to(torch.bfloat16), case["fmt"])
        n = case["n"] if kind == "linear" else 2 * case["inter"]
        s["w"] = _weight(g, n, k)
        s["bias"] = (0.5 * torch.randn(n, device=DEV, generator=g)).to(torch.bfloat16) if case.get("bias") else None
        s["residual"] = _hidden(g, case["rows"], n).to(torch.bfloat16) if case.get("residual") else None
    else:
        s["x"] = _hidden(g, case["rows"], k).to(torch.bfloat16)
        s["delta"] = (0.3 * torch.randn(case["rows"], k, device=DEV, generator=g)).to(torch.bfloat16)
        s["weight"] = (1.0 + 0.2 * torch.randn(k, device=DEV, generator=g)).to(torch.bfloat16)
        s["gate_up"] = _weight(g, 2 * case["inter"], k)
        s["down"] = _weight(g, k, case["inter"])
        s["sum"] = torch.empty_like(s["x"])
    return s


# ------------------------------------------------------------------ the plain form, in 32 bits
def _quantize(x, fmt):
    _, top, carry = FMT[fmt]
    v = x.float().reshape(x.shape[0], -1, BLOCK)
    amax = v.abs().amax(-1)
    # The exponent field of the largest magnitude, one more where its fraction is over that of the format's largest
    # value (1.75 or 1.5: the addition carries into the exponent), less that value's exponent.
    s = (((amax.view(torch.int32) + carry) >> 23) - top).clamp_min(1)
    y = v * ((254 - s) << 23).view(torch.float32).unsqueeze(-1)  # times 2^(127 - s): exact
    bad = ~torch.isfinite(v).all(-1)
    s = torch.where(bad, 255, s).to(torch.uint8)
    s = torch.nn.functional.pad(s, (0, -s.shape[1] % 4)).reshape(s.shape[0], -1, 4).transpose(0, 1).contiguous()
    y = torch.where(bad.unsqueeze(-1), 0.0, y).reshape(x.shape)
    if fmt == "e4m3":
        return y.to(torch.float8_e4m3fn), s
    a = y.abs()
    a = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2)))
    code = torch.where(a <= 2, 2 * a, torch.where(a <= 4, a + 2, 7.0)).to(torch.uint8) + 8 * (y < 0).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), s


def _values(q):
    """The values of (codes, scales) in 32 bits."""
    codes, scales = q
    if codes.dtype == torch.uint8:
        lut = torch.tensor(E2M1, device=codes.device)
        v = lut[torch.stack((codes & 15, codes >> 4), -1).to(torch.int32)].reshape(codes.shape[0], -1)
    else:
        v = codes.float()
    s = scales.transpose(0, 1).reshape(v.shape[0], -1)[:, :v.shape[1] // BLOCK]
    x = torch.where(s == 255, math.nan, (s.to(torch.int32) << 23).view(torch.float32))
    return (v.reshape(v.shape[0], -1, BLOCK) * x.unsqueeze(-1)).reshape(v.shape)


def _norm(s):
    x = s["x"] if s["delta"] is None else (s["x"].float() + s["delta"].float()).to(s["x"].dtype)
    f = x.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    return x, _quantize(y, "e4m3")


def _linear(x, w, bias=None, residual=None):
    y = _values(x) @ _values(w).t()
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return y.to(torch.bfloat16)


def _gate_up(x, w):
    g, u = (_values(x) @ _values(w).t()).chunk(2, -1)
    return _quantize(g / (1.0 + torch.exp(-g)) * u, "e4m3")


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "quantize":
        return _values(_quantize(s["x"], s["case"]["fmt"])).to(torch.bfloat16)
    if kind == "norm":
        x, q = _norm(s)
        return dict(sum=x, values=_values(q).to(torch.bfloat16))
    if kind == "linear":
        return _linear(s["x"], s["w"], s["bias"], s["residual"])
    if kind == "gate_up":
        return _values(_gate_up(s["x"], s["w"])).to(torch.bfloat16)
    x, q = _norm(s)
    return _linear(_gate_up(q, s["gate_up"]), s["down"], None, x)


# ------------------------------------------------------------------ the framework's operators
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ss-grpo_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)


def _framework(s):
    from flashgrpo_amd import kernels as K

    kind = s["case"]["kind"]
    if kind == "quantize":
        return K.mx_dequantize(K.mx_quantize(s["x"], s["case"]["fmt"]))
    if kind == "norm":
        x = s["x"] if s["delta"] is None else s["sum"]
        q = K.rmsnorm_mx(s["x"], s["weight"], s["eps"], delta=s["delta"], sum_out=None if s["delta"] is None else x)
        return dict(sum=x, values=K.mx_dequantize(q))
    if kind == "linear":
        return K.mx_linear(s["x"], s["w"], bias=s["bias"], residual=s["residual"])
    if kind == "gate_up":
        return K.mx_dequantize(K.mx_gate_up_swiglu(s["x"], s["w"]))
    q = K.rmsnorm_mx(s["x"], s["weight"], s["eps"], delta=s["delta"], sum_out=s["sum"])
    return K.mx_linear(K.mx_gate_up_swiglu(q, s["gate_up"]), s["down"], residual=s["sum"])


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------ the least work of one pass
def _mx_bytes(rows, k, fmt):
    return rows * k * (0.5 if fmt == "e2m1" else 1.0) + rows * k / BLOCK


def work(case):
    kind, rows, k = case["kind"], case["rows"], case["k"]
    e = 4 if case.get("dtype") == "fp32" else 2
    if kind == "quantize":  # rows in, codes and scales, the values out
        return dict(bytes=rows * k * (e + 2) + _mx_bytes(rows, k, case["fmt"]), flops=4.0 * rows * k)
    if kind == "norm":  # rows (and the addend) in, (the sum,) codes and scales and the values out
        return dict(bytes=rows * k * (e * (3 if case["delta"] else 1) + 2) + e * k + _mx_bytes(rows, k, "e4m3"), flops=8.0 * rows * k)
    if kind == "linear":
        n = case["n"]
        io = 2 * rows * n * (2 if case["residual"] else 1) + (2 * n if case["bias"] else 0)
        return dict(bytes=_mx_bytes(rows, k, case["fmt"]) + _mx_bytes(n, k, "e2m1") + io, flops=2.0 * rows * n * k)
    n = case["inter"]
    if kind == "gate_up":
        return dict(bytes=_mx_bytes(rows, k, case["fmt"]) + _mx_bytes(2 * n, k, "e2m1") + _mx_bytes(rows, n, "e4m3") + 2 * rows * n,
                    flops=4.0 * rows * n * k)
    # x and its addend in, the residual stream out, both weights
    return dict(bytes=6 * rows * k + 2 * k + _mx_bytes(3 * n, k, "e2m1"), flops=6.0 * rows * n * k)


# ------------------------------------------------------------------ from the definition, in 64 bits
def _two64(e):
    """2^e, from its bits: a power function may be off by its last one."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _grid64(y, low, bits):
    """y rounded to a binary floating format of `bits` fraction bits whose least exponent is `low`, ties to even."""
    e = (torch.frexp(y)[1] - 1).clamp_min(low)
    step = _two64(e - bits)
    return torch.round(y / step) * step


def _through64(v, fmt):
    """The values that v's MX form stands for."""
    v = v.double()
    most, low, bits = (448.0, -6, 3) if fmt == "e4m3" else (6.0, 0, 1)
    b = v.reshape(v.shape[0], -1, BLOCK)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True) / most)  # the least power of two not below m * 2^e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e).clamp_min(-126)
    x = _two64(e)
    return (_grid64(b / x, low, bits) * x).reshape(v.shape)


def _held64(q):
    codes, scales = q
    if codes.dtype == torch.uint8:
        c = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.int16, device=codes.device)
        c[:, 0::2], c[:, 1::2] = codes % 16, codes // 16
        m = c % 8
        v = torch.where(m < 2, m * 0.5, (1.0 + (m % 2) * 0.5) * _two64(m // 2 - 1)).double()
        v = torch.where(c >= 8, -v, v)
    else:
        v = codes.double()
    every = torch.cat(tuple(scales.double()), 1) if scales.shape[0] > 1 else scales[0].double()
    return v * _two64(every[:, :v.shape[1] // BLOCK] - 127).repeat_interleave(BLOCK, 1)


def _norm64(s):
    x = s["x"] if s["delta"] is None else (s["x"].double() + s["delta"].double()).to(s["x"].dtype)
    f = x.double()
    return x, _through64(f / torch.sqrt(f.pow(2).mean(-1, keepdim=True) + s["eps"]) * s["weight"].double(), "e4m3")


def _gate_up64(x, w):
    y = x @ w.t()
    n = y.shape[1] // 2
    return _through64(y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:], "e4m3")


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _through64(s["x"], case["fmt"])
    if kind == "norm":
        x, v = _norm64(s)
        return dict(sum=x.double(), values=v)
    if kind == "linear":
        y = _held64(s["x"]) @ _held64(s["w"]).t()
        y = y if s["bias"] is None else y + s["bias"].double()
        return y if s["residual"] is None else y + s["residual"].double()
    if kind == "gate_up":
        return _gate_up64(_held64(s["x"]), _held64(s["w"]))
    x, v = _norm64(s)
    return x.double() + _gate_up64(v, _held64(s["gate_up"])) @ _held64(s["down"]).t()
