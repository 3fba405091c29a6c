"""Dense layers in 8 bits: their operators as a serving program calls them.

A case is a dict of plain values. ``kind``:
  norm   the layer's output joins the residual stream, whose root-mean-square norm goes to the next
         projections in 8 bits, in 16 or both
  quant  rows become 8-bit operands: attention's outputs, or weights when they are loaded
  gemm   a projection of 8-bit rows by 8-bit weights
  ffn    the gated feed-forward block: gate and up projections, SwiGLU, down projection
  tail   what follows attention in a layer: norm, then the feed-forward block

8 bits are OCP MX: e4m3 codes with one power-of-two scale (e8m0) per 32 values of a row. A block's
scale is the smallest power of two, 2^-126 at least, of which its largest magnitude is at most 448
times; codes are rounded to nearest even. A block that holds an infinity or NaN has a NaN scale.
``codes`` are [rows, K]; ``scales`` lie as matrix instructions take them, [ceil(rows / 64), ceil(K / 128), 4, 64]:
that of block b of row r at [r / 64, b / 4, b % 4, r % 64], with unused places where rows or blocks end.
"""
import functools
import math
import os
import sys

import torch

own = False

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
BLOCK = 32  # values per scale
EPS = 1e-6


def listed():
    return [
        # one decode step of 16 sequences: the smallest call, launch and host cost
        dict(name="norm_step", kind="norm", dtype="bfloat16", stream="bfloat16", rows=16, cols=4096,
             y=False, mx=True),
        # a ragged chunk of a prompt; the stream is kept in 32 bits, a router reads the norm in 16
        dict(name="norm_chunk", kind="norm", dtype="float16", stream="float32", rows=499, cols=5120,
             y=True, mx=True),
        # a whole prompt batch
        dict(name="norm_prompts", kind="norm", dtype="bfloat16", stream="bfloat16", rows=8192,
             cols=7168, y=False, mx=True),
        # attention's outputs before their projection, from a buffer with wider rows
        dict(name="quant_rows", kind="quant", dtype="bfloat16", rows=2001, cols=4096, gap=1024),
        # a layer's weights when a model is loaded
        dict(name="quant_weights", kind="quant", dtype="float32", rows=14336, cols=4096, gap=0),
        # a projection in one decode step: the weight stream is everything
        dict(name="gemm_step", kind="gemm", dtype="bfloat16", M=16, N=4096, K=14336),
        # few odd rows, odd widths
        dict(name="gemm_odd", kind="gemm", dtype="float16", M=37, N=2051, K=1056),
        # a ragged chunk of a prompt
        dict(name="gemm_chunk", kind="gemm", dtype="bfloat16", M=500, N=4096, K=4096),
        # a whole prompt batch
        dict(name="gemm_prompts", kind="gemm", dtype="bfloat16", M=4096, N=4096, K=4096),
        # a decode batch at the MLP program's sizes
        dict(name="ffn_batch", kind="ffn", dtype="bfloat16", M=64, hidden=7168, inter=2048),
        # whole prompts: the largest call
        dict(name="ffn_prompts", kind="ffn", dtype="bfloat16", M=4096, hidden=4096, inter=11008),
        # one new token: five calls in a row that wait for each other
        dict(name="tail_token", kind="tail", dtype="bfloat16", M=1, hidden=4096, inter=11008),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quant", "gemm", "gemm", "gemm", "gemm", "ffn", "ffn", "ffn",
                       "tail"])
    h16 = rng.choice(["float16", "bfloat16"])
    if kind == "norm":
        y, mx = rng.choice([(False, True), (False, True), (True, True), (True, False)])
        return dict(kind=kind, dtype=h16, stream=rng.choice([h16, h16, "float32"]),
                    rows=_log(rng, 1, 8192), cols=BLOCK * _log(rng, 4, 256), y=y, mx=mx)
    if kind == "quant":
        return dict(kind=kind, dtype=rng.choice([h16, h16, "float32"]), rows=_log(rng, 1, 8192),
                    cols=BLOCK * _log(rng, 4, 448), gap=rng.choice([0, 0, 64, 1000]))
    if kind == "gemm":
        while True:  # any token count, any width of the result
            M, N, K = _log(rng, 1, 4096), _log(rng, 64, 14336), BLOCK * _log(rng, 4, 448)
            if M * N * K <= 4096 ** 3:
                return dict(kind=kind, dtype=h16, M=M, N=N, K=K)
    while True:
        M = _log(rng, 1, 4096 if kind == "ffn" else 256)
        hidden, inter = BLOCK * _log(rng, 16, 224), BLOCK * _log(rng, 16, 448)
        if M * hidden * inter <= 4096 * 4096 * 11008 // 4:
            return dict(kind=kind, dtype=h16, M=M, hidden=hidden, inter=inter)


def _activations(rows, cols, g):
    """Hidden states as layers make them: some dims much larger than the others."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return x * (1 + 15 * (torch.rand(cols, generator=g, device="cuda") < 0.02))


def _weights(rows, cols, g):
    w = torch.randn(rows, cols, generator=g, device="cuda") / math.sqrt(cols)
    return _quantise(w * (0.5 + torch.rand(rows, 1, generator=g, device="cuda")))


def _empty(rows, cols):
    scales = torch.zeros(-(-rows // 64), -(-cols // 128), 4, 64, dtype=torch.uint8, device="cuda")
    return (torch.zeros(rows, cols, dtype=torch.float8_e4m3fn, device="cuda"),
            scales.view(torch.float8_e8m0fnu))


def prepare(case, seed):
    dt = DT[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(kind=case["kind"])
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(rows, cols, g).to(dt)
        s["residual"] = (4 * _activations(rows, cols, g)).to(DT[case["stream"]])
        s["w"] = (1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).to(dt)
        s["stream"] = torch.zeros_like(s["residual"])
        s["y"] = torch.zeros_like(s["x"]) if case["y"] else None
        s["mx"] = _empty(rows, cols) if case["mx"] else (None, None)
    elif case["kind"] == "quant":
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(rows, cols + case["gap"], g).to(dt)[:, :cols]
        s["mx"] = _empty(rows, cols)
    elif case["kind"] == "gemm":
        s["a"] = _quantise(_activations(case["M"], case["K"], g))
        s["b"] = _weights(case["N"], case["K"], g)
        s["c"] = torch.zeros(case["M"], case["N"], dtype=dt, device="cuda")
    else:
        M, hidden, inter = case["M"], case["hidden"], case["inter"]
        x = _activations(M, hidden, g)
        s["gate"], s["up"] = _weights(inter, hidden, g), _weights(inter, hidden, g)
        s["down"] = _weights(hidden, inter, g)
        s["h"] = _empty(M, inter)
        s["c"] = torch.zeros(M, hidden, dtype=dt, device="cuda")
        if case["kind"] == "ffn":
            s["a"] = _quantise(x)
        else:
            s["x"] = x.to(dt)
            s["residual"] = (4 * _activations(M, hidden, g)).to(dt)
            s["w"] = (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(dt)
            s["stream"] = torch.zeros_like(s["residual"])
            s["y"], s["mx"] = None, _empty(M, hidden)
            s["w2"] = (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(dt)
            s["stream2"], s["y2"] = torch.zeros_like(s["residual"]), torch.zeros_like(s["x"])
    return s


@functools.cache
def _ops():
    path = os.path.join(os.getcwd(), "tilelang-tpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tilelang.jit.adapter.mi355x import ops
    return ops


def run(s):
    kind = s["kind"]
    if own:
        ops = _ops()
        if kind == "norm":
            ops.add_rmsnorm(s["x"], s["residual"], s["w"], s["stream"], EPS, s["y"], *s["mx"])
            return s["stream"], s["y"], s["mx"]
        if kind == "quant":
            ops.mx8_quant(s["x"], *s["mx"])
            return s["mx"]
        if kind == "gemm":
            ops.gemm_mx8(*s["a"], *s["b"], s["c"])
            return s["c"]
        a = s["a"] if kind == "ffn" else s["mx"]
        if kind == "tail":
            ops.add_rmsnorm(s["x"], s["residual"], s["w"], s["stream"], EPS, None, *s["mx"])
        ops.gemm_mx8_swiglu(*a, *s["gate"], *s["up"], *s["h"])
        ops.gemm_mx8(*s["h"], *s["down"], s["c"])
        if kind == "ffn":
            return s["c"]
        # the next layer's norm takes the block's output in
        ops.add_rmsnorm(s["c"], s["stream"], s["w2"], s["stream2"], EPS, s["y2"])
        return s["stream2"], s["y2"]
    if kind == "norm":
        _norm(s["x"], s["residual"], s["w"], s["stream"], s["y"], s["mx"])
        return s["stream"], s["y"], s["mx"]
    if kind == "quant":
        _put(s["mx"], _quantise(s["x"]))
        return s["mx"]
    if kind == "gemm":
        return s["c"].copy_(_product(s["a"], s["b"]))
    if kind == "tail":
        _norm(s["x"], s["residual"], s["w"], s["stream"], None, s["mx"])
    a = s["a"] if kind == "ffn" else s["mx"]
    gate, up = _product(a, s["gate"]), _product(a, s["up"])
    _put(s["h"], _quantise(up * gate / (1 + torch.exp(-gate))))
    s["c"].copy_(_product(s["h"], s["down"]))
    if kind == "ffn":
        return s["c"]
    _norm(s["c"], s["stream"], s["w2"], s["stream2"], s["y2"], (None, None))
    return s["stream2"], s["y2"]


# The plain forms


def _power(e):
    """2^e of whole numbers -126 .. 127, from its bits: exp2 may be off in the last place."""
    return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _quantise(x):
    """Codes and scales of rows x [M, K]."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    big = x.abs().amax(-1)
    m, p = torch.frexp(big)
    e = torch.where(m <= 0.875, p - 9, p - 8)  # big <= 448 2^e
    e = torch.where(big > 0, e, -126).clamp(-126, 120)  # 120: of the type's largest value
    fine = big < math.inf
    codes = torch.where(fine[..., None], x * _power(-e)[..., None], 0.0).flatten(-2)
    byte = torch.where(fine, e + 127, 255).to(torch.uint8)
    byte = torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4, 0, -byte.shape[0] % 64))
    byte = byte.unflatten(0, (-1, 64)).unflatten(2, (-1, 4)).permute(0, 2, 3, 1).contiguous()
    return codes.to(torch.float8_e4m3fn), byte.view(torch.float8_e8m0fnu)


def _put(out, mx):
    for o, t in zip(out, mx):
        o.copy_(t)


def _values(mx):
    codes, scales = mx
    byte = scales.view(torch.uint8).permute(0, 3, 1, 2).flatten(2).flatten(0, 1)
    byte = byte[:codes.shape[0], :codes.shape[1] // BLOCK].int()
    scale = torch.where(byte < 255, _power(byte - 127), math.nan)
    return (codes.float().unflatten(-1, (-1, BLOCK)) * scale[..., None]).flatten(-2)


def _product(a, b):
    return torch.matmul(_values(a), _values(b).T)


def _norm(x, residual, w, stream, y, mx):
    stream.copy_(x.float() + residual.float())
    h = stream.float()  # the norm is that of the stream as it is kept
    h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.float()
    if y is not None:
        y.copy_(h)
    if mx[0] is not None:
        _put(mx, _quantise(h))


def _mx_bytes(rows, cols):
    return rows * (cols + cols // BLOCK)


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, e = case["rows"] * case["cols"], SIZE[case["dtype"]]
        bytes_ = n * (e + 2 * SIZE[case["stream"]] + (e if case["y"] else 0)) + e * case["cols"]
        return {"bytes": bytes_ + (_mx_bytes(case["rows"], case["cols"]) if case["mx"] else 0), "flops": 0}
    if kind == "quant":
        n = case["rows"] * case["cols"]
        return {"bytes": n * SIZE[case["dtype"]] + _mx_bytes(case["rows"], case["cols"]), "flops": 0}
    if kind == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": _mx_bytes(M + N, K) + 2 * M * N, "flops": 2 * M * N * K}
    M, hidden, inter = case["M"], case["hidden"], case["inter"]
    block = {"bytes": _mx_bytes(2 * inter, hidden) + _mx_bytes(hidden, inter), "flops": 6 * M * hidden * inter}
    if kind == "ffn":  # rows in, result out
        return dict(block, bytes=block["bytes"] + _mx_bytes(M, hidden) + 2 * M * hidden)
    # rows and stream in; stream and norm out; two weights of norms
    return dict(block, bytes=block["bytes"] + 4 * 2 * M * hidden + 4 * hidden)


# The definition in 64 bits


def _exact_power(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_mx(x):
    """Codes' values of rows x, and scales [rows, K / 32], in 64 bits."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    big = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(big / 448)).clamp(-126, 127)
    e = torch.where(big > 448 * _exact_power(e), e + 1, torch.where(big <= 448 * _exact_power(e - 1), e - 1, e))
    e = e.clamp(-126, 127)
    y = x / _exact_power(e)
    top = y.abs().clamp(min=2.0 ** -6)
    n = torch.floor(torch.log2(top))
    n = torch.where(_exact_power(n) > top, n - 1, torch.where(_exact_power(n + 1) <= top, n + 1, n))
    step = _exact_power(n - 3)
    return (torch.round(y / step) * step).flatten(-2), _exact_power(e.squeeze(-1))


def _exact_out(x):
    """What the buffers hold: unused scales stay 0, which is 2^-127."""
    codes, scales = _exact_mx(x)
    rows, blocks = scales.shape
    out = torch.full((-(-rows // 64), -(-blocks // 4), 4, 64), 2.0 ** -127, dtype=torch.float64, device="cuda")
    r, b = (torch.arange(n, device="cuda") for n in (rows, blocks))
    out[r[:, None] // 64, b // 4, b % 4, r[:, None] % 64] = scales
    return codes, out


def _exact_values(codes, scales):
    """Values of rows in 64 bits; scales as _exact_mx gives them, or as the buffers hold them."""
    scales = scales.double()
    if scales.dim() > 2:
        r, b = (torch.arange(n, device="cuda") for n in (codes.shape[0], codes.shape[1] // BLOCK))
        scales = scales[r[:, None] // 64, b // 4, b % 4, r[:, None] % 64]
    return codes.double() * scales.repeat_interleave(BLOCK, -1)


def _exact_norm(x, residual, w, dt):
    stream = x.double() + residual.double()
    kept = stream.to(dt).double()
    rms = torch.sqrt(kept.pow(2).sum(-1, keepdim=True) / kept.shape[-1] + EPS)
    return stream, kept, kept / rms * w.double()


def _exact_ffn(a, s):
    gate, up = (a @ _exact_values(*s[w]).T for w in ("gate", "up"))
    h = _exact_values(*_exact_mx(up * gate * torch.sigmoid(gate)))
    return h @ _exact_values(*s["down"]).T


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        stream, _, y = _exact_norm(s["x"], s["residual"], s["w"], s["stream"].dtype)
        return stream, y if case["y"] else None, _exact_out(y) if case["mx"] else (None, None)
    if kind == "quant":
        return _exact_out(s["x"])
    if kind == "gemm":
        return _exact_values(*s["a"]) @ _exact_values(*s["b"]).T
    if kind == "ffn":
        return _exact_ffn(_exact_values(*s["a"]), s)
    dt = DT[case["dtype"]]
    _, kept, y = _exact_norm(s["x"], s["residual"], s["w"], dt)
    out = _exact_ffn(_exact_values(*_exact_mx(y)), s).to(dt)  # kept in 16 bits between the calls
    stream, _, y = _exact_norm(out, kept, s["w2"], dt)
    return stream, y
