"""The 4-bit K/V cache: its operators as a serving program calls them.

A case is a dict of plain values. ``kind``:
  attn   attention of the newest tokens of each sequence over its cached keys and values
  write  new K and V rows are quantised into their pages and read back as the values they hold
  read   the cached rows of whole sequences are read back for attention over unquantised K and V
  step   one decode step: the new rows are written, then attended with the rest of the cache

The cache is paged: ``codes`` uint8 [pages, 2, H_kv, page, D / 2] holds two e2m1 codes per byte (the
even dim in the low half; index 0 is K, 1 is V), ``scales`` uint8 [pages, 2, H_kv, D / 32, page] the
biased exponent of each 32 dims' power-of-two scale. A block's scale is the smallest power of two,
2^-126 at least, of which its largest magnitude is at most 7 times; codes are rounded to nearest even and
saturate at 6.
"""
import functools
import math
import os
import sys

import torch

own = False

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16}
BLOCK = 32  # dims per scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one short conversation: the smallest call, its latency counts
        dict(name="attn_one", kind="attn", dtype="bfloat16", B=1, T=1, H=32, Hkv=8, D=128, page=64,
             lo=1000, hi=1000),
        # a full serving batch of unequal lengths
        dict(name="attn_batch", kind="attn", dtype="bfloat16", B=64, T=1, H=32, Hkv=8, D=128,
             page=64, lo=512, hi=8192),
        # two long documents; the sum-exp goes to the merge with attention computed elsewhere
        dict(name="attn_long", kind="attn", dtype="bfloat16", B=2, T=1, H=64, Hkv=8, D=128, page=64,
             lo=100001, hi=131072, lse=True),
        # one K/V head per query head of 64 dims, small pages, short chats down to one token
        dict(name="attn_heads64", kind="attn", dtype="float16", B=24, T=1, H=16, Hkv=16, D=64,
             page=16, lo=1, hi=2047),
        # up to five drafted tokens per sequence are checked at once
        dict(name="attn_draft", kind="attn", dtype="float16", B=32, T=5, H=32, Hkv=4, D=128, page=32,
             lo=200, hi=4096),
        # chunks of two long prompts over what is cached of them
        dict(name="attn_chunk", kind="attn", dtype="bfloat16", B=2, T=1024, H=32, Hkv=8, D=128,
             page=64, lo=8192, hi=16384),
        # wide heads
        dict(name="attn_wide", kind="attn", dtype="bfloat16", B=12, T=1, H=16, Hkv=2, D=256,
             page=128, lo=1000, hi=6000),
        # the rows of one decode step
        dict(name="write_step", kind="write", dtype="bfloat16", B=32, T=1, H=32, Hkv=8, D=128,
             page=64, lo=100, hi=4000),
        # chunks of prompts behind what is there
        dict(name="write_prompt", kind="write", dtype="bfloat16", B=4, T=4096, H=32, Hkv=8, D=128,
             page=64, lo=4100, hi=6001),
        # eight cached prompts
        dict(name="read_prompt", kind="read", dtype="bfloat16", B=8, T=1, H=32, Hkv=8, D=128,
             page=64, lo=4000, hi=12000),
        # odd head counts, head dim and page size
        dict(name="read_odd", kind="read", dtype="float16", B=5, T=1, H=5, Hkv=5, D=96, page=24,
             lo=1, hi=701),
        # a decode step of a batch: write, then attend
        dict(name="step_batch", kind="step", dtype="bfloat16", B=48, T=1, H=32, Hkv=8, D=128,
             page=64, lo=1000, hi=5000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "attn", "write", "read", "step"])
    D = rng.choice([64, 96, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8, 8, 16])
    H = Hkv * rng.choice([1, 2, 4, 4, 7, 8, 16])
    page = rng.choice([16, 24, 32, 64, 64, 128])
    B = _log(rng, 1, 64)
    T = 1
    if kind == "write":
        T = rng.choice([1, _log(rng, 1, 2048)])
    elif kind in ("attn", "step"):
        T = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 8, 256)])
    # key values of the batch at most: those of the largest listed case of the kind
    most = (1 << 25) // (Hkv * D)
    B = min(B, max(1, (1 << 14) // (T * H // Hkv + 1) + 1))
    hi = max(1, min(_log(rng, 1, 65536), most // max(1, B * (1 + T * H // Hkv // 64))))
    hi = max(hi, T)
    lo = rng.choice([hi, max(1, hi // rng.choice([2, 3, 10])), 1])
    return dict(kind=kind, dtype=rng.choice(["float16", "bfloat16"]), B=B, T=T, H=H, Hkv=Hkv, D=D,
                page=page, lo=lo, hi=hi, lse=kind == "attn" and rng.random() < 0.3)


def _lengths(case):
    """Tokens of each sequence, and how many of them are new: the same for every seed."""
    B, T = case["B"], case["T"]
    n = [case["lo"] + (case["hi"] - case["lo"]) * i // max(1, B - 1) for i in range(B)]
    new = [max(1, T - (T * (B - 1 - i)) // (2 * B)) for i in range(B)] if T > 1 else [1] * B
    return n, [min(t, m) for t, m in zip(new, n)]


def _values(shape, g, dt):
    """Keys and values as a layer makes them: some dims much larger than the others."""
    x = torch.randn(shape, generator=g, device="cuda")
    wide = 1 + 7 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.04)
    return (x * wide).to(dt)


def prepare(case, seed):
    dt = DT[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, T, H, Hkv, D, page = (case[k] for k in ("B", "T", "H", "Hkv", "D", "page"))
    n, new = _lengths(case)
    order = torch.randperm(B, generator=g, device="cuda").tolist()
    n, new = [n[i] for i in order], [new[i] for i in order]
    per = -(-max(n) // page)
    pages = B * per + 3
    codes = torch.empty(pages, 2, Hkv, page, D // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(pages, 2, Hkv, D // BLOCK, page, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (2 * Hkv * page * D))
    for i in range(0, pages, step):
        c, e = _quantise(_values((min(step, pages - i), 2, Hkv, page, D), g, dt))
        codes[i:i + step] = c
        scales[i:i + step] = e.transpose(-1, -2)
    i32 = dict(dtype=torch.int32, device="cuda")
    qkv = torch.empty(B, T, (H + 2 * Hkv) * D, dtype=dt, device="cuda")  # a fused projection's rows
    qkv[..., :H * D] = torch.randn(B, T, H * D, generator=g, device="cuda").to(dt)
    qkv[..., H * D:] = _values((B, T, 2 * Hkv, D), g, dt).flatten(2)
    rows = n if case["kind"] == "read" else new
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    s = dict(kind=case["kind"], codes=codes, scales=scales, scale=D ** -0.5,
             table=torch.randperm(pages, generator=g, device="cuda")[:B * per].view(B, per).to(torch.int32),
             seqlens=torch.tensor(n, **i32), count=torch.tensor(new, **i32),
             start=torch.tensor([m - t for m, t in zip(n, new)], **i32), cu=torch.tensor(cu, **i32),
             q=qkv[..., :H * D].view(B, T, H, D), k=qkv[..., H * D:(H + Hkv) * D].view(B, T, Hkv, D),
             v=qkv[..., (H + Hkv) * D:].view(B, T, Hkv, D), longest=max(n))
    if case["kind"] in ("attn", "step"):
        s["out"] = torch.zeros(B, T, H, D, dtype=dt, device="cuda")
        s["lse"] = torch.zeros(B, T, H, device="cuda") if case.get("lse") else None
    else:
        s["k_out"], s["v_out"] = (torch.zeros(cu[-1], Hkv, D, dtype=dt, device="cuda") for _ in "kv")
    if own:
        ops = _ops()
        if "out" in s:
            need = ops.kv4_attn_workspace_bytes(B, T, H, Hkv, D)
            s["ws"] = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    return s


@functools.cache
def _ops():
    path = os.path.join(os.getcwd(), "tilelang-tpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tilelang.jit.adapter.mi355x import ops
    return ops


def run(s):
    if own:
        ops = _ops()
        kind = s["kind"]
        if kind in ("write", "step"):
            ops.kv4_append(s["k"], s["v"], s["start"], s["count"], s["table"], s["codes"], s["scales"])
        if kind in ("write", "read"):
            ops.kv4_read(s["codes"], s["scales"], s["table"], s["start"] if kind == "write" else None,
                         s["cu"], s["k_out"], s["v_out"])
            return s["k_out"], s["v_out"]
        ops.kv4_attn(s["q"], s["codes"], s["scales"], s["table"], s["seqlens"], s["out"], s["ws"],
                     s["scale"], count=s["count"], lse=s["lse"])
        return (s["out"],) if s["lse"] is None else (s["out"], s["lse"])
    if s["kind"] in ("write", "step"):
        _append(s)
    if s["kind"] in ("write", "read"):
        return _read(s)
    return _attend(s)


# The plain forms


def _quantise(x):
    """Codes [..., D / 2] and scale bytes [..., D / 32] of rows [..., D]."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    big = x.abs().amax(-1)
    m, p = torch.frexp(big)
    e = torch.where(m <= 0.875, p - 3, p - 2)  # big <= 7 2^e
    e = torch.where(big > 0, e, -126).clamp(-126, 125)
    y = (x * torch.exp2(-e.float()).unsqueeze(-1)).flatten(-2)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
            + (a >= 3.5) + (a > 5)) | (torch.signbit(y).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _dequantise(codes, scales):
    """Values [..., D] of codes [..., D / 2] and scale bytes [..., D / 32]."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    e = torch.exp2(scales.float() - 127).unsqueeze(-1)
    return (table[c].unflatten(-1, (-1, BLOCK)) * e).flatten(-2)


def _slots(s, start):
    """Of each row of cu: sequence, its index there, page and place in the page."""
    page = s["codes"].shape[3]
    i = torch.arange(s["k_out"].shape[0] if "k_out" in s else s["k"].shape[0] * s["k"].shape[1],
                     device="cuda", dtype=torch.int32)
    b = (torch.searchsorted(s["cu"], i, right=True) - 1).clamp(max=s["table"].shape[0] - 1)
    j = (i - s["cu"][b]).long()
    p = j + (0 if start is None else start[b].long())
    p = p.clamp(max=s["table"].shape[1] * page - 1)
    return b, j, s["table"][b, p // page].long(), p % page


def _append(s):
    b, j, pid, off = _slots(s, s["start"])
    live = j < s["count"][b]  # rows that pad the batch write the last new row once more
    j = torch.where(live, j, s["count"][b].long() - 1)
    p = s["start"][b].long() + j
    page = s["codes"].shape[3]
    pid, off = s["table"][b, p // page].long(), p % page
    for w, x in enumerate((s["k"], s["v"])):
        c, e = _quantise(x[b, j])
        s["codes"][pid, w, :, off] = c
        s["scales"][pid, w, :, :, off] = e


def _read(s):
    _, _, pid, off = _slots(s, s["start"] if s["kind"] == "write" else None)
    for w, out in enumerate((s["k_out"], s["v_out"])):
        out.copy_(_dequantise(s["codes"][pid, w, :, off], s["scales"][pid, w, :, :, off]))
    return s["k_out"], s["v_out"]


def _attend(s):
    q, out = s["q"], s["out"]
    B, T, H, D = q.shape
    Hkv, L = s["codes"].shape[2], s["longest"]
    pid = s["table"].long()
    c = s["codes"][pid].permute(2, 0, 3, 1, 4, 5).flatten(3, 4)[:, :, :, :L]
    e = s["scales"][pid].permute(2, 0, 3, 1, 5, 4).flatten(3, 4)[:, :, :, :L]
    k, v = _dequantise(c[0], e[0]), _dequantise(c[1], e[1])  # [B, Hkv, L, D]
    rows = q.float().view(B, T, Hkv, H // Hkv, D).transpose(1, 2).reshape(B, Hkv, -1, D)
    sc = torch.matmul(rows, k.transpose(-1, -2).contiguous()).view(B, Hkv, T, H // Hkv, L) * s["scale"]
    j = torch.arange(T, device="cuda")
    pos = (s["seqlens"] - s["count"])[:, None] + j  # [B, T]
    seen = torch.arange(L, device="cuda") <= pos[:, :, None]
    sc = sc.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, -1, L), v).view(B, Hkv, T, H // Hkv, D)
    o = torch.where(total > 0, o / total, 0.0).transpose(1, 2).reshape(B, T, H, D)
    live = (j < s["count"][:, None])[:, :, None]
    out.copy_(torch.where(live[..., None], o.to(out.dtype), out))
    if s["lse"] is None:
        return (out,)
    lse = (top * math.log2(math.e) + torch.log2(total)).squeeze(-1).transpose(1, 2).reshape(B, T, H)
    s["lse"].copy_(torch.where(live, lse, s["lse"]))
    return out, s["lse"]


def work(case):
    n, new = _lengths(case)
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    row = 2 * Hkv * (D // 2 + D // BLOCK)  # cache bytes of a token
    if case["kind"] == "read":
        return {"bytes": sum(n) * (row + 4 * Hkv * D), "flops": 0}
    write = sum(new) * (row + 4 * Hkv * D)
    if case["kind"] == "write":  # read back: the rows once more, and their values
        return {"bytes": write + sum(new) * (row + 4 * Hkv * D), "flops": 0}
    pairs = sum(t * m - t * (t - 1) // 2 for m, t in zip(n, new))
    attend = {"bytes": sum(n) * row + sum(new) * H * (4 * D + (4 if case.get("lse") else 0)),
              "flops": 4 * D * H * pairs}
    return attend if case["kind"] == "attn" else dict(attend, bytes=attend["bytes"] + write)


# The definition in 64 bits


def _exact_values(codes, scales):
    """Sign, exponent and fraction of each code, times its scale."""
    c = torch.stack((codes % 16, codes // 16), -1).flatten(-2).double()
    sign, c = torch.where(c >= 8, -1.0, 1.0), c % 8
    ex, half = torch.div(c, 2, rounding_mode="floor"), c % 2
    mag = torch.where(ex == 0, half / 2, (1 + half / 2) * 2.0 ** (ex - 1))
    return sign * mag * (2.0 ** (scales.double() - 127)).repeat_interleave(BLOCK, -1)


def _exact_rounded(x):
    """The values that rows x [..., D] have in the cache."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    big = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(big / 7)).clamp(-126, 125)
    e = torch.where(big > 7 * 2.0 ** e, e + 1, torch.where(big <= 7 * 2.0 ** (e - 1), e - 1, e))
    e = e.clamp(-126, 125)
    y = x / 2.0 ** e
    width = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return ((torch.round(y / width) * width).clamp(-6, 6) * 2.0 ** e).flatten(-2)


def _exact_cache(s, b, n):
    page = s["codes"].shape[3]
    p = torch.arange(n, device="cuda")
    pid, off = s["table"][b, p // page].long(), p % page
    return [_exact_values(s["codes"][pid, w, :, off], s["scales"][pid, w, :, :, off]) for w in (0, 1)]


def exact(case, seed):
    s = prepare(case, seed)
    kind, T = case["kind"], case["T"]
    n, new = s["seqlens"].tolist(), s["count"].tolist()
    if kind in ("write", "read"):
        got = [_exact_cache(s, b, m) if kind == "read" else
               [_exact_rounded(x[b, :t]) for x in (s["k"], s["v"])] for b, (m, t) in enumerate(zip(n, new))]
        return tuple(torch.cat([r[w] for r in got]) for w in (0, 1))
    H, Hkv = case["H"], case["Hkv"]
    out = s["out"].double()
    lse = torch.zeros(out.shape[:3], dtype=torch.float64, device="cuda")
    for b, (m, t) in enumerate(zip(n, new)):
        k, v = _exact_cache(s, b, m)
        if kind == "step":
            k[m - t:], v[m - t:] = _exact_rounded(s["k"][b, :t]), _exact_rounded(s["v"][b, :t])
        after = torch.arange(m, device="cuda") > torch.arange(m - t, m, device="cuda")[:, None]
        for h in range(H):
            one = h // (H // Hkv)
            sc = torch.matmul(s["q"][b, :t, h].double(), k[:, one].T.contiguous()) * case["D"] ** -0.5
            sc = torch.where(after, -math.inf, sc)
            out[b, :t, h] = torch.matmul(torch.softmax(sc, -1), v[:, one].contiguous())
            lse[b, :t, h] = torch.logsumexp(sc, -1) / math.log(2)
    return (out, lse) if case.get("lse") else (out,)
