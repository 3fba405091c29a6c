"""The 4-bit K/V cache's oracle (oracle/ref.py, kv4_*), pinned by checks that do not retype its formulas,
and the C entry points' refusals. CPU only."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

from oracle import ref
from tilelang.jit.adapter.mi355x import lib

EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -4


def test_values_follow_the_bits():
    """A code is sign, two exponent bits (bias 1), one fraction bit; exponent 0 is subnormal."""
    codes = np.arange(16, dtype=np.uint8)
    got = ref.kv4_dequantise_ref((codes | (codes << 4)).repeat(16).reshape(16, 16),
                                 np.full((16, 1), 130, np.uint8))
    for c in range(16):
        e, f = (c >> 1) & 3, c & 1
        mag = f * 0.5 if e == 0 else (1 + f * 0.5) * 2.0 ** (e - 1)
        assert (got[c] == (-1) ** (c >> 3) * mag * 8).all()


def test_quantised_is_nearest_and_the_scale_least():
    g = torch.Generator().manual_seed(5)
    x = torch.randn(400, 64, generator=g) * torch.exp(4 * torch.randn(400, 1, generator=g))
    x[0] = 0
    x = x.to(torch.bfloat16)
    codes, scales = ref.kv4_quantise_ref(x)
    v = x.double().numpy().reshape(400, 2, 32)
    q = ref.kv4_dequantise_ref(codes, scales).reshape(400, 2, 32)
    s = 2.0 ** (scales.astype(float) - 127)
    big = np.abs(v).max(-1)
    assert (big <= 7 * s).all() and ((big > 3.5 * s) | (scales == 1)).all()
    every = np.array([m * sg for m in ref.KV4_VALUES for sg in (1, -1)])
    near = np.abs(v[..., None] - every * s[..., None, None]).min(-1)
    assert np.array_equal(np.abs(v - q), near)
    assert (np.abs(v - q) <= s[..., None]).all()


def test_ties_take_the_even_code():
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    x = torch.zeros(1, 32)
    x[0, :7], x[0, 7] = torch.tensor(mids), 6.0  # scale 1
    codes, scales = ref.kv4_quantise_ref(x)
    assert scales[0, 0] == 127
    q = ref.kv4_dequantise_ref(codes, scales)[0]
    assert q[:7].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]


def test_what_is_not_finite():
    x = torch.ones(3, 64)
    x[0, 3], x[1, 40], x[2, 0], x[2, 1] = float("nan"), float("-inf"), -0.0, 3e38
    codes, scales = ref.kv4_quantise_ref(x)
    v = ref.kv4_dequantise_ref(codes, scales)
    assert np.isnan(v[0, :32]).all() and (v[0, 32:] == 1).all()
    assert v[1, 40] == -6 * 2.0 ** 125 and (v[1, 41:] == 0).all()
    assert np.signbit(v[2, 0]) and v[2, 0] == 0 and v[2, 1] == 6 * 2.0 ** 125


def test_append_in_steps_equals_at_once_and_reads_back():
    g = torch.Generator().manual_seed(6)
    B, T, Hkv, D, page, pages = 2, 13, 3, 64, 8, 7
    k, v = (torch.randn(B, T, Hkv, D, generator=g).to(torch.float16) for _ in "kv")
    bt = torch.randperm(pages, generator=g)[:6].view(2, 3).int().numpy()
    empty = (np.full((pages, 2, Hkv, page, D // 2), 0xA5, np.uint8),
             np.full((pages, 2, Hkv, D // 32, page), 0x5A, np.uint8))
    start, count = np.array([2, 11]), np.array([13, 13])  # sequence 1 ends at the table's 24th position
    once = ref.kv4_append_ref(k, v, start, count, bt, *empty)
    step = empty
    for j in range(T):
        step = ref.kv4_append_ref(k[:, j:j + 1], v[:, j:j + 1], start + j, np.array([1, 1]), bt, *step)
    assert all(np.array_equal(a, b) for a, b in zip(once, step))
    kk, vv = ref.kv4_rows_ref(*once, bt, 0, 2, 13)
    for got, x in ((kk, k), (vv, v)):
        assert np.array_equal(got, ref.kv4_dequantise_ref(*ref.kv4_quantise_ref(x[0])))
    assert (ref.kv4_rows_ref(*once, bt, 1, 22, 5)[0][2:] == 0).all()  # beyond the table
    used = {(int(bt[b, p // page]), p % page) for b, s in ((0, 2), (1, 11)) for p in range(s, min(24, s + 13))}
    for pid, off in itertools.product(range(pages), range(page)):
        if (pid, off) not in used:
            assert (once[0][pid, :, :, off] == 0xA5).all() and (once[1][pid, :, :, :, off] == 0x5A).all()


@pytest.mark.parametrize("causal", [True, False])
def test_attention_is_softmax_over_the_rows(causal):
    g = torch.Generator().manual_seed(7)
    B, T, H, Hkv, D, page, pages = 2, 4, 6, 2, 32, 8, 6
    codes = torch.randint(0, 256, (pages, 2, Hkv, page, D // 2), generator=g).byte().numpy()
    scales = torch.randint(124, 128, (pages, 2, Hkv, D // 32, page), generator=g).byte().numpy()
    bt = torch.randperm(pages, generator=g).view(2, 3).int().numpy()
    q = torch.randn(B, T, H, D, generator=g)
    seqlens, count = [19, 2], [3, 4]
    out, lse = ref.kv4_attn_ref(q, codes, scales, bt, seqlens, count, 0.2, causal)
    for b in range(B):
        k, v = (torch.from_numpy(x) for x in ref.kv4_rows_ref(codes, scales, bt, b, 0, seqlens[b]))
        for j, h in itertools.product(range(count[b]), range(H)):
            n = seqlens[b] - count[b] + j + 1 if causal else seqlens[b]
            if n <= 0:
                assert (out[b, j, h] == 0).all() and lse[b, j, h] == -np.inf
                continue
            s = (k[:n, h // 3] @ q[b, j, h].double()) * 0.2
            assert np.allclose(out[b, j, h], torch.softmax(s, 0) @ v[:n, h // 3], atol=1e-12)
            assert np.isclose(lse[b, j, h], torch.logsumexp(s, 0) / np.log(2), atol=1e-12)
    assert np.isnan(out[0, 3]).all()


P = ctypes.c_void_p(0x1000)


def _pool(**kw):
    a = dict(codes=P, cs=2 * 8 * 64 * 64, scales=P, ss=2 * 8 * 4 * 64, pages=10, bt=P, mp=4, page=64)
    a.update({k: v for k, v in kw.items() if k in a})
    return a


def _append(**kw):
    p = _pool(**kw)
    a = dict(k=P, v=P, kb=8192, kr=1024, vb=8192, vr=1024, dt=lib.BF16, start=P, count=P, B=2, T=8, Hkv=8, D=128)
    a.update({k: v for k, v in kw.items() if k in a})
    return lib.load().tlm_kv4_append(a["k"], a["v"], a["kb"], a["kr"], a["vb"], a["vr"], a["dt"], a["start"],
                                     a["count"], p["bt"], p["mp"], p["page"], p["codes"], p["cs"], p["scales"],
                                     p["ss"], p["pages"], a["B"], a["T"], a["Hkv"], a["D"], None)


def _read(**kw):
    p = _pool(**kw)
    a = dict(start=None, cu=P, k=P, v=P, B=2, total=8, Hkv=8, D=128, dt=lib.BF16)
    a.update({k: v for k, v in kw.items() if k in a})
    return lib.load().tlm_kv4_read(p["codes"], p["cs"], p["scales"], p["ss"], p["pages"], p["bt"], p["mp"],
                                   p["page"], a["start"], a["cu"], a["k"], a["v"], a["B"], a["total"], a["Hkv"],
                                   a["D"], a["dt"], None)


def _attn(**kw):
    p = _pool(**kw)
    a = dict(q=P, qb=4096, qr=4096, sl=P, count=None, o=P, lse=None, ws=P, wb=1 << 40, B=2, T=1, H=32, Hkv=8,
             D=128, causal=1, scale=0.1, dt=lib.BF16)
    a.update({k: v for k, v in kw.items() if k in a})
    return lib.load().tlm_kv4_attn(a["q"], a["qb"], a["qr"], p["codes"], p["cs"], p["scales"], p["ss"],
                                   p["pages"], p["bt"], p["mp"], p["page"], a["sl"], a["count"], a["o"], a["lse"],
                                   a["ws"], a["wb"], a["B"], a["T"], a["H"], a["Hkv"], a["D"], a["causal"],
                                   a["scale"], a["dt"], None)


ODD = ctypes.c_void_p(0x1008)
SHARED = [
    (dict(codes=None), EINVAL, "null"), (dict(scales=None), EINVAL, "null"), (dict(bt=None), EINVAL, "null"),
    (dict(codes=ODD), EINVAL, "aligned"), (dict(scales=ctypes.c_void_p(0x1004)), EINVAL, "aligned"),
    (dict(page=0), EINVAL, "sizes"), (dict(mp=0), EINVAL, "sizes"), (dict(pages=0), EINVAL, "sizes"),
    (dict(B=-1), EINVAL, "sizes"), (dict(Hkv=0), EINVAL, "sizes"), (dict(D=0), EINVAL, "sizes"),
    (dict(D=100), EUNSUPPORTED, "multiple of 32"), (dict(D=288), EUNSUPPORTED, "up to 256"),
    (dict(page=20), EUNSUPPORTED, "multiple of 8"), (dict(mp=1 << 40), EINVAL, "too large"),
    (dict(B=1 << 30), EINVAL, "too large"),
    (dict(cs=2 * 8 * 64 * 64 - 16), EINVAL, "stride"), (dict(cs=2 * 8 * 64 * 64 + 8), EINVAL, "stride"),
    (dict(ss=2 * 8 * 4 * 64 - 8), EINVAL, "stride"), (dict(ss=2 * 8 * 4 * 64 + 4), EINVAL, "stride"),
]


@pytest.mark.parametrize("call", [_append, _read, _attn])
@pytest.mark.parametrize("kw,code,word", SHARED)
def test_pool_refusals(call, kw, code, word):
    assert call(**kw) == code
    assert word in lib.load().tlm_last_error().decode()


@pytest.mark.parametrize("call,kw,code,word", [
    (_append, dict(k=None), EINVAL, "null"), (_append, dict(v=None), EINVAL, "null"),
    (_append, dict(start=None), EINVAL, "null"), (_append, dict(count=None), EINVAL, "null"),
    (_append, dict(dt=lib.F32), EUNSUPPORTED, "dtype"), (_append, dict(k=ODD), EINVAL, "aligned"),
    (_append, dict(kr=1028), EINVAL, "aligned"), (_append, dict(vb=-8), EINVAL, "sizes"),
    (_append, dict(T=-1), EINVAL, "sizes"),
    (_read, dict(cu=None), EINVAL, "null"), (_read, dict(k=None), EINVAL, "null"),
    (_read, dict(v=ODD), EINVAL, "aligned"), (_read, dict(dt=lib.F8E4M3), EUNSUPPORTED, "dtype"),
    (_read, dict(total=-1), EINVAL, "sizes"), (_read, dict(total=1 << 31), EINVAL, "sizes"),
    (_attn, dict(q=None), EINVAL, "null"), (_attn, dict(sl=None), EINVAL, "null"),
    (_attn, dict(o=None), EINVAL, "null"), (_attn, dict(dt=lib.F32), EUNSUPPORTED, "dtype"),
    (_attn, dict(qr=4100), EINVAL, "aligned"), (_attn, dict(q=ODD), EINVAL, "aligned"),
    (_attn, dict(o=ODD), EINVAL, "aligned"), (_attn, dict(lse=ctypes.c_void_p(0x1002)), EINVAL, "aligned"),
    (_attn, dict(H=33), EINVAL, "multiple of H_kv"), (_attn, dict(H=0), EINVAL, "sizes"),
    (_attn, dict(T=-1), EINVAL, "sizes"), (_attn, dict(T=1 << 30), EINVAL, "too large"),
])
def test_refusals(call, kw, code, word):
    assert call(**kw) == code
    assert word in lib.load().tlm_last_error().decode()


def test_empty_calls_do_nothing():
    assert _append(B=0) == 0 and _append(T=0) == 0
    assert _read(B=0) == 0 and _read(total=0) == 0
    assert _attn(B=0) == 0 and _attn(T=0) == 0


def test_empty_calls_take_null_rows():
    none = dict(k=None, v=None, q=None, o=None)
    for no in (dict(B=0, bt=None, start=None, count=None, sl=None), dict(T=0)):
        assert _append(**none, **no) == 0 and _attn(**none, **no, ws=None, wb=0) == 0
    assert _read(total=0, k=None, v=None) == 0 and _read(B=0, total=0, bt=None, k=None, v=None) == 0


@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 64), (32, 8, 128), (7, 1, 96), (16, 2, 256), (64, 1, 128), (2000, 1000, 32)])
def test_workspace_of_a_chunk_is_enough_for_steps(H, Hkv, D):
    size = lib.load().tlm_kv4_attn_workspace_bytes
    sizes = [size(3, T, H, Hkv, D) for T in (1, 2, 3, 5, 8, 17, 40, 200, 5000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert size(100, 8, H, Hkv, D) == size(1, 8, H, Hkv, D)
    assert size(0, 1, H, Hkv, D) == 0


@pytest.mark.parametrize("call", [_append, _read, _attn])
def test_more_sequences_than_their_numbers_hold(call):
    """From 2^31 - 2^16 sequences on, the number of one and the depth of a grid would pass 2^31 together."""
    small = dict(mp=1, Hkv=1, H=1, page=8, cs=8 * 128, ss=2 * 8 * 4)
    for B in (2 ** 31 - 2 ** 16, 2 ** 31 - 100):
        assert call(B=B, **small) == EINVAL
        assert "sequences" in lib.load().tlm_last_error().decode()
