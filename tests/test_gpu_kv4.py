"""The 4-bit K/V cache on the GPU: tlm_kv4_append and tlm_kv4_read bit for bit and tlm_kv4_attn within
its roundings of oracle/ref.py's kv4_* (float64), and runs of them together."""
import numpy as np
import pytest
import torch

from oracle import ref
from tilelang.jit.adapter.mi355x import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16


def _i32(v):
    return torch.as_tensor(np.asarray(v), dtype=torch.int32).to(DEV)


def _pools(pages, Hkv, page, D, seed=0, lo=122, hi=127):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (pages, 2, Hkv, page, D // 2), generator=g).byte(),
            torch.randint(lo, hi, (pages, 2, Hkv, D // 32, page), generator=g).byte())


def _append(k, v, start, count, bt, codes, scales):
    c, s = codes.to(DEV), scales.to(DEV)
    ops.kv4_append(k.to(DEV), v.to(DEV), _i32(start), _i32(count), _i32(bt), c, s)
    return c.cpu().numpy(), s.cpu().numpy()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hkv,D,page", [(1, 32, 8), (8, 128, 64), (3, 96, 24), (2, 256, 16), (5, 64, 40)])
def test_append_bit_exact(dtype, Hkv, D, page):
    g = torch.Generator().manual_seed(11)
    B, T, per = 5, 70, -(-150 // page)
    k, v = ((torch.randn(B, T, Hkv, D, generator=g) * torch.exp(3 * torch.randn(B, T, Hkv, 1, generator=g))).to(dtype)
            for _ in "kv")
    pages = B * per + 3
    bt = torch.randperm(pages, generator=g)[:B * per].view(B, per).int().numpy()
    start = np.array([0, 5, per * page - 33, 63, 64], np.int32)  # sequence 2 runs out of its table
    count = np.array([70, 0, 70, 1, 200], np.int32)              # 200: more than T
    codes, scales = _pools(pages, Hkv, page, D)
    got = _append(k, v, start, count, bt, codes, scales)
    exp = ref.kv4_append_ref(k, v, start, count, bt, codes.numpy(), scales.numpy())
    assert np.array_equal(got[0], exp[0]) and np.array_equal(got[1], exp[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_every_value(dtype):
    """Every 16-bit pattern as the block's only value, and beside a larger one (rounding at each scale)."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.zeros(1, 1024, 8, 256, dtype=dtype)
    x.view(-1, 32)[:, 0] = bits
    y = x.clone()
    y.view(-1, 32)[:, 1] = torch.ldexp(bits.abs().nan_to_num(0, 0, 0).float(), torch.arange(65536) % 5).to(dtype)
    codes, scales = _pools(16, 8, 64, 256)
    bt = np.arange(16, dtype=np.int32).reshape(1, 16)
    got = _append(x, y, [0], [1024], bt, codes, scales)
    exp = ref.kv4_append_ref(x, y, [0], [1024], bt, codes.numpy(), scales.numpy())
    assert np.array_equal(got[0], exp[0]) and np.array_equal(got[1], exp[1])


def test_append_corrupt_tables_and_positions():
    g = torch.Generator().manual_seed(12)
    k, v = (torch.randn(3, 20, 2, 64, generator=g).to(BF16) for _ in "kv")
    bt = np.array([[1, -5, 3], [1 << 30, 0, 4], [2, 5, -2147483648]], np.int32)
    start, count = np.array([4, 0, -7], np.int32), np.array([20, 20, 20], np.int32)
    codes, scales = _pools(4, 2, 8, 64)  # pages 4 and 5 do not exist
    got = _append(k, v, start, count, bt, codes, scales)
    exp = ref.kv4_append_ref(k, v, start, count, bt, codes.numpy(), scales.numpy())
    assert np.array_equal(got[0], exp[0]) and np.array_equal(got[1], exp[1])


def _layers(pages, layers, Hkv, page, D):
    """Pools of one layer out of several that alternate page by page."""
    codes = torch.full((pages, layers, 2, Hkv, page, D // 2), 0x11, dtype=torch.uint8, device=DEV)
    scales = torch.full((pages, layers, 2, Hkv, D // 32, page), 0x22, dtype=torch.uint8, device=DEV)
    return codes, scales


def test_append_and_read_slices():
    """K and V as slices of one projection's rows, pools as one layer of several; the rest stays."""
    g = torch.Generator().manual_seed(13)
    B, T, H, Hkv, D, page = 3, 9, 4, 2, 64, 16
    qkv = torch.randn(B, T + 2, (H + 2 * Hkv) * D, generator=g).to(BF16).to(DEV)[:, 1:-1]
    k = qkv[..., H * D:(H + Hkv) * D].view(B, T, Hkv, D)
    v = qkv[..., (H + Hkv) * D:].view(B, T, Hkv, D)
    codes, scales = _layers(4, 3, Hkv, page, D)
    bt, start, count = _i32([[3], [0], [2]]), _i32([2, 0, 7]), _i32([9, 4, 9])
    ops.kv4_append(k, v, start, count, bt, codes[:, 1], scales[:, 1])
    exp = ref.kv4_append_ref(k.cpu(), v.cpu(), [2, 0, 7], [9, 4, 9], bt.cpu().numpy(),
                             np.full((4, 2, Hkv, page, D // 2), 0x11, np.uint8),
                             np.full((4, 2, Hkv, D // 32, page), 0x22, np.uint8))
    assert np.array_equal(codes[:, 1].cpu().numpy(), exp[0])
    assert np.array_equal(scales[:, 1].cpu().numpy(), exp[1])
    for i in (0, 2):
        assert (codes[:, i] == 0x11).all() and (scales[:, i] == 0x22).all()
    cu = _i32([0, 9, 13, 22])
    ko, vo = (torch.empty(22, Hkv, D, dtype=BF16, device=DEV) for _ in "kv")
    ops.kv4_read(codes[:, 1], scales[:, 1], bt, start, cu, ko, vo)
    for got, x in ((ko, k), (vo, v)):
        x = torch.cat([x[b, :n] for b, n in enumerate((9, 4, 9))]).cpu()
        assert np.array_equal(got.double().cpu().numpy(), ref.kv4_dequantise_ref(*ref.kv4_quantise_ref(x)))


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
@pytest.mark.parametrize("Hkv,D,page", [(1, 32, 8), (8, 128, 64), (3, 96, 24), (2, 256, 16)])
def test_read_bit_exact(dtype, Hkv, D, page):
    g = torch.Generator().manual_seed(14)
    B, per = 5, 6
    pages = B * per
    codes, scales = _pools(pages, Hkv, page, D, 15, 0, 256)  # every scale, NaN among them
    bt = torch.randperm(pages, generator=g).view(B, per).int().numpy()
    bt[1, 2], bt[3, 0] = -1, pages
    n = [2 * page + 3, 4 * page, 0, 1, per * page + 5]  # the last reads past its table
    start = [0, 3, 7, 2 * page, 0]
    cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    for first in (None, start):
        outs = [torch.full((int(cu[-1]) + 3, Hkv, D), 7.0, dtype=dtype, device=DEV) for _ in "kv"]
        ops.kv4_read(codes.to(DEV), scales.to(DEV), _i32(bt), None if first is None else _i32(first), _i32(cu),
                     *outs)
        for w, out in enumerate(outs):
            exp = np.concatenate([ref.kv4_rows_ref(codes.numpy(), scales.numpy(), bt, b,
                                                   0 if first is None else start[b], n[b])[w] for b in range(B)])
            with np.errstate(all="ignore"):  # one rounding, as torch's cast of the fp64 value
                exp = torch.from_numpy(exp).to(dtype)
            assert torch.equal(out[:len(exp)].cpu().nan_to_num(123.0, posinf=456.0, neginf=-456.0),
                               exp.nan_to_num(123.0, posinf=456.0, neginf=-456.0))
            assert (out[len(exp):] == 7).all()


def _attn_case(dtype, B, T, H, Hkv, D, page, lens, seed=0, pages=None, q_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    per = max(1, -(-max(lens) // page))
    pages = pages or B * per + 2
    x = torch.randn(pages, 2, Hkv, page, D, generator=g)
    x[..., ::17] *= 6
    codes, scales = ref.kv4_quantise_ref(x)
    codes, scales = torch.from_numpy(codes), torch.from_numpy(np.ascontiguousarray(scales.swapaxes(-1, -2)))
    bt = torch.randperm(pages, generator=g)[:B * per].view(B, per).int().numpy()
    q = (torch.randn(B, T, H, D, generator=g) * q_scale).to(dtype)
    return q, codes, scales, bt


def _stale(codes, scales, bt, lens, page):
    """NaN in every place that no sequence uses."""
    codes, scales = codes.clone(), scales.clone()
    live = torch.zeros(codes.shape[0], page, dtype=torch.bool)
    for b, n in enumerate(lens):
        p = np.arange(n)
        live[torch.from_numpy(bt[b, p // page].astype(np.int64)), torch.from_numpy(p % page)] = True
    scales[~live[:, None, None, None, :].expand_as(scales)] = 255
    codes[~live[:, None, None, :, None].expand_as(codes)] = 0
    return codes, scales


def _run(q, codes, scales, bt, lens, count=None, causal=True, scale=None, lse=True, ws_fill=0xFF):
    B, T, H, D = q.shape
    out = torch.full((B, T, H, D), 9.0, dtype=q.dtype, device=DEV)
    z = torch.full((B, T, H), 9.0, device=DEV) if lse else None
    need = ops.kv4_attn_workspace_bytes(B, T, H, codes.shape[2], D)
    ws = torch.full((max(16, need),), ws_fill, dtype=torch.uint8, device=DEV)  # all ones: NaN
    ops.kv4_attn(q.to(DEV), codes.to(DEV), scales.to(DEV), _i32(bt), _i32(lens), out, ws,
                 D ** -0.5 if scale is None else scale, None if count is None else _i32(count), causal, z)
    torch.cuda.synchronize()
    return out.cpu(), None if z is None else z.cpu()


def _check(q, codes, scales, bt, lens, count=None, causal=True, scale=None, got=None):
    """Within the kernel's roundings of the float64 result. A score is a sum of D exact products in fp32 (q
    and the cached values are exact in its operands): off by at most (D + 2) 2^-24 of the sum of
    magnitudes A. A weight is off by that times ln 2 log2 e = 1, by exp2 (1 ulp, and its argument's
    rounding against a reference within the scores' range: 2 A 2^-24) and by its rounding where it multiplies V: with fp16
    queries two bf16 terms (2^-17), with bf16 ones fp16 (half a step is 2^-11, and half of fp16's smallest, 2^-25, where
    the largest weight is 2^11 at least: n 2^-36 of the largest |v| of the dim in all; where the key that has the
    weight has a V of 0, as in one of 64 keys at 57 bits above the others, that is more than the rest).
    Numerator and denominator are sums of up to n weights, (n + 64) 2^-24 each; the quotient is
    rounded once: by eps / 2, or half of the smallest subnormal, tiny eps / 2 (an output of 4.5e-7 is
    0.46 of fp16's 2^-24 steps off its nearest multiple: no fp16 value is nearer)."""
    B, T, H, D = q.shape
    sm = D ** -0.5 if scale is None else scale
    page = codes.shape[3]
    c, s = codes.numpy(), scales.numpy()
    exp, lse = ref.kv4_attn_ref(q, c, s, bt, lens, count, sm, causal)
    # sum p |v| / l, and the largest sum of magnitudes of a score, by the same reference on |v| and |q|, |k|
    mag = c.copy()
    mag[:, 1] &= 0x77
    spread, _ = ref.kv4_attn_ref(q, mag, s, bt, lens, count, sm, causal)
    out, z = got if got is not None else _run(q, codes, scales, bt, lens, count, causal, scale)
    eps = torch.finfo(q.dtype).eps / 2
    least = torch.finfo(q.dtype).tiny * eps
    weight = 2.0 ** -11 if q.dtype == BF16 else 2.0 ** -16
    for b in range(B):
        n = max(0, min(int(lens[b]), bt.shape[1] * page))
        m = T if count is None else max(0, min(int(count[b]), T))
        k, v = ref.kv4_rows_ref(c, s, bt, b, 0, n)
        k = np.abs(k).repeat(H // codes.shape[2], 1).transpose(1, 2, 0)
        a = np.abs(q[b, :m].double().numpy()).transpose(1, 0, 2) @ k * abs(sm) if n else np.zeros((H, m, 1))
        a = a.max(-1).T[..., None]  # [m, H, 1]
        v = np.nan_to_num(np.abs(v)).max(0, initial=0.0).repeat(H // codes.shape[2], 0)  # [H, D]
        small = n * 2.0 ** -36 * v if q.dtype == BF16 else 0.0
        rel = 2 * ((D + 4) * 2.0 ** -24 * a + 2.0 ** -23 + (n + 64) * 2.0 ** -24) + weight
        x, e = out[b, :m].double().numpy(), exp[b, :m]
        # beyond the type's range values become infinite, surely so by more than they may be off
        lim, most = eps * (1 + 2 ** -10) * np.abs(e) + rel * spread[b, :m], torch.finfo(q.dtype).max * (1 + eps)
        inf = np.abs(e) - lim > most
        assert (x[inf] == np.copysign(np.inf, e[inf])).all()
        inf |= np.isinf(x) & (np.abs(e) + lim > most)
        x, e = np.where(inf, 0.0, x), np.where(inf, 0.0, e)
        bad = np.abs(x - e) > eps * (1 + 2 ** -10) * np.abs(e) + rel * spread[b, :m] + small + least
        assert not bad.any(), (b, np.abs(x - e).max())
        assert np.array_equal(np.isnan(x), np.isnan(e))
        assert (out[b, m:] == 9).all()
        if z is not None:
            zz, ee = z[b, :m].double().numpy(), lse[b, :m]
            fin = np.isfinite(ee)
            assert np.array_equal(zz[~fin & ~np.isnan(ee)], ee[~fin & ~np.isnan(ee)])
            lim = (rel[..., 0] + 2.0 ** -22 * (np.abs(np.where(fin, ee, 0)) + 4)) * 1.5
            assert (np.abs(zz[fin] - ee[fin]) <= lim[fin]).all()
            assert (z[b, m:] == 9).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attn_head_dims(dtype, D):
    lens = [1, 33, 500]
    q, c, s, bt = _attn_case(dtype, 3, 1, 8, 2, D, 16, lens, D)
    _check(q, *_stale(c, s, bt, lens, 16), bt, lens)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (5, 5), (7, 1), (16, 1), (17, 1), (33, 1), (64, 2), (128, 1), (24, 3)])
def test_attn_head_groups(H, Hkv):
    lens = [70, 1, 259]
    q, c, s, bt = _attn_case(BF16, 3, 1, H, Hkv, 128, 64, lens, H)
    _check(q, *_stale(c, s, bt, lens, 64), bt, lens)


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 1000])
def test_attn_pages(page):
    lens = [1, 7, 8, 31, 32, 33, 63, 64, 65, 127, 129, 300]
    q, c, s, bt = _attn_case(F16, 12, 1, 8, 2, 64, page, lens, page)
    _check(q, *_stale(c, s, bt, lens, page), bt, lens)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,H,Hkv,D", [(2, 8, 8, 64), (5, 32, 4, 128), (17, 4, 2, 96), (64, 8, 2, 128), (130, 3, 1, 256)])
def test_attn_several_new_tokens(T, H, Hkv, D, causal):
    """Chunks of T with fewer of them in some sequences; sequences shorter than their new tokens, whose
    first rows see nothing when causal; rows past count untouched."""
    lens, count = [T, 300, T // 2, 0, 450], [T, max(1, T - 1), T, T, 0]
    q, c, s, bt = _attn_case(BF16, 5, T, H, Hkv, D, 16, lens, T)
    _check(q, *_stale(c, s, bt, lens, 16), bt, lens, count, causal)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attn_long_and_short_together(dtype):
    lens = [6000, 1, 0, 40, 3333, 2, 900]
    q, c, s, bt = _attn_case(dtype, 7, 1, 16, 4, 128, 64, lens, 3)
    _check(q, *_stale(c, s, bt, lens, 64), bt, lens)


def test_attn_many_sequences():
    lens = [(7 * i) % 41 for i in range(700)]
    q, c, s, bt = _attn_case(F16, 700, 1, 4, 2, 64, 8, lens, 4)
    _check(q, *_stale(c, s, bt, lens, 8), bt, lens)


def test_attn_lengths_past_the_table_and_below_zero():
    q, c, s, bt = _attn_case(BF16, 3, 2, 8, 2, 64, 16, [64, 64, 64], 5)
    _check(q, c, s, bt, [1000, -3, 2147483647])
    _check(q, c, s, bt, [64, 10, 64], count=[-1, 1000, 2])


def test_attn_missing_pages_read_as_zeros():
    q, c, s, bt = _attn_case(F16, 3, 1, 8, 2, 128, 16, [100, 90, 48], 6)
    bt[0, 2], bt[1, 0], bt[2, 2] = -1, c.shape[0], 2147483647
    _check(q, c, s, bt, [100, 90, 48])
    bt[2] = -7  # a sequence of zeros: its output is 0, its sum-exp log2 of its length
    _check(q, c, s, bt, [100, 90, 48])


def test_attn_same_page_twice():
    """Pages that two sequences share (a common prefix) and one that a sequence holds twice."""
    lens = [80, 95, 70]
    q, c, s, bt = _attn_case(BF16, 3, 1, 8, 4, 128, 16, lens, 7)
    bt[1, :3] = bt[0, :3]
    bt[2, 3] = bt[2, 0]
    _check(q, c, s, bt, lens)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attn_sharp_and_large_scores(dtype):
    """Scores in the thousands: softmax picks single keys; and a scale of 0: the mean of V."""
    lens = [700, 33, 5]
    q, c, s, bt = _attn_case(dtype, 3, 1, 8, 2, 128, 64, lens, 8, q_scale=200.0)
    _check(q, c, s, bt, lens, scale=1.0)
    _check(q, c, s, bt, lens, scale=0.0)
    _check(q, c, s, bt, lens, scale=-0.5)


def test_attn_growing_scores():
    """Every tile's maximum far above the last one's, and far below it."""
    lens = [1500, 1500]
    q, c, s, bt = _attn_case(BF16, 2, 1, 4, 1, 64, 16, lens, 9)
    q = torch.ones_like(q)
    c[:, 0] = 0x22  # K: ones
    for p in range(1500):
        for b, up in ((0, p), (1, 1499 - p)):
            s[int(bt[b, p // 16]), 0, :, :, p % 16] = 118 + up // 100
    _check(q, c, s, bt, lens, scale=1.0)


def test_attn_nan_and_extreme_blocks():
    """A NaN block of K or V in sight makes the rows that see it NaN, and only those; K's scales at both ends."""
    lens = [100, 100, 100, 100]
    q, c, s, bt = _attn_case(BF16, 4, 3, 4, 2, 64, 16, lens, 10)
    s[int(bt[0, 98 // 16]), 0, 1, 0, 98 % 16] = 255  # K of sequence 0, position 98, head 1: queries 1 and 2
    s[int(bt[1, 0]), 1, 0, 1, 3] = 255               # V of sequence 1, head 0, dims 32 ..
    s[int(bt[2, 1]), 0, :, :, 5] = 1                 # a key of nothing
    out, lse = _run(q, c, s, bt, lens)
    nan = torch.zeros(4, 3, 4, 64, dtype=torch.bool)
    nan[0, 1:, 2:] = True
    nan[1, :, :2, 32:] = True
    assert torch.equal(out.isnan(), nan)
    keep = [2, 3]
    _check(q[keep], c, s, bt[keep], [100, 100], got=(out[keep], lse[keep]))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,T,H,Hkv", [(64, 1, 8, 2), (128, 1, 4, 4), (128, 9, 8, 2), (256, 1, 8, 1), (96, 3, 4, 2)])
def test_attn_scales_outside_fp16(dtype, D, T, H, Hkv):
    """Blocks of K and V whose values fp16 does not hold, from some tile on, in single tiles and in the last one; and
    blocks of zeros."""
    lens = [900, 333, 64, 31]
    q, c, s, bt = _attn_case(dtype, 4, T, H, Hkv, D, 16, lens, D + T)
    page = lambda b, p: (int(bt[b, p // 16]), p % 16)
    for b, first, n in ((0, 500, 3), (0, 890, 10), (1, 0, 2), (1, 332, 1), (3, 5, 1)):
        for p in range(first, first + n):
            i, off = page(b, p)
            s[i, 1, :, :, off] = torch.tensor([60, 100, 141, 200])[p % 4]  # V
            s[i, 0, :, 0, off] = torch.tensor([1, 40, 108, 90])[p % 4]     # K: next to nothing
    i, off = page(2, 40)
    s[i, 0, :, :, off] = 143  # a key of up to 6 2^16, seen by queries scaled down
    q[2] = (q[2].float() * 2.0 ** -12).to(dtype)
    i, off = page(0, 100)
    c[i, :, :, off], s[i, :, :, :, off] = 0, 1  # zeros
    _check(q, *_stale(c, s, bt, lens, 16), bt, lens)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H,Hkv,D", [(5, 4, 2, 128), (40, 4, 1, 64), (3, 8, 8, 256), (6, 2, 1, 96)])
def test_attn_nan_of_later_tokens(dtype, T, H, Hkv, D):
    """A NaN of V or K at a position makes NaN of the queries at and behind it, and of none before it."""
    lens = [77, T, 200]
    q, c, s, bt = _attn_case(dtype, 3, T, H, Hkv, D, 16, lens, T + 31)
    clean = _run(q, c, s, bt, lens)
    at = [lens[0] - 2, lens[1] - 1, lens[2] - T]  # seen by the last two, the last, all
    for b, p in enumerate(at):
        s[int(bt[b, p // 16]), 1 if b != 1 else 0, Hkv - 1, D // 32 - 1, p % 16] = 255
    out, lse = _run(q, c, s, bt, lens)
    nan = torch.zeros(out.shape, dtype=torch.bool)
    head = H - H // Hkv
    nan[0, T - 2:, head:, D - 32:] = True
    nan[1, T - 1:, head:] = True
    nan[2, :, head:, D - 32:] = True
    assert torch.equal(out.isnan(), nan)
    assert torch.equal(lse.isnan(), nan.all(-1))
    # the others as before, but for the form in which the tile was computed
    eps = torch.finfo(dtype).eps
    err = (out.float() - clean[0].float()).abs()[~nan]
    assert (err <= 2 * eps * clean[0].float().abs()[~nan] + 2.0 ** -9 * clean[0].float().abs().max()).all()


def test_attn_strided_queries_and_layers():
    g = torch.Generator().manual_seed(15)
    B, T, H, Hkv, D, page = 3, 2, 8, 2, 64, 16
    lens = [30, 77, 5]
    q, c, s, bt = _attn_case(BF16, B, T, H, Hkv, D, page, lens, 11)
    codes, scales = _layers(c.shape[0], 3, Hkv, page, D)
    codes[:, 2], scales[:, 2] = c.to(DEV), s.to(DEV)
    wide = torch.randn(B, T + 1, (H + 4) * D, generator=g).to(BF16).to(DEV)
    wide[:, 1:, 2 * D:(2 + H) * D] = q.flatten(2).to(DEV)
    view = wide[:, 1:, 2 * D:(2 + H) * D].view(B, T, H, D)
    out = torch.full((B, T, H, D), 9.0, dtype=BF16, device=DEV)
    ws = torch.empty(max(16, ops.kv4_attn_workspace_bytes(B, T, H, Hkv, D)), dtype=torch.uint8, device=DEV)
    ops.kv4_attn(view, codes[:, 2], scales[:, 2], _i32(bt), _i32(lens), out, ws, D ** -0.5)
    _check(q, c, s, bt, lens, got=(out.cpu(), None))


def test_pools_past_4_gb():
    """Pages behind the 4 GB of their pool, written, read and attended."""
    Hkv, page, D = 8, 128, 128
    pages = (1 << 32) // (Hkv * page * D) + 3
    codes = torch.empty(pages, 2, Hkv, page, D // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(pages, 2, Hkv, D // 32, page, dtype=torch.uint8, device=DEV)
    g = torch.Generator().manual_seed(16)
    k, v = (torch.randn(1, 200, Hkv, D, generator=g).to(BF16) for _ in "kv")
    bt = np.array([[pages - 1, pages - 2]], np.int32)
    ops.kv4_append(k.to(DEV), v.to(DEV), _i32([0]), _i32([200]), _i32(bt), codes, scales)
    ko, vo = (torch.empty(200, Hkv, D, dtype=BF16, device=DEV) for _ in "kv")
    ops.kv4_read(codes, scales, _i32(bt), None, _i32([0, 200]), ko, vo)
    for got, x in ((ko, k), (vo, v)):
        assert np.array_equal(got.double().cpu().numpy(), ref.kv4_dequantise_ref(*ref.kv4_quantise_ref(x[0])))
    q = torch.randn(1, 1, 16, D, generator=g).to(BF16)
    out = torch.empty(1, 1, 16, D, dtype=BF16, device=DEV)
    ws = torch.empty(max(16, ops.kv4_attn_workspace_bytes(1, 1, 16, Hkv, D)), dtype=torch.uint8, device=DEV)
    ops.kv4_attn(q.to(DEV), codes, scales, _i32(bt), _i32([200]), out, ws, D ** -0.5)
    _check(q, codes[-2:].cpu(), scales[-2:].cpu(), np.array([[1, 0]], np.int32), [200], got=(out.cpu(), None))


def _prompt_and_steps(dtype, H, Hkv, D, page, prompts, chunk, steps):
    """Prompts written and attended chunk by chunk, then decode steps: every output against the oracle on the
    cache as it then is."""
    g = torch.Generator().manual_seed(17)
    B = len(prompts)
    per = -(-(max(prompts) + steps) // page)
    codes, scales = (x.to(DEV) for x in _pools(B * per, Hkv, page, D, 18, 255, 256))  # NaN: nothing written yet
    bt = torch.randperm(B * per, generator=g).view(B, per).int().numpy()
    have = np.zeros(B, np.int64)
    goal = np.array(prompts)
    ws = torch.empty(max(16, ops.kv4_attn_workspace_bytes(B, chunk, H, Hkv, D)), dtype=torch.uint8, device=DEV)
    while steps >= 0:
        T = chunk if (have < goal).any() else 1
        new = np.minimum(goal - have, T) if T > 1 else np.ones(B, np.int64)
        q = torch.randn(B, T, H, D, generator=g).to(dtype)
        k, v = (torch.randn(B, T, Hkv, D, generator=g).to(dtype) for _ in "kv")
        ops.kv4_append(k.to(DEV), v.to(DEV), _i32(have), _i32(new), _i32(bt), codes, scales)
        have += new
        out = torch.full((B, T, H, D), 9.0, dtype=dtype, device=DEV)
        ops.kv4_attn(q.to(DEV), codes, scales, _i32(bt), _i32(have), out, ws, D ** -0.5, _i32(new))
        _check(q, codes.cpu(), scales.cpu(), bt, have, new, got=(out.cpu(), None))
        steps -= T == 1
    return codes, scales, bt, have, g


def test_prompt_then_decode_steps():
    dtype, H, Hkv, D, page = BF16, 8, 2, 128, 16
    codes, scales, bt, have, g = _prompt_and_steps(dtype, H, Hkv, D, page, [100, 37, 64], 40, 3)
    # the prompt read back for attention over unquantised rows gives the same attention: all but the 16-bit
    # weights of that kernel (eps / 2 of each) are in the bound of the cache's own
    cu = np.concatenate([[0], np.cumsum(have)]).astype(np.int32)
    total = int(cu[-1])
    ko, vo = (torch.empty(total, Hkv, D, dtype=dtype, device=DEV) for _ in "kv")
    ops.kv4_read(codes, scales, _i32(bt), None, _i32(cu), ko, vo)
    T = 8
    q = torch.randn(3, T, H, D, generator=g).to(dtype)
    flat, o = q.flatten(0, 1).to(DEV), torch.empty(3 * T, H, D, dtype=dtype, device=DEV)
    ops.flash_attn_varlen_fwd(flat, ko, vo, _i32([0, T, 2 * T, 3 * T]), _i32(cu), T, o, True, D ** -0.5)
    out, _ = _run(q, codes.cpu(), scales.cpu(), bt, have)
    spread = vo.abs().max().item()
    assert (o.view_as(out).cpu().float() - out.float()).abs().max().item() <= 4 * torch.finfo(dtype).eps * spread


def test_prompt_then_decode_steps_f16_odd():
    _prompt_and_steps(F16, 9, 3, 96, 24, [50, 3, 77], 33, 2)


def test_same_bits_again_and_on_two_streams():
    lens = [3000, 100, 1700, 5]
    q, c, s, bt = _attn_case(BF16, 4, 1, 32, 8, 128, 64, lens, 19)
    args = (q.to(DEV), c.to(DEV), s.to(DEV), _i32(bt), _i32(lens))
    need = max(16, ops.kv4_attn_workspace_bytes(4, 1, 32, 8, 128))
    first = torch.empty_like(args[0])
    ops.kv4_attn(*args, first, torch.empty(need, dtype=torch.uint8, device=DEV), 0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(first) for _ in range(6)] for _ in streams]
    spaces = [torch.empty(need, dtype=torch.uint8, device=DEV) for _ in streams]
    for i in range(6):
        for st, o, w in zip(streams, outs, spaces):
            with torch.cuda.stream(st):
                ops.kv4_attn(*args, o[i], w, 0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for os in outs for o in os)


def test_decode_step_in_a_graph():
    """Append and attention captured once, replayed with other rows, lengths and tables; each replay equals the
    eager calls."""
    g = torch.Generator().manual_seed(20)
    B, H, Hkv, D, page = 4, 16, 4, 128, 32
    lens = [200, 64, 1000, 1]
    q, c, s, bt = _attn_case(BF16, B, 1, H, Hkv, D, page, [1040] * 4, 21)
    c, s, q, bt = c.to(DEV), s.to(DEV), q.to(DEV), _i32(bt)
    k, v = (torch.randn(B, 1, Hkv, D, generator=g).to(BF16).to(DEV) for _ in "kv")
    start, sl, one = _i32(lens), _i32(lens) + 1, _i32([1] * B)
    out = torch.empty_like(q)
    ws = torch.empty(max(16, ops.kv4_attn_workspace_bytes(B, 1, H, Hkv, D)), dtype=torch.uint8, device=DEV)

    def step(out, c, s, ws):
        ops.kv4_append(k, v, start, one, bt, c, s)
        ops.kv4_attn(q, c, s, bt, sl, out, ws, D ** -0.5)

    step(out, c, s, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out, c, s, ws)
    c2, s2, ws2, out2 = c.clone(), s.clone(), torch.empty_like(ws), torch.empty_like(out)
    for i in range(5):
        q.copy_(torch.randn(q.shape, generator=g))
        k.copy_(torch.randn(k.shape, generator=g))
        v.copy_(torch.randn(v.shape, generator=g))
        n = torch.randint(0, 1039, (B,), generator=g).int()
        start.copy_(n)
        sl.copy_(n + 1)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        step(out2, c2, s2, ws2)
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.equal(c, c2) and torch.equal(s, s2), i


def test_ops_refusals():
    q, c, s, bt = _attn_case(BF16, 2, 1, 8, 2, 64, 16, [20, 20], 22)
    q, c, s, bt, sl = q.to(DEV), c.to(DEV), s.to(DEV), _i32(bt), _i32([20, 20])
    out, ws = torch.empty_like(q), torch.empty(1 << 24, dtype=torch.uint8, device=DEV)
    k = torch.zeros(2, 1, 2, 64, dtype=BF16, device=DEV)
    one = _i32([1, 1])
    bad = [
        lambda: ops.kv4_attn(q.cpu(), c, s, bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q[..., :32], c, s, bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q.transpose(2, 3).contiguous().transpose(2, 3), c, s, bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q[:, :, :7], c, s, bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q, c[:, :1], s, bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q, c, s[:, :, :, :1], bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q, c.int(), s, bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q, c.transpose(2, 3).contiguous().transpose(2, 3), s, bt, sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q, c, s, bt.long(), sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q, c, s, bt[:1], sl, out, ws, 0.1),
        lambda: ops.kv4_attn(q, c, s, bt, sl[:1], out, ws, 0.1),
        lambda: ops.kv4_attn(q, c, s, bt, sl, out.float(), ws, 0.1),
        lambda: ops.kv4_attn(q, c, s, bt, sl, out, ws, 0.1, count=one[:1]),
        lambda: ops.kv4_attn(q, c, s, bt, sl, out, ws, 0.1, lse=torch.empty(2, 1, 8, device=DEV, dtype=BF16)),
        lambda: ops.kv4_append(k, k[:1], one, one, bt, c, s),
        lambda: ops.kv4_append(k, k.half(), one, one, bt, c, s),
        lambda: ops.kv4_append(k, k, one.long(), one, bt, c, s),
        lambda: ops.kv4_append(k[:, :, :1], k[:, :, :1], one, one, bt, c, s),
        lambda: ops.kv4_read(c, s, bt, None, one, k[0], k[0]),
        lambda: ops.kv4_read(c, s, bt, None, _i32([0, 1, 2]), k[:, 0], k[:1, 0]),
        lambda: ops.kv4_read(c, s, bt, one.long(), _i32([0, 1, 2]), k[:, 0], k[:, 0].clone()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError(i)


@pytest.mark.parametrize("seed", range(24))
def test_attn_random(seed):
    """Batches, heads, dims, pages, lengths and new tokens at random: how the work is cut depends on all of them."""
    r = np.random.RandomState(100 + seed)
    D = int(r.choice([32, 64, 96, 128, 160, 192, 224, 256]))
    Hkv = int(r.choice([1, 2, 3, 8]))
    H = Hkv * int(r.choice([1, 2, 4, 5, 8, 17]))
    page = int(r.choice([8, 16, 24, 32, 48, 64]))
    B = int(r.choice([1, 2, 5, 20, 65, 130]))
    T = int(r.choice([1, 1, 2, 7, 40])) if B <= 20 else int(r.choice([1, 3]))
    top = int(np.exp(r.uniform(0, np.log(20000 // B))))
    lens = r.randint(0, top + 1, B)
    lens[r.randint(B)] = max(1, top)
    count = r.randint(0, T + 1, B) if r.rand() < 0.5 else None
    dtype = BF16 if r.rand() < 0.5 else F16
    q, c, s, bt = _attn_case(dtype, B, T, H, Hkv, D, page, list(lens), seed)
    _check(q, *_stale(c, s, bt, lens, page), bt, lens, count, bool(r.rand() < 0.7))


@pytest.mark.parametrize("H,Hkv,D", [(1000, 1000, 32), (1040, 520, 160)])
def test_attn_more_kv_heads_than_workgroups_at_once(H, Hkv, D):
    lens = [100, 0, 37]
    q, c, s, bt = _attn_case(BF16, 3, 1, H, Hkv, D, 8, lens, 31)
    _check(q, *_stale(c, s, bt, lens, 8), bt, lens)
    _check(q, c, s, bt, [0, 0, 0])
    _check(q[:1], c, s, bt[:1], [0])
    _check(q[:1], c, s, bt[:1], [1])


def test_attn_large_pages():
    lens = [16500, 8199, 8201]
    q, c, s, bt = _attn_case(F16, 3, 2, 2, 1, 32, 8200, lens, 32)
    _check(q, *_stale(c, s, bt, lens, 8200), bt, lens)


def test_attn_one_query_for_all_sequences():
    """An expanded batch: a batch stride of 0."""
    lens = [300, 5, 64]
    q, c, s, bt = _attn_case(BF16, 1, 3, 8, 2, 64, 16, [300] * 3, 33, pages=60)
    bt = np.arange(57, dtype=np.int32).reshape(3, 19)
    qd = q.to(DEV).expand(3, 3, 8, 64)
    out, z = torch.empty(3, 3, 8, 64, dtype=BF16, device=DEV), torch.empty(3, 3, 8, device=DEV)
    ws = torch.empty(ops.kv4_attn_workspace_bytes(3, 3, 8, 2, 64), dtype=torch.uint8, device=DEV)
    ops.kv4_attn(qd, c.to(DEV), s.to(DEV), _i32(bt), _i32(lens), out, ws, 0.125, lse=z)
    _check(q.expand(3, 3, 8, 64).contiguous(), c, s, bt, lens, got=(out.cpu(), z.cpu()))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attn_scores_of_minus_infinity(dtype):
    """A query that gives all keys -inf is answered like one without keys; a score of +inf or NaN makes its row NaN. Their
    neighbours in the tile are as without them."""
    lens = [200, 200]
    q, c, s, bt = _attn_case(dtype, 2, 1, 8, 2, 64, 16, lens, 34)
    q[:, :, :, 0] = 0
    c[:, 0, :, :, 0] = c[:, 0, :, :, 0] & 0xF0 | 2    # dim 0 of K: 1
    want = _run(q, c, s, bt, lens)
    bad = q.clone()
    bad[0, 0, 2, 0] = -torch.inf
    bad[0, 0, 6, 0], bad[1, 0, 1, 0], bad[1, 0, 7, 0] = -torch.inf, torch.inf, torch.nan
    out, z = _run(bad, c, s, bt, lens)
    for b, h in ((0, 2), (0, 6)):
        assert (out[b, 0, h] == 0).all() and z[b, 0, h] == -torch.inf
    assert out[1, 0, 1].isnan().all() and out[1, 0, 7].isnan().all() and z[1, 0, 7].isnan()
    keep = torch.ones(2, 8, dtype=torch.bool)
    keep[0, 2] = keep[0, 6] = keep[1, 1] = keep[1, 7] = False
    assert torch.equal(out[:, 0][keep], want[0][:, 0][keep]) and torch.equal(z[:, 0][keep], want[1][:, 0][keep])

    one = c.clone()  # one key's dim 0 is -1: its score is +inf
    p = int(bt[0, 150 // 16])
    one[p, 0, :, 150 % 16, 0] = one[p, 0, :, 150 % 16, 0] & 0xF0 | 10
    out, z = _run(bad, one, s, bt, lens)
    assert out[0, 0, 2].isnan().all()


def test_empty_batches_and_steps():
    q, c, s, bt = _attn_case(BF16, 2, 1, 8, 2, 64, 16, [20, 20], 35)
    c, s, bt, n = c.to(DEV), s.to(DEV), _i32(bt), _i32([20, 20])
    before = c.clone(), s.clone()
    ws = torch.empty(1 << 22, dtype=torch.uint8, device=DEV)
    for B, T in ((0, 1), (2, 0), (0, 0)):
        x, kv = torch.empty(B, T, 8, 64, dtype=BF16, device=DEV), torch.empty(B, T, 2, 64, dtype=BF16, device=DEV)
        ops.kv4_append(kv, kv, n[:B], n[:B], bt[:B], c, s)
        ops.kv4_attn(x, c, s, bt[:B], n[:B], x.clone(), ws, 0.1, count=n[:B], lse=torch.empty(B, T, 8, device=DEV))
        ops.kv4_read(c, s, bt[:B], None, torch.zeros(B + 1, dtype=torch.int32, device=DEV), kv.flatten(0, 1),
                     kv.flatten(0, 1))
    torch.cuda.synchronize()
    assert torch.equal(c, before[0]) and torch.equal(s, before[1])


@pytest.mark.parametrize("B,D,Hkv", [(1, 128, 8), (2, 256, 2), (3, 256, 1), (1, 64, 1), (5, 128, 2), (2, 32, 90)])
def test_attn_few_units_per_workgroup(B, D, Hkv):
    """Lengths from none to more units than there are workgroups."""
    q, c, s, bt = _attn_case(BF16, B, 1, 2 * Hkv, Hkv, D, 64, [36000 // B // Hkv + 900] * B, 36)
    for n in (0, 1, 128, 129, 600, 36000 // B // Hkv + 900):
        lens = [max(0, n - 70 * b) for b in range(B)]
        _check(q, c, s, bt, lens)


@pytest.mark.parametrize("B,T,H,Hkv,causal", [(1, 700, 6, 2, True), (1, 515, 8, 1, False), (2, 300, 7, 1, True), (33, 40, 4, 2, True)])
def test_attn_many_row_tiles(B, T, H, Hkv, causal):
    """Chunks of more row tiles than a wave has lanes for the sequence, of unequal numbers of tokens."""
    lens = [T + 100 - 37 * b % 120 for b in range(B)]
    count = [T - 13 * b % T for b in range(B)]
    q, c, s, bt = _attn_case(BF16, B, T, H, Hkv, 64, 16, lens, 37)
    _check(q, *_stale(c, s, bt, lens, 16), bt, lens, count, causal)


@pytest.mark.parametrize("dtype,B,T,Hkv,D", [(BF16, 3, 4000, 9, 128), (F16, 2, 4100, 5, 256), (BF16, 1, 9000, 1, 128)])
def test_append_many_rows(dtype, B, T, Hkv, D):
    """Enough rows for more heads in flight, and heads that do not divide."""
    g = torch.Generator().manual_seed(38)
    per = T // 64 + 1
    k, v = (torch.randn(B, T, Hkv, D, generator=g).to(dtype) for _ in "kv")
    bt = torch.randperm(B * per, generator=g).view(B, per).int().numpy()
    start, count = np.arange(B, dtype=np.int32) * 20, np.array([T, T - 1, 5], np.int32)[:B]
    codes, scales = _pools(B * per, Hkv, 64, D)
    got = _append(k, v, start, count, bt, codes, scales)
    exp = ref.kv4_append_ref(k, v, start, count, bt, codes.numpy(), scales.numpy())
    assert np.array_equal(got[0], exp[0]) and np.array_equal(got[1], exp[1])


def test_read_of_more_than_2_30_sequences():
    """Where the sum of two sequences' numbers does not fit 32 bits: all empty but the last ones."""
    B, Hkv, D, page, pages = (1 << 30) + 5, 1, 32, 8, 3
    codes, scales = _pools(pages, Hkv, page, D, 39)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    cu[-3:] = _i32([5, 5, 12])
    bt = torch.full((B, 1), -1, dtype=torch.int32, device=DEV)
    bt[-3:, 0] = _i32([2, -1, 0])
    outs = [torch.full((14, Hkv, D), 7.0, dtype=F16, device=DEV) for _ in "kv"]
    ops.kv4_read(codes.to(DEV), scales.to(DEV), bt, None, cu, *outs)
    outs = [x.cpu() for x in outs]
    del cu, bt
    torch.cuda.empty_cache()
    last = np.array([[2], [-1], [0]], np.int32)
    for w, out in enumerate(outs):
        exp = np.concatenate([ref.kv4_rows_ref(codes.numpy(), scales.numpy(), last, b, 0, n)[w]
                              for b, n in ((0, 5), (2, 7))])
        assert np.array_equal(out[:12].double().numpy(), exp) and (out[12:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,T,H,Hkv,codes", [(64, 3, 4, 2, 0x10), (128, 9, 8, 2, 0x00), (256, 1, 2, 1, 0x21), (32, 2, 8, 1, 0x77)])
def test_attn_scale_bytes_253_and_254_of_v_are_nan(dtype, D, T, H, Hkv, codes):
    """In a tile that every query sees whole, in one that only later queries see and in one of the slower form, alone and
    together: NaN of the queries that see the block, as from byte 255."""
    lens = [200, 200, 333, 200, 40]
    q, c, s, bt = _attn_case(dtype, 5, T, H, Hkv, D, 16, lens, D + T + 40)
    for b, p, byte in ((0, 10, 253), (1, 199, 254), (2, 40, 254), (2, 332, 253), (3, 70, 253)):
        i, off = int(bt[b, p // 16]), p % 16
        s[i, 1, Hkv - 1, p % (D // 32), off] = byte
        c[i, 1, Hkv - 1, off] = codes
    for w in (0, 1):  # next to nothing and beyond fp16, so that all of sequence 3 is in the slower form
        s[int(bt[3, 0]), w, :, :, 0] = 60
    out = _run(q, c, s, bt, lens)
    s255 = s.clone()
    s255[:, 1][s255[:, 1] >= 253] = 255
    _check(q, c, s255, bt, lens, got=out)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page", [8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("D,T,H,Hkv", [(64, 1, 96, 96), (128, 9, 128, 64)])
def test_attn_missing_pages_after_full_rings(D, T, H, Hkv, page, dtype):
    """Pages outside the pool between others, in whole tiles and in the last one, where every stage of a wave's ring has
    held codes before: few ranges of 6 units or more for each of many K/V heads (of which the first and the last are
    compared)."""
    lens = [3000, 1700, 905]
    g = torch.Generator().manual_seed(page + D)
    per = -(-lens[0] // page)
    c, s = _pools(3 * per + 2, Hkv, page, D, page)
    bt = torch.randperm(3 * per + 2, generator=g)[:3 * per].view(3, per).int().numpy()
    q = torch.randn(3, T, H, D, generator=g).to(dtype)
    c, s = _stale(c, s, bt, lens, page)
    none = [-1, c.shape[0], -2147483648, 2147483647]
    last = [(n - 1) // page for n in lens]
    for b in range(3):
        for p in range(640 // page + b, last[b], 5 if page < 128 else 3):
            bt[b, p] = none[p % 4]
    bt[1, last[1]] = -1  # the masked tile's own page
    out, z = _run(q, c, s, bt, lens)
    for kv in (0, Hkv - 1):
        own = slice(kv * (H // Hkv), (kv + 1) * (H // Hkv))
        _check(q[:, :, own], c[:, :, kv:kv + 1], s[:, :, kv:kv + 1], bt, lens, scale=D ** -0.5,
               got=(out[:, :, own], z[:, :, own]))


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("B", [1022, 1023, 1024, 2000])
def test_read_many_sequences(B, first):
    """As many sequence starts as are searched in LDS, one fewer, one more, and twice as many; empty sequences among them, at
    both ends too."""
    Hkv, D, page, per = 1, 32, 8, 2
    g = torch.Generator().manual_seed(B)
    codes, scales = _pools(B * per, Hkv, page, D, B)
    bt = torch.randperm(B * per, generator=g).view(B, per).int().numpy()
    n = torch.randint(0, 9, (B,), generator=g).numpy()
    n[:3] = n[-2:] = n[B // 2:B // 2 + 5] = 0
    start = torch.randint(0, 9, (B,), generator=g).numpy() if first else np.zeros(B, np.int64)
    cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    outs = [torch.full((int(cu[-1]) + 2, Hkv, D), 7.0, dtype=BF16, device=DEV) for _ in "kv"]
    ops.kv4_read(codes.to(DEV), scales.to(DEV), _i32(bt), _i32(start) if first else None, _i32(cu), *outs)
    rows = [ref.kv4_rows_ref(codes.numpy(), scales.numpy(), bt, b, int(start[b]), int(n[b])) for b in range(B)]
    for w, out in enumerate(outs):
        exp = np.concatenate([r[w] for r in rows])
        assert np.array_equal(out[:len(exp)].double().cpu().numpy(), exp) and (out[len(exp):] == 7).all()


def test_append_more_sequences_than_a_grid_is_deep():
    B, Hkv, D, page = 65540, 1, 32, 8
    g = torch.Generator().manual_seed(41)
    k, v = (torch.randn(B, 1, Hkv, D, generator=g).to(BF16) for _ in "kv")
    codes, scales = _pools(B, Hkv, page, D)
    bt = torch.randperm(B, generator=g).view(B, 1).int().numpy()
    start, count = (torch.randint(0, m, (B,), generator=g).int().numpy() for m in (page, 2))
    start[-4:], count[-4:] = [0, 7, 3, 8], [1, 1, 0, 1]  # the last sequence is full
    got = _append(k, v, start, count, bt, codes, scales)
    exp = ref.kv4_append_ref(k, v, start, count, bt, codes.numpy(), scales.numpy())
    assert np.array_equal(got[0], exp[0]) and np.array_equal(got[1], exp[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_read_back_and_attended(dtype):
    """Rows appended, read back and given to tlm_flash_attn_varlen_fwd: within that kernel's roundings of the float64
    attention over the cache, and tlm_kv4_attn on the same rows within its own.

    tlm_flash_attn_varlen_fwd rounds each weight to dtype (eps / 2 of it) and sums the rounded or the unrounded ones (eps / 2
    of the quotient at most); its scores are fp32 sums of D exact products, off by (D + 4) 2^-24 of the sum of their
    magnitudes A, and a weight by that times 2; the sums of n terms are off by (n + 64) 2^-24 of the sum of magnitudes
    each. Its weights are relative to a maximum that a row has had, so the small ones of fp16 may fall among subnormal
    numbers: half a step of those is 2^-25, n times, of the largest |v|. The output is rounded once."""
    g = torch.Generator().manual_seed(42)
    H, Hkv, D, page, T = 8, 2, 128, 16, 8
    have = np.array([103, 40, 67, 8])
    B, per = len(have), 7
    codes, scales = (x.to(DEV) for x in _pools(B * per, Hkv, page, D, 43, 255, 256))
    bt = torch.randperm(B * per, generator=g).view(B, per).int().numpy()
    k, v = (torch.randn(B, int(have.max()), Hkv, D, generator=g).to(dtype) for _ in "kv")
    ops.kv4_append(k.to(DEV), v.to(DEV), _i32([0] * B), _i32(have), _i32(bt), codes, scales)
    cu = np.concatenate([[0], np.cumsum(have)]).astype(np.int32)
    ko, vo = (torch.empty(int(cu[-1]), Hkv, D, dtype=dtype, device=DEV) for _ in "kv")
    ops.kv4_read(codes, scales, _i32(bt), None, _i32(cu), ko, vo)
    q = torch.randn(B, T, H, D, generator=g).to(dtype)
    o = torch.empty(B * T, H, D, dtype=dtype, device=DEV)
    ops.flash_attn_varlen_fwd(q.flatten(0, 1).to(DEV), ko, vo, _i32([T * b for b in range(B + 1)]), _i32(cu), T, o, True,
                              D ** -0.5)
    c, s = codes.cpu(), scales.cpu()
    _check(q, c, s, bt, have)
    exp, _ = ref.kv4_attn_ref(q, c.numpy(), s.numpy(), bt, have, None, D ** -0.5)
    mag = c.clone()
    mag[:, 1] &= 0x77
    spread, _ = ref.kv4_attn_ref(q, mag.numpy(), s.numpy(), bt, have, None, D ** -0.5)
    eps = torch.finfo(dtype).eps
    n = int(have.max())
    for b in range(B):
        kk, vv = ref.kv4_rows_ref(c.numpy(), s.numpy(), bt, b, 0, int(have[b]))
        kk = np.abs(kk).repeat(H // Hkv, 1).transpose(1, 2, 0)
        a = (np.abs(q[b].double().numpy()).transpose(1, 0, 2) @ kk * D ** -0.5).max(-1).T[..., None]  # [T, H, 1]
        rel = eps + 2 * ((D + 4) * 2.0 ** -24 * a + 2.0 ** -23 + (n + 64) * 2.0 ** -24)
        small = n * 2.0 ** -25 * np.abs(vv).max() if dtype == F16 else 0.0
        lim = eps / 2 * (1 + 2 ** -7) * np.abs(exp[b]) + rel * spread[b] + small
        err = np.abs(o.view(B, T, H, D)[b].double().cpu().numpy() - exp[b])
        assert (err <= lim).all(), (b, (err / lim).max())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,T,H,Hkv", [(64, 1, 4, 1), (128, 9, 8, 2), (256, 1, 2, 2)])
@pytest.mark.parametrize("power", [10, 19, 21, 22, 23, 24, 25, 27, 30, 40, 90, 118])
def test_attn_scores_whose_steps_are_wide(power, D, T, H, Hkv, dtype):
    """Scores of +-1.375 D 2^(power - 7) whose neighbours in fp32 are up to 2^96 apart: one key is half or twice as far as the
    others, so its V is the output, exactly (a weight's rounding is far below half a step of the output), and its score
    the log2 of the sum. The key comes first, last, between and alone; its scores above 0 and below."""
    lens = [600, 300, 1, 40, 33, 600]
    at = [599 - (T - 1), 0, 0, 17, 31 - (T - 1), 350]
    q, c, s, bt = _attn_case(dtype, 6, T, H, Hkv, D, 16, [600 + T] * 6, 44)
    lens = [n + T - 1 for n in lens]  # every query sees the key
    c[:, 1] |= 0x11  # no zeros in V
    s[:, 1] = 127 + torch.randint(-3, 3, s[:, 1].shape, generator=torch.Generator().manual_seed(45)).to(torch.uint8)
    q = torch.full_like(q, 1.375)  # no power of two: the product with log2 e is rounded
    for sign in (1, -1):
        c[:, 0], s[:, 0] = (0x22 if sign > 0 else 0xAA), 120  # K: +-1 2^-7
        for b in range(6):
            s[int(bt[b, at[b] // 16]), 0, :, :, at[b] % 16] = 120 + sign
        out, z = _run(q, c, s, bt, lens, scale=2.0 ** power)
        top = sign * 1.375 * D * 2.0 ** (power - 7 + sign)
        for b in range(6):
            v = ref.kv4_rows_ref(c.numpy(), s.numpy(), bt, b, at[b], 1)[1][0].repeat(H // Hkv, 0)  # [H, D]
            x = out[b].double().numpy()
            assert np.array_equal(x, np.broadcast_to(v, x.shape)), (sign, b)
            assert (np.abs(z[b].double().numpy() / (top / np.log(2)) - 1) < 2.0 ** -21).all(), (sign, b)
