"""The 4-bit KV cache on the GPU against plain 64-bit implementations: stored
values and page bytes exactly, attention within a bound on the rounding errors
(tests/_compress_oracle.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import b2pa
from tests import _compress_oracle as co
from tests._helpers import random_tables

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = list(HALF_STEP)


def _np(t):
    return t.detach().double().cpu().numpy()


def _i32(x, dev):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)


def _table(tables, dev, width=None):
    width = width or max(1, max(len(t) for t in tables))
    a = np.full((len(tables), width), -1, np.int32)
    for b, t in enumerate(tables):
        a[b, : len(t)] = t
    return _i32(a, dev)


def _rows(rng, shape):
    """Rows whose groups span many magnitudes, some of them zero."""
    x = rng.standard_normal(shape)
    x *= np.exp2(rng.integers(-6, 5, shape[:-1] + (1,)))
    x[..., ::37] *= 8
    x[rng.random(shape[:-1]) < 0.05] = 0
    return x


def _pools(rng, NB, H, bs, D):
    """Packed K and V pools (numpy), with the values they stand for."""
    k, v = _rows(rng, (NB, H, bs, D)), _rows(rng, (NB, H, bs, D)) * 0.25
    return co.pack_pages(k, False), co.pack_pages(v, True), co.stored(k), co.stored(v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs,H", [(64, 8, 1), (64, 16, 8), (128, 16, 3), (128, 32, 5), (256, 16, 2), (256, 8, 1)])
def test_append_and_read(cuda_device, dtype, D, bs, H):
    rng = np.random.default_rng(D + bs)
    T, starts, lens = 23, [0, 5, bs - 1, 40, 7], [23, 1, 17, 0, 30]        # 30: clamped to T
    B = len(starts)
    ends = [s + min(n, T) for s, n in zip(starts, lens)]
    NB = sum(-(-e // bs) for e in ends) + 3
    tables = random_tables(rng, ends, NB, bs)
    k = torch.from_numpy(_rows(rng, (B, T, H, D))).to(dtype).to(cuda_device).transpose(1, 2)
    v = torch.from_numpy(_rows(rng, (B, T, H, D))).to(dtype).to(cuda_device).transpose(1, 2)
    before = rng.integers(0, 256, (2, NB, H, bs, D * 9 // 16)).astype(np.uint8)
    kp, vp = (torch.from_numpy(x).to(cuda_device) for x in before)
    want_k, want_v = before[0].copy(), before[1].copy()
    for pool, new, values in ((want_k, _np(k), False), (want_v, _np(v), True)):
        c, s = co.quantise(new)
        for b in range(B):
            for t in range(min(lens[b], T)):
                pos = starts[b] + t
                page = pool[tables[b][pos // bs]].reshape(H, -1)
                u = (c[b, :, t].astype(np.int16) + 8).astype(np.uint8)
                r = pos % bs
                page[:, r * D // 2: (r + 1) * D // 2] = u[:, 0::2] | (u[:, 1::2] << 4)
                sc = page[:, bs * D // 2:]
                if values:
                    sc.reshape(H, D // 16, bs)[:, :, r] = s[b, :, t]
                else:
                    sc.reshape(H, bs, D // 16)[:, r] = s[b, :, t]
    table = _table(tables, cuda_device)
    out = torch.full((B,), -7, dtype=torch.int64, device=cuda_device)
    b2pa.kv4_append(k, v, kp, vp, table, _i32(starts, cuda_device), _i32(lens, cuda_device), out)
    assert np.array_equal(kp.cpu().numpy(), want_k) and np.array_equal(vp.cpu().numpy(), want_v)
    assert out.tolist() == ends
    n = [min(x, T) for x in lens]
    rk, rv = b2pa.kv4_read(kp, vp, table, _i32(starts, cuda_device), _i32(n, cuda_device), T, dtype)
    live = (np.arange(T) < np.array(n)[:, None])[:, None, :, None]
    assert np.array_equal(_np(rk), np.where(live, co.stored(_np(k)), 0))
    assert np.array_equal(_np(rv), np.where(live, co.stored(_np(v)), 0))
    assert b2pa.read_status(cuda_device) == 0


def test_append_borders(cuda_device):
    """Every border of the two roundings, its fp32 neighbours, saturation, subnormal scales, NaN and infinity."""
    tops = []
    grid = co.GRID
    for i in range(1, len(grid)):
        t = np.float32((grid[i] + grid[i - 1]) / 2 * 7)
        tops += [np.nextafter(t, np.float32(0)), t, np.nextafter(t, np.float32(1e9))]
    rows = np.zeros((len(tops), 64), np.float32)
    for i, t in enumerate(tops):
        s = grid[co.scale_bytes(np.array([float(t)]))[0]]
        rows[i, 0] = t
        for m in range(7):
            x = np.float32((m + 0.5) * s)
            rows[i, 1 + 2 * m: 3 + 2 * m] = [np.nextafter(x, np.float32(0)), x]
            rows[i, 17 + 2 * m: 19 + 2 * m] = [-x, -np.nextafter(x, np.float32(1e9))]
        rows[i, 16] = -t
    extra = np.zeros((6, 64), np.float32)
    extra[0, :4] = [1e30, -1e5, 64512, 3]
    extra[1, 3], extra[1, 20] = np.nan, -np.inf
    extra[2, :3] = [1e-7, -2e-6, 1e-40]
    extra[3, 0] = np.float32(3.4e38)
    extra[4, :2] = [2.0 ** -16, -2.0 ** -17]
    rows = np.concatenate([rows, extra])
    n = len(rows)
    x = torch.from_numpy(rows).to(cuda_device).view(1, 1, n, 64)
    pages = -(-n // 16)
    kp = torch.zeros(pages, 1, 16, 36, dtype=torch.uint8, device=cuda_device)
    vp = torch.zeros_like(kp)
    table = _i32(np.arange(pages)[None], cuda_device)
    zero, cnt = _i32([0], cuda_device), _i32([n], cuda_device)
    b2pa.kv4_append(x, -x, kp, vp, table, zero, cnt)
    k, v = b2pa.kv4_read(kp, vp, table, zero, cnt, n, torch.float32)
    np.testing.assert_array_equal(_np(k)[0, 0], co.stored(rows))
    np.testing.assert_array_equal(_np(v)[0, 0], co.stored(-rows))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_borders_of_16_bits(cuda_device, dtype):
    """Every finite value as a group's largest; every border (k + 1/2) s of every scale s that the type holds with its
    neighbours, both signs; ranges of values against scales from subnormal to saturated."""
    tops = torch.arange(2 ** 15, dtype=torch.int16).view(dtype)
    tops = tops[torch.isfinite(tops)]
    rows = list(torch.cat([tops[:, None], -tops[:, None] / 2, tops.new_zeros(len(tops), 14)], 1))
    up, down = torch.tensor(float("inf")), torch.tensor(float("-inf"))
    for code in range(1, 226):
        s = float(co.GRID[code])
        x = torch.tensor([(k + 0.5) * s for k in range(7)]).to(dtype)
        x = torch.cat([x, torch.nextafter(x, up.to(dtype)), torch.nextafter(x, down.to(dtype))])[None]
        top = torch.full((1, 4), 7 * s, dtype=torch.float64).clamp(max=65504.0).to(dtype)
        flat = torch.cat([x, -x], 1).flatten()
        for i in range(0, 42, 14):
            rows.append(torch.cat([top[0, :2], flat[i: i + 14]]))
    for scale in (1e-7, 3e-6, 2e-5, 1.0, 1e4, 6e4):
        steps = torch.linspace(-1, 1, 15 * 200, dtype=torch.float64).view(200, 15) * scale
        rows += list(torch.cat([torch.full((200, 1), scale, dtype=torch.float64), steps], 1).to(dtype))
    x = torch.stack(rows)
    x = torch.cat([x, x.new_zeros(-len(x) % 4, 16)]).view(1, 1, -1, 64).to(cuda_device)
    n = x.shape[2]
    kp = torch.zeros(-(-n // 16), 1, 16, 36, dtype=torch.uint8, device=cuda_device)
    vp, table = torch.zeros_like(kp), _i32(np.arange(len(kp))[None], cuda_device)
    zero, cnt = _i32([0], cuda_device), _i32([n], cuda_device)
    b2pa.kv4_append(x, -x, kp, vp, table, zero, cnt)
    k, v = b2pa.kv4_read(kp, vp, table, zero, cnt, n, torch.float32)
    np.testing.assert_array_equal(_np(k), co.stored(_np(x)))
    np.testing.assert_array_equal(_np(v), co.stored(-_np(x)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_takes_any_strides(cuda_device, dtype):
    """Channel-strided, misaligned and broadcast sources."""
    gen = torch.Generator().manual_seed(2)
    base = torch.randn(2, 5, 130, 6, generator=gen).to(dtype).to(cuda_device)
    k = base[:, :, 1:129, :4].permute(0, 3, 1, 2)                 # [2, 4, 5, 128]: channel stride 6
    v = torch.randn(2, 5, 129, generator=gen).to(dtype).to(cuda_device)[:, None, :, 1:].expand(2, 4, 5, 128)
    kp = torch.zeros(2, 4, 8, 72, dtype=torch.uint8, device=cuda_device)
    vp = torch.zeros_like(kp)
    table = _i32([[1], [0]], cuda_device)
    s, n = _i32([3, 0], cuda_device), _i32([5, 4], cuda_device)
    b2pa.kv4_append(k, v, kp, vp, table, s, n)
    rk, rv = b2pa.kv4_read(kp, vp, table, s, n, 5, dtype)
    live = (np.arange(5) < np.array([5, 4])[:, None])[:, None, :, None]
    assert np.array_equal(_np(rk), np.where(live, co.stored(_np(k)), 0))
    assert np.array_equal(_np(rv), np.where(live, co.stored(_np(v)), 0))


def _attend_case(dev, *, lens, cur, H, D, bs, dtype, T, seed, q_scale=1.0, width=None, tables=None, q=None):
    rng = np.random.default_rng(seed)
    B = len(lens)
    NB = sum(-(-L // bs) for L in lens) + 5
    kp, vp, k, v = _pools(rng, NB, H, bs, D)
    tables = tables or random_tables(rng, lens, NB, bs)
    if q is None:
        q = torch.from_numpy(_rows(rng, (B, T, H, D)) * q_scale).to(dtype).to(dev).transpose(1, 2)
    fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4
    out = fn(q, torch.from_numpy(kp).to(dev), torch.from_numpy(vp).to(dev), _table(tables, dev, width),
             _i32(lens, dev), _i32(cur, dev))
    refs, bounds = [], []
    for b in range(B):
        K, V = co.rows_of(k, tables[b], lens[b]), co.rows_of(v, tables[b], lens[b])
        hidden = [j for j in range(lens[b]) if tables[b][j // bs] < 0]
        p, size = co.softmax_rows(_np(q)[b], K, cur[b], D ** -0.5, hidden)
        ref = np.einsum("htn,nhd->htd", p, V)
        refs.append(ref)
        bounds.append(co.output_bound(ref, HALF_STEP[dtype], D, size, lens[b], np.abs(V).max(initial=0.0)))
    return out, np.stack(refs), np.stack(bounds), dict(kp=kp, vp=vp, k=k, v=v, tables=tables, q=q)


def _check(out, ref, bound):
    err = np.abs(_np(out) - ref)
    assert (err <= bound).all(), f"worst error {err.max()} at {np.unravel_index(err.argmax(), err.shape)}, " \
                                 f"{(err / bound).max():.2f} of its bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs,H", [(64, 8, 3), (64, 16, 8), (64, 32, 1), (128, 8, 2), (128, 16, 5), (128, 32, 4),
                                    (256, 8, 1), (256, 16, 3), (256, 32, 2)])
def test_decode(cuda_device, dtype, D, bs, H):
    lens = [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 100, 300]
    out, ref, bound, _ = _attend_case(cuda_device, lens=lens, cur=[1] * len(lens), H=H, D=D, bs=bs, dtype=dtype, T=1,
                                      seed=D + bs + H)
    _check(out, ref, bound)
    assert b2pa.read_status(cuda_device) == 0


@pytest.mark.parametrize("T", [1, 3])
def test_nothing_visible(cuda_device, T):
    """Empty sequences and current lengths past the sequence leave zero rows; 0 and 2 shift what is seen."""
    lens, cur = [0, 1, 15, 16, 33, 5, 9, 0], [1, 1, 0, 2, 3, 20, 9, 0]
    out, ref, bound, _ = _attend_case(cuda_device, lens=lens, cur=cur, H=2, D=64, bs=16, dtype=torch.float32, T=T,
                                      seed=3)
    _check(out, ref, bound)
    assert not out[0].any() and not out[5].any() and not out[7].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L", [(1, 5000), (2, 2777), (40, 700)])
def test_decode_long(cuda_device, dtype, B, L):
    lens = [L - 13 * b for b in range(B)]
    out, ref, bound, _ = _attend_case(cuda_device, lens=lens, cur=[1] * B, H=4, D=128, bs=16, dtype=dtype, T=1, seed=L)
    _check(out, ref, bound)


@pytest.mark.parametrize("dtype,D,H,longest", [(torch.float32, 64, 8, 1040), (torch.bfloat16, 128, 8, 700),
                                               (torch.float16, 256, 6, 600), (torch.bfloat16, 64, 8, 500)])
def test_decode_of_many(cuda_device, dtype, D, H, longest):
    """More CTAs than the GPU holds at once, with and without the order by length; equal lengths and empty ones."""
    rng = np.random.default_rng(longest)
    lens = rng.integers(longest // 8, longest, 64).tolist()
    lens[5:9] = [longest] * 4
    lens[20:23], lens[63] = [0, 1, 0], longest
    out, ref, bound, _ = _attend_case(cuda_device, lens=lens, cur=[1] * 64, H=H, D=D, bs=16, dtype=dtype, T=1, seed=D)
    _check(out, ref, bound)
    assert b2pa.read_status(cuda_device) == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 60])
def test_fp32_precision(cuda_device, D, T):
    """Even rows (unit normal, outputs a thirtieth of a value): fp32 outputs are right as a whole to 2^-19.

    With |logit| under 8, two halves of q and fp32 sums leave a logit off by 2^-21 at most in the mean square, the
    weights by e^ that; n = 1,000 independent roundings of the sums of p v add 2^-24 * 1000^(1/2) * 4 at most
    relative to |out|.  Sums that carry an offset of the codes (5e-5 before they were kept apart) show."""
    rng = np.random.default_rng(D)
    H, bs, n = 2, 16, 1000
    NB = -(-n // bs)
    k, v = rng.standard_normal((NB, H, bs, D)), rng.standard_normal((NB, H, bs, D))
    q = torch.from_numpy(rng.standard_normal((1, H, T, D))).float().to(cuda_device)
    fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4
    out = fn(q, torch.from_numpy(co.pack_pages(k, False)).to(cuda_device),
             torch.from_numpy(co.pack_pages(v, True)).to(cuda_device), _i32(np.arange(NB)[None], cuda_device),
             _i32([n], cuda_device), _i32([T], cuda_device))
    p, _ = co.softmax_rows(_np(q)[0], co.rows_of(co.stored(k), range(NB), n), T, D ** -0.5)
    ref = np.einsum("htn,nhd->htd", p, co.rows_of(co.stored(v), range(NB), n))
    assert np.linalg.norm(_np(out)[0] - ref) <= 2.0 ** -19 * np.linalg.norm(ref)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [1, 60, 200])
@pytest.mark.parametrize("p", [-9, 6, 9, 12])
@pytest.mark.parametrize("lost", [False, True])
def test_fp32_precision_of_unlike_magnitudes(cuda_device, D, T, p, lost):
    """Queries times 2^-p on keys times 2^p: powers of two, which leave codes, logits and so the bound of
    test_fp32_precision as they are.  A query's low half that is a subnormal shows (7e-5 for p = 12).  With ``lost``
    the last row, which is padding, is not finite and stays alone."""
    rng = np.random.default_rng(D)
    H, bs, n = 2, 16, 1000
    NB = -(-n // bs)
    k, v = rng.standard_normal((NB, H, bs, D)) * 2.0 ** p, rng.standard_normal((NB, H, bs, D))
    q = torch.from_numpy(rng.standard_normal((1, H, T, D)) * 2.0 ** -p).float().to(cuda_device)
    live = T - 1 if lost and T > 1 else T
    q[:, :, live:, 3] = float("inf")
    fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4
    out = fn(q, torch.from_numpy(co.pack_pages(k, False)).to(cuda_device),
             torch.from_numpy(co.pack_pages(v, True)).to(cuda_device), _i32(np.arange(NB)[None], cuda_device),
             _i32([n], cuda_device), _i32([live], cuda_device))
    w, _ = co.softmax_rows(_np(q)[0, :, :live], co.rows_of(co.stored(k), range(NB), n), live, D ** -0.5)
    ref = np.einsum("htn,nhd->htd", w, co.rows_of(co.stored(v), range(NB), n))
    assert np.linalg.norm(_np(out)[0, :, :live] - ref) <= 2.0 ** -19 * np.linalg.norm(ref)
    assert torch.isnan(out[:, :, live:]).all()


@pytest.mark.parametrize("dtype,D,most", [(torch.float32, 64, 2.0 ** -17), (torch.float32, 128, 2.0 ** -17),
                                          (torch.float32, 256, 2.0 ** -17), (torch.bfloat16, 64, 2.0 ** -7),
                                          (torch.bfloat16, 128, 2.0 ** -7), (torch.bfloat16, 256, 2.0 ** -8),
                                          (torch.float16, 256, 2.0 ** -10)])
@pytest.mark.parametrize("T", [1, 60])
@pytest.mark.parametrize("at", [0, 700])
def test_one_key_draws_nearly_all(cuda_device, dtype, D, most, T, at):
    """One key with a logit 10 to 14 above the others' and a value of zero, so that the output is made of weights of
    about 2^-20 of the largest; the output as a whole.

    fp32: those weights are split with a rounding of 2^-38 of the largest, 2^-18.6 of themselves in the mean square; the
    far logit's own roundings (14 log2 e in fp32, and the scale's) are 2^-19.3 of every weight, the others' logits 2^-20,
    the exponential 2^-22, and the sums over 1,000 keys 2^-19 as in test_fp32_precision: 2^-17.1 together.  16-bit
    outputs round to half a step, and the prefill weights before that: to the operand type (head_dim 64 and 128), or to
    11 bits."""
    rng = np.random.default_rng(D)
    H, bs, n = 2, 16, 1000
    NB = -(-n // bs)
    k, v = rng.standard_normal((NB, H, bs, D)) / 4, rng.standard_normal((NB, H, bs, D))
    q = rng.standard_normal((1, H, T, D))
    k[..., :16] = 0                      # a group of its own, with the far key's 2^a in channel 0
    q[..., :16] = 0
    a = 4
    k[at // bs, :, at % bs] = 0
    k[at // bs, :, at % bs, 0] = 7 * 2.0 ** a   # code 7 of scale 2^a: exact
    q[..., 0] = 2.0 ** round(np.log2(12 * D ** 0.5 / (7 * 2.0 ** a)))
    far = 7 * 2.0 ** a * q[0, 0, 0, 0] * D ** -0.5
    assert 9 < far < 16
    v[at // bs, :, at % bs] = 0
    q = torch.from_numpy(q).to(dtype).to(cuda_device)
    fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4
    out = fn(q, torch.from_numpy(co.pack_pages(k, False)).to(cuda_device),
             torch.from_numpy(co.pack_pages(v, True)).to(cuda_device), _i32(np.arange(NB)[None], cuda_device),
             _i32([n], cuda_device), _i32([T], cuda_device))
    p, _ = co.softmax_rows(_np(q)[0], co.rows_of(co.stored(k), range(NB), n), T, D ** -0.5)
    ref = np.einsum("htn,nhd->htd", p, co.rows_of(co.stored(v), range(NB), n))
    assert np.linalg.norm(_np(out)[0] - ref) <= most * np.linalg.norm(ref)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.float32, 128), (torch.bfloat16, 256),
                                     (torch.float16, 128)])
def test_prefill_long(cuda_device, dtype, D):
    """Few queries on many keys (keys split between CTAs), and more queries than one CTA takes."""
    for T, lens in ((5, [6000, 4001]), (201, [201, 900])):
        cur = [T] * 2
        out, ref, bound, _ = _attend_case(cuda_device, lens=lens, cur=cur, H=2, D=D, bs=16, dtype=dtype, T=T, seed=T)
        _check(out, ref, bound + (0 if dtype == torch.float32 else HALF_STEP[dtype] * np.abs(ref).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs,H", [(64, 16, 3), (128, 8, 2), (256, 32, 1)])
def test_append_many_is_append_one_by_one(cuda_device, dtype, D, bs, H):
    """A long ragged prompt batch (an odd number of slots) leaves the pages that its tokens leave one at a time, and
    reads back alike."""
    rng = np.random.default_rng(D)
    B, T = 9, 151
    starts, lens = [0, 1, bs - 1, 7, 0, 3, 64, 0, 2], [151, 150, 1, 0, 77, 151, 8, 2, 149]
    ends = [a + n for a, n in zip(starts, lens)]
    NB = sum(-(-e // bs) for e in ends) + 2
    table = _table(random_tables(rng, ends, NB, bs), cuda_device)
    k, v = (torch.from_numpy(_rows(rng, (B, T, H, D))).to(dtype).to(cuda_device).transpose(1, 2) for _ in range(2))
    pools = [torch.full((NB, H, bs, D * 9 // 16), 5, dtype=torch.uint8, device=cuda_device) for _ in range(4)]
    b2pa.kv4_append(k, v, *pools[:2], table, _i32(starts, cuda_device), _i32(lens, cuda_device))
    for t in range(T):
        live = [int(t < n) for n in lens]
        b2pa.kv4_append(k[:, :, t:t + 1], v[:, :, t:t + 1], *pools[2:], table,
                        _i32([a + t for a in starts], cuda_device), _i32(live, cuda_device))
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    args = table, _i32(starts, cuda_device), _i32(lens, cuda_device), T, dtype
    live = (np.arange(T) < np.array(lens)[:, None])[:, None, :, None]
    for got, x in zip(b2pa.kv4_read(*pools[:2], *args), (k, v)):
        assert np.array_equal(_np(got), np.where(live, co.stored(_np(x)), 0))


@pytest.mark.parametrize("B", [2, 9])
def test_read_of_lengths_past_its_slots(cuda_device, B):
    """Lengths above T are T, for an odd number of slots whose table ends with the last one; one or two tokens a CTA."""
    rng = np.random.default_rng(B)
    T, D, bs, H, pages = 143, 64, 16, 2, 9  # positions 1 .. 143
    kp, vp, k, v = _pools(rng, B * pages, H, bs, D)
    table = np.arange(B * pages).reshape(B, pages)
    out = b2pa.kv4_read(torch.from_numpy(kp).to(cuda_device), torch.from_numpy(vp).to(cuda_device),
                        _i32(table, cuda_device), _i32([1] * B, cuda_device), _i32([T + 1, 500] + [T] * (B - 2), cuda_device),
                        T, torch.float32)
    for got, x in zip(out, (k, v)):
        want = [co.rows_of(x, ids, pages * bs)[1:].transpose(1, 0, 2) for ids in table]
        assert np.array_equal(_np(got), np.stack(want))
    assert b2pa.read_status(cuda_device) == 0


def test_decode_offsets_past_32_bits(cuda_device):
    """Pages at byte offsets past 2^32 of the pool."""
    H, D, bs = 8, 128, 32
    page = H * bs * 72
    NB = (1 << 32) // page + 40
    kp = torch.empty(NB, H, bs, 72, dtype=torch.uint8, device=cuda_device)
    vp = torch.empty_like(kp)
    rng = np.random.default_rng(5)
    lens = [70, 1000]
    tables = [[NB - 1 - i for i in range(3)], [NB - 4 - i for i in range(32)]]
    ids = tables[0] + tables[1]
    k, v = _rows(rng, (len(ids), H, bs, D)), _rows(rng, (len(ids), H, bs, D))
    kp[ids], vp[ids] = (torch.from_numpy(co.pack_pages(x, y)).to(cuda_device) for x, y in ((k, False), (v, True)))
    q = torch.from_numpy(_rows(rng, (2, H, 1, D))).to(torch.float16).to(cuda_device)
    out = b2pa.paged_attention_decode_kv4(q, kp, vp, _table(tables, cuda_device), _i32(lens, cuda_device),
                                          _i32([1, 1], cuda_device))
    at = 0
    for b, n in enumerate(lens):
        mine = list(range(at, at + len(tables[b])))
        at += len(mine)
        K, V = co.rows_of(co.stored(k), mine, n), co.rows_of(co.stored(v), mine, n)
        p, size = co.softmax_rows(_np(q)[b], K, 1, D ** -0.5)
        ref = np.einsum("htn,nhd->htd", p, V)
        _check(out[b], ref, co.output_bound(ref, 2.0 ** -11, D, size, n, np.abs(V).max()))


def test_far_logits(cuda_device):
    """Logits in the hundreds: the running maximum carries the sums."""
    out, ref, bound, _ = _attend_case(cuda_device, lens=[333, 40], cur=[1, 1], H=2, D=128, bs=16, dtype=torch.float32,
                                      T=1, seed=9, q_scale=30.0)
    _check(out, ref, bound)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.float32, 128), (torch.float32, 256),
                                     (torch.bfloat16, 128), (torch.bfloat16, 256), (torch.float16, 256)])
@pytest.mark.parametrize("T", [1, 50])
@pytest.mark.parametrize("far", [1e5, 3e5, 2e6, 3e7, 1e9])
def test_logits_in_the_millions(cuda_device, dtype, D, T, far):
    """Logits whose own rounding is of the size of usual logits: a query's largest wins by far more than that, and its
    key's value row comes out, to half a step."""
    rng = np.random.default_rng(D)
    H, bs, n = 2, 16, 500
    NB = -(-n // bs)
    k, v = rng.standard_normal((NB, H, bs, D)) * 4096, rng.standard_normal((NB, H, bs, D))
    q = rng.standard_normal((1, H, T, D)) * min(far, 3e7 if dtype == torch.float16 else far) / 4096
    q = torch.from_numpy(q).to(dtype).to(cuda_device)
    fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4
    out = _np(fn(q, torch.from_numpy(co.pack_pages(k, False)).to(cuda_device),
                 torch.from_numpy(co.pack_pages(v, True)).to(cuda_device), _i32(np.arange(NB)[None], cuda_device),
                 _i32([n], cuda_device), _i32([T], cuda_device)))[0]
    K, V = co.rows_of(co.stored(k), range(NB), n), co.rows_of(co.stored(v), range(NB), n)
    z = np.einsum("htd,nhd->htn", _np(q)[0], K) * D ** -0.5
    z = np.where(np.arange(n) < n - T + 1 + np.arange(T)[:, None], z, -np.inf)
    first, second = np.sort(z, -1)[..., -1], np.sort(z, -1)[..., -2]
    clear = first - second > 40 + 2.0 ** -16 * np.abs(_np(q)[0]).max() * np.abs(K).max() * D ** 0.5
    assert clear.mean() > 0.9
    ref = np.take_along_axis(V.transpose(1, 0, 2), z.argmax(-1)[..., None], 1)
    assert not np.isnan(out).any()
    # the 16-bit prefill of head_dim 64 and 128 rounds the winner's weight, which is not exactly 1 here, to the operand
    # type and its sum not: half a step more (one unit in 2^8 or 2^11 is twice that weight's largest rounding)
    steps = 2 if T > 1 and D < 256 and dtype != torch.float32 else 1
    assert (np.abs(out - ref) <= steps * HALF_STEP[dtype] * np.abs(ref) + 2.0 ** -22 * np.abs(V).max())[clear].all()


def test_scales_far_apart(cuda_device):
    """Value scales over their whole range within one sequence, small first and large first."""
    rng = np.random.default_rng(4)
    D, bs, n = 64, 16, 160
    for order in (1, -1):
        v = rng.standard_normal((10, 1, bs, D)) * np.exp2(np.linspace(-14, 13, 10))[::order, None, None, None]
        k = rng.standard_normal((10, 1, bs, D))
        kp, vp = co.pack_pages(k, False), co.pack_pages(v, True)
        q = torch.from_numpy(rng.standard_normal((1, 1, 1, D))).float().to(cuda_device)
        table = _i32(np.arange(10)[None], cuda_device)
        for m in (n, 16, 32, 1):
            out = b2pa.paged_attention_decode_kv4(q, torch.from_numpy(kp).to(cuda_device),
                                                  torch.from_numpy(vp).to(cuda_device), table,
                                                  _i32([m], cuda_device), _i32([1], cuda_device))
            K, V = co.rows_of(co.stored(k), range(10), m), co.rows_of(co.stored(v), range(10), m)
            p, size = co.softmax_rows(_np(q)[0], K, 1, D ** -0.5)
            ref = np.einsum("htn,nhd->htd", p, V)
            _check(out[0], ref, co.output_bound(ref, 2.0 ** -24, D, size, m, np.abs(V).max()))


def test_nan_reaches_only_its_own(cuda_device):
    """A NaN group of V makes its channels NaN; one of K the head's output; both only where the key is seen.  Stale
    NaN rows behind the sequence and of other heads are not read."""
    rng = np.random.default_rng(6)
    D, bs, H = 128, 16, 3
    k, v = rng.standard_normal((4, H, bs, D)), rng.standard_normal((4, H, bs, D))
    v[1, 0, 3, 40] = np.nan          # sequence 0, position 19, head 0, group 2
    k[2, 1, 0, 7] = np.inf           # sequence 1, position 0, head 1
    k[1, :, 9] = np.nan              # sequence 0, position 25: behind its length
    v[1, :, 9] = np.nan
    kp, vp = (torch.from_numpy(co.pack_pages(x, y)).to(cuda_device) for x, y in ((k, False), (v, True)))
    q = torch.from_numpy(rng.standard_normal((2, H, 1, D))).float().to(cuda_device)
    table = _i32([[0, 1], [2, 3]], cuda_device)
    for T in (1, 2):
        fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4
        out = fn(q.expand(2, H, T, D).contiguous(), kp, vp, table, _i32([25, 18], cuda_device),
                 _i32([T, T], cuda_device))
        bad = torch.isnan(out)
        assert bad[0, 0, :, 32:48].all() and not bad[0, 0, :, :32].any() and not bad[0, 0, :, 48:].any()
        assert not bad[0, 1:].any()
        assert bad[1, 1].all() and not bad[1, 0].any() and not bad[1, 2].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (128, 8), (256, 32)])
def test_nan_behind_the_mask(cuda_device, dtype, D, bs):
    """Within a chunk: NaN groups of V at the last position and of K at the one before reach only the queries that see
    them; a padded query that is NaN reaches nothing."""
    rng = np.random.default_rng(16)
    H, n, T = 2, 150, 70
    NB = -(-n // bs)
    clean_k, clean_v = rng.standard_normal((NB, H, bs, D)), rng.standard_normal((NB, H, bs, D))
    k, v = clean_k.copy(), clean_v.copy()
    at = lambda j: (j // bs, 0, j % bs)  # noqa: E731
    v[at(n - 1)][5] = np.nan
    k[at(n - 2)][20] = np.inf
    q = torch.from_numpy(rng.standard_normal((1, H, T + 3, D))).to(dtype).to(cuda_device)
    q[:, :, T:] = float("nan")
    table, lens, cur = _i32(np.arange(NB)[None], cuda_device), _i32([n], cuda_device), _i32([T], cuda_device)
    pools = [[torch.from_numpy(co.pack_pages(x, y)).to(cuda_device) for x, y in ((a, False), (b, True))]
             for a, b in ((clean_k, clean_v), (k, v))]
    p, size = co.softmax_rows(_np(q)[0, :, :T], co.rows_of(co.stored(clean_k), range(NB), n), T, D ** -0.5)
    V = co.rows_of(co.stored(clean_v), range(NB), n)
    ref = np.einsum("htn,nhd->htd", p, V)
    # (the unpacked pages' 16-bit kernels round the weights to the operand type, as in test_prefill)
    bound = co.output_bound(ref, HALF_STEP[dtype], D, size, n, np.abs(V).max()) \
        + (0 if dtype == torch.float32 else HALF_STEP[dtype] * np.abs(ref).max())
    for kp, vp, lost in ((0, 0, ()), (1, 1, ((T - 2, slice(None)), (T - 1, slice(None)))), (0, 1, ((T - 1, slice(0, 16)),)),
                         (1, 0, ((T - 2, slice(None)), (T - 1, slice(None))))):
        out = _np(b2pa.paged_attention_prefill_kv4(q, pools[kp][0], pools[vp][1], table, lens, cur))[0, :, :T]
        want = np.zeros(ref.shape, bool)
        for t, ch in lost:
            want[0, t, ch] = True
        assert np.array_equal(np.isnan(out), want), (kp, vp)
        assert (np.abs(out - ref) <= bound)[~want].all(), (kp, vp)
    w = torch.zeros(NB, H, bs, device=cuda_device)
    got = b2pa.accumulate_key_weights(q, pools[0][0], w, table, lens, cur, out=torch.zeros_like(w))
    assert got.sum().item() == pytest.approx(H * T, rel=1e-5)
    bad = b2pa.accumulate_key_weights(q, pools[1][0], w, table, lens, cur, out=torch.zeros_like(w))
    assert torch.equal(bad[:, 1], got[:, 1]) and torch.isnan(bad[:, 0].flatten()[:n]).all()


def test_far_queries(cuda_device):
    """fp32 queries past 2^15, and a row of them that is not finite, on keys small enough for usual logits."""
    rng = np.random.default_rng(26)
    for D in (64, 128):
        H, bs, n, T = 2, 16, 90, 33
        NB = -(-n // bs)
        k, v = rng.standard_normal((NB, H, bs, D)) * 2.0 ** -14, rng.standard_normal((NB, H, bs, D))
        q = rng.standard_normal((1, H, T, D)) * 2.0 ** 15
        qt = torch.from_numpy(q).float().to(cuda_device)
        qt[0, 1, 4, 7] = float("inf")
        out = b2pa.paged_attention_prefill_kv4(
            qt, *(torch.from_numpy(co.pack_pages(x, y)).to(cuda_device) for x, y in ((k, False), (v, True))),
            _i32(np.arange(NB)[None], cuda_device), _i32([n], cuda_device), _i32([T], cuda_device))
        p, size = co.softmax_rows(_np(torch.from_numpy(q).float())[0], co.rows_of(co.stored(k), range(NB), n), T, D ** -0.5)
        V = co.rows_of(co.stored(v), range(NB), n)
        ref = np.einsum("htn,nhd->htd", p, V)
        bound = co.output_bound(ref, 2.0 ** -24, D, size, n, np.abs(V).max())
        ok = np.ones((H, T), bool)
        ok[1, 4] = False
        assert (np.abs(_np(out)[0] - ref) <= bound)[ok].all() and np.isnan(_np(out)[0][~ok]).all()


def test_bad_pages(cuda_device):
    """Unset pages are not seen; ids past the pool are not read and are reported."""
    NB = 5 + 4
    for bad, code in ((-1, 0), (NB + 3, b2pa._lib.STATUS_CODES["B2PA_ERR_BAD_BLOCK_ID"])):
        b2pa.clear_status(cuda_device)
        lens = [64]
        rng = np.random.default_rng(1)
        kp, vp, k, v = _pools(rng, NB, 2, 16, 64)
        q = torch.from_numpy(_rows(rng, (1, 2, 1, 64))).float().to(cuda_device)
        args = (torch.from_numpy(kp).to(cuda_device), torch.from_numpy(vp).to(cuda_device),
                _table([[3, bad, 1, 0]], cuda_device), _i32(lens, cuda_device), _i32([1], cuda_device))
        K, V = co.rows_of(k, [3, 0, 1, 0], 64), co.rows_of(v, [3, 0, 1, 0], 64)
        p, size = co.softmax_rows(_np(q)[0], K, 1, 0.125, hidden=range(16, 32))
        ref = np.einsum("htn,nhd->htd", p, V)
        bound = co.output_bound(ref, 2.0 ** -24, 64, size, 64, np.abs(V).max())
        _check(b2pa.paged_attention_decode_kv4(q, *args)[0], ref, bound)
        assert b2pa.read_status(cuda_device) == code
        b2pa.clear_status(cuda_device)
        _check(b2pa.paged_attention_prefill_kv4(q, *args)[0], ref, bound)
        assert b2pa.read_status(cuda_device) == code
    b2pa.clear_status(cuda_device)
    # a length past the table: the table's rows are seen, and it is reported
    out = b2pa.paged_attention_decode_kv4(q, args[0], args[1], _table([[3, 2]], cuda_device), _i32([40], cuda_device),
                                          _i32([1], cuda_device))
    K, V = co.rows_of(k, [3, 2], 32), co.rows_of(v, [3, 2], 32)
    p, size = co.softmax_rows(_np(q)[0], K, 0, 0.125)
    ref = np.einsum("htn,nhd->htd", p, V)
    _check(out[0], ref, co.output_bound(ref, 2.0 ** -24, 64, size, 32, np.abs(V).max()))
    assert b2pa.read_status(cuda_device) == b2pa._lib.STATUS_CODES["B2PA_ERR_BAD_BLOCK_ID"]
    b2pa.clear_status(cuda_device)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs,H", [(64, 16, 4), (64, 8, 1), (128, 16, 2), (128, 32, 3), (256, 16, 1)])
def test_prefill(cuda_device, dtype, D, bs, H):
    """Chunks of 70 on prefixes, a padded row, a chunk without prefix."""
    cur = [70, 64, 1, 70]
    lens = [70, 64 + 33, 1 + 300, 70 + 129]
    out, ref, bound, _ = _attend_case(cuda_device, lens=lens, cur=cur, H=H, D=D, bs=bs, dtype=dtype, T=70, seed=D + bs)
    # the plain pools' 16-bit kernels round the softmax weights to the operand type: one half step more of max|v|
    _check(out, ref, bound + (0 if dtype == torch.float32 else HALF_STEP[dtype] * np.abs(ref).max()))
    assert b2pa.read_status(cuda_device) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_prefill_on_a_wide_table(cuda_device, dtype):
    """Tables for 65,000 tokens in pages of 8, with CTAs enough that none shares its keys."""
    out, ref, bound, _ = _attend_case(cuda_device, lens=[90], cur=[3], H=160, D=64, bs=8, dtype=dtype, T=3, seed=2,
                                      width=8120)
    _check(out, ref, bound + (0 if dtype == torch.float32 else HALF_STEP[dtype] * np.abs(ref).max()))


def test_streams_layouts_and_capture(cuda_device):
    """Strided q, a wide table, a non-current stream, and two graphs replayed after the inputs changed."""
    args = dict(lens=[50, 333], cur=[1, 1], H=4, D=128, bs=16, dtype=torch.bfloat16, T=1)
    out, ref, bound, st = _attend_case(cuda_device, seed=1, width=40, **args)
    _check(out, ref, bound)
    dev = cuda_device
    kp, vp = (torch.from_numpy(st[x]).to(dev) for x in ("kp", "vp"))
    table, lens, one = _table(st["tables"], dev), _i32(args["lens"], dev), _i32([1, 1], dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = b2pa.paged_attention_decode_kv4(st["q"], kp, vp, table, lens, one)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(other, out)
    q1, q2 = st["q"].clone(), st["q"].clone()
    graphs, outs = [], []
    for q in (q1, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(b2pa.paged_attention_decode_kv4(q, kp, vp, table, lens, one))
        graphs.append(g)
    q2.mul_(-1.5)
    wanted = [b2pa.paged_attention_decode_kv4(q, kp, vp, table, lens, one) for q in (q1, q2)]
    s1, s2 = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in ((s1, graphs[0]), (s2, graphs[1])):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wanted[0]) and torch.equal(outs[1], wanted[1])
    # a misaligned q is copied, not refused
    odd = torch.zeros(st["q"].numel() + 1, dtype=torch.bfloat16, device=dev)[1:].view(st["q"].shape)
    odd.copy_(st["q"])
    assert torch.equal(b2pa.paged_attention_decode_kv4(odd, kp, vp, table, lens, one), out)


def test_nothing_to_do(cuda_device):
    """Empty batches, chunks without tokens and pools without blocks: empty results, and the lengths all the same."""
    dev = cuda_device
    kp, vp = (torch.zeros(4, 2, 16, 36, dtype=torch.uint8, device=dev) for _ in range(2))
    t, five = _i32([[0, 1]], dev), _i32([5], dev)
    none, no_table = _i32(np.zeros(0), dev), torch.zeros(0, 2, dtype=torch.int32, device=dev)
    out = torch.full((1,), -7, dtype=torch.int64, device=dev)
    rows = torch.zeros(1, 2, 0, 64, device=dev)
    b2pa.kv4_append(rows, rows, kp, vp, t, five, five, out)
    assert out.tolist() == [5]
    assert b2pa.kv4_read(kp, vp, t, five, five, 0, torch.float32)[0].shape == (1, 2, 0, 64)
    assert b2pa.paged_attention_prefill_kv4(rows, kp, vp, t, five, five).shape == (1, 2, 0, 64)
    for T in (1, 3):
        rows = torch.zeros(0, 2, T, 64, device=dev)
        b2pa.kv4_append(rows, rows, kp, vp, no_table, none, none)
        fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4
        assert fn(rows, kp, vp, no_table, none, none).shape == (0, 2, T, 64)
        w = torch.ones(4, 2, 16, device=dev)
        assert b2pa.accumulate_key_weights(rows, kp, w, no_table, none, none).eq(1).all()
        # no pages at all
        for dtype in DTYPES:
            q = torch.ones(1, 2, T, 64, dtype=dtype, device=dev)
            assert not fn(q, kp, vp, t[:, :0], _i32([0], dev), _i32([T], dev)).any()
        assert b2pa.accumulate_key_weights(q, kp, w, t[:, :0], _i32([0], dev), _i32([T], dev)).eq(1).all()
    assert b2pa.evict_by_weight(kp, vp, w, no_table, none, 4).shape == (0, 2, 4)
    assert b2pa.evict_by_weight(kp, vp, w, t[:, :0], _i32([0], dev), 4).eq(-1).all()
    assert not kp.any() and not vp.any() and b2pa.read_status(dev) == 0


def test_refusals(cuda_device):
    dev = cuda_device
    kp = torch.zeros(4, 2, 16, 36, dtype=torch.uint8, device=dev)
    q = torch.zeros(1, 2, 1, 64, device=dev)
    t, one = _i32([[0, 1]], dev), _i32([1], dev)
    ok = (q, kp, kp.clone(), t, one, one)
    b2pa.paged_attention_decode_kv4(*ok)
    with pytest.raises(TypeError):
        b2pa.paged_attention_decode_kv4(q, q, q, t, one, one)
    with pytest.raises(TypeError):
        b2pa.paged_attention_decode_kv4(q.double(), *ok[1:])
    with pytest.raises(ValueError):
        b2pa.paged_attention_decode_kv4(torch.zeros(1, 3, 1, 64, device=dev), *ok[1:])
    with pytest.raises(ValueError):
        b2pa.paged_attention_decode_kv4(torch.zeros(1, 2, 1, 128, device=dev), *ok[1:])
    with pytest.raises(ValueError):
        b2pa.paged_attention_decode_kv4(torch.zeros(1, 2, 3, 64, device=dev), *ok[1:])
    with pytest.raises(ValueError):
        b2pa.paged_attention_decode_kv4(q, kp, kp, t, _i32([1, 1], dev), one)
    with pytest.raises(ValueError):
        b2pa.paged_attention_decode_kv4(q, kp, kp, _i32([[0], [1]], dev), one, one)
    with pytest.raises(TypeError):
        b2pa.kv4_read(kp.transpose(0, 1), kp, t, one, one, 4, torch.float32)
    with pytest.raises(TypeError):
        b2pa.kv4_read(kp, kp, t, one, one, 4, torch.float64)
    with pytest.raises(RuntimeError, match="block_size"):
        bad = torch.zeros(4, 2, 12, 36, dtype=torch.uint8, device=dev)
        b2pa.paged_attention_decode_kv4(q, bad, bad, t, one, one)
    assert b2pa.read_status(dev) == 0
