"""Key weights and eviction on the GPU against plain 64-bit implementations,
and the cache objects over a run of steps: prompt, decode steps, eviction,
more steps, on plain and 4-bit pools."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import b2pa
from oracle import model as om
from tests import _compress_oracle as co
from tests._helpers import random_tables
from tests.test_gpu_kv4 import DTYPES, _i32, _np, _rows, _table
from tests.test_gpu_kv4 import HALF_STEP

pytestmark = pytest.mark.gpu


def _weights_case(dev, *, lens, cur, T, H, D, bs, dtype, kv4, window, seed, in_place=False):
    rng = np.random.default_rng(seed)
    B = len(lens)
    NB = sum(-(-n // bs) for n in lens) + 3
    tables = random_tables(rng, lens, NB, bs)
    k = _rows(rng, (NB, H, bs, D))
    if kv4:
        pool, k = torch.from_numpy(co.pack_pages(k, False)).to(dev), co.stored(k)
    else:
        pool = torch.from_numpy(k).to(dtype).to(dev)
        k = _np(pool)
    q = torch.from_numpy(_rows(rng, (B, T, H, D))).to(dtype).to(dev).transpose(1, 2)
    w = torch.from_numpy(rng.random((NB, H, bs)) / 50).float().to(dev)
    out = w.clone() if in_place else torch.full_like(w, 7.0)
    want = _np(out)
    bound = np.zeros_like(want)
    for b in range(B):
        n, m = lens[b], min(cur[b], T)
        if n == 0:
            continue
        p, size = co.softmax_rows(_np(q)[b], co.rows_of(k, tables[b], n), cur[b], D ** -0.5)
        first = max(0, m - window) if window else 0
        add = p[:, first: max(m, first)].sum(1)
        for j in range(n):
            at = tables[b][j // bs], slice(None), j % bs
            want[at] = _np(w)[at] + add[:, j]
            # each weight's relative error, one rounding per addend, and the stored sum's own
            bound[at] = add[:, j] * (co.weight_error(D, size, n) + (T + 2) * 2.0 ** -23) + 2.0 ** -24 * want[at] \
                + 2.0 ** -30
    got = b2pa.accumulate_key_weights(q, pool, out if in_place else w, _table(tables, dev), _i32(lens, dev),
                                      _i32(cur, dev), window=window or None, out=None if in_place else out)
    assert got is out
    err = np.abs(_np(got) - want)
    assert (err <= bound).all(), f"worst {err.max()}, {np.max(err / np.maximum(bound, 1e-30)):.2f} of its bound"
    assert b2pa.read_status(dev) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("D,bs,H", [(64, 16, 3), (128, 8, 2), (128, 32, 1), (256, 16, 2)])
def test_key_weights(cuda_device, dtype, kv4, D, bs, H):
    _weights_case(cuda_device, lens=[1, 16, 17, 130, 333], cur=[1] * 5, T=1, H=H, D=D, bs=bs, dtype=dtype, kv4=kv4,
                  window=0, seed=1, in_place=True)
    _weights_case(cuda_device, lens=[66, 67 + 40, 3 + 200, 70], cur=[66, 67, 3, 70], T=70, H=H, D=D, bs=bs,
                  dtype=dtype, kv4=kv4, window=0, seed=2)
    _weights_case(cuda_device, lens=[66, 67 + 40, 3 + 200, 70], cur=[66, 67, 3, 70], T=70, H=H, D=D, bs=bs,
                  dtype=dtype, kv4=kv4, window=17, seed=3, in_place=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32])
def test_key_weights_small_heads(cuda_device, dtype, D):
    for T in (1, 21):
        _weights_case(cuda_device, lens=[T, T + 31, T + 100], cur=[T, T, max(1, T - 3)], T=T, H=3, D=D, bs=16,
                      dtype=dtype, kv4=False, window=0, seed=D)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("T", [1, 40])
def test_key_weights_precision(cuda_device, dtype, kv4, T):
    """Even rows (unit normal): the bound on a weight is a few 2^-12, so a product with one rounded half would show."""
    rng = np.random.default_rng(12)
    H, D, bs, n = 2, 64, 16, 200
    NB = -(-n // bs)
    k = rng.standard_normal((NB, H, bs, D))
    if kv4:
        pool, k = torch.from_numpy(co.pack_pages(k, False)).to(cuda_device), co.stored(k)
    else:
        pool = torch.from_numpy(k).to(dtype).to(cuda_device)
        k = _np(pool)
    q = torch.from_numpy(rng.standard_normal((1, H, T, D))).to(dtype).to(cuda_device)
    w = torch.zeros(NB, H, bs, device=cuda_device)
    dev = cuda_device
    b2pa.accumulate_key_weights(q, pool, w, _i32(np.arange(NB)[None], dev), _i32([n], dev), _i32([T], dev))
    p, size = co.softmax_rows(_np(q)[0], co.rows_of(k, range(NB), n), T, D ** -0.5)
    assert size < 20
    got = co.rows_of(_np(w)[..., None], range(NB), n)[..., 0].T
    want = p.sum(1)
    assert (np.abs(got - want) <= want * (co.weight_error(D, size, n) + (T + 2) * 2.0 ** -23) + 2.0 ** -30).all()
    # as a whole the roundings are independent: a tenth of their bound
    assert np.linalg.norm(got - want) <= 0.1 * co.weight_error(D, size, n) * np.linalg.norm(want)


@pytest.mark.parametrize("T", [1, 4])
def test_key_weights_nothing_counts(cuda_device, T):
    """Empty sequences, no counted query, and queries that see nothing."""
    _weights_case(cuda_device, lens=[0, 9, 5, 30, 40], cur=[0, 0, 20, 1, 2], T=T, H=2, D=64, bs=16,
                  dtype=torch.float32, kv4=False, window=0, seed=5)
    _weights_case(cuda_device, lens=[0, 9, 5, 30, 40], cur=[0, 0, 20, 1, 2], T=T, H=2, D=64, bs=16,
                  dtype=torch.bfloat16, kv4=True, window=1, seed=5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,n,T", [(1, 4000, 1), (1, 3333, 300), (24, 500, 1), (2, 1500, 130)])
def test_key_weights_long(cuda_device, dtype, B, n, T):
    lens = [n - 7 * b for b in range(B)]
    _weights_case(cuda_device, lens=lens, cur=[T] * B, T=T, H=4, D=64, bs=16, dtype=dtype, kv4=False, window=0, seed=n)
    _weights_case(cuda_device, lens=lens, cur=[T] * B, T=T, H=4, D=64, bs=16, dtype=dtype, kv4=True, window=0, seed=n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_key_weights_many_queries(cuda_device, dtype, kv4, D):
    """Several tiles of queries, with a window that begins inside one; one query past a tile, one past half of it."""
    for T, window in ((300, 0), (300, 150), (129, 0), (65, 0), (200, 64)):
        _weights_case(cuda_device, lens=[T, T + 211, 150], cur=[T, T - 5, 150 if T > 150 else 30], T=T, H=2, D=D, bs=16,
                      dtype=dtype, kv4=kv4, window=window, seed=T + window)


@pytest.mark.parametrize("longest", [200, 600])
@pytest.mark.parametrize("dtype,kv4,D", [(torch.float32, False, 64), (torch.bfloat16, True, 64),
                                         (torch.bfloat16, False, 128), (torch.float16, False, 256),
                                         (torch.float16, False, 32)])
def test_key_weights_of_many(cuda_device, dtype, kv4, D, longest):
    """More CTAs than the GPU holds at once, with and without the order by length; equal lengths and empty ones."""
    rng = np.random.default_rng(longest)
    lens = rng.integers(longest // 8, longest, 64).tolist()
    lens[5:9] = [longest] * 4
    lens[20:23], lens[63] = [0, 1, 0], longest
    _weights_case(cuda_device, lens=lens, cur=[1] * 64, T=1, H=10, D=D, bs=16, dtype=dtype, kv4=kv4, window=0, seed=7)


@pytest.mark.parametrize("kv4", [False, True])
@pytest.mark.parametrize("T", [1, 3])
def test_key_weights_wide_table(cuda_device, kv4, T):
    """A table far wider than its sequences (more keys than logits fit on chip) gives what a narrow one gives."""
    dev, H, D, bs = cuda_device, 2, 64, 16
    rng = np.random.default_rng(3)
    lens = [333, 40]
    tables = random_tables(rng, lens, 30, bs)
    k = rng.standard_normal((30, H, bs, D))
    pool = torch.from_numpy(co.pack_pages(k, False)).to(dev) if kv4 else torch.from_numpy(k).to(torch.float16).to(dev)
    q = torch.from_numpy(rng.standard_normal((2, H, T, D))).to(torch.float16).to(dev)
    w = torch.zeros(30, H, bs, device=dev)
    narrow, wide = (b2pa.accumulate_key_weights(q, pool, w, _table(tables, dev, width), _i32(lens, dev),
                                                _i32([T, T], dev), out=torch.zeros_like(w)) for width in (None, 20000))
    # the same products, summed in another order: n roundings of a sum of exponentials and one of its logarithm
    torch.testing.assert_close(wide, narrow, rtol=(333 + 16) * 2.0 ** -24, atol=0)
    assert narrow.sum().item() == pytest.approx(2 * H * T, rel=1e-4)


def test_two_graphs_and_a_side_stream(cuda_device):
    """Weights and eviction on another stream, and in two captured graphs that replay at the same time."""
    dev, H, D, bs, T = cuda_device, 2, 64, 16, 30
    rng = np.random.default_rng(21)
    lens, cur = [200, 90], [T, T]
    table, n, c = _i32([list(range(13)), list(range(13, 26))], dev), _i32(lens, dev), _i32(cur, dev)

    def inputs(seed):
        gen = torch.Generator().manual_seed(seed)
        return [torch.randn(*shape, generator=gen).to(dev) for shape in
                ((2, H, T, D), (26, H, bs, D), (26, H, bs, D))] + [torch.rand(26, H, bs, generator=gen).to(dev)]

    def work(q, k, v, w):
        b2pa.accumulate_key_weights(q, k, w, table, n, c)
        return b2pa.evict_by_weight(k, v, w, table, n, 50, 10)

    sets = [inputs(0), inputs(1)]
    want = []
    for x in sets:
        y = [t.clone() for t in x]
        want.append([work(*y)] + y)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        y = [t.clone() for t in sets[0]]
        got = [work(*y)] + y
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    live = [[t.clone() for t in x] for x in sets]
    graphs, outs = [], []
    for x in live:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(*x))
        graphs.append(g)
    streams = [torch.cuda.Stream(dev) for _ in graphs]
    for _ in range(5):
        for x, y in zip(live, sets):
            for a, b in zip(x, y):
                a.copy_(b)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, o, y in zip(live, outs, want):
            assert all(torch.equal(a, b) for a, b in zip([o] + x, y))


def _evict_case(dev, *, lens, keep, recent, H, D, bs, dtype, kv4, seed, fresh, weights=None):
    rng = np.random.default_rng(seed)
    B = len(lens)
    pages = [-(-n // bs) for n in lens]
    new_pages = [-(-min(n, keep) // bs) for n in lens]
    NB = sum(pages) + sum(new_pages) + 2
    perm = [int(x) for x in rng.permutation(NB)]
    tables = [[perm.pop() for _ in range(p)] for p in pages]
    outs = [[perm.pop() for _ in range(p)] for p in new_pages] if fresh else tables
    if kv4:
        k, v = (rng.integers(0, 256, (NB, H, bs, D * 9 // 16)).astype(np.uint8) for _ in range(2))
        kp, vp = (torch.from_numpy(x).to(dev) for x in (k, v))
    else:
        kp, vp = (torch.randn(NB, H, bs, D, generator=torch.Generator().manual_seed(seed + i)).to(dtype).to(dev)
                  for i in range(2))
        k, v = (x.cpu().clone().view(torch.uint8).numpy() for x in (kp, vp))
    w = rng.random((NB, H, bs)).astype(np.float32) if weights is None else weights(rng, (NB, H, bs))
    wt = torch.from_numpy(w.copy()).to(dev)
    width = -(-keep // bs)
    got = b2pa.evict_by_weight(kp, vp, wt, _table(tables, dev), _i32(lens, dev), keep, recent,
                               _table(outs, dev, width) if fresh else None).cpu().numpy()
    # row views of the pools: per page and head, slot-major segments
    def segments(pool, values):
        if not kv4:
            return [pool.reshape(NB, H, bs, -1)]
        flat = pool.reshape(NB, H, -1)
        s = flat[..., bs * D // 2:]
        s = s.reshape(NB, H, D // 16, bs).transpose(0, 1, 3, 2) if values else s.reshape(NB, H, bs, D // 16)
        return [flat[..., : bs * D // 2].reshape(NB, H, bs, D // 2), s]

    want = [k.copy(), v.copy(), w.copy()]
    src = segments(k, False) + segments(v, True) + [w[..., None]]
    dst = segments(want[0], False) + segments(want[1], True) + [want[2][..., None]]
    kept = np.full((B, H, keep), -1)
    for b, n in enumerate(lens):
        m = min(n, keep)
        for h in range(H):
            flat = w[np.array(tables[b], dtype=int), h].reshape(-1)[:n] if n else np.zeros(0)
            sel = co.evict(flat, keep, recent)
            kept[b, h, : len(sel)] = sel
            if not fresh and n <= keep:
                continue
            rows = [[s[tables[b][j // bs], h, j % bs].copy() for j in sel] for s in src]
            for r in range(-(-m // bs) * bs):
                for d, row in zip(dst, rows):
                    d[outs[b][r // bs], h, r % bs] = row[r] if r < m else 0
    assert np.array_equal(got, kept)
    for a, x in ((kp, want[0]), (vp, want[1])):
        assert np.array_equal(a.cpu().contiguous().view(torch.uint8).numpy().reshape(x.shape), x)
    assert np.array_equal(wt.cpu().numpy(), want[2], equal_nan=True)
    assert b2pa.read_status(dev) == 0


@pytest.mark.parametrize("fresh", [False, True], ids=["in_place", "out_table"])
@pytest.mark.parametrize("dtype,kv4,D,bs,H", [
    (torch.float32, False, 64, 16, 3), (torch.float32, False, 16, 8, 2), (torch.bfloat16, False, 128, 16, 2),
    (torch.float16, False, 16, 32, 1), (torch.float16, False, 256, 8, 1), (torch.bfloat16, False, 32, 16, 4),
    (None, True, 64, 16, 3), (None, True, 128, 8, 2), (None, True, 256, 32, 1)])
def test_evict(cuda_device, fresh, dtype, kv4, D, bs, H):
    for keep, recent in ((1, 0), (1, 1), (7, 3), (16, 16), (33, 100), (40, 0), (64, 13)):
        _evict_case(cuda_device, lens=[0, 1, 16, 33, 40, 41, 150, 300], keep=keep, recent=recent, H=H, D=D, bs=bs,
                    dtype=dtype, kv4=kv4, seed=keep, fresh=fresh)


@pytest.mark.parametrize("fresh", [False, True], ids=["in_place", "out_table"])
@pytest.mark.parametrize("dtype,kv4,D", [(torch.float32, False, 64), (torch.bfloat16, False, 128), (None, True, 64),
                                         (None, True, 256)])
def test_evict_many_heads(cuda_device, fresh, dtype, kv4, D):
    """Short sequences of many heads (one launch), to few tokens and to more than a chunk of rows."""
    for keep, recent in ((5, 5), (150, 20), (400, 0)):
        _evict_case(cuda_device, lens=[0, 3, 150, 151, 407, 512, 33, 260, 400, 401], keep=keep, recent=recent, H=16, D=D,
                    bs=16, dtype=dtype, kv4=kv4, seed=keep, fresh=fresh)
    _evict_case(cuda_device, lens=[300] * 10, keep=64, recent=0, H=16, D=D, bs=16, dtype=dtype, kv4=kv4, seed=1,
                fresh=fresh, weights=_ties)


def _ties(rng, shape):
    return np.floor(rng.random(shape) * 3).astype(np.float32)


def _special(rng, shape):
    w = rng.standard_normal(shape).astype(np.float32) * np.float32(1e-3)
    pick = rng.random(shape)
    for lo, x in ((0.0, np.nan), (0.05, np.inf), (0.1, -np.inf), (0.15, 0.0), (0.2, -0.0), (0.25, 1e-42), (0.3, 3e38)):
        w[(pick >= lo) & (pick < lo + 0.05)] = x
    return w


@pytest.mark.parametrize("weights", [_ties, _special, lambda rng, shape: np.zeros(shape, np.float32)],
                         ids=["ties", "special", "zeros"])
def test_evict_ties_and_special_weights(cuda_device, weights):
    for keep, recent in ((5, 2), (64, 0), (100, 10), (257, 7)):
        _evict_case(cuda_device, lens=[300, 64, 1100], keep=keep, recent=recent, H=2, D=64, bs=16,
                    dtype=torch.bfloat16, kv4=False, seed=keep, fresh=False, weights=weights)


@pytest.mark.parametrize("n,keep", [(9000, 1500), (60000, 30000), (60001, 17)])
def test_evict_long(cuda_device, n, keep):
    """Chunks that overlap their destinations, and sequences past what shared memory holds."""
    _evict_case(cuda_device, lens=[n, 100], keep=keep, recent=5, H=1, D=64, bs=32, dtype=torch.float16, kv4=False,
                seed=n, fresh=False)


def test_evict_bad_pages(cuda_device):
    dev = cuda_device
    kp = torch.randn(4, 1, 16, 64, device=dev)
    vp, w = torch.randn_like(kp), torch.rand(4, 1, 16, device=dev)
    before = kp.clone()
    bad = b2pa._lib.STATUS_CODES["B2PA_ERR_BAD_BLOCK_ID"]
    for table, n in (([[0, 9, 2]], 48), ([[0, -1, 2]], 48), ([[0, 1]], 40)):
        b2pa.clear_status(dev)
        b2pa.evict_by_weight(kp, vp, w, _i32(table, dev), _i32([n], dev), 20, 20)
        assert b2pa.read_status(dev) == bad
    assert torch.equal(kp[3], before[3])
    b2pa.clear_status(dev)


def test_evict_refusals(cuda_device):
    dev = cuda_device
    kp, w = torch.zeros(4, 2, 16, 64, device=dev), torch.zeros(4, 2, 16, device=dev)
    t, n = _i32([[0, 1]], dev), _i32([20], dev)
    for bad in (dict(keep=0), dict(keep=4, recent=-1), dict(keep=17, out_table=_i32([[3]], dev)),
                dict(keep=2 ** 32 + 4)):
        with pytest.raises(ValueError):
            b2pa.evict_by_weight(kp, kp.clone(), w, t, n, **bad)
    with pytest.raises(ValueError):
        b2pa.evict_by_weight(kp, kp.clone(), w.double(), t, n, 4)
    with pytest.raises(ValueError):
        b2pa.evict_by_weight(kp, kp[:, :1].contiguous(), w, t, n, 4)
    with pytest.raises(TypeError):
        b2pa.accumulate_key_weights(torch.zeros(1, 2, 1, 64, device=dev, dtype=torch.bfloat16), kp, w, t, n, n)
    with pytest.raises(ValueError):
        b2pa.accumulate_key_weights(torch.zeros(1, 2, 1, 64, device=dev), kp, w, t, n, n, window=0)


@pytest.mark.parametrize("kv4", [False, True], ids=["plain", "kv4"])
def test_offsets_past_32_bits(cuda_device, kv4):
    """Every call on pages at the far end of pools of more than 2^32 bytes (plain: 2^31 elements) gives what it gives
    on small pools."""
    dev, H, D, bs = cuda_device, 8, 128, 32
    cols, dtype = (72, torch.uint8) if kv4 else (D, torch.float16)
    block = H * bs * cols * (1 if kv4 else 2)
    NB, n = (1 << 32) // block + 40, 20
    gen = torch.Generator().manual_seed(1)
    small = [torch.randint(0, 200, (n, H, bs, cols), generator=gen, dtype=torch.uint8).to(dev) if kv4 else
             torch.randn(n, H, bs, cols, generator=gen).to(dtype).to(dev) for _ in range(2)]
    w_small = torch.rand(n, H, bs, generator=gen).to(dev)
    big = [torch.empty(NB, H, bs, cols, dtype=dtype, device=dev) for _ in range(2)]
    w_big = torch.empty(NB, H, bs, device=dev)
    for a, b in zip(big + [w_big], small + [w_small]):
        a[NB - n:] = b
    ids = torch.randperm(n, generator=gen).to(torch.int32).to(dev).view(2, n // 2)
    lens, T = _i32([300, 211], dev), 40
    q = torch.randn(2, H, T, D, generator=gen).to(torch.float16).to(dev)
    rows = torch.randn(2, H, T, D, generator=gen).to(torch.float16).to(dev)
    got = []
    for (kp, vp), w, table in ((small, w_small, ids), (big, w_big, ids + (NB - n))):
        res = []
        if kv4:
            b2pa.kv4_append(rows, -rows, kp, vp, table, lens - T, _i32([T, 7], dev))
            res += b2pa.kv4_read(kp, vp, table, lens - T, _i32([T, T], dev), T, torch.float32)
            res.append(b2pa.paged_attention_prefill_kv4(q, kp, vp, table, lens, _i32([T, T], dev)))
            res.append(b2pa.paged_attention_decode_kv4(q[:, :, :1], kp, vp, table, lens, _i32([1, 1], dev)))
        for x in (q, q[:, :, :1]):
            b2pa.accumulate_key_weights(x, kp, w, table, lens, _i32([x.shape[2]] * 2, dev))
        res.append(b2pa.evict_by_weight(kp, vp, w, table, lens, 100, 10))
        got.append(res + [t[-n:] for t in (kp, vp, w)])
    for a, b in zip(*got):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert b2pa.read_status(dev) == 0


@pytest.mark.parametrize("T", [1, 9])
def test_arguments_that_need_conversion(cuda_device, T):
    """64-bit lengths, strided lengths, tables that are slices, columns or 64-bit, misaligned and channel-strided
    queries: the same results as plain arguments, from every call."""
    dev, H, D, bs, B = cuda_device, 2, 64, 16, 3
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randint(0, 200, (12, H, bs, 36), generator=gen, dtype=torch.uint8).to(dev) for _ in range(2))
    w = torch.rand(12, H, bs, generator=gen).to(dev)
    q = torch.randn(B, H, T, D, generator=gen).to(dev)
    table = _i32(np.arange(12).reshape(3, 4), dev)
    lens, cur, start = _i32([60, 33, 9], dev), _i32([T] * 3, dev), _i32([3, 0, 40], dev)
    wide = torch.zeros(B, 9, dtype=torch.int32, device=dev)
    wide[:, 2:6] = table
    odd = torch.zeros(q.numel() + 1, device=dev)[1:].view(q.shape).copy_(q)
    every = torch.zeros(*q.shape[:3], 2 * D, device=dev)[..., ::2].copy_(q)
    strided = torch.stack([lens, lens], 1)[:, 0]
    fn = b2pa.paged_attention_decode_kv4 if T == 1 else b2pa.paged_attention_prefill_kv4

    def run(q, table, lens, cur, start):
        pools = [t.clone() for t in (k, v, w)]
        out = [fn(q, *pools[:2], table, lens, cur)]
        b2pa.accumulate_key_weights(q, pools[0], pools[2], table, lens, cur)
        b2pa.accumulate_key_weights(q, pools[0], pools[2], table, lens, cur, window=2)
        out += b2pa.kv4_read(*pools[:2], table, start, cur, T, torch.float32)
        b2pa.kv4_append(q, q, *pools[:2], table, start, cur)
        out.append(b2pa.evict_by_weight(*pools, table, lens, 20, 3))
        return out + pools

    want = run(q, table, lens, cur, start)
    for args in ((q, table.long(), lens.long(), cur.long(), start.long()), (q, wide[:, 2:6], strided, cur, start),
                 (q, torch.stack([table, table], 2)[..., 0], lens, cur, start), (odd, table, lens, cur, start),
                 (every, table, lens, cur, start)):
        assert all(torch.equal(a, b) for a, b in zip(run(*args), want))
    assert b2pa.read_status(dev) == 0


def test_counts_past_32_bits(cuda_device):
    """``recent`` and ``window`` of any size mean all of them; a batch cut to any number keeps what it has."""
    dev = cuda_device
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(3, 2, 16, 64, generator=gen).to(dev) for _ in range(2))
    w, q = torch.rand(3, 2, 16, generator=gen).to(dev), torch.randn(1, 2, 5, 64, generator=gen).to(dev)
    t, n, five = _i32([[2, 0, 1]], dev), _i32([40], dev), _i32([5], dev)
    assert b2pa.evict_by_weight(k, v, w, t, n, 7, 2 ** 32 + 1).tolist() == [[list(range(33, 40))] * 2]
    n = _i32([7], dev)
    for window in (5, 2 ** 31, 2 ** 32 + 1):
        assert torch.equal(b2pa.accumulate_key_weights(q, k, w, t, n, five, window=window, out=torch.zeros_like(w)),
                           b2pa.accumulate_key_weights(q, k, w, t, n, five, out=torch.zeros_like(w)))
    pool = b2pa.LayerBlockPool(16, 3, 1.5)
    pool.track_key_weights(2 ** 32 + 1)
    state = b2pa.PagedKVCacheState(pool)
    cache = b2pa.BatchedPagedKVCache([state], pool)
    cache.append_batch(q, q, [5])
    b2pa.paged_attention("b200_paged", q, cache, [5])
    assert pool.key_weights.sum().item() == pytest.approx(10, rel=1e-5)
    assert cache.evict(2 ** 40).tolist() == [[list(range(5))] * 2] and state.seq_len == 5


@pytest.mark.parametrize("kv4", [False, True], ids=["plain", "kv4"])
@pytest.mark.parametrize("fused", [False, True])
def test_run_of_steps(cuda_device, kv4, fused):
    """Ragged prompts, decode steps, an eviction, more steps (the block tables regrow), against dense 64-bit
    bookkeeping: outputs, key weights, kept positions, lengths and freed blocks."""
    dev, H, D, bs = cuda_device, 3, 64, 16
    rng = np.random.default_rng(8)
    pool = (b2pa.Kv4BlockPool if kv4 else b2pa.LayerBlockPool)(bs, 3, 1.5)
    pool.track_key_weights()
    states = [b2pa.PagedKVCacheState(pool) for _ in range(3)]
    K = [np.zeros((0, H, D)) for _ in range(3)]
    V = [np.zeros((0, H, D)) for _ in range(3)]
    W = [np.zeros((H, 0)) for _ in range(3)]
    err = [0.0] * 3

    def step(which, lengths, T):
        cache = b2pa.BatchedPagedKVCache([states[i] for i in which], pool)
        x = [torch.from_numpy(rng.standard_normal((len(which), T, H, D))).float().to(dev).transpose(1, 2)
             for _ in range(3)]
        got_lens = cache.append_batch(x[1], x[2], lengths)
        out = b2pa.paged_attention("b200_paged", x[0], cache, lengths)
        for i, b in enumerate(which):
            m = lengths[i]
            new = [_np(t)[i, :, :m].transpose(1, 0, 2) for t in x[1:]]
            if kv4:
                new = [co.stored(t) for t in new]
            K[b], V[b] = np.concatenate([K[b], new[0]]), np.concatenate([V[b], new[1]])
            n = len(K[b])
            assert int(got_lens[i]) == n == states[b].seq_len
            p, size = co.softmax_rows(_np(x[0])[i], K[b], m, D ** -0.5)
            ref = np.einsum("htn,nhd->htd", p, V[b])
            bound = co.output_bound(ref, 2.0 ** -24, D, size, n, np.abs(V[b]).max())
            assert (np.abs(_np(out)[i, :, :m] - ref[:, :m]) <= bound[:, :m]).all()
            W[b] = np.concatenate([W[b], np.zeros((H, n - W[b].shape[1]))], 1) + p[:, :m].sum(1)
            err[b] += m * co.weight_error(D, size, n) + 2.0 ** -20
            kw = _np(pool.key_weights)
            mine = co.rows_of(kw[..., None], states[b].block_ids, n)[..., 0].T
            assert (np.abs(mine - W[b]) <= err[b] * np.maximum(W[b], 2.0 ** -10)).all()

    prev = b2pa.set_fused_append(fused)
    try:
        step([0, 1, 2], [40, 17, 33], 40)
        for _ in range(5):
            step([0, 1, 2], [1, 1, 1], 1)
        cache = b2pa.BatchedPagedKVCache([states[0], states[2]], pool)
        free, held = len(pool.free_block_ids), [len(s.block_ids) for s in states]
        mine = {b: co.rows_of(_np(pool.key_weights)[..., None], states[b].block_ids, len(K[b]))[..., 0].T
                for b in (0, 2)}
        kept = cache.evict(20, recent=6).cpu().numpy()
        for i, b in enumerate((0, 2)):
            sel = np.stack([co.evict(mine[b][h], 20, 6) for h in range(H)])
            assert np.array_equal(kept[i], sel)
            K[b], V[b] = (np.stack([x[sel[h], h] for h in range(H)], 1) for x in (K[b], V[b]))
            W[b] = np.stack([W[b][h, sel[h]] for h in range(H)])
            assert states[b].seq_len == 20 and len(states[b].block_ids) == 2
        assert len(pool.free_block_ids) - free == held[0] + held[2] - 4
        for t in (pool.k_blocks, pool.v_blocks, pool.key_weights):  # freed pages are zero again
            assert not t[pool.free_block_ids].any()
        for _ in range(14):
            step([2, 0], [1, 1], 1)
        step([0, 1, 2], [3, 20, 20], 20)
        assert torch.equal(cache.evict(10 ** 6)[:, 0, 0].cpu(), torch.zeros(2, dtype=torch.int32))  # nothing leaves
    finally:
        b2pa.set_fused_append(prev)
    with pytest.raises(ValueError, match="twice"):
        b2pa.BatchedPagedKVCache([states[0], states[0]], pool).evict(4)
    assert b2pa.read_status(dev) == 0


@pytest.mark.parametrize("kv4", [False, True], ids=["plain", "kv4"])
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("T", [1, 6])
def test_device_lengths_of_any_layout(cuda_device, kv4, fused, T):
    """Current lengths on the device as a column, as one expanded value and in 64 bits: outputs and key weights are
    those of the plain tensor."""
    dev, H, D, B = cuda_device, 2, 64, 3
    rng = np.random.default_rng(T)
    prompt, q, k, v = (torch.from_numpy(rng.standard_normal((B, H, n, D))).float().to(dev) for n in (9, T, T, T))
    base = torch.full((B,), max(1, T - 2), dtype=torch.int32, device=dev)
    column = torch.stack([base, torch.full_like(base, 77)], 1)[:, 0]
    expanded = base[:1].expand(B)
    got = []
    prev = b2pa.set_fused_append(fused)
    try:
        for lengths in (base, column, expanded, base.long(), column.long()):
            pool = (b2pa.Kv4BlockPool if kv4 else b2pa.LayerBlockPool)(16, 8, 2.0)
            pool.track_key_weights()
            cache = b2pa.BatchedPagedKVCache([b2pa.PagedKVCacheState(pool) for _ in range(B)], pool)
            cache.append_batch(prompt, prompt, [9, 5, 7])
            b2pa.paged_attention("b200_paged", prompt, cache, [9, 5, 7])
            cache.append_batch(k, v, lengths)
            got.append((b2pa.paged_attention("b200_paged", q, cache, lengths), pool.key_weights))
    finally:
        b2pa.set_fused_append(prev)
    for out, weights in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(weights, got[0][1])
    with pytest.raises(ValueError, match="lengths"):
        b2pa.paged_attention("b200_paged", q, cache, base[:2])
    with pytest.raises(ValueError):
        b2pa.paged_attention("b200_paged", q, cache, base[:1].expand(B, B))
    assert b2pa.read_status(dev) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,bs", [(64, 8), (128, 16), (256, 32)])
def test_run_on_4_bit_pools_of_every_type(cuda_device, dtype, D, bs):
    """The cache objects on 4-bit pools for rows of every type and width: a ragged prompt, decode steps with and
    without a DecodeStep, an eviction, a second chunk; outputs and key weights against 64-bit bookkeeping."""
    dev, H, B = cuda_device, 2, 3
    rng = np.random.default_rng(D)
    pool = b2pa.Kv4BlockPool(bs, 4, 1.5)
    pool.track_key_weights()
    states = [b2pa.PagedKVCacheState(pool) for _ in range(B)]
    K = [np.zeros((0, H, D)) for _ in range(B)]
    V = [np.zeros((0, H, D)) for _ in range(B)]
    W = [np.zeros((H, 0)) for _ in range(B)]
    err = [0.0] * B

    def step(lengths, T):
        cache = b2pa.BatchedPagedKVCache(states, pool)
        q, k, v = (torch.from_numpy(rng.standard_normal((B, T, H, D))).to(dtype).to(dev).transpose(1, 2)
                   for _ in range(3))
        cache.append_batch(k, v, lengths)
        out = b2pa.paged_attention("b200_paged", q, cache, lengths)
        assert out.dtype == dtype and pool.k_blocks.dtype == torch.uint8
        for b, m in enumerate(lengths):
            new = [co.stored(_np(t)[b, :, :m].transpose(1, 0, 2)) for t in (k, v)]
            K[b], V[b] = np.concatenate([K[b], new[0]]), np.concatenate([V[b], new[1]])
            n = len(K[b])
            assert n == states[b].seq_len
            p, size = co.softmax_rows(_np(q)[b], K[b], m, D ** -0.5)
            ref = np.einsum("htn,nhd->htd", p, V[b])
            bound = co.output_bound(ref, HALF_STEP[dtype], D, size, n, np.abs(V[b]).max())
            if T > 1 and dtype != torch.float32:  # weights rounded to the operand type, as in test_prefill
                bound = bound + HALF_STEP[dtype] * np.abs(ref).max()
            assert (np.abs(_np(out)[b, :, :m] - ref[:, :m]) <= bound[:, :m]).all()
            W[b] = np.concatenate([W[b], np.zeros((H, n - W[b].shape[1]))], 1) + p[:, :m].sum(1)
            err[b] += m * co.weight_error(D, size, n) + 2.0 ** -20
            mine = co.rows_of(_np(pool.key_weights)[..., None], states[b].block_ids, n)[..., 0].T
            assert (np.abs(mine - W[b]) <= err[b] * np.maximum(W[b], 2.0 ** -10)).all()

    step([37, 5, 22], 37)
    plan = None
    for i in range(4):
        if i % 2 == 0:
            step([1] * B, 1)
        else:
            grown = [s.seq_len for s in states]
            plan = b2pa.DecodeStep([states], plan)
            with plan:
                q, k, v = (torch.from_numpy(rng.standard_normal((B, H, 1, D))).to(dtype).to(dev) for _ in range(3))
                cache = b2pa.BatchedPagedKVCache(states, pool)
                cache.append_batch(k, v, 1)
                out = b2pa.paged_attention("b200_paged", q, cache, 1)
            plan = plan.meta
            for b in range(B):
                K[b], V[b] = (np.concatenate([x[b], co.stored(_np(t)[b].transpose(1, 0, 2))]) for x, t in ((K, k), (V, v)))
                assert len(K[b]) == grown[b] + 1 == states[b].seq_len
                p, size = co.softmax_rows(_np(q)[b], K[b], 1, D ** -0.5)
                ref = np.einsum("htn,nhd->htd", p, V[b])
                assert (np.abs(_np(out)[b] - ref) <= co.output_bound(ref, HALF_STEP[dtype], D, size, len(K[b]),
                                                                     np.abs(V[b]).max())).all()
                W[b] = np.concatenate([W[b], np.zeros((H, 1))], 1) + p.sum(1)
                err[b] += co.weight_error(D, size, len(K[b])) + 2.0 ** -20
    kept = b2pa.BatchedPagedKVCache(states, pool).evict(16, recent=5).cpu().numpy()
    for b in range(B):
        n = min(16, len(K[b]))
        sel = kept[b][:, :n]
        assert (np.diff(sel) > 0).all() and states[b].seq_len == n
        # the best by the sums, within their error
        for h in range(H):
            gone = np.setdiff1d(np.arange(len(K[b])), sel[h])
            old = sel[h][sel[h] < len(K[b]) - 5]
            if len(gone) and len(old):
                assert W[b][h, gone].max() <= W[b][h, old].min() * (1 + 4 * err[b]) + 2.0 ** -10 * err[b]
        K[b], V[b] = (np.stack([x[sel[h], h] for h in range(H)], 1) for x in (K[b], V[b]))
        W[b] = np.stack([W[b][h, sel[h]] for h in range(H)])
    step([3, 9, 1], 9)
    step([1] * B, 1)
    assert b2pa.read_status(dev) == 0


@pytest.mark.parametrize("kv4", [False, True], ids=["plain", "kv4"])
def test_device_lengths_of_any_shape(cuda_device, kv4):
    """One request's length as a scalar, and a column of lengths as [B, 1]."""
    dev, H, D, B = cuda_device, 2, 64, 2
    x = torch.randn(B, H, 7, D, generator=torch.Generator().manual_seed(1)).to(dev)
    pool = (b2pa.Kv4BlockPool if kv4 else b2pa.LayerBlockPool)(16, 8, 2.0)
    states = [b2pa.PagedKVCacheState(pool) for _ in range(B)]
    both = b2pa.BatchedPagedKVCache(states, pool)
    both.append_batch(x, x, [7, 4])
    want = b2pa.paged_attention("b200_paged", x, both, [7, 4])
    lens = torch.tensor([[7], [4]], device=dev)
    assert torch.equal(b2pa.paged_attention("b200_paged", x, both, lens), want)
    one = b2pa.BatchedPagedKVCache(states[:1], pool)
    assert torch.equal(b2pa.paged_attention("b200_paged", x[:1], one, lens[0, 0]), want[:1])


def _model(dev, kv4):
    made = []

    def tracking_pool(*args):  # "mixed": the first layer's pages 4-bit, the second's plain
        made.append((b2pa.Kv4BlockPool if kv4 is True or (kv4 == "mixed" and not made) else b2pa.LayerBlockPool)(*args))
        made[-1].track_key_weights()
        return made[-1]

    back = om.b2pa_backend()
    back.pool_cls = tracking_pool
    om.set_seed(11)
    return om.TinyLM(300, 128, 2, 3, 256, 512, back, kv_block_size=16, kv_pool_initial_blocks=64,
                     kv_pool_growth_factor=2.0).to(dev).eval()


@torch.no_grad()
@pytest.mark.parametrize("kv4", [False, True, "mixed"], ids=["plain", "kv4", "mixed"])
def test_decoder_graph_with_eviction(cuda_device, kv4):
    """FusedDecoder under DecodeGraph with tracking pools gives, bit for bit, the logits, pools and key weights of the
    same steps run eagerly in a DecodeStep, through an eviction of every layer between replays."""
    dev = cuda_device
    lengths = [40, 25, 33]
    runs = []
    for mode in ("eager", "graph"):
        model = _model(dev, kv4)
        prompt = torch.randint(0, 300, (3, 40), generator=torch.Generator().manual_seed(3)).to(dev)
        cur = torch.tensor(lengths, device=dev)
        logits, caches = model(prompt, position_offset=0, current_lengths=cur)
        layer_states = [list(c.states) for c in caches]
        assert all(st[0].pool.key_weights.any() for st in layer_states)
        nxt = torch.argmax(logits[torch.arange(3, device=dev), cur - 1, :], dim=-1)
        batches = [b2pa.BatchedPagedKVCache(list(st), st[0].pool) for st in layer_states]
        dec = b2pa.FusedDecoder(model, max_batch=4)
        ids, pos = nxt.clone(), cur.clone()
        graph = b2pa.DecodeGraph(lambda: dec.step(ids, pos, batches)) if mode == "graph" else None
        meta, seen = None, []
        for s in range(24):
            if s == 12:
                for c in batches:
                    c.evict(24, recent=8)
            if graph:
                lg, _ = graph(layer_states)
            else:
                step = b2pa.DecodeStep(layer_states, meta)
                with step:
                    lg, _ = dec.step(ids, pos, batches)
                meta = step.meta
            seen.append(lg.clone())
            ids.copy_(torch.randint(0, 300, (3,), generator=torch.Generator().manual_seed(s)).to(dev))
            pos.add_(1)
        assert all(s.seq_len == 36 for st in layer_states for s in st)
        runs.append((seen, [(st[0].pool.k_blocks, st[0].pool.v_blocks, st[0].pool.key_weights) for st in layer_states],
                     [[s.block_ids for s in st] for st in layer_states]))
        if graph:
            assert graph.replays >= 20
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.equal(a, b)
    assert runs[0][2] == runs[1][2]
    for x, y in zip(runs[0][1], runs[1][1]):
        assert all(torch.equal(a, b) for a, b in zip(x, y))
    assert b2pa.read_status(dev) == 0


@torch.no_grad()
def test_executor_bounds_every_cache(cuda_device):
    """FusedDecodeExecutor with evict_keep: requests run to their end on bounded caches."""
    from oracle import serving as osv

    dev = cuda_device
    model = _model(dev, True)
    ex = osv.ModelExecutors(model, dev)
    reqs = osv.generate_requests(4, 1000.0, 300, [osv.WorkloadProfile("x", 60, 100, 40, 40, 1.0)], seed=2)
    decode = b2pa.FusedDecodeExecutor(model, dev, max_batch=4, evict_keep=48, evict_recent=16, evict_slack=8)
    longest = []

    def step(requests, *args, **kw):
        out = decode(requests, *args, **kw)
        longest.append(max(s.seq_len for r in requests for s in r.kv_caches))
        return out

    done, _ = osv.ContinuousScheduler(4, 128, 512).run(reqs, ex.prefill, step, ex.release)
    assert len(done) == 4 and all(len(r.generated_token_ids) == 40 for r in done)
    assert longest and max(longest) < 48 + 8
    assert b2pa.read_status(dev) == 0


@torch.no_grad()
def test_executor_refuses_layers_that_do_not_track(cuda_device):
    """A layer that does not track key weights is refused before the step: nothing has moved, and with the layers in
    step the same requests go on without eviction."""
    from oracle import serving as osv

    dev = cuda_device
    model = _model(dev, False)
    ex = osv.ModelExecutors(model, dev)
    reqs = osv.generate_requests(2, 1000.0, 300, [osv.WorkloadProfile("x", 60, 60, 20, 20, 1.0)], seed=2)
    bounded = b2pa.FusedDecodeExecutor(model, dev, max_batch=2, evict_keep=32, evict_slack=1)
    free = b2pa.FusedDecodeExecutor(model, dev, max_batch=2)
    refused = []

    def step(requests, *args, **kw):
        pool = requests[0].kv_caches[1].pool
        pool.key_weights = None  # the second layer stops tracking
        before = [(s.seq_len, list(s.block_ids)) for r in requests for s in r.kv_caches]
        tokens = [list(r.generated_token_ids) for r in requests]
        with pytest.raises(RuntimeError, match="track"):
            bounded(requests, *args, **kw)
        assert before == [(s.seq_len, list(s.block_ids)) for r in requests for s in r.kv_caches]
        assert tokens == [list(r.generated_token_ids) for r in requests]
        refused.append(1)
        return free(requests, *args, **kw)

    done, _ = osv.ContinuousScheduler(2, 128, 512).run(reqs, ex.prefill, step, ex.release)
    assert refused and len(done) == 2 and all(len(r.generated_token_ids) == 20 for r in done)
    assert b2pa.read_status(dev) == 0


@pytest.mark.parametrize("scale", [0.0, -0.3, 0.2])
@pytest.mark.parametrize("T", [1, 5, 140])
@pytest.mark.parametrize("kind,D", [("f32", 64), ("f32", 128), ("bf16", 64), ("f16", 128), ("f32", 32), ("bf16", 16),
                                    ("kv4", 64), ("kv4", 128), ("kv4", 256)])
def test_any_scale(cuda_device, scale, T, kind, D):
    """The C entries' scale may be zero (every visible key counts alike) or negative: key weights, and on 4-bit pools
    the attention."""
    dev, H, bs, n = cuda_device, 2, 16, 173
    rng = np.random.default_rng(D + T)
    NB = -(-n // bs)
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "kv4": torch.float32}[kind]
    k, v = rng.standard_normal((2, NB, H, bs, D))
    if kind == "kv4":
        pool, vpool = (torch.from_numpy(co.pack_pages(x, y)).to(dev) for x, y in ((k, False), (v, True)))
        k, v = co.stored(k), co.stored(v)
    else:
        pool = torch.from_numpy(k).to(dtype).to(dev)
        k = _np(pool)
    q = torch.from_numpy(rng.standard_normal((1, H, T, D))).to(dtype).to(dev)
    w = torch.zeros(NB, H, bs, device=dev)
    table, lens, cur = _i32(np.arange(NB)[None], dev), _i32([n], dev), _i32([T], dev)
    code = b2pa._lib.dtype_code(dtype)
    pool_code = b2pa._lib.DTYPE_KV4 if kind == "kv4" else code
    lib, status, stream = b2pa._lib.load(), b2pa._lib.status_buffer(dev).data_ptr(), b2pa._lib.stream_handle(dev)
    ws = torch.empty(lib.b2pa_key_weights_workspace_size(1, H, T, D, NB, bs, code, pool_code) + 256, dtype=torch.uint8,
                     device=dev)
    strides = b2pa._lib.strides4(q)
    assert 0 == lib.b2pa_key_weights(q.data_ptr(), strides, pool.data_ptr(), pool_code, NB, table.data_ptr(), NB, NB,
                                     lens.data_ptr(), cur.data_ptr(), 0, w.data_ptr(), w.data_ptr(), 1, H, T, D, bs,
                                     scale, code, ws.data_ptr(), ws.numel(), status, stream)
    K = co.rows_of(k, range(NB), n)
    p, _ = co.softmax_rows(_np(q)[0] * np.sign(scale), K, T, abs(scale))
    size = abs(scale) * float(np.einsum("htd,nhd->htn", np.abs(_np(q)[0]), np.abs(K)).max())
    got = co.rows_of(_np(w)[..., None], range(NB), n)[..., 0].T
    want = p.sum(1)
    assert (np.abs(got - want) <= want * (co.weight_error(D, size, n) + (T + 2) * 2.0 ** -23) + 2.0 ** -30).all()
    if kind != "kv4":
        return
    out = torch.empty_like(q)
    if T == 1:
        assert 0 == lib.b2pa_paged_decode_kv4(
            q.data_ptr(), strides, pool.data_ptr(), vpool.data_ptr(), NB, table.data_ptr(), NB, NB, lens.data_ptr(),
            cur.data_ptr(), out.data_ptr(), strides, 1, H, D, bs, scale, code, status, stream)
    else:
        ws = torch.empty(lib.b2pa_paged_prefill_kv4_workspace_size(1, H, T, D, NB, bs, code) + 256, dtype=torch.uint8,
                         device=dev)
        assert 0 == lib.b2pa_paged_prefill_kv4(
            q.data_ptr(), strides, pool.data_ptr(), vpool.data_ptr(), NB, table.data_ptr(), NB, NB, lens.data_ptr(),
            cur.data_ptr(), out.data_ptr(), strides, 1, H, T, D, bs, scale, code, ws.data_ptr(), ws.numel(), status, stream)
    V = co.rows_of(v, range(NB), n)
    ref = np.einsum("htn,nhd->htd", p, V)
    assert (np.abs(_np(out)[0] - ref) <= co.output_bound(ref, 2.0 ** -24, D, size, n, np.abs(V).max())).all()


@pytest.mark.parametrize("dtype,kv4,D", [
    (torch.float32, False, 32), (torch.float32, False, 64), (torch.float32, True, 64), (torch.float32, False, 128),
    (torch.bfloat16, False, 64), (torch.bfloat16, True, 128), (torch.float16, False, 128), (torch.float16, True, 256),
    (torch.bfloat16, False, 256), (torch.bfloat16, False, 16)])
@pytest.mark.parametrize("T", [1, 50])
@pytest.mark.parametrize("far", [1e5, 5e5, 2e6, 3e7])
def test_key_weights_of_far_logits(cuda_device, dtype, kv4, D, T, far):
    """Logits whose own rounding is of the size of usual logits: a query whose largest is far ahead gives that key a
    weight of one, whatever the size of the logit."""
    dev, H, bs, n = cuda_device, 6, 16, 500
    rng = np.random.default_rng(D)
    NB = -(-n // bs)
    big = 64.0 if dtype == torch.float16 and not kv4 else 4096.0
    k = rng.standard_normal((NB, H, bs, D)) * big
    if kv4:
        pool, k = torch.from_numpy(co.pack_pages(k, False)).to(dev), co.stored(k)
    else:
        pool = torch.from_numpy(k).to(dtype).to(dev)
        k = _np(pool)
    far = min(far, 1e4 * big) if dtype == torch.float16 else far
    q = torch.from_numpy(rng.standard_normal((1, H, T, D)) * far / big).to(dtype).to(dev)
    w = torch.zeros(NB, H, bs, device=dev)
    b2pa.accumulate_key_weights(q, pool, w, _i32(np.arange(NB)[None], dev), _i32([n], dev), _i32([T], dev))
    K = co.rows_of(k, range(NB), n)
    z = np.einsum("htd,nhd->htn", _np(q)[0], K) * D ** -0.5
    z = np.where(np.arange(n) < n - T + 1 + np.arange(T)[:, None], z, -np.inf)
    first, second = np.sort(z, -1)[..., -1], np.sort(z, -1)[..., -2]
    clear = first - second > 40 + 2.0 ** -16 * np.abs(_np(q)[0]).max() * np.abs(K).max() * D ** 0.5
    assert clear.mean() > 0.6
    got = co.rows_of(_np(w)[..., None], range(NB), n)[..., 0].T          # [H, n]
    least = np.zeros((H, n))
    for h in range(H):
        np.add.at(least[h], z[h].argmax(-1)[clear[h]], 1.0)
    unclear = (~clear).sum(1)[:, None]
    # a weight is 2^0 over a sum of it alone: exact but for the exponential's 2^-22 and a rounding per addend
    assert (got >= least * (1 - (T + 4) * 2.0 ** -22)).all()
    assert (got <= least + unclear + (T + 4) * 2.0 ** -22 * (least + 1)).all()
