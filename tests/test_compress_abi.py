"""The cache-compression entry points refuse bad arguments with status codes,
before anything reaches a GPU, and their plain oracle is self-consistent.  No
kernel runs here."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from b2pa import _lib
from tests import _compress_oracle as co


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        import __graft_entry__

        __graft_entry__.build()
    return _lib.load()


def _i64(t):
    return (ctypes.c_int64 * 4)(*t)


# made-up, never dereferenced addresses: every call below is refused on the host
BASE = dict(q=4096, qs=(64, 64, 64, 1), kp=8192, vp=16384, nb=10, pt=32, pts=4, mp=4, sl=64, cl=128, out=32768,
            os=(64, 64, 64, 1), B=1, H=1, T=4, D=64, bs=16, dt=0, ws=256, wsb=1 << 30)


def _append(lib, **kw):
    a = {**BASE, **kw}
    return lib.b2pa_kv4_append(a["q"], _i64(a["qs"]), a["out"], _i64(a["os"]), a["kp"], a["vp"], a["nb"], a["pt"],
                               a["pts"], a["mp"], a["sl"], a["cl"], None, a["B"], a["H"], a["T"], a["D"], a["bs"],
                               a["dt"], None, None)


def _read(lib, **kw):
    a = {**BASE, **kw}
    return lib.b2pa_kv4_read(a["kp"], a["vp"], a["nb"], a["pt"], a["pts"], a["mp"], a["sl"], a["cl"], a["q"],
                             _i64(a["qs"]), a["out"], _i64(a["os"]), a["B"], a["H"], a["T"], a["D"], a["bs"], a["dt"],
                             None, None)


def _decode(lib, **kw):
    a = {**BASE, **kw}
    return lib.b2pa_paged_decode_kv4(a["q"], _i64(a["qs"]), a["kp"], a["vp"], a["nb"], a["pt"], a["pts"], a["mp"],
                                     a["sl"], a["cl"], a["out"], _i64(a["os"]), a["B"], a["H"], a["D"], a["bs"], 0.125,
                                     a["dt"], None, None)


def _prefill(lib, **kw):
    a = {**BASE, **kw}
    return lib.b2pa_paged_prefill_kv4(a["q"], _i64(a["qs"]), a["kp"], a["vp"], a["nb"], a["pt"], a["pts"], a["mp"],
                                      a["sl"], a["cl"], a["out"], _i64(a["os"]), a["B"], a["H"], a["T"], a["D"],
                                      a["bs"], 0.125, a["dt"], a["ws"], a["wsb"], None, None)


def _weights(lib, **kw):
    a = {**BASE, "pd": 0, "win": 0, "w": 65536, **kw}
    return lib.b2pa_key_weights(a["q"], _i64(a["qs"]), a["kp"], a["pd"], a["nb"], a["pt"], a["pts"], a["mp"], a["sl"],
                                a["cl"], a["win"], a["w"], a["out"], a["B"], a["H"], a["T"], a["D"], a["bs"], 0.125,
                                a["dt"], a["ws"], a["wsb"], None, None)


def _evict(lib, **kw):
    a = {**BASE, "pd": 0, "w": 65536, "ot": None, "ots": 0, "keep": 8, "recent": 2, "kept": 1 << 20, **kw}
    return lib.b2pa_evict(a["kp"], a["vp"], a["pd"], a["w"], a["nb"], a["pt"], a["pts"], a["mp"], a["ot"], a["ots"],
                          a["sl"], a["keep"], a["recent"], a["kept"], a["B"], a["H"], a["D"], a["bs"], None, None)


@pytest.mark.parametrize("call", [_append, _read, _decode, _prefill])
def test_common_refusals(lib, call):
    assert call(lib, H=0) == -1
    assert call(lib, B=-1) == -1
    assert call(lib, dt=7) == -2
    assert call(lib, dt=3) == -2                     # rows outside the cache are never 4-bit
    assert call(lib, D=32) == -2 and call(lib, D=96) == -2
    assert call(lib, bs=12) == -2
    assert call(lib, pts=2) == -1                    # row stride < max_pages
    assert call(lib, pt=0) == -1
    assert call(lib, kp=0) == -1
    assert call(lib, kp=8200) == -2                  # pool not 16-byte aligned
    assert call(lib, q=0) == -1 and call(lib, out=0) == -1
    assert call(lib, B=70000) == -2
    assert call(lib, mp=1 << 28, pts=1 << 28) == -2  # positions past 2^31
    assert call(lib, B=0) == 0                       # nothing to do
    assert b"B=0" not in lib.b2pa_last_error_string()


def test_attention_refusals(lib):
    for call in (_decode, _prefill):
        assert call(lib, qs=(64, 64, 64, 2)) == -2
        assert call(lib, q=4100) == -2               # rows not 16-byte aligned
        assert call(lib, qs=(66, 66, 66, 1)) == -2
    assert _prefill(lib, wsb=16) == -4
    assert _prefill(lib, ws=0) == -4
    assert _prefill(lib, ws=264) == -4
    assert _read(lib, os=(64, 64, 64, 2)) == -2


def test_key_weights_refusals(lib):
    assert _weights(lib, pd=1) == -2                 # bf16 pool, fp32 q
    assert _weights(lib, D=48) == -2
    assert _weights(lib, pd=3, D=32) == -2           # 4-bit pages have no head_dim 32
    assert _weights(lib, win=-1) == -1
    assert _weights(lib, w=0) == -1 and _weights(lib, out=0) == -1
    assert _weights(lib, kp=8200) == -2
    assert _weights(lib, wsb=4) == -4
    assert _weights(lib, T=0) == 0


def test_evict_refusals(lib):
    assert _evict(lib, keep=-1) == -1 and _evict(lib, recent=-1) == -1
    assert _evict(lib, pd=5) == -2 and _evict(lib, D=48) == -2
    assert _evict(lib, w=0) == -1 and _evict(lib, kept=0) == -1 and _evict(lib, sl=0) == -1
    assert _evict(lib, w=65544) == -2                # weights not 16-byte aligned
    assert _evict(lib, ot=64, ots=1, keep=17) == -1  # one page of 16 slots a row
    assert _evict(lib, keep=0) == 0 and _evict(lib, B=0) == 0


def test_python_refusals_without_a_gpu():
    import b2pa

    kp = torch.zeros(4, 2, 16, 36, dtype=torch.uint8)
    t = torch.zeros(1, 4, dtype=torch.int32)
    one = torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 2, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        b2pa.kv4_append(q, q, kp, kp, t, one, one)
    with pytest.raises(RuntimeError, match="CUDA"):
        b2pa.paged_attention_decode_kv4(q, kp, kp, t, one, one)
    with pytest.raises(RuntimeError, match="CUDA"):
        b2pa.evict_by_weight(q, q, torch.zeros(1, 2, 1), t, one, 4)
    with pytest.raises(ValueError, match="head_dim"):
        b2pa.Kv4BlockPool(16, 4, 2.0).ensure_initialized(2, 32, torch.float32, torch.device("meta"))
    pool = b2pa.LayerBlockPool(16, 4, 2.0)
    with pytest.raises(ValueError, match="window"):
        pool.track_key_weights(window=0)
    cache = b2pa.BatchedPagedKVCache([b2pa.PagedKVCacheState(pool)], pool)
    with pytest.raises(RuntimeError, match="track"):
        cache.evict(4)
    with pytest.raises(ValueError, match="keep"):
        cache.evict(0)


def test_kv4_pool_bookkeeping_on_meta():
    """Allocation, growth and byte counts of a 4-bit pool: as the plain pool's, at 4.5 bits a value."""
    import b2pa

    pool = b2pa.Kv4BlockPool(16, 2, 2.0)
    pool.track_key_weights()
    k = torch.empty(1, 3, 40, 128, device="meta", dtype=torch.bfloat16)
    cache = b2pa.BatchedPagedKVCache([b2pa.PagedKVCacheState(pool)], pool)
    cache.append_batch(k, k, [40])
    assert pool.capacity_blocks == 4 and cache.states[0].block_ids == [1, 0, 3]
    assert pool.k_blocks.shape == (4, 3, 16, 72) and pool.k_blocks.dtype == torch.uint8
    assert pool.key_weights.shape == (4, 3, 16)
    assert pool.bytes_per_block() == 2 * 3 * 16 * 72
    assert cache.live_bytes() == 40 * 3 * 72 * 2


def test_evicting_before_the_first_append():
    """A pool that tracks and holds nothing is told from one that does not track."""
    import b2pa

    pool = b2pa.LayerBlockPool(16, 2, 2.0)
    cache = b2pa.BatchedPagedKVCache([b2pa.PagedKVCacheState(pool)], pool)
    with pytest.raises(RuntimeError, match="does not track"):
        cache.evict(4)
    pool.track_key_weights()
    with pytest.raises(RuntimeError, match="before its first append"):
        cache.evict(4)


def test_oracle_quantiser():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((64, 128)) * np.exp(rng.uniform(-12, 12, (64, 1)))).astype(np.float32)
    y = co.stored(x)
    g, s = x.reshape(64, 8, 16), co.SCALES[co.quantise(x)[1]]
    # half a step of s everywhere the group's maximum fits 7.5 s, and the scale within half a step of max / 7
    top = np.abs(g).max(-1)
    ok = (top / 7 > 2.0 ** -14) & (top / 7 < 9216)
    assert ok.any()
    assert (np.abs(y.reshape(g.shape) - g).max(-1) <= s / 2 * (1 + 1e-9))[ok].all()
    assert (np.abs(s - top / 7) <= top / 7 / 16 * (1 + 1e-9))[ok].all()
    for t in (torch.float16, torch.bfloat16):
        assert np.array_equal(torch.from_numpy(y).to(t).double().numpy(), y)  # exact in 16 bits
    bad = x[:1].copy()
    bad[0, 5], bad[0, 40] = np.nan, np.inf
    r = co.stored(bad).reshape(8, 16)
    assert np.isnan(r[0]).all() and np.isnan(r[2]).all() and np.isfinite(np.delete(r, [0, 2], 0)).all()


def test_extension_module_is_the_running_pytorchs(lib, monkeypatch):
    """A module built for another PyTorch is not loaded: a warning, and every call is declined to the longer way."""
    assert torch.__version__ in _lib.calls_path().name and _lib.calls_path().exists()
    assert _lib.calls().__file__ == str(_lib.calls_path())
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    monkeypatch.setattr(_lib, "_calls", None)
    with pytest.warns(RuntimeWarning, match="not built"):
        calls = _lib.calls()
    assert calls.kv4_append(1, 2) is NotImplemented and calls.set_status(0, 0) is NotImplemented
    assert _lib.calls() is calls


def test_short_calls_decline(lib):
    """The extension module's functions launch nothing and raise nothing on what they do not take: CPU tensors, other
    objects, missing arguments."""
    calls = _lib.calls()
    x = torch.zeros(1, 2, 1, 64)
    for name in ("kv4_append", "kv4_read", "decode_kv4", "prefill_kv4", "key_weights", "evict"):
        fn = getattr(calls, name)
        for n in range(10):
            assert fn(*[x] * n) is NotImplemented
            assert fn(*[None] * n) is NotImplemented
            assert fn(*["x", 3, x, None, 2 ** 70][:n]) is NotImplemented
