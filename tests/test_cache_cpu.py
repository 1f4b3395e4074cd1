"""The 4-bit key/value cache without a GPU: the oracle's own properties and everything that is refused on the host."""
import ctypes

import numpy as np
import pytest
import torch

from cobalt_amd import KVCache, KVRows, _lib, ops
from oracle import cache_ref as R


def test_held_values_are_within_half_a_step():
    g = np.random.default_rng(0)
    x = (g.standard_normal((40, 3, 128)) * np.exp(g.standard_normal((1, 3, 128)))).astype(np.float16).astype(np.float32)
    for group in (32, 64, 128):
        k, v = R.held(x, -x, group)
        for y, z in ((k, x), (v, -x)):
            w = z.reshape(40, 3, -1, group)
            # the step is rounded to fp16, and 15 of it may end short of the largest value by 15 half steps of fp16
            step = (w.max(-1) - w.min(-1)) / 15
            slack = (0.5 + 16 * 2.0 ** -11) * step + 2.0 ** -11 * np.abs(w).max(-1)
            assert (np.abs(y - z).reshape(w.shape).max(-1) <= slack).all()
            assert len(np.unique(y[0, 0, :group])) <= 16


def test_oracle_attention_by_hand():
    k, v = np.zeros((3, 2)), np.array([[1.0, 0], [2, 0], [6, 0]])
    o, *_ = R.attention(np.ones((3, 2)), k, v, np.arange(3), np.ones(3, bool), 1.0)
    np.testing.assert_allclose(o[:, 0], [1, 1.5, 3])
    o, *_ = R.attention(np.ones((3, 2)), k, v, np.arange(3), np.ones(3, bool), 1.0, window=1, sinks=1)
    np.testing.assert_allclose(o[:, 0], [1, 1.5, 3.5])
    o, *_ = R.attention(np.ones((1, 2)), k, v, np.array([-1]), np.ones(3, bool), 1.0)
    assert not o.any()


def _cache(**kw):
    d = dict(k_codes=0x1000, v_codes=0x2000, k_meta=0x3000, v_meta=0x4000, pages=10, page=16, heads=2, head_dim=128, group=32)
    return _lib.CbkCache(**{**d, **kw})


def _rows(**kw):
    d = dict(table=0x5000, ld_table=4, lens=0x6000, starts=None, seqs=2, table_cols=4, tokens=2)
    return _lib.CbkRows(**{**d, **kw})


def _write(c, r, k=0x7000, kr=256, kh=128, dt=1):
    return _lib.lib().cbk_cache_write(ctypes.byref(c), ctypes.byref(r), k, kr, kh, 0x8000, 256, 128, dt, None)


def _read(c, r, k=0x7000, kr=256, kh=128, dt=1):
    return _lib.lib().cbk_cache_read(ctypes.byref(c), ctypes.byref(r), k, kr, kh, 0x8000, 256, 128, dt, None)


def _attend(c, r, q=0x7000, qr=512, qh=128, out=0x8000, dt=1, heads=4, scale=1.0, window=0, sinks=0, ws=0x10000, room=1 << 40):
    return _lib.lib().cbk_cache_attention(ctypes.byref(c), ctypes.byref(r), q, qr, qh, out, 512, 128, dt, heads, scale, window, sinks,
                                          ws, room, None)


BAD_CACHE = [(dict(head_dim=96), -2), (dict(head_dim=0), -2), (dict(group=16), -2), (dict(group=48), -2), (dict(head_dim=64, group=128), -2),
             (dict(page=8), -2), (dict(page=48), -2), (dict(page=512), -2), (dict(page=0), -2), (dict(pages=0), -3), (dict(pages=1 << 31), -3),
             (dict(heads=0), -3), (dict(k_codes=None), -1), (dict(v_meta=None), -1), (dict(v_codes=0x2008), -4), (dict(k_meta=0x3004), -4)]
BAD_ROWS = [(dict(seqs=-1), -3), (dict(tokens=-1), -3), (dict(tokens=1 << 30, seqs=1), -3), (dict(tokens=3), -3), (dict(seqs=0), -3),
            (dict(ld_table=3), -3), (dict(table_cols=-1, ld_table=0), -3), (dict(table_cols=1 << 28, ld_table=1 << 28), -3),
            (dict(table=None), -1), (dict(lens=None), -1), (dict(lens=0x6002), -4), (dict(table=0x5001), -4), (dict(starts=0x9002), -4)]


@pytest.mark.parametrize("call", [_write, _read, _attend])
def test_entry_points_refuse_bad_descriptions_before_any_launch(call):
    for kw, want in BAD_CACHE:
        assert call(_cache(**kw), _rows()) == want, kw
    for kw, want in BAD_ROWS:
        assert call(_cache(), _rows(**kw)) == want, kw
    L = _lib.lib()
    assert L.cbk_cache_write(None, None, None, 0, 0, None, 0, 0, 1, None) == -1
    # nothing to do: no launch either
    assert call(_cache(), _rows(tokens=0)) == 0
    assert call(_cache(), _rows(seqs=0, tokens=5, starts=0x9000)) == 0


def test_entry_points_refuse_bad_tensors_before_any_launch():
    for call in (_write, _read):
        assert call(_cache(), _rows(), k=None) == -1
        assert call(_cache(), _rows(), k=0x7008) == -4
        assert call(_cache(), _rows(), kr=260) == -4
        assert call(_cache(), _rows(), kh=132) == -4
        assert call(_cache(), _rows(), kr=-256) == -3
        assert call(_cache(), _rows(), dt=3) == -5
    assert _write(_cache(), _rows(), dt=0) == -5                     # float32 comes out of the cache, but does not go in
    assert _attend(_cache(), _rows(), q=None) == -1
    assert _attend(_cache(), _rows(), out=None) == -1
    assert _attend(_cache(), _rows(), q=0x7008) == -4
    assert _attend(_cache(), _rows(), qr=516) == -4
    assert _attend(_cache(), _rows(), dt=0) == -5
    for heads in (0, -2, 3):
        assert _attend(_cache(), _rows(), heads=heads) == -3
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert _attend(_cache(), _rows(), scale=scale) == -3
    assert _attend(_cache(), _rows(), window=-1) == -3
    assert _attend(_cache(), _rows(), sinks=-1) == -3
    assert _attend(_cache(), _rows(), ws=0x10010) == -4
    big = _rows(table_cols=1000, ld_table=1000)
    need = _lib.lib().cbk_cache_attention_workspace_bytes(ctypes.byref(_cache()), ctypes.byref(big), 4)
    assert need > 0
    assert _attend(_cache(), big, room=need - 1) == -6
    assert _attend(_cache(), big, ws=None, room=0) == -6


def test_entry_points_refuse_what_would_pass_their_integers():
    most = (1 << 30) // 16
    for call in (_write, _read, _attend):
        assert call(_cache(), _rows(table_cols=most + 1, ld_table=most + 1)) == -3
    assert _lib.lib().cbk_cache_attention_workspace_bytes(ctypes.byref(_cache()), ctypes.byref(_rows(table_cols=most, ld_table=most)), 4) > 0
    for call in (_write, _read):
        assert call(_cache(heads=4096), _rows(tokens=1 << 17, seqs=1)) == -3          # 2^36 numbers
    assert _attend(_cache(), _rows(), heads=2 * 257) == -3
    assert _attend(_cache(), _rows(), scale=1e-31) == -3 and _attend(_cache(), _rows(), scale=1e31) == -3
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    c = KVCache(3, 2, 64, page=32, device="cpu")
    for scale in (1e-31, 1e31, -1.0, float("nan")):
        with pytest.raises(ValueError):
            ops.cache_attention(c, x, c.rows([[0, 1], [2, -1]], [40, 7]), scale=scale)


def test_sizes():
    L = _lib.lib()
    c = _cache(pages=7, page=64, heads=3, head_dim=256, group=64)
    assert L.cbk_cache_code_bytes(ctypes.byref(c)) == 7 * 64 * 3 * 128
    assert L.cbk_cache_meta_bytes(ctypes.byref(c)) == 7 * 64 * 3 * 4 * 4
    assert L.cbk_cache_code_bytes(ctypes.byref(_cache(group=48))) == 0
    for kw in (dict(head_dim=80), dict(group=16), dict(page=20), dict(pages=0), dict(heads=0), dict(head_dim=64, group=128)):
        args = {**dict(pages=2, heads=2, head_dim=128), **kw}
        with pytest.raises(ValueError):
            KVCache(**args, device="cpu")
    k = KVCache(3, 2, 64, page=32, group=64, device="cpu")
    assert k.nbytes() == 2 * (3 * 2 * 32 * 32 + 3 * 2 * 32 * 4) and not k.k_codes.any() and not k.v_meta.any()
    r = k.rows([[0, 1], [2, -1]], torch.tensor([40, 7]), [0, 1, 2])
    assert isinstance(r, KVRows) and all(t.dtype == torch.int32 for t in r) and k.rows([[0]], [1]).starts is None


def test_ops_refuse_a_cache_on_the_cpu():
    c = KVCache(3, 2, 64, page=32, device="cpu")
    r = c.rows([[0, 1], [2, -1]], [40, 7])
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    for call in (lambda: ops.cache_write(c, x, x, r), lambda: ops.cache_read(c, r, 2), lambda: ops.cache_attention(c, x, r)):
        with pytest.raises(_lib.CbkError):
            call()


def test_ops_refuse_tensors_that_require_a_gradient():
    c = KVCache(3, 2, 64, page=32, device="cpu")
    r = c.rows([[0, 1], [2, -1]], [40, 7])
    x, y = torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, 2, 64, dtype=torch.float16, requires_grad=True)
    calls = (lambda: ops.cache_attention(c, y, r), lambda: ops.cache_attention(c, x, r, out=y), lambda: ops.cache_write(c, y, x, r),
             lambda: ops.cache_write(c, x, y, r), lambda: ops.cache_read(c, r, 2, out=(x, y)))
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(_lib.CbkError):             # as any other call: the cache is not on the GPU
            call()


def test_rows_of_integers_that_int32_does_not_hold():
    c = KVCache(3, 2, 64, page=32, device="cpu")
    for table in ([[0, 1 << 32], [-(1 << 33), 1]], torch.tensor([[0, 1 << 32], [-(1 << 33), 1]])):
        r = c.rows(table, [(1 << 32) + 5, 7], torch.tensor([0, 1, 1 << 40]))
        assert r.table.tolist() == [[0, (1 << 31) - 1], [-(1 << 31), 1]]        # neither is a page of the pool
        assert r.lens.tolist() == [(1 << 31) - 1, 7] and r.starts.tolist() == [0, 1, (1 << 31) - 1]
    for t in (torch.int8, torch.int16, torch.uint8, torch.uint16, torch.uint32, torch.int64):
        assert c.rows(torch.tensor([[0, 2]], dtype=t), torch.tensor([100], dtype=t)).table.tolist() == [[0, 2]]
    for bad in ([[0.5, 1.0]], torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.bool)):
        with pytest.raises(TypeError, match="table must be integers"):
            c.rows(bad, [3])
    with pytest.raises(TypeError, match="lens must be integers"):
        c.rows([[0, 1]], [3.7])
    r = c.rows(torch.zeros(0, 2, dtype=torch.int32), [], [0])
    assert r.lens.dtype == torch.int32 and r.lens.shape == (0,)
