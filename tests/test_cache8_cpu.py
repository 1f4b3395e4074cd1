"""The 8-bit key/value cache and the tables of pages without a GPU: the oracle's own properties and everything that is refused on the host."""
import ctypes

import numpy as np
import pytest
import torch

from cobalt_amd import KVCache8, KVPages, KVRows, _lib, ops
from oracle import cache8_ref as R8
from oracle import cache_ref as R


def test_the_oracles_e4m3_is_torchs():
    x = torch.cat([torch.linspace(-448, 448, 100001), torch.linspace(-1, 1, 20001) * 2.0 ** -5]).double()
    want = x.float().to(torch.float8_e4m3fn).double()
    assert (torch.from_numpy(R8.e4m3(x.float().double().numpy())) == want).all()
    for e in range(-15, 8):
        assert R8.exponent(448 * 2.0 ** e) == e and R8.exponent(np.nextafter(448 * 2.0 ** e, np.inf)) == min(e + 1, 7)
    assert R8.exponent(0.0) == -15


def test_held_values_are_within_half_a_step():
    """Written at once or token by token: three bits behind the first of each value, steps of 2^-9 of the scale at least."""
    g = np.random.default_rng(0)
    x = (g.standard_normal((40, 3, 64)) * np.exp(2 * g.standard_normal((40, 1, 1)))).astype(np.float16).astype(np.float32)
    for steps in ([40], [1] * 40, [3, 30, 7]):
        for block in (16, 32):
            p, at = R8.Pool(2, 3, 64, 32, block), 0
            for n in steps:
                at += n
                p.write([[1, 0]], [at], [0, n], x[at - n:at], -x[at - n:at])
            k, v, there = p.read([[1, 0]], 0, range(40))
            assert there.all()
            for y, z in ((k, x), (v, -x)):
                top = np.stack([np.abs(z[i:i + block]).max((0, 2)) for i in range(0, 40, block)]).repeat(block, 0)[:40, :, None]
                # one rounding, or as many as the scale grew: of those past the first each by half the steps that the scale has by then
                slack = np.maximum(np.abs(z) * 2.0 ** -4, top * 2.0 ** -8 * 2.0 ** -9) * (1 if len(steps) == 1 else 2)
                assert (np.abs(y - z) <= slack + 2.0 ** -25).all()


def test_the_oracles_attention_is_the_other_caches():
    g = np.random.default_rng(1)
    q, k, v = (g.standard_normal((n, 8)) for n in (5, 30, 30))
    there = g.random(30) < 0.8
    for kw in ({}, dict(window=7), dict(window=3, sinks=4)):
        a = R.attention(q, k, v, np.arange(25, 30), there, 0.3, **kw)
        b = R8.attention(q, k, v, np.arange(25, 30), there, 0.3, **kw)
        np.testing.assert_allclose(a[0], b[0], atol=1e-12)
        np.testing.assert_allclose(a[2], b[2], atol=1e-12)
        assert (b[1] >= a[1] - 1e-9).all() and (b[3] <= a[3] + 1e-12).all()
    o, *_ = R8.attention(q, k, v, np.full(5, -1), there, 1.0)
    assert not o.any()


def _cache(**kw):
    d = dict(k_codes=0x1000, v_codes=0x2000, scales=0x3000, pages=10, page=16, heads=2, head_dim=128, block=16)
    return _lib.CbkCache8(**{**d, **kw})


def _rows(**kw):
    d = dict(table=0x5000, ld_table=4, lens=0x6000, starts=None, seqs=2, table_cols=4, tokens=2)
    return _lib.CbkRows(**{**d, **kw})


def _write(c, r, k=0x7000, kr=256, kh=128, dt=1):
    return _lib.lib().cbk_cache_eight_write(ctypes.byref(c), ctypes.byref(r), k, kr, kh, 0x8000, 256, 128, dt, None)


def _read(c, r, k=0x7000, kr=256, kh=128, dt=1):
    return _lib.lib().cbk_cache_eight_read(ctypes.byref(c), ctypes.byref(r), k, kr, kh, 0x8000, 256, 128, dt, None)


def _attend(c, r, q=0x7000, qr=512, qh=128, out=0x8000, dt=1, heads=4, scale=1.0, window=0, sinks=0, ws=0x10000, room=1 << 40):
    return _lib.lib().cbk_cache_eight_attention(ctypes.byref(c), ctypes.byref(r), q, qr, qh, out, 512, 128, dt, heads, scale, window, sinks,
                                           ws, room, None)


BAD_CACHE = [(dict(head_dim=96), -2), (dict(head_dim=0), -2), (dict(block=8), -2), (dict(block=48, page=64), -2), (dict(block=32), -2),
             (dict(block=0), -2), (dict(page=8), -2), (dict(page=48), -2), (dict(page=512), -2), (dict(page=0), -2), (dict(pages=0), -3),
             (dict(pages=1 << 31), -3), (dict(heads=0), -3), (dict(heads=4097), -3), (dict(k_codes=None), -1), (dict(scales=None), -1),
             (dict(v_codes=0x2008), -4), (dict(scales=0x3004), -4)]
BAD_ROWS = [(dict(seqs=-1), -3), (dict(tokens=-1), -3), (dict(tokens=1 << 30, seqs=1), -3), (dict(tokens=3), -3), (dict(seqs=0), -3),
            (dict(ld_table=3), -3), (dict(table_cols=-1, ld_table=0), -3), (dict(table_cols=1 << 28, ld_table=1 << 28), -3),
            (dict(table=None), -1), (dict(lens=None), -1), (dict(lens=0x6002), -4), (dict(table=0x5001), -4), (dict(starts=0x9002), -4)]


@pytest.mark.parametrize("call", [_write, _read, _attend])
def test_entry_points_refuse_bad_descriptions_before_any_launch(call):
    for kw, want in BAD_CACHE:
        assert call(_cache(**kw), _rows()) == want, kw
    for kw, want in BAD_ROWS:
        assert call(_cache(), _rows(**kw)) == want, kw
    assert _lib.lib().cbk_cache_eight_write(None, None, None, 0, 0, None, 0, 0, 1, None) == -1
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
        assert call(_cache(heads=4096), _rows(tokens=1 << 17, seqs=1)) == -3          # 2^29 rows and heads
    assert _write(_cache(), _rows(), dt=0) == -5                     # float32 comes out of the cache, but does not go in
    assert _attend(_cache(), _rows(), q=None) == -1
    assert _attend(_cache(), _rows(), out=None) == -1
    assert _attend(_cache(), _rows(), q=0x7008) == -4
    assert _attend(_cache(), _rows(), qr=516) == -4
    assert _attend(_cache(), _rows(), dt=0) == -5
    for heads in (0, -2, 3, 2 * 257):
        assert _attend(_cache(), _rows(), heads=heads) == -3
    for scale in (0.0, -1.0, float("nan"), float("inf"), 1e-31, 1e31):
        assert _attend(_cache(), _rows(), scale=scale) == -3
    assert _attend(_cache(), _rows(), window=-1) == -3
    assert _attend(_cache(), _rows(), sinks=-1) == -3
    assert _attend(_cache(), _rows(), ws=0x10010) == -4
    big = _rows(table_cols=1000, ld_table=1000)
    need = _lib.lib().cbk_cache_eight_attention_workspace_bytes(ctypes.byref(_cache()), ctypes.byref(big), 4)
    assert need > 0
    assert _attend(_cache(), big, room=need - 1) == -6
    assert _attend(_cache(), big, ws=None, room=0) == -6
    most = (1 << 30) // 16
    for call in (_write, _read, _attend):
        assert call(_cache(), _rows(table_cols=most + 1, ld_table=most + 1)) == -3


def test_sizes():
    L = _lib.lib()
    c = _cache(pages=7, page=64, heads=3, head_dim=256, block=32)
    assert L.cbk_cache_eight_code_bytes(ctypes.byref(c)) == 7 * 64 * 3 * 256
    assert L.cbk_cache_eight_scale_bytes(ctypes.byref(c)) == 7 * 3 * 2 * 8
    assert L.cbk_cache_eight_code_bytes(ctypes.byref(_cache(block=48))) == 0
    for kw in (dict(head_dim=80), dict(block=8), dict(block=128), dict(page=20), dict(pages=0), dict(heads=0)):
        args = {**dict(pages=2, heads=2, head_dim=128), **kw}
        with pytest.raises(ValueError):
            KVCache8(**args, device="cpu")
    k = KVCache8(3, 2, 64, page=32, block=16, device="cpu")
    assert k.nbytes() == 2 * (3 * 2 * 32 * 64) + 3 * 2 * 2 * 8 and not k.k_codes.any() and not k.scales.any()
    r = k.rows([[0, 1], [2, -1]], torch.tensor([40, 7]), [0, 1, 2])
    assert isinstance(r, KVRows) and all(t.dtype == torch.int32 for t in r)


def test_ops_refuse_a_cache_on_the_cpu():
    c = KVCache8(3, 2, 64, page=32, device="cpu")
    r = c.rows([[0, 1], [2, -1]], [40, 7])
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    for call in (lambda: ops.cache_write(c, x, x, r), lambda: ops.cache_read(c, r, 2), lambda: ops.cache_attention(c, x, r),
                 lambda: ops.cache_slots(c, r, 2)):
        with pytest.raises(_lib.CbkError):
            call()
    y = x.clone().requires_grad_()
    for call in (lambda: ops.cache_write(c, y, x, r), lambda: ops.cache_read(c, r, 2, out=(x, y)), lambda: ops.cache_attention(c, y, r)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()


# ------------------------------------------------------------------ tables of pages
def _pages(**kw):
    d = dict(table=0x5000, ld_table=4, lens=0x6000, free_pages=0x7000, free_count=0x8000, pages=10, seqs=2, table_cols=4, page=16)
    return _lib.CbkPages(**{**d, **kw})


def _resize(p, want=0x9000, starts=0xa000, ws=0x10000, room=1 << 20):
    return _lib.lib().cbk_cache_pages(ctypes.byref(p), want, starts, ws, room, None)


def test_tables_refuse_bad_descriptions_before_any_launch():
    for kw, want in [(dict(page=8), -2), (dict(page=48), -2), (dict(page=512), -2), (dict(pages=0), -3), (dict(pages=1 << 31), -3),
                     (dict(seqs=-1), -3), (dict(seqs=1 << 24), -3), (dict(table_cols=5), -3), (dict(table_cols=-1, ld_table=0), -3),
                     (dict(table_cols=(1 << 26) + 1, ld_table=1 << 27), -3), (dict(table=None), -1), (dict(lens=None), -1),
                     (dict(free_pages=None), -1), (dict(free_count=None), -1), (dict(lens=0x6001), -4), (dict(free_pages=0x7002), -4)]:
        assert _resize(_pages(**kw)) == want, kw
    assert _resize(_pages(), want=None) == -1
    assert _resize(_pages(), want=0x9002) == -4 and _resize(_pages(), starts=0xa001) == -4 and _resize(_pages(), ws=0x10010) == -4
    assert _lib.lib().cbk_cache_pages_workspace_bytes(ctypes.byref(_pages())) == 0
    for kw in (dict(seqs=2000), dict(seqs=100, table_cols=100, ld_table=100)):
        need = _lib.lib().cbk_cache_pages_workspace_bytes(ctypes.byref(_pages(**kw)))
        assert need > 0
        assert _resize(_pages(**kw), room=need - 1) == -6 and _resize(_pages(**kw), ws=None) == -6
    assert _resize(_pages(seqs=1 << 16, table_cols=1 << 15, ld_table=1 << 15)) == -3              # 2^31 entries
    assert _resize(_pages(seqs=0)) == 0                             # nothing to do
    assert _lib.lib().cbk_cache_pages(None, None, None, None, 0, None) == -1


def test_slots_refuse_bad_descriptions_before_any_launch():
    call = lambda r, pages=10, page=16, slots=0x7000, pos=0x8000: _lib.lib().cbk_cache_slots(ctypes.byref(r), pages, page, slots, pos, None)
    for kw, want in BAD_ROWS:
        assert call(_rows(**kw)) == want, kw
    for page in (0, 8, 24, 512):
        assert call(_rows(), page=page) == -2
    assert call(_rows(), pages=0) == -3 and call(_rows(), pages=1 << 31) == -3
    assert call(_rows(), slots=0x7004) == -4 and call(_rows(), pos=0x8002) == -4
    assert call(_rows(tokens=0)) == 0 and call(_rows(), slots=None, pos=None) == 0


def test_tables_of_python():
    for kw in (dict(pages=0), dict(seqs=0), dict(max_len=0), dict(page=24), dict(pages=1 << 31), dict(max_len=(1 << 30) + 1)):
        with pytest.raises(ValueError):
            KVPages(**{**dict(pages=10, seqs=3, max_len=100, page=16), **kw}, device="cpu")
    t = KVPages(10, 3, 100, page=16, device="cpu")
    assert t.table.shape == (3, 7) and bool((t.table == -1).all()) and not t.lens.any()
    assert t.free.tolist() == list(range(9, -1, -1)) and t.count.tolist() == [10]
    with pytest.raises(_lib.CbkError):
        ops.cache_pages(t, torch.zeros(3, dtype=torch.int32))
    for bad in (torch.zeros(3), torch.zeros(2, dtype=torch.int32), [1, 2, 3]):
        with pytest.raises((TypeError, ValueError, _lib.CbkError)):
            ops.cache_pages(t, bad)


def test_the_oracles_tables_by_hand():
    t = R8.Tables(6, 3, 64, 16)
    assert t.resize([20, 0, 17]) == [0, 20, 20, 37] and t.table == [[0, 1, -1, -1], [-1] * 4, [2, 3, -1, -1]]
    assert t.resize([0, 33, 18]) == [0, 0, 33, 34] and t.table == [[-1] * 4, [0, 1, 4, -1], [2, 3, -1, -1]]
    assert t.count == 1 and t.free[0] == 5
    assert t.resize([40, 33, 34]) == [0, 0, 0, 0] and t.lens == [0, 33, 18]     # three, then one more: the first does not fit, nor any behind it
    assert t.resize([-1, 65, 40]) == [0, 0, 0, 22] and t.lens == [0, 33, 40]
    assert t.slots([0, 0, 2, 4], 5) == ([15 + 16, 4 * 16, 5 * 16 + 6, 5 * 16 + 7, -1], [31, 32, 38, 39, 0])
