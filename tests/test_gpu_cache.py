"""The 4-bit key/value cache on the GPU against its definition: writing, reading back, attention.

What is held is defined to the bit (float32 steps), and read back as float32 it is compared bit for bit.  Attention is
compared with the definition in float64 within the error of its 16-bit operands.  With u = 2^-11 (half a step of fp16): keys and values
are rounded once, and for bf16 so may be the queries with the scale of the scores in them, so a score is off by at most u (bf16: 2u + u^2)
times scale sum_d |q_d k_d| =: reach (float32 sums and the exponential
add less than 2^-16 for the scores here, which stay below 64), and p by another u; weights that are off by a factor 1 + e_j, |e_j| <= e,
move the normalised sum by at most e / (1 - e) sum_j p_j |v_j - o|; the rounded values by u sum_j p_j |v_j|;
the result is rounded to its type, and an fp16 one may be subnormal (2^-25)."""
import numpy as np
import pytest
import torch

from cobalt_amd import KVCache, KVRows, _lib, ops
from oracle import cache_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -11
SCORE = {torch.float16: U, torch.bfloat16: 2 * U + U * U}           # of reach
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Setup:
    """Sequences of the given lengths whose tokens are all in the cache, on pages handed out in a shuffled order."""

    def __init__(self, lens, heads, dim, page, group, dtype, seed=0, spare=2, fill=None, outliers=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.dim, self.page, self.group, self.dtype, self.g = lens, heads, dim, page, group, dtype, g
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        cols = max(need + [1]) + 1
        table = [[-1] * cols for _ in lens]
        at = 0
        for b, n in enumerate(need):
            table[b][:n] = order[at:at + n]
            at += n
        self.unused = order[at:]
        self.table = ints(table).view(len(lens), cols)
        total = sum(lens)
        chan = torch.exp(0.5 * torch.randn(heads, dim, generator=g)) if outliers else 1.0
        self.k = (torch.randn(total, heads, dim, generator=g) * chan).to(dtype)
        self.v = torch.randn(total, heads, dim, generator=g).to(dtype)
        if fill:
            fill(self)
        self.cut = np.concatenate([[0], np.cumsum(lens)]).astype(int)
        self.cache = KVCache(self.pages, heads, dim, page=page, group=group, device=DEV)
        ops.cache_write(self.cache, self.k.to(DEV), self.v.to(DEV), KVRows(self.table, ints(lens), ints(self.cut.tolist())))
        self.hk, self.hv = R.held(self.k.float().numpy(), self.v.float().numpy(), group)

    def rows(self, new):
        return KVRows(self.table, ints(self.lens), ints(np.concatenate([[0], np.cumsum(new)]).astype(int).tolist()))

    def check(self, q, out, new, scale=None, window=None, sinks=0, there=None):
        """q, out [rows, heads * ratio, dim] of the newest `new` tokens of each sequence."""
        scale = scale or self.dim ** -0.5
        ratio = q.shape[1] // self.heads
        qn, on = q.double().cpu().numpy(), out.double().cpu().numpy()
        at = 0
        for b, n in enumerate(new):
            pos = np.arange(self.lens[b] - n, self.lens[b])
            k, v = self.hk[self.cut[b]:self.cut[b + 1]], self.hv[self.cut[b]:self.cut[b + 1]]
            ok = np.ones(len(k), bool) if there is None else there[b]
            for h in range(q.shape[1]):
                o, spread, size, reach = R.attention(qn[at:at + n, h], k[:, h // ratio], v[:, h // ratio], pos, ok, scale, window, sinks)
                e = (SCORE[out.dtype] * reach + U + 2.0 ** -16)[:, None]
                tol = e / (1 - e) * spread + U * size
                tol = tol + HALF[out.dtype] * (np.abs(o) + tol) + 2.0 ** -25
                bad = ~(np.abs(on[at:at + n, h] - o) <= tol)
                assert not bad.any(), (f"sequence {b} (length {self.lens[b]}), head {h}: rows {np.flatnonzero(bad.any(1))[:8]}, "
                                       f"off by {np.abs(on[at:at + n, h] - o)[bad].max()}, allowed {tol[bad].min()}")
            at += n

    def attend(self, new, ratio, seed=1, **kw):
        q = torch.randn(sum(new), self.heads * ratio, self.dim, generator=torch.Generator().manual_seed(seed)).to(self.dtype).to(DEV)
        out = ops.cache_attention(self.cache, q, self.rows(new), **kw)
        self.check(q, out, new, **kw)
        return q, out


# ------------------------------------------------------------------ writing and reading back
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group,page,heads", [(64, 32, 16, 2), (64, 64, 64, 1), (128, 32, 16, 3), (128, 64, 256, 8), (128, 128, 32, 5),
                                                  (256, 32, 64, 1), (256, 64, 128, 4), (256, 128, 16, 2)])
def test_written_tokens_read_back_as_defined(dim, group, page, heads, dtype):
    lens = [1, 0, 17, 300, 15, 64]
    s = Setup(lens, heads, dim, page, group, dtype, seed=dim + group + page)
    rows = s.rows(lens)
    for t in (torch.float32, torch.float16, torch.bfloat16):
        k, v = ops.cache_read(s.cache, rows, sum(lens), t)
        assert torch.equal(k.cpu(), torch.from_numpy(s.hk).float().to(t))
        assert torch.equal(v.cpu(), torch.from_numpy(s.hv).float().to(t))
    # the newest tokens alone; rows behind the last sequence and in front of the first stay as they were
    new = [1, 0, 5, 33, 15, 2]
    starts = ints((np.concatenate([[0], np.cumsum(new)]) + 2).tolist())
    n = sum(new)
    k, v = (torch.full((n + 5, heads, dim), 7.0, device=DEV) for _ in range(2))
    ops.cache_read(s.cache, KVRows(s.table, ints(lens), starts), n + 5, torch.float32, out=(k, v))
    want = np.concatenate([np.arange(s.cut[b + 1] - m, s.cut[b + 1]) for b, m in enumerate(new)])
    assert torch.equal(k[2:2 + n].cpu(), torch.from_numpy(s.hk[want]).float())
    assert torch.equal(v[2:2 + n].cpu(), torch.from_numpy(s.hv[want]).float())
    for x in (k, v):
        assert bool((x[:2] == 7).all()) and bool((x[2 + n:] == 7).all())


def test_equal_numbers_of_rows_need_no_offsets():
    s = Setup([40, 9, 16, 100], 2, 128, 16, 32, torch.float16)
    a = ops.cache_read(s.cache, KVRows(s.table, ints(s.lens)), 12, torch.float32)
    b = ops.cache_read(s.cache, s.rows([3] * 4), 12, torch.float32)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q = torch.randn(12, 4, 128, device=DEV).half()
    assert torch.equal(ops.cache_attention(s.cache, q, KVRows(s.table, ints(s.lens))), ops.cache_attention(s.cache, q, s.rows([3] * 4)))


def test_values_at_the_ends_of_the_range():
    def fill(s):
        k, v = s.k, s.v
        k[0, 0] = 3.0                                               # constant groups: no step
        k[1, 0] = 0.0
        k[2, 0] = 1e30                                              # beyond what is held
        k[3, 0, ::2] = -3e38
        k[4, 0] = torch.linspace(0, 1, 128) * 1e-6                  # a step below fp16's normal numbers
        k[5, 0] = torch.linspace(0, 1, 128) * 1e-9                  # and below all of them
        k[6, 0] = 40000.0 + 8 * torch.arange(128)
        v[7, 0, 5] = float("inf")
        v[8, 0, 5] = float("-inf")
        k[9, 1, 77] = float("nan")                                  # the token's key and value of this head are NaN
        v[10, 0, 0] = float("nan")
        v[11, 0] = torch.arange(128) % 16                           # codes themselves
    s = Setup([20], 2, 128, 16, 32, torch.bfloat16, fill=fill)
    k, v = ops.cache_read(s.cache, s.rows([20]), 20, torch.float32)
    for got, want in ((k, s.hk), (v, s.hv)):
        np.testing.assert_array_equal(got.cpu().numpy(), want.astype(np.float32))
    assert bool(k[9, 1].isnan().all()) and bool(v[9, 1].isnan().all()) and not bool(k[9, 0].isnan().any())
    assert bool(torch.isfinite(k[2:9]).all()) and bool(torch.isfinite(v[2:9]).all())
    assert torch.equal(v[11, 0].cpu(), s.v[11, 0].float())
    for t in (torch.float16, torch.bfloat16):
        k16, _ = ops.cache_read(s.cache, s.rows([20]), 20, t)
        np.testing.assert_array_equal(k16.float().cpu().numpy(), torch.from_numpy(s.hk).float().to(t).float().numpy())


def test_scales_and_values_at_the_borders_of_rounding():
    """Ranges whose fifteenth lies exactly between two fp16 numbers, or a float32 step beside, and values between two codes."""
    g = torch.Generator().manual_seed(1)
    n = 20000
    lo = -torch.randint(1, 1 << 11, (n, 1, 1), generator=g) * 2.0 ** -5
    step = torch.randint(1 << 11, 1 << 12, (n, 1, 1), generator=g) * 2.0 ** -12     # 12 bits: every second one a tie

    def fill(s):
        s.k[:] = (lo + 15 * step * torch.rand(n, 1, 64, generator=g)).half()
        s.k[:, :, 0:1], s.k[:, :, 63:] = lo.half(), (lo + 15 * step).half()
        s.v[:] = (lo + step * (torch.randint(0, 31, (n, 1, 64), generator=g) / 2)).half()
        s.v[:, :, 0:1], s.v[:, :, 63:] = lo.half(), (lo + 15 * step).half()
    s = Setup([n], 1, 64, 256, 64, torch.float16, fill=fill)
    for t in (torch.float32, torch.float16):
        k, v = ops.cache_read(s.cache, s.rows([n]), n, t)
        assert torch.equal(k.cpu(), torch.from_numpy(s.hk).float().to(t))
        assert torch.equal(v.cpu(), torch.from_numpy(s.hv).float().to(t))


def test_a_write_touches_its_own_tokens_only():
    s = Setup([37, 20], 3, 128, 16, 64, torch.float16, spare=3)
    n = [2, 1]
    k, v = (torch.randn(3, 3, 128, device=DEV).half() for _ in range(2))
    ops.cache_write(s.cache, k, v, s.rows(n))
    a, b = ops.cache_read(s.cache, s.rows(s.lens), 57, torch.float32)
    hk, hv = R.held(k.float().cpu().numpy(), v.float().cpu().numpy(), 64)
    s.hk[[35, 36, 56]], s.hv[[35, 36, 56]] = hk, hv
    assert torch.equal(a.cpu(), torch.from_numpy(s.hk).float()) and torch.equal(b.cpu(), torch.from_numpy(s.hv).float())
    # no page, a page number outside the pool, a position behind the table: nothing is written and reads are 0
    ops.cache_write(s.cache, k[:2], v[:2], s.rows(n)._replace(starts=ints([0, 1, 2])))
    after = [t.clone() for t in s.cache.native()[:4]]
    for bad in (-1, s.pages, 1 << 30, -(1 << 31)):
        table = torch.full_like(s.table, bad)
        ops.cache_write(s.cache, k, v, s.rows(n)._replace(table=table))
        got = ops.cache_read(s.cache, s.rows(n)._replace(table=table), 3, torch.float32)
        assert not bool(got[0].any()) and not bool(got[1].any())
    for lens in ([1 << 30, (1 << 31) - 1], [0, 0], [-5, -(1 << 31)]):
        ops.cache_write(s.cache, k, v, s.rows(n)._replace(lens=ints(lens)))
    for x, y in zip(s.cache.native()[:4], after):
        assert torch.equal(x, y)


def test_strided_and_unaligned_inputs():
    s = Setup([50, 30], 2, 128, 32, 32, torch.float16, seed=4)
    n, rows = 10, KVRows(s.table, ints(s.lens))
    fused = torch.randn(n, 2 * 4 * 128 + 8, device=DEV).half()      # q | k | v of one projection, with a tail
    k = fused[:, 512:768].view(n, 2, 128)
    v = fused[:, 768:1024].view(n, 2, 128)
    ops.cache_write(s.cache, k, v, rows)
    a = ops.cache_read(s.cache, rows, n, torch.float32)
    hk, hv = R.held(k.float().cpu().numpy(), v.float().cpu().numpy(), 32)
    assert torch.equal(a[0].cpu(), torch.from_numpy(hk).float()) and torch.equal(a[1].cpu(), torch.from_numpy(hv).float())
    for make in (lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),              # heads outside
                 lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),              # channels not contiguous
                 lambda x: torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape)):   # 2 bytes off
        s.cache.k_codes.zero_()
        ops.cache_write(s.cache, make(k.contiguous()), make(v.contiguous()), rows)
        b = ops.cache_read(s.cache, rows, n, torch.float32)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    out = tuple(torch.zeros(2, n, 128, device=DEV).transpose(0, 1) for _ in range(2))
    ops.cache_read(s.cache, rows, n, torch.float32, out=out)
    assert torch.equal(out[0], a[0]) and torch.equal(out[1], a[1])
    one = k[:1].expand(n, 2, 128)                                   # the same keys n times: a row stride of 0
    ops.cache_write(s.cache, one, one, rows)
    b = ops.cache_read(s.cache, rows, n, torch.float32)
    assert torch.equal(b[0][0], b[0][-1]) and torch.equal(b[0], b[1])
    many = torch.randn(n, 3, 128, device=DEV).half()[:, 1:]         # rows further apart than they are long
    ops.cache_write(s.cache, many, many, rows)
    s2 = R.held(many.float().cpu().numpy(), many.float().cpu().numpy(), 32)
    assert torch.equal(ops.cache_read(s.cache, rows, n, torch.float32)[0].cpu(), torch.from_numpy(s2[0]).float())


# ------------------------------------------------------------------ attention
LENS = [1, 2, 15, 16, 17, 33, 127, 128, 129, 300, 513]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group,page,heads,ratio", [(64, 32, 16, 2, 4), (64, 64, 32, 1, 1), (128, 32, 64, 2, 4), (128, 64, 16, 1, 8),
                                                        (128, 128, 256, 3, 1), (128, 32, 32, 1, 16), (256, 64, 16, 1, 4), (256, 32, 128, 2, 2),
                                                        (256, 128, 64, 1, 3), (128, 32, 16, 1, 20)])
def test_one_token_of_each_sequence(dim, group, page, heads, ratio, dtype):
    s = Setup(LENS, heads, dim, page, group, dtype, seed=dim + group)
    s.attend([1] * len(LENS), ratio)


@pytest.mark.parametrize("dim,ratio", [(64, 3), (128, 4), (256, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (128, 130), (129, 4), (200, 1), (10 ** 9, 3), (2 ** 31 - 1, 0)])
def test_windows_and_sinks(dim, ratio, window, sinks):
    s = Setup(LENS, 2, dim, 16, 32, torch.float16, seed=window % 97)
    s.attend([1] * len(LENS), ratio, window=window, sinks=sinks)
    s.attend([min(n, 9) for n in LENS], ratio, window=window, sinks=sinks)


@pytest.mark.parametrize("dim,ratio,dtype", [(64, 4, torch.bfloat16), (128, 4, torch.float16), (128, 1, torch.bfloat16), (256, 8, torch.float16)])
def test_several_tokens_of_each_sequence(dim, ratio, dtype):
    s = Setup(LENS, 1, dim, 32, 64, dtype, seed=3)
    s.attend([min(n, 1 + i) for i, n in enumerate(LENS)], ratio)
    s.attend([0, 2, 0, 0, 17, 3, 0, 1, 0, 0, 0], ratio)


@pytest.mark.parametrize("dim,ratio,dtype,window,sinks", [(64, 2, torch.float16, None, 0), (128, 4, torch.bfloat16, None, 0),
                                                          (128, 3, torch.float16, 50, 4), (256, 2, torch.bfloat16, None, 0), (256, 1, torch.float16, 140, 0)])
def test_whole_prompts(dim, ratio, dtype, window, sinks):
    s = Setup([1, 130, 0, 257, 64, 400], 2, dim, 16, 32, dtype, seed=8)
    s.attend(s.lens, ratio, window=window, sinks=sinks)
    s.attend([0, 70, 0, 200, 1, 399], ratio, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group,page", [(64, 32, 16), (64, 64, 64), (128, 32, 16), (128, 64, 32), (128, 128, 256), (256, 32, 16), (256, 64, 64), (256, 128, 32)])
def test_prompts_of_every_format(dim, group, page, dtype):
    s = Setup([1, 75, 0, 300, 64], 2, dim, page, group, dtype, seed=dim * group)
    s.attend(s.lens, 3)
    s.attend([0, 40, 0, 130, 64], 2, window=48, sinks=5)


@pytest.mark.parametrize("dim,group,dtype", [(64, 64, torch.float16), (128, 32, torch.bfloat16), (256, 64, torch.float16)])
def test_many_prompts(dim, group, dtype):
    """More tiles of rows than the chip holds workgroups: one workgroup each."""
    g = np.random.default_rng(1)
    s = Setup([int(x) for x in g.integers(0, 70, 1100)], 1, dim, 16, group, dtype, seed=16)
    s.attend(s.lens, 1)


@pytest.mark.parametrize("dim,dtype", [(64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16), (256, torch.float16)])
def test_chunks_behind_long_histories_are_cut_and_joined(dim, dtype):
    s = Setup([7000, 40, 2600], 1, dim, 32, 32, dtype, seed=15)
    s.attend([60, 40, 33], 4)
    s.attend([70, 1, 100], 2, window=1500, sinks=100)


@pytest.mark.parametrize("lens,heads,ratio", [([20011], 1, 4), ([9000, 3, 12345], 2, 2), ([4097], 8, 4)])
def test_long_histories_are_cut_and_joined(lens, heads, ratio):
    s = Setup(lens, heads, 128, 64, 32, torch.bfloat16, seed=5)
    _, a = s.attend([1] * len(lens), ratio)
    s.attend([1] * len(lens), ratio, window=5000, sinks=200)
    s.attend([min(n, 3) for n in lens], ratio)


def test_many_sequences():
    """More sequences than a workgroup has threads, most of them short, some empty."""
    g = np.random.default_rng(0)
    lens = [int(x) for x in g.integers(0, 40, 700)]
    lens[300] = 1500
    s = Setup(lens, 1, 64, 16, 32, torch.float16, seed=6)
    s.attend([min(n, 1) for n in lens], 2)
    k, v = ops.cache_read(s.cache, s.rows([min(n, 2) for n in lens]), sum(min(n, 2) for n in lens), torch.float32)
    want = np.concatenate([np.arange(s.cut[b + 1] - min(n, 2), s.cut[b + 1]) for b, n in enumerate(lens)]).astype(int)
    assert torch.equal(k.cpu(), torch.from_numpy(s.hk[want]).float())


def test_rows_that_see_nothing_are_zero():
    s = Setup([100, 40, 30], 2, 128, 16, 32, torch.float16)
    q = torch.randn(5, 4, 128, device=DEV).half()
    out = ops.cache_attention(s.cache, q, KVRows(torch.full_like(s.table, -1), ints(s.lens), ints([0, 1, 3, 5])))
    assert not bool(out.any())
    out = ops.cache_attention(s.cache, q, KVRows(s.table, ints([0, 0, 0]), ints([0, 1, 3, 5])))
    assert not bool(out.any())
    out = ops.cache_attention(s.cache, q, KVRows(s.table[:, :0], ints(s.lens), ints([0, 1, 3, 5])))
    assert not bool(out.any())
    # more rows than tokens: those in front of the sequence see nothing, the others what they should
    out = ops.cache_attention(s.cache, q, KVRows(s.table[:1], ints([2]), ints([0, 5])))
    assert not bool(out[:3].any()) and bool((out[3:] != 0).any(-1).all())
    s.lens, s.cut = [2], np.array([0, 2])
    s.check(q[3:], out[3:], [2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,seqs", [(4096, 1), (70, 1), (3000, 3), (4096, 20)])
def test_rows_of_no_sequence_at_all(rows, seqs, dtype):
    """Every sequence of the call is without rows, however many the call has, in front of them, behind them or between none."""
    s = Setup([2000] * seqs, 2, 128, 64, 32, dtype, seed=3)
    q = torch.randn(rows, 8, 128, device=DEV).to(dtype)
    for at in (0, 1000, rows):
        out = torch.full_like(q, 9)
        ops.cache_attention(s.cache, q, KVRows(s.table, ints(s.lens), ints([at] * (seqs + 1))), out=out)
        assert bool((out == 9).all())
    starts = [0] * (seqs + 1)
    starts[-1] = 5                                                  # and with five rows of the last one
    out = torch.full_like(q, 9)
    ops.cache_attention(s.cache, q, KVRows(s.table, ints(s.lens), ints(starts)), out=out)
    assert bool((out[5:] == 9).all())
    s.check(q[:5], out[:5], [0] * (seqs - 1) + [5])


def test_missing_pages_are_not_seen():
    s = Setup([200, 90], 1, 128, 16, 32, torch.bfloat16, seed=2)
    there = [np.ones(200, bool), np.ones(90, bool)]
    table = s.table.clone()
    for b, i in ((0, 0), (0, 5), (0, 12), (1, 2), (1, 5)):          # first, inner and last pages
        table[b, i] = -1 if i % 2 else s.pages + 3
        there[b][16 * i:16 * i + 16] = False
    q = torch.randn(6, 4, 128, device=DEV).bfloat16()
    out = ops.cache_attention(s.cache, q, KVRows(table, ints(s.lens), ints([0, 4, 6])))
    s.check(q, out, [4, 2], there=there)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_nan_reaches_the_rows_that_see_it_only(dim):
    def fill(s):
        s.v[70, 0, 3] = float("nan")
        s.k[100, 0, 3] = float("nan")
    s = Setup([128], 1, dim, 16, 32, torch.float16, fill=fill)
    q = torch.randn(128, 2, dim, device=DEV).half()
    out = ops.cache_attention(s.cache, q, s.rows([128]))
    nan = out.isnan()
    assert not bool(nan[:70].any()) and bool(nan[70:].all())
    out = ops.cache_attention(s.cache, q, s.rows([128]), window=20)
    assert set(torch.nonzero(out.isnan().any(-1).any(-1)).view(-1).tolist()) == set(range(70, 90)) | set(range(100, 120))
    # a NaN or an infinity in a query stays in its row
    q[5, 1, 7], q[6, 0, 0] = float("nan"), float("inf")
    out = ops.cache_attention(s.cache, q[:40], s.rows([128])._replace(lens=ints([40]), starts=ints([0, 40])))
    nan = out.isnan().any(-1)
    assert bool(nan[5, 1]) and bool(nan[6, 0]) and int(nan.sum()) == 2


def test_what_stands_behind_the_last_token_does_not_matter():
    s = Setup([37, 100], 2, 128, 64, 32, torch.float16, seed=9)
    q = torch.randn(4, 4, 128, device=DEV).half()
    rows = KVRows(s.table, ints(s.lens), ints([0, 3, 4]))
    a = ops.cache_attention(s.cache, q, rows)
    junk = KVRows(s.table, ints([64, 128]), ints([0, 27, 55]))      # the rest of the last pages: NaN and large values
    x = torch.full((55, 2, 128), 6e4, device=DEV).half()
    x[::2] = float("nan")
    ops.cache_write(s.cache, x, x, junk)
    assert torch.equal(a, ops.cache_attention(s.cache, q, rows))
    # bits that no write leaves there
    m = s.cache.v_meta.view(torch.int32).view(s.pages, 2, 4, 64)
    p = int(s.table[0, 0])
    m[p, :, :, 37:] = -1
    assert torch.equal(a, ops.cache_attention(s.cache, q, rows))


def test_large_and_small_queries():
    s = Setup([300], 1, 128, 32, 32, torch.bfloat16, outliers=False)
    q = torch.randn(4, 2, 128, device=DEV)
    q[0] *= 2.0 ** 100
    q[1] *= 2.0 ** -100
    q[2] = 0
    q = q.bfloat16()
    out = ops.cache_attention(s.cache, q, s.rows([4]))
    s.check(q[1:], out[1:], [3])                                    # (weights all but equal)
    top = (s.hk[:297, 0] @ q[0].double().cpu().numpy().T).argmax(0)  # one token takes all
    for h in range(2):
        np.testing.assert_allclose(out[0, h].double().cpu().numpy(), s.hv[top[h], 0], rtol=2.0 ** -8 + 2.0 ** -11, atol=1e-30)
    for scale in (1e-4, 0.5):
        out = ops.cache_attention(s.cache, q[2:], s.rows([2]), scale=scale)
        s.check(q[2:], out, [2], scale=scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [4, 64])
def test_rows_of_all_sizes_side_by_side(n, dtype):
    """Rows from the smallest to the largest numbers of their type, in one product with ordinary ones; scales from 1e-6 to 30."""
    s = Setup([300], 1, 128, 32, 32, dtype, outliers=False, seed=3)
    g = torch.Generator().manual_seed(5)
    base = torch.randn(n, 2, 128, generator=g)
    low, high = (-22, 13) if dtype == torch.float16 else (-120, 60)
    size = torch.linspace(low, high, 2 * n).view(2, n).t().round()
    q = (base * 2.0 ** size[..., None]).to(dtype).to(DEV)
    out = ops.cache_attention(s.cache, q, s.rows([n]))
    small = (size.amax(1) < 2).to(DEV)                              # (scores below 64, as the bound wants them)
    qd = q.double().cpu().numpy()
    for i in range(n):
        pos = 300 - n + i
        for h in range(2):
            sc = s.hk[:pos + 1, 0] @ qd[i, h] * 128 ** -0.5
            if np.abs(sc).max() < 40:
                o, spread, sz, reach = R.attention(qd[i:i + 1, h], s.hk[:, 0], s.hv[:, 0], np.array([pos]), np.ones(300, bool), 128 ** -0.5)
                e = SCORE[dtype] * reach[0] + U + 2.0 ** -16
                tol = e / (1 - e) * spread + U * sz
                tol = tol + HALF[dtype] * (np.abs(o) + tol) + 2.0 ** -25
                assert (np.abs(out[i, h].double().cpu().numpy() - o[0]) <= tol[0]).all(), (i, h)
            # one token takes all, by 200 more than two scores can be off, each by its share of the largest sum of magnitudes
            elif np.sort(sc)[-1] - np.sort(sc)[-2] > 200 + 2 * SCORE[dtype] * (np.abs(s.hk[:pos + 1, 0]) @ np.abs(qd[i, h])).max() * 128 ** -0.5:
                want = s.hv[sc.argmax(), 0]
                assert (np.abs(out[i, h].double().cpu().numpy() - want) <= (HALF[dtype] + U + 2.0 ** -16) * np.abs(want) + 1e-6).all(), (i, h)
            else:
                assert bool(torch.isfinite(out[i, h]).all())
    assert bool(small.any())
    ones = torch.full((n, 2, 128), 2.0 ** 13, device=DEV).to(dtype)    # all of one sign: their sum leaves fp16's range
    out = ops.cache_attention(s.cache, ones, s.rows([n]))
    assert bool(torch.isfinite(out).all())
    for scale in (1e-6, 0.02, 3.0, 30.0):
        q = (torch.randn(n, 2, 128, generator=g) * min(1.0, 0.05 / scale)).to(dtype).to(DEV)
        s.check(q, ops.cache_attention(s.cache, q, s.rows([n]), scale=scale), [n], scale=scale)


@pytest.mark.parametrize("large", [300.0, 4096.0, 60000.0])
@pytest.mark.parametrize("dim,n,heads", [(64, 4, 2), (128, 4, 2), (256, 4, 2), (64, 700, 8), (128, 700, 8), (256, 700, 8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_large_channel_leaves_the_small_ones(dtype, dim, n, heads, large):
    """One channel of the queries thousands of times the others, over a group of keys that are 0: the scores are the others' alone.  Rows that pass 2^8 leave
    [2^7, 2^8) and are held with steps of 2^-24, so that each element is off by 2^-25 max(1, large / 2^7) at most; bf16 ones may have the scale in them."""
    def fill(s):
        s.k *= 4
        s.k[..., :32] = 0
    s = Setup([700], heads, dim, 64, 32, dtype, outliers=False, seed=11, fill=fill)
    q = 0.05 * torch.randn(n, 2 * heads, dim, generator=torch.Generator().manual_seed(12))
    q[..., 5] = large
    q = q.to(dtype)
    out = ops.cache_attention(s.cache, q.to(DEV), s.rows([n]))
    scale, qn, on = dim ** -0.5, q.double().numpy(), out.double().cpu().numpy()
    for h in range(0, 2 * heads, 2 * heads - 1):
        k = s.hk[:, h // 2]
        o, spread, size, reach = R.attention(qn[:, h], k, s.hv[:, h // 2], np.arange(700 - n, 700), np.ones(700, bool), scale)
        e = (SCORE[dtype] * reach + U + 2.0 ** -16)[:, None] + 2.0 ** -25 * max(1.0, large / 2 ** 7 * scale) * np.abs(k).sum(1).max()
        tol = e / (1 - e) * spread + U * size
        tol = tol + HALF[dtype] * (np.abs(o) + tol) + 2.0 ** -25
        assert (np.abs(on[:, h] - o) <= tol).all(), (h, (np.abs(on[:, h] - o) / tol).max())


def test_one_token_outweighs_a_long_history():
    """Weights 2^-20 of the largest, 30000 of them: 3 % of the sum, in p that fp16 could not tell from 0 as it is."""
    def fill(s):
        s.k[:, 0] = 0
        s.k[777, 0, 0] = 20 * np.log(2) / 128 ** -0.5 / 8
        s.v[:, 0] = 1.0
        s.v[777, 0] = 0.0
    s = Setup([30001], 1, 128, 64, 32, torch.float16, fill=fill)
    q = torch.zeros(1, 1, 128, device=DEV).half()
    q[0, 0, 0] = 8
    s.check(q, ops.cache_attention(s.cache, q, s.rows([1])), [1])


def test_strides_and_rows_behind_the_last_sequence():
    s = Setup([50, 30], 2, 128, 32, 32, torch.float16, seed=4)
    rows = KVRows(s.table, ints(s.lens), ints([0, 3, 5]))
    fused = torch.randn(8, 6 * 128 + 8, device=DEV).half()
    q = fused[:, :512].view(8, 4, 128)
    want = ops.cache_attention(s.cache, q[:5].contiguous(), rows)
    s.check(q[:5], want, [3, 2])
    out = torch.full((4, 8, 128), 9.0, device=DEV).half().transpose(0, 1)
    assert ops.cache_attention(s.cache, q, rows, out=out) is out
    assert torch.equal(out[:5], want) and bool((out[5:] == 9).all())
    off = torch.cat([q.new_zeros(1), q[:5].reshape(-1)])[1:].view(5, 4, 128)
    assert torch.equal(ops.cache_attention(s.cache, off, rows), want)
    assert ops.cache_attention(s.cache, q[:0], rows._replace(starts=ints([0, 0, 0]))).shape == (0, 4, 128)
    empty = KVRows(s.table[:0], ints([]), ints([0]))
    assert ops.cache_attention(s.cache, q[:0], empty).shape == (0, 4, 128)
    out.fill_(9.0)
    ops.cache_attention(s.cache, q, empty, out=out)                 # rows of no sequence
    assert bool((out == 9).all())


def test_calls_repeat_bit_for_bit():
    s = Setup([5000, 700, 1], 2, 128, 64, 32, torch.bfloat16, seed=11)
    q, a = s.attend([1, 1, 1], 4)
    for _ in range(3):
        torch.empty(64 << 20, dtype=torch.uint8, device=DEV).fill_(255)   # what the workspace comes back as
        assert torch.equal(a, ops.cache_attention(s.cache, q, s.rows([1, 1, 1])))


def test_a_table_of_more_than_four_gigabytes():
    heads, dim, page = 4, 256, 256
    pages = (1 << 32) // (heads * page * dim // 2) + 9
    s = Setup([700, 513], heads, dim, page, 128, torch.float16, spare=0)
    cache = KVCache(pages, heads, dim, page=page, group=128, device=DEV)
    table = s.table.clone()
    table[table >= 0] += pages - s.pages
    ops.cache_write(cache, s.k.to(DEV), s.v.to(DEV), KVRows(table, ints(s.lens), ints(s.cut.tolist())))
    k, v = ops.cache_read(cache, KVRows(table, ints(s.lens), ints(s.cut.tolist())), 1213, torch.float32)
    assert torch.equal(k.cpu(), torch.from_numpy(s.hk).float()) and torch.equal(v.cpu(), torch.from_numpy(s.hv).float())
    q = torch.randn(2, 8, dim, device=DEV).half()
    out = ops.cache_attention(cache, q, KVRows(table, ints(s.lens)))
    s.check(q, out, [1, 1])
    assert not bool(cache.k_codes[:1 << 20].any())                  # (a wrapped offset would have landed there)


# ------------------------------------------------------------------ as a program uses them
def test_steps_in_a_graph_follow_the_lengths():
    """A recorded step (write, then attend) replayed over growing sequences, each against the eager calls."""
    s = Setup([130, 60], 2, 128, 16, 32, torch.float16, seed=12)
    lens, table = ints(s.lens), torch.full((2, 12), -1, dtype=torch.int32, device=DEV)
    table[:, :s.table.shape[1]] = s.table
    table[0, 9], table[1, 4] = s.unused[0], s.unused[1]
    rows = KVRows(table, lens)
    k, v, q = (torch.zeros(2, h, 128, device=DEV).half() for h in (2, 2, 8))

    def step():
        ops.cache_write(s.cache, k, v, rows)
        return ops.cache_attention(s.cache, q, rows, window=100, sinks=3)

    def inputs(i):
        g = torch.Generator(device=DEV).manual_seed(i)
        lens.add_(1)
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    start = lens.clone()
    with torch.cuda.stream(side):
        inputs(0)
        step()
        lens.copy_(start)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    arrays = s.cache.native()[:4]
    for i in range(6):
        keep = [t.clone() for t in arrays]
        inputs(i)
        graph.replay()
        torch.cuda.synchronize()
        got, held = out.clone(), [t.clone() for t in arrays]
        for t, x in zip(arrays, keep):
            t.copy_(x)
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        for t, x in zip(arrays, held):
            assert torch.equal(t, x)


def test_two_graphs_of_one_memory_pool():
    """Their workspaces are the same memory: replayed in turn, with eager calls between, both answer as eager calls do."""
    s = Setup([5000, 2600], 4, 128, 64, 32, torch.float16, seed=21)
    calls = []
    for new, window in (([1, 1], None), ([700, 500], None), ([3, 2], 300)):
        q = torch.randn(sum(new), 16, 128, device=DEV).half()
        rows = s.rows(new)
        calls.append((q, rows, window, ops.cache_attention(s.cache, q, rows, window=window)))
        if sum(new) < 10:
            s.check(q, calls[-1][3], new, window=window)
    torch.cuda.synchronize()
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for q, rows, window, want in calls:
        out, graph = torch.zeros_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            ops.cache_attention(s.cache, q, rows, window=window, out=out)
        graphs.append((graph, out, want))
    for i in range(4):
        for graph, out, want in graphs if i % 2 else graphs[::-1]:
            out.fill_(5)
            graph.replay()
            torch.empty(16 << 20, dtype=torch.uint8, device=DEV).fill_(255)
            assert torch.equal(out, want)
        q, rows, window, want = calls[i % 3]
        assert torch.equal(ops.cache_attention(s.cache, q, rows, window=window), want)


def test_two_streams_at_once():
    a, b = (Setup([3000, 200], 2, 128, 64, 32, torch.float16, seed=i) for i in (20, 21))
    q = [torch.randn(2, 8, 128, device=DEV).half() for _ in range(2)]
    want = [ops.cache_attention(s.cache, x, s.rows([1, 1])) for s, x in zip((a, b), q)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.cache_attention(s.cache, q[i], s.rows([1, 1])))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x, want[i])


def test_operators_refuse_what_does_not_fit():
    s = Setup([20, 30], 2, 128, 16, 32, torch.float16)
    r = s.rows([1, 1])
    q, k = torch.zeros(2, 4, 128, device=DEV).half(), torch.zeros(2, 2, 128, device=DEV).half()
    att, wr, rd = ops.cache_attention, ops.cache_write, ops.cache_read
    with pytest.raises(_lib.CbkError):
        att(s.cache, q.cpu(), r)
    with pytest.raises(_lib.CbkError):
        att(s.cache, q, r._replace(lens=r.lens.cpu()))
    with pytest.raises(_lib.CbkError):
        wr(s.cache, k, k.cpu(), r)
    with pytest.raises(TypeError):
        att(s.cache, q.float(), r)
    with pytest.raises(TypeError):
        att(s.cache, q, r._replace(lens=r.lens.long()))
    for bad in (q[:, :3], q[..., :64], q[0], q.view(2, 1, 512)):
        with pytest.raises(ValueError):
            att(s.cache, bad, r)
    for kw in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            att(s.cache, q, r, **kw)
    for rows in (r._replace(starts=r.starts[:2]), r._replace(table=r.table[:1]), r._replace(table=r.table[0]), r._replace(table=r.table.t().contiguous().t())):
        with pytest.raises(ValueError):
            att(s.cache, q, rows)
    with pytest.raises(ValueError):
        att(s.cache, q.new_zeros(3, 4, 128), KVRows(r.table, r.lens))
    for out in (torch.zeros(2, 4, 128, device=DEV), q.new_zeros(3, 4, 128), q.new_zeros(1, 4, 128).expand(2, 4, 128),
                q.new_zeros(2, 1, 128).expand(2, 4, 128), q.new_zeros(2, 4, 132)[..., :128], q.new_zeros(2, 4, 256)[..., ::2]):
        with pytest.raises(ValueError):
            att(s.cache, q, r, out=out)
    for a, b in ((k, k.bfloat16()), (k, k[:1]), (k.float(), k.float()), (k[:, :1], k)):
        with pytest.raises(ValueError):
            wr(s.cache, a, b, r)
    with pytest.raises(ValueError):
        rd(s.cache, r, -1)
    with pytest.raises(TypeError):
        rd(s.cache, r, 2, torch.int8)
    with pytest.raises(ValueError):
        rd(s.cache, r, 2, torch.float16, out=(k, k[:1]))


def test_operators_refuse_outputs_that_are_inputs():
    s = Setup([20, 30], 2, 128, 16, 32, torch.float16)
    r = s.rows([1, 1])
    q, k = torch.zeros(2, 4, 128, device=DEV).half(), torch.zeros(2, 2, 128, device=DEV).half()
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_attention(s.cache, q, r, out=q)
    with pytest.raises(ValueError, match="output each"):
        ops.cache_read(s.cache, r, 2, torch.float16, out=(k, k))
    s.cache.v_meta = s.cache.v_meta.cpu()
    with pytest.raises(ValueError, match="one device"):
        ops.cache_write(s.cache, k, k, r)


@pytest.mark.parametrize("dim,ratio,dtype", [(64, 256, torch.float16), (128, 100, torch.bfloat16), (128, 256, torch.float16)])
def test_many_query_heads_on_one(dim, ratio, dtype):
    Setup([700, 30], 1, dim, 32, 32, dtype, seed=ratio).attend([3, 30], ratio)
    Setup([5000], 2, dim, 32, 64, dtype, seed=ratio).attend([9], ratio, window=300, sinks=3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 300])
def test_the_smallest_and_largest_scales(n, dtype):
    """Scores of nothing: the mean.  Scores of 2^20 and more: the tokens of the largest alone, since keys of one value a token are held
    and multiplied exactly, equal ones alike, and the others lie 2^21 lower: the error is that of the rounded values and result."""
    s = Setup([700], 2, 128, 64, 32, dtype, seed=n, fill=lambda s: s.k.copy_((torch.arange(700) % 128 / 16).to(dtype)[:, None, None].expand_as(s.k)))
    q = torch.ones(n, 4, 128, device=DEV).to(dtype)
    s.check(q, ops.cache_attention(s.cache, q, s.rows([n]), scale=1e-30), [n], scale=1e-30)
    out = ops.cache_attention(s.cache, q, s.rows([n]), scale=2.0 ** 20).double().cpu().numpy()
    for h in range(4):
        o, _, size, _ = R.attention(q[:, h].double().cpu().numpy(), s.hk[:, h // 2], s.hv[:, h // 2], np.arange(700 - n, 700), np.ones(700, bool), 2.0 ** 20)
        tol = (U + 2.0 ** -16) * size
        tol = tol + HALF[dtype] * (np.abs(o) + tol) + 2.0 ** -25
        assert (np.abs(out[:, h] - o) <= tol).all()


@pytest.mark.parametrize("seed,large", [(i, False) for i in range(12)] + [(i, True) for i in range(13, 18)])
def test_calls_of_all_kinds(seed, large):
    """Drawn calls: sequences without tokens or rows, more rows than tokens, tables that end before the sequence does or name pages that are
    not there, rows in front of the first sequence and behind the last, windows, sinks, strides, both kernels."""
    g = torch.Generator().manual_seed(1000 + seed)
    draw = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    pick = lambda *x: x[draw(0, len(x) - 1)]
    dim, dtype, page, heads, ratio = pick(64, 128, 256), pick(torch.float16, torch.bfloat16), pick(16, 32, 64, 256), draw(1, 3), pick(1, 2, 3, 4, 7)
    group = pick(32, 64, 128) if dim > 64 else pick(32, 64)
    seqs = draw(1, 70) if seed % 4 == 0 else draw(1, 5)
    lens = [draw(0, 40) if seqs > 5 or draw(0, 3) == 0 else draw(100, 2500) for _ in range(seqs)]
    s = Setup(lens, heads, dim, page, group, dtype, seed=seed)
    most = pick(3, 70, 700)
    new = [draw(0, min(n + 5, most)) for n in lens]
    if large:                                                       # enough rows and heads for the kernel of many rows
        heads, ratio, lens = 4, pick(4, 5), [draw(1000, 1600) for _ in range(2)] + [draw(0, 60), draw(1000, 2500)]
        s = Setup(lens, heads, dim, page, group, dtype, seed=seed)
        new = [draw(400, 600), draw(400, 1005), draw(0, 60), draw(400, 600)]
    table = s.table.cpu()
    cols = draw(max(1, table.shape[1] // 2), table.shape[1])
    there = []
    for b, n in enumerate(lens):
        for i in range(table.shape[1]):
            if draw(0, 9) == 0:
                table[b, i] = pick(-1, -7, s.pages, 2 ** 31 - 1)
        pages = torch.where((table[b] >= 0) & (table[b] < s.pages), 1, 0).bool()
        pages[cols:] = False
        there.append(pages.repeat_interleave(page)[:n].numpy())
    front, behind = draw(0, 3), draw(0, 3)
    starts = ints((np.concatenate([[0], np.cumsum(new)]) + front).tolist())
    wide = torch.full((table.shape[0], table.shape[1] + 2), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    rows = KVRows(wide.to(DEV)[:, :cols], ints(lens), starts)
    window, sinks = pick((None, 0), (None, 0), (1, 0), (17, 3), (200, 40), (1000, 0))
    total = sum(new)
    q = torch.randn(total + front + behind, heads * ratio, dim, generator=g).to(dtype).to(DEV)
    out = torch.full((heads * ratio, total + front + behind, dim), 9.0, device=DEV, dtype=dtype).transpose(0, 1)
    ops.cache_attention(s.cache, q, rows, window=window, sinks=sinks, out=out)
    assert bool((out[:front] == 9).all()) and bool((out[front + total:] == 9).all())
    s.check(q[front:front + total], out[front:front + total], new, window=window, sinks=sinks, there=there)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [4, 300])
def test_a_query_that_is_no_number_stays_alone(n, dtype):
    s = Setup([3000, 2000], 2, 128, 64, 32, dtype, seed=n)
    q = torch.randn(2 * n, 8, 128, generator=torch.Generator().manual_seed(2)).to(dtype)
    q[1, 3, 7], q[2, 5, 100], q[n, 0, 0] = float("nan"), float("inf"), float("-inf")
    out = ops.cache_attention(s.cache, q.to(DEV), s.rows([n, n]))
    for r, h in ((1, 3), (2, 5), (n, 0)):
        assert bool(out[r, h].isnan().all())
        q[r, h], out[r, h] = 0, s_mean(s, r, h, n).to(out)         # (a query of zeros: the mean of the values it sees)
    s.check(q, out, [n, n])


def s_mean(s, r, h, n):
    b = r // n
    v = s.hv[s.cut[b]:s.cut[b + 1] - n + r % n + 1, h // 4]
    return torch.from_numpy(v.mean(0)).to(s.dtype)


def _bytes_of(x):
    """The addresses of a tensor's elements, in elements of its storage."""
    at = x.storage_offset()
    for n, step in zip(x.shape, x.stride()):
        at = (np.asarray(at)[..., None] + np.arange(n) * step)
    return set(at.reshape(-1).tolist())


def test_outputs_that_overlap_in_part_are_refused():
    """Views of one buffer as query and output, and as the two outputs of a read: wherever they share a byte the call is refused, and
    columns, planes and pieces of one tensor that do not are taken."""
    s = Setup([20, 30], 2, 64, 16, 32, torch.float16)
    n, r = 6, s.rows([3, 3])
    buf = torch.zeros(8 * n * 2 * 64, device=DEV).half()
    view = lambda at, rs, hs: buf[at:].as_strided((n, 2, 64), (rs, hs, 1), at)
    want = ops.cache_read(s.cache, r, n)

    def both(a, b):
        share = bool(_bytes_of(a) & _bytes_of(b))
        try:
            ops.cache_read(s.cache, r, n, out=(a, b))
            taken = True
            assert torch.equal(a, want[0]) and torch.equal(b, want[1])
        except ValueError as e:
            assert "overlap" in str(e)
            taken = False
        x = torch.randn(n, 2, 64, device=DEV).half()
        a.copy_(x)
        try:
            ops.cache_attention(s.cache, a, r, out=b)
            assert torch.equal(b, ops.cache_attention(s.cache, x, r))
            assert taken
        except ValueError as e:
            assert "overlap" in str(e) and not taken
        assert not (share and taken)
        return taken

    for a, b, ok in (((0, 128, 64), (128, 128, 64), False),             # a row further on
                     ((0, 128, 64), (64, 128, 64), False), ((128, 128, 64), (0, 128, 64), False), ((0, 128, 64), (0, 128, 64), False),
                     ((0, 128, 64), (n * 128, 128, 64), True), ((n * 128, 128, 64), (0, 128, 64), True),      # one behind the other
                     ((0, 256, 64), (128, 256, 64), True), ((128, 256, 64), (0, 256, 64), True),              # columns of one row
                     ((0, 256, 64), (64, 256, 64), False), ((0, 256, 128), (64, 256, 128), True),             # heads in turn
                     ((0, 256, 64), (3 * 256 + 128, 256, 64), True), ((3 * 256, 256, 64), (0, 256, 64), False),
                     ((0, 64, n * 64), (2 * n * 64, 64, n * 64), True), ((0, 64, 2 * n * 64), (n * 64, 64, 2 * n * 64), True),   # planes
                     ((0, 64, 2 * n * 64), (n * 64 - 64, 64, 2 * n * 64), False), ((0, 128, 64), (64, 64, n * 64), False)):
        assert both(view(*a), view(*b)) == ok, (a, b)
    g = np.random.default_rng(3)
    taken = 0
    for _ in range(60):                                                 # and drawn ones
        def one():
            if g.random() < 0.5:
                hs = int(g.choice([64, 72, 128]))
                return view(int(g.integers(0, 60)) * 8, int(g.choice([hs + 64, 256, 384])), hs)
            rs = int(g.choice([64, 72, 128]))
            return view(int(g.integers(0, 60)) * 8, rs, int(g.choice([(n - 1) * rs + 64, 1024])))
        taken += both(one(), one())
    assert taken
