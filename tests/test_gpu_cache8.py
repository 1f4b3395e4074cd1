"""The 8-bit key/value cache on the GPU against its definition: writing (block by block, a scale that grows), reading back,
attention.

What is held is defined to the bit, fp16 and bf16 hold it exactly, and it is compared bit for bit.  Attention is compared with the
definition in float64.  Keys and values are exact as operands.  With u = 2^-11 (half a step of fp16): for bf16 the queries, with the scale of the
scores in them, may be rounded once, so a score is off by at most u times scale sum_d |q_d k_d| =: reach, and p is rounded once, u; fp16
queries are exact and p is two fp16 (2^-22 of it).  In float32, at 2^-24 a step: a score is a sum of dim products (dim 2^-24 of reach, in any order), then two products
and one sum (scores here stay below 64 log2 e = 93: 3 * 93 * 2^-24 < 2^-15.9), the exponential adds 2^-22; a p below what fp16 holds is lost, 2^-32 of the
largest for each of n tokens.  Weights that are off by a factor 1 + e_j, |e_j| <= e, move the normalised sum by at most
e / (1 - e) sum_j p_j |v_j - o|; sums over n tokens in float32, n / 32 + 64 steps one behind the other, are off by that many times 2^-24 of
sum_j p_j |v_j|; the result is rounded to its type, and an fp16 one may be subnormal (2^-25)."""
import numpy as np
import pytest
import torch

from cobalt_amd import KVCache8, KVRows, _lib, ops
from oracle import cache8_ref as R8

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -11
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cut(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(int).tolist()


def bound(o, spread, size, reach, dim, n, dtype):
    """What a row of `dtype` may be off by (above)"""
    e = (U if dtype == BF16 else 0.0) * reach + dim * 2.0 ** -24 * reach + 2.0 ** -15.9 + (U if dtype == BF16 else 2.0 ** -22) + 2.0 ** -22 + n * 2.0 ** -32
    e = np.asarray(e)[..., None]
    tol = e / (1 - e) * spread + (n / 32 + 64) * 2.0 ** -24 * size
    return tol + HALF[dtype] * (np.abs(o) + tol) + 2.0 ** -25


class Setup:
    """Sequences of the given lengths whose tokens are all in the cache, written at once, on pages handed out in a shuffled order."""

    def __init__(self, lens, heads, dim, page, block, dtype, seed=0, spare=2, fill=None, outliers=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.dim, self.page, self.block, self.dtype, self.g = lens, heads, dim, page, block, dtype, g
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
        self.cut = cut(lens)
        self.cache = KVCache8(self.pages, heads, dim, page=page, block=block, device=DEV)
        self.ref = R8.Pool(self.pages, heads, dim, page, block)
        self.write(self.k, self.v, lens, lens)

    def write(self, k, v, lens, new):
        ops.cache_write(self.cache, k.to(DEV), v.to(DEV), KVRows(self.table, ints(lens), ints(cut(new))))
        self.ref.write(self.table.tolist(), lens, cut(new), k.float().cpu().numpy(), v.float().cpu().numpy())
        self.lens = lens
        self.cut = cut(lens)
        self.refresh()

    def refresh(self):
        held = [self.ref.read(self.table.tolist(), b, range(n)) for b, n in enumerate(self.lens)]
        self.hk, self.hv = (np.concatenate([h[i] for h in held]) if held else np.zeros((0, self.heads, self.dim)) for i in range(2))

    def rows(self, new):
        return KVRows(self.table, ints(self.lens), ints(cut(new)))

    def check_held(self, types=(torch.float32, F16, BF16)):
        for t in types:
            k, v = ops.cache_read(self.cache, self.rows(self.lens), sum(self.lens), t)
            assert k.dtype == t
            np.testing.assert_array_equal(k.float().cpu().numpy(), self.hk.astype(np.float32))
            np.testing.assert_array_equal(v.float().cpu().numpy(), self.hv.astype(np.float32))

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
                o, spread, size, reach = R8.attention(qn[at:at + n, h], k[:, h // ratio], v[:, h // ratio], pos, ok, scale, window, sinks)
                tol = bound(o, spread, size, reach, self.dim, self.lens[b], out.dtype)
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
FORMS = [(64, 16, 16, 2), (64, 64, 64, 1), (64, 32, 256, 3), (128, 16, 16, 3), (128, 16, 256, 8), (128, 32, 32, 5), (128, 64, 64, 2), (128, 128, 128, 1),
         (128, 256, 256, 2), (256, 16, 64, 1), (256, 32, 32, 4), (256, 64, 128, 1), (256, 128, 128, 2), (256, 256, 256, 1)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,block,page,heads", FORMS)
def test_written_tokens_read_back_as_defined(dim, block, page, heads, dtype):
    lens = [1, 0, 17, 300, 15, 64]
    s = Setup(lens, heads, dim, page, block, dtype, seed=dim + block + page)
    s.check_held()
    # the newest tokens alone; rows behind the last sequence and in front of the first stay as they were
    new = [1, 0, 5, 33, 15, 2]
    n = sum(new)
    k, v = (torch.full((n + 5, heads, dim), 7.0, device=DEV) for _ in range(2))
    ops.cache_read(s.cache, KVRows(s.table, ints(lens), ints([x + 2 for x in cut(new)])), n + 5, torch.float32, out=(k, v))
    want = np.concatenate([np.arange(s.cut[b + 1] - m, s.cut[b + 1]) for b, m in enumerate(new)])
    np.testing.assert_array_equal(k[2:2 + n].cpu().numpy(), s.hk[want].astype(np.float32))
    np.testing.assert_array_equal(v[2:2 + n].cpu().numpy(), s.hv[want].astype(np.float32))
    for x in (k, v):
        assert bool((x[:2] == 7).all()) and bool((x[2 + n:] == 7).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,block,page,heads", FORMS)
def test_a_blocks_scale_grows_with_its_tokens(dim, block, page, heads, dtype):
    """Sequences that grow by odd steps, of magnitudes that change by powers of two, up and down; the older tokens follow."""
    g = torch.Generator().manual_seed(dim * block + page)
    s = Setup([3, 0, 40], heads, dim, page, block, dtype, seed=7)
    grow = [[1, 1, 1], [5, 17, 3], [0, 2, 30], [33, 0, 1], [1, 15, 16], [64, 7, 0], [1, 1, 1]]
    most = [a + sum(x[i] for x in grow) for i, a in enumerate(s.lens)]
    pages = sum(-(-n // page) for n in most) + s.pages
    cache = KVCache8(pages, heads, dim, page=page, block=block, device=DEV)     # of pages for all that comes
    for a, b in zip(cache.native()[:3], s.cache.native()[:3]):
        a[:b.numel()] = b
    ref = R8.Pool(pages, heads, dim, page, block)
    for i in range(2):
        ref.codes[i][:s.pages], ref.scale[i][:s.pages] = s.ref.codes[i], s.ref.scale[i]
    table = [[x for x in row if x >= 0] for row in s.table.tolist()]
    fresh = iter(range(s.pages, pages))
    for b in range(3):
        while len(table[b]) * page < most[b]:
            table[b].append(next(fresh))
    cols = max(map(len, table)) + 1
    s.table = ints([t + [-1] * (cols - len(t)) for t in table])
    s.cache, s.ref, s.pages = cache, ref, pages
    for i, new in enumerate(grow):
        size = 2.0 ** torch.randint(-9, 7, (sum(new), heads, 1), generator=g)
        k, v = ((torch.randn(sum(new), heads, dim, generator=g) * size).to(dtype) for _ in range(2))
        s.write(k, v, [a + b for a, b in zip(s.lens, new)], new)
        s.check_held((torch.float32,) if i % 3 else (F16, BF16))


def test_a_block_begins_anew_with_its_first_token():
    s = Setup([20], 1, 64, 16, 16, F16, fill=lambda s: s.k.mul_(1000.0))
    before = s.ref.scale[0].max()
    small = torch.full((4, 1, 64), 0.01).half()
    s.write(small, small, [20], [4])                                # tokens 16 .. 19: the page's second block from its first token
    s.check_held()
    assert before > s.ref.scale[0][s.table[0, 1].item(), 0, 0] == 2.0 ** -15
    s.write(small[:1] * 3, small[:1], [20], [1])                    # and its last token again, in its scale
    s.check_held()
    assert s.ref.scale[0][s.table[0, 1].item(), 0, 0] == 2.0 ** -13


def test_values_at_the_ends_of_the_range():
    def fill(s):
        k, v = s.k, s.v
        k[:], v[:] = 0.0, 0.0
        k[0], v[0] = 448.0 * 2.0 ** -15, 0.0138                     # the last of the smallest scale, and just beyond
        k[16], v[16] = 448.0, 450.0
        k[32], v[32] = 1e30, -3e38                                  # beyond what is held
        k[33], v[33] = 1.0, 57344.0
        k[48, 0, 5], v[48, 0, 5] = float("inf"), float("-inf")
        k[64, 1, 7] = float("nan")                                  # the token's key and value of this head are NaN, and count nothing
        k[64, 1, 8] = 50000.0
        k[65] = 1.0
        v[65] = 2.0
        v[80, 0, 0] = float("nan")
        k[96] = torch.linspace(0, 1, 128) * 1e-6                    # below the smallest scale's steps and between them
        v[96] = torch.linspace(-1, 1, 128) * 2.0 ** -22
        k[112] = torch.arange(128) * 2.0 ** -9                      # subnormal codes, ties among them
        k[112, :, 0] = 448.0
        k[113] = (torch.arange(128) + 0.5) * 2.0 ** -9
    s = Setup([130], 2, 128, 16, 16, BF16, fill=fill)
    s.check_held()
    k, v = ops.cache_read(s.cache, s.rows([130]), 130, torch.float32)
    assert bool(k[64, 1].isnan().all()) and bool(v[64, 1].isnan().all()) and not bool(k[64, 0].isnan().any())
    assert bool(k[80, 0].isnan().all()) and bool(v[80, 0].isnan().all()) and int(k.isnan().sum()) == 256
    assert bool((k[32] == 57344).all()) and bool((v[32] == -57344).all()) and float(k[48, 0, 5]) == 57344 and float(v[48, 0, 5]) == -57344
    assert s.ref.scale[0][s.table[0, 4].item(), 0, 1] == 2.0 ** -8  # of 1.0, not of the NaN's neighbour
    assert bool((k[65] == 1).all()) and bool((v[33] == 57344).all())
    # a scale that grows under tokens that are NaN leaves them NaN
    s.write(torch.full((1, 2, 128), 5000.0).bfloat16(), torch.full((1, 2, 128), 1.0).bfloat16(), [67], [1])
    s.lens, s.cut = [130], [0, 130]
    s.refresh()
    s.check_held()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_every_16_bit_number_is_rounded_as_defined(dtype):
    """Every finite number below 57344 under every scale: a block's first value sets the scale."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype).float()
    x = bits[torch.isfinite(bits) & (bits.abs() <= 57344)]
    for e in range(-15, 8):
        top = 448.0 * 2.0 ** e
        y = x[x.abs() <= top]
        n = -(-y.numel() // 255)
        y = torch.cat([y, y.new_zeros(n * 255 - y.numel())]).view(n, 255)
        y = torch.cat([torch.full((n, 1), top), y], 1).view(n, 1, 256).to(dtype)
        cache = KVCache8(n // 16 + 1, 1, 256, page=16, block=16, device=DEV)
        rows = cache.rows([list(range(n // 16 + 1))], [n], [0, n])
        y = y.to(DEV)
        ops.cache_write(cache, y, -y, rows)
        k, v = ops.cache_read(cache, rows, n, torch.float32)
        want = R8.e4m3(y.double().cpu().numpy() / 2.0 ** e) * 2.0 ** e
        np.testing.assert_array_equal(k.cpu().numpy(), want.astype(np.float32))
        assert torch.equal(k, -v)


@pytest.mark.parametrize("up", [1, 2, 3, 5, 9, 14, 22])
def test_every_code_follows_a_scale_that_grows(up):
    """All 255 codes under scales that grow by 2^up: exact down to the smallest numbers, which round once more."""
    codes = torch.tensor(sorted({float(x) for n, m in ((448, 200001), (1, 4097)) for x in R8.e4m3(np.linspace(-n, n, m))}))
    assert codes.numel() == 253                                     # (0 has two)
    low = min(-15, 7 - up)
    x = torch.cat([codes * 2.0 ** low, torch.zeros(3)]).view(1, 1, 256).to(BF16)
    s = Setup([1], 1, 256, 16, 16, BF16, fill=lambda s: (s.k.copy_(x), s.v.copy_(-x)))
    s.check_held()
    np.testing.assert_array_equal(s.hk[0, 0], x[0, 0].double().numpy())
    big = torch.full((1, 1, 256), 448.0 * 2.0 ** (low + up)).to(BF16)
    s.write(big, big, [2], [1])
    s.check_held()


def test_equal_numbers_of_rows_need_no_offsets():
    s = Setup([40, 9, 16, 100], 2, 128, 16, 16, F16)
    a = ops.cache_read(s.cache, KVRows(s.table, ints(s.lens)), 12, torch.float32)
    b = ops.cache_read(s.cache, s.rows([3] * 4), 12, torch.float32)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q = torch.randn(12, 4, 128, device=DEV).half()
    assert torch.equal(ops.cache_attention(s.cache, q, KVRows(s.table, ints(s.lens))), ops.cache_attention(s.cache, q, s.rows([3] * 4)))
    k, v = (torch.randn(12, 2, 128).half() for _ in range(2))
    ops.cache_write(s.cache, k.to(DEV), v.to(DEV), KVRows(s.table, ints(s.lens)))
    s.ref.write(s.table.tolist(), s.lens, cut([3] * 4), k.float().numpy(), v.float().numpy())
    s.refresh()
    s.check_held()


@pytest.mark.parametrize("block", [16, 64])
def test_rows_of_many_blocks_and_of_few(block):
    """Calls whose workgroups walk through all that begins among their rows (long runs, short ones between, empty sequences), and calls
    with a workgroup a row."""
    g = np.random.default_rng(block)
    lens = [int(x) for x in g.integers(0, 30, 300)] + [9000, 1, 2, 4000] + [int(x) for x in g.integers(0, 3, 200)]
    s = Setup(lens, 1, 64, 64, block, BF16, seed=5)
    s.check_held((torch.float32,))
    new = [min(n, int(x)) for n, x in zip(lens, g.integers(0, 4, len(lens)))]
    k, v = ((torch.randn(sum(new), 1, 64) * 8).bfloat16() for _ in range(2))
    s.write(k, v, lens, new)
    s.check_held((BF16,))


def test_many_empty_sequences_between():
    """A million sequences, of which a few have rows, some of them one behind the other; and rows in front of the first and behind the last."""
    seqs, page = 1 << 20, 16
    have = {0: 5, 1: 1, 77777: 20, 77778: 3, 500000: 33, seqs - 1: 2}
    lens = torch.zeros(seqs, dtype=torch.int32)
    new = torch.zeros(seqs, dtype=torch.int64)
    table = torch.full((seqs, 3), -1, dtype=torch.int32)
    at, small = 0, []
    for b, n in have.items():
        lens[b] = new[b] = n
        table[b, :-(-n // page)] = torch.arange(at, at + -(-n // page), dtype=torch.int32)
        at += -(-n // page)
        small.append(n)
    starts = (torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]) + 2).int()
    rows = KVRows(table.to(DEV), lens.to(DEV), starts.to(DEV))
    total = sum(small) + 5
    k, v = (torch.randn(total, 1, 64).half() for _ in range(2))
    cache, ref = KVCache8(at, 1, 64, page=page, device=DEV), R8.Pool(at, 1, 64, page, 16)
    ops.cache_write(cache, k.to(DEV), v.to(DEV), rows)
    ref.write([table[b].tolist() for b in have], small, [x + 2 for x in cut(small)], k.float().numpy(), v.float().numpy())
    out = tuple(torch.full((total, 1, 64), 7.0, device=DEV) for _ in range(2))
    ops.cache_read(cache, rows, total, torch.float32, out=out)
    held = [ref.read([table[b].tolist() for b in have], i, range(n)) for i, n in enumerate(small)]
    for i in range(2):
        np.testing.assert_array_equal(out[i][2:-3].cpu().numpy(), np.concatenate([h[i] for h in held]).astype(np.float32))
        assert bool((out[i][:2] == 7).all()) and bool((out[i][-3:] == 7).all())
    slots, positions = ops.cache_slots(cache, rows, total)
    want = [int(table[b, j // page]) * page + j % page for b, n in have.items() for j in range(n)]
    assert slots.tolist() == [-1, -1] + want + [-1] * 3 and positions.tolist() == [0, 0] + [j for n in small for j in range(n)] + [0] * 3


def test_a_write_touches_its_own_blocks_only():
    s = Setup([37, 20], 3, 128, 16, 16, F16, spare=3)
    k, v = (torch.randn(3, 3, 128).half() for _ in range(2))
    s.write(k, v, [37, 20], [2, 1])
    s.check_held()
    # no page, a page number outside the pool, a position behind the table: nothing is written and reads are 0
    after = [t.clone() for t in s.cache.native()[:3]]
    n, k, v = [2, 1], k.to(DEV) * 100, v.to(DEV) * 100
    for bad in (-1, s.pages, 1 << 30, -(1 << 31)):
        table = torch.full_like(s.table, bad)
        ops.cache_write(s.cache, k, v, s.rows(n)._replace(table=table))
        got = ops.cache_read(s.cache, s.rows(n)._replace(table=table), 3, torch.float32)
        assert not bool(got[0].any()) and not bool(got[1].any())
    for lens in ([1 << 30, (1 << 31) - 1], [0, 0], [-5, -(1 << 31)]):
        ops.cache_write(s.cache, k, v, s.rows(n)._replace(lens=ints(lens)))
    for starts in ([3, 3, 3], [0, 0, 0], [4, 9, 100], [-5, -3, 0]):
        ops.cache_write(s.cache, k, v, s.rows(n)._replace(starts=ints(starts)))
    for x, y in zip(s.cache.native()[:3], after):
        assert torch.equal(x, y)


def test_more_rows_than_tokens():
    s = Setup([40, 5], 2, 128, 16, 16, F16)
    k, v = (torch.randn(9, 2, 128).half() for _ in range(2))
    ops.cache_write(s.cache, k.to(DEV), v.to(DEV), KVRows(s.table, ints([40, 5]), ints([0, 2, 9])))
    s.ref.write(s.table.tolist(), [40, 5], [0, 2, 9], k.float().numpy(), v.float().numpy())
    s.refresh()
    s.check_held((torch.float32,))
    a, b = ops.cache_read(s.cache, KVRows(s.table, ints([40, 5]), ints([0, 2, 9])), 9, torch.float32)
    assert not bool(a[2:4].any()) and not bool(b[2:4].any())        # rows in front of the sequence
    np.testing.assert_array_equal(a[4:].cpu().numpy(), s.hk[40:].astype(np.float32))


def test_strided_and_unaligned_inputs():
    s = Setup([50, 30], 2, 128, 32, 16, F16, seed=4)
    n, rows = 10, KVRows(s.table, ints(s.lens))
    fused = torch.randn(n, 2 * 4 * 128 + 8, device=DEV).half()      # q | k | v of one projection, with a tail
    k = fused[:, 512:768].view(n, 2, 128)
    v = fused[:, 768:1024].view(n, 2, 128)
    keep = [t.clone() for t in s.cache.native()[:3]]
    s.write(k.cpu(), v.cpu(), s.lens, [5, 5])
    s.check_held((torch.float32,))
    want = ops.cache_read(s.cache, rows, n, torch.float32)

    def restore():
        for t, x in zip(s.cache.native()[:3], keep):
            t.copy_(x)
    for make in (lambda x: x, lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),             # heads outside
                 lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),                          # channels not contiguous
                 lambda x: torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(x.shape)):           # 2 bytes off
        restore()
        ops.cache_write(s.cache, make(k), make(v), rows)
        b = ops.cache_read(s.cache, rows, n, torch.float32)
        assert torch.equal(want[0], b[0]) and torch.equal(want[1], b[1])
    out = tuple(torch.zeros(2, n, 128, device=DEV).transpose(0, 1) for _ in range(2))
    ops.cache_read(s.cache, rows, n, torch.float32, out=out)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    one = k[:1].expand(n, 2, 128)                                   # the same keys n times: a row stride of 0
    ops.cache_write(s.cache, one, one, rows)
    b = ops.cache_read(s.cache, rows, n, torch.float32)
    assert torch.equal(b[0][0], b[0][4])
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_read(s.cache, rows, n, torch.float32, out=(out[0], out[0]))


# ------------------------------------------------------------------ attention
LENS = [1, 2, 15, 16, 17, 33, 127, 128, 129, 300, 513]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,block,page,heads,ratio", [(64, 16, 16, 2, 4), (64, 32, 32, 1, 1), (128, 16, 64, 2, 4), (128, 16, 16, 1, 8), (128, 128, 256, 3, 1),
                                                        (128, 32, 32, 1, 16), (256, 16, 16, 1, 4), (256, 64, 128, 2, 2), (256, 256, 256, 1, 3), (128, 16, 16, 1, 20)])
def test_one_token_of_each_sequence(dim, block, page, heads, ratio, dtype):
    s = Setup(LENS, heads, dim, page, block, dtype, seed=dim + block)
    s.attend([1] * len(LENS), ratio)


@pytest.mark.parametrize("dim,ratio", [(64, 3), (128, 4), (256, 2)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (128, 130), (129, 4), (200, 1), (10 ** 9, 3), (2 ** 31 - 1, 0)])
def test_windows_and_sinks(dim, ratio, window, sinks):
    s = Setup(LENS, 2, dim, 16, 16, F16, seed=window % 97)
    s.attend([1] * len(LENS), ratio, window=window, sinks=sinks)
    s.attend([min(n, 9) for n in LENS], ratio, window=window, sinks=sinks)


@pytest.mark.parametrize("dim,ratio,dtype", [(64, 4, BF16), (128, 4, F16), (128, 1, BF16), (256, 8, F16)])
def test_several_tokens_of_each_sequence(dim, ratio, dtype):
    s = Setup(LENS, 1, dim, 32, 32, dtype, seed=3)
    s.attend([min(n, 1 + i) for i, n in enumerate(LENS)], ratio)
    s.attend([0, 2, 0, 0, 17, 3, 0, 1, 0, 0, 0], ratio)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,block,page", [(64, 16, 16), (64, 64, 64), (128, 16, 16), (128, 32, 64), (128, 256, 256), (256, 16, 32), (256, 128, 128)])
def test_prompts_of_every_format(dim, block, page, dtype):
    """Enough rows for the kernel that takes tiles of 256, with short and empty sequences between."""
    s = Setup([1, 875, 0, 300, 1064], 4, dim, page, block, dtype, seed=dim * block)
    s.attend(s.lens, 4)
    s.attend([0, 640, 0, 130, 1064], 4, window=48, sinks=5)


@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (256, F16)])
def test_small_prompts(dim, dtype):
    s = Setup([1, 130, 0, 257, 64, 400], 2, dim, 16, 16, dtype, seed=8)
    s.attend(s.lens, 2)
    s.attend([0, 70, 0, 200, 1, 399], 3, window=50, sinks=4)


@pytest.mark.parametrize("dim,block,dtype", [(64, 16, F16), (128, 64, BF16)])
def test_many_prompts(dim, block, dtype):
    """More tiles of rows than the chip holds workgroups: one workgroup each."""
    g = np.random.default_rng(1)
    s = Setup([int(x) for x in g.integers(0, 70, 1100)], 1, dim, 64, block, dtype, seed=16)
    s.attend(s.lens, 1)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (128, BF16), (256, F16)])
def test_chunks_behind_long_histories_are_cut_and_joined(dim, dtype):
    s = Setup([7000, 40, 2600], 4, dim, 32, 32, dtype, seed=15)
    s.attend([260, 40, 133], 4)
    s.attend([270, 1, 100], 4, window=1500, sinks=100)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,page,block", [(64, 64, 16), (128, 16, 16), (128, 64, 64)])
def test_drafts_of_more_than_sixteen_rows_a_head(dim, page, block, dtype):
    """Tiles of 32 rows, which long histories take: part of one, two sixteens, more than a tile; some of their pages missing, and a NaN."""
    def fill(s):
        s.v[5200 + 4100 - 3, 2, 1] = float("nan")                  # seen by the second sequence's last three rows
    s = Setup([5200, 4100, 17, 5000, 0, 3000], 8, dim, page, block, dtype, seed=dim + block, fill=fill)
    new = [5, 8, 5, 9, 0, 1]
    q, out = s.attend([5, 0, 5, 9, 0, 8], 4)
    s.attend([5, 0, 5, 9, 0, 8], 4, window=1000, sinks=70)
    q = torch.randn(sum(new), 32, dim, device=DEV).to(dtype)
    out = ops.cache_attention(s.cache, q, s.rows(new))
    nan = out.isnan().any(-1)
    assert bool(nan[10:13, 8:12].all()) and int(nan.sum()) == 12
    there = [np.ones(n, bool) for n in s.lens]
    table = s.table.clone()
    for b, i in ((0, 3), (3, 0), (3, 5000 // page)):
        table[b, i] = -1
        there[b][page * i:page * i + page] = False
    new = [5, 0, 5, 9, 0, 8]
    q = torch.randn(sum(new), 32, dim, device=DEV).to(dtype)
    s.check(q, ops.cache_attention(s.cache, q, s.rows(new)._replace(table=table)), new, there=there)


@pytest.mark.parametrize("lens,heads,ratio", [([20011], 1, 4), ([9000, 3, 12345], 2, 2), ([4097], 8, 4)])
def test_long_histories_are_cut_and_joined(lens, heads, ratio):
    s = Setup(lens, heads, 128, 64, 16, BF16, seed=5)
    s.attend([1] * len(lens), ratio)
    s.attend([1] * len(lens), ratio, window=5000, sinks=200)
    s.attend([min(n, 3) for n in lens], ratio)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_one_tile_in_hundreds_of_pieces(dim, dtype):
    s = Setup([70001], 1, dim, 128, 32, dtype, seed=7)
    s.attend([1], 1)
    s.attend([1], 16)
    s.attend([5], 3, window=60000, sinks=10)



@pytest.mark.parametrize("lens,heads,dim", [([1000] + [700, 1, 90] * 13, 8, 128), ([2000] + [1300, 0, 500, 129] * 25, 8, 64), ([1300, 2000, 20] * 25, 8, 128)])
def test_histories_of_some_length_in_one_piece(lens, heads, dim):
    """Enough sequences of medium length that no history is cut."""
    s = Setup(lens, heads, dim, 64, 16, BF16, seed=8)
    s.attend([min(n, 1) for n in lens], 4)
    s.attend([min(n, 1) for n in lens], 4, window=600, sinks=100)
    s.attend([min(n, 3) for n in lens], 4)
    s.attend([min(n, 7) for n in lens], 4)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_drafts_over_many_and_over_long_histories(dim, dtype):
    """Tiles of 32 rows, in one piece and cut, their last rows empty."""
    s = Setup([1100, 800, 40] * 13 + [1100], 8, dim, 64, 16, dtype, seed=3)
    s.attend([min(n, 3) for n in s.lens], 8)
    s.attend([min(n, 3) for n in s.lens], 8, window=700, sinks=3)
    s = Setup([11000, 300, 9000, 10000, 8000, 9500, 11000], 8, dim, 64, 64, dtype, seed=4)
    s.attend([5, 3, 7, 5, 6, 5, 5], 4)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompts_and_chunks_of_them(dim, dtype):
    """The kernel for many rows, a tile of rows one workgroup's and cut."""
    s = Setup([900, 300, 0, 500], 8, dim, 64, 16, dtype, seed=5)
    s.attend([900, 300, 0, 500], 4)
    s.attend([900, 300, 0, 500], 4, window=200, sinks=5)
    s = Setup([3001, 700], 8, dim, 64, 32, dtype, seed=6)
    s.attend([300, 500], 4)
    s.attend([300, 500], 4, window=2500, sinks=100)


def test_many_sequences():
    """More sequences than a workgroup has threads, most of them short, some empty."""
    g = np.random.default_rng(0)
    lens = [int(x) for x in g.integers(0, 40, 700)]
    lens[300] = 1500
    s = Setup(lens, 1, 64, 16, 16, F16, seed=6)
    s.attend([min(n, 1) for n in lens], 2)


@pytest.mark.parametrize("heads,dim", [(1, 64), (4, 128)])
def test_many_short_prompts(heads, dim):
    g = np.random.default_rng(1)
    s = Setup([int(x) for x in g.integers(0, 60, 600)], heads, dim, 16, 16, BF16, seed=9)
    s.attend(s.lens, 8)
    s.attend([(n + 1) // 2 for n in s.lens], 8, window=10, sinks=2)


def test_rows_that_see_nothing_are_zero():
    s = Setup([100, 40, 30], 2, 128, 16, 16, F16)
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
    s.lens, s.cut = [2], [0, 2]
    s.check(q[3:], out[3:], [2])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,seqs", [(4096, 1), (70, 1), (3000, 3), (4096, 20)])
def test_rows_of_no_sequence_at_all(rows, seqs, dtype):
    s = Setup([500] * seqs, 2, 128, 64, 64, dtype, seed=3)
    q = torch.randn(rows, 8, 128, device=DEV).to(dtype)
    table = torch.cat([s.table, torch.full((seqs, 40), -1, dtype=torch.int32, device=DEV)], 1)
    for at in (0, 1000, rows):
        out = torch.full_like(q, 9)
        ops.cache_attention(s.cache, q, KVRows(table, ints(s.lens), ints([at] * (seqs + 1))), out=out)
        assert bool((out == 9).all())
    starts = [0] * (seqs + 1)
    starts[-1] = 5                                                  # and with five rows of the last one
    out = torch.full_like(q, 9)
    ops.cache_attention(s.cache, q, KVRows(table, ints(s.lens), ints(starts)), out=out)
    assert bool((out[5:] == 9).all())
    s.check(q[:5], out[:5], [0] * (seqs - 1) + [5])


@pytest.mark.parametrize("many", [False, True])
def test_missing_pages_are_not_seen(many):
    s = Setup([200, 90, 1500], 2, 128, 16, 16, BF16, seed=2)
    there = [np.ones(n, bool) for n in s.lens]
    table = s.table.clone()
    for b, i in ((0, 0), (0, 5), (0, 12), (1, 2), (1, 5), (2, 7), (2, 80)):          # first, inner and last pages
        table[b, i] = -1 if i % 2 else s.pages + 3
        there[b][16 * i:16 * i + 16] = False
    new = [200, 90, 1500] if many else [4, 2, 1]
    q = torch.randn(sum(new), 8, 128, device=DEV).bfloat16()
    out = ops.cache_attention(s.cache, q, KVRows(table, ints(s.lens), ints(cut(new))))
    s.check(q, out, new, there=there)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads", [1, 32])
def test_a_nan_reaches_the_rows_that_see_it_only(dim, heads):
    def fill(s):
        s.v[70, 0, 3] = float("nan")
        s.k[100, 0, 3] = float("nan")
    s = Setup([1100], heads, dim, 16, 16, F16, fill=fill)
    q = torch.randn(1100, 4 * heads, dim, device=DEV).half()
    out = ops.cache_attention(s.cache, q, s.rows([1100]))
    nan = out.isnan().any(-1)
    assert not bool(nan[:70].any()) and bool(nan[70:, :4].all()) and not bool(nan[:, 4:].any())
    out = ops.cache_attention(s.cache, q, s.rows([1100]), window=20)
    assert set(torch.nonzero(out.isnan().any(-1).any(-1)).view(-1).tolist()) == set(range(70, 90)) | set(range(100, 120))
    # a NaN or an infinity in a query stays in its row
    q[5, 1, 7], q[6, 0, 0] = float("nan"), float("inf")
    out = ops.cache_attention(s.cache, q[:40], s.rows([1100])._replace(lens=ints([40]), starts=ints([0, 40])))
    nan = out.isnan().any(-1)
    assert bool(nan[5, 1]) and bool(nan[6, 0]) and int(nan.sum()) == 2


@pytest.mark.parametrize("new", [[3, 1], [1030, 1]])
def test_what_stands_behind_the_last_token_does_not_matter(new):
    s = Setup([1037, 100], 8, 128, 64, 16, F16, seed=9)
    q = torch.randn(sum(new), 32, 128, device=DEV).half()
    rows = KVRows(s.table, ints(s.lens), ints(cut(new)))
    a = ops.cache_attention(s.cache, q, rows)
    # bytes that no write leaves there, in the rest of the last pages: NaN
    for b, n in enumerate(s.lens):
        p, at = int(s.table[b, n // 64]), n % 64
        kc, vc = (t.view(s.pages, 8, -1) for t in s.cache.native()[:2])
        kc[p].view(8, 64, 128)[:, at:] = 0x7f
        v4 = vc[p].view(8, 16, 128, 4)
        v4[:, (at + 3) // 4:] = 0xff
        if at % 4:
            v4[:, at // 4, :, at % 4:] = 0x7f
    assert torch.equal(a, ops.cache_attention(s.cache, q, rows))


def test_stale_values_under_a_larger_scale_do_not_matter():
    """A page that has been another sequence's: its codes of 448 stand behind the last token, under the largest scale."""
    s = Setup([16], 1, 128, 16, 16, F16, fill=lambda s: (s.k.fill_(448.0), s.v.fill_(448.0)))
    x = torch.full((3, 1, 128), 57344.0).half()
    s.write(x * 0.001, x, [3], [3])
    q = torch.randn(3, 4, 128, device=DEV).half() * 0.01
    out = ops.cache_attention(s.cache, q, s.rows([3]))
    assert bool(torch.isfinite(out).all())
    s.check(q, out, [3])


def test_large_and_small_queries():
    s = Setup([300], 1, 128, 32, 32, BF16, outliers=False)
    q = torch.randn(4, 2, 128, device=DEV)
    q[0] *= 2.0 ** 100
    q[1] *= 2.0 ** -100
    q[2] = 0
    q = q.bfloat16()
    out = ops.cache_attention(s.cache, q, s.rows([4]))
    s.check(q[1:], out[1:], [3])                                    # (weights all but equal)
    top = (s.hk[:297, 0] @ q[0].double().cpu().numpy().T).argmax(0)  # one token takes all
    for h in range(2):
        np.testing.assert_allclose(out[0, h].double().cpu().numpy(), s.hv[top[h], 0], rtol=2.0 ** -8, atol=1e-30)
    for scale in (1e-4, 0.5):
        out = ops.cache_attention(s.cache, q[2:], s.rows([2]), scale=scale)
        s.check(q[2:], out, [2], scale=scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,heads", [(4, 1), (64, 1), (1100, 16)])
def test_rows_of_all_sizes_side_by_side(n, heads, dtype):
    """Rows from the smallest to the largest numbers of their type, in one product with ordinary ones; scales from 1e-6 to 30."""
    s = Setup([1200], heads, 128, 32, 32, dtype, outliers=False, seed=3)
    g = torch.Generator().manual_seed(5)
    base = torch.randn(n, 2 * heads, 128, generator=g)
    low, high = (-22, 13) if dtype == F16 else (-120, 60)
    size = torch.linspace(low, high, 2 * n).view(2, n).t().round().repeat(1, heads)
    q = (base * 2.0 ** size[..., None]).to(dtype).to(DEV)
    out = ops.cache_attention(s.cache, q, s.rows([n]))
    qd = q.double().cpu().numpy()
    for i in range(0, n, max(1, n // 64)):
        pos = 1200 - n + i
        for h in range(2):
            sc = s.hk[:pos + 1, 0] @ qd[i, h] * 128 ** -0.5
            if np.abs(sc).max() < 40:
                o, spread, sz, reach = R8.attention(qd[i:i + 1, h], s.hk[:, 0], s.hv[:, 0], np.array([pos]), np.ones(1200, bool), 128 ** -0.5)
                assert (np.abs(out[i, h].double().cpu().numpy() - o[0]) <= bound(o, spread, sz, reach, 128, 1200, dtype)[0]).all(), (i, h)
            # one token takes all, by 200 more than two scores can be off, each by its share of the largest sum of magnitudes
            elif np.sort(sc)[-1] - np.sort(sc)[-2] > 200 + 2 * (U + 2.0 ** -16) * (np.abs(s.hk[:pos + 1, 0]) @ np.abs(qd[i, h])).max() * 128 ** -0.5:
                want = s.hv[sc.argmax(), 0]
                assert (np.abs(out[i, h].double().cpu().numpy() - want) <= (HALF[dtype] + 2.0 ** -16) * np.abs(want) + 1e-6).all(), (i, h)
            else:
                assert bool(torch.isfinite(out[i, h]).all())
    ones = torch.full((n, 2 * heads, 128), 2.0 ** 13, device=DEV).to(dtype)
    out = ops.cache_attention(s.cache, ones, s.rows([n]))
    assert bool(torch.isfinite(out).all())
    if n < 100:
        for scale in (1e-6, 0.02, 3.0, 30.0):
            q = (torch.randn(n, 2, 128, generator=g) * min(1.0, 0.05 / scale)).to(dtype).to(DEV)
            s.check(q, ops.cache_attention(s.cache, q, s.rows([n]), scale=scale), [n], scale=scale)


@pytest.mark.parametrize("large", [300.0, 4096.0, 60000.0, 2.0 ** 20])
@pytest.mark.parametrize("dim,n,heads", [(64, 4, 2), (128, 4, 2), (256, 4, 2), (64, 1100, 16), (128, 1100, 16), (256, 1100, 16)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_large_channel_leaves_the_small_ones(dtype, dim, n, heads, large):
    """One channel of the queries thousands of times the others, over keys that are 0 there: the scores are the others' alone.  fp16 queries are exact operands;
    bf16 ones are held with steps of 2^-24, times what leaves the largest in [2^14, 2^15), so that each is off by 2^-25 max(1, large / 2^14) at most."""
    if dtype == F16 and large > 65504:
        large = 65504.0

    def fill(s):
        s.k *= 4
        s.k[..., 5] = 0
    s = Setup([1100], heads, dim, 64, 32, dtype, outliers=False, seed=11, fill=fill)
    q = 0.05 * torch.randn(n, 2 * heads, dim, generator=torch.Generator().manual_seed(12))
    q[..., 5] = large
    q = q.to(dtype)
    out = ops.cache_attention(s.cache, q.to(DEV), s.rows([n]))
    scale, qn, on = dim ** -0.5, q.double().numpy(), out.double().cpu().numpy()
    for h in range(0, 2 * heads, 2 * heads - 1):
        o, spread, size, reach = R8.attention(qn[:, h], s.hk[:, h // 2], s.hv[:, h // 2], np.arange(1100 - n, 1100), np.ones(1100, bool), scale)
        tol = bound(o, spread, size, reach, dim, 1100, dtype)
        if dtype == BF16:
            e = 2.0 ** -25 * max(1.0, large / 2 ** 14) * np.abs(s.hk[:, h // 2]).sum(1).max()
            tol = tol + 1.01 * e / (1 - e) * spread
        assert (np.abs(on[:, h] - o) <= tol).all(), (h, (np.abs(on[:, h] - o) / tol).max())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scales_at_the_ends_of_their_range(dtype):
    s = Setup([1100], 16, 128, 32, 32, dtype, outliers=False, seed=3)
    for n in (1, 1100):
        q = torch.randn(n, 32, 128, device=DEV).to(dtype)
        out = ops.cache_attention(s.cache, q, s.rows([n]), scale=1e-30)          # weights all equal
        want = np.cumsum(s.hv, 0)[1100 - n:] / np.arange(1100 - n + 1, 1101)[:, None, None]
        size = np.cumsum(np.abs(s.hv), 0)[1100 - n:] / np.arange(1100 - n + 1, 1101)[:, None, None]
        got = out.double().cpu().numpy().reshape(n, 16, 2, 128)
        tol = (1100 / 32 + 64) * 2.0 ** -24 * size + HALF[dtype] * np.abs(want) * 1.01 + 2.0 ** -25 + 2.0 ** -15 * size
        assert (np.abs(got - want[:, :, None]) <= tol[:, :, None]).all()
        out = ops.cache_attention(s.cache, q, s.rows([n]), scale=1e30)           # one token takes all
        assert bool(torch.isfinite(out).all())


def test_one_token_outweighs_a_long_history():
    """Weights 2^-20 of the largest, 30000 of them: 3 % of the sum, in p that fp16 could not tell from 0 as it is."""
    def fill(s):
        s.k[:, 0] = 0
        s.k[777, 0, 0] = 20 * np.log(2) / 128 ** -0.5 / 8
        s.v[:, 0] = 1.0
        s.v[777, 0] = 0.0
    s = Setup([30001], 1, 128, 64, 16, F16, fill=fill)
    q = torch.zeros(1, 1, 128, device=DEV).half()
    q[0, 0, 0] = 8
    s.check(q, ops.cache_attention(s.cache, q, s.rows([1])), [1])


def test_strides_and_rows_behind_the_last_sequence():
    s = Setup([50, 30], 2, 128, 32, 32, F16, seed=4)
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
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_attention(s.cache, q, rows, out=q)


def test_calls_repeat_bit_for_bit():
    s = Setup([5000, 700, 1], 2, 128, 64, 64, BF16, seed=11)
    q, a = s.attend([1, 1, 1], 4)
    for _ in range(3):
        torch.empty(64 << 20, dtype=torch.uint8, device=DEV).fill_(255)   # what the workspace comes back as
        assert torch.equal(a, ops.cache_attention(s.cache, q, s.rows([1, 1, 1])))


def test_a_pool_of_more_than_four_gigabytes():
    heads, dim, page = 4, 256, 256
    pages = (1 << 32) // (heads * page * dim) + 9
    s = Setup([700, 513], heads, dim, page, 128, F16, spare=0)
    cache = KVCache8(pages, heads, dim, page=page, block=128, device=DEV)
    table = s.table.clone()
    table[table >= 0] += pages - s.pages
    every = KVRows(table, ints(s.lens), ints(s.cut))
    ops.cache_write(cache, s.k.to(DEV), s.v.to(DEV), every)
    k, v = ops.cache_read(cache, every, 1213, torch.float32)
    np.testing.assert_array_equal(k.cpu().numpy(), s.hk.astype(np.float32))
    np.testing.assert_array_equal(v.cpu().numpy(), s.hv.astype(np.float32))
    q = torch.randn(2, 8, dim, device=DEV).half()
    s.check(q, ops.cache_attention(cache, q, KVRows(table, ints(s.lens))), [1, 1])
    q = torch.randn(1213, 32, dim, device=DEV).half()
    s.check(q[700:], ops.cache_attention(cache, q, every)[700:], [0, 513])
    assert not bool(cache.k_codes[:1 << 20].any())                  # (a wrapped offset would have landed there)


# ------------------------------------------------------------------ as a program uses them
def test_steps_in_a_graph_follow_the_lengths():
    """A recorded step (write, then attend) replayed over growing sequences, each against the eager calls."""
    s = Setup([130, 60], 2, 128, 16, 16, F16, seed=12)
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
            t.copy_(torch.randn(t.shape, generator=g, device=DEV) * (1 + i))

    arrays = s.cache.native()[:3]
    keep = [t.clone() for t in arrays]
    start = lens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        inputs(0)
        step()
        lens.copy_(start)
    torch.cuda.current_stream().wait_stream(side)
    for t, x in zip(arrays, keep):
        t.copy_(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
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
    s = Setup([5000, 2600], 4, 128, 64, 64, F16, seed=21)
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
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_calls_on_another_stream():
    s = Setup([3000, 700], 4, 128, 64, 16, BF16, seed=22)
    q = torch.randn(2, 16, 128, device=DEV).bfloat16()
    want = ops.cache_attention(s.cache, q, s.rows([1, 1]))
    rows = s.rows([1, 1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(ops.cache_attention(s.cache, q, rows))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_refusals_on_the_device():
    s = Setup([40], 2, 128, 16, 16, F16)
    x = torch.randn(1, 2, 128, device=DEV).half()
    rows = s.rows([1])
    with pytest.raises(_lib.CbkError):
        ops.cache_write(s.cache, x.cpu(), x.cpu(), rows)
    with pytest.raises(ValueError):
        ops.cache_write(s.cache, x, x.bfloat16(), rows)
    with pytest.raises(ValueError):
        ops.cache_write(s.cache, x[:, :1], x[:, :1], rows)
    with pytest.raises(ValueError):
        ops.cache_attention(s.cache, torch.randn(1, 3, 128, device=DEV).half(), rows)
    with pytest.raises(TypeError):
        ops.cache_attention(s.cache, x.float(), rows)
    s.cache.scales = s.cache.scales[:-8]
    with pytest.raises(ValueError, match="do not hold"):
        ops.cache_attention(s.cache, x, rows)
