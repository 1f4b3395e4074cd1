"""Attention over the 4-bit cache, the kernel for many rows: every form of it (head size, group, type) in both ways of dealing out the work,
and what is special to rows, tokens and scores.  Each case states the plan it is for and is held to it: a call of many rows whose tiles are cut
wants a workspace of 256 shares of two parts of 256 rows, one in whole tiles wants none under a table of more than 1024 tokens.

The definition is computed in float64 here, row by row of a head at once.  Bounds, with u = 2^-11: as in test_gpu_cache.py for bf16.  For fp16 calls
codes, queries and weights are not rounded to 16 bits at all, so only float32 is left of a score: with reach = scale sum_d |q_d| (|k_d| + 2 |m_d|), m the
group's minimum, at most D + 3 D/G + 16 roundings of 2^-23 of it, the sums of q as two fp16 (2^-22 of them, and 2^-25 of the largest minimum where they are
subnormal: 2^-25 scale D/G max |m|, or 2^-20 D/G where the scale is in them), 2^-20 for exponential and weight.  A row of n tokens sums n weights and products:
(n + 16) 2^-23 of sum_j p_j |v_j|; weights below 2^-25 / 2^7.5 of the largest are lost, n 2^-32 of the largest value.  Values are rounded once (u), unless they
are fp16 numbers.  The spread sum_j p_j |v_j - o| is bounded by the root of the weighted variance."""
import ctypes

import numpy as np
import pytest
import torch

from cobalt_amd import KVRows, _lib, ops
from test_gpu_cache import DEV, HALF, SCORE, U, Setup, ints

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
FORMS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


def plan_of(s, rows, count, q_heads):
    c, r = s.cache, _lib.CbkRows(table=16, ld_table=rows.table.shape[1], lens=16, starts=16, seqs=rows.lens.numel(), table_cols=rows.table.shape[1], tokens=count)
    d = _lib.CbkCache(16, 16, 16, 16, c.pages, c.page, c.heads, c.head_dim, c.group)
    need = _lib.lib().cbk_cache_attention_workspace_bytes(ctypes.byref(d), ctypes.byref(r), q_heads)
    if need == 256 * 32 + 256 * 2 * 256 * (c.head_dim + 4) * 4:
        return "cut"
    return "whole" if need == 0 and rows.table.shape[1] * c.page > 1024 else "few"


def rows_of(s, new, span, front=0):
    """The rows of the newest `new` tokens under a table for `span` tokens."""
    cols = -(-span // s.page)
    table = torch.full((len(s.lens), cols), -1, dtype=torch.int32, device=DEV)
    n = min(cols, s.table.shape[1])
    table[:, :n] = s.table[:, :n]
    return KVRows(table, ints(s.lens), ints((np.concatenate([[0], np.cumsum(new)]) + front).astype(int).tolist()))


def check(s, q, out, new, scale=None, window=None, sinks=0, there=None, exact_values=False, skip=()):
    scale = scale or s.dim ** -0.5
    ratio, dt, D, GS = q.shape[1] // s.heads, out.dtype, s.dim, s.dim // s.group
    at = 0
    for b, n in enumerate(new):
        L = s.lens[b]
        pos = torch.arange(L - n, L, device=DEV)[:, None]
        j = torch.arange(L, device=DEV)[None, :]
        seen = j <= pos
        if window:
            seen = seen & ((j > pos - window) | (j < sinks))
        if there is not None:
            seen = seen & torch.from_numpy(there[b]).to(DEV)[None, :]
        cut = slice(s.cut[b], s.cut[b + 1])
        for h in range(q.shape[1]) if n else ():
            k, v = (torch.from_numpy(x[cut, h // ratio].copy()).to(DEV) for x in (s.hk, s.hv))
            low = s.k[cut, h // ratio].float().clamp(-65280, 65280).view(L, GS, -1).amin(-1).half().double().abs().to(DEV)
            x = q[at:at + n, h].double()
            t = (x @ k.T) * scale
            t = t.masked_fill(~seen, -torch.inf)
            top = t.amax(1, keepdim=True)
            p = torch.exp(t - torch.where(top == -torch.inf, 0.0, top))
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            o, size = p @ v, p @ v.abs()
            spread = ((p @ v.square()) - o.square()).clamp_min(0).sqrt()
            count = seen.sum(1, keepdim=True).double()
            bare = scale * (x.abs() @ k.abs().T).masked_fill(~seen, 0).amax(1, keepdim=True)
            if dt == BF16:
                e = SCORE[dt] * bare + U + 2.0 ** -16
                sums = U * size
            else:
                mins = low.repeat_interleave(s.group, 1)
                reach = scale * (x.abs() @ (k.abs() + 2 * mins).T).masked_fill(~seen, 0).amax(1, keepdim=True)
                e = (D + 3 * GS + 16) * 2.0 ** -23 * reach + 2.0 ** -22 * reach + GS * (2.0 ** -25 * scale * float(low.max()) + 2.0 ** -20) + 2.0 ** -20
                sums = (0 if exact_values else U) * size
            tol = e / (1 - e).clamp_min(1e-3) * spread + sums + (count + 16) * 2.0 ** -23 * size + count * 2.0 ** -32 * float(v.abs().max())
            tol = tol + HALF[dt] * (o.abs() + tol) + 2.0 ** -25
            got = out[at:at + n, h].double()
            bad = ~((got - o).abs() <= tol)
            for r, head in skip:
                if head == h and at <= r < at + n:
                    bad[r - at] = False
            assert not bool(bad.any()), (f"sequence {b} (length {L}), head {h}: rows {torch.nonzero(bad.any(1)).flatten()[:8].tolist()}, off by "
                                         f"{(got - o).abs()[bad].max().item()}, allowed {tol[bad].min().item()}, worst {((got - o).abs() / tol).max().item()}")
        at += n


def attend(s, new, ratio, span, plan, seed=1, q=None, **kw):
    exact_values = kw.pop("exact_values", False)
    rows = rows_of(s, new, span)
    if q is None:
        q = torch.randn(sum(new), s.heads * ratio, s.dim, generator=torch.Generator().manual_seed(seed)).to(s.dtype).to(DEV)
    assert plan_of(s, rows, q.shape[0], q.shape[1]) == plan
    out = ops.cache_attention(s.cache, q, rows, **kw)
    check(s, q, out, new, exact_values=exact_values, **kw)
    return q, out, rows


# ------------------------------------------------------------------ every form, both ways
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,group", FORMS)
def test_whole_tiles(dim, group, dtype):
    s = Setup([1290, 5, 1200], 3, dim, {32: 16, 64: 64, 128: 256}[group], group, dtype, seed=dim + group)
    attend(s, s.lens, 4, 1290, "whole")
    attend(s, s.lens, 4, 1290, "whole", window=200, sinks=4)
    attend(s, s.lens, 4, 1290, "whole", window=300, sinks=0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,group", FORMS)
def test_cut_tiles(dim, group, dtype):
    s = Setup([2100, 5, 0, 1303], 3, dim, {32: 32, 64: 16, 128: 128}[group], group, dtype, seed=dim * group)
    attend(s, [601, 5, 0, 900], 4, 4096, "cut")
    attend(s, [601, 5, 0, 900], 4, 4096, "cut", window=128, sinks=130)
    attend(s, [601, 0, 0, 1000], 4, 4096, "cut", window=1000, sinks=1)


@pytest.mark.parametrize("dim,group,dtype", [(64, 64, F16), (128, 32, BF16), (256, 128, F16), (256, 64, BF16)])
def test_many_short_prompts_in_whole_tiles(dim, group, dtype):
    """More tiles of rows than three for every workgroup of the chip: whole ones, whatever the table holds."""
    g = np.random.default_rng(1)
    s = Setup([int(x) for x in g.integers(0, 90, 70)], 8, dim, 16, group, dtype, seed=16)
    attend(s, s.lens, 4, 4096, "whole")
    attend(s, s.lens, 4, 4096, "whole", window=20, sinks=2)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (128, BF16), (256, F16)])
def test_chunks_behind_long_histories(dim, dtype):
    s = Setup([9000, 300, 5000], 2, dim, 32, 32, dtype, seed=15)
    attend(s, [400, 300, 333], 4, 9100, "cut")
    attend(s, [500, 1, 100], 4, 16384, "cut", window=1500, sinks=100)


@pytest.mark.parametrize("ratio", [1, 2, 5, 16, 100, 256])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (256, F16)])
def test_query_heads_on_one(dim, dtype, ratio):
    tokens = {1: 3000, 2: 1500, 5: 1100}.get(ratio, 300)
    s = Setup([tokens, 70], 3 if ratio < 100 else 1, dim, 32, 32, dtype, seed=ratio)
    attend(s, s.lens, ratio, 16384, "cut")


# ------------------------------------------------------------------ rows, tokens and pages
@pytest.mark.parametrize("plan", ["whole", "cut"])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16), (256, BF16)])
def test_pages_that_are_not_there_and_rows_before_the_sequence(dim, dtype, plan):
    s = Setup([1200, 1400, 40], 3, dim, 16, 32, dtype, seed=2)
    g = np.random.default_rng(4)
    new = [1100, 1400, 40] if plan == "whole" else [700, 500, 40]
    rows = rows_of(s, new, 1400 if plan == "whole" else 6000, front=3)
    table, there = rows.table.cpu(), []
    for b, n in enumerate(s.lens):
        gone = g.random(table.shape[1]) < 0.15
        gone[0] = b == 0
        table[b, torch.from_numpy(gone)] = [-1, s.pages, -9][b]
        there.append(~np.repeat(gone, 16)[:n])
    total = sum(new)
    q = torch.randn(total + 5, 12, dim, generator=torch.Generator().manual_seed(7)).to(dtype).to(DEV)
    rows = rows._replace(table=table.to(DEV))
    assert plan_of(s, rows, total + 5, 12) == plan
    out = torch.full((12, total + 5, dim), 9.0, device=DEV, dtype=dtype).transpose(0, 1)
    ops.cache_attention(s.cache, q, rows, window=600, sinks=20, out=out)
    assert bool((out[:3] == 9).all()) and bool((out[3 + total:] == 9).all())
    check(s, q[3:3 + total], out[3:3 + total], new, window=600, sinks=20, there=there)
    # more rows than tokens: the first see nothing
    out = ops.cache_attention(s.cache, q, rows_of(s, new, 1400 if plan == "whole" else 6000)._replace(lens=ints([50, 100, 40])))
    assert not bool(out[:new[0] - 50].any()) and not bool(out[new[0]:new[0] + new[1] - 100].any()) and bool((out[new[0] - 50:new[0]] != 0).any(-1).all())
    assert not bool(ops.cache_attention(s.cache, q, rows._replace(table=torch.full_like(rows.table, -1)))[3:3 + total].any())
    assert not bool(ops.cache_attention(s.cache, q, rows._replace(lens=torch.zeros_like(rows.lens)))[3:3 + total].any())


@pytest.mark.parametrize("plan", ["whole", "cut"])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (128, F16), (256, F16), (256, BF16)])
def test_a_nan_reaches_the_rows_that_see_it_only(dim, dtype, plan):
    def fill(s):
        s.v[700, 0, 3] = float("nan")
        s.k[1000, 1, 3] = float("nan")
    s = Setup([1300], 4, dim, 16, 32, dtype, fill=fill)
    q = torch.randn(1300, 16, dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    rows = rows_of(s, [1300], 1300 if plan == "whole" else 8000)
    assert plan_of(s, rows, 1300, 16) == plan
    nan = ops.cache_attention(s.cache, q, rows).isnan()
    for head, first in ((0, 700), (1, 1000), (2, 1300), (3, 1300)):
        x = nan[:, 4 * head:4 * head + 4]
        assert not bool(x[:first].any()) and bool(x[first:].all())
    out = ops.cache_attention(s.cache, q, rows, window=20)
    for head, first in ((0, 700), (1, 1000)):
        x = out[:, 4 * head:4 * head + 4].isnan().any(-1).any(-1)
        assert torch.nonzero(x).flatten().tolist() == list(range(first, first + 20))


@pytest.mark.parametrize("plan", ["whole", "cut"])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (128, BF16), (128, F16), (256, F16), (256, BF16)])
def test_what_stands_behind_the_last_token_does_not_matter(dim, dtype, plan):
    """NaN, large values and bits that no write leaves in the rest of the last page and on the pages behind it."""
    s = Setup([1330], 4, dim, 16, 32, dtype, seed=9, fill=lambda s: (s.k[1290:].fill_(float("nan")), s.v[1290::2].fill_(6e4)))
    s.lens, s.cut = [1290], np.array([0, 1290])
    q = torch.randn(1290, 16, dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    rows = rows_of(s, [1290], 1296 if plan == "whole" else 8000)
    assert plan_of(s, rows, 1290, 16) == plan
    a = ops.cache_attention(s.cache, q, rows)
    check(s, q, a, [1290])
    s.cache.v_meta.view(torch.int32).view(s.pages, 4, dim // 32, 16)[int(s.table[0, 80]), :, :, 10:] = -1
    s.cache.k_meta.view(torch.int32).view(s.pages, 4, dim // 32, 16)[int(s.table[0, 80]), :, :, 10:] = -1
    assert torch.equal(a, ops.cache_attention(s.cache, q, rows))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("plan", ["whole", "cut"])
def test_queries_that_are_no_numbers_stay_alone(dtype, plan):
    s = Setup([1300, 1200], 4, 128, 64, 32, dtype, seed=3)
    new = [1300, 1200] if plan == "whole" else [400, 500]
    q = torch.randn(sum(new), 16, 128, generator=torch.Generator().manual_seed(2)).to(dtype)
    bad = [(1, 3), (2, 5), (new[0], 0), (300, 15), (350, 15)]
    for (r, h), x in zip(bad, (float("nan"), float("inf"), float("-inf"), float("inf"), float("-inf"))):
        q[r, h, 7 * h] = x
    q = q.to(DEV)
    rows = rows_of(s, new, 1300 if plan == "whole" else 8000)
    assert plan_of(s, rows, sum(new), 16) == plan
    out = ops.cache_attention(s.cache, q, rows)
    for r, h in bad:
        assert bool(out[r, h].isnan().all())
    clean = q.clone()
    for r, h in bad:
        clean[r, h] = 0
    check(s, clean, out, new, skip=bad)
    assert not bool(ops.cache_attention(s.cache, q, rows._replace(lens=torch.zeros_like(rows.lens))).any())      # and nothing is seen: 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("plan", ["few", "whole"])
def test_an_infinite_query_over_keys_of_one_sign(dtype, plan):
    """Scores that are all infinite have no softmax, whatever their sign."""
    s = Setup([1290], 4, 128, 64, 32, dtype, seed=3, fill=lambda s: s.k[:, :, 5].abs_().add_(1))
    n = 4 if plan == "few" else 1290
    q = torch.randn(n, 16, 128, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    bad = [(0, 0), (1, 3), (3, 14)]
    for (r, h), x in zip(bad, (float("-inf"), float("inf"), float("-inf"))):
        q[r, h, 5] = x
    rows = rows_of(s, [n], 1290)
    assert plan_of(s, rows, n, 16) == plan
    out = ops.cache_attention(s.cache, q, rows)
    for r, h in bad:
        assert bool(out[r, h].isnan().all())
        q[r, h] = 0
    check(s, q, out, [n], skip=bad)


# ------------------------------------------------------------------ scores
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,group", [(64, 32), (128, 64), (256, 128)])
@pytest.mark.parametrize("scale", [1e-30, 2.0 ** 20])
def test_the_smallest_and_largest_scales(dim, group, scale, dtype):
    """Scores of nothing: the mean.  Scores of 2^20 and more: the tokens of the largest alone, since keys of one value a token are held
    and multiplied exactly, equal ones alike, and the others lie 2^21 lower."""
    s = Setup([1400], 4, dim, 64, group, dtype, fill=lambda s: s.k.copy_((torch.arange(1400) % 128 / 16).to(dtype)[:, None, None].expand_as(s.k)))
    q = torch.ones(700, 16, dim, device=DEV).to(dtype)
    rows = rows_of(s, [700], 8000)
    assert plan_of(s, rows, 700, 16) == "cut"
    out = ops.cache_attention(s.cache, q, rows, scale=scale)
    for h in range(16):
        v = torch.from_numpy(s.hv[:, h // 4].copy()).to(DEV)
        key = torch.arange(1400, device=DEV) % 128 if scale > 1 else torch.zeros(1400, device=DEV)
        seen = torch.arange(1400, device=DEV)[None, :] <= torch.arange(700, 1400, device=DEV)[:, None]
        best = torch.where(seen, key[None, :], -1).amax(1, keepdim=True)
        w = (seen & (key[None, :] == best)).double()
        w = w / w.sum(1, keepdim=True)
        o, size = w @ v, w @ v.abs()
        tol = (U + 2.0 ** -16 + (1400 + 16) * 2.0 ** -23) * size
        tol = tol + HALF[dtype] * (o.abs() + tol) + 2.0 ** -25
        assert bool(((out[:, h].double() - o).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_of_all_sizes_side_by_side(dim, dtype):
    """Rows of queries from the smallest to the largest numbers for which scores stay below 60, in one product with ordinary ones."""
    s = Setup([1300], 4, dim, 32, 32, dtype, outliers=False, seed=3)
    g = torch.Generator().manual_seed(5)
    low = -24 if dtype == F16 else -120
    size = torch.linspace(low, 2, 1300 * 16).view(16, 1300).t().round()
    q = (torch.randn(1300, 16, dim, generator=g).clamp(-3, 3) * 2.0 ** size[..., None]).to(dtype).to(DEV)
    attend(s, [1300], 4, 1300, "whole", q=q)
    for scale in (1e-6, 0.02, 3.0, 30.0):
        x = (torch.randn(600, 16, dim, generator=g) * min(1.0, 0.05 / scale)).to(dtype).to(DEV)
        attend(s, [600], 4, 8000, "cut", q=x, scale=scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_large_scores_that_rise_and_fall(dim, dtype):
    """One token takes all of a row: scores of both signs up to 43000 (as exponents of 2), whose maximum moves on from tile to tile."""
    def fill(s):
        s.k[:] = 0
        s.k[:, :, 1::2] = (0.25 * torch.arange(1400) % 4).to(dtype)[:, None, None]
        size = torch.arange(0, 1400, 6) // 6
        s.k[::6, :, 0] = (size * (1 - 2 * (size % 2)))[:, None].to(dtype)
    s = Setup([1400], 4, dim, 32, 32, dtype, fill=fill)
    q = torch.zeros(1400, 16, dim)
    q[:, ::2, 0], q[:, 1::2, 0] = 128.0, -128.0
    q = q.to(dtype).to(DEV)
    for new, span, plan in ((1400, 1400, "whole"), (600, 8000, "cut")):
        rows = rows_of(s, [new], span)
        assert plan_of(s, rows, new, 16) == plan
        out = ops.cache_attention(s.cache, q[:new], rows, scale=1.0)
        for h in range(16):
            k = torch.from_numpy(s.hk[:, h // 4].copy()).to(DEV)
            t = q[:new, h].double() @ k.T
            t = t.masked_fill(torch.arange(1400, device=DEV)[None, :] > torch.arange(1400 - new, 1400, device=DEV)[:, None], -torch.inf)
            first, at = t.max(1)
            rest = t.scatter(1, at[:, None], -torch.inf).amax(1)
            alone = first - rest > 60 + 2 * SCORE[dtype] * t.masked_fill(t == -torch.inf, 0).abs().amax(1)   # (the next lies 256 lower)
            o = torch.from_numpy(s.hv[:, h // 4].copy()).to(DEV)[at]
            tol = (U + 2.0 ** -16) * o.abs()
            tol = tol + HALF[dtype] * (o.abs() + tol) + 2.0 ** -25
            ok = (out[:, h].double() - o).abs() <= tol
            assert bool(ok[alone].all()) and int(alone.sum()) > new * 0.9, (h, int(alone.sum()))
            assert bool(torch.isfinite(out[:, h]).all())


@pytest.mark.parametrize("plan", ["few", "cut"])
@pytest.mark.parametrize("size,scale,unit", [(30, 1e30, -14), (100, 1.0, -14), (-30, 1e30, 0), (126, 1e-30, 0), (127, 1.0, -14)])
def test_large_queries_times_large_scales(size, scale, unit, plan):
    """bf16 queries of 2^size whose product with the scale may pass float32, over keys that bring the scores back into it."""
    s = Setup([1300], 4, 128, 64, 32, BF16, fill=lambda s: s.k.copy_((torch.arange(1300) % 16 * 2.0 ** unit).to(BF16)[:, None, None].expand_as(s.k)))
    n = 4 if plan == "few" else 600
    q = torch.zeros(n, 16, 128)
    q[:, :, 40] = 2.0 ** size
    rows = rows_of(s, [n], 1300 if plan == "few" else 8000)
    assert plan_of(s, rows, n, 16) == plan
    out = ops.cache_attention(s.cache, q.bfloat16().to(DEV), rows, scale=scale)
    key = torch.arange(1300, device=DEV) % 16
    seen = torch.arange(1300, device=DEV)[None, :] <= torch.arange(1300 - n, 1300, device=DEV)[:, None]
    w = (seen & (key[None, :] == 15)).double()                      # the largest alone: the others lie far below
    w = w / w.sum(1, keepdim=True)
    for h in range(16):
        v = torch.from_numpy(s.hv[:, h // 4].copy()).to(DEV)
        o = w @ v
        tol = (U + 2.0 ** -16 + 1400 * 2.0 ** -23) * (w @ v.abs())
        tol = tol + HALF[BF16] * (o.abs() + tol) + 2.0 ** -25
        assert bool(((out[:, h].double() - o).abs() <= tol).all())


# ------------------------------------------------------------------ what fp16 calls promise
def _whole_numbers(s):
    """Values from -8 to 7, which are held as they are."""
    s.v[:] = torch.randint(-8, 8, s.v.shape, generator=torch.Generator().manual_seed(11)).half()
    v = s.v.view(s.v.shape[0], s.heads, -1, s.group)
    v[..., 0], v[..., 1] = -8, 7


def _codes(s):
    """Keys whose held values are no fp16 numbers, rounded alike in all channels a query takes: minimum -1 in the even channels and 15 steps
    of an 11-bit scale above it in the odd ones."""
    s.k[:, :, 0::2] = -1.0
    s.k[:, :, 1::2] = (2.0 + 0.04 * torch.rand(s.k.shape[0], s.heads, 1, generator=torch.Generator().manual_seed(12))).half()
    _whole_numbers(s)


@pytest.mark.parametrize("plan", ["few", "whole", "cut"])
@pytest.mark.parametrize("dim,group", FORMS)
def test_codes_queries_and_weights_are_not_rounded(dim, group, plan):
    """Rows of few tokens show it: what is off is not averaged there.  Scores about 40, 5 and 0.2."""
    n = {"few": 24, "whole": 1290, "cut": 300}[plan]
    s = Setup([n], 4, dim, 64, group, F16, fill=_codes, seed=1)
    assert np.array_equal(s.hv, s.v.double().numpy())
    span = {"few": 1100, "whole": n, "cut": 16384}[plan]
    g = torch.Generator().manual_seed(2)
    one_sign = torch.zeros(n, 16, dim)
    one_sign[:, :, 1::2] = 40.0 * dim ** -0.5 * (1 + 0.1 * torch.rand(n, 16, 1, generator=g))
    for q in (one_sign, 0.3 * torch.randn(n, 16, dim, generator=g), 0.01 * torch.randn(n, 16, dim, generator=g)):
        attend(s, [n], 4, span, plan, q=q.half().to(DEV), exact_values=True)


def _tie(near):
    """A scale near the given one and an fp16 number whose product, with log2 e in it, is a tie of fp16 once rounded to float32, and rounds the other way
    where it is exact."""
    log2e, f = np.float32(1.44269504088896341), np.float32
    for i in range(1025, 2048):
        x = np.float16(2 * i / 1024)
        for t in range(3, 400, 2):
            tie = f(near * float(x) * float(log2e)) * (1 + t / 4096)
            step = 2.0 ** (np.floor(np.log2(tie)) - 10)
            tie = f((np.floor(tie / step) + 0.5) * step)
            for scale in (f(float(tie) / float(x) / float(log2e)) * (1 + f(2) ** -23 * f(k)) for k in (-1, 0, 1)):
                fold = scale * log2e
                exact = float(fold) * float(x)                      # (24 and 11 bits: exact in float64)
                if f(exact) == tie and exact != float(tie) and np.float16(f(exact)) != np.float16(exact):
                    return float(scale), float(x)
    raise AssertionError


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32), (256, 128)])
@pytest.mark.parametrize("plan", ["few", "whole", "cut"])
def test_a_sum_of_queries_that_is_a_tie(dim, group, plan):
    """The sum of a query over a group times the scale goes into two fp16: the second has to be the rest of the very first, also where that could be
    rounded either way.  Keys whose minima are large and whose product with the query is small show a step of it."""
    scale, x = _tie(dim ** -0.5)

    def fill(s):
        low = -200 * torch.rand(s.k.shape[0], s.heads, 1, generator=torch.Generator().manual_seed(4))
        s.k[:] = (low * torch.rand(s.k.shape, generator=torch.Generator().manual_seed(5))).half()
        s.k.view(s.k.shape[0], s.heads, -1, s.group)[..., 3:4] = low.half()[..., None]
        s.k.view(s.k.shape[0], s.heads, -1, s.group)[..., 9] = 0
        _whole_numbers(s)
    n = {"few": 24, "whole": 1290, "cut": 300}[plan]
    s = Setup([n], 4, dim, 64, group, F16, fill=fill)
    q = torch.zeros(n, 16, dim)
    q.view(n, 16, -1, group)[..., 9] = x
    q[:, ::3, 9] = -x
    attend(s, [n], 4, {"few": 1100, "whole": n, "cut": 16384}[plan], plan, q=q.half().to(DEV), scale=scale, exact_values=True)


@pytest.mark.parametrize("scale", [1e-8, 1e-6, 1e-4, 0.01, 0.1, 1.3])
@pytest.mark.parametrize("dim,group", [(64, 32), (128, 32), (128, 128), (256, 32)])
@pytest.mark.parametrize("plan", ["few", "cut"])
def test_small_scales_over_large_keys(dim, group, scale, plan):
    """Scores that a small scale brings down from large keys: the minima are as large as the keys, and the scale must not cost their sums a digit."""
    def fill(s):
        g = torch.Generator().manual_seed(1)
        s.k[:] = (torch.randn(s.k.shape, generator=g) * 20000 * torch.rand(s.k.shape[0], s.heads, 1, generator=g)).clamp(-60000, 60000).half()
        _whole_numbers(s)
    s = Setup([300], 4, dim, 64, group, F16, fill=fill)
    n = 24 if plan == "few" else 300
    q = (torch.randn(n, 16, dim, generator=torch.Generator().manual_seed(2)) * min(0.02, 1e-4 / scale)).half().to(DEV)
    attend(s, [n], 4, 1100 if plan == "few" else 16384, plan, q=q, scale=scale, exact_values=True)


def test_a_call_of_many_rows_among_recorded_ones():
    """As it is against the definition, and the same from a graph whose pool a call of few rows shares."""
    s = Setup([5000, 2600], 4, 128, 64, 32, F16, seed=21)
    q, want, rows = attend(s, [700, 500], 4, 5056, "cut")
    few = s.rows([1, 1])
    x = q[:2].clone()
    torch.cuda.synchronize()
    pool, graphs = torch.cuda.graph_pool_handle(), []
    for args, answer in (((q, rows), want), ((x, few), ops.cache_attention(s.cache, x, few))):
        out, graph = torch.zeros_like(answer), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, pool=pool):
            ops.cache_attention(s.cache, *args, out=out)
        graphs.append((graph, out, answer))
    for _ in range(3):
        for graph, out, answer in graphs:
            out.fill_(5)
            graph.replay()
            torch.empty(16 << 20, dtype=torch.uint8, device=DEV).fill_(255)
            torch.cuda.synchronize()
            assert torch.equal(out, answer)
