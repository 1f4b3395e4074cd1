"""Tables of pages that follow the lengths asked for, and the places of a step's rows, on the GPU against the same done one page after the
other.  Everything is whole numbers, and has to be equal."""
import random

import pytest
import torch

from cobalt_amd import KVCache, KVCache8, KVPages, KVRows, _lib, ops
from oracle import cache8_ref as R8
from oracle import cache_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Pair:
    """The tables on the device and the oracle's"""

    def __init__(self, pages, seqs, max_len, page):
        self.pool, self.ref = KVPages(pages, seqs, max_len, page=page, device=DEV), R8.Tables(pages, seqs, max_len, page)

    def resize(self, want):
        rows = ops.cache_pages(self.pool, ints(want))
        starts = self.ref.resize(want)
        assert rows.table is self.pool.table and rows.lens is self.pool.lens
        assert rows.starts.tolist() == starts
        self.check()
        n = starts[-1]
        for count in {n, n + 3, max(n - 2, 0)}:
            slots, positions = ops.cache_slots(self.pool, rows, count)
            assert slots.dtype == torch.int64 and positions.dtype == torch.int32
            want_slots, want_positions = self.ref.slots(starts, count)
            assert slots.tolist() == want_slots and positions.tolist() == want_positions
        return rows

    def check(self):
        assert self.pool.lens.tolist() == self.ref.lens
        assert self.pool.table.tolist() == self.ref.table
        assert self.pool.count.item() == self.ref.count
        assert self.pool.free.tolist() == self.ref.free


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("seqs,max_len", [(1, 1), (1, 5000), (7, 100), (64, 1000), (100, 20000), (1500, 60), (1024, 900), (3000, 300)])
def test_lengths_that_come_and_go(seqs, max_len, page):
    rng = random.Random(seqs * max_len + page)
    per = -(-max_len // page)
    t = Pair(max(1, int(seqs * per * 0.6)), seqs, max_len, page)
    for i in range(8 if seqs < 1000 else 4):
        want = []
        for n in t.ref.lens:
            x = rng.random()
            want.append(0 if x < 0.15 else rng.randint(0, max_len) if x < 0.4 else min(max_len, n + rng.randint(1, 5)) if x < 0.8 else
                        max(0, n - rng.randint(0, 20)) if x < 0.9 else n if x < 0.95 else -1)
        t.resize(want)
    t.resize([0] * seqs)
    assert t.ref.count == t.pool.pages and sorted(t.ref.free) == list(range(t.pool.pages))


def test_pages_come_off_the_stack_in_order():
    t = Pair(10, 3, 100, 16)
    rows = t.resize([20, 0, 33])
    assert rows.table[:, :3].tolist() == [[0, 1, -1], [-1, -1, -1], [2, 3, 4]] and rows.starts.tolist() == [0, 20, 20, 53]
    t.resize([0, 16, 34])                                           # page 0 is on top
    assert t.pool.table[1, 0] == 0 and t.pool.lens.tolist() == [0, 16, 34]
    rows = t.resize([0, 17, 34])
    assert rows.table[1, :2].tolist() == [0, 1] and rows.starts.tolist() == [0, 0, 1, 1]


def test_a_step_and_back_leaves_everything_as_it_was():
    rng = random.Random(3)
    t = Pair(900, 200, 3000, 64)
    t.resize([rng.randint(0, 400) for _ in range(200)])
    keep = [x.clone() for x in t.pool.native()[:4]]
    had = list(t.ref.lens)
    t.resize([max(0, n + rng.randint(-200, 200)) for n in had])
    t.resize(had)
    assert torch.equal(t.pool.table, keep[0]) and torch.equal(t.pool.lens, keep[1]) and torch.equal(t.pool.count, keep[3])
    n = int(keep[3])
    assert torch.equal(t.pool.free[:n], keep[2][:n])


def test_what_the_pool_or_the_table_does_not_hold():
    t = Pair(6, 4, 100, 16)                                         # rows of 7 entries
    t.resize([30, 10, 0, 16])                                       # four pages
    rows = t.resize([30, 30, 40, 20])                               # one, three and one more: the pool has two
    assert t.pool.lens.tolist() == [30, 30, 0, 16] and rows.starts.tolist() == [0, 0, 20, 20, 20]
    t.resize([30, 30, 0, 20])
    t.resize([113, 0, 5, -1])                                       # 113 tokens would be eight pages: refused, alone
    assert t.pool.lens.tolist() == [30, 0, 5, 20]
    t.resize([-1, -7, -(1 << 31), (1 << 31) - 1])
    assert t.pool.lens.tolist() == [30, 0, 5, 20]
    t.resize([0, 100, 0, 0])                                        # what goes back is there for the others of the call: seven, of six
    assert t.pool.lens.tolist() == [0, 0, 0, 0]
    t.resize([0, 96, 0, 0])
    assert t.pool.lens.tolist() == [0, 96, 0, 0] and int(t.pool.count) == 0


def test_lengths_of_the_pool_itself_and_offsets_given():
    t = Pair(10, 3, 100, 16)
    t.resize([20, 5, 33])
    starts = torch.full((4,), 7, dtype=torch.int32, device=DEV)
    rows = ops.cache_pages(t.pool, t.pool.lens, starts=starts)
    assert rows.starts.data_ptr() == starts.data_ptr() and starts.tolist() == [0, 0, 0, 0]
    t.check()


def test_tables_that_do_not_belong_to_their_pool_stay_inside_it():
    t = KVPages(8, 2, 100, page=16, device=DEV)
    guard = [x.numel() for x in t.native()[:4]]
    for lens, count, want in (([100, 100], 8, [0, 0]), ([100, 3], 100, [0, 50]), ([-5, 1 << 30], -3, [100, 0]), ([50, 50], 8, [100, 100])):
        t.lens.copy_(ints(lens))
        t.count.fill_(count)
        t.table.fill_(1 << 30)
        rows = ops.cache_pages(t, ints(want))
        ops.cache_slots(t, rows, 50)
        torch.cuda.synchronize()
        assert 0 <= int(t.count) <= 8
    assert guard == [x.numel() for x in t.native()[:4]]


@pytest.mark.parametrize("seqs,cols,pages", [(2, 7, 8), (300, 20, 50), (200, 50, 900), (1024, 9, 100), (1500, 8, 64), (70000, 3, 1000)])
def test_nothing_around_the_arrays_of_a_table_is_touched(seqs, cols, pages):
    """Lengths, counts, entries and stacks of all kinds, as no pool has them, in one launch and in two: the arrays stand in one buffer, with other numbers between."""
    rng, page, cap = random.Random(seqs), 16, 16 * cols
    sizes = {"table": seqs * cols, "lens": seqs, "free": pages, "count": 1, "starts": seqs + 1, "want": seqs}
    gap, at, place = 64, 64, {}
    for name, n in sizes.items():
        place[name] = (at, at + n)
        at += n + gap
    buffer = torch.full((at,), 0x5a5a5a5a, dtype=torch.int32, device=DEV)
    part = {name: buffer[a:b] for name, (a, b) in place.items()}
    t = KVPages(pages, seqs, cap, page=page, device=DEV)
    t.table, t.lens, t.free, t.count = part["table"].view(seqs, cols), part["lens"], part["free"], part["count"]
    between = torch.ones(at, dtype=torch.bool, device=DEV)
    for a, b in place.values():
        between[a:b] = False
    ends = [-(1 << 31), -1, 0, 1, cap - 1, cap, cap + 1, 1 << 30, (1 << 31) - 1]
    some = lambda n, top: [rng.choice(ends) if rng.random() < 0.3 else rng.randint(0, top) for _ in range(n)]
    entries, stack = ints(some(sizes["table"], pages)), ints(some(pages, pages))
    for count in (pages, 0, -3, pages // 2, 10 * pages, -(1 << 31), (1 << 31) - 1):
        for lens, want in (([cap] * seqs, [0] * seqs), ([0] * seqs, [cap] * seqs), (some(seqs, cap), some(seqs, cap)), ([1] * seqs, some(seqs, 40)), (some(seqs, 40), [-1] * seqs)):
            for name, x in (("lens", ints(lens)), ("want", ints(want)), ("count", ints([count])), ("table", entries), ("free", stack)):
                part[name].copy_(x)
            rows = ops.cache_pages(t, part["want"], starts=part["starts"])
            ops.cache_slots(t, rows, 50)
            assert bool((buffer[between] == 0x5a5a5a5a).all())
            assert part["want"].tolist() == want
            assert 0 <= int(t.count) <= pages and 0 <= int(t.lens.min()) and int(t.lens.max()) <= cap


def test_offsets_of_no_sequences():
    t = KVPages(8, 1, 64, page=16, device=DEV)
    t.table, t.lens = t.table[:0], t.lens[:0]
    starts = torch.full((3,), 7, dtype=torch.int32, device=DEV)
    rows = ops.cache_pages(t, ints([]), starts=starts[:1])
    assert rows.starts.tolist() == [0] and starts.tolist() == [0, 7, 7]
    assert ops.cache_pages(t, ints([])).starts.tolist() == [0] and int(t.count) == 8


def test_slots_of_rows_of_all_kinds():
    table = ints([[3, 1, -1, 70], [0, 2, 9, -5], [4, 5, 6, 7]])
    pool = KVPages(8, 3, 64, page=16, device=DEV)
    rows = KVRows(table, ints([60, 2, 70]), ints([2, 32, 37, 49]))
    slots, positions = ops.cache_slots(pool, rows, 52)
    want_s, want_p = [-1] * 52, [0] * 52
    for b, (n, s0, s1) in enumerate([(60, 2, 32), (2, 32, 37), (70, 37, 49)]):
        for x in range(s0, s1):
            j = n - (s1 - x)
            want_p[x] = max(j, 0)
            page = table[b, j // 16].item() if 0 <= j < 64 else -1
            want_s[x] = page * 16 + j % 16 if 0 <= page < 8 else -1
    assert slots.tolist() == want_s and positions.tolist() == want_p
    # equally many each, none at all, more than a workgroup has
    s, p = ops.cache_slots(pool, KVRows(table, ints([5, 20, 64])), 9)
    assert s.tolist() == [50, 51, 52, 33, 34, 35, 125, 126, 127] and p.tolist() == [2, 3, 4, 17, 18, 19, 61, 62, 63]
    assert ops.cache_slots(pool, KVRows(table, ints([5, 20, 64])), 0)[0].shape == (0,)
    s, p = ops.cache_slots(pool, KVRows(table[:0], ints([]), ints([0])), 5000)
    assert bool((s == -1).all()) and not bool(p.any())


@pytest.mark.parametrize("seqs", [1, 3, 600, 20000])
def test_slots_of_many_rows(seqs):
    g = torch.Generator().manual_seed(seqs)
    n = torch.randint(0, 200000 // seqs + 2, (seqs,), generator=g) * (torch.rand(seqs, generator=g) < 0.7)
    lens = n + torch.randint(0, 300, (seqs,), generator=g)
    cols = -(-int(lens.max()) // 64) if int(lens.max()) else 1
    table = torch.randint(0, 1 << 20, (seqs, cols), generator=g, dtype=torch.int32)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)])
    total = int(starts[-1])
    b = torch.repeat_interleave(torch.arange(seqs), n)
    j = lens[b] - n[b] + torch.arange(total) - starts[b]
    want = table[b, j // 64].long() * 64 + j % 64
    pool = KVPages(1 << 20, 1, 64, page=64, device=DEV)
    s, p = ops.cache_slots(pool, KVRows(table.to(DEV), lens.int().to(DEV), starts.int().to(DEV)), total + 11)
    assert torch.equal(s[:total].cpu(), want) and torch.equal(p[:total].cpu(), j.int())
    assert bool((s[total:] == -1).all()) and not bool(p[total:].any())


def test_places_beyond_32_bits():
    pool = KVPages(1 << 24, 1, 1 << 20, page=256, device=DEV)
    table = torch.full((1, 4096), (1 << 24) - 1, dtype=torch.int32, device=DEV)
    s, p = ops.cache_slots(pool, KVRows(table, ints([1 << 20]), ints([0, 2])), 2)
    assert s.tolist() == [(((1 << 24) - 1) << 8) + 254, (((1 << 24) - 1) << 8) + 255] and p.tolist() == [(1 << 20) - 2, (1 << 20) - 1]


@pytest.mark.parametrize("kind", ["4bit", "8bit"])
def test_requests_through_tables_cache_and_attention(kind):
    """A server's life on one pool: requests come, decode, are cut back and end; every step's attention against the definition over what
    the pool held for it."""
    g, rng = torch.Generator().manual_seed(1), random.Random(1)
    heads, dim, page = 2, 64, 16
    tables = KVPages(40, 5, 200, page=page, device=DEV)
    cache = KVCache(40, heads, dim, page=page, device=DEV) if kind == "4bit" else KVCache8(40, heads, dim, page=page, device=DEV)
    ref = R8.Tables(40, 5, 200, page)
    text = [[], [], [], [], []]                                     # every token's (key, value)
    for step in range(12):
        want = []
        for b in range(5):
            x = rng.random()
            want.append(rng.randint(1, 150) if not text[b] else 0 if x < 0.15 else max(1, len(text[b]) - rng.randint(1, 4)) if x < 0.3 else
                        len(text[b]) + 1)
        rows = ops.cache_pages(tables, ints(want))
        starts = ref.resize(want)
        k, v = (torch.randn(starts[-1], heads, dim, generator=g).half() for _ in range(2))
        for b in range(5):
            text[b] = text[b][:ref.lens[b]] + [(k[t], v[t]) for t in range(starts[b], starts[b + 1])]
            assert len(text[b]) == ref.lens[b]
        ops.cache_write(cache, k.to(DEV), v.to(DEV), rows)
        q = torch.randn(starts[-1], 4, dim, generator=g).half()
        out = ops.cache_attention(cache, q.to(DEV), rows)
        slots, positions = ops.cache_slots(cache, rows, starts[-1])
        assert positions.tolist() == ref.slots(starts, starts[-1])[1]
        for b in range(5):
            n, new = ref.lens[b], starts[b + 1] - starts[b]
            if not n:
                continue
            hk, hv = (x.cpu().double().numpy() for x in ops.cache_read(cache, KVRows(tables.table[b:b + 1].contiguous(), ints([n]), ints([0, n])), n, torch.float32))
            for x, i in ((hk, 0), (hv, 1)):                         # what is held is near what was written
                y = torch.stack([t[i] for t in text[b]]).double().numpy()
                assert abs(x - y).max() < (0.4 if kind == "4bit" else 0.26)
            for h in range(4):
                at = slice(starts[b], starts[b + 1])
                o, spread, size, reach = R8.attention(q[at, h].double().numpy(), hk[:, h // 2], hv[:, h // 2], range(n - new, n), abs(hk[:, 0, 0]) >= 0, 0.125)
                assert (abs(out[at, h].double().cpu().numpy() - o) <= 0.002 * (1 + abs(o))).all()
    assert tables.table.tolist() == ref.table


@pytest.mark.parametrize("kind", ["4bit", "8bit"])
@pytest.mark.parametrize("lens,starts,counts", [([40, 70, 33], [0, 5, 30, 42], [36, 20, 5, 3, 41]), ([40, 70, 33], [-3, 5, 30, 42], [36, 42]),
                                                ([350, 400, 330], [0, 300, 620, 930], [800, 450, 929]), ([7, 40, 20], [0, 12, 30, 70], [50, 69])])
def test_rows_that_the_call_does_not_have(kind, lens, starts, counts):
    """Offsets that end behind the call's rows: those that are there are written, read and attended over as the tokens that `cache_slots` names."""
    heads, dim, page = 2, 64, 16
    per = [-(-n // page) for n in lens]
    cols = max(per) + 1
    table = [[sum(per[:b]) + i if i < per[b] else -1 for i in range(cols)] for b in range(len(lens))]
    make = (lambda: KVCache(sum(per), heads, dim, page=page, device=DEV)) if kind == "4bit" else (lambda: KVCache8(sum(per), heads, dim, page=page, device=DEV))
    rows = KVRows(ints(table), ints(lens), ints(starts))
    full = KVRows(rows.table, rows.lens, ints([0, lens[0], lens[0] + lens[1], sum(lens)]))
    bits = 1 << torch.arange(dim) % 10
    named = lambda n: 1.0 + ((torch.arange(n)[:, None, None] & bits) != 0).expand(n, heads, dim).half()      # a row's number in its channels, 1 and 2
    number = lambda x: ((x.cpu()[..., :10] > 1.5) * bits[:10]).sum(-1) - (x.cpu()[..., 0] < 0.5).int()       # (nothing held: -1)
    first = torch.zeros(sum(lens), heads, dim)                      # values: 1 for each sequence's first token, of its mean a row tells how many it sees
    first[[0, lens[0], lens[0] + lens[1]]] = 1
    whole = make()
    ops.cache_write(whole, torch.zeros(sum(lens), heads, dim).half().to(DEV), first.half().to(DEV), full)
    for n in counts:
        want = [-1] * sum(lens)
        pos = []
        for t in range(n):
            b = max(i for i in range(3) if starts[i] <= t)
            pos.append(lens[b] - (starts[b + 1] - t))
            if pos[-1] >= 0:
                want[sum(lens[:b]) + pos[-1]] = t
        slots, positions = ops.cache_slots(whole, rows, n)
        assert positions.tolist() == [max(j, 0) for j in pos]
        cache = make()
        x = named(n).to(DEV)
        ops.cache_write(cache, x, x, rows)
        for held in ops.cache_read(cache, full, sum(lens), torch.float32):
            assert number(held).tolist() == [[w, w] for w in want]
        for held in ops.cache_read(cache, rows, n, torch.float32):
            assert number(held).tolist() == [[t if j >= 0 else -1] * heads for t, j in enumerate(pos)]
        for ratio in (1, 16):                                       # few rows a sequence, and many
            out = ops.cache_attention(whole, torch.zeros(n, heads * ratio, dim).half().to(DEV), rows).double().cpu()
            seen = torch.where(out > 0, 1 / out.clamp(min=1e-9), torch.zeros_like(out))
            # 1 / (pos + 1), of weights and a result that fp16 rounds: 2^-10 off at most, of 400 less than a half
            assert torch.equal(seen.round().long(), torch.tensor([max(j + 1, 0) for j in pos])[:, None, None].expand_as(out))


def test_a_recorded_step_takes_pages_as_it_grows():
    tables = KVPages(30, 3, 120, page=16, device=DEV)
    ref = R8.Tables(30, 3, 120, 16)
    want = ints([30, 1, 15])
    ops.cache_pages(tables, want)
    ref.resize([30, 1, 15])

    def step():
        want.add_(1)
        rows = ops.cache_pages(tables, want)
        return rows.starts, *ops.cache_slots(tables, rows, 4)
    keep = [x.clone() for x in (*tables.native()[:4], want)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y in zip((*tables.native()[:4], want), keep):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        starts, slots, positions = step()
    for i in range(100):
        graph.replay()
        if i % 7 == 0:
            torch.empty(1 << 20, dtype=torch.uint8, device=DEV).fill_(255)
        if i == 40:                                                 # an eager step between
            torch.cuda.synchronize()
            ref_starts = ref.resize(want.tolist())
            step()
        s = ref.resize(want.tolist())
        assert starts.tolist() == s if i != 40 else True
        assert tables.table.tolist() == ref.table and tables.lens.tolist() == ref.lens
        if i != 40:
            assert (slots.tolist(), positions.tolist()) == ref.slots(s, 4)


def test_refusals():
    t = KVPages(10, 3, 100, page=16, device=DEV)
    lens = ints([1, 2, 3])
    with pytest.raises(_lib.CbkError):
        ops.cache_pages(t, lens.cpu())
    with pytest.raises(TypeError):
        ops.cache_pages(t, lens.long())
    with pytest.raises(ValueError):
        ops.cache_pages(t, lens[:2])
    with pytest.raises(ValueError):
        ops.cache_pages(t, lens, starts=ints([0, 0, 0]))
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_pages(t, lens, starts=t.table.view(-1)[:4])
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_pages(t, t.free[:3])
    both = torch.zeros(4, dtype=torch.int32, device=DEV)
    t.lens = both[:3]
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_pages(t, both[1:])
    with pytest.raises(ValueError, match="unit stride"):
        ops.cache_pages(t, ints([1, 2, 3, 4, 5, 6])[::2])
    rows = ops.cache_pages(t, lens)
    with pytest.raises(ValueError):
        ops.cache_slots(t, rows, -1)
    with pytest.raises(_lib.CbkError):
        ops.cache_slots(t, rows._replace(lens=rows.lens.cpu()), 3)
    with pytest.raises(TypeError):
        ops.cache_slots(t, rows._replace(lens=rows.lens.long()), 3)
    with pytest.raises(ValueError):
        ops.cache_slots(t, rows._replace(starts=None), 4)
    t.free = t.free[:-1]
    with pytest.raises(ValueError, match="do not hold"):
        ops.cache_pages(t, lens)
