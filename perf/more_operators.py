"""What the operators of the 8-bit key/value cache and of its page tables are measured on, and the same operators in
plain torch.

A case names a use:

  write    the newest tokens of every sequence go into the cache, and the blocks they stand in come back as the values
           the cache then holds for them (older tokens of a block follow its scale)
  read     tokens that are in the cache, as dense tensors
  attend   attention of the newest tokens, which the cache holds too: one token a sequence, a few, or a prompt
  pages    requests come, grow, lose rejected drafts and end: the table of every sequence's pages follows the lengths
           asked for, and, so that a pass finds what the last one found, goes back to the lengths before
  slots    where the rows of a step go, as places of the pool, and their positions

Caches: `seqs` sequences whose lengths are spread over `length` and whose newest tokens (the rows of the call) over `new`
(0: all of them), `q_heads` query heads on `heads` cache heads of `dim` channels, `page` tokens a page, `block` tokens a
scale, `window` (0: none) and `sinks` of the visible range.  Tables: of `seqs` sequences a share `done` ends, a share
`fresh` begins, the others gain `new` tokens or, a share `back`, lose some; `room` is the pool's size against
what the longest of the two states needs (below 1: some requests find no pages).  Slots: `pad` rows behind the last sequence's.

Head counts and head sizes are those of the benchmark's Mistral-7B and Gemma-3-27B shaped layers (32 and 8,
32 and 16, 128 channels), of the tests' small decoder (4 and 2, 64 channels), and 256 channels; lengths are generic.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
TOP = 57344.0                                                       # larger magnitudes are held as this one
LEAST, MOST = -15, 7                                                # exponents of a block's scale


def _cache(name, use, seqs, length, new, heads, q_heads, dim, page, block, dtype, window=0, sinks=0, lens_seed=0):
    return dict(name=name, use=use, seqs=seqs, length_lo=length[0], length_hi=length[1], new_lo=new[0], new_hi=new[1],
                heads=heads, q_heads=q_heads, dim=dim, page=page, block=block, dtype=dtype, window=window, sinks=sinks,
                lens_seed=lens_seed)


def _pages(name, seqs, length, new, page, done, fresh, back, room, lens_seed=0):
    return dict(name=name, use="pages", seqs=seqs, length_lo=length[0], length_hi=length[1], new_lo=new[0], new_hi=new[1],
                page=page, done=done, fresh=fresh, back=back, room=room, lens_seed=lens_seed)


def _slots_case(name, seqs, length, new, page, pad, lens_seed=0):
    return dict(name=name, use="slots", seqs=seqs, length_lo=length[0], length_hi=length[1], new_lo=new[0], new_hi=new[1],
                page=page, pad=pad, lens_seed=lens_seed)


def listed():
    return [
        # one decode step's keys and values of 32 sequences: the cost of the calls themselves
        _cache("write_step", "write", 32, (1, 4000), (1, 1), 8, 32, 128, 64, 16, "f16", lens_seed=1),
        # chunks of prompts of odd lengths enter the cache, most in the middle of a block
        _cache("write_chunks", "write", 8, (3000, 9000), (1000, 6000), 8, 32, 128, 64, 32, "bf16", lens_seed=2),
        # long prefixes handed to a program that wants them dense
        _cache("read_long", "read", 2, (30000, 50000), (0, 0), 16, 32, 128, 128, 128, "bf16", lens_seed=3),
        # one sequence, one token, a short history: latency alone
        _cache("attend_one", "attend", 1, (700, 700), (1, 1), 8, 32, 128, 64, 16, "f16"),
        # a decode step of a serving batch with histories of all lengths
        _cache("attend_batch", "attend", 32, (1, 8192), (1, 1), 8, 32, 128, 64, 16, "bf16", lens_seed=5),
        # two very long histories: too few rows to fill the chip without cutting the length
        _cache("attend_long", "attend", 2, (100000, 140000), (1, 1), 8, 32, 128, 256, 64, "f16", lens_seed=6),
        # a few drafted tokens of each sequence checked at once, wide heads, a window with four first tokens kept
        _cache("attend_draft", "attend", 12, (300, 9000), (2, 6), 4, 16, 256, 32, 32, "bf16", 2048, 4, lens_seed=7),
        # a whole prompt of a layer
        _cache("attend_prompt", "attend", 1, (4096, 4096), (4096, 4096), 8, 32, 128, 64, 16, "bf16"),
        # a decode step of a small serving batch: two requests end, two begin, the others gain a token
        _pages("pages_step", 32, (1, 4000), (1, 1), 64, 0.06, 0.06, 0.0, 1.5, lens_seed=9),
        # a large batch turns over: long prompts come in, drafts are taken back, the pool is short of pages
        _pages("pages_turnover", 1024, (1, 60000), (1, 8), 16, 0.15, 0.15, 0.2, 0.97, lens_seed=10),
        # places and positions of one token of every sequence, in a step recorded for more rows than it has
        _slots_case("slots_step", 48, (1, 4000), (1, 1), 64, 16, lens_seed=11),
        # and of many prompts of all lengths
        _slots_case("slots_prompts", 500, (1, 4000), (0, 0), 16, 0, lens_seed=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        use = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend", "pages", "pages", "slots"])
        hi = _log(rng, 1, 140000)
        lo = hi if rng.random() < 0.2 else max(1, int(hi * rng.random()))
        if use == "pages":
            seqs = _log(rng, 1, 4096)
            new = (1, 1) if rng.random() < 0.5 else (1, _log(rng, 2, 64))
            case = _pages("", seqs, (lo, hi), new, rng.choice([16, 32, 64, 128, 256]), round(0.3 * rng.random(), 2),
                          round(0.3 * rng.random(), 2), rng.choice([0.0, round(0.5 * rng.random(), 2)]),
                          rng.choice([0.9, 1.0, 1.2, 2.0]), rng.randrange(1 << 20))
            if work(case)["bytes"] <= 3e7:
                del case["name"]
                return case
            continue
        kind = rng.choice(["one", "one", "few", "chunk", "all"]) if use != "read" else rng.choice(["chunk", "all"])
        if kind == "one":
            new = (1, 1)
        elif kind == "few":
            new = (1, rng.randint(2, 8))
        elif kind == "chunk":
            n = _log(rng, 8, 4096)
            new = (max(1, int(n * rng.random())), n)
        else:
            new = (0, 0)
        page = rng.choice([16, 32, 64, 128, 256])
        if use == "slots":
            case = _slots_case("", _log(rng, 1, 4096), (lo, hi), new, page, rng.choice([0, 0, _log(rng, 1, 512)]), rng.randrange(1 << 20))
            lens = _lengths(case)
            if sum(r for _, r in lens) <= 1000000 and sum(n for n, _ in lens) <= 4e7:
                del case["name"]
                return case
            continue
        dim = rng.choice([64, 128, 128, 128, 256])
        heads = rng.choice([1, 2, 4, 8, 8, 16])
        ratio = rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
        block = rng.choice([b for b in (16, 32, 64, 128, 256) if b <= page])
        window, sinks = 0, 0
        if use == "attend" and rng.random() < 0.35:
            window, sinks = _log(rng, 16, 8192), rng.choice([0, 1, 4, 64])
        case = _cache("", use, _log(rng, 1, 64), (lo, hi), new, heads, heads * ratio, dim, page, block, rng.choice(["f16", "bf16"]), window,
                      sinks, rng.randrange(1 << 20))
        del case["name"]
        rows = sum(n for _, n in _lengths(case))
        held = sum(n for n, _ in _lengths(case)) * heads * dim
        if rows <= 20000 and rows * case["q_heads"] * dim <= 8e7 and held <= 2.4e8 and work(case)["flops"] <= 1.3e11:
            return case


# ------------------------------------------------------------------ shapes
def _lengths(case):
    """(length, rows) of every sequence: a property of the case, so that its work does not change with the seed."""
    rng = random.Random(case["lens_seed"])
    out = []
    for _ in range(case["seqs"]):
        n = rng.randint(case["length_lo"], case["length_hi"])
        out.append((n, min(n, rng.randint(case["new_lo"], case["new_hi"])) if case["new_hi"] else n))
    return out


def _requests(case):
    """(length, length asked for) of every sequence, pages of the pool, tokens that a sequence's table has room for."""
    rng = random.Random(case["lens_seed"])
    out = []
    for _ in range(case["seqs"]):
        n, x, gain = rng.randint(case["length_lo"], case["length_hi"]), rng.random(), rng.randint(case["new_lo"], case["new_hi"])
        if x < case["done"]:
            out.append((n, 0))
        elif x < case["done"] + case["fresh"]:
            out.append((0, n))
        elif x < case["done"] + case["fresh"] + case["back"]:
            out.append((n, max(0, n - gain)))
        else:
            out.append((n, n + gain))
    need = lambda i: sum(-(-x[i] // case["page"]) for x in out)
    pages = max(need(0), int(max(need(0), need(1)) * case["room"]), 1)      # (the state before has its pages)
    return out, pages, case["length_hi"] + case["new_hi"]


def _visible(length, rows, window, sinks):
    """Keys that the newest `rows` tokens of a sequence see, summed, and how many different ones there are."""
    first = length - rows
    if not window:
        return rows * first + rows * (rows + 1) // 2, length
    pairs = 0
    for p in range(first, length):
        lo = max(0, p + 1 - window)
        pairs += p + 1 - lo + min(lo, sinks)
    lo = max(0, first + 1 - window)
    return pairs, length - lo + min(lo, sinks)


def _touched(lens, block):
    """(length, tokens from the beginning of the first block that a sequence's newest rows stand in)."""
    return [(n, n - (n - r) // block * block) for n, r in lens]


def work(case):
    if case["use"] == "pages":
        reqs, pages, most = _requests(case)
        moved = sum(abs(-(-a // case["page"]) - -(-b // case["page"])) for a, b in reqs)
        table = case["seqs"] * -(-most // case["page"])
        # twice: lengths in and out, starts, a page moved is read and written; once: the table between the two is handed out
        return {"bytes": 2 * (4 * 4 * case["seqs"] + 8 * moved) + 8 * table, "flops": 0}
    lens = _lengths(case)
    rows = sum(n for _, n in lens)
    if case["use"] == "slots":
        held = sum(-(-n // case["page"]) - (n - r) // case["page"] for n, r in lens)
        return {"bytes": 12 * (rows + case["pad"]) + 8 * case["seqs"] + 4 * held, "flops": 0}
    token = 2 * case["heads"] * case["dim"]                                              # bytes of a token in the cache, but for the scales
    scale = 2 * case["heads"] * 4 / case["block"]
    dense = 2 * case["heads"] * case["dim"] * 2                                          # of its keys and values in 16 bits
    if case["use"] == "write":
        back = sum(n for _, n in _touched(lens, case["block"]))
        return {"bytes": int(rows * (dense + token + scale) + back * (dense + token + scale)), "flops": 0}
    if case["use"] == "read":
        return {"bytes": int(sum(n for _, n in _touched(lens, case["block"])) * (dense + token + scale)), "flops": 0}
    seen = [_visible(n, r, case["window"], case["sinks"]) for n, r in lens]
    size = sum(k for _, k in seen) * (token + scale) + 2 * rows * case["q_heads"] * case["dim"] * 2
    return {"bytes": int(size), "flops": 4 * case["q_heads"] * case["dim"] * sum(p for p, _ in seen)}


# ------------------------------------------------------------------ inputs
def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def _table(case, lens, g):
    """Pages are handed out in no order; the table's unused entries hold no page."""
    need = [-(-n // case["page"]) for n, _ in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _inputs(case, seed):
    """Keys have channels of different magnitude and a few outliers, as behind a rotary embedding."""
    g = torch.Generator(device=DEV).manual_seed(1000 * seed + 17)
    dt, H, D = TYPES[case["dtype"]], case["heads"], case["dim"]
    lens = _lengths(case)
    total, rows = sum(n for n, _ in lens), sum(r for _, r in lens)
    channel = torch.exp(0.4 * torch.randn(H, D, generator=g, device=DEV))
    channel[:, torch.randint(0, D, (max(1, D // 64),), generator=g, device=DEV)] *= 6.0
    k = torch.empty(total, H, D, dtype=dt, device=DEV)
    v = torch.empty(total, H, D, dtype=dt, device=DEV)
    for i in range(0, total, 32768):
        n = min(32768, total - i)
        k[i:i + n] = torch.randn(n, H, D, generator=g, device=DEV) * channel
        v[i:i + n] = torch.randn(n, H, D, generator=g, device=DEV)
    q = torch.randn(rows, case["q_heads"], D, generator=g, device=DEV).to(dt)
    table, pages = _table(case, lens, g)
    return dict(k=k, v=v, q=q, table=table, pages=pages, lens=lens)


def _cut(counts):
    """Offsets of sequences that are packed one behind the other."""
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def _newest(lens):
    """Positions of the newest rows among all tokens, packed sequence behind sequence."""
    whole = _cut([n for n, _ in lens])
    return torch.cat([torch.arange(whole[b + 1] - r, whole[b + 1], device=DEV) for b, (_, r) in enumerate(lens)])


def _lives(case, seed):
    """Lengths that the sequences had before, so that the pool's pages lie in no order."""
    rng = random.Random(seed)
    return [rng.randint(0, n) for n, _ in _requests(case)[0]]


def prepare(case, seed):
    if case["use"] == "pages":
        return _prepare_pages(case, seed)
    if case["use"] == "slots":
        g = torch.Generator(device=DEV).manual_seed(1000 * seed + 17)
        lens = _lengths(case)
        table, pages = _table(case, lens, g)
        st = dict(case=case, table=table, pages=pages, tokens=_ints([n for n, _ in lens]), starts=_ints(_cut([r for _, r in lens])),
                  count=sum(r for _, r in lens) + case["pad"])
        if own:
            from cobalt_amd import KVPages, KVRows
            st["pool"] = KVPages(pages, len(lens), case["length_hi"], page=case["page"], device=DEV)
            st["rows"] = KVRows(table, st["tokens"], st["starts"])
        return st
    x = _inputs(case, seed)
    lens = x["lens"]
    st = dict(case=case, lens=lens, q=x["q"], table=x["table"])
    newest = _newest(lens)
    st["k"], st["v"] = x["k"][newest], x["v"][newest]
    st["tokens"], st["starts"] = _ints([n for n, _ in lens]), _ints(_cut([r for _, r in lens]))
    # what the cache holds before: everything, or, of a write, all but the newest tokens
    before = [(n - r, n - r) if case["use"] == "write" else (n, n) for n, r in lens]
    older = torch.ones(x["k"].shape[0], dtype=torch.bool, device=DEV)
    if case["use"] == "write":
        older[newest] = False
    if own:
        from cobalt_amd import KVCache8, KVRows, ops
        st["cache"] = KVCache8(x["pages"], case["heads"], case["dim"], page=case["page"], block=case["block"], device=DEV)
        st["rows"] = KVRows(st["table"], st["tokens"], st["starts"])
        back = [r for _, r in _touched(lens, case["block"])]
        st["back"], st["count"] = KVRows(st["table"], st["tokens"], _ints(_cut(back))), sum(back)
        if sum(n for n, _ in before):
            ops.cache_write(st["cache"], x["k"][older], x["v"][older],
                            KVRows(st["table"], _ints([n for n, _ in before]), _ints(_cut([n for n, _ in before]))))
    else:
        slots, H, D = x["pages"] * case["page"], case["heads"], case["dim"]
        for name in ("k", "v"):
            st[name + "_codes"] = torch.zeros(slots, H, D, dtype=torch.uint8, device=DEV)
            st[name + "_scale"] = torch.zeros(slots // case["block"], H, device=DEV)
            whole = _cut([n for n, _ in lens])
            for b, (n, _) in enumerate(before):
                for i in range(0, n, 32768):                                # (whole blocks)
                    at = torch.arange(i, min(n, i + 32768), device=DEV)
                    _store(st, name, _slots(st, b, at), at, x[name][whole[b] + at])
    return st


# ------------------------------------------------------------------ plain form: the cache
def _slots(st, b, positions):
    page = st["case"]["page"]
    return st["table"][b][positions // page].long() * page + positions % page


def _scale(top):
    """The smallest power of two s with top <= 448 s, in the scales' range."""
    m, e = torch.frexp(top)
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(top == 0, torch.full_like(e, LEAST), e).clamp(LEAST, MOST)
    return torch.ldexp(torch.ones_like(top), e)


def _codes(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _store(st, name, slots, positions, x):
    """A block's scale grows with what comes in, and the codes of its older tokens follow; with its first token it begins anew."""
    block, codes, scale = st["case"]["block"], st[name + "_codes"], st[name + "_scale"]
    f = x.float().clamp(-TOP, TOP)
    which, place = torch.unique(slots // block, return_inverse=True)
    top = torch.zeros(which.numel(), f.shape[1], device=DEV)
    top.scatter_reduce_(0, place[:, None].expand(-1, f.shape[1]), f.abs().amax(-1), "amax")
    anew = torch.zeros(which.numel(), dtype=torch.bool, device=DEV)
    anew[place[positions % block == 0]] = True
    was = scale[which].masked_fill(anew[:, None], 0.0)
    now = torch.maximum(was, _scale(top))
    older = which[:, None] * block + torch.arange(block, device=DEV)
    codes[older] = _codes(_values(codes[older]) * (was / now)[:, None, :, None])
    scale[which] = now
    codes[slots] = _codes(f / now[place][:, :, None])


def _load(st, name, slots):
    return _values(st[name + "_codes"][slots]) * st[name + "_scale"][slots // st["case"]["block"]][:, :, None]


def _plain_attend(st):
    c = st["case"]
    H, R, D, dt = c["heads"], c["q_heads"] // c["heads"], c["dim"], TYPES[c["dtype"]]
    out, at = [], 0
    for b, (n, rows) in enumerate(st["lens"]):
        first = n - rows
        for r0 in range(0, rows, 1024):
            r1 = min(rows, r0 + 1024)
            p = torch.arange(first + r0, first + r1, device=DEV)
            lo = max(0, first + r0 + 1 - c["window"]) if c["window"] else 0
            j = torch.arange(lo, first + r1, device=DEV)
            if lo:
                j = torch.cat([torch.arange(min(lo, c["sinks"]), device=DEV), j])
            slots = _slots(st, b, j)
            k, v = _load(st, "k", slots).transpose(0, 1), _load(st, "v", slots).transpose(0, 1).contiguous()   # [H, keys, D]
            q = st["q"][at + r0:at + r1].float().view(r1 - r0, H, R, D).permute(1, 2, 0, 3).reshape(H, R * (r1 - r0), D)
            s = torch.matmul(q, k.transpose(1, 2).contiguous()) * (D ** -0.5)
            seen = j[None, :] <= p[:, None]
            if c["window"]:
                seen &= (j[None, :] > p[:, None] - c["window"]) | (j[None, :] < c["sinks"])
            s = s.view(H, R, r1 - r0, -1).masked_fill(~seen, float("-inf"))
            e = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(e.view(H, R * (r1 - r0), -1), v).view(H, R, r1 - r0, D) / e.sum(-1, keepdim=True)
            out.append(o.permute(2, 0, 1, 3).reshape(r1 - r0, H * R, D).to(dt))
        at += rows
    return torch.cat(out)


# ------------------------------------------------------------------ plain form: tables and slots
def _prepare_pages(case, seed):
    reqs, pages, most = _requests(case)
    st = dict(case=case, had=_ints([a for a, _ in reqs]), want=_ints([b for _, b in reqs]))
    if own:
        from cobalt_amd import KVPages, ops
        st["pool"] = KVPages(pages, len(reqs), most, page=case["page"], device=DEV)
        ops.cache_pages(st["pool"], _ints(_lives(case, seed)))
        ops.cache_pages(st["pool"], st["had"])
    else:
        st["table"] = torch.full((len(reqs), -(-most // case["page"])), -1, dtype=torch.int32, device=DEV)
        st["lens"] = torch.zeros(len(reqs), dtype=torch.int32, device=DEV)
        st["free"] = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=DEV)      # the last one is handed out first
        st["count"] = _ints([pages])
        _plain_pages(st, _ints(_lives(case, seed)))
        _plain_pages(st, st["had"])
    return st


def _spread(counts):
    """(sequence, number within it) of `counts` things of every sequence, one behind the other."""
    b = torch.repeat_interleave(torch.arange(counts.numel(), device=DEV), counts)
    return b, torch.arange(b.numel(), device=DEV) - (torch.cumsum(counts, 0) - counts)[b]


def _plain_pages(st, want):
    """Pages that sequences no longer need go back on the stack, the first one on top; then sequences take theirs from the top, in
    order, those for which the pages last.  Returns where the new rows of each begin."""
    page, table, lens, free = st["case"]["page"], st["table"], st["lens"].long(), st["free"]
    want = want.long()
    have, need = (lens + page - 1) // page, (want + page - 1) // page
    gone, more = (have - need).clamp(min=0), (need - have).clamp(min=0)
    count = st["count"][0].long() + gone.sum()
    b, i = _spread(gone)
    free[count - 1 - torch.arange(b.numel(), device=DEV)] = table[b, need[b] + i]
    table[b, need[b] + i] = -1
    served = (torch.cumsum(more, 0) <= count) | (more == 0)
    more = more * served
    b, i = _spread(more)
    table[b, have[b] + i] = free[count - 1 - torch.arange(b.numel(), device=DEV)]
    now = torch.where(served, want, lens)
    st["lens"].copy_(now)
    st["count"][0] = count - more.sum()
    starts = torch.zeros(lens.numel() + 1, dtype=torch.int32, device=DEV)
    starts[1:] = torch.cumsum((now - lens).clamp(min=0), 0)
    return starts


def _plain_slots(st):
    page, starts, lens = st["case"]["page"], st["starts"].long(), st["tokens"].long()
    t = torch.arange(st["count"], device=DEV)
    b = torch.searchsorted(starts, t, right=True) - 1
    none = b >= lens.numel()
    b = b.clamp(max=lens.numel() - 1)
    pos = (lens - starts[1:])[b] + t
    p = pos.masked_fill(none, 0)
    slots = st["table"][b, p // page].long() * page + p % page
    return slots.masked_fill(none, -1), p.int()


# ------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    use = c["use"]
    if use == "pages":
        return _run_pages(state)
    if own:
        from cobalt_amd import ops
        if use == "slots":
            return ops.cache_slots(state["pool"], state["rows"], state["count"])
        if use == "write":
            ops.cache_write(state["cache"], state["k"], state["v"], state["rows"])
        if use in ("write", "read"):
            return ops.cache_read(state["cache"], state["back"], state["count"], TYPES[c["dtype"]])
        return ops.cache_attention(state["cache"], state["q"], state["rows"], window=c["window"] or None, sinks=c["sinks"])
    if use == "slots":
        return _plain_slots(state)
    if use == "attend":
        return _plain_attend(state)
    lens = state["lens"]
    if use == "write":
        at = [torch.arange(n - r, n, device=DEV) for n, r in lens]
        slots, at = torch.cat([_slots(state, b, a) for b, a in enumerate(at)]), torch.cat(at)
        _store(state, "k", slots, at, state["k"])
        _store(state, "v", slots, at, state["v"])
    slots = torch.cat([_slots(state, b, torch.arange(n - r, n, device=DEV)) for b, (n, r) in enumerate(_touched(lens, c["block"]))])
    return _load(state, "k", slots).to(TYPES[c["dtype"]]), _load(state, "v", slots).to(TYPES[c["dtype"]])


def _run_pages(st):
    """The table and the lengths asked for, as a copy: the state goes back to where it was."""
    if own:
        from cobalt_amd import ops
        pool = st["pool"]
        rows = ops.cache_pages(pool, st["want"])
        there = pool.table.clone(), pool.lens.clone(), rows.starts
        back = ops.cache_pages(pool, st["had"])
        return (*there, pool.table, pool.lens, pool.free, pool.count, back.starts)
    starts = _plain_pages(st, st["want"])
    there = st["table"].clone(), st["lens"].clone(), starts
    back = _plain_pages(st, st["had"])
    return (*there, st["table"], st["lens"], st["free"], st["count"], back)


# ------------------------------------------------------------------ the definition in 64 bits
def _rounded(x):
    """x to three bits behind the first one, steps of 2^-9 at least, ties to even."""
    e = torch.floor(torch.log2(torch.clamp(x.abs(), min=2.0 ** -30))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(x / step) * step


def _exponent(top):
    """The least e with top <= 448 * 2^e, by trying them."""
    e = torch.full_like(top, LEAST)
    for i in range(LEAST, MOST):
        e = torch.where(top > 448.0 * 2.0 ** i, torch.full_like(e, i + 1), e)
    return e


def _held(x, block, new):
    """The values the cache holds for the tokens x [tokens, H, D] of one sequence, in float64: all but the newest `new` written at
    once, then those."""
    n, H, D = x.shape
    blocks = -(-n // block)
    f = torch.zeros(blocks * block, H, D, dtype=torch.float64, device=x.device)
    f[:n] = x.double().clamp(-TOP, TOP)
    late = torch.arange(blocks * block, device=x.device) >= n - new
    size = f.abs().amax(2)
    tops = lambda mask: (size * mask[:, None]).view(blocks, block, H).amax(1)                    # [blocks, H]
    e0, e1 = _exponent(tops(~late)), _exponent(tops(late))
    some = late.view(blocks, block)
    e1 = torch.where(some[:, :1], e1, torch.where(some.any(1, keepdim=True), torch.maximum(e0, e1), e0))
    wide = lambda e: torch.exp2(e).repeat_interleave(block, 0)[:, :, None]
    s0, s1 = wide(e0), wide(e1)
    old = _rounded(_rounded(f / s0) * (s0 / s1)) * s1
    return torch.where(late[:, None, None], _rounded(f / s1) * s1, old)[:n]


def exact(case, seed):
    if case["use"] == "pages":
        return _exact_pages(case, seed)
    if case["use"] == "slots":
        return _exact_slots(case, seed)
    x = _inputs(case, seed)
    lens, block = x["lens"], case["block"]
    ends = _cut([n for n, _ in lens])
    if case["use"] != "attend":
        out = {"k": [], "v": []}
        for b, (n, back) in enumerate(_touched(lens, block)):
            for name in out:
                out[name].append(_held(x[name][ends[b]:ends[b + 1]], block, lens[b][1] if case["use"] == "write" else n)[n - back:])
        return torch.cat(out["k"]), torch.cat(out["v"])
    H, R, D = case["heads"], case["q_heads"] // case["heads"], case["dim"]
    out = torch.zeros(x["q"].shape[0], H, R, D, dtype=torch.float64, device=DEV)
    q = x["q"].double().view(-1, H, R, D)
    t0, r0 = 0, 0
    for n, rows in lens:
        for h in range(H):
            k, v = (_held(x[name][t0:t0 + n, h:h + 1], block, n)[:, 0] for name in ("k", "v"))
            for i in range(0, rows, 512):
                m = min(512, rows - i)
                pos = torch.arange(n - rows + i, n - rows + i + m, device=DEV).repeat_interleave(R)[:, None]
                key = torch.arange(n, device=DEV)[None, :]
                s = (q[r0 + i:r0 + i + m, h].reshape(m * R, D) @ k.T) / math.sqrt(D)
                hidden = key > pos
                if case["window"]:
                    hidden |= (key <= pos - case["window"]) & (key >= case["sinks"])
                s[hidden] = -math.inf
                out[r0 + i:r0 + i + m, h] = (torch.softmax(s, 1) @ v).view(m, R, D)
        t0, r0 = t0 + n, r0 + rows
    return out.view(-1, H * R, D)


def _exact_pages(case, seed):
    """One request after the other, with a stack of page numbers."""
    reqs, pages, most = _requests(case)
    page = case["page"]
    table = np.full((len(reqs), -(-most // page)), -1, np.int64)
    free, count, lens = list(range(pages - 1, -1, -1)), pages, [0] * len(reqs)

    def resize(want):
        nonlocal count
        need = [-(-n // page) for n in want]
        have = [-(-n // page) for n in lens]
        gone = [int(table[b, i]) for b in range(len(want)) for i in range(need[b], have[b])]
        for b in range(len(want)):
            table[b, need[b]:max(have[b], need[b])] = -1
        for p in reversed(gone):
            free[count] = p
            count += 1
        left, asked, starts = count, 0, [0]
        for b in range(len(want)):
            more = max(need[b] - have[b], 0)
            asked += more
            gained = 0
            if more == 0 or asked <= left:
                for i in range(more):
                    count -= 1
                    table[b, have[b] + i] = free[count]
                gained, lens[b] = max(want[b] - lens[b], 0), want[b]
            starts.append(starts[-1] + gained)
        return starts

    resize(_lives(case, seed))
    resize([a for a, _ in reqs])
    starts = resize([b for _, b in reqs])
    there = table.copy(), np.array(lens), np.array(starts)
    back = resize([a for a, _ in reqs])
    return tuple(torch.as_tensor(np.asarray(x), dtype=torch.float64, device=DEV)
                 for x in (*there, table, np.array(lens), np.array(free), np.array([count]), np.array(back)))


def _exact_slots(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000 * seed + 17)
    lens = _lengths(case)
    table = _table(case, lens, g)[0].cpu().numpy().astype(np.int64)
    slots, positions = [], []
    for b, (n, r) in enumerate(lens):
        p = np.arange(n - r, n)
        slots.append(table[b][p // case["page"]] * case["page"] + p % case["page"])
        positions.append(p)
    slots.append(np.full(case["pad"], -1))
    positions.append(np.zeros(case["pad"], np.int64))
    return tuple(torch.as_tensor(np.concatenate(x), dtype=torch.float64, device=DEV) for x in (slots, positions))
