"""What the operators of the 4-bit key/value cache are measured on, and the same operators in plain torch.

A case names a use:

  write    the newest tokens of every sequence go into the cache, and come back as the values it holds for
           them (a prompt's own attention then sees what later steps will see)
  read     tokens that are in the cache, as dense tensors
  attend   attention of the newest tokens, which the cache holds too: one token a sequence, a few, or a prompt

and its shape: `seqs` sequences whose lengths are spread over `length` and whose newest tokens (the rows of
the call) over `new` (0: all of them), `q_heads` query heads on `heads` cache heads of `dim` channels, `page`
tokens a page, `group` channels a scale, `window` (0: none) and `sinks` of the visible range.

Head counts and head sizes are those of the benchmark's Mistral-7B and Gemma-3-27B shaped layers (32 and 8,
32 and 16, 128 channels), of the tests' small decoder (4 and 2, 64 channels), and 256 channels; lengths are generic.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
TOP = 65280.0                                                       # larger magnitudes are held as this one


def _case(name, use, seqs, length, new, heads, q_heads, dim, page, group, dtype, window=0, sinks=0, lens_seed=0):
    return dict(name=name, use=use, seqs=seqs, length_lo=length[0], length_hi=length[1], new_lo=new[0], new_hi=new[1],
                heads=heads, q_heads=q_heads, dim=dim, page=page, group=group, dtype=dtype, window=window, sinks=sinks,
                lens_seed=lens_seed)


def listed():
    return [
        # one decode step's keys and values of 32 sequences: the cost of the calls themselves
        _case("write_step", "write", 32, (1, 4000), (1, 1), 8, 32, 128, 64, 32, "f16", lens_seed=1),
        # a batch of prompts of odd lengths enters the cache
        _case("write_prompts", "write", 9, (1, 4500), (0, 0), 16, 32, 128, 32, 64, "bf16", lens_seed=2),
        # short prefixes of a small decoder back as dense tensors
        _case("read_prefix", "read", 5, (1, 900), (0, 0), 2, 4, 64, 16, 32, "f16", lens_seed=3),
        # long prefixes handed to a program that wants them dense
        _case("read_long", "read", 2, (30000, 50000), (0, 0), 8, 32, 128, 128, 128, "bf16", lens_seed=4),
        # one sequence, one token, a short history: latency alone
        _case("attend_one", "attend", 1, (700, 700), (1, 1), 8, 32, 128, 64, 32, "f16"),
        # a decode step of a serving batch with histories of all lengths
        _case("attend_batch", "attend", 32, (1, 8192), (1, 1), 8, 32, 128, 64, 64, "bf16", lens_seed=6),
        # two very long histories: too few rows to fill the chip without cutting the length
        _case("attend_long", "attend", 2, (100000, 140000), (1, 1), 8, 32, 128, 256, 32, "bf16", lens_seed=7),
        # a layer with a sliding window and four first tokens kept, one token each
        _case("attend_window", "attend", 16, (6000, 30000), (1, 1), 16, 32, 128, 32, 128, "f16", 4096, 4, lens_seed=8),
        # a few drafted tokens of each sequence checked at once, wide heads
        _case("attend_draft", "attend", 12, (300, 5000), (2, 6), 4, 16, 256, 32, 64, "bf16", lens_seed=9),
        # a whole prompt of a layer
        _case("attend_prompt", "attend", 1, (4096, 4096), (4096, 4096), 8, 32, 128, 64, 64, "bf16"),
        # prompts that arrive in chunks behind what the cache holds already, three query heads on one
        _case("attend_chunks", "attend", 6, (1500, 9000), (1, 1500), 8, 24, 64, 16, 64, "f16", lens_seed=11),
        # long prompts through a layer with a sliding window
        _case("attend_window_prompt", "attend", 2, (5000, 9000), (0, 0), 16, 32, 128, 64, 128, "bf16", 1024, 4, lens_seed=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        use = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend", "attend"])
        dim = rng.choice([64, 128, 128, 128, 256])
        heads = rng.choice([1, 2, 4, 8, 8, 16])
        ratio = rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
        page, group = rng.choice([16, 32, 64, 128, 256]), rng.choice([g for g in (32, 64, 128) if g <= dim])
        seqs = _log(rng, 1, 64)
        hi = _log(rng, 1, 140000)
        lo = hi if rng.random() < 0.2 else max(1, int(hi * rng.random()))
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
        window, sinks = 0, 0
        if use == "attend" and rng.random() < 0.35:
            window, sinks = _log(rng, 16, 8192), rng.choice([0, 1, 4, 64])
        case = _case("", use, seqs, (lo, hi), new, heads, heads * ratio, dim, page, group, rng.choice(["f16", "bf16"]), window,
                     sinks, rng.randrange(1 << 20))
        del case["name"]
        rows = sum(n for _, n in _lengths(case))
        w = work(case)
        held = sum(n for n, _ in _lengths(case)) * heads * dim
        if rows <= 20000 and rows * case["q_heads"] * dim <= 8e7 and held <= 2.6e8 and w["flops"] <= 1.3e11:
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


def work(case):
    lens = _lengths(case)
    rows = sum(n for _, n in lens)
    token = 2 * case["heads"] * (case["dim"] // 2 + 4 * (case["dim"] // case["group"]))   # bytes of a token in the cache
    dense = 2 * case["heads"] * case["dim"] * 2                                          # and of its keys and values in 16 bits
    if case["use"] == "write":
        return {"bytes": rows * (2 * dense + token), "flops": 0}
    if case["use"] == "read":
        return {"bytes": rows * (dense + token), "flops": 0}
    seen = [_visible(n, r, case["window"], case["sinks"]) for n, r in lens]
    size = sum(k for _, k in seen) * token + 2 * rows * case["q_heads"] * case["dim"] * 2
    return {"bytes": size, "flops": 4 * case["q_heads"] * case["dim"] * sum(p for p, _ in seen)}


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Keys have channels of different magnitude and a few outliers, as behind a rotary embedding; pages are
    handed out in no order; the table's unused entries hold no page."""
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
    need = [-(-n // case["page"]) for n, _ in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return dict(k=k, v=v, q=q, table=table, pages=pages, lens=lens)


def _cut(lens, which):
    """Offsets of the sequences in a packed tensor: of whole sequences (0) or of their newest rows (1)."""
    out = [0]
    for x in lens:
        out.append(out[-1] + x[which])
    return out


def _newest(lens):
    """Positions of the newest rows among all tokens, packed sequence behind sequence."""
    whole = _cut(lens, 0)
    return torch.cat([torch.arange(whole[b + 1] - r, whole[b + 1], device=DEV) for b, (_, r) in enumerate(lens)])


def prepare(case, seed):
    x = _inputs(case, seed)
    lens = x["lens"]
    st = dict(case=case, lens=lens, q=x["q"])
    newest = _newest(lens)
    st["k"], st["v"] = x["k"][newest], x["v"][newest]
    ints = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
    st["table"], st["tokens"] = x["table"], ints([n for n, _ in lens])
    st["starts"] = ints(_cut(lens, 1))
    if own:
        from cobalt_amd import KVCache, KVRows, ops
        st["cache"] = KVCache(x["pages"], case["heads"], case["dim"], page=case["page"], group=case["group"], device=DEV)
        st["rows"] = KVRows(st["table"], st["tokens"], st["starts"])
        if case["use"] != "write":
            ops.cache_write(st["cache"], x["k"], x["v"], KVRows(st["table"], st["tokens"], ints(_cut(lens, 0))))
    else:
        slots, H, D, G = x["pages"] * case["page"], case["heads"], case["dim"], case["group"]
        for name in ("k", "v"):
            st[name + "_codes"] = torch.zeros(slots, H, D // 2, dtype=torch.uint8, device=DEV)
            st[name + "_meta"] = torch.zeros(slots, H, D // G, 2, dtype=torch.float16, device=DEV)
            if case["use"] != "write":
                whole = _cut(lens, 0)
                for b, (n, _) in enumerate(lens):
                    for i in range(0, n, 32768):
                        at = torch.arange(i, min(n, i + 32768), device=DEV)
                        _store(st, name, _slots(st, b, at), x[name][whole[b] + at])
    return st


# ------------------------------------------------------------------ plain form
def _slots(st, b, positions):
    page = st["case"]["page"]
    return st["table"][b][positions // page].long() * page + positions % page


def _store(st, name, slots, x):
    G = st["case"]["group"]
    f = x.float().clamp(-TOP, TOP).unflatten(-1, (-1, G))
    low = f.amin(-1, keepdim=True).half()
    scale = ((f.amax(-1, keepdim=True) - low.float()) / 15.0).half()
    step = torch.where(scale == 0, torch.ones_like(scale), scale).float()
    code = torch.where(scale == 0, torch.zeros_like(f), ((f - low.float()) / step).round().clamp(0, 15))
    code = code.to(torch.uint8).flatten(-2)
    st[name + "_codes"][slots] = code[..., 0::2] | (code[..., 1::2] << 4)
    st[name + "_meta"][slots] = torch.cat([scale, low], -1)


def _load(st, name, slots):
    packed, meta = st[name + "_codes"][slots], st[name + "_meta"][slots].float()
    code = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    return (code.unflatten(-1, (-1, st["case"]["group"])) * meta[..., :1] + meta[..., 1:]).flatten(-2)


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


def _plain_new_slots(st):
    return torch.cat([_slots(st, b, torch.arange(n - r, n, device=DEV)) for b, (n, r) in enumerate(st["lens"])])


# ------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    use, dt = c["use"], TYPES[c["dtype"]]
    if own:
        from cobalt_amd import ops
        if use == "write":
            ops.cache_write(state["cache"], state["k"], state["v"], state["rows"])
        if use in ("write", "read"):
            return ops.cache_read(state["cache"], state["rows"], state["k"].shape[0], dt)
        return ops.cache_attention(state["cache"], state["q"], state["rows"], window=c["window"] or None, sinks=c["sinks"])
    if use == "attend":
        return _plain_attend(state)
    slots = _plain_new_slots(state)
    if use == "write":
        _store(state, "k", slots, state["k"])
        _store(state, "v", slots, state["v"])
    return _load(state, "k", slots).to(dt), _load(state, "v", slots).to(dt)


# ------------------------------------------------------------------ the definition in 64 bits
def _held(x, group):
    """The values the cache holds for x, in float64.  Which code, scale and minimum a value gets is a decision of
    the definition (scale and minimum are rounded to 16 bits, from a range taken in 32); the values follow exactly."""
    rows, H, D = x.shape
    f = torch.clamp(x.double(), -TOP, TOP).reshape(rows, H, D // group, group)
    m = f.min(dim=3).values.half()
    s = ((f.max(dim=3).values - m.double()).float() / 15.0).half()
    m, s = m.double()[..., None], s.double()[..., None]
    c = torch.round((f - m) / torch.where(s == 0, torch.ones_like(s), s))
    return (m + torch.clamp(c, 0, 15) * s).reshape(rows, H, D)


def exact(case, seed):
    x = _inputs(case, seed)
    lens, group = x["lens"], case["group"]
    newest = _newest(lens)
    if case["use"] in ("write", "read"):
        return _held(x["k"][newest], group), _held(x["v"][newest], group)
    H, R, D = case["heads"], case["q_heads"] // case["heads"], case["dim"]
    out = torch.zeros(newest.numel(), H, R, D, dtype=torch.float64, device=DEV)
    q = x["q"].double().view(-1, H, R, D)
    t0, r0 = 0, 0
    for n, rows in lens:
        for h in range(H):
            k, v = _held(x["k"][t0:t0 + n, h:h + 1], group)[:, 0], _held(x["v"][t0:t0 + n, h:h + 1], group)[:, 0]
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
