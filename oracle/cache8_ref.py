"""The 8-bit key/value cache and the tables of pages, in numpy and plain Python: one token, one block, one page at a time."""
import numpy as np

TOP, LEAST, MOST = 57344.0, -15, 7


def e4m3(x):
    """float64 magnitudes up to 448 rounded to e4m3: three bits behind the first, steps of 2^-9 at least, ties to even."""
    a = np.abs(x)
    e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0)
    step = np.exp2(e - 3.0)
    return np.rint(x / step) * step


def exponent(top):
    """The least e with top <= 448 * 2^e."""
    e = LEAST
    while e < MOST and top > 448.0 * 2.0 ** e:
        e += 1
    return e


class Pool:
    """codes[i][page, token, head] (i: keys, values; as numbers), scale[i][page, block, head] (0: none yet), nan[page, token, head]"""

    def __init__(self, pages, heads, dim, page, block):
        self.pages, self.heads, self.dim, self.page, self.block = pages, heads, dim, page, block
        self.codes = [np.zeros((pages, page, heads, dim)) for _ in range(2)]
        self.scale = [np.zeros((pages, page // block, heads)) for _ in range(2)]
        self.nan = np.zeros((pages, page, heads), bool)

    def places(self, table, b, positions):
        """[(page or -1, token in it)]"""
        out = []
        for p in positions:
            i = p // self.page
            n = int(table[b][i]) if 0 <= p and i < len(table[b]) else -1
            out.append((n if 0 <= n < self.pages else -1, p % self.page))
        return out

    def write(self, table, lens, starts, k, v):
        """k, v: float32 images of 16-bit numbers [rows, heads, dim]"""
        for b in range(len(lens)):
            n = starts[b + 1] - starts[b]
            places = self.places(table, b, range(lens[b] - n, lens[b]))
            at = 0
            while at < n:
                page, tok = places[at]
                run = min(self.block - tok % self.block, n - at)
                if page >= 0:
                    self._run(page, tok, k[starts[b] + at:starts[b] + at + run], v[starts[b] + at:starts[b] + at + run])
                at += run

    def _run(self, page, tok, k, v):
        """Rows of one block: tokens tok .. of the page"""
        block, n = tok // self.block, len(k)
        first = block * self.block
        mine = np.zeros(self.page, bool)
        mine[tok:tok + n] = True
        others = ~mine
        others[:first] = others[first + self.block:] = False
        bad = (np.isnan(k) | np.isnan(v)).any(-1)                       # [rows, heads]
        self.nan[page, tok:tok + n] = bad
        for h in range(self.heads):
            for i, x in enumerate((k[:, h].astype(np.float64), v[:, h].astype(np.float64))):
                x = np.where(bad[:, h, None], 0.0, np.clip(np.nan_to_num(x, nan=0.0, posinf=TOP, neginf=-TOP), -TOP, TOP))
                s = 2.0 ** exponent(np.abs(x).max())
                was = self.scale[i][page, block, h]
                if tok != first:
                    s = max(s, was)
                    if s != was:
                        self.codes[i][page, others, h] = e4m3(self.codes[i][page, others, h] * (was / s))
                self.scale[i][page, block, h] = s
                self.codes[i][page, tok:tok + n, h] = e4m3(x / s)

    def read(self, table, b, positions):
        """(keys, values, there) of tokens of a sequence, float64 [tokens, heads, dim]"""
        places = self.places(table, b, positions)
        out = [np.zeros((len(places), self.heads, self.dim)) for _ in range(2)]
        for j, (page, tok) in enumerate(places):
            if page >= 0:
                for i in range(2):
                    out[i][j] = self.codes[i][page, tok] * self.scale[i][page, tok // self.block][:, None]
                    out[i][j][self.nan[page, tok]] = np.nan
        return out[0], out[1], np.array([p >= 0 for p, _ in places], bool)


class Tables:
    """KVPages, one page after the other"""

    def __init__(self, pages, seqs, max_len, page):
        self.page, self.cols = page, -(-max_len // page)
        self.table = [[-1] * self.cols for _ in range(seqs)]
        self.lens, self.free, self.count = [0] * seqs, list(range(pages - 1, -1, -1)), pages

    def resize(self, want):
        """-> where the new rows of each sequence begin"""
        pages_of = lambda n: -(-n // self.page)
        want = [n if w < 0 or pages_of(w) > self.cols else w for w, n in zip(want, self.lens)]
        gone = []
        for b, w in enumerate(want):
            for i in range(pages_of(w), pages_of(self.lens[b])):
                gone.append(self.table[b][i])
                self.table[b][i] = -1
        for p in reversed(gone):
            self.free[self.count] = p
            self.count += 1
        left, asked, starts = self.count, 0, [0]
        for b, w in enumerate(want):
            have, need = pages_of(self.lens[b]), pages_of(w)
            asked += max(need - have, 0)
            gained = 0
            if need <= have or asked <= left:
                for i in range(have, need):
                    self.count -= 1
                    self.table[b][i] = self.free[self.count]
                gained = max(w - self.lens[b], 0)
                self.lens[b] = w
            starts.append(starts[-1] + gained)
        return starts

    def slots(self, starts, rows):
        """(slots, positions) of the rows of a step"""
        slots, positions = [-1] * rows, [0] * rows
        for b in range(len(self.lens)):
            n = starts[b + 1] - starts[b]
            for t in range(starts[b], min(starts[b + 1], rows)):
                j = self.lens[b] - n + t - starts[b]
                positions[t] = max(j, 0)
                if j >= 0 and j // self.page < self.cols and self.table[b][j // self.page] >= 0:
                    slots[t] = self.table[b][j // self.page] * self.page + j % self.page
        return slots, positions


def attention(q, k, v, pos, there, scale, window=None, sinks=0):
    """q [rows, D], k / v [tokens, D] float64, pos [rows] -> (o, spread, size, reach): o [rows, D] and, for the error of a computation
    with rounded weights, sqrt(sum_j p_j (v_j - o)^2) >= sum_j p_j |v_j - o|, sum_j p_j |v_j| and the largest scale sum_d |q_d k_jd| of a row."""
    rows, tokens = len(q), len(k)
    j = np.arange(tokens)
    o, spread, size, reach = np.zeros((rows, v.shape[1])), np.zeros((rows, v.shape[1])), np.zeros((rows, v.shape[1])), np.zeros(rows)
    for i in range(0, rows, 256):
        at = slice(i, min(rows, i + 256))
        p = np.asarray(pos)[at, None]
        seen = (j[None, :] <= p) & there[None, :]
        if window:
            seen &= (j[None, :] > p - window) | (j[None, :] < sinks)
        some = seen.any(1)
        if not some.any():
            continue
        s = np.where(seen, scale * (q[at] @ k.T), -np.inf)
        e = np.exp(s - np.where(some, s.max(1, initial=-np.inf), 0.0)[:, None])
        e /= np.maximum(e.sum(1), 1e-300)[:, None]
        o[at] = e @ v
        spread[at] = np.sqrt(np.maximum(e @ (v * v) - o[at] ** 2, 0.0)) + 1e-9 * np.abs(o[at])
        size[at] = e @ np.abs(v)
        reach[at] = scale * np.where(seen, np.abs(q[at]) @ np.abs(k).T, 0.0).max(1)
    return o, spread, size, reach
