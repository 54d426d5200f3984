"""The 4-bit cache and attention over it in numpy and 64 bits, from the layout
and the formulas that include/phobos_hip.h states: a pool is a byte array that
tokens are written into and read out of one at a time."""
import numpy as np


class Pool:
    def __init__(self, pages, heads, D, P, fill=0xFF):
        self.pages, self.heads, self.D, self.P = pages, heads, D, P
        self.data = np.full((pages, heads, P * (D + 8)), fill, np.uint8)

    def _codes_at(self, v, slot):
        """Byte index of each element's code in a head's part of a page."""
        d = np.arange(self.D)
        if not v:
            return slot * (self.D // 2) + d // 2
        word = (slot // 4 * (self.D // 8) + d // 8) * 4 + slot % 4
        return self.P * self.D // 2 + word * 4 + d % 8 // 2

    def _param_at(self, v, slot):
        return self.P * self.D + (4 * self.P if v else 0) + 4 * slot

    def write(self, page, head, slot, v, codes, scale, low):
        at, part = self._codes_at(v, slot), self.data[page, head]
        part[at[0::2]] = codes[0::2] | codes[1::2] << 4
        p = self._param_at(v, slot)
        part[p:p + 4] = np.array([scale, low], np.float16).view(np.uint8)

    def raw(self, page, head, slot, v):
        """(codes, scale, minimum)."""
        at, part = self._codes_at(v, slot), self.data[page, head]
        codes = part[at] >> (4 * (np.arange(self.D) % 2)).astype(np.uint8) & 15
        p = self._param_at(v, slot)
        scale, low = part[p:p + 4].view(np.float16)
        return codes, scale, low

    def value(self, page, head, slot, v):
        codes, scale, low = self.raw(page, head, slot, v)
        return codes * np.float64(scale) + np.float64(low)


def quantise(x):
    """(codes, scale, minimum) of one row."""
    x = np.asarray(x, np.float64)
    low = np.float16(np.float32(x.min()))
    scale = np.float16(np.float32((x.max() - x.min()) / 15))
    scale = max(scale, np.float16(2.0 ** -24))
    codes = np.clip(np.rint((x - np.float64(low)) / np.float64(scale)), 0, 15).astype(np.uint8)
    return codes, scale, low


def rows_of(b, lens, starts, max_q, rows, cap):
    """(tokens, [(row, position)]) of sequence b of a call."""
    n = min(max(int(lens[b]), 0), cap)
    if starts is None:
        first, count = b * max_q, max_q
    else:
        first, count = int(starts[b]), min(max(int(starts[b + 1]) - int(starts[b]), 0), max_q)
    return n, [(first + i, n - count + i) for i in range(count) if 0 <= first + i < rows]


def page_of(pool, table, b, token):
    page = int(table[b, token // pool.P])
    return page if 0 <= page < pool.pages else -1


def attention(pool, table, lens, starts, max_q, max_len, q, scale, causal):
    """(O, seen, bound): outputs in f64, which rows are in the call, and how
    far each output may be off by the arithmetic the header states, before its
    last rounding."""
    rows, Hq, D = q.shape
    R = Hq // pool.heads
    out = np.zeros((rows, Hq, D))
    off = np.zeros((rows, Hq, D))
    seen = np.zeros(rows, bool)
    for b in range(len(lens)):
        n, mine = rows_of(b, lens, starts, max_q, rows, min(max_len, table.shape[1] * pool.P))
        pages = [page_of(pool, table, b, t) for t in range(n)]
        there = np.array([p >= 0 for p in pages], bool)
        for h in range(pool.heads):
            k, v = np.zeros((n, D)), np.zeros((n, D))
            ks, vs = np.zeros((n, 2)), np.zeros((n, 2))
            for t in range(n):
                if there[t]:
                    k[t], v[t] = (pool.value(pages[t], h, t % pool.P, x) for x in (False, True))
                    ks[t], vs[t] = (pool.raw(pages[t], h, t % pool.P, x)[1:] for x in (False, True))
            kmag = 15 * np.abs(ks[:, 0]) + np.abs(ks[:, 1])  # of a code times scale, and of a minimum
            vmag = 15 * np.abs(vs[:, 0]) + np.abs(vs[:, 1])
            for row, pos in mine:
                seen[row] = True
                use = there & ((np.arange(n) <= pos) if causal else True)
                if not use.any():
                    continue
                for r in range(R):
                    x = q[row, h * R + r].astype(np.float64)
                    s = scale * (k[use] @ x)
                    p = np.exp(s - s.max())
                    l = p.sum()
                    out[row, h * R + r] = p @ v[use] / l
                    # scores: D+6 roundings of f32 and an f32 query's 22 bits
                    ds = abs(scale) * np.abs(x).sum() * kmag[use] * ((D + 6) * 2.0 ** -24 + 2.0 ** -22)
                    # weights: exp2 and its argument to 2 steps, 22 bits, a sum
                    # of n terms above and below; relative
                    rel = ds + ds.max() + (np.abs(s) + np.abs(s).max()) * 2.0 ** -22 + \
                        (2 * use.sum() + 16) * 2.0 ** -24 + 2.0 ** -21
                    off[row, h * R + r] = 1.01 * (p * rel * vmag[use]).sum() / l
    return out, seen, off
