"""The paged 8-bit cache in NumPy: tables by plain loops, quantisation and attention in 64 bits."""
import numpy as np

from ksearch_b200 import E4M3, I8

QMAX = {I8: 127.0, E4M3: 448.0}


def _e4m3_values():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[(c & 127) == 127] = 448.0        # the NaN patterns read as 448
    return np.where((c >= 128) & ((c & 127) != 127), -v, v)


E4M3_VALUES = _e4m3_values()


def decode(codes, fmt):
    """Codes (uint8) as f64."""
    return codes.view(np.int8).astype(np.float64) if fmt == I8 else E4M3_VALUES[codes]


def encode(y, fmt):
    """Nearest codes of values over their scale, ties to even; infinities at the ends, NaN as 0."""
    y = np.clip(np.where(np.isnan(y), 0.0, y), -QMAX[fmt], QMAX[fmt])
    if fmt == I8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    a = np.abs(y)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
    a = np.rint(a / 2.0 ** (e - 3)) * 2.0 ** (e - 3)
    codes = np.searchsorted(E4M3_VALUES[:127], a).astype(np.uint8)
    assert np.array_equal(E4M3_VALUES[codes], a)
    return codes | (np.signbit(y).astype(np.uint8) << 7)


def scale_for(amax, fmt):
    """The least power of two from 2^-100 to 2^100 that amax fits under."""
    e = -100
    while e < 100 and amax > QMAX[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e


class Tables:
    """What PageTables does, one sequence after the other."""

    def __init__(self, n_seqs, max_blocks, n_pages, page, max_rows):
        self.n_seqs, self.max_blocks, self.n_pages, self.page, self.max_rows = n_seqs, max_blocks, n_pages, page, max_rows
        self.lens = np.zeros(n_seqs, np.int64)
        self.tables = np.full((n_seqs, max_blocks), -1, np.int64)
        self.stack = list(range(n_pages - 1, -1, -1))
        self.rows = []          # (seq, pos, slot)
        self.jobs = []          # (first row, rows, slot, pos)
        self.row_start = np.zeros(n_seqs + 1, np.int64)

    def step(self, new):
        new = np.asarray(new, np.int64)
        cap = self.max_blocks * self.page
        status = 0
        for n, have in zip(new, self.lens):
            status = max(status, 4 if n < 0 or not 0 <= have <= cap else 3 if n > self.max_rows else 2 if have + n > cap else 0)
        if status < 3 and new.sum() > self.max_rows:
            status = 3
        blocks = lambda t: -(-t // self.page)  # noqa: E731
        if status == 0 and sum(blocks(t + n) - blocks(t) for t, n in zip(self.lens, new)) > len(self.stack):
            status = 1
        self.rows, self.jobs = [], []
        self.row_start[:] = 0
        if status:
            return status
        for s in range(self.n_seqs):
            for b in range(blocks(self.lens[s]), blocks(self.lens[s] + new[s])):
                self.tables[s, b] = self.stack.pop()
            for i in range(new[s]):
                pos = self.lens[s] + i
                slot = self.tables[s, pos // self.page] * self.page + pos % self.page
                if i == 0 or pos % self.page == 0:
                    self.jobs.append([len(self.rows), 0, slot, pos])
                self.jobs[-1][1] += 1
                self.rows.append((s, pos, slot))
            self.lens[s] += new[s]
            self.row_start[s + 1] = len(self.rows)
        return 0

    def trim(self, keep):
        back = []
        for s in range(self.n_seqs):
            if 0 <= keep[s] < self.lens[s]:
                lo, hi = -(-keep[s] // self.page), -(-self.lens[s] // self.page)
                back += self.tables[s, lo:hi].tolist()
                self.tables[s, lo:hi] = -1
                self.lens[s] = keep[s]
        self.stack += back[::-1]


class Cache:
    def __init__(self, n_pages, page, n_kv, hd, fmt):
        self.n_pages, self.page, self.n_kv, self.hd, self.fmt = n_pages, page, n_kv, hd, fmt
        self.codes = [np.zeros((n_pages, n_kv, page, hd), np.uint8) for _ in range(2)]
        self.scales = [np.zeros((n_pages, n_kv), np.float64) for _ in range(2)]

    def append(self, tables, k, v):
        """k, v [rows, n_kv, hd] (f64 of what is appended) by the jobs of the last step."""
        for which, x in enumerate((k, v)):
            for row, n, slot, _ in tables.jobs:
                p, off = divmod(int(slot), self.page)
                for h in range(self.n_kv):
                    y = x[row:row + n, h].astype(np.float64)
                    fine = np.abs(y[np.isfinite(y)])
                    s = scale_for(fine.max() if fine.size else 0.0, self.fmt)
                    codes = self.codes[which][p, h]
                    if off:
                        held = self.scales[which][p, h]
                        if held > s:
                            s = held
                        elif held < s:
                            codes[:off] = encode(decode(codes[:off], self.fmt) * (held / s), self.fmt)
                    codes[off:off + n] = encode(y / s, self.fmt)
                    self.scales[which][p, h] = s

    def values(self, which, pages, h):
        """f64 rows of a head over a run of pages."""
        c = decode(self.codes[which][pages, h], self.fmt) * np.clip(self.scales[which][pages, h], 2.0 ** -100, 2.0 ** 100)[:, None, None]
        return c.reshape(-1, self.hd)


def attention(cache, table, length, rows, q, scale, window):
    """q [rows, n_q, hd] of one sequence in f64 -> out, and for each (row, head) the largest sum |q_d k_d| of a seen position
    and sum p |v| over the seen ones: what a tolerance is made of."""
    n_q, hd = q.shape[1], cache.hd
    G = n_q // cache.n_kv
    out, spread, weight = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape)
    pages = np.asarray(table[:max(0, -(-length // cache.page))], np.int64)
    for h in range(cache.n_kv):
        K, V = cache.values(0, pages, h)[:length], cache.values(1, pages, h)[:length]
        for r in range(rows):
            p = length - rows + r
            lo = max(0, p - window + 1) if window else 0
            if p < lo:
                continue
            k, v = K[lo:p + 1], V[lo:p + 1]
            for g in range(G):
                x = q[r, h * G + g]
                s = k @ x * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h * G + g] = w @ v
                spread[r, h * G + g] = (np.abs(k) @ np.abs(x)).max() * abs(scale)
                weight[r, h * G + g] = w @ np.abs(v)
    return out, spread, weight


def norm_rope(x, w, cos_sin, eps):
    """x [rows, heads, hd] -> RMS norm (w: weights or None) and, with weights, RoPE, in f64."""
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
    if w is None:
        return y
    y = y * np.asarray(w, np.float64)
    half = x.shape[-1] // 2
    c, s = cos_sin[:, None, :half], cos_sin[:, None, half:]
    return np.concatenate([y[..., :half] * c - y[..., half:] * s, y[..., :half] * s + y[..., half:] * c], -1)
