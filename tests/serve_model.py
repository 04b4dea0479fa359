"""The batched serving operators (include/uq_serve.h) in 64-bit numpy, and
bounds on the kernels' distance from them."""
import numpy as np

import uq
from uq import serve

U32 = 2.0 ** -24  # half a step of f32, relative
DTYPE = {"f32": (uq.DType.F32, np.float32), "f16": (uq.DType.F16, np.float16)}


class Cache:
    """Pools in pages, page tables and a batch's rows, on the host and (upload) on the device."""

    def __init__(self, rng, dtype, kv, hd, page, rows, lens, pad=0, spare=2, shared=0, scale=1.0, room=0):
        self.dtype, self.kv, self.hd, self.page, self.rows, self.lens = dtype, kv, hd, page, list(rows), list(lens)
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.n_rows = int(self.start[-1]) + pad
        whole = shared // page
        need = [max(0, -(-x // page) - whole) for x in lens]
        self.max_pages = max(whole + max(need + [1]), room // page)  # room: positions of a table that is longer than it need be
        self.n_pages = whole + sum(need) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(rows), self.max_pages), -1, np.int32)
        at = whole
        for b, k in enumerate(need):
            self.table[b, :whole] = order[:whole]
            self.table[b, whole:whole + k] = order[at:at + k]
            at += k
        t = DTYPE[dtype][1]
        shape = (self.n_pages, kv, page, hd)
        self.k = (scale * rng.standard_normal(shape)).astype(t)
        self.v = (scale * rng.standard_normal(shape)).astype(t)
        if shared % page:
            for b in range(1, len(rows)):
                for c in (self.k, self.v):
                    if need[b] and need[0]:
                        c[self.table[b, whole], :, :shared % page] = c[self.table[0, whole], :, :shared % page]

    def slots(self, b, n):
        """(page, slot) of positions 0 .. n - 1 of sequence b, and which exist."""
        p = np.arange(n)
        idx = p // self.page
        page = np.where(idx < self.max_pages, self.table[b, np.minimum(idx, self.max_pages - 1)], -1)
        return page, p % self.page, (page >= 0) & (page < self.n_pages)

    def upload(self):
        self.d_k, self.d_v, self.d_start, self.d_len, self.d_table = (
            uq.DeviceArray.from_numpy(a) for a in (self.k, self.v, self.start, np.array(self.lens, np.int32), self.table))
        pages = serve.KvPages(self.d_k, self.d_v, DTYPE[self.dtype][0], self.n_pages, self.page, self.kv, self.hd)
        batch = serve.SeqBatch(len(self.rows), self.n_rows, self.d_start, self.d_len, self.d_table, self.max_pages)
        return pages, batch

    def row_positions(self):
        """(sequence, position) of every row of a sequence."""
        return [(b, self.lens[b] - n + i) for b, n in enumerate(self.rows) for i in range(n)]


def attention(c, q, heads, scale, gate=None):
    """(out, bound) in 64 bits: rows of no sequence are NaN in both.

    The bound: a score is off by e = |scale| sum |q k| (2^-22 + (hd + 4) 2^-24) (two-term queries, hd products
    summed in f32, its factor), and by the rounding of its exponent; so a weight is off by a factor within 2 e +
    8 2^-24 of 1 (e in the exponent of the weight and of the largest; exp2 and the two-term weight within 2^-22
    together). Sums of n positions take at most n + 64 roundings (the parts' joins among them), for o and for l.
    Everything is relative to sum p |v|, at least as large as each output; the gate multiplies all of it."""
    out = np.full((c.n_rows, heads, c.hd), np.nan)
    bound = np.full(out.shape, np.nan)
    group = heads // c.kv
    r = 0
    for b, n in enumerate(c.rows):
        for i in range(n):
            pos = c.lens[b] - n + i
            page, slot, ok = c.slots(b, max(0, pos + 1))
            page, slot = page[ok], slot[ok]
            for h in range(heads):
                if not len(page):
                    out[r, h], bound[r, h] = 0.0, 0.0
                    continue
                k, v = (a[page, h // group, slot].astype(np.float64) for a in (c.k, c.v))
                qh = q[r, h].astype(np.float64)
                s = scale * (k @ qh)
                e = abs(scale) * (np.abs(k) @ np.abs(qh)) * (2.0 ** -22 + (c.hd + 4) * U32)
                p = np.exp(s - s.max())
                p /= p.sum()
                A = p @ np.abs(v)
                out[r, h] = p @ v
                rel = 2 * e.max() + (8 + 2 * (len(p) + 64)) * U32
                bound[r, h] = rel * A + 1e-30
            r += 1
    if gate is not None:
        g = 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
        out, bound = out * g, bound * g + np.abs(out * g) * 4 * U32
    return out, bound


def verify(p, q, tokens, u, rows):
    """(accepted, next) by the definition, sums in order in f64."""
    def weight(w):
        return np.where((w > 0) & np.isfinite(w), w, 0.0)

    vocab, acc, nxt, a = p.shape[1], [], [], 0
    for n in rows:
        if n == 0:
            acc.append(0)
            nxt.append(-1)
            continue
        r = a
        while r + 1 < a + n:
            x = int(tokens[r + 1])
            with np.errstate(invalid="ignore"):
                if not (0 <= x < vocab and float(u[r]) * (1.0 if q is None else float(q[r, x])) < float(p[r, x])):
                    break
            r += 1
        plain = weight(p[r].astype(np.float64))
        w = plain
        if r + 1 < a + n:
            if q is None:
                w = plain.copy()
                if 0 <= tokens[r + 1] < vocab:
                    w[tokens[r + 1]] = 0.0
            else:
                w = weight(p[r].astype(np.float64) - q[r].astype(np.float64))
        if not w.sum() > 0:
            w = plain
        c = np.cumsum(w)
        last = float(u[a + n - 1])
        has = np.nonzero(w > 0)[0]
        if not len(has):
            nxt.append(-1)
        elif not last < 1:
            nxt.append(int(has[-1]))
        else:
            hit = has[c[has] > max(last, 0.0) * c[-1]]
            nxt.append(int(hit[0]) if len(hit) else int(has[-1]))
        acc.append(r - a)
        a += n
    return np.array(acc, np.int32), np.array(nxt, np.int32)
