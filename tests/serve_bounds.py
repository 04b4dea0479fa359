"""What the paged attention's results may differ by from 64 bits: the bounds of include/uq_serve.h with their parts
apart, for inputs that leave only some of them (sums of one product, equal weights), and the two f16 terms of an f16
cache's queries and weights on the CPU."""
import numpy as np

import serve_model as M

U32 = M.U32
QUERY_FLOOR = 2.0 ** -38  # of a query's largest value: half a step of the least f16 (2^-25), the largest held at 2^13 or more
FEW_FLOOR = 2.0 ** -39    # of a row's largest weight, blocks of 16 and 32 queries: held at 2^14
MANY_FLOOR = 2.0 ** -33   # blocks of 64 and 128: held at 2^8 or more


def score_error(c, q, k, scale, roundings):
    """Of q k scale: f32 sums of `roundings` terms; an f16 cache: two-term queries."""
    size = np.abs(q) @ np.abs(k).T
    e = size * roundings * U32
    if c.dtype == "f16":
        e += size * 2.0 ** -22 + QUERY_FLOOR * np.abs(q).max(-1, keepdims=True) * np.abs(k).sum(-1)
    return abs(scale) * e


def attention(c, q, heads, scale, roundings=None, floor=MANY_FLOOR, sums=None):
    """(out, bound) in 64 bits, as serve_model.attention, for the rows of sequences, many queries at a time. roundings:
    of a score's sum, head_dim + 4 where they are not known to be fewer; sums: of o and of l, n + 64 likewise."""
    out = np.zeros((c.n_rows, heads, c.hd))
    bound = np.zeros(out.shape)
    group = heads // c.kv
    r = 0
    for b, n in enumerate(c.rows):
        page, slot, ok = c.slots(b, max(0, c.lens[b]))
        where = np.nonzero(ok)[0]
        for j in range(c.kv):
            K, V = (a[page[ok], j, slot[ok]].astype(np.float64) for a in (c.k, c.v))
            for i in range(n):
                m = int(np.searchsorted(where, c.lens[b] - n + i, side="right"))
                if m == 0:
                    continue
                h = slice(j * group, (j + 1) * group)
                x, k, v = q[r + i, h].astype(np.float64), K[:m], V[:m]
                s = scale * (x @ k.T)
                e = score_error(c, x, k, scale, c.hd + 4 if roundings is None else roundings).max(-1, keepdims=True)
                p = np.exp(s - s.max(-1, keepdims=True))  # of the largest weight
                l = p.sum(-1, keepdims=True)
                out[r + i, h] = p @ v / l
                rel = 2 * e + (8 + 2 * (m + 64 if sums is None else sums)) * U32
                bound[r + i, h] = rel * (p @ np.abs(v)) / l + 1e-30
                if c.dtype == "f16":
                    bound[r + i, h] += floor * np.abs(v).sum(0) / l
        r += n
    return out, bound


def terms(x, n):
    """x as n f16 terms."""
    y = np.zeros_like(x)
    for _ in range(n):
        y = y + (x - y).astype(np.float16).astype(np.float64)
    return y


def attention_in_terms(c, q, heads, scale, query_terms=2, weight_terms=2, hold=8):
    """The results with queries and weights in that many terms, everything else in 64 bits: a query's largest value
    held between 2^13 and 2^15, the largest weight at 2^hold."""
    out = np.zeros((c.n_rows, heads, c.hd))
    group = heads // c.kv
    for r, (b, pos) in enumerate(c.row_positions()):
        page, slot, ok = c.slots(b, pos + 1)
        for h in range(heads):
            k, v = (a[page[ok], h // group, slot[ok]].astype(np.float64) for a in (c.k, c.v))
            x = q[r, h].astype(np.float64)
            to = 2.0 ** (14 - np.frexp(np.abs(x).max())[1])
            s = scale * (k @ (terms(x * to, query_terms) / to))
            p = np.exp(s - s.max()) * 2.0 ** hold
            out[r, h] = (terms(p, weight_terms) @ v) / p.sum()
    return out


# Shapes that take each kernel (f16; tables long enough not to be a workgroup's): heads, kv, rows, and the weights' floor.
KERNELS = {"16": (4, 2, [1], FEW_FLOOR), "32": (48, 2, [1], FEW_FLOOR), "64": (12, 1, [4], MANY_FLOOR), "128": (20, 1, [7], MANY_FLOOR)}
ROOM = 1 << 18


def one_each(rng, hd, kernel, dtype="f16"):
    """A cache whose keys and values have one value that is not zero, each position another: a score is one product,
    a result the weight of one position."""
    heads, kv, rows, floor = KERNELS[kernel]
    n = min(hd, 61)
    c = M.Cache(rng, dtype, kv, hd, 16, rows, [n], room=ROOM)
    c.k[:], c.v[:] = 0, 0
    page, slot, _ = c.slots(0, n)
    for j in range(kv):
        c.k[page, j, slot, rng.permutation(hd)[:n]] = rng.uniform(0.5, 2, n) * rng.choice([-1, 1], n)
        c.v[page, j, slot, rng.permutation(hd)[:n]] = 1
    q = (rng.uniform(1, 2, (c.n_rows, heads, hd)) * rng.choice([-1, 1], (c.n_rows, heads, hd))).astype(np.float32)
    return c, q, heads, floor


def one_large(rng, hd, kernel):
    """Queries with one value 2^20 times the others, of a channel that the keys do not have."""
    heads, kv, rows, floor = KERNELS[kernel]
    c = M.Cache(rng, "f16", kv, hd, 16, rows, [50], room=ROOM)
    q = rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)
    q[:, :, 7] = 3.1e6
    c.k[..., 7] = 0
    return c, q, heads, floor


def one_sees_all(rng, hd, kernel, least=16):
    """One weight far above many equal ones, 2^-least of it and a little: the small ones together weigh as much."""
    heads, kv, rows, floor = KERNELS[kernel]
    n = 4000
    c = M.Cache(rng, "f16", kv, hd, 16, rows, [n], room=ROOM)
    c.k[:], c.v[:] = 0, 0
    page, slot, _ = c.slots(0, n)
    c.k[page[5], :, slot[5], 0] = 1
    c.v[page[5], :, slot[5], 0] = 1
    c.v[page[6:], :, slot[6:], 1] = 1
    q = np.zeros((c.n_rows, heads, hd), np.float32)
    q[:, :, 0] = (least - np.log2(1.37)) * np.log(2)
    return c, q, heads, floor


def every_position(rng, dtype, rows, heads, n, hd=64, shared=0):
    """Queries of zero over n positions: every position weighs the same, and the values, small whole numbers, say which
    were added how often: position p adds 1 + (t // 1024) % 3 to columns t % 32 and 32 + (t // 32) % 32 of its tile t of
    32. Returns (cache, queries, exact results, tolerance). A sum takes at most 800 roundings of f32 in o and as many in
    l (of its workgroup's tiles one after another, of the workgroups)."""
    c = M.Cache(rng, dtype, 1, hd, 256, rows, [n - i for i in range(len(rows))], shared=shared)
    p = np.arange(n)
    t = p // 32
    value = np.zeros((n, hd))
    value[p, t % 32] = 1 + t // 1024 % 3
    value[p, 32 + t // 32 % 32] = 1 + t // 1024 % 3
    c.k[:], c.v[:] = 0, 0
    total = np.cumsum(value, 0)
    for b in range(len(rows)):
        page, slot, ok = c.slots(b, c.lens[b])
        assert ok.all()
        c.v[page, 0, slot] = value[:c.lens[b]]
        c.k[page, 0, slot] = rng.standard_normal((c.lens[b], hd))
    want = np.stack([total[pos] / (pos + 1) for _, pos in c.row_positions()])
    return c, np.zeros((c.n_rows, heads, hd), np.float32), value, np.repeat(want[:, None], heads, 1), 2 * 800 * U32 * want[:, None]
