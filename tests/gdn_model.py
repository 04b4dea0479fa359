"""The GatedDeltaNet operators of batched serving and the log probabilities
(include/uq_serve.h) in 64-bit numpy, with bounds on the kernels' distance
from them."""
import numpy as np

import uq
from uq import serve

U = 2.0 ** -24  # half a step of f32, relative
EPS = 1e-6


class Case:
    """The rows of a batch, its states in slots, and what the two operators take."""

    def __init__(self, seed, nqk, nv, hd, taps, rows, frm=None, to=None, spare=1, pad=0, decay=(-6.5, 1.5)):
        rng = self.rng = np.random.default_rng(seed)
        self.nqk, self.nv, self.hd, self.taps, self.rows = nqk, nv, hd, taps, list(rows)
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.n, self.n_rows, self.ch = int(self.start[-1]), int(self.start[-1]) + pad, (2 * nqk + nv) * hd
        self.slots = len(rows) + spare
        own = rng.permutation(self.slots)[:len(rows)]
        self.frm = np.array(own if frm is None else frm, np.int32)
        self.to = np.array(own if to is None else to, np.int32)

        def normal(*s):
            return rng.standard_normal(s).astype(np.float32)

        N = self.n_rows
        self.win, self.state = normal(self.slots, taps, self.ch), 0.3 * normal(self.slots, nv, hd, hd)
        self.qkv, self.conv1d = normal(N, self.ch), 0.5 * normal(self.ch, taps)
        self.beta_raw, self.alpha = normal(N, nv), 3 * normal(N, nv)
        self.dt_bias, self.a = normal(nv), -np.exp(rng.random(nv)).astype(np.float32)
        x = normal(N, 2 * nqk + nv, hd)
        x[:, :2 * nqk] /= np.linalg.norm(x[:, :2 * nqk].astype(np.float64), axis=-1, keepdims=True).astype(np.float32)
        self.q, self.k, self.v = (np.ascontiguousarray(p) for p in (x[:, :nqk], x[:, nqk:2 * nqk], x[:, 2 * nqk:]))
        self.gate = -np.exp(rng.uniform(*decay, (N, nv))).astype(np.float32)
        self.beta = rng.random((N, nv)).astype(np.float32)
        self.z, self.norm, self.scale = normal(N, nv, hd), (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32), hd ** -0.5

    def seqs(self):
        """(sequence, its rows' slice, state it begins with: a slot or None, slot it ends in or None)"""
        def slot(i):
            return int(i) if 0 <= i < self.slots else None

        for b, n in enumerate(self.rows):
            if n:
                yield b, slice(int(self.start[b]), int(self.start[b + 1])), slot(self.frm[b]), slot(self.to[b])

    def upload(self):
        dev = uq.DeviceArray.from_numpy
        self.d_win, self.d_state, self.d_start, self.d_from, self.d_to = (
            dev(a) for a in (self.win, self.state, self.start, self.frm, self.to))
        states = serve.GdnStates(self.d_win, self.d_state, self.slots, self.nqk, self.nv, self.hd, self.taps, self.d_from, self.d_to)
        return states, serve.SeqBatch(len(self.rows), self.n_rows, self.d_start)


def silu(x):
    return x / (1 + np.exp(-x))


def conv(c):
    """(out, bound), (beta, bound), (gate, bound), windows; rows of no sequence NaN.

    The convolution's products and sums: (taps + 1) U of the sum of the products' sizes. silu: its slope is at most
    1.1, and of its value 4 U for the exponential, 1 + it, the reciprocal and the product 2 U each at most. A head's
    norm: 7 sums a lane and over lanes and a root, half of them each, and a root, quotient and product of 2 U at most."""
    out = np.full((c.n_rows, c.ch), np.nan)
    tol = out.copy()
    win = c.win.astype(np.float64)
    w = c.conv1d.astype(np.float64).T
    for b, r, f, t in c.seqs():
        old = c.win[f, :c.taps - 1].astype(np.float64) if f is not None else np.zeros((c.taps - 1, c.ch))
        x = np.concatenate([old, c.qkv[r].astype(np.float64)])
        n = r.stop - r.start
        parts = [x[k:k + n] * w[k] for k in range(c.taps)]
        s, size = sum(parts), sum(np.abs(p) for p in parts)
        y = silu(s)
        e = 1.1 * (c.taps + 1) * U * size + 12 * U * np.abs(y)
        h, he = (a.reshape(n, -1, c.hd) for a in (y, e))
        q, qe = h[:, :2 * c.nqk], he[:, :2 * c.nqk]
        norm = np.linalg.norm(q, axis=-1, keepdims=True)
        ne = np.linalg.norm(qe, axis=-1, keepdims=True)
        big = np.maximum(norm, EPS)
        he[:, :2 * c.nqk] = qe / big + np.abs(q) / big * (ne / big + 16 * U)
        h[:, :2 * c.nqk] = q / big
        out[r], tol[r] = y, e + 1e-37
        if t is not None:
            win[t, :c.taps - 1] = x[n:]
    x = c.alpha.astype(np.float64) + c.dt_bias
    sp = np.logaddexp(0, x)
    gate = sp * c.a
    beta = 1 / (1 + np.exp(-c.beta_raw.astype(np.float64)))
    # the sum's rounding and that of its size's exponential; 12 roundings of the value
    gtol = np.abs(c.a) * (U * np.abs(x) + 12 * U * sp) + 1e-37
    return (out, tol), (beta, 10 * U * beta + 1e-37), (gate, gtol), win


def rule(c, finish=True):
    """(out, bound), (states, bound) of the rule, row after row in 64 bits; rows of no sequence NaN.

    The bound follows the computation in chunks of 64 rows, which takes in that row by row. A row's correction d = U
    is off by its product with the state and the value (c1 = (hd + 96) U of the sizes multiplied: at most hd + 64
    f32 additions and operands within 2^-22), and, solved through the inverse T of the chunk's triangle, by
    64 U |I + A| |T| |X| more. As keys have norm 1 and betas and decays are at most 1, a row's step does not enlarge
    an earlier state's error (2-norm of a column), so errors E of the columns add up, decayed:
        E <- e^g E + |k| residual + 8 U |S|,
    and at a chunk's end by c1 |K|^T |U|. Outputs are off by |q| E and c1 of the products' sizes. The norm and the
    gate pass that on to first order, 24 U of the value more."""
    N, hd = c.n_rows, c.hd
    out, tol = np.full((N, c.nv, hd), np.nan), np.full((N, c.nv, hd), np.nan)
    states, stol = c.state.astype(np.float64), np.zeros(c.state.shape)
    c1 = (hd + 96) * U
    k64, q64, v64 = (a.astype(np.float64) for a in (c.k, c.q, c.v))
    g64, b64 = c.gate.astype(np.float64), c.beta.astype(np.float64)
    for _, r, f, t in c.seqs():
        for h in range(c.nv):
            hq = h % c.nqk
            S = c.state[f, h].astype(np.float64) if f is not None else np.zeros((hd, hd))
            E = np.zeros(hd)
            for lo in range(r.start, r.stop, 64):
                rows = range(lo, min(lo + 64, r.stop))
                K, Q, V, be = k64[rows, hq], q64[rows, hq], v64[rows, h], b64[rows, h]
                G = np.cumsum(g64[rows, h])
                D = np.exp(np.minimum(0, G[:, None] - G[None, :]))
                A = np.tril(be[:, None] * D * (K @ K.T), -1)
                P = np.tril(D * (Q @ K.T))
                T = np.linalg.inv(np.eye(len(be)) + A)
                X = be[:, None] * (V - np.exp(G)[:, None] * (K @ S))
                through = 64 * U * (np.abs(np.eye(len(be)) + A) @ (np.abs(T) @ np.abs(X)))
                Uu = T @ X
                S0, M0 = S, np.linalg.norm(S, axis=0)
                for i, row in enumerate(rows):
                    S = np.exp(g64[row, h]) * S
                    M = np.linalg.norm(S, axis=0)
                    d = be[i] * (V[i] - K[i] @ S)
                    S = S + np.outer(K[i], d)
                    E = np.exp(g64[row, h]) * E + c1 * be[i] * (np.abs(V[i]) + M) + through[i] + 8 * U * np.linalg.norm(S, axis=0)
                    out[row, h] = c.scale * (Q[i] @ S)
                    nq = np.linalg.norm(Q[i])
                    sizes = nq * (np.exp(G[i]) * M0 + np.linalg.norm(S, axis=0)) + np.abs(P[i]) @ np.abs(Uu)
                    tol[row, h] = c.scale * (nq * E + c1 * sizes)
                last = np.exp(G[-1] - G)
                E = E + c1 * (np.linalg.norm((np.abs(K) * last[:, None]).T @ np.abs(Uu), axis=0) + np.exp(G[-1]) * M0)
            if t is not None:
                states[t, h], stol[t, h] = S, E[None, :] + 4 * U * np.abs(S)
    if finish:
        o, e = out, tol
        ms = (o * o).mean(-1, keepdims=True) + EPS
        by = 1 / np.sqrt(ms)
        y = o * by * c.norm
        ye = np.abs(by * c.norm) * (e + np.abs(o) * (np.abs(o) * e).mean(-1, keepdims=True) / ms)
        zs = silu(c.z.astype(np.float64))
        out = y * zs
        tol = ye * np.abs(zs) + 24 * U * np.abs(out)
    return (out, tol + 1e-37), (states, stol)


def logprobs(x, tokens, scale, n_top):
    """dict of results and tol_logprob, tol_entropy, tol_top for one row after another.

    Sums: at most 4 in a tile's parts, 3 of them, 16 tiles with a rescaling of 3 roundings each, 6 levels of lanes,
    16 parts a lane and their rescalings, 6 levels again: under 112 roundings, of the sum's size. A term's exponent is
    off by three roundings of itself, the exponential by 2."""
    out = {k: [] for k in ("logprob", "rank", "entropy", "top_id", "top_logprob", "tol_logprob", "tol_entropy", "tol_top")}
    vocab = x.shape[1]
    for row, t in zip(x, tokens):
        a = row.astype(np.float64)
        bad = np.isnan(a).any() or np.isposinf(a).any()
        possible = np.nonzero(a > -np.inf)[0]
        order = np.lexsort((np.arange(vocab), -a)) if not bad else np.array([], int)
        inside = 0 <= t < vocab
        ids = np.full(n_top, -1)
        lps, tols = np.full(n_top, -np.inf), np.zeros(n_top)
        if bad:
            lp = ent = np.nan
            lps[:] = np.nan
            tl = te = 0.0
        elif not len(possible):
            lp, ent, tl, te = -np.inf, 0.0, 0.0, 0.0
        else:
            m = a.max()
            d = np.float64(np.float32(scale)) * (m - a[possible])
            e = np.exp(-d)
            ln = np.log(e.sum())
            p = e / e.sum()
            base = U * (112 + 4 * (p @ d) + 2 * abs(ln))
            ent = ln + p @ d
            te = base + U * (112 * (p @ d) + 4 * (p @ (d * d)) + 4 * abs(ent) + 4)

            def one(i):
                di = np.float64(np.float32(scale)) * (m - a[i])
                return -di - ln, base + U * (2 * di + 2 * abs(di + ln))

            lp, tl = one(t) if inside else (-np.inf, 0.0)
            for j, i in enumerate(order[:min(n_top, len(possible))]):
                ids[j] = i
                lps[j], tols[j] = one(i)
        rank = int(np.sum(a > a[t]) + np.sum(a[:t] == a[t])) if inside and not bad else -1
        for k, val in zip(out, (lp, rank, ent, ids, lps, tl, te, tols)):
            out[k].append(val)
    return {k: np.array(v) for k, v in out.items()}
