"""GPU tests of the batched gated delta rule (include/uq_serve.h) with gates
above 0, which make a state larger: by rows and by chunks."""
import numpy as np
import pytest

import gdn_model as M
from test_gpu_gdn_serve import Rule

pytestmark = pytest.mark.gpu

U = M.U


def rule(c):
    """(out, bound), (states, bound) in 64 bits, row after row, without norm and gate.

    gdn_model.rule's bound with decays that may be above 1: a row's step takes an error on by e^g at most (keys of norm
    1, betas to 1). What a chunk's operands lose below its largest value, 2^-39 of a bound on it that is a power of 2,
    is a term of its own, as rows differ by their decays: the bound on X is max |v| + hd max |k| max e^G max |S|, that on
    U its largest."""
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
                D = np.exp(np.tril(G[:, None] - G[None, :]))
                A = np.tril(be[:, None] * D * (K @ K.T), -1)
                P = np.tril(D * (Q @ K.T))
                T = np.linalg.inv(np.eye(len(be)) + A)
                X = be[:, None] * (V - np.exp(G)[:, None] * (K @ S))
                through = 64 * U * (np.abs(np.eye(len(be)) + A) @ (np.abs(T) @ np.abs(X)))
                Uu = T @ X
                lost_x = 2.0 ** -38 * (np.abs(V).max(0) + hd * np.abs(K).max() * np.exp(G.max()) * np.abs(S).max(0))
                lost_u = 2.0 ** -38 * np.abs(Uu).max(0)
                M0 = np.linalg.norm(S, axis=0)
                for i, row in enumerate(rows):
                    S = np.exp(g64[row, h]) * S
                    m = np.linalg.norm(S, axis=0)
                    d = be[i] * (V[i] - K[i] @ S)
                    S = S + np.outer(K[i], d)
                    size = np.linalg.norm(S, axis=0)
                    E = (np.exp(g64[row, h]) * E + be[i] * (c1 * (np.abs(V[i]) + m + np.exp(G[i]) * M0) + lost_x) + through[i] + 8 * U * size)
                    out[row, h] = c.scale * (Q[i] @ S)
                    nq = np.linalg.norm(Q[i])
                    sizes = nq * (np.exp(G[i]) * M0 + size) + np.abs(P[i]) @ np.abs(Uu)
                    tol[row, h] = c.scale * (nq * E + c1 * sizes + np.abs(P[i]).sum() * lost_u)
                last = np.exp(G[-1] - G)
                Kl = np.abs(K) * last[:, None]
                E = E + c1 * (np.linalg.norm(Kl.T @ np.abs(Uu), axis=0) + np.exp(G[-1]) * M0) + Kl.sum() * lost_u
            if t is not None:
                states[t, h], stol[t, h] = S, E[None, :] + 4 * U * np.abs(S)
    return (out, tol + 1e-37), (states, stol)


@pytest.mark.parametrize("hd,rows,frm", [(64, [150, 1, 40, 5], None), (128, [130, 64, 3], None), (64, [70, 200], [-1, -1])])
def test_gates_above_zero(hd, rows, frm):
    """States that grow and decay in turns, single rows that multiply them, and a chunk's first and last row that do."""
    c = M.Case(131, 2, 4, hd, 4, rows, frm=frm)
    i = np.arange(c.n_rows)[:, None]
    c.gate[:] = 0.12 * np.sin(i / 9 + np.arange(c.nv))
    c.gate[20], c.gate[63], c.gate[64], c.gate[90:92] = 2.5, 1.5, 1.0, -2.0
    r = Rule(c, 0, (False, False))
    r.run()
    out, st = r.results()
    (want, tol), (ws, wt) = rule(c)
    assert np.all(np.abs(out - want) <= tol), np.max(np.abs(out - want) / tol)
    assert np.all(np.abs(st - ws) <= wt)


def test_one_gate_above_zero_is_seen_by_its_head_alone():
    c = M.Case(132, 2, 4, 64, 4, [100, 70])
    c.gate[33, 2] = 0.7
    r = Rule(c, 0, (False, False))
    r.run()
    out, st = r.results()
    (want, tol), (ws, wt) = rule(c)
    assert np.all(np.abs(out - want) <= tol) and np.all(np.abs(st - ws) <= wt)
