"""GPU tests of the GatedDeltaNet layers' batched operators (include/uq_serve.h)
beside the layer's own step of one token, in a row with the projections and the
log probabilities, over scales far from 1, and as a process's first calls."""
import os
import subprocess
import sys

import numpy as np
import pytest

import gdn_model as M
import uq
from test_gpu_gdn_serve import MARK, Conv, Rule, bits, dev, hip_of_bench, host
from test_gpu_layers import SMALL, Model, nodes_of
from uq import layer as L
from uq import serve

pytestmark = pytest.mark.gpu


def view(d, floats):
    v = type("View", (), {})()
    v.ptr, v.nbytes = d.ptr.value + 4 * floats, 0
    return v


def test_first_calls_of_a_process_captured():
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "gdn_capture_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr


# ------------------------------------------------------------------------- the layer's step

@pytest.mark.parametrize("split", [[70, 1, 4, 15], [1] * 5 + [85], [40, 50]])
def test_batch_of_a_layer_equals_its_steps(split):
    """Tokens through the layer's step one after another, and the same tokens' projections in a few calls with another
    sequence beside them: the windows bit for bit, convolution, norms and gates within the bounds of both, and from the
    step's own heads the normed and gated results and the state."""
    m = Model(SMALL, seed=91)
    c, d = m.cfg, m.d
    nqk, nv, hd, taps, nt = c.n_qk_heads, c.n_v_heads, c.head_dim_linear, c.conv_kernel, sum(split)
    ch = d.channels
    rng = np.random.default_rng(4)
    X = rng.standard_normal((nt, c.n_embd)).astype(np.float32)
    win, state = dev(np.zeros((taps, ch), np.float32)), dev(np.zeros((nv, hd, hd), np.float32))
    ws, dl = uq.DeviceArray(4 * L.ws_floats(d)), uq.DeviceArray(4 * c.n_embd)
    names = ["z", "beta_raw", "alpha", "beta", "gate", "conv_silu", "final"]
    step = {n: [] for n in names + ["qkv"]}
    for t in range(nt):
        dx = dev(X[t])
        L.gdn_step(d, m.gw, win, state, dx, dl, ws)
        for n, a in nodes_of(d, ws, names).items():
            step[n].append(a)
        step["qkv"].append(host(win, np.empty((taps, ch), np.float32))[-1])
    step = {n: np.stack(a) for n, a in step.items()}
    last_win, last_state = host(win, np.empty((taps, ch), np.float32)), host(state, np.empty((nv, hd, hd), np.float32))
    h = m.gh

    def case(n, at):
        """Those tokens in slot 1, from the second call on its state too, beside 3 rows of another sequence."""
        p = M.Case(92, nqk, nv, hd, taps, [n, 3], frm=[1 if at else -1, 0], to=[1, 2], spare=1)
        p.conv1d = h["ssm_conv1d"].reshape(ch, taps)
        p.dt_bias, p.a, p.norm = h["ssm_dt_bias"], h["ssm_a"], h["ssm_norm"]
        rows = slice(at, at + n)
        p.qkv[:n], p.beta_raw[:n], p.alpha[:n] = step["qkv"][rows], step["beta_raw"][rows], step["alpha"][rows]
        heads = step["conv_silu"][rows]
        p.q[:n], p.k[:n], p.v[:n] = (heads[:, a:b].reshape(n, -1, hd) for a, b in ((0, nqk * hd), (nqk * hd, 2 * nqk * hd), (2 * nqk * hd, ch)))
        p.beta[:n], p.gate[:n], p.z[:n] = step["beta"][rows], step["gate"][rows], step["z"][rows].reshape(n, nv, hd)
        return p

    at, w, s = 0, None, None
    exact = case(nt, 0)  # the whole in 64 bits
    (want, tol), (wst, wtol) = M.rule(exact)
    for n in split:
        p = case(n, at)
        if at:
            p.win[1], p.state[1] = w, s
        conv = Conv(p)
        conv.run()
        (_, ot), (_, bt), (_, gt), _ = M.conv(p)
        go, gb, gg, gw = conv.results()
        rule = Rule(p, n)  # whose copies of windows and states are its own
        rule.run()
        for got, ref, bound in ((go, step["conv_silu"], ot), (gb, step["beta"], bt), (gg, step["gate"], gt)):
            assert np.all(np.abs(got[:n] - ref[at:at + n]) <= 2 * bound[:n]), (n, np.max(np.abs(got[:n] - ref[at:at + n]) / bound[:n]))
        out, st = rule.results()
        w, s = gw[1], st[1]
        # calls' ends round the state once more each, inside the bound of chunks' ends
        assert np.all(np.abs(out[:n] - want[at:at + n]) <= 2 * tol[at:at + n])
        assert np.all(np.abs(out[:n].reshape(n, -1) - step["final"][at:at + n]) <= 3 * tol[at:at + n].reshape(n, -1))
        at += n
    assert np.array_equal(bits(w[:taps - 1]), bits(last_win[:taps - 1]))
    assert np.all(np.abs(s - wst[1]) <= 2 * wtol[1]) and np.all(np.abs(s - last_state) <= 3 * wtol[1])
    m.free()


def test_drafts_scored_and_taken():
    """Two turns of a server: a prompt and drafted tokens through convolution and rule, which leave no state; their heads
    through a projection and the log probabilities of given tokens; then the accepted rows again, which do."""
    nqk, nv, hd, vocab, top = 2, 4, 64, 1777, 7
    rng = np.random.default_rng(5)
    c = M.Case(93, nqk, nv, hd, 4, [70, 4, 1], frm=[-1, 1, 2], to=[0, -1, 2])
    n = c.n_rows
    head = uq.Weights(rng.standard_normal((vocab, nv * hd)).astype(np.float32) * 0.2, uq.DType.F32, nv * hd, vocab)
    conv, rule = Conv(c), Rule(c, 0)
    rule.states, rule.batch = conv.states, conv.batch
    qk = nqk * hd
    rule.heads = serve.GdnHeads(view(conv.out, 0), c.ch, view(conv.out, qk), c.ch, view(conv.out, 2 * qk), c.ch, conv.gate, conv.beta, c.scale,
                                dev(c.norm), M.EPS, dev(c.z), nv * hd)
    logits = uq.DeviceArray(4 * n * vocab)
    tokens = rng.integers(0, vocab, n).astype(np.int32)
    lp, rank, ids, tops = (uq.DeviceArray(4 * k) for k in (n, n, n * top, n * top))
    out = serve.LogProbs(lp, rank, None, ids, tops, top)
    lws = uq.DeviceArray(serve.logprobs_ws_bytes(n, vocab, top))
    d_tokens = dev(tokens)

    def turn():
        conv.run()
        rule.run()
        uq.gemm(head, n, rule.out, logits)
        serve.logprobs_d(out, logits, d_tokens, n, vocab, lws)

    state = conv.states._bufs[1]
    for accepted in (2, 4):
        before = host(state, c.state)
        turn()
        x = host(logits, np.empty((n, vocab), np.float32))
        ref = M.logprobs(x, tokens, 1.0, top)
        assert np.all(np.abs(host(lp, np.empty(n, np.float32)) - ref["logprob"]) <= ref["tol_logprob"])
        assert np.array_equal(host(rank, np.empty(n, np.int32)), ref["rank"])
        assert np.array_equal(host(ids, np.empty((n, top), np.int32)), ref["top_id"])
        first = host(rule.out, c.z)
        after = host(state, c.state)
        assert np.array_equal(bits(after[[1, 3]]), bits(before[[1, 3]])) and not np.array_equal(after[2], before[2])
        # the accepted rows of the second sequence alone, which end in its slot: the same results
        start, to = conv.batch._bufs[0], conv.states._bufs[3]
        start.upload(np.array([70, 70, 70 + accepted, 70 + accepted], np.int32))
        to.upload(np.array([0, 1, 2], np.int32))
        conv.run()
        rule.run()
        again, later = host(rule.out, c.z), host(state, c.state)
        assert np.array_equal(bits(again[70:70 + accepted]), bits(first[70:70 + accepted]))
        assert np.array_equal(bits(later[[0, 2, 3]]), bits(after[[0, 2, 3]])) and not np.array_equal(later[1], after[1])
        start.upload(c.start)
        to.upload(c.to)


def test_two_streams_at_once():
    """Calls of two streams, each with states and a workspace of its own, under way at the same time."""
    hip = hip_of_bench()
    streams = [hip.stream(), hip.stream()]
    cases = [M.Case(99, 2, 4, 128, 4, [200, 1, 70], frm=[0, 1, 2], to=[3, 4, 5], spare=3),
             M.Case(100, 2, 6, 64, 4, [90, 5, 300], frm=[0, 1, 2], to=[3, 4, 5], spare=3)]
    runs = [(Conv(c), Rule(c, 0)) for c in cases]
    hip.sync()
    want = []
    for conv, rule in runs:
        conv.run()
        rule.run()
        want.append((host(conv.out, conv.c.qkv), *rule.results()))
        for d in (conv.out, rule.out):
            d.upload(np.full(d.nbytes // 4, MARK, np.float32))
    hip.sync()
    for _ in range(6):
        for (conv, rule), s in zip(runs, streams):
            conv.run(s)
            rule.run(s)
    hip.sync()
    for (conv, rule), (out, heads, st) in zip(runs, want):
        got, gs = rule.results()
        assert np.array_equal(bits(host(conv.out, conv.c.qkv)), bits(out))
        assert np.array_equal(bits(got), bits(heads)) and np.array_equal(bits(gs), bits(st))


# ------------------------------------------------------------------------- scales

ROWS = [1, 5, 33, 150]


def plain(change=None, hd=64):
    """Results without norm and gate of a case whose arrays `change` has scaled. Every sequence begins with a state: that
    of none is 0, whatever its scale."""
    c = M.Case(94, 2, 4, hd, 4, ROWS, decay=(-6, 0))
    if change:
        change(c)
    r = Rule(c, 0, (False, False))
    r.run()
    return r.results()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [-70, -20, 20, 90])
def test_rule_is_linear_in_values_and_state(power, hd):
    """By powers of 2 bit for bit: every scale that the kernels choose is one."""
    def change(c):
        c.v *= np.float32(2.0 ** power)
        c.state *= np.float32(2.0 ** power)

    want, ws = plain(hd=hd)
    got, gs = plain(change, hd)
    assert np.array_equal(bits(got), bits(np.ldexp(want, power))) and np.array_equal(bits(gs), bits(np.ldexp(ws, power)))


def test_rule_has_a_scale_for_each_column():
    power = (np.arange(64) * 37 % 101 - 50).astype(np.int32)

    def change(c):
        c.v[:] = np.ldexp(c.v, power)
        c.state[:] = np.ldexp(c.state, power)

    want, ws = plain()
    got, gs = plain(change)
    assert np.array_equal(bits(got), bits(np.ldexp(want, power))) and np.array_equal(bits(gs), bits(np.ldexp(ws, power)))


@pytest.mark.parametrize("power", [-12, 3, 20])
def test_rule_of_keys_of_other_norms(power):
    """Keys 2^p times larger, betas 4^-p and states 2^-p times: A is the same, corrections are 4^-p times, results 2^-p."""
    def change(c):
        c.k *= np.float32(2.0 ** power)
        c.beta *= np.float32(4.0 ** -power)
        c.state *= np.float32(2.0 ** -power)

    want, ws = plain()
    got, gs = plain(change)
    assert np.array_equal(bits(got), bits(np.ldexp(want, -power))) and np.array_equal(bits(gs), bits(np.ldexp(ws, -power)))


def test_rule_of_nothing_and_after_it():
    """States, values, keys, queries and betas of zeros, for a chunk each, leave zeros or what the formula leaves."""
    c = M.Case(95, 1, 2, 64, 4, [64 * 7, 40], frm=[-1, 0])
    c.v[:64] = 0
    c.k[64:128] = 0
    c.q[128:192] = 0
    c.beta[192:256] = 0
    c.gate[256:320] = -np.inf
    c.v[320:384], c.gate[320:384] = 0, 0
    r = Rule(c, 0)
    r.run()
    with np.errstate(all="ignore"):
        c.gate = np.maximum(c.gate, -3000)  # e^-3000 is 0 in 64 bits too
        out, _ = r.check()
    assert np.all(out[:64] == 0) and np.all(out[128:192] == 0)


def test_rule_of_values_far_smaller_than_the_state():
    """A state of 1 that is forgotten, and values that are 2^-10 of it: what is left is theirs. In the chunk of 64 rows
    that the state ends in, the values that U solves for keep 2^-39 of |v| + 64 |k| |S| < 2^6 in largest values, twice
    that for its power of 2: 2^-32, below the bound's 160 2^-24 of values of 2^-14."""
    c = M.Case(96, 1, 1, 64, 4, [128], frm=[0], to=[0])
    c.v *= np.float32(2.0 ** -10)
    c.gate[10] = -1000
    r = Rule(c, 0, (False, False))
    r.run()
    out, st = r.results()
    (want, tol), (ws, wt) = M.rule(c, False)
    assert np.all(np.abs(out[:10] - want[:10]) <= tol[:10])
    # after the row the model begins anew: the same rows as a sequence of their own
    d = M.Case(96, 1, 1, 64, 4, [118], frm=[-1], to=[0])
    for name in ("q", "k", "v", "gate", "beta"):
        setattr(d, name, np.ascontiguousarray(getattr(c, name)[10:]))
    (want, tol), (ws, wt) = M.rule(d, False)
    ratio = np.abs(out[64:] - want[54:]) / tol[54:]
    assert np.all(np.abs(out[64:] - want[54:]) <= 2 * tol[54:]), ratio.max()
    assert np.all(np.abs(st[0] - ws[0]) <= 2 * wt[0])


@pytest.mark.parametrize("nqk,nv,hd,rows", [(4, 32, 64, [35] * 19 + [90]), (2, 34, 128, [70, 1, 33] * 6 + [40] * 7)])
def test_rule_of_many_heads(nqk, nv, hd, rows):
    """Many value heads of a key head in one workgroup, one after another; single rows between."""
    r = Rule(M.Case(98, nqk, nv, hd, 4, rows), 0)
    r.run()
    r.check()


def test_rows_of_no_sequence_between():
    """Row starts that leave rows out before, between and behind: as they were."""
    c = M.Case(97, 2, 2, 64, 4, [50, 3], pad=70)
    r = Rule(c, 0)
    start = np.array([20, 70, 73], np.int32)
    for name in ("q", "k", "v", "gate", "beta", "z"):
        a = getattr(c, name)
        a[20:73] = a[:53].copy()
    r = Rule(c, 0)
    c.d_start.upload(start)
    r.run()
    out, _ = r.results()
    ref = M.Case(97, 2, 2, 64, 4, [50, 3], pad=70)
    (want, tol), _ = M.rule(ref)
    assert np.all(np.abs(out[20:73] - want[:53]) <= tol[:53])
    assert np.all(out[:20] == MARK) and np.all(out[73:] == MARK)
