"""GPU tests of a server's turn of drafts over GatedDeltaNet layers
(include/uq_serve.h): several sequences draft, each has another number of rows
accepted, and a second call over the same rows takes windows and states on,
the refused rows as sequences of their own that begin with and leave nothing."""
import numpy as np
import pytest

import gdn_model as M
from test_gpu_gdn_serve import MARK, Conv, Rule, bits, dev, hip_of_bench, host
from uq import serve

pytestmark = pytest.mark.gpu


def of_kept(c, kept):
    """The batch of a step's rows, each sequence as its kept rows and its refused ones: starts, slots."""
    start, frm, to = [0], [], []
    for b, n in enumerate(c.rows):
        lo = int(c.start[b])
        start += [lo + kept[b], lo + n]
        frm += [int(c.frm[b]), -1]
        to += [b, -1]
    return tuple(np.array(a, np.int32) for a in (start, frm, to))


def heads_of(c, conv):
    at = []
    for floats in (0, c.nqk * c.hd, 2 * c.nqk * c.hd):
        v = type("View", (), {})()
        v.ptr, v.nbytes = conv.out.ptr.value + 4 * floats, 0
        at.append(v)
    return serve.GdnHeads(at[0], c.ch, at[1], c.ch, at[2], c.ch, conv.gate, conv.beta, c.scale, dev(c.norm), M.EPS, dev(c.z), c.nv * c.hd)


@pytest.mark.parametrize("rows,kept,hd", [
    ([5, 5, 4, 1, 6], [2, 3, 4, 1, 1], 64), ([5, 3, 5], [1, 1, 5], 128), ([70, 5, 90, 4], [70, 2, 90, 3], 64), ([40, 80, 33], [25, 7, 33], 64)])
def test_each_sequence_keeps_its_own_rows(rows, kept, hd):
    """Against 64 bits: the second call's windows are the inputs bit for bit, and its states those of the kept rows alone."""
    n = len(rows)
    c = M.Case(111, 2, 4, hd, 4, rows, frm=[-1] + list(range(1, n)), to=[-1] * n, spare=1, pad=2)
    conv, rule = Conv(c), Rule(c, 0)
    conv.run()
    rule.heads, rule.states, rule.batch = heads_of(c, conv), conv.states, conv.batch
    rule.run()
    first, before = host(rule.out, c.z), host(conv.states._bufs[1], c.state)
    assert np.array_equal(bits(before), bits(c.state)), "drafts leave no state"
    start, frm, to = of_kept(c, kept)
    d_frm, d_to = dev(frm), dev(to)
    states = serve.GdnStates(conv.states._bufs[0], conv.states._bufs[1], c.slots, c.nqk, c.nv, c.hd, c.taps, d_frm, d_to)
    batch = serve.SeqBatch(2 * n, c.n_rows, dev(start))
    ws = type(rule.ws)(serve.gdn_rule_ws_bytes(states, batch, 0))
    conv.out.upload(np.full(c.qkv.shape, MARK, np.float32))
    serve.gdn_conv_d(states, batch, conv.rows)
    heads, beta, gate = (host(a, like) for a, like in ((conv.out, c.qkv), (conv.beta, c.beta), (conv.gate, c.gate)))
    serve.gdn_rule_d(rule.out, states, batch, rule.heads, ws)
    got, st, win = host(rule.out, c.z), host(conv.states._bufs[1], c.state), host(conv.states._bufs[0], c.win)

    def alone():
        """The kept rows alone, closed up, each sequence into its slot."""
        k = M.Case(111, 2, 4, hd, 4, kept, frm=c.frm, to=list(range(n)), spare=1)
        pick = np.concatenate([np.arange(c.start[b], c.start[b] + kept[b]) for b in range(n)])
        k.win, k.state, k.conv1d, k.dt_bias, k.a, k.norm = c.win, c.state, c.conv1d, c.dt_bias, c.a, c.norm
        for name in ("qkv", "beta_raw", "alpha", "z"):
            setattr(k, name, np.ascontiguousarray(getattr(c, name)[pick]))
        return k, pick

    k, pick = alone()
    (want, tol), _, _, kept_win = M.conv(k)
    assert np.all(np.abs(heads[pick] - want) <= tol)
    assert np.array_equal(win, kept_win.astype(np.float32))
    # the rule of the kernel's own heads, so that the bound is the rule's alone
    q, kk, v = np.split(heads[pick].reshape(len(pick), -1, hd), [c.nqk, 2 * c.nqk], 1)
    k.q, k.k, k.v, k.beta, k.gate = q, kk, v, beta[pick], gate[pick]
    (want, tol), (ws64, wtol) = M.rule(k)
    assert np.all(np.abs(got[pick] - want) <= tol)
    assert np.all(np.abs(st - ws64) <= wtol)
    if max(rows) < 24:  # row by row in both calls
        assert np.array_equal(bits(got[pick]), bits(first[pick]))
    assert np.all(got[c.n:] == MARK)


def test_a_captured_turn():
    """Twice as many sequences as draft, captured once: starts and slots are set for the turn on the device."""
    hip = hip_of_bench()
    s = hip.stream()
    rows = [5, 5, 5]
    c = M.Case(112, 2, 4, 64, 4, rows, frm=[0, 1, 2], to=[-1] * 3, spare=1)
    conv, eager = Conv(c), Conv(c)
    d_start, d_frm, d_to = (dev(np.zeros(k, np.int32)) for k in (7, 6, 6))
    batch = serve.SeqBatch(6, c.n_rows, d_start)
    run = []
    for x in (conv, eager):
        st = serve.GdnStates(x.states._bufs[0], x.states._bufs[1], c.slots, c.nqk, c.nv, c.hd, c.taps, d_frm, d_to)
        out = dev(np.full(c.z.shape, MARK, np.float32))
        ws = type(out)(serve.gdn_rule_ws_bytes(st, batch, 5))
        h = heads_of(c, x)

        def call(stream=None, x=x, st=st, out=out, ws=ws, h=h):
            serve.gdn_conv_d(st, batch, x.rows, stream)
            serve.gdn_rule_d(out, st, batch, h, ws, 5, stream)

        run.append((call, st, out))
    hip.sync()
    g = hip.capture(s, lambda: run[0][0](s))
    rng = np.random.default_rng(2)
    for turn, kept in enumerate(([5, 5, 5], [1, 2, 3], [1, 1, 1], [4, 5, 1])):
        start, frm, to = of_kept(c, kept)
        x = rng.standard_normal(c.qkv.shape).astype(np.float32)
        for d, a in ((d_start, start), (d_frm, frm), (d_to, to), (conv.rows._bufs[0], x), (eager.rows._bufs[0], x)):
            d.upload(a)
        hip.sync()
        hip.launch_graph(g, s)
        hip.sync()
        run[1][0]()
        for i, like in ((0, c.win), (1, c.state)):
            assert np.array_equal(bits(host(run[0][1]._bufs[i], like)), bits(host(run[1][1]._bufs[i], like))), turn
        assert np.array_equal(bits(host(run[0][2], c.z)), bits(host(run[1][2], c.z))), turn
