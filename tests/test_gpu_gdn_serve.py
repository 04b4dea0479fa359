"""GPU tests of the GatedDeltaNet layers' operators of batched serving
(include/uq_serve.h) against 64-bit models (gdn_model.py): head shapes, taps,
ragged and padded batches, slots, values that are not finite, other streams,
graphs, and the operators in a row."""
import os
import sys

import numpy as np
import pytest

import gdn_model as M
import uq
from uq import serve

pytestmark = pytest.mark.gpu
MARK = np.float32(7.0)


def dev(a):
    return uq.DeviceArray.from_numpy(a)


def host(d, like):
    uq.synchronize()
    return d.download(like.dtype, like.size).reshape(like.shape)


def bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.int32)


def hip_of_bench():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if root not in sys.path:
        sys.path.insert(0, root)
    import bench

    return bench.Hip()


class Conv:
    """A case's convolution on the device."""

    def __init__(self, c, pads=(0, 0)):
        self.c = c
        wide = np.full((c.n_rows, c.ch + pads[0]), MARK, np.float32)
        wide[:, :c.ch] = c.qkv
        raw = [np.full((c.n_rows, c.nv + pads[1]), MARK, np.float32) for _ in range(2)]
        raw[0][:, :c.nv], raw[1][:, :c.nv] = c.beta_raw, c.alpha
        self.out, self.beta, self.gate = (dev(np.full(s, MARK, np.float32)) for s in ((c.n_rows, c.ch), (c.n_rows, c.nv), (c.n_rows, c.nv)))
        self.states, self.batch = c.upload()
        self.rows = serve.GdnRows(dev(wide), c.ch + pads[0], dev(c.conv1d), M.EPS, self.out, dev(raw[0]), dev(raw[1]), dev(c.dt_bias), dev(c.a),
                                  self.beta, self.gate, c.nv + pads[1])

    def run(self, stream=None):
        serve.gdn_conv_d(self.states, self.batch, self.rows, stream)

    def results(self):
        c = self.c
        return host(self.out, np.empty((c.n_rows, c.ch), np.float32)), host(self.beta, c.beta), host(self.gate, c.gate), host(c.d_win, c.win)


class Rule:
    """A case's delta rule on the device; its queries, keys and values in rows of one array, `pad` floats apart."""

    def __init__(self, c, most=0, finish=(True, True), pad=0):
        self.c, self.most = c, most
        N, wide = c.n_rows, c.ch + pad
        x = np.full((N, wide), MARK, np.float32)
        x[:, :c.ch] = np.concatenate([a.reshape(N, -1) for a in (c.q, c.k, c.v)], 1)
        self.x, self.out = dev(x), dev(np.full((N, c.nv, c.hd), MARK, np.float32))
        z = np.full((N, c.nv * c.hd + pad), MARK, np.float32)
        z[:, :c.nv * c.hd] = c.z.reshape(N, -1)

        def at(floats):
            v = type("View", (), {})()
            v.ptr, v.nbytes = self.x.ptr.value + 4 * floats, 0
            return v

        qk = c.nqk * c.hd
        self.heads = serve.GdnHeads(at(0), wide, at(qk), wide, at(2 * qk), wide, dev(c.gate), dev(c.beta), c.scale, dev(c.norm) if finish[0] else None,
                                    M.EPS, dev(z) if finish[1] else None, c.nv * c.hd + pad)
        self.states, self.batch = c.upload()
        self.ws = uq.DeviceArray(serve.gdn_rule_ws_bytes(self.states, self.batch, most))
        self.ws.upload(np.full(self.ws.nbytes, 0xFF, np.uint8))

    def run(self, stream=None):
        serve.gdn_rule_d(self.out, self.states, self.batch, self.heads, self.ws, self.most, stream)

    def results(self):
        c = self.c
        return host(self.out, np.empty((c.n_rows, c.nv, c.hd), np.float32)), host(c.d_state, c.state)

    def check(self, finish=True):
        out, st = self.results()
        (want, tol), (ws, wt) = M.rule(self.c, finish)
        n = self.c.n
        assert np.all(np.abs(out[:n] - want[:n]) <= tol[:n]), np.nanmax(np.abs(out[:n] - want[:n]) / tol[:n])
        assert np.all(out[n:] == MARK), "rows of no sequence"
        assert np.all(np.abs(st - ws) <= wt), np.max(np.abs(st - ws) - wt)
        return out, st


# ------------------------------------------------------------------------- the convolution

@pytest.mark.parametrize("nqk,nv,hd,taps,rows,pad,pads", [
    (1, 1, 64, 4, [1], 0, (0, 0)), (2, 4, 64, 4, [3, 0, 17, 1, 16, 33], 2, (5, 1)), (3, 3, 128, 2, [1, 2, 40], 0, (0, 0)),
    (2, 6, 64, 9, [1, 7, 8, 9, 50], 1, (1, 3)), (1, 5, 128, 5, [4, 3, 2, 1], 0, (0, 0)), (16, 32, 128, 4, [1, 5, 20], 0, (0, 0)),
    (2, 2, 64, 4, [2] * 300, 3, (0, 0)), (2, 2, 64, 3, [0, 0, 0, 90] + [0] * 300 + [1, 19], 0, (0, 0))])
def test_conv(nqk, nv, hd, taps, rows, pad, pads):
    c = M.Case(nqk * 100 + taps, nqk, nv, hd, taps, rows, pad=pad)
    d = Conv(c, pads)
    d.run()
    (out, ot), (beta, bt), (gate, gt), win = M.conv(c)
    go, gb, gg, gw = d.results()
    n = c.n
    assert np.all(np.abs(go[:n] - out[:n]) <= ot[:n]), np.max(np.abs(go[:n] - out[:n]) / ot[:n])
    assert np.all(np.abs(gb[:n] - beta[:n]) <= bt[:n]) and np.all(np.abs(gg[:n] - gate[:n]) <= gt[:n])
    assert all(np.all(a[n:] == MARK) for a in (go, gb, gg)), "rows of no sequence"
    assert np.array_equal(gw, win.astype(np.float32)), "windows are inputs, bit for bit"


def test_conv_slots():
    """A new sequence, two continuations of one slot, one that leaves nothing, and slots that are none."""
    c = M.Case(5, 2, 4, 64, 4, [2, 3, 1, 20, 5], frm=[-1, 3, 3, 99, 0], to=[1, 2, 5, -7, 0], spare=1)
    d = Conv(c)
    d.run()
    (out, ot), _, _, win = M.conv(c)
    go, _, _, gw = d.results()
    assert np.all(np.abs(go - out) <= ot) and np.array_equal(gw, win.astype(np.float32))


def test_conv_without_gates():
    c = M.Case(6, 1, 2, 64, 4, [5, 2])
    states, batch = c.upload()
    out = dev(np.full((c.n_rows, c.ch), MARK, np.float32))
    serve.gdn_conv_d(states, batch, serve.GdnRows(dev(c.qkv), c.ch, dev(c.conv1d), M.EPS, out))
    (want, tol), _, _, _ = M.conv(c)
    assert np.all(np.abs(host(out, c.qkv) - want) <= tol)


def test_conv_extremes():
    """Silu and gates far out, heads of zeros and of values whose squares vanish, and values that are not finite, which
    stay in the rows and heads that they belong to."""
    c = M.Case(7, 2, 4, 64, 4, [12, 9])
    c.conv1d[:] = 0
    c.conv1d[:, 3] = 1
    c.qkv[0], c.qkv[1], c.qkv[2] = 0, 1e-30, np.linspace(-200, 200, c.ch)
    c.alpha[0], c.alpha[1], c.alpha[2] = 1e4, -1e4, np.array([-80, 80, -20, 20])
    c.beta_raw[0], c.beta_raw[1] = 100, -100
    d = Conv(c)
    d.run()
    (out, ot), (beta, bt), (gate, gt), _ = M.conv(c)
    go, gb, gg, _ = d.results()
    assert np.all(np.abs(go - out) <= ot) and np.all(np.abs(gb - beta) <= bt) and np.all(np.abs(gg - gate) <= gt)
    c = M.Case(8, 2, 4, 64, 4, [12, 9])
    clean = Conv(c)
    clean.run()
    want = clean.results()[0]
    c.qkv[4, 70], c.qkv[4, 300] = np.nan, np.inf
    d = Conv(c)
    d.run()
    got = d.results()[0]
    hit = np.zeros(got.shape, bool)
    hit[4:8, 64:128] = True
    hit[4:8, 300] = True
    assert np.array_equal(bits(got)[~hit], bits(want)[~hit]) and np.isnan(got[4:8, 64:128]).all() and not np.isfinite(got[4:8, 300]).all()


def test_conv_in_turns_is_conv_at_once():
    """Rows of a sequence in several calls: the same bits, through the window."""
    c = M.Case(9, 2, 2, 64, 4, [40], frm=[0], to=[0])
    d = Conv(c)
    d.run()
    want, wb, wg, ww = d.results()
    got, at = [], 0
    for n in (1, 2, 16, 1, 17, 3):
        part = M.Case(9, 2, 2, 64, 4, [n], frm=[0], to=[0])
        part.conv1d, part.dt_bias, part.a = c.conv1d, c.dt_bias, c.a
        part.win = c.win if at == 0 else win
        part.qkv, part.beta_raw, part.alpha = c.qkv[at:at + n], c.beta_raw[at:at + n], c.alpha[at:at + n]
        p = Conv(part)
        p.run()
        o, _, _, win = p.results()
        got.append(o)
        at += n
    assert np.array_equal(bits(np.concatenate(got)), bits(want)) and np.array_equal(bits(win), bits(ww))


# ------------------------------------------------------------------------- the rule

FEW = [(1, 1, 64, [1]), (2, 4, 128, [1] * 5), (2, 6, 64, [3, 0, 5, 1, 9]), (16, 32, 128, [1, 2]), (3, 3, 128, [4, 17, 16, 33]),
       (1, 3, 64, [1] * 130)]


@pytest.mark.parametrize("finish", [(True, True), (False, False), (True, False), (False, True)])
@pytest.mark.parametrize("nqk,nv,hd,rows", FEW[1:4])
def test_rule_of_few_rows_with_and_without_norm_and_gate(nqk, nv, hd, rows, finish):
    c = M.Case(nv + hd, nqk, nv, hd, 4, rows, pad=1)
    r = Rule(c, max(rows), finish)
    r.run()
    out, _ = r.results()
    (o, ot), _ = M.rule(c, False)
    if finish[0]:
        ms = (o * o).mean(-1, keepdims=True) + M.EPS
        ot = np.abs(c.norm) / np.sqrt(ms) * (ot + np.abs(o) * (np.abs(o) * ot).mean(-1, keepdims=True) / ms)
        o = o / np.sqrt(ms) * c.norm
    if finish[1]:
        zs = M.silu(c.z.astype(np.float64))
        o, ot = o * zs, ot * np.abs(zs)
    n = c.n
    assert np.all(np.abs(out[:n] - o[:n]) <= ot[:n] + 24 * M.U * np.abs(o[:n]) + 1e-37)
    assert np.all(out[n:] == MARK)


@pytest.mark.parametrize("nqk,nv,hd,rows", FEW)
@pytest.mark.parametrize("pad", [0, 3])
def test_rule_of_few_rows(nqk, nv, hd, rows, pad):
    r = Rule(M.Case(hd + len(rows), nqk, nv, hd, 4, rows, pad=2), max(rows), pad=pad)
    r.run()
    r.check()


@pytest.mark.parametrize("nqk,nv,hd,rows,pad", [
    (1, 1, 64, [64], 0), (2, 4, 128, [65, 31, 32, 33, 1], 5), (1, 3, 64, [300, 0, 40, 7, 128, 63], 1), (3, 3, 128, [129, 100], 0),
    (2, 2, 64, [40] * 40 + [1] * 300 + [70], 2), (16, 16, 64, [1, 200, 1], 0), (1, 2, 128, [1030], 3)])
def test_rule_of_many_rows(nqk, nv, hd, rows, pad):
    c = M.Case(nv + hd + len(rows), nqk, nv, hd, 4, rows, pad=pad)
    for most in (0, max(rows)):
        r = Rule(c, most, pad=pad)
        r.run()
        r.check()


def test_rule_of_many_rows_without_norm_and_gate():
    r = Rule(M.Case(41, 2, 4, 128, 4, [70, 3, 200]), 0, (False, False), 1)
    r.run()
    r.check(False)


def test_rule_of_many_rows_hardly_forgetting():
    """Decays near 1 and far from each other over many chunks: the state is as old as the sequence."""
    r = Rule(M.Case(42, 1, 2, 64, 4, [700], decay=(-12, 0)), 0)
    r.run()
    r.check()


@pytest.mark.parametrize("most", [0, 1, 10 ** 6])
def test_rule_of_more_rows_than_it_was_told(most):
    r = Rule(M.Case(21, 2, 4, 64, 4, [1, 90, 3]), most)
    r.run()
    r.check()


@pytest.mark.parametrize("rows", [[2, 3, 1, 20, 5], [70, 100, 33, 64, 130]])
def test_rule_slots(rows):
    c = M.Case(22, 2, 4, 64, 4, rows, frm=[-1, 3, 3, 99, 0], to=[1, 2, 5, -7, 0])
    r = Rule(c, max(rows))
    r.run()
    r.check()


def test_rule_repeats_its_bits():
    c = M.Case(23, 2, 4, 128, 4, [1, 5, 100], frm=[0, 1, 2], to=[3, 3, 3], spare=2)
    r = Rule(c, 100)
    seen = []
    for _ in range(3):
        r.run()
        seen.append(r.results()[0])
    assert all(np.array_equal(bits(s), bits(seen[0])) for s in seen[1:])


def test_rule_gates_and_betas_at_their_ends():
    """No decay and whole corrections, all forgotten at a row, decays that vanish and ones that hardly are."""
    c = M.Case(24, 2, 4, 64, 4, [7, 90])
    c.gate[:], c.beta[:] = 0, 1
    c.gate[3], c.gate[20] = -1e30, -np.inf
    c.gate[40:60] = -1e-6
    c.gate[60:64], c.gate[64:70] = -200, -50
    c.beta[5], c.beta[30:33] = 0, 0
    r = Rule(c, 90)
    r.run()
    with np.errstate(all="ignore"):
        c.gate = np.maximum(c.gate, -3000)  # e^-3000 is 0 in 64 bits too; sums of infinities are not numbers
        r.check()


def test_rule_of_equal_keys():
    """One key again and again: what a row writes the next corrects whole."""
    for seed, beta in ((25, 1.0), (26, 0.5)):
        c = M.Case(seed, 1, 2, 64, 4, [150, 6])
        c.k[:] = c.k[0]
        c.gate[:], c.beta[:] = -1e-3, beta
        r = Rule(c, 150)
        r.run()
        r.check()


@pytest.mark.parametrize("rows,at", [([9, 4], 5), ([150, 3], 70), ([150, 3], 64), ([150, 3], 63)])
@pytest.mark.parametrize("what", ["q", "k", "v", "beta", "gate"])
def test_rule_values_that_are_not_finite(rows, at, what):
    """They reach nothing before their row, no other head's results and no other sequence's."""
    mk = lambda: M.Case(27, 2, 4, 64, 4, rows)  # noqa: E731
    a = Rule(mk(), max(rows))
    a.run()
    want, ws = a.results()
    c = mk()
    x = getattr(c, what)
    x[(at, 1) + (0,) * (x.ndim - 2)] = np.nan if what != "v" else np.inf
    b = Rule(c, max(rows))
    b.run()
    got, gs = b.results()
    mine = [1, 3] if what in "qk" else [1]
    other = [h for h in range(4) if h not in mine]
    assert np.array_equal(bits(got[:at]), bits(want[:at])) and np.array_equal(bits(got[:, other]), bits(want[:, other]))
    assert np.array_equal(bits(got[rows[0]:]), bits(want[rows[0]:])), "the other sequence"
    assert np.array_equal(bits(gs[:, other]), bits(ws[:, other]))
    if what in ("k", "gate"):
        assert np.isnan(got[at:rows[0], mine]).all()


def test_rule_in_turns():
    """A sequence in several calls, few and many rows, is the sequence at once within the bound; drafts leave the state
    they began with when they end nowhere."""
    c = M.Case(28, 2, 4, 64, 4, [200], frm=[0], to=[0])
    (want, tol), (ws, wt) = M.rule(c)
    state, at = c.state, 0
    for n in (1, 5, 64, 100, 30):
        p = M.Case(28, 2, 4, 64, 4, [n], frm=[0], to=[-1])
        for name in ("q", "k", "v", "gate", "beta", "z"):
            setattr(p, name, np.ascontiguousarray(getattr(c, name)[at:at + n]))
        p.norm, p.state = c.norm, state
        r = Rule(p, n)
        r.run()
        first, st = r.results()
        assert np.array_equal(bits(st), bits(state)), "nowhere"
        r.c.d_to.upload(np.zeros(1, np.int32))
        r.run()
        out, state = r.results()
        assert np.array_equal(bits(out), bits(first))
        # the turns' ends round the state once more each: inside the bound of the chunks' ends
        assert np.all(np.abs(out - want[at:at + n]) <= 2 * tol[at:at + n])
        at += n
    assert np.all(np.abs(state - ws) <= 2 * wt)


def test_rule_beyond_32_bit_offsets():
    """Slots more than 2^32 bytes apart: a state pool of 4.5 GB."""
    nv, hd = 16, 128
    slots = 4400  # of 1 MB
    c = M.Case(29, 2, nv, hd, 4, [2, 80], frm=[0, 1], to=[0, 1], spare=0)
    small = Rule(c, 80)
    small.run()
    want, ws = small.results()
    pool = uq.DeviceArray(4 * slots * nv * hd * hd)
    per = 4 * nv * hd * hd
    place = [slots - 1, slots - 2]
    L = uq.lib()
    for i, p in enumerate(place):
        a = np.ascontiguousarray(c.state[i])
        assert L.uq_memcpy_htod(pool.ptr.value + p * per, a.ctypes.data, a.nbytes, None) == 0
        uq.synchronize()
    d_slots = dev(np.array(place, np.int32))
    st = serve.GdnStates(None, pool, slots, 2, nv, hd, 4, d_slots, d_slots)
    serve.gdn_rule_d(small.out, st, small.batch, small.heads, small.ws, 80)
    out, _ = small.results()
    assert np.array_equal(bits(out), bits(want))
    got = np.empty_like(c.state[0])
    for i, p in enumerate(place):
        assert L.uq_memcpy_dtoh(got.ctypes.data, pool.ptr.value + p * per, got.nbytes, None) == 0
        assert np.array_equal(bits(got), bits(ws[i]))
    pool.free()


# ------------------------------------------------------------------------- together

def test_replays_follow_the_rows():
    """One graph of convolution and rule; between the replays row starts, slots and inputs change on the device, with
    eager calls between, and every replay is the eager call."""
    hip = hip_of_bench()
    s = hip.stream()
    base = M.Case(31, 2, 4, 64, 4, [40, 60, 28], pad=0)
    d, r = Conv(base), Rule(base, 0)
    r.states, r.batch = d.states, d.batch
    eager_d, eager_r = Conv(base), Rule(base, 0)
    eager_r.states, eager_r.batch = eager_d.states, eager_d.batch
    # the rule's rows are the convolution's results
    qk = 2 * 64

    def of(conv):
        v = [type("View", (), {})() for _ in range(3)]
        for x, o in zip(v, (0, qk, 2 * qk)):
            x.ptr = conv.out.ptr.value + 4 * o
        return serve.GdnHeads(v[0], base.ch, v[1], base.ch, v[2], base.ch, conv.gate, conv.beta, base.scale, dev(base.norm), M.EPS, dev(base.z), 256)

    r.heads, eager_r.heads = of(d), of(eager_d)
    hip.sync()
    g = hip.capture(s, lambda: [d.run(s), r.run(s)])
    rng = np.random.default_rng(1)
    dstart, estart = d.batch._bufs[0], eager_d.batch._bufs[0]
    conv_case, eager_case = d.c, eager_d.c
    for i, rows in enumerate(([40, 60, 28], [1, 1, 1], [128, 0, 0], [0, 100, 7], [0, 0, 0])):
        start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        x = rng.standard_normal(base.qkv.shape).astype(np.float32)
        slots = rng.permutation(4)[:3].astype(np.int32)
        for conv, rule, st, to in ((d, r, dstart, d.states._bufs), (eager_d, eager_r, estart, eager_d.states._bufs)):
            conv.rows._bufs[0].upload(x)
            st.upload(start)
            to[2].upload(slots)
            to[3].upload(slots)
            conv.out.upload(np.full(base.qkv.shape, MARK, np.float32))
            rule.out.upload(np.full((base.n_rows, 4, 64), MARK, np.float32))
        hip.sync()
        hip.launch_graph(g, s)
        hip.sync()
        eager_d.run()
        eager_r.run()
        for a, b, like in ((d.out, eager_d.out, base.qkv), (r.out, eager_r.out, base.z), (to_of(d, 0), to_of(eager_d, 0), base.win),
                           (to_of(d, 1), to_of(eager_d, 1), base.state)):
            assert np.array_equal(bits(host(a, like)), bits(host(b, like))), f"replay {i}"


def to_of(conv, i):
    return conv.states._bufs[i]


def test_two_streams_at_once():
    hip = hip_of_bench()
    cases = [M.Case(33, 2, 4, 64, 4, [90, 1, 70]), M.Case(34, 1, 3, 128, 4, [1] * 20 + [65])]
    streams, work, want = [hip.stream(), hip.stream()], [], []
    for c in cases:
        c.to = np.full(len(c.rows), -1, np.int32)
        r = Rule(c, 0)
        r.run()
        want.append(r.results()[0])
        work.append(r)
    hip.sync()
    for _ in range(5):
        for s, r in zip(streams, work):
            r.run(s)
    hip.sync()
    for r, w in zip(work, want):
        assert np.array_equal(bits(r.results()[0]), bits(w))
