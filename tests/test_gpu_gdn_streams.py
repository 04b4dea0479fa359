"""GPU tests of the GatedDeltaNet layers' batched operators (include/uq_serve.h)
on two streams at once, with everything that a call writes cleared before."""
import numpy as np
import pytest

import gdn_model as M
from test_gpu_gdn_serve import MARK, Conv, Rule, bits, hip_of_bench, host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("most", [0, 1])
def test_calls_of_two_streams_leave_what_each_alone_leaves(most):
    """Results, gates, windows and states, for many rows (most 0) and row by row (1); then the buffers hold MARK, and each
    stream's only call under way fills them again."""
    hip = hip_of_bench()
    streams = [hip.stream(), hip.stream()]
    cases = [M.Case(161, 2, 4, 128, 4, [200, 1, 70], frm=[0, 1, -1], to=[3, 4, 5], spare=3),
             M.Case(162, 2, 6, 64, 4, [90, 5, 130], frm=[-1, 1, 2], to=[3, 4, 5], spare=3)]
    runs = [(Conv(c), Rule(c, most)) for c in cases]

    def written(conv, rule):
        """(buffer, values to begin with)"""
        c = conv.c
        state, win = c.state.copy(), c.win.copy()
        state[3:], win[3:] = MARK, MARK
        return [(conv.out, np.full(c.qkv.shape, MARK, np.float32)), (conv.beta, np.full(c.beta.shape, MARK, np.float32)),
                (conv.gate, np.full(c.gate.shape, MARK, np.float32)), (conv.states._bufs[0], win),
                (rule.out, np.full(c.z.shape, MARK, np.float32)), (rule.states._bufs[1], state)]

    def clear():
        for r in runs:
            for d, a in written(*r):
                d.upload(a)
        hip.sync()

    clear()
    for conv, rule in runs:
        conv.run()
        rule.run()
    hip.sync()
    want = [[host(d, a) for d, a in written(*r)] for r in runs]
    for w, r in zip(want, runs):
        assert all(not np.array_equal(x, a) for x, (_, a) in zip(w, written(*r)))
    for turn in range(3):
        clear()
        for s, (conv, rule) in zip(streams, runs):
            conv.run(s)
            rule.run(s)
        hip.sync()
        for w, r in zip(want, runs):
            assert all(np.array_equal(bits(host(d, a)), bits(x)) for x, (d, a) in zip(w, written(*r))), turn
