"""Child process for tests/test_gpu_gdn_layer.py: the first calls of the
recurrent layers' operators in a fresh process, captured into two HIP graphs
that share their workspaces (the kernels' LDS limits are raised while the
stream is being captured), replayed in turns and compared bit for bit with
eager calls.

    python tests/gdn_capture_child.py   (exit 0 when all replays match)
"""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "unltd-inference_amd"), os.path.join(ROOT, "tests")]

import numpy as np  # noqa: E402

import bench  # noqa: E402
import gdn_model as M  # noqa: E402
import uq  # noqa: E402
from test_gpu_gdn_serve import Conv, Rule, bits, host  # noqa: E402
from uq import serve  # noqa: E402


def main():
    hip = bench.Hip()
    s = hip.stream()
    cases = [M.Case(50 + hd, 2, 4, hd, 4, rows, frm=[0, 1, 2], to=[3, 3, 3]) for hd, rows in ((128, [100, 1, 40]), (64, [70, 3, 90]))]
    runs = [(Conv(c), Rule(c, 0)) for c in cases]
    ws = uq.DeviceArray(max(r.ws.nbytes for _, r in runs))
    vocab = 5000
    x = uq.DeviceArray.from_numpy(np.random.default_rng(1).standard_normal((6, vocab)).astype(np.float32))
    lp, ids = uq.DeviceArray(4 * 6 * 4), uq.DeviceArray(4 * 6 * 4)
    lws = uq.DeviceArray(serve.logprobs_ws_bytes(6, vocab, 4))
    for _, r in runs:
        r.ws = ws
        r.c.d_to.upload(np.full(3, -1, np.int32))  # the states stay for every replay

    def call(i, stream):
        runs[i][0].run(stream)
        runs[i][1].run(stream)
        serve.logprobs_d(serve.LogProbs(None, None, None, ids, lp, 4), x, None, 6, vocab, lws, 1.0, 0, stream)

    like = [np.empty((c.n_rows, c.nv, c.hd), np.float32) for c in cases]
    hip.sync()
    print("inputs staged; capturing the first calls", file=sys.stderr, flush=True)
    graphs = [hip.capture(s, lambda i=i: call(i, s)) for i in range(2)]
    got = []
    for i in (0, 1, 0, 1, 1, 0):
        runs[i][1].out.upload(np.full(like[i].shape, 7, np.float32))
        lp.upload(np.zeros(24, np.float32))
        hip.launch_graph(graphs[i], s)
        hip.sync()
        got.append((i, host(runs[i][1].out, like[i]), host(lp, np.empty(24, np.float32))))
    for i, out, p in got:
        call(i, None)
        assert np.array_equal(bits(out), bits(host(runs[i][1].out, like[i]))), i
        assert np.array_equal(bits(p), bits(host(lp, np.empty(24, np.float32)))), i
    print("replays match", file=sys.stderr, flush=True)


if __name__ == "__main__":
    main()
