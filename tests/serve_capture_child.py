"""Child process for tests/test_gpu_serve.py: the first calls of batched serving
in a fresh process, captured into a HIP graph (the kernels' LDS limits are
raised while the stream is being captured), replayed twice and compared bit
for bit with eager calls.

    python tests/serve_capture_child.py   (exit 0 when all replays match)
"""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "unltd-inference_amd"), os.path.join(ROOT, "tests")]

import numpy as np  # noqa: E402

import bench  # noqa: E402
import serve_model as M  # noqa: E402
import uq  # noqa: E402
from uq import serve  # noqa: E402


def main():
    hip = bench.Hip()
    s = hip.stream()
    rng = np.random.default_rng(1)
    heads, kv, hd, vocab = 8, 2, 256, 5000
    calls, outs = [], []
    # one token each over a short table; over a long one; a prompt's chunk (the kernel of many queries); an f32 cache
    for dtype, rows, lens, room in (("f16", [1, 1], [30, 90], 0), ("f16", [1, 2], [500, 90], 1 << 16),
                                    ("f16", [60], [300], 1 << 16), ("f32", [30], [200], 1 << 16)):
        c = M.Cache(rng, dtype, kv, hd, 16, rows, lens, room=room)
        pages, batch = c.upload()
        q, k, v = (uq.DeviceArray.from_numpy(rng.standard_normal((c.n_rows, w, hd)).astype(np.float32)) for w in (heads, kv, kv))
        qo, out = (uq.DeviceArray(4 * c.n_rows * heads * hd) for _ in range(2))
        hr = serve.HeadRows(heads, q, heads * hd, hd, qo, k, kv * hd, v, kv * hd, rope="imrope", n_rot=64, theta_scale=0.6)
        ws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, heads))

        def call(stream, pages=pages, batch=batch, hr=hr, qo=qo, out=out, ws=ws):
            serve.kv_append_d(pages, batch, hr, stream)
            serve.attn_paged_d(out, qo, pages, batch, heads, 0.06, ws, stream=stream)

        calls.append(call)
        outs.append(out)
    p = rng.random((5, vocab)).astype(np.float32)
    dp = uq.DeviceArray.from_numpy(p)
    tok, u, start = (uq.DeviceArray.from_numpy(a) for a in (np.arange(5, dtype=np.int32), rng.random(5).astype(np.float32) * 0.1,
                                                           np.array([0, 3, 5], np.int32)))
    b = serve.SeqBatch(2, 5, start)
    acc, nxt, vws = uq.DeviceArray(8), uq.DeviceArray(8), uq.DeviceArray(serve.draft_verify_ws_bytes(b, vocab))
    calls.append(lambda stream: serve.draft_verify_d(acc, nxt, dp, None, tok, u, b, vocab, vws, stream=stream))
    outs += [acc, nxt]
    hip.sync()
    print("inputs staged; capturing the first calls", file=sys.stderr, flush=True)
    g = hip.capture(s, lambda: [call(s) for call in calls])
    replays = []
    for _ in range(2):
        for d in outs:
            d.upload(np.full(d.nbytes, 0xFF, np.uint8))
        hip.launch_graph(g, s)
        hip.sync()
        replays.append([d.download(np.int32) for d in outs])
    for call in calls:
        call(None)
    hip.sync()
    eager = [d.download(np.int32) for d in outs]
    ok = all(np.array_equal(a, b) for r in replays for a, b in zip(r, eager))
    print("replays equal eager calls:", ok, flush=True)
    return 0 if ok else 1


if __name__ == "__main__":
    sys.exit(main())
