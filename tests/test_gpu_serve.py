"""GPU tests of batched serving (include/uq_serve.h) against 64-bit models
(serve_model.py) and, where f32 bits are promised, against the oracle's norm
and rotations: types, head shapes, page sizes, lengths, padded batches, pages
that are none, values that are not finite where a row may not see them, other
streams, graphs, and the operators in a row."""
import os
import subprocess
import sys

import numpy as np
import pytest

import oracle as O
import serve_model as M
import uq
from uq import layer as L
from uq import ops, serve
from test_gpu_layers import SMALL, Model, nodes_of

pytestmark = pytest.mark.gpu


def host(d, like):
    uq.synchronize()
    return d.download(like.dtype, like.size).reshape(like.shape)


def dev(a):
    return uq.DeviceArray.from_numpy(a)


def rotated(kind, x, n_rot, freqs, theta, pos):
    if kind == "none" or n_rot == 0:
        return x
    if kind == "imrope":
        return O.rope_imrope(x, n_rot, theta, pos)
    y = x.copy()
    if kind == "llama":
        y[:n_rot] = O.rope_llama(x[:n_rot], freqs, pos)
    else:
        y[:n_rot] = O.rope_neox(x[:n_rot], freqs, pos)
    return y


def ulps(a, b):
    a, b = (np.ascontiguousarray(x, np.float32).view(np.int32).astype(np.int64) for x in (a, b))
    a, b = (np.where(x < 0, -(x & 0x7FFFFFFF), x) for x in (a, b))
    return int(np.abs(a - b).max()) if a.size else 0


# ------------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype,heads,kv,hd,page,rows,lens,rope,n_rot,norm,pad", [
    ("f16", 16, 4, 256, 64, [1], [2999], "imrope", 64, True, 0),
    ("f32", 16, 4, 256, 16, [3, 0, 5, 1], [3, 9, 700, 1], "imrope", 64, True, 2),
    ("f16", 6, 2, 128, 1, [4, 2], [17, 2], "neox", 128, True, 1),
    ("f32", 8, 8, 64, 4096, [2] * 70, list(range(2, 72)), "llama", 32, True, 0),
    ("f16", 3, 1, 512, 8, [9, 1], [4000, 40], "neox", 510, True, 0),
    ("f16", 5, 5, 64, 32, [33], [33], "none", 0, False, 3),
    ("f32", 4, 2, 128, 32, [300], [1000], "llama", 128, False, 0)])
def test_append_rows_are_the_norm_and_the_rotation(dtype, heads, kv, hd, page, rows, lens, rope, n_rot, norm, pad):
    rng = np.random.default_rng(hd + len(rows))
    c = M.Cache(rng, dtype, kv, hd, page, rows, lens, pad=pad)
    n, eps, theta = c.n_rows, 1e-6, 1e7 ** (-2.0 / max(n_rot, 1))
    freqs = (1e4 ** (-np.arange(max(1, n_rot // 2)) / max(1, n_rot // 2))).astype(np.float32)
    qh, qr = 2 * hd + 3, heads * (2 * hd + 3) + 5  # rows start at any float
    kr, vr = kv * hd + 7, kv * hd + 1
    qf, kf, vf = (rng.standard_normal((n, w)).astype(np.float32) for w in (qr, kr, vr))
    wq, wk = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    out0 = np.full((n, heads, hd), 7.0, np.float32)
    d_out, bufs = dev(out0), [dev(a) for a in (qf, kf, vf, wq, wk, freqs)]
    pages, batch = c.upload()
    hr = serve.HeadRows(heads, bufs[0], qr, qh, d_out, bufs[1], kr, bufs[2], vr, bufs[3] if norm else None,
                        bufs[4] if norm else None, eps, rope, n_rot, bufs[5], theta)
    serve.kv_append_d(pages, batch, hr)
    got, gk, gv = host(d_out, out0), host(c.d_k, c.k), host(c.d_v, c.v)
    want, wantk, wantv = out0.copy(), c.k.copy(), c.v.copy()
    for r, (b, pos) in enumerate(c.row_positions()):
        def prep(x, w):
            return rotated(rope, O.rmsnorm(x, w, eps) if norm else x, n_rot, freqs[:n_rot // 2], theta, pos)

        for h in range(heads):
            want[r, h] = prep(qf[r, h * qh:h * qh + hd], wq)
        pg, sl, ok = c.slots(b, pos + 1)
        assert ok[-1]
        for j in range(kv):
            wantk[pg[-1], j, sl[-1]] = prep(kf[r, j * hd:(j + 1) * hd], wk).astype(wantk.dtype)
            wantv[pg[-1], j, sl[-1]] = vf[r, j * hd:(j + 1) * hd].astype(wantv.dtype)
    # bit for bit but for the rotation's f64 sine and cosine (1 ulp where another libm's last bit turns the rounding)
    assert ulps(got, want) <= (1 if rope != "none" else 0)
    assert np.array_equal(gv.view(np.uint8), wantv.view(np.uint8)), "values are copied or rounded to nearest"
    if dtype == "f32":
        assert ulps(gk, wantk) <= (1 if rope != "none" else 0)
    else:  # an ulp of f32 moves a value to the next f16 at most
        assert np.max(np.abs(gk.astype(np.float64) - wantk) - 2.0 ** -10 * np.abs(wantk.astype(np.float64))) <= 2.0 ** -24
        assert np.mean(gk != wantk) < 1e-3
    for d in bufs + [d_out]:
        d.free()


def test_append_against_64_bits():
    """The formula in f64: a normed and rotated value is off by the f32 roundings of its scale (5: the mean, eps,
    the root, the quotient, the f64 sum's), its two products and the rotation's result."""
    rng = np.random.default_rng(5)
    heads, kv, hd, n_rot = 4, 2, 256, 256
    c = M.Cache(rng, "f32", kv, hd, 16, [6], [100000])
    q, k, v = (rng.standard_normal((6, m, hd)).astype(np.float32) for m in (heads, kv, kv))
    w = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)
    freqs = (1e4 ** (-np.arange(128) / 128)).astype(np.float32)
    d_out, bufs = dev(np.zeros_like(q)), [dev(a) for a in (q, k, v, w, freqs)]
    pages, batch = c.upload()
    serve.kv_append_d(pages, batch, serve.HeadRows(heads, bufs[0], heads * hd, hd, d_out, bufs[1], kv * hd, bufs[2], kv * hd,
                                                   bufs[3], bufs[3], 1e-6, "neox", n_rot, bufs[4]))
    got, gk = host(d_out, q), host(c.d_k, c.k)
    for r in range(6):
        pos = 100000 - 6 + r
        pg, sl, _ = c.slots(0, pos + 1)
        for x, y in [(q[r], got[r]), (k[r], gk[pg[-1], :, sl[-1]])]:
            x = x.astype(np.float64)
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w
            ang = pos * freqs.astype(np.float64)
            a, b = x[:, :128], x[:, 128:]
            want = np.concatenate([a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)], -1)
            size = np.concatenate([np.hypot(a, b)] * 2, -1)
            assert np.all(np.abs(y - want) <= 9 * 2.0 ** -24 * size)


def test_append_leaves_out_what_has_no_slot():
    """Pages that are none, positions beyond the table, negative positions and lengths, rows of no sequence: their
    keys and values go nowhere; queries are made for every row at a position."""
    rng = np.random.default_rng(6)
    heads, kv, hd, page = 2, 1, 64, 4
    c = M.Cache(rng, "f16", kv, hd, page, [3, 2, 2, 1, 2], [8, 4, 1, -5, 30], pad=1)
    assert c.max_pages == 8
    c.table[0, 1] = c.n_pages  # positions 4 .. 7 of sequence 0: three rows without a page
    c.table[4, 7] = -7  # positions 28, 29
    c.lens[1] = 33  # position 32 lies beyond the table
    c.table[1, 7] = c.table[1, 0]  # position 31 has a page
    q, k, v = (rng.standard_normal((c.n_rows, m, hd)).astype(np.float32) for m in (heads, kv, kv))
    out0 = np.full_like(q, 7.0)
    d_out, bufs = dev(out0), [dev(a) for a in (q, k, v)]
    pages, batch = c.upload()
    serve.kv_append_d(pages, batch, serve.HeadRows(heads, bufs[0], heads * hd, hd, d_out, bufs[1], kv * hd, bufs[2], kv * hd))
    got, gk, gv = host(d_out, q), host(c.d_k, c.k), host(c.d_v, c.v)
    want, wk, wv = out0.copy(), c.k.copy(), c.v.copy()
    want[[0, 1, 2, 3, 4, 6, 8, 9]] = q[[0, 1, 2, 3, 4, 6, 8, 9]]  # row 5: position -1; row 7: length -5; row 10: none
    wk[c.table[1, 7], :, 3], wv[c.table[1, 7], :, 3] = k[3], v[3]
    wk[c.table[2, 0], :, 0], wv[c.table[2, 0], :, 0] = k[6], v[6]
    for a, b in ((got, want), (gk, wk), (gv, wv)):
        assert np.array_equal(a, b)


def test_append_in_place_and_queries_or_keys_alone():
    rng = np.random.default_rng(7)
    heads, kv, hd = 3, 3, 64
    c = M.Cache(rng, "f32", kv, hd, 8, [5], [21])
    q, k, v = (rng.standard_normal((5, heads, hd)).astype(np.float32) for _ in range(3))
    w = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float32)
    pages, batch = c.upload()
    dq, dk, dv, dw = (dev(a) for a in (q, k, v, w))
    both = dev(np.zeros_like(q))
    args = dict(d_q_norm=dw, d_k_norm=dw, rope="imrope", n_rot=32, theta_scale=0.7)
    serve.kv_append_d(pages, batch, serve.HeadRows(heads, dq, heads * hd, hd, both, dk, kv * hd, dv, kv * hd, **args))
    want, wk, wv = host(both, q), host(c.d_k, c.k), host(c.d_v, c.v)
    pages2, batch2 = c.upload()
    serve.kv_append_d(pages2, batch2, serve.HeadRows(heads, d_k=dk, k_row=kv * hd, d_v=dv, v_row=kv * hd, **args))
    assert np.array_equal(host(c.d_k, c.k), wk) and np.array_equal(host(c.d_v, c.v), wv)
    serve.kv_append_d(pages2, batch2, serve.HeadRows(heads, dq, heads * hd, hd, dq, **args))
    assert np.array_equal(host(dq, q), want)
    assert not np.array_equal(want, q)


# ------------------------------------------------------------------------- attention

def attend(c, q, heads, scale, shared=0, gate=None, stream=None, out=None):
    pages, batch = c.upload()
    d_q = dev(q)
    out0 = np.full(q.shape, 7.0, np.float32) if out is None else out
    d_out = dev(out0)
    ws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, heads, shared))
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))  # what a workspace held before does not matter
    extra = {}
    if gate is not None:
        wide = np.zeros((c.n_rows, heads, 2 * c.hd), np.float32)
        wide[:, :, c.hd:] = gate
        d_g = dev(wide)
        view = type("View", (), {})()
        view.ptr = d_g.ptr.value + 4 * c.hd
        extra = dict(d_gate=view, gate_row=2 * heads * c.hd, gate_head=2 * c.hd)
    serve.attn_paged_d(d_out, d_q, pages, batch, heads, scale, ws, shared_len=shared, stream=stream, **extra)
    got = host(d_out, out0)
    serve.attn_paged_d(d_out, d_q, pages, batch, heads, scale, ws, shared_len=shared, stream=stream, **extra)
    again = host(d_out, out0)
    assert int(np.sum(got.view(np.int32) != again.view(np.int32))) == 0, "a call repeated gives the same bits"
    for d in (d_q, d_out, ws):
        d.free()
    return got


def check(c, q, heads, scale, shared=0, gate=None, what=""):
    got = attend(c, q, heads, scale, shared, gate)
    want, bound = M.attention(c, q, heads, scale, gate)
    n = int(c.start[-1])
    assert np.all(got[n:] == 7.0), "rows behind the last sequence are left as they were"
    err = np.abs(got[:n] - want[:n])
    bad = ~(err <= bound[:n])
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} outside, rows {sorted(set(np.nonzero(bad)[0]))[:8]}, "
                           f"worst {np.nanmax(err):.3g} of {np.nanmax(np.abs(want[:n])):.3g}")
    scale_ = np.abs(want[:n]).max()
    print(f"{what}: worst {err.max() / scale_ if scale_ else 0:.3g} of the largest, bound {bound[:n].max() / scale_ if scale_ else 0:.3g}",
          flush=True)


# Positions of the page tables: no more than the batch needs (short ones: a workgroup takes a block by itself), and many
# (blocks are divided, and joined; more than 32 queries of a KV head are another kernel's).
ROOM = [0, 1 << 16]

SHAPES = [
    # heads, kv, hd, page, rows, lens, shared, pad
    (16, 4, 256, 64, [1], [700], 0, 0),
    (16, 4, 256, 64, [1], [1], 0, 2),
    (4, 4, 64, 16, [1] * 9, [1, 2, 15, 16, 17, 127, 128, 129, 1000], 0, 1),
    (12, 2, 128, 32, [4, 1, 0, 3, 5], [4, 33, 50, 600, 65], 0, 0),
    (8, 1, 512, 16, [1, 3], [200, 77], 0, 0),
    (24, 1, 64, 8, [1, 2], [130, 259], 0, 0),  # 24 queries of a KV head: blocks of one row's heads
    (6, 2, 256, 1, [2, 1], [70, 5], 0, 0),  # a page a position
    (4, 2, 128, 4096, [40], [1333], 0, 0),  # a chunk of a prompt
    (3, 1, 64, 16, [97], [97], 0, 3),  # a whole prompt
    (16, 4, 256, 64, [1] * 6, [1030, 1100, 1025, 1500, 1024, 1300], 1024, 0),
    (12, 2, 128, 32, [4, 2, 1, 3], [333, 350, 334, 400], 331, 1),  # the shared part ends inside a page
    (4, 2, 64, 16, [3, 5, 2], [50, 51, 64], 49, 0),  # rows at positions inside the shared part
    (8, 2, 64, 16, [20, 1], [200, 140], 128, 0),
    # blocks of 64 and 128 queries of a KV head (f16): chunks, whole prompts, the batch over shared positions
    (16, 4, 256, 64, [33], [700], 0, 1),
    (12, 4, 256, 16, [50, 0, 7, 90], [300, 20, 1000, 90], 0, 2),
    (8, 2, 128, 32, [129, 40], [129, 777], 0, 0),
    (4, 4, 64, 16, [200, 130], [260, 131], 0, 0),
    (6, 2, 64, 8, [70], [333], 0, 0),
    (16, 4, 256, 64, [1] * 30, list(range(1000, 1030)), 1000, 0),
    (4, 2, 128, 16, [20] * 7, [620, 610, 650, 600, 608, 601, 640], 599, 3),
    (8, 1, 64, 1, [3] * 11, [140 + 9 * i for i in range(11)], 130, 0),
    (5, 1, 256, 32, [40, 20], [35, 64], 0, 0),  # more rows than positions
    (16, 4, 256, 64, [1] * 20 + [70], [60 + 7 * i for i in range(21)], 50, 0),  # shared and own on different kernels
    # blocks of 32 queries: 17 to 32 of a KV head, more where the cache is f32
    (20, 1, 128, 32, [1] * 3, [50, 200, 333], 0, 0),
    (24, 1, 256, 16, [1, 1], [40, 700], 0, 1),
    (32, 1, 64, 8, [1, 0, 1], [1, 5, 64], 0, 0),
    (8, 1, 128, 16, [3] * 4, [64, 90, 61, 150], 60, 0),
    (16, 8, 64, 16, [1] * 100, [2601 + i % 7 for i in range(100)], 2600, 2),  # f32: shared on 32, own on 16
    # shared positions enough for the blocks of many queries
    (16, 4, 256, 64, [1] * 25, [9300 + i % 3 for i in range(25)], 9290, 0),
    (32, 2, 128, 16, [3] * 10, [3910 + 7 * i for i in range(10)], 3900, 1)]


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention_against_64_bits(dtype, case, room):
    heads, kv, hd, page, rows, lens, shared, pad = SHAPES[case]
    rng = np.random.default_rng(100 + case)
    c = M.Cache(rng, dtype, kv, hd, page, rows, lens, pad=pad, shared=shared, room=room)
    q = (2 * rng.standard_normal((c.n_rows, heads, hd))).astype(np.float32)
    gate = rng.standard_normal(q.shape).astype(np.float32) if case % 2 else None
    check(c, q, heads, 1 / np.sqrt(hd), shared, gate, f"{dtype} {SHAPES[case]}")


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype,seqs", [("f16", 300), ("f32", 600)])
def test_attention_of_many_sequences(dtype, seqs, room):
    """More sequences than a workgroup's threads, some without rows or positions."""
    rng = np.random.default_rng(seqs)
    rows = rng.integers(0, 3, seqs)
    lens = np.where(rng.random(seqs) < 0.1, rows, rows + rng.integers(0, 60, seqs))
    c = M.Cache(rng, dtype, 1, 64, 16, rows, lens, pad=1, room=room)
    q = rng.standard_normal((c.n_rows, 2, 64)).astype(np.float32)
    check(c, q, 2, 0.125, what=f"{dtype} {seqs} sequences")


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("shared", [0, 24])
def test_attention_passes_over_what_no_row_sees(dtype, shared, room):
    """Slots behind the lengths, unused pages, later rows' positions and pages that are none hold NaN, infinities
    and the type's lowest value: the results are those without them. A row without any position is zero."""
    rng = np.random.default_rng(21)
    rows, lens = [6, 3, 4, 2, 3], [70, 33, 2, 41, 60]
    if shared:
        lens[2] = 26
    c = M.Cache(rng, dtype, 2, 128, 8, rows, lens, shared=shared, room=room)
    lens = c.lens
    q = rng.standard_normal((c.n_rows, 4, 128)).astype(np.float32)
    used = np.zeros(c.k.shape[:3], bool)
    for b, n in enumerate(lens):
        pg, sl, ok = c.slots(b, n)
        used[pg, :, sl] = True
    for a in (c.k, c.v):
        hole = a[~used]
        hole[:] = np.array([np.nan, np.inf, -np.inf, np.finfo(a.dtype).min], a.dtype)[np.arange(hole.size).reshape(hole.shape) % 4]
        a[~used] = hole
    c.table[3, 3 if shared else 1] = c.n_pages + 3  # positions 24 .. 31 (8 .. 15) of sequence 3 are nowhere
    c.table[4, 3:] = -1
    if not shared:
        c.table[4, :] = -1  # nothing is left of sequence 4
    want, bound = M.attention(c, q, 4, 0.1)
    # only the last row of each sequence sees its last position
    for b, n in enumerate(lens):
        pg, sl, ok = c.slots(b, n)
        if ok[-1] and n - 1 >= shared:
            c.k[pg[-1], 0, sl[-1]], c.v[pg[-1], 0, sl[-1]] = np.nan, np.inf
            c.k[pg[-1], 1, sl[-1], 3], c.v[pg[-1], 1, sl[-1], ::2] = -np.inf, np.nan
    got = attend(c, q, 4, 0.1, shared)
    last = c.start[1:] - 1
    free = np.setdiff1d(np.arange(c.n_rows), last)
    assert np.all(np.abs(got[free] - want[free]) <= bound[free])
    if not shared:
        assert np.all(got[free[-2:]] == 0.0) and np.all(got[last[-1]] == 0.0), "no position left"
        assert np.all(got[9:11] == 0.0), "negative positions"
    for b in (0, 1):
        assert not np.isfinite(got[last[b]]).all(), "a row that sees them shows it"


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_with_a_value_not_finite_that_some_rows_see(dtype, room):
    """Position 40 of 45 holds values of NaN, infinity and numbers: rows before it are untouched, rows from it on
    are not finite in those columns alone."""
    rng = np.random.default_rng(22)
    c = M.Cache(rng, dtype, 1, 64, 16, [9], [45], room=room)
    q = rng.standard_normal((9, 2, 64)).astype(np.float32)
    clean, bound = M.attention(c, q, 2, 0.125)
    pg, sl, _ = c.slots(0, 45)
    c.v[pg[40], 0, sl[40], 5] = np.nan
    c.v[pg[40], 0, sl[40], 9] = np.inf
    got = attend(c, q, 2, 0.125)
    assert np.all(np.abs(got[:4] - clean[:4]) <= bound[:4])
    cols = np.ones(64, bool)
    cols[[5, 9]] = False
    assert np.all(np.abs(got[4:, :, cols] - clean[4:, :, cols]) <= bound[4:, :, cols])
    assert np.isnan(got[4:, :, 5]).all() and not np.isfinite(got[4:, :, 9]).any()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,lens", [([1, 1], [1, 33]), ([50, 1], [50, 129])])
def test_attention_keeps_a_nan_that_is_all_a_tile_shows(dtype, rows, lens, room):
    """The only position that a row sees, or the only one in the last tile that it sees, has a key of NaN."""
    rng = np.random.default_rng(28)
    c = M.Cache(rng, dtype, 1, 64, 16, rows, lens, room=room)
    for b, pos in ((0, 0), (1, lens[1] - 1)):
        pg, sl, _ = c.slots(b, pos + 1)
        c.k[pg[-1], :, sl[-1]] = np.nan
    got = attend(c, rng.standard_normal((sum(rows), 2, 64)).astype(np.float32), 2, 0.125)
    assert np.isnan(got).all()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_of_large_and_small_numbers(dtype, room):
    """Scores of thousands (one weight is all), queries of 1e-30 and 1e30, keys of zero, the largest f16."""
    rng = np.random.default_rng(23)
    c = M.Cache(rng, dtype, 2, 64, 16, [1, 1, 1, 1], [100, 200, 300, 50], room=room)
    q = rng.standard_normal((4, 4, 64)).astype(np.float32)
    q[0] *= 1000
    q[1] *= 1e-30
    q[2] = 0
    pg, sl, _ = c.slots(3, 50)
    c.k[pg, :, sl] = 0
    c.v[pg, :, sl] = 65504
    q[3] *= 1e30
    got = attend(c, q, 4, 0.125)
    want, bound = M.attention(c, q, 4, 0.125)
    # a score of thousands is off by more than the weights bear: the least bound is that of values' size
    assert np.all(np.abs(got[1:] - want[1:]) <= bound[1:])
    one = np.abs(got[0] - want[0]) <= np.maximum(bound[0], 1e-4)
    assert one.all()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-30])
def test_attention_with_any_scale(dtype, scale, room):
    """Turned round, the mean of the values, nearly the mean: blocks of few and of many queries."""
    rng = np.random.default_rng(29)
    c = M.Cache(rng, dtype, 2, 64, 16, [1, 30], [90, 200], room=room)
    check(c, rng.standard_normal((31, 6, 64)).astype(np.float32), 6, scale, what=f"{dtype} scale {scale}")


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_of_many_queries_large_and_not_finite(dtype, room):
    """Queries of 1e30, 1e-30 and 0 among others, and of NaN and infinity, whose own results show it and no others."""
    rng = np.random.default_rng(30)
    c = M.Cache(rng, dtype, 1, 128, 16, [40], [300], room=room)
    q = rng.standard_normal((40, 4, 128)).astype(np.float32)
    clean = q.copy()
    q[3] *= 1e-30
    q[4] = 0
    q[5, 1] *= 1e5
    bad = [(7, 0), (8, 3), (39, 2)]
    for (r, h), x in zip(bad, (np.nan, np.inf, -np.inf)):
        q[r, h, 11] = x
    got = attend(c, q, 4, 0.1)
    clean[[3, 4, 5]] = q[[3, 4, 5]]
    want, bound = M.attention(c, clean, 4, 0.1)
    good = np.ones((40, 4), bool)
    for r, h in bad:
        good[r, h] = False
        assert not np.isfinite(got[r, h]).any()
    bound[5, 1] = np.maximum(bound[5, 1], 1e-3)  # scores of 1e5: which weight is all may turn on their last bits
    good[5, 1] = False
    assert np.all(np.abs(got - want)[good] <= bound[good])
    assert np.isfinite(got[5, 1]).all()


@pytest.mark.parametrize("rows", [[1, 2], [40, 30]])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_without_pages_or_rows(dtype, rows):
    """A cache of no pages, a table of none: zeros. A batch whose rows are all none: nothing is written."""
    n = sum(rows)
    q = dev(np.ones((n, 4, 64), np.float32))
    start, zero = dev(np.array([0, rows[0], n], np.int32)), dev(np.zeros(3, np.int32))
    lens, table = dev(np.array([100, 70], np.int32)), dev(np.arange(14, dtype=np.int32))
    some = dev(np.ones((14, 2, 16, 64), M.DTYPE[dtype][1]))
    like = np.empty((n, 4, 64), np.float32)
    for shared in (0, 33):
        for kv, batch, want in [
                (serve.KvPages(None, None, M.DTYPE[dtype][0], 0, 16, 2, 64), serve.SeqBatch(2, n, start, lens, table, 7), 0.0),
                (serve.KvPages(some, some, M.DTYPE[dtype][0], 14, 16, 2, 64), serve.SeqBatch(2, n, zero, lens, table, 7), 7.0),
                (serve.KvPages(some, some, M.DTYPE[dtype][0], 14, 16, 2, 64), serve.SeqBatch(2, n, start, lens), 0.0)]:
            if shared and not batch.max_pages:
                continue
            out = dev(np.full(like.shape, 7.0, np.float32))
            ws = uq.DeviceArray(serve.attn_paged_ws_bytes(kv, batch, 4, shared))
            serve.attn_paged_d(out, q, kv, batch, 4, 0.125, ws, shared_len=shared)
            assert np.all(host(out, like) == want)


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_in_a_pool_beyond_32_bits(dtype, room):
    """Pages whose values lie 2^32 and more bytes and elements into the arrays, appended to and read, by few queries
    and by many (a page number of them would be another page's in 32 bits)."""
    hd, page, heads = 128, 16, 4
    elem = 2 if dtype == "f16" else 4
    per = page * hd  # elements of a page (one KV head)
    n_pages = (1 << 32) // per + 64
    rows, lens = [40, 1], [200, 150]
    rng = np.random.default_rng(31)
    c = M.Cache(rng, dtype, 1, hd, page, rows, lens, spare=0, room=room)
    high = n_pages - 1 - np.arange(c.n_pages)  # page x of the small cache is this page of the large one
    d_k, d_v = uq.DeviceArray(n_pages * per * elem), uq.DeviceArray(n_pages * per * elem)

    lo = int(high[-1]) * per * elem
    for d, a in ((d_k, c.k), (d_v, c.v)):
        buf = np.ascontiguousarray(a[::-1])
        uq._check(uq.lib().uq_memcpy_htod(d.ptr.value + lo, buf.ctypes.data, buf.nbytes, None))
        uq.synchronize()
    pages = serve.KvPages(d_k, d_v, M.DTYPE[dtype][0], n_pages, page, 1, hd)
    table = np.where(c.table >= 0, high[c.table], -1).astype(np.int32)
    batch = serve.SeqBatch(2, 41, dev(c.start), dev(np.array(lens, np.int32)), dev(table), c.max_pages)
    q, k, v = (rng.standard_normal((41, w, hd)).astype(np.float32) for w in (heads, 1, 1))
    dq, dk, dv = dev(q), dev(k), dev(v)
    out = dev(np.zeros_like(q))
    serve.kv_append_d(pages, batch, serve.HeadRows(d_k=dk, k_row=hd, d_v=dv, v_row=hd))
    for r, (b, pos) in enumerate(c.row_positions()):
        pg, sl, _ = c.slots(b, pos + 1)
        c.k[pg[-1], :, sl[-1]], c.v[pg[-1], :, sl[-1]] = k[r], v[r]
    ws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, heads))
    serve.attn_paged_d(out, dq, pages, batch, heads, 0.1, ws)
    want, bound = M.attention(c, q, heads, 0.1)
    assert np.all(np.abs(host(out, q) - want) <= bound)
    for d in (d_k, d_v):
        d.free()


@pytest.mark.parametrize("room", ROOM)
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,lens,shared", [([3, 1], [70, 90], 48), ([50, 40], [90, 140], 40), ([70], [150], 0)])
def test_attention_in_place_from_any_float(dtype, rows, lens, shared, room):
    """d_out = d_q, four bytes off any alignment."""
    rng = np.random.default_rng(32)
    c = M.Cache(rng, dtype, 2, 64, 16, rows, lens, shared=shared, room=room)
    q = rng.standard_normal((c.n_rows, 4, 64)).astype(np.float32)
    want = attend(c, q, 4, 0.125, shared)
    pages, batch = c.upload()
    buf = dev(np.concatenate([[5.0], q.ravel(), [6.0]]).astype(np.float32))
    view = type("View", (), {})()
    view.ptr = buf.ptr.value + 4
    ws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, 4, shared))
    serve.attn_paged_d(view, view, pages, batch, 4, 0.125, ws, shared_len=shared)
    got = host(buf, np.empty(q.size + 2, np.float32))
    assert got[0] == 5.0 and got[-1] == 6.0
    assert np.array_equal(got[1:-1].view(np.int32), want.ravel().view(np.int32))


def test_two_calls_at_once():
    """Two batches on two streams, each with its workspace, again and again: each call's bits are those it has alone."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(__file__))))
    import bench
    hip = bench.Hip()
    streams = [hip.stream(), hip.stream()]
    rng = np.random.default_rng(33)
    work = []
    for dtype, heads, kv, hd, rows, lens, shared in [("f16", 8, 2, 128, [1] * 5 + [60], [2000, 30, 500, 77, 900, 400], 0),
                                                     ("f16", 16, 4, 256, [2] * 20, list(range(700, 720)), 690)]:
        c = M.Cache(rng, dtype, kv, hd, 16, rows, lens, shared=shared)
        q = rng.standard_normal((c.n_rows, heads, hd)).astype(np.float32)
        want = attend(c, q, heads, 0.1, shared)
        pages, batch = c.upload()
        ws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, heads, shared))
        outs = [dev(np.zeros_like(q)) for _ in range(10)]
        work.append((pages, batch, dev(q), outs, ws, heads, shared, want, c))
    hip.sync()
    for i in range(10):
        for s, (pages, batch, dq, outs, ws, heads, shared, want, c) in zip(streams, work):
            serve.attn_paged_d(outs[i], dq, pages, batch, heads, 0.1, ws, shared_len=shared, stream=s)
    hip.sync()
    for pages, batch, dq, outs, ws, heads, shared, want, c in work:
        for o in outs:
            assert np.array_equal(host(o, want).view(np.int32), want.view(np.int32))


@pytest.mark.parametrize("room", ROOM)
def test_two_graphs_share_a_workspace(room):
    """Replayed in turn on one stream, with eager calls of the same workspace between: a call leaves nothing behind
    that another needs."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(__file__))))
    import bench
    hip = bench.Hip()
    s = hip.stream()
    rng = np.random.default_rng(34)
    work = []
    for rows, lens, shared in [([1, 1, 1], [900, 33, 410], 0), ([40, 1], [300, 280], 256)]:
        c = M.Cache(rng, "f16", 2, 128, 16, rows, lens, shared=shared, room=room)
        q = rng.standard_normal((c.n_rows, 8, 128)).astype(np.float32)
        want = attend(c, q, 8, 0.1, shared)
        work.append((*c.upload(), dev(q), dev(np.zeros_like(q)), shared, want, c))
    ws = uq.DeviceArray(max(serve.attn_paged_ws_bytes(w[0], w[1], 8, w[4]) for w in work))
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))

    def step(w, stream):
        serve.attn_paged_d(w[3], w[2], w[0], w[1], 8, 0.1, ws, shared_len=w[4], stream=stream)

    hip.sync()
    graphs = [hip.capture(s, lambda w=w: step(w, s)) for w in work]  # the kernels' first call for these shapes
    for i in range(6):
        w = work[i % 2]
        w[3].upload(np.full(w[5].shape, 7.0, np.float32))
        if i % 3 == 2:
            step(work[1 - i % 2], None)
        hip.sync()
        hip.launch_graph(graphs[i % 2], s)
        hip.sync()
        assert np.array_equal(host(w[3], w[5]).view(np.int32), w[5].view(np.int32)), f"replay {i}"


def test_attention_does_not_depend_on_the_other_sequences():
    """A sequence by itself and in a batch: the same up to the order of the sums."""
    rng = np.random.default_rng(24)
    c = M.Cache(rng, "f16", 4, 128, 16, [1, 4, 2], [500, 90, 1500])
    q = rng.standard_normal((7, 8, 128)).astype(np.float32)
    both = attend(c, q, 8, 0.1)
    one = M.Cache(np.random.default_rng(1), "f16", 4, 128, 16, [4], [90])
    one.k, one.v, one.n_pages, one.max_pages = c.k, c.v, c.n_pages, c.max_pages
    one.table = c.table[1:2]
    got = attend(one, q[1:5], 8, 0.1)
    _, bound = M.attention(one, q[1:5], 8, 0.1)
    assert np.all(np.abs(got - both[1:5]) <= 2 * bound)


def test_attention_over_a_long_cache():
    """70000 positions, f16: the bound of their number still holds where rows are spread over many workgroups."""
    rng = np.random.default_rng(25)
    c = M.Cache(rng, "f16", 1, 64, 256, [2], [70001])
    q = (3 * rng.standard_normal((2, 4, 64))).astype(np.float32)
    check(c, q, 4, 0.125, what="70001 positions")


def test_attention_in_place_and_on_another_stream():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(__file__))))
    import bench
    rng = np.random.default_rng(26)
    c = M.Cache(rng, "f32", 2, 64, 16, [2, 1], [300, 40])
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    want = attend(c, q, 4, 0.125)
    hip = bench.Hip()
    s = hip.stream()
    pages, batch = c.upload()
    d_q = dev(q)
    ws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, 4))
    hip.sync()
    serve.attn_paged_d(d_q, d_q, pages, batch, 4, 0.125, ws, stream=s)
    hip.ok(hip.h.hipStreamSynchronize(s), "hipStreamSynchronize")
    got = host(d_q, q)
    assert np.array_equal(got.view(np.int32), want.view(np.int32))


@pytest.mark.parametrize("room", ROOM)
def test_attention_captured_follows_lengths_and_pages(room):
    """One graph of append and attention; between the replays the lengths, pages and rows change on the device, and
    eager work with a workspace of its own runs."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(__file__))))
    import bench
    hip = bench.Hip()
    s = hip.stream()
    heads, kv, hd, page = 8, 2, 128, 16
    rng = np.random.default_rng(27)
    c = M.Cache(rng, "f16", kv, hd, page, [1, 2, 1], [200, 130, 9], pad=2, spare=20, room=room)
    pages, batch = c.upload()
    n = c.n_rows
    bufs = [uq.DeviceArray(4 * n * w * hd) for w in (heads, kv, kv, heads, heads)]
    dq, dk, dv, dqo, dout = bufs
    ws, other = (uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, heads)) for _ in range(2))
    hr = serve.HeadRows(heads, dq, heads * hd, hd, dqo, dk, kv * hd, dv, kv * hd, rope="imrope", n_rot=64, theta_scale=0.6)

    def step(stream=None, w=ws):
        serve.kv_append_d(pages, batch, hr, stream=stream)
        serve.attn_paged_d(dout, dqo, pages, batch, heads, 0.1, w, stream=stream)

    g = hip.capture(s, lambda: step(s))
    for r in range(4):
        x = [rng.standard_normal((n, w, hd)).astype(np.float32) for w in (heads, kv, kv)]
        for d, a in zip((dq, dk, dv), x):
            d.upload(a)
        lens = np.array([200 + r, 130 + 40 * r, 9 if r < 2 else 1], np.int32)
        start = np.array([0, 1, 3, 4] if r != 1 else [0, 2, 2, 5], np.int32)
        table = c.table.copy()
        table[1, 8:8 + 9] = np.random.default_rng(r).permutation(np.setdiff1d(np.arange(c.n_pages), c.table[[0, 2]]))[:min(9, c.max_pages - 8)][:table[1, 8:17].size]
        c.d_len.upload(lens)
        c.d_start.upload(start)
        c.d_table.upload(table)
        dout.upload(np.full(n * heads * hd, 7.0, np.float32))
        k0, v0 = host(c.d_k, c.k), host(c.d_v, c.v)
        hip.sync()
        step(w=other)
        want, wk = host(dout, x[0]), host(c.d_k, c.k)
        c.d_k.upload(k0)
        c.d_v.upload(v0)
        dout.upload(np.full(n * heads * hd, 7.0, np.float32))
        hip.sync()
        hip.launch_graph(g, s)
        hip.sync()
        assert np.array_equal(host(dout, x[0]).view(np.int32), want.view(np.int32)), f"replay {r}"
        assert np.array_equal(host(c.d_k, c.k).view(np.int16), wk.view(np.int16)), f"replay {r} keys"
        assert np.all(want[int(start[-1]):] == 7.0)


# ------------------------------------------------------------------------- verification

def run_verify(p, q, tokens, u, rows, p_pad=0, q_pad=0, pad_rows=0):
    n, vocab = p.shape
    wide = np.full((n, vocab + p_pad), 3.0, np.float32)
    wide[:, :vocab] = p
    dq = None
    if q is not None:
        wq = np.full((n, vocab + q_pad), 3.0, np.float32)
        wq[:, :vocab] = q
        dq = dev(wq)
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    d_start = dev(start)
    batch = serve.SeqBatch(len(rows), n, d_start)
    acc, nxt = dev(np.full(len(rows), 77, np.int32)), dev(np.full(len(rows), 77, np.int32))
    ws = uq.DeviceArray(max(16, serve.draft_verify_ws_bytes(batch, vocab)))
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
    serve.draft_verify_d(acc, nxt, dev(wide), dq, dev(np.asarray(tokens, np.int32)), dev(np.asarray(u, np.float32)), batch, vocab, ws,
                         p_row=vocab + p_pad, q_row=vocab + q_pad)
    like = np.zeros(len(rows), np.int32)
    return host(acc, like), host(nxt, like)


def probabilities(rng, n, vocab, sharp=3.0):
    x = sharp * rng.standard_normal((n, vocab))
    p = np.exp(x - x.max(-1, keepdims=True))
    return (p / p.sum(-1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("vocab,rows,draft,pads", [
    (7, [1, 4, 0, 2], True, (0, 0)), (1, [3, 1], True, (0, 0)), (2047, [5] * 9, True, (1, 3)), (2048, [8, 1, 3], False, (0, 0)),
    (2049, [8] * 20, True, (5, 0)), (32003, [1, 2, 3, 4, 5, 0], False, (0, 0)), (152064, [5, 1, 5], True, (0, 64)),
    (600001, [2, 3], True, (0, 0))])
def test_verify_against_64_bits(vocab, rows, draft, pads):
    rng = np.random.default_rng(vocab + len(rows))
    n = sum(rows)
    p = probabilities(rng, n, vocab)
    q = probabilities(rng, n, vocab) * 0.5 + p * 0.5 if draft else None
    tokens = rng.integers(0, vocab, n)
    for r in range(n - 1):  # drafts of likely tokens, so that runs are accepted
        if rng.random() < 0.8:
            tokens[r + 1] = rng.choice(vocab, p=(p[r] / p[r].astype(np.float64).sum()).astype(np.float64) / (p[r] / p[r].astype(np.float64).sum()).astype(np.float64).sum())
    u = rng.random(n).astype(np.float32) * (1.0 if draft else 0.1)
    got = run_verify(p, q, tokens, u, rows, *pads)
    want = M.verify(p, q, tokens, u, rows)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (got, want)


def test_verify_ties_and_edges():
    """Probabilities that are sums of powers of two: running sums are exact, a number on a border goes to the next
    token; equality refuses."""
    vocab = 5000
    p = np.zeros((8, vocab), np.float32)
    q = np.zeros_like(p)
    p[:, [3, 2500, 4999]] = [0.25, 0.5, 0.25]
    q[:, [3, 2500]] = [0.5, 0.5]
    rows = [1] * 8
    u = np.array([0.0, 0.25, 0.2499999, 0.75, 0.74999994, 0.99999994, 1.0, np.nan], np.float32)
    acc, nxt = run_verify(p, q, np.zeros(8), u, rows)
    assert acc.tolist() == [0] * 8 and nxt.tolist() == [3, 2500, 3, 4999, 2500, 4999, 4999, 4999]
    # u q = p refuses (0.5 * 0.5 = 0.25), just below accepts; after the refusal only token 4999 has p > q
    tokens = [0, 3, 0, 3]
    acc, nxt = run_verify(p[:4], q[:4], tokens, [0.5, 0.9, np.nextafter(np.float32(0.5), np.float32(0)), 0.3], [2, 2])
    assert acc.tolist() == [0, 1] and nxt.tolist() == [4999, 2500]
    # certain drafts: the refused token is left out
    acc, nxt = run_verify(p[:2], None, [0, 2500], [0.5, 0.6], [2])
    assert acc.tolist() == [0] and nxt.tolist() == [4999]
    # certain drafts of a certain target: refused only by u = 1, and then nothing is left but p itself
    one = np.zeros((2, vocab), np.float32)
    one[:, 11] = 1
    acc, nxt = run_verify(one, None, [0, 11], [1.0, 0.6], [2])
    assert acc.tolist() == [0] and nxt.tolist() == [11]
    acc, nxt = run_verify(one, one, [0, 11], [0.99, -3.0], [2])
    assert acc.tolist() == [1] and nxt.tolist() == [11]
    # drafted tokens outside the vocabulary are refused
    acc, nxt = run_verify(one, None, [0, vocab], [0.0, 0.6], [2])
    assert acc.tolist() == [0] and nxt.tolist() == [11]
    acc, nxt = run_verify(one, one * 0.5, [0, -1], [0.0, 0.6], [2])
    assert acc.tolist() == [0] and nxt.tolist() == [11]


def test_verify_weights_that_are_none():
    vocab = 4100
    p = np.zeros((5, vocab), np.float32)
    p[0, [5, 4000]] = [np.nan, 0.5]
    p[1, [5, 4000, 4001]] = [np.inf, 0.5, -1.0]
    p[2] = -1.0
    p[3, 4099] = 1e-38
    p[4] = np.nan
    acc, nxt = run_verify(p, None, np.zeros(5), np.full(5, 0.9), [1] * 5)
    assert acc.tolist() == [0] * 5 and nxt.tolist() == [4000, 4000, -1, 4099, -1]


def test_verify_captured():
    """Replays follow the tokens, numbers, probabilities and row starts of the time."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(__file__))))
    import bench
    hip = bench.Hip()
    s = hip.stream()
    rng = np.random.default_rng(35)
    vocab, n = 3001, 12
    like = np.zeros(3, np.int32)
    d_p, d_q, d_tok, d_u = (uq.DeviceArray(4 * k) for k in (n * vocab, n * vocab, n, n))
    d_start, acc, nxt = dev(np.zeros(4, np.int32)), dev(like), dev(like)
    batch = serve.SeqBatch(3, n, d_start)
    ws = uq.DeviceArray(serve.draft_verify_ws_bytes(batch, vocab))
    hip.sync()
    g = hip.capture(s, lambda: serve.draft_verify_d(acc, nxt, d_p, d_q, d_tok, d_u, batch, vocab, ws, stream=s))
    for rows in ([4, 4, 4], [1, 0, 8], [0, 0, 0], [12, 0, 0]):
        p = probabilities(rng, n, vocab, 2.0)
        q = probabilities(rng, n, vocab, 2.0) * 0.3 + p * 0.7
        tok = np.array([rng.integers(0, vocab)] + [int(np.argmax(p[r] * rng.random(vocab))) for r in range(n - 1)], np.int32)
        u = rng.random(n).astype(np.float32)
        for d, a in ((d_p, p), (d_q, q), (d_tok, tok), (d_u, u), (d_start, np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))):
            d.upload(a)
        hip.sync()
        hip.launch_graph(g, s)
        hip.sync()
        want = M.verify(p, q, tok, u, rows)
        assert np.array_equal(host(acc, like), want[0]) and np.array_equal(host(nxt, like), want[1]), rows


# ------------------------------------------------------------------------- together

def test_first_calls_of_a_process_captured():
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "serve_capture_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_paged_attention_of_a_layer_equals_its_step(dtype):
    """Tokens of a conversation through the attention layer's step, and their own projections through append and
    attention over pages: the f32 cache's rows are the contiguous cache's bit for bit, the gated attention agrees
    within the bound."""
    m = Model(SMALL, seed=81)
    c, d = m.cfg, m.d
    nt, ctx = 9, 16
    nh, nkv, hd = c.n_head, c.n_head_kv, c.head_dim
    rng = np.random.default_rng(3)
    X = rng.standard_normal((nt, c.n_embd)).astype(np.float32)
    kc, vc = uq.DeviceArray(4 * ctx * nkv * hd), uq.DeviceArray(4 * ctx * nkv * hd)
    ws, dl = uq.DeviceArray(4 * L.ws_floats(d, ctx)), uq.DeviceArray(4 * c.n_embd)
    qf, kr, vr, gated = (np.empty((nt, w), np.float32) for w in (2 * nh * hd, nkv * hd, nkv * hd, nh * hd))
    for t in range(nt):
        dx = dev(X[t])
        L.attn_step(d, m.aw, kc, vc, ctx, t, dx, dl, ws)
        nodes = nodes_of(d, ws, ["qfull", "k_raw", "gated"], ctx)
        qf[t], kr[t], gated[t] = nodes["qfull"], nodes["k_raw"], nodes["gated"]
    uq.synchronize()
    K = kc.download(np.float32, ctx * nkv * hd).reshape(ctx, nkv, hd)
    V = vc.download(np.float32, ctx * nkv * hd).reshape(ctx, nkv, hd)
    vr[:] = V[:nt].reshape(nt, -1)
    cache = M.Cache(rng, dtype, nkv, hd, 4, [6, 0, 3], [6, 0, 9], pad=1, spare=3)  # a prompt of 6, then 3 drafted
    cache.table[2, :2] = cache.table[0, :2]  # the same conversation: its first six positions' pages
    pages, batch = cache.upload()

    def padded(a):
        return dev(np.concatenate([a, np.zeros((1, a.shape[1]), np.float32)]))

    dqf, dk, dv, wq, wk = padded(qf), padded(kr), padded(vr), dev(m.ah["attn_q_norm"]), dev(m.ah["attn_k_norm"])
    dq, dout = uq.DeviceArray(4 * 10 * nh * hd), dev(np.full((10, nh, hd), 7.0, np.float32))
    aws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, nh))
    serve.kv_append_d(pages, batch, serve.HeadRows(nh, dqf, 2 * nh * hd, 2 * hd, dq, dk, nkv * hd, dv, nkv * hd, wq, wk, 1e-6,
                                                   "imrope", c.n_rot, None, c.theta_scale))
    view = type("View", (), {})()
    view.ptr = dqf.ptr.value + 4 * hd
    serve.attn_paged_d(dout, dq, pages, batch, nh, c.kq_scale, aws, d_gate=view, gate_row=2 * nh * hd, gate_head=2 * hd)
    got = host(dout, np.empty((10, nh, hd), np.float32))
    q = host(dq, np.empty((10, nh, hd), np.float32))
    cache.k, cache.v = host(cache.d_k, cache.k), host(cache.d_v, cache.v)
    pg, sl, ok = cache.slots(2, nt)
    assert ok.all()
    for a, b in ((cache.k, K), (cache.v, V)):
        assert np.array_equal(a[pg, :, sl], b[:nt].astype(a.dtype)), "cache rows"
    gate = np.concatenate([qf.reshape(nt, nh, 2, hd)[:, :, 1], np.zeros((1, nh, hd), np.float32)])
    want, bound = M.attention(cache, q, nh, c.kq_scale, gate)
    assert np.all(np.abs(got[:nt] - want[:nt]) <= bound[:nt])
    if dtype == "f32":
        assert np.all(np.abs(got[:nt].reshape(nt, -1) - gated) <= bound[:nt].reshape(nt, -1) + 4 * M.U32 * np.abs(gated))
    assert np.all(got[nt:] == 7.0)
    m.free()


def test_append_attend_verify_together():
    """A step of drafted tokens over a shared prompt, the operators in a row on one stream, and the same step again:
    the rows that verification accepts stay, the lengths follow, refused rows' slots are written over."""
    rng = np.random.default_rng(91)
    heads, kv, hd, page, vocab, shared = 4, 2, 64, 16, 999, 40
    rows, lens = [4, 2, 4], [44 + 4, 60, 41 + 4]
    c = M.Cache(rng, "f16", kv, hd, page, rows, lens, shared=shared, spare=4)
    n = c.n_rows
    head = uq.Weights(rng.standard_normal((vocab, heads * hd)).astype(np.float32) * 0.2, uq.DType.F32, heads * hd, vocab)
    pages, batch = c.upload()
    dq, dk, dv, dqo, dout = (uq.DeviceArray(4 * n * w * hd) for w in (heads, kv, kv, heads, heads))
    dlog, dp, dqp = (uq.DeviceArray(4 * n * vocab) for _ in range(3))
    acc, nxt, dtok, du = (uq.DeviceArray(4 * k) for k in (3, 3, n, n))
    ws = uq.DeviceArray(serve.attn_paged_ws_bytes(pages, batch, heads, shared))
    vws = uq.DeviceArray(serve.draft_verify_ws_bytes(batch, vocab))
    hr = serve.HeadRows(heads, dq, heads * hd, hd, dqo, dk, kv * hd, dv, kv * hd, rope="imrope", n_rot=32, theta_scale=0.7)
    start = [0, 4, 6, 10]
    for step in range(3):
        x = [rng.standard_normal((n, w, hd)).astype(np.float32) for w in (heads, kv, kv)]
        tok, u = rng.integers(0, vocab, n).astype(np.int32), (rng.random(n) * 0.02).astype(np.float32)
        qp = probabilities(rng, n, vocab, 1.0)
        for d, a in zip((dq, dk, dv, dtok, du, dqp), x + [tok, u, qp]):
            d.upload(a)
        serve.kv_append_d(pages, batch, hr)
        serve.attn_paged_d(dout, dqo, pages, batch, heads, 0.125, ws, shared_len=shared)
        uq.gemm(head, n, dout, dlog)
        ops.softmax_d(dp, dlog, vocab, n, 1.0)
        serve.draft_verify_d(acc, nxt, dp, dqp, dtok, du, batch, vocab, vws)
        q, out, p = (host(d, np.empty(s, np.float32)) for d, s in ((dqo, (n, heads, hd)), (dout, (n, heads, hd)), (dp, (n, vocab))))
        c.k, c.v = host(c.d_k, c.k), host(c.d_v, c.v)
        want, bound = M.attention(c, q, heads, 0.125)
        assert np.all(np.abs(out - want) <= bound), f"step {step}"
        for r, (b, pos) in enumerate(c.row_positions()):
            pg, sl, _ = c.slots(b, pos + 1)
            assert np.array_equal(c.v[pg[-1], :, sl[-1]], x[2][r].astype(np.float16))
        a, t = host(acc, np.empty(3, np.int32)), host(nxt, np.empty(3, np.int32))
        wa, wt = M.verify(p, qp, tok, u, rows)
        assert np.array_equal(a, wa) and np.array_equal(t, wt)
        # the next step's rows: the drawn token and new drafts, behind what was accepted
        room = c.max_pages * page
        c.lens = [min(room, ln - r + int(k) + 1 + r) for ln, r, k in zip(c.lens, rows, a)]
        for b, ln in enumerate(c.lens):
            for i in range(-(-ln // page)):
                if c.table[b, i] < 0:
                    c.table[b, i] = np.setdiff1d(np.arange(c.n_pages), c.table)[0]
        c.d_len.upload(np.array(c.lens, np.int32))
        c.d_table.upload(c.table)
