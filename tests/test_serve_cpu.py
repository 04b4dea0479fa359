"""Batched serving (include/uq_serve.h) without a GPU: what is refused before
any launch, workspace sizes, and the index arithmetic that the kernels and the
CPU emulation share (uq_serve_index.h)."""
import ctypes as C

import numpy as np
import pytest

import serve_model as M
import uq
from uq import serve


class At:
    """An address that nothing is read from before the refusal."""

    def __init__(self, ptr=4096, nbytes=1 << 40):
        self.ptr, self.nbytes = ptr, nbytes


A = At()


def pages(**over):
    s = dict(d_k=A, d_v=A, dtype=uq.DType.F16, n_pages=100, page_size=16, n_head_kv=2, head_dim=128)
    return serve.KvPages(**dict(s, **over))


def batch(**over):
    s = dict(n_seqs=3, n_rows=7, d_row_start=A, d_len=A, d_pages=A, max_pages=20)
    return serve.SeqBatch(**dict(s, **over))


def heads(**over):
    s = dict(n_head=4, d_q=A, q_row=512, q_head=128, d_q_out=At(8192), d_k=A, k_row=256, d_v=A, v_row=256, rope="imrope", n_rot=64,
             theta_scale=0.5)
    return serve.HeadRows(**dict(s, **over))


def refused(kind, fn, *a, text="", **k):
    with pytest.raises(uq.UqError) as e:
        fn(*a, **k)
    assert e.value.kind == kind and text in str(e.value), str(e.value)


BAD_PAGES = [("DTYPE", dict(dtype=uq.DType.Q8_0)), ("DTYPE", dict(dtype=uq.DType.Q4K)), ("ARG", dict(head_dim=96)), ("ARG", dict(head_dim=0)),
             ("ARG", dict(page_size=0)), ("ARG", dict(page_size=24)), ("ARG", dict(page_size=131072)), ("ARG", dict(n_head_kv=0)),
             ("ARG", dict(n_pages=1 << 27)), ("ARG", dict(d_k=None)), ("ARG", dict(d_v=None)), ("ARG", dict(d_v=At(4104)))]
BAD_BATCH = [("ARG", dict(n_seqs=65536)), ("ARG", dict(n_rows=(1 << 24) + 1)), ("ARG", dict(d_row_start=None)), ("ARG", dict(d_len=None)),
             ("ARG", dict(d_pages=None)), ("ARG", dict(max_pages=1 << 27))]


@pytest.mark.parametrize("kind,over", BAD_PAGES)
def test_bad_pages_are_refused(kind, over):
    refused(kind, serve.kv_append_d, pages(**over), batch(), heads())
    refused(kind, serve.attn_paged_d, A, A, pages(**over), batch(), 4, 1.0, A)
    assert serve.attn_paged_ws_bytes(pages(**over), batch(), 4) == 0


@pytest.mark.parametrize("kind,over", BAD_BATCH)
def test_bad_batches_are_refused(kind, over):
    refused(kind, serve.kv_append_d, pages(), batch(**over), heads())
    refused(kind, serve.attn_paged_d, A, A, pages(), batch(**over), 4, 1.0, A)
    assert serve.attn_paged_ws_bytes(pages(), batch(**over), 4) == 0


@pytest.mark.parametrize("kind,over", [
    ("LEN", dict(n_head=3)), ("LEN", dict(n_head=0)), ("ARG", dict(n_head=1 << 17, q_row=1 << 25)), ("ARG", dict(d_q_out=None)), ("LEN", dict(q_head=127)),
    ("LEN", dict(q_row=511)), ("ARG", dict(d_v=None)), ("LEN", dict(k_row=255)), ("LEN", dict(v_row=0)), ("LEN", dict(n_rot=63)),
    ("LEN", dict(n_rot=130)), ("ARG", dict(rope="neox")), ("ARG", dict(rope="llama")), ("ARG", dict(d_q_out=A, q_row=1024, q_head=256))])
def test_bad_heads_are_refused(kind, over):
    refused(kind, serve.kv_append_d, pages(), batch(), heads(**over))


def test_unknown_rotation_and_null_structs_are_refused():
    h = heads()
    h.rope = 4
    refused("ARG", serve.kv_append_d, pages(), batch(), h)
    h.rope = -1
    refused("ARG", serve.kv_append_d, pages(), batch(), h)
    L = uq.lib()
    assert L.uq_kv_append_d(None, batch()._at, heads()._at, None) == 4
    assert L.uq_kv_append_d(pages()._at, None, heads()._at, None) == 4
    p, b = pages(), batch()
    assert L.uq_kv_append_d(p._at, b._at, None, None) == 4
    assert L.uq_attn_paged_ws_bytes(None, b._at, 4, 0) == 0 and L.uq_draft_verify_ws_bytes(None, 10) == 0


def test_attention_refusals():
    p, b = pages(), batch()
    refused("LEN", serve.attn_paged_d, A, A, p, b, 3, 1.0, A)
    refused("LEN", serve.attn_paged_d, A, A, p, b, 0, 1.0, A)
    refused("ARG", serve.attn_paged_d, At(None), A, p, b, 4, 1.0, A)
    refused("ARG", serve.attn_paged_d, A, At(None), p, b, 4, 1.0, A)
    refused("ARG", serve.attn_paged_d, A, A, p, b, 4, 1.0, At(None))
    refused("ARG", serve.attn_paged_d, A, A, p, b, 4, 1.0, At(4104), text="aligned")
    refused("ARG", serve.attn_paged_d, A, A, p, b, 4, 1.0, A, shared_len=321, text="beyond a table")
    for shared in (0, 320):
        need = serve.attn_paged_ws_bytes(p, b, 4, shared)
        assert need > 0
        refused("ARG", serve.attn_paged_d, A, A, p, b, 4, 1.0, At(nbytes=need - 1), shared_len=shared, text="workspace")
    refused("ARG", serve.attn_paged_d, A, A, p, batch(n_rows=1 << 24), 1 << 15, 1.0, A)
    refused("ARG", serve.attn_paged_d, A, A, p, batch(n_rows=(1 << 23) + 2), 4, 1.0, A)  # a grid of 2^32 threads
    assert serve.attn_paged_ws_bytes(p, batch(n_rows=1 << 15), 1 << 10) > 0
    refused("ARG", serve.attn_paged_d, A, A, p, batch(n_rows=(1 << 15) + 1), 1 << 10, 1.0, A, text="2^25")
    for scale in (float("nan"), float("inf"), -float("inf")):
        refused("ARG", serve.attn_paged_d, A, A, p, b, 4, scale, A, text="kq_scale")


def test_verification_refusals():
    b = serve.SeqBatch(2, 5, A)
    ok = dict(d_accepted=A, d_next=A, d_p=A, d_q=A, d_tokens=A, d_u=A, batch=b, vocab=100, ws=A)
    for name in ("d_accepted", "d_next", "d_p", "d_tokens", "d_u"):
        refused("ARG", serve.draft_verify_d, **dict(ok, **{name: At(None)}))
    refused("ARG", serve.draft_verify_d, **dict(ok, vocab=0), p_row=100)
    refused("ARG", serve.draft_verify_d, **dict(ok, vocab=(1 << 24) + 1))
    refused("LEN", serve.draft_verify_d, **ok, p_row=99)
    refused("LEN", serve.draft_verify_d, **ok, q_row=99)
    refused("ARG", serve.draft_verify_d, **dict(ok, ws=At(nbytes=serve.draft_verify_ws_bytes(b, 100) - 1)))
    refused("ARG", serve.draft_verify_d, **dict(ok, ws=At(4104)))
    refused("ARG", serve.draft_verify_d, **dict(ok, batch=serve.SeqBatch(2, 5, None)))


def test_empty_batches_need_no_device():
    p = pages()
    for b in (batch(n_seqs=0, n_rows=0), batch(n_rows=0)):
        serve.attn_paged_d(A, A, p, b, 4, 1.0, A)
        serve.kv_append_d(p, b, heads())
    serve.kv_append_d(p, batch(), serve.HeadRows())  # neither queries nor keys
    serve.draft_verify_d(A, A, A, A, A, A, serve.SeqBatch(0, 0, None), 10, A)


# ------------------------------------------------------------------------- indexes

def emu():
    E = uq.emu()
    I, LL, P = C.c_int, C.c_longlong, C.c_void_p
    E.uq_emu_seq_rows.argtypes = [I, I, I, P]
    E.uq_emu_seq_len.argtypes = [I, I]
    E.uq_emu_page_row.argtypes = [I, I, I, I, I, I]
    E.uq_emu_run_start.argtypes, E.uq_emu_run_start.restype = [LL, I, I], LL
    E.uq_emu_run_owner.argtypes = [LL, I, LL]
    E.uq_emu_blocks_of.argtypes = [I, I, I]
    return E


def test_row_starts_and_lengths_are_bounded():
    E, out = emu(), np.zeros(2, np.int32)

    def rows(a, b, n):
        E.uq_emu_seq_rows(a, b, n, out.ctypes.data_as(C.c_void_p))
        return out.tolist()

    assert rows(3, 7, 10) == [3, 4] and rows(7, 3, 10)[1] == 0 and rows(5, 5, 10)[1] == 0
    for a in (-5, 0, 3, 10, 11, 2 ** 31 - 1, -2 ** 31):
        for b in (-5, 0, 3, 10, 11, 2 ** 31 - 1, -2 ** 31):
            lo, n = rows(a, b, 10)
            assert 0 <= lo <= 10 and n >= 0 and lo + n <= 10
    assert [E.uq_emu_seq_len(x, 64) for x in (-1, 0, 5, 64, 65, 2 ** 31 - 1)] == [0, 0, 5, 64, 64, 64]


@pytest.mark.parametrize("n_pages,kv,log2", [(1, 1, 0), (7, 3, 0), (5, 2, 4), (2 ** 15 - 1, 4, 14)])
def test_page_rows_are_the_layout(n_pages, kv, log2):
    E, ps = emu(), 1 << log2
    for page in {0, n_pages // 2, n_pages - 1}:
        for j in range(kv):
            for pos in {0, 1, ps - 1, ps, 3 * ps + ps // 2, 2 ** 31 - 1}:
                assert E.uq_emu_page_row(n_pages, kv, log2, page, j, pos) == (page * kv + j) * ps + pos % ps < 2 ** 31
    for page in (-1, n_pages, 2 ** 31 - 1, -2 ** 31):
        assert E.uq_emu_page_row(n_pages, kv, log2, page, 0, 0) == -1, "no page"


@pytest.mark.parametrize("T,G", [(1, 1), (5, 5), (17, 5), (512, 512), (1000, 512), (8191, 512), (3 * 2 ** 33 + 1, 512)])
def test_every_unit_has_one_owner(T, G):
    E = emu()
    edges = [E.uq_emu_run_start(T, G, w) for w in range(G + 1)]
    assert edges[0] == 0 and edges[-1] == T and all(a < b for a, b in zip(edges, edges[1:])), "no empty runs while G <= T"
    for w in range(G):
        for u in {edges[w], edges[w + 1] - 1, (edges[w] + edges[w + 1] - 1) // 2}:
            assert E.uq_emu_run_owner(T, G, u) == w


@pytest.mark.parametrize("group,RB", [(1, 16), (3, 16), (4, 16), (24, 16), (4, 128), (8, 64)])
def test_blocks_hold_every_query(group, RB):
    E = emu()
    for n in (0, 1, 2, 15, 16, 17, 40, 127, 128, 129, 1 << 24):
        blocks = E.uq_emu_blocks_of(n, group, RB)
        assert blocks * RB >= n * group > (blocks - 1) * RB or n == blocks == 0


def test_the_model_reads_pages_as_the_layout_says():
    rng = np.random.default_rng(1)
    c = M.Cache(rng, "f32", 2, 64, 4, [1, 2], [9, 6])
    page, slot, ok = c.slots(0, 9)
    assert ok.all() and slot.tolist() == [0, 1, 2, 3] * 2 + [0] and len(set(page.tolist())) == 3
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    out, bound = M.attention(c, q, 4, 0.125)
    p = c.table[1, 0]
    k, v = c.k[[p, p, p, p, c.table[1, 1]], 1, [0, 1, 2, 3, 0]], c.v[[p, p, p, p, c.table[1, 1]], 1, [0, 1, 2, 3, 0]]
    s = k.astype(np.float64) @ q[1, 3] * 0.125
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[1, 3], w @ v, rtol=1e-12) and bound.shape == out.shape
