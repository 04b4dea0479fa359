"""Batched serving over a paged KV cache (include/uq_serve.h): the new rows of
several sequences, their keys and values in pages, attention over them and
the verification of drafted tokens. Buffers are uq.DeviceArray or anything
with the same `ptr` and `nbytes`."""
from __future__ import annotations

import ctypes as C

from . import DeviceArray, _check, lib

ROPE = {"none": 0, "llama": 1, "neox": 2, "imrope": 3}


def _p(a):
    return None if a is None else a.ptr


class _Struct(C.Structure):
    """Holds on to the buffers that its pointers name."""

    def _keep(self, *bufs):
        self._bufs = bufs
        self._at = C.addressof(self)


class KvPages(_Struct):
    """uq_kv_pages: d_k, d_v are [n_pages][n_head_kv][page_size][head_dim] of dtype (F32 or F16)."""
    _fields_ = [("d_k", C.c_void_p), ("d_v", C.c_void_p), ("dtype", C.c_int), ("n_pages", C.c_size_t),
                ("page_size", C.c_size_t), ("n_head_kv", C.c_size_t), ("head_dim", C.c_size_t)]

    def __init__(self, d_k: DeviceArray, d_v: DeviceArray, dtype: int, n_pages: int, page_size: int, n_head_kv: int,
                 head_dim: int):
        super().__init__(_p(d_k), _p(d_v), int(dtype), n_pages, page_size, n_head_kv, head_dim)
        self._keep(d_k, d_v)


class SeqBatch(_Struct):
    """uq_seq_batch: rows d_row_start[b] .. d_row_start[b + 1] - 1 are the last of sequence b's d_len[b] positions,
    whose pages are d_pages[b]. Verification needs neither lengths nor pages."""
    _fields_ = [("n_seqs", C.c_size_t), ("n_rows", C.c_size_t), ("d_row_start", C.c_void_p), ("d_len", C.c_void_p),
                ("d_pages", C.c_void_p), ("max_pages", C.c_size_t)]

    def __init__(self, n_seqs: int, n_rows: int, d_row_start: DeviceArray, d_len: DeviceArray | None = None,
                 d_pages: DeviceArray | None = None, max_pages: int = 0):
        super().__init__(n_seqs, n_rows, _p(d_row_start), _p(d_len), _p(d_pages), max_pages)
        self._keep(d_row_start, d_len, d_pages)


class HeadRows(_Struct):
    """uq_head_rows: the heads of a batch's rows as the projections leave them; strides in floats. rope: none, llama,
    neox (both with d_freqs) or imrope (with theta_scale)."""
    _fields_ = [("n_head", C.c_size_t), ("d_q", C.c_void_p), ("q_row", C.c_size_t), ("q_head", C.c_size_t),
                ("d_q_out", C.c_void_p), ("d_k", C.c_void_p), ("k_row", C.c_size_t), ("d_v", C.c_void_p),
                ("v_row", C.c_size_t), ("d_q_norm", C.c_void_p), ("d_k_norm", C.c_void_p), ("eps", C.c_float),
                ("rope", C.c_int), ("n_rot", C.c_size_t), ("d_freqs", C.c_void_p), ("theta_scale", C.c_double)]

    def __init__(self, n_head: int = 0, d_q: DeviceArray | None = None, q_row: int = 0, q_head: int = 0,
                 d_q_out: DeviceArray | None = None, d_k: DeviceArray | None = None, k_row: int = 0,
                 d_v: DeviceArray | None = None, v_row: int = 0, d_q_norm: DeviceArray | None = None,
                 d_k_norm: DeviceArray | None = None, eps: float = 1e-6, rope: str = "none", n_rot: int = 0,
                 d_freqs: DeviceArray | None = None, theta_scale: float = 0.0):
        super().__init__(n_head, _p(d_q), q_row, q_head, _p(d_q_out), _p(d_k), k_row, _p(d_v), v_row, _p(d_q_norm),
                         _p(d_k_norm), eps, ROPE[rope], n_rot, _p(d_freqs), theta_scale)
        self._keep(d_q, d_q_out, d_k, d_v, d_q_norm, d_k_norm, d_freqs)


def kv_append_d(kv: KvPages, batch: SeqBatch, heads: HeadRows, stream=None) -> None:
    """uq_kv_append_d"""
    _check(lib().uq_kv_append_d(kv._at, batch._at, heads._at, stream))


def attn_paged_ws_bytes(kv: KvPages, batch: SeqBatch, n_head: int, shared_len: int = 0) -> int:
    """uq_attn_paged_ws_bytes: bytes of the attention's workspace (0 for arguments that it refuses)."""
    return lib().uq_attn_paged_ws_bytes(kv._at, batch._at, n_head, shared_len)


def attn_paged_d(d_out: DeviceArray, d_q: DeviceArray, kv: KvPages, batch: SeqBatch, n_head: int, kq_scale: float,
                 ws: DeviceArray, shared_len: int = 0, d_gate: DeviceArray | None = None, gate_row: int = 0,
                 gate_head: int = 0, stream=None) -> None:
    """uq_attn_paged_d: d_out, d_q are [n_rows][n_head][head_dim]; the first shared_len positions are every
    sequence's."""
    _check(lib().uq_attn_paged_d(d_out.ptr, d_q.ptr, kv._at, batch._at, n_head, shared_len, kq_scale, _p(d_gate),
                                 gate_row, gate_head, ws.ptr, ws.nbytes, stream))


def draft_verify_ws_bytes(batch: SeqBatch, vocab: int) -> int:
    """uq_draft_verify_ws_bytes"""
    return lib().uq_draft_verify_ws_bytes(batch._at, vocab)


def draft_verify_d(d_accepted: DeviceArray, d_next: DeviceArray, d_p: DeviceArray, d_q: DeviceArray | None,
                   d_tokens: DeviceArray, d_u: DeviceArray, batch: SeqBatch, vocab: int, ws: DeviceArray,
                   p_row: int = 0, q_row: int = 0, stream=None) -> None:
    """uq_draft_verify_d: probabilities d_p (d_q: the drafts' own, None for certain drafts) are [n_rows][vocab], rows
    p_row (q_row) floats apart (0: vocab)."""
    _check(lib().uq_draft_verify_d(d_accepted.ptr, d_next.ptr, d_p.ptr, p_row or vocab, _p(d_q), q_row or vocab,
                                   d_tokens.ptr, d_u.ptr, batch._at, vocab, ws.ptr, ws.nbytes, stream))
