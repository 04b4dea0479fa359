"""The limits of batched serving's shapes (include/uq_serve.h) to the last value that is taken."""
import pytest

from test_serve_cpu import A, batch, heads, pages, refused
from uq import serve


@pytest.mark.parametrize("page_size", [1, 16, 4096, 65536])
def test_tables_end_before_positions_leave_an_int(page_size):
    """The attention counts positions in tiles of up to 128 and looks up tiles ahead: within 2^16 of 2^31 those counts
    would leave a 32-bit integer."""
    p = pages(page_size=page_size, n_pages=100)
    most = (2 ** 31 - 2 ** 16) // page_size
    assert serve.attn_paged_ws_bytes(p, batch(max_pages=most), 4) > 0
    assert serve.attn_paged_ws_bytes(p, batch(max_pages=most), 4, most * page_size) > 0
    for more in (most + 1, (2 ** 31 - 1) // page_size):
        if more > most:
            assert serve.attn_paged_ws_bytes(p, batch(max_pages=more), 4) == 0
            refused("ARG", serve.attn_paged_d, A, A, p, batch(max_pages=more), 4, 1.0, A, text="positions")
            refused("ARG", serve.kv_append_d, p, batch(max_pages=more), heads(), text="positions")
