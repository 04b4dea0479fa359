// Index arithmetic of the paged cache and of the batch, shared by the kernels
// and the CPU emulation: every number that comes from device memory (row
// starts, lengths, page numbers) is bounded here before it becomes an address.
#pragma once

#include <cstdint>

#include "uq_bits.h"

namespace uq {

// Rows [lo, lo + n) of a sequence; n is 0 where the starts do not ascend.
// Starts outside [0, n_rows] are moved into it.
struct SeqRows {
    int lo, n;
};
UQ_HD SeqRows seq_rows(int a, int b, int n_rows) {
    a = a < 0 ? 0 : a > n_rows ? n_rows : a;
    b = b < 0 ? 0 : b > n_rows ? n_rows : b;
    return SeqRows{a, b > a ? b - a : 0};
}

// A sequence's length: lengths below 0 hold nothing, those beyond the table
// end with it (cap = max_pages * page_size, at most 2^31 - 2^16).
UQ_HD int seq_len(int len, int cap) { return len < 0 ? 0 : len > cap ? cap : len; }

// Page geometry: the row of (page, kv head, slot) counts head_dim values.
struct PageMap {
    int n_pages, n_head_kv, log2_page;
};
UQ_HD bool page_ok(const PageMap &m, int page) { return (unsigned)page < (unsigned)m.n_pages; }
// Row of position pos in page `page` (page_ok) of KV head j; below 2^31.
UQ_HD int page_row(const PageMap &m, int page, int j, int pos) {
    return (int)((((unsigned)page * (unsigned)m.n_head_kv + (unsigned)j) << m.log2_page) |
                 ((unsigned)pos & ((1u << m.log2_page) - 1u)));
}

// ---- the attention's work list ---------------------------------------------
// Queries of a KV head are numbered row * group + head: block rb holds numbers
// [rb * RB, (rb + 1) * RB). A sequence of n rows has ceil(n * group / RB)
// blocks, each over `units` units of keys, for every KV head; units of all
// sequences (the shared positions' first) are numbered through, block by
// block, head by head, and G workgroups take equal runs of them.
UQ_HD int blocks_of(int n, int group, int RB) { return (int)(((long long)n * group + RB - 1) / RB); }
UQ_HD long long run_start(long long T, int G, int w) { return (long long)w * T / G; }
// The workgroup whose run holds unit u < T.
UQ_HD int run_owner(long long T, int G, long long u) { return (int)(((u + 1) * G - 1) / T); }

}  // namespace uq
