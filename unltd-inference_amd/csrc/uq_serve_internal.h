// Shared by the batched-serving kernels (uq_serve.hip, uq_attn_paged.hip) and
// their C ABI (uq_serve_abi.cpp): the batch as the kernels see it, and the
// index arithmetic that the host checks and the CPU tests run as well.
#pragma once

#include "../../include/uq_serve.h"
#include "uq_serve_index.h"

#include <hip/hip_runtime.h>

namespace uq {

struct BatchView {
    int n_seqs, n_rows, max_pages;
    const int32_t *row_start, *len, *pages;
};

// The cache's geometry (uq_serve_index.h's PageMap) and its arrays.
struct PagesView {
    PageMap map;
    int n_head_kv, head_dim;
    bool f16;
    void *k, *v;
};

hipError_t launch_kv_append(const PagesView &kv, const BatchView &b, const uq_head_rows &h, hipStream_t s);

struct AttnPagedArgs {
    float *out;
    const float *q;
    int n_head, shared_len;
    float scale;
    const float *gate;
    size_t gate_row, gate_head;
};
size_t attn_paged_ws_bytes(const PagesView &kv, const BatchView &b, int n_head, int shared_len);
hipError_t launch_attn_paged(const PagesView &kv, const BatchView &b, const AttnPagedArgs &a, void *ws, hipStream_t s);

size_t draft_verify_ws_bytes(int n_seqs, int vocab);
hipError_t launch_draft_verify(int32_t *accepted, int32_t *next, const float *p, size_t p_row, const float *q,
                               size_t q_row, const int32_t *tokens, const float *u, const BatchView &b, int vocab,
                               void *ws, hipStream_t s);

}  // namespace uq
