// C ABI of batched serving (include/uq_serve.h): argument checks, then the
// launches of uq_serve.hip and uq_attn_paged.hip.
#include <climits>
#include <cmath>
#include <cstdint>
#include <exception>

#include "uq_internal.h"
#include "uq_serve_internal.h"

using uq::set_error;

#define UQ_TRY(call)                \
    do {                            \
        const uq_status st_ = call; \
        if (st_) return st_;        \
    } while (0)

namespace {

uq_status hip_st(hipError_t e, const char *what) { return e == hipSuccess ? UQ_OK : uq::hip_error(e, what); }

constexpr size_t kMaxRows = 1u << 23;  // of a call: a grid of 256 threads each stays below 2^32
constexpr size_t kMaxSeqs = 65535;     // a grid dimension of the verification
constexpr size_t kMaxPairs = 1u << 25; // rows times heads of the attention: a grid of 64 threads each, likewise
constexpr size_t kMaxVocab = 1u << 24;
// Positions of a table: the kernels' int counts run up to a block of tiles past the last one.
constexpr size_t kMaxPositions = (size_t)INT_MAX + 1 - 65536;

// need_len: the call reads lengths and pages as well as row starts.
uq_status view_batch(const char *fn, const uq_seq_batch *b, bool need_len, uq::BatchView *v) {
    if (!b) return set_error(UQ_ERR_ARG, "%s: null batch", fn);
    if (b->n_seqs > kMaxSeqs) return set_error(UQ_ERR_ARG, "%s: %zu sequences above %zu", fn, b->n_seqs, kMaxSeqs);
    if (b->n_rows > kMaxRows) return set_error(UQ_ERR_ARG, "%s: %zu rows above %zu", fn, b->n_rows, kMaxRows);
    if (b->n_seqs && !b->d_row_start) return set_error(UQ_ERR_ARG, "%s: null row starts", fn);
    if (need_len && b->n_seqs && !b->d_len) return set_error(UQ_ERR_ARG, "%s: null lengths", fn);
    if (need_len && b->n_seqs && b->max_pages && !b->d_pages) return set_error(UQ_ERR_ARG, "%s: null page table", fn);
    *v = uq::BatchView{(int)b->n_seqs, (int)b->n_rows, 0, b->d_row_start, b->d_len, b->d_pages};
    return UQ_OK;
}

uq_status view_pages(const char *fn, const uq_kv_pages *kv, const uq_seq_batch *b, uq::PagesView *v, uq::BatchView *bv) {
    if (!kv) return set_error(UQ_ERR_ARG, "%s: null cache", fn);
    if (kv->dtype != UQ_F32 && kv->dtype != UQ_F16)
        return set_error(UQ_ERR_DTYPE, "%s: cache dtype %d is neither F32 nor F16", fn, (int)kv->dtype);
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256 && kv->head_dim != 512)
        return set_error(UQ_ERR_ARG, "%s: head_dim %zu is not 64, 128, 256 or 512", fn, kv->head_dim);
    if (kv->page_size == 0 || kv->page_size > 65536 || (kv->page_size & (kv->page_size - 1)))
        return set_error(UQ_ERR_ARG, "%s: page_size %zu is not a power of two up to 65536", fn, kv->page_size);
    if (kv->n_head_kv == 0 || kv->n_head_kv > 1024)
        return set_error(UQ_ERR_ARG, "%s: n_head_kv %zu outside 1 .. 1024", fn, kv->n_head_kv);
    const size_t per = kv->n_head_kv * kv->page_size;  // below 2^27
    if (kv->n_pages > (size_t)INT_MAX / per)
        return set_error(UQ_ERR_ARG, "%s: %zu pages of %zu rows reach 2^31 rows", fn, kv->n_pages, per);
    if (kv->n_pages && (!kv->d_k || !kv->d_v)) return set_error(UQ_ERR_ARG, "%s: null cache array", fn);
    if (((uintptr_t)kv->d_k | (uintptr_t)kv->d_v) % 16)
        return set_error(UQ_ERR_ARG, "%s: cache arrays are not 16-byte aligned", fn);
    UQ_TRY(view_batch(fn, b, true, bv));
    if (b->max_pages > kMaxPositions / kv->page_size)
        return set_error(UQ_ERR_ARG, "%s: a table of %zu pages of %zu has more than 2^31 - 2^16 positions", fn,
                         b->max_pages, kv->page_size);
    bv->max_pages = (int)b->max_pages;
    int lg = 0;
    while (((size_t)1 << lg) < kv->page_size) lg++;
    *v = uq::PagesView{uq::PageMap{(int)kv->n_pages, (int)kv->n_head_kv, lg}, (int)kv->n_head_kv, (int)kv->head_dim,
                       kv->dtype == UQ_F16, kv->d_k, kv->d_v};
    return UQ_OK;
}

uq_status check_heads(const char *fn, size_t n_head, const uq::PagesView &kv) {
    if (n_head == 0 || n_head % (size_t)kv.n_head_kv)
        return set_error(UQ_ERR_LEN, "%s: n_head %zu is not a multiple of n_head_kv %d", fn, n_head, kv.n_head_kv);
    if (n_head > 65536) return set_error(UQ_ERR_ARG, "%s: n_head %zu above 65536", fn, n_head);
    return UQ_OK;
}

// The attention's arguments as far as its workspace depends on them.
uq_status view_attn(const char *fn, const uq_kv_pages *kv, const uq_seq_batch *b, size_t n_head, size_t shared_len,
                    uq::PagesView *pv, uq::BatchView *bv) {
    UQ_TRY(view_pages(fn, kv, b, pv, bv));
    UQ_TRY(check_heads(fn, n_head, *pv));
    if (b->n_rows * n_head > kMaxPairs)
        return set_error(UQ_ERR_ARG, "%s: %zu rows of %zu heads above 2^25", fn, b->n_rows, n_head);
    if (shared_len > b->max_pages * kv->page_size)
        return set_error(UQ_ERR_ARG, "%s: shared_len %zu beyond a table of %zu positions", fn, shared_len,
                         b->max_pages * kv->page_size);
    return UQ_OK;
}

}  // namespace

extern "C" {

uq_status uq_kv_append_d(const uq_kv_pages *kv, const uq_seq_batch *batch, const uq_head_rows *h, void *stream) {
    const char *fn = "kv_append_d";
    uq::PagesView pv;
    uq::BatchView bv;
    UQ_TRY(view_pages(fn, kv, batch, &pv, &bv));
    if (!h) return set_error(UQ_ERR_ARG, "%s: null heads", fn);
    if (h->d_q) {
        UQ_TRY(check_heads(fn, h->n_head, pv));
        if (!h->d_q_out) return set_error(UQ_ERR_ARG, "%s: queries without d_q_out", fn);
        if (h->n_head > 1 && h->q_head < kv->head_dim)
            return set_error(UQ_ERR_LEN, "%s: q_head %zu below head_dim %zu", fn, h->q_head, kv->head_dim);
        if (batch->n_rows > 1 && h->q_row < (h->n_head - 1) * h->q_head + kv->head_dim)
            return set_error(UQ_ERR_LEN, "%s: q_row %zu below the heads of a row", fn, h->q_row);
        if (h->d_q_out == h->d_q && batch->n_rows &&
            ((batch->n_rows > 1 && h->q_row != h->n_head * kv->head_dim) ||
             (h->n_head > 1 && h->q_head != kv->head_dim)))
            return set_error(UQ_ERR_ARG, "%s: d_q_out is d_q with other strides", fn);
    }
    if (h->d_k) {
        const size_t wide = kv->n_head_kv * kv->head_dim;
        if (!h->d_v) return set_error(UQ_ERR_ARG, "%s: keys without values", fn);
        if (batch->n_rows > 1 && (h->k_row < wide || h->v_row < wide))
            return set_error(UQ_ERR_LEN, "%s: k_row %zu or v_row %zu below %zu", fn, h->k_row, h->v_row, wide);
    }
    if (h->rope < UQ_ROPE_NONE || h->rope > UQ_ROPE_IMROPE)
        return set_error(UQ_ERR_ARG, "%s: unknown rotation %d", fn, (int)h->rope);
    if (h->rope != UQ_ROPE_NONE) {
        if (h->n_rot % 2 || h->n_rot > kv->head_dim)
            return set_error(UQ_ERR_LEN, "%s: n_rot %zu is odd or above head_dim %zu", fn, h->n_rot, kv->head_dim);
        if (h->rope != UQ_ROPE_IMROPE && h->n_rot && !h->d_freqs)
            return set_error(UQ_ERR_ARG, "%s: rotation without frequencies", fn);
    }
    return hip_st(uq::launch_kv_append(pv, bv, *h, (hipStream_t)stream), fn);
}

size_t uq_attn_paged_ws_bytes(const uq_kv_pages *kv, const uq_seq_batch *batch, size_t n_head, size_t shared_len) {
    uq::PagesView pv;
    uq::BatchView bv;
    if (view_attn("attn_paged_ws_bytes", kv, batch, n_head, shared_len, &pv, &bv)) return 0;
    return uq::attn_paged_ws_bytes(pv, bv, (int)n_head, (int)shared_len);
}

uq_status uq_attn_paged_d(float *d_out, const float *d_q, const uq_kv_pages *kv, const uq_seq_batch *batch,
                          size_t n_head, size_t shared_len, float kq_scale, const float *d_gate, size_t gate_row,
                          size_t gate_head, void *d_ws, size_t ws_bytes, void *stream) {
    const char *fn = "attn_paged_d";
    uq::PagesView pv;
    uq::BatchView bv;
    UQ_TRY(view_attn(fn, kv, batch, n_head, shared_len, &pv, &bv));
    if (!std::isfinite(kq_scale)) return set_error(UQ_ERR_ARG, "%s: kq_scale is not finite", fn);
    if (batch->n_rows == 0 || batch->n_seqs == 0) return UQ_OK;
    if (!d_out || !d_q || !d_ws) return set_error(UQ_ERR_ARG, "%s: null device pointer", fn);
    if ((uintptr_t)d_ws % 16) return set_error(UQ_ERR_ARG, "%s: the workspace is not 16-byte aligned", fn);
    const size_t need = uq::attn_paged_ws_bytes(pv, bv, (int)n_head, (int)shared_len);
    if (ws_bytes < need) return set_error(UQ_ERR_ARG, "%s: workspace of %zu bytes below %zu", fn, ws_bytes, need);
    const uq::AttnPagedArgs a{d_out, d_q, (int)n_head, (int)shared_len, kq_scale, d_gate, gate_row, gate_head};
    try {
        return hip_st(uq::launch_attn_paged(pv, bv, a, d_ws, (hipStream_t)stream), fn);
    } catch (const std::exception &e) {  // the record of raised LDS limits is the one allocation
        return set_error(UQ_ERR_HIP, "%s: %s", fn, e.what());
    }
}

size_t uq_draft_verify_ws_bytes(const uq_seq_batch *batch, size_t vocab) {
    uq::BatchView bv;
    if (view_batch("draft_verify_ws_bytes", batch, false, &bv) || vocab == 0 || vocab > kMaxVocab) return 0;
    return uq::draft_verify_ws_bytes(bv.n_seqs, (int)vocab);
}

uq_status uq_draft_verify_d(int32_t *d_accepted, int32_t *d_next, const float *d_p, size_t p_row, const float *d_q,
                            size_t q_row, const int32_t *d_tokens, const float *d_u, const uq_seq_batch *batch,
                            size_t vocab, void *d_ws, size_t ws_bytes, void *stream) {
    const char *fn = "draft_verify_d";
    uq::BatchView bv;
    UQ_TRY(view_batch(fn, batch, false, &bv));
    if (vocab == 0 || vocab > kMaxVocab) return set_error(UQ_ERR_ARG, "%s: vocab %zu outside 1 .. 2^24", fn, vocab);
    if (p_row < vocab || (d_q && q_row < vocab))
        return set_error(UQ_ERR_LEN, "%s: a row stride (%zu, %zu) below vocab %zu", fn, p_row, q_row, vocab);
    if (bv.n_seqs == 0) return UQ_OK;
    if (!d_accepted || !d_next || (bv.n_rows && (!d_p || !d_tokens || !d_u)) || !d_ws)
        return set_error(UQ_ERR_ARG, "%s: null device pointer", fn);
    if ((uintptr_t)d_ws % 16) return set_error(UQ_ERR_ARG, "%s: the workspace is not 16-byte aligned", fn);
    const size_t need = uq::draft_verify_ws_bytes(bv.n_seqs, (int)vocab);
    if (ws_bytes < need) return set_error(UQ_ERR_ARG, "%s: workspace of %zu bytes below %zu", fn, ws_bytes, need);
    return hip_st(uq::launch_draft_verify(d_accepted, d_next, d_p, p_row, d_q, q_row, d_tokens, d_u, bv, (int)vocab,
                                          d_ws, (hipStream_t)stream),
                  fn);
}

}  // extern "C"
