/*
 * uq_serve.h -- batched serving over a paged KV cache: the new rows (tokens)
 * of several sequences of different lengths through the parts of an attention
 * layer that depend on their positions and of a GatedDeltaNet layer that
 * depend on their states, the verification of drafted tokens and the log
 * probabilities of given ones. No counterpart in the reference, which runs one
 * sequence over contiguous caches and states
 * (crates/unltd-generation/src/qwen35_forward.rs:333-543, :585-671) and
 * decodes greedily (greedy.rs:18-65).
 *
 *   rows -> projections (uq_gemm / uq_gemm_q8k over all rows)
 *        -> an attention layer:
 *             uq_kv_append_d   (q / k norms, rotation, k and v into the pages)
 *             uq_attn_paged_d  (attention of the rows over the pages, gate)
 *           a GatedDeltaNet layer:
 *             uq_gdn_conv_d    (convolution, silu, q / k norms, gates)
 *             uq_gdn_rule_d    (gated delta rule, gated norm)
 *        -> output projection, FFN, head
 *        -> uq_softmax_d, uq_draft_verify_d; uq_logprobs_d
 *
 * Every entry point takes device pointers of the current HIP device and a
 * stream of it (NULL: its null stream), is asynchronous on that stream,
 * allocates nothing, copies nothing to the host and can be captured into a
 * HIP graph from its first call on. Structs are read during the call;
 * lengths, row starts and page tables are read on the device when the call
 * runs, so that a captured call follows them. Workspaces belong to the
 * caller: calls that may overlap need one each.
 */
#ifndef UQ_SERVE_H
#define UQ_SERVE_H

#include "uq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A paged cache of one attention layer. A page holds page_size consecutive
 * positions of one sequence (or of several that share them) for every KV
 * head: both arrays are [n_pages][n_head_kv][page_size][head_dim], 16-byte
 * aligned. UQ_F32 (the type of the contiguous caches) or UQ_F16. */
typedef struct uq_kv_pages {
    void *d_k, *d_v;
    uq_dtype dtype;
    size_t n_pages;   /* n_pages * n_head_kv * page_size below 2^31 */
    size_t page_size; /* a power of two, at most 65536 */
    size_t n_head_kv; /* at most 1024 */
    size_t head_dim; /* 64, 128, 256 or 512 */
} uq_kv_pages;

/* The new rows of a batch. Rows d_row_start[b] .. d_row_start[b+1] - 1 are
 * the last positions of sequence b, which holds d_len[b] positions with
 * them: row d_row_start[b] + i is position
 *   d_len[b] - (d_row_start[b+1] - d_row_start[b]) + i.
 * d_row_start ascends from 0; rows behind d_row_start[n_seqs] (a batch padded
 * to n_rows) belong to no sequence, and what a call writes for rows is left
 * as it was for them. A sequence may have no rows.
 * Position p of sequence b is slot p % page_size of page
 * d_pages[b * max_pages + p / page_size]. A page number outside [0, n_pages)
 * and a position beyond the table hold nothing: appending there writes
 * nothing, attention passes over them. */
typedef struct uq_seq_batch {
    size_t n_seqs, n_rows; /* at most 65535, 2^23 */
    const int32_t *d_row_start; /* [n_seqs + 1] */
    const int32_t *d_len;       /* [n_seqs] */
    const int32_t *d_pages;     /* [n_seqs][max_pages] */
    size_t max_pages;           /* max_pages * page_size at most 2^31 - 2^16 */
} uq_seq_batch;

/* Position rotation of a head's first n_rot values, as the per-row entry
 * points of uq_ops.h turn them, bit for bit. */
typedef enum uq_rope {
    UQ_ROPE_NONE = 0,
    UQ_ROPE_LLAMA = 1,  /* pairs (2i, 2i+1) by position * d_freqs[i] (uq_rope_llama) */
    UQ_ROPE_NEOX = 2,   /* pairs (i, i + n_rot/2) by position * d_freqs[i] (uq_rope_neox) */
    UQ_ROPE_IMROPE = 3  /* every third of those pairs by position * theta_scale^i (uq_rope_imrope) */
} uq_rope;

/* The heads of a batch's rows before the attention, as the projections leave
 * them. Strides are in floats. */
typedef struct uq_head_rows {
    size_t n_head;       /* query heads, a multiple of n_head_kv */
    const float *d_q;    /* head h of row r at r * q_row + h * q_head; NULL: no queries */
    size_t q_row, q_head;
    float *d_q_out;      /* [n_rows][n_head][head_dim]; may be d_q where the strides are the same */
    const float *d_k;    /* KV head j of row r at r * k_row + j * head_dim; NULL: no keys and no values */
    size_t k_row;
    const float *d_v;    /* likewise; not NULL where d_k is not */
    size_t v_row;
    const float *d_q_norm, *d_k_norm; /* rms norm weights [head_dim]; NULL: no norm */
    float eps;
    uq_rope rope;
    size_t n_rot;        /* even, at most head_dim */
    const float *d_freqs; /* [n_rot / 2] (LLAMA, NEOX) */
    double theta_scale;  /* (IMROPE) */
} uq_head_rows;

/* One pass over the heads of every row: queries normed (uq_rmsnorm's
 * numerics) and rotated to their positions into d_q_out, keys normed,
 * rotated and written to the row's slot of the cache, values written as they
 * are. f32 rows are uq_rmsnorm's and the rotations' bit for bit; an f16 cache
 * takes them rounded to nearest even (past 65519 infinite).
 * A row at a negative position is left out. Two rows of one slot (the same
 * page given to two sequences) leave the bits of either.
 * The sources may not overlap the cache or each other's outputs.
 * Errors: UQ_ERR_ARG (null pointers, shapes beyond the limits above, a
 * cache array not 16-byte aligned), UQ_ERR_DTYPE, UQ_ERR_LEN (n_head no
 * multiple of n_head_kv, n_rot odd or above head_dim, a row stride below
 * the row). */
uq_status uq_kv_append_d(const uq_kv_pages *kv, const uq_seq_batch *batch, const uq_head_rows *heads, void *stream);

/* Causal attention of every row over the pages of its sequence: for query
 * head h with KV head h / (n_head / n_head_kv),
 *   s[p] = kq_scale * q_h . K[p],   p = 0 .. the row's position
 *   out_h = sum over p of exp(s[p] - max s) V[p] / sum over p of exp(s[p] - max s).
 * d_q and d_out are [n_rows][n_head][head_dim] and may be the same array.
 * d_gate, if not NULL: out_h is multiplied by sigmoid(d_gate[r * gate_row +
 * h * gate_head + i]), the gated attention of qwen35_forward.rs:677-684.
 *
 * shared_len > 0: positions 0 .. shared_len - 1 are the same in every
 * sequence (a common document or system prompt). They are read through the
 * first sequence's pages, once for the rows of the whole batch; the
 * results are those of shared_len = 0 up to the order of the sums. Other
 * sequences' table entries of whole shared pages are not read.
 *
 * Numerics: f32 results of f32 sums over exact products of weights and of
 * queries times the mantissa of kq_scale log2 e (over an f32 cache rounded to
 * f32), in a fixed order: a call repeated gives the same bits. Over an f16
 * cache each of them is two f16 terms, within 2^-22 of it and, where it is
 * small, a step of f16's least numbers: a value of a query within 2^-38 of the
 * query's largest, a weight within 2^-33 of the row's largest (2^-25 for
 * scores beyond 2^22). So values below 2^-16 of a query's largest, and weights
 * below 2^-11 of the row's, have fewer bits than 22.
 * Scores times log2 e beyond f32's range are infinite.
 * What a row does not see (later positions, slots behind the length, pages
 * that are none) does not enter, whatever it holds. A row that sees no
 * position, or only scores of -infinity, is zero. Queries, and keys or values
 * that a row sees, which are not finite make its results NaN or infinite,
 * keys of a score of -infinity excepted.
 *
 * The workspace (uq_attn_paged_ws_bytes, 16-byte aligned) does not depend on
 * the lengths. uq_attn_paged_ws_bytes returns 0 for arguments that the call
 * refuses. Errors: UQ_ERR_ARG (also a workspace too small, shared_len beyond
 * the table, n_rows * n_head above 2^25 or kq_scale not finite), UQ_ERR_DTYPE,
 * UQ_ERR_LEN (n_head no multiple of n_head_kv). */
size_t uq_attn_paged_ws_bytes(const uq_kv_pages *kv, const uq_seq_batch *batch, size_t n_head, size_t shared_len);
uq_status uq_attn_paged_d(float *d_out, const float *d_q, const uq_kv_pages *kv, const uq_seq_batch *batch,
                          size_t n_head, size_t shared_len, float kq_scale, const float *d_gate, size_t gate_row,
                          size_t gate_head, void *d_ws, size_t ws_bytes, void *stream);

/* Verification of drafted tokens against the target's probabilities. The
 * rows of sequence b are its last known token and k = rows - 1 drafted
 * tokens after it: d_tokens[r] is row r's token, d_p [n_rows][vocab] (p_row
 * floats apart) the target's probabilities of what follows it, d_q the
 * distribution that the following token was drafted from (the last row's is
 * not read; NULL: the drafts are certain). With r = the sequence's first row,
 * i = 0, 1, ...: the draft x = d_tokens[r + i + 1] is accepted if
 *   d_u[r + i] * q[r + i][x] < p[r + i][x]   (exact; q = 1 for certain drafts),
 * up to the first that is not. d_accepted[b] is the number accepted and
 * d_next[b] the token after them, drawn from the weights w of row r +
 * d_accepted[b] with the sequence's last number u = d_u[r + k]: the least
 * token whose sum w[0] + .. + w[token] (64-bit) exceeds u * sum w, where
 *   w = p                  when every draft was accepted,
 *   w = max(p - q, 0)      after a refusal (certain drafts: p without x),
 *   w = p                  where that leaves no weight.
 * Weights that are NaN, negative or infinite count as zero; with no weight at
 * all d_next is -1; u at or above 1, or NaN, takes the last token with
 * weight, and below 0 the first. A drafted token outside [0, vocab) is
 * refused. A sequence without rows gives 0 and -1.
 * Only n_seqs, n_rows and d_row_start of the batch are read.
 * Errors: UQ_ERR_ARG (null pointers, a workspace too small, vocab 0 or above
 * 2^24), UQ_ERR_LEN (a row stride below vocab). */
size_t uq_draft_verify_ws_bytes(const uq_seq_batch *batch, size_t vocab);
uq_status uq_draft_verify_d(int32_t *d_accepted, int32_t *d_next, const float *d_p, size_t p_row, const float *d_q,
                            size_t q_row, const int32_t *d_tokens, const float *d_u, const uq_seq_batch *batch,
                            size_t vocab, void *d_ws, size_t ws_bytes, void *stream);

/* The states of one GatedDeltaNet layer, a slot for each sequence: what
 * uq_gdn_layer_step_d carries from token to token, one after another.
 * Sequence b begins with the state of slot d_from[b] (outside [0, n_slots):
 * zeros, a new sequence) and leaves its last one in slot d_to[b] (outside:
 * nowhere, as for drafts that are not verified yet: a second call over the
 * same rows takes the state on, in which each sequence is its accepted rows
 * and its refused ones a sequence behind it, from nothing to nowhere). Several
 * sequences may begin with one slot, as continuations of one prompt do. Two
 * sequences that end in one slot leave there any part of either's state; one
 * that begins with a slot that another of the call ends in gets unspecified
 * results. A sequence without rows writes nothing. */
typedef struct uq_gdn_states {
    float *d_conv;  /* [n_slots][conv_kernel][channels], channels = (2 n_qk_heads + n_v_heads) head_dim:
                       rows 0 .. conv_kernel - 2 are the last inputs; the last row is neither read nor written */
    float *d_state; /* [n_slots][n_v_heads][head_dim][head_dim], 16-byte aligned */
    size_t n_slots; /* n_slots * n_v_heads below 2^31 */
    size_t n_qk_heads, n_v_heads; /* 1 .. 1024 each; value head h has query and key head h % n_qk_heads */
    size_t head_dim;              /* 64 or 128 */
    size_t conv_kernel;           /* 2 .. 9 */
    const int32_t *d_from, *d_to; /* [n_seqs] */
} uq_gdn_states;

/* A batch's rows before the convolution, as the projections leave them.
 * Strides are in floats. */
typedef struct uq_gdn_rows {
    const float *d_qkv; /* [n_rows][channels], rows qkv_row apart: query heads, key heads, value heads */
    size_t qkv_row;
    const float *d_conv1d; /* [channels][conv_kernel] */
    float eps;             /* of the q / k norms */
    float *d_out;          /* [n_rows][channels] */
    const float *d_beta_raw, *d_alpha; /* [n_rows][n_v_heads], rows raw_row apart; both NULL: no gates */
    size_t raw_row;                    /* 0: n_v_heads */
    const float *d_dt_bias, *d_a; /* [n_v_heads] */
    float *d_beta, *d_gate;       /* [n_rows][n_v_heads] */
} uq_gdn_rows;

/* The convolution of every row over its sequence's last conv_kernel inputs
 * (those before its rows from the window), silu, and the query and key heads
 * divided by max(their 2-norm, eps) (steps 4 and 5 of recr_layer,
 * qwen35_forward.rs:427-464); the windows taken on; and the rows' gates
 * (:405-419): beta = sigmoid(beta_raw), gate = softplus(alpha + dt_bias) a.
 *
 * Numerics: f32, the convolution's sum in the taps' order and alpha + dt_bias
 * rounded once; silu, the norms and the gates of these add up to 16 roundings
 * (2^-24) of their values; silu below 2^-119 may be 0. Norms' sums of squares
 * beyond f32's range are infinite, as uq_l2_norm_rows'. A row's values that are
 * not finite reach the rows that convolve them and, in query and key heads, the
 * head.
 * d_out may not overlap the rows or the windows. Only n_seqs, n_rows and
 * d_row_start of the batch are read, and d_conv, not d_state.
 * Errors: UQ_ERR_ARG (null pointers, shapes beyond the limits above),
 * UQ_ERR_LEN (n_v_heads no multiple of n_qk_heads, a row stride below the
 * row). */
uq_status uq_gdn_conv_d(const uq_gdn_states *states, const uq_seq_batch *batch, const uq_gdn_rows *rows, void *stream);

/* A batch's rows before the delta rule. Strides are in floats. */
typedef struct uq_gdn_heads {
    const float *d_q, *d_k; /* head h of row r at r * q_row (k_row) + h * head_dim, h < n_qk_heads */
    const float *d_v;       /* likewise, h < n_v_heads */
    size_t q_row, k_row, v_row;
    const float *d_gate, *d_beta; /* [n_rows][n_v_heads] */
    float scale;
    const float *d_norm; /* rms norm weights [head_dim]; NULL: no norm */
    float eps;
    const float *d_z; /* head h of row r at r * z_row + h * head_dim; NULL: no gate */
    size_t z_row;
} uq_gdn_heads;

/* The gated delta rule (uq_gdn_fused_step, uq_ops.h) of every row of a
 * sequence in order, for each value head h with its query q, key k, value v,
 * gate g and beta:
 *   S <- exp(g) S;  S <- S + k (beta (v - S^T k))^T;  out = scale S^T q,
 * then, where given, out <- rmsnorm(out) d_norm and out <- out silu(d_z), the
 * gated norm of qwen35_forward.rs:495-511. d_out is [n_rows][n_v_heads]
 * [head_dim] and may not overlap the inputs or the states.
 *
 * most_rows: the most rows of a sequence, where the caller knows it (0: it
 * does not). It decides how the call is divided, not what rows it takes: a
 * sequence may have more. Sequences of few rows take them one by one, those
 * of many (from 24 in a small batch, from 48 in a large one) in chunks of 64
 * whose products run on the matrix cores:
 *   (I + A) U = diag(beta) (V - diag(e^G) K S),  A[i][j] = beta_i e^(G_i - G_j) k_i.k_j  (j < i),
 *   out = scale (diag(e^G) Q S + P U),           P[i][j] = e^(G_i - G_j) q_i.k_j         (j <= i),
 *   S <- e^G_63 S + (diag(e^(G_63 - G)) K)^T U,  G the running sum of the gates.
 * Both are deterministic; they differ by the order of f32 sums and by the
 * chunks' operands, as below. The gates' sums are held in 64 bits,
 * exponentials are of differences.
 *
 * Numerics: f32 sums. By chunks the products' operands are two f16 terms each,
 * within 2^-22 of a value or 2^-39 of the largest of its row (K, Q, T, P) or
 * column (U); for S and V - diag(e^G) K S, of a bound on the largest of a
 * column: the sum of the terms' sizes, sums over products by their number
 * times the largest. For keys of norm 1, gates at most 0 and betas of 0 to 1
 * no error grows, however many rows; results are off by some 1e-6 of the
 * largest; gates above 0 take an error on with the state. Values 2^20 times
 * smaller than others of their chunk and column, as after a gate that has all
 * forgotten, lose bits that row by row they keep.
 * Results, and e to the sum of a chunk's gates up to a row, beyond f32's range:
 * unspecified for the sequence's head from the start of those 64 rows on.
 * Values that are not finite make the results of their head from their row on,
 * and its state, NaN, infinite or unspecified; earlier rows, other heads and
 * other sequences do not see them.
 *
 * Only n_seqs, n_rows and d_row_start of the batch are read, and d_state, not
 * d_conv. The workspace (uq_gdn_rule_ws_bytes, 16-byte aligned) does not
 * depend on the row starts; uq_gdn_rule_ws_bytes returns 0 for arguments that
 * the call refuses. Errors: UQ_ERR_ARG (null pointers, shapes beyond the limits
 * above, a workspace too small, scale not finite), UQ_ERR_LEN (n_v_heads no
 * multiple of n_qk_heads, a row stride below the row, v_row above 2^24). */
size_t uq_gdn_rule_ws_bytes(const uq_gdn_states *states, const uq_seq_batch *batch, size_t most_rows);
uq_status uq_gdn_rule_d(float *d_out, const uq_gdn_states *states, const uq_seq_batch *batch,
                        const uq_gdn_heads *heads, size_t most_rows, void *d_ws, size_t ws_bytes, void *stream);

/* Results of uq_logprobs_d; any may be NULL. */
typedef struct uq_logprobs {
    float *d_logprob;     /* [n_rows]: the given token's */
    int32_t *d_rank;      /* [n_rows]: tokens before it in the order below */
    float *d_entropy;     /* [n_rows], in nats */
    int32_t *d_top_id;    /* [n_rows][n_top]: the first tokens in that order */
    float *d_top_logprob; /* [n_rows][n_top] */
    size_t n_top;         /* 0 .. 64 */
} uq_logprobs;

/* Of every row of logits x (rows x_row floats apart) the logarithms of the
 * probabilities softmax(scale x): those of the tokens d_tokens[r], the
 * entropy -sum p log p (p log p = 0 where p is 0), and the n_top likeliest
 * tokens. Tokens are ordered by their logits, the largest first, equal ones
 * by their number. d_tokens may be NULL where neither d_logprob nor d_rank is
 * wanted.
 * A logit of -infinity is a token that cannot follow: its log probability is
 * -infinity, and it is no alternative. Log probabilities below f32's range are
 * -infinity, too. Alternatives that there are not are -1 with -infinity. A row
 * without any possible token has entropy 0. A token outside [0, vocab) has log
 * probability -infinity and rank -1. A row with a logit that is NaN or
 * +infinity has NaN for log probabilities and entropy, and -1 for ranks and
 * alternatives.
 * Numerics: f32; the sums over the vocabulary run in a fixed order, up to 2^20
 * tokens none of more than 112 roundings. Ranks and alternatives are exact.
 * Errors: UQ_ERR_ARG (null pointers, vocab 0 or above 2^24, n_rows above 2^23,
 * n_rows * vocab above 2^39, n_top above 64, scale not positive or above
 * 2^127, a workspace too small or not 16-byte aligned), UQ_ERR_LEN (x_row
 * below vocab). */
size_t uq_logprobs_ws_bytes(size_t n_rows, size_t vocab, size_t n_top);
uq_status uq_logprobs_d(const uq_logprobs *out, const float *d_x, size_t x_row, const int32_t *d_tokens, size_t n_rows,
                        size_t vocab, float scale, void *d_ws, size_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* UQ_SERVE_H */
