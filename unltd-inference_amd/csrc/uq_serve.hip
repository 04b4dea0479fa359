// Batched serving: preparation and append of a batch's heads
// (uq_kv_append_d) and the verification of drafted tokens
// (uq_draft_verify_d). The attention over the pages is uq_attn_paged.hip.
#include <algorithm>
#include <climits>

#include "uq_device.h"
#include "uq_serve_internal.h"

namespace uq {

namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any float

// ---- heads of a row ---------------------------------------------------------

constexpr int kAppTPB = 256;
constexpr int kAppMaxHd = 512;

// The row's sequence, position and page, found by the whole workgroup at once
// (one round trip for the starts and lengths, one for the page) and left in
// LDS. pos -1: the row belongs to no sequence or lies at a negative position.
struct RowAt {
    int seq, pos, page;
};

__device__ __forceinline__ void find_row(const BatchView &b, const PageMap &m, int row, RowAt *at) {
    if (threadIdx.x == 0) *at = RowAt{-1, -1, -1};
    __syncthreads();
    for (int i = threadIdx.x; i < b.n_seqs; i += kAppTPB) {
        const SeqRows r = seq_rows(b.row_start[i], b.row_start[i + 1], b.n_rows);
        if (row < r.lo || row >= r.lo + r.n) continue;
        const int cap = b.max_pages << m.log2_page, len = b.len[i];
        const int pos = len - r.n + (row - r.lo);
        int page = -1;
        if (len >= 0 && pos >= 0 && pos < cap) page = b.pages[(size_t)i * b.max_pages + (pos >> m.log2_page)];
        *at = RowAt{i, len >= 0 ? pos : -1, page};
    }
    __syncthreads();
}

// E consecutive floats of a row from any float on.
template <int E>
__device__ __forceinline__ void load_row(float (&v)[E], const float *p) {
    if constexpr (E >= 4) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const f4u f = *(const f4u *)(p + e);
#pragma unroll
            for (int i = 0; i < 4; i++) v[e + i] = f[i];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = p[e];
    }
}
template <int E>
__device__ __forceinline__ void store_row(float *p, const float (&v)[E]) {
    if constexpr (E >= 4) {
#pragma unroll
        for (int e = 0; e < E; e += 4) *(f4u *)(p + e) = f4u{v[e], v[e + 1], v[e + 2], v[e + 3]};
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) p[e] = v[e];
    }
}
// Rounded to nearest even, as one store of 2 E bytes (rows are 2 E-byte aligned).
template <int E>
__device__ __forceinline__ void store_half(_Float16 *p, const float (&v)[E]) {
    typedef _Float16 hE __attribute__((ext_vector_type(E)));
    if constexpr (E == 1) {
        *p = (_Float16)v[0];
    } else {
        hE h;
#pragma unroll
        for (int e = 0; e < E; e++) h[e] = (_Float16)v[e];
        *(hE *)p = h;
    }
}

// rms norm of a row held E values a lane (uq_rmsnorm's bits): the sequential
// f64 sum of the f32 squares as the wave's tree with the bound of
// seq_sum_f32 (uq_device.h), or, undecided, replayed in order with each value
// taken from its lane.
template <int E>
__device__ __forceinline__ void norm_row(float (&v)[E], const float (&w)[E], float eps) {
    constexpr int n = 64 * E;
    double s = 0.0;
#pragma unroll
    for (int e = 0; e < E; e++) s += (double)__fmul_rn(v[e], v[e]);
    const double S = wave_sum_d(s), dn = (double)n, er = (double)(n + 66) * 0x1p-52 * S;
    float mean = (float)((S - er) / dn);
    if (__float_as_uint(mean) != __float_as_uint((float)((S + er) / dn))) {  // wave-uniform
        double q = 0.0;
        for (int l = 0; l < 64; l++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float t = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v[e]), l));
                q += (double)__fmul_rn(t, t);
            }
        mean = (float)(q / dn);
    }
    const float scale = __fdiv_rn(1.0f, sqrtf_cr(__fadd_rn(mean, eps)));
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = __fmul_rn(__fmul_rn(v[e], scale), w[e]);
}

struct AppendArgs {
    uq_head_rows h;
    PagesView kv;
    BatchView b;
};

// One workgroup for a row's heads blockIdx.y, blockIdx.y + gridDim.y, ...: the
// row's angles once (f64 sine and cosine, as the per-row rotations take
// them; they cost as much as a head's whole norm), kept in LDS, then a wave a
// head: E = HD / 64 values a lane, norm in registers, rotation through the
// wave's own LDS row, one store. Memory bounds it (4024 rows of 24 heads of
// 256 values: 47 us, 4.2 TB/s; from the chip's cache 35), or for a few rows a
// launch (4.6 us, 5.9 with its start).
template <int HD, bool F16>
__global__ __launch_bounds__(kAppTPB) void kv_append_kernel(AppendArgs a) {
    constexpr int E = HD / 64, NW = kAppTPB / 64;
    __shared__ RowAt at;
    __shared__ double2 turn[kAppMaxHd / 2];
    __shared__ float rowv[NW][HD];
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uq_head_rows &h = a.h;
    const int nq = h.d_q ? (int)h.n_head : 0, nk = h.d_k ? a.kv.n_head_kv : 0, step_u = NW * (int)gridDim.y;
    auto load = [&](float (&v)[E], int u) {
        const float *src = u < nq        ? h.d_q + (size_t)row * h.q_row + (size_t)u * h.q_head
                           : u >= nq + nk ? h.d_v + (size_t)row * h.v_row + (size_t)(u - nq - nk) * HD
                                          : h.d_k + (size_t)row * h.k_row + (size_t)(u - nq) * HD;
        load_row<E>(v, src + E * lane);
    };
    int u = wave + NW * (int)blockIdx.y;
    float v[E], ahead[E];  // a head under way while the one before it is worked on, the first while the row is looked for
    if (u < nq + 2 * nk) load(ahead, u);
    find_row(a.b, a.kv.map, row, &at);
    const int pos = at.pos, page = at.page;
    if (pos < 0) return;
    const int half = (int)h.n_rot / 2, step = h.rope == UQ_ROPE_IMROPE ? 3 : 1;
    const int turns = h.rope == UQ_ROPE_NONE ? 0 : (half + step - 1) / step;
    for (int t = threadIdx.x; t < turns; t += kAppTPB) {
        double angle = (double)pos;
        if (h.rope == UQ_ROPE_IMROPE)
            for (int i = 0; i < 3 * t; i++) angle *= h.theta_scale;
        else
            angle *= (double)h.d_freqs[t];
        double sn, cs;
        sincos(angle, &sn, &cs);
        turn[t] = make_double2(sn, cs);
    }
    __syncthreads();
    const bool cached = page_ok(a.kv.map, page);
    for (; u < nq + 2 * nk; u += step_u) {
        const bool isq = u < nq, isv = u >= nq + nk;
        const int j = isq ? u : isv ? u - nq - nk : u - nq;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = ahead[e];
        if (u + step_u < nq + 2 * nk) load(ahead, u + step_u);
        if (!isq && !cached) continue;  // the whole wave
        if (!isv) {
            const float *w = isq ? h.d_q_norm : h.d_k_norm;
            if (w) {
                float wv[E];
                load_row<E>(wv, w + E * lane);
                norm_row<E>(v, wv, h.eps);
            }
            if (turns) {
                float *rv = rowv[wave];
#pragma unroll
                for (int e = 0; e < E; e++) rv[E * lane + e] = v[e];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                for (int t = lane; t < turns; t += 64) {
                    const int x = h.rope == UQ_ROPE_LLAMA ? 2 * t : step * t;
                    const int y = h.rope == UQ_ROPE_LLAMA ? x + 1 : x + half;
                    const double2 tr = turn[t];
                    const double x0 = (double)rv[x], x1 = (double)rv[y];
                    rv[x] = (float)fma(tr.y, x0, -(tr.x * x1));
                    rv[y] = (float)fma(tr.x, x0, tr.y * x1);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int e = 0; e < E; e++) v[e] = rv[E * lane + e];
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (isq) {
            store_row<E>(h.d_q_out + ((size_t)row * h.n_head + j) * HD + E * lane, v);
        } else {
            const size_t o = (size_t)page_row(a.kv.map, page, j, pos) * HD + E * lane;
            if constexpr (F16)
                store_half<E>((_Float16 *)(isv ? a.kv.v : a.kv.k) + o, v);
            else
                store_row<E>((float *)(isv ? a.kv.v : a.kv.k) + o, v);
        }
    }
}

// ---- verification -------------------------------------------------------------

constexpr int kVerTPB = 256;
constexpr int kVerChunk = 512;  // tokens that a wave sums: 8 a lane

struct VerifyArgs {
    int32_t *accepted, *next;
    const float *p, *q;
    size_t p_row, q_row;
    const int32_t *tokens;
    const float *u;
    BatchView b;
    int vocab, chunks;
    int run;        // chunks of a wave
    double2 *sums;  // [n_seqs][chunks]: the chunk's weight after a refusal, and of p alone
    int4 *heads;    // [n_seqs]: first row, rows, accepted, the bits of the number that draws
};

// A weight that is NaN, negative or infinite counts as zero.
__device__ __forceinline__ double weight(double w) { return w > 0.0 && w < (double)INFINITY ? w : 0.0; }

struct Row {
    size_t row;   // the row that is drawn from
    int accepted, last;  // last: index of the sequence's last row
    bool ended;   // every draft was accepted
    int x;        // the refused token (certain drafts)
};

__device__ __forceinline__ Row row_at(const VerifyArgs &a, const SeqRows &r, int accepted) {
    Row o;
    o.row = (size_t)r.lo + accepted;
    o.accepted = accepted;
    o.last = r.lo + r.n - 1;
    o.ended = accepted == r.n - 1;
    o.x = !o.ended && !a.q ? a.tokens[o.row + 1] : -1;
    return o;
}
// The first refused draft of a sequence's rows r, by one wave: the products
// are exact in f64 (24 x 24 bits).
__device__ __forceinline__ int first_refused(const VerifyArgs &a, const SeqRows &r) {
    const int k = r.n - 1, lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < k; i0 += 64) {
        const int i = i0 + lane;
        bool ok = true;
        if (i < k) {
            const size_t row = (size_t)r.lo + i;
            const int x = a.tokens[row + 1];
            const double u = (double)a.u[row];
            ok = false;
            if ((unsigned)x < (unsigned)a.vocab) {
                const double q = a.q ? (double)a.q[row * a.q_row + x] : 1.0;
                ok = u * q < (double)a.p[row * a.p_row + x];
            }
        }
        const unsigned long long no = __ballot(!ok);
        if (no) return i0 + __builtin_ctzll(no);
    }
    return k;
}

// Weights of token t: after a refusal, and of p.
__device__ __forceinline__ double2 weights(const VerifyArgs &a, const Row &o, int t, float p, float q) {
    double w = (double)p;
    if (!o.ended) w = a.q ? (double)p - (double)q : t == o.x ? 0.0 : w;
    return make_double2(weight(w), weight((double)p));
}

// Sums of the chunks of one sequence's row, `run` of them a wave, which finds
// the row by itself (three round trips, so a wave takes several chunks where
// there are many; the next chunk is under way while one is summed). p and q
// are read once here, and the drawn token's chunk once more by
// verify_draw_kernel. No barrier. 64 sequences of 152064 tokens: 14 us, 5.5
// TB/s; one: 4 us.
__global__ __launch_bounds__(kVerTPB) void verify_sum_kernel(VerifyArgs a) {
    const int s = blockIdx.y, lane = threadIdx.x & 63;
    const int c0 = (int)(blockIdx.x * (kVerTPB / 64) + (threadIdx.x >> 6)) * a.run, c1 = min(a.chunks, c0 + a.run);
    const SeqRows r = seq_rows(a.b.row_start[s], a.b.row_start[s + 1], a.b.n_rows);
    if (r.n == 0 && c0 == 0 && lane == 0) a.heads[s] = make_int4(r.lo, 0, 0, 0);
    if (r.n == 0 || c0 >= c1) return;
    const Row o = row_at(a, r, first_refused(a, r));
    if (c0 == 0 && lane == 0) a.heads[s] = make_int4(r.lo, r.n, o.accepted, __float_as_int(a.u[r.lo + r.n - 1]));
    const float *p = a.p + o.row * a.p_row, *q = a.q && !o.ended ? a.q + o.row * a.q_row : p;
    f4u vp[2], vq[2];
    auto load = [&](int c) {  // tokens 256 j + 4 lane .. of the chunk
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int t = c * kVerChunk + 256 * j + 4 * lane;
            if (t + 4 <= a.vocab) {
                vp[j] = *(const f4u *)(p + t);
                vq[j] = *(const f4u *)(q + t);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    vp[j][e] = t + e < a.vocab ? p[t + e] : 0.0f;
                    vq[j][e] = t + e < a.vocab ? q[t + e] : 0.0f;
                }
            }
        }
    };
    load(c0);
    for (int c = c0; c < c1; c++) {
        f4u p2[2], q2[2];
#pragma unroll
        for (int j = 0; j < 2; j++) p2[j] = vp[j], q2[j] = vq[j];
        if (c + 1 < c1) load(c + 1);
        double x = 0.0, y = 0.0;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double2 w = weights(a, o, c * kVerChunk + 256 * j + 4 * lane + e, p2[j][e], q2[j][e]);
                x += w.x, y += w.y;
            }
        x = wave_sum_d(x);
        y = wave_sum_d(y);
        if (lane == 0) a.sums[(size_t)s * a.chunks + c] = make_double2(x, y);
    }
}

// Inclusive sum of v over the wave's lanes in their order (a fixed tree: rows of 16, then the rows before).
__device__ __forceinline__ double wave_scan_d(double v) {
    v += dpp_d<0x111>(v);       // row_shr:1
    v += dpp_d<0x112>(v);       // row_shr:2
    v += dpp_d<0x114>(v);       // row_shr:4
    v += dpp_d<0x118>(v);       // row_shr:8
    v += dpp_d<0x142, 0xA>(v);  // row_bcast:15 into rows 1, 3
    v += dpp_d<0x143, 0xC>(v);  // row_bcast:31 into rows 2, 3
    return v;
}

// Where a lane's run of weights passes the threshold: the first with weight whose sum exceeds it, or else the last
// with weight.
struct Passed {
    int at;       // -1: no weight
    double base;  // the sum before it
    bool over;
};
__device__ __forceinline__ void pass(Passed &o, double &run, int i, double w, double thr) {
    if (o.over || !(w > 0.0)) return;
    o.at = i;
    o.base = run;
    run += w;
    o.over = run > thr;
}
// The lane that holds the draw; -1: no weight in any.
__device__ __forceinline__ int drawing_lane(const Passed &o) {
    const unsigned long long over = __ballot(o.over), some = __ballot(o.at >= 0);
    return over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
}

// One wave a sequence: the chunk that the threshold falls in, then the token
// in it. Rounded running sums need not ascend where a weight is zero or at the
// joints of the tree, so a token needs weight of its own to be drawn, and
// where no sum exceeds the threshold the last one with weight is it. The
// time is round trips (a lane's chunks' sums, one after another; the refused
// token; its chunk of p and q): a wave needs no barriers between them (64
// sequences of 152064 tokens: 4.5 us; a workgroup of four waves with its scans
// in LDS: 15).
constexpr int kKeep = 8;  // chunks' sums of a lane read once, and kept (in scratch memory): a vocabulary of 2^18
__global__ __launch_bounds__(64) void verify_draw_kernel(VerifyArgs a) {
    const int s = blockIdx.x, lane = threadIdx.x;
    // every lane a run of chunks
    const double2 *sums = a.sums + (size_t)s * a.chunks;
    const int per = (a.chunks + 63) / 64, c0 = min(a.chunks, lane * per), c1 = min(a.chunks, c0 + per);
    double2 keep[kKeep], t = make_double2(0.0, 0.0);
#pragma unroll
    for (int i = 0; i < kKeep; i++) keep[i] = c0 + i < c1 ? sums[c0 + i] : make_double2(0.0, 0.0);
    const int4 head = a.heads[s];
#pragma unroll
    for (int i = 0; i < kKeep; i++) t.x += keep[i].x, t.y += keep[i].y;  // a sequence without rows: of anything, not used
    for (int c = c0 + kKeep; c < c1; c++) t.x += sums[c].x, t.y += sums[c].y;
    const SeqRows r{head.x, head.y};
    if (lane == 0) a.accepted[s] = head.z;
    if (r.n == 0) {
        if (lane == 0) a.next[s] = -1;
        return;
    }
    const Row o = row_at(a, r, head.z);
    double inc = wave_scan_d(t.x), total = __shfl(inc, 63);
    const bool plain = !(total > 0.0);  // no weight after the refusal: p itself
    if (plain) inc = wave_scan_d(t.y), total = __shfl(inc, 63);
    double u = (double)__int_as_float(head.w);
    u = u >= 0.0 ? u : u < 0.0 ? 0.0 : 1.0;  // NaN as 1
    const double thr = u >= 1.0 ? (double)INFINITY : u * total;
    Passed chunk{-1, 0.0, false};
    double run = inc - (plain ? t.y : t.x);
#pragma unroll
    for (int i = 0; i < kKeep; i++) pass(chunk, run, c0 + i, plain ? keep[i].y : keep[i].x, thr);
    for (int c = c0 + kKeep; c < c1; c++) pass(chunk, run, c, plain ? sums[c].y : sums[c].x, thr);
    int from = drawing_lane(chunk);
    if (from < 0) {
        if (lane == 0) a.next[s] = -1;
        return;
    }
    // the chunk's tokens: eight neighbours a lane
    const float *p = a.p + o.row * a.p_row, *q = a.q && !o.ended ? a.q + o.row * a.q_row : p;
    const int x0 = __shfl(chunk.at, from) * kVerChunk + 8 * lane;
    float vp[8], vq[8];
    if (x0 + 8 <= a.vocab) {
        load_row<8>(vp, p + x0);
        load_row<8>(vq, q + x0);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            vp[e] = x0 + e < a.vocab ? p[x0 + e] : 0.0f;
            vq[e] = x0 + e < a.vocab ? q[x0 + e] : 0.0f;
        }
    }
    double w[8], mine = 0.0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const double2 v = weights(a, o, x0 + e, vp[e], vq[e]);
        w[e] = plain ? v.y : v.x;
        mine += w[e];
    }
    Passed token{-1, 0.0, false};
    run = __shfl(chunk.base, from) + (wave_scan_d(mine) - mine);
#pragma unroll
    for (int e = 0; e < 8; e++) pass(token, run, x0 + e, w[e], thr);
    from = drawing_lane(token);
    const int drawn = __shfl(token.at, max(from, 0));
    if (lane == 0) a.next[s] = drawn;
}

}  // namespace

hipError_t launch_kv_append(const PagesView &kv, const BatchView &b, const uq_head_rows &h, hipStream_t s) {
    if (b.n_rows == 0 || b.n_seqs == 0) return hipSuccess;
    const int units = (h.d_q ? (int)h.n_head : 0) + (h.d_k ? 2 * kv.n_head_kv : 0);
    if (units == 0) return hipSuccess;
    const int most = (units + kAppTPB / 64 - 1) / (kAppTPB / 64);
    int split = (512 + b.n_rows - 1) / b.n_rows;
    split = split < 1 ? 1 : split > most ? most : split;
    const AppendArgs a{h, kv, b};
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)b.n_rows, (unsigned)split), dim3(kAppTPB), 0, s, a);
        return hipGetLastError();
    };
    switch (kv.head_dim) {
    case 64: return kv.f16 ? go(kv_append_kernel<64, true>) : go(kv_append_kernel<64, false>);
    case 128: return kv.f16 ? go(kv_append_kernel<128, true>) : go(kv_append_kernel<128, false>);
    case 256: return kv.f16 ? go(kv_append_kernel<256, true>) : go(kv_append_kernel<256, false>);
    case 512: return kv.f16 ? go(kv_append_kernel<512, true>) : go(kv_append_kernel<512, false>);
    }
    return hipErrorInvalidValue;
}

size_t draft_verify_ws_bytes(int n_seqs, int vocab) {
    return (size_t)n_seqs * ((((size_t)vocab + kVerChunk - 1) / kVerChunk) * sizeof(double2) + sizeof(int4));
}

hipError_t launch_draft_verify(int32_t *accepted, int32_t *next, const float *p, size_t p_row, const float *q,
                               size_t q_row, const int32_t *tokens, const float *u, const BatchView &b, int vocab,
                               void *ws, hipStream_t s) {
    if (b.n_seqs == 0) return hipSuccess;
    const int chunks = (vocab + kVerChunk - 1) / kVerChunk;
    // one chunk a wave up to two rounds of 8 workgroups a CU, then up to 8
    const long long waves = (long long)chunks * b.n_seqs;
    const int run = (int)std::min(8LL, std::max(1LL, waves / (2 * 8 * 256 * (kVerTPB / 64))));
    const VerifyArgs a{accepted, next, p, q, p_row, q_row, tokens, u, b, vocab, chunks, run,
                       (double2 *)ws, (int4 *)((double2 *)ws + (size_t)b.n_seqs * chunks)};
    const int per = kVerTPB / 64 * run;
    hipLaunchKernelGGL(verify_sum_kernel, dim3((unsigned)((chunks + per - 1) / per), (unsigned)b.n_seqs), dim3(kVerTPB), 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(verify_draw_kernel, dim3((unsigned)b.n_seqs), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace uq
