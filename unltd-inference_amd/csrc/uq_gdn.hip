// Batched serving of GatedDeltaNet layers: the convolution of a batch's rows
// with its windows, norms and gates (uq_gdn_conv_d), and the gated delta rule
// over its states (uq_gdn_rule_d).
#include <algorithm>
#include <climits>
#include <type_traits>


#include "uq_device.h"
#include "uq_internal.h"
#include "uq_mfma.h"
#include "uq_serve_internal.h"

namespace uq {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any float

// Sum over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float rows16_sum(float v) {
    auto two = [&](const auto &r) { return __uint_as_float(r[0]) + __uint_as_float(r[1]); };
    v = two(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return two(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}
// Sum over LANES neighbouring lanes (16 or 32), in all of them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp_f<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp_f<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp_f<0x141>(v);  // row_half_mirror
    v += dpp_f<0x140>(v);  // row_mirror
    if constexpr (LANES == 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}
// Inclusive sum over the wave's lanes.
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ int dpp_i(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROW_MASK, 0xF, true);
}
__device__ __forceinline__ int wave_scan_i(int v) {
    v += dpp_i<0x111>(v);       // row_shr:1
    v += dpp_i<0x112>(v);       // row_shr:2
    v += dpp_i<0x114>(v);       // row_shr:4
    v += dpp_i<0x118>(v);       // row_shr:8
    v += dpp_i<0x142, 0xA>(v);  // row_bcast:15 into rows 1, 3
    v += dpp_i<0x143, 0xC>(v);  // row_bcast:31 into rows 2, 3
    return v;
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// x / (1 + e^-x), by the hardware's power of 2 and reciprocal (1 ulp each). e^-x is 2^t c, t = -x log2 e rounded and c
// what that and the constant's own rounding leave: far below 0, where t is large, 2^t alone would be off by |t| 2^-24. Where
// the product overflows 2^t is 0 or infinite, and c need only be a number.
__device__ __forceinline__ float silu(float x) {
    const float t = -1.44269502f * x;
    const float c = fminf(fmaf(fmaf(-1.44269502f, x, -t), 0.693147181f, fmaf(x, -1.33497589e-8f, 1.0f)), 2.0f);
    return x * __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(t), c, 1.0f));
}

// Sequences of at least `least` rows are cut into tiles of T rows, numbered
// through; every wave finds its tile's by itself, 256 sequences at a time.
struct Tile {
    int seq, lo, n, first;  // -1: there is none; the sequence's rows, and the tile's first row among them
};
template <int T>
__device__ __forceinline__ Tile find_tile(const BatchView &b, int tile, int least) {
    const int lane = threadIdx.x & 63;
    int run = 0;
    for (int c = 0; c < b.n_seqs; c += 256) {
        const int i0 = c + 4 * lane;
        int start[5], count[4], mine = 0;
#pragma unroll
        for (int e = 0; e < 5; e++) start[e] = b.row_start[min(i0 + e, b.n_seqs)];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const SeqRows r = seq_rows(start[e], start[e + 1], b.n_rows);
            count[e] = i0 + e < b.n_seqs && r.n >= least ? (r.n + T - 1) / T : 0;
            mine += count[e];
        }
        const int upto = wave_scan_i(mine), all = lane_of(upto, 63);
        if (tile < run + all) {
            int at = run + upto - mine;
            Tile t{-1, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (tile >= at && tile < at + count[e]) {
                    const SeqRows r = seq_rows(start[e], start[e + 1], b.n_rows);
                    t = Tile{i0 + e, r.lo, r.n, (tile - at) * T};
                }
                at += count[e];
            }
            const unsigned long long here = __ballot(t.seq >= 0);
            if (!here) return t;
            const int from = __builtin_ctzll(here);
            return Tile{lane_of(t.seq, from), lane_of(t.lo, from), lane_of(t.n, from), lane_of(t.first, from)};
        }
        run += all;
    }
    return Tile{-1, 0, 0, 0};
}

// Sequences of at least `least` rows that go by chunks, numbered through: l of
// them lie before this one. Its chunks' slots in the workspace begin at
// lo / 64 + l, so that none share one and none needs the others' counts.
struct Long {
    int seq, lo, n, slot;  // seq -1: there is none
};
constexpr int kChunk = 64;
UQ_HD int chunk_slot(int lo, int l) { return lo / kChunk + l; }
// SLOT: the sequence that holds slot `want`; else the one that `want` lie before.
template <bool SLOT>
__device__ __forceinline__ Long find_long(const BatchView &b, int want, int least) {
    const int lane = threadIdx.x & 63;
    int run = 0;
    for (int c = 0; c < b.n_seqs; c += 256) {
        const int i0 = c + 4 * lane;
        int start[5], mine = 0;
#pragma unroll
        for (int e = 0; e < 5; e++) start[e] = b.row_start[min(i0 + e, b.n_seqs)];
        SeqRows r[4];
        bool is[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            r[e] = seq_rows(start[e], start[e + 1], b.n_rows);
            is[e] = i0 + e < b.n_seqs && r[e].n >= least;
            mine += is[e];
        }
        const int upto = wave_scan_i(mine);
        int l = run + upto - mine;
        Long t{-1, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int slot = chunk_slot(r[e].lo, l);
            if (is[e] && t.seq < 0 && (SLOT ? want >= slot && want < slot + (r[e].n + kChunk - 1) / kChunk : l == want))
                t = Long{i0 + e, r[e].lo, r[e].n, slot};
            l += is[e];
        }
        const unsigned long long here = __ballot(t.seq >= 0);
        if (here) {
            const int from = __builtin_ctzll(here);
            return Long{lane_of(t.seq, from), lane_of(t.lo, from), lane_of(t.n, from), lane_of(t.slot, from)};
        }
        run += lane_of(upto, 63);
    }
    return Long{-1, 0, 0, 0};
}

// ---- the convolution --------------------------------------------------------

constexpr int kConvTPB = 256;
constexpr int kConvRows = 16;  // of a tile: more than the taps before a row, so that only a sequence's first tile reads the window

struct ConvArgs {
    StatesView st;
    BatchView b;
    uq_gdn_rows r;
    int groups;  // of 256 channels
};

// A wave takes 256 channels (four neighbours a lane) of a tile's rows, the
// taps and the last inputs in registers; one more takes the tile's gates. The
// wave of a sequence's first tile also takes the window on, whose old values
// it alone reads. Memory bounds it: 6010 rows of 8192 channels 84 us, 4.7 TB/s;
// other taps than 4 hold nine in registers, three waves a SIMD and not five: 87 us with 3 of them, 150 with 8.
template <int CK>  // taps, 0: any up to 9
__global__ __launch_bounds__(kConvTPB) void gdn_conv_kernel(ConvArgs a) {
    constexpr int MT = CK ? CK : 9, H = MT - 1, STEP = 4;
    const int taps = CK ? CK : a.st.taps, skip = MT - taps;  // places before the first tap
    const unsigned per = (unsigned)(a.groups + kConvTPB / 64) / (kConvTPB / 64), i = blockIdx.y * gridDim.x + blockIdx.x, tile = i / per;
    const int lane = threadIdx.x & 63, group = uniform((int)(i - tile * per) * (kConvTPB / 64) + (int)(threadIdx.x >> 6));
    if (group > a.groups) return;
    const Tile t = find_tile<kConvRows>(a.b, (int)tile, 1);
    if (t.seq < 0) return;
    const int nn = min(kConvRows, t.n - t.first);
    const size_t row0 = (size_t)t.lo + t.first;
    if (group == a.groups) {
        if (!a.r.d_alpha) return;
        for (int i = lane; i < nn * a.st.nv; i += 64) {
            const int r = i / a.st.nv, h = i - r * a.st.nv;
            const size_t in = (row0 + r) * a.r.raw_row + h, o = (row0 + r) * a.st.nv + h;
            const float x = a.r.d_alpha[in] + a.r.d_dt_bias[h];
            a.r.d_beta[o] = __fdiv_rn(1.0f, 1.0f + expf(-a.r.d_beta_raw[in]));
            a.r.d_gate[o] = (fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x)))) * a.r.d_a[h];
        }
        return;
    }
    const int channels = a.st.channels, c = group * 256 + 4 * lane;
    const bool in = c < channels;  // whole heads: channels are a multiple of 64
    const int cc = in ? c : 0;
    float tap[4][MT];
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
        for (int k = 0; k < MT; k++) tap[e][k] = k >= skip ? a.r.d_conv1d[(size_t)(cc + e) * taps + k - skip] : 0.0f;
    const float *qkv = a.r.d_qkv + cc;
    auto at_row = [&](size_t row) { return (f4) * (const f4u *)(qkv + row * a.r.qkv_row); };
    // old[j]: the input H - j rows before the tile's first
    f4 old[H];
    const int from = a.st.from[t.seq], to = a.st.to[t.seq];
    const bool has = (unsigned)from < (unsigned)a.st.n_slots;
#pragma unroll
    for (int j = 0; j < H; j++) {
        old[j] = f4{0.f, 0.f, 0.f, 0.f};
        if (j < skip) continue;
        if (t.first > 0)
            old[j] = at_row(row0 - H + j);
        else if (has)
            old[j] = *(const f4u *)(a.st.conv + ((size_t)from * taps + j - skip) * channels + cc);
    }
    if (t.first == 0 && (unsigned)to < (unsigned)a.st.n_slots && in) {
        // the last taps - 1 of [the window; the rows]
#pragma unroll
        for (int j = 0; j < H; j++) {
            if (j < skip) continue;
            const int p = t.n + j;
            f4 w;
            if (p >= H) {
                w = at_row((size_t)t.lo + p - H);
            } else {
                w = old[0];
#pragma unroll
                for (int k = 1; k < H; k++)
                    if (k == p) w = old[k];
            }
            *(f4u *)(a.st.conv + ((size_t)to * taps + j - skip) * channels + c) = w;
        }
    }
    const bool norm = c < 2 * a.st.nqk * a.st.hd;
    f4 x[H + STEP];  // the last inputs, then the step's rows
#pragma unroll
    for (int j = 0; j < H; j++) x[j] = old[j];
    f4 next[STEP];
#pragma unroll
    for (int u = 0; u < STEP; u++) next[u] = at_row(row0 + min(u, nn - 1));
    for (int r = 0; r < nn; r += STEP) {
#pragma unroll
        for (int u = 0; u < STEP; u++) x[H + u] = next[u];
#pragma unroll
        for (int u = 0; u < STEP; u++) next[u] = at_row(row0 + min(r + STEP + u, nn - 1));
#pragma unroll
        for (int u = 0; u < STEP; u++) {
            f4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float s = 0.0f;
#pragma unroll
                for (int k = 0; k < MT; k++)
                    if (k >= skip) s = fmaf(x[u + k][e], tap[e][k], s);
                y[e] = silu(s);
            }
            float sq = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) sq = fmaf(y[e], y[e], sq);
            sq = a.st.hd == 64 ? lanes_sum<16>(sq) : lanes_sum<32>(sq);
            const float root = sqrtf(sq), by = norm ? 1.0f / (root < a.r.eps ? a.r.eps : root) : 1.0f;  // a NaN stays one
            if (in && r + u < nn) *(f4u *)(a.r.d_out + (row0 + r + u) * channels + c) = y * by;
        }
#pragma unroll
        for (int j = 0; j < H; j++) x[j] = x[j + STEP];
    }
}

// ---- the delta rule, row by row -----------------------------------------------

struct RuleArgs {
    float *out;
    StatesView st;
    BatchView b;
    uq_gdn_heads h;
    int chunked;      // sequences of at least so many rows go by chunks
    int longs, slots; // of those at most, and of their chunks
    int parts;        // workgroups of a chunk and key head
    int singles;      // workgroups of half the sequences that go row by row, a multiple of 8
    uint8_t *ws;      // [slots][nv] ChunkWs
    uint8_t *kq;      // [slots][nqk] keys, then queries
};

// The epilogue of a head's row: rms norm and gate, lane l its values
// (HD / 64) l and on; E of them.
template <int HD>
__device__ __forceinline__ void finish_row(const RuleArgs &a, size_t row, int head, float (&v)[HD / 64]) {
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63;
    if (a.h.d_norm) {
        float sq = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) sq = fmaf(v[e], v[e], sq);
        const float by = 1.0f / sqrtf(wave_sum(sq) / (float)HD + a.h.eps);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = v[e] * by * a.h.d_norm[E * lane + e];
    }
    if (a.h.d_z) {
        const float *z = a.h.d_z + row * a.h.z_row + (size_t)head * HD + E * lane;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] *= silu(z[e]);
    }
    float *o = a.out + (row * a.st.nv + head) * HD + E * lane;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = v[e];
}

// One workgroup a sequence and value head, a wave 32 of its columns: lane l
// has columns 4 (l % 8) .. + 3 of rows (HD / 8) (l / 8) and on. A column's
// two products, with k and with q, are formed of the state before the row,
//     S^T k = e^g (S_0^T k),   S^T q = e^g (S_0^T q) + (q.k) d,
// so that their sums over the lanes run side by side, and no wave waits for
// another but for the norm. The state passes through registers once, which
// bounds it for few rows: 64 sequences of one row, 32 heads of 128, 58 us or
// 4.7 TB/s. Each further row of one sequence takes 1.1 us.
constexpr int kRowBuf = 16;  // rows whose results wait for the norm
template <int HD>
__device__ __forceinline__ void rule_rows(const RuleArgs &a, int seq, int head, float (*buf)[HD]) {
    constexpr int R = HD / 8, NW = HD / 32;
    const int hq = head % a.st.nqk;
    const SeqRows rows = seq_rows(a.b.row_start[seq], a.b.row_start[seq + 1], a.b.n_rows);
    if (rows.n == 0 || rows.n >= a.chunked) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i0 = (lane >> 3) * R, j0 = 32 * wave + 4 * (lane & 7);
    const int from = a.st.from[seq], to = a.st.to[seq];
    const bool finish = a.h.d_norm || a.h.d_z;
    f4 S[R];
    if ((unsigned)from < (unsigned)a.st.n_slots) {
        const float *s = a.st.state + (((size_t)from * a.st.nv + head) * HD + i0) * HD + j0;
#pragma unroll
        for (int r = 0; r < R; r++) S[r] = *(const f4 *)(s + (size_t)r * HD);
    } else {
#pragma unroll
        for (int r = 0; r < R; r++) S[r] = f4{0.f, 0.f, 0.f, 0.f};
    }
    struct Row {
        f4 k[R / 4], v;
        float g, b;
    };
    f4 q[R / 4];
    auto load_q = [&](int i) {
        const float *p = a.h.d_q + ((size_t)rows.lo + i) * a.h.q_row + (size_t)hq * HD + i0;
#pragma unroll
        for (int u = 0; u < R / 4; u++) q[u] = *(const f4u *)(p + 4 * u);
    };
    auto load = [&](Row &x, int i) {
        const size_t row = (size_t)rows.lo + i;
        const float *k = a.h.d_k + row * a.h.k_row + (size_t)hq * HD + i0;
#pragma unroll
        for (int u = 0; u < R / 4; u++) x.k[u] = *(const f4u *)(k + 4 * u);
        x.v = *(const f4u *)(a.h.d_v + row * a.h.v_row + (size_t)head * HD + j0);
        x.g = a.h.d_gate[row * a.st.nv + head];
        x.b = a.h.d_beta[row * a.st.nv + head];
    };
    Row x, next;
    load(x, 0), load_q(0);
    for (int i = 0; i < rows.n; i++) {
        const int then = min(i + 1, rows.n - 1);
        load(next, then);
        const float eg = expf(x.g);
        f4 sk{0.f, 0.f, 0.f, 0.f}, sq = sk, d, o;
        float qk = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float k = x.k[r / 4][r % 4], qr = q[r / 4][r % 4];
            qk = fmaf(qr, k, qk);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                sk[e] = fmaf(k, S[r][e], sk[e]);
                sq[e] = fmaf(qr, S[r][e], sq[e]);
            }
        }
        load_q(then);
        auto over_rows = [](float v) { return rows16_sum(v + dpp_f<0x128>(v)); };  // row_ror:8: lanes l, l ^ 8, l ^ 16, ..
        qk = over_rows(qk);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            d[e] = x.b * (x.v[e] - eg * over_rows(sk[e]));
            o[e] = a.h.scale * fmaf(qk, d[e], eg * over_rows(sq[e]));
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int e = 0; e < 4; e++) S[r][e] = fmaf(x.k[r / 4][r % 4], d[e], eg * S[r][e]);
        if (!finish) {
            if (lane < 8) *(f4u *)(a.out + (((size_t)rows.lo + i) * a.st.nv + head) * HD + j0) = o;
        } else {
            const int at = i % kRowBuf;
            if (lane < 8) *(f4 *)&buf[at][j0] = o;
            if (at == kRowBuf - 1 || i == rows.n - 1) {
                __syncthreads();
                for (int r = wave; r <= at; r += NW) {
                    float v[HD / 64];
#pragma unroll
                    for (int e = 0; e < HD / 64; e++) v[e] = buf[r][HD / 64 * lane + e];
                    finish_row<HD>(a, (size_t)rows.lo + i - at + r, head, v);
                }
                __syncthreads();
            }
        }
        x = next;
    }
    if ((unsigned)to < (unsigned)a.st.n_slots) {
        float *s = a.st.state + (((size_t)to * a.st.nv + head) * HD + i0) * HD + j0;
#pragma unroll
        for (int r = 0; r < R; r++) *(f4 *)(s + (size_t)r * HD) = S[r];
    }
}

// Workgroup i of the even (odd: 1) sequences' in a kernel of 256 threads. Both kernels of the chunks take half: each
// leaves compute units free where chunks are few, and the states' way from memory and back is what these need.
template <int HD>
__device__ __forceinline__ void rule_rows_of(const RuleArgs &a, unsigned i, int odd, float (*buf)[HD]) {
    const unsigned seq = 2 * (i / a.st.nv) + odd;
    if (threadIdx.x < 2 * HD && seq < (unsigned)a.b.n_seqs) rule_rows<HD>(a, (int)seq, (int)(i % a.st.nv), buf);  // whole waves
}
template <int HD>
__global__ __launch_bounds__(2 * HD) void gdn_rows_kernel(RuleArgs a) {
    __shared__ __align__(16) float buf[kRowBuf][HD];
    rule_rows<HD>(a, (int)blockIdx.y, (int)blockIdx.x, buf);
}

// ---- the delta rule by chunks ---------------------------------------------------
//
// Of 64 rows with the state S before them and G_i the gates' sum up to row i,
// the corrections U solve
//     (I + A) U = diag(beta) (V - diag(e^G) K S),  A[i][j] = beta_i e^(G_i - G_j) k_i.k_j  (j < i),
// and  out = scale (diag(e^G) Q S + P U),          P[i][j] = e^(G_i - G_j) q_i.k_j         (j <= i),
//      S <- e^G_63 S + K^T (diag(e^(G_63 - G)) U).
// What does not depend on S, T = (I + A)^-1 diag(beta) and P, is formed for all
// chunks at once (gdn_prep_kernel); gdn_chunks_kernel then takes a sequence's
// chunks one after another, by columns of a head's state, as nothing of
// another column enters one; gdn_finish_kernel applies norm and gate. 509 rows
// of 32 heads take 11.5, 24 and 7.5 us, three prompts of 5241 rows 60, 146 and 45.
//
// The products run on the f16 matrix cores with two terms of each operand,
// h + l = x 2^s within 2^-22 of it: s brings the largest value of a row (left
// operands) or column (right ones), or a bound on it, to 2^13 .. 2^14, so that
// values down to 2^-16 of it keep 22 bits and what is lost below is 2^-39 of
// it. The products h h, h l and l h are exact and summed in f32; l l is left
// out, 2^-22 of the product at most. The three take 48 clocks for 16 x 16 x 32,
// where the f32 matrix cores take 256: with those 509 rows of 32 heads took 81
// us, and 70 when the second kernel was put on the others.
//
// A 16x16x32 product's depth is summed over lane / 16 and 8 values a lane, of
// tiles 2 p and 2 p + 1: values 4 (lane / 16) .. + 3 of each. A result's rows
// lie so over the lanes, so that a pair of results is a right operand as it is.
//
// A row with a key, beta or gate that is not finite leaves the products
// (first: the first such row), and so do rows of a column from its first
// correction on that is not: 0 times NaN would carry it to earlier rows.
// Their results are set to NaN.

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((vector_size(16)));

// Left operands in the workspace, pieces of 1 KB: [tile of 16 rows][pair of tiles in depth][h, l][64 lanes][8 f16].
// The keys are read by columns as well (read_columns), 4 rows of 4 pieces of 4 columns at a time: those lie in
// different banks when a piece's rows are turned by 4 for each group of columns.
__device__ __forceinline__ int place(int m, int g) { return 16 * g + ((m + 4 * g) & 15); }
struct ChunkWs {  // of a chunk and value head, in bytes
    static constexpr int T = 0, P = 12 * 1024, vec = 24 * 1024;  // 6 pieces of h and l each: tile_piece
    // vec, floats: factors of the rows of K S (e^G with the keys' scale), of T's product for the state (e^(G_63 - G) with
    // the keys' scale and T's), of Q S, and of T's and P's rows; then e^G_63, the first row that is left out and the
    // largest of gx
    static constexpr int gx = 0, gg = 64, gq = 128, gt = 192, gp = 256, whole = 320, first = 321, top = 322;
    static constexpr int bytes = 26 * 1024;
};
__device__ __forceinline__ int tile_piece(int tile, int pair) { return tile < 2 ? tile : 2 * tile - 2 + pair; }
constexpr int kq_bytes(int hd) { return kChunk * hd * 4; }  // of the keys or queries of a chunk

constexpr float kLeastGate = -1000.0f;  // e^-1000 of any f32 is 0: gates below it are taken as it, so that differences are numbers

__device__ __forceinline__ bool finite32(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }
__device__ __forceinline__ uint32_t size_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }  // NaN above infinity
template <int N>
__device__ __forceinline__ uint32_t size_bits(const f4 (&v)[N]) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) r = max(r, size_bits(v[i][e]));
    return r;
}
// Over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ uint32_t rows16_max(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
    v = max(v, dpp_u<0xB1>(v));
    v = max(v, dpp_u<0x4E>(v));
    v = max(v, dpp_u<0x141>(v));
    return rows16_max(max(v, dpp_u<0x140>(v)));
}
// The exponent ex that brings values of at most this size below 2^14: x 2^(14 - ex). Sizes below 2^-100 as it, 0 among
// them, whose own exponent is 0, as if a column of zeros (a new sequence's state) held values near 1.
__device__ __forceinline__ int scale_of(uint32_t bits) {
    const int ex = __builtin_amdgcn_frexp_expf(__uint_as_float(bits));
    return bits ? max(-100, ex) : -100;
}
__device__ __forceinline__ float scale_up(int ex) { return ldexpf(1.0f, 14 - ex); }
__device__ __forceinline__ float scale_down(int ex) { return ldexpf(1.0f, ex - 14); }
// The same of a 2^i + b 2^j, a bound that may lie beyond f32's range where what it bounds does not, formed in 64 bits. At
// 2^141 scale_down ends, far above what f32 holds.
__device__ __forceinline__ int scale_of_sum(double a, int i, float b, int j) {
    const double sum = ldexp(a, i) + ldexp((double)b, j) + 0x1p-200;
    return min(141, max(-100, __builtin_amdgcn_frexp_exp(sum)));
}
// The two terms of a pair of tiles, each rounded to the nearest. A pair of conversions, back, a difference: three
// instructions a value of 4 clocks each, where a product and sum of mixed precision for each term takes 8 each.
__device__ __forceinline__ void two_terms(const f4 &a, const f4 &b, h8 &h, h8 &l) {
    typedef float f8 __attribute__((ext_vector_type(8)));
    const f8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    h = __builtin_convertvector(v, h8);
    l = __builtin_convertvector(v - __builtin_convertvector(h, f8), h8);
}
__device__ __forceinline__ void two_terms(const f4 &a, const f4 &b, float s, h8 &h, h8 &l) { two_terms(a * s, b * s, h, l); }
// The largest size of N tiles' values, a NaN's above all. As floats' order is that of their bits, for those above zero as
// signed, for those below as unsigned: an instruction a value, where floats, made canonical first, take one and a half.
template <int N>
__device__ __forceinline__ float top_of(const f4 (&v)[N]) {
    int above[2] = {0, 0};
    uint32_t below[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2 * N; i++) {
        const uint32_t x = __float_as_uint(v[i / 2][i % 2 * 2]), y = __float_as_uint(v[i / 2][i % 2 * 2 + 1]);
        above[i % 2] = max(above[i % 2], max((int)x, (int)y));
        below[i % 2] = max(below[i % 2], max(x, y));
    }
    return __uint_as_float(max((uint32_t)max(above[0], above[1]), max(below[0], below[1]) & 0x7FFFFFFFu));
}
// Nothing that depends on v moves up across this point.
template <int N>
__device__ __forceinline__ void hold(f4 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) __asm__ volatile("" : "+v"(v[i]));
}
__device__ __forceinline__ f4 mfma4(const f4 &a, const f4 &b, f4 c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f4 mfma_h(const h8 &a, const h8 &b, const f4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Column J of -A, a lane's row of it in the quarter's lane J, times the inverse's row J.
template <int J>
__device__ __forceinline__ void eliminate(const f4 &a, f4 &v) {
    const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[J % 4]), __float_as_uint(v[J % 4]), false, false);
    const unsigned h = half[J / 8];
    const auto row = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    const float x = __uint_as_float(row[J / 4 % 2]);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = fmaf(dpp_f<0x150 + J>(a[e]), x, v[e]);  // row_newbcast:J
    if constexpr (J < 14) eliminate<J + 1>(a, v);
}
constexpr int kPrepTPB = 256;
template <int HD>
struct PrepLds {
    static constexpr int planes = kq_bytes(HD), tiles = 2 * 10 * 1024;  // the keys; A below the diagonal (6) and the inverses (4), twice
    __align__(16) uint8_t space[planes > tiles ? planes : tiles];
    double G[4][kChunk];  // of the wave
    float beta[4][kChunk];
    int ex_k[kChunk], ex_q[kChunk], bad[4];
};
// T and P of a chunk, and the keys and queries in two terms, a workgroup the
// value heads of one query and key head. Wave w has rows 16 w .. + 15 of both;
// all see the keys' pieces in the LDS. It takes tiles (r, w), r >= w, of K K^T
// and (r, w), r <= w, of K Q^T, five for each wave, and keeps them for the
// heads. Every result lies as the operand that it is next: lane (m, g) has
// values 4 g .. + 3 of column m, which is a row's piece of the transposed. So
// tile (i, j) of A is the left operand A_ij^T, K Q^T has P's rows, and T's row
// of tiles i is formed from the diagonal back,
//     T_ij^T = -T_jj^T sum over j < k <= i of A_kj^T T_ik^T,
// by wave i from A and the diagonal's inverses alone. What it reads and writes
// bounds it for many chunks, at 4 TB/s.
template <int HD>
__device__ __forceinline__ void rule_prep(const RuleArgs &a, int slot, int hq, int part, PrepLds<HD> &l) {
    constexpr int KP = HD / 32;
    const Long s = find_long<true>(a.b, slot, a.chunked);
    if (s.seq < 0) return;
    const int c0 = (slot - s.slot) * kChunk, n = min(kChunk, s.n - c0);
    const size_t row0 = (size_t)s.lo + c0;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6)), m = lane & 15, g = lane >> 4, mine = 16 * wave + m;
    const float *gates = a.h.d_gate + (row0 + min(lane, n - 1)) * a.st.nv, *betas = a.h.d_beta + (row0 + min(lane, n - 1)) * a.st.nv;
    const int step = a.parts * a.st.nqk;
    int head = hq + part * a.st.nqk;
    float gate = gates[head], bt = betas[head];
    int exk, exq;  // of the wave's rows
    h8 kh[KP], kl[KP], qh[KP], ql[KP];
    {
        const size_t row = row0 + min(mine, n - 1);
        const float *pk = a.h.d_k + row * a.h.k_row + (size_t)hq * HD + 4 * g, *pq = a.h.d_q + row * a.h.q_row + (size_t)hq * HD + 4 * g;
        f4 k[2 * KP], q[2 * KP];
#pragma unroll
        for (int c = 0; c < 2 * KP; c++) k[c] = *(const f4u *)(pk + 16 * c);
#pragma unroll
        for (int c = 0; c < 2 * KP; c++) q[c] = *(const f4u *)(pq + 16 * c);
        const uint32_t top_k = rows16_max(size_bits(k)), top_q = rows16_max(size_bits(q));
        __asm__ volatile("" : "+v"(gate), "+v"(bt));  // asked for before the stores below, behind which they would wait
        const unsigned long long no = __ballot(top_k >= 0x7F800000u);  // rows with a key that is not finite
        exk = scale_of(top_k), exq = scale_of(top_q);
        if (g == 0) l.ex_k[mine] = exk, l.ex_q[mine] = exq;
        if (lane == 0) l.bad[wave] = (int)(no & 0xFFFF);
        h8 *to = (h8 *)(a.kq + ((size_t)slot * a.st.nqk + hq) * 2 * kq_bytes(HD)) + wave * KP * 128 + place(m, g);
        h8 *lk = (h8 *)l.space + wave * KP * 128 + place(m, g);
#pragma unroll
        for (int p = 0; p < KP; p++) {
            two_terms(k[2 * p], k[2 * p + 1], scale_up(exk), kh[p], kl[p]);
            two_terms(q[2 * p], q[2 * p + 1], scale_up(exq), qh[p], ql[p]);
            lk[p * 128] = kh[p];
            lk[p * 128 + 64] = kl[p];
        }
        if (part == 0) {
#pragma unroll
            for (int p = 0; p < KP; p++) {
                to[p * 128] = kh[p];
                to[p * 128 + 64] = kl[p];
                to[kq_bytes(HD) / 16 + p * 128] = qh[p];
                to[kq_bytes(HD) / 16 + p * 128 + 64] = ql[p];
            }
        }
    }
    __syncthreads();
    const f4 zero{0.f, 0.f, 0.f, 0.f};
    f4 dk[4], dq[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        f4 k0 = zero, k1 = zero, q0 = zero, q1 = zero;
        const h8 *x = (const h8 *)l.space + r * KP * 128 + place(m, g);
#pragma unroll
        for (int p = 0; p < KP; p++) {
            const h8 xh = x[p * 128], xl = x[p * 128 + 64];
            if (r >= wave) {
                k0 = mfma_h(xh, kh[p], k0);
                k1 = mfma_h(xh, kl[p], k1);
                k1 = mfma_h(xl, kh[p], k1);
            }
            if (r <= wave) {
                q0 = mfma_h(xh, qh[p], q0);
                q1 = mfma_h(xh, ql[p], q1);
                q1 = mfma_h(xl, qh[p], q1);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int ex = l.ex_k[16 * r + 4 * g + e] - 28;
            dk[r][e] = ldexpf(k0[e] + k1[e], ex + exk);
            dq[r][e] = a.h.scale * ldexpf(q0[e] + q1[e], ex + exq);
        }
    }
    const unsigned long long bad_k = (unsigned long long)(uint32_t)(l.bad[0] | l.bad[1] << 16) | (unsigned long long)(uint32_t)(l.bad[2] | l.bad[3] << 16) << 32;
    const float back_k = scale_down(l.ex_k[lane]), back_q = a.h.scale * scale_down(l.ex_q[lane]);
    __syncthreads();  // the keys are read
    double *const G = l.G[wave];
    float *const beta = l.beta[wave];
    f4 *tiles = (f4 *)l.space + lane;  // tile (i, j) of A at i (i - 1) / 2 + j, the inverse of (i, i) at 6 + i
    for (int turn = 0; head < a.st.nv; head += step, turn ^= 1) {
        uint8_t *ws = a.ws + ((size_t)slot * a.st.nv + head) * ChunkWs::bytes;
        float *vec = (float *)(ws + ChunkWs::vec);
        f4 *at = tiles + turn * 10 * 64;
        const bool in = lane < n;
        float gt = in ? gate : 0.0f;
        const float b = in ? bt : 0.0f;
        if (gt < kLeastGate) gt = kLeastGate;
        const int other = min(head + step, a.st.nv - 1);
        gate = gates[other], bt = betas[other];
        const bool ok = finite32(gt) && finite32(b);
        const unsigned long long bad = __ballot(!ok) | bad_k;
        const int first = bad ? __builtin_ctzll(bad) : kChunk;
        double sum = ok ? (double)gt * 1.4426950408889634 : 0.0;  // by ln 2: powers of 2 are one instruction
        sum += dpp_d<0x111>(sum);
        sum += dpp_d<0x112>(sum);
        sum += dpp_d<0x114>(sum);
        sum += dpp_d<0x118>(sum);
        sum += dpp_d<0x142, 0xA>(sum);
        sum += dpp_d<0x143, 0xC>(sum);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's lanes alone read and write these
        G[lane] = sum;
        beta[lane] = lane < first ? b : 0.0f;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's lanes alone read and write these
        auto power = [](double x) { return __builtin_amdgcn_exp2f((float)x); };
        // P's tiles of the wave's row and A's of its column
        const double Gm = G[mine];
        f4 diag = zero, P[4], T[4], below[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const f4 be = *(const f4 *)&beta[16 * r + 4 * g];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = 16 * r + 4 * g + e;
                const float x = (float)(G[i] - Gm), by = __builtin_amdgcn_exp2f(i <= mine ? -x : x);  // from the earlier row to the later
                P[r][e] = i <= mine ? by * dq[r][e] : 0.0f;
                below[r][e] = i > mine && i < first ? be[e] * by * dk[r][e] : 0.0f;
                if (r == wave) diag[e] = -below[r][e];
            }
            T[r] = zero;
        }
#pragma unroll
        for (int r = 1; r < 4; r++)
            if (r > wave) at[(r * (r - 1) / 2 + wave) * 64] = below[r];
        // the diagonal tile's inverse, lane (m, g) column m of rows 4 g and on; a row that is done goes to all of them
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = 4 * g + e == m ? 1.0f : 0.0f;
        eliminate<0>(diag, v);
        at[(6 + wave) * 64] = v;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float *d = (const float *)(at - lane + (6 + wave) * 64);
            const float x = d[(16 * (m >> 2) + 4 * g + e) * 4 + (m & 3)];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i == wave) T[i][e] = x;
        }
#pragma unroll
        for (int j = 2; j >= 0; j--) {
            if (j >= wave) continue;
            f4 sum2 = zero;
#pragma unroll
            for (int k = j + 1; k < 4; k++)
                if (k <= wave) sum2 = mfma4(at[(k * (k - 1) / 2 + j) * 64], T[k], sum2);
            T[j] = -mfma4(at[(6 + j) * 64], sum2, zero);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) T[r] *= *(const f4 *)&beta[16 * r + 4 * g];
        __asm__ volatile("" : "+v"(gate), "+v"(bt));  // likewise
        // rows of T and P in two terms
        const int pairs = wave < 2 ? 1 : 2;
        auto store = [&](const f4 (&y)[4], int what) {
            const int ex = scale_of(rows16_max(size_bits(y)));
            h8 *to = (h8 *)(ws + what) + lane;
#pragma unroll
            for (int p = 0; p < 2; p++) {
                if (p >= pairs) continue;
                h8 h, lo;
                two_terms(y[2 * p], y[2 * p + 1], scale_up(ex), h, lo);
                to[tile_piece(wave, p) * 128] = h;
                to[tile_piece(wave, p) * 128 + 64] = lo;
            }
            return scale_down(ex);
        };
        const float back_t = store(T, ChunkWs::T), back_p = store(P, ChunkWs::P);
        const double last = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(sum), 63), __builtin_amdgcn_readlane(__double2loint(sum), 63));
        if (g == 0) {
            vec[ChunkWs::gt + mine] = back_t;
            vec[ChunkWs::gp + mine] = back_p;
            vec[ChunkWs::gg + mine] = power(last - Gm) * scale_down(exk) * back_t;
        }
        if (wave == 0) {
            const float gx = power(sum) * back_k;
            vec[ChunkWs::gx + lane] = gx;
            const uint32_t top = wave_top(__float_as_uint(gx));
            if (lane == 0) vec[ChunkWs::top] = __uint_as_float(top);
        } else if (wave == 1) {
            vec[ChunkWs::gq + lane] = power(sum) * back_q;
        } else if (wave == 2 && lane == 63) {
            vec[ChunkWs::whole] = power(sum);
            *(int *)(vec + ChunkWs::first) = first;
        }
    }
}
// The chunks' workgroups, which the next kernel waits for, then those of sequences that go row by row.
template <int HD>
__global__ __launch_bounds__(kPrepTPB, 3) void gdn_prep_kernel(RuleArgs a) {
    __shared__ union Lds {
        PrepLds<HD> prep;
        float buf[kRowBuf][HD];
    } l;
    const unsigned per = (unsigned)a.parts * a.st.nqk, chunks = a.slots * per, i = blockIdx.y * gridDim.x + blockIdx.x, in = i % per;
    if (i < chunks)
        rule_prep<HD>(a, (int)(i / per), (int)(in % a.st.nqk), (int)(in / a.st.nqk), l.prep);
    else
        rule_rows_of<HD>(a, i - chunks, 0, l.buf);
}

// The transposing LDS read: of the 16 lanes' 16 x 4 values, lane i gets value i % 4 of lanes 4 j + i / 4, j < 4.
__device__ __forceinline__ h4 read_columns(const uint8_t *p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(uintptr_t)(
                                      (__attribute__((address_space(3))) const uint8_t *)p)));
}

// A sequence's chunks in order, a workgroup 32 columns of a head. Two waves take
// the state on, 16 columns each, all of a column's values in registers; two
// more the results of the same columns, for which the former leave the state
// before a chunk and the corrections, both as operands, in the LDS. Left
// operands come to the LDS once for all, brought by the results' waves, whose
// way is the shorter: between the chunk's two barriers P and the next chunk's
// keys and factors, then its queries and T. One wave a SIMD: products and the
// vector instructions between them are ordered so that the latter run while
// the matrix cores work. A chunk takes a state's wave 5300 clocks, 1800 of them
// products; the operands' terms and what waits for one another are the rest.
constexpr int kChunkCols = 32;
// Workgroups of columns, one a compute unit, that go before the sequences that go row by row; most of the others, of
// sequences that there may be, find none.
constexpr int kFirstChains = 256;
template <int HD>
struct ChunkLds {
    static constexpr int KB = kq_bytes(HD), Q = 2 * KB, T = 3 * KB, P = T + ChunkWs::P, vec = T + ChunkWs::vec, vec_bytes = ChunkWs::bytes - ChunkWs::vec;  // keys and factors twice
    static constexpr int S = vec + 2 * vec_bytes, U = S + 2 * HD * 64, one = U + 2 * 4096, bytes = one + 2 * 256;  // of two waves
};
template <int HD>
__global__ __launch_bounds__(256, 1) void gdn_chunks_kernel(RuleArgs a) {
    using L = ChunkLds<HD>;
    constexpr int KP = HD / 32, ST = HD / 16, NB = HD / kChunkCols, KB = L::KB;
    extern __shared__ __align__(1024) uint8_t lds[];
    // a head's column blocks on one XCD (workgroup i runs on XCD i % 8), whose L2 they share their operands in
    unsigned i = blockIdx.y * gridDim.x + blockIdx.x;
    if (i >= (unsigned)kFirstChains) {
        if (i - kFirstChains < (unsigned)a.singles) return rule_rows_of<HD>(a, i - kFirstChains, 1, (float (*)[HD])lds);
        i -= a.singles;
    }
    const int xcd = i & 7, at = i >> 3, pair = at / NB * 8 + xcd, head = pair % a.st.nv, hq = head % a.st.nqk;
    if (pair >= a.longs * a.st.nv) return;
    const Long s = find_long<false>(a.b, pair / a.st.nv, a.chunked);
    if (s.seq < 0) return;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6)), m = lane & 15, g = lane >> 4, half = wave & 1;
    const int col = at % NB * kChunkCols + 16 * half + m, chunks = (s.n + kChunk - 1) / kChunk;
    const f4 zero{0.f, 0.f, 0.f, 0.f};
    uint8_t *const ls = lds + L::S + half * HD * 64 + 16 * lane, *const lu = lds + L::U + half * 4096 + 16 * lane;
    float *const one = (float *)(lds + L::one) + half * 64;  // of each column: the scales of its state and of U, its largest value, the row where U ends
    // Values and results of a chunk's rows through a buffer that ends with the sequence: what lies behind is 0, and
    // not written. A chunk's offsets stay below 2^32 (row strides below 2^24).
    auto rows_of = [&](const float *p, uint32_t row, int c) {
        return buf_rsrc(p + (size_t)c * kChunk * row, 4 * ((uint32_t)(min(kChunk, s.n - c * kChunk) - 1) * row + HD));
    };
    // Products of a pair of tiles' depth of four tiles of rows; an operand is read a step before it is used. Turned, a
    // lane has a row's values 4 g and on, as they are stored, and not four rows' of a column.
    struct Rows {
        h8 h[4], l[4];
    };
    auto read_rows = [&](Rows &x, const uint8_t *l, int p) {
#pragma unroll
        for (int t = 0; t < 4; t++) x.h[t] = *(const h8 *)(l + (t * KP + p) * 2048);
#pragma unroll
        for (int t = 0; t < 4; t++) x.l[t] = *(const h8 *)(l + (t * KP + p) * 2048 + 1024);
    };
    auto times = [&](const Rows &x, const h8 &h, const h8 &l, f4 (&r)[4], auto turned) {
#pragma unroll
        for (int k = 0; k < 3; k++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const h8 &y = k < 2 ? x.h[t] : x.l[t], &z = k == 1 ? l : h;
                r[t] = decltype(turned)::value ? mfma_h(z, y, r[t]) : mfma_h(y, z, r[t]);
            }
    };
    // a triangle's product: pair 0 of all four tiles of rows, pair 1 of the last two
    struct Tri {
        h8 h[6], l[6];
    };
    auto read_tri = [&](Tri &y, int what) {
#pragma unroll
        for (int i = 0; i < 6; i++) {
            y.h[i] = *(const h8 *)(lds + what + i * 2048 + 16 * lane);
            y.l[i] = *(const h8 *)(lds + what + i * 2048 + 1024 + 16 * lane);
        }
    };
    auto triangle = [&](const Tri &y, const h8 (&h)[2], const h8 (&l)[2], f4 (&d)[4], auto turned) {
#pragma unroll
        for (int t = 0; t < 4; t++) d[t] = zero;
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int k = 0; k < 3; k++)
#pragma unroll
                for (int t = 2 * p; t < 4; t++) {
                    const h8 &u = k < 2 ? y.h[tile_piece(t, p)] : y.l[tile_piece(t, p)], &z = k == 1 ? l[p] : h[p];
                    d[t] = decltype(turned)::value ? mfma_h(z, u, d[t]) : mfma_h(u, z, d[t]);
                }
    };
    auto factors = [&](f4 (&f)[4], int c, int what) {
#pragma unroll
        for (int t = 0; t < 4; t++) f[t] = *(const f4 *)(lds + L::vec + (c & 1) * L::vec_bytes + 4 * (what + 16 * t + 4 * g));
    };
#define STEP __builtin_amdgcn_sched_barrier(0)
// N times a product, R reads of the LDS and M vector instructions
#define MIX(N, R, M)                                             \
    _Pragma("unroll") for (int mix = 0; mix < (N); mix++) {      \
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);       \
        __builtin_amdgcn_sched_group_barrier(0x100, (R), 0);     \
        __builtin_amdgcn_sched_group_barrier(0x002, (M), 0);     \
    }
    const uint8_t *ws = a.ws + ((size_t)s.slot * a.st.nv + head) * ChunkWs::bytes + 1024 * half + 16 * lane;
    const uint8_t *kq = a.kq + ((size_t)s.slot * a.st.nqk + hq) * 2 * KB + 1024 * half + 16 * lane;
    const size_t ws_step = (size_t)a.st.nv * ChunkWs::bytes, kq_step = (size_t)a.st.nqk * 2 * KB;
    // the wave's half of a chunk's pieces of 1 KB
    constexpr int NK = KB / 2048, NT = ChunkWs::P / 2048;
    static_assert(L::vec_bytes == 2048, "a piece for each wave");
    auto fetch = [&](const uint8_t *from, int to, int i) { dma16(from + 2048 * i, lds + to + 1024 * half + 2048 * i); };
    // queries and T
    auto fetch_after = [&](int c) {
#pragma unroll
        for (int i = 0; i < NK; i++) fetch(kq + c * kq_step + KB, L::Q, i);
#pragma unroll
        for (int i = 0; i < NT; i++) fetch(ws + c * ws_step, L::T, i);
    };
    if (wave >= 2) {  // the results
        const uint32_t out_row = (uint32_t)(a.st.nv * HD), o_at = 4 * (m * out_row + col - m + 4 * g);
        float *out = a.out + ((size_t)s.lo * a.st.nv + head) * HD;
#pragma unroll
        for (int i = 0; i < NK; i++) fetch(kq, 0, i), fetch(kq + KB, L::Q, i);
#pragma unroll
        for (int i = 0; i < NT; i++) fetch(ws, L::T, i);
        fetch(ws + ChunkWs::vec, L::vec, 0);
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint8_t *query_at = lds + L::Q + 16 * place(m, g);
        // the last chunk's products, and their columns' and rows' factors
        f4 o[4], r[4], down_u, stop;
        float fp[4];
        auto store = [&](int c) {
            const auto bo = rows_of(out, out_row, c);
            int least = kChunk;
#pragma unroll
            for (int e = 0; e < 4; e++) least = min(least, __float_as_int(stop[e]));
            const bool bad = __ballot(least < kChunk);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                f4 y;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = fmaf(fp[t] * r[t][e], down_u[e], o[t][e]);
                if (bad) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (16 * t + m >= __float_as_int(stop[e])) y[e] = __uint_as_float(0x7FC00000u);
                }
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4v, y), bo, o_at + 64 * t * out_row, 0, 0);
            }
        };
        for (int c = 0; c < chunks; c++) {
            const int next = min(c + 1, chunks - 1), into = (c + 1) & 1;  // the last chunk brings itself again, and waits for it at the end
            wait_vm_barrier<0>();
            if (c > 0) store(c - 1);
            h8 sh[KP], sl[KP];
#pragma unroll
            for (int p = 0; p < KP; p++) sh[p] = *(const h8 *)(ls + 2048 * p), sl[p] = *(const h8 *)(ls + 2048 * p + 1024);
            Rows ra, rb;
            read_rows(ra, query_at, 0);
            const f4 down_s = *(const f4 *)(one + 4 * g);
            float fq[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const float *vec = (const float *)(lds + L::vec + (c & 1) * L::vec_bytes) + 16 * t + m;
                fq[t] = vec[ChunkWs::gq], fp[t] = vec[ChunkWs::gp], o[t] = zero;
            }
            STEP;
#pragma unroll
            for (int i = 0; i < NT; i++) fetch(ws + c * ws_step + ChunkWs::P, L::P, i);
#pragma unroll
            for (int i = 0; i < NK; i++) fetch(kq + next * kq_step, into * KB, i);
            fetch(ws + next * ws_step + ChunkWs::vec, L::vec + into * L::vec_bytes, 0);
            STEP;
#pragma unroll
            for (int p = 0; p < KP; p++) {
                Rows &now = p % 2 ? rb : ra, &then = p % 2 ? ra : rb;
                if (p + 1 < KP) read_rows(then, query_at, p + 1);
                times(now, sh[p], sl[p], o, std::true_type{});
                MIX(8, 1, 1);
                STEP;
            }
#pragma unroll
            for (int t = 0; t < 4; t++) o[t] *= fq[t] * down_s;
            // the state's largest value, of its first terms, as whose scale's bound it serves
            typedef unsigned short w8 __attribute__((ext_vector_type(8)));
            w8 top = __builtin_bit_cast(w8, sh[0]) & (unsigned short)0x7FFF;
#pragma unroll
            for (int p = 1; p < KP; p++) top = __builtin_elementwise_max(top, (w8)(__builtin_bit_cast(w8, sh[p]) & (unsigned short)0x7FFF));
            uint32_t largest = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) largest = max(largest, (uint32_t)top[e]);
            one[16 + m] = (float)__builtin_bit_cast(_Float16, (unsigned short)rows16_max(largest));
            STEP;
            wait_vm_barrier<NK + 1>();  // P is there, the state and the queries are read; the corrections are there
            f4 u[4];
#pragma unroll
            for (int t = 0; t < 4; t++) u[t] = *(const f4 *)(lu + 1024 * t);
            Tri tri;
            read_tri(tri, L::P);
            f4 ft[4];
            factors(ft, c, ChunkWs::gt);
            down_u = *(const f4 *)(one + 32 + 4 * g), stop = *(const f4 *)(one + 48 + 4 * g);
            STEP;
            fetch_after(next);
            STEP;
#pragma unroll
            for (int t = 0; t < 4; t++) u[t] *= ft[t];
            const int ex_u = scale_of(rows16_max(__float_as_uint(top_of(u))));
            h8 uh[2], ul[2];
#pragma unroll
            for (int p = 0; p < 2; p++) two_terms(u[2 * p], u[2 * p + 1], scale_up(ex_u), uh[p], ul[p]);
            const float down = scale_down(ex_u);
            f4 by;  // of the columns that the lane has of the products
#pragma unroll
            for (int e = 0; e < 4; e++) by[e] = __shfl(down, 4 * g + e);
            triangle(tri, uh, ul, r, std::true_type{});
            down_u *= by;
        }
        store(chunks - 1);
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what the last chunk brought lands before the wave leaves
        return;
    }
    const int from = a.st.from[s.seq], to = a.st.to[s.seq];
    const size_t mine = (size_t)(4 * g) * HD + col;  // the lane's first value of a state
    f4 S[ST];
#pragma unroll
    for (int t = 0; t < ST; t++) S[t] = zero;
    if ((unsigned)from < (unsigned)a.st.n_slots) {
        const float *p = a.st.state + ((size_t)from * a.st.nv + head) * HD * HD + mine;
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) S[t][e] = p[(16 * t + e) * HD];
    }
    const uint32_t v_row = (uint32_t)a.h.v_row, v_at = 4 * (4 * g * v_row + col);
    const float *V = a.h.d_v + (size_t)s.lo * a.h.v_row + (size_t)head * HD;
    f4 v[4];
    auto load_v = [&](int c) {
        const auto b = rows_of(V, v_row, c);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) v[t][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, v_at + 4 * (16 * t + e) * v_row, 0, 0));
    };
    h8 sh[KP], sl[KP];
    // A column's state is held in units of 2^(ex_s - 14). Its scale is set before the values are known, by a bound on the
    // largest, as is that of X: of a sum's terms, of which f32's errors are parts of 2^-24. A bound 64 times too large
    // costs 2^-33 of it.
    int ex_s;
    auto state_terms = [&](int p) {
        two_terms(S[2 * p], S[2 * p + 1], sh[p], sl[p]);
        *(h8 *)(ls + 2048 * p) = sh[p];
        *(h8 *)(ls + 2048 * p + 1024) = sl[p];
    };
    auto column_top = [&](float v) { return rows16_max(__float_as_uint(v)); };
    auto units = [&](int ex) {
#pragma unroll
        for (int t = 0; t < ST; t++) S[t] *= ldexpf(1.0f, ex);
    };
    load_v(0);
    ex_s = scale_of(column_top(top_of(S)));
    units(14 - ex_s);
#pragma unroll
    for (int p = 0; p < KP; p++) state_terms(p);
    one[m] = scale_down(ex_s);
    for (int c = 0; c < chunks; c++) {
        const uint8_t *lk = lds + (c & 1) * KB, *row_at = lk + 16 * place(m, g);
        const int next = min(c + 1, chunks - 1);
        lds_barrier();  // the keys, T and the factors are there, and the state's terms
        Rows ra, rb;
        f4 x[4], r[4] = {zero, zero, zero, zero}, fx[4], fg[4];
        read_rows(ra, row_at, 0);
        const float *vec = (const float *)(lds + L::vec + (c & 1) * L::vec_bytes);
        const float whole = vec[ChunkWs::whole], top_x = vec[ChunkWs::top];
        const int first_bad = *(const int *)(vec + ChunkWs::first);
        STEP;
        // the scale of X while the keys come: at most |v| + |e^G k| |S|
        hold(v);
        uint32_t top_v = column_top(top_of(v));
        if (__ballot(top_v >= 0x7F800000u)) {  // of the finite ones, whose rows may come before
            f4 w[4];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) w[t][e] = finite32(v[t][e]) ? v[t][e] : 0.0f;
            top_v = column_top(top_of(w));
        }
        int ex_x = scale_of_sum(top_x, ex_s + 14 + (HD == 128 ? 7 : 6), __uint_as_float(top_v), 0);
        factors(fx, c, ChunkWs::gx);
        STEP;
        Tri tri;
#pragma unroll
        for (int p = 0; p < KP; p++) {
            Rows &now = p % 2 ? rb : ra, &then = p % 2 ? ra : rb;
            if (p + 1 < KP)
                read_rows(then, row_at, p + 1);
            else
                read_tri(tri, L::T), factors(fg, c, ChunkWs::gg);
            times(now, sh[p], sl[p], r, std::false_type{});
            if (p == KP - 1) {
                hold(fx);
                const float up = scale_up(ex_x), by = ldexpf(-1.0f, min(ex_s - ex_x, 127));  // beyond it all of fx is 0
#pragma unroll
                for (int t = 0; t < 4; t++) fx[t] *= by, x[t] = v[t] * up;
            }
            MIX(12, 1, 3);
            STEP;
        }
        // X = V - diag(e^G) K S, in units of 2^(ex_x - 14)
        h8 xh[2], xl[2], gh[2], gl[2];
#pragma unroll
        for (int p = 0; p < 2; p++) {
#pragma unroll
            for (int t = 2 * p; t < 2 * p + 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[t][e] = fmaf(fx[t][e], r[t][e], x[t][e]);
            two_terms(x[2 * p], x[2 * p + 1], xh[p], xl[p]);
        }
        STEP;
        f4 u[4], ug[4];  // U, in X's units and of T's rows
        triangle(tri, xh, xl, u, std::false_type{});
        load_v(next);
        const int first = uniform(first_bad);
        STEP;
        // A correction that is not finite makes what it is multiplied with in the last row NaN or infinite, by 0 too
        int stop = first;  // the column's rows from here on are not numbers
        if (first < kChunk || __ballot(!finite32(u[3][3])) != 0) {
#pragma unroll
            for (int t = 3; t >= 0; t--)
#pragma unroll
                for (int e = 3; e >= 0; e--)
                    if (!finite32(x[t][e])) stop = min(stop, 16 * t + 4 * g + e);
            stop = min(stop, __shfl_xor(stop, 16));
            stop = min(stop, __shfl_xor(stop, 32));
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) x[t][e] = 16 * t + 4 * g + e < stop ? x[t][e] : 0.0f;
            const int ex = scale_of(column_top(top_of(x)));
            ex_x += ex - 14;
#pragma unroll
            for (int p = 0; p < 2; p++) two_terms(x[2 * p], x[2 * p + 1], scale_up(ex), xh[p], xl[p]);
            triangle(tri, xh, xl, u, std::false_type{});
        }
        // S <- e^G_63 S + K^T (e^(G_63 - G) U), two tiles of the state at a time: the keys by columns, rows 4 g + m / 4
        // of tile 2 p + (0, 1), columns 4 (m % 4) and on of state tile i
        struct Cols {
            h8 h[2][2], l[2][2];
        };
        const uint8_t *col_at = lk + 16 * place(4 * g + (m >> 2), m & 3);
        auto read_tiles = [&](Cols &k, int i0) {
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint8_t *y = col_at + (2 * p * KP + i0 / 2) * 2048 + 8 * j;
                    k.h[p][j] = __builtin_shufflevector(read_columns(y), read_columns(y + KP * 2048), 0, 1, 2, 3, 4, 5, 6, 7);
                    k.l[p][j] = __builtin_shufflevector(read_columns(y + 1024), read_columns(y + KP * 2048 + 1024), 0, 1, 2, 3, 4, 5, 6, 7);
                }
        };
        Cols cols[2];
        read_tiles(cols[0], 0);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            ug[t] = u[t] * fg[t];
            *(f4 *)(lu + 1024 * t) = u[t];
        }
        one[32 + m] = scale_down(ex_x);
        one[48 + m] = __int_as_float(stop);
        const uint32_t top_g = column_top(top_of(ug));
        const int ex_g = scale_of(top_g);
        const float up_g = scale_up(ex_g);
        two_terms(ug[0], ug[1], up_g, gh[0], gl[0]);
        STEP;
        lds_barrier();  // the corrections are there
        const float top_s = one[16 + m] + 0x1p-24f;  // f16 takes values to 0 below half of that
        f4 d[2][2];
        float keep = 0.0f, add = 0.0f;
        auto update = [&](int q) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[2 * q + t][e] = fmaf(d[q % 2][t][e], add, S[2 * q + t][e] * keep);
            state_terms(q);
        };
#pragma unroll
        for (int q = 0; q < KP; q++) {
            const Cols &k = cols[q % 2];
            if (q + 1 < KP) read_tiles(cols[(q + 1) % 2], 2 * q + 2);
            d[q % 2][0] = d[q % 2][1] = zero;
            if (q == 0) two_terms(ug[2], ug[3], up_g, gh[1], gl[1]);
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int y = 0; y < 3; y++)
#pragma unroll
                    for (int t = 0; t < 2; t++) d[q % 2][t] = mfma_h(y < 2 ? k.h[p][t] : k.l[p][t], y == 1 ? gl[p] : gh[p], d[q % 2][t]);
            if (q == 0) {
                // what the sum's terms amount to at most; those of K^T U by the operands' scales and the depth
                const int to = scale_of_sum((double)top_s * whole, ex_s - 14, __uint_as_float(top_g), ex_x + 6);
                keep = ldexpf(whole, ex_s - to), add = ldexpf(1.0f, ex_g + ex_x - 14 - to);
                ex_s = to;
                one[m] = scale_down(ex_s);
            } else {
                update(q - 1);
            }
            MIX(12, 2, 5);
            STEP;
        }
        update(KP - 1);
        if (__ballot(stop < kChunk)) {
            const float nan = __uint_as_float(0x7FC00000u);
            if (stop < kChunk)
#pragma unroll
                for (int i = 0; i < ST; i++) S[i] = f4{nan, nan, nan, nan};
#pragma unroll
            for (int p = 0; p < KP; p++) state_terms(p);
        }
    }
    units(ex_s - 14);
#undef MIX
#undef STEP
    if ((unsigned)to < (unsigned)a.st.n_slots) {
        float *p = a.st.state + ((size_t)to * a.st.nv + head) * HD * HD + mine;
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) p[(16 * t + e) * HD] = S[t][e];
    }
}

// The epilogue of the rows that went by chunks: a workgroup a chunk and head,
// HD / 4 lanes a row, several rows of a lane under way. Memory bounds it: 5241
// rows of 32 heads 45 us, 5.6 TB/s.
template <int HD>
__global__ __launch_bounds__(256) void gdn_finish_kernel(RuleArgs a) {
    constexpr int PER = HD / 4, STEP = 256 / PER, N = kChunk / STEP;  // threads of a row, rows at a time, rows of a thread
    const unsigned i = blockIdx.y * gridDim.x + blockIdx.x;
    const int slot = (int)(i / a.st.nv), head = (int)(i % a.st.nv), r0 = threadIdx.x / PER, o = 4 * (threadIdx.x % PER);
    if (slot >= a.slots) return;
    const Long s = find_long<true>(a.b, slot, a.chunked);
    if (s.seq < 0) return;
    const int c0 = (slot - s.slot) * kChunk, n = min(kChunk, s.n - c0);
    const size_t row0 = (size_t)s.lo + c0;
    f4 v[N], z[N], w{1.f, 1.f, 1.f, 1.f};
    if (a.h.d_norm) w = *(const f4u *)(a.h.d_norm + o);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const size_t row = row0 + min(r0 + STEP * i, n - 1);
        v[i] = *(const f4u *)(a.out + (row * a.st.nv + head) * HD + o);
        if (a.h.d_z) z[i] = *(const f4u *)(a.h.d_z + row * a.h.z_row + (size_t)head * HD + o);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (a.h.d_norm) {
            float sq = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) sq = fmaf(v[i][e], v[i][e], sq);
            v[i] *= (1.0f / sqrtf(lanes_sum<PER>(sq) / (float)HD + a.h.eps)) * w;
        }
        if (a.h.d_z) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[i][e] *= silu(z[i][e]);
        }
        if (r0 + STEP * i < n) *(f4u *)(a.out + ((row0 + r0 + STEP * i) * a.st.nv + head) * HD + o) = v[i];
    }
}

}  // namespace

// So many workgroups, of which a kernel numbers those across first.
static dim3 grid_of(size_t n) {
    const size_t across = std::min(n, (size_t)1 << 22);
    return dim3((unsigned)across, (unsigned)((n + across - 1) / across));
}

hipError_t launch_gdn_conv(const StatesView &st, const BatchView &b, const uq_gdn_rows &r, hipStream_t s) {
    if (b.n_rows == 0 || b.n_seqs == 0) return hipSuccess;
    const ConvArgs a{st, b, r, (st.channels + 255) / 256};
    const unsigned per = kConvTPB / 64, tiles = (unsigned)(b.n_rows / kConvRows + std::min(b.n_seqs, b.n_rows));
    // A tile's channels one after another: rows are often a power of 2 apart, and a column of tiles would meet in few of
    // the memory's channels. 6010 rows of 8192 channels so took 82 us, and 94 the other way round.
    const dim3 grid = grid_of((size_t)tiles * (((unsigned)a.groups + per) / per));
    if (st.taps == 4)
        hipLaunchKernelGGL(gdn_conv_kernel<4>, grid, dim3(kConvTPB), 0, s, a);
    else
        hipLaunchKernelGGL(gdn_conv_kernel<0>, grid, dim3(kConvTPB), 0, s, a);
    return hipGetLastError();
}

namespace {
// Sequences of this many rows and more go by chunks. One alone takes as long by chunks at 64 rows as at 20, and row by
// row is quicker where many share the chip. Heads of 128, rows and us row by row / by chunks: 1 sequence of 32 heads,
// 24: 30 / 23; 8, 32: 45 / 46; 64, 32: 203 / 275, 48: 288 / 286; 300, 64: 1586 / 1460.
int chunk_least(const StatesView &st, const BatchView &b) {
    const long long heads = (long long)b.n_seqs * st.nv;
    return heads <= 64 ? 24 : heads <= 1024 ? 32 : 48;
}
// How many sequences can go by chunks, and the slots of their chunks; 0 where none is expected to.
struct Plan {
    int least, longs, slots;
};
Plan plan_of(const StatesView &st, const BatchView &b, size_t most_rows) {
    const int least = chunk_least(st, b);
    if (b.n_rows < least || (most_rows && most_rows < (size_t)least)) return Plan{INT_MAX, 0, 0};
    const int longs = std::min(b.n_seqs, b.n_rows / least);
    return Plan{least, longs, b.n_rows / kChunk + longs + 1};
}
}  // namespace

size_t gdn_rule_ws_bytes(const StatesView &st, const BatchView &b, size_t most_rows) {
    return 16 + (size_t)plan_of(st, b, most_rows).slots * (st.nv * (size_t)ChunkWs::bytes + st.nqk * (size_t)(2 * kq_bytes(st.hd)));
}

template <int HD>
hipError_t launch_rule(RuleArgs a, hipStream_t s) {
    if (!a.longs) {
        hipLaunchKernelGGL(gdn_rows_kernel<HD>, dim3((unsigned)a.st.nv, (unsigned)a.b.n_seqs), dim3(2 * HD), 0, s, a);
        return hipGetLastError();
    }
    constexpr size_t lds = ChunkLds<HD>::bytes;
    const auto kernel = gdn_chunks_kernel<HD>;
    if (hipError_t e = allow_lds((const void *)kernel, lds)) return e;
    const size_t pairs = (size_t)a.longs * a.st.nv, seqs = a.b.n_seqs, nv = a.st.nv;
    // The value heads of a key head one after another, or all at once where all find room on the chip: 509 rows 11.5 us
    // against 14. More of them would keep sequences that go row by row from it: 34 against 31 for 1021 rows beside 40.
    a.parts = a.slots * nv <= 3 * 256 ? a.st.nv / a.st.nqk : 1;
    a.singles = (int)((seqs / 2 * nv + 7) / 8 * 8);
    hipLaunchKernelGGL(gdn_prep_kernel<HD>, grid_of((size_t)a.slots * a.parts * a.st.nqk + (seqs + 1) / 2 * nv), dim3(kPrepTPB), 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(kernel, grid_of(std::max((size_t)kFirstChains, (pairs + 7) / 8 * 8 * (HD / kChunkCols)) + a.singles), dim3(256), lds, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    if (a.h.d_norm || a.h.d_z) hipLaunchKernelGGL(gdn_finish_kernel<HD>, grid_of((size_t)a.slots * a.st.nv), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_gdn_rule(float *out, const StatesView &st, const BatchView &b, const uq_gdn_heads &h, size_t most_rows,
                           void *ws, hipStream_t s) {
    if (b.n_rows == 0 || b.n_seqs == 0) return hipSuccess;
    const Plan p = plan_of(st, b, most_rows);
    const RuleArgs a{out, st, b, h, p.least, p.longs, p.slots, 1, 0, (uint8_t *)ws, (uint8_t *)ws + (size_t)p.slots * st.nv * ChunkWs::bytes};
    return st.hd == 128 ? launch_rule<128>(a, s) : launch_rule<64>(a, s);
}

}  // namespace uq
