// Batched serving of GatedDeltaNet layers: the convolution of a batch's rows
// with its windows, norms and gates (uq_gdn_conv_d), and the gated delta rule
// over its states (uq_gdn_rule_d).
#include <algorithm>
#include <climits>

#include "uq_device.h"
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

// x / (1 + e^-x). The quotient by the hardware's reciprocal (1 ulp).
__device__ __forceinline__ float silu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + expf(-x)); }

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
// it alone reads.
template <int CK>  // taps, 0: any up to 9
__global__ __launch_bounds__(kConvTPB) void gdn_conv_kernel(ConvArgs a) {
    constexpr int MT = CK ? CK : 9, H = MT - 1, STEP = 4;
    const int taps = CK ? CK : a.st.taps, skip = MT - taps;  // places before the first tap
    const int lane = threadIdx.x & 63, group = uniform((int)(blockIdx.y * (kConvTPB / 64) + (threadIdx.x >> 6)));
    if (group > a.groups) return;
    const Tile t = find_tile<kConvRows>(a.b, (int)blockIdx.x, 1);
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
                    if (k >= skip) s = __fadd_rn(s, __fmul_rn(x[u + k][e], tap[e][k]));
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
    float *ws;        // [slots][nv][kChunkFloats]
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
// bounds it for few rows.
constexpr int kRowBuf = 16;  // rows whose results wait for the norm
template <int HD>
__global__ __launch_bounds__(2 * HD) void gdn_rows_kernel(RuleArgs a) {
    constexpr int R = HD / 8, NW = HD / 32;
    __shared__ float buf[kRowBuf][HD];
    const int head = blockIdx.x, seq = blockIdx.y, hq = head % a.st.nqk;
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
        f4 q[R / 4], k[R / 4], v;
        float g, b;
    };
    auto load = [&](Row &x, int i) {
        const size_t row = (size_t)rows.lo + i;
        const float *q = a.h.d_q + row * a.h.q_row + (size_t)hq * HD + i0, *k = a.h.d_k + row * a.h.k_row + (size_t)hq * HD + i0;
#pragma unroll
        for (int u = 0; u < R / 4; u++) x.q[u] = *(const f4u *)(q + 4 * u), x.k[u] = *(const f4u *)(k + 4 * u);
        x.v = *(const f4u *)(a.h.d_v + row * a.h.v_row + (size_t)head * HD + j0);
        x.g = a.h.d_gate[row * a.st.nv + head];
        x.b = a.h.d_beta[row * a.st.nv + head];
    };
    Row x, next;
    load(x, 0);
    for (int i = 0; i < rows.n; i++) {
        load(next, min(i + 1, rows.n - 1));
        const float eg = expf(x.g);
        f4 sk{0.f, 0.f, 0.f, 0.f}, sq = sk, d, o;
        float qk = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float k = x.k[r / 4][r % 4], q = x.q[r / 4][r % 4];
            qk = fmaf(q, k, qk);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                sk[e] = fmaf(k, S[r][e], sk[e]);
                sq[e] = fmaf(q, S[r][e], sq[e]);
            }
        }
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

// ---- the delta rule by chunks ---------------------------------------------------
//
// Of 64 rows with the state S before them and G_i the gates' sum up to row i,
// the corrections U solve
//     (I + A) U = diag(beta) (V - diag(e^G) K S),  A[i][j] = beta_i e^(G_i - G_j) k_i.k_j  (j < i),
// and  out = scale (diag(e^G) Q S + P U),          P[i][j] = e^(G_i - G_j) q_i.k_j         (j <= i),
//      S <- e^G_63 S + K^T (diag(e^(G_63 - G)) U).
// What does not depend on S, T = (I + A)^-1 diag(beta) and P, is formed for all
// chunks at once (gdn_prep_kernel); gdn_chunks_kernel then takes a sequence's
// chunks one after another, 16 columns of a head's state a workgroup, which
// nothing of another column enters.
//
// Products run on the f32 matrix cores, 16x16x4, whose depth is a sum over k
// = lane / 16: taken as 4 (lane / 16) + e in the e-th of four products, the left
// operand is 4 neighbours of a row, one load, and a product's result (rows 4
// (lane / 16) + e, column lane % 16) is a right operand as it is.
//
// A row with a key, beta or gate that is not finite leaves the products
// (first: the first such row), and so do rows of a column from its first
// correction on that is not: 0 times NaN would carry it to earlier rows.
// Their results are set to NaN.

struct ChunkWs {  // of a chunk and head, in floats
    static constexpr int T = 0, P = kChunk * kChunk, ge = 2 * kChunk * kChunk, gl = ge + kChunk, first = gl + kChunk;
};
constexpr int kChunkFloats = ChunkWs::first + 4;
constexpr float kLeastGate = -1000.0f;  // e^-1000 of any f32 is 0: gates below it are taken as it, so that differences are numbers

__device__ __forceinline__ bool finite32(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }
__device__ __forceinline__ f4 mfma4(const f4 &a, const f4 &b, f4 c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// T and P of a chunk and head. The 10 tiles on and below the diagonal of K K^T
// and Q K^T are five for each wave: column w of the one and 3 - w of the
// other. The triangle's inverse: a wave inverts a diagonal tile row after row,
// a column a lane, then goes down its column of tiles,
//     T_ij = -T_ii sum over j <= k < i of A_ik T_kj,
// as substitution would, in whose order errors do not grow.
constexpr int kPrepTPB = 256;
template <int HD>
__global__ __launch_bounds__(kPrepTPB) void gdn_prep_kernel(RuleArgs a) {
    constexpr int KC = HD / 16, LD = kChunk + 4;
    __shared__ __align__(16) float A[kChunk][LD], D[4][16][20];
    __shared__ double G[kChunk];
    __shared__ float beta[kChunk];
    __shared__ unsigned bad_k[4];
    __shared__ unsigned long long bad_g;
    const int head = blockIdx.y, hq = head % a.st.nqk;
    const Long s = find_long<true>(a.b, (int)blockIdx.x, a.chunked);
    if (s.seq < 0) return;
    const int c0 = ((int)blockIdx.x - s.slot) * kChunk, n = min(kChunk, s.n - c0);
    const size_t row0 = (size_t)s.lo + c0;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6)), m = lane & 15, g = lane >> 4;
    float *ws = a.ws + ((size_t)blockIdx.x * a.st.nv + head) * kChunkFloats;
    auto frag = [&](f4 (&f)[KC], const float *p, size_t stride, int tile) {
        const float *r = p + (row0 + min(16 * tile + m, n - 1)) * stride + (size_t)hq * HD + 4 * g;
#pragma unroll
        for (int c = 0; c < KC; c++) f[c] = *(const f4u *)(r + 16 * c);
    };
    auto product = [&](const f4 (&x)[KC], const f4 (&y)[KC]) {
        f4 s0{0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
        for (int c = 0; c < KC; c += 2) s0 = mfma4(x[c], y[c], s0), s1 = mfma4(x[c + 1], y[c + 1], s1);
        return s0 + s1;
    };
    f4 y[KC], x[KC];
    frag(y, a.h.d_k, a.h.k_row, wave);
    if (wave == 0) {
        const bool in = lane < n;
        float gt = in ? a.h.d_gate[(row0 + lane) * a.st.nv + head] : 0.0f, bt = in ? a.h.d_beta[(row0 + lane) * a.st.nv + head] : 0.0f;
        if (gt < kLeastGate) gt = kLeastGate;
        const bool ok = finite32(gt) && finite32(bt);
        const unsigned long long no = __ballot(!ok);
        double sum = ok ? (double)gt : 0.0;
        sum += dpp_d<0x111>(sum);
        sum += dpp_d<0x112>(sum);
        sum += dpp_d<0x114>(sum);
        sum += dpp_d<0x118>(sum);
        sum += dpp_d<0x142, 0xA>(sum);
        sum += dpp_d<0x143, 0xC>(sum);
        G[lane] = sum;
        beta[lane] = ok ? bt : 0.0f;
        if (lane == 0) bad_g = no;
        const double last = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(sum), 63), __builtin_amdgcn_readlane(__double2loint(sum), 63));
        ws[ChunkWs::ge + lane] = expf((float)sum);
        ws[ChunkWs::gl + lane] = expf((float)(last - sum));
    }
    {
        bool ok = true;
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) ok = ok && finite32(y[c][e]);
        const unsigned long long no = __ballot(!ok);
        if (lane == 0) bad_k[wave] = (unsigned)((no | no >> 16 | no >> 32 | no >> 48) & 0xFFFF);
    }
    __syncthreads();
    const unsigned long long bad = bad_g | bad_k[0] | (unsigned long long)bad_k[1] << 16 | (unsigned long long)bad_k[2] << 32 | (unsigned long long)bad_k[3] << 48;
    const int first = bad ? __builtin_ctzll(bad) : kChunk;
    if (threadIdx.x == 0) *(int *)(ws + ChunkWs::first) = first;
    // A's tiles (r, wave), then P's (r, 3 - wave), r not above their column
    auto decay = [&](int i, int j) { return expf((float)(G[i] - G[j])); };
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if (r < wave) continue;
        frag(x, a.h.d_k, a.h.k_row, r);
        const f4 d = product(x, y);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = 16 * r + 4 * g + e, j = 16 * wave + m;
            A[i][j] = j < i && i < first ? beta[i] * decay(i, j) * d[e] : 0.0f;
        }
    }
    frag(y, a.h.d_k, a.h.k_row, 3 - wave);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if (r < 3 - wave) continue;
        frag(x, a.h.d_q, a.h.q_row, r);
        const f4 d = product(x, y);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int i = 16 * r + 4 * g + e, j = 16 * (3 - wave) + m;
            ws[ChunkWs::P + i * kChunk + j] = j <= i ? a.h.scale * decay(i, j) * d[e] : 0.0f;
        }
    }
    __syncthreads();
    // the diagonal tile's inverse, column m in every lane of it
    {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float sum = i == m ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; j++) sum = fmaf(-A[16 * wave + i][16 * wave + j], v[j], sum);
            v[i] = sum;
        }
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (g == i / 4) D[wave][i][m] = v[i];
    }
    __syncthreads();
    f4 t[4];
    const float bm = 16 * wave + m < first ? beta[16 * wave + m] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i < wave) continue;
        if (i == wave) {
#pragma unroll
            for (int e = 0; e < 4; e++) t[i][e] = D[wave][4 * g + e][m];
        } else {
            f4 sum{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < i; k++)
                if (k >= wave) sum = mfma4(*(const f4 *)&A[16 * i + m][16 * k + 4 * g], t[k], sum);
            const f4 zero{0.f, 0.f, 0.f, 0.f};
            t[i] = -mfma4(*(const f4 *)&D[i][m][4 * g], sum, zero);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) ws[ChunkWs::T + (16 * i + 4 * g + e) * kChunk + 16 * wave + m] = t[i][e] * bm;
    }
}

// A sequence's chunks in order: four waves, wave w rows 16 w and on of the
// chunk and HD / 4 rows of the state. Operands of the next chunk are loaded as
// soon as this one's are used.
constexpr int kColumns = 16;
template <int HD>
__global__ __launch_bounds__(256, 1) void gdn_chunks_kernel(RuleArgs a) {
    constexpr int KC = HD / 16, ST = HD / 64, NB = HD / kColumns;
    __shared__ f4 lS[KC][64], lX[4][64], lU[4][64];
    __shared__ int lBad[4];
    // a head's column blocks on one XCD (workgroup i runs on XCD i % 8), whose L2 they share their operands in
    const int xcd = blockIdx.x & 7, at = blockIdx.x >> 3, pair = at / NB * 8 + xcd, head = pair % a.st.nv, hq = head % a.st.nqk;
    if (pair >= a.longs * a.st.nv) return;
    const Long s = find_long<false>(a.b, pair / a.st.nv, a.chunked);
    if (s.seq < 0) return;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6)), m = lane & 15, g = lane >> 4;
    const int col = at % NB * kColumns + m;
    const int chunks = (s.n + kChunk - 1) / kChunk;
    f4 S[ST];
    const int from = a.st.from[s.seq], to = a.st.to[s.seq];
    auto state_row = [&](int t) { return HD / 4 * wave + 16 * t + 4 * g; };
#pragma unroll
    for (int t = 0; t < ST; t++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            S[t][e] = (unsigned)from < (unsigned)a.st.n_slots
                          ? a.st.state[(((size_t)from * a.st.nv + head) * HD + state_row(t) + e) * HD + col]
                          : 0.0f;
    f4 k[KC], q[KC], T[4], P[4], kt[ST][4], v, ge, gl[4];
    float whole;
    int first;
    // a chunk's row, the last one where there is none: what has no row has beta 0 and corrections of 0
    auto row_of = [&](int c, int r) { return (size_t)s.lo + min(c * kChunk + r, s.n - 1); };
    auto ws_of = [&](int c) { return a.ws + ((size_t)(s.slot + c) * a.st.nv + head) * kChunkFloats; };
    auto load_k = [&](int c) {
        const float *p = a.h.d_k + row_of(c, 16 * wave + m) * a.h.k_row + (size_t)hq * HD + 4 * g;
#pragma unroll
        for (int i = 0; i < KC; i++) k[i] = *(const f4u *)(p + 16 * i);
    };
    auto load_q = [&](int c) {
        const float *p = a.h.d_q + row_of(c, 16 * wave + m) * a.h.q_row + (size_t)hq * HD + 4 * g;
#pragma unroll
        for (int i = 0; i < KC; i++) q[i] = *(const f4u *)(p + 16 * i);
    };
    auto load_v = [&](int c) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = a.h.d_v[row_of(c, 16 * wave + 4 * g + e) * a.h.v_row + (size_t)head * HD + col];
        ge = *(const f4 *)(ws_of(c) + ChunkWs::ge + 16 * wave + 4 * g);
        first = *(const int *)(ws_of(c) + ChunkWs::first);
    };
    auto load_t = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i <= wave) T[i] = *(const f4 *)(ws_of(c) + ChunkWs::T + (16 * wave + m) * kChunk + 16 * i + 4 * g);
    };
    auto load_p = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i <= wave) P[i] = *(const f4 *)(ws_of(c) + ChunkWs::P + (16 * wave + m) * kChunk + 16 * i + 4 * g);
    };
    auto load_kt = [&](int c) {  // K transposed: rows of the state, 4 neighbouring rows of the chunk
#pragma unroll
        for (int i = 0; i < 4; i++) {
            gl[i] = *(const f4 *)(ws_of(c) + ChunkWs::gl + 16 * i + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float *p = a.h.d_k + row_of(c, 16 * i + 4 * g + e) * a.h.k_row + (size_t)hq * HD + HD / 4 * wave + m;
#pragma unroll
                for (int t = 0; t < ST; t++) kt[t][i][e] = p[16 * t];
            }
        }
        whole = ws_of(c)[ChunkWs::ge + kChunk - 1];
    };
    load_k(0), load_v(0), load_q(0), load_t(0), load_p(0), load_kt(0);
    const f4 zero{0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < chunks; c++) {
        const int next = min(c + 1, chunks - 1);
#pragma unroll
        for (int t = 0; t < ST; t++) lS[ST * wave + t][lane] = S[t];
        __syncthreads();
        // X = V - diag(e^G) K S
        f4 s0 = zero, s1 = zero;
#pragma unroll
        for (int i = 0; i < KC; i += 2) s0 = mfma4(k[i], lS[i][lane], s0), s1 = mfma4(k[i + 1], lS[i + 1][lane], s1);
        load_k(next);
        f4 x;
        bool ok = true;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[e] = fmaf(-ge[e], s0[e] + s1[e], v[e]);
            ok = ok && finite32(x[e]);
        }
        const int to_bad = first;
        const f4 eg = ge;
        load_v(next);
        lX[wave][lane] = x;
        const bool any = __ballot(!ok) != 0;
        if (lane == 0) lBad[wave] = any;
        s0 = zero, s1 = zero;
#pragma unroll
        for (int i = 0; i < KC; i += 2) s0 = mfma4(q[i], lS[i][lane], s0), s1 = mfma4(q[i + 1], lS[i + 1][lane], s1);
        load_q(next);
        __syncthreads();
        // U = T X
        const bool bad = uniform(lBad[0] | lBad[1] | lBad[2] | lBad[3]) || to_bad < kChunk;
        int stop = to_bad;  // the column's rows from here on are not numbers
        if (bad) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 3; e >= 0; e--)
                    if (!finite32(lX[i][lane][e])) stop = min(stop, 16 * i + 4 * g + e);
            stop = min(stop, __shfl_xor(stop, 16));
            stop = min(stop, __shfl_xor(stop, 32));
        }
        f4 u = zero;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i > wave) continue;
            f4 xi = lX[i][lane];
            if (bad) {
#pragma unroll
                for (int e = 0; e < 4; e++) xi[e] = 16 * i + 4 * g + e < stop ? xi[e] : 0.0f;
            }
            u = mfma4(T[i], xi, u);
        }
        load_t(next);
        lU[wave][lane] = u;
        f4 o;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = eg[e] * a.h.scale * (s0[e] + s1[e]);
        __syncthreads();
        // out and the state
        f4 ub[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ub[i] = lU[i][lane];
            if (i <= wave) o = mfma4(P[i], ub[i], o);
        }
        load_p(next);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int r = 16 * wave + 4 * g + e;
            const float w = bad && r >= stop ? __uint_as_float(0x7FC00000u) : o[e];
            if (c * kChunk + r < s.n) a.out[(((size_t)s.lo + c * kChunk + r) * a.st.nv + head) * HD + col] = w;
        }
#pragma unroll
        for (int t = 0; t < ST; t++) S[t] *= whole;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const f4 ug = ub[i] * gl[i];
#pragma unroll
            for (int t = 0; t < ST; t++) S[t] = mfma4(kt[t][i], ug, S[t]);
        }
        if (bad && stop < kChunk) {
#pragma unroll
            for (int t = 0; t < ST; t++) S[t] = f4{1.f, 1.f, 1.f, 1.f} * __uint_as_float(0x7FC00000u);
        }
        load_kt(next);
    }
    if ((unsigned)to < (unsigned)a.st.n_slots) {
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) a.st.state[(((size_t)to * a.st.nv + head) * HD + state_row(t) + e) * HD + col] = S[t][e];
    }
}

// The epilogue of the rows that went by chunks: a workgroup a chunk and head.
template <int HD>
__global__ __launch_bounds__(256) void gdn_finish_kernel(RuleArgs a) {
    const int head = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Long s = find_long<true>(a.b, (int)blockIdx.x, a.chunked);
    if (s.seq < 0) return;
    const int c0 = ((int)blockIdx.x - s.slot) * kChunk, n = min(kChunk, s.n - c0);
    for (int r = wave; r < n; r += 4) {
        const size_t row = (size_t)s.lo + c0 + r;
        float v[HD / 64];
#pragma unroll
        for (int e = 0; e < HD / 64; e++) v[e] = a.out[(row * a.st.nv + head) * HD + HD / 64 * lane + e];
        finish_row<HD>(a, row, head, v);
    }
}

}  // namespace

hipError_t launch_gdn_conv(const StatesView &st, const BatchView &b, const uq_gdn_rows &r, hipStream_t s) {
    if (b.n_rows == 0 || b.n_seqs == 0) return hipSuccess;
    const ConvArgs a{st, b, r, (st.channels + 255) / 256};
    const unsigned per = kConvTPB / 64, tiles = (unsigned)(b.n_rows / kConvRows + std::min(b.n_seqs, b.n_rows));
    const dim3 grid(tiles, ((unsigned)a.groups + per) / per);
    if (st.taps == 4)
        hipLaunchKernelGGL(gdn_conv_kernel<4>, grid, dim3(kConvTPB), 0, s, a);
    else
        hipLaunchKernelGGL(gdn_conv_kernel<0>, grid, dim3(kConvTPB), 0, s, a);
    return hipGetLastError();
}

// Sequences of this many rows and more go by chunks.
constexpr int kChunkLeast = 32;

namespace {
// How many sequences can go by chunks, and the slots of their chunks; 0 where none is expected to.
struct Plan {
    int longs, slots;
};
Plan plan_of(const BatchView &b, size_t most_rows) {
    if (b.n_rows < kChunkLeast || (most_rows && most_rows < (size_t)kChunkLeast)) return Plan{0, 0};
    const int longs = std::min(b.n_seqs, b.n_rows / kChunkLeast);
    return Plan{longs, b.n_rows / kChunk + longs + 1};
}
}  // namespace

size_t gdn_rule_ws_bytes(const StatesView &st, const BatchView &b, size_t most_rows) {
    return 16 + (size_t)plan_of(b, most_rows).slots * st.nv * kChunkFloats * sizeof(float);
}

template <int HD>
hipError_t launch_rule(RuleArgs a, bool some, hipStream_t s) {
    if (a.longs) {
        const dim3 chunks((unsigned)a.slots, (unsigned)a.st.nv);
        hipLaunchKernelGGL(gdn_prep_kernel<HD>, chunks, dim3(kPrepTPB), 0, s, a);
        if (hipError_t e = hipGetLastError()) return e;
        const long long pairs = (long long)a.longs * a.st.nv, groups = (pairs + 7) / 8 * 8 * (HD / kColumns);
        hipLaunchKernelGGL(gdn_chunks_kernel<HD>, dim3((unsigned)groups), dim3(256), 0, s, a);
        if (hipError_t e = hipGetLastError()) return e;
        if (a.h.d_norm || a.h.d_z) {
            hipLaunchKernelGGL(gdn_finish_kernel<HD>, chunks, dim3(256), 0, s, a);
            if (hipError_t e = hipGetLastError()) return e;
        }
    }
    if (some) {
        hipLaunchKernelGGL(gdn_rows_kernel<HD>, dim3((unsigned)a.st.nv, (unsigned)a.b.n_seqs), dim3(2 * HD), 0, s, a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

hipError_t launch_gdn_rule(float *out, const StatesView &st, const BatchView &b, const uq_gdn_heads &h, size_t most_rows,
                           void *ws, hipStream_t s) {
    if (b.n_rows == 0 || b.n_seqs == 0) return hipSuccess;
    const Plan p = plan_of(b, most_rows);
    const RuleArgs a{out, st, b, h, p.longs ? kChunkLeast : INT_MAX, p.longs, p.slots, (float *)ws};
    return st.hd == 128 ? launch_rule<128>(a, true, s) : launch_rule<64>(a, true, s);
}

}  // namespace uq
