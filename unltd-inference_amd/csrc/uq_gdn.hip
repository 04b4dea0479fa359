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
    int chunked;  // sequences of at least so many rows go by chunks
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

size_t gdn_rule_ws_bytes(const StatesView &st, const BatchView &b, size_t most_rows) { return 16; }

hipError_t launch_gdn_rule(float *out, const StatesView &st, const BatchView &b, const uq_gdn_heads &h, size_t most_rows,
                           void *ws, hipStream_t s) {
    if (b.n_rows == 0 || b.n_seqs == 0) return hipSuccess;
    const RuleArgs a{out, st, b, h, INT_MAX};
    const dim3 grid((unsigned)st.nv, (unsigned)b.n_seqs);
    if (st.hd == 128)
        hipLaunchKernelGGL(gdn_rows_kernel<128>, grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(gdn_rows_kernel<64>, grid, dim3(128), 0, s, a);
    return hipGetLastError();
}

}  // namespace uq
