// Attention over paged caches on blocks of many queries (a prompt's chunk, or
// a batch over positions that it shares): 32 queries a wave, 2 or 4 waves a
// block over the same tiles of positions, whose keys and values all waves
// take from LDS.
//
// Matrix products bound it: with two f16 terms 8 HD flops a query and
// position, 2048 matrix cycles a wave and tile of 8192 values, which takes
// 1.92 us at full load (1.1 PFLOP/s; the clock falls to 2.1 GHz). So a wave
// holds as many queries as its registers do (32: their terms, the sums and
// two tiles' scores), LDS is read once for each, and everything else lies in
// the shadow of the products: the first product of tile t + 1 runs while tile
// t's weights are formed, the second takes over while the other half is. A
// tile then costs the LDS 160 KB of a CU's traffic in 4000 cycles. 509 rows of
// 16 heads of 256 values over 4096 positions: 92 us; 48 rows of them over
// 16384 shared positions: 53 us, in two blocks of 128 queries a KV head with
// the second half empty; 25 MB of records written at its end.
#include "uq_attn_paged.h"
#include "uq_mfma.h"

namespace uq {

namespace {

constexpr float kRef = 8.0f;    // weights are held times 2^8 or more (small ones within 2^-25, half the least f16):
constexpr float kMove = 15.0f;  // the reference moves where one would pass 2^15

__device__ __forceinline__ float half_max(float v) {  // over the lanes l, l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// What a wave wrote to LDS, it may read.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The value is formed before this point and used after it: keeps products and the work between them, which no other
// instruction orders, in the steps they are written in.
template <class T>
__device__ __forceinline__ void pin(T &v) {
    __asm__ volatile("" : "+v"(v));
}

// The transposing LDS read: of the 16 lanes' 16 x 4 values, lane i gets value i % 4 of lanes 4 j + i / 4, j < 4. With
// lane 4 r + q at values 4 q .. of row r, that is column i of the four rows.
__device__ __forceinline__ u2 read_columns(const uint8_t *p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(uintptr_t)(
                                      (__attribute__((address_space(3))) uint8_t *)p)));
}

// Tiles of NP positions lie in LDS as rows of HD / 8 pieces of 16 bytes, brought there without passing registers.
// Piece c of row r is at c ^ (r & 7) of the keys, so that the 32 rows of a product's operand lie in different banks,
// and at c ^ 2 (r & 3) of the values, so that the four rows of a transposing read do.
template <int HD, int QW>
struct Many {
    static constexpr int NP = 8192 / HD, ST = NP / 32, KC = HD / 16, DT = HD / 32, KP = NP / 16, RB = 32 * QW, NT = 64 * QW;
    static constexpr int kTile = NP * HD * 2;  // 16 KB
    static constexpr int LI = 16 / QW;         // loads of a wave a tile, 1 KB each
    static constexpr int D = QW == 4 ? 2 : 1;  // iterations that a load has to arrive: what LDS holds, at one workgroup
    static constexpr int NB = D + 1;           // a CU of four waves or two of two
    static constexpr int CT = 2048 / NP;       // tiles whose rows are looked up at a time, and those ahead of them
    static constexpr int AHEAD = D + 3;
    static constexpr int kOver = 7;  // 13 us against 1.9 us a tile
    static constexpr size_t kLds = 2 * NB * kTile;
};

template <int HD, int QW>
__global__ __launch_bounds__(64 * QW, 1) void attn_many_kernel(AttnArgs A) {
    using M = Many<HD, QW>;
    constexpr int NP = M::NP, ST = M::ST, KC = M::KC, DT = M::DT, KP = M::KP, RB = M::RB, NT = M::NT;
    extern __shared__ __align__(1024) uint8_t lds[];   // keys of NB tiles, values of NB
    __shared__ int rows[(M::CT + M::AHEAD) * NP];    // rows of the positions of CT tiles and those ahead, 0 for none
    __shared__ uint32_t have[(M::CT + M::AHEAD) * ST];  // which are
    __shared__ int unfinite;          // some tile holds values that are not finite and that not every query sees
    __shared__ int row_lim[RB];
    __shared__ int red[QW];
    __shared__ WalkLds walk_lds;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int wave = uniform(tid >> 6);
    const int nkv = A.kv.n_head_kv;
    const PageMap &map = A.kv.map;

    Walk<NT, NP, M::kOver, 1> X;
    if (!X.find(A, walk_lds)) return;
    while (X.next(A)) {
        const Work &w = X.w;
        const int seq = X.seq, rb = X.rb, kvh = X.kvh, un = X.un, count = X.count;
        const int nq = min(RB, w.n * A.group - rb * RB);
        const bool active = wave * 32 < nq;

        // ---- the queries' last positions
        __syncthreads();  // the block before is done with LDS
        for (int i = tid; i < RB; i += NT) {
            int lim = -1;
            if (seq >= 0 && i < nq && w.len >= 0) lim = max(-1, w.len - w.n + (rb * RB + i) / A.group);
            row_lim[i] = lim;
        }
        if (seq < 0) {
            __syncthreads();
            const int q0 = rb * RB, q1 = q0 + nq;
            for (int i = tid; i < A.b.n_seqs; i += NT) {
                const SeqRows sr = seq_rows(A.b.row_start[i], A.b.row_start[i + 1], A.b.n_rows);
                const int len = A.b.len[i];
                const int a = max(q0, sr.lo * A.group), b = min(q1, (sr.lo + sr.n) * A.group);
                for (int q = a; q < b; q++) row_lim[q - q0] = len >= 0 ? max(-1, len - sr.n + q / A.group - sr.lo) : -1;
            }
        }
        if (tid == 0) unfinite = 0;
        __syncthreads();
        const int mine = wave * 32 + n, num = rb * RB + mine;
        const bool in = mine < nq;
        const int lim = row_lim[mine];
        int lim_min = in ? lim : INT_MAX;
        lim_min = lanes_min<32>(lim_min);
        if (lane == 0) red[wave] = lim_min;

        // ---- tiles t = 0 .. count - 1 of positions p0 + NP t
        const int first = w.base + un * NP;
        const int32_t *table = A.b.pages + (seq < 0 ? (size_t)0 : (size_t)seq * A.b.max_pages);
        const _Float16 *K = (const _Float16 *)A.kv.k, *V = (const _Float16 *)A.kv.v;
        int cb = 0;  // first of the tiles in rows
        auto look_up = [&]() {
            for (int x = tid; x < (M::CT + M::AHEAD) * NP; x += NT) {
                const int pos = first + cb * NP + x;
                const int page = cb + x / NP < count && pos < w.end ? table[pos >> map.log2_page] : -1;
                const bool ok = page_ok(map, page);
                rows[x] = ok ? page_row(map, page, kvh, pos) : 0;
                const unsigned long long m = __ballot(ok);
                if ((lane & 31) == 0) have[x >> 5] = (uint32_t)(m >> (lane & 32));
            }
        };
        look_up();

        // ---- queries: two f16 terms in the order of the first product's right operand
        // 16 at a time by way of the wave's part of LDS: rows are read whole, and by the lanes of a query from there
        const int at_q = (w.lo + (in ? num / A.group : rb * RB / A.group)) * A.a.n_head + kvh * A.group + (in ? num : rb * RB) % A.group;
        h8 qh[KC], ql[KC];
        float fac;
        uint8_t *const own = lds + wave * 16384;
        {
            constexpr int LQ = HD / 4, RL = 64 / LQ, J = 16 / RL;  // lanes of a query, queries of a load, loads
            int exps = 15;
            f4 vs[2][J];
#pragma unroll
            for (int j = 0; j < 2 * J; j++)
                vs[j / J][j % J] = *(const f4u *)(A.a.q + (size_t)__shfl(at_q, j * RL + lane / LQ) * HD + 4 * (lane % LQ));
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const f4 (&v)[J] = vs[g];
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const int q = j * RL + lane / LQ;
                    uint32_t top = 0;
#pragma unroll
                    for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(v[j][e]) & 0x7FFFFFFFu);
                    top = lanes_max<LQ>(top);
                    // |q| < 2^ex; not finite: left as it is, its terms are not finite either
                    const int ex = top > 0 && top < 0x7F800000u ? __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 15;
                    const int ex_n = __shfl(ex, (n & (RL - 1)) * LQ);  // of query n, where it is of this load
                    if (n >> 4 == g && (n & 15) / RL == j) exps = ex_n;
                    h4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        _Float16 a, b;
                        product_terms(ldexpf(v[j][e], 15 - ex), A.scale_m, a, b);
                        hi[e] = a, lo[e] = b;
                    }
                    uint8_t *to = own + q * HD * 2 + ((((lane % LQ) >> 1) ^ (q & 7)) << 4) + 8 * (lane & 1);
                    *(h4 *)to = hi;
                    *(h4 *)(to + 16 * HD * 2) = lo;
                }
                wave_fence();
                if (n >> 4 == g) {
#pragma unroll
                    for (int c = 0; c < KC; c++) {
                        const uint8_t *from = own + (n & 15) * HD * 2 + (((2 * c + h) ^ (n & 7)) << 4);
                        qh[c] = *(const h8 *)from;
                        ql[c] = *(const h8 *)(from + 16 * HD * 2);
                    }
                }
                wave_fence();
            }
            fac = score_factor(A.scale_e + exps - 15);
        }

        // Tile t into buffer b of the keys or values: LI loads a wave; what is no position brings any row. Their rows
        // are read ahead, so that the LDS answers them all at once.
        auto rows_of = [&](int t, int (&r)[M::LI]) {
#pragma unroll
            for (int i = 0; i < M::LI; i++) r[i] = rows[(t - cb) * NP + ((wave * M::LI + i) * 64 + lane) / (HD / 8)];
        };
        auto address = [](const _Float16 *base, int row, int piece) {  // a row's bytes are a multiple of its pieces'
            constexpr int LG = HD == 64 ? 7 : HD == 128 ? 8 : 9;
            const uint32_t lo = ((uint32_t)row << LG) | (piece << 4), hi = (uint32_t)row >> (32 - LG);
            return (const uint8_t *)base + (((uint64_t)hi << 32) | lo);
        };
        auto load_keys = [&](int i, int r, int b) {
            const int x = (wave * M::LI + i) * 64 + lane, piece = (x % (HD / 8)) ^ ((x / (HD / 8)) & 7);
            dma16(address(K, r, piece), lds + b * M::kTile + (wave * M::LI + i) * 1024);
        };
        auto load_values = [&](int i, int r, int b) {
            const int x = (wave * M::LI + i) * 64 + lane, piece = (x % (HD / 8)) ^ (2 * ((x / (HD / 8)) & 3));
            dma16(address(V, r, piece), lds + (M::NB + b) * M::kTile + (wave * M::LI + i) * 1024);
        };
        auto all_have = [&](int t) {
            uint32_t all = ~0u;
#pragma unroll
            for (int i = 0; i < ST; i++) all &= have[(t - cb) * ST + i];
            return all == ~0u;
        };
        int lim_all = 0;  // the least of the block's, once the waves have met
        // Values of positions that are none become zeros, and so does what is not finite where some query may not
        // see it (it is added at the end for those that do). Every wave is behind a barrier after it.
        auto mend_values = [&](int t, int b, bool full) {
            if (full && first + t * NP + NP - 1 <= lim_all) return;
            for (int x = tid; x < NP * HD / 8; x += NT) {
                u4 *at = (u4 *)(lds + (M::NB + b) * M::kTile) + x;
                const int y = (t - cb) * NP + x / (HD / 8);
                const bool ok = (have[y >> 5] >> (y & 31)) & 1;
                u4 z = *at;
                bool fin = true;
#pragma unroll
                for (int d = 0; d < 4; d++) {
                    const bool lo = (z[d] & 0x7C00u) != 0x7C00u, hi = (z[d] & 0x7C000000u) != 0x7C000000u;
                    fin = fin && lo && hi;
                    z[d] = (ok && lo ? z[d] & 0x0000FFFFu : 0u) | (ok && hi ? z[d] & 0xFFFF0000u : 0u);
                }
                if (!ok || !fin) *at = z;
                if (ok && !fin) unfinite = 1;
            }
            __syncthreads();
        };
        f16x acc[DT], s[ST], sn[ST];
        float a = INFINITY, l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[d][r] = 0.0f;
        h8 ph[KP], pl[KP];
        // The first product in 16 steps of two matrix instructions, its operand read two steps ahead; between(q) is
        // other work in the shadow of step q. Nothing moves from one step to another.
        auto scores = [&](int b, f16x (&o)[ST], auto between) {
            const uint8_t *kb[4];  // pieces 8 x + 2 c + h of row n: a constant apart for every x (and 32 rows on)
#pragma unroll
            for (int c = 0; c < 4; c++) kb[c] = lds + b * M::kTile + n * HD * 2 + (((2 * c + h) ^ (n & 7)) << 4);
            auto at = [&](int q) { return *(const h8 *)(kb[(q / ST) & 3] + 32 * (q % ST) * HD * 2 + (q / ST >> 2) * 128); };
            h8 k[3];
            k[0] = at(0), k[1] = at(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < 16; q++) {
                const int c = q / ST, i = q % ST;
                if (q + 2 < 16) k[(q + 2) % 3] = at(q + 2);
                if (c == 0) {
#pragma unroll
                    for (int r = 0; r < 16; r++) o[i][r] = 0.0f;
                }
                o[i] = mfma(k[q % 3], qh[c], o[i]);
                pin(o[i]);
                between(q);
                o[i] = mfma(k[q % 3], ql[c], o[i]);
                pin(o[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        static_assert(KC * ST == 16 && KP * DT == 16, "16 steps of either product, whatever the head");

        // A tile's scores, their largest given: what a query does not see becomes -infinity, the reference moves where a
        // weight would grow too large (rarely after the first tiles: the sums are multiplied then).
        auto settle = [&](int t, float top, bool full) {
            const int p0 = first + t * NP;
            if (!full || p0 + NP - 1 > lim_min) {
                top = -INFINITY;
#pragma unroll
                for (int i = 0; i < ST; i++) {
                    const uint32_t hv = have[(t - cb) * ST + i] >> (4 * h);
                    const int room = lim - p0 - 32 * i - 4 * h;
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int x = 8 * (r >> 2) + (r & 3);
                        const bool sees = ((hv >> x) & 1) && x <= room;
                        s[i][r] = sees ? s[i][r] : -INFINITY;
                        top = fmaxf(top, s[i][r]);
                    }
                }
            }
            top = half_max(top) * fac;
            const bool move = top + a > kMove;  // not where both are infinite: nothing seen yet
            if (__any(move)) {
                const float na = move ? reference(top, kRef) : a;
                const float corr = move ? exp2_hw(na - a) : 1.0f;
                a = na;
                l *= corr;
#pragma unroll
                for (int d = 0; d < DT; d++) acc[d] *= corr;
            }
        };
        // Two weights and their two terms.
        auto weights = [&](int e, float ref) {
            const float x = exp2_hw(fmaf(s[e >> 4][e & 15], fac, ref)), y = exp2_hw(fmaf(s[e >> 4][(e & 15) + 1], fac, ref));
            l += x;
            l += y;
            const _Float16 hx = (_Float16)x, hy = (_Float16)y;
            ph[e >> 3][e & 7] = hx, ph[e >> 3][(e & 7) + 1] = hy;
            pl[e >> 3][e & 7] = (_Float16)fmaf((float)hx, -1.0f, x), pl[e >> 3][(e & 7) + 1] = (_Float16)fmaf((float)hy, -1.0f, y);
        };

        __syncthreads();
#pragma unroll
        for (int i = 0; i < QW; i++) lim_all = i == 0 ? red[0] : min(lim_all, red[i]);
        int rk[M::LI], rv[M::LI];
        for (int t = 0; t <= M::D; t++) {
            rows_of(t, rk);
#pragma unroll
            for (int i = 0; i < M::LI; i++) {
                load_keys(i, rk[i], t);
                if (t < M::D) load_values(i, rk[i], t);
            }
        }
        wait_vm_barrier<0>();
        bool full = all_have(0);
        mend_values(0, 0, full);
        if (active) {
            scores(0, s, [](int) {});
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < ST; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) top = fmaxf(top, s[i][r]);
            settle(0, top, full);
        }
        rows_of(1 + M::D, rk);
        rows_of(M::D, rv);
        __syncthreads();  // tile 0's keys are read: the first iteration loads over them

        int b0 = 0;  // t % NB
        for (int t = 0; t < count; t++) {
            const int b1 = b0 + 1 == M::NB ? 0 : b0 + 1, bl = b0 == 0 ? M::NB - 1 : b0 - 1;  // of t + 1 and t + D
            // into the buffers of tile t's keys and of tile t - 1's values, which are used up
            auto load = [&](int q) {
                if (q < M::LI)
                    load_keys(q, rk[q], b0);
                else if (q < 2 * M::LI)
                    load_values(q - M::LI, rv[q - M::LI], bl);
            };
            full = all_have(t + 1);
            if (active) {
                // The next tile's scores on the matrix cores (of no tile behind the last: not used), in their shadow the
                // loads and the first half of this tile's weights; then the second product, with the other half (whose
                // slots it reaches after 8 steps) and the next scores' largest.
                const float ref = a == INFINITY ? 0.0f : a;
                scores(b1, sn, [&](int q) {
                    load(q);
                    if (ST == 4)
                        weights(2 * q, ref);
                    else if (q & 1 && q < 8 * ST)
                        weights(q - 1, ref);
                    pin(l);
                });
                // values 32 d .. of positions 16 p + 8 x + 4 h ..: lane 4 r + q of sixteen at value 4 q of row r
                const int vr = 4 * h + ((lane >> 2) & 3), vq = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
                const uint8_t *vb[2];
#pragma unroll
                for (int d = 0; d < 2; d++)
                    vb[d] = lds + (M::NB + b0) * M::kTile + vr * HD * 2 + 8 * (lane & 1) + (((4 * d + vq) ^ (2 * (vr & 3))) << 4);
                auto at = [&](int q) {
                    const int p = q / DT, d = q % DT;
                    const uint8_t *x = vb[d & 1] + 16 * p * HD * 2 + (d >> 1) * 128;
                    const u2 x0 = read_columns(x), x1 = read_columns(x + 8 * HD * 2);
                    return __builtin_bit_cast(h8, u4{x0[0], x0[1], x1[0], x1[1]});
                };
                h8 v[3];
                v[0] = at(0), v[1] = at(1);
                __builtin_amdgcn_sched_barrier(0);
                float top = -INFINITY;
#pragma unroll
                for (int q = 0; q < 16; q++) {
                    const int p = q / DT, d = q % DT;
                    if (q + 2 < 16) v[(q + 2) % 3] = at(q + 2);
                    acc[d] = mfma(v[q % 3], ph[p], acc[d]);
                    pin(acc[d]);
                    if (q < 8) {
                        if constexpr (ST == 1) {
                            if (q & 1) weights(8 + q - 1, ref);
                        } else {
#pragma unroll
                            for (int e = 0; e < ST; e += 2) weights(8 * ST + q * ST + e, ref);
                        }
                        pin(l);
                    } else {
#pragma unroll
                        for (int e = 2 * (q - 8) * ST; e < 2 * (q - 7) * ST; e++) {
                            top = fmaxf(top, sn[e >> 4][e & 15]);
                            s[e >> 4][e & 15] = sn[e >> 4][e & 15];
                        }
                        pin(top);
                    }
                    acc[d] = mfma(v[q % 3], pl[p], acc[d]);
                    pin(acc[d]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (t + 1 < count) settle(t + 1, top, full);
            } else {
#pragma unroll
                for (int q = 0; q < 2 * M::LI; q++) load(q);
            }
            rows_of(t + 2 + M::D, rk);
            rows_of(t + 1 + M::D, rv);
            wait_vm_barrier<(M::D - 1) * 2 * M::LI>();
            if (t + 1 < count) mend_values(t + 1, b1, full);
            if (t + 1 - cb == M::CT && t + 1 < count) {
                __syncthreads();  // the waves are done with the rows of these tiles
                cb = t + 1;
                look_up();
                __syncthreads();
                rows_of(t + 2 + M::D, rk);
                rows_of(t + 1 + M::D, rv);
            }
            b0 = b1;
        }
        wait_vm_barrier<0>();

        // ---- values that are not finite, left out by mend_values because a query that may not see them would take
        // 0 * NaN from them: for the queries that see them (any weight: the sum is infinite or NaN all the same)
        if (unfinite && active) {
            for (int t = 0; t < count; t++) {
                const int p0 = first + t * NP;
                for (int y = 0; y < NP && p0 + y < w.end; y++) {
                    const int page = table[(p0 + y) >> map.log2_page];
                    if (!page_ok(map, page)) continue;
                    const bool sees = p0 + y <= lim;
                    const _Float16 *vp = V + (size_t)page_row(map, page, kvh, p0 + y) * HD;
#pragma unroll
                    for (int d = 0; d < DT; d++) {
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const int m = 8 * (r >> 2) + 4 * h + (r & 3);
                            const float v = (float)vp[32 * d + m];
                            if (sees && !(fabsf(v) < INFINITY)) acc[d][r] += v;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }

        // ---- results
        l += __shfl_xor(l, 32);
        const bool starts = X.starts, whole = starts && X.ends;
        const bool done = whole && A.a.shared_len == 0;
        if (active) {
            // by way of LDS, 128 values of the 32 queries at a time, to store them row by row
            const int idx = done ? at_q
                            : whole ? (int)rec_whole(A, seq >= 0, 0, 0) + at_q
                                    : (int)rec_part(A.part[seq >= 0], X.me, starts, mine);
            const float mul = !done ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            if (!done && in && h == 0) A.rec_al[idx] = make_float2(a, l);
            float *const dst = done ? A.a.out : A.rec_o;
            constexpr int W = HD < 128 ? HD : 128, LW = W / 4, RW = 64 / LW;  // values, lanes of a row, rows of a store
#pragma unroll
            for (int d0 = 0; d0 < HD; d0 += W) {
#pragma unroll
                for (int d = 0; d < W / 32; d++)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f16x &x = acc[d0 / 32 + d];
                        *(f4 *)(own + n * W * 4 + (((8 * d + r / 2 + h) ^ (n & 7)) << 4)) = f4{x[r], x[r + 1], x[r + 2], x[r + 3]} * mul;
                    }
                wave_fence();
                auto store = [&](int j, bool gated) {
                    const int q = j + lane / LW, c = lane % LW;
                    f4 y = *(const f4 *)(own + q * W * 4 + ((c ^ (q & 7)) << 4));
                    const int to = __shfl(idx, q);
                    if (wave * 32 + q >= nq) return;
                    if (gated) {
                        const float *z = A.a.gate + (size_t)(to / A.a.n_head) * A.a.gate_row + (size_t)(to % A.a.n_head) * A.a.gate_head + d0 + 4 * c;
#pragma unroll
                        for (int e = 0; e < 4; e++) y[e] *= sigmoid1(z[e]);
                    }
                    *(f4u *)(dst + (size_t)to * HD + d0 + 4 * c) = y;
                };
                if (done && A.a.gate) {
#pragma unroll 1
                    for (int j = 0; j < 32; j += RW) store(j, true);
                } else {
#pragma unroll 8
                    for (int j = 0; j < 32; j += RW) store(j, false);
                }
                wave_fence();
            }
        }
        if (starts && tid < nq) {  // a block has half as many queries as the workgroup threads
            const int num = rb * RB + tid;
            put_seg(A, seq >= 0, w.lo + num / A.group, kvh * A.group + num % A.group,
                    done ? kDone : whole ? kWhole : X.me,
                    done || whole ? 0 : X.last(), tid);
        }
    }
}

template <int HD, int QW>
hipError_t launch(const AttnArgs &A, hipStream_t s) {
    auto *k = attn_many_kernel<HD, QW>;
    if (hipError_t e = allow_lds((const void *)k, Many<HD, QW>::kLds)) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)A.part[A.first].G), dim3(64 * QW), (Many<HD, QW>::kLds), s, A);
    return hipGetLastError();
}

}  // namespace

bool attn_many_ok(const PagesView &kv) {
    return kv.f16 && kv.head_dim <= 256 && kv.map.n_pages > 0;  // head_dim 512: its sums do not fit a wave's registers
}

hipError_t launch_attn_many(const AttnArgs &A, hipStream_t s) {
    const int rows = A.part[A.first].rows;
    if (!attn_many_ok(A.kv) || (rows != 64 && rows != 128)) return hipErrorInvalidValue;
    switch (A.kv.head_dim) {
    case 64: return rows == 64 ? launch<64, 2>(A, s) : launch<64, 4>(A, s);
    case 128: return rows == 64 ? launch<128, 2>(A, s) : launch<128, 4>(A, s);
    case 256: return rows == 64 ? launch<256, 2>(A, s) : launch<256, 4>(A, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace uq
