// Attention of a batch's rows over a paged cache (uq_attn_paged_d).
//
// With scores s[p] = kq_scale q.K[p] of a query, one pass over the keys keeps
// a reference a and the sums
//     l = sum 2^(s[p] log2 e + a),   o = sum 2^(s[p] log2 e + a) V[p],
// where -a follows the largest s log2 e seen so far (o and l are multiplied by
// 2^(a' - a) when it moves), and the result is o / l. Parts over other
// positions join the same way.
//
// Few queries: the cache is read from memory once for 16 or 32 queries of a
// KV head, so that bounds it where there is much of it (65536 positions of 4
// KV heads of 256 f32 values: 5.1 TB/s with the start and end, 6.2 in the
// loop); where there is little, its round trips do: lengths, page numbers,
// tiles, the waves' sums (one tile a wave: 8 to 12 us).
#include <cmath>

#include "uq_attn_paged.h"

namespace uq {

namespace {

constexpr int kTPB = 256;
constexpr int kWaves = kTPB / 64;
constexpr int kCUs = 256;
// Workgroups of attn_paged_kernel a CU: its registers' (32 queries of 256 values: 128 for the sums alone) and LDS's limit.
constexpr int few_per_cu(int hd, int rt) { return hd == 512 || (hd == 256 && rt == 2) ? 1 : 2; }
constexpr int kOver = 3;           // a block's start and end in tiles: 8 us against 2.7 us a tile at full load

template <bool F16, int HD>
struct Geo;
// f16 cache: tiles of 32 positions, 16x16x32 products; a lane holds 8
// consecutive values of K, 8 (HD 64: 4) of V.
template <int HD>
struct Geo<true, HD> {
    static constexpr int NP = 32, PT = 2, KC = HD / 32, DL = HD == 64 ? 4 : 8, NH = HD / (16 * DL), VS = 8;
};
// f32 cache: tiles of 16 positions, 16x16x4 products; 4 consecutive values.
template <int HD>
struct Geo<false, HD> {
    static constexpr int NP = 16, PT = 1, KC = HD / 16, DL = 4, NH = HD / 64, VS = 4;
};

// Over the lanes l, l ^ 16, l ^ 32, l ^ 48.
template <class Op>
__device__ __forceinline__ float rows16(float v, Op op) {
    auto two = [&](const auto &r) { return op(__uint_as_float(r[0]), __uint_as_float(r[1])); };
    v = two(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return two(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}
__device__ __forceinline__ float row16_max(float v) {
    return rows16(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float row16_sum(float v) {
    return rows16(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ bool finite32(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

// A wave's part of a block: scores, running reference and sums over its
// tiles of the positions.
//
// Scores are formed transposed, S^T = K Q^T (16 positions x 16 queries a
// tile), so that a lane holds one query's scores (column n = lane & 15) of
// positions 4 (lane >> 4) + i; with the position order of the second
// product's depth chosen to match (slot 8 g + j of a 32-deep product is
// position 4 g + j of tile j / 4), the weights are its right operand where
// they are, and o^T = V^T P^T (values x queries) needs V's values of 8
// positions a lane: rows are loaded 16 bytes a lane and paired by v_perm, one
// a register. No value crosses lanes but the maximum and row numbers.
//
// f16 cache: a query is scaled by a power of two to at most 2^15, times the
// mantissa of the scale and log2 e, and split into two f16 terms, a weight
// (times 2^14) likewise: within 2^-22 of the value and half a step of the least
// f16, 2^-38 of a query's largest value (held at 2^13 or more) and 2^-39 of the
// largest weight. Products are exact and summed in f32. f32 cache: the f32
// matrix products.
//
// RT is 1 or 2: of 16 or 32 queries of a KV head, columns n and n + 16.
template <bool F16, int HD, int RT>
struct Wave {
    using G = Geo<F16, HD>;
    f4 acc[RT][G::NH][G::DL];
    float a[RT], l[RT];  // reference, this lane's share of l

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int y = 0; y < RT; y++) {
#pragma unroll
            for (int h = 0; h < G::NH; h++)
#pragma unroll
                for (int j = 0; j < G::DL; j++) acc[y][h][j] = f4{0.f, 0.f, 0.f, 0.f};
            a[y] = INFINITY;
            l[y] = 0.0f;
        }
    }
};

template <bool F16, int HD>
struct Tile {
    using G = Geo<F16, HD>;
    using KV = std::conditional_t<F16, h8, f4>;
    using VV = std::conditional_t<!F16, f4, std::conditional_t<G::DL == 8, u4, u2>>;
    KV k[G::PT][G::KC];
    VV v[G::VS][G::NH];
};
// A tile's first position, the row of position lane & (NP - 1), the lanes
// whose position exists.
struct Place {
    int p0, row;
    unsigned long long have;
};

template <bool F16, int HD, int RT>
__global__ __launch_bounds__(kTPB, few_per_cu(HD, RT)) void attn_paged_kernel(AttnArgs A) {
    using G = Geo<F16, HD>;
    using E = std::conditional_t<F16, _Float16, float>;
    constexpr int NP = G::NP, MS = HD + 4, ROWS = 16 * RT;  // a unit is a wave's tile
    constexpr float kShift = F16 ? 14.0f : 0.0f;
    extern __shared__ __align__(1024) uint8_t lds[];  // the block's queries; the waves' sums at its end
    __shared__ float row_c[ROWS];         // factor of a query's scores, a power of two (times log2 e)
    __shared__ int row_lim[ROWS];         // its last position, -1: none
    __shared__ float2 wave_al[kWaves][ROWS];
    __shared__ WalkLds walk_lds;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = uniform(tid >> 6);
    const int nkv = A.kv.n_head_kv;
    const PageMap &map = A.kv.map;

    Walk<kTPB, NP, kOver, kWaves> X;
    if (!X.find(A, walk_lds)) return;
    Wave<F16, HD, RT> W;
    while (X.next(A)) {
        const Work &w = X.w;
        const int seq = X.seq, rb = X.rb, kvh = X.kvh, un = X.un, nq = min(ROWS, w.n * A.group - rb * ROWS);
        // the last position that a query of the block sees, for all that is known without its rows
        const int seen = seq < 0 ? INT_MAX - 1 : w.len - w.n + (rb * ROWS + nq - 1) / A.group;
        const int end = min(w.end, max(0, seen + 1));
        const int count = min(X.count, max(0, (end - w.base + NP - 1) / NP - un));
        const int32_t *table = A.b.pages + (seq < 0 ? (size_t)0 : (size_t)seq * A.b.max_pages);
        const E *K = (const E *)A.kv.k, *V = (const E *)A.kv.v;
        auto page_of = [&](int it) {  // of position lane & (NP - 1) of tile it
            const int pos = w.base + (un + it) * NP + (lane & (NP - 1));
            return it < count && pos < end ? page_at(A, table, pos) : -1;
        };
        int page = page_of(wave), ahead = page_of(wave + kWaves);  // on their way while the queries are

        // ---- the block's queries into LDS, in the order of the products' right operand
        __syncthreads();  // the waves' sums of the block before are read
#pragma unroll
        for (int y = 0; y < RT; y++) {
            const int r = (tid >> 4) + 16 * y, part = tid & 15, num = rb * ROWS + r;
            const bool in = r < nq;
            const int row = w.lo + (in ? num / A.group : 0);
            const float *q = A.a.q + ((size_t)row * A.a.n_head + (size_t)kvh * A.group + (in ? num % A.group : 0)) * HD;
            if (seq < 0) {
                if (part == 0) row_lim[r] = -1;
            } else if (part == 0) {
                row_lim[r] = in && w.len >= 0 ? max(-1, w.len - w.n + (row - w.lo)) : -1;
            }
            float fac = score_factor(A.scale_e);
            if constexpr (F16) {
                constexpr int C = (HD / 8 + 15) / 16;
                float v[C][8];
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const int ch = part + 16 * c;
                    const bool has = in && ch < HD / 8;
#pragma unroll
                    for (int x = 0; x < 8; x += 4) {
                        const f4u f = has ? *(const f4u *)(q + 8 * ch + x) : f4u{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            v[c][x + e] = f[e];
                            top = max(top, __float_as_uint(f[e]) & 0x7FFFFFFFu);
                        }
                    }
                }
                top = lanes_max<16>(top);
                // |q| < 2^ex; not finite: left as it is, its terms are not finite either
                const int ex = top > 0 && top < 0x7F800000u ? __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 15;
                fac = score_factor(A.scale_e + ex - 15);
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const int ch = part + 16 * c;
                    h8 hi, lo;
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        _Float16 a, b;
                        product_terms(ldexpf(v[c][x], 15 - ex), A.scale_m, a, b);
                        hi[x] = a, lo[x] = b;
                    }
                    if (ch < HD / 8) {
                        h8 *dst = (h8 *)lds + y * HD * 4 + (ch >> 2) * 128 + (ch & 3) * 16 + (r & 15);
                        dst[0] = hi;
                        dst[64] = lo;
                    }
                }
            } else {
                const float m = ldexpf(A.scale_m, A.scale_e - min(127, max(-126, A.scale_e)));  // what the factor leaves
#pragma unroll
                for (int c = 0; c < HD / 64; c++) {
                    const int ch = part + 16 * c;
                    ((f4 *)lds)[y * HD * 4 + (ch >> 2) * 64 + (ch & 3) * 16 + (r & 15)] = in ? (f4) * (const f4u *)(q + 4 * ch) * m : f4{0.f, 0.f, 0.f, 0.f};
                }
            }
            if (part == 0) row_c[r] = fac;
            if (seq < 0) {  // the block's rows are of any sequences: each row's is looked for by 16 threads
                __syncthreads();
                for (int i = part; in && i < A.b.n_seqs; i += 16) {
                    const SeqRows sr = seq_rows(A.b.row_start[i], A.b.row_start[i + 1], A.b.n_rows);
                    if (row < sr.lo || row >= sr.lo + sr.n) continue;
                    const int len = A.b.len[i];
                    row_lim[r] = len >= 0 ? max(-1, len - sr.n + (row - sr.lo)) : -1;
                }
            }
        }
        __syncthreads();
        int lim[RT], lim_min = INT_MAX;
        float fac[RT];
#pragma unroll
        for (int y = 0; y < RT; y++) {
            lim[y] = row_lim[n + 16 * y];
            fac[y] = row_c[n + 16 * y];
            if (n + 16 * y < nq) lim_min = min(lim_min, lim[y]);
        }
        lim_min = uniform(lanes_min<16>(lim_min));
        W.reset();
        bool unfinite = false;  // values that are not finite were left out where some query may not see them
        // A tile's keys and values in registers. The next tile's keys are on their way while this one's values are
        // multiplied, and its values while its own keys are, in the same registers; the loads are issued without a
        // branch (what is no position loads any row), so that they need not be waited for at one.
        Tile<F16, HD> T;
        auto place = [&](Place &x, int it, int page) {
            const bool there = page_ok(map, page);
            x.p0 = w.base + (un + it) * NP;
            x.row = there ? page_row(map, page, kvh, x.p0 + (lane & (NP - 1))) : 0;
            x.have = __ballot(there);
        };
        auto row_at = [](const Place &x, int lane4, int more) {  // of lane lane4 / 4 + more
            return __builtin_amdgcn_ds_bpermute(lane4 + 4 * more, x.row);
        };
        auto fetch_keys = [&](const Place &x) {
            using KV = typename Tile<F16, HD>::KV;
#pragma unroll
            for (int t = 0; t < G::PT; t++) {
                const KV *kp = (const KV *)(K + (size_t)row_at(x, 4 * n, 16 * t) * HD) + g;
#pragma unroll
                for (int c = 0; c < G::KC; c++) T.k[t][c] = kp[4 * c];
            }
        };
        auto fetch_values = [&](const Place &x) {
            using VV = typename Tile<F16, HD>::VV;
#pragma unroll
            for (int i = 0; i < G::VS; i++) {
                const E *vp = V + (size_t)row_at(x, 16 * g, 16 * (i >> 2) + (i & 3)) * HD + G::DL * n;
#pragma unroll
                for (int h = 0; h < G::NH; h++) T.v[i][h] = *(const VV *)(vp + 16 * G::DL * h);
            }
        };
        if (map.n_pages > 0 && wave < count) {  // else there is nothing to load from, or for
          Place cur, nxt;
          place(cur, wave, page);
          fetch_keys(cur);
          fetch_values(cur);
          for (int it = wave; it < count; it += kWaves) {
            place(nxt, it + kWaves, ahead);
            ahead = page_of(it + 2 * kWaves);
            const unsigned long long have = cur.have;
            const int p0 = cur.p0;
            const bool edge = have != ~0ull || p0 + NP - 1 > lim_min;
            const uint32_t hv = (uint32_t)have >> (4 * g);  // bit 16 t + i: position 16 t + 4 g + i

            // scores, in two sums (f32: four, of a piece's four values): each rounds fewer terms at smaller size (f16, 256
            // values, 8000 positions: off by 5.1e-7 of the result, one sum 7.7e-7; f32: 5.2e-7, 1.3e-6; no slower)
            f4 s[RT][G::PT], more[RT][F16 ? G::PT : 3];
#pragma unroll
            for (int y = 0; y < RT; y++)
#pragma unroll
                for (int t = 0; t < G::PT; t++) s[y][t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = 0; y < RT; y++)
#pragma unroll
                for (int e = 0; e < (F16 ? G::PT : 3); e++) more[y][e] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < G::KC; c++)
#pragma unroll
                for (int y = 0; y < RT; y++) {
                    if constexpr (F16) {
                        const h8 *q = (const h8 *)lds + y * HD * 4 + c * 128 + lane;
                        const h8 qh = q[0], ql = q[64];
#pragma unroll
                        for (int t = 0; t < G::PT; t++) {
                            f4 &to = c % 2 ? more[y][t] : s[y][t];
                            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(T.k[t][c], qh, to, 0, 0, 0);
                            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(T.k[t][c], ql, to, 0, 0, 0);
                        }
                    } else {
                        const f4 q = ((const f4 *)lds)[y * HD * 4 + c * 64 + lane];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            f4 &to = e == 0 ? s[y][0] : more[y][e - 1];
                            to = __builtin_amdgcn_mfma_f32_16x16x4f32(T.k[0][c][e], q[e], to, 0, 0, 0);
                        }
                    }
                }
            if constexpr (F16) {
#pragma unroll
                for (int y = 0; y < RT; y++)
#pragma unroll
                    for (int t = 0; t < G::PT; t++) s[y][t] += more[y][t];
            } else {
#pragma unroll
                for (int y = 0; y < RT; y++) s[y][0] = (s[y][0] + more[y][0]) + (more[y][1] + more[y][2]);
            }

            __builtin_amdgcn_sched_barrier(0);
            fetch_keys(nxt);
            __builtin_amdgcn_sched_barrier(0);

            // weights: slot x = 4 t + i is position p0 + 16 t + 4 g + i
            float p[RT][4 * G::PT];
#pragma unroll
            for (int y = 0; y < RT; y++) {
                const int room = lim[y] - p0 - 4 * g;
                if (edge) {
#pragma unroll
                    for (int t = 0; t < G::PT; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            s[y][t][i] = ((hv >> (16 * t + i)) & 1) & (uint32_t)(16 * t + i <= room) ? s[y][t][i] : -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int t = 0; t < G::PT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) top = fmaxf(top, s[y][t][i]);
                top = row16_max(top) * fac[y];
                const float na = fminf(W.a[y], kShift == 0.0f ? -top : reference(top, kShift));
                const float corr = na == INFINITY ? 1.0f : exp2_hw(na - W.a[y]);
                W.a[y] = na;
                W.l[y] *= corr;
#pragma unroll
                for (int t = 0; t < G::PT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // no score above -infinity: no weight, but a NaN stays one
                        const float z = s[y][t][i];
                        const float v = na == INFINITY ? (z == z ? 0.0f : z) : exp2_hw(fmaf(z, fac[y], na));
                        p[y][4 * t + i] = v;
                        W.l[y] += v;
                    }
#pragma unroll
                for (int h = 0; h < G::NH; h++)
#pragma unroll
                    for (int j = 0; j < G::DL; j++) W.acc[y][h][j] *= corr;
            }

            // values: slot x of a lane is position p0 + 16 (x / 4) + 4 g + x % 4
            if constexpr (F16) {
                constexpr int D2 = G::DL / 2;
                auto &v = T.v;
                if (edge) {
#pragma unroll
                    for (int x = 0; x < G::VS; x++) {
                        const bool ok = (hv >> (16 * (x >> 2) + (x & 3))) & 1;
                        bool fin = true;
#pragma unroll
                        for (int h = 0; h < G::NH; h++)
#pragma unroll
                            for (int d = 0; d < D2; d++) {
                                const uint32_t z = v[x][h][d];
                                const bool lo = (z & 0x7C00u) != 0x7C00u, hi = (z & 0x7C000000u) != 0x7C000000u;
                                fin = fin && lo && hi;
                                v[x][h][d] = (ok && lo ? z & 0x0000FFFFu : 0u) | (ok && hi ? z & 0xFFFF0000u : 0u);
                            }
                        unfinite = unfinite || (ok && !fin);
                    }
                }
                h8 ph[RT], pl[RT];
#pragma unroll
                for (int y = 0; y < RT; y++)
#pragma unroll
                    for (int x = 0; x < 8; x++) {
                        ph[y][x] = (_Float16)p[y][x];
                        pl[y][x] = (_Float16)(p[y][x] - (float)ph[y][x]);
                    }
#pragma unroll
                for (int h = 0; h < G::NH; h++)
#pragma unroll
                    for (int j = 0; j < G::DL; j++) {
                        u4 f;
#pragma unroll
                        for (int x = 0; x < 4; x++)
                            f[x] = __builtin_amdgcn_perm(v[2 * x + 1][h][j >> 1], v[2 * x][h][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
                        const h8 vf = __builtin_bit_cast(h8, f);
#pragma unroll
                        for (int y = 0; y < RT; y++) {
                            W.acc[y][h][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[y], W.acc[y][h][j], 0, 0, 0);
                            W.acc[y][h][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[y], W.acc[y][h][j], 0, 0, 0);
                        }
                    }
            } else {
                auto &v = T.v;
                if (edge) {
#pragma unroll
                    for (int x = 0; x < G::VS; x++) {
                        const bool ok = (hv >> x) & 1;
                        bool fin = true;
#pragma unroll
                        for (int h = 0; h < G::NH; h++)
#pragma unroll
                            for (int d = 0; d < 4; d++) {
                                const bool one = finite32(v[x][h][d]);
                                fin = fin && one;
                                v[x][h][d] = ok && one ? v[x][h][d] : 0.0f;
                            }
                        unfinite = unfinite || (ok && !fin);
                    }
                }
#pragma unroll
                for (int x = 0; x < G::VS; x++)
#pragma unroll
                    for (int h = 0; h < G::NH; h++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int y = 0; y < RT; y++)
                                W.acc[y][h][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[x][h][j], p[y][x], W.acc[y][h][j], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            fetch_values(nxt);
            cur = nxt;
          }
          if (__any(unfinite)) {
              // A query that may not see them would have taken 0 * NaN from them; those that do take them now (any
              // weight: the sum is infinite or NaN all the same).
              for (int it = wave; it < count; it += kWaves)
                  for (int x = 0; x < NP; x++) {
                      const int pos = w.base + (un + it) * NP + x;
                      const int pg = pos < end ? page_at(A, table, pos) : -1;
                      if (!page_ok(map, pg)) continue;
                      const E *vp = V + (size_t)page_row(map, pg, kvh, pos) * HD;
#pragma unroll
                      for (int h = 0; h < G::NH; h++)
#pragma unroll
                          for (int i = 0; i < 4; i++) {
#pragma unroll
                              for (int j = 0; j < G::DL; j++) {
                                  const float v = (float)vp[h * 16 * G::DL + (4 * g + i) * G::DL + j];
#pragma unroll
                                  for (int y = 0; y < RT; y++)
                                      if (pos <= lim[y] && !finite32(v)) W.acc[y][h][j][i] += v;
                              }
                              __builtin_amdgcn_sched_barrier(0);
                          }
                  }
          }
        }

        // ---- the waves' sums joined: references, then o scaled to the least of them
#pragma unroll
        for (int y = 0; y < RT; y++) {
            W.l[y] = row16_sum(W.l[y]);
            if (lane < 16) wave_al[wave][lane + 16 * y] = make_float2(W.a[y], W.l[y]);
        }
        __syncthreads();  // also: every wave is done with the queries in LDS
        float *sums = (float *)lds + (size_t)wave * ROWS * MS;
#pragma unroll
        for (int y = 0; y < RT; y++) {
            const int q = n + 16 * y;
            float amin = INFINITY;
#pragma unroll
            for (int i = 0; i < kWaves; i++) amin = fminf(amin, wave_al[i][q].x);
            const float to = W.a[y] == INFINITY ? 0.0f : exp2_hw(amin - W.a[y]);
            if (q < nq) {
#pragma unroll
                for (int h = 0; h < G::NH; h++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < G::DL; j += 4) {
                            const f4 *o = W.acc[y][h];
                            *(f4 *)(sums + q * MS + h * 16 * G::DL + (4 * g + i) * G::DL + j) =
                                f4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]} * to;
                        }
            }
        }
        __syncthreads();
        const bool starts = X.starts, whole = starts && X.ends, done = whole && A.a.shared_len == 0;
        for (int x = tid; x < nq * (HD / 4); x += kTPB) {
            const int r = x / (HD / 4), d = x % (HD / 4) * 4, num = rb * ROWS + r;
            float ar = INFINITY, lr = 0.0f;
            f4 o = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kWaves; i++) ar = fminf(ar, wave_al[i][r].x);
#pragma unroll
            for (int i = 0; i < kWaves; i++) {
                const float2 al = wave_al[i][r];
                lr += al.y * (al.x == INFINITY ? 0.0f : exp2_hw(ar - al.x));  // l is NaN where it says so
                o += *(const f4 *)((const float *)lds + ((size_t)i * ROWS + r) * MS + d);
            }
            const int row = w.lo + num / A.group, head = kvh * A.group + num % A.group;
            if (done) {
                const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
                f4 y = o * inv;
                if (A.a.gate) {
                    const float *z = A.a.gate + (size_t)row * A.a.gate_row + (size_t)head * A.a.gate_head + d;
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] *= sigmoid1(z[e]);
                }
                *(f4u *)(A.a.out + ((size_t)row * A.a.n_head + head) * HD + d) = y;
            } else {
                const size_t rec = whole ? rec_whole(A, seq >= 0, row, head) : rec_part(A.part[seq >= 0], X.me, starts, r);
                *(f4 *)(A.rec_o + rec * HD + d) = o;
                if (d == 0) A.rec_al[rec] = make_float2(ar, lr);
            }
        }
        if (starts && !A.alone && tid < nq) {
            const int num = rb * ROWS + tid;
            put_seg(A, seq >= 0, w.lo + num / A.group, kvh * A.group + num % A.group,
                    done ? kDone : whole ? kWhole : X.me, done || whole ? 0 : X.last(), tid);
        }
    }
}

template <int E>
struct Floats {
    typedef float V __attribute__((ext_vector_type(E)));
    typedef float At __attribute__((ext_vector_type(E), aligned(4)));  // from any float on
};
template <>
struct Floats<1> {
    typedef float V, At;
};

// Joins the records of a row and head (its part of the shared positions, then
// its own) where the workgroups have not written the result themselves: the
// least reference first, then the sums. What it takes is round trips (row
// starts, lengths and seg; references; then a wave's records one after
// another, two trips each: the part's base and rows from the arguments, and
// the record), so a row and head has a workgroup of 16 or 4 waves that take
// every 16th or 4th record while there are few of them, and one wave of a
// workgroup's four where there are many with few records. 16 pairs of 6 records: 5 us, of 128: 12; 8144 pairs of 4
// or 5: 14.5 us (37 MB read, 8 written).
template <int HD, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void attn_join_kernel(AttnArgs A, int pairs) {
    constexpr int E = HD / 64, PER = WAVES == 1 ? 4 : 1;  // values of a lane, pairs of a workgroup
    using Values = typename Floats<E>::V;
    using ValuesAt = typename Floats<E>::At;
    __shared__ float red[WAVES], redl[WAVES];
    __shared__ __align__(32) float part[WAVES][WAVES == 1 ? 1 : HD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int pair = (int)blockIdx.x * PER + (WAVES == 1 ? wave : 0);
    if (pair >= pairs) return;  // a wave by itself (WAVES 1), else none
    const int row = pair / A.a.n_head, head = pair % A.a.n_head;
    int2 sg[2];
#pragma unroll
    for (int c = 0; c < 2; c++) sg[c] = A.seg[((size_t)c * A.b.n_rows + row) * A.a.n_head + head];
    int seq = -1, len = 0;
    SeqRows its{0, 0};
    for (int i0 = 0; i0 < A.b.n_seqs && seq < 0; i0 += 64) {
        const int i = i0 + lane;
        SeqRows r{0, 0};
        int l = 0;
        if (i < A.b.n_seqs) {
            r = seq_rows(A.b.row_start[i], A.b.row_start[i + 1], A.b.n_rows);
            l = A.b.len[i];
        }
        const unsigned long long any = __ballot(row >= r.lo && row < r.lo + r.n);
        if (any) {
            const int at = __builtin_ctzll(any);
            seq = i0 + at;
            its = SeqRows{__builtin_amdgcn_readlane(r.lo, at), __builtin_amdgcn_readlane(r.n, at)};
            len = __builtin_amdgcn_readlane(l, at);
        }
    }
    if (seq < 0) return;
    // the two parts: records first .. first + count - 1 of workgroups, or one whole record
    int count[2] = {0, 0}, first[2] = {0, 0}, slot[2] = {0, 0};
#pragma unroll
    for (int c = 0; c < 2; c++) {
        if (c == 0 && A.a.shared_len == 0) continue;
        if (c == 1) {
            const Work w = work_of<1>(A, seq, its, len);
            const int num = (row - w.lo) * A.group + head % A.group;
            if (w.units == 0 || seen_units<1>(A, w, num / A.part[1].rows) == 0) continue;
        }
        const int last = min(sg[c].y >> 8, A.part[c].G - 1);
        if (sg[c].x == kDone) return;
        first[c] = sg[c].x;
        slot[c] = min(sg[c].y & 255, A.part[c].rows - 1);
        count[c] = first[c] == kWhole ? 1 : first[c] < 0 ? 0 : max(0, last - first[c] + 1);
    }
    const int total = count[0] + count[1];
    auto rec = [&](int i) {
        const int c = i >= count[0], k = c ? i - count[0] : i;
        return first[c] == kWhole ? rec_whole(A, c, row, head) : rec_part(A.part[c], first[c] + k, k == 0, slot[c]);
    };
    const int begin = WAVES == 1 ? 0 : wave;
    // the references of 64 records of this wave at a time
    const int at0 = begin + WAVES * lane;
    const float2 al0 = at0 < total ? A.rec_al[rec(at0)] : make_float2(INFINITY, 0.0f);
    float amin = al0.x;
    for (int i = at0 + 64 * WAVES; i < total; i += 64 * WAVES) amin = fminf(amin, A.rec_al[rec(i)].x);
    amin = lanes_min<64>(amin);
    if constexpr (WAVES > 1) {
        if (lane == 0) red[wave] = amin;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; i++) amin = fminf(amin, red[i]);
    }
    float l = 0.0f;
    Values o = (Values)0.0f;
    for (int i0 = begin; i0 < total; i0 += 64 * WAVES) {
        const int mine = i0 + WAVES * lane;
        float f = 0.0f;
        if (mine < total) {
            const float2 al = i0 == begin ? al0 : A.rec_al[rec(mine)];
            f = al.x == INFINITY ? 0.0f : exp2_hw(amin - al.x);
            l += f * al.y;
        }
        const int n = min(64, (total - i0 + WAVES - 1) / WAVES);
        for (int k = 0; k < n; k++) {
            const Values x = *(const Values *)(A.rec_o + rec(i0 + WAVES * k) * HD + E * lane);
            const float fk = __int_as_float(lane_of(__float_as_int(f), k));
            o += fk * x;
        }
    }
    l = wave_sum(l);
    if constexpr (WAVES > 1) {
        if (lane == 0) redl[wave] = l;
        *(Values *)&part[wave][E * lane] = o;
        __syncthreads();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < WAVES; i++) l += redl[i];
        for (int d = threadIdx.x; d < HD; d += 64 * WAVES) {
            float y = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; i++) y += part[i][d];
            y = l == 0.0f ? 0.0f : y * (1.0f / l);
            if (A.a.gate) y *= sigmoid1(A.a.gate[(size_t)row * A.a.gate_row + (size_t)head * A.a.gate_head + d]);
            A.a.out[((size_t)row * A.a.n_head + head) * HD + d] = y;
        }
    } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        Values y = l == 0.0f ? (Values)0.0f : o * inv;
        if (A.a.gate) {
            const ValuesAt z = *(const ValuesAt *)(A.a.gate + (size_t)row * A.a.gate_row + (size_t)head * A.a.gate_head + E * lane);
            if constexpr (E == 1) {
                y *= sigmoid1(z);
            } else {
#pragma unroll
                for (int e = 0; e < E; e++) y[e] *= sigmoid1(z[e]);
            }
        }
        *(ValuesAt *)(A.a.out + ((size_t)row * A.a.n_head + head) * HD + E * lane) = y;
    }
}

// The workspace's parts, and how the parts of the work are launched.
struct Plan {
    size_t al, seg, bytes;
    bool apart;  // the shared positions in a launch of their own
    AttnArgs A;
};

// Queries of a block for the R queries of a KV head of one of n_seqs sequences
// (the mean) over at most `positions`: 64 or 128 on attn_many_kernel, else 16
// or 32 on attn_paged_kernel. 32 read the cache half as often (us, 16 | 32;
// f16, 32 sequences of 20 queries: 79 | 68; f32, of 40: 117 | 106; 509 rows of
// one, f32: 500 | 370; 48 rows with 16384 shared, f32: 300 | 180), but
//  - take longer over few tiles (`few` a CU), and so does attn_many_kernel: f16,
//    chunks of 33 rows of 4 heads of 256 values over 1500 positions: 35 with
//    16, 40; over 4096: 52, 42; of 128 values, 129 rows over 1500: 28, 30; 200:
//    34, 31. The more where shared positions need a launch apart from own ones
//    in blocks of 16: 25 rows of 16 heads of 128 values, 3000: 29, 43; 48 rows,
//    4000: 43, 47; 20 rows of 32 heads, 16000: 89, 58. f32, 14 rows of 12
//    heads, 12000: 43, 50; 20000: 65, 61;
//  - leave a CU one workgroup for 256 f32 values, which reads too slowly from
//    memory unless the blocks are of one or two sequences (32 sequences of 64
//    queries: 220 | 274; 8 of 256: 345 | 382; 2 of 1024: 655 | 458).
int block_rows(const PagesView &kv, size_t R, int n_seqs, size_t positions, bool shared) {
    const size_t tiles = n_seqs * ((R + 15) / 16) * kv.n_head_kv * (positions / (kv.f16 ? 32 : 16));  // of 16 queries
    const size_t few = kv.f16 ? shared ? 28 : std::min(20, 2048 / kv.head_dim) : shared ? 64 : 28;
    if (R <= 16 || kv.head_dim == 512 || tiles < few * kCUs) return 16;
    if (R > 32 && attn_many_ok(kv)) return R > 64 ? 128 : 64;
    return !kv.f16 && kv.head_dim == 256 && n_seqs > 2 ? 16 : 32;
}
int block_groups(const PagesView &kv, int rows) {
    if (rows <= 32) return kCUs * few_per_cu(kv.head_dim, rows / 16);
    return rows == 64 ? 2 * kCUs : kCUs;  // 2 or 4 waves, a SIMD's registers each
}

Plan plan(const PagesView &kv, const BatchView &b, const AttnPagedArgs &a) {
    const int group = a.n_head / kv.n_head_kv;
    const size_t queries = (size_t)b.n_rows * group;
    Plan p{};
    AttnArgs &A = p.A;
    A.a = a, A.kv = kv, A.b = b, A.group = group;
    A.scale_m = (float)std::frexp((double)a.scale * M_LOG2E, &A.scale_e);
    const size_t own = (queries + b.n_seqs - 1) / b.n_seqs, cap = (size_t)b.max_pages << kv.map.log2_page;
    // A block of few positions in a workgroup of its own, shared positions with it, saves the join: 9 us for 14 (13
    // rows over 14 positions), 15 for 36 (15 rows, 83 positions shared, up to 512). What a workgroup reads alone takes
    // as long as a join at 0.3 to 0.5 MB (f16, 256 values, up to 384 positions: 17.6 for 19.5; 736: 24 for 18).
    const size_t most = (size_t)320 * 1024 / (2 * kv.head_dim * (kv.f16 ? 2 : 4));
    A.alone = cap <= most && (b.n_seqs + queries / 16) * kv.n_head_kv <= 4 * kCUs;
    if (A.alone) {
        A.common = a.shared_len, A.a.shared_len = 0;
        A.part[0].rows = A.part[1].rows = 16;
    } else {
        A.part[1].rows = block_rows(kv, own, b.n_seqs, cap, false);
        A.part[0].rows = a.shared_len ? std::max(A.part[1].rows, block_rows(kv, queries, 1, a.shared_len, true)) : A.part[1].rows;
    }
    for (Part &x : A.part) x.G = block_groups(kv, x.rows);
    auto groups_recs = [&](const Part &x) { return (size_t)2 * x.G * x.rows; };
    size_t recs = A.alone ? 0 : groups_recs(A.part[1]);
    p.apart = A.part[0].rows != A.part[1].rows;
    if (p.apart) A.part[0].base = recs, recs += groups_recs(A.part[0]);
    A.whole = recs;
    if (A.a.shared_len) recs += (size_t)2 * b.n_rows * a.n_head;
    p.al = recs * kv.head_dim * sizeof(float);
    p.seg = p.al + recs * sizeof(float2);
    p.bytes = A.alone ? 16 : p.seg + (size_t)2 * b.n_rows * a.n_head * sizeof(int2);
    return p;
}

template <bool F16, int HD, int RT>
hipError_t launch(const AttnArgs &A, hipStream_t s) {
    constexpr size_t lds = (size_t)kWaves * 16 * RT * (HD + 4) * 4;
    static_assert(lds >= (size_t)HD * 64 * RT, "the queries fit where the sums go");
    static_assert(few_per_cu(HD, RT) * (lds + 2048) <= 160 * 1024, "LDS");
    auto *k = attn_paged_kernel<F16, HD, RT>;
    if (hipError_t e = allow_lds((const void *)k, lds)) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)A.part[A.first].G), dim3(kTPB), lds, s, A);
    return hipGetLastError();
}

template <bool F16>
hipError_t launch_few(const AttnArgs &A, hipStream_t s) {
    const bool two = A.part[A.first].rows == 32;
    switch (A.kv.head_dim) {
    case 64: return two ? launch<F16, 64, 2>(A, s) : launch<F16, 64, 1>(A, s);
    case 128: return two ? launch<F16, 128, 2>(A, s) : launch<F16, 128, 1>(A, s);
    case 256: return two ? launch<F16, 256, 2>(A, s) : launch<F16, 256, 1>(A, s);
    case 512: return launch<F16, 512, 1>(A, s);
    }
    return hipErrorInvalidValue;
}

template <int HD>
hipError_t join(const AttnArgs &A, hipStream_t s) {
    const int pairs = A.b.n_rows * A.a.n_head;  // at most 2^25
    if (pairs > 16 * kCUs)
        hipLaunchKernelGGL((attn_join_kernel<HD, 1>), dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, s, A, pairs);
    else if (pairs > 4 * kCUs)
        hipLaunchKernelGGL((attn_join_kernel<HD, 4>), dim3((unsigned)pairs), dim3(256), 0, s, A, pairs);
    else
        hipLaunchKernelGGL((attn_join_kernel<HD, 16>), dim3((unsigned)pairs), dim3(1024), 0, s, A, pairs);
    return hipGetLastError();
}

hipError_t launch_join(const AttnArgs &A, hipStream_t s) {
    switch (A.kv.head_dim) {
    case 64: return join<64>(A, s);
    case 128: return join<128>(A, s);
    case 256: return join<256>(A, s);
    case 512: return join<512>(A, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

size_t attn_paged_ws_bytes(const PagesView &kv, const BatchView &b, int n_head, int shared_len) {
    if (b.n_rows == 0 || b.n_seqs == 0) return 16;
    AttnPagedArgs a{};
    a.n_head = n_head, a.shared_len = shared_len;
    return plan(kv, b, a).bytes;
}

hipError_t launch_attn_paged(const PagesView &kv, const BatchView &b, const AttnPagedArgs &a, void *ws, hipStream_t s) {
    if (b.n_rows == 0 || b.n_seqs == 0) return hipSuccess;
    Plan p = plan(kv, b, a);
    AttnArgs &A = p.A;
    A.rec_o = (float *)ws;
    A.rec_al = (float2 *)((uint8_t *)ws + p.al);
    A.seg = (int2 *)((uint8_t *)ws + p.seg);
    auto go = [&](int first, int last) {
        A.first = first, A.last = last;
        return A.part[first].rows > 32 ? launch_attn_many(A, s) : kv.f16 ? launch_few<true>(A, s) : launch_few<false>(A, s);
    };
    if (p.apart)
        if (hipError_t e = go(0, 0)) return e;
    if (hipError_t e = go(A.a.shared_len && !p.apart ? 0 : 1, 1)) return e;
    return A.alone ? hipSuccess : launch_join(A, s);
}

}  // namespace uq
