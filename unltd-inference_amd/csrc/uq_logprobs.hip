// Log probabilities of given tokens, their ranks, the entropy and the
// likeliest alternatives of rows of logits (uq_logprobs_d).
//
// One pass over a row: with m the largest logit seen so far and c = scale
// log2 e a lane keeps
//     l = sum 2^(c (x - m)),   s = sum 2^(c (x - m)) c (x - m),
// from which log p(t) = scale (x_t - m) - ln l and the entropy
// ln l - ln 2 s / l; parts of a row join by 2^(c (m' - m)). The differences
// are formed before the product, so that logits of any size, the type's lowest
// value among them, do not lose the small ones. At scales below 1, which bring
// differences beyond f32's range back into it, they are those of halves.
//
// Rows are cut into runs of tiles of 1024 values, a wave each, without
// barriers. Memory bounds it where there is much of it: 1021 rows of 152064
// 110 us, 5.7 TB/s. One row with its 20 likeliest tokens is 13 us: two launches,
// 5 and 7, of steps that wait for one another.
#include <algorithm>
#include <cfloat>

#include "uq_device.h"
#include "uq_serve_internal.h"

namespace uq {

namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any float

constexpr int kTPB = 256, kTile = 1024, kVals = kTile / 64;
constexpr float kLeast = -300.0f;  // 2^-300 is 0: exponents below it are taken as it, so that no 0 times infinity arises

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// What a wave leaves of its run.
struct Part {
    float m, l, s;
    int before;  // tokens before the given one
    int kept, unused;  // keys
};

struct Args {
    uq_logprobs out;
    const float *x;
    size_t x_row;
    const int32_t *tokens;
    int n_rows, vocab, n_top, tiles, run, parts;  // tiles of a row, of a wave; waves of a row
    // a logit's factor in a difference, 1 or 1/2, and by what the difference becomes an exponent of e, of 2
    float pre, scale, c;
    Part *part;      // [n_rows][parts]
    uint64_t *keys;  // [n_rows][parts][64]
    __device__ __forceinline__ float minus(float x, float y) const { return fmaf(x, pre, -(y * pre)); }
};

// A token's key is its logit as an integer in the order of its size, then the complement of its number. 0 is none.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 as +0
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
constexpr uint32_t kLowest = 0x00800000u;  // ordered(-infinity) + 1: neither it nor a NaN that is below it is kept

// What the wave's lanes have written to the LDS is read by others behind this point.
__device__ __forceinline__ void lanes_see() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// Keys in the LDS, the first n_top (64 at most) of those offered among them. Only when they overflow are they put in
// order, and the first n_top kept: a wave's run mostly ends before.
constexpr int kPool = 128;  // 64 are free after that, as many as one call offers
struct Pool {
    uint64_t *at;
    int n_top, count = 0;
    uint32_t least = kLowest;  // logits below it are not among the first
    bool full = false;         // n_top keys are kept, of which the last has the logit `least`
    __device__ __forceinline__ Pool(uint64_t *p, int n) : at(p), n_top(n) {}
    // Puts the keys in order and keeps the first n_top. A key's place is how many are larger: keys differ, as a token is seen once.
    __device__ __forceinline__ void order() {
        const int lane = threadIdx.x & 63;
        lanes_see();
        const uint64_t k0 = lane < count ? at[lane] : 0, k1 = lane + 64 < count ? at[lane + 64] : 0;
        int p0 = 0, p1 = 0;
        for (int j = 0; j < min(count, 64); j++) {
            const uint64_t k = lane_of(k0, j);
            p0 += k > k0;
            p1 += k > k1;
        }
        for (int j = 0; j < count - 64; j++) {
            const uint64_t k = lane_of(k1, j);
            p0 += k > k0;
            p1 += k > k1;
        }
        if (lane < count && p0 < n_top) at[p0] = k0;
        if (lane + 64 < count && p1 < n_top) at[p1] = k1;
        count = min(count, n_top);
        lanes_see();
    }
    // LATER: tokens after all that were offered before, which go before them where logits are equal.
    template <bool LATER>
    __device__ __forceinline__ void take(uint64_t key, bool in) {
        unsigned long long b = __ballot(in);
        if (!b) return;
        if (count + __builtin_popcountll(b) > kPool) {
            order();
            full = true;
            least = max(least, (uint32_t)uniform((int)(at[n_top - 1] >> 32)) + (LATER ? 1 : 0));
            in = in && (uint32_t)(key >> 32) >= least;
            b = __ballot(in);
        }
        const int slot = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
        if (in) at[count + slot] = key;
        count += __builtin_popcountll(b);
    }
};

// A bound that at least n lanes' values reach (its upper 16 bits are those of the n-th largest, the rest 0).
__device__ __forceinline__ uint32_t reached_by(uint32_t v, int n) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t more = t | 1u << bit;
        if (__builtin_popcountll(__ballot(v >= more)) >= n) t = more;
    }
    return t;
}

// How many of the lanes' values reach t, and the largest such t for n of them, but for its lowest bits, which are 0.
template <int N>
__device__ __forceinline__ int reaching(const uint32_t (&v)[N], uint32_t t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; i++) n += __builtin_popcountll(__ballot(v[i] >= t));
    return n;
}
template <int LOWEST, int N>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&v)[N], int n) {
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= LOWEST; bit--) {
        const uint32_t more = t | 1u << bit;
        if (reaching(v, more) >= n) t = more;
    }
    return t;
}
// The first n of a tile's values (token 256 j + 4 lane + e in o[4 j + e]): others become 0. Returns the last one's size, 0
// if n values are not as large as `least`: then all stay.
__device__ __forceinline__ uint32_t first_of(uint32_t (&o)[kVals], int n, uint32_t least) {
    const uint32_t t = reached_by<0>(o, n);
    if (t < least) return 0;
    int room = n - reaching(o, t + 1);
#pragma unroll
    for (int j = 0; j < kVals; j += 4) {
        int rank = 0, all = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const unsigned long long b = __ballot(o[j + e] == t);
            rank = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, rank));
            all += __builtin_popcountll(b);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool tie = o[j + e] == t;
            if (o[j + e] < t || (tie && rank >= room)) o[j + e] = 0;
            rank += tie;
        }
        room -= all;
    }
    return t;
}

template <bool TOP>
__global__ __launch_bounds__(kTPB) void logprobs_kernel(Args a) {
    const int lane = threadIdx.x & 63;
    const int w = uniform((int)(blockIdx.x * (kTPB / 64) + (threadIdx.x >> 6)));
    const int row = w / a.parts, part = w - row * a.parts;
    if (row >= a.n_rows) return;
    const float *x = a.x + (size_t)row * a.x_row;
    const int t0 = part * a.run, t1 = min(a.tiles, t0 + a.run);
    float v[kVals], next[kVals];
    auto load = [&](float (&d)[kVals], int tile) {  // token 256 j + 4 lane + e of the tile in d[4 j + e]
#pragma unroll
        for (int j = 0; j < kVals / 4; j++) {
            const int i = tile * kTile + 256 * j + 4 * lane;
            if (i + 4 <= a.vocab) {
                const f4u f = *(const f4u *)(x + i);
#pragma unroll
                for (int e = 0; e < 4; e++) d[4 * j + e] = f[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) d[4 * j + e] = i + e < a.vocab ? x[i + e] : -INFINITY;
            }
        }
    };
    load(v, t0);
    const int token = a.tokens ? uniform(a.tokens[row]) : -1;
    const bool ranked = (unsigned)token < (unsigned)a.vocab;
    const float given = ranked ? x[token] : INFINITY;
    float m = -FLT_MAX, l = 0.0f, s = 0.0f;
    int before = 0;
    __shared__ uint64_t pools[TOP ? kTPB / 64 : 1][kPool];
    Pool pool(pools[TOP ? threadIdx.x >> 6 : 0], a.n_top);
    for (int t = t0; t < t1; t++) {
        if (t + 1 < t1) load(next, t + 1);
        float top = v[0];
#pragma unroll
        for (int i = 1; i < kVals; i++) top = fmaxf(top, v[i]);
        if (__ballot(top > m)) {
            const float to = fmaxf(m, top), d = fmaxf(a.minus(m, to) * a.c, kLeast), f = exp2_hw(d);
            s = f * fmaf(d, l, s);
            l *= f;
            m = to;
        }
        float tl[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ts[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kVals; i++) {
            const float d = a.minus(v[i], m) * a.c, e = exp2_hw(d);
            tl[i % 4] += e;
            ts[i % 4] = fmaf(e, fmaxf(d, kLeast), ts[i % 4]);
        }
        l += (tl[0] + tl[1]) + (tl[2] + tl[3]);
        s += (ts[0] + ts[1]) + (ts[2] + ts[3]);
        if (ranked) {
            const int first = t * kTile;
            if (token >= first + kTile) {
#pragma unroll
                for (int i = 0; i < kVals; i++) before += __builtin_popcountll(__ballot(v[i] >= given));
            } else if (token < first) {
#pragma unroll
                for (int i = 0; i < kVals; i++) before += __builtin_popcountll(__ballot(v[i] > given));
            } else {
#pragma unroll
                for (int i = 0; i < kVals; i++) {
                    const int id = first + 256 * (i / 4) + 4 * lane + i % 4;
                    before += __builtin_popcountll(__ballot(v[i] > given || (v[i] == given && id < token)));
                }
            }
        }
        if constexpr (TOP) {
            // Values below a bound that n_top lanes reach with their largest cannot be among the first. Where that leaves
            // more than fit, for n_top near 64 (of 1024 values 43 for 32, 236 for 64) or for equal logits, a bound that n_top
            // values reach; then, for equal ones, the tile's first alone.
            const uint32_t most = ordered(top);
            const unsigned long long over = __ballot(most >= pool.least);
            if (over) {
                if (__builtin_popcountll(over) >= a.n_top) pool.least = max(pool.least, reached_by(most, a.n_top));
                uint32_t o[kVals];
#pragma unroll
                for (int i = 0; i < kVals; i++) o[i] = v[i] == v[i] ? ordered(v[i]) : 0;
                if (__builtin_popcountll(__ballot(most >= pool.least)) > 32 && pool.count + reaching(o, pool.least) > kPool) {
                    pool.least = max(pool.least, reached_by<16>(o, a.n_top));
                    if (reaching(o, pool.least) > a.n_top + 32) {
                        const uint32_t last = first_of(o, a.n_top, pool.least);
                        if (last) pool.least = last, pool.full = true;
                    }
                }
#pragma unroll
                for (int i = 0; i < kVals; i++)
                    pool.take<false>((uint64_t)o[i] << 32 | (uint32_t)~(t * kTile + 256 * (i / 4) + 4 * lane + i % 4), o[i] >= pool.least);
                if (pool.full) {  // later tokens of equal logits come after those kept
                    pool.least += 1;
                    pool.full = false;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kVals; i++) v[i] = next[i];
    }
    // the lanes' sums
    const float all = [&] {
        float r = m;
        for (int d = 1; d < 64; d *= 2) r = fmaxf(r, __shfl_xor(r, d));
        return r;
    }();
    const float d = fmaxf(a.minus(m, all) * a.c, kLeast), f = exp2_hw(d);
    s = wave_sum(f * fmaf(d, l, s));
    l = wave_sum(f * l);
    const size_t o = (size_t)row * a.parts + part;
    if constexpr (TOP)
        if (pool.count > 64) pool.order();
    lanes_see();
    if (lane == 0) a.part[o] = Part{all, l, s, before, pool.count, 0};
    if constexpr (TOP)
        if (lane < pool.count) a.keys[o * 64 + lane] = pool.at[lane];
}

// A wave a row: joins its parts and writes the results.
template <bool TOP>
__global__ __launch_bounds__(64) void logprobs_join_kernel(Args a) {
    const int row = blockIdx.x, lane = threadIdx.x;
    const Part *parts = a.part + (size_t)row * a.parts;
    float m = -FLT_MAX, l = 0.0f, s = 0.0f;
    int before = 0;
    constexpr int P = 4;  // parts of a lane at a time
    uint32_t most[P] = {0, 0, 0, 0};
    for (int i0 = 0; i0 < a.parts; i0 += 64 * P) {
        Part p[P];
#pragma unroll
        for (int j = 0; j < P; j++) p[j] = parts[min(i0 + 64 * j + lane, a.parts - 1)];
#pragma unroll
        for (int j = 0; j < P; j++) {
            if (i0 + 64 * j + lane >= a.parts) continue;
            const float to = fmaxf(m, p[j].m), d = fmaxf(a.minus(m, to) * a.c, kLeast), dp = fmaxf(a.minus(p[j].m, to) * a.c, kLeast);
            const float f = exp2_hw(d), fp = exp2_hw(dp);
            s = f * fmaf(d, l, s) + fp * fmaf(dp, p[j].l, p[j].s);
            l = f * l + fp * p[j].l;
            m = to;
            before += p[j].before;
            most[j] = max(most[j], ordered(p[j].m));
        }
    }
    float all = m;
    for (int d = 1; d < 64; d *= 2) all = fmaxf(all, __shfl_xor(all, d));
    const float d = fmaxf(a.minus(m, all) * a.c, kLeast), f = exp2_hw(d);
    s = wave_sum(f * fmaf(d, l, s));
    l = wave_sum(f * l);
    for (int k = 1; k < 64; k *= 2) before += __shfl_xor(before, k);
    const bool sound = l == l && l < INFINITY;  // no NaN and no infinite logit
    const float ln_l = logf(l), nan = __uint_as_float(0x7FC00000u);
    auto log_p = [&](float x) { return !sound ? nan : l > 0.0f ? fmaf(a.minus(x, all), a.scale, -ln_l) : -INFINITY; };
    if (lane == 0) {
        const int token = a.tokens ? a.tokens[row] : -1;
        const bool in = (unsigned)token < (unsigned)a.vocab;
        if (a.out.d_logprob)
            a.out.d_logprob[row] = in ? log_p(a.x[(size_t)row * a.x_row + token]) : sound ? -INFINITY : nan;
        if (a.out.d_rank) a.out.d_rank[row] = in && sound ? before : -1;
        // the terms are not positive but for their roundings
        if (a.out.d_entropy) a.out.d_entropy[row] = !sound ? nan : l > 0.0f ? fmaxf(0.0f, ln_l - 0.693147182f * (s / l)) : 0.0f;
    }
    if constexpr (TOP) {
        // as within a wave's run: n_top parts reach the bound with their largest, and the others are not read
        __shared__ uint64_t kept[kPool];
        Pool pool(kept, a.n_top);
        if (a.parts >= a.n_top) pool.least = max(pool.least, reached_by<16>(most, a.n_top));
        const uint64_t *keys = a.keys + (size_t)row * a.parts * 64;
        for (int i0 = 0; i0 < a.parts; i0 += 64) {
            const int i = min(i0 + lane, a.parts - 1);
            const int count = parts[i].kept;
            const uint32_t largest = i0 + lane < a.parts ? ordered(parts[i].m) : 0;
            unsigned long long over = __ballot(largest >= pool.least);
            constexpr int N = 16;  // parts at a time
            while (over) {
                uint64_t k[N];
#pragma unroll
                for (int j = 0; j < N; j++) {
                    const int from = over ? __builtin_ctzll(over) : 0, n = over ? __builtin_amdgcn_readlane(count, from) : 0;
                    k[j] = lane < n ? keys[(size_t)(i0 + from) * 64 + lane] : 0;
                    over &= over - 1;
                }
                uint32_t o[N];
#pragma unroll
                for (int j = 0; j < N; j++) o[j] = (uint32_t)(k[j] >> 32);
                if (a.n_top > 32 && pool.count + reaching(o, pool.least) > kPool) pool.least = max(pool.least, reached_by<16>(o, a.n_top));
#pragma unroll
                for (int j = 0; j < N; j++) pool.take<true>(k[j], o[j] >= pool.least);
                over &= __ballot(largest >= pool.least);
            }
        }
        pool.order();
        const uint64_t mine = lane < pool.count ? kept[lane] : 0;
        if (lane < a.n_top) {
            const bool is = sound && mine != 0;
            const uint32_t u = (uint32_t)(mine >> 32);
            const float x = __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
            const size_t o = (size_t)row * a.n_top + lane;
            if (a.out.d_top_id) a.out.d_top_id[o] = is ? (int)~(uint32_t)mine : -1;
            if (a.out.d_top_logprob) a.out.d_top_logprob[o] = !sound ? nan : is ? log_p(x) : -INFINITY;
        }
    }
}

// Tiles of a wave: one, so that waves are many and short, or two of 65536 and more. 1021 rows of 152064 take 110 us with
// one, 112 with two or four and 129 with 16, and with their 20 likeliest tokens, of which two tiles leave as many as one,
// 159, 145, 171 and 170; 200 rows with 64 of them 91 with one and 115 with two.
struct Shape {
    int tiles, run, parts;
};
Shape shape_of(int n_rows, int vocab) {
    Shape s;
    s.tiles = (vocab + kTile - 1) / kTile;
    const long long all = (long long)s.tiles * n_rows;
    s.run = all >= 65536 ? 2 : 1;
    s.parts = (s.tiles + s.run - 1) / s.run;
    return s;
}

}  // namespace

size_t logprobs_ws_bytes(int n_rows, int vocab, int n_top) {
    const Shape s = shape_of(n_rows, vocab);
    return (size_t)n_rows * s.parts * (sizeof(Part) + (n_top ? 64 * sizeof(uint64_t) : 0));
}

hipError_t launch_logprobs(const uq_logprobs &out, const float *x, size_t x_row, const int32_t *tokens, int n_rows,
                           int vocab, float scale, void *ws, hipStream_t s) {
    if (n_rows == 0) return hipSuccess;
    const Shape h = shape_of(n_rows, vocab);
    const bool top = out.n_top && (out.d_top_id || out.d_top_logprob);
    Part *part = (Part *)ws;
    const float pre = scale < 1.0f ? 0.5f : 1.0f, by = scale / pre;
    const Args a{out,     x,     x_row,   tokens, n_rows, vocab, top ? (int)out.n_top : 0,
                 h.tiles, h.run, h.parts, pre,    by,     (float)(by * 1.4426950408889634), part, (uint64_t *)(part + (size_t)n_rows * h.parts)};
    const long long waves = (long long)n_rows * h.parts, per = kTPB / 64;
    const dim3 grid((unsigned)((waves + per - 1) / per));
    if (top)
        hipLaunchKernelGGL(logprobs_kernel<true>, grid, dim3(kTPB), 0, s, a);
    else
        hipLaunchKernelGGL(logprobs_kernel<false>, grid, dim3(kTPB), 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    if (top)
        hipLaunchKernelGGL(logprobs_join_kernel<true>, dim3((unsigned)n_rows), dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL(logprobs_join_kernel<false>, dim3((unsigned)n_rows), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace uq
