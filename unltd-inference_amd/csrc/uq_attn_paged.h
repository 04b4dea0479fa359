// Shared by the attention kernels over paged caches (uq_attn_paged.hip: blocks
// of few queries; uq_attn_many.hip: of many): the work list, its division
// into workgroups' runs and the records that join them.
#pragma once

#include <algorithm>
#include <climits>
#include <type_traits>

#include "uq_attn_ref.h"
#include "uq_attn_ref.h"
#include "uq_device.h"
#include "uq_internal.h"
#include "uq_serve_internal.h"

namespace uq {

// One of the two parts of the work: the shared positions with the rows of the
// whole batch (part 0), or every sequence's own positions with its rows (1).
// Both may be one launch (the same G, rows and base).
struct Part {
    int rows;     // queries of a block
    int G;        // workgroups
    size_t base;  // first of the workgroups' records
};

struct AttnArgs {
    AttnPagedArgs a;
    PagesView kv;
    BatchView b;
    int group;
    float scale_m;    // kq_scale log2 e = scale_m 2^scale_e: the queries take the mantissa (0.5 to 1, signed), the
    int scale_e;      // exponent is a factor of their scores (uq_attn_ref.h)
    int common;       // positions that part 1 reads through the first sequence's pages (shared, but not a part)
    bool alone;       // every block has a workgroup of its own: no records, no join
    int first, last;  // the launch's parts
    Part part[2];
    size_t whole;   // first of the rows' own records
    float *rec_o;   // records: [..][HD] sums o ...
    float2 *rec_al; // ... with (a, l)
    int2 *seg;      // [part][row][head]: where the units of its block lie (put_seg)
};

// uq_attn_many.hip: part A.first (= A.last) on blocks of A.part[].rows = 64 or
// 128 queries (an f16 cache, head_dim 64, 128 or 256).
bool attn_many_ok(const PagesView &kv);
hipError_t launch_attn_many(const AttnArgs &A, hipStream_t s);

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any float
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));


// Where a block's units lie: in one workgroup that wrote the results itself,
// in one whose record is the row's own, or in several workgroups' records.
constexpr int kDone = -1, kWhole = -2;

// Records: two blocks of rows for each workgroup (its run's first block where
// that began earlier, its last where that goes on), then one per row and
// head of each part.
__device__ __forceinline__ size_t rec_part(const Part &p, int w, int second, int n) {
    return p.base + ((size_t)w * 2 + second) * p.rows + n;
}
__device__ __forceinline__ size_t rec_whole(const AttnArgs &A, int part, int row, int head) {
    return A.whole + ((size_t)part * A.b.n_rows + row) * A.a.n_head + head;
}

// What the workgroup that starts a block notes for each of its queries: the
// first workgroup with units of the block, or kDone or kWhole, the last one,
// and the query's place among the block's records.
__device__ __forceinline__ void put_seg(const AttnArgs &A, int part, int row, int head, int first, int last, int slot) {
    A.seg[((size_t)part * A.b.n_rows + row) * A.a.n_head + head] = make_int2(first, last << 8 | slot);
}

// The sequence of one part of the work: s = -1 is the shared positions with
// the rows of the whole batch.
struct Work {
    int lo, n, len;      // rows, length as given
    int base, end;       // positions [base, end)
    int units, blocks;
};

template <int U>
__device__ __forceinline__ Work work_of(const AttnArgs &A, int s, const SeqRows &r, int len) {
    const int cap = A.b.max_pages << A.kv.map.log2_page;
    Work w = s < 0 ? Work{r.lo, r.n, 0, 0, A.a.shared_len, 0, 0} : Work{r.lo, r.n, len, A.a.shared_len, seq_len(len, cap), 0, 0};
    w.units = w.end > w.base ? (w.end - w.base + U - 1) / U : 0;
    w.blocks = blocks_of(w.n, A.group, A.part[s >= 0].rows);
    return w;
}
template <int U>
__device__ __forceinline__ Work work_of(const AttnArgs &A, int s) {
    if (s < 0) return work_of<U>(A, s, seq_rows(0, A.b.row_start[A.b.n_seqs], A.b.n_rows), 0);
    return work_of<U>(A, s, seq_rows(A.b.row_start[s], A.b.row_start[s + 1], A.b.n_rows), A.b.len[s]);
}

// The units of a block of a sequence's own positions up to the last one that
// a row of it sees, given how many of the sequence's rows lie before the
// block's end.
template <int U>
__device__ __forceinline__ int seen_to(const Work &w, int rows) {
    const int end = min(w.end, max(0, w.len - w.n + min(w.n, rows)));
    return end > w.base ? (end - w.base + U - 1) / U : 0;
}
template <int U>
__device__ __forceinline__ int seen_units(const AttnArgs &A, const Work &w, int rb) {
    return seen_to<U>(w, ((rb + 1) * A.part[1].rows - 1) / A.group + 1);  // below 2^26: n_rows n_head is at most 2^25
}
// Their sum over the blocks, without a division a block; `more` for each with any.
template <int U>
__device__ __forceinline__ long long seen_sum(const AttnArgs &A, const Work &w, int more) {
    const int RB = A.part[1].rows, step = RB / A.group, rest = RB % A.group;
    int rows = (RB - 1) / A.group + 1, left = (RB - 1) % A.group;
    long long t = 0;
    for (int rb = 0; rb < w.blocks; rb++) {
        const int units = seen_to<U>(w, rows);
        t += A.alone ? 1 : units > 0 ? units + more : 0;
        rows += step, left += rest;
        if (left >= A.group) rows++, left -= A.group;
    }
    return t;
}

// The page of a position of a sequence's own part, whose table's row is given.
__device__ __forceinline__ int page_at(const AttnArgs &A, const int32_t *table, int pos) {
    return (pos < A.common ? A.b.pages : table)[pos >> A.kv.map.log2_page];
}

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long uniform(long long v) {
    const unsigned lo = (unsigned)uniform((int)v), hi = (unsigned)uniform((int)(v >> 32));
    return (long long)((unsigned long long)hi << 32 | lo);
}

// Inclusive sum over the wave's lanes, and a reduction over LANES neighbouring lanes (16, 32 or 64) in all of them,
// without a round trip to the LDS.
template <int CTRL, int ROW_MASK = 0xF>
__device__ __forceinline__ long long dpp_l(long long v) {
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROW_MASK, 0xF, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROW_MASK, 0xF, true);
    return (long long)hi << 32 | lo;
}
__device__ __forceinline__ long long wave_scan_l(long long v) {
    v += dpp_l<0x111>(v);       // row_shr:1
    v += dpp_l<0x112>(v);       // row_shr:2
    v += dpp_l<0x114>(v);       // row_shr:4
    v += dpp_l<0x118>(v);       // row_shr:8
    v += dpp_l<0x142, 0xA>(v);  // row_bcast:15 into rows 1, 3
    v += dpp_l<0x143, 0xC>(v);  // row_bcast:31 into rows 2, 3
    return v;
}
template <int LANES, class Op>
__device__ __forceinline__ uint32_t lanes_of(uint32_t v, Op op) {
    v = op(v, dpp_u<0xB1>(v));   // quad_perm [1,0,3,2]
    v = op(v, dpp_u<0x4E>(v));   // quad_perm [2,3,0,1]
    v = op(v, dpp_u<0x141>(v));  // row_half_mirror
    v = op(v, dpp_u<0x140>(v));  // row_mirror
    if constexpr (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    if constexpr (LANES == 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    return v;
}
// The largest bit pattern; the least signed integer; the least float.
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    return lanes_of<LANES>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int LANES>
__device__ __forceinline__ int lanes_min(int v) {
    return (int)lanes_of<LANES>((uint32_t)v, [](uint32_t a, uint32_t b) { return (uint32_t)min((int)a, (int)b); });
}
template <int LANES>
__device__ __forceinline__ float lanes_min(float v) {
    return __uint_as_float(lanes_of<LANES>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ long long lane_of(long long v, int lane) {
    return (long long)lane_of((int)(v >> 32), lane) << 32 | (unsigned)lane_of((int)v, lane);
}

// The walk of a workgroup of TPB threads over its run of the work. Every block
// of a KV head counts OVER units beside its units of U positions: what its
// start and end cost, so that a run with two of them has less else to do.
// They lie before the units; a run that ends among them leaves the block to
// the next one.
//
// The shared positions by themselves are `blocks` alike, and where the
// workgroups divide well among them every run lies in one block of one KV
// head, and the runs of all blocks over the same positions go to one XCD at a
// time (workgroup i runs on XCD i % 8), whose L2 then reads each tile once (48
// rows of 16 heads behind 65536 positions: 207 to 191 us).
//
// What find reads are all row starts and lengths, by every
// workgroup: one round trip to the L2, where another kernel for a plan would
// cost a launch.
struct WalkLds {
    long long scan[4], off;
    int index, work[7];
};
template <int TPB, int U, int OVER, int PAR>
struct Walk {
    int runs, me, over;        // runs of all workgroups, this one's; units counted for a block's start and end
    int seq, rb, units;        // where the next block is looked for
    long long T, u, u1, off;   // all units, the rest of this run, the next unit's place among its block's (all KV heads)
    Work w;
    // the block at hand
    int kvh, un, count;  // its KV head, the first of its units here and how many
    bool starts, ends;   // whether those begin and end it
    long long end;       // its last unit among all

    __device__ __forceinline__ int units_of(const AttnArgs &A, int b) const {
        return seq < 0 ? w.units : seen_units<U>(A, w, b);
    }
    __device__ __forceinline__ static int each_of(const AttnArgs &A, int n, int over) {  // of n units, for a KV head
        return A.alone ? 1 : n > 0 ? n + over : 0;
    }
    __device__ __forceinline__ static long long cost(const AttnArgs &A, int n, int over) {
        return (long long)A.kv.n_head_kv * each_of(A, n, over);
    }
    // Units before item c + tid and its own (of items c .. c + TPB - 1 with value(i) each); returns those up to c + TPB
    template <class Value>
    __device__ static __forceinline__ long long scan(WalkLds &lds, int c, int n, long long run, long long &mine, long long &before,
                                                     Value value) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        mine = c + tid < n ? value(c + tid) : 0;
        const long long inc = wave_scan_l(mine);
        __syncthreads();
        if (lane == 63) lds.scan[wave] = inc;
        __syncthreads();
        before = run + inc - mine;
#pragma unroll
        for (int k = 0; k < TPB / 64; k++) {
            if (k < wave) before += lds.scan[k];
            run += lds.scan[k];
        }
        return run;
    }
    // Few sequences (and few blocks of one): every wave looks by itself, and there is no barrier.
    __device__ bool find(const AttnArgs &A, WalkLds &lds) {
        const int tid = threadIdx.x, lane = tid & 63, parts = A.b.n_seqs + 1;
        const bool few = parts <= 64;
        Work mine_w{};
        auto value = [&](int i) {
            if (i > 0 ? A.last == 0 : A.first == 1) return 0LL;
            mine_w = work_of<U>(A, i - 1);
            if (mine_w.units == 0 && !A.alone) return 0LL;
            return i == 0 ? cost(A, mine_w.units, OVER) * mine_w.blocks : A.kv.n_head_kv * seen_sum<U>(A, mine_w, OVER);
        };
        long long mine = 0, before = 0, run = 0;
        T = 0;
        if (few) {
            mine = lane < parts ? value(lane) : 0;
            const long long inc = wave_scan_l(mine);
            before = inc - mine;
            T = lane_of(inc, 63);
        } else {
            for (int c = 0; c < parts; c += TPB) T = scan(lds, c, parts, T, mine, before, value);
            T = uniform(T);
        }
        // no empty runs between others, and none of fewer units than the workgroup takes at a time
        runs = (int)min((long long)A.part[A.first].G, A.alone ? T : (T + PAR - 1) / PAR);
        me = (int)blockIdx.x;
        over = OVER;
        if (A.last == 0) {
            const Work all = work_of<U>(A, -1);
            const int nkv = A.kv.n_head_kv, of = 8 / min(8, nkv & -nkv);  // J * nkv is a multiple of 8
            const int J = all.blocks == 0 || all.blocks > runs / nkv ? 0 : min(all.units, runs / (nkv * all.blocks)) / of * of;
            if (J > 0 && all.units / J <= T / runs + OVER) {
                over = 0;
                T = (long long)all.blocks * nkv * all.units;
                runs = J * nkv * all.blocks;
                const int i = me >> 3, at = i / all.blocks * 8 + (me & 7);  // the positions' run among all KV heads'
                me = me < runs ? i % all.blocks * nkv * J + at : runs;
            }
        }
        if (me >= runs) return false;
        u = run_start(T, runs, me);
        u1 = run_start(T, runs, me + 1);
        if (A.last == 0) {
            seq = -1;
            off = u;
            w = work_of<U>(A, -1);
            w = Work{uniform(w.lo), uniform(w.n), uniform(w.len), uniform(w.base), uniform(w.end), uniform(w.units), uniform(w.blocks)};
        } else if (few) {
            const int at = __builtin_ctzll(__ballot(mine > 0 && before <= u && u < before + mine) | 1ull << 63);
            seq = at - 1;
            off = u - lane_of(before, at);
            w = Work{lane_of(mine_w.lo, at), lane_of(mine_w.n, at), lane_of(mine_w.len, at), lane_of(mine_w.base, at),
                     lane_of(mine_w.end, at), lane_of(mine_w.units, at), lane_of(mine_w.blocks, at)};
        } else {
            auto keep = [&](int i) {
                lds.index = i - 1, lds.off = u - before;
                lds.work[0] = mine_w.lo, lds.work[1] = mine_w.n, lds.work[2] = mine_w.len, lds.work[3] = mine_w.base;
                lds.work[4] = mine_w.end, lds.work[5] = mine_w.units, lds.work[6] = mine_w.blocks;
            };
            if (parts <= TPB) {
                if (mine > 0 && before <= u && u < before + mine) keep(tid);
            } else {
                for (int c = 0; c < parts; c += TPB) {
                    run = scan(lds, c, parts, run, mine, before, value);
                    if (mine > 0 && before <= u && u < before + mine) keep(c + tid);
                }
            }
            __syncthreads();
            seq = uniform(lds.index);
            off = uniform(lds.off);
            w = Work{uniform(lds.work[0]), uniform(lds.work[1]), uniform(lds.work[2]), uniform(lds.work[3]),
                     uniform(lds.work[4]), uniform(lds.work[5]), uniform(lds.work[6])};
        }
        rb = 0;
        auto block = [&](int b) { return cost(A, units_of(A, b), over); };
        if (w.blocks > 64) {  // the block, likewise
            run = 0;
            for (int c = 0; c < w.blocks; c += TPB) {
                run = scan(lds, c, w.blocks, run, mine, before, block);
                if (mine > 0 && before <= off && off < before + mine) lds.index = c + tid, lds.off = off - before;
                if (off < run) break;  // the same for every thread
            }
            __syncthreads();
            rb = uniform(lds.index);
            off = uniform(lds.off);
        } else if (w.blocks > 1) {
            mine = lane < w.blocks ? block(lane) : 0;
            before = wave_scan_l(mine) - mine;
            rb = __builtin_ctzll(__ballot(mine > 0 && before <= off && off < before + mine) | 1ull << 63);
            off -= lane_of(before, rb);
        }
        units = units_of(A, rb);
        return true;
    }
    // The next block with units of this run; false: none.
    __device__ __forceinline__ bool next(const AttnArgs &A) {
        while (u < u1) {
            const int each = each_of(A, units, over);
            if (off >= (long long)A.kv.n_head_kv * each) {
                off -= (long long)A.kv.n_head_kv * each;
                if (++rb >= w.blocks) {
                    do {
                        if (++seq >= A.b.n_seqs) return false;  // the batch changed under the call
                        w = work_of<U>(A, seq);
                    } while (w.blocks == 0);
                    rb = 0;
                }
                units = units_of(A, rb);
                continue;
            }
            kvh = off >> 31 ? (int)(off / each) : (int)off / each;
            const int at = (int)(off - (long long)kvh * each), upto = (int)min((long long)each, at + (u1 - u));
            un = max(0, at - over);
            count = max(0, upto - over) - un;
            starts = un == 0, ends = upto == each;
            end = u + each - at - 1;
            u += upto - at;
            off += upto - at;
            if (A.alone) {
                un = 0, count = units, starts = ends = true;
                return true;
            }
            if (count > 0) return true;
        }
        return false;
    }
    // The workgroup that ends the block at hand.
    __device__ __forceinline__ int last() const { return run_owner(T, runs, end); }
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The two f16 terms of a b, not rounded to f32 before. The first is taken from a register: where the compiler sees the
// product, it converts it from f32 in one place and from the exact product in another, and the terms do not match.
__device__ __forceinline__ void product_terms(float a, float b, _Float16 &hi, _Float16 &lo) {
    float v = a * b;
    __asm__("" : "+v"(v));
    hi = (_Float16)v;
    lo = (_Float16)fmaf(a, b, -(float)hi);
}

}  // namespace
}  // namespace uq
