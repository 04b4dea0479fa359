// Shared by the attention kernels over paged caches (uq_attn_paged.hip: blocks
// of few queries; uq_attn_many.hip: of many): the work list, its division
// into workgroups' runs and the records that join them.
#pragma once

#include <algorithm>
#include <climits>
#include <type_traits>

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

constexpr float kLog2e = 1.44269504088896340736f;

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
        t += units > 0 ? units + more : 0;
        rows += step, left += rest;
        if (left >= A.group) rows++, left -= A.group;
    }
    return t;
}

// A value that is the same in every lane, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long long uniform(long long v) {
    const unsigned lo = (unsigned)uniform((int)v), hi = (unsigned)uniform((int)(v >> 32));
    return (long long)((unsigned long long)hi << 32 | lo);
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
// time (workgroup i runs on XCD i % 8), whose L2 then reads each tile once:
// XXX
//
// What find reads are all row starts and lengths, by every
// workgroup: one round trip to the L2, where another kernel for a plan would
// cost a launch.
struct WalkLds {
    long long scan[4], off;
    int index, work[7];
};
template <int TPB, int U, int OVER>
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
    __device__ __forceinline__ static long long cost(const AttnArgs &A, int n, int over) {
        return n > 0 ? (long long)A.kv.n_head_kv * (n + over) : 0;
    }
    // Units before item c + tid and its own (of items c .. c + TPB - 1 with value(i) each); returns those up to c + TPB
    template <class Value>
    __device__ static __forceinline__ long long scan(WalkLds &lds, int c, int n, long long run, long long &mine, long long &before,
                                                     Value value) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        mine = c + tid < n ? value(c + tid) : 0;
        long long inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long long up = __shfl_up(inc, d);
            if (lane >= d) inc += up;
        }
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
    __device__ bool find(const AttnArgs &A, WalkLds &lds) {
        const int tid = threadIdx.x, parts = A.b.n_seqs + 1;
        Work mine_w{};
        auto value = [&](int i) {
            if (i > 0 ? A.last == 0 : A.first == 1) return 0LL;
            mine_w = work_of<U>(A, i - 1);
            if (mine_w.units == 0) return 0LL;
            return i == 0 ? cost(A, mine_w.units, OVER) * mine_w.blocks : A.kv.n_head_kv * seen_sum<U>(A, mine_w, OVER);
        };
        long long mine = 0, before = 0, run = 0;
        T = 0;
        for (int c = 0; c < parts; c += TPB) T = scan(lds, c, parts, T, mine, before, value);
        T = uniform(T);
        runs = (int)min((long long)A.part[A.first].G, T);  // no empty runs between others
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
                run = 0;
                mine = threadIdx.x == 0 ? T : 0, before = 0, mine_w = all;
            }
        }
        if (me >= runs) return false;
        u = run_start(T, runs, me);
        u1 = run_start(T, runs, me + 1);
        auto keep = [&](int i) {
            lds.index = i - 1, lds.off = u - before;
            lds.work[0] = mine_w.lo, lds.work[1] = mine_w.n, lds.work[2] = mine_w.len, lds.work[3] = mine_w.base;
            lds.work[4] = mine_w.end, lds.work[5] = mine_w.units, lds.work[6] = mine_w.blocks;
        };
        if (parts <= TPB || over == 0) {
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
        rb = 0;
        if (w.blocks > 1) {  // the block, likewise
            run = 0;
            for (int c = 0; c < w.blocks; c += TPB) {
                run = scan(lds, c, w.blocks, run, mine, before, [&](int b) { return cost(A, units_of(A, b), over); });
                if (mine > 0 && before <= off && off < before + mine) lds.index = c + tid, lds.off = off - before;
                if (off < run) break;  // the same for every thread
            }
            __syncthreads();
            rb = uniform(lds.index);
            off = uniform(lds.off);
        }
        units = units_of(A, rb);
        return true;
    }
    // The next block with units of this run; false: none.
    __device__ __forceinline__ bool next(const AttnArgs &A) {
        while (u < u1) {
            const int each = units > 0 ? units + over : 0;
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
            if (count > 0) return true;
        }
        return false;
    }
    // The workgroup that ends the block at hand.
    __device__ __forceinline__ int last() const { return run_owner(T, runs, end); }
};

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace
}  // namespace uq
