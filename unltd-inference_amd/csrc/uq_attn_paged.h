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
    bool many;        // part 1 runs on attn_many_kernel
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
__device__ __forceinline__ Work work_of(const AttnArgs &A, int s) {
    Work w;
    const int cap = A.b.max_pages << A.kv.map.log2_page;
    if (s < 0) {
        const SeqRows r = seq_rows(0, A.b.row_start[A.b.n_seqs], A.b.n_rows);
        w = Work{r.lo, r.n, 0, 0, A.a.shared_len, 0, 0};
    } else {
        const SeqRows r = seq_rows(A.b.row_start[s], A.b.row_start[s + 1], A.b.n_rows);
        const int len = A.b.len[s];
        w = Work{r.lo, r.n, len, A.a.shared_len, seq_len(len, cap), 0, 0};
    }
    w.units = w.end > w.base ? (w.end - w.base + U - 1) / U : 0;
    w.blocks = blocks_of(w.n, A.group, A.part[s >= 0].rows);
    return w;
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
    return seen_to<U>(w, ((rb + 1) * A.part[1].rows - 1) / A.group + 1);  // below 2^30: n_rows n_head is below 2^29
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

// A workgroup's run: units [u, u1) of T, the first of them off units into
// sequence seq (-1: the shared positions).
struct Run {
    long long T, u, u1, off;
    int runs, seq;
    Work work;  // of seq
};
struct RunLds {
    long long scan[4], off;
    int seq, work[7];
};
// The run of this workgroup (of TPB threads), by a scan over the sequences'
// units (count(s, work of s); every workgroup reads all row starts and lengths: one round
// trip to the L2, where another kernel for a plan would cost a launch). False:
// none.
template <int TPB, int U, class Count>
__device__ bool find_run(const AttnArgs &A, Count count, RunLds &lds, Run &r) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, parts = A.b.n_seqs + 1;
    // units of sequence i - 1 and of those before it, for i = c + tid; returns the total up to c + TPB
    Work w{};
    auto scan = [&](int c, long long run, long long &mine, long long &before) {
        const int i = c + tid;
        mine = 0;
        if (i < parts && (i > 0 ? A.last == 1 : A.first == 0)) {
            w = work_of<U>(A, i - 1);
            mine = count(i - 1, w);
        }
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
        for (int k = 0; k < TPB / 64; k++) {
            if (k < wave) before += lds.scan[k];
            run += lds.scan[k];
        }
        return run;
    };
    auto keep = [&](int s, long long b) {
        lds.seq = s, lds.off = r.u - b;
        lds.work[0] = w.lo, lds.work[1] = w.n, lds.work[2] = w.len, lds.work[3] = w.base, lds.work[4] = w.end;
        lds.work[5] = w.units, lds.work[6] = w.blocks;
    };
    long long mine = 0, before = 0;
    r.T = 0;
    for (int c = 0; c < parts; c += TPB) r.T = scan(c, r.T, mine, before);
    r.T = uniform(r.T);
    r.runs = (int)min((long long)A.part[A.first].G, r.T);  // no empty runs between others
    if ((int)blockIdx.x >= r.runs) return false;
    r.u = run_start(r.T, r.runs, (int)blockIdx.x);
    r.u1 = run_start(r.T, r.runs, (int)blockIdx.x + 1);
    if (parts <= TPB) {
        if (mine > 0 && before <= r.u && r.u < before + mine) keep(tid - 1, before);
    } else {
        long long run = 0;
        for (int c = 0; c < parts; c += TPB) {
            run = scan(c, run, mine, before);
            if (mine > 0 && before <= r.u && r.u < before + mine) keep(c + tid - 1, before);
        }
    }
    __syncthreads();
    r.seq = uniform(lds.seq);
    r.off = uniform(lds.off);
    r.work = Work{uniform(lds.work[0]), uniform(lds.work[1]), uniform(lds.work[2]), uniform(lds.work[3]),
                  uniform(lds.work[4]), uniform(lds.work[5]), uniform(lds.work[6])};
    return true;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace
}  // namespace uq
