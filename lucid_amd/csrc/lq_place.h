// lq_place.h -- where packed tokens and cached positions live.  Every index that a kernel takes
// from device memory (starts, lengths, page numbers) is checked here before it becomes an
// address, so the rules are plain host code too.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define LQ_PLACE __host__ __device__ __forceinline__
#else
#define LQ_PLACE inline
#endif

namespace lq {

// Workgroups of a launch in two dimensions.  A launch takes fewer than 2^32 work items in x: rows of 2^22
// workgroups (of 512 threads at most), the last row in part past the end, as many rows as it takes
// (65535 at most, that is 2.7e11 workgroups: more than the memory has rows for).
struct Workgroups {
    uint32_t x, y;
};
constexpr int64_t WORKGROUPS_X = (int64_t)1 << 22;
LQ_PLACE Workgroups workgroups(int64_t n) {
    return n <= WORKGROUPS_X ? Workgroups{(uint32_t)n, 1}
                             : Workgroups{(uint32_t)WORKGROUPS_X, (uint32_t)((n + WORKGROUPS_X - 1) / WORKGROUPS_X)};
}
LQ_PLACE int64_t workgroup_index(uint32_t x, uint32_t y) { return (int64_t)y * WORKGROUPS_X + x; }

// The last of `seqs` (>= 1) sequences whose start is at or before t (the first one if none is).
// Any contents of starts[0 .. seqs - 1] give a number in [0, seqs).
LQ_PLACE int64_t sequence_of(const int32_t* starts, int64_t seqs, int64_t t) {
    int64_t lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Row (in rows of hd values) of head 0 of a position in the pool [pages][Hkv][page][hd], or -1
// when the position is negative, past the table's row or in a page outside the pool.  Head h is
// h * page rows further.
LQ_PLACE int64_t position_row(int64_t pos, const int32_t* table_row, int64_t table_stride, int64_t pages, int64_t Hkv,
                              int64_t page) {
    if (pos < 0) return -1;
    const int64_t col = pos / page;
    if (col >= table_stride) return -1;
    const int64_t id = table_row[col];
    if (id < 0 || id >= pages) return -1;
    return id * Hkv * page + (pos - col * page);
}

// Sequence and position of packed token t that is being appended (starts NULL: one token per
// sequence); false when it belongs to no sequence.  The sequence's length counts its new tokens.
LQ_PLACE bool token_place(int64_t t, const int32_t* starts, int64_t seqs, const int32_t* lengths, int64_t& s,
                          int64_t& pos) {
    s = t;
    int64_t fresh = 1, i = 0;
    if (starts) {
        s = sequence_of(starts, seqs, t);
        i = t - starts[s];
        fresh = (int64_t)starts[s + 1] - starts[s];
        if (i < 0 || i >= fresh) return false;
    }
    pos = (int64_t)lengths[s] - fresh + i;
    return true;
}

// Rows of one sequence of a packed pair (q, k), kept inside the totals whatever the starts hold,
// and the keys a query of it sees.
struct Packed {
    int64_t q0, nq, k0, nk;
};
LQ_PLACE Packed packed_sequence(const int32_t* qs, const int32_t* ks, int64_t s, int64_t total_q, int64_t total_k) {
    Packed p;
    const int64_t qa = qs[s], qb = qs[s + 1], ka = ks[s], kb = ks[s + 1];
    p.q0 = qa < 0 ? 0 : qa > total_q ? total_q : qa;
    p.nq = (qb > total_q ? total_q : qb) - p.q0;
    if (p.nq < 0) p.nq = 0;
    p.k0 = ka < 0 ? 0 : ka > total_k ? total_k : ka;
    p.nk = (kb > total_k ? total_k : kb) - p.k0;
    if (p.nk < 0) p.nk = 0;
    return p;
}
LQ_PLACE int64_t keys_seen(const Packed& p, int64_t i, bool causal) {
    const int64_t n = causal ? p.nk - p.nq + i + 1 : p.nk;
    return n < 0 ? 0 : n > p.nk ? p.nk : n;
}

}  // namespace lq
