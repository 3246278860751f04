// lq_paged.h -- what the kernels over a paged key-value cache share: the places of appended tokens, the
// rules of a row's codes, the plan that spreads attention over workgroups, a wave's sums and their meeting.
#pragma once

#include <type_traits>

#include "lq_attn.h"
#include "lq_place.h"

namespace lq {

// ------------------------------------------------------------------------------ append

struct AppendArgs {
    const void *k, *v;
    int64_t ld, tokens;
    const int32_t* starts;
    int64_t seqs, Hkv, hd;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    void *kp, *vp;
    void *ks, *vs;  // float32 of int8 rows, bfloat16 of 4-bit ones
    int64_t pages, page;
};

// Row of packed token t's head 0 in the pool, or -1 when it has no place.
__device__ __forceinline__ int64_t token_row(const AppendArgs& a, int64_t t) {
    int64_t s, pos;
    if (!token_place(t, a.starts, a.seqs, a.lengths, s, pos)) return -1;
    return position_row(pos, a.table + s * a.table_stride, a.table_stride, a.pages, a.Hkv, a.page);
}

// Eight source values as float32, and eight values stored.
template <class Src>
__device__ __forceinline__ void load8(const typename Src::T* p, float (&x)[8]) {
    if constexpr (Src::code == LQ_F32) {
        const vf4 lo = __builtin_nontemporal_load(reinterpret_cast<const vf4*>(p));
        const vf4 hi = __builtin_nontemporal_load(reinterpret_cast<const vf4*>(p) + 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = lo[j];
            x[j + 4] = hi[j];
        }
    } else {
        const u4v w = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(p));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f2v u = unpack2(Src{}, w[j]);
            x[2 * j] = u[0];
            x[2 * j + 1] = u[1];
        }
    }
}

// int8 rows: scale = max|x| / 127, code = rne(x * (127 / max|x|)); a row whose largest magnitude is below
// 127 / FLT_MAX (or 0) is stored as zeros; one that holds an infinity or NaN gets a scale that is not
// finite, so that it reads back as NaN or infinity.
struct RowScale {
    float inv, scale;
    __device__ __forceinline__ explicit RowScale(int32_t top) {  // the largest |x| as bits (NaN above infinity)
        const float amax = __builtin_bit_cast(float, top);
        inv = 127.0f / amax;
        const bool zero = amax == amax && !(inv < INFINITY);
        scale = zero ? 0.0f : amax / 127.0f;
        if (zero) inv = 0.0f;
    }
    __device__ __forceinline__ int code(float x) const {
        const float c = rne(x * inv);
        return c == c ? (int)fminf(fmaxf(c, -127.0f), 127.0f) : 0;
    }
};
__device__ __forceinline__ int32_t magnitude(float x) { return __builtin_bit_cast(int32_t, x) & 0x7fffffff; }

// ------------------------------------------------------------------------------ attention

struct PagedArgs {
    const void* q;
    int64_t ldq;
    int B, H, Hkv, hd, group, qtiles;
    const void *k, *v;
    const void *ks, *vs;  // float32 of int8 rows, bfloat16 of 4-bit ones
    int64_t pages;
    int page;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    float scale;
    void* out;
    int out_f32;
    int q_vec;          // q may be read 16 bytes at a time
    int groups;         // workgroups that share all positions evenly; 0: one per sequence and key head
    int2* pieces;       // [B][key head and tile of query heads]: first piece's slot, number of pieces
    float *part_o, *part_ml;
};

constexpr int PG_K = 32;        // positions of a wave's tile
constexpr int PG_I8_WAVES = 4;  // waves of a workgroup over an int8 cache

// Length of sequence b within its table (positions past it are an error: `over`).
__device__ __forceinline__ int sequence_length(const PagedArgs& a, int b, bool& over) {
    const int64_t cap = min(a.table_stride * a.page, (int64_t)(INT32_MAX - 4096));
    const int len = max(a.lengths[b], 0);
    over = len > cap;
    return over ? (int)cap : len;
}

// The kernels share this plan.  The work is a line of steps (WAVES tiles of 32 positions, of 64 over 4-bit pages): all steps
// of the first sequence's first key head (and tile of 16 query heads), then of its next one, and so
// on.  Each workgroup takes an equal part of the line (PAIRS: one of two sizes), whatever the sequences' lengths, and works
// through the pieces of sequences in it one after the other.  A piece costs some microseconds of dependent
// loads before its first tile, which counts as START steps on the line (without it 64 sequences of 256 to
// 8191 positions took 128 us, with it 110).  Where parts of 256 or 512 positions are enough for all, each
// lies within one sequence instead.  A piece that is
// a whole sequence is written at once, others go to the workspace (a workgroup has two at most, its first
// and its last) and are joined by a second launch.  With short sequences (`groups` 0) a workgroup takes
// one of them whole and there is no second launch.
//
// Within a piece each wave takes every WAVES-th tile with a maximum, sum and accumulators of its own, and
// the waves meet at the end: no barrier inside the loop.
//   S^T = K Q^T (v_mfma 16x16x32): K is the A operand, row l (and 16 + l) in lane (l, g), which receives
//   positions 4 g + i (and 16 + 4 g + i) of query l;
//   O^T += V^T P^T: those weights are the B operand as they are; V comes from the wave's LDS, whose
//   transposing read gives lane (l, g) dim l of the same positions.
// A weight enters as 16-bit terms: two hold 22 bits of it in fp16 and 16 in bfloat16, which is more than a
// 16-bit output keeps; a float32 output takes a third one in bfloat16 (24 bits).  The products are free
// beside the loads.
struct Piece {
    int b, h0, hk, heads, begin, end, len;
    bool over, whole;
    int64_t slot;
};

// n / d of numbers that are seldom past 32 bits: the longer division is a few hundred instructions.
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
    return (n | d) >> 32 ? n / d : (int64_t)((uint32_t)n / (uint32_t)d);
}
// What lane `i` of the wave holds, the same in all.
__device__ __forceinline__ int64_t of_lane(int64_t v, int i) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)v, i), hi = __builtin_amdgcn_readlane((int)(v >> 32), i);
    return (int64_t)((uint64_t)hi << 32 | lo);
}
// The sum over this lane and those below it.
template <int FROM, int ROWS>
__device__ __forceinline__ int64_t add_moved(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)v, FROM, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), FROM, ROWS, 0xF, false);
    return v + (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t wave_upto(int64_t v) {
    v = add_moved<0x111, 0xF>(v);  // row_shr: 1, 2, 4, 8
    v = add_moved<0x112, 0xF>(v);
    v = add_moved<0x114, 0xF>(v);
    v = add_moved<0x118, 0xF>(v);
    v = add_moved<0x142, 0xA>(v);    // lane 15 of the row before, into rows 1 and 3
    return add_moved<0x143, 0xC>(v);  // lane 31, into rows 2 and 3
}

// The line of steps as a workgroup walks it.
template <int WAVES, int TILE = PG_K>
struct Line {
    static constexpr int STEP = WAVES * TILE, NT = 64 * WAVES;
    static constexpr int PART = STEP < 256 ? 256 / STEP : 1, PART2 = STEP < 512 ? 512 / STEP : 1;  // 256, 512 positions
    // a start is 256 positions' time; over 4-bit pages, which pass faster, 512 (1 / 2 / 3 / 5 steps of 256: 64 sequences of
    // up to 8191 positions 49.1 / 46.8 / 48.3 / 52.3 us, long ones alike)
    static constexpr int START = TILE == 64 ? 2 * PART : PART;
    static_assert((PART & (PART - 1)) == 0 && (PART2 & (PART2 - 1)) == 0, "masks");
    int64_t share, at, stop, start;  // steps of a workgroup; next step, end and start of this part
    // Over 4-bit pages the later of two workgroups on a CU is the slower one: the older waves issue first (even parts ended
    // after 34 and 43 us).  A workgroup of the first half takes 5/8 of the two's steps: long sequences 47.5 -> 44.3 us,
    // 64 of up to 8191 46.8 -> 43.6 (1/2 in whole steps: 47.3 and 45.0, 11/16: 46.8 and 45.7; priorities that
    // change with every tile: 45.1 and 44.3).  Calls of both kinds, even parts / 5/8: 32 dims 30.5 / 29.0 and 31.2 / 28.8
    // us, 64 dims 37 / 34.4 and 37.2 / 34.3, 96 dims 46.2 / 43.8 and 43.6 / 41.2, 128 dims 54.2 / 52.9 and 51.3 / 48.8.  That
    // takes workgroups n and n + groups / 2 to share a CU; where other work holds the CUs the first half end later instead.
    int64_t half, late;  // workgroups of the first half; steps of one of the second
    int64_t base;        // first step of sequence b
    static constexpr bool PAIRS = TILE == 64;  // two workgroups to a CU up to 128 dims
    int b, len, steps, heads;  // heads: key heads times tiles of 16 query heads
    int cost;                  // places of one head of sequence b on the line
    int unit, lead;            // steps that a part is a multiple of (0: any), places before a head's first step
    bool over;

    __device__ __forceinline__ void sequence(const PagedArgs& a, int i) {
        b = i;
        len = sequence_length(a, i, over);
        steps = (len + STEP - 1) / STEP;
        places();
    }
    __device__ __forceinline__ void places() { cost = unit ? (steps + unit - 1) & -unit : steps ? steps + START : 0; }
    // Finds the part of this workgroup; `scan` holds WAVES + 1 numbers.
    __device__ __forceinline__ void init(const PagedArgs& a, int64_t* scan) {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        heads = a.Hkv * a.qtiles;
        unit = 0;
        if (a.groups == 0) {
            lead = START;
            const uint32_t n = (uint32_t)workgroup(), i = n / (uint32_t)heads;
            start = at = stop = base = 0;
            if (i >= (uint32_t)a.B) return;
            sequence(a, (int)i);
            start = at = (int64_t)(n - i * heads) * cost;
            stop = at + cost;
            return;
        }
        if (a.B <= 64) return init_alone(a);
        const int per = (a.B + NT - 1) / NT, first = min(tid * per, a.B), last = min(first + per, a.B);
        // parts of 256 or 512 positions, if the workgroups suffice: none then has two pieces (a thread counts no
        // further than 2^20 parts, more than there are workgroups)
        int64_t n256 = 0, n512 = 0;
        for (int i = first; i < last; ++i) {
            sequence(a, i);
            n256 += (int64_t)heads * ((steps + PART - 1) / PART);
            n512 += (int64_t)heads * ((steps + PART2 - 1) / PART2);
        }
        int small = wave_add((int)min(n256, (int64_t)1 << 20)), large = wave_add((int)min(n512, (int64_t)1 << 20));
        if (lane == 0) scan[wave] = (int64_t)small << 32 | large;
        __syncthreads();
        small = large = 0;
        for (int w = 0; w < WAVES; ++w) {
            small += (int)(scan[w] >> 32);
            large += (int)scan[w];
        }
        unit = small <= a.groups ? PART : large <= a.groups ? PART2 : 0;
        lead = unit ? 0 : START;
        int64_t mine = 0;
        for (int i = first; i < last; ++i) {
            sequence(a, i);
            mine += (int64_t)heads * cost;
        }
        const int64_t upto = wave_upto(mine);
        __syncthreads();
        if (lane == 63) scan[wave] = upto;
        __syncthreads();
        int64_t before = upto - mine, total = 0;
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) before += scan[w];
            total += scan[w];
        }
        total = of_lane(total, 0);
        part_of(a, total);
        if (at >= stop) return;
        __syncthreads();
        if (at >= before && at < before + mine) {  // one thread's sequences
            scan[0] = before;
            scan[1] = first;
        }
        __syncthreads();
        base = of_lane(scan[0], 0);
        sequence(a, (int)of_lane(scan[1], 0));
        advance(a);
    }
    // The same for up to 64 sequences, one a lane: each wave for itself, without a barrier, each length loaded once.  A
    // workgroup has its part after 2400 cycles; with the scan over the workgroup, a search in LDS and 64-bit
    // divisions it had it after 6500 (32 sequences of up to 2047 positions of 4 bits: 16.1 us, 17.4 with those).
    __device__ __forceinline__ void init_alone(const PagedArgs& a) {
        const int lane = threadIdx.x & 63;
        sequence(a, min(lane, a.B - 1));
        if (lane >= a.B) steps = 0;
        auto parts = [&](int of) {
            return wave_add((int)min((int64_t)heads * ((steps + of - 1) / of), (int64_t)1 << 20));
        };
        unit = parts(PART) <= a.groups ? PART : parts(PART2) <= a.groups ? PART2 : 0;
        lead = unit ? 0 : START;
        places();
        const int64_t mine = (int64_t)heads * cost, upto = wave_upto(mine);
        part_of(a, of_lane(upto, 63));
        if (at >= stop) return;
        const int from = __builtin_ctzll(__ballot(at >= upto - mine && at < upto));
        base = of_lane(upto - mine, from);
        b = from;
        len = __builtin_amdgcn_readlane(len, from);
        steps = __builtin_amdgcn_readlane(steps, from);
        cost = __builtin_amdgcn_readlane(cost, from);
        over = __builtin_amdgcn_readlane((int)over, from);
    }
    __device__ __forceinline__ void part_of(const PagedArgs& a, int64_t total) {
        const int64_t n = blockIdx.x;
        share = unit ? unit : quotient(total + a.groups - 1, a.groups);
        start = n * share;
        int64_t mine = share;
        if constexpr (PAIRS) {
            half = a.groups / 2;
            late = share;
            if (!unit && a.hd <= 128) {
                const int64_t pair = quotient(total + half - 1, half);
                share = min(pair, (pair * 5 + 4) / 8);
                late = pair - share;
                start = min(n, half) * share + max(n - half, (int64_t)0) * late;
                mine = n < half ? share : late;
            }
        }
        start = at = min(start, total);
        stop = min(at + mine, total);
    }
    // The workgroup with place x of the line.
    __device__ __forceinline__ int owner(int64_t x) const {
        if constexpr (PAIRS) {
            if (x >= half * share) return (int)(half + quotient(x - half * share, late));
        }
        return (int)quotient(x, share);
    }
    __device__ __forceinline__ void advance(const PagedArgs& a) {
        while (at >= base + (int64_t)heads * cost) {
            base += (int64_t)heads * cost;
            sequence(a, b + 1);
        }
    }
    // The next piece; false when the part is done.  Uniform over the workgroup.
    __device__ __forceinline__ bool next(const PagedArgs& a, Piece& p) {
        while (at < stop) {
            advance(a);
            const int hq = (int)quotient(at - base, cost), x0 = (int)(at - base - (int64_t)hq * cost);
            const int x1 = (int)min((int64_t)cost, x0 + (stop - at));
            const int s0 = max(x0 - lead, 0), s1 = min(x1 - lead, steps);
            const bool first = at == start;
            at += x1 - x0;
            if (s1 <= 0) continue;  // nothing but the start of a sequence whose steps come in the next part
            const int qt = hq % a.qtiles;
            p.b = b;
            p.hk = hq / a.qtiles;
            p.heads = min(16, a.group - 16 * qt);
            p.h0 = p.hk * a.group + 16 * qt;
            p.len = len;
            p.over = over;
            p.begin = s0 * STEP;
            p.end = min(s1 * STEP, len);
            p.whole = s1 - s0 == steps;
            p.slot = 2 * (int64_t)blockIdx.x + (first ? 0 : 1);
            if (a.groups && s0 == 0 && threadIdx.x == 0) {  // for the join
                const int64_t end = base + (int64_t)hq * cost + lead + steps - 1;  // its last step
                const int more = p.whole ? 0 : owner(end) - (int)blockIdx.x;
                a.pieces[(int64_t)b * heads + hq] = make_int2((int)p.slot, more + 1);
            }
            return true;
        }
        return false;
    }
};

// Sequences without a position: 0, or NaN where only the table is missing.
template <int WAVES, class Q>
__device__ __forceinline__ void paged_empty(const PagedArgs& a) {
    const int64_t row = (int64_t)a.H * a.hd;
    for (int64_t b = workgroup(); b < a.B; b += (int64_t)gridDim.x * gridDim.y) {
        bool over;
        if (sequence_length(a, (int)b, over) > 0) continue;
        const float y = over ? __builtin_nanf("") : 0.0f;
        const int heads = a.Hkv * a.qtiles;
        if (a.groups)
            for (int e = threadIdx.x; e < heads; e += 64 * WAVES) a.pieces[b * heads + e] = make_int2(0, 0);
        for (int64_t e = threadIdx.x; e < row; e += 64 * WAVES) {
            if (a.out_f32) static_cast<float*>(a.out)[b * row + e] = y;
            else static_cast<typename Q::T*>(a.out)[b * row + e] = Q::store(y);
        }
    }
}

// Eight dims from d on of query head h0 + min(l, heads - 1), zeros past the head dim.
__device__ __forceinline__ u4v paged_query(const PagedArgs& a, const Piece& w, int l, int d, int hd) {
    u4v f = {0, 0, 0, 0};
    if (d >= hd) return f;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + w.b * a.ldq + (int64_t)(w.h0 + min(l, w.heads - 1)) * hd + d;
    if (a.q_vec) return *reinterpret_cast<const u4v*>(q);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j >> 1] |= (uint32_t)q[j] << (16 * (j & 1));
    return f;
}

// Statistics and accumulators of a wave: 16 queries, DT * 16 dims.
template <int DT, class P>
struct Sums {
    vf4 o[DT];
    float m, l;
    __device__ __forceinline__ Sums() : m(-INFINITY), l(0.0f) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = vf4{0.f, 0.f, 0.f, 0.f};
    }
    // Scores (of n positions from this lane's 4 g on, -inf past them) to weights relative to the
    // running maximum; the accumulators follow it only when it has risen by more than 2^RESCALE_AT.
    __device__ __forceinline__ void weights(vf4 (&sc)[2], float sl2, bool whole, int n) {
        float mx = -INFINITY;
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!whole && 16 * T + i >= n) sc[T][i] = -INFINITY;
                mx = fmaxf(mx, sc[T][i]);
            }
        mx = quarter_max(mx) * sl2;
        if (__any(mx > m + RESCALE_AT)) {
            const float mn = fmaxf(m, weight_reference<P>(mx));
            const float corr = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] *= corr;
        }
        const float base = m == -INFINITY ? 0.0f : m - WEIGHT_SHIFT<P>;
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[T][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[T][i], sl2, -base));
                l += sc[T][i];
            }
    }
    // O^T += V^T P^T, V at LDS `v_at` with rows of VROW bytes swizzled by swz; `all`: every bit of the weights
    template <int VROW, class F>
    __device__ __forceinline__ void accumulate(const vf4 (&w)[2], uint32_t v_at, F swz, bool all) {
        const bool third = P::code == LQ_BF16 && all;
        u4v ph, pl;
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t u = pack2(P{}, w[T][2 * i], w[T][2 * i + 1]);
                const f2v r = unpack2(P{}, u);
                ph[2 * T + i] = u;
                pl[2 * T + i] = pack2(P{}, w[T][2 * i] - r[0], w[T][2 * i + 1] - r[1]);
            }
        const int lane = threadIdx.x & 63, vi = lane & 15, row = 4 * (lane >> 4) + (vi >> 2);
        auto values = [&](int d) __attribute__((always_inline)) {
            const uint32_t at = v_at + row * VROW + (((2 * d + ((vi & 3) >> 1)) ^ swz(row)) << 4) + 8 * (vi & 1);
            const u2v lo = lds_read_tr(at), hi = lds_read_tr(at + 16 * VROW);
            return u4v{lo[0], lo[1], hi[0], hi[1]};
        };
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const u4v v = values(d);
            o[d] = mfma_16x16x32(P{}, v, ph, o[d]);
            o[d] = mfma_16x16x32(P{}, v, pl, o[d]);
        }
        if (third) {  // apart, so that the loop above stays one block
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f2v r = unpack2(P{}, ph[2 * T + i]), e = unpack2(P{}, pl[2 * T + i]);
                    ph[2 * T + i] = pack2(P{}, w[T][2 * i] - r[0] - e[0], w[T][2 * i + 1] - r[1] - e[1]);
                }
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = mfma_16x16x32(P{}, values(d), ph, o[d]);
        }
    }
};

// Dim d of row r's sum over a piece, key by key: for values that hold an infinity, which the second term
// of a weight turned into NaN.  M: the piece's maximum.
template <class Q>
__device__ __forceinline__ float paged_sum_again(const PagedArgs& a, const Piece& w, int r, int d, float M) {
    const typename Q::T* q = static_cast<const typename Q::T*>(a.q) + w.b * a.ldq + (int64_t)(w.h0 + r) * a.hd;
    const int32_t* table = a.table + (int64_t)w.b * a.table_stride;
    const float base = M == -INFINITY ? 0.0f : M - WEIGHT_SHIFT<Q>;
    float x = 0.0f;
    for (int key = w.begin; key < w.end; ++key) {
        const int64_t row0 = position_row(key, table, a.table_stride, a.pages, a.Hkv, a.page);
        if (row0 < 0) return __builtin_nanf("");
        const int64_t row = row0 + (int64_t)w.hk * a.page;
        const typename Q::T* k = static_cast<const typename Q::T*>(a.k) + row * a.hd;
        float s = 0.0f;
        for (int i = 0; i < a.hd; ++i) s = __builtin_fmaf(Q::load(q[i]), Q::load(k[i]), s);
        const float f = __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.scale * LOG2E, -base));
        x = __builtin_fmaf(f, Q::load(static_cast<const typename Q::T*>(a.v)[row * a.hd + d]), x);
    }
    return x;
}

// The waves' sums meet: wave w's lie at LDS lds + w * SLOT (16 queries of OROW floats each), and the
// workgroup writes the output or its part of it.  AGAIN: the pages hold values of type Q, infinities among
// them; pages of codes are not read that way.
template <bool AGAIN, int WAVES, int SLOT, int DT, class Q, class P>
__device__ __forceinline__ void paged_finish(const PagedArgs& a, const Piece& w, uint8_t* lds, float (*ml)[2][16],
                                             Sums<DT, P>& s, bool bad) {
    constexpr int OROW = 16 * DT + 4;
    static_assert(16 * OROW * 4 <= SLOT, "the sums fit the wave's LDS");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4, hd = a.hd;
    float l = quarter_sum(s.l);
    if (__any(bad)) l = __builtin_nanf("");
    float* so = reinterpret_cast<float*>(lds + wave * SLOT);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<vf4*>(so + l16 * OROW + 16 * d + 4 * g) = s.o[d];
    if (g == 0) {
        ml[wave][0][l16] = s.m;
        ml[wave][1][l16] = l;
    }
    __syncthreads();
    for (int e = tid; e < w.heads * hd; e += 64 * WAVES) {
        const int r = e / hd, d = e - r * hd;
        float M = -INFINITY;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) M = fmaxf(M, ml[v][0][r]);
        const float base = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, x = 0.0f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            const float f = __builtin_amdgcn_exp2f(ml[v][0][r] - base);
            L = __builtin_fmaf(f, ml[v][1][r], L);
            x = __builtin_fmaf(f, reinterpret_cast<const float*>(lds + v * SLOT)[r * OROW + d], x);
        }
        if constexpr (AGAIN)
            if (!(fabsf(x) < INFINITY) && L == L) x = paged_sum_again<Q>(a, w, r, d, M);
        if (w.whole) {
            const int64_t at = ((int64_t)w.b * a.H + w.h0 + r) * hd + d;
            if (a.out_f32) static_cast<float*>(a.out)[at] = x / L;
            else static_cast<typename Q::T*>(a.out)[at] = Q::store(x / L);
        } else {
            a.part_o[(16 * w.slot + r) * hd + d] = x;
            if (d == 0) {
                a.part_ml[2 * (16 * w.slot + r)] = M;
                a.part_ml[2 * (16 * w.slot + r) + 1] = L;
            }
        }
    }
    __syncthreads();  // the next piece fills this LDS again
}

// V rows in LDS: 16-byte chunk c of row r lies at chunk c ^ v_swz(r), so that the transposing reads (4 rows,
// 2 chunks for 16 lanes) and the writes spread over the banks; K rows (16 lanes read 16 rows): c ^ k_swz(r).
template <int HDP>
__device__ __forceinline__ int k_swz(int r) {
    return HDP == 64 ? (r >> 1) & 7 : HDP % 128 == 0 ? r & 15 : r & 7;
}
template <int HDP>
__device__ __forceinline__ int v_swz(int r) {
    return HDP == 64 ? 2 * ((r >> 1) & 3) : HDP % 128 == 0 ? 2 * (r & 7) : 2 * (r & 3);
}

}  // namespace lq
