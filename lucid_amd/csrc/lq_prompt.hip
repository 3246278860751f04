// lq_prompt.hip -- attention over packed prompts of different lengths, with grouped heads.
//
// Sequence s owns rows q_starts[s] .. q_starts[s + 1] - 1 of q and k_starts[s] .. of k / v.  With
// `causal`, query i of nq sees keys 0 .. nk - nq + i (the queries are the last nq of nk
// positions); a query that sees no key has the output 0.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_attn.h"
#include "lq_dma.h"
#include "lq_place.h"

namespace lq {
namespace {

struct PromptArgs {
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv;
    const int32_t *qs, *ks;
    int64_t seqs, total_q, total_k, H, Hkv, hd;
    int causal;
    float scale;
    void* out;
};

// Query t of head h (key head hk) over keys k0 .. k0 + len - 1, by one wave: 64 keys at a time, a lane
// scores one key, then adds its dims (lane, lane + 64, ...) of the weighted values.  Reads nothing
// but the keys seen, element by element: for operands that no vector fits, and for queries whose
// tiles hold infinities or NaN.
template <class E, class Out>
__device__ __forceinline__ void attend_row(const PromptArgs& a, int64_t t, int h, int hk, int64_t k0, int64_t len) {
    constexpr int PARTS = ATTN_MAX_HD / 64;
    const int lane = threadIdx.x & 63, hd = (int)a.hd;
    const typename E::T* q = static_cast<const typename E::T*>(a.q) + t * a.ldq + (int64_t)h * hd;
    const typename E::T* k = static_cast<const typename E::T*>(a.k) + k0 * a.ldk + (int64_t)hk * hd;
    const typename E::T* v = static_cast<const typename E::T*>(a.v) + k0 * a.ldv + (int64_t)hk * hd;
    const float fit = E::code == LQ_BF16 ? exp2f(WEIGHT_SHIFT<E>) : 1.0f;  // sums of the largest values stay finite
    float m = -INFINITY, l = 0.0f, acc[PARTS] = {};
    for (int64_t kb = 0; kb < len; kb += 64) {
        const int n = (int)min((int64_t)64, len - kb);
        float s = -INFINITY;
        if (lane < n) {
            const typename E::T* kr = k + (kb + lane) * a.ldk;
            s = 0.0f;
            for (int d = 0; d < hd; ++d) s = __builtin_fmaf(E::load(q[d]), E::load(kr[d]), s);
            s *= a.scale * LOG2E;
        }
        float mx = s;
        for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
        mx = fmaxf(mx, m);
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float e = lane < n ? __builtin_amdgcn_exp2f(s - base) * fit : 0.0f;
        const float corr = __builtin_amdgcn_exp2f(m - base);
        m = mx;
        l = l * corr + ln_wave_sum(e);
#pragma unroll
        for (int c = 0; c < PARTS; ++c) acc[c] *= corr;
        for (int j = 0; j < n; ++j) {
            const float p = __shfl(e, j, 64);
#pragma unroll
            for (int c = 0; c < PARTS; ++c)
                if (lane + 64 * c < hd) acc[c] = __builtin_fmaf(p, E::load(v[(kb + j) * a.ldv + lane + 64 * c]), acc[c]);
        }
    }
    typename Out::T* o = static_cast<typename Out::T*>(a.out) + (t * a.H + h) * hd;
#pragma unroll
    for (int c = 0; c < PARTS; ++c)
        if (lane + 64 * c < hd) o[lane + 64 * c] = Out::store(len > 0 ? acc[c] / l : 0.0f);
}

// One wave per (head, query).
template <class E, class Out>
__global__ __launch_bounds__(64) void prompt_rows_kernel(PromptArgs a) {
    const int64_t t = blockIdx.y + (int64_t)blockIdx.z * 65535;
    if (t >= a.total_q) return;
    const int64_t sq = sequence_of(a.qs, a.seqs, t);
    const Packed pk = packed_sequence(a.qs, a.ks, sq, a.total_q, a.total_k);
    if (t < pk.q0 || t >= pk.q0 + pk.nq) return;
    attend_row<E, Out>(a, t, blockIdx.x, blockIdx.x / (int)(a.H / a.Hkv), pk.k0, keys_seen(pk, t - pk.q0, a.causal));
}

// ------------------------------------------------------------------------- the tile kernel

constexpr int PT_WAVES = 4, PT_K = 64;  // waves of a workgroup, keys of a tile

// Sequence and query block of workgroup index n; false past the last block.  Under the causal mask later
// blocks have more keys, and the longest work starts first: up to 64 sequences, block L of every
// sequence that has one before any block L - 1 (at the count of blocks from L on, which a search
// finds); with more, blocks last to first within each sequence.  Every wave finds it by itself, a lane
// for each of 64 sequences, and takes the sequence's rows from that lane.
template <int QB>
__device__ __forceinline__ bool find_block(const PromptArgs& a, int64_t n, Packed& pk, int64_t& blk) {
    const int lane = threadIdx.x & 63;
    Packed mine{0, 0, 0, 0};  // this lane's sequence
    auto blocks = [&](int64_t s) {
        if (s >= a.seqs) return 0;
        mine = packed_sequence(a.qs, a.ks, s, a.total_q, a.total_k);
        return (int)((mine.nq + QB - 1) / QB);
    };
    auto take = [&](int l) {  // the rows of lane l's sequence, in scalar registers
        pk.q0 = __builtin_amdgcn_readlane((int)mine.q0, l);
        pk.nq = __builtin_amdgcn_readlane((int)mine.nq, l);
        pk.k0 = __builtin_amdgcn_readlane((int)mine.k0, l);
        pk.nk = __builtin_amdgcn_readlane((int)mine.nk, l);
    };
    if (a.seqs <= 64) {
        const int cnt = blocks(lane);
        auto from = [&](int level) { return wave_add(max(cnt - level, 0)); };  // blocks at or past a level
        if (n >= from(0)) return false;
        int lo = 0, hi = wave_max(cnt);  // from(lo) > n >= from(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (from(mid) > n) lo = mid; else hi = mid;
        }
        uint64_t has = __ballot(cnt > lo);
        for (int64_t k = n - from(lo + 1); k > 0; --k) has &= has - 1;
        take(__builtin_ctzll(has));
        blk = lo;
        return true;
    }
    for (int64_t base = 0; base < a.seqs; base += 64) {
        int upto = blocks(base + lane);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d, 64);
            if (lane >= d) upto += o;
        }
        const int all = __builtin_amdgcn_readlane(upto, 63);
        if (n < all) {
            const int l = __builtin_ctzll(__ballot(upto > n));
            take(l);
            blk = __builtin_amdgcn_readlane(upto, l) - 1 - n;
            return true;
        }
        n -= all;
    }
    return false;
}

// A workgroup of four waves; SPLIT of them share 32 queries and take 64 / SPLIT keys of a tile each, so
// that it has QB = 128 / SPLIT queries.  K and V tiles are copied to LDS one ahead (three ahead, with one
// workgroup to a CU, was no faster where few workgroups run and slower elsewhere).
//   S^T = K Q^T (v_mfma 32x32x16): a lane receives 16 keys of one query, so the softmax statistics are one
//   number a lane;
//   O^T += V^T P^T: those weights are the B operand as they are (no exchange between lanes), and V^T is
//   what the transposing read of the V rows gives.  A rescale is one factor a lane.
// The scores of the next tile are on the matrix cores while the vector unit makes this tile's weights (one
// wave's exponentials beside its own products: 12288 tokens, 32 heads of 128 in bfloat16, 1192 -> 1135
// us; an order of the two forced by scheduling hints 1155).
// What bounds it: at that size 1100 TFLOP/s, where a library product of 16384^3 reaches 1326 on this
// card; the card keeps 1.6 to 1.9 GHz under this load, at which the matrix cores are busy 61% of the
// time and the vector unit 54% (exponentials, sums and roundings of the weights, only in part beside
// the products).  Short sequences add some 4 us of dependent loads to every workgroup.
template <int HDP, int SPLIT, class E, class Out>
__global__ __launch_bounds__(64 * PT_WAVES, HDP <= 64 ? 3 : HDP <= 128 ? 2 : 1) void prompt_tile_kernel(PromptArgs a) {
    constexpr int QB = 32 * PT_WAVES / SPLIT;
    constexpr int CPR = HDP / 8;                                // 16-byte chunks of a row
    constexpr int TILE = PT_K * HDP * 2;                        // bytes of a K (or V) tile
    constexpr int COPIES = PT_K * CPR / (64 * PT_WAVES);        // 16-byte copies of a lane per tile
    constexpr int KS = HDP / 16, DT = HDP / 32, KT = PT_K / 32 / SPLIT;
    // A weight enters its product in 16 bits: once rounded for a 16-bit output (one more rounding of the size of
    // the output's own; a second term would be half as many products again, and they bound the kernel);
    // as two terms in fp16 (22 bits), three in bfloat16 (24 bits), for a float32 output.
    constexpr int TERMS = Out::code != LQ_F32 ? 1 : E::code == LQ_F16 ? 2 : 3;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TILE];
    __shared__ int odd_values[PT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hh = lane >> 5;
    const uint32_t group = (uint32_t)(a.H / a.Hkv);
    const uint32_t id = (uint32_t)workgroup(), n = id / (uint32_t)a.H, hx = id - n * (uint32_t)a.H;
    // consecutive workgroups (on consecutive XCDs) take different key heads: an XCD's L2 then
    // serves few of them
    const int hk = hx % (uint32_t)a.Hkv, h = hk * group + hx / (uint32_t)a.Hkv;
    Packed pk;
    int64_t blk;
    if (!find_block<QB>(a, n, pk, blk)) return;
    blk = __builtin_amdgcn_readfirstlane((int)blk);
    const bool causal = a.causal != 0;
    const int kg = wave % SPLIT, k32 = 64 / SPLIT * kg;  // this wave's keys of a tile begin at k32
    const int64_t qb = blk * QB, qw = qb + 32 * (wave / SPLIT);  // first query of the workgroup, of the wave
    const int hd = (int)a.hd;

    // B operand of S^T = K Q^T: query qw + col, dims 16 s + 8 hh ..
    u4v qf[KS];
    {
        const int64_t qi = min(qw + col, pk.nq - 1);
        const uint16_t* qr = static_cast<const uint16_t*>(a.q) + (pk.q0 + qi) * a.ldq + (int64_t)h * hd;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * hh;
            qf[s] = d < hd ? *reinterpret_cast<const u4v*>(qr + d) : u4v{0, 0, 0, 0};
        }
    }
    // keys seen by this lane's query, by the wave's first and last one, and by the workgroup
    const int lim = (int)keys_seen(pk, qw + col, causal);
    const int seen_first = (int)keys_seen(pk, qw, causal);
    const int seen_wave = qw < pk.nq ? (int)keys_seen(pk, qw + 31, causal) : 0;
    const int seen_all = (int)keys_seen(pk, min(qb + QB, pk.nq) - 1, causal);
    const int tiles = (seen_all + PT_K - 1) / PT_K;

    // copies: lane of copy j of its wave fills LDS slot (j * waves + wave) * 64 + lane; slot x of row
    // r holds chunk x ^ swizzle(r), so that the reads below spread over the banks
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds);
    uint32_t koff[COPIES], voff[COPIES];
    const uint32_t ldk = (uint32_t)a.ldk * 2, ldv = (uint32_t)a.ldv * 2;
    // (64 banks: 16 rows' 16-byte chunks at a time for K, 4 rows' 64 bytes for V; no conflicts at 64, 128 and 256)
    auto k_swz = [](int r) { return CPR == 8 ? (r >> 1) & 7 : CPR % 16 == 0 ? r & 15 : r & 7; };
    auto v_swz = [](int r) { return CPR == 8 ? 4 * ((r >> 1) & 1) : CPR % 16 == 0 ? 4 * (r & 3) : 4 * (r & 1); };
#pragma unroll
    for (int j = 0; j < COPIES; ++j) {
        const int slot = (j * PT_WAVES + wave) * 64 + lane, r = slot / CPR, x = slot % CPR;
        const int ck = x ^ k_swz(r), cv = x ^ v_swz(r);
        koff[j] = 8 * ck < hd ? r * ldk + ck * 16 : 0x80000000u;  // past the head dim: out of range, read as 0
        voff[j] = 8 * cv < hd ? r * ldv + cv * 16 : 0x80000000u;
    }
    const char* kbase = static_cast<const char*>(a.k) + (pk.k0 * a.ldk + (int64_t)hk * hd) * 2;
    const char* vbase = static_cast<const char*>(a.v) + (pk.k0 * a.ldv + (int64_t)hk * hd) * 2;
    auto issue = [&](int t, const char* src, uint32_t ld, const uint32_t (&off)[COPIES], uint32_t at)
                     __attribute__((always_inline)) {
        if (t >= tiles) return;
        const int rows = (int)min((int64_t)PT_K, pk.nk - (int64_t)t * PT_K);  // at least 1
        const v4i r = buffer_rsrc(src + (int64_t)t * PT_K * ld, (uint32_t)((rows - 1) * ld + 2 * hd));
        const uint32_t to = lds0 + (t & 1) * 2 * TILE + at + wave * 1024;
#pragma unroll
        for (int j = 0; j < COPIES; ++j) lds_dma16_fresh(r, off[j], to + j * PT_WAVES * 1024);
    };
    auto issue_k = [&](int t) __attribute__((always_inline)) { issue(t, kbase, ldk, koff, 0); };
    auto issue_v = [&](int t) __attribute__((always_inline)) { issue(t, vbase, ldv, voff, TILE); };

    f16v o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const float sl2 = a.scale * LOG2E;
    // reads of K: row col of a 32-key block, chunk 2 s + hh; of V: rows 4 hh + (i >> 2) (+ 8), see lds_read_tr
    const uint32_t krow = lds0 + (k32 + col) * HDP * 2;
    const int vi = lane & 15, vr = 4 * hh + (vi >> 2), vc = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);
    const uint32_t vrow = lds0 + TILE + (k32 + vr) * HDP * 2 + 8 * (vi & 1);

    const int open = qw < pk.nq ? min(seen_first / PT_K, tiles) : 0;  // tiles whose keys every query of the wave sees
    const int mine = (seen_wave + PT_K - 1) / PT_K;                   // tiles with a key that some query of it sees
    auto scores = [&](int t, f16v (&sc)[KT]) __attribute__((always_inline)) {
        const uint32_t at = krow + (t & 1) * 2 * TILE;
#pragma unroll
        for (int b = 0; b < KT; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[b][i] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int b = 0; b < KT; ++b)
                sc[b] = mfma_32x32x16(E{}, lds_read16(at + b * 32 * HDP * 2 + (((2 * s + hh) ^ k_swz(col)) << 4)),
                                      qf[s], sc[b]);
    };
    auto mask = [&](int t, f16v (&sc)[KT]) __attribute__((always_inline)) {
        const int left = lim - t * PT_K - k32 - 4 * hh;
#pragma unroll
        for (int b = 0; b < KT; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (32 * b + 8 * (i >> 2) + (i & 3) >= left) sc[b][i] = -INFINITY;
    };
    // the running maximum over a tile's scores; the accumulators follow it only when it has risen by
    // more than 2^RESCALE_AT
    auto maximum = [&](const f16v (&sc)[KT]) __attribute__((always_inline)) {
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < KT; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[b][i]);
        mx = half_max(mx) * sl2;
        if (__any(mx > m + RESCALE_AT)) {
            const float mn = fmaxf(m, weight_reference<E>(mx));
            const float corr = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= corr;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= corr;
        }
    };
    // Tile t, whose scores are `sc`: the scores of tile t + 1 go to the matrix cores while the vector unit makes
    // this tile's weights, then the weights meet V.  MASKED where some query of the wave does not see
    // some key of tile t or t + 1.
    auto step = [&](int t, f16v (&sc)[KT], f16v (&next)[KT], auto masked) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        wait_vmcnt<0>();
        block_barrier();  // K of t + 1 and V of t have landed; every wave is done with K of t and V of t - 1
        issue_k(t + 2);
        issue_v(t + 1);
        if (MASKED && t >= mine) return;
        const bool more = !MASKED || t + 1 < mine;
        if (more) scores(t + 1, next);
        const float base = m == -INFINITY ? 0.0f : m - WEIGHT_SHIFT<E>;
        u4v p[TERMS][2 * KT];
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < KT; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][i], sl2, -base));
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][i + 1], sl2, -base));
                l += x;
                sum += y;
                float u = x, v = y;  // what the terms so far leave
#pragma unroll
                for (int n = 0; n < TERMS; ++n) {
                    const uint32_t w = pack2(E{}, u, v);
                    p[n][2 * b + (i >> 3)][(i & 7) >> 1] = w;
                    if (n + 1 < TERMS) {
                        const f2v r = unpack2(E{}, w);
                        u -= r[0];
                        v -= r[1];
                    }
                }
            }
        l += sum;
        const uint32_t vt = vrow + (t & 1) * 2 * TILE;
        auto value = [&](int d, int ks) __attribute__((always_inline)) {
            const uint32_t at = vt + ks * 16 * HDP * 2 + (((4 * d + vc) ^ v_swz(vr)) << 4);
            const u2v lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * HDP * 2);
            return u4v{lo[0], lo[1], hi[0], hi[1]};
        };
#pragma unroll
        for (int ks = 0; ks < 2 * KT; ++ks)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const u4v v = value(d, ks);
#pragma unroll
                for (int n = 0; n < TERMS; ++n) o[d] = mfma_32x32x16(E{}, v, p[n][ks], o[d]);
            }
        if (more) {
            if (MASKED && t + 1 >= open) mask(t + 1, next);
            maximum(next);
        }
    };
    f16v sa[KT], sb[KT];
    if (tiles > 0) {
        issue_k(0);
        wait_vmcnt<0>();
        block_barrier();
        issue_k(1);
        issue_v(0);
        if (mine > 0) {
            scores(0, sa);
            if (open == 0) mask(0, sa);
            maximum(sa);
        }
    }
    int t = 0;
    for (; t + 2 < open; t += 2) {
        step(t, sa, sb, std::false_type{});
        step(t + 1, sb, sa, std::false_type{});
    }
    for (; t < tiles; ++t) {
        step(t, sa, sb, std::true_type{});
#pragma unroll
        for (int b = 0; b < KT; ++b) sa[b] = sb[b];
    }
    // An infinity or NaN among the values has met weights it must not meet: the 0 of a key that is not seen, the
    // second or third term of a weight.  It left a sum that is not finite; such queries are computed again.
    bool odd = false;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) odd |= !(fabsf(o[d][i]) < INFINITY);
    bool again = __any(odd);
    l = half_sum(l);
    if constexpr (SPLIT > 1) {  // the waves of a query meet in the first of them
        constexpr int WORDS = (16 * DT + 2) * 64;
        static_assert(PT_WAVES / SPLIT * (SPLIT - 1) * WORDS * 4 <= 4 * TILE, "the sums fit the tiles' LDS");
        float* sums = reinterpret_cast<float*>(lds) + wave / SPLIT * (SPLIT - 1) * WORDS + lane;
        block_barrier();  // every wave is done with the tiles
        if (kg > 0) {
            float* mine = sums + (kg - 1) * WORDS;
            mine[0] = m;
            mine[64] = l;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) mine[64 * (2 + 16 * d + i)] = o[d][i];
        }
        if (lane == 0) odd_values[wave] = again;
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int w = 1; w < SPLIT; ++w) {
            const float* other = sums + (w - 1) * WORDS;
            again |= odd_values[wave + w] != 0;
            const float mn = fmaxf(m, other[0]), base = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(other[0] - base);
            m = mn;
            l = __builtin_fmaf(l, f, g * other[64]);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] = __builtin_fmaf(o[d][i], f, g * other[64 * (2 + 16 * d + i)]);
        }
    }
    if (again) {  // the wave's queries once more, one by one
        for (int64_t i = qw; i < min(qw + 32, pk.nq); ++i)
            attend_row<E, Out>(a, pk.q0 + i, h, hk, pk.k0, keys_seen(pk, i, causal));
        return;
    }
    const float r = seen_all > 0 && lim > 0 ? 1.0f / l : 0.0f;
    const int64_t qi = qw + col;
    if (qi < pk.nq) {
        typename Out::T* orow = static_cast<typename Out::T*>(a.out) + ((pk.q0 + qi) * a.H + h) * hd;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int dim = 32 * d + 2 * i + 4 * hh;
                if (dim < hd) {
                    if constexpr (Out::code == LQ_F32) {
                        *reinterpret_cast<vf4*>(orow + dim) = vf4{o[d][i] * r, o[d][i + 1] * r, o[d][i + 2] * r,
                                                                  o[d][i + 3] * r};
                    } else {
                        *reinterpret_cast<u2v*>(orow + dim) = u2v{pack2(E{}, o[d][i] * r, o[d][i + 1] * r),
                                                                  pack2(E{}, o[d][i + 2] * r, o[d][i + 3] * r)};
                    }
                }
            }
    }
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

int lq_prompt_attention(const void* d_q, int64_t ldq, const void* d_k, int64_t ldk, const void* d_v, int64_t ldv,
                        int type, const int32_t* d_q_starts, const int32_t* d_k_starts, int64_t seqs, int64_t total_q,
                        int64_t total_k, int64_t H, int64_t Hkv, int64_t hd, int causal, float scale, void* d_out,
                        int out_type, void* stream) {
    LQ_REQUIRE(is_half_type(type), "lq_prompt_attention: q, k and v must be fp16 or bfloat16");
    LQ_REQUIRE(out_type == type || out_type == LQ_F32, "lq_prompt_attention: out must be of q's type or float32");
    LQ_REQUIRE(seqs >= 0 && total_q >= 0 && total_k >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && hd > 0 &&
                   ldq >= H * hd && ldk >= Hkv * hd && ldv >= Hkv * hd && H <= 65535 && seqs < 0x7fffffff &&
                   total_q <= 0x7fffffff && total_k <= 0x7fffffff,
               "lq_prompt_attention: bad shape");
    if (hd % 8 != 0 || hd > ATTN_MAX_HD)
        return set_error(LQ_ERR_UNSUPPORTED, "lq_prompt_attention: head dim must be a multiple of 8, 256 at most");
    LQ_REQUIRE(scale > 0.0f && scale < INFINITY, "lq_prompt_attention: scale must be positive and finite");
    if (seqs == 0 || total_q == 0) return LQ_OK;
    LQ_REQUIRE(d_q && d_q_starts && d_k_starts && d_out && ((d_k && d_v) || total_k == 0),
               "lq_prompt_attention: NULL pointer");
    const PromptArgs a{d_q, d_k, d_v, ldq, ldk, ldv, d_q_starts, d_k_starts, seqs, total_q, total_k, H, Hkv, hd,
                       causal, scale, d_out};
    const hipStream_t st = as_stream(stream);
    // 16-byte copies and loads: bases and rows aligned to them, offsets of a tile's rows within 31 bits
    const bool vec = aligned16(d_q) && aligned16(d_k) && aligned16(d_v) && aligned16(d_out) && ldq % 8 == 0 &&
                     ldk % 8 == 0 && ldv % 8 == 0 && ldk < (1 << 23) && ldv < (1 << 23);
    auto blocks = [&](int64_t qb) { return (total_q + (qb - 1) * (seqs < total_q ? seqs : total_q)) / qb * H; };
    if (vec && blocks(64) <= 0x7fffffff) {
        // Enough workgroups to fill the chip twice over: 128 queries each.  Fewer: 64 queries each with the keys
        // split over two waves, which shortens the longest chain of tiles (one sequence of 3845 with 8 heads of
        // 128: 87 us with 128 queries, 66 with 64; 34 of up to 3483 with 2 heads: 81 and 64; at twice as
        // many workgroups no difference).
        const bool many = blocks(128) >= 2 * 512;
        const dim3 tiles = grid_of(blocks(many ? 128 : 64)), wg(64 * PT_WAVES);
        with_half(type, [&](auto e) {
            using E = decltype(e);
            auto go = [&](auto w, auto o) {
                constexpr int W = decltype(w)::value;
                using O = decltype(o);
                if (many) hipLaunchKernelGGL((prompt_tile_kernel<W, 1, E, O>), tiles, wg, 0, st, a);
                else hipLaunchKernelGGL((prompt_tile_kernel<W, 2, E, O>), tiles, wg, 0, st, a);
            };
            auto width = [&](auto o) {
                if (hd <= 64) go(std::integral_constant<int, 64>{}, o);
                else if (hd <= 128) go(std::integral_constant<int, 128>{}, o);
                else if (hd <= 192) go(std::integral_constant<int, 192>{}, o);
                else go(std::integral_constant<int, 256>{}, o);
            };
            if (out_type == LQ_F32) width(ElemF32{});
            else width(E{});
        });
        note_path(many ? "prompt tile 128" : "prompt tile 64");
        return launch_status("lq_prompt_attention");
    }
    note_path("prompt rows");
    const dim3 grid((unsigned)H, (unsigned)(total_q < 65535 ? total_q : 65535), (unsigned)((total_q + 65534) / 65535));
    with_half(type, [&](auto e) {
        using E = decltype(e);
        if (out_type == LQ_F32)
            hipLaunchKernelGGL((prompt_rows_kernel<E, ElemF32>), grid, dim3(64), 0, st, a);
        else
            hipLaunchKernelGGL((prompt_rows_kernel<E, E>), grid, dim3(64), 0, st, a);
    });
    return launch_status("lq_prompt_attention");
}

}  // extern "C"
