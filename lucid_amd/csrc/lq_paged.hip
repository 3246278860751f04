// lq_paged.hip -- a key-value cache in pages: appending new tokens' keys and values, and the
// attention of one new token per sequence over its pages.
//
// Layout.  k / v pages [pages][Hkv][page][hd] (fp16, bfloat16, int8 codes with one float32
// scale per row in [pages][Hkv][page], or 4-bit codes with bfloat16 scales and biases: lq_u4.h); table [seqs][table_stride] of page numbers; position p
// of sequence s is slot p % page of page table[s][p / page].  A head's rows of one page lie next
// to each other, so the attention of a head streams page * hd contiguous values.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_dma.h"
#include "lq_paged_u4.h"
#include "lq_u4.h"

namespace lq {
namespace {

// ------------------------------------------------------------------------------ append

// One thread per value, for rows that 16-byte accesses do not fit.
template <class Src, class Dst>
__global__ __launch_bounds__(256) void append_any_kernel(AppendArgs a) {
    const int64_t per = a.Hkv * a.hd;
    const int64_t t = workgroup();
    if (t >= a.tokens) return;
    const int64_t row = token_row(a, t);
    if (row < 0) return;
    for (int64_t e = threadIdx.x; e < 2 * per; e += blockDim.x) {
        const bool is_v = e >= per;
        const int64_t w = is_v ? e - per : e;
        const int64_t h = w / a.hd, d = w - h * a.hd;
        const float x = Src::load(static_cast<const typename Src::T*>(is_v ? a.v : a.k)[t * a.ld + w]);
        static_cast<typename Dst::T*>(is_v ? a.vp : a.kp)[(row + h * a.page) * a.hd + d] = Dst::store(x);
    }
}

// TOK tokens per workgroup.  A thread keeps one place of the rows (k or v, head, eight dims) and
// moves it for every token, the loads of all of them in flight together.  Bound by HBM: 20452 tokens of
// 8 heads of 128 in bfloat16 33 us, 5.0 TB/s read and written (one thread per value 87 us); up to 4096
// tokens one a workgroup, so that there are workgroups enough.
template <int TOK, class Src, class Dst>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    __shared__ int64_t rows[TOK];
    const int64_t t0 = workgroup() * TOK;
    if (threadIdx.x < TOK) rows[threadIdx.x] = t0 + threadIdx.x < a.tokens ? token_row(a, t0 + threadIdx.x) : -1;
    __syncthreads();
    const uint32_t hd8 = (uint32_t)a.hd >> 3, per = (uint32_t)a.Hkv * hd8;
    for (uint32_t e = threadIdx.x; e < 2 * per; e += 256) {
        const bool is_v = e >= per;
        const uint32_t w = is_v ? e - per : e, h = w / hd8, d = (w - h * hd8) * 8;
        const typename Src::T* src = static_cast<const typename Src::T*>(is_v ? a.v : a.k) + t0 * a.ld + (int64_t)w * 8;
        typename Dst::T* dst = static_cast<typename Dst::T*>(is_v ? a.vp : a.kp) + (int64_t)h * a.page * a.hd + d;
        float x[TOK][8];
#pragma unroll
        for (int i = 0; i < TOK; ++i)
            if (rows[i] >= 0) load8<Src>(src + i * a.ld, x[i]);
#pragma unroll
        for (int i = 0; i < TOK; ++i)
            if (rows[i] >= 0) {
                u4v o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = pack2(Dst{}, x[i][2 * j], x[i][2 * j + 1]);
                *reinterpret_cast<u4v*>(dst + rows[i] * a.hd) = o;
            }
    }
}

// One wave per (token, head, k or v), element by element.
template <class Src>
__global__ __launch_bounds__(64) void append_i8_any_kernel(AppendArgs a) {
    const int64_t n = workgroup(), t = n / (2 * a.Hkv);
    if (t >= a.tokens) return;
    const int64_t row = token_row(a, t);
    if (row < 0) return;
    const int64_t h = (n - t * 2 * a.Hkv) >> 1;
    const bool is_v = n & 1;
    const typename Src::T* src = static_cast<const typename Src::T*>(is_v ? a.v : a.k) + t * a.ld + h * a.hd;
    const int64_t r = row + h * a.page;
    int32_t top = 0;
    for (int64_t d = threadIdx.x; d < a.hd; d += 64) top = max(top, magnitude(Src::load(src[d])));
    const RowScale rs(wave_max(top));
    int8_t* dst = static_cast<int8_t*>(is_v ? a.vp : a.kp) + r * a.hd;
    for (int64_t d = threadIdx.x; d < a.hd; d += 64) dst[d] = (int8_t)rs.code(Src::load(src[d]));
    if (threadIdx.x == 0) static_cast<float*>(is_v ? a.vs : a.ks)[r] = rs.scale;
}

// LPR lanes per row of hd <= 8 LPR values, eight values a lane; one workgroup per token.
template <int LPR, class Src>
__global__ __launch_bounds__(256) void append_i8_kernel(AppendArgs a) {
    const int64_t t = workgroup();
    if (t >= a.tokens) return;
    const int64_t row = token_row(a, t);
    if (row < 0) return;
    const uint32_t d = (threadIdx.x % LPR) * 8;
    // every lane of a wave takes the same number of rounds: the exchange below needs them all
    constexpr uint32_t PER = 64 / LPR;
    const uint32_t rounded = ((uint32_t)a.Hkv * 2 + PER - 1) / PER * PER;
    for (uint32_t e = threadIdx.x / LPR; e < rounded; e += 256 / LPR) {
        const bool is_v = e & 1, mine = e < (uint32_t)a.Hkv * 2 && d < (uint32_t)a.hd;
        const uint32_t h = e >> 1;
        float x[8] = {};
        const typename Src::T* src = static_cast<const typename Src::T*>(is_v ? a.v : a.k) + t * a.ld;
        if (mine) load8<Src>(src + (int64_t)h * a.hd + d, x);
        int32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude(x[j]));
#pragma unroll
        for (int off = LPR / 2; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
        const RowScale rs(top);
        if (!mine) continue;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= (uint32_t)(rs.code(x[j]) & 0xff) << (8 * (j & 3));
        const int64_t r = row + (int64_t)h * a.page;
        *reinterpret_cast<u2v*>(static_cast<int8_t*>(is_v ? a.vp : a.kp) + r * a.hd + d) = u2v{w[0], w[1]};
        if (d == 0) static_cast<float*>(is_v ? a.vs : a.ks)[r] = rs.scale;
    }
}

// ------------------------------------------------------------------------------ attention

// positions of a wave between two looks into the table
template <int WAVES>
constexpr int PG_IDS = WAVES > 4 ? 128 : 512;

// fp16 / bfloat16 cache.  K and V tiles are copied to the wave's LDS 16 bytes a lane, NST tiles deep: the
// copies of a row are one contiguous access, they need no registers, and a wave waits only for
// its oldest tile.  The byte offsets of PG_IDS positions at a time are looked up before their copies.
// Bound by HBM: 64 sequences of 256 to 8191 positions, 8 heads of 128, 110 us with the join (5.4 TB/s); of
// 8192 each 336 us (6.4 TB/s).  Rows loaded to registers, 64 bytes of each at a time: 130 us, the
// first.
template <int HDP, int WAVES, int NST, bool EXACT, class Q>
__global__ __launch_bounds__(64 * WAVES) void paged_copy_kernel(PagedArgs a) {
    constexpr int CPR = HDP / 8, COPIES = PG_K * CPR / 64, KS = HDP / 32, DT = HDP / 16;
    constexpr int ROW = HDP * 2, TILE = PG_K * ROW, SLOT = 2 * NST * TILE;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[WAVES * SLOT];
    __shared__ int64_t offsets[WAVES][PG_IDS<WAVES>];
    __shared__ float ml[WAVES][2][16];
    __shared__ int64_t scan[WAVES + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    const int hd = EXACT ? HDP : a.hd;
    Line<WAVES> line;
    line.init(a, scan);
    const uint32_t slot = (uint32_t)reinterpret_cast<uintptr_t>(lds) + wave * SLOT;
    // copy i of a tile: LDS chunk 64 i + lane, row (64 i + lane) / CPR
    int kch[COPIES], vch[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
        const int r = (64 * i + lane) / CPR, x = (64 * i + lane) % CPR;
        kch[i] = (x ^ k_swz<HDP>(r)) * 16;
        vch[i] = (x ^ v_swz<HDP>(r)) * 16;
    }
    const char* kp = static_cast<const char*>(a.k);
    const char* vp = static_cast<const char*>(a.v);
    // every copy instruction covers a whole row at least, so that some lane of it is on whatever the head
    // dim: the waits below count instructions
    auto issue = [&](int t) __attribute__((always_inline)) {
        const uint32_t to = slot + (t % NST) * 2 * TILE;
        int64_t off[COPIES];
#pragma unroll
        for (int i = 0; i < COPIES; ++i) off[i] = offsets[wave][t * PG_K + (64 * i + lane) / CPR];
#pragma unroll
        for (int i = 0; i < COPIES; ++i)
            if (EXACT || kch[i] < 2 * hd) lds_copy16(kp + off[i] + kch[i], to + i * 1024);
#pragma unroll
        for (int i = 0; i < COPIES; ++i)
            if (EXACT || vch[i] < 2 * hd) lds_copy16(vp + off[i] + vch[i], to + TILE + i * 1024);
    };
    const float sl2 = a.scale * LOG2E;
    for (Piece w; line.next(a, w);) {
        if (!EXACT) {  // chunks past the head dim are never copied and stay zeros
            for (int i = lane; i < SLOT / 16; i += 64) reinterpret_cast<u4v*>(lds + wave * SLOT)[i] = u4v{0, 0, 0, 0};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        u4v qf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = paged_query(a, w, l16, 32 * s + 8 * g, hd);
        const int32_t* table = a.table + (int64_t)w.b * a.table_stride;
        Sums<DT, Q> sums;
        bool bad = w.over || a.pages == 0;
        constexpr int STEP = WAVES * PG_K;
        for (int sub = w.begin; sub < w.end && a.pages > 0; sub += WAVES * PG_IDS<WAVES>) {
            const int stop = min(sub + WAVES * PG_IDS<WAVES>, w.end);
            const int first = sub + wave * PG_K;
            const int tiles = first < stop ? (stop - first + STEP - 1) / STEP : 0;
            for (int e = lane; e < tiles * PG_K; e += 64) {
                const int key = first + (e / PG_K) * STEP + (e % PG_K);
                int64_t off = 0;  // row 0 stands in past the end and for a bad page: its score and values are dropped
                if (key < stop) {
                    const uint32_t col = (uint32_t)key / (uint32_t)a.page;
                    const int id = table[col];  // the length lies within the table
                    if (id >= 0 && id < a.pages)
                        off = (((int64_t)id * a.Hkv + w.hk) * a.page + (key - (int)(col * (uint32_t)a.page))) * (2 * hd);
                    else
                        bad = true;
                }
                offsets[wave][e] = off;
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int t = 0; t < NST; ++t)
                if (t < tiles) issue(t);
            for (int t = 0; t < tiles; ++t) {
                const int later = min(NST - 1, tiles - 1 - t);  // tiles that may still be on their way
                static_assert(NST <= 4 && 2 * (NST - 1) * COPIES < 64, "the counter's range");
                if (later == 0) wait_vmcnt<0>();
                else if (later == 1) wait_vmcnt<2 * COPIES>();
                else if (later == 2) wait_vmcnt<(NST > 2 ? 4 : 0) * COPIES>();
                else wait_vmcnt<(NST > 3 ? 6 : 0) * COPIES>();
                asm volatile("" ::: "memory");
                const uint32_t kt = slot + (t % NST) * 2 * TILE, vt = kt + TILE;
                const int left = stop - (first + t * STEP);  // positions of this tile that exist
                vf4 sc[2];
#pragma unroll
                for (int T = 0; T < 2; ++T) {
                    sc[T] = vf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < KS; ++s)
                        sc[T] = mfma_16x16x32(Q{}, lds_read16(kt + (16 * T + l16) * ROW +
                                                              (((4 * s + g) ^ k_swz<HDP>(l16)) << 4)),
                                              qf[s], sc[T]);
                }
                const bool whole = left >= PG_K;
                sums.weights(sc, sl2, whole, left - 4 * g);
                if (!whole) {  // values past the end as zeros: their weight 0 must meet no infinity or NaN
                    const int r = lane & 31;
                    if (r >= left)
                        for (int c = lane >> 5; c < CPR; c += 2)
                            *reinterpret_cast<lds_u4v*>(vt + r * ROW + c * 16) = u4v{0, 0, 0, 0};
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                }
                sums.template accumulate<ROW>(sc, vt, v_swz<HDP>, a.out_f32 != 0);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile is read: its LDS may be filled again
                if (t + NST < tiles) issue(t + NST);
            }
        }
        paged_finish<true, WAVES, SLOT, DT, Q>(a, w, lds, ml, sums, bad);
    }
    paged_empty<WAVES, Q>(a);
}

// int8 cache.  Codes are exact in 16 bits: they are loaded to registers (a tile ahead), widened there,
// and V goes to the wave's LDS as bfloat16.  The key's scale multiplies the score, the value's scale
// the weight, which is bfloat16 for its range.  131071 positions and a second sequence, 8 heads of 128: 79
// us with the join (4.9 TB/s).  No unit is full there: the vector unit is busy 44% of the time (one and a
// half instructions a code; with the compiler's own conversions 125 us) and the matrix cores 9%, while the
// waves, two to a SIMD with a tile ahead each, wait for loads half of theirs.
template <int HDP, bool EXACT, class Q>
__global__ __launch_bounds__(64 * PG_I8_WAVES, HDP <= 64 ? 3 : HDP <= 128 ? 2 : 1) void paged_i8_kernel(PagedArgs a) {
    using P = ElemBF16;
    constexpr int WAVES = PG_I8_WAVES, KS = HDP / 32, HALF = HDP / 64, DT = HDP / 16;
    constexpr int ROW = HDP * 2, TILE = PG_K * ROW, OTILE = 16 * (HDP + 4) * 4;
    constexpr int SLOT = (TILE > OTILE ? TILE : OTILE) + 256;  // + 64 scales
    __shared__ __attribute__((aligned(16))) uint8_t lds[WAVES * SLOT];
    __shared__ float ml[WAVES][2][16];
    __shared__ int64_t scan[WAVES + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    const int hd = EXACT ? HDP : a.hd;
    Line<WAVES> line;
    line.init(a, scan);
    const float sl2 = a.scale * LOG2E;
    uint8_t* slot = lds + wave * SLOT;
    float* scales = reinterpret_cast<float*>(slot + SLOT - 256);
    const uint32_t slot_at = (uint32_t)reinterpret_cast<uintptr_t>(slot);
    for (Piece w; line.next(a, w);) {
        // dims of this lane's eight slots in step s of the first product: a load brings 16 codes
        auto dims = [&](int s) { return 64 * (s >> 1) + 16 * g + 8 * (s & 1); };
        u4v qf[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = paged_query(a, w, l16, dims(s), hd);
        const int32_t* table = a.table + (int64_t)w.b * a.table_stride;
        // page number of a position, -1 past the end
        auto page_of = [&](int key) -> int { return key < w.end ? table[(uint32_t)key / (uint32_t)a.page] : -1; };
        bool bad = w.over || a.pages == 0;
        // a tile in registers: rows l16 and 16 + l16 of K and V, and their scales
        u4v kr[2][HALF], vr[2][HALF];
        float ksc[2], vsc[2];
        auto fetch = [&](int key0, const int (&id)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                const int key = key0 + 16 * T + l16;
                const bool ok = id[T] >= 0 && id[T] < a.pages;
                bad |= key < w.end && !ok;
                // row 0 stands in: its scores and values are dropped
                const int64_t row = ok ? ((int64_t)id[T] * a.Hkv + w.hk) * a.page + (uint32_t)key % (uint32_t)a.page : 0;
                const int8_t* kp = static_cast<const int8_t*>(a.k) + row * hd;
                const int8_t* vp = static_cast<const int8_t*>(a.v) + row * hd;
                ksc[T] = static_cast<const float*>(a.ks)[row];
                vsc[T] = static_cast<const float*>(a.vs)[row];
                auto load = [&](const int8_t* p, int d) {
                    if constexpr (EXACT) return *reinterpret_cast<const u4v*>(p + d);
                    const u2v lo = *reinterpret_cast<const u2v*>(p + (d < hd ? d : 0));
                    const u2v hi = *reinterpret_cast<const u2v*>(p + (d + 8 < hd ? d + 8 : 0));
                    return u4v{lo[0], lo[1], hi[0], hi[1]};
                };
#pragma unroll
                for (int s = 0; s < HALF; ++s) {
                    kr[T][s] = load(kp, 64 * s + 16 * g);
                    vr[T][s] = load(vp, 64 * s + 16 * g);
                }
            }
        };
        Sums<DT, P> sums;
        constexpr int STEP = WAVES * PG_K;
        int key0 = w.begin + wave * PG_K;
        if (a.pages > 0 && key0 < w.end) {
            int id[2], next[2];
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                id[T] = page_of(key0 + 16 * T + l16);
                next[T] = page_of(key0 + STEP + 16 * T + l16);
            }
            fetch(key0, id);
            for (; key0 < w.end; key0 += STEP) {
                const int left = w.end - key0;
                const bool whole = left >= PG_K;
                vf4 sc[2];
#pragma unroll
                for (int T = 0; T < 2; ++T) {
                    sc[T] = vf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        const uint32_t lo = kr[T][s >> 1][2 * (s & 1)], hi = kr[T][s >> 1][2 * (s & 1) + 1];
                        const u2v x = widen4(Q{}, lo), y = widen4(Q{}, hi);
                        // codes past hd meet zeros
                        sc[T] = mfma_16x16x32(Q{}, u4v{x[0], x[1], y[0], y[1]}, qf[s], sc[T]);
                    }
                }
#pragma unroll
                for (int T = 0; T < 2; ++T) {
                    const int r = 16 * T + l16;
#pragma unroll
                    for (int s = 0; s < KS; ++s) {
                        const uint32_t lo = vr[T][s >> 1][2 * (s & 1)], hi = vr[T][s >> 1][2 * (s & 1) + 1];
                        const u2v x = widen4(P{}, lo), y = widen4(P{}, hi);
                        *reinterpret_cast<u4v*>(slot + r * ROW + (((dims(s) >> 3) ^ v_swz<HDP>(r)) << 4)) =
                            u4v{x[0], x[1], y[0], y[1]};
                    }
                    scales[r] = ksc[T];
                    scales[32 + r] = r < left ? vsc[T] : 0.0f;  // codes are finite: a weight of 0 drops them
                }
                // the next tile, and the page numbers of the one after it
                if (key0 + STEP < w.end) {
                    id[0] = next[0];
                    id[1] = next[1];
#pragma unroll
                    for (int T = 0; T < 2; ++T) next[T] = page_of(key0 + 2 * STEP + 16 * T + l16);
                    fetch(key0 + STEP, id);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's LDS writes, before any lane reads them
#pragma unroll
                for (int T = 0; T < 2; ++T) {
                    const vf4 f = *reinterpret_cast<const vf4*>(scales + 16 * T + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[T][i] *= f[i];
                }
                sums.weights(sc, sl2, whole, left - 4 * g);
#pragma unroll
                for (int T = 0; T < 2; ++T) {
                    const vf4 f = *reinterpret_cast<const vf4*>(scales + 32 + 16 * T + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[T][i] *= f[i];
                }
                sums.template accumulate<ROW>(sc, slot_at, v_swz<HDP>, a.out_f32 != 0);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads, before the next tile's writes
            }
        }
        paged_finish<false, WAVES, SLOT, DT, Q>(a, w, lds, ml, sums, bad);
    }
    paged_empty<WAVES, Q>(a);
}

// The pieces of one (sequence, query head) joined by one workgroup: hd / 4 lanes take four dims each
// of every (256 / (hd / 4))-th piece, and these sums meet in LDS.
template <class Q>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
    __shared__ float f[256], red[4];
    __shared__ vf4 sums[256];
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.x, b = blockIdx.y;
    const int heads = a.Hkv * a.qtiles, hk = h / a.group, hq = hk * a.qtiles + (h - hk * a.group) / 16;
    const int2 info = a.pieces[(int64_t)b * heads + hq];
    const int used = info.y, row = (h - hk * a.group) % 16;
    if (used <= 1) return;  // written already
    // the first piece, then the first ones of the workgroups that follow
    auto piece = [&](int s) { return (int64_t)16 * (s == 0 ? info.x : (info.x & ~1) + 2 * s) + row; };
    const int64_t at = (int64_t)b * a.H + h;
    const f2v* ml = reinterpret_cast<const f2v*>(a.part_ml);  // maximum and sum of a piece's row
    const float* po = a.part_o;
    const int quads = a.hd / 4, teams = 256 / quads, team = tid / quads, d = (tid - team * quads) * 4;
    // a thread's first pieces and every piece's statistics are on their way before anything waits
    constexpr int AHEAD = 8;
    vf4 p[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const int s = team + i * teams;
        p[i] = vf4{0.f, 0.f, 0.f, 0.f};
        if (team < teams && s < used) p[i] = *reinterpret_cast<const vf4*>(po + piece(s) * a.hd + d);
    }
    f2v mine = tid < used ? ml[piece(tid)] : f2v{-INFINITY, 0.0f};
    float M = mine[0];
    for (int s = tid + 256; s < used; s += 256) M = fmaxf(M, ml[piece(s)][0]);
    M = unkey(wave_max(fkey(M)));
    if (lane == 0) red[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    vf4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < used; s0 += 256) {
        const int n = min(256, used - s0);
        __syncthreads();
        if (s0 > 0) mine = tid < n ? ml[piece(s0 + tid)] : f2v{-INFINITY, 0.0f};
        const float e = tid < n ? __builtin_amdgcn_exp2f(mine[0] - base) : 0.0f;
        f[tid] = e;
        const float w = ln_wave_sum(tid < n ? e * mine[1] : 0.0f);
        if (lane == 0) red[tid >> 6] = w;
        __syncthreads();
        L += (red[0] + red[1]) + (red[2] + red[3]);
        if (team >= teams) continue;
        int s = team;
        if (s0 == 0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i, s += teams)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (s < n) x[j] = __builtin_fmaf(f[s], p[i][j], x[j]);
        }
#pragma unroll 4
        for (; s < n; s += teams) {
            const vf4 q = *reinterpret_cast<const vf4*>(po + piece(s0 + s) * a.hd + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = __builtin_fmaf(f[s], q[j], x[j]);
        }
    }
    sums[tid] = x;
    __syncthreads();
    if (team == 0) {
        for (int t = 1; t < teams; ++t) x += sums[t * quads + tid];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y = x[i] / L;
            if (a.out_f32) static_cast<float*>(a.out)[at * a.hd + d + i] = y;
            else static_cast<typename Q::T*>(a.out)[at * a.hd + d + i] = Q::store(y);
        }
    }
}

// Workgroups of a call over long sequences: as many as run at a time (two to a CU, one past 128 dims; three of
// the int8 kernel up to 64: 69 sequences of up to 39768, 2 heads of 64, 59 -> 55 us).
// Up to PG_ALONE positions each workgroup takes a sequence whole: the plan and the second launch would cost
// more than they give.  Whole against shared, us a call, 16-bit rows of 64 / 128 dims, ragged lengths:
//   sequences x key heads      8                    256                   1024
//   longest 512     7.0-14.3 / 13.2-17.5   8.7-16.2 / 14.3-19.3   21.0-27.4 / 28.4-35.6
//   longest 1024   10.4-15.1 / 20.4-17.7  12.8-17.4 / 22.8-21.7   35.6-34.8 / 48.2-45.7
//   longest 2048   16.7-14.9 / 35.0-18.0  19.3-23.1 / 37.2-29.6   68.2-57.2 / 94.1-76.4
// (at 1024 rows of 128 dims lose up to 15% by it; int8 rows are alike.)
constexpr int PG_GROUPS = 512, PG_GROUPS_I8_64 = 768, PG_GROUPS_WIDE = 256, PG_ALONE = 1024;
// bytes of the table of pieces, and the slots of a call (two to a workgroup)
int64_t pieces_bytes(int64_t units) { return (units * (int64_t)sizeof(int2) + 15) / 16 * 16; }
int paged_groups(int64_t hd, bool i8) {
    return hd <= 64 && i8 ? PG_GROUPS_I8_64 : hd <= 128 ? PG_GROUPS : PG_GROUPS_WIDE;
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

int lq_paged_kv_append(const void* d_k, const void* d_v, int src_type, int64_t ld, int64_t tokens,
                       const int32_t* d_starts, int64_t seqs, int64_t Hkv, int64_t hd, const int32_t* d_table,
                       int64_t table_stride, const int32_t* d_lengths, void* d_k_pages, void* d_v_pages,
                       int cache_type, void* d_k_scale, void* d_v_scale, int64_t pages, int64_t page,
                       void* stream) {
    LQ_REQUIRE(is_float_type(src_type), "lq_paged_kv_append: source must be float32, fp16 or bfloat16");
    LQ_REQUIRE(is_half_type(cache_type) || cache_type == LQ_I8 || cache_type == LQ_U4,
               "lq_paged_kv_append: cache must be fp16, bfloat16, int8 or 4 bits");
    if (cache_type == LQ_U4)  // the append with rotation, of nothing
        return paged_append_rotary("lq_paged_kv_append", nullptr, 0, d_k, d_v, ld, src_type, tokens, d_starts, seqs, 0,
                                   Hkv, hd, nullptr, 0, 0, 0, d_table, table_stride, d_lengths, nullptr, 0, nullptr, 0,
                                   LQ_F16, d_k_pages, d_v_pages, cache_type, d_k_scale, d_v_scale, pages, page, stream);
    LQ_REQUIRE(tokens >= 0 && seqs >= 0 && Hkv > 0 && hd > 0 && Hkv <= 65535 && hd <= 65535 && ld >= Hkv * hd &&
                   table_stride >= 0 && pages >= 0 && page > 0 && tokens <= 0x7fffffff && seqs <= 0x7fffffff &&
                   table_stride <= 0x7fffffff && pages <= 0x7fffffff && page <= 0x7fffffff,
               "lq_paged_kv_append: bad shape");
    LQ_REQUIRE(d_starts || tokens == seqs, "lq_paged_kv_append: without starts there is one token per sequence");
    if (tokens == 0 || seqs == 0 || table_stride == 0 || pages == 0) return LQ_OK;
    LQ_REQUIRE(d_k && d_v && d_table && d_lengths && d_k_pages && d_v_pages, "lq_paged_kv_append: NULL pointer");
    LQ_REQUIRE(cache_type != LQ_I8 || (d_k_scale && d_v_scale), "lq_paged_kv_append: an int8 cache needs scales");
    const AppendArgs a{d_k, d_v, ld, tokens, d_starts, seqs, Hkv, hd, d_table, table_stride, d_lengths,
                       d_k_pages, d_v_pages, d_k_scale, d_v_scale, pages, page};
    const hipStream_t st = as_stream(stream);
    // eight values of a row at a time: heads of whole eights, bases and rows 16-byte aligned
    const uintptr_t ends = reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v) |
                           reinterpret_cast<uintptr_t>(d_k_pages) | reinterpret_cast<uintptr_t>(d_v_pages);
    const bool vec = hd % 8 == 0 && (ends & 15) == 0 && ld * elem_size(src_type) % 16 == 0 && Hkv * hd < (1 << 28);
    with_float(src_type, [&](auto s) {
        using S = decltype(s);
        const dim3 one = grid_of(tokens);
        if (cache_type == LQ_I8) {
            if (vec && hd <= 64) hipLaunchKernelGGL((append_i8_kernel<8, S>), one, dim3(256), 0, st, a);
            else if (vec && hd <= 128) hipLaunchKernelGGL((append_i8_kernel<16, S>), one, dim3(256), 0, st, a);
            else if (vec && hd <= 256) hipLaunchKernelGGL((append_i8_kernel<32, S>), one, dim3(256), 0, st, a);
            else
                hipLaunchKernelGGL((append_i8_any_kernel<S>), grid_of(tokens * 2 * Hkv), dim3(64), 0, st, a);
            return;
        }
        with_half(cache_type, [&](auto c) {
            using C = decltype(c);
            if (!vec) hipLaunchKernelGGL((append_any_kernel<S, C>), one, dim3(256), 0, st, a);
            else if (tokens <= 4 * 1024) hipLaunchKernelGGL((append_kernel<1, S, C>), one, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((append_kernel<4, S, C>), grid_of((tokens + 3) / 4), dim3(256), 0, st, a);
        });
    });
    return launch_status("lq_paged_kv_append");
}

size_t lq_paged_attention_workspace_size(int64_t B, int64_t H, int64_t Hkv, int64_t hd, int64_t max_length) {
    if (B <= 0 || H <= 0 || Hkv <= 0 || hd <= 0 || max_length <= PG_ALONE) return 0;
    return (size_t)pieces_bytes(B * Hkv * ((H / Hkv + 15) / 16)) +
           (size_t)2 * paged_groups(hd, true) * 16 * (hd + 2) * sizeof(float);  // of either kind of cache
}

int lq_paged_attention(const void* d_q, int q_type, int64_t ldq, int64_t B, int64_t H, int64_t Hkv, int64_t hd,
                       const void* d_k_pages, const void* d_v_pages, int cache_type, const void* d_k_scale,
                       const void* d_v_scale, int64_t pages, int64_t page, const int32_t* d_table,
                       int64_t table_stride, const int32_t* d_lengths, int64_t max_length, float scale, void* d_out,
                       int out_type, void* d_workspace, size_t workspace_bytes, void* stream) {
    LQ_REQUIRE(is_half_type(q_type), "lq_paged_attention: q must be fp16 or bfloat16");
    LQ_REQUIRE(cache_type == q_type || cache_type == LQ_I8 || cache_type == LQ_U4,
               "lq_paged_attention: the cache must be of q's type, int8 or 4 bits");
    LQ_REQUIRE(out_type == q_type || out_type == LQ_F32, "lq_paged_attention: out must be of q's type or float32");
    LQ_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && hd > 0 && ldq >= H * hd && pages >= 0 && page > 0 &&
                   table_stride >= 0 && max_length >= 0 && B <= 65535 && H <= 65535 && table_stride <= 0x7fffffff &&
                   pages <= 0x7fffffff && page <= 0x7fffffff && max_length <= 0x7fffffff,
               "lq_paged_attention: bad shape");
    if (hd % 8 != 0 || hd > ATTN_MAX_HD)
        return set_error(LQ_ERR_UNSUPPORTED, "lq_paged_attention: head dim must be a multiple of 8, 256 at most");
    if (cache_type == LQ_U4 && hd % U4_GROUP != 0)
        return set_error(LQ_ERR_UNSUPPORTED, "lq_paged_attention: head dims of a 4-bit cache are multiples of 32");
    LQ_REQUIRE(scale > 0.0f && scale < INFINITY, "lq_paged_attention: scale must be positive and finite");
    if (B == 0) return LQ_OK;
    LQ_REQUIRE(d_q && d_lengths && d_out && (d_table || table_stride == 0) && ((d_k_pages && d_v_pages) || pages == 0),
               "lq_paged_attention: NULL pointer");
    LQ_REQUIRE(cache_type == q_type || pages == 0 || (d_k_scale && d_v_scale),
               "lq_paged_attention: a cache of codes needs scales");
    LQ_REQUIRE(cache_type != LQ_U4 || (aligned16(d_k_scale) && aligned16(d_v_scale)),
               "lq_paged_attention: the scales of a 4-bit cache must be 16-byte aligned");
    LQ_REQUIRE(aligned16(d_k_pages) && aligned16(d_v_pages), "lq_paged_attention: pages must be 16-byte aligned");
    const bool alone = max_length <= PG_ALONE;
    LQ_REQUIRE(alone || (d_workspace && aligned16(d_workspace) &&
                         workspace_bytes >= lq_paged_attention_workspace_size(B, H, Hkv, hd, max_length)),
               "lq_paged_attention: workspace too small or not 16-byte aligned");
    const int group = (int)(H / Hkv), qtiles = (group + 15) / 16;
    const int groups = alone ? 0 : paged_groups(hd, cache_type == LQ_I8);
    const int64_t units = B * Hkv * qtiles;
    LQ_REQUIRE(units <= 0x7fffffff, "lq_paged_attention: too many workgroups");
    char* ws = static_cast<char*>(d_workspace);
    float* part_o = alone ? nullptr : reinterpret_cast<float*>(ws + pieces_bytes(units));
    const PagedArgs a{d_q, ldq, (int)B, (int)H, (int)Hkv, (int)hd, group, qtiles, d_k_pages, d_v_pages, d_k_scale,
                      d_v_scale, pages, (int)page, d_table, table_stride, d_lengths, scale, d_out, out_type == LQ_F32,
                      aligned16(d_q) && ldq % 8 == 0, groups, reinterpret_cast<int2*>(ws), part_o,
                      alone ? nullptr : part_o + (int64_t)2 * groups * 16 * hd};
    const dim3 grid = grid_of(alone ? units : groups);
    const hipStream_t st = as_stream(stream);
    // A few short sequences: as many waves each as the LDS holds tiles for, to hide more of the latency (8 sequences
    // of up to 640, 8 heads of 64: 9.4 us a call with four waves, 7.8 with eight); else two, two workgroups to a CU.
    const bool few = alone && units <= 256;
    note_path(!alone ? "paged shared" : few ? "paged whole few" : "paged whole");
    with_half(q_type, [&](auto q) {
        using Q = decltype(q);
        auto i8 = [&](auto w, auto exact) {
            hipLaunchKernelGGL((paged_i8_kernel<decltype(w)::value, decltype(exact)::value, Q>), grid,
                               dim3(64 * PG_I8_WAVES), 0, st, a);
        };
        auto copy = [&](auto w, auto waves, auto nst, auto exact) {
            hipLaunchKernelGGL((paged_copy_kernel<decltype(w)::value, decltype(waves)::value, decltype(nst)::value,
                                                  decltype(exact)::value, Q>),
                               grid, dim3(64 * decltype(waves)::value), 0, st, a);
        };
        const std::integral_constant<int, 2> two{};
        const std::integral_constant<int, 4> four{};
        const std::integral_constant<int, 8> eight{};
        const std::integral_constant<int, 64> w64{};
        const std::integral_constant<int, 128> w128{};
        const std::integral_constant<int, 192> w192{};
        const std::integral_constant<int, 256> w256{};
        if (cache_type == LQ_U4) {
            paged_u4_launch(a, q_type, few, grid, st);
        } else if (cache_type == LQ_I8) {
            if (hd == 64) i8(w64, std::true_type{});
            else if (hd == 128) i8(w128, std::true_type{});
            else if (hd < 64) i8(w64, std::false_type{});
            else if (hd < 128) i8(w128, std::false_type{});
            else if (hd <= 192) i8(w192, std::false_type{});
            else i8(w256, std::false_type{});
        } else if (hd <= 64) {
            if (few) hd == 64 ? copy(w64, eight, two, std::true_type{}) : copy(w64, eight, two, std::false_type{});
            else hd == 64 ? copy(w64, two, four, std::true_type{}) : copy(w64, two, four, std::false_type{});
        } else if (hd <= 128) {
            if (few) hd == 128 ? copy(w128, four, two, std::true_type{}) : copy(w128, four, two, std::false_type{});
            else hd == 128 ? copy(w128, two, two, std::true_type{}) : copy(w128, two, two, std::false_type{});
        } else if (hd <= 192) {
            copy(w192, two, two, std::false_type{});
        } else {
            copy(w256, two, two, std::false_type{});
        }
        if (alone) return;
        const dim3 rows((unsigned)H, (unsigned)B);
        hipLaunchKernelGGL((paged_join_kernel<Q>), rows, dim3(256), 0, st, a);
    });
    return launch_status("lq_paged_attention");
}

}  // extern "C"
