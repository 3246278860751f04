// lq_paged_u4.hip -- attention of one new token per sequence over pages that hold 4 bits a value.
//
// A key is K_d = ks_g c_d + kb_g for the 32 dims of a group g, a value V_d = vs c_d + vb for all its dims, so
//   q.K     = sum_g ks_g (q_g . c_g) + kb_g sum(q_g)
//   sum w V = sum w (vs c) + sum w vb:
// the products run on codes, exact in 16 bits, and the scales and biases enter beside them in float32.  A group is as deep as
// one matrix instruction (16x16x32), so its scale multiplies that instruction's result; a value's scale
// multiplies its weight, and its bias adds one number to all dims of a query.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_dma.h"
#include "lq_paged_u4.h"
#include "lq_u4.h"

namespace lq {
namespace {

constexpr int U4_TILE = 64;   // positions of a wave's tile
constexpr int U4_NST = 2;     // tiles on their way

// What the sums of a wave are relative to, all in whole powers of two, which round nothing:
// * weights to the running maximum of a query's scores, to the next whole number above it in log2 units (the exponents of
//   the weights that count stay near 0);
// * scales and biases to the largest of the wave's values, 2^large.  What leaves the wave is in their own units again, or in
//   2^U4_DOWN of them for a reference as much higher where they are as large as 2^U4_LARGE: the sums of a million values of
//   1e36, or of 4096 of bfloat16's largest, are finite then, as over the other caches, and the smallest keep their bits;
// * a weight times its value's scale, which enters a product in fp16, to the largest one that the query has met: as 2^lift
//   times it, between 2^U4_SET and 2^U4_LIMIT for the largest; what fp16 drops (half its least step) is 2^-35 of that.  The
//   largest product and not the largest scale decides: a row that attention ignores costs the others nothing.
constexpr int U4_LARGE = 80, U4_DOWN = 20, U4_SET = 10, U4_LIMIT = 15;

// The low half of byte I of a word, a signed number, over 16 in float32 (its bits).
template <int I>
__device__ __forceinline__ uint32_t nibble_to_f32(uint32_t w) {
    uint32_t f;
#define LQ_NIBBLE(i)                                                                                     \
    asm("v_cvt_off_f32_i4_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_" #i : "=v"(f) : "v"(w))
    if constexpr (I == 0) LQ_NIBBLE(0);
    if constexpr (I == 1) LQ_NIBBLE(1);
    if constexpr (I == 2) LQ_NIBBLE(2);
    if constexpr (I == 3) LQ_NIBBLE(3);
#undef LQ_NIBBLE
    return f;
}

// Eight values of type E for the codes c of a word, in four registers; pair p holds codes p and p + 4.  A code lies in
// the mantissa under the exponent that gives it its weight: 16 + c, one shift and one and-or for two codes.  CENTRE: in
// fp16 one addition more for c - 7.5; in bfloat16, which has none of pairs, (c - 8) / 16 by conversions of a signed nibble.
// An and-or takes no literal, so mask and exponent are kept in registers whose values the compiler does not see.
template <class E, bool CENTRE>
struct Widen8 {
    static constexpr float ADDED = !CENTRE ? 16.0f : E::code == LQ_F16 ? -7.5f : -8.0f;  // to a code
    static constexpr float TIMES = CENTRE && E::code == LQ_BF16 ? 0.0625f : 1.0f;        // and their sum
    uint32_t mask, exponent;
    __device__ __forceinline__ Widen8()
        : mask(E::code == LQ_F16 ? 0x03c003c0u : 0x00780078u), exponent(E::code == LQ_F16 ? 0x4c004c00u : 0x41804180u) {
        asm("" : "+s"(mask), "+v"(exponent));
    }
    __device__ __forceinline__ u4v operator()(uint32_t w) const {
        if constexpr (E::code == LQ_BF16 && CENTRE) {
            const uint32_t even = w ^ 0x88888888u, odd = even >> 4;  // two's complement of c - 8
            auto pair = [](uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); };
            return u4v{pair(nibble_to_f32<0>(even), nibble_to_f32<2>(even)), pair(nibble_to_f32<0>(odd), nibble_to_f32<2>(odd)),
                       pair(nibble_to_f32<1>(even), nibble_to_f32<3>(even)), pair(nibble_to_f32<1>(odd), nibble_to_f32<3>(odd))};
        }
        if constexpr (E::code == LQ_BF16)
            return u4v{((w << 3) & mask) | exponent, ((w >> 1) & mask) | exponent, ((w >> 5) & mask) | exponent,
                       ((w >> 9) & mask) | exponent};
        u4v v = {((w << 6) & mask) | exponent, ((w << 2) & mask) | exponent, ((w >> 2) & mask) | exponent,
                 ((w >> 6) & mask) | exponent};
        if constexpr (CENTRE) {
            typedef _Float16 h2v __attribute__((ext_vector_type(2)));
            const h2v down = {(_Float16)-23.5f, (_Float16)-23.5f};
#pragma unroll
            for (int p = 0; p < 4; ++p) v[p] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2v, (uint32_t)v[p]) + down);
        }
        return v;
    }
};

typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef __attribute__((address_space(3))) uint16_t lds_u16;
typedef __attribute__((address_space(3))) float lds_f32;
typedef __attribute__((address_space(3))) vf4 lds_vf4;
typedef __attribute__((address_space(3))) int64_t lds_i64;

// Transposing read of codes: of each 16 lanes, lane i points at the 16 codes of row i and receives column i of the
// 16 rows, row j in nibble j.
__device__ __forceinline__ v2i lds_read_tr4(uint32_t at) {
    return __builtin_amdgcn_ds_read_tr4_b64_v2i32(reinterpret_cast<lds_v2i*>(at));
}

// One lane's place in the page table: a column and a slot in its page, moved a whole step at a time.
struct Place {
    int col, slot;
    __device__ __forceinline__ void start(uint32_t key, uint32_t page) {
        col = (int)(key / page);
        slot = (int)(key - (uint32_t)col * page);
    }
    __device__ __forceinline__ void advance(int cols, int slots, int page) {
        col += cols;
        slot += slots;
        if (slot >= page) {
            slot -= page;
            ++col;
        }
    }
};

// G: groups of 32 dims.  The plan of the other caches (lq_paged.h) with tiles of 64 positions; within a tile lane
// (l, g) holds the scores and weights of query l at positions 16 g + 4 T + i: row r of the first product's
// operand T is position 16 (r / 4) + 4 T + r % 4, and the transposing read brings a lane the codes of its dim at just
// these 16 positions.
// Keys' codes meet queries in the queries' type.  Queries of bfloat16 enter times a power of two, which goes into the
// scores' factor and halves the exponent of their largest: products with keys of the inverse size stay in float32's
// range, and no dim above 2^-126 of the largest loses a bit.  Values' codes meet weights in fp16.  A weight enters times its
// value's scale, relative to the largest such product so far (U4_SET), as two terms (within 2^-23 of it); sums and
// maximum stay float32.
// A code c enters as 16 + c.  What that adds to a score is taken off where the biases come in: one instruction more
// multiplies the row's scales and biases, bfloat16 as they are stored, by minus the queries' sums times 16 and by their
// sums, in three bfloat16 terms each (24 bits).  An output gets 16 + c less 23.5, by a row of that, and 7.5 scales more
// from the biases: the rounding of a weight then meets codes around 0, not around 7.5.
// A float32 output is worth codes around 0 in both products (Widen8), so that no sum grows by what is taken off later: 2-norm
// of the error of 300 to 131071 positions 1.2e-7 to 6e-7 of the output's (bfloat16 keys' codes as 16 + c: 5e-7 to 2e-6).
// With 16 + c in both it is 3e-5 at 131071 positions, whose values cancel: 1.01 times what rounding alone gives an fp16
// output.  64 sequences of up to 8191 positions take 52 us in float32, 47 in fp16.
// With one term to a weight of a 16-bit output, and 256 + c for half of a key's codes, those took 46 us: the error of
// fp16 outputs over long sequences was 1.4 times what their rounding alone gives.
// A tile comes to the wave's LDS by copies of codes, scales, biases and the page numbers of a later tile; the wave waits for
// the older of two tiles alone.
// 1.47 million positions and key heads of 128 dims (218 MB, 31 us of reading): 51 us and 5.1 for the join.  No unit is
// full: a workgroup's first tile comes after 8.3 us in the median, 14.2 at most (the plan, the page numbers, the copies:
// none of which can be earlier than the one before), the vector unit is busy 55% of the time, the matrix cores 17%, and
// the waves, two to a SIMD, wait 23% of theirs.  64 sequences of up to 8191 (172 MB): 47 us and 5.8, of which
// workgroups' second pieces cost a fifth.  Products on vector instructions, a key to a lane: 98 and 6.4 ms.
// Scores by 4x4x4 products, which have no idle rows for four query heads to a key head, in an earlier form: long
// ones 2% faster, but 58 instead of 49 us for the 64 sequences and 20 instead of 16 for 32 of up to 2047, as every lane
// then lays out a whole query.
// CENTRE: for a float32 output.
// ALIGNED: pages of whole tiles: a tile lies in one page, its addresses are a scalar and a constant of the lane.
template <int G, int WAVES, bool CENTRE, bool ALIGNED, class Q>
__global__ __launch_bounds__(64 * WAVES, WAVES == 4 && G > 4 ? 1 : 2) void paged_u4_kernel(PagedArgs a) {
    using P = ElemF16;
    using B = ElemBF16;
    constexpr int HD = 32 * G, DT = 2 * G, OPS = G <= 4 ? 1 : 2;
    constexpr int NST = U4_NST, ROW = 16 * G, CODES = U4_TILE * ROW, KMETA = U4_TILE * 4 * G, VMETA = U4_TILE * 4;
    constexpr int KM = 2 * CODES, VM = KM + KMETA, TILE = VM + VMETA;
    constexpr int VBIAS = NST * TILE, IDS = VBIAS + VMETA, ROWS = IDS + NST * 256, SLOT = ROWS + 512;
    constexpr bool WIDE = G % 4 == 0;  // the scales of keys 16 bytes a lane
    constexpr int KM_COPIES = WIDE ? G / 4 : G, COPIES = 2 * G + KM_COPIES + 2;
    static_assert((NST - 1) * COPIES < 64, "the counter's range");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[WAVES * SLOT];
    __shared__ float ml[WAVES][2][16];
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // scalar, and what follows from it
    Line<WAVES, U4_TILE> line;
    line.init(a, reinterpret_cast<int64_t*>(lds));
    const Widen8<P, CENTRE> value_codes;
    const auto key_codes = [&] {
        if constexpr (Q::code == LQ_BF16) return Widen8<Q, CENTRE>{};
        else return value_codes;
    }();
    constexpr int STEP = WAVES * U4_TILE;
    const int page = a.page, cols = STEP / page, slots = STEP - cols * page;
    const uint32_t slot = (uint32_t)reinterpret_cast<uintptr_t>(lds) + wave * SLOT;
    const char *kp = static_cast<const char*>(a.k), *vp = static_cast<const char*>(a.v);
    const char *kmp = static_cast<const char*>(a.ks), *vmp = static_cast<const char*>(a.vs);
    // chunk c of row r lies at place c ^ swz(r): the 16 rows of a read spread over the banks
    constexpr bool POW2 = (G & (G - 1)) == 0;
    auto swz = [](int r) { return POW2 ? ((r >> 2) ^ (r >> 4)) & 3 & (G - 1) : 0; };
    // where this lane reads: its row of operand T = 0 (T is 4 rows further, its swizzle T ^ that of row 0), and its row
    // of values
    const int kr = 16 * (l16 >> 2) + (l16 & 3), vr = 16 * g + l16;
    uint32_t kat[POW2 ? G : 1], vat[POW2 ? G : 1];
#pragma unroll
    for (int x = 0; x < (POW2 ? G : 1); ++x) {
        kat[x] = kr * ROW + ((POW2 ? x ^ ((l16 >> 2) & (G - 1)) : 0) << 4) + 4 * g;
        vat[x] = CODES + vr * ROW + ((POW2 ? x ^ swz(vr) : 0) << 4);
    }
    auto key_at = [&](int T, int s) { return (POW2 ? kat[(s ^ T) & (G - 1)] : kat[0] + 16 * s) + 4 * T * ROW; };
    auto value_at = [&](int d) { return (POW2 ? vat[(d >> 1) & (G - 1)] : vat[0] + 16 * (d >> 1)) + 8 * (d & 1); };
    uint32_t tile_off[G];  // of the chunk that this lane copies, in a tile of consecutive rows
#pragma unroll
    for (int i = 0; i < G; ++i) {
        const int r = (64 * i + lane) / G, c = ((64 * i + lane) % G) ^ swz(r);
        tile_off[i] = r * ROW + 16 * c;
    }
    for (Piece w; line.next(a, w);) {
        __syncthreads();  // the plan's numbers are read: their LDS may be filled
        // the same in all lanes, but found in vector registers
        w.b = __builtin_amdgcn_readfirstlane(w.b);
        w.hk = __builtin_amdgcn_readfirstlane(w.hk);
        w.begin = __builtin_amdgcn_readfirstlane(w.begin);
        w.end = __builtin_amdgcn_readfirstlane(w.end);
        const int32_t* table = a.table + (int64_t)w.b * a.table_stride;
        const int first = w.begin + wave * U4_TILE;
        const int tiles = a.pages > 0 && first < w.end ? (w.end - first + STEP - 1) / STEP : 0;
        bool bad = w.over || a.pages == 0;
        vf4 o[DT], ones = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = vf4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.0f, vbias = 0.0f;
        int lift = 1024, large = -127;  // of this lane's query: above what any product needs; of the wave
        // this lane's position in the tile that is issued next, and in the one whose page number is fetched next
        int key = first + lane;
        Place at, ahead;
        at.start((uint32_t)(ALIGNED ? first : key), (uint32_t)page);
        ahead = at;
        const int last = (int)((uint32_t)(w.end - 1) / (uint32_t)page);  // the last column with a position
        auto fetch_id = [&](int t) __attribute__((always_inline)) {
            lds_copy4(table + min(ahead.col, last), slot + IDS + (t % NST) * 256);
            ahead.advance(cols, slots, page);
        };
        // tile t, whose page numbers have come; row 0 stands in past the end and for a bad page: its scores and values
        // are dropped
        auto issue = [&](int t) __attribute__((always_inline)) {
            const uint32_t to = slot + (t % NST) * TILE;
            const int id = (int)*reinterpret_cast<lds_u32*>(slot + IDS + (t % NST) * 256 + 4 * lane);
            if constexpr (ALIGNED) {
                const int one = __builtin_amdgcn_readfirstlane(id);
                const bool ok = one >= 0 && one < a.pages;
                bad |= !ok;
                const int64_t row =
                    ok ? ((int64_t)one * a.Hkv + w.hk) * page + __builtin_amdgcn_readfirstlane(at.slot) : 0;
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    lds_copy16_from(kp + row * ROW, tile_off[i], to + i * 1024);
                    lds_copy16_from(vp + row * ROW, tile_off[i], to + CODES + i * 1024);
                }
#pragma unroll
                for (int i = 0; i < KM_COPIES; ++i) {
                    if constexpr (WIDE)
                        lds_copy16_from(kmp + row * (4 * G) + i * 1024, 16 * lane, to + KM + i * 1024);
                    else lds_copy4_from(kmp + row * (4 * G) + i * 256, 4 * lane, to + KM + i * 256);
                }
                lds_copy4_from(vmp + row * 4, 4 * lane, to + VM);
                fetch_id(t + NST);
                at.advance(cols, slots, page);
                return;
            }
            const bool ok = id >= 0 && id < a.pages;
            bad |= key < w.end && !ok;
            const int64_t row = key < w.end && ok ? ((int64_t)id * a.Hkv + w.hk) * page + at.slot : 0;
            *reinterpret_cast<lds_i64*>(slot + ROWS + 8 * lane) = row;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const int r = (64 * i + lane) / G, c = ((64 * i + lane) % G) ^ swz(r);
                const int64_t off = *reinterpret_cast<lds_i64*>(slot + ROWS + 8 * r) * ROW + 16 * c;
                lds_copy16(kp + off, to + i * 1024);
                lds_copy16(vp + off, to + CODES + i * 1024);
            }
#pragma unroll
            for (int i = 0; i < KM_COPIES; ++i) {
                const int r = (64 * i + lane) / KM_COPIES, c = (64 * i + lane) % KM_COPIES;
                const char* from = kmp + *reinterpret_cast<lds_i64*>(slot + ROWS + 8 * r) * (4 * G);
                if constexpr (WIDE) lds_copy16(from + 16 * c, to + KM + i * 1024);
                else lds_copy4(from + 4 * c, to + KM + i * 256);
            }
            lds_copy4(vmp + row * 4, to + VM);
            fetch_id(t + NST);
            key += STEP;
            at.advance(cols, slots, page);
        };
        // the first page numbers and the queries are on their way together, then the first tiles while the queries are
        // laid out
        if (tiles > 0) {
#pragma unroll
            for (int t = 0; t < NST; ++t) fetch_id(t);
        }
        u4v q[G];
#pragma unroll
        for (int s = 0; s < G; ++s) q[s] = paged_query(a, w, l16, 32 * s + 8 * g, HD);
#pragma unroll
        for (int s = 0; s < G; ++s) asm volatile("" : "+v"(q[s]));  // loaded here
        wait_vmcnt<0>();
        asm volatile("" ::: "memory");
        if (tiles > 0) {
#pragma unroll
            for (int t = 0; t < NST; ++t)
                if (t < tiles) issue(t);
        }
        // queries in the order of the codes' pairs, and the sums of each group
        float sl2 = a.scale * LOG2E;
        if constexpr (Q::code == LQ_BF16) {
            uint32_t top = 0;
#pragma unroll
            for (int s = 0; s < G; ++s)
#pragma unroll
                for (int p = 0; p < 4; ++p) top = max(top, max(q[s][p] & 0x7fffu, (q[s][p] >> 16) & 0x7fffu));
            // half of the largest value's exponent, where the scores' factor stays above float32's end
            const int e = max(((int)(__float_as_uint(quarter_max(__uint_as_float(top << 16))) >> 23) - 127) >> 1,
                              -126 - ((int)(__float_as_uint(sl2) >> 23) - 127));
            sl2 = __builtin_amdgcn_ldexpf(sl2, e);
            const float by = __builtin_amdgcn_ldexpf(1.0f / key_codes.TIMES, -e);
#pragma unroll
            for (int s = 0; s < G; ++s)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const f2v u = unpack2(Q{}, q[s][p]);
                    q[s][p] = pack2(Q{}, u[0] * by, u[1] * by);
                }
        }
        u4v qf[G], qsum[OPS];
#pragma unroll
        for (int i = 0; i < OPS; ++i) qsum[i] = u4v{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < G; ++s) {
            float sum = 0.0f;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const f2v u = unpack2(Q{}, q[s][p]);
                sum += u[0] + u[1];
            }
#pragma unroll
            for (int p = 0; p < 4; ++p)  // halves of words p / 2 and p / 2 + 2
                qf[s][p] = __builtin_amdgcn_perm(q[s][2 + (p >> 1)], q[s][p >> 1], p & 1 ? 0x07060302u : 0x05040100u);
            sum = quarter_sum(sum) * key_codes.TIMES;
            // lane group g holds the g-th of three terms of the sum, and of what the codes' offsets add, negative
            auto term = [&](float x) {
                const float t0 = unpack2(B{}, pack2(B{}, x, 0.0f))[0], r1 = x - t0;
                const float t1 = unpack2(B{}, pack2(B{}, r1, 0.0f))[0];
                return g == 0 ? t0 : g == 1 ? t1 : g == 2 ? r1 - t1 : 0.0f;
            };
            const uint32_t both = pack2(B{}, term(sum), term(-key_codes.ADDED * sum));
            const int at = G <= 4 ? G + s : 8 + s;
            qsum[0][(s >> 1) & 3] |= s & 1 ? both & 0xffff0000u : both >> 16;      // with the scales
            qsum[at >> 3][(at >> 1) & 3] |= at & 1 ? both << 16 : both & 0xffffu;  // with the biases
        }
        for (int t = 0; t < tiles; ++t) {
            if (t + 1 == tiles) wait_vmcnt<0>();
            else wait_vmcnt<COPIES>();
            static_assert(NST == 2, "the waits above");
            asm volatile("" ::: "memory");
            const uint32_t tile = slot + (t % NST) * TILE, meta_at = tile + KM + kr * 4 * G, four_at = tile + 64 * g;
            const int left = w.end - (first + t * STEP);  // positions of this tile that exist
            // Reads come in batches ahead of their use, and each operand T's products beside the sums of the one
            // before: left to itself the compiler waits for every read and every product in turn.  A wave's LDS
            // operations keep their order, so a write needs no wait before the read that follows.
            u4v meta[4][OPS];  // scales and biases of the rows this lane feeds, in one operand or in two
            uint32_t code[4][G];
            float ks[G];
#pragma unroll
            for (int T = 0; T < 4; ++T) {
                const uint32_t from = meta_at + 4 * T * 4 * G;
#pragma unroll
                for (int i = 0; i < OPS; ++i) meta[T][i] = u4v{0, 0, 0, 0};
                if constexpr (G == 4) {
                    meta[T][0] = *reinterpret_cast<lds_u4v*>(from);
                } else if constexpr (G < 4) {
#pragma unroll
                    for (int i = 0; i < G; ++i) meta[T][0][i] = *reinterpret_cast<lds_u32*>(from + 4 * i);
                } else {
#pragma unroll
                    for (int i = 0; i < 2 * G; ++i)
                        meta[T][i / G][(i % G) >> 1] |= (uint32_t)*reinterpret_cast<lds_u16*>(from + 2 * i)
                                                        << (16 * ((i % G) & 1));
                }
            }
#pragma unroll
            for (int s = 0; s < G; ++s)
                ks[s] = bf16_bits_to_f32(*reinterpret_cast<lds_u16*>(tile + KM + lane * 4 * G + 2 * s));
            const uint32_t vw = *reinterpret_cast<lds_u32*>(tile + VM + 4 * lane);
#pragma unroll
            for (int T = 0; T < 4; ++T)
#pragma unroll
                for (int s = 0; s < G; ++s) code[T][s] = *reinterpret_cast<lds_u32*>(tile + key_at(T, s));
            asm volatile("" ::: "memory");
            // the scales and the values' biases as float32, [group][position], over the bytes that every lane has read;
            // codes are finite: a weight of 0 drops what lies past the end once its scale and bias are 0
#pragma unroll
            for (int s = 0; s < G; ++s) *reinterpret_cast<lds_f32*>(tile + KM + 256 * s + 4 * lane) = ks[s];
            const int mine = lane < left ? (int)(max(vw & 0x7fffu, vw >> 16 & 0x7fffu) >> 7) - 127 : -127;
            if (__any(mine > large)) {
                const int to = __builtin_amdgcn_readfirstlane(wave_max(mine));
                vbias = __builtin_amdgcn_ldexpf(vbias, large - to);
                lift += to - large;
                large = to;
            }
            const float vs = lane < left ? __builtin_amdgcn_ldexpf(bf16_bits_to_f32((uint16_t)vw), -large) : 0.0f;
            *reinterpret_cast<lds_f32*>(tile + VM + 4 * lane) = vs;
            *reinterpret_cast<lds_f32*>(slot + VBIAS + 4 * lane) =
                lane < left ? __builtin_fmaf(7.5f, vs, __builtin_amdgcn_ldexpf(bf16_bits_to_f32((uint16_t)(vw >> 16)), -large)) : 0.0f;
            asm volatile("" ::: "memory");
            vf4 sc[4], x[2][G], f[2][G];
            auto factors = [&](int T) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < G; ++s) f[T & 1][s] = *reinterpret_cast<lds_vf4*>(four_at + KM + 256 * s + 16 * T);
            };
            factors(0);
#pragma unroll
            for (int T = 0; T < 5; ++T) {
                if (T < 4) {
                    sc[T] = mfma_16x16x32(B{}, meta[T][0], qsum[0], vf4{0.f, 0.f, 0.f, 0.f});
                    if constexpr (OPS == 2) sc[T] = mfma_16x16x32(B{}, meta[T][1], qsum[1], sc[T]);
#pragma unroll
                    for (int s = 0; s < G; ++s)
                        x[T & 1][s] = mfma_16x16x32(Q{}, key_codes(code[T][s]), qf[s], vf4{0.f, 0.f, 0.f, 0.f});
                }
                if (T > 0) {
#pragma unroll
                    for (int s = 0; s < G; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sc[T - 1][i] = __builtin_fmaf(f[(T - 1) & 1][s][i], x[(T - 1) & 1][s][i], sc[T - 1][i]);
                }
                if (T + 1 < 4) factors(T + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            // what the values need, read beside the weights
            v2i vcode[DT];
            vf4 vf[4], vb[4];
#pragma unroll
            for (int T = 0; T < 4; ++T) {
                vf[T] = *reinterpret_cast<lds_vf4*>(four_at + VM + 16 * T);
                vb[T] = *reinterpret_cast<lds_vf4*>(slot + VBIAS + 64 * g + 16 * T);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) vcode[d] = lds_read_tr4(tile + value_at(d));
            __builtin_amdgcn_sched_barrier(0);
            if (left < U4_TILE) {
#pragma unroll
                for (int T = 0; T < 4; ++T)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (16 * g + 4 * T + i >= left) sc[T][i] = -INFINITY;
                        asm volatile("" : "+v"(sc[T][i]));  // in the branch: not sixteen selects for every tile
                    }
            }
            // weights relative to the running maximum, which may lag by 2^RESCALE_AT
            float mx = -INFINITY;
#pragma unroll
            for (int T = 0; T < 4; ++T)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[T][i]);
            mx = quarter_max(mx) * sl2;
            if (__any(mx > m + RESCALE_AT)) {
                const float to = fmaxf(m, ceilf(mx)), finite = to == -INFINITY ? 0.0f : to;
                const float corr = __builtin_amdgcn_exp2f(m - finite);
                lift += (int)fminf(finite - m, 4096.0f);  // the products' reference stays where it was
                m = to;
                l *= corr;
                vbias *= corr;
            }
            const float from = m == -INFINITY ? 0.0f : m;
            float most = 0.0f;  // the largest weight times its value's scale
#pragma unroll
            for (int T = 0; T < 4; ++T) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[T][i], sl2, -from));
                    l += e;
                    vbias = __builtin_fmaf(e, vb[T][i], vbias);
                    sc[T][i] = e * vf[T][i];
                    most = fmaxf(most, fabsf(sc[T][i]));
                }
            }
            most = quarter_max(most);
            if (__any(__builtin_amdgcn_ldexpf(most, lift) >= ldexpf(1.0f, U4_LIMIT))) {
                const int to = min(lift, U4_SET + 127 - (int)(__float_as_uint(most) >> 23));
                const float f = __builtin_amdgcn_ldexpf(1.0f, to - lift);
                lift = to;
#pragma unroll
                for (int i = 0; i < 4; ++i) ones[i] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][i] *= f;
            }
#pragma unroll
            for (int T = 0; T < 4; ++T)
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[T][i] = __builtin_amdgcn_ldexpf(sc[T][i], lift);
            // O^T += C^T P^T: word j of a transposed read holds positions 8 j .. of this lane's 16, pairs four apart
            u4v hi[2], lo[2];
            float minus = -1.0f;
            asm("" : "+v"(minus));  // a product with it reads a half of hi as it lies: no conversion
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float x = sc[2 * j][p], y = sc[2 * j + 1][p];
                    hi[j][p] = pack2(P{}, x, y);
                    const f2v u = unpack2(P{}, hi[j][p]);
                    lo[j][p] = pack2(P{}, __builtin_fmaf(u[0], minus, x), __builtin_fmaf(u[1], minus, y));
                }
            const u4v offset = {0x4de04de0u, 0x4de04de0u, 0x4de04de0u, 0x4de04de0u};  // 23.5
            if constexpr (!CENTRE) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    ones = mfma_16x16x32(P{}, offset, hi[j], ones);
                    ones = mfma_16x16x32(P{}, offset, lo[j], ones);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const u4v v = value_codes((uint32_t)vcode[d][j]);
                    o[d] = mfma_16x16x32(P{}, v, hi[j], o[d]);
                    o[d] = mfma_16x16x32(P{}, v, lo[j], o[d]);
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile is read: its LDS may be filled again
            if (t + NST < tiles) issue(t + NST);
        }
        wait_vmcnt<0>();  // page numbers fetched ahead
        // what all dims of a query share: the sum of its values' middles
        const float extra = quarter_sum(vbias);
        Sums<DT, P> sums;
        const int down = large >= U4_LARGE && fabsf(m) < 0x1p22f ? U4_DOWN : 0;
        sums.m = m + (float)down;
        sums.l = __builtin_amdgcn_ldexpf(l, -down);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sums.o[d][i] = __builtin_amdgcn_ldexpf(__builtin_amdgcn_ldexpf(o[d][i] - ones[0], -lift) + extra, large - down);
        paged_finish<false, WAVES, SLOT, DT, Q>(a, w, lds, ml, sums, bad);
    }
    paged_empty<WAVES, Q>(a);
}

}  // namespace

void paged_u4_launch(const PagedArgs& a, int q_type, bool few, dim3 grid, hipStream_t st) {
    with_half(q_type, [&](auto q) {
        using Q = decltype(q);
        auto launch = [&](auto groups, auto waves) {
            constexpr int G = decltype(groups)::value, W = decltype(waves)::value;
            auto all = [&](auto every) {
                constexpr bool CENTRE = decltype(every)::value;
                if (a.page % U4_TILE == 0)
                    hipLaunchKernelGGL((paged_u4_kernel<G, W, CENTRE, true, Q>), grid, dim3(64 * W), 0, st, a);
                else
                    hipLaunchKernelGGL((paged_u4_kernel<G, W, CENTRE, false, Q>), grid, dim3(64 * W), 0, st, a);
            };
            if (a.out_f32) all(std::true_type{});
            else all(std::false_type{});
        };
        // a few short sequences: eight waves each where the LDS holds their tiles, to hide more of the latency
        auto go = [&](auto groups) {
            if constexpr (decltype(groups)::value < 4) {
                if (few) return launch(groups, std::integral_constant<int, 8>{});
            }
            launch(groups, std::integral_constant<int, 4>{});
        };
        switch (a.hd / U4_GROUP) {
        case 1: go(std::integral_constant<int, 1>{}); break;
        case 2: go(std::integral_constant<int, 2>{}); break;
        case 3: go(std::integral_constant<int, 3>{}); break;
        case 4: go(std::integral_constant<int, 4>{}); break;
        case 5: go(std::integral_constant<int, 5>{}); break;
        case 6: go(std::integral_constant<int, 6>{}); break;
        case 7: go(std::integral_constant<int, 7>{}); break;
        default: go(std::integral_constant<int, 8>{}); break;
        }
    });
}

}  // namespace lq
