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
constexpr int U4_WAVES = 4;
constexpr int U4_NST = 2;     // tiles on their way

// Four registers of eight 16-bit values 16 + c for the codes c of a word; pair p holds codes p and p + 4.  A code
// under the exponent of 16 is one shift and one and-or for two of them.
__device__ __forceinline__ u4v widen8(ElemBF16, uint32_t w) {
    constexpr uint32_t M = 0x00780078u, B = 0x41804180u;
    return u4v{((w << 3) & M) | B, ((w >> 1) & M) | B, ((w >> 5) & M) | B, ((w >> 9) & M) | B};
}
__device__ __forceinline__ u4v widen8(ElemF16, uint32_t w) {
    constexpr uint32_t M = 0x03c003c0u, B = 0x4c004c00u;
    return u4v{((w << 6) & M) | B, ((w << 2) & M) | B, ((w >> 2) & M) | B, ((w >> 6) & M) | B};
}

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
// A tile comes to the wave's LDS by copies of codes, scales, biases and the page numbers of a later tile; the wave waits for
// its oldest tile alone.
template <int G, class Q>
__global__ __launch_bounds__(64 * U4_WAVES, G <= 4 ? 2 : 1) void paged_u4_kernel(PagedArgs a) {
    using P = ElemBF16;
    constexpr int HD = 32 * G, DT = 2 * G, WAVES = U4_WAVES, NST = U4_NST;
    constexpr int ROW = 16 * G, CODES = U4_TILE * ROW, KMETA = U4_TILE * 4 * G, VMETA = U4_TILE * 4;
    constexpr int TILE = 2 * CODES + KMETA + VMETA;
    constexpr bool WIDE = G % 4 == 0;                 // the scales of keys 16 bytes a lane
    constexpr int KCOPIES = WIDE ? G / 4 : G, COPIES = 2 * G + KCOPIES + 2;
    constexpr int IDS = NST * TILE, ROWS = IDS + NST * 256, VBIAS = ROWS + 512, SLOT = VBIAS + 256;
    static_assert((NST - 1) * COPIES < 64, "the counter's range");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[WAVES * SLOT];
    __shared__ float ml[WAVES][2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    Line<WAVES, U4_TILE> line;
    line.init(a, reinterpret_cast<int64_t*>(lds));
    constexpr int STEP = WAVES * U4_TILE;
    const int page = a.page, cols = STEP / page, slots = STEP - cols * page;
    const uint32_t slot = (uint32_t)reinterpret_cast<uintptr_t>(lds) + wave * SLOT;
    const float sl2 = a.scale * LOG2E;
    const char *kp = static_cast<const char*>(a.k), *vp = static_cast<const char*>(a.v);
    const char *kmp = static_cast<const char*>(a.ks), *vmp = static_cast<const char*>(a.vs);
    auto swz = [](int r) { return (G & (G - 1)) == 0 ? ((r >> 2) ^ (r >> 4)) & (G - 1) : 0; };
    for (Piece w; line.next(a, w);) {
        __syncthreads();  // the plan's numbers are read: their LDS may be filled
        // queries in the order of the codes' pairs, and the sums of each group
        u4v qf[G];
        vf4 start[G];
        u4v qsum = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < G; ++s) {
            const u4v q = paged_query(a, w, l16, 32 * s + 8 * g, HD);
            float sum = 0.0f;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const f2v u = unpack2(Q{}, q[p]);
                sum += u[0] + u[1];
            }
#pragma unroll
            for (int p = 0; p < 4; ++p)  // halves of words p / 2 and p / 2 + 2
                qf[s][p] = __builtin_amdgcn_perm(q[2 + (p >> 1)], q[p >> 1], p & 1 ? 0x07060302u : 0x05040100u);
            sum = quarter_sum(sum);
            start[s] = vf4{-16.0f * sum, -16.0f * sum, -16.0f * sum, -16.0f * sum};
            // 24 bits of the sum as three bfloat16 terms, lane group g the g-th: the biases' products in one instruction
            const float t0 = bf16_bits_to_f32(f32_to_bf16_bits(sum)), t1 = bf16_bits_to_f32(f32_to_bf16_bits(sum - t0));
            const float term = g == 0 ? t0 : g == 1 ? t1 : g == 2 ? sum - t0 - t1 : 0.0f;
            qsum[s >> 1] |= (uint32_t)f32_to_bf16_bits(term) << (16 * (s & 1));
        }
        const int32_t* table = a.table + (int64_t)w.b * a.table_stride;
        const int first = w.begin + wave * U4_TILE;
        const int tiles = a.pages > 0 && first < w.end ? (w.end - first + STEP - 1) / STEP : 0;
        bool bad = w.over || a.pages == 0;
        vf4 o[DT], ones = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = vf4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.0f, vbias = 0.0f;
        // this lane's position in the tile that is issued next, and in the one whose page numbers are fetched next
        int key = first + lane;
        Place at, ahead;
        at.start((uint32_t)key, (uint32_t)page);
        ahead = at;
        const int last = (int)((uint32_t)(w.end - 1) / (uint32_t)page);  // the last column with a position
        auto issue = [&](int t) __attribute__((always_inline)) {
            const uint32_t to = slot + (t % NST) * TILE, ids = slot + IDS + (t % NST) * 256;
            const int id = (int)*reinterpret_cast<lds_u32*>(ids + 4 * lane);
            const bool ok = id >= 0 && id < a.pages;
            bad |= key < w.end && !ok;
            // row 0 stands in past the end and for a bad page: its scores and values are dropped
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
            if constexpr (WIDE) {
#pragma unroll
                for (int i = 0; i < KCOPIES; ++i) {
                    const int r = (64 * i + lane) / KCOPIES, c = (64 * i + lane) % KCOPIES;
                    const int64_t off = *reinterpret_cast<lds_i64*>(slot + ROWS + 8 * r) * (4 * G) + 16 * c;
                    lds_copy16(kmp + off, to + 2 * CODES + i * 1024);
                }
            } else {
#pragma unroll
                for (int i = 0; i < KCOPIES; ++i) {
                    const int r = (64 * i + lane) / G, c = (64 * i + lane) % G;
                    const int64_t off = *reinterpret_cast<lds_i64*>(slot + ROWS + 8 * r) * (4 * G) + 4 * c;
                    lds_copy4(kmp + off, to + 2 * CODES + i * 256);
                }
            }
            lds_copy4(vmp + row * 4, to + 2 * CODES + KMETA);
            lds_copy4(table + min(ahead.col, last), ids);  // the tile NST later: this tile's numbers are read
            key += STEP;
            at.advance(cols, slots, page);
            ahead.advance(cols, slots, page);
        };
        if (tiles > 0) {
            // page numbers of the first tiles
#pragma unroll
            for (int t = 0; t < NST; ++t) {
                lds_copy4(table + min(ahead.col, last), slot + IDS + t * 256);
                ahead.advance(cols, slots, page);
            }
            wait_vmcnt<0>();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int t = 0; t < NST; ++t)
                if (t < tiles) issue(t);
        }
        for (int t = 0; t < tiles; ++t) {
            if (tiles - 1 - t == 0) wait_vmcnt<0>();
            else wait_vmcnt<COPIES>();
            static_assert(NST == 2, "the waits above");
            asm volatile("" ::: "memory");
            const uint32_t kt = slot + (t % NST) * TILE, vt = kt + CODES, km = vt + CODES, vm = km + KMETA;
            const int left = w.end - (first + t * STEP);  // positions of this tile that exist
            // biases of the rows this lane feeds to the matrix cores; the scales as float32, [group][position]
            u4v kb[4];
#pragma unroll
            for (int T = 0; T < 4; ++T) {
                const uint32_t r = 16 * (l16 >> 2) + 4 * T + (l16 & 3), from = km + r * 4 * G + 2 * G;
                kb[T] = u4v{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < G; s += 2) {
                    if constexpr (G % 2 == 0) kb[T][s >> 1] = *reinterpret_cast<lds_u32*>(from + 2 * s);
                    else
                        kb[T][s >> 1] = *reinterpret_cast<lds_u16*>(from + 2 * s) |
                                        (s + 1 < G ? (uint32_t)*reinterpret_cast<lds_u16*>(from + 2 * s + 2) << 16 : 0u);
                }
            }
            float ks[G];
#pragma unroll
            for (int s = 0; s < G; ++s)
                ks[s] = bf16_bits_to_f32(*reinterpret_cast<lds_u16*>(km + lane * 4 * G + 2 * s));
            const uint32_t vw = *reinterpret_cast<lds_u32*>(vm + 4 * lane);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int s = 0; s < G; ++s) *reinterpret_cast<lds_f32*>(km + 256 * s + 4 * lane) = ks[s];
            // codes are finite: a weight of 0 drops what lies past the end once its scale and bias are
            *reinterpret_cast<lds_f32*>(vm + 4 * lane) = lane < left ? bf16_bits_to_f32((uint16_t)vw) : 0.0f;
            *reinterpret_cast<lds_f32*>(slot + VBIAS + 4 * lane) = lane < left ? bf16_bits_to_f32((uint16_t)(vw >> 16)) : 0.0f;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            vf4 sc[4];
#pragma unroll
            for (int T = 0; T < 4; ++T) {
                const int r = 16 * (l16 >> 2) + 4 * T + (l16 & 3);
                sc[T] = mfma_16x16x32(P{}, kb[T], qsum, vf4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int s = 0; s < G; ++s) {
                    const uint32_t c = *reinterpret_cast<lds_u32*>(kt + r * ROW + ((s ^ swz(r)) << 4) + 4 * g);
                    const vf4 x = mfma_16x16x32(Q{}, widen8(Q{}, c), qf[s], start[s]);
                    const vf4 f = *reinterpret_cast<lds_vf4*>(km + 256 * s + 4 * (16 * g + 4 * T));
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[T][i] = __builtin_fmaf(f[i], x[i], sc[T][i]);
                }
            }
            // weights relative to the running maximum, as the other caches' kernels form them
            float mx = -INFINITY;
#pragma unroll
            for (int T = 0; T < 4; ++T)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (left < U4_TILE && 16 * g + 4 * T + i >= left) sc[T][i] = -INFINITY;
                    mx = fmaxf(mx, sc[T][i]);
                }
            mx = quarter_max(mx) * sl2;
            if (__any(mx > m + RESCALE_AT)) {
                const float mn = fmaxf(m, weight_reference<P>(mx));
                const float corr = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= corr;
                vbias *= corr;
#pragma unroll
                for (int i = 0; i < 4; ++i) ones[i] *= corr;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][i] *= corr;
            }
            const float base = m == -INFINITY ? 0.0f : m - WEIGHT_SHIFT<P>;
#pragma unroll
            for (int T = 0; T < 4; ++T) {
                const vf4 f = *reinterpret_cast<lds_vf4*>(vm + 4 * (16 * g + 4 * T));
                const vf4 b = *reinterpret_cast<lds_vf4*>(slot + VBIAS + 4 * (16 * g + 4 * T));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[T][i], sl2, -base));
                    l += e;
                    vbias = __builtin_fmaf(e, b[i], vbias);
                    sc[T][i] = e * f[i];
                }
            }
            // O^T += C^T P^T: word j of a transposed read holds positions 8 j .. of this lane's 16, pairs four apart
            u4v hi[2], lo[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float x = sc[2 * j][p], y = sc[2 * j + 1][p];
                    hi[j][p] = pack2(P{}, x, y);
                    const f2v u = unpack2(P{}, hi[j][p]);
                    lo[j][p] = pack2(P{}, x - u[0], y - u[1]);
                }
            const u4v sixteen = {0x41804180u, 0x41804180u, 0x41804180u, 0x41804180u};
            const int vr = 16 * g + l16;
            auto codes = [&](int d) __attribute__((always_inline)) {
                return lds_read_tr4(vt + vr * ROW + (((d >> 1) ^ swz(vr)) << 4) + 8 * (d & 1));
            };
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                ones = mfma_16x16x32(P{}, sixteen, hi[j], ones);
                ones = mfma_16x16x32(P{}, sixteen, lo[j], ones);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const v2i c = codes(d);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const u4v v = widen8(P{}, (uint32_t)c[j]);
                    o[d] = mfma_16x16x32(P{}, v, hi[j], o[d]);
                    o[d] = mfma_16x16x32(P{}, v, lo[j], o[d]);
                }
            }
            if (a.out_f32) {  // every bit of the weights
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const f2v u = unpack2(P{}, hi[j][p]), e = unpack2(P{}, lo[j][p]);
                        hi[j][p] = pack2(P{}, sc[2 * j][p] - u[0] - e[0], sc[2 * j + 1][p] - u[1] - e[1]);
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) ones = mfma_16x16x32(P{}, sixteen, hi[j], ones);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const v2i c = codes(d);
#pragma unroll
                    for (int j = 0; j < 2; ++j) o[d] = mfma_16x16x32(P{}, widen8(P{}, (uint32_t)c[j]), hi[j], o[d]);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile is read: its LDS may be filled again
            if (t + NST < tiles) issue(t + NST);
        }
        wait_vmcnt<0>();  // page numbers fetched ahead
        // what all dims of a query share: the sum of its values' biases, less the 16 of every code
        const float extra = quarter_sum(vbias) - ones[0];
        Sums<DT, P> sums;
        sums.m = m;
        sums.l = l;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums.o[d][i] = o[d][i] + extra;
        paged_finish<false, WAVES, SLOT, DT, Q>(a, w, lds, ml, sums, bad);
    }
    paged_empty<WAVES, Q>(a);
}

}  // namespace

void paged_u4_launch(const PagedArgs& a, int q_type, dim3 grid, hipStream_t st) {
    with_half(q_type, [&](auto q) {
        using Q = decltype(q);
        auto go = [&](auto groups) {
            hipLaunchKernelGGL((paged_u4_kernel<decltype(groups)::value, Q>), grid, dim3(64 * U4_WAVES), 0, st, a);
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
