// lq_paged.hip -- a key-value cache in pages: appending new tokens' keys and values, and the
// attention of one new token per sequence over its pages.
//
// Layout.  k / v pages [pages][Hkv][page][hd] (fp16, bfloat16, or int8 codes with one float32
// scale per row in [pages][Hkv][page]); table [seqs][table_stride] of page numbers; position p
// of sequence s is slot p % page of page table[s][p / page].  A head's rows of one page lie next
// to each other, so the attention of a head streams page * hd contiguous values.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "lq_attn.h"
#include "lq_place.h"

namespace lq {
namespace {

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
    float *ks, *vs;
    int64_t pages, page;
};

// Row of packed token t's head 0 in the pool, or -1 when it has no place.
__device__ __forceinline__ int64_t token_row(const AppendArgs& a, int64_t t) {
    int64_t s, pos;
    if (!token_place(t, a.starts, a.seqs, a.lengths, s, pos)) return -1;
    return position_row(pos, a.table + s * a.table_stride, a.table_stride, a.pages, a.Hkv, a.page);
}

// One thread per value, for rows that 16-byte accesses do not fit.
template <class Src, class Dst>
__global__ __launch_bounds__(256) void append_any_kernel(AppendArgs a) {
    const int64_t per = a.Hkv * a.hd;
    const int64_t t = blockIdx.x;
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

// TOK tokens per workgroup.  A thread keeps one place of the rows (k or v, head, eight dims) and
// moves it for every token, the loads of all of them in flight together.
template <int TOK, class Src, class Dst>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
    __shared__ int64_t rows[TOK];
    const int64_t t0 = (int64_t)blockIdx.x * TOK;
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

// One wave per (token, head, k or v), element by element.
template <class Src>
__global__ __launch_bounds__(64) void append_i8_any_kernel(AppendArgs a) {
    const int64_t t = blockIdx.x;
    const int64_t row = token_row(a, t);
    if (row < 0) return;
    const int h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const typename Src::T* src = static_cast<const typename Src::T*>(is_v ? a.v : a.k) + t * a.ld + h * a.hd;
    const int64_t r = row + h * a.page;
    int32_t top = 0;
    for (int64_t d = threadIdx.x; d < a.hd; d += 64) top = max(top, magnitude(Src::load(src[d])));
    const RowScale rs(wave_max(top));
    int8_t* dst = static_cast<int8_t*>(is_v ? a.vp : a.kp) + r * a.hd;
    for (int64_t d = threadIdx.x; d < a.hd; d += 64) dst[d] = (int8_t)rs.code(Src::load(src[d]));
    if (threadIdx.x == 0) (is_v ? a.vs : a.ks)[r] = rs.scale;
}

// LPR lanes per row of hd <= 8 LPR values, eight values a lane; one workgroup per token.
template <int LPR, class Src>
__global__ __launch_bounds__(256) void append_i8_kernel(AppendArgs a) {
    const int64_t t = blockIdx.x;
    const int64_t row = token_row(a, t);
    if (row < 0) return;
    const uint32_t d = (threadIdx.x % LPR) * 8;
    // every lane of a wave takes the same number of rounds: the exchange below needs them all
    for (uint32_t e = threadIdx.x / LPR; e < ((uint32_t)a.Hkv * 2 + 64 / LPR - 1) / (64 / LPR) * (64 / LPR); e += 256 / LPR) {
        const bool is_v = e & 1, mine = e < (uint32_t)a.Hkv * 2 && d < (uint32_t)a.hd;
        const uint32_t h = e >> 1;
        float x[8] = {};
        if (mine) load8<Src>(static_cast<const typename Src::T*>(is_v ? a.v : a.k) + t * a.ld + (int64_t)h * a.hd + d, x);
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
        if (d == 0) (is_v ? a.vs : a.ks)[r] = rs.scale;
    }
}

// ------------------------------------------------------------------------------ attention

struct PagedArgs {
    const void* q;
    int64_t ldq;
    int B, H, Hkv, hd, group, qtiles;
    const void *k, *v;
    const float *ks, *vs;
    int64_t pages;
    int page;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    float scale;
    void* out;
    int out_f32;
    int q_vec;          // q may be read 16 bytes at a time
    int chunk, splits;  // positions of a workgroup; chunk 0 .. splits - 1 (the last takes the rest)
    float *part_o, *part_ml;
};

constexpr int PG_WAVES = 4, PG_K = 32;  // waves of a workgroup, keys of a wave's tile

// Length of sequence b within its table (positions past it are an error: `over`), and the number
// of chunks it takes (the last one takes what the plan did not foresee).
__device__ __forceinline__ int sequence_length(const PagedArgs& a, int b, bool& over, int& used) {
    const int64_t cap = min(a.table_stride * a.page, (int64_t)(INT32_MAX - 4096));
    const int len = max(a.lengths[b], 0);
    over = len > cap;
    const int n = over ? (int)cap : len;
    used = min(a.splits, (int)(((int64_t)n + a.chunk - 1) / a.chunk));
    return n;
}

// Workgroup (key head and tile of 16 query heads, sequence, chunk of positions).  Each wave takes
// every fourth tile of 32 positions with a maximum, sum and accumulators of its own, and the
// waves meet at the end: no barrier inside the loop.
//   S^T = K Q^T (v_mfma 16x16x32): lane (l, g) loads the rows l and 16 + l of K straight into the A
//   operand and receives positions 4 g + i (and 16 + 4 g + i) of query l;
//   O^T += V^T P^T: those weights are the B operand as they are; V passes through the wave's LDS,
//   whose transposing read gives lane (l, g) dim l of the same positions.
// A weight enters as two 16-bit terms (about 16 significant bits): the products are free beside the
// loads.  An int8 cache's codes are exact in 16 bits; the key's scale multiplies the score, the
// value's scale the weight, which is then bfloat16 for its range.
template <int HDP, bool EXACT, class Q, class C>
__global__ __launch_bounds__(64 * PG_WAVES) void paged_tile_kernel(PagedArgs a) {
    constexpr bool I8 = C::code == LQ_I8;
    using P = std::conditional_t<I8, ElemBF16, Q>;  // type of the second product
    constexpr int KS = HDP / 32, DT = HDP / 16;
    constexpr int VROW = HDP * 2, VTILE = PG_K * VROW;            // bytes of a V row / tile in LDS
    constexpr int OROW = HDP + 4, OTILE = 16 * OROW * 4;          // floats of a query's row, bytes of a wave's sums
    constexpr int SLOT = (VTILE > OTILE ? VTILE : OTILE) + 256;   // + 64 scales
    __shared__ __attribute__((aligned(16))) uint8_t lds[PG_WAVES * SLOT];
    __shared__ float mls[PG_WAVES][2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    const int hk = blockIdx.x / a.qtiles, qt = blockIdx.x - hk * a.qtiles, b = blockIdx.y, split = blockIdx.z;
    const int hd = EXACT ? HDP : a.hd, heads = min(16, a.group - 16 * qt);
    const int h0 = hk * a.group + 16 * qt;
    bool bad;  // a position that has no page
    int used;
    const int len = sequence_length(a, b, bad, used);
    const int64_t first = (int64_t)split * a.chunk;
    if (split > 0 && split >= used) return;
    const int end = split == a.splits - 1 ? len : (int)min((int64_t)len, first + a.chunk);
    const int begin = (int)first;

    // dims of this lane's eight slots in step s of the first product
    auto dims = [&](int s) { return I8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };
    u4v qf[KS];
    {
        const uint16_t* qr = static_cast<const uint16_t*>(a.q) + b * a.ldq + (int64_t)(h0 + min(l16, heads - 1)) * hd;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = u4v{0, 0, 0, 0};
            if (EXACT || dims(s) < hd) {
                if (a.q_vec) {
                    qf[s] = *reinterpret_cast<const u4v*>(qr + dims(s));
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) qf[s][j >> 1] |= (uint32_t)qr[dims(s) + j] << (16 * (j & 1));
                }
            }
        }
    }
    const int32_t* table = a.table + (int64_t)b * a.table_stride;
    // page number of a position (-1: none), and the row of a position in the pool
    auto page_of = [&](int key) -> int {
        const uint32_t col = (uint32_t)key / (uint32_t)a.page;
        return key < end && col < a.table_stride ? table[col] : -1;
    };
    auto row_of = [&](int key, int id) -> int64_t {
        return ((int64_t)id * a.Hkv + hk) * a.page + (uint32_t)key % (uint32_t)a.page;
    };
    // a tile in registers: K (and V) rows l16 and 16 + l16, and their scales
    u4v kr[2][I8 ? KS / 2 : KS], vr[2][I8 ? KS / 2 : KS];
    float ksc[2], vsc[2];
    auto fetch = [&](int key0, const int (&id)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int T = 0; T < 2; ++T) {
            const int key = key0 + 16 * T + l16;
            const bool ok = id[T] >= 0 && id[T] < a.pages;
            bad |= key < end && !ok;
            const int64_t row = ok ? row_of(key, id[T]) : 0;  // row 0 stands in: its scores and values are dropped
            if constexpr (I8) {
                const int8_t* kp = static_cast<const int8_t*>(a.k) + row * hd;
                const int8_t* vp = static_cast<const int8_t*>(a.v) + row * hd;
                ksc[T] = a.ks[row];
                vsc[T] = a.vs[row];
#pragma unroll
                for (int s = 0; s < KS / 2; ++s) {
                    const int d = 64 * s + 16 * g;
                    if constexpr (EXACT) {
                        kr[T][s] = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(kp + d));
                        vr[T][s] = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(vp + d));
                    } else {
                        const u2v k0 = *reinterpret_cast<const u2v*>(kp + (d < hd ? d : 0));
                        const u2v k1 = *reinterpret_cast<const u2v*>(kp + (d + 8 < hd ? d + 8 : 0));
                        const u2v v0 = *reinterpret_cast<const u2v*>(vp + (d < hd ? d : 0));
                        const u2v v1 = *reinterpret_cast<const u2v*>(vp + (d + 8 < hd ? d + 8 : 0));
                        kr[T][s] = u4v{k0[0], k0[1], k1[0], k1[1]};
                        vr[T][s] = u4v{v0[0], v0[1], v1[0], v1[1]};
                    }
                }
            } else {
                const uint16_t* kp = static_cast<const uint16_t*>(a.k) + row * hd;
                const uint16_t* vp = static_cast<const uint16_t*>(a.v) + row * hd;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int d = EXACT || dims(s) < hd ? dims(s) : 0;
                    kr[T][s] = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(kp + d));
                    vr[T][s] = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(vp + d));
                }
            }
        }
    };

    vf4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = vf4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;
    const float sl2 = a.scale * LOG2E;
    uint8_t* slot = lds + wave * SLOT;
    float* scales = reinterpret_cast<float*>(slot + SLOT - 256);
    const uint32_t slot_at = (uint32_t)reinterpret_cast<uintptr_t>(slot);
    // 16-byte chunk c of V row r lies at chunk c ^ swz(r): the writes (16 rows, 4 chunks) and the
    // transposing reads (4 rows, 2 chunks a group) spread over the banks
    auto swz = [](int r) { return HDP == 64 ? 2 * ((r >> 1) & 3) : HDP % 128 == 0 ? 2 * (r & 7) : 2 * (r & 3); };
    const int vi = lane & 15, trow = 4 * g + (vi >> 2);
    constexpr float SHIFT = WEIGHT_SHIFT<P>;

    const int stride = PG_WAVES * PG_K;
    int key0 = begin + wave * PG_K;
    if (a.pages > 0 && key0 < end) {
        int id[2], next[2];
#pragma unroll
        for (int T = 0; T < 2; ++T) {
            id[T] = page_of(key0 + 16 * T + l16);
            next[T] = page_of(key0 + stride + 16 * T + l16);
        }
        fetch(key0, id);
        for (; key0 < end; key0 += stride) {
            const bool whole = key0 + PG_K <= end && __all(!bad);
            // scores
            vf4 sc[2];
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                sc[T] = vf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u4v kf;
                    if constexpr (I8) {
                        const u2v lo = widen4<Q>(kr[T][s >> 1][2 * (s & 1)]), hi = widen4<Q>(kr[T][s >> 1][2 * (s & 1) + 1]);
                        kf = u4v{lo[0], lo[1], hi[0], hi[1]};
                    } else {
                        kf = kr[T][s];
                    }
                    if (!EXACT && dims(s) >= hd) kf = u4v{0, 0, 0, 0};
                    sc[T] = mfma_16x16x32(Q{}, kf, qf[s], sc[T]);
                }
            }
            // V into the wave's LDS (rows past the end as zeros)
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                const int r = 16 * T + l16;
                const bool gone = !whole && (key0 + r >= end);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u4v w;
                    if constexpr (I8) {
                        const u2v lo = widen4<P>(vr[T][s >> 1][2 * (s & 1)]), hi = widen4<P>(vr[T][s >> 1][2 * (s & 1) + 1]);
                        w = u4v{lo[0], lo[1], hi[0], hi[1]};
                    } else {
                        w = vr[T][s];
                    }
                    if (gone || (!EXACT && dims(s) >= hd)) w = u4v{0, 0, 0, 0};
                    *reinterpret_cast<u4v*>(slot + r * VROW + (((dims(s) >> 3) ^ swz(r)) << 4)) = w;
                }
                if constexpr (I8) {
                    scales[r] = ksc[T];
                    scales[32 + r] = gone ? 0.0f : vsc[T];
                }
            }
            // the next tile, and the page numbers of the one after it
            if (key0 + stride < end) {
                id[0] = next[0];
                id[1] = next[1];
#pragma unroll
                for (int T = 0; T < 2; ++T) next[T] = page_of(key0 + 2 * stride + 16 * T + l16);
                fetch(key0 + stride, id);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's LDS writes, before any lane reads them
            // weights
            float mx = -INFINITY;
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                if constexpr (I8) sc[T] *= *reinterpret_cast<const vf4*>(scales + 16 * T + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!whole && key0 + 16 * T + 4 * g + i >= end) sc[T][i] = -INFINITY;
                    mx = fmaxf(mx, sc[T][i]);
                }
            }
            mx = quarter_max(mx) * sl2;
            if (__any(mx > m + RESCALE_AT)) {
                const float mn = fmaxf(m, mx);
                const float corr = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
                m = mn;
                l *= corr;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] *= corr;
            }
            const float base = m == -INFINITY ? 0.0f : m - SHIFT;
            u4v ph, pl;
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                vf4 w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[T][i], sl2, -base));
                    l += w[i];
                }
                if constexpr (I8) w *= *reinterpret_cast<const vf4*>(scales + 32 + 16 * T + 4 * g);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t u = pack2(P{}, w[2 * i], w[2 * i + 1]);
                    const f2v r = unpack2(P{}, u);
                    ph[2 * T + i] = u;
                    pl[2 * T + i] = pack2(P{}, w[2 * i] - r[0], w[2 * i + 1] - r[1]);
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const uint32_t at = slot_at + trow * VROW + (((2 * d + ((vi & 3) >> 1)) ^ swz(trow)) << 4) + 8 * (vi & 1);
                const u2v lo = lds_read_tr(at), hi = lds_read_tr(at + 16 * VROW);
                const u4v v = {lo[0], lo[1], hi[0], hi[1]};
                o[d] = mfma_16x16x32(P{}, v, ph, o[d]);
                o[d] = mfma_16x16x32(P{}, v, pl, o[d]);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads, before the next tile's writes
        }
    }
    l = quarter_sum(l);
    if (__any(bad || (a.pages == 0 && begin < end))) l = __builtin_nanf("");
    // the waves' sums meet
    float* so = reinterpret_cast<float*>(slot);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<vf4*>(so + l16 * OROW + 16 * d + 4 * g) = o[d];
    if (g == 0) {
        mls[wave][0][l16] = m;
        mls[wave][1][l16] = l;
    }
    __syncthreads();
    for (int e = tid; e < heads * hd; e += 64 * PG_WAVES) {
        const int r = e / hd, d = e - r * hd;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < PG_WAVES; ++w) M = fmaxf(M, mls[w][0][r]);
        const float base = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < PG_WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(mls[w][0][r] - base);
            L = __builtin_fmaf(f, mls[w][1][r], L);
            x = __builtin_fmaf(f, reinterpret_cast<const float*>(lds + w * SLOT)[r * OROW + d], x);
        }
        const int64_t at = (int64_t)b * a.H + h0 + r;
        if (used > 1) {
            const int64_t pt = at * a.splits + split;
            a.part_o[pt * hd + d] = x;
            if (d == 0) {
                a.part_ml[2 * pt] = M;
                a.part_ml[2 * pt + 1] = L;
            }
        } else {
            const float y = len || bad ? x / L : 0.0f;
            if (a.out_f32) static_cast<float*>(a.out)[at * hd + d] = y;
            else static_cast<typename Q::T*>(a.out)[at * hd + d] = Q::store(y);
        }
    }
}

// The chunks of one (sequence, query head) joined: one workgroup, a thread per dim, the chunks' factors in
// LDS 256 at a time.
template <class Q>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
    __shared__ float f[256], red[4];
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.x, b = blockIdx.y;
    bool over;
    int used;
    sequence_length(a, b, over, used);
    if (used <= 1) return;  // written by its one chunk
    const int64_t at = (int64_t)b * a.H + h;
    const float* ml = a.part_ml + 2 * at * a.splits;
    const float* po = a.part_o + at * a.splits * a.hd;
    float M = -INFINITY;
    for (int s = tid; s < used; s += 256) M = fmaxf(M, ml[2 * s]);
    for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    if (lane == 0) red[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, x = 0.0f;
    for (int s0 = 0; s0 < used; s0 += 256) {
        const int n = min(256, used - s0);
        __syncthreads();
        float w = 0.0f;
        if (tid < n) {
            const float e = __builtin_amdgcn_exp2f(ml[2 * (s0 + tid)] - base);
            f[tid] = e;
            w = e * ml[2 * (s0 + tid) + 1];
        }
        w = ln_wave_sum(w);
        if (lane == 0) red[tid >> 6] = w;
        __syncthreads();
        L += (red[0] + red[1]) + (red[2] + red[3]);
        if (tid < a.hd)
            for (int s = 0; s < n; ++s) x = __builtin_fmaf(f[s], po[(int64_t)(s0 + s) * a.hd + tid], x);
    }
    if (tid < a.hd) {
        const float y = x / L;
        if (a.out_f32) static_cast<float*>(a.out)[at * a.hd + tid] = y;
        else static_cast<typename Q::T*>(a.out)[at * a.hd + tid] = Q::store(y);
    }
}

// Positions of a workgroup and number of chunks: enough workgroups for the chip, whole tiles of
// every wave, and no more chunks than the bound of the lengths asks for.
struct Split {
    int chunk, splits;
};
Split plan_split(int64_t B, int64_t H, int64_t Hkv, int64_t max_length) {
    const int64_t rows = B * Hkv * ((H / Hkv + 15) / 16);
    constexpr int64_t STEP = PG_WAVES * PG_K, WANT = 2048, LEAST = 4 * STEP;
    int64_t chunk = rows > 0 ? (max_length * rows + WANT - 1) / WANT : 0;
    chunk = (chunk + STEP - 1) / STEP * STEP;
    if (chunk < LEAST) chunk = LEAST;
    if (chunk > (1 << 30)) chunk = 1 << 30;
    int64_t splits = (max_length + chunk - 1) / chunk;
    return {(int)chunk, (int)(splits < 1 ? 1 : splits)};
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

int lq_paged_kv_append(const void* d_k, const void* d_v, int src_type, int64_t ld, int64_t tokens,
                       const int32_t* d_starts, int64_t seqs, int64_t Hkv, int64_t hd, const int32_t* d_table,
                       int64_t table_stride, const int32_t* d_lengths, void* d_k_pages, void* d_v_pages,
                       int cache_type, float* d_k_scale, float* d_v_scale, int64_t pages, int64_t page,
                       void* stream) {
    LQ_REQUIRE(is_float_type(src_type), "lq_paged_kv_append: source must be float32, fp16 or bfloat16");
    LQ_REQUIRE(is_half_type(cache_type) || cache_type == LQ_I8,
               "lq_paged_kv_append: cache must be fp16, bfloat16 or int8");
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
        const dim3 one((unsigned)tokens);
        if (cache_type == LQ_I8) {
            if (vec && hd <= 64) hipLaunchKernelGGL((append_i8_kernel<8, S>), one, dim3(256), 0, st, a);
            else if (vec && hd <= 128) hipLaunchKernelGGL((append_i8_kernel<16, S>), one, dim3(256), 0, st, a);
            else if (vec && hd <= 256) hipLaunchKernelGGL((append_i8_kernel<32, S>), one, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((append_i8_any_kernel<S>), dim3((unsigned)tokens, (unsigned)(2 * Hkv)), dim3(64), 0, st, a);
            return;
        }
        with_half(cache_type, [&](auto c) {
            using C = decltype(c);
            if (!vec) hipLaunchKernelGGL((append_any_kernel<S, C>), one, dim3(256), 0, st, a);
            else if (tokens <= 4 * 1024) hipLaunchKernelGGL((append_kernel<1, S, C>), one, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((append_kernel<4, S, C>), dim3((unsigned)((tokens + 3) / 4)), dim3(256), 0, st, a);
        });
    });
    return launch_status("lq_paged_kv_append");
}

size_t lq_paged_attention_workspace_size(int64_t B, int64_t H, int64_t Hkv, int64_t hd, int64_t max_length) {
    if (B <= 0 || H <= 0 || Hkv <= 0 || hd <= 0 || max_length <= 0 || max_length > 0x7fffffff) return 0;
    const Split s = plan_split(B, H, Hkv, max_length);
    return s.splits > 1 ? (size_t)(B * H) * s.splits * (hd + 2) * sizeof(float) : 0;
}

int lq_paged_attention(const void* d_q, int q_type, int64_t ldq, int64_t B, int64_t H, int64_t Hkv, int64_t hd,
                       const void* d_k_pages, const void* d_v_pages, int cache_type, const float* d_k_scale,
                       const float* d_v_scale, int64_t pages, int64_t page, const int32_t* d_table,
                       int64_t table_stride, const int32_t* d_lengths, int64_t max_length, float scale, void* d_out,
                       int out_type, void* d_workspace, size_t workspace_bytes, void* stream) {
    LQ_REQUIRE(is_half_type(q_type), "lq_paged_attention: q must be fp16 or bfloat16");
    LQ_REQUIRE(cache_type == q_type || cache_type == LQ_I8, "lq_paged_attention: the cache must be of q's type or int8");
    LQ_REQUIRE(out_type == q_type || out_type == LQ_F32, "lq_paged_attention: out must be of q's type or float32");
    LQ_REQUIRE(B >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && hd > 0 && ldq >= H * hd && pages >= 0 && page > 0 &&
                   table_stride >= 0 && max_length >= 0 && B <= 65535 && H <= 65535 && table_stride <= 0x7fffffff &&
                   pages <= 0x7fffffff && page <= 0x7fffffff && max_length <= 0x7fffffff,
               "lq_paged_attention: bad shape");
    if (hd % 8 != 0 || hd > ATTN_MAX_HD)
        return set_error(LQ_ERR_UNSUPPORTED, "lq_paged_attention: head dim must be a multiple of 8, 256 at most");
    LQ_REQUIRE(scale > 0.0f && scale < INFINITY, "lq_paged_attention: scale must be positive and finite");
    if (B == 0) return LQ_OK;
    LQ_REQUIRE(d_q && d_lengths && d_out && (d_table || table_stride == 0) && ((d_k_pages && d_v_pages) || pages == 0),
               "lq_paged_attention: NULL pointer");
    LQ_REQUIRE(cache_type != LQ_I8 || pages == 0 || (d_k_scale && d_v_scale),
               "lq_paged_attention: an int8 cache needs scales");
    LQ_REQUIRE(aligned16(d_k_pages) && aligned16(d_v_pages), "lq_paged_attention: pages must be 16-byte aligned");
    const Split sp = plan_split(B, H, Hkv, max_length);
    LQ_REQUIRE(sp.splits == 1 || (d_workspace && workspace_bytes >=
                                      lq_paged_attention_workspace_size(B, H, Hkv, hd, max_length)),
               "lq_paged_attention: workspace too small");
    const int group = (int)(H / Hkv), qtiles = (group + 15) / 16;
    float* part_o = static_cast<float*>(d_workspace);
    const PagedArgs a{d_q, ldq, (int)B, (int)H, (int)Hkv, (int)hd, group, qtiles, d_k_pages, d_v_pages, d_k_scale,
                      d_v_scale, pages, (int)page, d_table, table_stride, d_lengths, scale, d_out, out_type == LQ_F32,
                      aligned16(d_q) && ldq % 8 == 0, sp.chunk, sp.splits, part_o, part_o ? part_o + B * H * sp.splits * hd : nullptr};
    const dim3 grid((unsigned)(Hkv * qtiles), (unsigned)B, (unsigned)sp.splits), wg(64 * PG_WAVES);
    const hipStream_t st = as_stream(stream);
    with_half(q_type, [&](auto q) {
        using Q = decltype(q);
        auto go = [&](auto w, auto exact, auto c) {
            hipLaunchKernelGGL((paged_tile_kernel<decltype(w)::value, decltype(exact)::value, Q, decltype(c)>), grid, wg,
                               0, st, a);
        };
        auto width = [&](auto c) {
            if (hd == 64) go(std::integral_constant<int, 64>{}, std::true_type{}, c);
            else if (hd == 128) go(std::integral_constant<int, 128>{}, std::true_type{}, c);
            else if (hd < 64) go(std::integral_constant<int, 64>{}, std::false_type{}, c);
            else if (hd < 128) go(std::integral_constant<int, 128>{}, std::false_type{}, c);
            else if (hd <= 192) go(std::integral_constant<int, 192>{}, std::false_type{}, c);
            else go(std::integral_constant<int, 256>{}, std::false_type{}, c);
        };
        if (cache_type == LQ_I8) width(ElemI8{});
        else width(Q{});
        if (sp.splits > 1)
            hipLaunchKernelGGL((paged_join_kernel<Q>), dim3((unsigned)H, (unsigned)B), dim3(256), 0, st, a);
    });
    return launch_status("lq_paged_attention");
}

}  // extern "C"
