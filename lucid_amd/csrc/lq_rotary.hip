// lq_rotary.hip -- queries and keys rotated by their positions, the keys and values appended to a paged cache;
// also the plain append to 4-bit pages.
//
//   (a, b) -> (a c - b s, b c + a s) for each pair of dims, angles from a float32 table by position.
//
// Every source value is read once and written once, in its new place and type; the rows of a token's angles serve all
// its heads from registers.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_paged_u4.h"
#include "lq_u4.h"

namespace lq {
namespace {

struct RotaryArgs {
    AppendArgs a;  // k, v and the cache
    const void* q;
    int64_t ldq;
    int H;
    const float* angles;
    int64_t positions;
    int rot, interleaved;
    void* qo;
    int64_t ldqo;
    void* ko;
    int64_t ldko;
};

enum { ROW_Q, ROW_K, ROW_V };

// Where a packed token goes.
struct Token {
    int64_t pos, row;  // position; row of its page (head 0), or -1
    bool turned;       // its position has angles
};
// False when it belongs to no sequence.
__device__ __forceinline__ bool find_token(const RotaryArgs& r, int64_t t, Token& k) {
    int64_t s;
    if (!token_place(t, r.a.starts, r.a.seqs, r.a.lengths, s, k.pos)) return false;
    k.turned = r.rot == 0 || (k.pos >= 0 && k.pos < r.positions);
    k.row = k.turned ? position_row(k.pos, r.a.table + s * r.a.table_stride, r.a.table_stride, r.a.pages, r.a.Hkv,
                                    r.a.page)
                     : -1;
    return true;
}

// Head h of a token's queries, keys or values.
template <class Src>
__device__ __forceinline__ const typename Src::T* source_row(const RotaryArgs& r, int64_t t, int kind, int h) {
    const void* p = kind == ROW_Q ? r.q : kind == ROW_K ? r.a.k : r.a.v;
    return static_cast<const typename Src::T*>(p) + t * (kind == ROW_Q ? r.ldq : r.a.ld) + (int64_t)h * r.a.hd;
}

// One wave per (token, head), value by value: for what 16-byte accesses do not fit.
template <class Src, class Out, class Cache>
__global__ __launch_bounds__(64) void rotary_any_kernel(RotaryArgs r) {
    const int64_t heads = r.H + 2 * r.a.Hkv, n = workgroup(), t = n / heads;
    if (t >= r.a.tokens) return;
    const int e = (int)(n - t * heads), lane = threadIdx.x, hd = (int)r.a.hd, half = r.rot / 2;
    const int kind = e < r.H ? ROW_Q : e < r.H + r.a.Hkv ? ROW_K : ROW_V;
    const int h = kind == ROW_Q ? e : kind == ROW_K ? e - r.H : e - r.H - (int)r.a.Hkv;
    Token k;
    if (!find_token(r, t, k)) return;
    const typename Src::T* x = source_row<Src>(r, t, kind, h);
    const int rot = kind == ROW_V ? 0 : r.rot;
    const float* cs = r.angles + (k.turned ? k.pos : 0) * r.rot;
    auto first = [&](int i) { return r.interleaved ? 2 * i : i; };
    auto second = [&](int i) { return r.interleaved ? 2 * i + 1 : i + half; };
    auto value = [&](int d) {
        const float u = Src::load(x[d]);
        if (d >= rot) return u;
        const bool is_b = r.interleaved ? (d & 1) : d >= half;
        const int i = r.interleaved ? d >> 1 : is_b ? d - half : d;
        const float w = Src::load(x[is_b ? first(i) : second(i)]), c = cs[i], s = cs[half + i];
        return is_b ? u * c + w * s : u * c - w * s;
    };
    if (kind != ROW_Q && k.row >= 0) {
        const int64_t row = k.row + h * r.a.page;
        void* pages = kind == ROW_K ? r.a.kp : r.a.vp;
        if constexpr (std::is_same_v<Cache, ElemI8>) {
            int32_t top = 0;
            for (int d = lane; d < hd; d += 64) top = max(top, magnitude(value(d)));
            const RowScale rs(wave_max(top));
            for (int d = lane; d < hd; d += 64) static_cast<int8_t*>(pages)[row * hd + d] = (int8_t)rs.code(value(d));
            if (lane == 0) static_cast<float*>(kind == ROW_K ? r.a.ks : r.a.vs)[row] = rs.scale;
        } else if constexpr (std::is_same_v<Cache, void>) {
            const int step = kind == ROW_K ? U4_GROUP : hd, groups = hd / step;
            uint16_t* meta = static_cast<uint16_t*>(kind == ROW_K ? r.a.ks : r.a.vs) + row * 2 * groups;
            for (int g = 0; g < groups; ++g) {
                float lo = INFINITY, hi = -INFINITY;
                for (int d = g * step + lane; d < (g + 1) * step; d += 64) {
                    const float v = value(d);
                    lo = fminf(lo, v);
                    hi = fabsf(v) < INFINITY ? fmaxf(hi, v) : INFINITY;
                }
                const Group4 q(-unkey(wave_max(fkey(-lo))), unkey(wave_max(fkey(hi))));
                if (lane == 0) {
                    meta[g] = f32_to_bf16_bits(q.scale);
                    meta[groups + g] = f32_to_bf16_bits(q.bias);
                }
                uint8_t* to = static_cast<uint8_t*>(pages) + row * (hd / 2);
                for (int b = g * step / 2 + lane; b < (g + 1) * step / 2; b += 64)
                    to[b] = (uint8_t)(q.code(value(2 * b)) | q.code(value(2 * b + 1)) << 4);
            }
        } else {
            for (int d = lane; d < hd; d += 64)
                static_cast<typename Cache::T*>(pages)[row * hd + d] = Cache::store(value(d));
        }
    }
    // the rotated rows last, a pair to a lane: they may lie in the source's place
    void* out = kind == ROW_Q ? r.qo : kind == ROW_K ? r.ko : nullptr;
    if (!out) return;
    typename Out::T* y = static_cast<typename Out::T*>(out) + t * (kind == ROW_Q ? r.ldqo : r.ldko) + (int64_t)h * hd;
    const float nan = __builtin_nanf("");
    for (int i = lane; i < half; i += 64) {
        const int p = first(i), q = second(i);
        const float u = Src::load(x[p]), w = Src::load(x[q]), c = k.turned ? cs[i] : nan, s = k.turned ? cs[half + i] : nan;
        y[p] = Out::store(u * c - w * s);
        y[q] = Out::store(w * c + u * s);
    }
    for (int d = rot + lane; d < hd; d += 64) y[d] = Out::store(k.turned ? Src::load(x[d]) : nan);
}

// Eight source values as they lie in memory.
template <class Src>
struct Raw8 {
    static constexpr int N = Src::code == LQ_F32 ? 8 : 4;
    uint32_t w[N];
    __device__ __forceinline__ void load(const typename Src::T* p) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u4v v = __builtin_nontemporal_load(reinterpret_cast<const u4v*>(p) + i / 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i + j] = v[j];
        }
    }
    __device__ __forceinline__ void unpack(float (&x)[8]) const {
        if constexpr (Src::code == LQ_F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __uint_as_float(w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f2v u = unpack2(Src{}, w[j]);
                x[2 * j] = u[0];
                x[2 * j + 1] = u[1];
            }
        }
    }
    __device__ __forceinline__ Raw8 of_lane_xor(int m) const {
        Raw8 r;
#pragma unroll
        for (int j = 0; j < N; ++j) r.w[j] = (uint32_t)__shfl_xor((int)w[j], m, 64);
        return r;
    }
};

// A workgroup takes AHEAD rows of a token a lane, lpr lanes (8, 16 or 32) to a row of hd <= 8 lpr values, eight values
// a lane.  A lane keeps its place in the row for every head, so the angles of its dims are loaded once.  The values are on
// their way before the token's place is looked up (a search, two numbers, a page number and the angles, each
// after the other).  swap: the lane whose place holds the partners differs by this bit; 0: the partners are loaded.
// Bound by HBM: 20452 tokens of 32 + 2 * 8 heads of 128 in bfloat16 106 us, 4.8 TB/s read and written, what a copy
// reaches (one row a lane in workgroups of 256: 133, with the partners loaded 168).
constexpr int RT_T = 64;  // threads; 128 or 256 of them, four rows a lane: 136 and 118 us
// Rows of a call from which a lane takes four: the loads of one hide nothing of the places' latency.  One / four rows a
// lane: 49152 rows alike, 98304 rows 13.7 / 10.6 us.
constexpr int64_t RT_ROWS = 1 << 16;
template <int AHEAD, class Src, class Out, class Cache>
__global__ __launch_bounds__(RT_T) void rotary_kernel(RotaryArgs r, int lpr, int swap, uint32_t groups) {
    const int64_t n = workgroup(), t = n / groups;
    if (t >= r.a.tokens) return;
    const int hd = (int)r.a.hd, half = r.rot / 2, Hkv = (int)r.a.Hkv, heads = r.H + 2 * Hkv;
    const int d = (threadIdx.x & (lpr - 1)) * 8;
    const int other = r.interleaved || d >= r.rot ? d : d < half ? d + half : d - half;  // the partners' dims
    auto kind_of = [&](int e) { return e < r.H ? ROW_Q : e < r.H + Hkv ? ROW_K : ROW_V; };
    auto head_of = [&](int e) { return e < r.H ? e : e < r.H + Hkv ? e - r.H : e - r.H - Hkv; };
    // rows e0 + i * round; those past the last are nobody's, but take part in the exchanges
    const int round = blockDim.x / lpr, e0 = (int)(n - t * groups) * AHEAD * round + threadIdx.x / lpr;
    Raw8<Src> raw[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        const int e = e0 + i * round;
#pragma unroll
        for (int j = 0; j < Raw8<Src>::N; ++j) raw[i].w[j] = 0;
        if (e < heads && d < hd) raw[i].load(source_row<Src>(r, t, kind_of(e), head_of(e)) + d);
    }
    Token k;
    if (!find_token(r, t, k)) return;
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        c[j] = 1.0f;
        s[j] = 0.0f;
    }
    if (d < r.rot && k.turned) {
        const float* cs = r.angles + k.pos * r.rot;
        if (r.interleaved) {
            const vf4 u = *reinterpret_cast<const vf4*>(cs + d / 2), w = *reinterpret_cast<const vf4*>(cs + half + d / 2);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                c[j] = u[j >> 1];
                s[j] = j & 1 ? w[j >> 1] : -w[j >> 1];
            }
        } else {
            const float* p = cs + (d < half ? d : d - half);
            const float sign = d < half ? -1.0f : 1.0f;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const vf4 u = *reinterpret_cast<const vf4*>(p + j), w = *reinterpret_cast<const vf4*>(p + half + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[j + i] = u[i];
                    s[j + i] = sign * w[i];
                }
            }
        }
    }
    auto row_of = [&](int e, const Raw8<Src>& in) __attribute__((always_inline)) {
        const int kind = kind_of(e), h = head_of(e);
        const bool mine = e < heads && d < hd;
        float x[8], y[8];
        in.unpack(x);
        if (r.interleaved) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = x[j ^ 1];
        } else if (swap) {
            in.of_lane_xor(swap).unpack(y);
        } else if (mine && kind != ROW_V) {
            Raw8<Src> p;
            p.load(source_row<Src>(r, t, kind, h) + other);
            p.unpack(y);
        }
        // a c - b s, and b c + a s: the sign is in s
        if (kind != ROW_V && d < r.rot) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * c[j] + y[j] * s[j];
        }
        if (mine && kind != ROW_V) {
            void* out = kind == ROW_Q ? r.qo : r.ko;
            if (out) {
                const int64_t at = t * (kind == ROW_Q ? r.ldqo : r.ldko) + (int64_t)h * hd + d;
                u4v o;
                const float nan = __builtin_nanf("");
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[j] = pack2(Out{}, k.turned ? x[2 * j] : nan, k.turned ? x[2 * j + 1] : nan);
                __builtin_nontemporal_store(o, reinterpret_cast<u4v*>(static_cast<typename Out::T*>(out) + at));
            }
        }
        const bool keep = mine && kind != ROW_Q && k.row >= 0;
        const int64_t row = k.row + (int64_t)h * r.a.page;
        void* pages = kind == ROW_K ? r.a.kp : r.a.vp;
        if constexpr (std::is_same_v<Cache, ElemI8>) {
            int32_t top = 0;
            if (mine) {
#pragma unroll
                for (int j = 0; j < 8; ++j) top = max(top, magnitude(x[j]));
            }
            for (int off = lpr / 2; off > 0; off >>= 1) top = max(top, __shfl_xor(top, off, 64));
            const RowScale rs(top);
            if (!keep) return;
            u2v w = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j >> 2] |= (uint32_t)(rs.code(x[j]) & 0xff) << (8 * (j & 3));
            *reinterpret_cast<u2v*>(static_cast<int8_t*>(pages) + row * hd + d) = w;
            if (d == 0) static_cast<float*>(kind == ROW_K ? r.a.ks : r.a.vs)[row] = rs.scale;
        } else if constexpr (std::is_same_v<Cache, void>) {
            float lo = INFINITY, hi = -INFINITY;
            if (mine) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    lo = fminf(lo, x[j]);
                    hi = fabsf(x[j]) < INFINITY ? fmaxf(hi, x[j]) : INFINITY;
                }
            }
            // the four lanes of a key's group, all lanes of a value's row; the rows of a wave may be of both kinds
            for (int off = 1; off < lpr; off <<= 1) {
                const float ol = __shfl_xor(lo, off, 64), oh = __shfl_xor(hi, off, 64);
                if (off < U4_GROUP / 8 || kind == ROW_V) {
                    lo = fminf(lo, ol);
                    hi = fmaxf(hi, oh);
                }
            }
            if (!keep) return;
            const Group4 q(lo, hi);
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) w |= q.code(x[j]) << (4 * j);
            reinterpret_cast<uint32_t*>(pages)[(row * hd + d) / 8] = w;
            const int groups = kind == ROW_K ? hd / U4_GROUP : 1;
            if (kind == ROW_K ? d % U4_GROUP == 0 : d == 0) {
                uint16_t* meta = static_cast<uint16_t*>(kind == ROW_K ? r.a.ks : r.a.vs) + row * 2 * groups +
                                 (kind == ROW_K ? d / U4_GROUP : 0);
                meta[0] = f32_to_bf16_bits(q.scale);
                meta[groups] = f32_to_bf16_bits(q.bias);
            }
        } else {
            if (!keep) return;
            u4v o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = pack2(Cache{}, x[2 * j], x[2 * j + 1]);
            *reinterpret_cast<u4v*>(static_cast<typename Cache::T*>(pages) + row * hd + d) = o;
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) row_of(e0 + i * round, raw[i]);
}

}  // namespace

int paged_append_rotary(const char* name, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv,
                        int src_type, int64_t tokens, const int32_t* starts, int64_t seqs, int64_t H, int64_t Hkv,
                        int64_t hd, const float* angles, int64_t positions, int64_t rot, int interleaved,
                        const int32_t* table, int64_t table_stride, const int32_t* lengths, void* q_out, int64_t ldqo,
                        void* k_out, int64_t ldko, int q_type, void* k_pages, void* v_pages, int cache_type,
                        void* k_scale, void* v_scale, int64_t pages, int64_t page, void* stream) {
    const std::string n = std::string(name) + ": ";
    LQ_REQUIRE(is_float_type(src_type), n + "source must be float32, fp16 or bfloat16");
    LQ_REQUIRE(is_half_type(q_type), n + "rotated rows must be fp16 or bfloat16");
    LQ_REQUIRE(cache_type == q_type || cache_type == LQ_I8 || cache_type == LQ_U4,
               n + "cache must be of the rotated rows' type, int8 or 4 bits");
    LQ_REQUIRE(tokens >= 0 && seqs >= 0 && H >= 0 && Hkv > 0 && hd > 0 && H <= 65535 && Hkv <= 65535 &&
                   ldkv >= Hkv * hd && (H == 0 || (ldq >= H * hd && ldqo >= H * hd)) && (!k_out || ldko >= Hkv * hd) &&
                   table_stride >= 0 && pages >= 0 && page > 0 && positions >= 0 && tokens <= 0x7fffffff &&
                   seqs <= 0x7fffffff && table_stride <= 0x7fffffff && pages <= 0x7fffffff && page <= 0x7fffffff,
               n + "bad shape");
    LQ_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= hd, n + "rotated dims must be even and within the head");
    if (hd > ATTN_MAX_HD) return set_error(LQ_ERR_UNSUPPORTED, n + "head dim above 256");
    if (cache_type == LQ_U4 && hd % U4_GROUP != 0)
        return set_error(LQ_ERR_UNSUPPORTED, n + "head dims of a 4-bit cache are multiples of 32");
    LQ_REQUIRE(starts || tokens == seqs, n + "without starts there is one token per sequence");
    if (tokens == 0 || seqs == 0) return LQ_OK;
    const bool stored = table_stride > 0 && pages > 0;  // else the rotation alone
    if (!stored && H == 0 && !k_out) return LQ_OK;
    LQ_REQUIRE(k && v && lengths && (H == 0 || (q && q_out)) && (rot == 0 || positions == 0 || angles) &&
                   (!stored || (table && k_pages && v_pages)),
               n + "NULL pointer");
    LQ_REQUIRE(!stored || is_half_type(cache_type) || (k_scale && v_scale), n + "a cache of codes needs scales");
    LQ_REQUIRE(cache_type != LQ_U4 || ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 3) == 0,
               n + "4-bit pages must be 4-byte aligned");
    LQ_REQUIRE((q_out != q || H == 0 || (q_type == src_type && ldqo == ldq)) &&
                   (!k_out || k_out != k || (q_type == src_type && ldko == ldkv)),
               n + "rotation in place needs equal types and strides");
    LQ_REQUIRE(!k_out || k_out != v, n + "the rotated keys cannot take the values' place");
    const RotaryArgs r{{k, v, ldkv, tokens, starts, seqs, Hkv, hd, table, stored ? table_stride : 0, lengths, k_pages,
                        v_pages, k_scale, v_scale, pages, page},
                       q, ldq, (int)H, angles, positions, (int)rot, interleaved != 0, q_out, ldqo, k_out, ldko};
    const hipStream_t st = as_stream(stream);
    // eight values at a time: their partners are eight values too, every base and row 16-byte aligned
    const int64_t se = elem_size(src_type);
    const uintptr_t ends = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                           reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                           reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(angles) |
                           (H ? reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) : 0);
    const int64_t strides = ldkv * se | (H ? ldq * se | ldqo * 2 : 0) | (k_out ? ldko * 2 : 0);
    const bool vec = hd % 8 == 0 && rot % (interleaved ? 8 : 16) == 0 && (ends & 15) == 0 && (strides & 15) == 0;
    const int64_t heads = H + 2 * Hkv;
    const int lpr = hd <= 64 ? 8 : hd <= 128 ? 16 : 32;
    const int64_t apart = rot / 16;  // lanes between partners: an exchange where that is a power of two
    const int swap = !interleaved && rot > 0 && (apart & (apart - 1)) == 0 ? (int)apart : 0;
    const bool few = tokens * heads < RT_ROWS;
    note_path(!vec ? "rotary single" : few ? "rotary" : "rotary four rows");
    with_float(src_type, [&](auto s) {
        using S = decltype(s);
        with_half(q_type, [&](auto o) {
            using O = decltype(o);
            auto go = [&](auto one, auto four, auto ak) {
                if (!vec) {
                    hipLaunchKernelGGL(ak, grid_of(tokens * heads), dim3(64), 0, st, r);
                    return;
                }
                const int64_t each = RT_T / lpr * (few ? 1 : 4), groups = (heads + each - 1) / each;
                const dim3 grid = grid_of(tokens * groups);
                if (few) hipLaunchKernelGGL(one, grid, dim3(RT_T), 0, st, r, lpr, swap, (uint32_t)groups);
                else hipLaunchKernelGGL(four, grid, dim3(RT_T), 0, st, r, lpr, swap, (uint32_t)groups);
            };
            if (cache_type == LQ_I8) go(rotary_kernel<1, S, O, ElemI8>, rotary_kernel<4, S, O, ElemI8>, rotary_any_kernel<S, O, ElemI8>);
            else if (cache_type == LQ_U4) go(rotary_kernel<1, S, O, void>, rotary_kernel<4, S, O, void>, rotary_any_kernel<S, O, void>);
            else go(rotary_kernel<1, S, O, O>, rotary_kernel<4, S, O, O>, rotary_any_kernel<S, O, O>);
        });
    });
    return launch_status(name);
}

}  // namespace lq

using namespace lq;

extern "C" {

int lq_paged_kv_append_rotary(const void* d_q, int64_t ldq, const void* d_k, const void* d_v, int64_t ldkv,
                              int src_type, int64_t tokens, const int32_t* d_starts, int64_t seqs, int64_t H,
                              int64_t Hkv, int64_t hd, const float* d_angles, int64_t positions, int64_t rot,
                              int interleaved, const int32_t* d_table, int64_t table_stride, const int32_t* d_lengths,
                              void* d_q_out, int64_t ldqo, void* d_k_out, int64_t ldko, int q_type, void* d_k_pages,
                              void* d_v_pages, int cache_type, void* d_k_scale, void* d_v_scale, int64_t pages,
                              int64_t page, void* stream) {
    return paged_append_rotary("lq_paged_kv_append_rotary", d_q, ldq, d_k, d_v, ldkv, src_type, tokens, d_starts, seqs,
                               H, Hkv, hd, d_angles, positions, rot, interleaved, d_table, table_stride, d_lengths,
                               d_q_out, ldqo, d_k_out, ldko, q_type, d_k_pages, d_v_pages, cache_type, d_k_scale,
                               d_v_scale, pages, page, stream);
}

}  // extern "C"
