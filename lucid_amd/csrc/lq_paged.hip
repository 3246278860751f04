// lq_paged.hip -- a key-value cache in pages: appending new tokens' keys and values, and the
// attention of one new token per sequence over its pages.
//
// Layout.  k / v pages [pages][Hkv][page][hd] (fp16, bfloat16, or int8 codes with one float32
// scale per row in [pages][Hkv][page]); table [seqs][table_stride] of page numbers; position p
// of sequence s is slot p % page of page table[s][p / page].  A head's rows of one page lie next
// to each other, so the attention of a head streams page * hd contiguous values.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

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

// One thread per value: the simplest form.
template <class Src, class Dst>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
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

// int8 rows: one wave per (token, head, k or v).  scale = max|x| / 127, code = rne(x * (127 /
// max|x|)); a row whose largest magnitude is below 127 / FLT_MAX (or 0) is stored as zeros; one
// that holds an infinity or NaN gets a scale that is not finite, so that it reads back as NaN.
template <class Src>
__global__ __launch_bounds__(64) void append_i8_kernel(AppendArgs a) {
    const int64_t t = blockIdx.x;
    const int64_t row = token_row(a, t);
    if (row < 0) return;
    const int h = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const typename Src::T* src = static_cast<const typename Src::T*>(is_v ? a.v : a.k) + t * a.ld + h * a.hd;
    const int64_t r = row + h * a.page;
    int32_t top = 0;  // integer order of |x| bits; NaN above infinity
    for (int64_t d = threadIdx.x; d < a.hd; d += 64)
        top = max(top, __builtin_bit_cast(int32_t, Src::load(src[d])) & 0x7fffffff);
    top = wave_max(top);
    const float amax = __builtin_bit_cast(float, top);
    const float inv = 127.0f / amax;
    const bool zero = !(inv < INFINITY) && amax == amax;
    int8_t* dst = static_cast<int8_t*>(is_v ? a.vp : a.kp) + r * a.hd;
    for (int64_t d = threadIdx.x; d < a.hd; d += 64) {
        const float c = rne(Src::load(src[d]) * inv);
        dst[d] = zero || c != c ? 0 : (int8_t)fminf(fmaxf(c, -127.0f), 127.0f);
    }
    if (threadIdx.x == 0) (is_v ? a.vs : a.ks)[r] = zero ? 0.0f : amax / 127.0f;
}

// ------------------------------------------------------------------------------ attention

struct PagedArgs {
    const void* q;
    int64_t ldq, B, H, Hkv, hd;
    const void *k, *v;
    const float *ks, *vs;
    int64_t pages, page;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    float scale;
    void* out;
};

// One workgroup per (head, sequence), 256 keys at a time: a thread scores one key, then a
// thread per dim adds the weighted values.
template <class Q, class Kv, class Out>
__global__ __launch_bounds__(256) void paged_rows_kernel(PagedArgs a) {
    __shared__ float qs[ATTN_MAX_HD];
    __shared__ float p[256];
    __shared__ int64_t rows[256];
    __shared__ float red[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t h = blockIdx.x, b = blockIdx.y, hk = h / (a.H / a.Hkv);
    const int hd = (int)a.hd;
    if (tid < hd) qs[tid] = Q::load(static_cast<const typename Q::T*>(a.q)[b * a.ldq + h * hd + tid]);
    const int64_t len = max(a.lengths[b], 0);
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int64_t k0 = 0; k0 < len; k0 += 256) {
        __syncthreads();
        const int64_t key = k0 + tid;
        float s = -INFINITY;
        if (key < len) {
            const int64_t r0 = position_row(key, a.table + b * a.table_stride, a.table_stride, a.pages, a.Hkv, a.page);
            const int64_t r = r0 < 0 ? -1 : r0 + hk * a.page;
            rows[tid] = r;
            s = __builtin_nanf("");
            if (r >= 0) {
                const typename Kv::T* kr = static_cast<const typename Kv::T*>(a.k) + r * hd;
                s = 0.0f;
                for (int d = 0; d < hd; ++d) s = __builtin_fmaf(qs[d], Kv::load(kr[d]), s);
                if (Kv::code == LQ_I8) s *= a.ks[r];
                s *= a.scale * LOG2E;
            }
        }
        // the block's maximum (a NaN stays in its own weight and reaches the sum)
        float mb = s;
        for (int off = 32; off > 0; off >>= 1) mb = fmaxf(mb, __shfl_xor(mb, off, 64));
        if (lane == 0) red[wave] = mb;
        __syncthreads();
        mb = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = fmaxf(m, mb);
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float e = key < len ? __builtin_amdgcn_exp2f(s - base) : 0.0f;
        const float corr = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        p[tid] = e;
        float sum = e;
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if (lane == 0) red[4 + wave] = sum;
        __syncthreads();
        l = l * corr + (red[4] + red[5] + red[6] + red[7]);
        acc *= corr;
        if (tid < hd) {
            const int n = (int)min((int64_t)256, len - k0);
            for (int j = 0; j < n; ++j) {
                const int64_t r = rows[j];
                if (r < 0) continue;
                float v = Kv::load(static_cast<const typename Kv::T*>(a.v)[r * hd + tid]);
                if (Kv::code == LQ_I8) v *= a.vs[r];
                acc = __builtin_fmaf(p[j], v, acc);
            }
        }
    }
    if (tid < hd)
        static_cast<typename Out::T*>(a.out)[(b * a.H + h) * hd + tid] = Out::store(len ? acc / l : 0.0f);
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
    with_float(src_type, [&](auto s) {
        using S = decltype(s);
        if (cache_type == LQ_I8) {
            hipLaunchKernelGGL((append_i8_kernel<S>), dim3((unsigned)tokens, (unsigned)(2 * Hkv)), dim3(64), 0, st, a);
        } else {
            with_half(cache_type, [&](auto c) {
                hipLaunchKernelGGL((append_kernel<S, decltype(c)>), dim3((unsigned)tokens), dim3(256), 0, st, a);
            });
        }
    });
    return launch_status("lq_paged_kv_append");
}

size_t lq_paged_attention_workspace_size(int64_t B, int64_t H, int64_t Hkv, int64_t hd, int64_t max_length) {
    (void)B, (void)H, (void)Hkv, (void)hd, (void)max_length;
    return 0;
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
                   pages <= 0x7fffffff && page <= 0x7fffffff,
               "lq_paged_attention: bad shape");
    if (hd % 8 != 0 || hd > ATTN_MAX_HD)
        return set_error(LQ_ERR_UNSUPPORTED, "lq_paged_attention: head dim must be a multiple of 8, 256 at most");
    LQ_REQUIRE(scale > 0.0f && scale < INFINITY, "lq_paged_attention: scale must be positive and finite");
    if (B == 0) return LQ_OK;
    LQ_REQUIRE(d_q && d_lengths && d_out && (d_table || table_stride == 0) && ((d_k_pages && d_v_pages) || pages == 0),
               "lq_paged_attention: NULL pointer");
    LQ_REQUIRE(cache_type != LQ_I8 || pages == 0 || (d_k_scale && d_v_scale),
               "lq_paged_attention: an int8 cache needs scales");
    const PagedArgs a{d_q, ldq, B, H, Hkv, hd, d_k_pages, d_v_pages, d_k_scale, d_v_scale, pages, page, d_table,
                      table_stride, d_lengths, scale, d_out};
    const dim3 grid((unsigned)H, (unsigned)B);
    const hipStream_t st = as_stream(stream);
    with_half(q_type, [&](auto q) {
        using Q = decltype(q);
        auto go = [&](auto kv, auto o) {
            hipLaunchKernelGGL((paged_rows_kernel<Q, decltype(kv), decltype(o)>), grid, dim3(256), 0, st, a);
        };
        if (cache_type == LQ_I8 && out_type == LQ_F32) go(ElemI8{}, ElemF32{});
        else if (cache_type == LQ_I8) go(ElemI8{}, Q{});
        else if (out_type == LQ_F32) go(Q{}, ElemF32{});
        else go(Q{}, Q{});
    });
    return launch_status("lq_paged_attention");
}

}  // extern "C"
