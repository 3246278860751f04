// lq_prompt.hip -- attention over packed prompts of different lengths, with grouped heads.
//
// Sequence s owns rows q_starts[s] .. q_starts[s + 1] - 1 of q and k_starts[s] .. of k / v.  With
// `causal`, query i of nq sees keys 0 .. nk - nq + i (the queries are the last nq of nk
// positions); a query that sees no key has the output 0.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_attn.h"
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

// One workgroup per (head, query), 256 keys at a time: the simplest form.
template <class E, class Out>
__global__ __launch_bounds__(256) void prompt_rows_kernel(PromptArgs a) {
    __shared__ float qv[ATTN_MAX_HD];
    __shared__ float p[256];
    __shared__ float red[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t h = blockIdx.x, t = blockIdx.y + (int64_t)blockIdx.z * 65535, hk = h / (a.H / a.Hkv);
    if (t >= a.total_q) return;
    const int hd = (int)a.hd;
    const int64_t sq = sequence_of(a.qs, a.seqs, t);
    const Packed pk = packed_sequence(a.qs, a.ks, sq, a.total_q, a.total_k);
    if (t < pk.q0 || t >= pk.q0 + pk.nq) return;
    const int64_t k0 = pk.k0, len = keys_seen(pk, t - pk.q0, a.causal);
    if (tid < hd) qv[tid] = E::load(static_cast<const typename E::T*>(a.q)[t * a.ldq + h * hd + tid]);
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int64_t kb = 0; kb < len; kb += 256) {
        __syncthreads();
        const int64_t key = kb + tid;
        float s = -INFINITY;
        if (key < len) {
            const typename E::T* kr = static_cast<const typename E::T*>(a.k) + (k0 + key) * a.ldk + hk * hd;
            s = 0.0f;
            for (int d = 0; d < hd; ++d) s = __builtin_fmaf(qv[d], E::load(kr[d]), s);
            s *= a.scale * LOG2E;
        }
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
            const int n = (int)min((int64_t)256, len - kb);
            const typename E::T* vr = static_cast<const typename E::T*>(a.v) + (k0 + kb) * a.ldv + hk * hd + tid;
            for (int j = 0; j < n; ++j) acc = __builtin_fmaf(p[j], E::load(vr[j * a.ldv]), acc);
        }
    }
    if (tid < hd) static_cast<typename Out::T*>(a.out)[(t * a.H + h) * hd + tid] = Out::store(len ? acc / l : 0.0f);
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
    const dim3 grid((unsigned)H, (unsigned)(total_q < 65535 ? total_q : 65535), (unsigned)((total_q + 65534) / 65535));
    with_half(type, [&](auto e) {
        using E = decltype(e);
        if (out_type == LQ_F32)
            hipLaunchKernelGGL((prompt_rows_kernel<E, ElemF32>), grid, dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL((prompt_rows_kernel<E, E>), grid, dim3(256), 0, st, a);
    });
    return launch_status("lq_prompt_attention");
}

}  // extern "C"
