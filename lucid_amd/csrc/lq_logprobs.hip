// lq_logprobs.hip -- log probabilities of given tokens under rows of logits, the rows' entropy and
// best alternatives, and the gradient of the first two in the logits.
//
//   lse = m + log sum_j e^(x_j - m),  m = max_j x_j        logprob = x_t - lse
//   entropy = -sum_j p_j log p_j = log S - (sum_j e^(d_j) d_j) / S,  d_j = x_j - m,  S = sum_j e^(d_j)
//   grad_j = g (1[j = t] - p_j) - ge p_j (log p_j + entropy),  p_j = e^(x_j - lse)
//
// A logit of -inf is a token that is not allowed: it has probability 0 and adds nothing to the
// entropy or the gradient.  A row that allows none has lse = -inf, log probabilities of -inf,
// entropy 0 and gradient 0.  A target outside [0, vocab) carries no loss: log probability 0 and
// no gradient through it.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_attn.h"

namespace lq {
namespace {

constexpr int LP_MAX_TOP = 64;

struct LogprobArgs {
    const void* x;
    int64_t ldx, rows, vocab;
    const int32_t* targets;
    int top;
    float *logprobs, *entropy, *lse, *top_logprobs;
    int32_t* top_ids;
};

// Order of alternatives as one integer: larger values first (NaN above everything, -0 equal to
// +0), then lower indices.  0 is below every candidate's key.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t index) {
    uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    u = v != v ? 0xfffffffeu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return ((uint64_t)u << 32) | (uint32_t)~index;
}
__device__ __forceinline__ uint32_t rank_index(uint64_t key) { return ~(uint32_t)key; }

// Log probability of a logit: -inf stays -inf in a row that allows nothing.
__device__ __forceinline__ float logprob_of(float x, float lse) { return x == -INFINITY && lse == lse ? x : x - lse; }

// One workgroup per row: the maximum, the sums, then one scan per alternative.
template <class E>
__global__ __launch_bounds__(256) void logprobs_rows_kernel(LogprobArgs a) {
    __shared__ float red[2][4];
    __shared__ uint64_t best[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x;
    const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ldx;
    float m = -INFINITY;
    for (int64_t j = tid; j < a.vocab; j += 256) m = fmaxf(m, E::load(x[j]));
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    __syncthreads();
    const float base = m == -INFINITY ? 0.0f : m;
    float s = 0.0f, ed = 0.0f;
    for (int64_t j = tid; j < a.vocab; j += 256) {
        const float d = E::load(x[j]) - base, e = __builtin_amdgcn_exp2f(d * LOG2E);
        s += e;
        ed = __builtin_fmaf(e, fmaxf(d, -1e4f), ed);
    }
    for (int off = 32; off > 0; off >>= 1) {
        s += __shfl_xor(s, off, 64);
        ed += __shfl_xor(ed, off, 64);
    }
    if (lane == 0) {
        red[0][wave] = s;
        red[1][wave] = ed;
    }
    __syncthreads();
    s = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    ed = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const float log_s = logf(s), lse = base + log_s;  // -inf for a row that allows nothing
    if (tid == 0) {
        if (a.lse) a.lse[r] = lse;
        if (a.entropy) a.entropy[r] = s == 0.0f ? 0.0f : log_s - ed / s;
        if (a.logprobs) {
            const int64_t t = a.targets[r];
            a.logprobs[r] = t >= 0 && t < a.vocab ? logprob_of(E::load(x[t]), lse) : 0.0f;
        }
    }
    uint64_t last = ~(uint64_t)0;
    for (int k = 0; k < a.top; ++k) {
        uint64_t b = 0;
        for (int64_t j = tid; j < a.vocab; j += 256) {
            const uint64_t key = rank_key(E::load(x[j]), (uint32_t)j);
            if (key < last && key > b) b = key;
        }
        for (int off = 32; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor(b, off, 64);
            b = o > b ? o : b;
        }
        if (lane == 0) best[wave] = b;
        __syncthreads();
        for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
        __syncthreads();
        last = b;
        if (tid == 0) {
            const int64_t j = rank_index(b);
            a.top_ids[r * a.top + k] = (int32_t)j;
            a.top_logprobs[r * a.top + k] = logprob_of(E::load(x[j]), lse);
        }
    }
}

struct LogprobGradArgs {
    const void* x;
    int64_t ldx, rows, vocab;
    const int32_t* targets;
    const float *lse, *entropy, *g_logprobs, *g_entropy;
    void* grad;
    int64_t ldg;
};

template <class E>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogprobGradArgs a) {
    const int64_t r = blockIdx.x;
    const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ldx;
    typename E::T* y = static_cast<typename E::T*>(a.grad) + r * a.ldg;
    const int64_t t = a.targets[r];
    const bool given = t >= 0 && t < a.vocab;
    const float g = given ? a.g_logprobs[r] : 0.0f, lse = a.lse[r];
    const float ge = a.g_entropy ? a.g_entropy[r] : 0.0f, H = a.g_entropy ? a.entropy[r] : 0.0f;
    const bool none = lse == -INFINITY;
    for (int64_t j = threadIdx.x; j < a.vocab; j += 256) {
        const float lp = E::load(x[j]) - lse, p = none ? 0.0f : __builtin_amdgcn_exp2f(lp * LOG2E);
        const float w = g + ge * (fmaxf(lp, -1e4f) + H);
        const float hot = !none && given && j == t ? g : 0.0f;
        y[j] = E::store(hot - p * w);
    }
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

size_t lq_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int64_t top) {
    (void)rows, (void)vocab, (void)top;
    return 0;
}

int lq_token_logprobs(const void* d_x, int type, int64_t ldx, int64_t rows, int64_t vocab, const int32_t* d_targets,
                      int64_t top, float* d_logprobs, float* d_entropy, float* d_lse, float* d_top_logprobs,
                      int32_t* d_top_ids, void* d_workspace, size_t workspace_bytes, void* stream) {
    LQ_REQUIRE(is_float_type(type), "lq_token_logprobs: logits must be float32, fp16 or bfloat16");
    LQ_REQUIRE(rows >= 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= 0x7fffffff && ldx >= vocab,
               "lq_token_logprobs: bad shape");
    LQ_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab,
               "lq_token_logprobs: at most 64 alternatives, and no more than the vocabulary holds");
    if (rows == 0) return LQ_OK;
    LQ_REQUIRE(d_x && (d_targets || !d_logprobs) && (top == 0 || (d_top_logprobs && d_top_ids)),
               "lq_token_logprobs: NULL pointer");
    const LogprobArgs a{d_x, ldx, rows, vocab, d_targets, (int)top, d_logprobs, d_entropy, d_lse, d_top_logprobs,
                        d_top_ids};
    with_float(type, [&](auto e) {
        hipLaunchKernelGGL((logprobs_rows_kernel<decltype(e)>), dim3((unsigned)rows), dim3(256), 0, as_stream(stream),
                           a);
    });
    return launch_status("lq_token_logprobs");
}

int lq_token_logprobs_backward(const void* d_x, int type, int64_t ldx, int64_t rows, int64_t vocab,
                               const int32_t* d_targets, const float* d_lse, const float* d_entropy,
                               const float* d_g_logprobs, const float* d_g_entropy, void* d_grad, int64_t ldg,
                               void* stream) {
    LQ_REQUIRE(is_float_type(type), "lq_token_logprobs_backward: logits must be float32, fp16 or bfloat16");
    LQ_REQUIRE(rows >= 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= 0x7fffffff && ldx >= vocab && ldg >= vocab,
               "lq_token_logprobs_backward: bad shape");
    if (rows == 0) return LQ_OK;
    LQ_REQUIRE(d_x && d_targets && d_lse && d_g_logprobs && d_grad && (d_entropy || !d_g_entropy),
               "lq_token_logprobs_backward: NULL pointer");
    LQ_REQUIRE(d_grad != d_x || ldg == ldx, "lq_token_logprobs_backward: in place needs equal strides");
    const LogprobGradArgs a{d_x, ldx, rows, vocab, d_targets, d_lse, d_entropy, d_g_logprobs, d_g_entropy, d_grad, ldg};
    with_float(type, [&](auto e) {
        hipLaunchKernelGGL((logprobs_grad_kernel<decltype(e)>), dim3((unsigned)rows), dim3(256), 0, as_stream(stream),
                           a);
    });
    return launch_status("lq_token_logprobs_backward");
}

}  // extern "C"
