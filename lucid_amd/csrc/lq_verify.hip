// lq_verify.hip -- verification of drafted tokens under a target's distribution, from given random numbers.
//
//   kept while u q(t) < p(t); the new token by the first j with W_j > u W, W_j the sums of max(p - q, 0) (or of p).
//   p = e^(x - lse), q likewise.
//
// Whole numbers come out, and a border between two of them decides: exponentials and sums are 64-bit, so that a sum
// in another order, off by some 2^-50, changes a token in one of 10^10 draws.
//
// Two launches: the first finds each sequence's row and sums parts of it (the only large read: one row of the
// target and one of the draft), the second finds the part that holds the border and the token in it.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_attn.h"

namespace lq {
namespace {

struct VerifyArgs {
    const void* x;
    int64_t ld;
    const float* lse;
    const void* d;  // the draft's logits, or NULL: certain drafts
    int64_t ldd;
    const float* dlse;
    const int32_t *drafts, *starts;
    int64_t seqs, rows;
    int vocab, parts;
    const float *accept, *sample;
    int32_t *tokens, *accepted;
    double2* sums;  // [seqs][parts]: of the weights max(p - q, 0) and of p
};

constexpr int VF_T = 256, VF_PART = 4096;  // threads of a workgroup, tokens of a part

// Rows of sequence s, kept inside the array whatever the starts hold.
__device__ __forceinline__ void sequence_rows(const VerifyArgs& a, int64_t s, int64_t& first, int64_t& n) {
    const int64_t lo = a.starts[s], hi = a.starts[s + 1];
    first = lo < 0 ? 0 : lo > a.rows ? a.rows : lo;
    n = (hi > a.rows ? a.rows : hi) - first;
    if (n < 0) n = 0;
}

template <class E>
__device__ __forceinline__ double probability(const void* x, int64_t ld, const float* lse, int64_t row, int64_t j) {
    return exp((double)E::load(static_cast<const typename E::T*>(x)[row * ld + j]) - (double)lse[row]);
}

// How many of a sequence's drafts are kept; every thread of a wave calls it, 64 drafts at a time.
template <class E>
__device__ __forceinline__ int64_t kept(const VerifyArgs& a, int64_t first, int64_t drafts) {
    const int lane = threadIdx.x & 63;
    for (int64_t i = 0; i < drafts; i += 64) {
        bool fails = false;
        if (i + lane < drafts) {
            const int64_t r = first + i + lane;
            const int32_t t = a.drafts[r];
            fails = true;
            if (t >= 0 && t < a.vocab) {
                const double q = a.d ? probability<E>(a.d, a.ldd, a.dlse, r, t) : 1.0;
                fails = !((double)a.accept[r] * q < probability<E>(a.x, a.ld, a.lse, r, t));
            }
        }
        const uint64_t m = __ballot(fails);
        if (m) return i + __builtin_ctzll(m);
    }
    return drafts;
}

// The weights of token j in a row: of what is left of p, and p.
template <class E>
struct Weights {
    const VerifyArgs& a;
    int64_t row;
    bool rejected;
    int32_t draft;
    __device__ __forceinline__ Weights(const VerifyArgs& a, int64_t row, bool rejected)
        : a(a), row(row), rejected(rejected), draft(rejected ? a.drafts[row] : -1) {}
    __device__ __forceinline__ double2 operator()(int j) const {
        const double p = probability<E>(a.x, a.ld, a.lse, row, j);
        if (!rejected) return make_double2(0.0, p);
        if (!a.d) return make_double2(j == draft ? 0.0 : p, p);
        const double w = p - probability<E>(a.d, a.ldd, a.dlse, row, j);
        return make_double2(w > 0.0 ? w : 0.0, p);
    }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

template <class E>
__global__ __launch_bounds__(VF_T) void verify_sums_kernel(VerifyArgs a) {
    __shared__ double2 red[VF_T / 64];
    const int64_t n = workgroup(), s = n / a.parts;
    if (s >= a.seqs) return;
    const int part = (int)(n - s * a.parts), tid = threadIdx.x;
    int64_t first, rows;
    sequence_rows(a, s, first, rows);
    const int64_t keep = rows > 0 ? kept<E>(a, first, rows - 1) : 0;
    if (part == 0 && tid == 0) a.accepted[s] = (int32_t)keep;
    if (rows == 0) return;
    const Weights<E> w(a, first + keep, keep < rows - 1);
    double2 sum = make_double2(0.0, 0.0);
    const int end = min(a.vocab, (part + 1) * VF_PART);
    for (int j = part * VF_PART + tid; j < end; j += VF_T) {
        const double2 v = w(j);
        sum.x += v.x;
        sum.y += v.y;
    }
    sum.x = wave_sum64(sum.x);
    sum.y = wave_sum64(sum.y);
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < VF_T / 64; ++i) {
            sum.x += red[i].x;
            sum.y += red[i].y;
        }
        a.sums[n] = sum;
    }
}

// First index of [0, n) whose inclusive sum of value(i) passes `at`, and the sum before it; the last index with
// a positive value where rounding leaves none; -1 where there is none.  n may be any number: each thread
// takes a run of ceil(n / VF_T).  Uniform over the workgroup.
struct Border {
    int index;
    double before;
};
template <class F>
__device__ __forceinline__ Border find_border(int n, double at, F value, double* scan, int* best, double* before) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (n + VF_T - 1) / VF_T, lo = min(tid * per, n), hi = min(lo + per, n);
    double mine = 0.0;
    int last = -1;
    for (int i = lo; i < hi; ++i) {
        const double v = value(i);
        mine += v;
        if (v > 0.0) last = i;
    }
    double upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
    }
    __syncthreads();
    if (lane == 63) scan[wave] = upto;
    if (tid == 0) {
        best[0] = n;
        best[1] = -1;
        *before = 0.0;
    }
    __syncthreads();
    double base = upto - mine;
    if (lane == 0) base = 0.0;  // exactly
    for (int w = 0; w < wave; ++w) base += scan[w];
    int found = n;
    double at_found = 0.0, run = base;
    for (int i = lo; i < hi; ++i) {
        const double v = value(i);
        if (found == n && v > 0.0 && run + v > at) {
            found = i;
            at_found = run;
        }
        run += v;
    }
    if (found < n) atomicMin(&best[0], found);
    if (last >= 0) atomicMax(&best[1], last);
    __syncthreads();
    Border b{best[0], 0.0};
    if (found == b.index && found < n) *before = at_found;
    if (b.index == n) b.index = best[1];
    __syncthreads();
    b.before = *before;
    return b;
}

template <class E>
__global__ __launch_bounds__(VF_T) void verify_token_kernel(VerifyArgs a) {
    __shared__ double values[VF_PART];
    __shared__ double scan[VF_T / 64], before;
    __shared__ int best[2];
    const int64_t s = workgroup();
    if (s >= a.seqs) return;
    const int tid = threadIdx.x;
    int64_t first, rows;
    sequence_rows(a, s, first, rows);
    if (rows == 0) return;
    const int64_t keep = a.accepted[s];
    const Weights<E> w(a, first + keep, keep < rows - 1);
    const double2* sums = a.sums + s * a.parts;
    // the totals, in one order for every thread
    double2 total = make_double2(0.0, 0.0);
    for (int i = 0; i < a.parts; ++i) {
        total.x += sums[i].x;
        total.y += sums[i].y;
    }
    const bool rest = total.x > 0.0;
    const double all = rest ? total.x : total.y, u = (double)a.sample[s];
    int token = -1;
    if (all > 0.0 && all < INFINITY) {
        const Border p = find_border(a.parts, u * all, [&](int i) { return rest ? sums[i].x : sums[i].y; }, scan, best,
                                     &before);
        if (p.index >= 0) {
            const int j0 = p.index * VF_PART, m = min(VF_PART, a.vocab - j0);
            for (int i = tid; i < m; i += VF_T) {
                const double2 v = w(j0 + i);
                values[i] = rest ? v.x : v.y;
            }
            __syncthreads();
            token = j0 + find_border(m, u * all - p.before, [&](int i) { return values[i]; }, scan, best, &before).index;
        }
    }
    for (int64_t i = tid; i < rows; i += VF_T)
        a.tokens[first + i] = i < keep ? a.drafts[first + i] : i == keep ? token : -1;
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

size_t lq_verify_drafts_workspace_size(int64_t seqs, int64_t vocab) {
    if (seqs <= 0 || vocab <= 0) return 0;
    return (size_t)seqs * (size_t)((vocab + VF_PART - 1) / VF_PART) * sizeof(double2);
}

int lq_verify_drafts(const void* d_logits, int type, int64_t ld, const float* d_lse, const void* d_draft_logits,
                     int64_t ldd, const float* d_draft_lse, const int32_t* d_drafts, const int32_t* d_starts,
                     int64_t seqs, int64_t rows, int64_t vocab, const float* d_accept_u, const float* d_sample_u,
                     int32_t* d_tokens, int32_t* d_accepted, void* d_workspace, size_t workspace_bytes, void* stream) {
    LQ_REQUIRE(is_float_type(type), "lq_verify_drafts: logits must be float32, fp16 or bfloat16");
    LQ_REQUIRE(seqs >= 0 && rows >= 0 && vocab > 0 && vocab <= (1 << 30) && ld >= vocab && seqs <= 0x7fffffff &&
                   rows <= 0x7fffffff && (!d_draft_logits || ldd >= vocab),
               "lq_verify_drafts: bad shape");
    LQ_REQUIRE(!d_draft_logits == !d_draft_lse, "lq_verify_drafts: the draft's logits and their lse come together");
    if (seqs == 0) return LQ_OK;
    LQ_REQUIRE(d_starts && d_accepted && d_sample_u, "lq_verify_drafts: NULL pointer");
    LQ_REQUIRE(rows == 0 || (d_logits && d_lse && d_drafts && d_accept_u && d_tokens), "lq_verify_drafts: NULL pointer");
    LQ_REQUIRE(d_workspace && aligned16(d_workspace) &&
                   workspace_bytes >= lq_verify_drafts_workspace_size(seqs, vocab),
               "lq_verify_drafts: workspace too small or not 16-byte aligned");
    const int parts = (int)((vocab + VF_PART - 1) / VF_PART);
    const VerifyArgs a{d_logits, ld, d_lse, d_draft_logits, ldd, d_draft_lse, d_drafts, d_starts, seqs, rows,
                       (int)vocab, parts, d_accept_u, d_sample_u, d_tokens, d_accepted,
                       static_cast<double2*>(d_workspace)};
    const hipStream_t st = as_stream(stream);
    with_float(type, [&](auto e) {
        using E = decltype(e);
        hipLaunchKernelGGL((verify_sums_kernel<E>), grid_of(seqs * parts), dim3(VF_T), 0, st, a);
        hipLaunchKernelGGL((verify_token_kernel<E>), grid_of(seqs), dim3(VF_T), 0, st, a);
    });
    return launch_status("lq_verify_drafts");
}

}  // extern "C"
