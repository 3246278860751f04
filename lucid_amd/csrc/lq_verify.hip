// lq_verify.hip -- verification of drafted tokens under a target's distribution, from given random numbers.
//
//   kept while u q(t) < p(t); the new token by the first j with W_j > u W, W_j the sums of max(p - q, 0) (or of p).
//   p = e^(x - lse), q likewise.
//
// Whole numbers come out, and a border between two of them decides: exponentials and sums are 64-bit, so that a sum
// in another order, off by some 2^-50, changes a token in one of 10^10 draws.
//
// Two launches: the first finds each sequence's row and sums runs of it (the only large read: one row of the
// target and one of the draft), the second finds the run that holds the border and the token in it.
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
    int vocab, runs;
    const float *accept, *sample;
    int32_t *tokens, *accepted;
    double2* sums;  // [seqs][runs]: of the weights max(p - q, 0) and of p
};

// Threads of a workgroup; tokens of a run, which one wave sums (sixteen to a lane) and one workgroup searches.
constexpr int VF_T = 256, VF_RUN = 1024;

// e^t for t <= 709, within a few 2^-52: t = k log 2 + r, |r| <= log(2) / 2, Taylor's sum to r^12 (the next term is
// 2^-52), the high and low part of log 2 taken off in turn.  NaN for NaN.
__device__ __forceinline__ double exp64(double t) {
    const double k = __builtin_rint(t * 1.4426950408889634);
    const double r = __builtin_fma(k, -2.3190468138462996e-17, __builtin_fma(k, -0.6931471805599453, t));
    double p = 1.0 / 479001600.0;
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return t < -746.0 ? 0.0 : ldexp(p, (int)k);
}

// Eight values from any address (rows of odd lengths).
template <class E>
__device__ __forceinline__ void load8_any(const typename E::T* p, float (&x)[8]) {
    if constexpr (E::code == LQ_F32) {
        vf4 v[2];
        __builtin_memcpy(v, p, 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[j >> 2][j & 3];
    } else {
        u4v w;
        __builtin_memcpy(&w, p, 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f2v u = unpack2(E{}, w[j]);
            x[2 * j] = u[0];
            x[2 * j + 1] = u[1];
        }
    }
}

// Rows of sequence s, kept inside the array whatever the starts hold.
__device__ __forceinline__ void sequence_rows(const VerifyArgs& a, int64_t s, int64_t& first, int64_t& n) {
    const int64_t lo = a.starts[s], hi = a.starts[s + 1];
    first = lo < 0 ? 0 : lo > a.rows ? a.rows : lo;
    n = (hi > a.rows ? a.rows : hi) - first;
    if (n < 0) n = 0;
}

template <class E>
__device__ __forceinline__ double probability(const void* x, int64_t ld, const float* lse, int64_t row, int64_t j) {
    return exp64((double)E::load(static_cast<const typename E::T*>(x)[row * ld + j]) - (double)lse[row]);
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

// The weights of eight tokens from j on in a row: of what is left of p, and p.  Past the vocabulary both are 0.
template <class E>
struct Weights {
    const typename E::T *x, *d;
    double lse, dlse;
    int vocab;
    bool rejected;
    int32_t draft;
    __device__ __forceinline__ Weights(const VerifyArgs& a, int64_t row, bool rejected)
        : x(static_cast<const typename E::T*>(a.x) + row * a.ld),
          d(rejected && a.d ? static_cast<const typename E::T*>(a.d) + row * a.ldd : nullptr), lse((double)a.lse[row]),
          dlse(rejected && a.d ? (double)a.dlse[row] : 0.0), vocab(a.vocab), rejected(rejected),
          draft(rejected ? a.drafts[row] : -1) {}
    template <int N>
    __device__ __forceinline__ void operator()(int j, double2 (&w)[N]) const {
        float u[N], v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = v[i] = -INFINITY;
        if (N == 8 && j + N <= vocab) {
            if constexpr (N == 8) {
                load8_any<E>(x + j, u);
                if (d) load8_any<E>(d + j, v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (j + i < vocab) {
                    u[i] = E::load(x[j + i]);
                    if (d) v[i] = E::load(d[j + i]);
                }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const double p = j + i < vocab ? exp64((double)u[i] - lse) : 0.0;
            double r = 0.0;
            if (rejected) {
                if (!d) r = j + i == draft ? 0.0 : p;
                else {
                    const double e = p - exp64((double)v[i] - dlse);
                    r = e > 0.0 ? e : 0.0;
                }
            }
            w[i] = make_double2(r, p);
        }
    }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// One wave per run.  verify_b64 (64 rows of 100003, twice): FIGURE
template <class E>
__global__ __launch_bounds__(VF_T) void verify_sums_kernel(VerifyArgs a) {
    const int64_t groups = (a.runs + VF_T / 64 - 1) / (VF_T / 64), n = workgroup(), s = n / groups;
    if (s >= a.seqs) return;
    const int lane = threadIdx.x & 63;
    const int run = __builtin_amdgcn_readfirstlane((int)(n - s * groups) * (VF_T / 64) + (threadIdx.x >> 6));
    int64_t first, rows;
    sequence_rows(a, s, first, rows);
    const int64_t keep = rows > 0 ? kept<E>(a, first, rows - 1) : 0;
    if (run == 0 && lane == 0) a.accepted[s] = (int32_t)keep;
    if (rows == 0 || run >= a.runs) return;
    const Weights<E> w(a, first + keep, keep < rows - 1);
    double2 sum = make_double2(0.0, 0.0);
#pragma unroll
    for (int i = 0; i < VF_RUN; i += 512) {
        double2 v[8];
        w(run * VF_RUN + i + 8 * lane, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            sum.x += v[k].x;
            sum.y += v[k].y;
        }
    }
    sum.x = wave_sum64(sum.x);
    sum.y = wave_sum64(sum.y);
    if (lane == 0) a.sums[s * a.runs + run] = sum;
}

// The inclusive sums over the workgroup's threads of one number each, and the sum of all.
__device__ __forceinline__ double block_scan(double mine, double* scan, double& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
    }
    __syncthreads();
    if (lane == 63) scan[wave] = upto;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < VF_T / 64; ++w) {
        if (w < wave) before += scan[w];
        total += scan[w];
    }
    return before + upto;
}

// The smallest of the threads' candidates, or where none has one (n) the largest of `last`.
__device__ __forceinline__ int first_of(int found, int n, int last, int* best) {
    __syncthreads();
    if (threadIdx.x == 0) {
        best[0] = n;
        best[1] = -1;
    }
    __syncthreads();
    if (found < n) atomicMin(&best[0], found);
    if (last >= 0) atomicMax(&best[1], last);
    __syncthreads();
    return best[0] < n ? best[0] : best[1];
}

// A workgroup per sequence.  Where rounding leaves no sum above the border, the last token with a weight is taken.
template <class E>
__global__ __launch_bounds__(VF_T) void verify_token_kernel(VerifyArgs a) {
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
    const double u = (double)a.sample[s];
    const double2* sums = a.sums + s * a.runs;
    // runs lo .. hi - 1 are this thread's
    const int per = (a.runs + VF_T - 1) / VF_T, lo = min(tid * per, a.runs), hi = min(lo + per, a.runs);
    double2 mine = make_double2(0.0, 0.0), total;
    for (int i = lo; i < hi; ++i) {
        const double2 v = sums[i];
        mine.x += v.x;
        mine.y += v.y;
    }
    const double upto_x = block_scan(mine.x, scan, total.x), upto_y = block_scan(mine.y, scan, total.y);
    const bool rest = total.x > 0.0;
    const double all = rest ? total.x : total.y, at = u * all;
    int token = -1;
    if (all > 0.0 && all < INFINITY) {
        double run = rest ? upto_x - mine.x : upto_y - mine.y, at_found = 0.0;
        int found = a.runs, last = -1;
        for (int i = lo; i < hi; ++i) {
            const double v = rest ? sums[i].x : sums[i].y;
            if (v > 0.0) {
                last = i;
                if (found == a.runs && run + v > at) {
                    found = i;
                    at_found = run;
                }
            }
            run += v;
        }
        const int part = first_of(found, a.runs, last, best);
        if (found == part) before = at_found;
        else if (last == part) before = -1.0;  // no border: every weight passes it, and the last one is taken
        __syncthreads();
        if (part >= 0) {
            const bool none = before < 0.0;
            const int j0 = part * VF_RUN;
            constexpr int EACH = VF_RUN / VF_T;
            double2 v[EACH];
            w(j0 + EACH * tid, v);
            double sum = 0.0, all_of_it;
#pragma unroll
            for (int i = 0; i < EACH; ++i) sum += rest ? v[i].x : v[i].y;
            double upto = block_scan(sum, scan, all_of_it) - sum + (none ? 0.0 : before);
            int pick = VF_RUN, tail = -1;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const double x = rest ? v[i].x : v[i].y;
                if (x > 0.0) {
                    tail = EACH * tid + i;
                    if (!none && pick == VF_RUN && upto + x > at) pick = tail;
                }
                upto += x;
            }
            token = j0 + first_of(pick, VF_RUN, tail, best);
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
    return (size_t)seqs * (size_t)((vocab + VF_RUN - 1) / VF_RUN) * sizeof(double2);
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
    const int runs = (int)((vocab + VF_RUN - 1) / VF_RUN);
    const VerifyArgs a{d_logits, ld, d_lse, d_draft_logits, ldd, d_draft_lse, d_drafts, d_starts, seqs, rows,
                       (int)vocab, runs, d_accept_u, d_sample_u, d_tokens, d_accepted,
                       static_cast<double2*>(d_workspace)};
    const hipStream_t st = as_stream(stream);
    with_float(type, [&](auto e) {
        using E = decltype(e);
        hipLaunchKernelGGL((verify_sums_kernel<E>), grid_of(seqs * ((runs + VF_T / 64 - 1) / (VF_T / 64))), dim3(VF_T), 0, st, a);
        hipLaunchKernelGGL((verify_token_kernel<E>), grid_of(seqs), dim3(VF_T), 0, st, a);
    });
    return launch_status("lq_verify_drafts");
}

}  // extern "C"
