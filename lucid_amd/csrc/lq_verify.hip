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

// Threads of a workgroup; tokens of a run, which one wave sums and one searches (eight to a lane).  Both launches, us,
// with runs of 512 / 1024 / 2048: 64 sequences of 8 rows of 100003 in bfloat16 21.4 / 22.5 / 28.1, 8 sequences of 5
// rows of 32000 in float32 with certain drafts 8.8 / 10.5 / 13.8.
constexpr int VF_T = 256, VF_RUN = 512;

// e^t within a few 2^-53: t = n log(2) / 64 + r, the high and low part of log(2) / 64 taken off in turn; 2^(n % 64 / 64)
// from a table in LDS, Taylor's sum of e^r to r^5 (|r| < 0.0055: the next term is 2^-54), 2^(n / 64) as an
// exponent.  0 below -745 and for NaN.  Coefficients are held in scalar registers whose values the compiler does not see:
// it would move each into place again for every exponential.
struct Exp64 {
    double by, lo, hi, c[4];
    const double* table;
    // `t`: 64 numbers of LDS, filled here by the workgroup's first wave; a barrier where there are others
    __device__ __forceinline__ explicit Exp64(double* t)
        : by(92.332482616893657), lo(-3.6235106466348430e-19), hi(-0.010830424696249145),
          c{0.5, 1.0 / 6.0, 1.0 / 24.0, 1.0 / 120.0}, table(t) {
        asm("" : "+s"(by), "+s"(lo), "+s"(hi));
#pragma unroll
        for (int i = 0; i < 4; ++i) asm("" : "+s"(c[i]));
        if (threadIdx.x < 64) t[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
    }
    __device__ __forceinline__ double operator()(double t) const {
        constexpr double SHIFT = 6755399441055744.0;  // 1.5 * 2^52: a sum with it is rounded to whole numbers
        t = fmax(t, -800.0);
        const double n = __builtin_fma(t, by, SHIFT), k = n - SHIFT;
        const double r = __builtin_fma(k, lo, __builtin_fma(k, hi, t));
        double p = __builtin_fma(c[3], r, c[2]);
        p = __builtin_fma(p, r, c[1]);
        p = __builtin_fma(p, r, c[0]);
        p = __builtin_fma(p, r, 1.0) * r;
        const int whole = (int)(uint32_t)__builtin_bit_cast(uint64_t, n);
        const double y = table[whole & 63];
        return __builtin_amdgcn_ldexp(__builtin_fma(y, p, y), whole >> 6);
    }
};

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
__device__ __forceinline__ double log_probability(const void* x, int64_t ld, const float* lse, int64_t row, int64_t j) {
    return (double)E::load(static_cast<const typename E::T*>(x)[row * ld + j]) - (double)lse[row];
}

// How many of a sequence's drafts are kept; every thread of a wave calls it, 64 drafts at a time.
template <class E>
__device__ __forceinline__ int64_t kept(const Exp64& e, const VerifyArgs& a, int64_t first, int64_t drafts) {
    const int lane = threadIdx.x & 63;
    for (int64_t i = 0; i < drafts; i += 64) {
        bool fails = false;
        if (i + lane < drafts) {
            const int64_t r = first + i + lane;
            const int32_t t = a.drafts[r];
            fails = true;
            if (t >= 0 && t < a.vocab) {
                const double q = a.d ? log_probability<E>(a.d, a.ldd, a.dlse, r, t) : 0.0;
                const double p = log_probability<E>(a.x, a.ld, a.lse, r, t);
                fails = !(q == q && (double)a.accept[r] * e(q) < e(p));
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
    const Exp64& exp;
    const typename E::T *x, *d;
    double lse, dlse;
    int vocab;
    bool rejected;
    int32_t draft;
    __device__ __forceinline__ Weights(const Exp64& exp, const VerifyArgs& a, int64_t row, bool rejected)
        : exp(exp), x(static_cast<const typename E::T*>(a.x) + row * a.ld),
          d(rejected && a.d ? static_cast<const typename E::T*>(a.d) + row * a.ldd : nullptr), lse((double)a.lse[row]),
          dlse(rejected && a.d ? (double)a.dlse[row] : 0.0), vocab(a.vocab), rejected(rejected),
          draft(rejected ? a.drafts[row] : -1) {}
    __device__ __forceinline__ void operator()(int j, double2 (&w)[8]) const {
        float u[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = v[i] = -INFINITY;
        if (j + 8 <= vocab) {
            load8_any<E>(x + j, u);
            if (d) load8_any<E>(d + j, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j + i < vocab) {
                    u[i] = E::load(x[j + i]);
                    if (d) v[i] = E::load(d[j + i]);
                }
        }
        double p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = exp((double)u[i] - lse);  // -inf past the vocabulary: 0
        if (d) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = make_double2(fmax(p[i] - exp((double)v[i] - dlse), 0.0), p[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = make_double2(rejected && j + i != draft ? p[i] : 0.0, p[i]);
        }
    }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// One wave per run, sixteen bytes a load.  64 rows of 100003 in bfloat16 and as many of the draft: 16.5 us.  That is 25.6
// MB (3.7 us) and 12.8 million exponentials of about 20 64-bit operations each (6.5 us), after some 4 us of dependent
// loads from the starts to the row that is summed.
template <class E>
__global__ __launch_bounds__(VF_T) void verify_sums_kernel(VerifyArgs a) {
    __shared__ double table[64];
    const Exp64 e(table);
    __syncthreads();
    const int64_t groups = (a.runs + VF_T / 64 - 1) / (VF_T / 64), n = workgroup(), s = n / groups;
    if (s >= a.seqs) return;
    const int lane = threadIdx.x & 63;
    const int run = __builtin_amdgcn_readfirstlane((int)(n - s * groups) * (VF_T / 64) + (threadIdx.x >> 6));
    int64_t first, rows;
    sequence_rows(a, s, first, rows);
    const int64_t keep = rows > 0 ? kept<E>(e, a, first, rows - 1) : 0;
    if (run == 0 && lane == 0) a.accepted[s] = (int32_t)keep;
    if (rows == 0 || run >= a.runs) return;
    const Weights<E> w(e, a, first + keep, keep < rows - 1);
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

// The sum of the lanes up to this one, and of all.
__device__ __forceinline__ double wave_scan64(double v, double& total) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    total = __shfl(v, 63, 64);
    return v;
}

// A wave per sequence, without a barrier: the run that holds the border, then the token in it.  4.9 us for 64 sequences
// of 196 runs: a chain of dependent loads, scans of 64-bit sums and eight exponentials.  Where rounding leaves
// no sum above the border, the last token with a weight is taken.
template <class E>
__global__ __launch_bounds__(64) void verify_token_kernel(VerifyArgs a) {
    __shared__ double table[64];
    const Exp64 e(table);
    __syncthreads();
    const int64_t s = workgroup();
    if (s >= a.seqs) return;
    const int lane = threadIdx.x;
    int64_t first, rows;
    sequence_rows(a, s, first, rows);
    if (rows == 0) return;
    const double u = (double)a.sample[s];
    const int64_t keep = a.accepted[s];
    const double2* sums = a.sums + s * a.runs;
    // runs lo .. hi - 1 are this lane's
    const int per = (a.runs + 63) / 64, lo = min(lane * per, a.runs), hi = min(lo + per, a.runs);
    double2 mine = make_double2(0.0, 0.0), total;
#pragma unroll 4
    for (int i = lo; i < hi; ++i) {
        const double2 v = sums[i];
        mine.x += v.x;
        mine.y += v.y;
    }
    const Weights<E> w(e, a, first + keep, keep < rows - 1);
    const double upto_x = wave_scan64(mine.x, total.x), upto_y = wave_scan64(mine.y, total.y);
    const bool rest = total.x > 0.0;
    const double all = rest ? total.x : total.y, at = u * all;
    int token = -1;
    if (all > 0.0 && all < INFINITY) {
        double upto = rest ? upto_x - mine.x : upto_y - mine.y, before = 0.0;
        int found = -1, last = -1;
#pragma unroll 4
        for (int i = lo; i < hi; ++i) {
            const double v = rest ? sums[i].x : sums[i].y;
            if (v > 0.0) {
                last = i;
                if (found < 0 && upto + v > at) {
                    found = i;
                    before = upto;
                }
            }
            upto += v;
        }
        uint64_t m = __ballot(found >= 0);
        const bool border = m != 0;
        if (!border) m = __ballot(last >= 0);  // one has, as the total is positive
        const int owner = border ? __builtin_ctzll(m) : 63 - __builtin_clzll(m);
        const int run = __shfl(border ? found : last, owner, 64);
        before = __shfl(before, owner, 64);
        constexpr int EACH = VF_RUN / 64;
        double v[EACH], sum = 0.0, all_of_it;
#pragma unroll
        for (int i = 0; i < EACH; i += 8) {
            double2 x[8];
            w(run * VF_RUN + EACH * lane + i, x);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[i + k] = rest ? x[k].x : x[k].y;
                sum += v[i + k];
            }
        }
        upto = wave_scan64(sum, all_of_it) - sum + before;
        found = last = -1;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (v[i] > 0.0) {
                last = EACH * lane + i;
                if (found < 0 && border && upto + v[i] > at) found = last;
            }
            upto += v[i];
        }
        m = __ballot(found >= 0);
        const bool there = m != 0;
        if (!there) m = __ballot(last >= 0);
        // a run is taken for its positive sum, so that some lane of it has a weight
        if (m) token = run * VF_RUN + __shfl(there ? found : last, there ? __builtin_ctzll(m) : 63 - __builtin_clzll(m), 64);
    }
    for (int64_t i = lane; i < rows; i += 64)
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
        hipLaunchKernelGGL((verify_token_kernel<E>), grid_of(seqs), dim3(64), 0, st, a);
    });
    return launch_status("lq_verify_drafts");
}

}  // extern "C"
