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
constexpr int64_t LP_MAX_VOCAB = (int64_t)1 << 30;

// Sums of one part of a row: its largest value, sum e^d and sum e^d d relative to it.
struct PartSums {
    float R, s, ed, pad;
};

struct LogprobArgs {
    const void* x;
    int64_t ldx, rows, vocab;
    const int32_t* targets;
    int top;
    float *logprobs, *entropy, *lse, *top_logprobs;
    int32_t* top_ids;
    int parts;        // workgroups of a row; past 1 the results go to the next two, for the join
    PartSums* sums;   // [rows][parts]
    uint64_t* keys;   // [rows][parts][top]
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

// 16 bytes of a row's elements as float32.
template <class E>
struct Chunk {
    static constexpr int N = 16 / (int)sizeof(typename E::T);
    float v[N];
};
template <class E>
__device__ __forceinline__ Chunk<E> widen(u4v w) {
    Chunk<E> c;
    if constexpr (E::code == LQ_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c.v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2v p = unpack2(E{}, w[i]);
            c.v[2 * i] = p[0];
            c.v[2 * i + 1] = p[1];
        }
    }
    return c;
}

// A row in 16-byte chunks of aligned addresses: chunk q holds elements q N - shift ... q N - shift +
// N - 1, of which the first and the last chunk may own only some.
template <class E>
struct Row {
    static constexpr int N = Chunk<E>::N;
    const typename E::T* x;
    int vocab, shift, chunks;
    __device__ __forceinline__ Row(const typename E::T* row, int64_t n) : x(row), vocab((int)n) {
        shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::T));
        chunks = (int)(((int64_t)vocab + shift + N - 1) / N);
    }
    __device__ __forceinline__ bool full(int q) const {
        return q * (int64_t)N >= shift && (q + 1) * (int64_t)N - shift <= vocab;
    }
    __device__ __forceinline__ int first(int q) const { return q * N - shift; }
    __device__ __forceinline__ u4v load(int q) const {
        return __builtin_nontemporal_load(reinterpret_cast<const u4v*>(x + first(q)));
    }
};

// A row as `head` single elements, `chunks` 16-byte chunks of aligned addresses and `tail` single elements.
template <class E>
struct Split {
    static constexpr int N = Chunk<E>::N;
    const typename E::T* x;
    int vocab, head, chunks, tail;
    __device__ __forceinline__ Split(const typename E::T* row, int64_t n) : x(row), vocab((int)n) {
        const int past = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::T));
        head = min((N - past) % N, vocab);
        chunks = (vocab - head) / N;
        tail = vocab - head - chunks * N;
    }
    __device__ __forceinline__ int first(int q) const { return head + q * N; }
    __device__ __forceinline__ u4v load(int q) const {
        return __builtin_nontemporal_load(reinterpret_cast<const u4v*>(x + first(q)));
    }
};

constexpr int LP_CAND = 512;  // alternatives collected before the last choice
constexpr int LP_PARTS = 16;  // parts of a row at most

// A row's results from its sums (written by the one thread that `writes`), and one alternative.
template <class E>
__device__ __forceinline__ float row_results(const LogprobArgs& a, int64_t r, float R, float s, float ed, bool writes) {
    const float log_s = logf(s), lse = (R == -INFINITY ? 0.0f : R) + log_s;  // -inf for a row that allows nothing
    if (writes) {
        if (a.lse) a.lse[r] = lse;
        if (a.entropy) a.entropy[r] = s == 0.0f ? 0.0f : log_s - ed / s;
        if (a.logprobs) {
            const int64_t t = a.targets[r];
            const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ldx;
            a.logprobs[r] = t >= 0 && t < a.vocab ? logprob_of(E::load(x[t]), lse) : 0.0f;
        }
    }
    return lse;
}
template <class E>
__device__ __forceinline__ void row_choice(const LogprobArgs& a, int64_t r, int at, int j, float lse) {
    a.top_ids[r * a.top + at] = j;
    a.top_logprobs[r * a.top + at] = logprob_of(E::load(static_cast<const typename E::T*>(a.x)[r * a.ldx + j]), lse);
}

// One workgroup per row, one pass over it.  A thread keeps a reference for its exponentials, the sums of e^d
// and of e^d d, and its largest value.  The reference follows the largest value when that has risen by more
// than 4, looked at once for four chunks: the sum of e^d d is rounded at the size that the largest value
// has relative to the reference, and the final change of reference takes most of it away again (past a rise
// of 16 only, the entropy of rows that one token rules was off by 100 half-steps of float32's 1, now by 4;
// 8 rows of 32000 float32 logits take 7.6 us for 7.36, past a rise of 2 7.66).  Chunks are summed before
// they are added: a sum that holds the row's largest value then loses the small ones by rounding only
// where a whole group of them is below 2^-25 of it.
//
// The alternatives come from those largest values: of 64 groups of threads, the top-th largest group
// maximum `cut` has at least `top` elements at or above it, and only threads whose own maximum
// reaches it can hold any.  Their chunks are read again (from the caches), elements at or above the
// cut collected and ranked against each other.  Where too many tie with the cut (masked tokens) the
// elements above it are collected alone and the ties taken in index order; rows with NaN or +inf,
// and rows where even those are too many, are searched once per alternative.
//
// 4096 rows of 100003 bfloat16 logits, eight alternatives: 148 us (5.5 TB/s).  Before the single elements
// at the ends left the loop: 159, with 256 threads to a row 171, with 1024 164, without alternatives
// 142.  Without the entropy it is no faster: the loads bound it.
template <int NT, class E>
__global__ __launch_bounds__(NT) void logprobs_kernel(LogprobArgs a) {
    constexpr int W = NT / 64, N = Chunk<E>::N, UNROLL = 4;
    __shared__ __attribute__((aligned(16))) float groups[64];  // largest values of NT / 64 neighbouring threads each
    __shared__ float red[2][W];
    __shared__ int s_who, s_count, s_wave[W];
    __shared__ int who[NT];
    __shared__ uint64_t cand[LP_CAND];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t id = (uint32_t)workgroup();
    const int64_t r = id / (uint32_t)a.parts;
    if (r >= a.rows) return;
    const int part = id - (uint32_t)r * (uint32_t)a.parts;
    // this workgroup's columns: whole chunks but for the last part's end
    const int64_t width = (a.vocab + (int64_t)a.parts * N - 1) / ((int64_t)a.parts * N) * N, c0 = part * width;
    const Split<E> row(static_cast<const typename E::T*>(a.x) + r * a.ldx + c0, min(width, a.vocab - c0));

    float ref = -INFINITY, base = 0.0f, top = -INFINITY, s = 0.0f, ed = 0.0f;  // base: ref, 0 while it is -inf
    auto largest = [](const Chunk<E>& c) __attribute__((always_inline)) {
        float m = c.v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) m = fmaxf(m, c.v[e]);
        return m;
    };
    auto follow = [&](float m) __attribute__((always_inline)) {
        top = fmaxf(top, m);
        if (m > ref + 4.0f) {
            const float f = s > 0.0f ? __builtin_amdgcn_exp2f((base - m) * LOG2E) : 0.0f;
            ed = f > 0.0f ? f * __builtin_fmaf(s, base - m, ed) : 0.0f;
            s *= f;
            ref = base = m;
        }
    };
    auto sums = [&](const Chunk<E>& c, float& cs, float& ce) __attribute__((always_inline)) {
        cs = ce = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = c.v[e] - base, p = __builtin_amdgcn_exp2f(d * LOG2E);
            cs += p;
            ce = __builtin_fmaf(p, fmaxf(d, -1000.0f), ce);  // p is 0 there: no 0 * inf
        }
    };
    auto add = [&](const Chunk<E>& c) __attribute__((always_inline)) {
        follow(largest(c));
        float cs, ce;
        sums(c, cs, ce);
        s += cs;
        ed += ce;
    };
    // the single elements of both ends: one each of the first threads, on their way during the loop
    Chunk<E> ends;
#pragma unroll
    for (int e = 0; e < N; ++e) ends.v[e] = -INFINITY;
    if (tid < row.head) ends.v[0] = E::load(row.x[tid]);
    if (tid < row.tail) ends.v[1] = E::load(row.x[row.vocab - row.tail + tid]);
    int q = tid;
    for (; q + (UNROLL - 1) * NT < row.chunks; q += UNROLL * NT) {
        u4v w[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) w[u] = row.load(q + u * NT);
        Chunk<E> c[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) c[u] = widen<E>(w[u]);
        static_assert(UNROLL == 4, "the sums below");
        follow(fmaxf(fmaxf(largest(c[0]), largest(c[1])), fmaxf(largest(c[2]), largest(c[3]))));
        float cs[UNROLL], ce[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) sums(c[u], cs[u], ce[u]);
        s += (cs[0] + cs[1]) + (cs[2] + cs[3]);
        ed += (ce[0] + ce[1]) + (ce[2] + ce[3]);
    }
    for (; q < row.chunks; q += NT) add(widen<E>(row.load(q)));
    if (tid < N) add(ends);

    {
        float g = top;
#pragma unroll
        for (int off = NT / 128; off > 0; off >>= 1) g = fmaxf(g, __shfl_xor(g, off, 64));
        if (tid % (NT / 64) == 0) groups[tid / (NT / 64)] = g;
        if (tid == 0) s_who = s_count = 0;
    }
    __syncthreads();
    // the row's largest value, and every thread's sums relative to it
    const float mine = groups[lane];
    const float R = unkey(wave_max(fkey(mine)));
    if (s > 0.0f) {
        const float f = __builtin_amdgcn_exp2f((base - R) * LOG2E);
        ed = f > 0.0f ? f * __builtin_fmaf(s, base - R, ed) : 0.0f;
        s *= f;
    }
    s = ln_wave_sum(s);
    ed = ln_wave_sum(ed);
    if (lane == 0) {
        red[0][wave] = s;
        red[1][wave] = ed;
    }
    float cut = -INFINITY;
    if (a.top) {  // every wave finds the same: the least group maximum that fewer than `top` exceed
        int above = 0;
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
            const vf4 o = *reinterpret_cast<const vf4*>(groups + j);
            above += (o[0] > mine) + (o[1] > mine) + (o[2] > mine) + (o[3] > mine);
        }
        cut = unkey(wave_min(above < a.top ? fkey(mine) : INT32_MAX));
        if (top >= cut) who[atomicAdd(&s_who, 1)] = tid;
    }
    __syncthreads();
    s = red[0][0];
    ed = red[1][0];
#pragma unroll
    for (int w = 1; w < W; ++w) {
        s += red[0][w];
        ed += red[1][w];
    }
    float lse = 0.0f;
    if (a.parts == 1) lse = row_results<E>(a, r, R, s, ed, tid == 0);
    else if (tid == 0) a.sums[id] = PartSums{R, s, ed, 0.0f};
    if (a.top == 0) return;

    auto put = [&](int at, uint64_t key) {
        if (a.parts > 1) a.keys[(int64_t)id * a.top + at] = key - (uint64_t)c0;  // the row's own index
        else row_choice<E>(a, r, at, (int)rank_index(key), lse);
    };
    if (s == s) {  // uniform: no NaN, no +inf in the row
        // the elements at or above the cut (past it, when `strict`) of the threads listed: a wave reads one
        // thread's chunks, a lane each
        const int holders = s_who;
        auto collect = [&](bool strict) {
            auto see = [&](float v, int j) __attribute__((always_inline)) {
                if (strict ? v > cut : v >= cut) {
                    const int at = atomicAdd(&s_count, 1);
                    if (at < LP_CAND) cand[at] = rank_key(v, (uint32_t)j);
                }
            };
            for (int i = wave; i < holders; i += W) {
                const int t = who[i];
                for (int64_t c = t + (int64_t)NT * lane; c < row.chunks; c += (int64_t)NT * 64) {
                    const Chunk<E> v = widen<E>(row.load((int)c));
#pragma unroll
                    for (int e = 0; e < N; ++e) see(v.v[e], row.first((int)c) + e);
                }
                if (lane == 0 && t < row.head) see(E::load(row.x[t]), t);
                if (lane == 1 && t < row.tail) see(E::load(row.x[row.vocab - row.tail + t]), row.vocab - row.tail + t);
            }
            __syncthreads();
            return s_count;
        };
        // each candidate's place is the number of larger ones (keys are distinct)
        auto rank_all = [&](int n) {
            for (int i = tid; i < n; i += NT) {
                const uint64_t key = cand[i];
                int at = 0;
                for (int j = 0; j < n; ++j) at += cand[j] > key;
                if (at < a.top) put(at, key);
            }
        };
        int n = collect(false);
        if (n <= LP_CAND) {
            rank_all(n);
            return;
        }
        __syncthreads();
        if (tid == 0) s_count = 0;
        __syncthreads();
        n = collect(true);
        if (n <= LP_CAND) {
            rank_all(n);
            int at = n;  // then the ties, the lowest indices first
            for (int64_t j0 = 0; j0 < row.vocab && at < a.top; j0 += NT) {
                const int64_t j = j0 + tid;
                const bool hit = j < row.vocab && E::load(row.x[j]) == cut;
                const uint64_t bits = __ballot(hit);
                __syncthreads();
                if (lane == 0) s_wave[wave] = __popcll(bits);
                __syncthreads();
                int before = at + __popcll(bits & (((uint64_t)1 << lane) - 1));
                int all = at;
                for (int w = 0; w < W; ++w) {
                    before += w < wave ? s_wave[w] : 0;
                    all += s_wave[w];
                }
                if (hit && before < a.top) put(before, rank_key(cut, (uint32_t)j));
                at = all;
            }
            return;
        }
    }
    uint64_t last = ~(uint64_t)0;
    for (int k = 0; k < a.top; ++k) {
        uint64_t b = 0;
        for (int64_t j = tid; j < row.vocab; j += NT) {
            const uint64_t key = rank_key(E::load(row.x[j]), (uint32_t)j);
            if (key < last && key > b) b = key;
        }
        for (int off = 32; off > 0; off >>= 1) {
            const uint64_t o = __shfl_xor(b, off, 64);
            b = o > b ? o : b;
        }
        __syncthreads();
        if (lane == 0) cand[wave] = b;
        __syncthreads();
        for (int w = 0; w < W; ++w) b = cand[w] > b ? cand[w] : b;
        last = b;
        if (tid == 0) put(k, b);
    }
}

// The parts of a row joined by one workgroup: sums in the parts' order, then every part's alternatives
// ranked against each other.
template <class E>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
    __shared__ uint64_t keys[LP_PARTS * LP_MAX_TOP];
    const int64_t r = blockIdx.x;
    const int n = a.parts * a.top;
    for (int i = threadIdx.x; i < n; i += 256) keys[i] = a.keys[r * n + i];
    const PartSums* p = a.sums + r * a.parts;
    float R = -INFINITY, s = 0.0f, ed = 0.0f;
    for (int i = 0; i < a.parts; ++i) R = fmaxf(R, p[i].R);
    for (int i = 0; i < a.parts; ++i) {
        if (p[i].s == 0.0f) continue;  // a part that allows nothing
        const float d = p[i].R - R, f = __builtin_amdgcn_exp2f(d * LOG2E);
        s = __builtin_fmaf(f, p[i].s, s);
        ed += f == 0.0f ? 0.0f : f * __builtin_fmaf(p[i].s, d, p[i].ed);
    }
    const float lse = row_results<E>(a, r, R, s, ed, threadIdx.x == 0);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        const uint64_t key = keys[i];
        int at = 0;
        for (int j = 0; j < n; ++j) at += keys[j] > key;
        if (at < a.top) row_choice<E>(a, r, at, (int)rank_index(key), lse);
    }
}

// Parts of a row: where there are fewer rows than CUs, and long ones, several workgroups share a row and a second
// launch joins them (one row of 200000 float32 logits 28.6 -> 12.9 us, of 128000 bfloat16 15.3 -> 10.2; 34
// rows of 159307 bfloat16 20.0 -> 12.6; a row of 65000 float32 11.0 -> 9.9; shorter ones lose).
int row_parts(int64_t rows, int64_t bytes) {
    if (rows <= 0 || rows > 128 || bytes < 131072) return 1;
    const int64_t n = bytes / 32768 < 256 / rows ? bytes / 32768 : 256 / rows;
    return n < 1 ? 1 : n > LP_PARTS ? LP_PARTS : (int)n;
}
size_t parts_bytes(int64_t rows, int parts, int64_t top) {
    return parts > 1 ? (size_t)rows * parts * (sizeof(PartSums) + (size_t)top * sizeof(uint64_t)) : 0;
}

struct LogprobGradArgs {
    const void* x;
    int64_t ldx, rows, vocab;
    const int32_t* targets;
    const float *lse, *entropy, *g_logprobs, *g_entropy;
    void* grad;
    int64_t ldg;
};

// What a row's elements have in common, and one element's gradient.
struct GradRow {
    float g, ge, H, lse;
    int64_t target;  // -1: none
    bool none;       // a row that allows nothing
    __device__ __forceinline__ GradRow(const LogprobGradArgs& a, int64_t r) {
        const int64_t t = a.targets[r];
        lse = a.lse[r];
        none = lse == -INFINITY;
        target = t >= 0 && t < a.vocab && !none ? t : -1;
        g = target >= 0 ? a.g_logprobs[r] : 0.0f;
        ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
        H = a.g_entropy ? a.entropy[r] : 0.0f;
    }
    __device__ __forceinline__ float at(float x, int64_t j) const {
        const float lp = x - lse, p = none ? 0.0f : __builtin_amdgcn_exp2f(lp * LOG2E);
        const float w = __builtin_fmaf(ge, fmaxf(lp, -1e4f) + H, g);  // p is 0 below: no 0 * inf
        return (j == target ? g : 0.0f) - p * w;
    }
};

constexpr int LG_CHUNKS = 4;  // 16-byte chunks of a thread

// Rows of x and grad that share their alignment: a workgroup takes 1024 chunks of a row.  Bound by HBM: 8192
// rows of 32000 bfloat16 logits 180 us, 5.8 TB/s read and written (element by element 404 us).
template <class E>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogprobGradArgs a) {
    constexpr int N = Chunk<E>::N;
    const int64_t r = blockIdx.y + (int64_t)blockIdx.z * 65535;
    if (r >= a.rows) return;
    const Row<E> row(static_cast<const typename E::T*>(a.x) + r * a.ldx, a.vocab);
    typename E::T* y = static_cast<typename E::T*>(a.grad) + r * a.ldg;
    const int q0 = blockIdx.x * (256 * LG_CHUNKS) + threadIdx.x;
    u4v w[LG_CHUNKS];
#pragma unroll
    for (int u = 0; u < LG_CHUNKS; ++u) {
        const int q = q0 + 256 * u;
        if (q < row.chunks && row.full(q)) w[u] = row.load(q);
    }
    const GradRow gr(a, r);
#pragma unroll
    for (int u = 0; u < LG_CHUNKS; ++u) {
        const int q = q0 + 256 * u;
        if (q >= row.chunks) break;
        const int j0 = row.first(q);
        if (row.full(q)) {
            const Chunk<E> c = widen<E>(w[u]);
            float o[N];
#pragma unroll
            for (int e = 0; e < N; ++e) o[e] = gr.at(c.v[e], j0 + e);
            u4v p;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (E::code == LQ_F32) p[i] = __builtin_bit_cast(uint32_t, o[i]);
                else p[i] = pack2(E{}, o[2 * i], o[2 * i + 1]);
            }
            __builtin_nontemporal_store(p, reinterpret_cast<u4v*>(y + j0));
        } else {
            for (int e = 0; e < N; ++e)
                if (j0 + e >= 0 && j0 + e < row.vocab) y[j0 + e] = E::store(gr.at(E::load(row.x[j0 + e]), j0 + e));
        }
    }
}

// Any alignment, element by element.
template <class E>
__global__ __launch_bounds__(256) void logprobs_grad_any_kernel(LogprobGradArgs a) {
    const int64_t r = workgroup();
    if (r >= a.rows) return;
    const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ldx;
    typename E::T* y = static_cast<typename E::T*>(a.grad) + r * a.ldg;
    const GradRow gr(a, r);
    for (int64_t j = threadIdx.x; j < a.vocab; j += 256) y[j] = E::store(gr.at(E::load(x[j]), j));
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

size_t lq_token_logprobs_workspace_size(int64_t rows, int64_t vocab, int64_t top) {
    if (rows <= 0 || vocab <= 0 || vocab > LP_MAX_VOCAB || top < 0 || top > LP_MAX_TOP) return 0;
    const size_t half = parts_bytes(rows, row_parts(rows, 2 * vocab), top);  // the type is not known here
    const size_t full = parts_bytes(rows, row_parts(rows, 4 * vocab), top);
    return half > full ? half : full;
}

int lq_token_logprobs(const void* d_x, int type, int64_t ldx, int64_t rows, int64_t vocab, const int32_t* d_targets,
                      int64_t top, float* d_logprobs, float* d_entropy, float* d_lse, float* d_top_logprobs,
                      int32_t* d_top_ids, void* d_workspace, size_t workspace_bytes, void* stream) {
    LQ_REQUIRE(is_float_type(type), "lq_token_logprobs: logits must be float32, fp16 or bfloat16");
    LQ_REQUIRE(rows >= 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= LP_MAX_VOCAB && ldx >= vocab,
               "lq_token_logprobs: bad shape");
    LQ_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab,
               "lq_token_logprobs: at most 64 alternatives, and no more than the vocabulary holds");
    if (rows == 0) return LQ_OK;
    LQ_REQUIRE(d_x && (d_targets || !d_logprobs) && (top == 0 || (d_top_logprobs && d_top_ids)),
               "lq_token_logprobs: NULL pointer");
    const int parts = row_parts(rows, vocab * elem_size(type));
    LQ_REQUIRE(parts == 1 || (d_workspace && aligned16(d_workspace) && workspace_bytes >= parts_bytes(rows, parts, top)),
               "lq_token_logprobs: workspace too small or not 16-byte aligned");
    PartSums* sums = parts > 1 ? static_cast<PartSums*>(d_workspace) : nullptr;
    const LogprobArgs a{d_x, ldx, rows, vocab, d_targets, (int)top, d_logprobs, d_entropy, d_lse, d_top_logprobs,
                        d_top_ids, parts, sums, parts > 1 ? reinterpret_cast<uint64_t*>(sums + rows * parts) : nullptr};
    note_path(parts > 1 ? "logprobs parts" : "logprobs rows");
    with_float(type, [&](auto e) {
        using E = decltype(e);
        const dim3 grid = grid_of(rows * parts);
        const hipStream_t st = as_stream(stream);
        const int64_t chunks = vocab * (int64_t)sizeof(typename E::T) / 16;
        if (chunks <= 256) hipLaunchKernelGGL((logprobs_kernel<64, E>), grid, dim3(64), 0, st, a);
        else if (chunks <= 1024) hipLaunchKernelGGL((logprobs_kernel<256, E>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((logprobs_kernel<512, E>), grid, dim3(512), 0, st, a);
        if (parts > 1) hipLaunchKernelGGL((logprobs_join_kernel<E>), dim3((unsigned)rows), dim3(256), 0, st, a);
    });
    return launch_status("lq_token_logprobs");
}

int lq_token_logprobs_backward(const void* d_x, int type, int64_t ldx, int64_t rows, int64_t vocab,
                               const int32_t* d_targets, const float* d_lse, const float* d_entropy,
                               const float* d_g_logprobs, const float* d_g_entropy, void* d_grad, int64_t ldg,
                               void* stream) {
    LQ_REQUIRE(is_float_type(type), "lq_token_logprobs_backward: logits must be float32, fp16 or bfloat16");
    LQ_REQUIRE(rows >= 0 && rows <= 0x7fffffff && vocab > 0 && vocab <= LP_MAX_VOCAB && ldx >= vocab && ldg >= vocab,
               "lq_token_logprobs_backward: bad shape");
    if (rows == 0) return LQ_OK;
    LQ_REQUIRE(d_x && d_targets && d_lse && d_g_logprobs && d_grad && (d_entropy || !d_g_entropy),
               "lq_token_logprobs_backward: NULL pointer");
    LQ_REQUIRE(d_grad != d_x || ldg == ldx, "lq_token_logprobs_backward: in place needs equal strides");
    const LogprobGradArgs a{d_x, ldx, rows, vocab, d_targets, d_lse, d_entropy, d_g_logprobs, d_g_entropy, d_grad, ldg};
    with_float(type, [&](auto e) {
        using E = decltype(e);
        constexpr int64_t S = sizeof(typename E::T), N = 16 / S;
        const hipStream_t st = as_stream(stream);
        if (((reinterpret_cast<uintptr_t>(d_x) - reinterpret_cast<uintptr_t>(d_grad)) & 15) == 0 &&
            (ldx - ldg) * S % 16 == 0) {
            const int64_t span = (vocab + 2 * (N - 1)) / N;  // chunks of a row at most
            const dim3 grid((unsigned)((span + 256 * LG_CHUNKS - 1) / (256 * LG_CHUNKS)),
                            (unsigned)(rows < 65535 ? rows : 65535), (unsigned)((rows + 65534) / 65535));
            hipLaunchKernelGGL((logprobs_grad_kernel<E>), grid, dim3(256), 0, st, a);
        } else {
            hipLaunchKernelGGL((logprobs_grad_any_kernel<E>), grid_of(rows), dim3(256), 0, st, a);
        }
    });
    return launch_status("lq_token_logprobs_backward");
}

}  // extern "C"
