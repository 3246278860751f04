// lq_rms.hip -- root-mean-square norm of rows with the residual's addition, out as floats or as 8-bit codes
// with a scale per row (the rows of a W8A8 product).
//
//   h = x + res (rounded to x's type, stored);  y = h / sqrt(mean h^2 + eps) * gamma;
//   codes: scale = max|y| / 127, code = rne(y * 127 / max|y|).
//
// A row stays in registers: x and the residual are read once, the sum and the output written once, and
// nothing else moves.  Bound by HBM: 4097 rows of 4096 in bfloat16 with a residual, 8-bit rows out, 23 us (5.1 TB/s read
// and written), 16384 rows of 8192 151 us (6.2); 8 rows of 512 take the 3 us of any launch.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include "lq_paged.h"

namespace lq {
namespace {

struct RmsArgs {
    const void *x, *res;
    void* sum;
    int64_t ldx, ldres, ldsum;
    const void* gamma;
    int gamma_type;
    float eps;
    int64_t rows;
    int D;
    void* y;
    int y_type;  // LQ_I8: codes
    int64_t ldy;
    float* scales;
};

__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
    if (type == LQ_F32) return static_cast<const float*>(p)[i];
    if (type == LQ_F16) return ElemF16::load(static_cast<const _Float16*>(p)[i]);
    return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int type, int64_t i, float v) {
    if (type == LQ_F32) static_cast<float*>(p)[i] = v;
    else if (type == LQ_F16) static_cast<_Float16*>(p)[i] = ElemF16::store(v);
    else static_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(v);
}

// Eight values that every row reads: kept in the caches.
template <class E>
__device__ __forceinline__ void load8_shared(const void* p, int d, float (&g)[8]) {
    const typename E::T* q = static_cast<const typename E::T*>(p) + d;
    if constexpr (E::code == LQ_F32) {
        const vf4 lo = reinterpret_cast<const vf4*>(q)[0], hi = reinterpret_cast<const vf4*>(q)[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            g[j] = lo[j];
            g[j + 4] = hi[j];
        }
    } else {
        const u4v w = *reinterpret_cast<const u4v*>(q);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f2v u = unpack2(E{}, w[j]);
            g[2 * j] = u[0];
            g[2 * j + 1] = u[1];
        }
    }
}

// Sum / maximum over the threads of a row.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = ln_wave_sum(v);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
        for (int w = 0; w < TPR / 64; ++w) v += red[w];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ int32_t row_max(int32_t v, float* red) {
    v = wave_max(v);
    if constexpr (TPR > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __int_as_float(v);
        __syncthreads();
        for (int w = 0; w < TPR / 64; ++w) v = max(v, __float_as_int(red[w]));
    }
    return v;
}

// The factors of a row: y = ldexp(h, shift) * r.  Squares of a row that leave float32's range are summed again of
// values scaled by a power of two.  sum(f): the row's sum of f(h)^2; top: its largest magnitude.
struct RowNorm {
    float r;
    int shift;
};
template <class Sum, class Top>
__device__ __forceinline__ RowNorm row_norm(float squares, float D, float eps, Sum sum, Top top) {
    const float ms = squares / D;
    if (ms < 1e30f && ms + eps > 1e-30f) return {1.0f / sqrtf(ms + eps), 0};
    if (ms != ms) return {ms, 0};  // NaN
    const int32_t m = top();
    const int e = max((m >> 23) - 127, -60);  // infinities: 128
    return {1.0f / sqrtf(sum(-e) / D + ldexpf(eps, -2 * e)), -e};
}

// TPR threads to a row of at most 8 TPR CH values, in registers.  VEC: chunks of eight values, 16 bytes and more a
// load; else single values, TPR apart, for rows of odd lengths or strides.
template <int TPR, int CH, bool VEC, class E>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_kernel(RmsArgs a) {
    constexpr int BLOCK = TPR < 256 ? 256 : TPR, N = 8 * CH;
    __shared__ float red[BLOCK / 64];
    const int tid = threadIdx.x % TPR;
    const int64_t row = workgroup() * (BLOCK / TPR) + threadIdx.x / TPR;
    if (row >= a.rows) return;  // whole waves; a workgroup of more than one wave to a row has one row
    const int D = a.D;
    auto place = [&](int k) { return VEC ? 8 * (tid + TPR * (k >> 3)) + (k & 7) : tid + TPR * k; };
    const typename E::T* x = static_cast<const typename E::T*>(a.x) + row * a.ldx;
    const typename E::T* res = a.res ? static_cast<const typename E::T*>(a.res) + row * a.ldres : nullptr;
    typename E::T* sum = a.sum ? static_cast<typename E::T*>(a.sum) + row * a.ldsum : nullptr;
    float h[N];
    if constexpr (VEC) {
        float o[N];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int d = place(8 * c);
            float u[8] = {}, w[8] = {};
            if (d < D) {
                load8<E>(x + d, u);
                if (res) load8<E>(res + d, w);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[8 * c + j] = u[j];
                o[8 * c + j] = w[j];
            }
        }
        if (res) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int d = place(8 * c);
                if constexpr (E::code == LQ_F32) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[8 * c + j] += o[8 * c + j];
                    if (sum && d < D) {
                        *reinterpret_cast<vf4*>(sum + d) = vf4{h[8 * c], h[8 * c + 1], h[8 * c + 2], h[8 * c + 3]};
                        *reinterpret_cast<vf4*>(sum + d + 4) = vf4{h[8 * c + 4], h[8 * c + 5], h[8 * c + 6], h[8 * c + 7]};
                    }
                } else {
                    u4v p;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[j] = pack2(E{}, h[8 * c + 2 * j] + o[8 * c + 2 * j], h[8 * c + 2 * j + 1] + o[8 * c + 2 * j + 1]);
                        const f2v u = unpack2(E{}, p[j]);
                        h[8 * c + 2 * j] = u[0];
                        h[8 * c + 2 * j + 1] = u[1];
                    }
                    if (sum && d < D) *reinterpret_cast<u4v*>(sum + d) = p;
                }
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int d = place(k);
            h[k] = 0.0f;
            if (d < D) {
                h[k] = E::load(x[d]);
                if (res) {
                    const typename E::T s = E::store(h[k] + E::load(res[d]));
                    if (sum) sum[d] = s;
                    h[k] = E::load(s);
                }
            }
        }
    }
    auto squares = [&](int shift) {
        float s[4] = {};
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float v = shift ? ldexpf(h[k], shift) : h[k];
            s[k & 3] = __builtin_fmaf(v, v, s[k & 3]);
        }
        return row_sum<TPR>((s[0] + s[1]) + (s[2] + s[3]), red);
    };
    const RowNorm n = row_norm(squares(0), (float)D, a.eps, squares, [&] {
        int32_t t = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) t = max(t, magnitude(h[k]));
        return row_max<TPR>(t, red);
    });
    if (n.shift)
#pragma unroll
        for (int k = 0; k < N; ++k) h[k] = ldexpf(h[k], n.shift);
    int32_t top = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        float g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = 1.0f;
        if (a.gamma) {
            const int d = place(8 * c);
            if constexpr (VEC) {
                if (d < D) {
                    if (a.gamma_type == LQ_F32) load8_shared<ElemF32>(a.gamma, d, g);
                    else if (a.gamma_type == LQ_F16) load8_shared<ElemF16>(a.gamma, d, g);
                    else load8_shared<ElemBF16>(a.gamma, d, g);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (place(8 * c + j) < D) g[j] = load_any(a.gamma, a.gamma_type, place(8 * c + j));
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[8 * c + j] = h[8 * c + j] * n.r * g[j];
            top = max(top, magnitude(h[8 * c + j]));
        }
    }
    if (a.y_type == LQ_I8) {
        // places past the row hold 0, or NaN where the row has an infinity
        const RowScale rs(row_max<TPR>(top, red));
        int8_t* q = static_cast<int8_t*>(a.y) + row * a.ldy;
        if (tid == 0) a.scales[row] = rs.scale;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if constexpr (VEC) {
                if (place(8 * c) < D) {
                    u2v w = {0, 0};
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j >> 2] |= (uint32_t)(rs.code(h[8 * c + j]) & 0xff) << (8 * (j & 3));
                    *reinterpret_cast<u2v*>(q + place(8 * c)) = w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (place(8 * c + j) < D) q[place(8 * c + j)] = (int8_t)rs.code(h[8 * c + j]);
            }
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if constexpr (VEC) {
            const int64_t at = row * a.ldy + place(8 * c);
            if (place(8 * c) < D) {
                if (a.y_type == LQ_F32) {
                    vf4* o = reinterpret_cast<vf4*>(static_cast<float*>(a.y) + at);
                    o[0] = vf4{h[8 * c], h[8 * c + 1], h[8 * c + 2], h[8 * c + 3]};
                    o[1] = vf4{h[8 * c + 4], h[8 * c + 5], h[8 * c + 6], h[8 * c + 7]};
                } else {
                    u4v p;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        p[j] = a.y_type == LQ_F16 ? pack2(ElemF16{}, h[8 * c + 2 * j], h[8 * c + 2 * j + 1])
                                                  : pack2(ElemBF16{}, h[8 * c + 2 * j], h[8 * c + 2 * j + 1]);
                    *reinterpret_cast<u4v*>(static_cast<uint16_t*>(a.y) + at) = p;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (place(8 * c + j) < D) store_any(a.y, a.y_type, row * a.ldy + place(8 * c + j), h[8 * c + j]);
        }
    }
}

// Rows that registers do not hold: read again on each pass, from the stored sum where there is one (each thread
// reads the places that it wrote).
template <class E>
__global__ __launch_bounds__(512) void rms_wide_kernel(RmsArgs a) {
    constexpr int TPR = 512;
    __shared__ float red[TPR / 64];
    const int64_t row = workgroup();
    if (row >= a.rows) return;
    const int D = a.D, tid = threadIdx.x;
    const typename E::T* x = static_cast<const typename E::T*>(a.x) + row * a.ldx;
    const typename E::T* res = a.res ? static_cast<const typename E::T*>(a.res) + row * a.ldres : nullptr;
    typename E::T* sum = a.sum ? static_cast<typename E::T*>(a.sum) + row * a.ldsum : nullptr;
    if (res && sum) {
        for (int d = tid; d < D; d += TPR) sum[d] = E::store(E::load(x[d]) + E::load(res[d]));
        x = sum;
        res = nullptr;
    }
    auto value = [&](int d) {
        const float v = E::load(x[d]);
        return res ? E::load(E::store(v + E::load(res[d]))) : v;
    };
    auto squares = [&](int shift) {
        float s = 0.0f;
        for (int d = tid; d < D; d += TPR) {
            const float v = ldexpf(value(d), shift);
            s = __builtin_fmaf(v, v, s);
        }
        return row_sum<TPR>(s, red);
    };
    const RowNorm n = row_norm(squares(0), (float)D, a.eps, squares, [&] {
        int32_t t = 0;
        for (int d = tid; d < D; d += TPR) t = max(t, magnitude(value(d)));
        return row_max<TPR>(t, red);
    });
    auto out = [&](int d) {
        return ldexpf(value(d), n.shift) * n.r * (a.gamma ? load_any(a.gamma, a.gamma_type, d) : 1.0f);
    };
    if (a.y_type != LQ_I8) {
        for (int d = tid; d < D; d += TPR) store_any(a.y, a.y_type, row * a.ldy + d, out(d));
        return;
    }
    int32_t top = 0;
    for (int d = tid; d < D; d += TPR) top = max(top, magnitude(out(d)));
    const RowScale rs(row_max<TPR>(top, red));
    if (tid == 0) a.scales[row] = rs.scale;
    int8_t* q = static_cast<int8_t*>(a.y) + row * a.ldy;
    for (int d = tid; d < D; d += TPR) q[d] = (int8_t)rs.code(out(d));
}

// Values of a row in registers.  Threads to a row, kernel us, bfloat16, few rows / many (8-bit rows from 4096 dims):
//   dims    rows         threads (chunks of eight each)
//    512    8 / 4096     64 (1): 2.9 / 5.0     256 (1): 3.2 / 7.6
//   1024    8 / 8192     64 (2): 3.3 / 13.4    256 (1): 3.3 / 16.6
//   2048    8 / 4096     64 (4): 4.6 / 13.1    256 (1): 3.4 / 14.4
//   4096    8 / 4097     64 (8): 6.9 / 26.5    256 (2): 4.0 / 23.1    512 (1): 3.5 / 24.0
//   8192    - / 4096    256 (4): 42.6          512 (2): 41.0         1024 (1): 51.6
//  16384    8 / 2048    256 (8): 7.6 / 48.0    512 (4): 5.5 / 44.7   1024 (2): 4.6 / 43.0
// (not 1024: a launch of 2^22 such workgroups and more would pass 2^32 threads)
constexpr int RMS_MAX = 16384;

int rms_launch(const RmsArgs& a, int type, hipStream_t st, const char* name) {
    const uintptr_t ends = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.res) |
                           reinterpret_cast<uintptr_t>(a.sum) | reinterpret_cast<uintptr_t>(a.gamma) |
                           reinterpret_cast<uintptr_t>(a.y);
    const int64_t e = elem_size(type), ye = elem_size(a.y_type);
    const int64_t strides = (a.ldx * e) | (a.res ? a.ldres * e : 0) | (a.sum ? a.ldsum * e : 0) |
                            (a.y_type == LQ_I8 ? 2 * a.ldy : a.ldy * ye);
    const bool vec = a.D % 8 == 0 && (ends & 15) == 0 && (strides & 15) == 0;
    with_float(type, [&](auto s) {
        using E = decltype(s);
        auto go = [&](auto tpr, auto ch) {
            constexpr int TPR = decltype(tpr)::value, CH = decltype(ch)::value, PER = TPR < 256 ? 256 / TPR : 1;
            const dim3 grid = grid_of((a.rows + PER - 1) / PER), block(TPR < 256 ? 256 : TPR);
            if (vec) hipLaunchKernelGGL((rms_kernel<TPR, CH, true, E>), grid, block, 0, st, a);
            else hipLaunchKernelGGL((rms_kernel<TPR, CH, false, E>), grid, block, 0, st, a);
        };
        const std::integral_constant<int, 64> t64{};
        const std::integral_constant<int, 256> t256{};
        const std::integral_constant<int, 512> t512{};
        const std::integral_constant<int, 4> c4{};
        const std::integral_constant<int, 1> c1{};
        const std::integral_constant<int, 2> c2{};
        note_path(a.D > RMS_MAX ? "rms wide" : vec ? "rms" : "rms single");
        if (a.D <= 512) go(t64, c1);
        else if (a.D <= 1024) go(t64, c2);
        else if (a.D <= 2048) go(t256, c1);
        else if (a.D <= 4096) go(t256, c2);
        else if (a.D <= 8192) go(t512, c2);
        else if (a.D <= RMS_MAX) go(t512, c4);
        else hipLaunchKernelGGL((rms_wide_kernel<E>), grid_of(a.rows), dim3(512), 0, st, a);
    });
    return launch_status(name);
}

// What both entry points ask of the arguments they share; 1: there is nothing to do.
int rms_check(const RmsArgs& a, int type, int64_t D, const std::string& name) {
    LQ_REQUIRE(is_float_type(type) && (!a.gamma || is_float_type(a.gamma_type)),
               name + ": x and gamma must be float32, fp16 or bfloat16");
    LQ_REQUIRE(a.rows >= 0 && D > 0 && D <= (1 << 30) && a.ldx >= D && a.ldy >= D && (!a.res || a.ldres >= D) &&
                   (!a.sum || a.ldsum >= D),
               name + ": bad shape");
    LQ_REQUIRE(a.eps > 0.0f && a.eps < INFINITY, name + ": eps must be positive and finite");
    if (a.rows == 0) return 1;
    LQ_REQUIRE(a.x && a.y && (a.y_type != LQ_I8 || a.scales), name + ": NULL pointer");
    LQ_REQUIRE((a.sum != a.x || a.ldsum == a.ldx) && (a.sum != a.res || a.ldsum == a.ldres),
               name + ": a sum in place has its operand's stride");
    LQ_REQUIRE(a.y != a.x && a.y != a.res && a.y != a.sum, name + ": the output must be apart from x, res and sum");
    return LQ_OK;
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

int lq_rms_norm(const void* d_x, int type, int64_t ldx, const void* d_res, int64_t ldres, void* d_sum, int64_t ldsum,
                const void* d_gamma, int gamma_type, float eps, int64_t rows, int64_t D, void* d_y, int y_type,
                int64_t ldy, void* stream) {
    LQ_REQUIRE(is_float_type(y_type), "lq_rms_norm: y must be float32, fp16 or bfloat16");
    const RmsArgs a{d_x, d_res, d_res ? d_sum : nullptr, ldx, ldres, ldsum, d_gamma, gamma_type, eps, rows, (int)D,
                    d_y, y_type, ldy, nullptr};
    if (const int rc = rms_check(a, type, D, "lq_rms_norm")) return rc < 0 ? rc : LQ_OK;
    return rms_launch(a, type, as_stream(stream), "lq_rms_norm");
}

int lq_rms_norm_quantize(const void* d_x, int type, int64_t ldx, const void* d_res, int64_t ldres, void* d_sum,
                         int64_t ldsum, const void* d_gamma, int gamma_type, float eps, int64_t rows, int64_t D,
                         int8_t* d_codes, int64_t ldc, float* d_scales, void* stream) {
    const RmsArgs a{d_x, d_res, d_res ? d_sum : nullptr, ldx, ldres, ldsum, d_gamma, gamma_type, eps, rows, (int)D,
                    d_codes, LQ_I8, ldc, d_scales};
    if (const int rc = rms_check(a, type, D, "lq_rms_norm_quantize")) return rc < 0 ? rc : LQ_OK;
    return rms_launch(a, type, as_stream(stream), "lq_rms_norm_quantize");
}

}  // extern "C"
