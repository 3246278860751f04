// lq_attn.h -- element types and row rules shared by the paged and the packed attention kernels
// and the log-probability kernels.
#pragma once

#include "lq_internal.h"

namespace lq {

typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));

// Storage types: `load` is exact, `store` rounds once to nearest even.
struct ElemF32 {
    typedef float T;
    static constexpr int code = LQ_F32;
    static __device__ __forceinline__ float load(T v) { return v; }
    static __device__ __forceinline__ T store(float v) { return v; }
};
struct ElemF16 {
    typedef _Float16 T;
    static constexpr int code = LQ_F16;
    static __device__ __forceinline__ float load(T v) { return (float)v; }
    static __device__ __forceinline__ T store(float v) { return __builtin_bit_cast(_Float16, f32_to_f16_rn(v)); }
};
struct ElemBF16 {
    typedef uint16_t T;
    static constexpr int code = LQ_BF16;
    static __device__ __forceinline__ float load(T v) { return bf16_bits_to_f32(v); }
    static __device__ __forceinline__ T store(float v) { return f32_to_bf16_bits(v); }
};
struct ElemI8 {
    typedef int8_t T;
    static constexpr int code = LQ_I8;
    static __device__ __forceinline__ float load(T v) { return (float)v; }
};

inline bool is_float_type(int t) { return t == LQ_F32 || t == LQ_F16 || t == LQ_BF16; }
inline bool is_half_type(int t) { return t == LQ_F16 || t == LQ_BF16; }
inline int64_t elem_size(int t) { return t == LQ_F32 ? 4 : t == LQ_I8 ? 1 : 2; }

// f(Elem{}) of a float type code (checked by the caller).
template <class F>
inline void with_float(int t, F f) {
    if (t == LQ_F32) f(ElemF32{});
    else if (t == LQ_F16) f(ElemF16{});
    else f(ElemBF16{});
}
template <class F>
inline void with_half(int t, F f) {
    if (t == LQ_F16) f(ElemF16{});
    else f(ElemBF16{});
}

constexpr float LOG2E = 1.44269504088896341f;
constexpr float LN2 = 0.693147180559945309f;
constexpr int ATTN_MAX_HD = 256;  // head dims of the attention kernels: multiples of 8 up to this

}  // namespace lq
