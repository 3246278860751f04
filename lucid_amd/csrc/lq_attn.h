// lq_attn.h -- element types and row rules shared by the paged and the packed attention kernels
// and the log-probability kernels.
#pragma once

#include "lq_internal.h"
#include "lq_place.h"

namespace lq {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

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

// The grid of n workgroups, and a workgroup's place in it (past the end in the last row's rest).
inline dim3 grid_of(int64_t n) {
    const Workgroups w = workgroups(n);
    return dim3(w.x, w.y);
}
__device__ __forceinline__ int64_t workgroup() { return workgroup_index(blockIdx.x, blockIdx.y); }

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

// Eight 16-bit values of either type in four registers, as the matrix instructions take them.
__device__ __forceinline__ f16v mfma_32x32x16(ElemF16, u4v a, u4v b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma_32x32x16(ElemBF16, u4v a, u4v b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}
__device__ __forceinline__ vf4 mfma_16x16x32(ElemF16, u4v a, u4v b, vf4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}
__device__ __forceinline__ vf4 mfma_16x16x32(ElemBF16, u4v a, u4v b, vf4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}
// Two values rounded to nearest even into one register, and back.
__device__ __forceinline__ uint32_t pack2(ElemF16, float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v{a, b}), h2v));
}
__device__ __forceinline__ uint32_t pack2(ElemBF16, float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v{a, b}), b2v));
}
__device__ __forceinline__ f2v unpack2(ElemF16, uint32_t w) {
    return __builtin_convertvector(__builtin_bit_cast(h2v, w), f2v);
}
__device__ __forceinline__ f2v unpack2(ElemBF16, uint32_t w) {
    return f2v{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
}
// A weight that enters a product in 16 bits is 2^WEIGHT_SHIFT times its value relative to the
// running maximum (which may lag by 2^RESCALE_AT): fp16 then resolves weights down to 2^-30 of
// the largest and stays below 2^14.  bfloat16 has float32's exponents, for its values too: the shift
// down keeps the sums of a million values of 1e36, or of 4096 of the type's largest, finite.
template <class E>
constexpr float WEIGHT_SHIFT = E::code == LQ_F16 ? 6.0f : -20.0f;
constexpr float RESCALE_AT = 8.0f;
// The reference of the weights for a largest score mx (log2 units).  In bfloat16 mx to 2^-13: the large shift is
// then exact on it (below 2^11), so that sums with different references stay comparable, and the largest
// weight, 2^-13 from a power of two at most, still rounds to it.
template <class E>
__device__ __forceinline__ float weight_reference(float mx) {
    if constexpr (E::code == LQ_BF16) return fabsf(mx) < 2048.0f ? rintf(mx * 8192.0f) * (1.0f / 8192.0f) : mx;
    return mx;
}

// The larger / the sum of the values that lanes l and l ^ 32 hold.
__device__ __forceinline__ float half_max(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// The largest / the sum of the values that the lanes 16 and 32 apart hold (four lanes).
__device__ __forceinline__ float quarter_max(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return half_max(fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])));
}
__device__ __forceinline__ float quarter_sum(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto p = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return half_sum(__uint_as_float(p[0]) + __uint_as_float(p[1]));
}

// Byte I of a word as a signed integer in float32.
template <int I>
__device__ __forceinline__ float byte_to_f32(uint32_t w) {
    float f;
#define LQ_BYTE(i)                                                                                        \
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_" #i : "=v"(f) : "v"(w))
    if constexpr (I == 0) LQ_BYTE(0);
    if constexpr (I == 1) LQ_BYTE(1);
    if constexpr (I == 2) LQ_BYTE(2);
    if constexpr (I == 3) LQ_BYTE(3);
#undef LQ_BYTE
    return f;
}
// Four int8 codes of a word as two words of 16-bit values, exact in both types.  fp16: the code + 128
// under the exponent of 1024 is 1152 + code; bfloat16: the upper halves of the float32 values (eight
// significant bits hold any code).
__device__ __forceinline__ u2v widen4(ElemF16, uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const h2v bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    const h2v lo = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias;
    const h2v hi = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias;
    return u2v{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
}
__device__ __forceinline__ u2v widen4(ElemBF16, uint32_t w) {
    const uint32_t a = __float_as_uint(byte_to_f32<0>(w)), b = __float_as_uint(byte_to_f32<1>(w));
    const uint32_t c = __float_as_uint(byte_to_f32<2>(w)), d = __float_as_uint(byte_to_f32<3>(w));
    return u2v{__builtin_amdgcn_perm(b, a, 0x07060302u), __builtin_amdgcn_perm(d, c, 0x07060302u)};
}

// Sum of an integer over the wave, the same in every lane, by register permutes (the pairings of
// ln_wave_sum).
__device__ __forceinline__ int wave_add(int v) {
    v += __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, true);   // quad_perm [1,0,3,2]
    v += __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, true);   // quad_perm [2,3,0,1]
    v += __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, true);  // row_half_mirror
    v += __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, true);  // row_mirror
    const auto p16 = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = (int)(p16[0] + p16[1]);
    const auto p32 = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    return (int)(p32[0] + p32[1]);
}

// LDS reads at a byte offset of the workgroup's LDS (written by copies the compiler does not see).
typedef __attribute__((address_space(3))) u4v lds_u4v;
typedef __attribute__((address_space(3))) s4v lds_s4v;
__device__ __forceinline__ u4v lds_read16(uint32_t at) { return *reinterpret_cast<lds_u4v*>(at); }
// Transposing read: of each 16 lanes, lane i points at four values of row i / 4 (columns 4 (i %
// 4) ..) and receives column i of the four rows.
__device__ __forceinline__ u2v lds_read_tr(uint32_t at) {
    return __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s4v*>(at)));
}

constexpr float LOG2E = 1.44269504088896341f;
constexpr float LN2 = 0.693147180559945309f;
constexpr int ATTN_MAX_HD = 256;  // head dims of the attention kernels: multiples of 8 up to this

}  // namespace lq
