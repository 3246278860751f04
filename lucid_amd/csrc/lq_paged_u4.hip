// lq_paged_u4.hip -- attention of one new token per sequence over pages that hold 4 bits a value.
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>

#include <algorithm>

#include "lq_paged_u4.h"
#include "lq_u4.h"

namespace lq {
namespace {

// One wave per (sequence, query head), a position at a time: the formula as it stands.
template <class Q>
__global__ __launch_bounds__(64) void paged_u4_simple_kernel(PagedArgs a) {
    const int lane = threadIdx.x, hd = a.hd, G = hd / U4_GROUP;
    for (int64_t n = blockIdx.x; n < (int64_t)a.B * a.H; n += gridDim.x) {
        const int b = (int)(n / a.H), h = (int)(n - (int64_t)b * a.H), hk = h / a.group;
        bool over, bad = false;
        const int len = sequence_length(a, b, over);
        float q[4], acc[4] = {}, m = -INFINITY, l = 0.0f;
        for (int j = 0; j < 4; ++j) {
            const int d = lane + 64 * j;
            q[j] = d < hd ? Q::load(static_cast<const typename Q::T*>(a.q)[b * a.ldq + (int64_t)h * hd + d]) : 0.0f;
        }
        for (int p = 0; p < len; ++p) {
            const int64_t row0 = position_row(p, a.table + (int64_t)b * a.table_stride, a.table_stride, a.pages, a.Hkv, a.page);
            if (row0 < 0) {
                bad = true;
                break;
            }
            const int64_t row = row0 + (int64_t)hk * a.page;
            auto value = [&](const void* pages, const void* meta, int groups, int d) {
                const uint8_t c = static_cast<const uint8_t*>(pages)[row * (hd / 2) + d / 2];
                const uint16_t* s = static_cast<const uint16_t*>(meta) + row * 2 * groups;
                const int g = d / (hd / groups);
                return __builtin_fmaf((float)(d & 1 ? c >> 4 : c & 15), bf16_bits_to_f32(s[g]), bf16_bits_to_f32(s[groups + g]));
            };
            float s = 0.0f, v[4];
            for (int j = 0; j < 4; ++j) {
                const int d = lane + 64 * j;
                v[j] = 0.0f;
                if (d >= hd) continue;
                s = __builtin_fmaf(q[j], value(a.k, a.ks, G, d), s);
                v[j] = value(a.v, a.vs, 1, d);
            }
            s = ln_wave_sum(s) * a.scale * LOG2E;
            const float mn = s > m ? s : m, base = mn == -INFINITY ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - base), e = __builtin_amdgcn_exp2f(s - base);
            m = mn;
            l = l * f + e;
            for (int j = 0; j < 4; ++j) acc[j] = acc[j] * f + e * v[j];
        }
        for (int j = 0; j < 4; ++j) {
            const int d = lane + 64 * j;
            if (d >= hd) continue;
            const float y = bad || over || (len > 0 && a.pages == 0) ? __builtin_nanf("") : len > 0 ? acc[j] / l : 0.0f;
            const int64_t at = n * hd + d;
            if (a.out_f32) static_cast<float*>(a.out)[at] = y;
            else static_cast<typename Q::T*>(a.out)[at] = Q::store(y);
        }
    }
}

}  // namespace

void paged_u4_launch(const PagedArgs& a, int q_type, dim3 grid, hipStream_t st) {
    with_half(q_type, [&](auto q) {
        using Q = decltype(q);
        hipLaunchKernelGGL((paged_u4_simple_kernel<Q>), dim3((unsigned)std::min<int64_t>((int64_t)a.B * a.H, 1 << 20)),
                           dim3(64), 0, st, a);
    });
}

}  // namespace lq
