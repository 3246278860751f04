// lq_paged_u4.h -- the append with rotation and the attention over 4-bit pages, for the entry points of lq_paged.hip.
#pragma once

#include "lq_paged.h"

namespace lq {

// lq_paged_kv_append_rotary, errors under `name` (lq_rotary.hip).
int paged_append_rotary(const char* name, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldkv,
                        int src_type, int64_t tokens, const int32_t* starts, int64_t seqs, int64_t H, int64_t Hkv,
                        int64_t hd, const float* angles, int64_t positions, int64_t rot, int interleaved,
                        const int32_t* table, int64_t table_stride, const int32_t* lengths, void* q_out, int64_t ldqo,
                        void* k_out, int64_t ldko, int q_type, void* k_pages, void* v_pages, int cache_type,
                        void* k_scale, void* v_scale, int64_t pages, int64_t page, void* stream);

// The kernel of attention over 4-bit pages (lq_paged_u4.hip); few: a few short sequences, one workgroup each.
void paged_u4_launch(const PagedArgs& a, int q_type, bool few, dim3 grid, hipStream_t st);

}  // namespace lq
