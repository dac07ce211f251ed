// Arguments of the kernels in rotary_cache.hip.
#pragma once

#include "sngguf_common.hpp"

namespace sngguf {

struct RotaryCacheArgs {
    // rotation (turns NULL: none)
    const double* turns;
    double magnitude;
    const int64_t* positions;
    int32_t pairs, interleaved;
    // rows [tokens][heads][dim], strides in elements
    const bf16_t *q, *k, *v;
    bf16_t *q_out, *k_out, *v_out;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, q_out_token, q_out_head, k_out_token, k_out_head;
    int64_t tokens;
    int32_t q_heads, k_heads, dim;
    int32_t wide;             // every row of every tensor starts at a 16-byte boundary
    int32_t tokens_per_block;
    // cache
    void *k_pages, *v_pages;
    uint16_t *k_scales, *v_scales;
    const int64_t* slots;
    int64_t slot_count;       // pages x page size
    int32_t page_shift, kv_heads;
};

int launch_rotary_cache(const RotaryCacheArgs& a, int cache, hipStream_t stream);
int launch_cache_read(const RotaryCacheArgs& a, bool q8, hipStream_t stream);

}  // namespace sngguf
