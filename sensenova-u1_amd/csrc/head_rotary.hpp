// Arguments of the kernel in head_rotary.hip.
#pragma once

#include "rotary_cache.hpp"

namespace sngguf {

constexpr int kMostParts = 4;

// Norm of single heads: parts of a head that each have a root mean square of their own
struct HeadNormArgs {
    const void* weight[kMostParts];      // 16-byte aligned
    int32_t elements[kMostParts];        // multiples of 8; behind the last part: 0
    float one_over[kMostParts];          // 1 / elements
    int32_t parts;                       // 0: none
    int32_t bf16;                        // weights are bf16, else fp32
    float eps;
};

struct HeadRotaryArgs : RotaryCacheArgs {
    const int32_t* axis;                 // [pairs], or NULL: all the first
    int32_t axes;
    int64_t axis_stride;                 // from a token's position to its next one
    int32_t parts, part[kMostParts];     // elements, together 2 x pairs
    int32_t lane_shift;                  // 2^lane_shift lanes have a head
    HeadNormArgs q_norm, k_norm;
};

int launch_head_rotary(const HeadRotaryArgs& a, int cache, hipStream_t stream);

}  // namespace sngguf
