// Arguments of the kernels in page_tables.hip.
#pragma once

#include "sngguf_common.hpp"

namespace sngguf {

struct PageSequence {        // of a step
    int32_t length, after;   // tokens before it and behind it
    int32_t pages, ring_at;  // pages before it; place in the ring of the first it gets
};

struct PageArgs {
    int32_t *pages, *lens, *held, *free;
    int64_t* cursor;
    int64_t sequences, tokens;
    int32_t width, ring, page_shift;
    // append
    const int32_t* added;
    int32_t *ends, *lens_out, *missing;
    int64_t *cursor_out, *positions, *slots;
    PageSequence* of;        // [sequences], scratch of the two-launch form
    // release, fork
    const uint8_t* done;
    const int32_t *parent, *common;
};

constexpr int64_t kOneLaunchSequences = 1024, kOneLaunchTokens = 4096;

int launch_page_append(const PageArgs& a, bool one, hipStream_t stream);
int launch_page_release(const PageArgs& a, hipStream_t stream);
int launch_page_fork(const PageArgs& a, hipStream_t stream);

}  // namespace sngguf
