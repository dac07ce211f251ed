// Attention of sequences that begin alike: what the kernels in attention_shared.hip are given.
#pragma once

#include "attention.hpp"

namespace sngguf {

constexpr int kSharedUnit = 128;     // common keys are taken in multiples of every kernel's key tile

// One of the launches that compute partial results: the common keys', the single tokens', the chunks'
struct SharedLaunch {
    int32_t rows, keys;              // of a tile
    int32_t min_rows, max_rows;      // of the sequences that it takes
    int32_t want, least;             // workgroups aimed at where keys are split; key tiles of a split at least
    int32_t split;
    int32_t slots;                   // workgroups of a key / value head
    int32_t* map;                    // [slots]
    float* partial;
};
constexpr int kSharedLaunches = 3;

struct SharedArgs {
    AttentionArgs a;                 // lengths, tensors
    const int32_t* groups;           // [group_count + 1]
    const int32_t* shared;           // [group_count]
    int32_t group_count;
    AttentionEntry* entries;         // [groups, then sequences]
    int32_t* group_of;               // [sequences]: group with common keys, or -1
    int32_t* sequence_of;            // [tokens_q], or NULL: token t is sequence t
    SharedLaunch launch[kSharedLaunches];
};

int launch_shared_plan(const SharedArgs& s, hipStream_t stream);
int launch_shared_join(const SharedArgs& s, int dim, hipStream_t stream);

}  // namespace sngguf
