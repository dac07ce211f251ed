// Attention of sequences that begin alike: what the kernels in attention_shared.hip are given.
#pragma once

#include "attention.hpp"

namespace sngguf {

constexpr int kSharedUnit = 128;     // common keys are taken in multiples of every kernel's key tile

// One of the launches that compute partial results: common keys of many rows; few rows, of common keys (where there is no first) and of
// sequences; many rows of sequences
struct SharedLaunch {
    int32_t row_shift, key_shift;    // 2^row_shift rows and 2^key_shift keys of a tile
    int32_t max_rows;                // of the sequences that the second takes; the third takes the others
    int32_t want, least;             // workgroups that run at once (0: keys are not split); key tiles of a split at least
    int32_t slots;                   // workgroups of a key / value head
    AttentionEntry* map;             // [slots]: what each does
    float* partial;
};
constexpr int kSharedLaunches = 3;

struct SharedArgs {
    AttentionArgs a;                 // lengths, tensors
    const int32_t* groups;           // [group_count + 1]
    const int32_t* shared;           // [group_count]
    int32_t group_count;
    AttentionEntry* entries;         // [groups, then sequences]
    int32_t* sequence_of;            // [tokens_q], or NULL: token t is sequence t
    SharedLaunch launch[kSharedLaunches];
};

int launch_shared_plan(const SharedArgs& s, hipStream_t stream);
int launch_shared_join(const SharedArgs& s, int dim, hipStream_t stream);

}  // namespace sngguf
