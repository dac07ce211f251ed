// Attention of new tokens over a paged cache in which groups of sequences begin with the same tokens: what a group has in common
// is read and multiplied once for all of its queries, what a sequence has of its own once for its queries.
//
// With the keys of a query in two sets, C (common) and O (own), and of each set the maximum m, the sum l = sum_j exp2(s_j - m) and the
// vector o = sum_j exp2(s_j - m) v_j:
//     out = (o_C 2^(m_C - m) + o_O 2^(m_O - m)) / (l_C 2^(m_C - m) + l_O 2^(m_O - m)),   m = max(m_C, m_O),
// which is how splits of a sequence are joined as well.  So the common tokens of a group are one more "sequence", whose queries are
// all of the group's and see all of its keys, for the attention kernels that there are; they write partial results, and a join sums each
// query's from both sequences.  Sequences of a group are neighbours, and so are their queries.
//
//  * The plan: lengths lie on the device, so a kernel of one workgroup finds how many tokens each group has in common (no more than
//    its sequences have in front of their new ones, in whole key tiles: what is left over is read as each one's own), deals the work
//    of each launch over its workgroups, and writes down for each of these what it does.  4.8 us, the time of its 900 instructions one after the
//    other.
//  * The join: half a wavefront lies along a query's elements and takes some partial results at a time.  Weights are scaled by 2^-16, so that
//    no sum leaves fp32 whose average does not (there are fewer than 2^16 splits).
// What is rounded is what the attention kernels round, weights in front of the product with the values (to bf16, or fp16 of an 8-bit cache), here by the maximum
// of their own set of keys; partial results and their sums are fp32.  Off by 0.0020 to 0.0023 of its norm in bf16 and 0.0017 in 8 bits, as without groups.
// Measured, 32 query and 8 key / value heads of 128, passes back to back: 64 single tokens over 16384 common keys and 1 to 400 of their own in bf16
// 59 us (sngguf_paged_attention 447): plan, common keys 28 (17 GFLOP in 256-row workgroups of eight key tiles, half of whose time is their start and
// 33 MB of partial results), own keys 14, join 9; 32 over 8192 and up to 900 in 8 bits 43 (73): plan, one launch of 30, join 6.
#include "attention_shared.hpp"

namespace sngguf {

namespace {

constexpr int kThreads = 256;
constexpr int32_t kOwn = 16;            // so many numbers a lane writes by itself, more all lanes of the wavefront
constexpr float kNever = 1e9f;

// The least of the wavefront's numbers (row shifts, then a row's last value handed on; lanes without a partner keep theirs)
__device__ __forceinline__ int32_t wave_min(int32_t x) {
#define SNGGUF_STEP(CONTROL, ROWS) x = min(x, __builtin_amdgcn_update_dpp(x, x, CONTROL, ROWS, 0xF, false));
    SNGGUF_STEP(0x111, 0xF)
    SNGGUF_STEP(0x112, 0xF)
    SNGGUF_STEP(0x114, 0xF)
    SNGGUF_STEP(0x118, 0xF)
    SNGGUF_STEP(0x142, 0xA)
    SNGGUF_STEP(0x143, 0xC)
#undef SNGGUF_STEP
    return __builtin_amdgcn_readlane(x, 63);
}

// Sum over the wavefront, in all lanes
__device__ __forceinline__ float wave_total(float x) {
#define SNGGUF_STEP(CONTROL, ROWS) x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CONTROL, ROWS, 0xF, false));
    SNGGUF_STEP(0x111, 0xF)
    SNGGUF_STEP(0x112, 0xF)
    SNGGUF_STEP(0x114, 0xF)
    SNGGUF_STEP(0x118, 0xF)
    SNGGUF_STEP(0x142, 0xA)
    SNGGUF_STEP(0x143, 0xC)
#undef SNGGUF_STEP
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// What a launch has to do, in a wavefront's entries
struct LaunchSums {
    float work;              // row tiles x key tiles
    uint32_t row_tiles, entries;
};

// An entry's launch (-1: none), its row tiles and key tiles
struct Entry {
    int launch;
    uint32_t row_tiles, key_tiles;
};
__device__ __forceinline__ Entry entry_of(const SharedLaunch* launch, const AttentionEntry& e, int group, bool common) {
    const uint32_t rows = (uint32_t)e.lq * (uint32_t)group;
    Entry x = {-1, 0, 0};
    if (rows == 0 || (common && e.lk == 0)) return x;
    const int l = common ? (launch[0].slots ? 0 : 1) : (int32_t)rows > launch[1].max_rows || launch[1].slots == 0 ? 2 : 1;
    if (launch[l].slots == 0) return x;
    const int row_shift = launch[l].row_shift, key_shift = launch[l].key_shift;
    x.launch = l;
    x.row_tiles = (rows + (1u << row_shift) - 1) >> row_shift;
    const int32_t lo = e.k0 >> key_shift, hi = (int32_t)(((int64_t)e.lk + (1 << key_shift) - 1) >> key_shift);
    x.key_tiles = hi > lo ? hi - lo : 1;
    return x;
}

}  // namespace

// W wavefronts.  ONE: there are no more entries than threads, and what a phase hands to the next stays in LDS and registers.
// It runs through once, on one compute unit, so its time is that of one instruction after the other: sums that do not depend on each other are
// side by side, and what is done once for each launch is done by as many lanes.
template <int W, bool ONE>
__global__ __launch_bounds__(64 * W) void attention_shared_plan_kernel(SharedArgs s) {
    constexpr int T = 64 * W;
    touch_arguments(s);
    __shared__ AttentionEntry held[ONE ? T : 1];
    __shared__ SharedLaunch launch[kSharedLaunches];
    __shared__ LaunchSums sums[W][kSharedLaunches];
    __shared__ uint32_t ups[W][kSharedLaunches];
    const AttentionArgs& a = s.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t groups = s.group_count, sequences = a.sequences;
    const int64_t all = (int64_t)groups + sequences;
    AttentionEntry* entries = ONE ? held : s.entries;         // groups, then sequences; `row` of a sequence: its group with common keys, or -1

    // (the first group's numbers are on their way while lengths are)
    int32_t group_0 = 0, group_1 = 0, group_shared = 0;
    if (wave < groups) group_0 = s.groups[wave], group_1 = s.groups[wave + 1], group_shared = s.shared[wave];
    if (tid < kSharedLaunches) launch[tid] = s.launch[tid];
#pragma unroll 1
    for (int64_t base = 0; base < sequences; base += T) {
        const int64_t i = base + tid;
        AttentionSequence q = {0, 0, 0, 0, 0};
        if (i < sequences) {
            q = attention_sequence(a, (int)i);
            entries[groups + i] = {(int32_t)q.q0, q.lq, 0, q.lk, -1, 1, -1, 0};
        }
        // (tokens of no sequence keep any number, and the join sees that they are not that one's)
        if (!s.sequence_of) continue;
        if (q.lq <= kOwn)
            for (int32_t j = 0; j < q.lq; j++) s.sequence_of[q.q0 + j] = (int32_t)i;
        for (uint64_t many = __ballot(q.lq > kOwn); many; many &= many - 1) {
            const int m = __builtin_ctzll(many);
            const int32_t q0 = __builtin_amdgcn_readlane((int)q.q0, m), lq = __builtin_amdgcn_readlane(q.lq, m), of = __builtin_amdgcn_readlane((int)i, m);
            for (int32_t j = lane; j < lq; j += 64) s.sequence_of[q0 + j] = of;
        }
    }
    __syncthreads();

    // ---- what a group has in common: a wavefront a group -------------------------------------------------------------------
#pragma unroll 1
    for (int64_t g = wave; g < groups; g += W) {
        // (numbers that are no cumulative counts stay within the tensors)
        int32_t e0 = group_0, e1 = group_1;
        const int32_t said = group_shared;
        if (g + W < groups) group_0 = s.groups[g + W], group_1 = s.groups[g + W + 1], group_shared = s.shared[g + W];
        e0 = e0 < 0 ? 0 : e0 > sequences ? sequences : e0;
        e1 = e1 < e0 ? e0 : e1 > sequences ? sequences : e1;
        // sequences without new tokens have no say; the first and the last of the others tell which queries are the group's
        int32_t least = 0x7FFFFFFF, row = -1, q0 = 0, q1 = 0, count = 0;
#pragma unroll 1
        for (int64_t base = e0; base < e1; base += 64) {
            AttentionEntry e = {};
            if (base + lane < e1) e = entries[groups + base + lane];
            const uint64_t live = __ballot(e.lq != 0);
            if (!live) continue;
            const int first = __builtin_ctzll(live), last = 63 - __builtin_clzll(live);
            least = min(least, wave_min(e.lq != 0 ? e.lk - e.lq : 0x7FFFFFFF));
            if (row < 0) row = (int32_t)base + first, q0 = __builtin_amdgcn_readlane(e.q0, first);
            q1 = __builtin_amdgcn_readlane(e.q0 + e.lq, last);
            count += __builtin_popcountll(live);
        }
        int32_t common = said < least ? said : least;
        common = common < 0 || count < 2 || q1 <= q0 ? 0 : common / kSharedUnit * kSharedUnit;
        if (lane == 0) entries[g] = {q0, common ? q1 - q0 : 0, 0, common, row, 1, -1, 0};
        if (common)
#pragma unroll 1
            for (int64_t i = (int64_t)e0 + lane; i < e1; i += 64) {
                entries[groups + i].k0 = common;
                entries[groups + i].row = (int32_t)g;
            }
    }
    __syncthreads();

    AttentionEntry e = {};
    Entry x = {-1, 0, 0};
    if (ONE && tid < all) {
        e = entries[tid];
        x = entry_of(launch, e, a.group, tid < groups);
    }
    // ---- all work of each launch, and how many key tiles of it a workgroup takes ---------------------------------------------
    {
        float work[kSharedLaunches] = {};
        uint32_t tiles[kSharedLaunches] = {}, entries_of[kSharedLaunches] = {};
        auto add = [&](const Entry& y) {
#pragma unroll
            for (int l = 0; l < kSharedLaunches; l++)
                if (l == y.launch) work[l] += (float)y.row_tiles * (float)y.key_tiles, tiles[l] += y.row_tiles, entries_of[l]++;
        };
        if constexpr (ONE) add(x);
        else
            for (int64_t v = tid; v < all; v += T) add(entry_of(launch, entries[v], a.group, v < groups));
#pragma unroll
        for (int l = 0; l < kSharedLaunches; l++) {
            const uint32_t count = wave_total(tiles[l]), some = wave_total(entries_of[l]);
            const float sum = wave_total(work[l]);
            if (lane == 0) sums[wave][l] = {sum, count, some};
        }
    }
    __syncthreads();
    // (lane l has launch l's.)  Workgroups of many rows are one or two a compute unit: as many as run at once.  Splits of c key tiles are at most one
    // more than their fraction for each row tile, so c = work / (workgroups - row tiles) does in any case; a single entry's are as many as fit.
    // Those of few rows are short, and some may follow others: the last split of a row tile is half as long as the others on average.
    float chunk_of = kNever;
    if (lane < kSharedLaunches && launch[lane].want) {
        float sum = 0.f, count = 0.f;
        uint32_t some = 0;
#pragma unroll
        for (int w = 0; w < W; w++) sum += sums[w][lane].work, count += (float)sums[w][lane].row_tiles, some += sums[w][lane].entries;
        const float want = (float)launch[lane].want;
        sum *= (float)a.kv_heads;
        count *= (float)a.kv_heads;
        float at_once = lane == 1 ? fmaxf(want - 0.5f * count, 0.5f * want) : some == 1 ? count * __builtin_floorf(want * __builtin_amdgcn_rcpf(count) * 1.00001f) : want - count;
        if (at_once > 0.f) chunk_of = __builtin_ceilf(fmaxf(sum * __builtin_amdgcn_rcpf(at_once) * 0.99999f, (float)launch[lane].least));
    }

    // ---- which workgroups take an entry ------------------------------------------------------------------------------------
    uint32_t before[kSharedLaunches] = {};
#pragma unroll 1
    for (int64_t base = 0; base < all; base += T) {
        const int64_t v = base + tid;
        if (base) __syncthreads();                               // (the counts of the turn before are read)
        if constexpr (!ONE) {
            x = {-1, 0, 0};
            if (v < all) {
                e = entries[v];
                x = entry_of(launch, e, a.group, v < groups);
            }
        }
        const int mine = x.launch < 0 ? 0 : x.launch;
        const float c = __shfl(chunk_of, mine);
        const uint32_t chunk = c < kNever ? (uint32_t)c : 0x7FFFFFFFu;
        const uint32_t splits = x.key_tiles > chunk ? (x.key_tiles + chunk - 1) / chunk : 1;
        const uint32_t slots = x.row_tiles * splits;             // (no launch: none)
        uint32_t up = 0;
#pragma unroll
        for (int l = 0; l < kSharedLaunches; l++) {
            const uint32_t sum = wave_scan(l == x.launch ? slots : 0);
            if (l == x.launch) up = sum;
            if (lane == 63) ups[wave][l] = sum;
        }
        __syncthreads();
        uint32_t in_front = mine == 0 ? before[0] : mine == 1 ? before[1] : before[2];
#pragma unroll
        for (int w = 0; w < W; w++) {
            if (w < wave) in_front += ups[w][mine];
#pragma unroll
            for (int l = 0; l < kSharedLaunches; l++) before[l] += ups[w][l];
        }
        int32_t count = 0, first = -1;
        if (v < all) {
            const bool common = v < groups;
            const int32_t room = launch[mine].slots;
            count = (int32_t)slots;
            first = (int32_t)(in_front + up) - count;
            e.splits = (int32_t)splits;
            e.flags = x.launch < 0 ? 0
                                   : mine << 8 | (common ? kEntryPartial | (x.row_tiles == 1 ? kEntryOnce : 0)
                                                         : kEntryCausal | kEntryOnce | (splits > 1 || e.row >= 0 ? kEntryPartial : 0));
            // (lengths that are none can need more workgroups than there are: the join passes over them)
            e.first = x.launch < 0 || first < 0 || (int64_t)first + count > room ? -1 : first;
            s.entries[v] = e;
            e.first = first;
            if (!common) e.row = (int32_t)(v - groups);
            if (first < 0 || first >= room) count = 0;
            else if ((int64_t)first + count > room) count = room - first;
            if (count <= kOwn) {
                AttentionEntry* map = launch[mine].map + first;
#pragma unroll 1
                for (int32_t k = 0; k < count; k++) map[k] = e;
            }
        }
#pragma unroll 1
        for (uint64_t many = __ballot(count > kOwn); many; many &= many - 1) {
            const int m = __builtin_ctzll(many), l = __builtin_amdgcn_readlane(mine, m), n = __builtin_amdgcn_readlane(count, m);
            const int32_t f = __builtin_amdgcn_readlane(first, m);
            const AttentionEntry y = {__builtin_amdgcn_readlane(e.q0, m),  __builtin_amdgcn_readlane(e.lq, m),     __builtin_amdgcn_readlane(e.k0, m),    __builtin_amdgcn_readlane(e.lk, m),
                                      __builtin_amdgcn_readlane(e.row, m), __builtin_amdgcn_readlane(e.splits, m), __builtin_amdgcn_readlane(e.first, m), __builtin_amdgcn_readlane(e.flags, m)};
            AttentionEntry* map = launch[l].map + f;
#pragma unroll 1
            for (int32_t k = lane; k < n; k += 64) map[k] = y;
        }
    }
    // workgroups beyond the last: entries without queries
#pragma unroll 1
    for (int l = 0; l < kSharedLaunches; l++) {
        const int32_t room = launch[l].slots;
        AttentionEntry* map = launch[l].map;
#pragma unroll 1
        for (int64_t i = (int64_t)(l == 0 ? before[0] : l == 1 ? before[1] : before[2]) + tid; i < room; i += T) map[i].lq = 0;
    }
}

// A query's partial results summed.  TEAMS half wavefronts have a query, eight or four of them a workgroup, or two (a wavefront, four a workgroup).
template <int DT, int TEAMS>
__global__ __launch_bounds__(TEAMS == 2 ? kThreads : 32 * TEAMS) void attention_shared_join_kernel(SharedArgs s) {
    constexpr int PER = DT / 32;             // elements of a lane
    constexpr int CHUNK = 2;                 // partial results that a team asks for at once (4: up to 1 us more in a pass, 8: 2 to 5)
    __shared__ float room[TEAMS > 2 ? TEAMS : 1][DT + 2];
    touch_arguments(s);
    const AttentionArgs& a = s.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, e = PER * (lane & 31);
    const int team = TEAMS > 2 ? (threadIdx.x >> 5) : half;
    const int64_t query = TEAMS > 2 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (query >= a.tokens_q * a.heads) return;
    const uint32_t token = (uint32_t)(query / a.heads), head = (uint32_t)(query - (int64_t)token * a.heads);
    const int32_t seq = s.sequence_of ? s.sequence_of[token] : (int32_t)token;
    if (seq < 0 || seq >= a.sequences) return;
    const AttentionEntry own = s.entries[s.group_count + seq];
    if (!(own.flags & kEntryPartial) || token - (uint32_t)own.q0 >= (uint32_t)own.lq) return;
    const uint32_t kv = head / (uint32_t)a.group, place = head - kv * (uint32_t)a.group;
    AttentionEntry common = {};
    common.first = -1;
    if (own.row >= 0) common = s.entries[own.row];

    // this query's row of an entry: its partial results are `step` apart
    struct Part {
        const float *o, *stats;
        int32_t splits;
        int64_t step;
    };
    auto part_of = [&](const AttentionEntry& x) -> Part {
        if (x.first < 0 || token - (uint32_t)x.q0 >= (uint32_t)x.lq) return {nullptr, nullptr, 0, 0};
        const int l = x.flags >> 8;
        const SharedLaunch& y = l == 0 ? s.launch[0] : l == 1 ? s.launch[1] : s.launch[2];
        const uint32_t row = (token - (uint32_t)x.q0) * (uint32_t)a.group + place, tile = row >> y.row_shift;
        const uint32_t tiles = ((uint32_t)x.lq * (uint32_t)a.group + (1u << y.row_shift) - 1) >> y.row_shift;
        // (the last row tile comes first)
        const int64_t slot = ((int64_t)x.first + (int64_t)(tiles - 1 - tile) * x.splits) * a.kv_heads + kv;
        const int64_t at = (slot << y.row_shift) + (row - (tile << y.row_shift));
        return {y.partial + at * DT, y.partial + (((int64_t)y.slots * a.kv_heads) << y.row_shift) * DT + at * 2, x.splits, (int64_t)a.kv_heads << y.row_shift};
    };
    const Part c = part_of(common), w = part_of(own);
    const int32_t parts = c.splits + w.splits;

    float o[PER], l = 0.f, m = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < PER; t++) o[t] = 0.f;
    for (int32_t p0 = team; p0 < parts; p0 += CHUNK * TEAMS) {
        float ms[CHUNK], ls[CHUNK], x[CHUNK][PER];
#pragma unroll
        for (int k = 0; k < CHUNK; k++) {
            // (behind the last, the first of these again, without weight)
            const int32_t p = p0 + TEAMS * k < parts ? p0 + TEAMS * k : p0;
            const bool is_common = p < c.splits;
            const int64_t at = (is_common ? p : p - c.splits) * (is_common ? c.step : w.step);
            const float2 st = *reinterpret_cast<const float2*>((is_common ? c.stats : w.stats) + at * 2);
            const float* from = (is_common ? c.o : w.o) + at * DT + e;
            ms[k] = p0 + TEAMS * k < parts ? st.x : -__builtin_inff();
            ls[k] = st.y;
            if constexpr (PER == 2) {
                const float2 v = *reinterpret_cast<const float2*>(from);
                x[k][0] = v.x, x[k][1] = v.y;
            } else {
#pragma unroll
                for (int t = 0; t < PER; t += 4) {
                    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(from + t);
#pragma unroll
                    for (int y = 0; y < 4; y++) x[k][t + y] = v[y];
                }
            }
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < CHUNK; k++) top = fmaxf(top, ms[k]);
        if (top == -__builtin_inff()) continue;       // (nothing seen)
        const float keep = __builtin_amdgcn_exp2f(m - top);
        m = top;
        l *= keep;
#pragma unroll
        for (int t = 0; t < PER; t++) o[t] *= keep;
#pragma unroll
        for (int k = 0; k < CHUNK; k++) {
            if (ms[k] == -__builtin_inff()) continue;  // (a weight of zero would make an infinity NaN)
            const float f = __builtin_amdgcn_exp2f(ms[k] - top) * 0x1p-16f;
            l += ls[k] * f;
#pragma unroll
            for (int t = 0; t < PER; t++) o[t] += x[k][t] * f;
        }
    }
    if constexpr (TEAMS > 2) {
#pragma unroll
        for (int t = 0; t < PER; t++) room[team][e + t] = o[t];
        if ((lane & 31) == 0) room[team][DT] = m, room[team][DT + 1] = l;
        __syncthreads();
        if (threadIdx.x >= 64) return;
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < TEAMS; i++) top = fmaxf(top, room[i][DT]);
        l = 0.f;
#pragma unroll
        for (int t = 0; t < PER; t++) o[t] = 0.f;
#pragma unroll
        for (int i = 0; i < TEAMS; i++) {
            if (room[i][DT] == -__builtin_inff()) continue;
            const float f = __builtin_amdgcn_exp2f(room[i][DT] - top);
            l += room[i][DT + 1] * f;
#pragma unroll
            for (int t = 0; t < PER; t++) o[t] += room[i][e + t] * f;
        }
    } else {
        const float other = __shfl_xor(m, 32), top = fmaxf(m, other);
        const float f = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - top);
        l *= f;
        l += __shfl_xor(l, 32);
#pragma unroll
        for (int t = 0; t < PER; t++) {
            o[t] *= f;
            o[t] += __shfl_xor(o[t], 32);
        }
    }
    if (half == 0 && e < a.dim) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bf16_t* out = a.out + (int64_t)token * a.out_token + (int64_t)head * a.out_head + e;
#pragma unroll
        for (int t = 0; t < PER; t += 2) *reinterpret_cast<uint32_t*>(out + t) = pack_bf16(o[t] * inv, o[t + 1] * inv);
    }
}

int launch_shared_plan(const SharedArgs& s, hipStream_t stream) {
    const int64_t entries = (int64_t)s.group_count + s.a.sequences;
    if (entries <= 256) attention_shared_plan_kernel<4, true><<<1, 256, 0, stream>>>(s);
    else attention_shared_plan_kernel<16, false><<<1, 1024, 0, stream>>>(s);
    return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;
}

// dim: of the kernels, 64, 128 or 256
int launch_shared_join(const SharedArgs& s, int dim, hipStream_t stream) {
    const int64_t queries = s.a.tokens_q * s.a.heads;
    // Passes with eight / four / two teams: 64 queries of many splits 37.2 / 40.5 / 48.2 us, 512 42.0 / 44.2 / 51.3; 2048 of 35 parts 59.4 / 59.0 /
    // 61.7, of 17 48.9 / 48.5 / 47.9; 4096 72.7 / 68.7 / 69.4; 6400 of 10 - / 64.7 / 59.2
    const int teams = queries <= 1024 ? 8 : queries <= 4096 ? 4 : 2;
    const dim3 grid((unsigned)(teams > 2 ? queries : (queries + 3) / 4));
#define SNGGUF_GO(D)                                                                                                    \
    if (dim == D) {                                                                                                     \
        if (teams == 8) attention_shared_join_kernel<D, 8><<<grid, 32 * 8, 0, stream>>>(s);                             \
        else if (teams == 4) attention_shared_join_kernel<D, 4><<<grid, 32 * 4, 0, stream>>>(s);                        \
        else attention_shared_join_kernel<D, 2><<<grid, kThreads, 0, stream>>>(s);                                      \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
    SNGGUF_GO(64)
    SNGGUF_GO(128)
    SNGGUF_GO(256)
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

}  // namespace sngguf
