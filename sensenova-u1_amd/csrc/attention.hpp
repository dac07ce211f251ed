// What the attention kernels share: their arguments, and how a launch's workgroups find their share of the work.
//
// The lengths of the sequences lie in device memory (a captured launch sees new ones at every replay), so the host knows
// only how many sequences and tokens there are at most.  Every workgroup scans the lengths itself, 64 sequences at a time,
// and finds its (sequence, row tile, key / value head, split) from its number; workgroups beyond the last one leave.
//
// A row is one (token, query head) pair of the heads that share a key / value head: row r of a sequence is token r / group,
// head r % group, so a tile of keys and values serves all heads of the group.
#pragma once

#include "sngguf_common.hpp"

namespace sngguf {

// Where a launch's sequences and workgroups are planned by a kernel in front of it (attention_shared.hip): a sequence, or the tokens that a
// group of sequences has in common as one whose queries are all of the group's.
struct AttentionEntry {
    int32_t q0, lq;         // its queries
    int32_t k0, lk;         // its keys: places [k0, lk), k0 a multiple of every kernel's key tile
    int32_t row;            // of the table of pages
    int32_t splits, first;  // workgroups (of a key / value head) of each row tile, number of the first one
    int32_t flags;
};
enum { kEntryCausal = 1, kEntryPartial = 2, kEntryOnce = 4 };

struct AttentionArgs {
    const bf16_t* q;        // [tokens_q][heads][dim]
    bf16_t* out;
    int64_t q_token, q_head, out_token, out_head;     // strides in elements
    // keys and values: packed rows ...
    const bf16_t *k, *v;    // [tokens_k][kv_heads][dim]
    int64_t k_token, k_head, v_token, v_head;
    const int32_t* ends_k;  // [sequences + 1]
    // ... or pages [pages][kv_heads][page][dim], scales [pages][kv_heads][dim / 32][page]
    const void *k_pages, *v_pages;
    const uint16_t *k_scales, *v_scales;
    const int32_t* table;   // [sequences][table_width], rows table_stride apart
    const int32_t* lens;    // [sequences]
    int64_t table_stride;
    int32_t pages, page_shift, table_width;
    const int32_t* ends_q;  // [sequences + 1], or NULL: one token each
    int32_t sequences;
    int64_t tokens_q, tokens_k;
    int32_t heads, kv_heads, group, dim;
    float scale_log2;       // softmax scale x log2(e)
    int32_t causal;
    int64_t window;         // 0: none
    int32_t min_rows, max_rows;   // rows of the sequences that this launch takes
    // split of a sequence's keys over workgroups (NULL: none)
    float* partial;         // [workgroups][tile rows][dim of the kernel], then [workgroups][tile rows][2]: maximum, sum
    int32_t want;           // workgroups that fill the device
    int32_t least;          // key tiles of a split at least
    int64_t grid;           // workgroups of the main launch
    // planned launches (NULL: every workgroup finds its own place)
    const AttentionEntry* map;   // [workgroups / kv_heads]: what each does; nothing where there are no queries
};

struct AttentionSequence {
    int64_t q0, k0;
    int32_t lq, lk;
    int32_t from;           // first key that counts, a multiple of the key tile
};

__device__ __forceinline__ AttentionSequence attention_sequence(const AttentionArgs& a, int i) {
    AttentionSequence s;
    s.from = 0;
    if (a.ends_q) {
        // (values that are no cumulative lengths stay within the tensors)
        int64_t e0 = a.ends_q[i], e1 = a.ends_q[i + 1];
        e0 = e0 < 0 ? 0 : e0 > a.tokens_q ? a.tokens_q : e0;
        e1 = e1 < e0 ? e0 : e1 > a.tokens_q ? a.tokens_q : e1;
        s.q0 = e0;
        s.lq = (int32_t)(e1 - e0);
    } else {
        s.q0 = i;
        s.lq = 1;
    }
    if (a.lens) {
        const int64_t cap = (int64_t)a.table_width << a.page_shift;
        int64_t n = a.lens[i];
        s.k0 = 0;
        s.lk = (int32_t)(n < 0 ? 0 : n > cap ? cap : n);
    } else {
        int64_t e0 = a.ends_k[i], e1 = a.ends_k[i + 1];
        e0 = e0 < 0 ? 0 : e0 > a.tokens_k ? a.tokens_k : e0;
        e1 = e1 < e0 ? e0 : e1 > a.tokens_k ? a.tokens_k : e1;
        s.k0 = e0;
        s.lk = (int32_t)(e1 - e0);
    }
    return s;
}

// Row tiles of a sequence, and key tiles that its rows see between them.
template <int ROWS, int KEYS>
__device__ __forceinline__ void attention_tiles(const AttentionArgs& a, const AttentionSequence& s, uint32_t& row_tiles, uint32_t& key_tiles) {
    const uint32_t rows = (uint32_t)s.lq * (uint32_t)a.group;     // (tokens_q x group is below 2^31)
    if ((int32_t)rows < a.min_rows || (int32_t)rows > a.max_rows) {
        row_tiles = key_tiles = 0;
        return;
    }
    row_tiles = (rows + ROWS - 1) / ROWS;
    int64_t lo = a.window ? (int64_t)s.lk - s.lq - a.window + 1 : 0;
    lo = lo < 0 ? 0 : lo / KEYS;
    const int64_t hi = ((int64_t)s.lk + KEYS - 1) / KEYS;
    key_tiles = (uint32_t)(hi > lo ? hi - lo : 1);
}

// x of the lanes up to this one added up, in the vector unit (row shifts, then a row's last value handed on)
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false);
    return x;
}
__device__ __forceinline__ uint32_t wave_total(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(x), 63); }

struct AttentionBlock {
    AttentionSequence s;
    int32_t seq, row_tile, split, splits, kv_head;
    int64_t slot;           // number of this workgroup's (combining: of split 0's) partial result; splits lie kv_heads apart
    bool there;
    bool causal, partial;   // partial: its result goes to be joined
    bool once;              // planned launches: nobody else reads its pages
};

// A planned workgroup's place
template <int ROWS>
__device__ __forceinline__ AttentionBlock attention_planned_block(const AttentionArgs& a, uint32_t id) {
    AttentionBlock b;
    b.kv_head = id % (uint32_t)a.kv_heads;
    const uint32_t want = id / (uint32_t)a.kv_heads;
    const AttentionEntry e = a.map[want];
    b.s.lq = __builtin_amdgcn_readfirstlane(e.lq);
    b.there = b.s.lq != 0;
    if (!b.there) return b;
    b.s.q0 = (uint32_t)__builtin_amdgcn_readfirstlane(e.q0);
    b.s.k0 = 0;
    b.s.lk = __builtin_amdgcn_readfirstlane(e.lk);
    b.s.from = __builtin_amdgcn_readfirstlane(e.k0);
    b.seq = __builtin_amdgcn_readfirstlane(e.row);
    b.splits = __builtin_amdgcn_readfirstlane(e.splits);
    const int32_t flags = __builtin_amdgcn_readfirstlane(e.flags);
    b.causal = flags & kEntryCausal;
    b.partial = flags & kEntryPartial;
    b.once = flags & kEntryOnce;
    const uint32_t within = want - (uint32_t)__builtin_amdgcn_readfirstlane(e.first), t = within / (uint32_t)b.splits;
    b.split = (int32_t)(within - t * (uint32_t)b.splits);
    b.row_tile = (int32_t)(((uint32_t)b.s.lq * (uint32_t)a.group + ROWS - 1) / ROWS - 1 - t);
    b.slot = id;
    return b;
}

// COMBINE: `id` counts (row tile, head) pairs and not (row tile, split, head) triples.
template <int ROWS, int KEYS, bool COMBINE>
__device__ __forceinline__ AttentionBlock attention_block(const AttentionArgs& a, uint32_t id) {
    const int lane = threadIdx.x & 63;
    AttentionBlock b;
    b.there = false;
    b.causal = a.causal;
    b.once = false;
    // heads of one row tile are neighbours: with 8 key / value heads each XCD keeps to one head's keys and values
    b.kv_head = id % (uint32_t)a.kv_heads;
    const uint32_t want = id / (uint32_t)a.kv_heads;
    uint32_t chunk = 0;     // key tiles of a split; 0: not split
    if (a.partial) {
        uint64_t total = 0, tiles = 0;
        for (int base = 0; base < a.sequences; base += 64) {
            uint64_t mine = 0;
            uint32_t rt = 0, kt = 0;
            if (base + lane < a.sequences) {
                attention_tiles<ROWS, KEYS>(a, attention_sequence(a, base + lane), rt, kt);
                mine = (uint64_t)rt * kt;
            }
            // (64 numbers of 25 bits add up within 32)
            if (__ballot(mine >> 25) == 0) {
                mine = wave_total((uint32_t)mine);
            } else {
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor((unsigned long long)mine, o);
            }
            total += mine;
            tiles += wave_total(rt);
        }
        // the last split of a row tile is half as long as the others on average: so many workgroups less, or the device would have
        // a few to do in a second round
        const uint64_t cut = tiles * a.kv_heads / 2, most = a.want;
        const uint64_t target = cut < most / 2 ? most - cut : most / 2;
        // (rounded up by one at most where the quotient is whole: the grid has room for `want`)
        const double exact = (double)(total * a.kv_heads) / (double)target;
        chunk = exact < 2147483647.0 ? (uint32_t)exact + 1 : 0x7FFFFFFFu;
        if (chunk < (uint32_t)a.least) chunk = a.least;
    }
    uint32_t before = 0, before_slots = 0;
    for (int base = 0; base < a.sequences; base += 64) {
        uint32_t rt = 0, kt = 0, splits = 1;
        AttentionSequence mine_s = {0, 0, 0, 0};
        if (base + lane < a.sequences) {
            mine_s = attention_sequence(a, base + lane);
            attention_tiles<ROWS, KEYS>(a, mine_s, rt, kt);
            if (chunk) splits = (kt + chunk - 1) / chunk;
            if (splits < 1) splits = 1;
        }
        const uint32_t slots = rt * splits, mine = COMBINE ? rt : slots;
        const uint32_t sum = wave_scan(mine), sum_slots = COMBINE ? wave_scan(slots) : sum;
        const uint64_t hit = __ballot(want >= before + sum - mine && want < before + sum);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const uint32_t first = before + (uint32_t)__builtin_amdgcn_readlane((int)(sum - mine), l);
            const uint32_t first_slot = before_slots + (uint32_t)__builtin_amdgcn_readlane((int)(sum_slots - slots), l);
            const uint32_t tiles = (uint32_t)__builtin_amdgcn_readlane((int)rt, l);
            b.seq = base + l;
            b.splits = __builtin_amdgcn_readlane((int)splits, l);
            const uint32_t within = want - first;
            const uint32_t t = COMBINE ? within : within / (uint32_t)b.splits;
            b.split = COMBINE ? 0 : (int32_t)(within - t * (uint32_t)b.splits);
            // the last rows of a causal sequence see the most keys: first.  (Sequences follow one another all the same: longest first over
            // all of them was 8 % faster for four prompts of 1000 tokens and 10 % slower for eight of 300 to 1700, whose keys and values
            // then no longer stay in an XCD's cache.)
            b.row_tile = (int32_t)(tiles - 1 - t);
            b.slot = ((int64_t)first_slot + (int64_t)t * b.splits + b.split) * a.kv_heads + b.kv_head;
            b.s.q0 = (uint32_t)__builtin_amdgcn_readlane((int)mine_s.q0, l);     // (both below 2^31)
            b.s.k0 = (uint32_t)__builtin_amdgcn_readlane((int)mine_s.k0, l);
            b.s.lq = __builtin_amdgcn_readlane(mine_s.lq, l);
            b.s.lk = __builtin_amdgcn_readlane(mine_s.lk, l);
            b.s.from = 0;
            b.partial = b.splits > 1;
            b.there = true;
            return b;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        before_slots += (uint32_t)__builtin_amdgcn_readlane((int)sum_slots, 63);
    }
    return b;
}

// Token of a row, and its head of the group
__device__ __forceinline__ int32_t attention_token(const AttentionArgs& a, int64_t row, int32_t& head) {
    const uint32_t token = (uint32_t)row / (uint32_t)a.group;
    head = (int32_t)((uint32_t)row - token * (uint32_t)a.group);
    return (int32_t)token;
}

// Keys [lo, hi) that some row of rows [r0, r1) of a sequence sees.
__device__ __forceinline__ void attention_keys(const AttentionArgs& a, const AttentionBlock& b, int64_t r0, int64_t r1, int32_t& lo, int32_t& hi) {
    const AttentionSequence& s = b.s;
    const int64_t back = (int64_t)s.lk - s.lq;
    lo = s.from;
    hi = s.lk;
    if (b.causal) {
        const int64_t last = back + (uint32_t)(r1 - 1) / (uint32_t)a.group + 1;
        if (last < hi) hi = (int32_t)(last < 0 ? 0 : last);
    }
    if (a.window) {
        const int64_t first = back + (uint32_t)r0 / (uint32_t)a.group - a.window + 1;
        if (first > lo) lo = (int32_t)(first < hi ? first : hi);
    }
}

enum { kPacked = 0, kPaged = 1, kPagedQ8 = 2 };       // where keys and values lie

// Row r over the keys [lo, hi) again, key by key, by one wavefront, and its result to where it goes (a row of `out`, or of a split's
// partial result for tiles of ROWS rows).  The matrix products multiply a value that a row does not see by a weight of zero,
// which takes it away unless it is an infinity or a NaN; and their weights may be as large as the limit above which they are set
// right, too much for values near the end of bf16.  So a row whose result is not finite is done again: what it sees counts, and
// nothing else.  A lane has a key's score, then all lanes lie along the elements of one value after the other; weights are
// scaled by 2^-31, so that no sum of values leaves fp32.  (UP: by which power of two the other splits' are.)
// A row that is NaN throughout ends where that is known, as all rows of a model that has gone NaN come here: 16384 tokens 10 ms, to the end
// 1.5 s.  One with an infinite element or some NaN is done to its end, 0.7 us a key with all wavefronts at it.
template <int DT, int SOURCE, int ROWS, int UP>
__device__ __forceinline__ void attention_row_again(const AttentionArgs& a, const AttentionBlock& b, int64_t r, int32_t lo, int32_t hi) {
    constexpr int PER = DT / 64;            // elements of a lane: lane, lane + 64, ...
    const int lane = threadIdx.x & 63;
    int32_t head;
    const int32_t token = attention_token(a, r, head), place = b.s.lk - b.s.lq + token;
    head += b.kv_head * a.group;
    const bf16_t* q = a.q + (b.s.q0 + token) * a.q_token + (int64_t)head * a.q_head;
    if (b.causal && place + 1 < hi) hi = place + 1;
    if (a.window && place - a.window + 1 > lo) lo = (int32_t)(place - a.window + 1);
    float m = -__builtin_inff(), l = 0.f, o[PER];
#pragma unroll
    for (int t = 0; t < PER; t++) o[t] = 0.f;
    for (int64_t base = lo; base < hi; base += 64) {
        const int count = hi - base < 64 ? (int)(hi - base) : 64;
        const int64_t key = base + (lane < count ? lane : count - 1);
        // elements in front of the key's and the value's first; 8-bit: also of the scales
        int64_t k_at, v_at, scale_at = 0;
        if constexpr (SOURCE == kPacked) {
            k_at = (b.s.k0 + key) * a.k_token + (int64_t)b.kv_head * a.k_head;
            v_at = (b.s.k0 + key) * a.v_token + (int64_t)b.kv_head * a.v_head;
        } else {
            int64_t page = a.table[(int64_t)b.seq * a.table_stride + (key >> a.page_shift)];
            page = (page < 0 ? 0 : page >= a.pages ? a.pages - 1 : page) * a.kv_heads + b.kv_head;
            const int64_t row = key & ((1 << a.page_shift) - 1);
            k_at = v_at = ((page << a.page_shift) + row) * a.dim;
            scale_at = (page * (a.dim >> 5) << a.page_shift) + row;
        }
        float s = 0.f;
        for (int e = 0; e < a.dim; e++) {
            float k;
            if constexpr (SOURCE == kPagedQ8)
                k = (float)static_cast<const int8_t*>(a.k_pages)[k_at + e] * f16_to_f32(a.k_scales[scale_at + ((int64_t)(e >> 5) << a.page_shift)]);
            else
                k = bf16_to_f32((SOURCE == kPacked ? a.k : static_cast<const bf16_t*>(a.k_pages))[k_at + e]);
            s = __builtin_fmaf(k, bf16_to_f32(q[e]), s);
        }
        s = lane < count ? s * a.scale_log2 : -__builtin_inff();
        float top = s;
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        top = fmaxf(top, m);
        const float from = top == -__builtin_inff() ? 0.f : top, keep = __builtin_amdgcn_exp2f(m - from);
        m = top;
        const float p = __builtin_amdgcn_exp2f(s - from - 31.f);
        l = l * keep + p;                   // (of this lane's keys)
        if (__any(l != l)) {                // a score is NaN, or more than one infinite: so is all of the row
            l = __builtin_nanf("");
#pragma unroll
            for (int t = 0; t < PER; t++) o[t] = l;
            break;
        }
#pragma unroll
        for (int t = 0; t < PER; t++) o[t] *= keep;
        for (int j = 0; j < count; j++) {
            const float pj = __shfl(p, j);
            const int64_t at = __shfl((long long)v_at, j), sc = SOURCE == kPagedQ8 ? __shfl((long long)scale_at, j) : 0;
#pragma unroll
            for (int t = 0; t < PER; t++) {
                const int e = lane + 64 * t;
                if (e >= a.dim) continue;
                float v;
                if constexpr (SOURCE == kPagedQ8)
                    v = (float)static_cast<const int8_t*>(a.v_pages)[at + e] * f16_to_f32(a.v_scales[sc + ((int64_t)(e >> 5) << a.page_shift)]);
                else
                    v = bf16_to_f32((SOURCE == kPacked ? a.v : static_cast<const bf16_t*>(a.v_pages))[at + e]);
                o[t] = __builtin_fmaf(pj, v, o[t]);
            }
        }
        bool done = true;                   // nothing that follows changes elements that are all NaN, and they do not need the sum
#pragma unroll
        for (int t = 0; t < PER; t++) done &= o[t] != o[t] || lane + 64 * t >= a.dim;
        if (__all(done)) break;
    }
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) l += __shfl_xor(l, x);
    const int64_t part = b.slot * ROWS + r - (int64_t)b.row_tile * ROWS;
    // A partial result is in the scale of the other splits', or, where an element would leave fp32 there, as it is with a maximum higher by
    // as much.
    constexpr float kBack = (float)(1ull << (31 + UP));
    bool far = false;
#pragma unroll
    for (int t = 0; t < PER; t++) far |= __builtin_isfinite(o[t]) && !__builtin_isfinite(o[t] * kBack);
    far = __any(far);
    const float back = far ? 1.f : kBack;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int t = 0; t < PER; t++) {
        const int e = lane + 64 * t;
        if (e >= a.dim) continue;
        if (b.partial) a.partial[part * DT + e] = o[t] * back;
        else a.out[(b.s.q0 + token) * a.out_token + (int64_t)head * a.out_head + e] = f32_to_bf16(o[t] * inv);
    }
    if (b.partial && lane == 0) {
        // (a row whose scores are NaN has no maximum, and the join passes over splits without one: any number, so that the sum gets there)
        float* st = a.partial + a.grid * ROWS * DT + part * 2;
        st[0] = l != l ? 0.f : far ? m + (31 + UP) : m;
        st[1] = l * back;
    }
}

int launch_attention_combine(const AttentionArgs& a, int rows, int keys, int dim, int64_t tiles, int64_t most_rows, hipStream_t stream);

}  // namespace sngguf
