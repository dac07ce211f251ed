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
//    of each launch over its workgroups, and writes down which workgroup does what.
//  * The join: half a wavefront lies along a query's elements and takes some partial results at a time.  Weights are scaled by 2^-16, so that
//    no sum leaves fp32 whose average does not (there are fewer than 2^16 splits).
#include "attention_shared.hpp"

namespace sngguf {

namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kThreads = 256;

__device__ __forceinline__ int32_t wave_min(int32_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor((unsigned long long)x, o);
    return x;
}

// Which launch takes an entry, its row tiles and key tiles
__device__ __forceinline__ int entry_tiles(const SharedArgs& s, const AttentionEntry& e, bool common, uint32_t& row_tiles, uint32_t& key_tiles) {
    const uint32_t rows = (uint32_t)e.lq * (uint32_t)s.a.group;
    row_tiles = key_tiles = 0;
    if (rows == 0 || (common && e.lk == 0)) return -1;
#pragma unroll
    for (int l = 0; l < kSharedLaunches; l++) {
        const SharedLaunch& x = s.launch[l];
        if ((l == 0) != common || x.slots == 0 || (int32_t)rows < x.min_rows || (int32_t)rows > x.max_rows) continue;
        row_tiles = (rows + (uint32_t)x.rows - 1) / (uint32_t)x.rows;
        const int32_t lo = e.k0 / x.keys, hi = (int32_t)(((int64_t)e.lk + x.keys - 1) / x.keys);
        key_tiles = hi > lo ? hi - lo : 1;
        return l;
    }
    return -1;
}

}  // namespace

__global__ __launch_bounds__(kPlanThreads) void attention_shared_plan_kernel(SharedArgs s) {
    __shared__ uint64_t sums[kPlanWaves][2 * kSharedLaunches];
    __shared__ uint32_t ups[kPlanWaves][kSharedLaunches];
    __shared__ int32_t firsts[kPlanThreads], counts[kPlanThreads];
    const AttentionArgs& a = s.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t groups = s.group_count, sequences = a.sequences;
    const int64_t all = (int64_t)groups + sequences;

    for (int64_t i = tid; i < sequences; i += kPlanThreads) {
        const AttentionSequence q = attention_sequence(a, (int)i);
        s.entries[groups + i] = {(int32_t)q.q0, q.lq, 0, q.lk, (int32_t)i, 1, -1, 0};
        s.group_of[i] = -1;
    }
    if (s.sequence_of)
        for (int64_t t = tid; t < a.tokens_q; t += kPlanThreads) s.sequence_of[t] = -1;
#pragma unroll
    for (int l = 0; l < kSharedLaunches; l++)
        for (int32_t i = tid; i < s.launch[l].slots; i += kPlanThreads) s.launch[l].map[i] = -1;
    __syncthreads();

    // ---- what a group has in common: a wavefront a group -------------------------------------------------------------------
    for (int64_t g = wave; g < groups; g += kPlanWaves) {
        // (numbers that are no cumulative counts stay within the tensors)
        int32_t e0 = s.groups[g], e1 = s.groups[g + 1];
        e0 = e0 < 0 ? 0 : e0 > sequences ? sequences : e0;
        e1 = e1 < e0 ? e0 : e1 > sequences ? sequences : e1;
        // sequences without new tokens have no say
        int32_t least = 0x7FFFFFFF, row = 0x7FFFFFFF, q0 = 0x7FFFFFFF, q1 = 0, count = 0;
        for (int64_t i = (int64_t)e0 + lane; i < e1; i += 64) {
            const AttentionEntry e = s.entries[groups + i];
            if (e.lq == 0) continue;
            least = min(least, e.lk - e.lq);
            row = min(row, (int32_t)i);
            q0 = min(q0, e.q0);
            q1 = max(q1, e.q0 + e.lq);
            count++;
        }
        least = wave_min(least);
        row = wave_min(row);
        q0 = wave_min(q0);
        q1 = -wave_min(-q1);
        const int32_t said = s.shared[g];
        int32_t common = said < least ? said : least;
        common = common < 0 ? 0 : common / kSharedUnit * kSharedUnit;
        if (wave_total((uint32_t)count) < 2) common = 0;
        if (lane == 0) s.entries[g] = {q0, common ? q1 - q0 : 0, 0, common, row, 1, -1, 0};
        if (common)
            for (int64_t i = (int64_t)e0 + lane; i < e1; i += 64) {
                s.entries[groups + i].k0 = common;
                s.group_of[i] = (int32_t)g;
            }
    }
    if (s.sequence_of)
        for (int64_t i = wave; i < sequences; i += kPlanWaves) {
            const AttentionEntry e = s.entries[groups + i];
            for (int32_t j = lane; j < e.lq; j += 64) s.sequence_of[e.q0 + j] = (int32_t)i;
        }
    __syncthreads();

    // ---- all work of each launch, and how many key tiles of it a workgroup takes ---------------------------------------------
    uint64_t sum[2 * kSharedLaunches] = {};
    for (int64_t v = tid; v < all; v += kPlanThreads) {
        uint32_t rt, kt;
        const int mine = entry_tiles(s, s.entries[v], v < groups, rt, kt);
#pragma unroll
        for (int l = 0; l < kSharedLaunches; l++)
            if (l == mine) sum[2 * l] += (uint64_t)rt * kt, sum[2 * l + 1] += rt;
    }
#pragma unroll
    for (int x = 0; x < 2 * kSharedLaunches; x++) {
        const uint64_t t = wave_sum64(sum[x]);
        if (lane == 0) sums[wave][x] = t;
    }
    __syncthreads();
    uint32_t chunk[kSharedLaunches];
#pragma unroll
    for (int l = 0; l < kSharedLaunches; l++) {
        uint64_t work = 0, tiles = 0;
#pragma unroll
        for (int w = 0; w < kPlanWaves; w++) work += sums[w][2 * l], tiles += sums[w][2 * l + 1];
        // the last split of a row tile is half as long as the others on average: so many workgroups less
        const SharedLaunch& x = s.launch[l];
        const uint64_t cut = tiles * a.kv_heads / 2, most = x.want;
        const uint64_t target = cut < most / 2 ? most - cut : most / 2 > 0 ? most / 2 : 1;
        const double exact = (double)(work * a.kv_heads) / (double)target;
        chunk[l] = !x.split || exact >= 2147483646.0 ? 0x7FFFFFFFu : (uint32_t)exact + 1;
        if (chunk[l] < (uint32_t)x.least) chunk[l] = x.least;
    }

    // ---- which workgroups take an entry ------------------------------------------------------------------------------------
    uint32_t before[kSharedLaunches] = {};
    for (int64_t base = 0; base < all; base += kPlanThreads) {
        const int64_t v = base + tid;
        uint32_t rt = 0, kt = 0, splits = 1, up[kSharedLaunches] = {};
        int mine = -1;
        AttentionEntry e = {};
        if (v < all) {
            e = s.entries[v];
            mine = entry_tiles(s, e, v < groups, rt, kt);
        }
#pragma unroll
        for (int l = 0; l < kSharedLaunches; l++) {
            if (l == mine) {
                splits = (kt + chunk[l] - 1) / chunk[l];
                if (splits < 1) splits = 1;
            }
            up[l] = wave_scan(l == mine ? rt * splits : 0);
            if (lane == 63) ups[wave][l] = up[l];
        }
        __syncthreads();
        int32_t first = -1, count = 0;
#pragma unroll
        for (int l = 0; l < kSharedLaunches; l++) {
            uint32_t in_front = before[l];
            for (int w = 0; w < kPlanWaves; w++) {
                if (w < wave) in_front += ups[w][l];
                before[l] += ups[w][l];
            }
            if (l == mine) {
                count = (int32_t)(rt * splits);
                first = (int32_t)(in_front + up[l]) - count;
                // (lengths that are none can need more workgroups than there are)
                if (first < 0 || (int64_t)first + count > s.launch[l].slots) first = -1, count = 0;
            }
        }
        if (mine >= 0) {
            const bool common = v < groups;
            e.splits = (int32_t)splits;
            e.first = first;
            e.flags = mine << 8 | (common ? kEntryPartial | (rt == 1 ? kEntryOnce : 0)
                                          : kEntryCausal | kEntryOnce | (splits > 1 || s.group_of[v - groups] >= 0 ? kEntryPartial : 0));
            s.entries[v] = e;
        }
        firsts[tid] = first;
        counts[tid] = mine < 0 ? 0 : count << 2 | mine;
        __syncthreads();
        for (int i = wave; i < kPlanThreads && base + i < all; i += kPlanWaves) {
            const int32_t n = counts[i] >> 2, f = firsts[i];
            int32_t* map = s.launch[0].map;
            if ((counts[i] & 3) == 1) map = s.launch[1].map;
            if ((counts[i] & 3) == 2) map = s.launch[2].map;
            for (int32_t j = lane; j < n; j += 64) map[f + j] = (int32_t)(base + i);
        }
        __syncthreads();
    }
}

// A query's partial results summed.  TEAMS half wavefronts have a query: two, or all eight of the workgroup where queries are few.
template <int DT, int TEAMS>
__global__ __launch_bounds__(kThreads) void attention_shared_join_kernel(SharedArgs s) {
    constexpr int PER = DT / 32;             // elements of a lane
    constexpr int CHUNK = 4;                 // partial results that a team asks for at once
    __shared__ float room[TEAMS > 2 ? TEAMS : 1][DT + 2];
    const AttentionArgs& a = s.a;
    const int lane = threadIdx.x & 63, half = lane >> 5, e = PER * (lane & 31);
    const int team = TEAMS > 2 ? (threadIdx.x >> 5) : half;
    const int64_t query = TEAMS > 2 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (query >= a.tokens_q * a.heads) return;
    const uint32_t token = (uint32_t)(query / a.heads), head = (uint32_t)(query - (int64_t)token * a.heads);
    const int32_t seq = s.sequence_of ? s.sequence_of[token] : (int32_t)token;
    if (seq < 0 || seq >= a.sequences) return;
    const AttentionEntry own = s.entries[s.group_count + seq];
    const int32_t g = s.group_of[seq];
    if (!(own.flags & kEntryPartial)) return;
    const uint32_t kv = head / (uint32_t)a.group, place = head - kv * (uint32_t)a.group;
    AttentionEntry common = {};
    common.first = -1;
    if (g >= 0) common = s.entries[g];

    // this query's row of an entry: its partial results are `step` apart
    struct Part {
        const float *o, *stats;
        int32_t splits;
        int64_t step;
    };
    auto part_of = [&](const AttentionEntry& x) -> Part {
        if (x.first < 0) return {nullptr, nullptr, 0, 0};
        const int l = x.flags >> 8;
        const SharedLaunch& y = l == 0 ? s.launch[0] : l == 1 ? s.launch[1] : s.launch[2];
        const uint32_t row = (token - (uint32_t)x.q0) * (uint32_t)a.group + place, tile = row / (uint32_t)y.rows;
        const uint32_t tiles = ((uint32_t)x.lq * (uint32_t)a.group + (uint32_t)y.rows - 1) / (uint32_t)y.rows;
        // (the last row tile comes first)
        const int64_t slot = ((int64_t)x.first + (int64_t)(tiles - 1 - tile) * x.splits) * a.kv_heads + kv;
        const int64_t at = slot * y.rows + (row - tile * (uint32_t)y.rows);
        return {y.partial + at * DT, y.partial + (int64_t)y.slots * a.kv_heads * y.rows * DT + at * 2, x.splits, (int64_t)a.kv_heads * y.rows};
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
    attention_shared_plan_kernel<<<1, kPlanThreads, 0, stream>>>(s);
    return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;
}

// dim: of the kernels, 64, 128 or 256
int launch_shared_join(const SharedArgs& s, int dim, hipStream_t stream) {
    const int64_t queries = s.a.tokens_q * s.a.heads;
    const bool wide = queries <= 1024;
    const dim3 grid((unsigned)(wide ? queries : (queries + 3) / 4));
#define SNGGUF_GO(D)                                                                                                    \
    if (dim == D) {                                                                                                     \
        if (wide) attention_shared_join_kernel<D, 8><<<grid, kThreads, 0, stream>>>(s);                                 \
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
