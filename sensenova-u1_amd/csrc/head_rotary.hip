// Heads of queries and keys normed and turned by several positions of their token, in one pass; keys and values to the paged
// cache in the same launch or not.
//
// With y = w x / sqrt(mean over the part of x^2 + eps) for each part of a head that is normed by itself (or y = x), and for
// pair i of rate f_i (turns a position) that belongs to axis a_i, at the token's position p[a_i]:
//     u' = u c - v s,  v' = v c + u s,   c = fp32(m cos(2 pi p[a_i] f_i)), s the same with the sine, m the table's magnitude,
// (u, v) two elements of y.  Pairs are neighbours, or lie half a part apart in each part of the head.  The angle is formed in 64
// bits and reduced to the nearest whole turn there; everything else is fp32, rounded to bf16 once (norm, weight and rotation
// by themselves would round three times, and be off by 1.7 times as much).
//
// Bound by memory: an element is two bytes in and two out, for some ten operations; and next by its instructions, which is why heads are divided
// as they are.  Neighbouring lanes have a head between them, its sums of squares are added up across them in the vector unit, and all of it is
// read before any of it is written, so a call may work in place.  A lane keeps to the same elements of all heads, so weights,
// cosines and sines are fetched once for a token.
//  * head_pairs_kernel, pairs half a part apart in parts of multiples of 16 elements: a lane has eight pairs, both of their elements, and a
//    workgroup up to four tokens.  4096 tokens of 40 heads of 128: 15.3 us (84 MB, 5.5 TB/s), with two norms a head 17.4; as eight elements a lane,
//    with the others from the lane that has them, and one token a workgroup 20.9 and 33.4.  5003 tokens of 32 query and 8 + 8 heads, two
//    norms, keys and values written in 8 bits: 28 us (113 MB, 4.0 TB/s).  One token: 3 us, all latency.
//  * head_rotary_kernel, neighbouring pairs, any parts or rows: a lane has eight elements; those that they are turned with, where they are not among
//    the eight, are read beside them.  Shapes for which the other is no form, so it is kept simple.
#include <type_traits>

#include "head_rotary.hpp"
#include "rotary_cache_device.hpp"

namespace sngguf {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;                                // heads of a lane that head_rotary_kernel asks for at once

enum { kNeighbours = 0, kAnyHalves = 1 };
enum { kNormNone = 0, kNormHalf = 1, kNormWide = 2 };     // weights: none, bf16, fp32

template <int CONTROL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CONTROL, 0xF, 0xF, false));
}

// Sum over 2^shift neighbouring lanes, the same in all of them (the mirrors exchange groups whose lanes already agree)
__device__ __forceinline__ float lanes_sum(float x, int shift) {
    if (shift > 0) x += dpp<0xB1>(x);
    if (shift > 1) x += dpp<0x4E>(x);
    if (shift > 2) x += dpp<0x141>(x);
    if (shift > 3) x += dpp<0x140>(x);
    if (shift > 4) x += __shfl_xor(x, 16);
    if (shift > 5) x += __shfl_xor(x, 32);
    return x;
}

// 1 / sqrt of the mean of squares: the instruction is off by a step at most; numbers below the smallest normal one, which it takes for zero, are
// scaled into its range
__device__ __forceinline__ float rstd_of(float sum, float one_over, float eps) {
    const float mean = __builtin_fmaf(sum, one_over, eps);
    const bool tiny = mean < 0x1p-100f;
    const float r = __builtin_amdgcn_rsqf(tiny ? mean * 0x1p64f : mean);
    return tiny ? r * 0x1p32f : r;
}

// Part of the norm that element e belongs to, and where it starts
__device__ __forceinline__ int norm_part(const HeadNormArgs& n, int e, int& start) {
    int p = 0;
    start = 0;
#pragma unroll
    for (int i = 0; i + 1 < kMostParts; i++)
        if (p == i && i + 1 < n.parts && e >= start + n.elements[i]) start += n.elements[i], p = i + 1;
    return p;
}
__device__ __forceinline__ const void* norm_weight(const HeadNormArgs& n, int p) { return p == 0 ? n.weight[0] : p == 1 ? n.weight[1] : p == 2 ? n.weight[2] : n.weight[3]; }
__device__ __forceinline__ float norm_one_over(const HeadNormArgs& n, int p) { return p == 0 ? n.one_over[0] : p == 1 ? n.one_over[1] : p == 2 ? n.one_over[2] : n.one_over[3]; }

// Position of a token that turns a pair.  Up to four axes: all of the token's positions are asked for beside the pair's axis.
__device__ __forceinline__ int64_t position_of(const HeadRotaryArgs& a, int pair, int64_t token) {
    const int64_t* at = a.positions + token;
    if (!a.axis || a.axes == 1) return at[0];
    int axis = a.axis[pair];
    if (a.axes <= 4) {
        int64_t p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = at[(i < a.axes ? i : a.axes - 1) * a.axis_stride];
        return axis <= 0 ? p[0] : axis == 1 ? p[1] : axis == 2 ? p[2] : p[3];
    }
    axis = axis < 0 ? 0 : axis >= a.axes ? a.axes - 1 : axis;
    return at[axis * a.axis_stride];
}

// What a lane keeps of a norm: weights of its eight elements and of their pairs' others, and the parts that they belong to
struct LaneNorm {
    float g[8], gz[8];
    int part;
    uint32_t z_parts;                                    // four bits each
};

}  // namespace

template <int LAYOUT, bool CACHE, bool NORM>
__global__ __launch_bounds__(kThreads) void head_rotary_kernel(HeadRotaryArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 cs_all[];    // [token][pair]
    const int tid = threadIdx.x, lanes = 1 << a.lane_shift, teams = kThreads >> a.lane_shift;
    const int team = tid >> a.lane_shift, e = 8 * (tid & (lanes - 1));
    const bool there = e < a.dim;
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_block;
    const int count = (int)(a.tokens - t0 < a.tokens_per_block ? a.tokens - t0 : a.tokens_per_block);
    const bool single = count == 1;
    const int turned = 2 * a.pairs;

    // ---- items: (token, head) pairs, dealt over the teams; the first ones' words are asked for before the angles are formed ----
    struct Item {
        int t, h;
        bool active;
    };
    auto item = [&](int i, int heads) -> Item {
        const bool active = i < count * heads;
        if (!active) return {0, 0, false};
        const int t = single ? 0 : (int)((uint32_t)i / (uint32_t)heads);
        return {t, i - t * heads, there};
    };
    auto q_row = [&](const Item& x) { return a.q + (t0 + x.t) * a.q_token + x.h * a.q_head; };
    const int others = CACHE ? 2 * a.kv_heads : a.k_heads;
    auto k_row = [&](const Item& x) -> const bf16_t* {
        if (CACHE && x.h >= a.kv_heads) return a.v + (t0 + x.t) * a.v_token + (x.h - a.kv_heads) * a.v_head;
        return a.k + (t0 + x.t) * a.k_token + x.h * a.k_head;
    };
    u32x4_t q_raw[kAhead], k_raw = {0u, 0u, 0u, 0u};
    auto load_q = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const Item x = item(i0 + u * teams + team, a.q_heads);
            q_raw[u] = u32x4_t{0u, 0u, 0u, 0u};
            if (x.active) q_raw[u] = load8(q_row(x) + e, a.wide);
        }
    };
    auto load_k = [&](int i0) {
        const Item x = item(i0 + team, others);
        k_raw = u32x4_t{0u, 0u, 0u, 0u};
        if (x.active) k_raw = load8(k_row(x) + e, a.wide);
    };
    load_q(0);
    load_k(0);

    // ---- which pairs this lane's elements belong to ----------------------------------------------------------------------
    int z_at[8], pairs_of[8];
    uint32_t seconds = 0, rotated = 0;
    if constexpr (LAYOUT == kAnyHalves) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            int start = 0, first = 0;
            z_at[j] = there ? e + j : 0;
            pairs_of[j] = 0;
#pragma unroll
            for (int p = 0; p < kMostParts; p++) {
                const int n = p < a.parts ? a.part[p] : 0, at = e + j - start;
                if (at >= 0 && at < n) {
                    const bool sec = at >= n / 2;
                    seconds |= sec ? 1u << j : 0u;
                    rotated |= 1u << j;
                    pairs_of[j] = first + (sec ? at - n / 2 : at);
                    z_at[j] = e + j + (sec ? -(n / 2) : n / 2);
                }
                start += n;
                first += n / 2;
            }
        }
    }

    // ---- weights -------------------------------------------------------------------------------------------------------
    auto weights = [&](const HeadNormArgs& n) -> LaneNorm {
        LaneNorm w;
        int start;
        w.part = norm_part(n, there ? e : 0, start);
        w.z_parts = 0;
        const void* at = norm_weight(n, w.part);
        const int off = (there ? e : 0) - start;
        if (n.parts == 0) {
#pragma unroll
            for (int j = 0; j < 8; j++) w.g[j] = w.gz[j] = 1.f;
            return w;
        }
        if (n.bf16) {
            unpack8(*reinterpret_cast<const u32x4_t*>(static_cast<const bf16_t*>(at) + off), w.g);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const f32x4_t v = *reinterpret_cast<const f32x4_t*>(static_cast<const float*>(at) + off + j);
#pragma unroll
                for (int y = 0; y < 4; y++) w.g[j + y] = v[y];
            }
        }
        if constexpr (LAYOUT == kNeighbours) {
#pragma unroll
            for (int j = 0; j < 8; j++) w.gz[j] = w.g[j ^ 1];
            w.z_parts = (uint32_t)w.part;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                int z_start;
                const int p = norm_part(n, z_at[j], z_start);
                const void* z = norm_weight(n, p);
                w.gz[j] = n.bf16 ? bf16_to_f32(static_cast<const bf16_t*>(z)[z_at[j] - z_start]) : static_cast<const float*>(z)[z_at[j] - z_start];
                w.z_parts |= (uint32_t)p << (4 * j);
            }
        }
        return w;
    };
    LaneNorm qw, kw;
    if constexpr (NORM) {
        qw = weights(a.q_norm);
        kw = weights(a.k_norm);
    }

    // ---- angles ----------------------------------------------------------------------------------------------------------
    for (int i = tid; i < count * a.pairs; i += kThreads) {
        const int t = single ? 0 : i / a.pairs, p = i - t * a.pairs;
        cs_all[i] = cos_sin(a.turns, p, position_of(a, p, t0 + t), a.magnitude);
    }
    __syncthreads();
    float c[8], s[8];                                    // of token `t_of`; an element is y c + z s
    int t_of = -1;
    auto turn_by = [&](int t) {
        if (t == t_of) return;
        t_of = t;
        const float2* cs = cs_all + t * a.pairs;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            c[j] = 1.f, s[j] = -0.f;                     // (not turned: x + -0 is x, also where x is a zero of either sign)
            if constexpr (LAYOUT == kNeighbours) {
                if (there && e + j < turned) c[j] = cs[(e + j) >> 1].x, s[j] = (j & 1) ? cs[(e + j) >> 1].y : -cs[(e + j) >> 1].y;
            } else {
                if (rotated >> j & 1) c[j] = cs[pairs_of[j]].x, s[j] = (seconds >> j & 1) ? cs[pairs_of[j]].y : -cs[pairs_of[j]].y;
            }
        }
    };

    // ---- eight elements of a head, normed and turned (all lanes of a wavefront come here together) -----------------------------
    auto turned8 = [&](u32x4_t raw, const bf16_t* row, const HeadNormArgs& n, const LaneNorm& w) -> u32x4_t {
        float x[8], z[8];
        unpack8(raw, x);
        if constexpr (LAYOUT == kNeighbours) {
#pragma unroll
            for (int j = 0; j < 8; j++) z[j] = there && e + j < turned ? x[j ^ 1] : 0.f;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) z[j] = row && (rotated >> j & 1) ? bf16_to_f32(row[z_at[j]]) : 0.f;
        }
        if constexpr (NORM) {
            if (n.parts) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) ss += x[j] * x[j];
                float r = 0.f, rz[LAYOUT == kAnyHalves ? 8 : 1] = {};
                for (int p = 0; p < n.parts; p++) {
                    const float rp = rstd_of(lanes_sum(there && w.part == p ? ss : 0.f, a.lane_shift), norm_one_over(n, p), n.eps);
                    if (w.part == p) r = rp;
#pragma unroll
                    for (int j = 0; j < (LAYOUT == kAnyHalves ? 8 : 1); j++)
                        if ((w.z_parts >> (4 * j) & 15u) == (uint32_t)p) rz[j] = rp;
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[j] = x[j] * r * w.g[j];
                    z[j] = z[j] * rz[LAYOUT == kAnyHalves ? j : 0] * w.gz[j];
                }
#pragma unroll
                for (int j = 0; j < 8; j++)              // (weights that are not finite)
                    if (LAYOUT == kNeighbours ? e + j >= turned : !(rotated >> j & 1)) z[j] = 0.f;
            }
        }
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = x[j] * c[j] + z[j] * s[j];
        return pack8(y);
    };

    for (int i0 = 0; i0 < count * a.q_heads; i0 += kAhead * teams) {
        if (i0) load_q(i0);
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const Item x = item(i0 + u * teams + team, a.q_heads);
            turn_by(x.t);
            const u32x4_t y = turned8(q_raw[u], x.active ? q_row(x) : nullptr, a.q_norm, qw);
            if (x.active) store8(a.q_out + (t0 + x.t) * a.q_out_token + x.h * a.q_out_head + e, y, a.wide);
        }
    }
    for (int i0 = 0; i0 < count * others; i0 += teams) {
        if (i0) load_k(i0);
        const Item x = item(i0 + team, others);
        turn_by(x.t);
        const u32x4_t y = turned8(k_raw, x.active && !(CACHE && x.h >= a.kv_heads) ? k_row(x) : nullptr, a.k_norm, kw);
        if (!x.active) continue;
        if constexpr (!CACHE) {
            store8(a.k_out + (t0 + x.t) * a.k_out_token + x.h * a.k_out_head + e, y, a.wide);
        } else {
            const int64_t slot = a.slots[t0 + x.t];
            // slots outside the cache (padding is marked by negative ones) are passed over; the lanes of a run agree
            if (slot < 0 || slot >= a.slot_count) continue;
            const bool value = x.h >= a.kv_heads;
            const int h = value ? x.h - a.kv_heads : x.h;
            void* pages = value ? a.v_pages : a.k_pages;
            uint16_t* scales = value ? a.v_scales : a.k_scales;
            const u32x4_t held = value ? k_raw : y;
            if (scales) cache_piece<true>(cache_place<true>(pages, scales, a, slot, h), a, e, held);
            else cache_piece<false>(cache_place<false>(pages, scales, a, slot, h), a, e, held);
        }
    }
}

// Eight pairs a lane: pieces a and b of eight elements each, (a_j, b_j) the pairs; elements behind the turned ones as pairs that are not turned.
// Rows start at 16-byte boundaries.
__device__ __forceinline__ u32x4_t piece_at(const bf16_t* p) { return *reinterpret_cast<const u32x4_t*>(p); }

// SHIFT: 2^SHIFT lanes have a head.  Known for normed heads of 80 to 128 elements, whose sums then need no choices (4096 tokens 17.5 against
// 18.2 us, one token 5.2 against 5.8 with its graph node; written in 8 bits level); -1: a.lane_shift says.
template <bool CACHE, int NORM, int SHIFT>
__global__ __launch_bounds__(kThreads) void head_pairs_kernel(HeadRotaryArgs a) {
    extern __shared__ __attribute__((aligned(16))) float2 cs_all[];    // [token][pair], then (CACHE) [team][dim] bf16
    touch_arguments(a);
    const int lane_shift = SHIFT >= 0 ? SHIFT : a.lane_shift;
    const int tid = threadIdx.x, lanes = 1 << lane_shift, teams = kThreads >> lane_shift;
    const int team = tid >> lane_shift, unit = tid & (lanes - 1);
    const bool there = 16 * unit < a.dim;
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_block;
    const int count = (int)(a.tokens - t0 < a.tokens_per_block ? a.tokens - t0 : a.tokens_per_block);
    const int turned = 2 * a.pairs;

    // ---- this lane's pieces --------------------------------------------------------------------------------------------------
    // (lanes behind the head's elements do what its first one does, so that nothing depends on them but the sums that they have no part in)
    const int of = there ? unit : 0;
    const bool rotates = 8 * of < a.pairs;
    int ea = turned + 16 * (of - (a.pairs >> 3)), eb = ea + 8, pair = 0;
    {
        int start = 0, first = 0;
#pragma unroll
        for (int p = 0; p < kMostParts; p++) {
            const int n = p < a.parts ? a.part[p] : 0, at = 8 * of - first;
            if (rotates && at >= 0 && at < n / 2) {
                ea = start + at;
                eb = ea + n / 2;
                pair = 8 * of;
            }
            start += n;
            first += n / 2;
        }
    }

    // ---- items: (token, head) pairs dealt over the teams, a lane's next kAhead on their way -----------------------------------
    struct Item {
        int t, h;
    };
    auto first_item = [&](int heads) -> Item {
        const int t = (int)((uint32_t)team / (uint32_t)heads);
        return {t, team - t * heads};
    };
    const int others = CACHE ? 2 * a.kv_heads : a.k_heads;
    const int q_hop = teams / a.q_heads, q_rest = teams - q_hop * a.q_heads, k_hop = others ? teams / others : 0, k_rest = teams - k_hop * others;
    auto next_item = [](const Item& x, int hop, int rest, int heads) -> Item {
        const int h = x.h + rest;
        return h >= heads ? Item{x.t + hop + 1, h - heads} : Item{x.t + hop, h};
    };
    struct Words {
        u32x4_t a, b;
    };
    auto words_at = [&](const bf16_t* p) -> Words { return {piece_at(p + ea), piece_at(p + eb)}; };
    // Loads have no branches of their own, since a lane whose words are on their way in another branch would wait for them: behind the last item
    // the first one's words again, which go nowhere; values, which go to the cache as they are, as pieces `unit` and `unit` + lanes.
    const int vb = 8 * (unit + lanes) < a.dim ? 8 * (unit + lanes) : 0;
    auto load_cached = [&](const Item& x, int64_t& slot) -> Words {
        const bool in = x.t < count;
        const int64_t token = t0 + (in ? x.t : 0);
        int h = in ? x.h : 0;
        const bool value = h >= a.kv_heads;
        h -= value ? a.kv_heads : 0;
        const bf16_t* p = (value ? a.v : a.k) + token * (value ? a.v_token : a.k_token) + h * (value ? a.v_head : a.k_head);
        slot = a.slots[token];
        return {piece_at(p + (value ? 8 * unit : ea)), piece_at(p + (value ? vb : eb))};
    };
    const Item x0 = first_item(a.q_heads);
    Item y = others ? first_item(others) : Item{count, 0};
    int64_t slot = -1;
    const Words q_raw = words_at(a.q + t0 * a.q_token + (x0.t < count ? x0.t * a.q_token + x0.h * a.q_head : 0));
    Words k_raw = {};
    if constexpr (CACHE) k_raw = load_cached(y, slot);
    else if (others) k_raw = words_at(a.k + t0 * a.k_token + (y.t < count ? y.t * a.k_token + y.h * a.k_head : 0));

    // ---- weights: asked for here, used behind the angles -----------------------------------------------------------------------
    struct Weights {
        u32x4_t word[NORM == kNormWide ? 4 : 2];         // pieces a and b
        int part_a, part_b;
    };
    auto ask_weights = [&](const HeadNormArgs& n) -> Weights {
        Weights w;
        int start_a, start_b;
        const int part_a = norm_part(n, ea, start_a), part_b = norm_part(n, eb, start_b), at_a = ea - start_a, at_b = eb - start_b;
        w.part_a = n.parts ? part_a : -1;
        w.part_b = n.parts ? part_b : -1;
        if (NORM == kNormNone) return w;
        if (n.parts == 0) {                              // heads without a norm beside others with one: times 1
            const uint32_t one = NORM == kNormWide ? 0x3F800000u : 0x3F803F80u;
#pragma unroll
            for (u32x4_t& x : w.word) x = u32x4_t{one, one, one, one};
            return w;
        }
        if constexpr (NORM == kNormWide) {
            const u32x4_t* pa = reinterpret_cast<const u32x4_t*>(static_cast<const float*>(norm_weight(n, part_a)) + at_a);
            const u32x4_t* pb = reinterpret_cast<const u32x4_t*>(static_cast<const float*>(norm_weight(n, part_b)) + at_b);
            w.word[0] = pa[0], w.word[1] = pa[1], w.word[2] = pb[0], w.word[3] = pb[1];
        } else {
            w.word[0] = piece_at(static_cast<const bf16_t*>(norm_weight(n, part_a)) + at_a);
            w.word[1] = piece_at(static_cast<const bf16_t*>(norm_weight(n, part_b)) + at_b);
        }
        return w;
    };
    auto weight_of = [](const Weights& w, int piece, int j) -> float {
        if constexpr (NORM == kNormWide) return __builtin_bit_cast(float, (uint32_t)w.word[2 * piece + j / 4][j & 3]);
        else return (j & 1) ? bf16hi_to_f32(w.word[piece][j / 2]) : bf16lo_to_f32(w.word[piece][j / 2]);
    };
    const Weights qw = ask_weights(a.q_norm), kw = ask_weights(a.k_norm);

    // ---- angles ----------------------------------------------------------------------------------------------------------------
    for (int i = tid; i < count * a.pairs; i += kThreads) {
        const int t = count == 1 ? 0 : i / a.pairs, p = i - t * a.pairs;
        cs_all[i] = cos_sin(a.turns, p, position_of(a, p, t0 + t), a.magnitude);
    }
    __syncthreads();

    // Both pieces normed and turned (all lanes of a wavefront come here together)
    auto turn = [&](Words raw, int t, const HeadNormArgs& n, const Weights& w) -> Words {
        float u[8], v[8];
        unpack8(raw.a, u);
        unpack8(raw.b, v);
        if constexpr (NORM != kNormNone) {
            float sa = 0.f, sb = 0.f, ra = n.parts ? 0.f : 1.f, rb = ra;
#pragma unroll
            for (int j = 0; j < 8; j++) sa = __builtin_fmaf(u[j], u[j], sa), sb = __builtin_fmaf(v[j], v[j], sb);
            if (!there) sa = sb = 0.f;
            auto part = [&](int p) {
                const float mine = (w.part_a == p ? sa : 0.f) + (w.part_b == p ? sb : 0.f);
                const float r = rstd_of(lanes_sum(mine, lane_shift), norm_one_over(n, p), n.eps);
                if (w.part_a == p) ra = r;
                if (w.part_b == p) rb = r;
            };
            // (one or two parts are the usual ones: side by side)
            part(0);
            part(1);
#pragma unroll 1
            for (int p = 2; p < n.parts; p++) part(p);
#pragma unroll
            for (int j = 0; j < 8; j++) u[j] = u[j] * ra * weight_of(w, 0, j), v[j] = v[j] * rb * weight_of(w, 1, j);
        } else if (!rotates) {
            return raw;
        }
        if (rotates) {
            const f32x4_t* cs = reinterpret_cast<const f32x4_t*>(cs_all + t * a.pairs + pair);
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const f32x4_t w2 = cs[j / 2];
#pragma unroll
                for (int i = j; i < j + 2; i++) {
                    const float c = w2[2 * (i - j)], s = w2[2 * (i - j) + 1], x = u[i], z = v[i];
                    if constexpr (NORM) {
                        u[i] = __builtin_fmaf(x, c, -(z * s));
                        v[i] = __builtin_fmaf(z, c, x * s);
                    } else {                             // (as the rotation by one position has it, to the bit)
                        u[i] = x * c - z * s;
                        v[i] = z * c + x * s;
                    }
                }
            }
        }
        return {pack8(u), pack8(v)};
    };

    // All items of the queries, or of the keys.  Where each team has one, its words are stored without a branch, as stores that may have been
    // skipped would have to be waited for with the loads in front of them.
    auto rows = [&](Item x, Words raw, int heads, int hop, int rest, const bf16_t* from, int64_t token, int64_t head, bf16_t* to, int64_t to_token, int64_t to_head,
                    const HeadNormArgs& n, const Weights& w) {
        const int items = count * heads;
        // how far an item's row is from the one before it, in the same run of heads or with one more token
        const int64_t step = hop * token + rest * head, wrap = token - heads * head, to_step = hop * to_token + rest * to_head, to_wrap = to_token - heads * to_head;
        const bf16_t* p = from + t0 * token + x.t * token + x.h * head;
        bf16_t* out = to + (t0 + x.t) * to_token + x.h * to_head;
        int i0 = 0;
        auto item = [&](auto all) {
            const Item next = next_item(x, hop, rest, heads);
            const bool wraps = next.t != x.t + hop;
            Words ahead;
            if (i0 + teams < items) {
                p += wraps ? step + wrap : step;
                ahead = words_at(next.t < count ? p : from + t0 * token);
            }
            const bool in = decltype(all)::value || x.t < count;
            const Words y = turn(raw, in ? x.t : 0, n, w);
            if (in) {
                *reinterpret_cast<u32x4_t*>(out + ea) = y.a;
                *reinterpret_cast<u32x4_t*>(out + eb) = y.b;
            }
            out += wraps ? to_step + to_wrap : to_step;
            x = next;
            raw = ahead;
            i0 += teams;
        };
        while (i0 + teams <= items) item(std::true_type());
        if (i0 < items) item(std::false_type());
    };
    rows(x0, q_raw, a.q_heads, q_hop, q_rest, a.q, a.q_token, a.q_head, a.q_out, a.q_out_token, a.q_out_head, a.q_norm, qw);
    if constexpr (!CACHE) {
        if (others) rows(y, k_raw, others, k_hop, k_rest, a.k, a.k_token, a.k_head, a.k_out, a.k_out_token, a.k_out_head, a.k_norm, kw);
        return;
    }
    const int k_items = count * others;
    bf16_t* room = reinterpret_cast<bf16_t*>(cs_all + a.tokens_per_block * a.pairs) + team * a.dim;
    for (int i0 = 0; i0 < k_items; i0 += teams) {
        const Item next = next_item(y, k_hop, k_rest, others);
        int64_t slot_ahead;
        const Words ahead = load_cached(next, slot_ahead);
        const bool value = y.h >= a.kv_heads;
        Words out = k_raw;
        if (__any(!value)) out = turn(k_raw, y.t < count ? y.t : 0, a.k_norm, kw);
        {
            // through LDS, so that four neighbouring lanes have a run of 32 elements (a head's lanes are one wavefront's)
            if (there && !value) {
                *reinterpret_cast<u32x4_t*>(room + ea) = out.a;
                *reinterpret_cast<u32x4_t*>(room + eb) = out.b;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int h = value ? y.h - a.kv_heads : y.h;
            // slots outside the cache (padding is marked by negative ones) are passed over; the lanes of a run agree
            if (y.t < count && slot >= 0 && slot < a.slot_count) {
                void* pages = value ? a.v_pages : a.k_pages;
                uint16_t* scales = value ? a.v_scales : a.k_scales;
                auto both = [&](auto q8_) {
                    constexpr bool Q8 = decltype(q8_)::value;
                    const CachePlace to = cache_place<Q8>(pages, scales, a, slot, h);
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const int e = 8 * (unit + half * lanes);
                        if (e >= a.dim) continue;
                        cache_piece<Q8>(to, a, e, value ? (half ? k_raw.b : k_raw.a) : *reinterpret_cast<const u32x4_t*>(room + e));
                    }
                };
                if (scales) both(std::integral_constant<bool, true>());
                else both(std::integral_constant<bool, false>());
            }
            __builtin_amdgcn_wave_barrier();             // (the room is written again)
        }
        y = next;
        k_raw = ahead;
        slot = slot_ahead;
    }
}

int launch_head_rotary(const HeadRotaryArgs& a0, int cache, hipStream_t stream) {
    HeadRotaryArgs a = a0;
    bool pairs = !a.interleaved && a.wide && a.dim % 16 == 0;
    for (int p = 0; p < a.parts; p++) pairs = pairs && a.part[p] % 16 == 0;
    if (a.q_norm.parts && a.k_norm.parts && a.q_norm.bf16 != a.k_norm.bf16) pairs = false;       // (weights of two types: the simple one)
    const int elements = pairs ? 16 : 8;                 // of a lane
    while ((elements << a.lane_shift) < a.dim) a.lane_shift++;
    if (pairs && cache && a.lane_shift < 2) a.lane_shift = 2;        // (four lanes for a run of the 8-bit cache)
    const int teams = kThreads >> a.lane_shift;
    const int64_t heads = (int64_t)a.q_heads + (cache ? 2 * a.kv_heads : a.k_heads);
    // as many tokens as give each team a head; where there are tokens enough for two workgroups a compute unit, up to four times as many, as
    // finding its elements and weights costs a workgroup as much as two heads do (40 normed heads, 1 / 2 / 4 tokens a workgroup: 4096 tokens
    // 27.9 / 21.0 / 17.4 us, 3000 22.2 / 17.6 / 14.3, 2048 16.6 / 12.6 / 12.3; eight: 33000 139.7 against 134.4)
    const int64_t fill = heads * 8 <= teams ? 8 : heads < teams ? teams / heads : 1;
    const int64_t spare = a.tokens / (512 * fill);
    const int64_t tokens = fill * (spare < 1 ? 1 : spare > 4 ? 4 : spare), room = 2048 / a.pairs;       // (16 KB of cosines and sines)
    a.tokens_per_block = (int32_t)(tokens < room ? tokens : room);
    const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    if (blocks * kThreads >= (int64_t)1 << 32) return SNGGUF_E_BADSHAPE;     // (threads of a launch are numbered with 32 bits)
    const bool norm = a.q_norm.parts || a.k_norm.parts;
    const size_t lds = (size_t)a.tokens_per_block * a.pairs * sizeof(float2) + (pairs && cache ? (size_t)teams * a.dim * 2 : 0);
    const dim3 grid((unsigned)blocks);
    const HeadNormArgs& one = a.q_norm.parts ? a.q_norm : a.k_norm;
    const int kind = !norm ? kNormNone : one.bf16 ? kNormHalf : kNormWide;
#define SNGGUF_GO(C)                                                                                                    \
    if ((cache != 0) == C) {                                                                                            \
        if (pairs && kind == kNormNone) head_pairs_kernel<C, kNormNone, -1><<<grid, kThreads, lds, stream>>>(a);        \
        else if (pairs && kind == kNormHalf && a.lane_shift == 3) head_pairs_kernel<C, kNormHalf, 3><<<grid, kThreads, lds, stream>>>(a); \
        else if (pairs && kind == kNormHalf) head_pairs_kernel<C, kNormHalf, -1><<<grid, kThreads, lds, stream>>>(a);   \
        else if (pairs) head_pairs_kernel<C, kNormWide, -1><<<grid, kThreads, lds, stream>>>(a);                        \
        else if (a.interleaved && norm) head_rotary_kernel<kNeighbours, C, true><<<grid, kThreads, lds, stream>>>(a);   \
        else if (a.interleaved) head_rotary_kernel<kNeighbours, C, false><<<grid, kThreads, lds, stream>>>(a);          \
        else if (norm) head_rotary_kernel<kAnyHalves, C, true><<<grid, kThreads, lds, stream>>>(a);                     \
        else head_rotary_kernel<kAnyHalves, C, false><<<grid, kThreads, lds, stream>>>(a);                              \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
    SNGGUF_GO(false)
    SNGGUF_GO(true)
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

}  // namespace sngguf
