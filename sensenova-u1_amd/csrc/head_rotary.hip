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
// Bound by memory: an element is two bytes in and two out, for some ten operations.  2^lane_shift neighbouring lanes have a head,
// 16 bytes each: its sums of squares are added up across them in the vector unit, and a lane gets its pairs' other elements from
// the lane that has them (parts that are no multiple of 16 elements: from memory, where they were just read).  All of a head is
// read before any of it is written, so a call may work in place.  A workgroup's lanes keep to the same elements of
// all heads, so weights, cosines and sines are fetched once for a token.
#include "head_rotary.hpp"
#include "rotary_cache_device.hpp"

namespace sngguf {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;                                // heads of a lane that are asked for at once

enum { kHalves = 0, kNeighbours = 1, kAnyHalves = 2 };   // parts of multiples of 16 elements; pairs next to each other; any parts

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

__device__ __forceinline__ float rstd_of(float sum, int elements, float eps) { return 1.0f / sqrtf(sum / (float)elements + eps); }

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
__device__ __forceinline__ int norm_elements(const HeadNormArgs& n, int p) { return p == 0 ? n.elements[0] : p == 1 ? n.elements[1] : p == 2 ? n.elements[2] : n.elements[3]; }

// What a lane keeps of a norm: weights of its eight elements and of their pairs' others, and the parts that they belong to
struct LaneNorm {
    float g[8], gz[8];
    int part, elements;
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
    // kHalves: pairs from `pair` on, the others in the lane `away` further; kAnyHalves: each element by itself
    int pair = 0, away = 0;
    bool second = false, rotates = there && e < turned;
    int z_at[8], pairs_of[8];
    uint32_t seconds = 0, rotated = 0;
    if constexpr (LAYOUT == kHalves) {
        int start = 0, first = 0;
#pragma unroll
        for (int p = 0; p < kMostParts; p++) {
            const int n = p < a.parts ? a.part[p] : 0;
            if (e >= start && e < start + n) {
                second = e - start >= n / 2;
                pair = first + (second ? e - start - n / 2 : e - start);
                away = second ? -(n / 16) : n / 16;
            }
            start += n;
            first += n / 2;
        }
    } else if constexpr (LAYOUT == kNeighbours) {
        pair = e >> 1;
    } else {
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
    const int z_lane = (tid & 63) + away;                // (a part lies in one head, and a head in one wavefront)

    // ---- weights -------------------------------------------------------------------------------------------------------
    auto weights = [&](const HeadNormArgs& n) -> LaneNorm {
        LaneNorm w;
        int start;
        w.part = norm_part(n, there ? e : 0, start);
        w.elements = norm_elements(n, w.part);
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
        if constexpr (LAYOUT == kHalves) {
#pragma unroll
            for (int j = 0; j < 8; j++) w.gz[j] = __shfl(w.g[j], z_lane);
            w.z_parts = (uint32_t)__shfl(w.part, z_lane);
        } else if constexpr (LAYOUT == kNeighbours) {
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
        int axis = a.axis ? a.axis[p] : 0;
        axis = axis < 0 ? 0 : axis >= a.axes ? a.axes - 1 : axis;
        cs_all[i] = cos_sin(a.turns, p, a.positions[axis * a.axis_stride + t0 + t], a.magnitude);
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
            if constexpr (LAYOUT == kHalves) {
                if (rotates) c[j] = cs[pair + j].x, s[j] = second ? cs[pair + j].y : -cs[pair + j].y;
            } else if constexpr (LAYOUT == kNeighbours) {
                if (there && e + j < turned) c[j] = cs[pair + j / 2].x, s[j] = (j & 1) ? cs[pair + j / 2].y : -cs[pair + j / 2].y;
            } else {
                if (rotated >> j & 1) c[j] = cs[pairs_of[j]].x, s[j] = (seconds >> j & 1) ? cs[pairs_of[j]].y : -cs[pairs_of[j]].y;
            }
        }
    };

    // ---- eight elements of a head, normed and turned (all lanes of a wavefront come here together) -----------------------------
    auto turned8 = [&](u32x4_t raw, const bf16_t* row, const HeadNormArgs& n, const LaneNorm& w) -> u32x4_t {
        float x[8], z[8];
        unpack8(raw, x);
        if constexpr (LAYOUT == kHalves) {
            u32x4_t other;
#pragma unroll
            for (int i = 0; i < 4; i++) other[i] = (uint32_t)__shfl((int)raw[i], z_lane);
            unpack8(other, z);
            if (!rotates) {
#pragma unroll
                for (int j = 0; j < 8; j++) z[j] = 0.f;
            }
        } else if constexpr (LAYOUT == kNeighbours) {
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
                if (LAYOUT != kAnyHalves && n.group) {
                    r = rstd_of(lanes_sum(ss, __builtin_ctz(n.group)), w.elements, n.eps);
                    if (n.parts == 1 || LAYOUT == kNeighbours) rz[0] = r;
                    else rz[0] = __shfl(r, z_lane);
                } else {
                    for (int p = 0; p < n.parts; p++) {
                        const float rp = rstd_of(lanes_sum(there && w.part == p ? ss : 0.f, a.lane_shift), norm_elements(n, p), n.eps);
                        if (w.part == p) r = rp;
#pragma unroll
                        for (int j = 0; j < (LAYOUT == kAnyHalves ? 8 : 1); j++)
                            if ((w.z_parts >> (4 * j) & 15u) == (uint32_t)p) rz[j] = rp;
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[j] = x[j] * r * w.g[j];
                    z[j] = z[j] * rz[LAYOUT == kAnyHalves ? j : 0] * w.gz[j];
                }
                if (LAYOUT == kHalves && !rotates) {     // (weights that are not finite)
#pragma unroll
                    for (int j = 0; j < 8; j++) z[j] = 0.f;
                } else if (LAYOUT != kHalves) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (LAYOUT == kNeighbours ? e + j >= turned : !(rotated >> j & 1)) z[j] = 0.f;
                }
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
            if (scales) cache_piece<true>(pages, scales, a, slot, h, e, held);
            else cache_piece<false>(pages, scales, a, slot, h, e, held);
        }
    }
}

int launch_head_rotary(const HeadRotaryArgs& a0, int cache, hipStream_t stream) {
    HeadRotaryArgs a = a0;
    while ((8 << a.lane_shift) < a.dim) a.lane_shift++;
    const int teams = kThreads >> a.lane_shift;
    const int64_t heads = (int64_t)a.q_heads + (cache ? 2 * a.kv_heads : a.k_heads);
    a.tokens_per_block = heads >= teams ? 1 : heads * 8 <= teams ? 8 : (int32_t)(teams / heads);
    const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    if (blocks * kThreads >= (int64_t)1 << 32) return SNGGUF_E_BADSHAPE;     // (threads of a launch are numbered with 32 bits)
    bool halves = !a.interleaved;
    for (int p = 0; p < a.parts; p++) halves = halves && a.part[p] % 16 == 0;
    const int layout = a.interleaved ? kNeighbours : halves ? kHalves : kAnyHalves;
    const bool norm = a.q_norm.parts || a.k_norm.parts;
    const size_t lds = (size_t)a.tokens_per_block * a.pairs * sizeof(float2);
#define SNGGUF_GO(L, C, N)                                                                                              \
    if (layout == L && (cache != 0) == C && norm == N) {                                                                \
        head_rotary_kernel<L, C, N><<<dim3((unsigned)blocks), kThreads, lds, stream>>>(a);                              \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
#define SNGGUF_GO_ALL(L) SNGGUF_GO(L, false, false) SNGGUF_GO(L, false, true) SNGGUF_GO(L, true, false) SNGGUF_GO(L, true, true)
    SNGGUF_GO_ALL(kHalves)
    SNGGUF_GO_ALL(kNeighbours)
    SNGGUF_GO_ALL(kAnyHalves)
#undef SNGGUF_GO_ALL
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

}  // namespace sngguf
