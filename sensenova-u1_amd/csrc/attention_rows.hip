// Attention of few rows over a paged cache: single new tokens, and short runs of them.
//
//     o = sum_j softmax_j(scale q . k_j) v_j  over the keys j of the sequence that the row sees
//
// in one pass over the keys with a running maximum m and sum l (in base 2: p_j = exp2(scale log2(e) q . k_j - m)).  Bound by
// the bytes of the cache, so a workgroup's wavefronts read keys and values straight into registers, in the order in which
// the matrix instructions want them, and never through LDS; each wavefront takes every fourth run of 32 keys with a maximum
// and a sum of its own, and the four are joined at the end.  Sequences are split over workgroups where there are few.
// Measured, 32 query and 8 key / value heads of 128: 24 tokens over 37 .. 9996 in 8 bits 49.5 us, 5.3 TB/s; one over 131071 in bf16
// 80 us, 6.6 TB/s (the same cache each time, which stays in the last-level cache in part; a kernel that only reads: 6.5); the join 6 to 7
// us more.  Short runs of new tokens are bound by their arithmetic, which one or two wavefronts a SIMD do not overlap: 8 new tokens each of 16
// sequences of 8000 in 8 bits 3.5 TB/s, 16 of 4 1.3.
//
// Per run of 32 keys and 16 rows (columns of the 16 x 16 x 32 instructions, lane % 16; lane group g = lane / 16):
//  * scores: K (16 keys x dim) times Q^T.  The order in which dim is summed is free: in 8 bits lane group g takes elements
//    [g DT / 4, (g + 1) DT / 4) of its key's row, in bf16 eight of every 32.  Matrix row 4 g + i of the first instruction is key
//    8 g + i, of the second key 8 g + 4 + i;
//  * so a lane's eight scores are of keys 8 g .. 8 g + 7, which is how the second product wants them: V^T (16 elements x 32
//    keys) times P^T, where lane group g holds keys 8 g .. 8 g + 7.  A lane reads DT / 16 neighbouring elements of those eight
//    rows, and instruction t takes element t of each.
// What is rounded: in bf16 the weights, to bf16, for the product with the values (the matrix instructions take both operands in one type;
// weights in two parts would be twice the instructions).  It is most of the error: one token over 131071 is off by 0.0023 of its norm from the
// definition, where fp32 weights and a result in bf16 are off by 0.0017.  An 8-bit cache is widened to fp16 (whole numbers are
// exact there, the product with the scale is rounded to 11 bits; values are within fp16 by the format) and multiplied in fp16, queries scaled
// into it by a power of two, with p scaled by 2^12: p down to 2^-36 of the largest still counts, and 11 bits are enough: 0.0017.
// The sum of a row's weights is of the fp32 ones: their roundings are to the nearest and cancel in a long sum, and the sum is done while the
// rounded ones are still being packed.  Scores, maxima, sums and the values' sums are fp32.
#include <type_traits>

#include "attention.hpp"

namespace sngguf {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kRun = 32;                    // keys of a wavefront's step
constexpr int kKeys = kRun * kWaves;        // keys of a workgroup's step

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

template <bool Q8> struct Operand { typedef bf16x8_t T; };
template <> struct Operand<true> { typedef f16x8_t T; };

__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4_t mfma(f16x8_t a, f16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)a, (_Float16)b});
}

// bytes 0, 1 (HIGH: 2, 3) of four int8 with their sign bits flipped -> two fp16 whole numbers: 0x6400 | u is 1024 + u
template <bool HIGH>
__device__ __forceinline__ f16x2_t whole_pair(uint32_t flipped) {
    const uint32_t w = __builtin_amdgcn_perm(0x64646464u, flipped, HIGH ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(f16x2_t, w) + f16x2_t{(_Float16)-1152.f, (_Float16)-1152.f};
}

// Words of the cache; ONCE: that one workgroup reads once, and no other does
template <bool ONCE, typename T> __device__ __forceinline__ T word_at(const uint8_t* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
    else return *reinterpret_cast<const T*>(p);
}

}  // namespace

// Workgroups that a compute unit takes at a time (as many wavefronts a SIMD: four a workgroup).  Heads of 256 elements: one, as two
// spill (32 single tokens over 4000 in bf16: 193 us against 297).
constexpr int rows_workgroups(int dt, int nt) { return nt * dt <= 128 ? 3 : nt * dt <= 256 && dt < 256 ? 2 : 1; }

// DT: elements of a head, rounded up (FULL: exactly).  NT: 16-row tiles.
template <int DT, bool FULL, bool Q8, int NT>
__global__ __launch_bounds__(kThreads, rows_workgroups(DT, NT)) void attention_rows_kernel(AttentionArgs a) {
    typedef typename Operand<Q8>::T op_t;
    constexpr int ROWS = 16 * NT;
    constexpr int KP = DT / 4;              // elements of a key that a lane reads
    constexpr int VP = DT / 16;             // elements of a value that a lane reads
    constexpr int KC = KP / 8;              // instructions of a score
    constexpr int KW = Q8 ? KC / 2 : KC;    // 16-byte words of a key
    constexpr int KR = DT / 128 > 0 ? DT / 128 : 1;   // scales of a key
    constexpr int VW = Q8 ? VP / 4 : VP / 2;          // dwords of a value
    constexpr int E = Q8 ? 1 : 2;           // bytes of an element
    // Pages that no other sequence has are read with the read-once hint, where a line is not asked for again much later (wider heads take a line
    // in four requests, heads between two kernels read pieces in place of those behind them).  16 tokens over 8000, each over a cache of
    // its own: 128 elements in bf16 92 us against 101, in 8 bits 59 against 62; 96 in bf16 84 against 81, 256 in 8 bits 134 against
    // 112.  Pages that sequences share come from a cache but for the first time: with the hint 8 sequences with 32768 tokens in common took
    // 141 us instead of 91 (8 bits 87, 70).  Who shares is asked only by tiles of 16 rows: a loop with both kinds of loads has four new
    // tokens each over 8000 2 to 5 % slower (60 us instead of 76 with the 8000 in common), eight new ones, in 32 rows, 6 to 12 %.  Heads of 64 in
    // 8 bits do not ask, which lose as much as they gain (16 over 8000 34.8 us, asking 37.4; 8 with 32768 in common 50.0, 48.0).
    constexpr bool HINT = FULL && DT <= 128, ASK = HINT && NT == 1 && !(Q8 && DT == 64);
    constexpr float kUp = Q8 ? 12.f : 0.f;
    constexpr float kLimit = Q8 ? 32768.f : 1e9f;
    extern __shared__ __attribute__((aligned(16))) float lds[];   // [wave][16][DT] sums, then [wave][ROWS][2]
    float* stats = lds + kWaves * 16 * DT;

    const AttentionBlock b = attention_block<ROWS, kKeys, false>(a, blockIdx.x);
    if (!b.there) return;
    const int dim = FULL ? DT : a.dim;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int64_t rows = (int64_t)b.s.lq * a.group;
    const int64_t r0 = (int64_t)b.row_tile * ROWS, r1 = r0 + ROWS < rows ? r0 + ROWS : rows;
    int32_t lo, hi;
    attention_keys(a, b.s, r0, r1, lo, hi);
    const int32_t back = b.s.lk - b.s.lq, most = b.s.lk - 1;

    // ---- this split's runs, and the cache's words of a run -----------------------------------------------------------------
    int32_t s0 = lo / kKeys, s1 = (hi + kKeys - 1) / kKeys;
    {
        const int32_t per = (s1 - s0 + b.splits - 1) / b.splits;
        s0 += per * b.split;
        s1 = s0 + per < s1 ? s0 + per : s1;
    }
    const int32_t end = s1 * kKeys < hi ? s1 * kKeys : hi;
    const int32_t page_mask = (1 << a.page_shift) - 1;
    const int32_t* table = a.table + (int64_t)b.seq * a.table_stride;
    auto page_of = [&](int32_t key) -> int32_t {
        const int32_t p = table[(key < most ? key : most) >> a.page_shift];
        return p < 0 ? 0 : p >= a.pages ? a.pages - 1 : p;
    };
    // key of matrix row `col` in the two score instructions: 8 (col / 4) + col % 4 (+ 4); values: keys 8 g .. 8 g + 7
    const int k_key = 8 * (col >> 2) + (col & 3), v_key = 8 * g;
    int k_e[KW];                            // (pieces behind dim: the first, whose elements meet queries of zero)
#pragma unroll
    for (int x = 0; x < KW; x++) {
        const int e = Q8 ? KP * g + 16 * x : 32 * x + 8 * g;
        k_e[x] = FULL || e < dim ? e : 0;
    }
    const int v_e = FULL || VP * col < dim ? VP * col : 0;      // (behind dim: never stored)
    u32x4_t k_raw[2][KW];
    uint16_t k_scale[2][KR];
    uint32_t v_raw[8][VW];
    u32x4_t v_scale;
    auto load_keys_as = [&](auto once_, int32_t key0, int32_t page) {
        constexpr bool ONCE = decltype(once_)::value;
        const int64_t at = (int64_t)page * a.kv_heads + b.kv_head;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int32_t key = key0 + k_key + 4 * i, row = (key < most ? key : most) & page_mask;
            const uint8_t* p = static_cast<const uint8_t*>(a.k_pages) + ((at << a.page_shift) + row) * (dim * E);
#pragma unroll
            for (int x = 0; x < KW; x++) k_raw[i][x] = word_at<ONCE, u32x4_t>(p + E * k_e[x]);
            if constexpr (Q8) {
                const uint16_t* sc = a.k_scales + (at * (dim >> 5) << a.page_shift) + row;
#pragma unroll
                for (int x = 0; x < KR; x++) k_scale[i][x] = sc[(int64_t)(k_e[x * (KW / KR)] >> 5) << a.page_shift];
            }
        }
    };
    auto load_values_as = [&](auto once_, int32_t key0, int32_t page) {
        constexpr bool ONCE = decltype(once_)::value;
        const int64_t at = (int64_t)page * a.kv_heads + b.kv_head;
        const int32_t lead = key0 + v_key < most ? key0 + v_key : most, row = lead & page_mask & ~7;
        const uint8_t* p = static_cast<const uint8_t*>(a.v_pages) + ((at << a.page_shift) + row) * (dim * E) + E * v_e;
        auto word = [&](int j, int r) {
            const uint8_t* q = p + r * (dim * E);
            if constexpr (VW == 1) v_raw[j][0] = word_at<ONCE, uint32_t>(q);
            else if constexpr (VW == 2) {
                const u32x2_t w = word_at<ONCE, u32x2_t>(q);
                v_raw[j][0] = w[0], v_raw[j][1] = w[1];
            } else {
#pragma unroll
                for (int x = 0; x < VW; x += 4) {
                    const u32x4_t w = word_at<ONCE, u32x4_t>(q + 4 * x);
#pragma unroll
                    for (int y = 0; y < 4; y++) v_raw[j][x + y] = w[y];
                }
            }
        };
        if (key0 + kRun <= b.s.lk) {
#pragma unroll
            for (int j = 0; j < 8; j++) word(j, j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int32_t last = (most & page_mask) - row;     // of these eight, or of the eight that are read in their place
                word(j, key0 + v_key + j <= most ? j : last);
            }
        }
        if constexpr (Q8) v_scale = *reinterpret_cast<const u32x4_t*>(a.v_scales + ((at * (dim >> 5) + (v_e >> 5)) << a.page_shift) + row);
    };
    typedef std::integral_constant<bool, false> Often;
    typedef std::integral_constant<bool, true> Once;
    bool once = false;
    // (the marks keep the compiler from making one load without the hint of the two)
    auto load_keys = [&](int32_t key0, int32_t page) {
        if constexpr (!ASK) {
            load_keys_as(std::integral_constant<bool, HINT>(), key0, page);
        } else if (once) {
            load_keys_as(Once(), key0, page);
            asm volatile("; once");
        } else {
            load_keys_as(Often(), key0, page);
        }
    };
    auto load_values = [&](int32_t key0, int32_t page) {
        if constexpr (!ASK) {
            load_values_as(std::integral_constant<bool, HINT>(), key0, page);
        } else if (once) {
            load_values_as(Once(), key0, page);
            asm volatile("; once");
        } else {
            load_values_as(Often(), key0, page);
        }
    };
    int32_t key0 = s0 * kKeys + wave * kRun;
    int32_t page_k = 0, page_v = 0;
    if (key0 < end) {
        page_k = page_of(key0 + (k_key & ~7));
        page_v = page_of(key0 + v_key);
        if constexpr (ASK) {
            // this split's first page, and what up to 63 other sequences have in its place: a common prompt is at the same place in all tables
            const int32_t other = (b.seq & ~63) + lane, at = (s0 * kKeys) >> a.page_shift;
            const bool there = other < a.sequences && other != b.seq;
            const int32_t mine = table[at], theirs = a.table[(int64_t)(there ? other : b.seq) * a.table_stride + at];
            once = __ballot(there && theirs == mine) == 0;
        }
        load_keys(key0, page_k);
        load_values(key0, page_v);
        page_k = page_of(key0 + kKeys + (k_key & ~7));
        page_v = page_of(key0 + kKeys + v_key);
    }

    // ---- queries: operand fragments, and which keys each column sees ---------------------------------------------------
    op_t qf[NT][KC];
    float c[NT];                            // scale_log2 x what the row was scaled by
    int32_t first[NT], last[NT];            // visible keys of the column's row, inclusive
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int64_t r = r0 + 16 * n + col;
        const int64_t rr = r < r1 ? r : r1 - 1;
        int32_t head;
        const int32_t token = attention_token(a, rr, head);
        head += b.kv_head * a.group;
        const bf16_t* q = a.q + (b.s.q0 + token) * a.q_token + (int64_t)head * a.q_head;
        const int32_t place = back + token;
        last[n] = a.causal && place < most ? place : most;
        first[n] = a.window && place - a.window + 1 > 0 ? (int32_t)(place - a.window + 1) : 0;
        u32x4_t raw[KC];
#pragma unroll
        for (int i = 0; i < KC; i++) {
            const int e = Q8 ? KP * g + 8 * i : 32 * i + 8 * g;
            raw[i] = FULL || e < dim ? *reinterpret_cast<const u32x4_t*>(q + e) : u32x4_t{0u, 0u, 0u, 0u};
        }
        c[n] = a.scale_log2;
        if constexpr (Q8) {
            // bf16 -> fp16: scaled by a power of two that brings the row's largest element into [1, 2)
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < KC; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t x = raw[i][j] & 0x7F807F80u;
                    top = max(top, max(x >> 16, x & 0xFFFFu));
                }
            top = max(top, (uint32_t)__shfl_xor((int)top, 16));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            const int ex = top == 0 ? 0 : (int)(top >> 7) - 127;
#pragma unroll
            for (int i = 0; i < KC; i++) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = pack_f16(__builtin_ldexpf(bf16lo_to_f32(raw[i][j]), -ex), __builtin_ldexpf(bf16hi_to_f32(raw[i][j]), -ex));
                qf[n][i] = __builtin_bit_cast(op_t, w);
            }
            c[n] = fmaxf(__builtin_ldexpf(c[n], ex), 1.2e-38f);
        } else {
#pragma unroll
            for (int i = 0; i < KC; i++) qf[n][i] = __builtin_bit_cast(op_t, raw[i]);
        }
    }
    // keys that every row of the tile sees
    const int32_t place0 = back + (int32_t)((uint32_t)r0 / (uint32_t)a.group), place1 = back + (int32_t)((uint32_t)(r1 - 1) / (uint32_t)a.group);
    const int32_t all_last = a.causal && place0 < most ? place0 : most;
    const int32_t all_first = a.window && place1 - a.window + 1 > 0 ? (int32_t)(place1 - a.window + 1) : 0;

    f32x4_t acc[NT][VP];
    float m[NT], l[NT], nb[NT];             // nb: what is added to a scaled score, kUp - m
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = -__builtin_inff();
        nb[n] = __builtin_inff();           // nothing known yet: whatever is formed with it is set right
        l[n] = 0.f;
#pragma unroll
        for (int t = 0; t < VP; t++) acc[n][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    for (; key0 < end; key0 += kKeys) {
        const bool more = key0 + kKeys < end;
        float sc[NT][8];
        {
            op_t kf[2][KC];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if constexpr (Q8) {
#pragma unroll
                    for (int x = 0; x < KW; x++) {
                        const _Float16 d = __builtin_bit_cast(_Float16, k_scale[i][x / (KW / KR)]);
                        const f16x2_t dd = {d, d};
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            u32x4_t f;
#pragma unroll
                            for (int z = 0; z < 2; z++) {
                                const uint32_t flipped = k_raw[i][x][2 * y + z] ^ 0x80808080u;
                                f[2 * z] = __builtin_bit_cast(uint32_t, whole_pair<false>(flipped) * dd);
                                f[2 * z + 1] = __builtin_bit_cast(uint32_t, whole_pair<true>(flipped) * dd);
                            }
                            kf[i][2 * x + y] = __builtin_bit_cast(op_t, f);
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < KC; x++) kf[i][x] = __builtin_bit_cast(op_t, k_raw[i][x]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                f32x4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int x = 0; x < KC; x++)
#pragma unroll
                    for (int i = 0; i < 2; i++) s[i] = mfma(kf[i][x], qf[n][x], s[i]);
#pragma unroll
                for (int j = 0; j < 8; j++) sc[n][j] = s[j >> 2][j & 3];
            }
        }
        if (more) load_keys(key0 + kKeys, page_k);
        if (key0 + kRun - 1 > all_last || key0 < all_first) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int32_t key = key0 + v_key + j;
                    if (key < first[n] || key > last[n]) sc[n][j] = -__builtin_inff();
                }
        }
        // weights with the maximum known so far; only where they run away are maximum, sums and weights set right
        float p[NT][8], sum[NT];
        bool fine = true;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            sum[n] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[n][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][j], c[n], nb[n]));
                sum[n] += p[n][j];
            }
            fine = fine && sum[n] <= kLimit;
        }
        if (__any(!fine)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float top = sc[n][0];
#pragma unroll
                for (int j = 1; j < 8; j++) top = fmaxf(top, sc[n][j]);
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                top = fmaxf(top * c[n], m[n]);
                const bool none = top == -__builtin_inff();
                const float base = none ? 0.f : top, keep = __builtin_amdgcn_exp2f(m[n] - base);
                m[n] = top;
                nb[n] = none ? __builtin_inff() : kUp - base;
                l[n] *= keep;
#pragma unroll
                for (int t = 0; t < VP; t++) acc[n][t] *= keep;
                sum[n] = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[n][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[n][j], c[n], kUp - base));
                    sum[n] += p[n][j];
                }
            }
        }
        op_t pf[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            l[n] += sum[n];
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = Q8 ? pack_f16(p[n][2 * j], p[n][2 * j + 1]) : pack_bf16(p[n][2 * j], p[n][2 * j + 1]);
            pf[n] = __builtin_bit_cast(op_t, w);
        }
        // vf: element t of keys 8 g .. 8 g + 7
        u32x4_t vf[VP];
        if constexpr (Q8) {
            if (key0 + kRun > b.s.lk) {
                // scales behind the last key were never written: not even a zero may meet them
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (key0 + v_key + j > most) v_scale[j >> 1] &= (j & 1) ? 0x0000FFFFu : 0xFFFF0000u;
            }
#pragma unroll
            for (int x = 0; x < VW; x++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t dw = v_scale[j];      // (a bit cast of a vector's element itself takes element 0)
                    const f16x2_t d = __builtin_bit_cast(f16x2_t, dw);
                    const uint32_t a0 = v_raw[2 * j][x] ^ 0x80808080u, a1 = v_raw[2 * j + 1][x] ^ 0x80808080u;
                    // pairs of elements of each key -> pairs of keys of each element
                    const uint32_t l0 = __builtin_bit_cast(uint32_t, whole_pair<false>(a0)), l1 = __builtin_bit_cast(uint32_t, whole_pair<false>(a1));
                    const uint32_t h0 = __builtin_bit_cast(uint32_t, whole_pair<true>(a0)), h1 = __builtin_bit_cast(uint32_t, whole_pair<true>(a1));
                    vf[4 * x][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(l1, l0, 0x05040100u)) * d);
                    vf[4 * x + 1][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(l1, l0, 0x07060302u)) * d);
                    vf[4 * x + 2][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(h1, h0, 0x05040100u)) * d);
                    vf[4 * x + 3][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(h1, h0, 0x07060302u)) * d);
                }
        } else {
#pragma unroll
            for (int x = 0; x < VW; x++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    vf[2 * x][j] = __builtin_amdgcn_perm(v_raw[2 * j + 1][x], v_raw[2 * j][x], 0x05040100u);
                    vf[2 * x + 1][j] = __builtin_amdgcn_perm(v_raw[2 * j + 1][x], v_raw[2 * j][x], 0x07060302u);
                }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int t = 0; t < VP; t++) acc[n][t] = mfma(__builtin_bit_cast(op_t, vf[t]), pf[n], acc[n][t]);
        if (more) {
            load_values(key0 + kKeys, page_v);
            page_k = page_of(key0 + 2 * kKeys + (k_key & ~7));
            page_v = page_of(key0 + 2 * kKeys + v_key);
        }
    }

    // ---- the four wavefronts' results --------------------------------------------------------------------------------
    uint32_t again = 0;                     // this wavefront's rows that are not finite: four of each 16
#pragma unroll
    for (int n = 0; n < NT; n++) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        if (g == 0) {
            stats[(wave * ROWS + 16 * n + col) * 2] = m[n];
            stats[(wave * ROWS + 16 * n + col) * 2 + 1] = l[n];
        }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; n++) {
        float top = -__builtin_inff(), mine;
#pragma unroll
        for (int w = 0; w < kWaves; w++) top = fmaxf(top, stats[(w * ROWS + 16 * n + col) * 2]);
        mine = m[n] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m[n] - top);
        // acc[n][t][i]: column col, element VP (4 g + i) + t
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < VP; t += 4)
                *reinterpret_cast<f32x4_t*>(lds + (wave * 16 + col) * DT + VP * (4 * g + i) + t) =
                    f32x4_t{acc[n][t][i] * mine, acc[n][t + 1][i] * mine, acc[n][t + 2][i] * mine, acc[n][t + 3][i] * mine};
        __syncthreads();
        // thread: row tid / 16 of the tile, elements VP (tid % 16) ...
        const int row = threadIdx.x >> 4, e = VP * (threadIdx.x & 15);
        const int64_t r = r0 + 16 * n + row;
        float odd = 0.f;
        if (r < r1 && e < dim) {
            float o[VP];
#pragma unroll
            for (int t = 0; t < VP; t++) {
                o[t] = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; w++) o[t] += lds[(w * 16 + row) * DT + e + t];
            }
            float rm = -__builtin_inff(), rl = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; w++) rm = fmaxf(rm, stats[(w * ROWS + 16 * n + row) * 2]);
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                const float wm = stats[(w * ROWS + 16 * n + row) * 2];
                if (wm != -__builtin_inff()) rl += stats[(w * ROWS + 16 * n + row) * 2 + 1] * __builtin_amdgcn_exp2f(wm - rm);
            }
            odd = rl * 0.f;
#pragma unroll
            for (int t = 0; t < VP; t++) odd = __builtin_fmaf(o[t], 0.f, odd);
            if (b.splits > 1) {
                float* part = a.partial + (b.slot * ROWS + 16 * n + row) * DT + e;
#pragma unroll
                for (int t = 0; t < VP; t += 4) *reinterpret_cast<f32x4_t*>(part + t) = f32x4_t{o[t], o[t + 1], o[t + 2], o[t + 3]};
                if (e == 0) {
                    float* st = a.partial + a.grid * ROWS * DT + (b.slot * ROWS + 16 * n + row) * 2;
                    st[0] = rm;
                    st[1] = rl;
                }
            } else {
                const float inv = rl == 0.f ? 0.f : 1.f / rl;
                int32_t head;
                const int32_t token = attention_token(a, r, head);
                head += b.kv_head * a.group;
                bf16_t* out = a.out + (b.s.q0 + token) * a.out_token + (int64_t)head * a.out_head + e;
#pragma unroll
                for (int t = 0; t < VP; t += 4)
                    *reinterpret_cast<u32x2_t*>(out + t) = u32x2_t{pack_bf16(o[t] * inv, o[t + 1] * inv), pack_bf16(o[t + 2] * inv, o[t + 3] * inv)};
            }
        }
        const uint64_t odd_lanes = __ballot(odd != 0.f);
#pragma unroll
        for (int i = 0; i < 4; i++) again |= (odd_lanes >> (16 * i) & 0xFFFFu) ? 1u << (4 * n + i) : 0u;
        __syncthreads();
    }
    // (this wavefront's stores above stay in front: these rows are written twice, and the second is what is left)
    while (again) {
        const int i = __builtin_ctz(again);
        again &= again - 1;
        attention_row_again<DT, Q8 ? kPagedQ8 : kPaged, ROWS, Q8 ? 12 : 0>(a, b, r0 + 16 * (i >> 2) + 4 * wave + (i & 3), s0 * kKeys, end);
    }
}

// A lane's elements of a row that is not finite again, split by split: what was read for a split behind the last may be an infinity, which a
// weight of zero makes NaN, and splits whose sums are within fp32 can have one together that is not, unless all weights are that
// much smaller (there are at most as many splits as workgroups, below 2^16).  A function of its own: in line it takes registers from the
// loads under way (three workgroups a compute unit instead of four: 16 sequences of 8 new tokens over 8000 84 us instead of 79).
template <int PER>
__device__ __attribute__((noinline)) void join_row_again(const float* stats, const float* part, int step, int dim, int splits, bf16_t* out) {
    float o[PER], l = 0.f, m = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < PER; t++) o[t] = 0.f;
    for (int s = 0; s < splits; s++) {
        const int64_t at = (int64_t)s * step;
        const float ms = stats[at * 2], ls = stats[at * 2 + 1], top = fmaxf(m, ms);
        if (top == -__builtin_inff()) continue;
        const float keep = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(ms - top) * 0x1p-16f;
        m = top;
        l = l * keep + ls * w;
#pragma unroll
        for (int t = 0; t < PER; t++) o[t] = o[t] * keep + part[at * dim + t] * w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int t = 0; t < PER; t += 2) *reinterpret_cast<uint32_t*>(out + t) = pack_bf16(o[t] * inv, o[t + 1] * inv);
}

// Joins the splits of rows.  WIDE: a workgroup a row; else a wavefront a row.  Half a wavefront lies along the row's elements and
// takes some splits at a time, all of whose words are asked for before any is used (behind the last split, those of the first
// again: a branch around a load would have the loads wait for each other): the launch is one latency long, and what it
// reads is little.
template <int ROWS, int KEYS, int DT, bool WIDE>
__global__ __launch_bounds__(kThreads) void attention_combine_kernel(AttentionArgs a) {
    constexpr int PER = DT / 32;            // elements of a lane
    constexpr int TEAMS = WIDE ? 2 * kWaves : 2;
    __shared__ float part[WIDE ? TEAMS : 1][DT + 2];
    const AttentionBlock b = attention_block<ROWS, KEYS, true>(a, blockIdx.x);
    // (lengths that are none can name more splits than there were workgroups)
    if (!b.there || b.splits < 2 || b.slot + (int64_t)(b.splits - 1) * a.kv_heads >= a.grid) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int half = lane >> 5, e = PER * (lane & 31), team = WIDE ? 2 * wave + half : half;
    const float* stats = a.partial + a.grid * ROWS * DT;
    const int64_t r0 = (int64_t)b.row_tile * ROWS, left = (int64_t)b.s.lq * a.group - r0;
    const int rows = left < ROWS ? (int)left : ROWS;
    // (the launch has as many workgroups as the caller takes for the most rows; more rows are taken in turn)
    for (int row = WIDE ? blockIdx.y : blockIdx.y * kWaves + wave; row < rows; row += gridDim.y * (WIDE ? 1 : kWaves)) {
        float o[PER], l = 0.f, m = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < PER; t++) o[t] = 0.f;
        auto join = [&](auto chunk_) {
            constexpr int CHUNK = decltype(chunk_)::value;
            for (int s0 = team; s0 < b.splits; s0 += CHUNK * TEAMS) {
                float ms[CHUNK], ls[CHUNK], x[CHUNK][PER];
#pragma unroll
                for (int k = 0; k < CHUNK; k++) {
                    const int s = s0 + TEAMS * k;
                    const int64_t at = (b.slot + (int64_t)(s < b.splits ? s : s0) * a.kv_heads) * ROWS + row;
                    const float2 st = *reinterpret_cast<const float2*>(stats + at * 2);
                    ms[k] = s < b.splits ? st.x : -__builtin_inff();
                    ls[k] = st.y;
                    const float* p = a.partial + at * DT + e;
                    if constexpr (PER == 2) {
                        const float2 v = *reinterpret_cast<const float2*>(p);
                        x[k][0] = v.x, x[k][1] = v.y;
                    } else {
#pragma unroll
                        for (int t = 0; t < PER; t += 4) {
                            const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p + t);
#pragma unroll
                            for (int y = 0; y < 4; y++) x[k][t + y] = v[y];
                        }
                    }
                }
                float top = m;
#pragma unroll
                for (int k = 0; k < CHUNK; k++) top = fmaxf(top, ms[k]);
                if (top == -__builtin_inff()) continue;       // (splits in which the row sees nothing)
                const float keep = __builtin_amdgcn_exp2f(m - top);
                m = top;
                l *= keep;
#pragma unroll
                for (int t = 0; t < PER; t++) o[t] *= keep;
#pragma unroll
                for (int k = 0; k < CHUNK; k++) {
                    const float w = __builtin_amdgcn_exp2f(ms[k] - top);
                    l += ls[k] * w;
#pragma unroll
                    for (int t = 0; t < PER; t++) o[t] += x[k][t] * w;
                }
            }
        };
        if (!WIDE || b.splits <= 2 * TEAMS) join(std::integral_constant<int, 2>());
        else join(std::integral_constant<int, DT == 256 ? 8 : 16>());
        // the teams' results: in LDS, or the wavefront's two halves
        if constexpr (WIDE) {
#pragma unroll
            for (int t = 0; t < PER; t++) part[team][e + t] = o[t];
            if ((lane & 31) == 0) part[team][DT] = m, part[team][DT + 1] = l;
            __syncthreads();
            if (wave == 0) {
                float top = -__builtin_inff();
#pragma unroll
                for (int w = 0; w < TEAMS; w++) top = fmaxf(top, part[w][DT]);
                l = 0.f;
#pragma unroll
                for (int t = 0; t < PER; t++) o[t] = 0.f;
#pragma unroll
                for (int w = 0; w < TEAMS; w++) {
                    const float f = part[w][DT] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(part[w][DT] - top);
                    l += part[w][DT + 1] * f;
#pragma unroll
                    for (int t = 0; t < PER; t++) o[t] += part[w][e + t] * f;
                }
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
        float odd = l * 0.f;
#pragma unroll
        for (int t = 0; t < PER; t++) odd = __builtin_fmaf(o[t], 0.f, odd);
        if ((!WIDE || wave == 0) && half == 0 && e < a.dim) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int64_t r = r0 + row;
            int32_t head;
            const int32_t token = attention_token(a, r, head);
            head += b.kv_head * a.group;
            bf16_t* out = a.out + (b.s.q0 + token) * a.out_token + (int64_t)head * a.out_head + e;
#pragma unroll
            for (int t = 0; t < PER; t += 2) *reinterpret_cast<uint32_t*>(out + t) = pack_bf16(o[t] * inv, o[t + 1] * inv);
            if (odd != 0.f)
                join_row_again<PER>(stats + (b.slot * ROWS + row) * 2, a.partial + (b.slot * ROWS + row) * DT + e, a.kv_heads * ROWS, DT, b.splits, out);
        }
        if constexpr (WIDE) __syncthreads();       // (part is written again)
    }
}

// tiles: (row tile, head) pairs at most; most_rows: of a tile, as far as is known
int launch_attention_combine(const AttentionArgs& a, int rows, int keys, int dim, int64_t tiles, int64_t most_rows, hipStream_t stream) {
    const unsigned count = (unsigned)(most_rows < rows ? most_rows : rows);
    // few rows have many splits each; many rows few: four rows a wavefront, as finding its place costs a workgroup more than they do
#define SNGGUF_GO(R, K, D)                                                                                              \
    if (rows == R && keys == K && dim == D) {                                                                           \
        constexpr bool kWide = R <= 64;                                                                                 \
        attention_combine_kernel<R, K, D, kWide><<<dim3((unsigned)tiles, kWide ? count : (count + 4 * kWaves - 1) / (4 * kWaves)), kThreads, 0, stream>>>(a); \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
#define SNGGUF_GO_DIM(R, K) SNGGUF_GO(R, K, 64) SNGGUF_GO(R, K, 128) SNGGUF_GO(R, K, 256)
    SNGGUF_GO_DIM(16, 128)
    SNGGUF_GO_DIM(32, 128)
    SNGGUF_GO_DIM(64, 128)
    SNGGUF_GO_DIM(128, 64)
    SNGGUF_GO(256, 64, 64)
    SNGGUF_GO(256, 64, 128)
    SNGGUF_GO(256, 64, 256)
#undef SNGGUF_GO_DIM
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

// dim: of the kernel, 64, 128 or 256; rows: of a tile, 16, 32 or (up to 128 elements) 64
int launch_attention_rows(const AttentionArgs& a, int rows, int dim, bool q8, hipStream_t stream) {
#define SNGGUF_GO(D, F, Q, N)                                                                                           \
    if (dim == D && (a.dim == D) == F && q8 == Q && rows == 16 * N) {                                                   \
        constexpr int kLds = (kWaves * 16 * D + kWaves * 16 * N * 2) * 4;                                               \
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&attention_rows_kernel<D, F, Q, N>), \
                                                           hipFuncAttributeMaxDynamicSharedMemorySize, kLds);           \
        if (attr != hipSuccess) return SNGGUF_E_LAUNCH;                                                                 \
        attention_rows_kernel<D, F, Q, N><<<dim3((unsigned)a.grid), kThreads, kLds, stream>>>(a);                       \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
#define SNGGUF_GO_TYPES(D, N) SNGGUF_GO(D, true, false, N) SNGGUF_GO(D, false, false, N) SNGGUF_GO(D, true, true, N) SNGGUF_GO(D, false, true, N)
    SNGGUF_GO_TYPES(64, 1)
    SNGGUF_GO_TYPES(64, 2)
    SNGGUF_GO_TYPES(64, 4)
    SNGGUF_GO_TYPES(128, 1)
    SNGGUF_GO_TYPES(128, 2)
    SNGGUF_GO_TYPES(128, 4)
    SNGGUF_GO_TYPES(256, 1)
    SNGGUF_GO_TYPES(256, 2)
#undef SNGGUF_GO_TYPES
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

}  // namespace sngguf
