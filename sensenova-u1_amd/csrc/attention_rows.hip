// Attention of few rows over a paged cache: single new tokens, and short runs of them.
//
//     o = sum_j softmax_j(scale q . k_j) v_j  over the keys j of the sequence that the row sees
//
// in one pass over the keys with a running maximum m and sum l (in base 2: p_j = exp2(scale log2(e) q . k_j - m)).  Bound by
// the bytes of the cache, so a workgroup's wavefronts read keys and values straight into registers, in the order in which
// the matrix instructions want them, and never through LDS; each wavefront takes every fourth run of 32 keys with a maximum
// and a sum of its own, and the four are joined at the end.  Sequences are split over workgroups where there are few.
//
// Per run of 32 keys and 16 rows (columns of the 16 x 16 x 32 instructions, lane % 16; lane group g = lane / 16):
//  * scores: K (16 keys x dim) times Q^T.  The order in which dim is summed is free: lane group g takes elements
//    [g DT / 4, (g + 1) DT / 4) of its key's row, which are contiguous.  Matrix row 4 g + i of the first instruction is key
//    8 g + i, of the second key 8 g + 4 + i;
//  * so a lane's eight scores are of keys 8 g .. 8 g + 7, which is how the second product wants them: V^T (16 elements x 32
//    keys) times P^T, where lane group g holds keys 8 g .. 8 g + 7.  A lane reads DT / 16 neighbouring elements of those eight
//    rows, and instruction t takes element t of each.
// An 8-bit cache is widened to fp16 (whole numbers are exact there, the product with the scale is rounded to 11 bits; values are
// within fp16 by the format) and multiplied in fp16, with p scaled by 2^12: p down to 2^-36 of the largest still counts.
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

}  // namespace

// DT: elements of a head, rounded up.  NT: 16-row tiles.
template <int DT, bool Q8, int NT>
__global__ __launch_bounds__(kThreads) void attention_rows_kernel(AttentionArgs a) {
    typedef typename Operand<Q8>::T op_t;
    constexpr int ROWS = 16 * NT;
    constexpr int KP = DT / 4;              // elements of a key that a lane reads
    constexpr int VP = DT / 16;             // elements of a value that a lane reads
    constexpr int KC = KP / 8;              // instructions of a score
    extern __shared__ __attribute__((aligned(16))) float lds[];   // [wave][16][DT] sums, then [wave][ROWS][2]
    float* stats = lds + kWaves * 16 * DT;

    const AttentionBlock b = attention_block<ROWS, kKeys, false>(a, blockIdx.x);
    if (!b.there) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int64_t rows = (int64_t)b.s.lq * a.group;
    const int64_t r0 = (int64_t)b.row_tile * ROWS, r1 = r0 + ROWS < rows ? r0 + ROWS : rows;
    int32_t lo, hi;
    attention_keys(a, b.s, r0, r1, lo, hi);
    const int32_t back = b.s.lk - b.s.lq;

    // ---- queries: operand fragments, and which keys each column sees ---------------------------------------------------
    op_t qf[NT][KC];
    float c[NT];                            // scale_log2 x what the row was scaled by
    int32_t first[NT], last[NT];            // visible keys of the column's row, inclusive
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int64_t r = r0 + 16 * n + col;
        const bool there = r < r1;
        const int64_t rr = there ? r : r0;
        const int32_t token = (int32_t)(rr / a.group), head = b.kv_head * a.group + (int32_t)(rr - (int64_t)token * a.group);
        const bf16_t* q = a.q + (b.s.q0 + token) * a.q_token + (int64_t)head * a.q_head;
        const int32_t place = back + token;
        last[n] = !there ? -1 : a.causal && place < b.s.lk - 1 ? place : b.s.lk - 1;
        first[n] = a.window && place - a.window + 1 > 0 ? (int32_t)(place - a.window + 1) : 0;
        u32x4_t raw[KC];
#pragma unroll
        for (int i = 0; i < KC; i++) {
            const int e = KP * g + 8 * i;
            raw[i] = there && e < a.dim ? *reinterpret_cast<const u32x4_t*>(q + e) : u32x4_t{0u, 0u, 0u, 0u};
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
                    const uint32_t h = x >> 16, l = x & 0xFFFFu;
                    top = top > h ? top : h;
                    top = top > l ? top : l;
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

    f32x4_t acc[NT][VP];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n] = -__builtin_inff();
        l[n] = 0.f;
#pragma unroll
        for (int t = 0; t < VP; t++) acc[n][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    // ---- this split's steps --------------------------------------------------------------------------------------------
    int32_t s0 = lo / kKeys, s1 = (hi + kKeys - 1) / kKeys;
    {
        const int32_t per = (s1 - s0 + b.splits - 1) / b.splits;
        s0 += per * b.split;
        s1 = s0 + per < s1 ? s0 + per : s1;
    }
    const int32_t page_mask = (1 << a.page_shift) - 1;
    // key of matrix row `col` in the two score instructions: 8 (col / 4) + col % 4 (+ 4); values: keys 8 g .. 8 g + 7
    const int k_key = 8 * (col >> 2) + (col & 3), v_key = 8 * g;
    const int v_e = VP * col < a.dim ? VP * col : 0;      // (columns behind dim: any finite-or-not values of the same row, never stored)
    const int64_t run_stride = (int64_t)1 << a.page_shift;
    for (int32_t s = s0; s < s1; s++) {
        const int32_t key0 = s * kKeys + wave * kRun;
        if (key0 >= hi) break;
        const bool edge = key0 + kRun > b.s.lk;
        // -- keys
        int64_t kat[2];
        {
            const int32_t lead = min(key0 + (k_key & ~7), b.s.lk - 1);
            const int64_t page = (attention_page(a, b.seq, lead) * a.kv_heads + b.kv_head) << a.page_shift;
            kat[0] = page + (min(key0 + k_key, b.s.lk - 1) & page_mask);
            kat[1] = page + (min(key0 + k_key + 4, b.s.lk - 1) & page_mask);
        }
        op_t kf[2][KC];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if constexpr (Q8) {
                const int64_t pg = kat[i] >> a.page_shift, row = kat[i] & page_mask;
                const uint16_t* sc = a.k_scales + (pg * (a.dim >> 5) << a.page_shift) + row;
                const uint8_t* p = static_cast<const uint8_t*>(a.k_pages) + kat[i] * a.dim;
#pragma unroll
                for (int x = 0; x < KC / 2; x++) {
                    const int e = KP * g + 16 * x < a.dim ? KP * g + 16 * x : 0;
                    const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p + e);
                    const _Float16 d = __builtin_bit_cast(_Float16, sc[(e >> 5) * run_stride]);
                    const f16x2_t dd = {d, d};
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        u32x4_t f;
#pragma unroll
                        for (int z = 0; z < 2; z++) {
                            const uint32_t flipped = w[2 * y + z] ^ 0x80808080u;
                            f[2 * z] = __builtin_bit_cast(uint32_t, whole_pair<false>(flipped) * dd);
                            f[2 * z + 1] = __builtin_bit_cast(uint32_t, whole_pair<true>(flipped) * dd);
                        }
                        kf[i][2 * x + y] = __builtin_bit_cast(op_t, f);
                    }
                }
            } else {
                const bf16_t* p = static_cast<const bf16_t*>(a.k_pages) + kat[i] * a.dim;
#pragma unroll
                for (int x = 0; x < KC; x++) {
                    const int e = KP * g + 8 * x < a.dim ? KP * g + 8 * x : 0;
                    kf[i][x] = __builtin_bit_cast(op_t, *reinterpret_cast<const u32x4_t*>(p + e));
                }
            }
        }
        // -- values: vf[t] holds element t of keys 8 g .. 8 g + 7
        op_t vf[VP];
        {
            const int32_t lead = min(key0 + v_key, b.s.lk - 1);
            const int64_t page = attention_page(a, b.seq, lead) * a.kv_heads + b.kv_head;
            const int32_t row = lead & page_mask & ~7;
            int32_t at[8];
#pragma unroll
            for (int j = 0; j < 8; j++) at[j] = min(key0 + v_key + j, b.s.lk - 1) & page_mask;
            if constexpr (Q8) {
                u32x4_t sw = *reinterpret_cast<const u32x4_t*>(a.v_scales + ((page * (a.dim >> 5) + (v_e >> 5)) << a.page_shift) + row);
                if (edge) {
                    // scales behind the last key were never written: not even a zero may meet them
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (key0 + v_key + j >= b.s.lk) sw[j >> 1] &= (j & 1) ? 0x0000FFFFu : 0xFFFF0000u;
                }
                const uint8_t* p = static_cast<const uint8_t*>(a.v_pages) + (page << a.page_shift) * a.dim + v_e;
                uint32_t w[8][VP / 4];
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int x = 0; x < VP / 4; x++) w[j][x] = *reinterpret_cast<const uint32_t*>(p + (int64_t)at[j] * a.dim + 4 * x) ^ 0x80808080u;
#pragma unroll
                for (int x = 0; x < VP / 4; x++) {
                    u32x4_t f[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t dw = sw[j];      // (a bit cast of a vector's element itself takes element 0)
                        const f16x2_t d = __builtin_bit_cast(f16x2_t, dw);
                        const uint32_t a0 = w[2 * j][x], a1 = w[2 * j + 1][x];
                        // pairs of elements of each key -> pairs of keys of each element
                        const uint32_t l0 = __builtin_bit_cast(uint32_t, whole_pair<false>(a0)), l1 = __builtin_bit_cast(uint32_t, whole_pair<false>(a1));
                        const uint32_t h0 = __builtin_bit_cast(uint32_t, whole_pair<true>(a0)), h1 = __builtin_bit_cast(uint32_t, whole_pair<true>(a1));
                        f[0][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(l1, l0, 0x05040100u)) * d);
                        f[1][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(l1, l0, 0x07060302u)) * d);
                        f[2][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(h1, h0, 0x05040100u)) * d);
                        f[3][j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(h1, h0, 0x07060302u)) * d);
                    }
#pragma unroll
                    for (int t = 0; t < 4; t++) vf[4 * x + t] = __builtin_bit_cast(op_t, f[t]);
                }
            } else {
                const bf16_t* p = static_cast<const bf16_t*>(a.v_pages) + (page << a.page_shift) * a.dim + v_e;
                uint32_t w[8][VP / 2];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t* pj = reinterpret_cast<const uint32_t*>(p + (int64_t)at[j] * a.dim);
#pragma unroll
                    for (int x = 0; x < VP / 2; x++) w[j][x] = pj[x];
                }
#pragma unroll
                for (int x = 0; x < VP / 2; x++) {
                    u32x4_t f0, f1;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        f0[j] = __builtin_amdgcn_perm(w[2 * j + 1][x], w[2 * j][x], 0x05040100u);
                        f1[j] = __builtin_amdgcn_perm(w[2 * j + 1][x], w[2 * j][x], 0x07060302u);
                    }
                    vf[2 * x] = __builtin_bit_cast(op_t, f0);
                    vf[2 * x + 1] = __builtin_bit_cast(op_t, f1);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            f32x4_t sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int x = 0; x < KC; x++) sc[i] = mfma(kf[i][x], qf[n][x], sc[i]);
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int32_t key = key0 + 8 * g + j;
                p[j] = key >= first[n] && key <= last[n] ? sc[j >> 2][j & 3] : -__builtin_inff();
            }
            float top = p[0];
#pragma unroll
            for (int j = 1; j < 8; j++) top = fmaxf(top, p[j]);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            top = fmaxf(top * c[n], m[n]);
            const float base = top == -__builtin_inff() ? 0.f : top;
            const float keep = __builtin_amdgcn_exp2f(m[n] - base);
            m[n] = top;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[j], c[n], -base));
                sum += p[j];
            }
            l[n] = l[n] * keep + sum;
            u32x4_t pw;
#pragma unroll
            for (int j = 0; j < 4; j++) pw[j] = Q8 ? pack_f16(p[2 * j] * 4096.f, p[2 * j + 1] * 4096.f) : pack_bf16(p[2 * j], p[2 * j + 1]);
            const op_t pf = __builtin_bit_cast(op_t, pw);
#pragma unroll
            for (int t = 0; t < VP; t++) {
                acc[n][t] *= keep;
                acc[n][t] = mfma(vf[t], pf, acc[n][t]);
            }
        }
    }

    // ---- the four wavefronts' results --------------------------------------------------------------------------------
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
        if constexpr (Q8) mine *= 1.f / 4096.f;
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
        if (r < r1 && e < a.dim) {
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
                const int32_t token = (int32_t)(r / a.group), head = b.kv_head * a.group + (int32_t)(r - (int64_t)token * a.group);
                bf16_t* out = a.out + (b.s.q0 + token) * a.out_token + (int64_t)head * a.out_head + e;
#pragma unroll
                for (int t = 0; t < VP; t += 4)
                    *reinterpret_cast<u32x2_t*>(out + t) = u32x2_t{pack_bf16(o[t] * inv, o[t + 1] * inv), pack_bf16(o[t + 2] * inv, o[t + 3] * inv)};
            }
        }
        __syncthreads();
    }
}

// Joins the splits of a row: one wavefront a row, lanes along its elements.
template <int ROWS, int KEYS, int DT>
__global__ __launch_bounds__(kThreads) void attention_combine_kernel(AttentionArgs a) {
    const AttentionBlock b = attention_block<ROWS, KEYS, true>(a, blockIdx.x);
    if (!b.there || b.splits < 2) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.y * kWaves + wave;
    const int64_t r = (int64_t)b.row_tile * ROWS + row;
    if (r >= (int64_t)b.s.lq * a.group) return;
    const float* stats = a.partial + a.grid * ROWS * DT;
    float top = -__builtin_inff();
    for (int s = 0; s < b.splits; s++) top = fmaxf(top, stats[((b.slot + (int64_t)s * a.kv_heads) * ROWS + row) * 2]);
    float o[DT / 64];
#pragma unroll
    for (int t = 0; t < DT / 64; t++) o[t] = 0.f;
    float l = 0.f;
    for (int s = 0; s < b.splits; s++) {
        const int64_t at = (b.slot + (int64_t)s * a.kv_heads) * ROWS + row;
        const float ms = stats[at * 2];
        if (ms == -__builtin_inff()) continue;
        const float w = __builtin_amdgcn_exp2f(ms - top);
        l += stats[at * 2 + 1] * w;
#pragma unroll
        for (int t = 0; t < DT / 64; t++) o[t] += a.partial[at * DT + 64 * t + lane] * w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int32_t token = (int32_t)(r / a.group), head = b.kv_head * a.group + (int32_t)(r - (int64_t)token * a.group);
    bf16_t* out = a.out + (b.s.q0 + token) * a.out_token + (int64_t)head * a.out_head;
#pragma unroll
    for (int t = 0; t < DT / 64; t++)
        if (64 * t + lane < a.dim) out[64 * t + lane] = f32_to_bf16(o[t] * inv);
}

int64_t attention_rows_keys() { return kKeys; }

// tiles: (row tile, head) pairs at most
int launch_attention_combine(const AttentionArgs& a, int rows, int keys, int dim, int64_t tiles, hipStream_t stream) {
#define SNGGUF_GO(R, K, D)                                                                                              \
    if (rows == R && keys == K && dim == D) {                                                                           \
        attention_combine_kernel<R, K, D><<<dim3((unsigned)tiles, R / kWaves), kThreads, 0, stream>>>(a);               \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
#define SNGGUF_GO_DIM(R, K) SNGGUF_GO(R, K, 64) SNGGUF_GO(R, K, 128) SNGGUF_GO(R, K, 256)
    SNGGUF_GO_DIM(16, 128)
    SNGGUF_GO_DIM(32, 128)
    SNGGUF_GO_DIM(64, 128)
    SNGGUF_GO_DIM(128, 64)
    SNGGUF_GO(256, 64, 64)
    SNGGUF_GO(256, 64, 128)
#undef SNGGUF_GO_DIM
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

int launch_attention_rows(const AttentionArgs& a, int rows, int dim, bool q8, hipStream_t stream) {
#define SNGGUF_GO(D, Q, N)                                                                                              \
    if (dim == D && q8 == Q && rows == 16 * N) {                                                                        \
        constexpr int kLds = (kWaves * 16 * D + kWaves * 16 * N * 2) * 4;                                               \
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&attention_rows_kernel<D, Q, N>), \
                                                           hipFuncAttributeMaxDynamicSharedMemorySize, kLds);           \
        if (attr != hipSuccess) return SNGGUF_E_LAUNCH;                                                                 \
        attention_rows_kernel<D, Q, N><<<dim3((unsigned)a.grid), kThreads, kLds, stream>>>(a);                          \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
#define SNGGUF_GO_DIM(D) SNGGUF_GO(D, false, 1) SNGGUF_GO(D, false, 2) SNGGUF_GO(D, false, 4) SNGGUF_GO(D, true, 1) SNGGUF_GO(D, true, 2) SNGGUF_GO(D, true, 4)
    SNGGUF_GO_DIM(64)
    SNGGUF_GO_DIM(128)
    SNGGUF_GO_DIM(256)
#undef SNGGUF_GO_DIM
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

}  // namespace sngguf
