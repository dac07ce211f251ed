// Attention of many rows: whole prompts over their own packed keys and values, and chunks of new tokens over a paged cache.
//
// A workgroup takes 128 rows of one sequence and key / value head (row = token x query heads of the group, so the heads that
// share keys and values share their tiles), four wavefronts of 32 rows, and walks over tiles of 64 keys in two LDS stages.
// One pass with a running maximum m and sum l, in base 2.  Bound by the matrix instructions (32 x 32 x 16):
//  * S^T = K Q^T: a lane holds sixteen of a row's 32 scores (row = lane % 32), so maxima and sums are taken in registers, and
//    the two halves of a row meet in one exchange.  Register i of lane half h is key 8 (i / 4) + 4 h + i % 4;
//  * O^T += V^T P^T wants eight keys of a row in each lane, in any order that V^T shares: those registers are taken as they
//    are, and V, which lies row by row in LDS, is read with the transposing read, four keys of one element at a time.
// In LDS a row's 16-byte pieces are permuted so that the eight or sixteen rows that one read touches lie in different banks;
// copies go from global memory to LDS directly, and permute on the global side.
// An 8-bit cache is widened on its way to LDS: fp16 there (see attention_rows.hip), and p is scaled by 2^12.
#include "attention.hpp"

namespace sngguf {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;
constexpr int kKeys = 64;

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

template <bool Q8> struct Operand { typedef bf16x8_t T; };
template <> struct Operand<true> { typedef f16x8_t T; };

__device__ __forceinline__ f32x16_t mfma(bf16x8_t a, bf16x8_t b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16_t mfma(f16x8_t a, f16x8_t b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)a, (_Float16)b});
}
template <bool HIGH>
__device__ __forceinline__ f16x2_t whole_pair(uint32_t flipped) {
    const uint32_t w = __builtin_amdgcn_perm(0x64646464u, flipped, HIGH ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(f16x2_t, w) + f16x2_t{(_Float16)-1152.f, (_Float16)-1152.f};
}

// The larger (the sum) of a value and that of the lane 32 away.
__device__ __forceinline__ float other_half(float x) {
    const u32x2_t r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t other = (threadIdx.x & 32) ? r[0] : r[1];
    return __builtin_bit_cast(float, other);
}

// A pointer that is the same in all lanes, in scalar registers.
__device__ __forceinline__ const uint8_t* uniform_ptr(const void* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const uint8_t*>(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
// 16 bytes a lane to 1 KB of LDS; the loop waits for these requests itself (s_waitcnt vmcnt(0) in front of its barrier)
__device__ __forceinline__ void copy_request(uint32_t lds, uint32_t off, const void* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

// What piece c of row r is exchanged with: rows that one read touches together get different pieces.
template <int DT>
__device__ __forceinline__ int swizzle(int r) {
    // 128-byte rows lie two to a line of the 64 banks, so that rows of one parity have to differ
    return DT == 64 ? ((((r >> 1) & 1) << 2) | ((r >> 2) & 3)) : (((r & 3) << 2) | ((r >> 2) & 3));
}

}  // namespace

enum { kPacked = 0, kPaged = 1, kPagedQ8 = 2 };

template <int DT, int SOURCE>
__global__ __launch_bounds__(kThreads) void attention_tiles_kernel(AttentionArgs a) {
    constexpr bool Q8 = SOURCE == kPagedQ8;
    typedef typename Operand<Q8>::T op_t;
    constexpr int PIECES = DT / 8;                     // of a row
    constexpr int TILE = kKeys * DT * 2;               // bytes
    constexpr int KS = DT / 16, DTILES = DT / 32;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // [stage][keys, values]

    const AttentionBlock b = attention_block<kRows, kKeys, false>(a, blockIdx.x);
    if (!b.there) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int64_t rows = (int64_t)b.s.lq * a.group;
    const int64_t r0 = (int64_t)b.row_tile * kRows, r1 = r0 + kRows < rows ? r0 + kRows : rows;
    int32_t lo, hi;
    attention_keys(a, b.s, r0, r1, lo, hi);
    const int32_t back = b.s.lk - b.s.lq;

    // ---- this lane's row: its query as operand fragments, and the keys that it sees ------------------------------------
    const int64_t r = r0 + 32 * wave + col;
    const bool there = r < r1;
    const int64_t rr = there ? r : r1 - 1;
    const int32_t token = (int32_t)(rr / a.group), head = b.kv_head * a.group + (int32_t)(rr - (int64_t)token * a.group);
    const int32_t place = back + token;
    const int32_t last = a.causal && place < b.s.lk - 1 ? place : b.s.lk - 1;
    const int32_t first = a.window && place - a.window + 1 > 0 ? (int32_t)(place - a.window + 1) : 0;
    op_t qf[KS];
    float c = a.scale_log2;
    {
        const bf16_t* q = a.q + (b.s.q0 + token) * a.q_token + (int64_t)head * a.q_head;
        u32x4_t raw[KS];
#pragma unroll
        for (int i = 0; i < KS; i++) {
            const int e = 16 * i + 8 * h;
            raw[i] = e < a.dim ? *reinterpret_cast<const u32x4_t*>(q + e) : u32x4_t{0u, 0u, 0u, 0u};
        }
        if constexpr (Q8) {
            // bf16 -> fp16: scaled by a power of two that brings the row's largest element into [1, 2)
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < KS; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t x = raw[i][j] & 0x7F807F80u;
                    top = max(top, max(x >> 16, x & 0xFFFFu));
                }
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            const int ex = top == 0 ? 0 : (int)(top >> 7) - 127;
#pragma unroll
            for (int i = 0; i < KS; i++) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = pack_f16(__builtin_ldexpf(bf16lo_to_f32(raw[i][j]), -ex), __builtin_ldexpf(bf16hi_to_f32(raw[i][j]), -ex));
                qf[i] = __builtin_bit_cast(op_t, w);
            }
            c = fmaxf(__builtin_ldexpf(c, ex), 1.2e-38f);
        } else {
#pragma unroll
            for (int i = 0; i < KS; i++) qf[i] = __builtin_bit_cast(op_t, raw[i]);
        }
    }

    // ---- this split's tiles -------------------------------------------------------------------------------------------
    int32_t s0 = lo / kKeys, s1 = (hi + kKeys - 1) / kKeys;
    {
        const int32_t per = (s1 - s0 + b.splits - 1) / b.splits;
        s0 += per * b.split;
        s1 = s0 + per < s1 ? s0 + per : s1;
    }
    // rows whose visible keys are the fewest: tiles inside these bounds need no mask
    const int64_t tail = r1 - 1;
    const int32_t place0 = back + (int32_t)(r0 / a.group), place1 = back + (int32_t)(tail / a.group);
    const int32_t all_last = a.causal && place0 < b.s.lk - 1 ? place0 : b.s.lk - 1;
    const int32_t all_first = a.window && place1 - a.window + 1 > 0 ? (int32_t)(place1 - a.window + 1) : 0;

    f32x16_t acc[DTILES];
#pragma unroll
    for (int t = 0; t < DTILES; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[t][i] = 0.f;
    float m = -__builtin_inff(), l = 0.f;

    // ---- tiles into LDS ------------------------------------------------------------------------------------------------
    // Sixteen rows a wavefront.  Rows behind the last key are the last key's: masked, but finite wherever the keys are.
    const int32_t page_mask = (1 << a.page_shift) - 1;
    constexpr int RQ = 1024 / (DT * 2);                // rows of one request (1 KB)
    constexpr int REQ = 16 / RQ;
    const int crow = lane / PIECES, cpiece = lane % PIECES;
    constexpr int QP = DT / 16;                        // 8-bit: 16-byte pieces of a row
    constexpr int QN = 16 * QP / 64;                   // ... a lane has of each tile
    u32x4_t kq[Q8 ? QN : 1], vq[Q8 ? QN : 1];
    uint16_t ksc[Q8 ? QN : 1], vsc[Q8 ? QN : 1];
    auto request = [&](int32_t tile, int stage) {
        const int32_t base = tile * kKeys + 16 * wave;
        const int32_t most = b.s.lk - 1;
        if constexpr (SOURCE == kPacked) {
            const int32_t lead = base < most ? base : most;
            const uint8_t* kb = uniform_ptr(a.k + (b.s.k0 + lead) * a.k_token + (int64_t)b.kv_head * a.k_head);
            const uint8_t* vb = uniform_ptr(a.v + (b.s.k0 + lead) * a.v_token + (int64_t)b.kv_head * a.v_head);
#pragma unroll
            for (int i = 0; i < REQ; i++) {
                const int row = RQ * i + crow;
                int piece = cpiece ^ swizzle<DT>(row);
                piece = 8 * piece < a.dim ? piece : 0;
                const int32_t at = base + row < most ? base + row - lead : most - lead;
                copy_request(lds_offset(lds + (2 * stage) * TILE + (16 * wave + RQ * i) * DT * 2), (uint32_t)(2 * (at * a.k_token + 8 * piece)), kb);
                copy_request(lds_offset(lds + (2 * stage + 1) * TILE + (16 * wave + RQ * i) * DT * 2), (uint32_t)(2 * (at * a.v_token + 8 * piece)), vb);
            }
        } else {
            // (sixteen rows lie in one page)
            const int32_t lead = base < most ? base : most;
            const int64_t page = __builtin_amdgcn_readfirstlane((int)attention_page(a, b.seq, lead));
            const int64_t at_page = page * a.kv_heads + b.kv_head;
            if constexpr (SOURCE == kPaged) {
                const uint8_t* kb = uniform_ptr(static_cast<const bf16_t*>(a.k_pages) + (at_page << a.page_shift) * a.dim);
                const uint8_t* vb = uniform_ptr(static_cast<const bf16_t*>(a.v_pages) + (at_page << a.page_shift) * a.dim);
#pragma unroll
                for (int i = 0; i < REQ; i++) {
                    const int row = RQ * i + crow;
                    int piece = cpiece ^ swizzle<DT>(row);
                    piece = 8 * piece < a.dim ? piece : 0;
                    const int32_t at = (base + row < most ? base + row : most) & page_mask;
                    const uint32_t off = (uint32_t)(2 * (at * a.dim + 8 * piece));
                    copy_request(lds_offset(lds + (2 * stage) * TILE + (16 * wave + RQ * i) * DT * 2), off, kb);
                    copy_request(lds_offset(lds + (2 * stage + 1) * TILE + (16 * wave + RQ * i) * DT * 2), off, vb);
                }
            } else {
                const uint8_t* kb = static_cast<const uint8_t*>(a.k_pages) + (at_page << a.page_shift) * a.dim;
                const uint8_t* vb = static_cast<const uint8_t*>(a.v_pages) + (at_page << a.page_shift) * a.dim;
                const uint16_t* ks = a.k_scales + (at_page * (a.dim >> 5) << a.page_shift);
                const uint16_t* vs = a.v_scales + (at_page * (a.dim >> 5) << a.page_shift);
#pragma unroll
                for (int i = 0; i < QN; i++) {
                    const int p = lane + 64 * i, row = p / QP;
                    int piece = p % QP;
                    piece = 16 * piece < a.dim ? piece : 0;
                    const int32_t at = (base + row < most ? base + row : most) & page_mask;
                    kq[i] = *reinterpret_cast<const u32x4_t*>(kb + at * a.dim + 16 * piece);
                    vq[i] = *reinterpret_cast<const u32x4_t*>(vb + at * a.dim + 16 * piece);
                    ksc[i] = ks[((piece >> 1) << a.page_shift) + at];
                    vsc[i] = vs[((piece >> 1) << a.page_shift) + at];
                }
            }
        }
    };
    // 8-bit tiles: widened from the registers that request() filled
    auto widen = [&](int stage) {
        if constexpr (Q8) {
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int i = 0; i < QN; i++) {
                    const int p = lane + 64 * i, row = p / QP, piece = p % QP;
                    const u32x4_t w = half ? vq[i] : kq[i];
                    const _Float16 d1 = __builtin_bit_cast(_Float16, half ? vsc[i] : ksc[i]);
                    const f16x2_t d = {d1, d1};
                    uint8_t* to = lds + (2 * stage + half) * TILE + (16 * wave + row) * DT * 2;
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        u32x4_t f;
#pragma unroll
                        for (int z = 0; z < 2; z++) {
                            const uint32_t flipped = w[2 * y + z] ^ 0x80808080u;
                            f[2 * z] = __builtin_bit_cast(uint32_t, whole_pair<false>(flipped) * d);
                            f[2 * z + 1] = __builtin_bit_cast(uint32_t, whole_pair<true>(flipped) * d);
                        }
                        *reinterpret_cast<u32x4_t*>(to + 16 * ((2 * piece + y) ^ swizzle<DT>(row))) = f;
                    }
                }
        }
    };

    // fragment addresses within a tile: keys: row col, piece 2 ks + h; values: key 4 h + (lane % 16) / 4, elements 16 ((lane %
    // 32) / 16) + 4 (lane % 4) ..., the rows of one transposing read being four keys
    const int vkey = 4 * h + ((lane & 15) >> 2), velem = 16 * ((lane & 31) >> 4) + 4 * (lane & 3);

    if (s0 < s1) {
        request(s0, 0);
        widen(0);
    }
    for (int32_t s = s0; s < s1; s++) {
        const int stage = (s - s0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (s + 1 < s1) request(s + 1, stage ^ 1);
        const uint8_t* kt = lds + (2 * stage) * TILE;
        const uint8_t* vt = kt + TILE;
        f32x16_t sc[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) sc[t][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int row = 32 * t + col;
                const op_t kf = *reinterpret_cast<const op_t*>(kt + row * DT * 2 + 16 * ((2 * ks + h) ^ swizzle<DT>(row)));
                sc[t] = mfma(kf, qf[ks], sc[t]);
            }
        }
        const int32_t key0 = s * kKeys;
        if (key0 + kKeys - 1 > all_last || key0 < all_first) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int32_t key = key0 + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
                    if (key < first || key > last) sc[t][i] = -__builtin_inff();
                }
        }
        float top = sc[0][0];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, sc[t][i]);
        top = fmaxf(top, other_half(top));
        top = fmaxf(top * c, m);
        const float base = top == -__builtin_inff() ? 0.f : top;
        const float keep = __builtin_amdgcn_exp2f(m - base);
        m = top;
        float sum = 0.f;
        op_t pf[4];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                u32x4_t w;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * half + 2 * j], c, -base));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * half + 2 * j + 1], c, -base));
                    sum += p0 + p1;
                    w[j] = Q8 ? pack_f16(p0 * 4096.f, p1 * 4096.f) : pack_bf16(p0, p1);
                }
                pf[2 * t + half] = __builtin_bit_cast(op_t, w);
            }
        l = l * keep + sum;
#pragma unroll
        for (int t = 0; t < DTILES; t++) {
            acc[t] *= keep;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                u32x2_t half[2];
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int row = 16 * x + 8 * y + vkey, e = 32 * t + velem;
                    half[y] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(
                        vt + row * DT * 2 + 16 * ((e >> 3) ^ swizzle<DT>(row)) + 2 * (e & 7))));
                }
                const u32x4_t w = {half[0][0], half[0][1], half[1][0], half[1][1]};
                acc[t] = mfma(__builtin_bit_cast(op_t, w), pf[x], acc[t]);
            }
        }
        if (s + 1 < s1) widen(stage ^ 1);
    }
    l += other_half(l);
    if (!there) return;
    // acc[t][i]: row `col`, element 32 t + 8 (i / 4) + 4 h + i % 4
    const float unit = Q8 ? 1.f / 4096.f : 1.f;
    if (b.splits > 1) {
        const int64_t at = b.slot * kRows + 32 * wave + col;
#pragma unroll
        for (int t = 0; t < DTILES; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f32x4_t*>(a.partial + at * DT + 32 * t + 2 * i + 4 * h) =
                    f32x4_t{acc[t][i] * unit, acc[t][i + 1] * unit, acc[t][i + 2] * unit, acc[t][i + 3] * unit};
        if (h == 0) {
            float* st = a.partial + a.grid * kRows * DT + at * 2;
            st[0] = m;
            st[1] = l;
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : unit / l;
    bf16_t* out = a.out + (b.s.q0 + token) * a.out_token + (int64_t)head * a.out_head;
#pragma unroll
    for (int t = 0; t < DTILES; t++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int e = 32 * t + 2 * i + 4 * h;
            if (e < a.dim)
                *reinterpret_cast<u32x2_t*>(out + e) = u32x2_t{pack_bf16(acc[t][i] * inv, acc[t][i + 1] * inv), pack_bf16(acc[t][i + 2] * inv, acc[t][i + 3] * inv)};
        }
}

int launch_attention_tiles(const AttentionArgs& a, int dim, int source, hipStream_t stream) {
#define SNGGUF_GO(D, S)                                                                                                 \
    if (dim == D && source == S) {                                                                                      \
        constexpr int kLds = 4 * kKeys * D * 2;                                                                         \
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&attention_tiles_kernel<D, S>), \
                                                           hipFuncAttributeMaxDynamicSharedMemorySize, kLds);           \
        if (attr != hipSuccess) return SNGGUF_E_LAUNCH;                                                                 \
        attention_tiles_kernel<D, S><<<dim3((unsigned)a.grid), kThreads, kLds, stream>>>(a);                            \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
#define SNGGUF_GO_DIM(D) SNGGUF_GO(D, kPacked) SNGGUF_GO(D, kPaged) SNGGUF_GO(D, kPagedQ8)
    SNGGUF_GO_DIM(64)
    SNGGUF_GO_DIM(128)
    SNGGUF_GO_DIM(256)
#undef SNGGUF_GO_DIM
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

}  // namespace sngguf
