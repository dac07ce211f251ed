// Attention of many rows: whole prompts over their own packed keys and values, and chunks of new tokens over a paged cache.
//
// A workgroup takes 128 or 256 rows of one sequence and key / value head (row = token x query heads of the group, so the heads
// that share keys and values share their tiles), 32 for each wavefront, and walks over tiles of 64 keys in a ring of LDS
// stages.  One pass with a running maximum m and sum l, in base 2.  Bound by the matrix instructions (32 x 32 x 16):
//  * S^T = K Q^T: a lane holds sixteen of a row's 32 scores (row = lane % 32).  Register i of lane half h is key 8 (i / 4) +
//    4 h + i % 4;
//  * O^T += V^T P^T wants eight keys of a row in each lane, in any order that V^T shares: those registers are taken as they
//    are, and V, which lies row by row in LDS, is read with the transposing read, four keys of one element at a time.
// In LDS a tile is blocks of 8 rows x 128 bytes, the order that one copy request (1 KB, global memory to LDS directly) makes of
// whole cache lines: piece by piece (16 bytes), and within a piece row by row, so that a read of one piece of many rows is
// contiguous and every address of a tile is a lane's constant and an immediate offset.  Pieces 2, 3, 6, 7 have the halves of
// their eight rows exchanged: the transposing read takes four pieces of four rows, which then fill all banks; blocks of
// neighbouring rows lie half a turn of the banks apart for the same reason.
//
// A step takes 32 keys, and three of them at once: the product with V of the step before, the weights of its own scores, and the
// scores of the step after depend on nothing of each other, so the vector instructions of the weights are dealt over the
// matrix instructions.  What would put the maximum in front of the weights is left out: they are formed with the maximum known
// so far, whatever the scores, and only if a row's 32 weights sum to more than a limit far within range (or to nothing that
// is a number) are maximum, sums and weights set right, behind the step.
// An 8-bit cache is widened on its way to LDS: fp16 there, and p is scaled by 2^12.
// What is rounded is what attention_rows.hip says, for its reasons.  Rounded bf16 weights are summed, as one instruction sums a packed pair;
// fp16 ones, rounded to 2^-11, before.  A prompt of 16384 is off by 0.0020 of its norm from the definition (fp32 weights: 0.0016), a chunk over an
// 8-bit cache by 0.0017 (0.0016).
//
// Measured, 32 query and 8 key / value heads of 128: a prompt of 16384 tokens 1.85 .. 1.94 ms, 1.13 .. 1.19 PFLOP/s (matrix cores busy 59 % of
// the cycles at 1.85 GHz; a large library product reaches 1.40 PFLOP/s); 1024 new tokens over 30000 in 8 bits 0.55 ms, 0.9 PFLOP/s.  A
// workgroup costs 8 us beside its tiles, 1.4 to 1.8 us each.  Level or slower: 64 rows a wavefront (half the LDS reads), eight
// fragments in the ring, a barrier that drains no reads, the two products in turn, 128 rows a workgroup (2.17 ms).
#include <type_traits>
#include <utility>

#include "attention.hpp"

namespace sngguf {

namespace {

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

// the same from an address of each lane's own
__device__ __forceinline__ void copy_request(uint32_t lds, const void* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}

// f(0), f(1), ... f(N - 1), each number a constant (an unrolled loop of this size is given up by the compiler)
template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>()), ...);
}

// From a row to the one `step` behind it: token and head of the group, without a division for each
struct RowWalk {
    uint32_t group, heads;
    int64_t hop, wrap;
    __device__ __forceinline__ RowWalk(uint32_t group, uint32_t step, int64_t token, int64_t head)
        : group(group), heads(step % group), hop((int64_t)(step / group) * token + (int64_t)(step % group) * head), wrap(token - (int64_t)group * head) {}
    template <typename P> __device__ __forceinline__ void next(P*& at, uint32_t& head) const {
        at += hop;
        head += heads;
        if (head >= group) at += wrap, head -= group;
    }
};

// Place of (row % 8, piece % 8) in its block, in pieces.
__device__ __forceinline__ int block_place(int row, int piece) { return 8 * (piece & 7) + ((row & 7) ^ (4 * ((piece >> 1) & 1))); }

template <int DT> struct Tile {
    static constexpr int kBlocks = (DT + 63) / 64;             // of eight rows
    static constexpr int kRowBlock = kBlocks * 1024 + 128;     // bytes from eight rows to the next
    static constexpr int kBytes = kKeys / 8 * kRowBlock;
};

}  // namespace

// W: wavefronts, of 32 rows each.  NS: LDS stages; stage i holds the keys of tile i and the values of tile i - 1.  PLANNED: a kernel in
// front of this one dealt the work.
template <int DT, int SOURCE, int W, int NS, bool PLANNED>
__global__ __launch_bounds__(64 * W, DT <= 128 || W == 8 ? 2 : 1) void attention_tiles_kernel(AttentionArgs a) {
    constexpr bool Q8 = SOURCE == kPagedQ8;
    typedef typename Operand<Q8>::T op_t;
    constexpr int ROWS = 32 * W;
    constexpr int TILE = Tile<DT>::kBytes, RB = Tile<DT>::kRowBlock, PB = Tile<DT>::kBlocks;
    constexpr int KS = DT / 16, DTILES = DT / 32;
    constexpr int DP = DT <= 64 ? 64 : DT <= 128 ? 128 : 256;   // elements of a row of a partial result
    constexpr int VF = 2 * DTILES, NF = VF + KS;       // operand fragments of a step: of values, in all
    constexpr int NP = 8;                              // pairs of weights of a step that a lane forms
    constexpr float kLimit = Q8 ? 32768.f : 1e9f;      // (fp16 weights are scaled by 2^12)
    constexpr float kUp = Q8 ? 12.f : 0.f;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // [stage][keys, values]

    AttentionBlock b;
    if constexpr (PLANNED) b = attention_planned_block<ROWS>(a, blockIdx.x);
    else b = attention_block<ROWS, kKeys, false>(a, blockIdx.x);
    if (!b.there) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int64_t rows = (int64_t)b.s.lq * a.group;
    const int64_t r0 = (int64_t)b.row_tile * ROWS, r1 = r0 + ROWS < rows ? r0 + ROWS : rows;
    int32_t lo, hi;
    attention_keys(a, b, r0, r1, lo, hi);
    const int32_t back = b.s.lk - b.s.lq;

    // ---- this split's tiles -------------------------------------------------------------------------------------------
    int32_t s0 = lo / kKeys, s1 = (hi + kKeys - 1) / kKeys;
    {
        const int32_t per = (s1 - s0 + b.splits - 1) / b.splits;
        s0 += per * b.split;
        s1 = s0 + per < s1 ? s0 + per : s1;
    }
    const int32_t count = s1 - s0;
    // rows whose visible keys are the fewest: tiles inside these bounds need no mask
    const int32_t place0 = back + (int32_t)((uint32_t)r0 / (uint32_t)a.group), place1 = back + (int32_t)((uint32_t)(r1 - 1) / (uint32_t)a.group);
    const int32_t all_last = b.causal && place0 < b.s.lk - 1 ? place0 : b.s.lk - 1;
    const int32_t all_first = a.window && place1 - a.window + 1 > 0 ? (int32_t)(place1 - a.window + 1) : 0;

    f32x16_t acc[DTILES];
#pragma unroll
    for (int t = 0; t < DTILES; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[t][i] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    float nb = __builtin_inff();     // what is added to a scaled score, kUp - m; nothing known yet: whatever is formed with it is set right

    // ---- tiles into LDS ------------------------------------------------------------------------------------------------
    // Rows behind the last key are the last key's: masked, but finite wherever the keys are.
    const int32_t page_mask = (1 << a.page_shift) - 1;
    constexpr int LOAD = kKeys / W;                    // rows of a tile that a wavefront brings, 8 or 16
    constexpr int REQ = LOAD / 8 * PB;                 // requests for them: blocks
    constexpr int QP = DT / 16;                        // 8-bit: 16-byte pieces of a row
    constexpr int QN = (LOAD * QP + 63) / 64;          // ... a lane has of each tile
    static_assert(LOAD % 8 == 0, "whole requests");
    u32x4_t held[2][Q8 ? QN : 1];
    uint16_t held_scale[2][Q8 ? QN : 1];
    // this lane's part of a request: row and piece of a block
    const int crow = (lane & 7) ^ (4 * ((lane >> 4) & 1)), cpiece = lane >> 3;
    const int64_t k_stride = SOURCE == kPacked ? a.k_token : a.dim, v_stride = SOURCE == kPacked ? a.v_token : a.dim;
    // byte offsets of this lane's pieces behind the first of the wavefront's rows, and the last row known to be there
    uint32_t coff[2][REQ];
    int32_t rows_there[2] = {-1, -1};
    auto set_offsets = [&](int half, int32_t spare) {
        spare = spare < LOAD - 1 ? spare : LOAD - 1;
        if (spare == rows_there[half]) return;
        rows_there[half] = spare;
#pragma unroll
        for (int j = 0; j < REQ; j++) {
            const int i = j / PB, p = j % PB, at = 8 * i + crow, row = at < spare ? at : spare;
            // (pieces behind dim: the first, whose elements meet queries of zero, or are never stored)
            coff[half][j] = (uint32_t)(2 * row * (int32_t)(half ? v_stride : k_stride)) + (64 * p + 8 * cpiece < a.dim ? 128 * p + 16 * cpiece : 0);
        }
    };
    const uint8_t* k_base = reinterpret_cast<const uint8_t*>(SOURCE == kPacked ? a.k + b.s.k0 * a.k_token + (int64_t)b.kv_head * a.k_head : nullptr);
    const uint8_t* v_base = reinterpret_cast<const uint8_t*>(SOURCE == kPacked ? a.v + b.s.k0 * a.v_token + (int64_t)b.kv_head * a.v_head : nullptr);
    const int32_t most = b.s.lk - 1;
    const int32_t* table = SOURCE == kPacked ? nullptr : a.table + (int64_t)b.seq * a.table_stride;
    // page of the wavefront's rows of a tile (they lie in one)
    auto page_of = [&](int32_t tile) -> int32_t {
        if constexpr (SOURCE == kPacked) return 0;
        const int32_t base = tile * kKeys + LOAD * wave, lead = base < most ? base : most;
        const int32_t p = *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(table + __builtin_amdgcn_readfirstlane(lead >> a.page_shift));
        return p < 0 ? 0 : p >= a.pages ? a.pages - 1 : p;
    };
    // where the wavefront's rows of a tile start, for the requests of half 0 (keys) or 1 (values)
    const uint8_t* from[2] = {nullptr, nullptr};
    auto aim = [&](int half, int32_t tile, int32_t page) {
        const int32_t base = tile * kKeys + LOAD * wave, lead = base < most ? base : most;
        const int32_t spare = most - lead;             // rows behind the first that there are
        if constexpr (SOURCE == kPacked) {
            from[half] = uniform_ptr((half ? v_base : k_base) + 2 * (int64_t)lead * (half ? v_stride : k_stride));
            set_offsets(half, spare);
        } else {
            const int64_t at_page = (int64_t)page * a.kv_heads + b.kv_head;
            const int64_t at = (at_page << a.page_shift) + (lead & page_mask);
            from[half] = uniform_ptr(static_cast<const uint8_t*>(half ? a.v_pages : a.k_pages) + at * a.dim * (Q8 ? 1 : 2));
            if constexpr (!Q8) {
                set_offsets(half, spare);
            } else {
                const uint16_t* scales = (half ? a.v_scales : a.k_scales) + (at_page * (a.dim >> 5) << a.page_shift) + (lead & page_mask);
#pragma unroll
                for (int i = 0; i < QN; i++) {
                    // neighbouring lanes have neighbouring rows, which lie in different banks when they are written to LDS (piece by
                    // piece they would all lie in the same ones: a chunk of 1024 over 30000 took 568 us instead of 540)
                    const int p = lane + 64 * i, row = p % LOAD < spare ? p % LOAD : spare;
                    int piece = p / LOAD;
                    piece = 16 * piece < a.dim ? piece : 0;
                    held[half][i] = *reinterpret_cast<const u32x4_t*>(from[half] + row * a.dim + 16 * piece);
                    held_scale[half][i] = scales[((piece >> 1) << a.page_shift) + row];
                }
            }
        }
    };
    const uint32_t lds0 = lds_offset(lds);
    // request j of REQ into the half of the stage at `stage`
    auto request = [&](int half, uint32_t stage, int j) {
        if constexpr (!Q8) copy_request(stage + half * TILE + (LOAD / 8 * wave + j / PB) * RB + (j % PB) * 1024, coff[half][j], from[half]);
    };
    // 8-bit tiles: widened from the registers that the request filled
    auto widen = [&](int half, uint32_t stage, int i) {
        if constexpr (Q8) {
            const int p = lane + 64 * i, row = LOAD * wave + p % LOAD, piece = p / LOAD;
            if (LOAD * QP % 64 != 0 && piece >= QP) return;
            const u32x4_t w = held[half][i];
            const _Float16 d1 = __builtin_bit_cast(_Float16, held_scale[half][i]);
            const f16x2_t d = {d1, d1};
            const uint32_t to = stage + half * TILE + (row >> 3) * RB + (piece >> 2) * 1024;
#pragma unroll
            for (int y = 0; y < 2; y++) {
                u32x4_t f;
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const uint32_t flipped = w[2 * y + z] ^ 0x80808080u;
                    f[2 * z] = __builtin_bit_cast(uint32_t, whole_pair<false>(flipped) * d);
                    f[2 * z + 1] = __builtin_bit_cast(uint32_t, whole_pair<true>(flipped) * d);
                }
                *(__attribute__((address_space(3))) u32x4_t*)(uintptr_t)(to + 16 * block_place(row, 2 * piece + y)) = f;
            }
        }
    };
    typedef std::integral_constant<int, 0> First;
    typedef std::integral_constant<int, 1> Second;

    // ---- fragments ---------------------------------------------------------------------------------------------------
    // keys: row 32 half + col, piece 2 ks + h; values: keys 32 half + 16 x + 8 y + 4 h + (lane % 16) / 4 (the rows of one transposing
    // read are four keys), elements 32 t + 16 ((lane % 32) / 16) + 4 (lane % 4) ...
    const uint32_t k_at[2] = {lds0 + (uint32_t)((col >> 3) * RB + 16 * block_place(col, h)), lds0 + (uint32_t)((col >> 3) * RB + 16 * block_place(col, 2 + h))};
    const uint32_t v_at = lds0 + (uint32_t)(TILE + 16 * block_place(4 * h + ((lane & 15) >> 2), 2 * ((lane & 31) >> 4) + ((lane & 3) >> 1)) + 8 * (lane & 1));
    // one lane's addresses in a stage; everything else is an immediate offset
    struct At {
        uint32_t k[2], v;
    };
    auto at_stage = [&](uint32_t stage) -> At {
        At x = {{k_at[0] + stage, k_at[1] + stage}, v_at + stage};
        asm volatile("" : "+v"(x.k[0]), "+v"(x.k[1]), "+v"(x.v));     // (or every address would be formed by itself)
        return x;
    };
    auto key_fragment = [&](const At& x, int half, int ks) -> op_t {
        return *(const __attribute__((address_space(3))) op_t*)(uintptr_t)(x.k[ks & 1] + 4 * half * RB + (ks >> 2) * 1024 + ((ks & 2) ? 512 : 0));
    };
    auto value_fragment = [&](const At& x, int half, int t, int y) -> op_t {
        u32x2_t part[2];
#pragma unroll
        for (int z = 0; z < 2; z++)
            part[z] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(uintptr_t)(
                x.v + (4 * half + 2 * y + z) * RB + (t >> 1) * 1024 + (t & 1) * 512)));
        return __builtin_bit_cast(op_t, u32x4_t{part[0][0], part[0][1], part[1][0], part[1][1]});
    };

    // ---- the first tile's keys, this lane's row: its query as operand fragments, and the keys that it sees -----------------------
    // Queries are asked for as tiles are, whole lines at a time, each wavefront its own rows, into the room of the stages behind the first, or of
    // all if keys come through registers (a lane that reads its own row takes a quarter of each line: seven prompts of 1 to 2047 tokens, 78.7 us, took
    // 80.9).  Read by lanes where the room is too small, and for heads of 256, whose loop then took 4 % longer.  Nothing else is asked for
    // before both are there.
    const int64_t my_row = r0 + 32 * wave + col;
    constexpr uint32_t kStage = 2 * TILE, kRing = NS * kStage;   // a stage: keys of tile i, values of tile i - 1
    constexpr bool QLDS = DT < 256 && (Q8 || (NS - 1) * kStage >= 4 * W * RB);
    constexpr uint32_t QROOM = Q8 ? 0 : kStage;
    const uint32_t group = (uint32_t)a.group, token0 = (uint32_t)r0 / group;
    int32_t page_k = 0, page_v = 0;
    op_t qf[KS];
    float c = a.scale_log2;
    int32_t first, last;
    {
        int32_t head;
        const int32_t token = attention_token(a, my_row < r1 ? my_row : r1 - 1, head);
        head += b.kv_head * a.group;
        const int32_t place = back + token;
        last = b.causal && place < most ? place : most;
        first = a.window && place - a.window + 1 > 0 ? (int32_t)(place - a.window + 1) : 0;
        u32x4_t raw[KS] = {};
        if (count > 0) {
            page_k = page_v = page_of(s0);
            aim(0, s0, page_k);
#pragma unroll
            for (int j = 0; j < REQ; j++) request(0, lds0, j);
            if constexpr (QLDS) {
                // row 32 wave + 8 i + crow of the tile; rows behind the last are its first
                const bf16_t* row0 = a.q + (b.s.q0 + token0) * a.q_token + (int64_t)(b.kv_head * a.group + (uint32_t)r0 - token0 * group) * a.q_head;
                const uint32_t r = (uint32_t)r0 + 32 * wave + crow;
                const uint32_t t = r / group;
                uint32_t g = r - t * group;
                const RowWalk walk(group, 8, a.q_token, a.q_head);
                const bf16_t* from = a.q + (b.s.q0 + t) * a.q_token + (int64_t)(b.kv_head * group + g) * a.q_head;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bf16_t* row = r + 8 * i < r1 ? from : row0;
#pragma unroll
                    for (int p = 0; p < PB; p++)
                        copy_request(lds0 + QROOM + (4 * wave + i) * RB + p * 1024, row + (64 * p + 8 * cpiece < a.dim ? 64 * p + 8 * cpiece : 0));
                    walk.next(from, g);
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                const At at = at_stage(QROOM + 4 * wave * RB);
#pragma unroll
                for (int i = 0; i < KS; i++) {
                    raw[i] = __builtin_bit_cast(u32x4_t, key_fragment(at, 0, i));
                    if (16 * i + 8 * h >= a.dim) raw[i] = u32x4_t{0u, 0u, 0u, 0u};
                }
            }
        }
        if constexpr (!QLDS) {
            const bf16_t* q = a.q + (b.s.q0 + token) * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
            for (int i = 0; i < KS; i++) {
                const int e = 16 * i + 8 * h;
                raw[i] = e < a.dim ? *reinterpret_cast<const u32x4_t*>(q + e) : u32x4_t{0u, 0u, 0u, 0u};
            }
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

    // ---- pieces of a step ----------------------------------------------------------------------------------------------
    typedef uint32_t weights_t[2][4];     // [16 keys][pair]
    auto mask = [&](f32x16_t& s, int32_t key0) {
        if (key0 + 31 > all_last || key0 < all_first) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int32_t key = key0 + 8 * (i >> 2) + 4 * h + (i & 3);
                if (key < first || key > last) s[i] = -__builtin_inff();
            }
        }
    };
    auto raise_pair = [&](const f32x16_t& s, float add, int p, float& p0, float& p1) {
        p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * p], c, add));
        p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * p + 1], c, add));
    };
    auto pack_pair = [&](weights_t& w, float& sum, int p, float p0, float p1) {
        if constexpr (Q8) {
            w[p / 4][p % 4] = pack_f16(p0, p1);
            sum += p0 + p1;
        } else {
            // (one instruction adds both of a pair; 8 bits: two, of weights whose rounding is an eighth of bf16's)
            const uint32_t both = pack_bf16(p0, p1);
            w[p / 4][p % 4] = both;
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, both), __builtin_bit_cast(bf16x2_t, 0x3F803F80u), sum, false);
        }
    };
    // maximum, sums and weights from the scores
    auto set_right = [&](const f32x16_t& s, weights_t& w, float& sum) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
        top = fmaxf(top, other_half(top));
        top = fmaxf(top * c, m);
        const bool none = top == -__builtin_inff();
        const float base = none ? 0.f : top, keep = __builtin_amdgcn_exp2f(m - base), add = kUp - base;
        m = top;
        nb = none ? __builtin_inff() : add;
        l *= keep;
#pragma unroll
        for (int t = 0; t < DTILES; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[t][i] *= keep;
        sum = 0.f;
#pragma unroll
        for (int p = 0; p < NP; p++) {
            float p0, p1;
            raise_pair(s, add, p, p0, p1);
            pack_pair(w, sum, p, p0, p1);
        }
    };
    auto weights_operand = [&](const weights_t& w, int x) -> op_t { return __builtin_bit_cast(op_t, u32x4_t{w[x][0], w[x][1], w[x][2], w[x][3]}); };

    op_t ring[4];
    // One step: values of keys 32 half ... of a stage times w0; weights of s into w1; scores of keys 32 half ... into s1.
    // The first three fragments are in the ring; the next step's are fetched by its end, from the same stage or from `next`, behind
    // the barrier that this needs.  beside(f): what else is done beside fragment f.
    auto step = [&](f32x16_t& s, f32x16_t& s1, const weights_t& w0, weights_t& w1, const At& at, const At& next, int32_t key0, auto half_, auto beside) {
        constexpr int half = decltype(half_)::value;
        mask(s, key0);
#pragma unroll
        for (int i = 0; i < 16; i++) s1[i] = 0.f;
        float sum = 0.f;
        // (a pair is packed one fragment after it was raised: the exponential's result is a while coming)
        constexpr int PF = (NP + NF - 1) / NF;         // pairs of a fragment at most
        float up[2][PF][2];
        auto pack_of = [&](auto f_) {
            constexpr int f = decltype(f_)::value, p0 = f * NP / NF, p1 = (f + 1) * NP / NF;
#pragma unroll
            for (int p = p0; p < p1; p++) pack_pair(w1, sum, p, up[f & 1][p - p0][0], up[f & 1][p - p0][1]);
        };
        each_of(
            [&](auto f_) {
                constexpr int f = decltype(f_)::value, g = f + 3;
                beside(f_);
                if constexpr (g < VF) ring[g & 3] = value_fragment(at, half, g % DTILES, g / DTILES);
                else if constexpr (g < NF) ring[g & 3] = key_fragment(at, half, g - VF);
                else ring[g & 3] = value_fragment(next, half ^ 1, (g - NF) % DTILES, (g - NF) / DTILES);
                if constexpr (f < VF) acc[f % DTILES] = mfma(ring[f & 3], weights_operand(w0, f / DTILES), acc[f % DTILES]);
                else s1 = mfma(ring[f & 3], qf[f - VF], s1);
                constexpr int p0 = f * NP / NF, p1 = (f + 1) * NP / NF;
#pragma unroll
                for (int p = p0; p < p1; p++) raise_pair(s, nb, p, up[f & 1][p - p0][0], up[f & 1][p - p0][1]);
                if constexpr (f > 0) pack_of(std::integral_constant<int, f - 1>());
            },
            std::make_integer_sequence<int, NF>());
        pack_of(std::integral_constant<int, NF - 1>());
        if (__any(!(sum <= kLimit))) set_right(s, w1, sum);
        l += sum;
    };
    auto scores = [&](const At& at, int half) -> f32x16_t {
        f32x16_t s = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) s = mfma(key_fragment(at, half, ks), qf[ks], s);
        return s;
    };
    auto values = [&](const weights_t& w, const At& at, int half) {
#pragma unroll
        for (int f = 0; f < VF; f++) acc[f % DTILES] = mfma(value_fragment(at, half, f % DTILES, f / DTILES), weights_operand(w, f / DTILES), acc[f % DTILES]);
    };

    if (count > 0) {
        weights_t wa, wb;
        float sum;
        // (behind the last tile: of the last, read by nobody, so that the loop neither asks whether there are more nor counts what is
        // under way)
        auto after = [&](uint32_t stage) { return stage + kStage < kRing ? stage + kStage : 0u; };
        // the requests of all stages but the NS - 2 last asked for have arrived, from every wavefront
        auto wait_stage = [&] {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * REQ * (NS - 2)) : "memory");
            __syncthreads();
        };
        auto aim_stage = [&](int32_t i) {
            const int32_t tk = s0 + (i < count ? i : count - 1), tv = s0 + (i <= count ? i : count) - 1;
            page_v = page_k;
            page_k = page_of(tk);
            aim(0, tk, page_k);
            aim(1, tv, page_v);
        };
        if constexpr (Q8) {
            __syncthreads();       // (every wavefront has its queries)
#pragma unroll
            for (int i = 0; i < QN; i++) widen(0, lds0, i);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int n = 1; n < NS; n++) {
            aim_stage(n);
#pragma unroll
            for (int j = 0; j < 2 * REQ; j++) request(j / REQ, lds0 + n * kStage, j % REQ);
        }
        At at = at_stage(0);
        f32x16_t sa = scores(at, 0), sb = scores(at, 1);
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 2 * QN; i++) widen(i / QN, lds0 + kStage, i % QN);
        }
        mask(sa, s0 * kKeys);
        set_right(sa, wa, sum);
        l += sum;
        wait_stage();
        uint32_t stage = kStage;                       // of tile i's keys
        uint32_t ahead = NS == 2 ? 0u : after(kStage); // the last one asked for
        at = at_stage(stage);
        ring[0] = value_fragment(at, 0, 0, 0);
        ring[1] = value_fragment(at, 0, 1 % DTILES, 1 / DTILES);
        ring[2] = value_fragment(at, 0, 2 % DTILES, 2 / DTILES);
        for (int32_t i = 1; i < count; i++) {
            if constexpr (NS > 2) ahead = after(ahead);
            else ahead = after(stage);
            stage = after(stage);
            const At next = at_stage(stage);
            aim_stage(i + NS - 1);
            const int32_t key0 = (s0 + i - 1) * kKeys + 32;
            const uint32_t to = lds0 + ahead;
            // requests and widened pieces are dealt over the fragments: close together they fill the memory pipeline's queue
            step(sb, sa, wa, wb, at, at, key0, First(), [&](auto f_) {
                constexpr int f = decltype(f_)::value;
#pragma unroll
                for (int j = f * REQ / NF; j < (f + 1) * REQ / NF; j++) request(0, to, j);
            });
            step(sa, sb, wb, wa, at, next, key0 + 32, Second(), [&](auto f_) {
                constexpr int f = decltype(f_)::value, before = NF - 3;
                if constexpr (f < before) {
#pragma unroll
                    for (int j = f * REQ / before; j < (f + 1) * REQ / before; j++) request(1, to, j);
                    if constexpr (Q8) {
#pragma unroll
                        for (int j = f * 2 * QN / before; j < (f + 1) * 2 * QN / before; j++) widen(j / QN, to, j % QN);
                    }
                }
                if constexpr (f == before) wait_stage();
            });
            at = next;
        }
        values(wa, at, 0);
        mask(sb, (s1 - 1) * kKeys + 32);
        set_right(sb, wb, sum);
        l += sum;
        values(wb, at, 1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // no request outlives the workgroup's LDS
    }

    // ---- out: acc[t][i]: this lane's row, element 32 t + 8 (i / 4) + 4 h + i % 4 ---------------------------------------------
    l += other_half(l);
    float odd = l * 0.f;
#pragma unroll
    for (int t = 0; t < DTILES; t++)
#pragma unroll
        for (int i = 0; i < 16; i++) odd = __builtin_fmaf(acc[t][i], 0.f, odd);
    const uint64_t odd_lanes = __ballot(odd != 0.f && my_row < r1);
    uint32_t again = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);      // the wavefront's rows that are not finite
    if (b.partial) {
        if (my_row < r1) {
            const int64_t at = b.slot * ROWS + (my_row - r0);
#pragma unroll
            for (int t = 0; t < DTILES; t++)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<f32x4_t*>(a.partial + at * DP + 32 * t + 2 * i + 4 * h) = f32x4_t{acc[t][i], acc[t][i + 1], acc[t][i + 2], acc[t][i + 3]};
            if (h == 0) {
                float* st = a.partial + a.grid * ROWS * DP + at * 2;
                st[0] = m;
                st[1] = l;
            }
        }
    } else {
        // through LDS (each wavefront its own rows, in the room of the stages), so that whole rows are written: a lane has eight bytes of
        // each of its row's pieces
        constexpr int OUT = 2 * DT + 16;                   // bytes of a row there; the padding spreads rows over the banks
        static_assert(ROWS * OUT <= NS * 2 * TILE, "room");
        __syncthreads();
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint8_t* room = lds + wave * 32 * OUT;
#pragma unroll
        for (int t = 0; t < DTILES; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<u32x2_t*>(room + col * OUT + 2 * (32 * t + 2 * i + 4 * h)) =
                    u32x2_t{pack_bf16(acc[t][i] * inv, acc[t][i + 1] * inv), pack_bf16(acc[t][i + 2] * inv, acc[t][i + 3] * inv)};
        __syncthreads();
        constexpr int LANES = DP / 8, AT_ONCE = 64 / LANES;   // lanes of a row, rows of an instruction
        const int e = 8 * (lane % LANES);
        uint32_t row = lane / LANES;
        const uint32_t r = (uint32_t)r0 + 32 * wave + row, t = r / group;
        uint32_t g = r - t * group;
        bf16_t* to = a.out + (b.s.q0 + t) * a.out_token + (int64_t)(b.kv_head * group + g) * a.out_head + e;
        const RowWalk walk(group, AT_ONCE, a.out_token, a.out_head);
#pragma unroll
        for (int i = 0; i < 32 / AT_ONCE; i++) {
            if (r + AT_ONCE * i < r1 && e < a.dim) *reinterpret_cast<u32x4_t*>(to) = *reinterpret_cast<const u32x4_t*>(room + (row + AT_ONCE * i) * OUT + 2 * e);
            walk.next(to, g);
        }
    }
    // (this wavefront's stores above stay in front: these rows are written twice, and the second is what is left)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    while (again) {
        const int i = __builtin_ctz(again);
        again &= again - 1;
        attention_row_again<DP, SOURCE, ROWS, Q8 ? 12 : 0>(a, b, r0 + 32 * wave + i, s0 * kKeys, s1 * kKeys < hi ? s1 * kKeys : hi);
    }
}

// dim: of the kernel, 64, 96, 128, 192 or 256; rows: of a workgroup, 128 or (up to 192 elements) 256
int launch_attention_tiles(const AttentionArgs& a, int rows, int dim, int source, hipStream_t stream) {
    const bool planned = a.map != nullptr;
#define SNGGUF_GO(D, S, W, N, P)                                                                                        \
    if (dim == D && source == S && rows == 32 * W && planned == P) {                                                    \
        constexpr int kLds = N * 2 * Tile<D>::kBytes;                                                                   \
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&attention_tiles_kernel<D, S, W, N, P>), \
                                                           hipFuncAttributeMaxDynamicSharedMemorySize, kLds);           \
        if (attr != hipSuccess) return SNGGUF_E_LAUNCH;                                                                 \
        attention_tiles_kernel<D, S, W, N, P><<<dim3((unsigned)a.grid), 64 * W, kLds, stream>>>(a);                     \
        return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;                                           \
    }
    // (three stages where a compute unit has room for them; 8-bit tiles pass through registers and need two)
#define SNGGUF_GO_PAGED(D, W, N, P) SNGGUF_GO(D, kPaged, W, N, P) SNGGUF_GO(D, kPagedQ8, W, 2, P)
#define SNGGUF_GO_DIM(D, W, N) SNGGUF_GO(D, kPacked, W, N, false) SNGGUF_GO_PAGED(D, W, N, false) SNGGUF_GO_PAGED(D, W, N, true)
    SNGGUF_GO_DIM(64, 4, 3)
    SNGGUF_GO_DIM(64, 8, 3)
    SNGGUF_GO_DIM(96, 4, 2)
    SNGGUF_GO_DIM(96, 8, 3)
    SNGGUF_GO_DIM(128, 4, 2)
    SNGGUF_GO_DIM(128, 8, 3)
    SNGGUF_GO_DIM(192, 4, 2)
    SNGGUF_GO_DIM(192, 8, 2)
    SNGGUF_GO_DIM(256, 4, 2)
#undef SNGGUF_GO_DIM
#undef SNGGUF_GO_PAGED
#undef SNGGUF_GO
    return SNGGUF_E_BADSHAPE;
}

}  // namespace sngguf
