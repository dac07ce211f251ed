// Rotary positions, and the paged cache of keys and values: written (with the rotation in the same launch or without),
// and read back.
//
// Rotation of a pair (x, y) at position p by its rate f (turns a position): with a = 2 pi p f,
//     x' = x c - y s,  y' = y c + x s,   c = fp32(m cos a), s = fp32(m sin a), m the table's magnitude.
// p f is formed in 64 bits and reduced to the nearest whole turn there: in 32 bits the angle of position 10^6 would be off by
// 0.06 rad.  Pairs are (2 i, 2 i + 1) or (i, i + pairs); elements behind the turned ones are copied.
//
// An 8-bit cache holds runs of 32 elements as Q8_0 does: d = fp16(max |x| / 127), whole numbers q = rint(x / d), value d q.
// d is at most 512, so that every value is within fp16 (the attention kernels multiply in fp16): larger magnitudes are held as
// +-65024.  A run with a NaN is held as NaN.
//
// All of it is bound by memory.  A workgroup takes a few tokens: its threads first make one (cosine, sine) pair each, in LDS,
// then work through the tokens' heads in pieces of 16 bytes.  8192 tokens of 40 heads of 128: 35.7 us, 4.7 TB/s; 5003 tokens of 32 query
// and 8 + 8 heads, keys and values written in 8 bits: 23.4 us, 4.8 TB/s; 40000 tokens read back: 53 us, 4.7 TB/s (nontemporal stores: 58).
#include "rotary_cache_device.hpp"

namespace sngguf {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ void turn(float& x, float& y, float2 w) {
    const float a = x * w.x - y * w.y, b = y * w.x + x * w.y;
    x = a;
    y = b;
}

// The eight elements from e on of a head that goes to the cache, turned; partners are read beside them.
__device__ __forceinline__ u32x4_t turned8(const bf16_t* head, int e, const RotaryCacheArgs& a, const float2* cs) {
    const u32x4_t own = load8(head + e, a.wide);
    const int turned = 2 * a.pairs;
    if (e >= turned) return own;
    float x[8], y[8];
    unpack8(own, x);
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[2 * i] = x[2 * i];
            y[2 * i + 1] = x[2 * i + 1];
            if (e + 2 * i < turned) turn(y[2 * i], y[2 * i + 1], cs[(e >> 1) + i]);
        }
        return pack8(y);
    }
    if ((a.pairs & 7) == 0) {
        const bool second = e >= a.pairs;
        const int at = second ? e - a.pairs : e;
        float z[8];
        unpack8(load8(head + (second ? at : e + a.pairs), a.wide), z);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 w = cs[at + i];
            y[i] = second ? x[i] * w.x + z[i] * w.y : x[i] * w.x - z[i] * w.y;
        }
        return pack8(y);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int k = e + i;
        y[i] = x[i];
        if (k < a.pairs) {
            const float2 w = cs[k];
            y[i] = x[i] * w.x - bf16_to_f32(head[k + a.pairs]) * w.y;
        } else if (k < turned) {
            const float2 w = cs[k - a.pairs];
            y[i] = x[i] * w.x + bf16_to_f32(head[k - a.pairs]) * w.y;
        }
    }
    return pack8(y);
}

// One unit of a head that goes to a tensor, which may be the tensor that it comes from: no other thread reads or writes the
// elements of this unit.  Neighbouring pairs: unit u is elements 8 u .. 8 u + 7.  Halves: the first ceil(pairs / 8) units are
// eight pairs each, the others eight of the elements behind the turned ones.
__device__ __forceinline__ void turn_unit(const bf16_t* from, bf16_t* to, int u, const RotaryCacheArgs& a, const float2* cs) {
    const int turned = 2 * a.pairs;
    if (a.interleaved) {
        const int e = 8 * u;
        u32x4_t v = load8(from + e, a.wide);
        if (e < turned) {
            float x[8];
            unpack8(v, x);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (e + 2 * i < turned) turn(x[2 * i], x[2 * i + 1], cs[(e >> 1) + i]);
            v = pack8(x);
        }
        store8(to + e, v, a.wide);
        return;
    }
    const int pair_units = (a.pairs + 7) >> 3;
    const bool wide = a.wide && (a.pairs & 7) == 0;
    if (u >= pair_units) {
        const int e = turned + 8 * (u - pair_units);
        if (wide) store8(to + e, load8(from + e, true), true);
        else
            for (int k = e; k < e + 8 && k < a.dim; k++) to[k] = from[k];
        return;
    }
    const int p = 8 * u;
    if (wide) {
        float x[8], y[8];
        unpack8(load8(from + p, true), x);
        unpack8(load8(from + p + a.pairs, true), y);
#pragma unroll
        for (int i = 0; i < 8; i++) turn(x[i], y[i], cs[p + i]);
        store8(to + p, pack8(x), true);
        store8(to + p + a.pairs, pack8(y), true);
        return;
    }
    for (int k = p; k < p + 8 && k < a.pairs; k++) {
        float x = bf16_to_f32(from[k]), y = bf16_to_f32(from[k + a.pairs]);
        turn(x, y, cs[k]);
        to[k] = f32_to_bf16(x);
        to[k + a.pairs] = f32_to_bf16(y);
    }
}

}  // namespace

// Items [0, units) of the heads [0, heads) of `count` tokens, dealt over the workgroup: f(token, head, unit).  Items of one
// head are neighbouring threads.
template <typename F>
__device__ __forceinline__ void each_unit(int count, int heads, int units, F f) {
    const int row0 = threadIdx.x / units, unit = threadIdx.x - row0 * units, step = kThreads / units;
    if (row0 >= step || heads == 0) return;
    int t = row0 / heads, h = row0 - t * heads;
    while (t < count) {
        f(t, h, unit);
        h += step;
        while (h >= heads) {
            h -= heads;
            t++;
        }
    }
}

// ROTARY: q (and k) are turned.  CACHE: 0 none, 1 bf16, 2 8-bit; k and v go to their slots.
template <bool ROTARY, int CACHE>
__global__ __launch_bounds__(kThreads) void rotary_cache_kernel(RotaryCacheArgs a) {
    extern __shared__ float2 cs_all[];
    const int tid = threadIdx.x;
    const int64_t t0 = (int64_t)blockIdx.x * a.tokens_per_block;
    const int count = (int)(a.tokens - t0 < a.tokens_per_block ? a.tokens - t0 : a.tokens_per_block);
    if constexpr (ROTARY) {
        for (int i = tid; i < count * a.pairs; i += kThreads) {
            const int t = i / a.pairs, p = i - t * a.pairs;
            cs_all[i] = cos_sin(a.turns, p, a.positions[t0 + t], a.magnitude);
        }
        __syncthreads();
        const int units = a.interleaved ? a.dim >> 3 : ((a.pairs + 7) >> 3) + ((a.dim - 2 * a.pairs + 7) >> 3);
        each_unit(count, CACHE ? a.q_heads : a.q_heads + a.k_heads, units, [&](int t, int h, int u) {
            if (h < a.q_heads)
                turn_unit(a.q + (t0 + t) * a.q_token + h * a.q_head, a.q_out + (t0 + t) * a.q_out_token + h * a.q_out_head, u, a, cs_all + t * a.pairs);
            else
                turn_unit(a.k + (t0 + t) * a.k_token + (h - a.q_heads) * a.k_head, a.k_out + (t0 + t) * a.k_out_token + (h - a.q_heads) * a.k_out_head, u, a,
                          cs_all + t * a.pairs);
        });
    }
    if constexpr (CACHE != 0) {
        each_unit(count, 2 * a.kv_heads, a.dim >> 3, [&](int t, int h, int u) {
            const int64_t slot = a.slots[t0 + t];
            // slots outside the cache (padding is marked by negative ones) are passed over; the lanes of a run agree
            if (slot < 0 || slot >= a.slot_count) return;
            if (h < a.kv_heads) {
                const bf16_t* p = a.k + (t0 + t) * a.k_token + h * a.k_head;
                cache_piece<CACHE == 2>(cache_place<CACHE == 2>(a.k_pages, a.k_scales, a, slot, h), a, 8 * u, ROTARY ? turned8(p, 8 * u, a, cs_all + t * a.pairs) : load8(p + 8 * u, a.wide));
            } else {
                h -= a.kv_heads;
                cache_piece<CACHE == 2>(cache_place<CACHE == 2>(a.v_pages, a.v_scales, a, slot, h), a, 8 * u, load8(a.v + (t0 + t) * a.v_token + h * a.v_head + 8 * u, a.wide));
            }
        });
    }
}

// Slots of the cache as bf16 rows [tokens][kv_heads][dim]; a slot outside the cache gives zeros.  The cache with the read-once hint: 40000
// tokens in 8 bits, another cache each pass, 53 us against 55 (the same one again at once, 55 against 48).
template <bool Q8>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(RotaryCacheArgs a) {
    const int pieces = a.dim >> 3;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t token = i / (pieces * a.kv_heads);
    if (token >= a.tokens) return;
    const int rest = (int)(i - token * (pieces * a.kv_heads)), h = rest / pieces, e = 8 * (rest - h * pieces);
    const int64_t slot = a.slots[token];
    const int64_t page = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
    const int64_t at = page * a.kv_heads + h;
#pragma unroll
    for (int half = 0; half < 2; half++) {
        const void* pages = half ? a.v_pages : a.k_pages;
        const uint16_t* scales = half ? a.v_scales : a.k_scales;
        bf16_t* out = (half ? a.v_out : a.k_out) + (token * a.kv_heads + h) * a.dim + e;
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (slot >= 0 && slot < a.slot_count) {
            if constexpr (Q8) {
                const u32x2_t q = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(static_cast<const int8_t*>(pages) + ((at << a.page_shift) + row) * a.dim + e));
                const float d = f16_to_f32(scales[((at * (a.dim >> 5) + (e >> 5)) << a.page_shift) + row]);
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = d * (float)(int8_t)(q[j >> 2] >> (8 * (j & 3)));
                v = pack8(x);
            } else {
                v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(static_cast<const bf16_t*>(pages) + ((at << a.page_shift) + row) * a.dim + e));
            }
        }
        *reinterpret_cast<u32x4_t*>(out) = v;
    }
}

int launch_rotary_cache(const RotaryCacheArgs& a0, int cache, hipStream_t stream) {
    RotaryCacheArgs a = a0;
    // one token a workgroup, whose angles serve all its heads (two or four: no faster at 8192 tokens of 40 heads), more where a token has
    // less than one unit for each thread
    const int64_t units = (int64_t)(a.q_heads + (cache ? 2 * a.kv_heads : a.k_heads)) * (a.dim >> 3);
    a.tokens_per_block = units >= kThreads ? 1 : units * 8 <= kThreads ? 8 : (int32_t)(kThreads / units);
    const int64_t blocks = (a.tokens + a.tokens_per_block - 1) / a.tokens_per_block;
    if (blocks * kThreads >= (int64_t)1 << 32) return SNGGUF_E_BADSHAPE;     // (threads of a launch are numbered with 32 bits)
    const dim3 grid((unsigned)blocks);
    const size_t lds = (size_t)a.tokens_per_block * a.pairs * sizeof(float2);
    if (a.turns) {
        if (cache == 0) rotary_cache_kernel<true, 0><<<grid, kThreads, lds, stream>>>(a);
        else if (cache == 1) rotary_cache_kernel<true, 1><<<grid, kThreads, lds, stream>>>(a);
        else rotary_cache_kernel<true, 2><<<grid, kThreads, lds, stream>>>(a);
    } else {
        if (cache == 1) rotary_cache_kernel<false, 1><<<grid, kThreads, 0, stream>>>(a);
        else rotary_cache_kernel<false, 2><<<grid, kThreads, 0, stream>>>(a);
    }
    return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;
}

int launch_cache_read(const RotaryCacheArgs& a, bool q8, hipStream_t stream) {
    const int64_t threads = a.tokens * a.kv_heads * (a.dim >> 3);
    const dim3 grid((unsigned)((threads + kThreads - 1) / kThreads));
    if (q8) cache_read_kernel<true><<<grid, kThreads, 0, stream>>>(a);
    else cache_read_kernel<false><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError() == hipSuccess ? SNGGUF_OK : SNGGUF_E_LAUNCH;
}

}  // namespace sngguf
