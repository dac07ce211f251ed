// What the kernels that turn heads and write the paged cache share: angles, pieces of eight elements, the 8-bit format.
#pragma once

#include "rotary_cache.hpp"

namespace sngguf {

__device__ __forceinline__ float2 cos_sin(const double* turns, int pair, int64_t position, double magnitude) {
    const double t = (double)position * turns[pair];
    double s, c;
    sincospi(2.0 * (t - rint(t)), &s, &c);
    return make_float2((float)(c * magnitude), (float)(s * magnitude));
}

// eight bf16 values <-> fp32
__device__ __forceinline__ void unpack8(u32x4_t p, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = bf16lo_to_f32(p[i]);
        x[2 * i + 1] = bf16hi_to_f32(p[i]);
    }
}
__device__ __forceinline__ u32x4_t pack8(const float (&x)[8]) {
    return u32x4_t{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
}

// Eight bf16 values of a head starting at element e; `wide`: 16-byte aligned.
__device__ __forceinline__ u32x4_t load8(const bf16_t* p, bool wide) {
    if (wide) return *reinterpret_cast<const u32x4_t*>(p);
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (uint32_t)p[2 * i] | ((uint32_t)p[2 * i + 1] << 16);
    return v;
}
__device__ __forceinline__ void store8(bf16_t* p, u32x4_t v, bool wide) {
    if (wide) {
        *reinterpret_cast<u32x4_t*>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        p[2 * i] = (bf16_t)v[i];
        p[2 * i + 1] = (bf16_t)(v[i] >> 16);
    }
}

// Eight elements into a run: four neighbouring lanes hold it.  Returns the whole numbers, and the scale for the run.
//
// q = rint(x / d) without a division for each: with r = 1 / d to a step, t = x r is off by at most 2^-22 of itself, and t + (x - t d) r by 2^-44,
// before it is rounded.  That gives the same whole number: x has 8 significant bits and d at most 11, so x / d is a half exactly, which the
// second t then is too, or further from one than 2^-13.  (Checked over all largest magnitudes of a run, all x up to them and r off by a step either way.)
// No whole number is beyond 127 then, but where d is held to 512 or rounded down by more than 2^-8 of itself, as a scale below the smallest
// normal one, 2^-14, may be: at 2^-24 by a third, where x / d is up to 190.  Only there are x held to 127 d.
// Largest magnitudes are compared as whole numbers, which bf16 without its sign is ordered as, NaN above all.
__device__ __forceinline__ u32x2_t quantise8(u32x4_t p, uint16_t& scale) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t magnitude = p[i] & 0x7FFF7FFFu;
        m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, magnitude));
    }
    uint32_t top_bits = m[0] > m[1] ? m[0] : m[1];
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const uint32_t other = o == 1 ? (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top_bits, 0xB1, 0xF, 0xF, false)
                                      : (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top_bits, 0x4E, 0xF, 0xF, false);
        top_bits = top_bits > other ? top_bits : other;
    }
    const float top = top_bits > 0x7F80u ? __builtin_nanf("") : __builtin_bit_cast(float, top_bits << 16);
    float d = top / 127.f;
    if (d > 512.f) d = 512.f;
    scale = f32_to_f16(d);
    d = f16_to_f32(scale);
    u32x2_t out = {0u, 0u};
    if (d > 0.f) {
        constexpr float kWhole = 12582912.f;           // 1.5 x 2^23: added to a small number, it rounds it to a whole one in its low bits
        const float r = __builtin_amdgcn_rcpf(d);
        float x[8];
        unpack8(p, x);
        if (d >= 512.f || d < 0x1p-14f) {
            const float most = 127.f * d;
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __builtin_amdgcn_fmed3f(x[i], -most, most);
        }
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float t = x[i] * r;
            q[i] = __builtin_bit_cast(uint32_t, __builtin_fmaf(__builtin_fmaf(-t, d, x[i]), r, t) + kWhole);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
            out[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0C0C0400u),
                                           __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0C0C0400u), 0x05040100u);
    }
    return out;
}

// Where a token's head lies in one half of the cache: its elements, and its first scale
struct CachePlace {
    uint8_t* row;
    uint16_t* scale;
};
template <bool Q8>
__device__ __forceinline__ CachePlace cache_place(void* pages, uint16_t* scales, const RotaryCacheArgs& a, int64_t slot, int head) {
    const uint32_t page = (uint32_t)(slot >> a.page_shift), row = (uint32_t)slot & ((1u << a.page_shift) - 1);
    const uint64_t at = (uint64_t)page * (uint32_t)a.kv_heads + (uint32_t)head;
    return {static_cast<uint8_t*>(pages) + ((at << a.page_shift) + row) * (uint32_t)(a.dim * (Q8 ? 1 : 2)), scales + ((at * (uint32_t)(a.dim >> 5) << a.page_shift) + row)};
}

// One piece (eight elements from e on) of a token's head into the cache.
template <bool Q8>
__device__ __forceinline__ void cache_piece(const CachePlace& to, const RotaryCacheArgs& a, int e, u32x4_t v) {
    if constexpr (Q8) {
        uint16_t scale;
        const u32x2_t q = quantise8(v, scale);
        *reinterpret_cast<u32x2_t*>(to.row + e) = q;
        if ((e & 31) == 0) to.scale[(uint32_t)(e >> 5) << a.page_shift] = scale;
    } else {
        *reinterpret_cast<u32x4_t*>(to.row + 2 * e) = v;
    }
}

}  // namespace sngguf
