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
// q = rint(x / d) without a division for each: with r = 1 / d to a step, t = x r is off by less than 2^-15, and q = rint(t) can
// be wrong only if x / d is that near to a half.  It then is one: x has 8 significant bits and d at most 11, so |x / d - (n + 1/2)|, a multiple
// of 2^-12 at least for numbers in reach, is 0 or more than that.  x - q d is exact, so 2 |x - q d| = d tells, and the even one is taken.
// (Largest magnitudes are compared as whole numbers, which bf16 without its sign is ordered as, NaN above all.)
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
        const float r = __builtin_amdgcn_rcpf(d), most = 127.f * d;
        float x[8];
        unpack8(p, x);
        uint32_t q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float within = __builtin_amdgcn_fmed3f(x[i], -most, most);
            const float u = within * r + kWhole;
            const float off = __builtin_fmaf(-(u - kWhole), d, within);
            q[i] = __builtin_bit_cast(uint32_t, u);
            if (2.f * __builtin_fabsf(off) == d && (q[i] & 1u)) q[i] += off > 0.f ? 1u : 0xFFFFFFFFu;
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
            out[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0C0C0400u),
                                           __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0C0C0400u), 0x05040100u);
    }
    return out;
}

// One piece (eight elements from e on) of a token's head into the cache.
template <bool Q8>
__device__ __forceinline__ void cache_piece(void* pages, uint16_t* scales, const RotaryCacheArgs& a, int64_t slot, int head, int e, u32x4_t v) {
    const int64_t page = slot >> a.page_shift, row = slot & ((1 << a.page_shift) - 1);
    const int64_t at = page * a.kv_heads + head;
    if constexpr (Q8) {
        uint16_t scale;
        const u32x2_t q = quantise8(v, scale);
        *reinterpret_cast<u32x2_t*>(static_cast<int8_t*>(pages) + ((at << a.page_shift) + row) * a.dim + e) = q;
        if ((e & 31) == 0) scales[((at * (a.dim >> 5) + (e >> 5)) << a.page_shift) + row] = scale;
    } else {
        *reinterpret_cast<u32x4_t*>(static_cast<bf16_t*>(pages) + ((at << a.page_shift) + row) * a.dim + e) = v;
    }
}

}  // namespace sngguf
