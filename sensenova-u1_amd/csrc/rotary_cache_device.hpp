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
__device__ __forceinline__ u32x2_t quantise8(u32x4_t p, uint16_t& scale) {
    float x[8];
    unpack8(p, x);
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        top = fmaxf(top, __builtin_fabsf(x[i]));
        bad |= x[i] != x[i];
    }
    if (bad) top = __builtin_nanf("");
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float t = __shfl_xor(top, o);
        top = (top != top || t != t) ? __builtin_nanf("") : fmaxf(top, t);
    }
    float d = top / 127.f;
    if (d > 512.f) d = 512.f;
    scale = f32_to_f16(d);
    d = f16_to_f32(scale);
    u32x2_t out = {0u, 0u};
    if (d > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float q = __builtin_rintf(x[i] / d);
            q = q > 127.f ? 127.f : q < -127.f ? -127.f : q;
            out[i >> 2] |= ((uint32_t)(int)q & 0xFFu) << (8 * (i & 3));
        }
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
