/*
 * The rows of a typed KV cache: conversions between f32 and the 16-bit (F16,
 * BF16) and 8-bit (Q8_K) elements of its pages.
 */
#pragma once
#include "q38_device.h"
#define Q38_LAYOUT_FN Q38_DEV
#include "../q38_kv_layout.h"

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 q38_bf16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t q38_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t q38_u32x4 __attribute__((ext_vector_type(4)));

/* The block of (page, kv head) in a slot's pool. */
template <int T>
Q38_DEV char *q38_kv_block(void *pool, int page, int head) {
    return static_cast<char *>(pool) + (size_t)page * q38_kv_page_bytes<T>() + head * q38_kv_block_bytes<T>();
}

Q38_DEV float *q38_kv_scales(char *block, int head) {
    return reinterpret_cast<float *>(block + q38_kv_scales_offset(head));
}

/* A 16-bit value of the type, rounded to nearest even (F16: past 65504 to
 * infinity), and back. */
template <int T>
Q38_DEV uint16_t q38_to16(float x) {
    if (T == Q38_KV_F16) return __builtin_bit_cast(uint16_t, (_Float16)x);
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}
template <int T>
Q38_DEV float q38_from16(uint16_t b) {
    if (T == Q38_KV_F16) return (float)__builtin_bit_cast(_Float16, b);
    return __uint_as_float((uint32_t)b << 16);
}

/* Dims d .. d + 3 (d a multiple of 4) of one token's key. */
template <int T>
Q38_DEV f32x4 q38_k_load4(char *block, int head, int t, int d) {
    const int i = q38_k_index<T>(t, d);
    f32x4 x;
    if (T == Q38_KV_Q8) {
        const uint32_t u = *reinterpret_cast<const uint32_t *>(block + i);
        const float s = q38_kv_scales(block, head)[t];
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = (float)((int)((u >> (8 * c)) & 255u) - 128) * s;
    } else {
        const q38_u32x2 u = *reinterpret_cast<const q38_u32x2 *>(block + 2 * i);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = q38_from16<T>((uint16_t)(u[c >> 1] >> (16 * (c & 1))));
    }
    return x;
}

/* Dims d .. d + 3 of the values of tokens t0 and t1, which share a pair of
 * tokens (2n, 2n + 1), maybe the same one twice. */
template <int T>
Q38_DEV void q38_v_load4(char *block, int head, int t0, int t1, int d, f32x4 &x0, f32x4 &x1) {
    const float s0 = T == Q38_KV_Q8 ? q38_kv_scales(block, head)[t0] : 0.0f;
    const float s1 = T == Q38_KV_Q8 ? q38_kv_scales(block, head)[t1] : 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int i = q38_v_index<T>(t0 & ~1, d + c);
        if (T == Q38_KV_Q8) {
            const uint32_t u = *reinterpret_cast<const uint16_t *>(block + i);
            x0[c] = (float)((int)((u >> (8 * (t0 & 1))) & 255u) - 128) * s0;
            x1[c] = (float)((int)((u >> (8 * (t1 & 1))) & 255u) - 128) * s1;
        } else {
            const uint32_t u = *reinterpret_cast<const uint32_t *>(block + 2 * i);
            x0[c] = q38_from16<T>((uint16_t)(u >> (16 * (t0 & 1))));
            x1[c] = q38_from16<T>((uint16_t)(u >> (16 * (t1 & 1))));
        }
    }
}

/* A head's 256 values held 4 per lane by a wave (lane l: 4l .. 4l + 3) as a
 * Q8_K block: the quants, and the scale (the same in every lane). */
Q38_DEV void q38_wave_q8k(f32x4 x, int (&q)[4], float &scale) {
    float big = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    big = q38_max16(big);
    {
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(big), __float_as_uint(big), false, false);
        big = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        const q38_halves h = q38_both_halves(big);
        big = fmaxf(h.a, h.b);
    }
    if (big == 0.0f) {
        q[0] = q[1] = q[2] = q[3] = 0;
        scale = 0.0f;
        return;
    }
    /* the first value of that size: the lowest lane holding one, its lowest
     * dim.  Only its sign is left to find. */
    const bool mine = fabsf(x.x) == big || fabsf(x.y) == big || fabsf(x.z) == big || fabsf(x.w) == big;
    const float cand = fabsf(x.x) == big ? x.x : fabsf(x.y) == big ? x.y : fabsf(x.z) == big ? x.z : x.w;
    const uint64_t holders = __ballot(mine);
    const float m = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(cand), holders ? __builtin_ctzll(holders) : 0));
    const float inverse = -127.0f / m;
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = min(q38_nearest_int(inverse * x[c]), 127);
    scale = 1.0f / inverse;
}
