/*
 * The rows of a typed KV cache: conversions between f32 and the 16-bit (F16,
 * BF16), 8-bit (Q8_K) and 4-bit (MXFP4) elements of its pages.
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

/* MXFP4.  The conversions take the scale as the power of two that a scale byte E
 * stands for (E = 255, which an infinity or NaN leaves: an infinity, and every
 * value of the block NaN). */
Q38_DEV uint8_t *q38_mx4_scales(char *block, int head) {
    return reinterpret_cast<uint8_t *>(block + q38_mx4_scales_offset(head));
}
typedef float q38_f32x2 __attribute__((ext_vector_type(2)));
Q38_DEV float q38_mx4_power(uint32_t e) { return __uint_as_float(e << 23); }
/* The scale byte of a block whose largest size has these bits: 2^(E - 127) is the
 * smallest power of two of which that is at most 7, the largest that rounds to a
 * code without being cut (6); from 2^-125, so that its values, from 2^-126 on, are
 * normal, to 2^125, so that they are finite.  Against the power below the largest
 * value's own alone, which cuts up to a quarter of it, the error of normal
 * values is 0.112 of their size, not 0.115. */
Q38_DEV uint32_t q38_mx4_exponent(uint32_t largest) {
    const uint32_t e = (largest + 0x1FFFFFu) >> 23;
    return largest >= 0x7F800000u ? 255u : min(max(e, 4u), 254u) - 2u;
}
/* Codes of two values in byte SEL of a word, nearest, halfway to the even code; and back. */
template <int SEL>
Q38_DEV uint32_t q38_mx4_pack(uint32_t word, float a, float b, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, a, b, scale, SEL);
}
template <int SEL>
Q38_DEV q38_f32x2 q38_mx4_pair(uint32_t word, float scale) {
    return __builtin_bit_cast(q38_f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, SEL));
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
    if constexpr (T == Q38_KV_MX4) {
        const uint32_t u = *reinterpret_cast<const uint16_t *>(block + (i >> 1));
        const float s = q38_mx4_power(q38_mx4_scales(block, head)[q38_mx4_k_scale(t, d)]);
        const q38_f32x2 a = q38_mx4_pair<0>(u, s), b = q38_mx4_pair<1>(u, s);
        x = f32x4{a[0], a[1], b[0], b[1]};
    } else if (T == Q38_KV_Q8) {
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
    if constexpr (T == Q38_KV_MX4) {
        /* a pair's bytes lie side by side, both hold dim d and its partner 16 away */
        const uint8_t *scales = q38_mx4_scales(block, head);
        const float p0 = q38_mx4_power(scales[q38_mx4_v_scale(t0, d)]), p1 = q38_mx4_power(scales[q38_mx4_v_scale(t1, d)]);
        const int half = (d >> 4) & 1;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t u = *reinterpret_cast<const uint16_t *>(block + (q38_v_index<T>(t0 & ~1, d + c) >> 1));
            const q38_f32x2 a = q38_mx4_pair<0>(u >> (8 * (t0 & 1)), p0), b = q38_mx4_pair<0>(u >> (8 * (t1 & 1)), p1);
            x0[c] = half ? a[1] : a[0];
            x1[c] = half ? b[1] : b[0];
        }
        return;
    }
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
