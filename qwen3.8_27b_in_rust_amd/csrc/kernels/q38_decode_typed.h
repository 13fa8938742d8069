/*
 * Decode over a cache of 16-, 8- or 4-bit rows: the kernel of
 * attn_decode_typed.hip (which says what it does and what it measured), of
 * attn_decode_mxfp4.hip and of attn_weigh.hip.
 */
#pragma once
#include <type_traits>

#include "q38_kv_types.h"
#include "q38_rope.h"

/* 1/sqrt(256) (ops.rs:869) times log2(e). */
#define Q38_SCORE_LOG2 0.09016844005556021f

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int kWaves = Q38_DECODE_TYPED_WAVES;
constexpr int kGroup = Q38_ATTN_GROUP;
/* A head's reference lies kRefBelow under the score that set it, and is raised
 * once a score passes that one by kRefSlack. */
template <int T>
constexpr bool kInBf16 = T == Q38_KV_BF16 || T == Q38_KV_MX4; /* operands and parts, else f16 */
template <int T>
constexpr float kRefBelow = kInBf16<T> ? 0.0f : 7.0f;
constexpr float kRefSlack = 8.0f;
/* f16 weights and queries: what their lower part is larger by (the upper one's
 * rounding leaves 2^-11 of them at most, 2^4 and 2^-1). */
template <int T>
constexpr float kLowUnit = kInBf16<T> ? 1.0f : 0x1p11f;
/* 8-bit rows, weight times scale: the largest one of a page that raises a
 * head's power of two becomes 2^6 .. 2^8 units of it, and up to 2^15 raise
 * nothing.  The powers' ends keep them, their inverses and a weight (2^15 at
 * most) over them normal, and the largest scale (2^121) times such a weight
 * within f16. */
constexpr float kWeightedMax = 0x1p15f;
constexpr int kWeightedBits = 8, kUnitMin = -112, kUnitMax = 121;

/* One page of one kv head as a wave holds it. */
template <int T>
struct Page {
    static constexpr int kLoads = T == Q38_KV_Q8 ? 4 : 8; /* 1 KiB loads of each of K and V */
    q38_u32x4 k[kLoads], v[kLoads];
    f32x4 ks, vs; /* 8-bit rows: the scales of tokens 4 (lane / 16) .. + 3 */
};
template <>
struct Page<Q38_KV_MX4> {
    static constexpr int kLoads = 2;
    q38_u32x4 k[kLoads], v[kLoads];
    q38_u32x2 ks;    /* scale bytes of token lane % 16, a byte per 32 dims */
    q38_u32x4 vs[2]; /* and of tokens 4 (lane / 16) .. + 3, a word per 32 dims */
};

/* Loads of a page's block go through a buffer resource that ends with it (8-bit
 * rows: with its scales), or of no size at all: past the wave's last page they
 * fetch nothing, without a branch that would make the compiler wait for every
 * load before it.  They are non-temporal, each page being read once: 128K tokens
 * of bf16 84 us against 100 without, Q8_K 47.5 against 54.6. */
Q38_DEV __amdgpu_buffer_rsrc_t block_rsrc(char *block, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(block, 0, bytes, 0x00027000);
}
Q38_DEV q38_u32x4 ld_block(__amdgpu_buffer_rsrc_t r, int at) {
    constexpr int kStream = 2; /* non-temporal */
    return __builtin_bit_cast(q38_u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kStream));
}

Q38_DEV q38_u32x2 ld_block8(__amdgpu_buffer_rsrc_t r, int at) {
    return __builtin_bit_cast(q38_u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 2));
}

/* A page's scores, lane (c, g)'s four tokens of column c: columns past the six heads lie
 * past the range, where nothing is stored (a branch instead of it would leave the count of outstanding accesses
 * open, and every wait for the page's values would wait for this store as well: 128K tokens of MXFP4, one layer again and
 * again, 42.4 us against 38.9).  MXFP4's are written through L2 (32K tokens 15.3 us against 16.4, and 128K 38.5 against 38.9);
 * other rows' stay there for a while (bf16 27.3 against 28.0 and 100 in both, Q8_K 19.1 against 18.7 and 56.8
 * against 57.5). */
template <int T>
Q38_DEV void put_scores(float *page, bool live, int c, int g, const float (&s)[4]) {
    constexpr int kPolicy = T == Q38_KV_MX4 ? 16 : 0;
    const __amdgpu_buffer_rsrc_t r = block_rsrc(reinterpret_cast<char *>(page), live ? Q38_SCORES_PAGE * 4 : 0);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(q38_u32x4, f32x4{s[0], s[1], s[2], s[3]}), r, (c * Q38_PAGE_TOKENS + 4 * g) * 4, 0, kPolicy);
}

template <int T, typename Args>
Q38_DEV void load_page(Page<T> &p, const Args &a, int page, bool live, int j, int lane) {
    const int scales = T == Q38_KV_MX4 ? q38_mx4_scales_offset(j) : q38_kv_scales_offset(j);
    const int bytes = !live                ? 0
                      : T == Q38_KV_Q8  ? scales + Q38_PAGE_TOKENS * 4
                      : T == Q38_KV_MX4 ? scales + Q38_MX4_SCALES
                                        : q38_kv_block_bytes<T>();
    const __amdgpu_buffer_rsrc_t k = block_rsrc(q38_kv_block<T>(a.kpool, page, j), bytes);
    const __amdgpu_buffer_rsrc_t v = block_rsrc(q38_kv_block<T>(a.vpool, page, j), bytes);
#pragma unroll
    for (int i = 0; i < Page<T>::kLoads; ++i) p.k[i] = ld_block(k, 1024 * i + 16 * lane);
    if constexpr (T == Q38_KV_Q8) {
        p.ks = __builtin_bit_cast(f32x4, ld_block(k, scales + 16 * (lane >> 4)));
        p.vs = __builtin_bit_cast(f32x4, ld_block(v, scales + 16 * (lane >> 4)));
    }
    if constexpr (T == Q38_KV_MX4) {
        p.ks = ld_block8(k, scales + 8 * (lane & 15));
#pragma unroll
        for (int i = 0; i < 2; ++i) p.vs[i] = ld_block(v, scales + 32 * (lane >> 4) + 16 * i);
    }
#pragma unroll
    for (int i = 0; i < Page<T>::kLoads; ++i) p.v[i] = ld_block(v, 1024 * i + 16 * lane);
}

/* Two biased bytes of u as two halves: 0x6400 | b is 1024 + b, and 1152 less
 * is the quant, both exact. */
template <uint32_t SEL>
Q38_DEV uint32_t halves_of(uint32_t u) {
    const f16x2 x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, SEL));
    return __builtin_bit_cast(uint32_t, x + f16x2{(_Float16)-1152.0f, (_Float16)-1152.0f});
}

/* Byte B of a word of codes as two bf16 values, exactly, and the scale that byte B of a word is. */
template <int B>
Q38_DEV uint32_t bf16_pair(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}
template <int B>
Q38_DEV float scale_byte(uint32_t e) {
    float r; /* (byte B << 23 in one operation; from C++ it is a shift and a mask) */
    static_assert(B >= 0 && B < 4, "a byte of a word");
    if (B == 0) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(23), "v"(e));
    if (B == 1) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(23), "v"(e));
    if (B == 2) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(23), "v"(e));
    if (B == 3) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(23), "v"(e));
    return r;
}

Q38_DEV float row_ror8(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));
}

/* The maximum over the four lanes of a column (l, l ^ 16, l ^ 32, l ^ 48). */
Q38_DEV float column_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const q38_halves h = q38_both_halves(x);
    return fmaxf(h.a, h.b);
}
Q38_DEV float column_sum(float x) {
    x = q38_pair_rows_sum(x);
    const q38_halves h = q38_both_halves(x);
    return h.a + h.b;
}

/* What a wave carries from page to page. */
struct State {
    float ref; /* column l % 16's reference, in log2 units */
    float l;   /* the sum of this lane's weights */
    int unit;   /* 8-bit rows: o is in units of 2^unit, in which a scaled weight fits f16 */
    float inv;  /* 2^-unit */
    f32x4 o[16]; /* o[n][i]: row 4 (l / 16) + i, dim 16 n + l % 16 */
};

template <int T>
Q38_DEV f32x4 mma_k(q38_u32x4 k, q38_u32x4 q, f32x4 c) {
    if (kInBf16<T>)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
}
template <int T>
Q38_DEV f32x4 mma_v(q38_u32x2 p, q38_u32x2 v, f32x4 c) {
    if (kInBf16<T>)
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, p), __builtin_bit_cast(s16x4, v), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, p), __builtin_bit_cast(f16x4, v), c, 0, 0, 0);
}

Q38_DEV uint32_t pack16(uint16_t lo, uint16_t hi) { return (uint32_t)hi << 16 | lo; }

/* Scores of a page's tokens, the softmax update, the weighted sum of its
 * values.  valid: tokens of the page that count (16 but for the sequence's
 * last page); first: nothing is summed yet. */
template <int T, bool kWeigh = false>
Q38_DEV void page_step(State &st, const Page<T> &p, const q38_u32x4 (*q)[8][64], float unscale, float above, int valid, bool first,
                       int lane, float *scores = nullptr) {
    const int c = lane & 15, g = lane >> 4;
    f32x4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
    /* the queries are read from LDS at every page: an index that the compiler
     * cannot see through keeps it from holding them in registers, 32 a part,
     * which the pages in flight need (8-bit pages leave room) */
    int ql = lane;
    if (T != Q38_KV_Q8) asm volatile("" : "+v"(ql));
    if (T == Q38_KV_Q8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const q38_u32x4 u = p.k[i];
            const q38_u32x4 a = {halves_of<0x04010400u>(u[0]), halves_of<0x04030402u>(u[0]), halves_of<0x04010400u>(u[1]),
                                 halves_of<0x04030402u>(u[1])};
            const q38_u32x4 b = {halves_of<0x04010400u>(u[2]), halves_of<0x04030402u>(u[2]), halves_of<0x04010400u>(u[3]),
                                 halves_of<0x04030402u>(u[3])};
            s0 = mma_k<T>(a, q[0][2 * i][ql], s0);
            s1 = mma_k<T>(b, q[0][2 * i + 1][ql], s1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f32x4 &s = T == Q38_KV_F16 && (i & 1) ? s1 : s0;
            s = mma_k<T>(p.k[i], q[0][i][ql], s);
            if (T == Q38_KV_BF16) s1 = mma_k<T>(p.k[i], q[1][i][ql], s1);
        }
    }
    float s[4];
    f32x4 ks = p.ks, vs = p.vs;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = s0[i] + s1[i];
        const float y = kInBf16<T> ? x : x * unscale;
        s[i] = y + row_ror8(y);
        if (T == Q38_KV_Q8) s[i] = s[i] * ks[i] * above;
        if (valid < 16 && 4 * g + i >= valid) {
            s[i] = -INFINITY;
            vs[i] = 0.0f;
        }
    }
    /* kept for the sums of weights, which need the whole context's maximum and sum first */
    if (kWeigh) put_scores<T>(scores, true, c, g, s);
    const float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
    auto scale_heads = [&](float f) { /* o by each head's factor */
        float fr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fr[i] = __shfl(f, 4 * g + i, 64);
#pragma unroll
        for (int n = 0; n < 16; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) st.o[n][i] *= fr[i];
    };
    float f = 1.0f;
    bool raised = __any(mx > st.ref + (kRefBelow<T> + kRefSlack));
    if (raised) {
        /* the page's maximum per head; heads that it does not raise keep theirs */
        const float top = column_max(mx) - kRefBelow<T>;
        const float ref = fmaxf(st.ref, top);
        f = st.ref == -INFINITY ? 0.0f : q38_exp2(st.ref - ref);
        st.l *= f;
        if (T == Q38_KV_Q8) {
            /* what o holds shrinks with the weights: its unit follows by whole
             * powers, the next above, and o is left up to twice as large */
            const float by = st.ref == -INFINITY ? 512.0f : fminf(ref - st.ref, 512.0f);
            const int unit = max(st.unit - (int)ceilf(by), kUnitMin);
            f = q38_exp2((float)(st.unit - unit) - by);
            st.unit = unit;
            st.inv = __builtin_amdgcn_ldexpf(1.0f, -unit);
        }
        st.ref = ref;
        if (T != Q38_KV_Q8 && !first) scale_heads(f);
    }
    float w[4], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = q38_exp2(s[i] - st.ref);
        sum += w[i];
    }
    st.l += sum;
    if (T == Q38_KV_Q8) {
        /* scales are signed (the largest value is quant -127).  A product past f32's
         * end raises the unit by 2^120, which leaves it 2^8 at least, and is looked
         * at once more; the second raise always does. */
        float x[4];
#pragma unroll
        for (int turn = 0;; ++turn) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = w[i] * st.inv * vs[i];
            const float big = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
            if (turn == 2 || !__any(big > kWeightedMax)) break;
            const int top = __builtin_amdgcn_frexp_expf(fminf(column_max(big), 0x1.fffffep127f));
            const int unit = min(st.unit + max(top - kWeightedBits, 0), kUnitMax);
            f = __builtin_amdgcn_ldexpf(f, st.unit - unit);
            raised = true;
            st.unit = unit;
            st.inv = __builtin_amdgcn_ldexpf(1.0f, -unit);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = x[i];
        /* once for both raises: two of these take registers that pages need */
        if (raised && !first) scale_heads(f);
    }

    /* the weights' parts: rows 0-5 the first (and, in a product of its own,
     * the third), rows 8-13 the second */
    q38_u32x2 a0, a1;
    const bool upper = c >= 8;
    if (kInBf16<T>) {
        uint32_t x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t hi = __float_as_uint(w[i]) & 0xFFFF0000u;
            const float r = w[i] - __uint_as_float(hi);
            const uint32_t mid = __float_as_uint(r) & 0xFFFF0000u;
            const float lo = r - __uint_as_float(mid);
            x[i] = upper ? mid : hi;
            y[i] = upper ? 0u : __float_as_uint(lo);
        }
        a0 = q38_u32x2{__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u)};
        a1 = q38_u32x2{__builtin_amdgcn_perm(y[1], y[0], 0x07060302u), __builtin_amdgcn_perm(y[3], y[2], 0x07060302u)};
    } else {
        uint16_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const _Float16 hi = (_Float16)w[i];
            const _Float16 lo = (_Float16)((w[i] - (float)hi) * kLowUnit<T>);
            x[i] = __builtin_bit_cast(uint16_t, upper ? lo : hi);
        }
        a0 = q38_u32x2{pack16(x[0], x[1]), pack16(x[2], x[3])};
    }
    /* values of tokens that do not count are cleared (8-bit ones are finite) */
    q38_u32x2 keep = {~0u, ~0u};
    if (T != Q38_KV_Q8 && valid < 16) {
        const int n = valid - 4 * g;
        keep = q38_u32x2{n <= 0 ? 0u : n == 1 ? 0xFFFFu : ~0u, n <= 2 ? 0u : n == 3 ? 0xFFFFu : ~0u};
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) {
        q38_u32x2 v;
        if (T == Q38_KV_Q8) {
            const uint32_t u = p.v[n >> 2][n & 3];
            v = q38_u32x2{halves_of<0x04010400u>(u), halves_of<0x04030402u>(u)};
        } else {
            v = q38_u32x2{p.v[n >> 1][2 * (n & 1)] & keep[0], p.v[n >> 1][2 * (n & 1) + 1] & keep[1]};
        }
        st.o[n] = mma_v<T>(a0, v, st.o[n]);
        if (T == Q38_KV_BF16) st.o[n] = mma_v<T>(a1, v, st.o[n]);
    }
}

/* The same for two pages of 4-bit rows at once, whose 32 tokens are the k of one
 * product: half the products of O, and one look at the running maxima for both.
 * valid: tokens of each that count; the bytes of the others are 0. */
Q38_DEV uint32_t upper_halves(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
template <bool kWeigh>
Q38_DEV void pair_step(State &st, const Page<Q38_KV_MX4> (&p)[2], const q38_u32x4 (*q)[8][64], int valid0, int valid1, bool first,
                       int lane, float *scores0, float *scores1) {
    constexpr int T = Q38_KV_MX4;
    const int c = lane & 15, g = lane >> 4;
    int ql = lane;
    asm volatile("" : "+v"(ql)); /* (as in page_step) */
    f32x4 s0[2] = {}, s1[2] = {};
    auto step = [&](auto b, int i) {
        constexpr int B = decltype(b)::value;
        const q38_u32x4 q0 = q[0][4 * i + B][ql], q1 = q[1][4 * i + B][ql];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t u = p[x].k[i][B];
            const float scale = scale_byte<B>(p[x].ks[i]);
            const q38_u32x4 a = {bf16_pair<0>(u, scale), bf16_pair<1>(u, scale), bf16_pair<2>(u, scale), bf16_pair<3>(u, scale)};
            s0[x] = mma_k<T>(a, q0, s0[x]);
            s1[x] = mma_k<T>(a, q1, s1[x]);
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        step(std::integral_constant<int, 0>(), i);
        step(std::integral_constant<int, 1>(), i);
        step(std::integral_constant<int, 2>(), i);
        step(std::integral_constant<int, 3>(), i);
    }
    float s[2][4];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y = s0[x][i] + s1[x][i];
            s[x][i] = y + row_ror8(y);
        }
    if (valid0 + valid1 < 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (4 * g + i >= valid0) s[0][i] = -INFINITY;
            if (4 * g + i >= valid1) s[1][i] = -INFINITY;
        }
    }
    if (kWeigh) {
        put_scores<T>(scores0, true, c, g, s[0]);
        put_scores<T>(scores1, valid1 > 0, c, g, s[1]);
    }
    const float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    if (__any(mx > st.ref + kRefSlack)) {
        const float ref = fmaxf(st.ref, column_max(mx));
        const float f = st.ref == -INFINITY ? 0.0f : q38_exp2(st.ref - ref);
        st.l *= f;
        st.ref = ref;
        if (!first) {
            float fr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) fr[i] = __shfl(f, 4 * g + i, 64);
#pragma unroll
            for (int n = 0; n < 16; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) st.o[n][i] *= fr[i];
        }
    }
    /* the weights' parts: rows 0-5 the first and, in a product of its own, the third, rows 8-13 the second */
    q38_u32x4 a0, a1;
    const bool upper = c >= 8;
    float sum = 0.0f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        float w[4], r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = q38_exp2(s[x][i] - st.ref);
            sum += e;
            const float rest = e - __uint_as_float(__float_as_uint(e) & 0xFFFF0000u);
            const float last = rest - __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
            w[i] = upper ? rest : e;
            r[i] = upper ? 0.0f : last;
        }
        a0[2 * x] = upper_halves(w[0], w[1]);
        a0[2 * x + 1] = upper_halves(w[2], w[3]);
        a1[2 * x] = upper_halves(r[0], r[1]);
        a1[2 * x + 1] = upper_halves(r[2], r[3]);
    }
    st.l += sum;
    /* a byte's two values are dims of two tiles: tokens are paired up for each */
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q38_u32x4 v0, v1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t u = p[x].v[i >> 2][i & 3], e = p[x].vs[i >> 2][i & 3];
            const uint32_t t0 = bf16_pair<0>(u, scale_byte<0>(e)), t1 = bf16_pair<1>(u, scale_byte<1>(e)),
                           t2 = bf16_pair<2>(u, scale_byte<2>(e)), t3 = bf16_pair<3>(u, scale_byte<3>(e));
            v0[2 * x] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
            v0[2 * x + 1] = __builtin_amdgcn_perm(t3, t2, 0x05040100u);
            v1[2 * x] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
            v1[2 * x + 1] = __builtin_amdgcn_perm(t3, t2, 0x07060302u);
        }
        st.o[2 * i] = mma_k<T>(a0, v0, st.o[2 * i]);
        st.o[2 * i + 1] = mma_k<T>(a0, v1, st.o[2 * i + 1]);
        st.o[2 * i] = mma_k<T>(a1, v0, st.o[2 * i]);
        st.o[2 * i + 1] = mma_k<T>(a1, v1, st.o[2 * i + 1]);
    }
}
/* The values of tokens from `valid` on as 0. */
Q38_DEV void clear_tail(Page<Q38_KV_MX4> &p, int valid, int lane) {
    const int n = min(max(valid - 4 * (lane >> 4), 0), 4);
    const uint32_t bytes = n == 4 ? ~0u : (1u << (8 * n)) - 1u;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            p.v[s][w] &= bytes;
            p.vs[s][w] &= bytes;
        }
}

/* The new token's rows in LDS as they are stored: the key's elements in order
 * of dims, the value's so that a lane's (dim 16 n + c for each tile n of one
 * load) lie in one word. */
struct NewRows {
    uint32_t k[Q38_ATTN_HEAD_DIM / 2], v[Q38_ATTN_HEAD_DIM / 2]; /* 16-bit elements, or bytes */
    float scale[2];
};
/* MXFP4: a row's codes, K as its 16-byte pieces and V a byte for each lane's pair of
 * dims and load, and its scale bytes. */
struct NewRowsMx4 {
    uint32_t k[Q38_ATTN_HEAD_DIM / 8], v[Q38_ATTN_HEAD_DIM / 8];
    uint8_t scale[2][8];
};
Q38_DEV int new_value_index_mx4(int d) { return ((d >> 7) * 16 + (d & 15)) * 4 + ((d >> 5) & 3); }
Q38_DEV int new_key_index_mx4(int d) { return (((d >> 7) * 4 + ((d >> 3) & 3)) * 4 + ((d >> 5) & 3)) * 4 + ((d & 7) >> 1); }
template <int T>
Q38_DEV int new_value_index(int d) {
    return T == Q38_KV_Q8 ? (d >> 6) * 64 + (d & 15) * 4 + ((d >> 4) & 3) : (d >> 5) * 32 + (d & 15) * 2 + ((d >> 4) & 1);
}

/* They take the place of token t in what the page held. */
template <int T>
Q38_DEV void put_new_token(Page<T> &p, const NewRows &row, int t, int lane) {
    const int c = lane & 15, g = lane >> 4;
    const bool key_lane = c == t, value_lane = g == (t >> 2);
    constexpr uint32_t kKeep = 0x07060504u; /* a word's own bytes */
#pragma unroll
    for (int s = 0; s < Page<T>::kLoads; ++s) {
        const q38_u32x4 kw = *reinterpret_cast<const q38_u32x4 *>(row.k + (s * 4 + g) * 4);
        if (key_lane) p.k[s] = kw;
        const uint32_t vw = row.v[s * 16 + c];
        if (T == Q38_KV_Q8) {
            const uint32_t sh = 8 * (t & 3);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t sel = (kKeep & ~(255u << sh)) | (uint32_t)w << sh;
                p.v[s][w] = __builtin_amdgcn_perm(p.v[s][w], vw, value_lane ? sel : kKeep);
            }
        } else {
            const uint32_t sh = 16 * (t & 1);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t sel = (kKeep & ~(0xFFFFu << sh)) | (w < 2 ? 0x0100u : 0x0302u) << sh;
                p.v[s][w] = __builtin_amdgcn_perm(p.v[s][w], vw, value_lane && ((t >> 1) & 1) == (w & 1) ? sel : kKeep);
            }
        }
    }
    if (T == Q38_KV_Q8) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (value_lane && (t & 3) == e) p.ks[e] = row.scale[0], p.vs[e] = row.scale[1];
    }
}

Q38_DEV void put_new_token(Page<Q38_KV_MX4> &p, const NewRowsMx4 &row, int t, int lane) {
    const int c = lane & 15, g = lane >> 4;
    const bool key_lane = c == t, value_lane = g == (t >> 2);
    const uint32_t sh = 8 * (t & 3);
    const q38_u32x2 ks = *reinterpret_cast<const q38_u32x2 *>(row.scale[0]), vs = *reinterpret_cast<const q38_u32x2 *>(row.scale[1]);
    if (key_lane) p.ks = ks;
    /* byte t % 4 of a word out of byte w of another */
    auto put = [&](uint32_t word, uint32_t from, int w) {
        const uint32_t sel = (0x07060504u & ~(255u << sh)) | (uint32_t)w << sh;
        return __builtin_amdgcn_perm(word, from, value_lane ? sel : 0x07060504u);
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const q38_u32x4 kw = *reinterpret_cast<const q38_u32x4 *>(row.k + (s * 4 + g) * 4);
        if (key_lane) p.k[s] = kw;
        const uint32_t vw = row.v[s * 16 + c];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            p.v[s][w] = put(p.v[s][w], vw, w);
            p.vs[s][w] = put(p.vs[s][w], vs[s], w);
        }
    }
}
/* Dims 4 lane .. + 3 of a key (which 0) or value to the page and to `row`. */
Q38_DEV void store_new_mx4(NewRowsMx4 &row, char *block, int j, int t, int which, int lane, f32x4 x) {
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) big = max(big, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    big = max(big, __float_as_uint(q38_row_move<0xB1>(__uint_as_float(big))));
    big = max(big, __float_as_uint(q38_row_move<0x4E>(__uint_as_float(big))));
    big = max(big, __float_as_uint(q38_row_move<0x141>(__uint_as_float(big)))); /* eight lanes hold a block */
    const uint32_t e = q38_mx4_exponent(big);
    const float scale = q38_mx4_power(e);
    const uint32_t code = q38_mx4_pack<1>(q38_mx4_pack<0>(0u, x[0], x[1], scale), x[2], x[3], scale);
    const int d = 4 * lane;
    if ((lane & 7) == 0) {
        row.scale[which][lane >> 3] = (uint8_t)e;
        q38_mx4_scales(block, j)[which ? q38_mx4_v_scale(t, d) : q38_mx4_k_scale(t, d)] = (uint8_t)e;
    }
    if (which == 0) {
        *reinterpret_cast<uint16_t *>(reinterpret_cast<char *>(row.k) + new_key_index_mx4(d)) = (uint16_t)code;
        *reinterpret_cast<uint16_t *>(block + (q38_k_index<Q38_KV_MX4>(t, d) >> 1)) = (uint16_t)code;
        return;
    }
    /* a byte holds dims 16 apart: the lane of the lower one puts it together */
    const uint32_t high = __shfl_xor(code, 4, 64);
    if (lane & 4) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint8_t b = (uint8_t)(((code >> (4 * i)) & 15u) | ((high >> (4 * i)) & 15u) << 4);
        reinterpret_cast<uint8_t *>(row.v)[new_value_index_mx4(d + i)] = b;
        reinterpret_cast<uint8_t *>(block)[q38_v_index<Q38_KV_MX4>(t, d + i) >> 1] = b;
    }
}

/* Workgroup barrier for LDS alone: loads of pages stay in flight across it
 * (__syncthreads() would wait for them). */
Q38_DEV void lds_barrier() { q38_barrier_vm<63>(); }

/* Dims 4 lane .. + 3 of column c's (and c + 8's) parts to the query operands:
 * operand i, lane 16 g + c holds the 8 dims that k step i's group g takes. */
template <int T>
Q38_DEV void store_query(q38_u32x4 (*q)[8][64], int c, int lane, f32x4 x) {
    const int d = 4 * lane;
    const int i = T == Q38_KV_Q8 ? 2 * (d >> 6) + ((d >> 3) & 1) : d >> 5;
    const int g = T == Q38_KV_Q8 ? (d >> 4) & 3 : (d >> 3) & 3;
    auto put = [&](int set, int col, const uint16_t (&e)[4]) {
        q38_u32x2 *at = reinterpret_cast<q38_u32x2 *>(&q[set][i][16 * g + col]) + ((d >> 2) & 1);
        *at = q38_u32x2{pack16(e[0], e[1]), pack16(e[2], e[3])};
    };
    uint16_t a[4], b[4], third[4], none[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (kInBf16<T>) {
            const uint32_t hi = __float_as_uint(x[e]) & 0xFFFF0000u;
            const float r = x[e] - __uint_as_float(hi);
            const uint32_t mid = __float_as_uint(r) & 0xFFFF0000u;
            a[e] = (uint16_t)(hi >> 16);
            b[e] = (uint16_t)(mid >> 16);
            third[e] = (uint16_t)(__float_as_uint(r - __uint_as_float(mid)) >> 16);
        } else {
            const _Float16 hi = (_Float16)x[e];
            a[e] = __builtin_bit_cast(uint16_t, hi);
            b[e] = __builtin_bit_cast(uint16_t, (_Float16)((x[e] - (float)hi) * kLowUnit<T>));
        }
    }
    put(0, c, a);
    put(0, c + 8, b);
    if (kInBf16<T>) {
        put(1, c, third);
        put(1, c + 8, none);
    }
}

/* The sequence of a split: b in the batch, its first split and their number. */
struct Where {
    int b, seq, pos, base, n;
};
/* One sequence's arguments under the names of a batch's. */
struct OneArgs {
    float *kpool, *vpool;
    const int32_t *page_table;
    const float *q, *k_new, *v_new, *gate;
    float *out, *part_o, *part_ml;
    const float *q_norm, *k_norm;
    float theta_scale;
    int32_t gate_head_stride, pos, split_tokens, total_splits;
    static constexpr int32_t pt_stride = 0;
};
Q38_DEV Where find(const OneArgs &a, int) { return {0, 0, a.pos, 0, a.total_splits}; }
Q38_DEV Where find(const q38_decode_typed_args &a, int g) {
    /* entries past n_seq are INT_MAX */
    int b = 0;
    for (int i0 = 1; i0 < a.n_seq; i0 += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) b += a.split_base[i0 + i] <= g ? 1 : 0;
    return {b, a.seq[b], a.pos[b], a.split_base[b], a.split_base[b + 1] - a.split_base[b]};
}

/* What the weights of six heads, of whose scores over the whole context top is the maximum and
 * inverse one over the sum, add to a split's n tokens.  pt: its first page's id;
 * last: the sequence's last position among them (past them where a later split has it), which a row
 * stored by the call starts anew as the sequence's token `token`. */
template <int kThreads>
Q38_DEV void add_weights(const float *top, const float *inverse, const float *scores, const int32_t *pt, float *weights, int32_t *tokens,
                         int n, int last, bool stored, int token) {
    for (int t = 4 * threadIdx.x; t < n; t += 4 * kThreads) {
        const float *sc = scores + (size_t)(t >> 4) * Q38_ATTN_KV_HEADS * Q38_SCORES_PAGE + (t & 15);
        const size_t at = (size_t)pt[t >> 4] * Q38_WEIGHTS_PAGE + (t & 15);
        f32x4 s[kGroup];
#pragma unroll
        for (int h = 0; h < kGroup; ++h) s[h] = q38_ld4(sc + h * Q38_PAGE_TOKENS);
        const f32x4 old = q38_ld4(weights + at);
        f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < kGroup; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_fmaf(q38_exp2(s[h][i] - top[h]), inverse[h], w[i]);
        if (t + 4 <= last) {
            q38_st4(weights + at, old + w);
            continue;
        }
        /* the last tokens: none behind the last, and a new one starts its sum */
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (t + i > last) break;
            const bool starts = t + i == last && stored;
            weights[at + i] = starts ? w[i] : old[i] + w[i];
            if (starts) tokens[at + i] = token;
        }
    }
}

/* Nothing beside the attention (q38_weigh_args: the scores too). */
struct NoSums {};

template <int T, bool kPre, typename Args, typename Sums = NoSums>
Q38_DEV void decode_typed(const Args &a, const Sums &sums = Sums()) {
    constexpr bool kWeigh = !std::is_same_v<Sums, NoSums>;
    constexpr int kQSets = kInBf16<T> ? 2 : 1;
    /* pages of a wave in registers: two 16-bit ones leave too few for the rest
     * (128K tokens 95 us against 85), 8-bit ones are half as large (1 / 2 / 3
     * pages: 49.9 / 47.5 / 48.8 us), 4-bit ones come in pairs (one / two of them:
     * 29.6 / 30.2) */
    constexpr int kDepth = T == Q38_KV_Q8 ? 2 : 1;
    constexpr int kPer = T == Q38_KV_MX4 ? 2 : 1; /* pages of a step */
    __shared__ q38_u32x4 q_frag[kQSets][8][64];
    __shared__ float q_unscale[8];
    __shared__ __attribute__((aligned(16))) std::conditional_t<T == Q38_KV_MX4, NewRowsMx4, NewRows> new_rows;
    __shared__ __attribute__((aligned(16))) float rope_cs[kPre ? kWaves : 1][32][2];
    __shared__ __attribute__((aligned(16))) float red_o[kWaves][kGroup][Q38_ATTN_HEAD_DIM];
    __shared__ __attribute__((aligned(16))) float red_m[8][kWaves], red_l[8][kWaves]; /* [column][wave] */
    __shared__ __attribute__((aligned(16))) float red_unit[8][kWaves]; /* of red_o */
    __shared__ float head_top[kGroup], head_inverse[kGroup]; /* over the whole context */
    static_assert(kWaves == 8 && kGroup == 6, "a wave per query head, one for the key and one for the value");

    const int g_split = blockIdx.x, j = blockIdx.y, tid = threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Where at_seq = find(a, g_split);
    const int b = at_seq.b, seq = at_seq.seq, pos = at_seq.pos, split = g_split - at_seq.base, nsplit = at_seq.n;
    const int t_begin = split * a.split_tokens, t_end = min(pos + 1, t_begin + a.split_tokens);
    const int n_pages = (t_end - t_begin + Q38_PAGE_TOKENS - 1) / Q38_PAGE_TOKENS;
    const bool has_pos = t_end == pos + 1;

    /* this wave's first page id through the scalar cache: as a vector load it
     * comes back to the workgroup's later waves behind the page loads of the
     * earlier ones (forming q and reading 1021 tokens took 9.6 us with it against
     * 9.75, Q8_K 10.0 against 10.1) */
    static_assert(Q38_MAX_SPLIT_TOKENS <= 64 * kWaves * Q38_PAGE_TOKENS, "a lane per page id");
    const int32_t *pt = a.page_table + (size_t)seq * a.pt_stride + (t_begin >> 4);
    const int first_page = pt[min(wave, n_pages - 1)];

    /* the rows that this wave forms: query head `wave`, or the new key or value */
    const int q_stride = kPre ? 2 * Q38_ATTN_HEAD_DIM : Q38_ATTN_HEAD_DIM;
    const bool forms_q = wave < kGroup;
    bool forms_new = false;
    /* (a wave that forms nothing loads head 0's) */
    const float *src = a.q + ((size_t)b * Q38_ATTN_HEADS + j * kGroup + (forms_q ? wave : 0)) * q_stride;
    const float *weight = a.q_norm;
    if (!forms_q) {
        /* (kept a branch: the other waves wait for none of these arguments) */
        asm volatile("");
        forms_new = a.k_new != nullptr && has_pos;
        if (forms_new) src = (wave == kGroup ? a.k_new : a.v_new) + (size_t)b * Q38_ATTN_KV_DIM + j * Q38_ATTN_HEAD_DIM;
        weight = a.k_norm;
    }
    f32x4 x = q38_ld4(src + 4 * lane), xw = {0.f, 0.f, 0.f, 0.f};
    if (kPre) xw = q38_ld4(weight + 4 * lane);
    __builtin_amdgcn_sched_barrier(0); /* on their way before the page id is waited for */
    /* the wave's first pages: no load from here to the first score sits under
     * a branch, so the rows above are waited for alone and the pages come in
     * while the queries are formed */
    Page<T> buf[kDepth][kPer];
    load_page<T>(buf[0][0], a, first_page, wave < n_pages, j, lane);
    /* all of its page ids, the i-th in lane i: pages wave, wave + 8, ... (64 of
     * them cover the largest split) */
    const int my_pages = pt[min(wave + kWaves * lane, n_pages - 1)];
    auto fetch = [&](Page<T> &p, int at) {
        load_page<T>(p, a, __builtin_amdgcn_readlane(my_pages, (at / kWaves) & 63), at < n_pages, j, lane);
    };
#pragma unroll
    for (int u = 1; u < kDepth * kPer; ++u) fetch(buf[u / kPer][u % kPer], wave + kWaves * u);

    if (kPre) {
        /* (every wave, so that the weights' load above stays before the pages':
         * under a branch it would sink into it) */
        int rope_pos = pos;
        if constexpr (kWeigh) rope_pos += sums.evicted[b];
        q38_rope_table_half(rope_cs[wave], lane & 31, rope_pos, a.theta_scale);
        /* the lanes read each other's entries below: LDS serves a wave in
         * order, the fence keeps the compiler to it */
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        f32x4 y = x;
        q38_norm_rope_row(y, xw, lane, rope_cs[wave]);
        if (wave <= kGroup) x = y; /* the value goes as it is */
    }
    if (forms_q) {
        x *= Q38_SCORE_LOG2;
        if (!kInBf16<T>) {
            float big = q38_max16(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
            big = column_max(big);
            /* exponent of the largest (129 at most, of infinity or NaN), kept where
             * 2^(10 - e) and its inverse are normal */
            const int e = max((int)(__float_as_uint(big) >> 23) - 126, -116);
            x *= __uint_as_float((uint32_t)(127 + 10 - e) << 23);
            if (lane == 0) q_unscale[wave] = __uint_as_float((uint32_t)(127 - 10 + e) << 23);
        }
        store_query<T>(q_frag, wave, lane, x);
    } else {
        store_query<T>(q_frag, wave, lane, f32x4{0.f, 0.f, 0.f, 0.f}); /* columns 6 and 7 */
        if (lane == 0) q_unscale[wave] = 1.0f;
        if (forms_new) {
            const int which = wave - kGroup;
            char *block = q38_kv_block<T>(which ? a.vpool : a.kpool, pt[(pos - t_begin) >> 4], j);
            const int t = pos & 15;
            if constexpr (T == Q38_KV_MX4) {
                store_new_mx4(new_rows, block, j, t, which, lane, x);
            } else {
                int qv[4] = {0, 0, 0, 0};
                float scale = 0.0f;
                if (T == Q38_KV_Q8) q38_wave_q8k(x, qv, scale);
                void *row = which ? new_rows.v : new_rows.k;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = 4 * lane + i;
                    const int to = which ? new_value_index<T>(d) : d;
                    const int at = which ? q38_v_index<T>(t, d) : q38_k_index<T>(t, d);
                    if (T == Q38_KV_Q8) {
                        static_cast<uint8_t *>(row)[to] = (uint8_t)(qv[i] + 128);
                        reinterpret_cast<uint8_t *>(block)[at] = (uint8_t)(qv[i] + 128);
                    } else {
                        static_cast<uint16_t *>(row)[to] = q38_to16<T>(x[i]);
                        reinterpret_cast<uint16_t *>(block)[at] = q38_to16<T>(x[i]);
                    }
                }
                if (T == Q38_KV_Q8 && lane == 0) {
                    new_rows.scale[which] = scale;
                    q38_kv_scales(block, j)[t] = scale;
                }
            }
        }
    }
    lds_barrier();
    const int c = lane & 15, g = lane >> 4;

    if (wave < n_pages) {
        /* the column's unit; 8-bit rows: one below 1 before the row's scale and one above after it (a query near f32's
         * end over small keys has products with its unit past that end, where the scores are not) */
        const float unit = q_unscale[c & 7], above = fmaxf(unit, 1.0f);
        const float unscale = (T == Q38_KV_Q8 ? fminf(unit, 1.0f) : unit) * (c < 8 ? 1.0f : 1.0f / kLowUnit<T>);
        State st;
        st.ref = -INFINITY;
        st.l = 0.0f;
        st.unit = kUnitMin;
        st.inv = __builtin_amdgcn_ldexpf(1.0f, -kUnitMin);
#pragma unroll
        for (int n = 0; n < 16; ++n) st.o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
        /* the only ways out are the gotos: a page's loads are behind the same
         * number of younger ones on every path, and are waited for alone */
        for (int i = wave;; i += kWaves * kDepth * kPer) {
#pragma unroll
            for (int u = 0; u < kDepth; ++u) {
                const int at = i + kWaves * kPer * u;
                if (at >= n_pages) goto done;
                float *scores = nullptr;
                if constexpr (kWeigh)
                    scores = sums.scores + (((size_t)g_split * (a.split_tokens >> 4) + at) * Q38_ATTN_KV_HEADS + j) * Q38_SCORES_PAGE;
                if constexpr (T == Q38_KV_MX4) {
                    int valid[2] = {Q38_PAGE_TOKENS, Q38_PAGE_TOKENS};
                    if (at + kWaves >= n_pages - 1) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const int page = at + kWaves * x;
                            if (page >= n_pages) valid[x] = 0; /* (it was loaded as zeros) */
                            if (page != n_pages - 1) continue;
                            valid[x] = t_end - t_begin - Q38_PAGE_TOKENS * page;
                            if (has_pos && a.k_new != nullptr) put_new_token(buf[u][x], new_rows, valid[x] - 1, lane);
                            clear_tail(buf[u][x], valid[x], lane);
                        }
                    }
                    pair_step<kWeigh>(st, buf[u], q_frag, valid[0], valid[1], at == wave, lane, scores,
                                      scores + kWaves * Q38_ATTN_KV_HEADS * Q38_SCORES_PAGE);
#pragma unroll
                    for (int x = 0; x < 2; ++x) fetch(buf[u][x], at + kWaves * (kPer * kDepth + x));
                } else {
                    int valid = Q38_PAGE_TOKENS;
                    if (at == n_pages - 1) {
                        valid = t_end - t_begin - Q38_PAGE_TOKENS * at;
                        if (has_pos && a.k_new != nullptr) put_new_token<T>(buf[u][0], new_rows, valid - 1, lane);
                    }
                    page_step<T, kWeigh>(st, buf[u][0], q_frag, unscale, above, valid, at == wave, lane, scores);
                    fetch(buf[u][0], at + kWaves * kDepth);
                }
            }
        }
    done:
        /* Both parts' rows added (lanes l and l ^ 32): exchanging tile n's upper
         * half for tile n + 1's lower one puts both tiles' pairs side by side, the
         * even tile's sums in the lower half of the wave, the odd one's in the
         * upper. */
        constexpr float kUnit = kInBf16<T> ? 1.0f : 0x1p-7f; /* 2^-kRefBelow */
        const float l = column_sum(st.l);
        if (lane < 8) {
            red_m[lane][wave] = st.ref + kRefBelow<T>;
            red_l[lane][wave] = l * kUnit;
            red_unit[lane][wave] = T == Q38_KV_Q8 ? __builtin_amdgcn_ldexpf(kUnit, st.unit) : kUnit;
        }
        float *out = &red_o[wave][4 * (g & 1)][16 * (g >> 1) + c];
#pragma unroll
        for (int n = 0; n < 16; n += 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(st.o[n][i]), __float_as_uint(st.o[n + 1][i]), false, false);
                if (i < 2 || (g & 1) == 0) /* heads 4 (g & 1) + i < 6 */
                    out[i * Q38_ATTN_HEAD_DIM + 16 * n] = __builtin_fmaf(__uint_as_float(r[1]), 1.0f / kLowUnit<T>, __uint_as_float(r[0]));
            }
        }
    }
    __syncthreads();

    /* a wave per head joins the waves' parts, lane l dims 4l .. 4l + 3 */
    if (wave >= kGroup && !(kWeigh && nsplit == 1)) return;
    if (wave < kGroup) {
        float M = -INFINITY, L = 0.0f;
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
        const int h = j * kGroup + wave;
        const size_t at = (size_t)h * Q38_ATTN_HEAD_DIM + 4 * lane;
        if (n_pages == 1) {
            M = red_m[wave][0];
            L = red_l[wave][0];
            O = q38_ld4(&red_o[0][wave][4 * lane]) * red_unit[wave][0];
        } else {
            float m[kWaves], f[kWaves];
            f32x4 o[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                m[w] = w < n_pages ? red_m[wave][w] : -INFINITY;
                o[w] = q38_ld4(&red_o[w][wave][4 * lane]);
                M = fmaxf(M, m[w]);
            }
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                f[w] = q38_exp2(m[w] - M);
                /* a wave without pages has left nothing there */
                L += w < n_pages ? red_l[wave][w] * f[w] : 0.0f;
                const float fu = f[w] * red_unit[wave][w];
#pragma unroll
                for (int e = 0; e < 4; ++e) O[e] = w < n_pages ? __builtin_fmaf(fu, o[w][e], O[e]) : O[e];
            }
        }
        if (nsplit == 1) {
            f32x4 r = O / L;
            if (a.gate != nullptr) {
                const f32x4 gate = q38_ld4(a.gate + ((size_t)b * Q38_ATTN_HEADS + h) * a.gate_head_stride + 4 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] *= q38_sigmoid(gate[e]);
            }
            q38_st4(a.out + (size_t)b * Q38_ATTN_Q_DIM + at, r);
            if (kWeigh && lane == 0) {
                head_top[wave] = M;
                head_inverse[wave] = 1.0f / L;
            }
        } else {
            q38_st4(a.part_o + (size_t)g_split * Q38_ATTN_Q_DIM + at, O);
            if (lane == 0) {
                a.part_ml[((size_t)g_split * Q38_ATTN_HEADS + h) * 2 + 0] = M;
                a.part_ml[((size_t)g_split * Q38_ATTN_HEADS + h) * 2 + 1] = L;
            }
        }
    }
    if constexpr (kWeigh) {
        if (nsplit != 1) return;
        /* the whole context: its sums without a second launch, once every wave's scores are stored */
        __builtin_amdgcn_s_waitcnt(0x0f70); /* vmcnt(0) */
        __syncthreads();
        const size_t head = (size_t)j * Q38_WEIGHTS_HEAD;
        add_weights<64 * kWaves>(head_top, head_inverse, sums.scores + ((size_t)g_split * (a.split_tokens >> 4) * Q38_ATTN_KV_HEADS + j) * Q38_SCORES_PAGE,
                                 pt, sums.weights + head, sums.tokens + head, t_end, pos, a.k_new != nullptr, pos + sums.evicted[b]);
    }
}

}  // namespace

/* name: a batch; name_one: one sequence; with pre, the pre step of full_core in the kernel. */
#define Q38_DECODE_KERNEL(name, T, PRE)                                                                             \
    extern "C" __global__ __launch_bounds__(64 * kWaves) void q38_attn_decode_##name(q38_decode_typed_args a) {     \
        decode_typed<T, PRE>(a);                                                                                    \
    }                                                                                                               \
    extern "C" __global__ __launch_bounds__(64 * kWaves) void q38_attn_decode_##name##_one(Q38_DECODE_ONE_PARAMS) { \
        decode_typed<T, PRE>(OneArgs{                                                                               \
            q38_global<float>(rows[2]), q38_global<float>(rows[3]), q38_global<const int32_t>(rows[0]),             \
            q38_global<const float>(rows[1]), rest.k_new, rest.v_new, rest.gate, rest.out, rest.part_o,             \
            rest.part_ml, q_norm, rest.k_norm, rest.theta_scale, span[3], span[0], span[1], span[2]});              \
    }
