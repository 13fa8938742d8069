/*
 * Rows of a ragged batch into and out of a typed cache's pages: the kernels of
 * kv_rows.hip (which says what they do and what they measured) and of
 * kv_rows_mxfp4.hip.
 */
#pragma once
#include "q38_kv_types.h"
#include "q38_rope.h"

namespace {

constexpr int kQuads = Q38_KV_ROWS_QUADS, kParts = Q38_KV_ROWS_PARTS;
constexpr int kThreads = 64 * Q38_ATTN_KV_HEADS * kQuads;
static_assert(kThreads == Q38_KV_ROWS_THREADS && 4 * kQuads * kParts == Q38_PAGE_TOKENS, "a wave per head and quad");

struct PageSpan {
    int t0, t1;   /* tokens of the page, [t0, t1) */
    int row0;     /* the batch's row of token t0 */
    int pos0;     /* and its position */
    int page;     /* physical page */
};

/* Page x of a batch: of the sequence whose rows from `first` on are n, whose
 * first row is `row`, first page page_base and page table starts at `table`. */
Q38_DEV PageSpan page_span(const int32_t *page_table, size_t table, int first, int n, int row, int page_base, int x) {
    const int lp = (first >> 4) + x - page_base;
    const int p0 = max(first, lp * Q38_PAGE_TOKENS);
    const int p1 = min(first + n, (lp + 1) * Q38_PAGE_TOKENS);
    return {p0 & 15, (p0 & 15) + p1 - p0, row + p0 - first, p0, page_table[table + lp]};
}
Q38_DEV PageSpan page_span(const q38_kv_rows_args &a, int x) {
    /* the sequence that holds page x: entries past n_seq are INT_MAX, so eight
     * are compared at a time, without a chain of dependent scalar loads */
    int b = 0;
    for (int i0 = 1; i0 < a.n_seq; i0 += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) b += a.page_base[i0 + i] <= x ? 1 : 0;
    return page_span(a.head.page_table, (size_t)a.seq[b] * a.head.pt_stride, a.pos0[b], a.row_base[b + 1] - a.row_base[b],
                     a.row_base[b], a.page_base[b], x);
}
Q38_DEV PageSpan page_span(const q38_kv_rows_few_args &a, int x) {
    int table = a.table[0], first = a.pos0[0], n = a.n_tokens[0], row = 0, page_base = 0;
    int pages = ((first + n - 1) >> 4) - (first >> 4) + 1;
    if (a.n_tokens[1] == 0) return page_span(a.head.page_table, (size_t)table, first, n, 0, 0, x);
#pragma unroll
    for (int i = 1; i < Q38_KV_ROWS_FEW; ++i) {
        const bool on = x >= page_base + pages; /* past the sequence before: never past the last */
        page_base += on ? pages : 0;
        row += on ? n : 0;
        table = on ? a.table[i] : table;
        first = on ? a.pos0[i] : first;
        n = on ? a.n_tokens[i] : n;
        pages = ((first + n - 1) >> 4) - (first >> 4) + 1;
    }
    return page_span(a.head.page_table, (size_t)table, first, n, row, page_base, x);
}

/* LDS of one wave: a quad's elements in page order, 16-bit (2 KiB) or 8-bit. */
typedef q38_u32x4 Stage[128];

/* The lanes of a wave read what others of it wrote: LDS serves a wave in
 * order, the fence keeps the compiler to it. */
Q38_DEV void stage_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

/* Place of (token i of the quad, dim d) in a stage, in elements: the page's
 * order with the other quads left out. */
template <int T>
Q38_DEV int stage_k(int i, int d) {
    if (T == Q38_KV_Q8) return ((d >> 4) * 4 + i) * 16 + (d & 15);
    if (T == Q38_KV_MX4) return (((d >> 7) * 4 + ((d >> 3) & 3)) * 4 + i) * 32 + ((d >> 5) & 3) * 8 + (d & 7);
    return ((d >> 3) * 4 + i) * 8 + (d & 7);
}
template <int T>
Q38_DEV int stage_v(int i, int d) {
    if (T == Q38_KV_Q8) return ((d >> 6) * 16 + (d & 15)) * 16 + ((d >> 4) & 3) * 4 + i;
    if (T == Q38_KV_MX4) return ((d >> 7) * 16 + (d & 15)) * 32 + ((d >> 5) & 3) * 8 + 2 * i + ((d >> 4) & 1);
    return ((d >> 5) * 16 + (d & 15)) * 8 + ((d >> 4) & 1) * 4 + i;
}
/* Piece p of a quad's stage in the block, in 16-byte pieces. */
Q38_DEV int piece_at(bool key, int quad, int p) {
    return key ? (p >> 2) * 16 + 4 * quad + (p & 3) : (p >> 4) * 64 + quad * 16 + (p & 15);
}

/* Four tokens' wave-wide sums or maxima at once: each step halves the values a
 * lane still carries, so that lane l ends with token l % 4's, in 7 operations
 * where four separate reductions take 24 -- and what follows (a division, a
 * root) is done once for all four. */
template <typename V, typename DPP1, typename DPP2, typename DPP4, typename DPP8, typename Join, typename Halves>
Q38_DEV V quad_reduce(const V (&s)[4], int lane, DPP1 xor1, DPP2 xor2, DPP4 by4, DPP8 ror8, Join join, Halves across) {
    const bool b0 = lane & 1, b1 = lane & 2;
    const V a = join(b0 ? s[1] : s[0], xor1(b0 ? s[0] : s[1]));
    const V c = join(b0 ? s[3] : s[2], xor1(b0 ? s[2] : s[3]));
    V r = join(b1 ? c : a, xor2(b1 ? a : c));
    r = join(r, by4(r));
    r = join(r, ror8(r));
    return across(r);
}
/* The sums are taken in q38_wave_sum_f64's order: a key's mean, and so its row, is
 * the same whichever kernel forms it. */
Q38_DEV double quad_sum_f64(const double (&s)[4], int lane) {
    return quad_reduce(
        s, lane, [](double x) { return q38_row_move_f64<0xB1>(x); }, [](double x) { return q38_row_move_f64<0x4E>(x); },
        [](double x) { return q38_row_xor4_f64(x); }, [](double x) { return q38_row_move_f64<0x128>(x); },
        [](double x, double y) { return x + y; },
        [](double x) { return q38_rows_sum_f64(x); });
}
Q38_DEV float quad_max(const float (&s)[4], int lane) {
    return quad_reduce(
        s, lane, [](float x) { return q38_row_move<0xB1>(x); }, [](float x) { return q38_row_move<0x4E>(x); },
        [](float x) { return q38_row_move<0x124>(x); }, [](float x) { return q38_row_move<0x128>(x); },
        [](float x, float y) { return fmaxf(x, y); },
        [](float x) {
            auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
            x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
            const q38_halves h = q38_both_halves(x);
            return fmaxf(h.a, h.b);
        });
}
/* Token i's value of one that lane l holds for token l % 4. */
Q38_DEV float quad_value(float x, int i) {
    return i == 0 ? q38_row_move<0x00>(x) : i == 1 ? q38_row_move<0x55>(x) : i == 2 ? q38_row_move<0xAA>(x) : q38_row_move<0xFF>(x);
}

/* RMSNorm and rotation of the quad's keys (q38_norm_rope4_cs, four at once).
 * Every f32 square is exact in f64, so a fused addition rounds as the plain one. */
Q38_DEV void norm_rope_quad(f32x4 (&x)[4], f32x4 w, int lane, const float (*cs)[32][2], const int (&t)[4]) {
    double ss[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ss[i] = (double)x[i].x * (double)x[i].x;
#pragma unroll
        for (int c = 1; c < 4; ++c) ss[i] = __builtin_fma((double)x[i][c], (double)x[i][c], ss[i]);
    }
    const float scale = q38_rms_scale_of(quad_sum_f64(ss, lane));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = x[i] * quad_value(scale, i) * w;
        q38_rope_row(x[i], lane, cs[t[i]]);
    }
}

/* The quad's Q8_K blocks (q38_wave_q8k, four at once): quants + 128 packed,
 * and in lane l token l % 4's scale. */
Q38_DEV float q8k_quad(const f32x4 (&x)[4], int lane, uint32_t (&b)[4]) {
    float up[4], down[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        up[i] = fmaxf(fmaxf(x[i].x, x[i].y), fmaxf(x[i].z, x[i].w));
        down[i] = fmaxf(fmaxf(-x[i].x, -x[i].y), fmaxf(-x[i].z, -x[i].w));
    }
    const float pos = quad_max(up, lane), neg = quad_max(down, lane);
    float m = pos > neg ? pos : -neg;
    if (__any(pos == neg && pos != 0.0f)) {
        /* the largest size with both signs: the first value of it decides */
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float big = quad_value(pos, i);
            const f32x4 v = x[i];
            const bool mine = fabsf(v.x) == big || fabsf(v.y) == big || fabsf(v.z) == big || fabsf(v.w) == big;
            const float cand = fabsf(v.x) == big ? v.x : fabsf(v.y) == big ? v.y : fabsf(v.z) == big ? v.z : v.w;
            const uint64_t holders = __ballot(mine);
            const float at = __uint_as_float(
                __builtin_amdgcn_readlane(__float_as_uint(cand), holders ? __builtin_ctzll(holders) : 0));
            if ((lane & 3) == i && pos == neg) m = at;
        }
    }
    const bool zero = pos == 0.0f && neg == 0.0f;
    const float inverse = zero ? 0.0f : -127.0f / m;
    const float scale = zero ? 0.0f : 1.0f / inverse;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float inv = quad_value(inverse, i);
        /* q38_nearest_int's sum holds the rounded quant in its low bits, and no
         * product rounds past 127 (|x| <= |m|), so its low byte is the quant;
         * plus 128 is the top bit turned.  (A block whose inverse scale
         * overflows gets 0, and has a scale of 0.) */
        uint32_t q[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) q[c] = __float_as_uint(inv * x[i][c] + 12582912.0f);
        b[i] = 0x80808080u ^ __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[3], q[2], 0x0C0C0400u),
                                                   __builtin_amdgcn_perm(q[1], q[0], 0x0C0C0400u), 0x05040100u);
    }
    return scale;
}

/* The quad's MXFP4 blocks: the codes of each token's four values, lowest first, in
 * 16 bits, and the scale byte of each token's block of 32 (8 lanes hold one). */
Q38_DEV void mx4_quad(const f32x4 (&x)[4], uint32_t (&code)[4], uint32_t (&e)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        /* sizes compared by their bits, where a NaN is larger than any number */
        auto bits = [&](int c) { return __float_as_uint(x[i][c]) & 0x7FFFFFFFu; };
        uint32_t big = max(max(bits(0), bits(1)), max(bits(2), bits(3)));
        big = max(big, __float_as_uint(q38_row_move<0xB1>(__uint_as_float(big))));
        big = max(big, __float_as_uint(q38_row_move<0x4E>(__uint_as_float(big))));
        big = max(big, __float_as_uint(q38_row_move<0x141>(__uint_as_float(big)))); /* the other four of the eight */
        e[i] = q38_mx4_exponent(big);
        const float scale = q38_mx4_power(e[i]);
        code[i] = q38_mx4_pack<1>(q38_mx4_pack<0>(0u, x[i][0], x[i][1], scale), x[i][2], x[i][3], scale);
    }
}
Q38_DEV void store_quad_mx4(char *block, Stage &stage, bool key, int head, int quad, int first, int last, int lane,
                            const f32x4 (&x)[4]) {
    constexpr int kPieces = 32;
    uint32_t code[4], e[4];
    mx4_quad(x, code, e);
    uint8_t *scales = q38_mx4_scales(block, head);
    const int mine = lane & 7; /* the token whose scale this lane stores, of 32 dims that its eight hold */
    if (mine >= first && mine < last) {
        const int t = 4 * quad + mine, d = 4 * lane;
        scales[key ? q38_mx4_k_scale(t, d) : q38_mx4_v_scale(t, d)] =
            (uint8_t)(mine == 0 ? e[0] : mine == 1 ? e[1] : mine == 2 ? e[2] : e[3]);
    }
    q38_u32x4 *out = reinterpret_cast<q38_u32x4 *>(block);
    char *at = reinterpret_cast<char *>(stage);
    if (key) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint16_t *>(at + stage_k<Q38_KV_MX4>(i, 4 * lane) / 2) = (uint16_t)code[i];
        stage_fence();
        if (lane < kPieces && (lane & 3) >= first && (lane & 3) < last) out[piece_at(true, quad, lane)] = stage[lane];
        return;
    }
    /* dims 16 apart share a byte: lanes 4 apart hold them, and each puts two of
     * their four dims together, all four tokens of one in a word */
    const bool upper = lane & 4;
    const uint32_t a01 = code[0] | code[1] << 16, a23 = code[2] | code[3] << 16;
    const uint32_t b01 = __shfl_xor(a01, 4, 64), b23 = __shfl_xor(a23, 4, 64);
    const uint32_t low01 = upper ? b01 : a01, low23 = upper ? b23 : a23, high01 = upper ? a01 : b01, high23 = upper ? a23 : b23;
    const int d0 = 32 * (lane >> 3) + 4 * (lane & 3);
    uint32_t word[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int sh = 4 * (upper ? 2 + k : k);
        const uint32_t x01 = ((low01 >> sh) & 0x000F000Fu) | ((high01 >> sh) & 0x000F000Fu) << 4;
        const uint32_t x23 = ((low23 >> sh) & 0x000F000Fu) | ((high23 >> sh) & 0x000F000Fu) << 4;
        word[k] = __builtin_amdgcn_perm(x23, x01, 0x06040200u);
    }
    if (first == 0 && last == 4) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            *reinterpret_cast<uint32_t *>(at + stage_v<Q38_KV_MX4>(0, d0 + (upper ? 2 : 0) + k) / 2) = word[k];
        stage_fence();
        if (lane < kPieces) out[piece_at(false, quad, lane)] = stage[lane];
        return;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i >= first && i < last)
                reinterpret_cast<uint8_t *>(block)[q38_v_index<Q38_KV_MX4>(4 * quad + i, d0 + (upper ? 2 : 0) + k) / 2] =
                    (uint8_t)(word[k] >> (8 * i));
}

template <int T>
Q38_DEV void store_quad(char *block, Stage &stage, bool key, int head, int quad, int first, int last, int lane, const f32x4 (&x)[4]) {
    /* tokens first .. last - 1 of the quad are the batch's */
    if constexpr (T == Q38_KV_MX4) {
        store_quad_mx4(block, stage, key, head, quad, first, last, lane, x);
        return;
    }
    if (T == Q38_KV_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i >= first && i < last)
                q38_st4(reinterpret_cast<float *>(block) + q38_k_index<T>(4 * quad + i, 4 * lane), x[i]);
        return;
    }
    uint32_t b[4][T == Q38_KV_Q8 ? 1 : 2]; /* token i's four elements */
    if (T == Q38_KV_Q8) {
        uint32_t q[4];
        const float scale = q8k_quad(x, lane, q);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i][0] = q[i];
        if (lane >= first && lane < last) q38_kv_scales(block, head)[4 * quad + lane] = scale;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                b[i][T == Q38_KV_Q8 ? 0 : h] =
                    (uint32_t)q38_to16<T>(x[i][2 * h]) | (uint32_t)q38_to16<T>(x[i][2 * h + 1]) << 16;
    }
    constexpr int kPieces = T == Q38_KV_Q8 ? 64 : 128;
    q38_u32x4 *out = reinterpret_cast<q38_u32x4 *>(block);
    if (key) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t *at = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(stage) +
                                                        stage_k<T>(i, 4 * lane) * (T == Q38_KV_Q8 ? 1 : 2));
            at[0] = b[i][0];
            if (T != Q38_KV_Q8) at[1] = b[i][T == Q38_KV_Q8 ? 0 : 1];
        }
        stage_fence();
#pragma unroll
        for (int p = lane; p < kPieces; p += 64)
            if ((p & 3) >= first && (p & 3) < last) out[piece_at(true, quad, p)] = stage[p];
        return;
    }
    /* the four tokens of each dim side by side */
    if (first == 0 && last == 4) {
        if (T == Q38_KV_Q8) {
            const uint32_t lo = __builtin_amdgcn_perm(b[1][0], b[0][0], 0x05010400u); /* dims 0, 1 of tokens 0, 1 */
            const uint32_t hi = __builtin_amdgcn_perm(b[1][0], b[0][0], 0x07030602u); /* dims 2, 3 */
            const uint32_t lo2 = __builtin_amdgcn_perm(b[3][0], b[2][0], 0x05010400u);
            const uint32_t hi2 = __builtin_amdgcn_perm(b[3][0], b[2][0], 0x07030602u);
            const uint32_t w[4] = {__builtin_amdgcn_perm(lo2, lo, 0x05040100u), __builtin_amdgcn_perm(lo2, lo, 0x07060302u),
                                   __builtin_amdgcn_perm(hi2, hi, 0x05040100u), __builtin_amdgcn_perm(hi2, hi, 0x07060302u)};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                *reinterpret_cast<uint32_t *>(reinterpret_cast<char *>(stage) + stage_v<T>(0, 4 * lane + c)) = w[c];
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int h = T == Q38_KV_Q8 ? 0 : c >> 1;
                const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
                q38_u32x2 w = {__builtin_amdgcn_perm(b[1][h], b[0][h], sel), __builtin_amdgcn_perm(b[3][h], b[2][h], sel)};
                *reinterpret_cast<q38_u32x2 *>(reinterpret_cast<char *>(stage) + 2 * stage_v<T>(0, 4 * lane + c)) = w;
            }
        }
        stage_fence();
#pragma unroll
        for (int p = lane; p < kPieces; p += 64) out[piece_at(false, quad, p)] = stage[p];
        return;
    }
    /* a quad that the batch holds in part: its own elements only */
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i < first || i >= last) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int at = q38_v_index<T>(4 * quad + i, 4 * lane + c);
            if (T == Q38_KV_Q8)
                reinterpret_cast<uint8_t *>(block)[at] = (uint8_t)(b[i][0] >> (8 * c));
            else
                reinterpret_cast<uint16_t *>(block)[at] = (uint16_t)(b[i][T == Q38_KV_Q8 ? 0 : c >> 1] >> (16 * (c & 1)));
        }
    }
}

template <int T, typename Args>
Q38_DEV void kv_append(const Args &a) {
    __shared__ __attribute__((aligned(16))) float cs[4 * kQuads][32][2];
    __shared__ Stage stages[T == Q38_KV_F32 ? 1 : kThreads / 64];
    const PageSpan sp = page_span(a, blockIdx.x / kParts);
    const int quad0 = blockIdx.x % kParts * kQuads;
    const bool key = blockIdx.y == 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int head = wave & 3, quad = quad0 + (wave >> 2);
    const bool turns = key && a.head.k_norm != nullptr;
    const int first = max(sp.t0 - 4 * quad, 0), last = min(sp.t1 - 4 * quad, 4);
    const bool live = first < last;
    const float *rows = static_cast<const float *>(key ? a.head.k_rows : a.head.v_rows) +
                        (size_t)sp.row0 * Q38_ATTN_KV_DIM + head * Q38_ATTN_HEAD_DIM + 4 * lane;
    f32x4 x[4], w = {0.f, 0.f, 0.f, 0.f};
    if (live) {
        /* a token that is not the batch's loads a neighbour's row, and is not stored */
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = q38_ld4_stream(rows + (size_t)(4 * quad + min(max(i, first), last - 1) - sp.t0) * Q38_ATTN_KV_DIM);
        if (turns) w = q38_ld4(a.head.k_norm + 4 * lane);
    }
    if (turns) {
        /* the page's angles: a half-wave per token */
        const int t = 4 * quad0 + (tid >> 5);
        if (tid < 128 * kQuads && t >= sp.t0 && t < sp.t1)
            q38_rope_table_half(cs[tid >> 5], lane & 31, sp.pos0 + t - sp.t0, a.head.theta_scale);
        __syncthreads();
    }
    if (!live) return;
    if (turns) {
        int t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = 4 * (wave >> 2) + min(max(i, first), last - 1);
        norm_rope_quad(x, w, lane, cs, t);
    }
    store_quad<T>(q38_kv_block<T>(key ? a.head.kpool : a.head.vpool, sp.page, head), stages[T == Q38_KV_F32 ? 0 : wave], key, head,
                  quad, first, last, lane, x);
}

/* OUT16: rows in the cache's 16 bits, moved as they are (T is BF16 for both).
 * The rows leave for a reader elsewhere, by non-temporal stores: 4096 tokens of
 * Q8_K 8.3 us against 11.3, 1531 of BF16 6.3 against 8.7, as they are stored 6.1
 * against 7.2 (a kernel that reads 4096 of them at once takes 1.2 us longer for
 * it).  The append's pages stay in the caches for the call that reads them next:
 * stored past them they cost 9.0 us instead of 9.9, and the gather after it 2
 * more. */
template <int T, bool OUT16, typename Args>
Q38_DEV void kv_gather(const Args &a) {
    __shared__ Stage stages[T == Q38_KV_F32 ? 1 : kThreads / 64];
    const PageSpan sp = page_span(a, blockIdx.x / kParts);
    const int quad0 = blockIdx.x % kParts * kQuads;
    const bool key = blockIdx.y == 0;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int head = wave & 3, quad = quad0 + (wave >> 2);
    const int first = max(sp.t0 - 4 * quad, 0), last = min(sp.t1 - 4 * quad, 4);
    if (first >= last) return;
    char *block = q38_kv_block<T>(key ? a.head.kpool : a.head.vpool, sp.page, head);
    const size_t row = (size_t)(sp.row0 + 4 * quad - sp.t0) * Q38_ATTN_KV_DIM + head * Q38_ATTN_HEAD_DIM + 4 * lane;
    void *rows = key ? a.head.k_rows : a.head.v_rows;
    f32x4 x[4];
    q38_u32x2 raw[4];
    if constexpr (T == Q38_KV_MX4) {
        q38_u32x4 *stage = stages[wave];
        const uint8_t *scales = q38_mx4_scales(block, head);
        uint32_t e[4];
        /* the last lanes load the first ones' pieces again */
        const q38_u32x4 piece = reinterpret_cast<const q38_u32x4 *>(block)[piece_at(key, quad, lane & 31)];
        if (key) {
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = scales[q38_mx4_k_scale(4 * quad + i, 4 * lane)];
        } else {
            const uint32_t u = *reinterpret_cast<const uint32_t *>(scales + q38_mx4_v_scale(4 * quad, 4 * lane));
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = (u >> (8 * i)) & 255u;
        }
        stage[lane & 31] = piece;
        stage_fence();
        const char *at = reinterpret_cast<const char *>(stage);
        uint32_t lo[4], hi[4]; /* byte i % 4 .. of token i: dims 0, 1 and 2, 3 */
        if (key) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = *reinterpret_cast<const uint16_t *>(at + stage_k<T>(i, 4 * lane) / 2);
                lo[i] = u;
                hi[i] = u >> 8;
            }
        } else {
            uint32_t u[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                u[c] = (*reinterpret_cast<const uint32_t *>(at + (stage_v<T>(0, 4 * lane + c) & ~1) / 2) >> (lane & 4)) & 0x0F0F0F0Fu;
            const uint32_t p01 = u[0] | u[1] << 4, p23 = u[2] | u[3] << 4; /* byte i: token i's */
#pragma unroll
            for (int i = 0; i < 4; ++i) lo[i] = p01 >> (8 * i), hi[i] = p23 >> (8 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float s = q38_mx4_power(e[i]);
            const q38_f32x2 a = q38_mx4_pair<0>(lo[i], s), b = q38_mx4_pair<0>(hi[i], s);
            x[i] = f32x4{a[0], a[1], b[0], b[1]};
        }
    } else if (T == Q38_KV_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = q38_ld4(reinterpret_cast<const float *>(block) + q38_k_index<T>(4 * quad + i, 4 * lane));
    } else {
        constexpr int kPieces = T == Q38_KV_Q8 ? 64 : 128;
        q38_u32x4 *stage = stages[T == Q38_KV_F32 ? 0 : wave];
        const q38_u32x4 *in = reinterpret_cast<const q38_u32x4 *>(block);
        q38_u32x4 piece[kPieces / 64];
        f32x4 scale = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kPieces / 64; ++k) piece[k] = in[piece_at(key, quad, lane + 64 * k)];
        if (T == Q38_KV_Q8) scale = q38_ld4(q38_kv_scales(block, head) + 4 * quad);
#pragma unroll
        for (int k = 0; k < kPieces / 64; ++k) stage[lane + 64 * k] = piece[k];
        stage_fence();
        const char *at = reinterpret_cast<const char *>(stage);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t e[4]; /* the token's four elements */
            if (key) {
                if (T == Q38_KV_Q8) {
                    const uint32_t u = *reinterpret_cast<const uint32_t *>(at + stage_k<T>(i, 4 * lane));
#pragma unroll
                    for (int c = 0; c < 4; ++c) e[c] = (u >> (8 * c)) & 255u;
                } else {
                    const q38_u32x2 u = *reinterpret_cast<const q38_u32x2 *>(at + 2 * stage_k<T>(i, 4 * lane));
#pragma unroll
                    for (int c = 0; c < 4; ++c) e[c] = (u[c >> 1] >> (16 * (c & 1))) & 0xFFFFu;
                }
            } else {
                /* the dim's four tokens in one read; the compiler keeps it for all i */
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (T == Q38_KV_Q8) {
                        const uint32_t u = *reinterpret_cast<const uint32_t *>(at + stage_v<T>(0, 4 * lane + c));
                        e[c] = (u >> (8 * i)) & 255u;
                    } else {
                        const q38_u32x2 u = *reinterpret_cast<const q38_u32x2 *>(at + 2 * stage_v<T>(0, 4 * lane + c));
                        e[c] = (u[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
                    }
                }
            }
            raw[i] = q38_u32x2{e[0] | e[1] << 16, e[2] | e[3] << 16};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                x[i][c] = T == Q38_KV_Q8 ? (float)((int)e[c] - 128) * scale[i] : q38_from16<T>((uint16_t)e[c]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i < first || i >= last) continue;
        if (OUT16)
            __builtin_nontemporal_store(raw[i], reinterpret_cast<q38_u32x2 *>(static_cast<uint16_t *>(rows) + row +
                                                                              (size_t)i * Q38_ATTN_KV_DIM));
        else
            q38_st4_stream(static_cast<float *>(rows) + row + (size_t)i * Q38_ATTN_KV_DIM, x[i]);
    }
}

}  // namespace

#define Q38_KV_APPEND_KERNEL(name, T)                                                                            \
    extern "C" __global__ __launch_bounds__(kThreads) void name(q38_kv_rows_args a) { kv_append<T>(a); }         \
    extern "C" __global__ __launch_bounds__(kThreads) void name##_few(q38_kv_rows_few_args a) { kv_append<T>(a); }
#define Q38_KV_GATHER_KERNEL(name, T, OUT16)                                                                     \
    extern "C" __global__ __launch_bounds__(kThreads) void name(q38_kv_rows_args a) { kv_gather<T, OUT16>(a); }  \
    extern "C" __global__ __launch_bounds__(kThreads) void name##_few(Q38_KV_GATHER_FEW_PARAMS) {                \
        kv_gather<T, OUT16>(                                                                                     \
            q38_kv_rows_few_args{{rest.kpool, rest.vpool, page_table, rest.k_rows, rest.v_rows, nullptr, 0.f, 0}, \
                                 {table[0], table[1], table[2], table[3]},                                  \
                                 {pos0[0], pos0[1], pos0[2], pos0[3]},                                           \
                                 {n_tokens[0], n_tokens[1], n_tokens[2], n_tokens[3]}});                         \
    }
