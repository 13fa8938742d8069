/*
 * The attention weights that a run of a prompt's queries gives to the cached
 * tokens, added to the sums of a tracking cache.
 *
 * Query u (position base_pos + u) sees positions up to its own: token t of a kv
 * head takes W[t] += sum_u sum_h exp2(s_uht - M_uh) / L_uh over the group's heads
 * h.  M and L need every position first: the first launch forms the scores and leaves
 * each column's (a query's head) maximum and sum over a split of the positions, the
 * second joins the splits' and adds.  A short context's scores are kept for it, 24 f32
 * a query and token; over a longer one they would write and read several times the bytes that the
 * keys have, and it forms them again on the matrix unit (q38_attn_observe in the host's
 * code has both sides' times).
 *
 * S^T = K Q^T as in the decode (q38_decode_typed.h: a cached value is an operand
 * as it stands, a query is split into parts whose sum it is), but with 16 real
 * columns a product.  f16 operands take a query's two parts (22 bits), bf16 ones
 * three, which are all of its 24 bits; two of them, rounded to nearest, leave 2^-16
 * of a query, and over scores of 60 some 3e-4 of a weight: only where the caller asks
 * for them (q38_set_observe_parts).
 * A workgroup keeps the parts of 16 queries' 96 columns in LDS; a wave holds kPages
 * pages of keys as operands and reads each part once for all of them (one page where it keeps
 * scores).  Groups of queries come one after the other in a workgroup of the second
 * launch, so that every sum has one owner and a fixed order.
 *
 * Measured: 32 queries over 32K tokens of MXFP4, formed twice, 34.1 us for the statistics
 * and 43.5 for the sums (26.6 and 33.4 with two parts).  The products of three parts are 38.7
 * GFLOP a launch, which keep the matrix unit busy for 3.775e7 cycles, 15 us on 1024 SIMDs: 45
 * and 35% (the keys, 19 MB, would take 3).  The rest is the vector unit's masks, exponentials and
 * sums over columns, 68 and 82 instructions a page and tile beside 24 products, and the
 * parts' way from LDS: the branches at each tile keep one tile's products from
 * running beside the exponentials of the one before.  7 queries over
 * 1000 tokens of bf16, scores kept, 8.1 and 3.5: 32 workgroups, a wave a page, bound by the
 * chains queries - parts in LDS - keys - join and scores - join - sums.
 */
#include "q38_decode_typed.h"

namespace {

constexpr int kTiles = Q38_OBSERVE_COLS / 16;
template <int T>
constexpr int kPagesOf = T == Q38_KV_Q8 ? Q38_OBSERVE_PAGES_Q8 : Q38_OBSERVE_PAGES;
static_assert(kTiles * 16 == Q38_OBSERVE_COLS, "whole tiles");

/* A step's operand of a tile, its four groups of 16 lanes 16 bytes further apart than
 * they are long: a wave stores one column of every step and group at once, which
 * would all lie in two banks. */
typedef q38_u32x4 Step[4][17];
template <int kParts>
struct Queries {
    Step part[kTiles][kParts][8];
    float unscale[Q38_OBSERVE_COLS];
};

/* Tiles of a group that hold a query. */
Q38_DEV int tiles_of(const q38_observe_args &a, int group) {
    return (min(a.n_tokens - group * Q38_OBSERVE_QUERIES, Q38_OBSERVE_QUERIES) * kGroup + 15) >> 4;
}

/* The group's queries as operands: columns 6 u + h, zero past the last query. */
template <int T, int kParts>
Q38_DEV void load_queries(Queries<kParts> &q, const q38_observe_args &a, int group, int j, int lane, int wave) {
    const int d = 4 * lane;
    const int i = T == Q38_KV_Q8 ? 2 * (d >> 6) + ((d >> 3) & 1) : d >> 5;
    const int g = T == Q38_KV_Q8 ? (d >> 4) & 3 : (d >> 3) & 3;
    constexpr int kRows = Q38_OBSERVE_COLS / kWaves;
    const int rows = tiles_of(a, group) * 16 / kWaves; /* of tiles that hold a query */
    f32x4 x[kRows];
#pragma unroll
    for (int n = 0; n < kRows; ++n) { /* (a branch a load would hold the loads up) */
        const int col = n * kWaves + wave, u = group * Q38_OBSERVE_QUERIES + col / kGroup, h = j * kGroup + col % kGroup;
        x[n] = q38_ld4(a.q + ((size_t)min(u, a.n_tokens - 1) * Q38_ATTN_HEADS + h) * Q38_ATTN_HEAD_DIM + d);
        if (u >= a.n_tokens) x[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int n = 0; n < kRows; ++n) {
        if (n >= rows) continue;
        const int col = n * kWaves + wave;
        f32x4 y = x[n] * Q38_SCORE_LOG2;
        float unscale = 1.0f;
        if (!kInBf16<T>) {
            /* as the decode scales a head: its largest value to 2^9..10 */
            const float big = column_max(q38_max16(fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)))));
            const int e = max((int)(__float_as_uint(big) >> 23) - 126, -116);
            y *= __uint_as_float((uint32_t)(127 + 10 - e) << 23);
            unscale = __uint_as_float((uint32_t)(127 - 10 + e) << 23);
        }
        if (lane == 0) q.unscale[col] = unscale;
        uint16_t p[kParts][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (kInBf16<T>) {
                float rest = y[e];
#pragma unroll
                for (int k = 0; k < kParts; ++k) {
                    const __bf16 part = (__bf16)rest;
                    p[k][e] = __builtin_bit_cast(uint16_t, part);
                    rest -= (float)part;
                }
            } else {
                const _Float16 hi = (_Float16)y[e];
                p[0][e] = __builtin_bit_cast(uint16_t, hi);
                p[1][e] = __builtin_bit_cast(uint16_t, (_Float16)((y[e] - (float)hi) * kLowUnit<T>));
            }
        }
#pragma unroll
        for (int k = 0; k < kParts; ++k)
            *(reinterpret_cast<q38_u32x2 *>(&q.part[col >> 4][k][i][g][col & 15]) + ((d >> 2) & 1)) =
                q38_u32x2{pack16(p[k][0], p[k][1]), pack16(p[k][2], p[k][3])};
    }
}

/* A page's keys as operands, and 8-bit rows' scales of tokens 4 (lane / 16) .. + 3. */
struct Keys {
    q38_u32x4 a[8];
    f32x4 scale;
};
template <int T>
Q38_DEV void load_keys(Keys &k, const char *kpool, int page, int j, int lane) {
    char *block = q38_kv_block<T>(const_cast<char *>(kpool), page, j);
    const q38_u32x4 *in = reinterpret_cast<const q38_u32x4 *>(block) + lane;
    if constexpr (T == Q38_KV_MX4) {
        const q38_u32x4 u[2] = {in[0], in[64]};
        const q38_u32x2 s = *reinterpret_cast<const q38_u32x2 *>(q38_mx4_scales(block, j) + 8 * (lane & 15));
        auto step = [&](uint32_t codes, float scale) {
            return q38_u32x4{bf16_pair<0>(codes, scale), bf16_pair<1>(codes, scale), bf16_pair<2>(codes, scale), bf16_pair<3>(codes, scale)};
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            k.a[4 * i] = step(u[i][0], scale_byte<0>(s[i]));
            k.a[4 * i + 1] = step(u[i][1], scale_byte<1>(s[i]));
            k.a[4 * i + 2] = step(u[i][2], scale_byte<2>(s[i]));
            k.a[4 * i + 3] = step(u[i][3], scale_byte<3>(s[i]));
        }
    } else if constexpr (T == Q38_KV_Q8) {
        q38_u32x4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = in[64 * i];
        k.scale = q38_ld4(q38_kv_scales(block, j) + 4 * (lane >> 4));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = u[i >> 1][2 * (i & 1)], y = u[i >> 1][2 * (i & 1) + 1];
            k.a[i] = q38_u32x4{halves_of<0x04010400u>(x), halves_of<0x04030402u>(x), halves_of<0x04010400u>(y), halves_of<0x04030402u>(y)};
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) k.a[i] = in[64 * i];
    }
}

/* Scores (log2 units) less `base` of kPages pages against a tile's 16 columns.
 * bf16 operands: all parts' products go into one sum that starts at -base. */
template <int T, int kPages, int kParts>
Q38_DEV void scores_of(const Keys (&k)[kPages], const Step (&part)[kParts][8], float unscale, float base, int lane, float (&s)[kPages][4]) {
    /* (an index that the compiler cannot see through: it would keep the parts of
     * all tiles in registers over the loop of pages) */
    asm volatile("" : "+v"(lane));
    constexpr int kSums = kInBf16<T> ? 1 : 2;
    const float first = kInBf16<T> ? -base : 0.0f;
    /* 8-bit rows: a query's unit below 1 before the row's scale and one above after it, as their product may pass f32's
     * end where the score does not */
    const float below = fminf(unscale, 1.0f), above = fmaxf(unscale, 1.0f);
    f32x4 c[kPages][kSums];
#pragma unroll
    for (int p = 0; p < kPages; ++p)
#pragma unroll
        for (int n = 0; n < kSums; ++n) c[p][n] = f32x4{first, first, first, first};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int n = 0; n < kParts; ++n) {
            const q38_u32x4 q = part[n][i][0][lane + (lane >> 4)];
#pragma unroll
            for (int p = 0; p < kPages; ++p) c[p][n % kSums] = mma_k<T>(k[p].a[i], q, c[p][n % kSums]);
        }
#pragma unroll
    for (int p = 0; p < kPages; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kInBf16<T>) {
                s[p][i] = c[p][0][i];
            } else {
                const float x = __builtin_fmaf(c[p][kSums - 1][i], 1.0f / kLowUnit<T>, c[p][0][i]);
                s[p][i] = T == Q38_KV_Q8 ? __builtin_fmaf(x * below * k[p].scale[i], above, -base) : __builtin_fmaf(x, unscale, -base);
            }
        }
}

/* Scores past the column's own position do not count.  page: the first of kPages that lie kWaves apart. */
template <int kPages>
Q38_DEV void mask(float (&s)[kPages][4], int page, int last, int g) {
#pragma unroll
    for (int p = 0; p < kPages; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (16 * (page + kWaves * p) + 4 * g + i > last) s[p][i] = -INFINITY;
}

struct Span {
    int begin, end; /* pages of the split */
    int last;       /* the cache's last page that a query sees */
};
Q38_DEV Span span_of(const q38_observe_args &a) {
    const int last = (a.base_pos + a.n_tokens - 1) >> 4, begin = blockIdx.x * a.split_pages;
    return {begin, min(begin + a.split_pages, last + 1), last};
}

/* A short context's scores (log2 units, -inf where a column does not see): group, kv head and page by page, a tile
 * as the lanes hold it. */
Q38_DEV float *kept_scores(const q38_observe_args &a, int group, int j, int page, int tile, int lane) {
    const int pages = ((a.base_pos + a.n_tokens - 1) >> 4) + 1;
    return a.scores + (((((size_t)group * Q38_ATTN_KV_HEADS + j) * pages + page) * kTiles + tile) * 64 + lane) * 4;
}

template <int T, int kPages, int kParts>
Q38_DEV void observe_stats(const q38_observe_args &a) {
    __shared__ __attribute__((aligned(16))) Queries<kParts> q;
    const int j = blockIdx.y, group = a.group0 + blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const Span sp = span_of(a);
    const int tiles = tiles_of(a, group);
    load_queries<T>(q, a, group, j, lane, wave);
    __syncthreads();
    float M[kTiles], L[kTiles], unscale[kTiles];
    int last[kTiles]; /* the column's own position */
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        const int u = group * Q38_OBSERVE_QUERIES + (16 * t + c) / kGroup;
        M[t] = -INFINITY;
        L[t] = 0.0f;
        unscale[t] = q.unscale[16 * t + c];
        last[t] = u < a.n_tokens ? a.base_pos + u : -1;
    }
    for (int page = sp.begin + wave; page < sp.end; page += kWaves * kPages) {
        Keys k[kPages];
#pragma unroll
        for (int p = 0; p < kPages; ++p) load_keys<T>(k[p], a.kpool, a.page_row[min(page + kWaves * p, sp.end - 1)], j, lane);
        /* pages past the split's end, and positions that some column does not see */
        const bool masks = page + kWaves * (kPages - 1) >= sp.end ||
                           16 * (page + kWaves * (kPages - 1)) + 15 > a.base_pos + group * Q38_OBSERVE_QUERIES;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            if (t >= tiles) continue;
            /* against the column's reference so far, which is raised, as the decode's is, once a score passes it by
             * kRefSlack */
            float s[kPages][4];
            const bool none = M[t] == -INFINITY;
            const float base = none ? 0.0f : M[t];
            scores_of<T>(k, q.part[t], unscale[t], base, lane, s);
            if (masks) mask(s, page, min(last[t], 16 * sp.end - 1), g);
            if constexpr (kPages == 1) q38_st4(kept_scores(a, blockIdx.z, j, page, t, lane), f32x4{s[0][0], s[0][1], s[0][2], s[0][3]} + base);
            float top = -INFINITY;
#pragma unroll
            for (int p = 0; p < kPages; ++p) top = fmaxf(top, fmaxf(fmaxf(s[p][0], s[p][1]), fmaxf(s[p][2], s[p][3])));
            if (__any(top > (none ? -INFINITY : kRefSlack))) {
                const float by = none ? (top == -INFINITY ? 0.0f : top) : fmaxf(top, 0.0f);
                if (!none || top != -INFINITY) M[t] = base + by;
                L[t] *= none ? 0.0f : q38_exp2(-by); /* (a first reference below -128 has no finite power: 0 times it is none) */
#pragma unroll
                for (int p = 0; p < kPages; ++p)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[p][i] -= by;
            }
            float sum = 0.0f;
#pragma unroll
            for (int p = 0; p < kPages; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += q38_exp2(s[p][i]);
            L[t] += sum;
        }
    }
    /* the waves' in the queries' place */
    __syncthreads();
    float(*red)[Q38_OBSERVE_COLS][2] = reinterpret_cast<float(*)[Q38_OBSERVE_COLS][2]>(&q);
    static_assert(sizeof(float) * kWaves * Q38_OBSERVE_COLS * 2 <= sizeof(q), "the waves' columns fit");
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        const float top = column_max(M[t]);
        const float sum = column_sum(M[t] == -INFINITY ? 0.0f : L[t] * q38_exp2(M[t] - top));
        if (g == 0) {
            red[wave][16 * t + c][0] = top;
            red[wave][16 * t + c][1] = sum;
        }
    }
    __syncthreads();
    if (tid >= Q38_OBSERVE_COLS) return;
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, red[w][tid][0]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
        sum += red[w][tid][0] == -INFINITY ? 0.0f : red[w][tid][1] * q38_exp2(red[w][tid][0] - top);
    float *out = a.part_ml + ((((size_t)blockIdx.z * Q38_ATTN_KV_HEADS + j) * Q38_OBSERVE_COLS + tid) * a.n_splits + blockIdx.x) * 2;
    out[0] = top;
    out[1] = sum;
}

/* A column's maximum, and one over its sum. */
typedef float Stats[Q38_OBSERVE_COLS][2];

/* at_group: the group's place in part_ml; u0: its first query. */
Q38_DEV void join_stats(Stats &stat, const q38_observe_args &a, int at_group, int u0, int j, int tid) {
    /* the splits' maxima and sums joined, four threads a column (a wave a column
     * took 2 us longer a group) */
    const int col = tid >> 2;
    if (col < Q38_OBSERVE_COLS) {
        constexpr int kEach = 64 / 4;
        const float *ml = a.part_ml + (((size_t)at_group * Q38_ATTN_KV_HEADS + j) * Q38_OBSERVE_COLS + col) * a.n_splits * 2;
        float m[kEach], l[kEach], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int at = 4 * n + (tid & 3);
            m[n] = -INFINITY;
            l[n] = 0.0f;
            if (at < a.n_splits) {
                m[n] = ml[2 * at];
                l[n] = ml[2 * at + 1];
            }
        }
#pragma unroll
        for (int n = 0; n < kEach; ++n) top = fmaxf(top, m[n]);
        top = fmaxf(top, q38_dpp<0xB1>(top));
        top = fmaxf(top, q38_dpp<0x4E>(top));
        /* a split that the column sees nothing of has a maximum of -inf */
#pragma unroll
        for (int n = 0; n < kEach; ++n) sum += m[n] != -INFINITY ? l[n] * q38_exp2(m[n] - top) : 0.0f;
        sum += q38_dpp<0xB1>(sum);
        sum += q38_dpp<0x4E>(sum);
        const bool in = u0 + col / kGroup < a.n_tokens;
        if ((tid & 3) == 0) {
            stat[col][0] = in ? top : 0.0f;
            stat[col][1] = in ? 1.0f / sum : 0.0f;
        }
    }
}

template <int T, int kPages, int kParts>
Q38_DEV void observe_sums(const q38_observe_args &a) {
    __shared__ __attribute__((aligned(16))) Queries<kParts> q;
    __shared__ Stats stat;
    const int j = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const Span sp = span_of(a);
    for (int group = 0; group < a.n_groups; ++group) {
        const int u0 = group * Q38_OBSERVE_QUERIES, tiles = tiles_of(a, group);
        /* (the same in every wave) a split that only later groups see */
        if (16 * sp.begin > a.base_pos + min(u0 + Q38_OBSERVE_QUERIES, a.n_tokens) - 1) continue;
        __syncthreads(); /* the group before is done with q and stat */
        load_queries<T>(q, a, group, j, lane, wave);
        join_stats(stat, a, group, u0, j, tid);
        __syncthreads();
        for (int page = sp.begin + wave; page < sp.end; page += kWaves * kPages) {
            Keys k[kPages];
#pragma unroll
            for (int p = 0; p < kPages; ++p) load_keys<T>(k[p], a.kpool, a.page_row[min(page + kWaves * p, sp.end - 1)], j, lane);
            const bool masks = page + kWaves * (kPages - 1) >= sp.end || 16 * (page + kWaves * (kPages - 1)) + 15 > a.base_pos + u0;
            float w[kPages][4] = {};
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                if (t >= tiles) continue;
                float s[kPages][4];
                /* (read from LDS for each set of pages: six tiles' are too many registers) */
                int col = 16 * t + c;
                asm volatile("" : "+v"(col));
                scores_of<T>(k, q.part[t], q.unscale[col], stat[col][0], lane, s);
                if (masks) {
                    const int u = u0 + col / kGroup;
                    mask(s, page, min(u < a.n_tokens ? a.base_pos + u : -1, 16 * sp.end - 1), g);
                }
                const float inverse = stat[col][1];
#pragma unroll
                for (int p = 0; p < kPages; ++p)
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[p][i] = __builtin_fmaf(q38_exp2(s[p][i]), inverse, w[p][i]);
            }
#pragma unroll
            for (int p = 0; p < kPages; ++p) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[p][i] = q38_sum16(w[p][i]);
            }
            /* lane 16 g + p adds page p's tokens 4 g .. + 3 (all at once: one after the other each waits for its sum) */
            f32x4 add = {w[0][0], w[0][1], w[0][2], w[0][3]};
#pragma unroll
            for (int p = 1; p < kPages; ++p)
                if (c == p) add = f32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
            const int t0 = 16 * (page + kWaves * c) + 4 * g, end = min(a.base_pos + a.n_tokens, 16 * sp.end);
            if (c < kPages && t0 < end) {
                float *sums = a.weights + (size_t)a.page_row[page + kWaves * c] * Q38_WEIGHTS_PAGE + j * Q38_WEIGHTS_HEAD + 4 * g;
                const f32x4 now = q38_ld4(sums) + add;
                if (t0 + 4 <= end) {
                    q38_st4(sums, now);
                } else {
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        if (t0 + i < end) sums[i] = now[i];
                }
            }
        }
    }
}

/* The sums of a short context: a wave a page, from the scores that the statistics left. */
Q38_DEV void observe_add(const q38_observe_args &a) {
    __shared__ Stats stat;
    const int j = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int end = a.base_pos + a.n_tokens, pages = (end + 15) >> 4, page = blockIdx.x * kWaves + wave;
    const bool live = page < pages;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    for (int at = 0; at < a.n_groups; ++at) {
        const int group = a.group0 + at, tiles = tiles_of(a, group);
        f32x4 s[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) s[t] = q38_ld4(kept_scores(a, at, j, live ? page : 0, min(t, tiles - 1), lane));
        __syncthreads(); /* the group before is done with stat */
        join_stats(stat, a, at, group * Q38_OBSERVE_QUERIES, j, tid);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            if (t >= tiles) continue;
            const float top = stat[16 * t + c][0], inverse = stat[16 * t + c][1];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_fmaf(q38_exp2(s[t][i] - top), inverse, w[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = q38_sum16(w[i]);
    const int t0 = 16 * page + 4 * g;
    if (c != 0 || t0 >= end) return;
    float *sums = a.weights + (size_t)a.page_row[page] * Q38_WEIGHTS_PAGE + j * Q38_WEIGHTS_HEAD + 4 * g;
    const f32x4 now = q38_ld4(sums) + w;
    if (t0 + 4 <= end) {
        q38_st4(sums, now);
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (t0 + i < end) sums[i] = now[i];
    }
}

}  // namespace

#define Q38_OBSERVE_STATS(name, T, PAGES, PARTS)                                                                 \
    extern "C" __global__ __launch_bounds__(64 * kWaves) void q38_observe_stats_##name(q38_observe_args a) {     \
        observe_stats<T, PAGES, PARTS>(a);                                                                       \
    }
#define Q38_OBSERVE_SUMS(name, T, PARTS)                                                                         \
    extern "C" __global__ __launch_bounds__(64 * kWaves) void q38_observe_sums_##name(q38_observe_args a) {      \
        observe_sums<T, kPagesOf<T>, PARTS>(a);                                                                  \
    }
#define Q38_OBSERVE_KERNELS(name, suffix, T, PARTS)              \
    Q38_OBSERVE_STATS(name##suffix, T, kPagesOf<T>, PARTS)       \
    Q38_OBSERVE_STATS(name##_short##suffix, T, 1, PARTS)         \
    Q38_OBSERVE_SUMS(name##suffix, T, PARTS)
Q38_OBSERVE_KERNELS(f16, , Q38_KV_F16, 2)
Q38_OBSERVE_KERNELS(bf16, , Q38_KV_BF16, 2)
Q38_OBSERVE_KERNELS(bf16, _few, Q38_KV_BF16, 3)
Q38_OBSERVE_KERNELS(q8k, , Q38_KV_Q8, 2)
Q38_OBSERVE_KERNELS(mxfp4, , Q38_KV_MX4, 2)
Q38_OBSERVE_KERNELS(mxfp4, _few, Q38_KV_MX4, 3)
extern "C" __global__ __launch_bounds__(64 * kWaves) void q38_observe_add(q38_observe_args a) { observe_add(a); }
