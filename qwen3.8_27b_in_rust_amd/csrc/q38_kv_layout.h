/*
 * Element order of a KV cache's pages, by row type.
 *
 * A page of one kv head (a block) holds 16 tokens of 256 values, ordered as
 * the matrix unit's operands want them, so that a decode wave's loads are
 * contiguous kilobytes whose registers feed the products as they are:
 *  - K, the A operand of S^T = K Q^T on 16 x 16 x 32 tiles (lane l: token
 *    l % 16, eight dims from 8 (l / 16) of each 32): [dim / 32][dim / 8 % 4]
 *    [token][dim % 8]; 8-bit rows, two such steps to a 16-byte load:
 *    [dim / 64][dim / 16 % 4][token][dim % 16];
 *  - V, the B operand of O = P V on 16 x 16 x 16 tiles (lane l: dim l % 16
 *    of a 16-dim tile, tokens 4 (l / 16) .. + 3), two tiles to a 16-byte
 *    load: [dim / 32][token / 4][dim % 16][dim / 16 % 2][token % 4]; 8-bit
 *    rows, four tiles: [dim / 64][token / 4][dim % 16][dim / 16 % 4][token % 4].
 * Q8_K: a token's 256 values of one head are one Q8_K block -- the first
 * value m of largest magnitude sets the scale 1 / (-127 / m), quants are
 * round-to-nearest-even of x * (-127 / m) capped at 127 -- kept as quant +
 * 128 in a byte (the decode kernel makes f16 of it without a sign step).  The
 * f32 scales, [head][token], follow the page's four blocks, so that every
 * block starts on a cache line.
 * MXFP4: 32 of a token's values share a scale byte E, a value is its 4-bit code's
 * (sign, and 0, 0.5, 1, 1.5, 2, 3, 4, 6) times 2^(E - 127).  A word of eight codes,
 * lowest first, is what a conversion to the matrix unit's operands takes:
 *  - K, four steps of 32 dims to a 16-byte load, as above:
 *    [dim / 128][dim / 8 % 4][token][dim / 32 % 4][dim % 8];
 *  - V, one byte of a lane holds its dims of two 16-dim tiles (one scale for
 *    both), a word four tokens': [dim / 128][token / 4][dim % 16][dim / 32 % 4]
 *    [token % 4][dim / 16 % 2].
 * The scale bytes follow the four blocks, 128 to a head: K [token][dim / 32], the
 * eight of a lane's token in one load; V [token / 4][dim / 32][token % 4], as its words'
 * bytes lie.  A block that an infinity or NaN got into has E = 255.
 */
#ifndef Q38_KV_LAYOUT_H
#define Q38_KV_LAYOUT_H

#include "q38_kargs.h"

#ifndef Q38_LAYOUT_FN
#define Q38_LAYOUT_FN inline
#endif

enum { Q38_KV_F32 = 0, Q38_KV_F16 = 1, Q38_KV_BF16 = 2, Q38_KV_Q8 = 3, Q38_KV_MX4 = 4 };

template <int T>
Q38_LAYOUT_FN constexpr int q38_kv_page_bytes() {
    return T == Q38_KV_F32 ? Q38_KV_PAGE_F32 : T == Q38_KV_Q8 ? Q38_KV_PAGE_Q8 : T == Q38_KV_MX4 ? Q38_KV_PAGE_MX4 : Q38_KV_PAGE_16;
}
/* Of a block: one kv head's values. */
template <int T>
Q38_LAYOUT_FN constexpr int q38_kv_block_bytes() {
    return T == Q38_KV_MX4 ? Q38_PAGE_TOKENS * Q38_ATTN_HEAD_DIM / 2
                           : Q38_PAGE_TOKENS * Q38_ATTN_HEAD_DIM * (T == Q38_KV_F32 ? 4 : T == Q38_KV_Q8 ? 1 : 2);
}
/* Q8_K: a block's scales, in bytes after its first quant. */
Q38_LAYOUT_FN int q38_kv_scales_offset(int head) {
    return (Q38_ATTN_KV_HEADS - head) * Q38_PAGE_TOKENS * Q38_ATTN_HEAD_DIM + head * Q38_PAGE_TOKENS * 4;
}

/* MXFP4: a block's scale bytes, likewise, and the place of one of them. */
enum { Q38_MX4_SCALES = Q38_PAGE_TOKENS * Q38_ATTN_HEAD_DIM / 32 };
Q38_LAYOUT_FN int q38_mx4_scales_offset(int head) {
    return (Q38_ATTN_KV_HEADS - head) * q38_kv_block_bytes<Q38_KV_MX4>() + head * Q38_MX4_SCALES;
}
Q38_LAYOUT_FN int q38_mx4_k_scale(int t, int d) { return t * 8 + (d >> 5); }
Q38_LAYOUT_FN int q38_mx4_v_scale(int t, int d) { return (t >> 2) * 32 + (d >> 5) * 4 + (t & 3); }

/* Element offset of (token, dim) in a block (MXFP4: in codes of 4 bits). */
template <int T>
Q38_LAYOUT_FN int q38_k_index(int t, int d) {
    if (T == Q38_KV_F32) return t * 256 + d;
    if (T == Q38_KV_Q8) return ((d >> 6) * 64 + ((d >> 4) & 3) * 16 + t) * 16 + (d & 15);
    if (T == Q38_KV_MX4) return ((d >> 7) * 64 + ((d >> 3) & 3) * 16 + t) * 32 + ((d >> 5) & 3) * 8 + (d & 7);
    return ((d >> 5) * 64 + ((d >> 3) & 3) * 16 + t) * 8 + (d & 7);
}
template <int T>
Q38_LAYOUT_FN int q38_v_index(int t, int d) {
    if (T == Q38_KV_F32) return t * 256 + d;
    if (T == Q38_KV_Q8) return ((d >> 6) * 64 + (t >> 2) * 16 + (d & 15)) * 16 + ((d >> 4) & 3) * 4 + (t & 3);
    if (T == Q38_KV_MX4)
        return ((d >> 7) * 64 + (t >> 2) * 16 + (d & 15)) * 32 + ((d >> 5) & 3) * 8 + (t & 3) * 2 + ((d >> 4) & 1);
    return ((d >> 5) * 64 + (t >> 2) * 16 + (d & 15)) * 8 + ((d >> 4) & 1) * 4 + (t & 3);
}

#endif
