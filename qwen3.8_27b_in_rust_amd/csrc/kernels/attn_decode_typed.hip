/*
 * Full-attention GQA decode over a paged KV cache of 16-bit or 8-bit rows
 * (gfx950, wave64): the path of attn_decode.hip (full_core,
 * src/model/ops.rs:813-940) over a cache that holds each row rounded to its
 * type.
 *
 * A workgroup streams one kv head's pages of one context split once for the
 * group's 6 query heads, a wave per page, and the split's partials are joined
 * by q38_attn_decode_merge.  Half or a quarter of the f32 bytes come in per
 * row, and the vector unit no longer keeps up with them (12 multiply-adds a
 * value and the conversions), so the products run on the matrix unit, in f32
 * class precision although its operands have 16 bits:
 *  - S^T = K Q^T, 16 tokens x 16 columns.  A cached value is an operand as it
 *    stands (an 8-bit quant as a whole number in f16, its row's scale applied
 *    to the score).  A query is split into parts whose sum it is -- f16 hi and
 *    lo (22 bits, after a power of two per head brings the largest to 2^9..10,
 *    clear of f16's ends; lo taken 2^11 times as large, so that f16's fixed step
 *    below 2^-14 is 2^-45 of the largest or less and a small one on a large key keeps its
 *    bits), or bf16 hi, mid and lo (24 bits) -- and the 6 heads
 *    fill columns 0-5 with one part and 8-13 with another, so two parts cost
 *    one product; a rotation of the 16 lanes by 8 adds them up.
 *  - O = P V, 16 rows x 16 dims.  The lanes that hold a score are those that
 *    supply its weight as an operand (C's column l % 16, rows 4 (l / 16) + i
 *    are A's row l % 16, k 4 (l / 16) + i), so the weights never leave their
 *    registers; they are split like the queries, into rows 0-5 and 8-13, and held
 *    to 2^-36 of their unit (2^-43 of the largest weight) or to 22 bits.
 *    8-bit rows: the value's scale goes into its weight, over a power of two
 *    per head that follows the largest product of the two, so that a row of
 *    large values without weight takes nothing from the others.
 *  - softmax in base 2 against a reference per head that is raised (and O and
 *    the sum rescaled) only when a score passes the one that set it by 2^8, so
 *    most pages rescale nothing.  In f16 the weights are taken 2^7 times as
 *    large, up to 2^15, which leaves their small parts more of its range; the
 *    partials leave without that factor.
 * An infinity in a row that counts meets a lower part that may be 0 or of the
 * other sign: NaN, in the heads of a key, in the dim of a value (16-bit rows).
 * A row's position past the sequence's end counts nothing whatever it holds:
 * its scores are -inf and its values, which a weight of 0 would not keep NaN
 * out of, are cleared.
 *
 * Measured (us of a whole pass with its merge; one sequence, 600 MB of caches in
 * turn, so that nothing is in the last level's cache; forming q in the
 * kernel adds under 1): bf16 rows 17 tokens 4.8, 1021 8.3, 4096 10.5, 32K 26.1 (5.1
 * TB/s), 128K 85.9 (6.2 TB/s, what pages read once in any order reach); Q8_K 5.3,
 * 8.5, 10.0, 17.6 and 47.1 (5.8 TB/s).  One cache again and again, 1021 to 128K: 8.0,
 * 8.7, 25.7, 83.9 and 8.2, 9.0, 16.4, 46.9.  Long 16-bit contexts are bound by memory,
 * Q8_K ones by memory and the 266 vector instructions a page and head that mostly
 * turn bytes into operands; short ones by the two launches and the chain
 * arguments - page id - page - scores - join, 3-4 us of them.
 */
#include "q38_decode_typed.h"

Q38_DECODE_KERNEL(f16, Q38_KV_F16, false)
Q38_DECODE_KERNEL(f16_pre, Q38_KV_F16, true)
Q38_DECODE_KERNEL(bf16, Q38_KV_BF16, false)
Q38_DECODE_KERNEL(bf16_pre, Q38_KV_BF16, true)
Q38_DECODE_KERNEL(q8k, Q38_KV_Q8, false)
Q38_DECODE_KERNEL(q8k_pre, Q38_KV_Q8, true)
