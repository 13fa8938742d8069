/*
 * Rows of a ragged batch into and out of the pages of a cache of MXFP4 rows
 * (q38_kv_rows.h: the kernels of kv_rows.hip, whose norm, rotation, tiles of tokens
 * and ways through LDS these share).
 *
 * A block's scale is a power of two from its largest magnitude alone (the smallest
 * of which that has at most 7: 6 is then the nearest code for what lies above it too, as 7
 * is halfway to the 8 that would be next), so eight lanes of four values agree on it by three
 * maxima, and one conversion instruction rounds two values to nearest, ties to the
 * even code.  Rounding happens once, from the f32 row.
 *
 * Measured: 4096 tokens in 8.6 us, 33.6 MB in and 4.5 out, 4.4 TB/s (a copy's 38 MB
 * would take 6.1; 312 vector instructions a wave of keys and values on average do the rest), and back
 * as f32 in 6.5, 38 MB, 5.8 TB/s; 1531 tokens of 12 sequences to 16 bits 6.6 and 5.0, of
 * which the launches' start takes some 3 each.
 */
#include "q38_kv_rows.h"

Q38_KV_APPEND_KERNEL(q38_kv_append_mxfp4, Q38_KV_MX4)
Q38_KV_GATHER_KERNEL(q38_kv_gather_mxfp4, Q38_KV_MX4, false)
