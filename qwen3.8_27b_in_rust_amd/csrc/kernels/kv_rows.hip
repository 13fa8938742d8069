/*
 * Rows of a ragged batch into and out of the pages of a typed KV cache.
 *
 * Append: key rows are RMSNormed (f64 sum of squares) and rotated on the way
 * (or stored as they are, without a norm weight), value rows stored as they
 * are, both converted to the cache's type once.  Gather is the inverse: the
 * values that the rows stand for as f32, or 16-bit rows as they are stored.
 *
 * Both move bytes: 4 KB of f32 a row and half or a quarter of that in the
 * page.  A workgroup of 8 waves serves half a page of one sequence; a wave has
 * four tokens (a quad) of one kv head, lane l the dims 4l .. 4l + 3 of each.
 * All its loads go out at once -- four workgroups a CU keep the memory busy --
 * and the quad's part of the page is put together in the wave's own LDS, where
 * the page's element order (q38_kv_layout.h) makes it 16-byte pieces: of one
 * token for K, of all four for V.  The rotation angles are formed once per token,
 * by a workgroup whose waves share them (half as many heads in one, and the
 * angles twice, took 13.4 us where this took 12.5).  A workgroup for a whole page
 * leaves the keys' arithmetic to half as many CUs where there are few pages,
 * one for a quarter costs its start too often: 1531 tokens of 12 sequences to
 * bf16 7.7 us, 6.7 by halves, 7.0 by quarters, and back 6.3, 6.0, 6.4; 4096 to
 * Q8_K 9.9, 9.2, 9.3 and back 7.6, 7.5, 8.0; to bf16 9.4, 10.1, 11.2.
 *
 * Measured (us, calls of one kind in turn over buffers that no cache holds):
 * 4096 tokens to Q8_K 9.2 (42 MB) and back 7.4 (5.7 TB/s); 1531 tokens of 12
 * sequences to bf16 6.8 and back 5.2; 6 tokens to f16 4.1 and back 3.8, which
 * is what the launches of so small calls take on the host.  (Traced in turn with
 * each other, 4096 tokens take the kernels 10.1 and 6.7.)
 * Keys are held up by their arithmetic as much as by memory: the angles and,
 * per token and head, the f64 sum, the rotation and the quantiser are some
 * 500 instructions a wave and quad (1500 with four reductions one by one,
 * 19 us).
 */
#include "q38_kv_rows.h"

Q38_KV_APPEND_KERNEL(q38_kv_append_f32, Q38_KV_F32)
Q38_KV_APPEND_KERNEL(q38_kv_append_f16, Q38_KV_F16)
Q38_KV_APPEND_KERNEL(q38_kv_append_bf16, Q38_KV_BF16)
Q38_KV_APPEND_KERNEL(q38_kv_append_q8k, Q38_KV_Q8)
Q38_KV_GATHER_KERNEL(q38_kv_gather_f32, Q38_KV_F32, false)
Q38_KV_GATHER_KERNEL(q38_kv_gather_f16, Q38_KV_F16, false)
Q38_KV_GATHER_KERNEL(q38_kv_gather_bf16, Q38_KV_BF16, false)
Q38_KV_GATHER_KERNEL(q38_kv_gather_q8k, Q38_KV_Q8, false)
/* 16-bit rows as they are stored, F16 or BF16. */
Q38_KV_GATHER_KERNEL(q38_kv_gather_16, Q38_KV_BF16, true)
