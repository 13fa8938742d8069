/*
 * Decode over a cache of MXFP4 rows: the path of attn_decode_typed.hip
 * (q38_decode_typed.h holds both) with a step of its own.
 *
 * A value is a 4-bit code times its block's power of two, and the conversion
 * instructions turn two codes and a scale into two bf16 that hold the product
 * exactly: so scales cost no instruction after that, operands are bf16, and
 * queries and weights have the three bf16 parts (24 bits) that bf16 rows' have.
 * A page of 16 tokens is half the k of a P V product of 16 x 16 x 32, and 16-bit
 * rows take the 16 x 16 x 16 one for it; here a wave takes two pages a step, whose 32
 * tokens fill the longer product: half as many of them, and one rescaling and
 * reference for both (128K tokens 29.6 us against 36.4 a page at a time, 1021
 * tokens 6.2 against 7.9; two steps' pages in registers instead of one 30.2 and
 * 8.3: a page's rows are 4.25 KiB, and 8 waves of two fetch 68 KiB ahead as it is).
 * A row's position past the sequence's end has its codes and scales cleared.
 *
 * Measured (us of a whole pass with its merge; one sequence, 600 MB of layers in
 * turn / one layer again and again): 17 tokens 4.9 / 4.9, 1021 8.5 / 8.5, 4096 9.6 /
 * 9.1, 32K 14.7 / 13.1, 128K 30.7 / 29.5 (4.6 TB/s of rows; the steady part runs at
 * 6.1, what pages read once reach, and 5.6 us are start and join).  Reads past L2
 * are the pages' and 1% more (128K: 1.118e6 requests of 128 bytes for 142.6 MB).
 * 244 vector instructions a page and head keep pace with the pages; 16 sequences
 * of 2K to 32K take 46 us for 200 MB: splits of one size, of which a sequence's last
 * one is seldom full.
 */
#include "q38_decode_typed.h"

Q38_DECODE_KERNEL(mxfp4, Q38_KV_MX4, false)
Q38_DECODE_KERNEL(mxfp4_pre, Q38_KV_MX4, true)
