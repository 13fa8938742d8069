/*
 * Decode over a cache of MXFP4 rows (q38_decode_typed.h: the kernels of
 * attn_decode_typed.hip).
 */
#include "q38_decode_typed.h"

Q38_DECODE_KERNEL(mxfp4, Q38_KV_MX4, false)
Q38_DECODE_KERNEL(mxfp4_pre, Q38_KV_MX4, true)
