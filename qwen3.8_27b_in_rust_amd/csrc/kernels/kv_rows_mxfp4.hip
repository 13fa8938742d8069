/*
 * Rows of a ragged batch into and out of the pages of a cache of MXFP4 rows
 * (q38_kv_rows.h: the kernels of kv_rows.hip).
 */
#include "q38_kv_rows.h"

Q38_KV_APPEND_KERNEL(q38_kv_append_mxfp4, Q38_KV_MX4)
Q38_KV_GATHER_KERNEL(q38_kv_gather_mxfp4, Q38_KV_MX4, false)
