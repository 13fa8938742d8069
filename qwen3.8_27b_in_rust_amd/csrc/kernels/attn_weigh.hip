/*
 * Decode over a cache that adds up the attention weights of its tokens.
 *
 * A cached token's sum, per kv head, takes the softmax weight that each of the
 * group's 6 query heads gives it: W[t] += sum_h exp2(s_ht - M_h) / L_h.  M_h
 * and L_h are known only when every split has run, so the decode kernel
 * (q38_decode_typed.h) leaves its scores, 24 bytes a token and kv head, and
 * the launch that joins the splits' outputs turns them into weights beside it: a
 * workgroup per (split, kv head) joins the splits' maxima and sums for its six
 * heads and adds what each token gets.  A sequence of one split has both at its
 * workgroups' end, and they add there: where all sequences have one there is no
 * second launch.  Each sum has one owner, so the order of additions is fixed.
 * Scores are 96 bytes a token against the 1088 to 4096 of its rows.  (To form them
 * again in the second launch would read the keys twice, 512 to 2048 bytes a token.)
 *
 * Measured (us of a whole pass with its merge, 600 MB of layers in turn; beside it a
 * cache that tracks nothing): bf16 rows 17 tokens 6.2 (4.8), 1021 10.0 (8.3), 32K 29.2 (26.1), 128K 102 (86);
 * Q8_K 6.7 (5.3), 10.3 (8.5), 21.2 (17.6), 57 (47); MXFP4 6.9 (4.9), 10.4 (8.5), 17.3 (14.7), 39 (31).
 * (17 tokens with the sums in a launch of their own: 8.9, 9.5 and 10.0.)
 * Of 128K tokens' 12.6 MB of scores most of what they cost is their writing between the
 * pages' loads (bf16 86 us without; kept in LDS to the split's end 93, but 0.5 to 0.9
 * longer up to 32K tokens, and nothing gained for MXFP4).
 */
#include "q38_decode_typed.h"
#include "q38_merge.h"

#define Q38_WEIGH_KERNEL(name, T, PRE)                                                                      \
    extern "C" __global__ __launch_bounds__(64 * kWaves) void q38_attn_weigh_##name(q38_decode_typed_args a, \
                                                                                   q38_weigh_args w) {      \
        decode_typed<T, PRE>(a, w);                                                                         \
    }
Q38_WEIGH_KERNEL(f16, Q38_KV_F16, false)
Q38_WEIGH_KERNEL(f16_pre, Q38_KV_F16, true)
Q38_WEIGH_KERNEL(bf16, Q38_KV_BF16, false)
Q38_WEIGH_KERNEL(bf16_pre, Q38_KV_BF16, true)
Q38_WEIGH_KERNEL(q8k, Q38_KV_Q8, false)
Q38_WEIGH_KERNEL(q8k_pre, Q38_KV_Q8, true)
Q38_WEIGH_KERNEL(mxfp4, Q38_KV_MX4, false)
Q38_WEIGH_KERNEL(mxfp4_pre, Q38_KV_MX4, true)

namespace {

/* Workgroup (split g, kv head j): the tokens of the split. */
Q38_DEV void add_split(const q38_merge_args &m, const q38_weigh_merge_args &a, int g, int j) {
    __shared__ float top[kGroup], inverse[kGroup];
    int b = 0;
    while (b + 1 < m.n_seq && m.split_base[b + 1] <= g) ++b;
    const int base = m.split_base[b], n = m.split_base[b + 1] - base;
    if (n == 1) return; /* the decode kernel has added them */
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int h = wave; h < kGroup; h += 4) {
        /* the head's maximum and sum over all splits */
        const float *ml = m.part_ml + ((size_t)base * Q38_ATTN_HEADS + j * kGroup + h) * 2;
        float M = -INFINITY, L = 0.0f;
        for (int s = lane; s < n; s += 64) M = fmaxf(M, ml[(size_t)s * Q38_ATTN_HEADS * 2]);
        M = column_max(q38_max16(M));
        for (int s = lane; s < n; s += 64)
            L = __builtin_fmaf(ml[(size_t)s * Q38_ATTN_HEADS * 2 + 1], q38_exp2(ml[(size_t)s * Q38_ATTN_HEADS * 2] - M), L);
        L = column_sum(q38_sum16(L));
        if (lane == 0) {
            top[h] = M;
            inverse[h] = 1.0f / L;
        }
    }
    __syncthreads();
    const int t_begin = (g - base) * a.split_tokens, last = a.pos[b] - t_begin;
    const size_t head = (size_t)j * Q38_WEIGHTS_HEAD;
    add_weights<256>(top, inverse, a.scores + ((size_t)g * (a.split_tokens >> 4) * Q38_ATTN_KV_HEADS + j) * Q38_SCORES_PAGE,
                     a.page_table + (size_t)a.seq[b] * a.pt_stride + (t_begin >> 4), a.weights + head, a.tokens + head,
                     min(last + 1, a.split_tokens), last, a.appended != 0, a.pos[b] + a.evicted[b]);
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void q38_attn_weigh_merge(q38_merge_args m, q38_weigh_merge_args a) {
    constexpr int kMerges = Q38_ATTN_HEADS * 4;
    const int x = blockIdx.x;
    if (x >= m.n_seq * kMerges) {
        const int y = x - m.n_seq * kMerges;
        add_split(m, a, y >> 2, y & 3);
        return;
    }
    const int b = x / kMerges, rest = x - b * kMerges, base = m.split_base[b], n = m.split_base[b + 1] - base;
    if (n > 1) merge_splits(m, b, base, n, rest >> 2, rest & 3);
}
