/*
 * Decode over a cache that adds up the attention weights of its tokens.
 *
 * A cached token's sum, per kv head, takes the softmax weight that each of the
 * group's 6 query heads gives it: W[t] += sum_h exp2(s_ht - M_h) / L_h.  M_h
 * and L_h are known only when every split has run, so the decode kernel
 * (q38_decode_typed.h) leaves its scores, 24 bytes a token and kv head, and
 * the launch that joins the splits' outputs turns them into weights beside it: a
 * workgroup per (split, kv head) joins the splits' maxima and sums for its six
 * heads and adds what each token gets.  Each sum has one owner, so the order of
 * additions is fixed.  Scores are 96 bytes a token against the 1088 to 4096 of
 * its rows.  (To form them again in the second launch would read the keys twice, 512 to
 * 2048 bytes a token.)
 *
 * Measured (us of a whole pass with its merge, 600 MB of layers in turn; beside it a
 * cache that tracks nothing): bf16 rows 1021 tokens 9.6 (8.3), 32K 29.4 (26.1), 128K 104 (86);
@@ */
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
Q38_DEV void add_weights(const q38_merge_args &m, const q38_weigh_merge_args &a, int g, int j) {
    __shared__ float top[kGroup], inverse[kGroup];
    int b = 0;
    while (b + 1 < m.n_seq && m.split_base[b + 1] <= g) ++b;
    const int base = m.split_base[b], n = m.split_base[b + 1] - base;
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
    const int pos = a.pos[b], t_begin = (g - base) * a.split_tokens, t_end = min(pos + 1, t_begin + a.split_tokens);
    const int32_t *pt = a.page_table + (size_t)a.seq[b] * a.pt_stride + (t_begin >> 4);
    const float *scores = a.scores + ((size_t)g * (a.split_tokens >> 4) * Q38_ATTN_KV_HEADS + j) * Q38_SCORES_PAGE;
    for (int t = 4 * tid; t < t_end - t_begin; t += 4 * 256) {
        const float *sc = scores + (size_t)(t >> 4) * Q38_ATTN_KV_HEADS * Q38_SCORES_PAGE + (t & 15);
        const size_t at = (size_t)pt[t >> 4] * Q38_WEIGHTS_PAGE + j * Q38_WEIGHTS_HEAD + (t & 15);
        f32x4 s[kGroup];
#pragma unroll
        for (int h = 0; h < kGroup; ++h) s[h] = q38_ld4(sc + h * Q38_PAGE_TOKENS);
        const f32x4 old = q38_ld4(a.weights + at);
        f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < kGroup; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __builtin_fmaf(q38_exp2(s[h][i] - top[h]), inverse[h], w[i]);
        if (t_begin + t + 4 <= pos) {
            q38_st4(a.weights + at, old + w);
            continue;
        }
        /* the last tokens: none behind pos, and a new one starts its sum */
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = t_begin + t + i;
            if (p > pos) break;
            const bool starts = p == pos && a.appended;
            a.weights[at + i] = starts ? w[i] : old[i] + w[i];
            if (starts) a.tokens[at + i] = pos + a.evicted[b];
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void q38_attn_weigh_merge(q38_merge_args m, q38_weigh_merge_args a) {
    constexpr int kMerges = Q38_ATTN_HEADS * 4;
    const int x = blockIdx.x;
    if (x >= m.n_seq * kMerges) {
        const int y = x - m.n_seq * kMerges;
        add_weights(m, a, y >> 2, y & 3);
        return;
    }
    const int b = x / kMerges, rest = x - b * kMerges, base = m.split_base[b], n = m.split_base[b + 1] - base;
    if (n > 1) merge_splits(m, b, base, n, rest >> 2, rest & 3);
}
