/*
 * Full-attention GQA decode over a paged KV cache of 16-bit or 8-bit rows
 * (gfx950, wave64): the same path as over f32 rows (attn_decode.hip; full_core,
 * src/model/ops.rs:813-940), whose cache holds each row rounded to its type.
 */
#include "q38_kv_types.h"
#include "q38_rope.h"

/* 1/sqrt(256) (ops.rs:869) times log2(e). */
#define Q38_SCORE_LOG2 0.09016844005556021f

namespace {

template <int T, bool kPre>
Q38_DEV void decode_typed(const q38_decode_args &a) {
    __shared__ __attribute__((aligned(16))) float q[Q38_ATTN_GROUP][Q38_ATTN_HEAD_DIM];
    __shared__ float row[2][Q38_ATTN_HEAD_DIM];
    __shared__ float p[Q38_ATTN_GROUP][Q38_PAGE_TOKENS];
    __shared__ float cs[32][2];
    const int g = blockIdx.x, j = blockIdx.y, tid = threadIdx.x;
    int b = 0;
    while (b + 1 < a.n_seq && a.split_base[b + 1] <= g) ++b;
    const int seq = a.seq[b], pos = a.pos[b];
    const int split = g - a.split_base[b], nsplit = a.split_base[b + 1] - a.split_base[b];
    const int t_begin = split * a.split_tokens, t_end = min(pos + 1, t_begin + a.split_tokens);
    const int32_t *pt = a.page_table + (size_t)seq * a.pt_stride;
    const int lane = tid & 63, wave = tid >> 6;
    const int q_stride = kPre ? 2 * Q38_ATTN_HEAD_DIM : Q38_ATTN_HEAD_DIM;
    const float *qb = a.q + ((size_t)b * Q38_ATTN_HEADS + j * Q38_ATTN_GROUP) * q_stride;
    if (kPre) {
        if (tid < 64) q38_rope_table(cs, lane, pos, a.theta_scale);
        __syncthreads();
    }
    for (int hh = wave; hh < Q38_ATTN_GROUP; hh += 4) {
        f32x4 x = q38_ld4(qb + hh * q_stride + 4 * lane);
        if (kPre) q38_norm_rope4_cs(x, q38_ld4(a.q_norm + 4 * lane), lane, cs);
        q38_st4(&q[hh][4 * lane], x * Q38_SCORE_LOG2);
    }
    if (a.k_new != nullptr && t_end == pos + 1 && wave < 2) {
        /* the new token's row: wave 0 the key, wave 1 the value */
        const float *src = (wave ? a.v_new : a.k_new) + (size_t)b * Q38_ATTN_KV_DIM + j * Q38_ATTN_HEAD_DIM;
        f32x4 x = q38_ld4(src + 4 * lane);
        if (kPre && wave == 0) q38_norm_rope4_cs(x, q38_ld4(a.k_norm + 4 * lane), lane, cs);
        char *block = q38_kv_block<T>(wave ? a.vpool : a.kpool, pt[pos >> 4], j);
        const int t = pos & 15;
        int qv[4];
        float scale = 0.0f;
        if (T == Q38_KV_Q8) {
            q38_wave_q8k(x, qv, scale);
            if (lane == 0) q38_kv_scales(block)[t] = scale;
        }
        for (int c = 0; c < 4; ++c) {
            const int i = wave ? q38_v_index<T>(t, 4 * lane + c) : q38_k_index<T>(t, 4 * lane + c);
            if (T == Q38_KV_Q8)
                reinterpret_cast<uint8_t *>(block)[i] = (uint8_t)(qv[c] + 128);
            else
                reinterpret_cast<uint16_t *>(block)[i] = q38_to16<T>(x[c]);
        }
        __threadfence();
    }
    __syncthreads();
    float m[Q38_ATTN_GROUP], l[Q38_ATTN_GROUP], o[Q38_ATTN_GROUP];
    for (int hh = 0; hh < Q38_ATTN_GROUP; ++hh) m[hh] = -INFINITY, l[hh] = o[hh] = 0.0f;
    for (int tb = t_begin; tb < t_end; tb += Q38_PAGE_TOKENS) {
        const int page = pt[tb >> 4], n = min(Q38_PAGE_TOKENS, t_end - tb);
        char *kb = q38_kv_block<T>(a.kpool, page, j), *vb = q38_kv_block<T>(a.vpool, page, j);
        if (tid < Q38_ATTN_GROUP * Q38_PAGE_TOKENS) {
            const int hh = tid >> 4, t = tid & 15;
            float s = 0.0f;
            if (t < n)
                for (int d = 0; d < Q38_ATTN_HEAD_DIM; ++d)
                    s = __builtin_fmaf(q[hh][d], q38_kv_value<T>(kb, q38_k_index<T>(t, d), t), s);
            p[hh][t] = t < n ? s : -INFINITY;
        }
        __syncthreads();
        for (int hh = 0; hh < Q38_ATTN_GROUP; ++hh) {
            float mx = m[hh];
            for (int t = 0; t < n; ++t) mx = fmaxf(mx, p[hh][t]);
            const float f = q38_exp2(m[hh] - mx);
            l[hh] *= f;
            o[hh] *= f;
            m[hh] = mx;
            for (int t = 0; t < n; ++t) {
                const float w = q38_exp2(p[hh][t] - mx);
                l[hh] += w;
                o[hh] = __builtin_fmaf(w, q38_kv_value<T>(vb, q38_v_index<T>(t, tid), t), o[hh]);
            }
        }
        __syncthreads();
    }
    for (int hh = 0; hh < Q38_ATTN_GROUP; ++hh) {
        const int h = j * Q38_ATTN_GROUP + hh;
        if (nsplit == 1) {
            float r = o[hh] / l[hh];
            if (a.gate != nullptr)
                r *= q38_sigmoid(a.gate[((size_t)b * Q38_ATTN_HEADS + h) * a.gate_head_stride + tid]);
            a.out[(size_t)b * Q38_ATTN_Q_DIM + h * Q38_ATTN_HEAD_DIM + tid] = r;
        } else {
            a.part_o[((size_t)g * Q38_ATTN_HEADS + h) * Q38_ATTN_HEAD_DIM + tid] = o[hh];
            if (tid == 0) {
                a.part_ml[((size_t)g * Q38_ATTN_HEADS + h) * 2 + 0] = m[hh];
                a.part_ml[((size_t)g * Q38_ATTN_HEADS + h) * 2 + 1] = l[hh];
            }
        }
    }
}

}  // namespace

#define Q38_DECODE_KERNELS(name, T)                                                                     \
    extern "C" __global__ __launch_bounds__(256) void q38_attn_decode_##name(q38_decode_args a) {       \
        decode_typed<T, false>(a);                                                                      \
    }                                                                                                   \
    extern "C" __global__ __launch_bounds__(256) void q38_attn_decode_##name##_pre(q38_decode_args a) { \
        decode_typed<T, true>(a);                                                                       \
    }
Q38_DECODE_KERNELS(f16, Q38_KV_F16)
Q38_DECODE_KERNELS(bf16, Q38_KV_BF16)
Q38_DECODE_KERNELS(q8k, Q38_KV_Q8)
