/*
 * Rows of a ragged batch into and out of the pages of a typed KV cache.
 *
 * Append: key rows are RMSNormed (f64 sum of squares) and rotated on the way
 * (or stored as they are, without a norm weight), value rows stored as they
 * are, both converted to the cache's type once.  Gather is the inverse: the
 * values that the rows stand for as f32, or 16-bit rows as they are stored.
 *
 * A workgroup serves one page of one sequence, a wave per kv head; lane l of
 * a wave holds dims 4l .. 4l + 3 of the wave's head.
 */
#include "q38_kv_types.h"
#include "q38_rope.h"

namespace {

struct PageSpan {
    int t0, t1;   /* tokens of the page, [t0, t1) */
    int row0;     /* the batch's row of token t0 */
    int pos0;     /* and its position */
    int page;     /* physical page */
};

Q38_DEV PageSpan page_span(const q38_kv_rows_args &a, int x) {
    int b = 0;
    while (b + 1 < a.n_seq && a.page_base[b + 1] <= x) ++b;
    const int first = a.pos0[b], n = a.row_base[b + 1] - a.row_base[b];
    const int lp = (first >> 4) + x - a.page_base[b];
    const int p0 = max(first, lp * Q38_PAGE_TOKENS);
    const int p1 = min(first + n, (lp + 1) * Q38_PAGE_TOKENS);
    return {p0 & 15, (p0 & 15) + p1 - p0, a.row_base[b] + p0 - first, p0,
            a.page_table[(size_t)a.seq[b] * a.pt_stride + lp]};
}

template <int T>
Q38_DEV void store_row(char *block, bool key, int t, int lane, f32x4 x) {
    if (T == Q38_KV_Q8) {
        int q[4];
        float scale;
        q38_wave_q8k(x, q, scale);
        uint8_t *out = reinterpret_cast<uint8_t *>(block);
        if (lane == 0) q38_kv_scales(block)[t] = scale;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = 4 * lane + c;
            out[key ? q38_k_index<T>(t, d) : q38_v_index<T>(t, d)] = (uint8_t)(q[c] + 128);
        }
        return;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int d = 4 * lane + c;
        const int i = key ? q38_k_index<T>(t, d) : q38_v_index<T>(t, d);
        if (T == Q38_KV_F32)
            reinterpret_cast<float *>(block)[i] = x[c];
        else
            reinterpret_cast<uint16_t *>(block)[i] = q38_to16<T>(x[c]);
    }
}

template <int T>
Q38_DEV void kv_append(const q38_kv_rows_args &a) {
    __shared__ float cs[Q38_PAGE_TOKENS][32][2];
    const PageSpan sp = page_span(a, blockIdx.x);
    const bool key = blockIdx.y == 0;
    const int lane = threadIdx.x & 63, head = threadIdx.x >> 6;
    const bool turns = key && a.k_norm != nullptr;
    if (turns) {
        /* the page's angles: a half-wave per token */
        for (int t = sp.t0 + (int)(threadIdx.x >> 5); t < sp.t1; t += 8)
            q38_rope_table(cs[t], lane & 31, sp.pos0 + t - sp.t0, a.theta_scale);
        __syncthreads();
    }
    const float *rows = static_cast<const float *>(key ? a.k_rows : a.v_rows);
    char *block = q38_kv_block<T>(key ? a.kpool : a.vpool, sp.page, head);
    const f32x4 w = turns ? q38_ld4(a.k_norm + 4 * lane) : f32x4{0.f, 0.f, 0.f, 0.f};
    for (int t = sp.t0; t < sp.t1; ++t) {
        f32x4 x = q38_ld4(rows + (size_t)(sp.row0 + t - sp.t0) * Q38_ATTN_KV_DIM + head * Q38_ATTN_HEAD_DIM + 4 * lane);
        if (turns) q38_norm_rope4_cs(x, w, lane, cs[t]);
        store_row<T>(block, key, t, lane, x);
    }
}

template <int T, bool k16>
Q38_DEV void kv_gather(const q38_kv_rows_args &a) {
    const PageSpan sp = page_span(a, blockIdx.x);
    const bool key = blockIdx.y == 0;
    const int lane = threadIdx.x & 63, head = threadIdx.x >> 6;
    char *block = q38_kv_block<T>(key ? a.kpool : a.vpool, sp.page, head);
    void *rows = key ? a.k_rows : a.v_rows;
    for (int t = sp.t0; t < sp.t1; ++t) {
        const size_t at = (size_t)(sp.row0 + t - sp.t0) * Q38_ATTN_KV_DIM + head * Q38_ATTN_HEAD_DIM + 4 * lane;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = 4 * lane + c;
            const int i = key ? q38_k_index<T>(t, d) : q38_v_index<T>(t, d);
            if (k16)
                static_cast<uint16_t *>(rows)[at + c] = reinterpret_cast<const uint16_t *>(block)[i];
            else
                static_cast<float *>(rows)[at + c] = q38_kv_value<T>(block, i, t);
        }
    }
}

}  // namespace

#define Q38_KV_ROWS_KERNELS(name, T)                                                                        \
    extern "C" __global__ __launch_bounds__(256) void q38_kv_append_##name(q38_kv_rows_args a) { kv_append<T>(a); } \
    extern "C" __global__ __launch_bounds__(256) void q38_kv_gather_##name(q38_kv_rows_args a) {            \
        kv_gather<T, false>(a);                                                                             \
    }
Q38_KV_ROWS_KERNELS(f32, Q38_KV_F32)
Q38_KV_ROWS_KERNELS(f16, Q38_KV_F16)
Q38_KV_ROWS_KERNELS(bf16, Q38_KV_BF16)
Q38_KV_ROWS_KERNELS(q8k, Q38_KV_Q8)

/* 16-bit rows as they are stored, F16 or BF16. */
extern "C" __global__ __launch_bounds__(256) void q38_kv_gather_16(q38_kv_rows_args a) {
    kv_gather<Q38_KV_BF16, true>(a);
}
