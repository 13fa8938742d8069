/*
 * The splits of a decode call joined: attn_decode.hip's merge kernels and
 * attn_weigh.hip's.
 */
#pragma once
#include "q38_device.h"

namespace {

/* Combine the splits of each (sequence, head): rescale every partial to the
 * common max, sum, normalise, gate.  Workgroup (b, h, dq): dq picks 64 of
 * the 256 dims, so 96 workgroups share a sequence's merge.  Thread (sl, dl)
 * merges splits sl, sl + 16, ... of dims 4dl..4dl+3 online (running max,
 * sum and output in registers); up to 8 splits' (m, l, o) are loaded at
 * once, so a merge of up to 128 splits costs one memory round trip.  The 16
 * per-thread results of each dim quad then meet in LDS. */
template <typename Args>
Q38_DEV void merge_splits(const Args &a, int b, int base, int n, int h, int dq) {
    constexpr int kBatch = 8;
    __shared__ f32x4 red_o[16][16];
    __shared__ float red_m[16][16];
    __shared__ float red_l[16][16];
    const int tid = threadIdx.x;
    const int dl = tid & 15;
    const int sl = tid >> 4;
    const int d = dq * 64 + 4 * dl;
    const size_t o_step = (size_t)Q38_ATTN_HEADS * Q38_ATTN_HEAD_DIM;
    const float *po = a.part_o + ((size_t)base * Q38_ATTN_HEADS + h) * Q38_ATTN_HEAD_DIM + d;
    const float *pml = a.part_ml + ((size_t)base * Q38_ATTN_HEADS + h) * 2;
    /* the gate of the 4 output dims this thread may store, loaded with the
     * partials rather than after them */
    const size_t off = (size_t)b * Q38_ATTN_Q_DIM + h * Q38_ATTN_HEAD_DIM + d;
    const bool gated = a.gate != nullptr;
    const f32x4 gt = gated && sl == 0 ? q38_ld4(a.gate + ((size_t)b * Q38_ATTN_HEADS + h) * a.gate_head_stride + d)
                                      : f32x4{0.f, 0.f, 0.f, 0.f};

    float M = -INFINITY, L = 0.0f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = sl; s0 < n; s0 += 16 * kBatch) {
        float m[kBatch], l[kBatch];
        f32x4 o[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int s = s0 + 16 * k;
            const bool in = s < n;
            const int sc = in ? s : s0; /* a split known to exist */
            m[k] = in ? pml[(size_t)sc * Q38_ATTN_HEADS * 2] : -INFINITY;
            l[k] = pml[(size_t)sc * Q38_ATTN_HEADS * 2 + 1];
            o[k] = q38_ld4(po + (size_t)sc * o_step);
        }
        float mx = M;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) mx = fmaxf(mx, m[k]);
        if (mx != -INFINITY) {
            const float f = q38_exp2(M - mx); /* 0 while M is -inf */
            L *= f;
            O *= f;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const float w = q38_exp2(m[k] - mx); /* 0 for absent or empty splits */
                L = __builtin_fmaf(w, l[k], L);
                O = q38_fma4(w, o[k], O);
            }
            M = mx;
        }
    }
    red_o[sl][dl] = O;
    red_m[sl][dl] = M;
    red_l[sl][dl] = L;
    __syncthreads();
    if (sl == 0) {
        float Mt = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) Mt = fmaxf(Mt, red_m[i][dl]);
        float Lt = 0.0f;
        f32x4 Ot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float mi = red_m[i][dl];
            const float w = mi == -INFINITY ? 0.0f : q38_exp2(mi - Mt);
            Lt = __builtin_fmaf(w, red_l[i][dl], Lt);
            Ot = q38_fma4(w, red_o[i][dl], Ot);
        }
        f32x4 r = Ot / Lt;
        if (gated) {
            r.x *= q38_sigmoid(gt.x);
            r.y *= q38_sigmoid(gt.y);
            r.z *= q38_sigmoid(gt.z);
            r.w *= q38_sigmoid(gt.w);
        }
        q38_st4(a.out + off, r);
    }
}

}  // namespace
