/*
 * RMSNorm and the partial rotation of 256-dim query and key heads, shared by
 * the decode kernels and the cache's row kernels: one set of roundings, so a
 * key comes out the same whichever kernel appends it.
 */
#pragma once
#include "q38_device.h"

/* RoPE angles of one position: pair p gets theta_p = position * scale^p by p
 * repeated f32 multiplications (the reference's rounding), and cs[p] = (cos,
 * sin) of it; lane p < 32 of the calling half-wave forms pair p, every lane
 * running the whole chain and keeping its own term of it (a loop of p steps
 * costs a branch a step). */
Q38_DEV void q38_rope_table(float (*cs)[2], int lane, int position, float theta_scale) {
    float theta = (float)position, mine = theta;
#pragma unroll
    for (int i = 1; i < 32; ++i) {
        theta *= theta_scale;
        mine = lane == i ? theta : mine;
    }
    float sine, cosine;
    sincosf(mine, &sine, &cosine);
    if (lane < 32) {
        cs[lane][0] = cosine;
        cs[lane][1] = sine;
    }
}

/* RoPE on dims 0..63 (ops.rs:595-610: pairs (p, p+32), theta_0 = position,
 * theta_{p+1} = theta_p * 1e7^(-2/64) by repeated f32 multiplication) of one
 * 256-dim head held 4 dims per lane by a whole wave (lane l: dims 4l ..
 * 4l+3), with the angles' cosines and sines from a q38_rope_table */
Q38_DEV void q38_rope_lanes_cs(f32x4 &x, int l, const float (*cs)[2]) {
    f32x4 partner;
#pragma unroll
    for (int c = 0; c < 4; ++c) partner[c] = __shfl_xor(x[c], 8, 64);
    if (l < 16) {
        const int p0 = 4 * (l & 7);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float cosine = cs[p0 + c][0];
            const float sine = cs[p0 + c][1];
            if (l < 8) {
                const float x0 = x[c], x1 = partner[c];
                x[c] = x0 * cosine - x1 * sine;
            } else {
                const float x0 = partner[c], x1 = x[c];
                x[c] = x0 * sine + x1 * cosine;
            }
        }
    }
}

/* RMS scale of a 256-dim head from its f64 sum of squares */
Q38_DEV float q38_rms_scale_of(double ss) {
    const float mean = (float)(ss / (double)Q38_ATTN_HEAD_DIM);
    return 1.0f / sqrtf(mean + 1e-6f);
}

/* The same for a head held by a half-wave, lane li: dims 4li .. 4li+3 (x0)
 * and 128 + 4li .. (x1); the angles from a q38_rope_table. */
Q38_DEV void q38_norm_rope8(f32x4 &x0, f32x4 &x1, f32x4 w0, f32x4 w1, int li, const float (*cs)[2]) {
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < 4; ++c) ss += (double)x0[c] * (double)x0[c] + (double)x1[c] * (double)x1[c];
    const float scale = q38_rms_scale_of(q38_sum32_f64(ss));
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        x0[c] = x0[c] * scale * w0[c];
        x1[c] = x1[c] * scale * w1[c];
    }
    q38_rope_lanes_cs(x0, li, cs);
}

/* RMSNorm with weight w (rms_scale / rmsnorm_inplace, ops.rs:476-498: f64 sum
 * of squares, eps 1e-6), then the RoPE of q38_rope_lanes_cs, of a head held 4
 * dims per lane by a whole wave.  Every f32 square is exact in f64, its sums are
 * not: two orders of them give the same f32 mean unless it lies within some
 * 2^-50 of halfway between two.  The forms of a whole wave (this, q38_norm_rope_row, the
 * append's) add in one order and agree bit for bit; a half-wave's
 * (q38_norm_rope8) adds in another. */
Q38_DEV void q38_norm_rope4_cs(f32x4 &x, f32x4 w, int lane, const float (*cs)[2]) {
    double ss = (double)x.x * (double)x.x + (double)x.y * (double)x.y + (double)x.z * (double)x.z +
                (double)x.w * (double)x.w;
    const float scale = q38_rms_scale_of(q38_wave_sum_f64(ss));
#pragma unroll
    for (int c = 0; c < 4; ++c) x[c] = x[c] * scale * w[c];
    q38_rope_lanes_cs(x, lane, cs);
}

/* q38_rope_table for a half-wave whose lane li is the wave's lane li or li + 32:
 * which lanes keep a step's angle is a constant mask rather than a comparison. */
Q38_DEV void q38_rope_table_half(float (*cs)[2], int li, int position, float theta_scale) {
    float theta = (float)position, mine = theta;
#pragma unroll
    for (int i = 1; i < 32; ++i) {
        theta *= theta_scale;
        mine = __builtin_amdgcn_inverse_ballot_w64(1ull << i | 1ull << (i + 32)) ? theta : mine;
    }
    float sine, cosine;
    sincosf(mine, &sine, &cosine);
    cs[li][0] = cosine;
    cs[li][1] = sine;
}

/* q38_rope_lanes_cs with the partner lane (l ^ 8) reached inside its row of 16. */
Q38_DEV void q38_rope_row(f32x4 &x, int lane, const float (*cs)[2]) {
    f32x4 partner;
#pragma unroll
    for (int c = 0; c < 4; ++c) partner[c] = q38_row_move<0x128>(x[c]);
    if (lane < 16) {
        const f32x4 *p = reinterpret_cast<const f32x4 *>(&cs[4 * (lane & 7)][0]);
        const f32x4 p0 = p[0], p1 = p[1];
        const float cosine[4] = {p0[0], p0[2], p1[0], p1[2]}, sine[4] = {p0[1], p0[3], p1[1], p1[3]};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            /* lanes 0-7 hold dims 0 .. 31, lanes 8-15 their partners 32 .. 63 */
            const float own = x[c] * cosine[c], other = partner[c] * sine[c];
            x[c] = lane < 8 ? own - other : other + own;
        }
    }
}

/* q38_norm_rope4_cs by row moves, its sums in the same order.  Every f32 square
 * is exact in f64, so a fused addition rounds as the plain one. */
Q38_DEV void q38_norm_rope_row(f32x4 &x, f32x4 w, int lane, const float (*cs)[2]) {
    double ss = (double)x.x * (double)x.x;
#pragma unroll
    for (int c = 1; c < 4; ++c) ss = __builtin_fma((double)x[c], (double)x[c], ss);
    ss += q38_row_move_f64<0xB1>(ss);
    ss += q38_row_move_f64<0x4E>(ss);
    ss += q38_row_move_f64<0x141>(ss);
    ss += q38_row_move_f64<0x140>(ss);
    x = x * q38_rms_scale_of(q38_rows_sum_f64(ss)) * w;
    q38_rope_row(x, lane, cs);
}
