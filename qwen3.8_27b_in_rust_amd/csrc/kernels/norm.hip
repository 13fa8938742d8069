/*
 * The residual's addition, the layer norm and its 8-bit form, one pass over
 * a row (gfx950, wave64): h = x + residual, y = h * (1 / sqrt(mean(h^2) +
 * 1e-6)) * w (accumulate ops.rs:547-560, rmsnorm ops.rs:476-498: f64 sum of
 * squares), and y's Q8_K blocks (quantize_q8_k, src/kernel/quant.rs:97-128).
 */
#include "q38_kv_types.h"

namespace {

Q38_DEV double block_sum_f64(double x, double *part, int waves) {
    x = q38_wave_sum_f64(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < waves; ++w) s += part[w];
    return s;
}

}  // namespace

/* grid (n_tokens), 256 threads. */
extern "C" __global__ __launch_bounds__(256) void q38_add_rms_norm(q38_norm_args a) {
    __shared__ double part[4];
    const int t = blockIdx.x, width = a.width;
    const size_t row = (size_t)t * width;
    double ss = 0.0;
    for (int d = threadIdx.x; d < width; d += 256) {
        const float h = a.residual != nullptr ? a.x[row + d] + a.residual[row + d] : a.x[row + d];
        ss += (double)h * (double)h;
    }
    const float mean = (float)(block_sum_f64(ss, part, 4) / (double)width);
    const float scale = 1.0f / sqrtf(mean + 1e-6f);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int blocks = width / Q38_Q8K_BLOCK;
    int8_t *quants = static_cast<int8_t *>(a.q8k);
    int16_t *sums = reinterpret_cast<int16_t *>(quants + (size_t)a.n_tokens * width);
    float *scales = reinterpret_cast<float *>(sums + (size_t)a.n_tokens * blocks * 16);
    /* a wave per 256 values, lane l: 4l .. 4l + 3 */
    for (int b = wave; b * 256 < width; b += 4) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = b * 256 + 4 * lane + c;
            if (d >= width) continue;
            const float h = a.residual != nullptr ? a.x[row + d] + a.residual[row + d] : a.x[row + d];
            y[c] = h * scale * a.weight[d];
            if (a.sum != nullptr) a.sum[row + d] = h;
            if (a.y != nullptr) a.y[row + d] = y[c];
        }
        if (a.q8k == nullptr) continue;
        int q[4];
        float qs;
        q38_wave_q8k(y, q, qs);
        const size_t k = (size_t)t * blocks + b;
        int s = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            quants[k * 256 + 4 * lane + c] = (int8_t)q[c];
            s += q[c];
        }
        s += __builtin_amdgcn_update_dpp(0, s, 0xB1, 0xF, 0xF, false);
        s += __builtin_amdgcn_update_dpp(0, s, 0x4E, 0xF, 0xF, false);
        if ((lane & 3) == 0) sums[k * 16 + (lane >> 2)] = (int16_t)s;
        if (lane == 0) scales[k] = qs;
    }
}

/* The values that Q8_K rows stand for: grid (ceil(n_tokens * width / 1024)),
 * 256 threads, 4 values each. */
extern "C" __global__ __launch_bounds__(256) void q38_dequantize_q8k(q38_dequantize_args a) {
    const size_t n = (size_t)a.n_tokens * a.width;
    const size_t i = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x);
    if (i >= n) return;
    const char *base = static_cast<const char *>(a.q8k);
    const uint32_t u = *reinterpret_cast<const uint32_t *>(base + i);
    const float s = reinterpret_cast<const float *>(base + n + n / 8)[i >> 8];
    f32x4 v;
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = (float)(int8_t)(u >> (8 * c)) * s;
    q38_st4(a.out + i, v);
}
