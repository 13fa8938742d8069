/*
 * The residual's addition, the layer norm and its 8-bit form, one pass over
 * a row (gfx950, wave64): h = x + residual, y = h * (1 / sqrt(mean(h^2) +
 * 1e-6)) * w (accumulate ops.rs:547-560, rmsnorm ops.rs:476-498: f64 sum of
 * squares), and y's Q8_K blocks (quantize_q8_k, src/kernel/quant.rs:97-128).
 */
#include "q38_kv_types.h"

namespace {

/* The sum over the workgroup, the same in every thread. */
template <int NT>
Q38_DEV double block_sum_f64(double x, double *part) {
    x = q38_wave_sum_f64(x);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) s += part[w];
    return s;
}

Q38_DEV float norm_scale(double ss, int width) {
    const float mean = (float)(ss / (double)width);
    return 1.0f / sqrtf(mean + 1e-6f);
}

Q38_DEV double square_sum(f32x4 h) {
    return (double)h.x * (double)h.x + (double)h.y * (double)h.y + (double)h.z * (double)h.z + (double)h.w * (double)h.w;
}

/* Where a row's Q8_K blocks go. */
struct Q8kRow {
    int8_t *quants;
    int16_t *sums;
    float *scales;
};
Q38_DEV Q8kRow q8k_row(const q38_norm_args &a, int t) {
    const size_t n = (size_t)a.n_tokens * a.width, row = (size_t)t * a.width;
    int8_t *base = static_cast<int8_t *>(a.q8k);
    int16_t *sums = reinterpret_cast<int16_t *>(base + n);
    return {base + row, sums + row / 16, reinterpret_cast<float *>(sums + n / 16) + row / 256};
}

/* Block b of a row, held 4 values per lane by a wave. */
Q38_DEV void store_q8k(const Q8kRow &r, int b, int lane, f32x4 y) {
    int q[4];
    float scale;
    q38_wave_q8k(y, q, scale);
    reinterpret_cast<uint32_t *>(r.quants)[b * 64 + lane] =
        (uint32_t)(q[0] & 255) | (uint32_t)(q[1] & 255) << 8 | (uint32_t)(q[2] & 255) << 16 | (uint32_t)(q[3] & 255) << 24;
    int s = q[0] + q[1] + q[2] + q[3];
    s += __builtin_amdgcn_update_dpp(0, s, 0xB1, 0xF, 0xF, false);
    s += __builtin_amdgcn_update_dpp(0, s, 0x4E, 0xF, 0xF, false);
    if ((lane & 3) == 0) r.sums[b * 16 + (lane >> 2)] = (int16_t)s;
    if (lane == 0) r.scales[b] = scale;
}

/* A workgroup of NT threads per row, the row in registers: thread i holds
 * dims 4 (i + NT v) .. + 3, so a wave's v-th vectors are 256 consecutive dims,
 * a Q8_K block.  Every load is issued at once and every value read once, so
 * the kernel runs at the memory's rate: 4096 rows of 5120 with all outputs
 * (17.14 bytes a value) 67 us, 5.4 TB/s, 512 rows of 12288 to 20480 5.3 to 5.6
 * TB/s, rows and outputs that no cache holds; one row 3.5 us a call among others (the
 * kernel 3.3), where an empty launch takes about as long.  A first version that read its row twice and value by value took 187 us. */
template <int NT, int V>
Q38_DEV void norm_row(const q38_norm_args &a) {
    __shared__ double part[NT / 64];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 63, width = a.width;
    const size_t row = (size_t)t * width;
    const bool adds = a.residual != nullptr;
    /* 1024 threads of long rows: the weights come after the rows' registers are
     * added up, kAhead of them and one more a step, so that 64 registers do and
     * a CU holds two rows (509 rows of 17408 22.8 us against 26.6, one row 6.7
     * against 6.9; at 256 threads the same costs 70.0 against 67.9) */
    constexpr bool kLate = NT == 1024 && V > 3;
    constexpr int kAhead = 3;
    f32x4 h[V], r[V], w[V];
    /* threads past the row load its last vector and leave it out: no load
     * sits under a branch, so all of them are in flight together.  Nothing
     * reads these rows again, and loads that say so (non-temporal) keep them
     * from pushing the outputs out of the caches: 509 rows of 17408 from HBM
     * 28.7 us against 35.1, 256 rows 15.1 against 18.9; from the last level's
     * cache, as right after a small copy, they are slower (27.5 against 22.8,
     * 1024 rows of 5120 18.3 against 14.3), and with the residual's row
     * there and x's in HBM the two are even (after its producer 14.2 and 14.5 at
     * 256 rows of 5120, 87.1 and 87.5 at 4096) */
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = min(4 * (tid + NT * v), width - 4);
        h[v] = q38_ld4_stream(a.x + row + d);
        if (!kLate) w[v] = q38_ld4(a.weight + d);
    }
    if (adds) {
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = q38_ld4_stream(a.residual + row + min(4 * (tid + NT * v), width - 4));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] += r[v];
    }
    if (kLate) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int v = 0; v < kAhead; ++v) w[v] = q38_ld4(a.weight + min(4 * (tid + NT * v), width - 4));
    }
    double ss = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const double s = square_sum(h[v]);
        ss += 4 * (tid + NT * v) < width ? s : 0.0;
    }
    const float scale = norm_scale(block_sum_f64<NT>(ss, part), width);
    const Q8kRow q = q8k_row(a, t);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int d = 4 * (tid + NT * v);
        if (kLate && v + kAhead < V) w[v + kAhead] = q38_ld4(a.weight + min(4 * (tid + NT * (v + kAhead)), width - 4));
        if (d - 4 * lane >= width) break; /* past the row for the whole wave */
        const f32x4 y = h[v] * scale * w[v];
        if (d < width) {
            if (a.sum != nullptr) q38_st4(a.sum + row + d, h[v]);
            if (a.y != nullptr) q38_st4(a.y + row + d, y);
        }
        /* the width is a multiple of 256: the wave's 256 dims are all there */
        if (a.q8k != nullptr) store_q8k(q, d >> 8, lane, y);
        /* one block's quantiser at a time: run together they take registers
         * that more rows in flight need */
        __builtin_amdgcn_sched_barrier(0);
    }
}

/* Rows that are not whole aligned vectors, or too long for registers: the row
 * is read again after its sum (from the cache), value by value. */
Q38_DEV void norm_row_any(const q38_norm_args &a) {
    __shared__ double part[16];
    const int t = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, width = a.width;
    const size_t row = (size_t)t * width;
    double ss = 0.0;
    for (int d = threadIdx.x; d < width; d += 1024) {
        const float h = a.residual != nullptr ? a.x[row + d] + a.residual[row + d] : a.x[row + d];
        ss += (double)h * (double)h;
    }
    const float scale = norm_scale(block_sum_f64<1024>(ss, part), width);
    const Q8kRow q = q8k_row(a, t);
    /* a wave per 256 values, lane l: 4l .. 4l + 3.  A thread reads again only
     * what no other writes, so an output may be an input's own row. */
    for (int b = wave; b * 256 < width; b += 16) {
        f32x4 h = {0.f, 0.f, 0.f, 0.f}, y = h;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = b * 256 + 4 * lane + c;
            if (d < width) h[c] = a.residual != nullptr ? a.x[row + d] + a.residual[row + d] : a.x[row + d];
            if (d < width) y[c] = h[c] * scale * a.weight[d];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = b * 256 + 4 * lane + c;
            if (a.sum != nullptr && d < width) a.sum[row + d] = h[c];
            if (a.y != nullptr && d < width) a.y[row + d] = y[c];
        }
        if (a.q8k != nullptr) store_q8k(q, b, lane, y);
    }
}

}  // namespace

#define Q38_NORM_KERNEL(NT, V)                                                                              \
    extern "C" __global__ __launch_bounds__(NT, NT == 1024 ? 8 : 1) /* (waves a SIMD) */                    \
    void q38_add_rms_norm_##NT##_##V(Q38_NORM_PARAMS) {                                                     \
        norm_row<NT, V>(Q38_NORM_ARGS);                               \
    }
Q38_NORM_KERNEL(256, 1)
Q38_NORM_KERNEL(256, 2)
Q38_NORM_KERNEL(256, 3)
Q38_NORM_KERNEL(256, 4)
Q38_NORM_KERNEL(256, 5)
Q38_NORM_KERNEL(1024, 1)
Q38_NORM_KERNEL(1024, 2)
Q38_NORM_KERNEL(1024, 3)
Q38_NORM_KERNEL(1024, 4)
Q38_NORM_KERNEL(1024, 5)
extern "C" __global__ __launch_bounds__(1024) void q38_add_rms_norm_any(Q38_NORM_PARAMS) {
    norm_row_any(Q38_NORM_ARGS);
}

/* The values that Q8_K rows stand for: grid (ceil(n_tokens * width / 1024)),
 * 256 threads, 4 values each. */
extern "C" __global__ __launch_bounds__(256) void q38_dequantize_q8k(Q38_DEQUANTIZE_PARAMS) {
    const size_t total = (size_t)n[0] * n[1];
    const size_t i = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x);
    if (i >= total) return;
    const char *base = static_cast<const char *>(q8k);
    const uint32_t u = *reinterpret_cast<const uint32_t *>(base + i);
    const float s = reinterpret_cast<const float *>(base + total + total / 8)[i >> 8];
    f32x4 v;
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = (float)(int8_t)(u >> (8 * c)) * s;
    q38_st4(out + i, v);
}
