/*
 * The sums of attention weights of a tracking cache: in and out of its pages,
 * and the eviction of the tokens that have the least.
 */
#include "q38_kv_types.h"

namespace {

/* A wave a page, lane 4 t + j token t of kv head j: rows are whole lines. */
Q38_DEV void copy_weights(const q38_kv_weights_args &a) {
    const int x = 4 * blockIdx.x + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (x >= a.page_base[a.n_seq]) return;
    int b = 0;
    for (int i0 = 1; i0 < a.n_seq; i0 += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) b += a.page_base[i0 + i] <= x ? 1 : 0;
    const int first = a.pos0[b], n = a.row_base[b + 1] - a.row_base[b];
    const int lp = (first >> 4) + x - a.page_base[b], t = lane >> 2, j = lane & 3, p = lp * Q38_PAGE_TOKENS + t;
    if (p < first || p >= first + n) return;
    const size_t at = (size_t)a.page_table[(size_t)a.seq[b] * a.pt_stride + lp] * Q38_WEIGHTS_PAGE + j * Q38_PAGE_TOKENS + t;
    const size_t row = (size_t)(a.row_base[b] + p - first) * Q38_ATTN_KV_HEADS + j;
    if (a.to_pages) {
        a.weights[at] = a.weight_rows != nullptr ? a.weight_rows[row] : 0.0f;
        a.tokens[at] = a.token_rows != nullptr ? a.token_rows[row] : p + a.evicted[b];
    } else {
        if (a.weight_rows != nullptr) a.weight_rows[row] = a.weights[at];
        if (a.token_rows != nullptr) a.token_rows[row] = a.tokens[at];
    }
}

/* Order of eviction as a whole number: larger stays.  Tokens from first_recent on
 * above all, then by weight, both zeros alike, NaN below every number. */
Q38_DEV uint32_t rank_of(float w, int token, int first_recent) {
    if (token >= first_recent) return ~0u;
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kThreads = 1024, kWaves = kThreads / 64;

/* Exclusive sum over the workgroup's threads, and the total. */
Q38_DEV uint32_t scan(uint32_t x, uint32_t *lds, uint32_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t y = __shfl_up(sum, d, 64);
        if (lane >= d) sum += y;
    }
    __syncthreads(); /* lds may still be read from the call before */
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const uint32_t y = lds[w];
        before += w < wave ? y : 0;
        total += y;
    }
    return before + sum - x;
}

/* The n_keep ranks that stay of n: the n_keep-th largest found digit by digit
 * (eight bits a pass over the sums), then in one more pass which tokens those are --
 * all above it, and of those that equal it the first -- and where the holes below
 * n_keep and the tokens that fill them lie.  A thread has a page's 16 tokens. */
Q38_DEV void select(const q38_evict_args &a) {
    __shared__ uint32_t hist[kWaves][256];
    __shared__ uint32_t lds[kWaves], found[2];
    const int x = blockIdx.x, b = blockIdx.y, slot = x >> 2, j = x & 3, tid = threadIdx.x, wave = tid >> 6;
    const int n = a.n_tokens[b], keep = a.n_keep[b], recent = a.first_recent[b], pages = (n + 15) >> 4;
    if (keep >= n) {
        if (tid == 0) a.counts[(size_t)b * gridDim.x + x] = 0;
        return;
    }
    const int32_t *pt = a.page_table + (size_t)a.seq[b] * a.pt_stride;
    const float *weights = a.weights + (size_t)slot * a.slot_weights + j * Q38_PAGE_TOKENS;
    const int32_t *tokens = a.tokens + (size_t)slot * a.slot_weights + j * Q38_PAGE_TOKENS;
    auto load = [&](int page, uint32_t (&rank)[16]) {
        const size_t at = (size_t)pt[page] * Q38_WEIGHTS_PAGE;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 w = q38_ld4(weights + at + 4 * i);
            const q38_i32x4 t = *reinterpret_cast<const q38_i32x4 *>(tokens + at + 4 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) rank[4 * i + e] = rank_of(w[e], t[e], recent);
        }
    };
    uint32_t prefix = 0, left = (uint32_t)keep; /* the largest digits so far, and ranks to take among those that share them */
    for (int shift = 24; keep > 0 && shift >= 0; shift -= 8) {
        for (int i = tid; i < kWaves * 256; i += kThreads) (&hist[0][0])[i] = 0;
        __syncthreads();
        for (int page = tid; page < pages; page += kThreads) {
            uint32_t rank[16];
            load(page, rank);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (16 * page + i < n && (shift == 24 || rank[i] >> (shift + 8) == prefix >> (shift + 8)))
                    atomicAdd(&hist[wave][(rank[i] >> shift) & 255u], 1u);
        }
        __syncthreads();
        /* thread d: how many have digit 255 - d */
        uint32_t count = 0, total;
        if (tid < 256)
#pragma unroll
            for (int w = 0; w < kWaves; ++w) count += hist[w][255 - tid];
        const uint32_t above = scan(count, lds, total);
        if (tid < 256 && above < left && above + count >= left) {
            found[0] = 255 - tid;
            found[1] = left - above;
        }
        __syncthreads();
        prefix |= found[0] << shift;
        left = found[1];
    }
    /* prefix: the smallest rank that stays; left of those that equal it do */
    int32_t *holes = a.moves + ((size_t)b * gridDim.x + x) * 2 * a.max_moves, *sources = holes + a.max_moves;
    uint32_t equal_before = 0, holes_before = 0, sources_before = 0;
    for (int page0 = 0; page0 < pages; page0 += kThreads) {
        const int page = page0 + tid;
        uint32_t above = 0, equal = 0, total;
        if (page < pages) {
            uint32_t rank[16];
            load(page, rank);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool in = 16 * page + i < n && keep > 0;
                above |= (in && rank[i] > prefix ? 1u : 0u) << i;
                equal |= (in && rank[i] == prefix ? 1u : 0u) << i;
            }
        }
        uint32_t rest = equal_before + scan((uint32_t)__popc(equal), lds, total);
        equal_before += total;
        uint32_t stays = above;
        for (uint32_t e = equal; e != 0 && rest < left; ++rest, e &= e - 1) stays |= e & (0u - e);
        const int below = min(max(keep - 16 * page, 0), 16), count = min(max(n - 16 * page, 0), 16);
        const uint32_t low = (1u << below) - 1u, all = (1u << count) - 1u;
        uint32_t hole = ~stays & low & all, source = stays & ~low & all;
        const uint32_t h = scan((uint32_t)__popc(hole), lds, total);
        int at = (int)(holes_before + h);
        holes_before += total;
        for (; hole != 0; hole &= hole - 1) holes[at++] = 16 * page + __builtin_ctz(hole);
        const uint32_t s = scan((uint32_t)__popc(source), lds, total);
        at = (int)(sources_before + s);
        sources_before += total;
        for (; source != 0; source &= source - 1) sources[at++] = 16 * page + __builtin_ctz(source);
    }
    if (tid == 0) a.counts[(size_t)b * gridDim.x + x] = (int32_t)holes_before;
}

/* A row of one kv head from one place to another: a wave.  K moves in its 16-byte
 * pieces, V in the units that hold one token's values alone. */
template <int T>
Q38_DEV void move_row(const char *from, int t0, char *to, int t1, bool key, int head, int lane) {
    if (key) {
        constexpr int kPieces = T == Q38_KV_MX4 ? 8 : T == Q38_KV_Q8 ? 16 : 32;
        if (lane < kPieces)
            reinterpret_cast<q38_u32x4 *>(to)[lane * 16 + t1] = reinterpret_cast<const q38_u32x4 *>(from)[lane * 16 + t0];
    } else {
#pragma unroll
        for (int i = 0; i < (T == Q38_KV_MX4 ? 2 : 4); ++i) {
            if constexpr (T == Q38_KV_MX4) {
                const int u = 64 * i + lane, d = (u >> 4) * 32 + (u & 15);
                to[q38_v_index<T>(t1, d) >> 1] = from[q38_v_index<T>(t0, d) >> 1];
            } else if constexpr (T == Q38_KV_Q8) {
                to[q38_v_index<T>(t1, 64 * i + lane)] = from[q38_v_index<T>(t0, 64 * i + lane)];
            } else {
                reinterpret_cast<uint16_t *>(to)[q38_v_index<T>(t1, 64 * i + lane)] =
                    reinterpret_cast<const uint16_t *>(from)[q38_v_index<T>(t0, 64 * i + lane)];
            }
        }
    }
    if constexpr (T == Q38_KV_Q8) {
        if (lane == 0) q38_kv_scales(to, head)[t1] = q38_kv_scales(const_cast<char *>(from), head)[t0];
    }
    if constexpr (T == Q38_KV_MX4) {
        const uint8_t *s = q38_mx4_scales(const_cast<char *>(from), head);
        uint8_t *r = q38_mx4_scales(to, head);
        if (lane < 8)
            r[key ? q38_mx4_k_scale(t1, 32 * lane) : q38_mx4_v_scale(t1, 32 * lane)] =
                s[key ? q38_mx4_k_scale(t0, 32 * lane) : q38_mx4_v_scale(t0, 32 * lane)];
    }
}

/* Holes lie below n_keep and the rows that fill them from there on: no row is read
 * that another move writes, so the moves run in any order, in place. */
template <int T>
Q38_DEV void move_rows(const q38_evict_args &a) {
    const int x = blockIdx.y, b = blockIdx.z, slot = x >> 2, j = x & 3;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int count = a.counts[(size_t)b * gridDim.y + x], begin = blockIdx.x * Q38_EVICT_ROWS;
    const int32_t *holes = a.moves + ((size_t)b * gridDim.y + x) * 2 * a.max_moves, *sources = holes + a.max_moves;
    const int32_t *pt = a.page_table + (size_t)a.seq[b] * a.pt_stride;
    char *k = a.kpool + (size_t)slot * a.slot_bytes, *v = a.vpool + (size_t)slot * a.slot_bytes;
    for (int i = begin + wave; i < min(begin + Q38_EVICT_ROWS, count); i += 4) {
        const int p1 = holes[i], p0 = sources[i], g0 = pt[p0 >> 4], g1 = pt[p1 >> 4], t0 = p0 & 15, t1 = p1 & 15;
        move_row<T>(q38_kv_block<T>(k, g0, j), t0, q38_kv_block<T>(k, g1, j), t1, true, j, lane);
        move_row<T>(q38_kv_block<T>(v, g0, j), t0, q38_kv_block<T>(v, g1, j), t1, false, j, lane);
        if (lane == 0) {
            const size_t from = (size_t)slot * a.slot_weights + (size_t)g0 * Q38_WEIGHTS_PAGE + j * Q38_PAGE_TOKENS + t0;
            const size_t to = (size_t)slot * a.slot_weights + (size_t)g1 * Q38_WEIGHTS_PAGE + j * Q38_PAGE_TOKENS + t1;
            a.weights[to] = a.weights[from];
            a.tokens[to] = a.tokens[from];
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void q38_kv_weights_copy(q38_kv_weights_args a) { copy_weights(a); }
extern "C" __global__ __launch_bounds__(kThreads) void q38_kv_evict_select(q38_evict_args a) { select(a); }
extern "C" __global__ __launch_bounds__(256) void q38_kv_evict_move_f16(q38_evict_args a) { move_rows<Q38_KV_F16>(a); }
extern "C" __global__ __launch_bounds__(256) void q38_kv_evict_move_bf16(q38_evict_args a) { move_rows<Q38_KV_BF16>(a); }
extern "C" __global__ __launch_bounds__(256) void q38_kv_evict_move_q8k(q38_evict_args a) { move_rows<Q38_KV_Q8>(a); }
extern "C" __global__ __launch_bounds__(256) void q38_kv_evict_move_mxfp4(q38_evict_args a) { move_rows<Q38_KV_MX4>(a); }
