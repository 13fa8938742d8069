/*
 * The sums of attention weights of a tracking cache: in and out of its pages,
 * and the eviction of the tokens that have the least.
 *
 * Eviction is two launches.  The first finds, in each slot and kv head by itself, the
 * n_keep largest ranks of n and lists the holes below n_keep and the rows that go
 * there; the second moves those rows.  So n - n_keep rows at most are read, and no
 * more than n_keep written, and what stays below n_keep is not touched: packing all
 * rows in order would move every row behind the first hole, and its
 * reads and writes would lie in one another's way.
 *
 * Measured: a layer of 32K tokens to 8K, bf16: lists 22.3 us (four workgroups, one a kv head;
 * 16 layers' are 64 beside each other, in 24), 24.6K rows moved in
 * 24-30, for 81 MB read and 35 written past L2, 3.9-4.8 TB/s.  (The rows have 25 MB: their bytes
 * lie in nine of ten lines of the pages they come from.)  Eight sequences of 250 to
 * 4003 tokens of Q8_K to 60% of them 11.5 and 13.4.
 */
#include <type_traits>

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
    const size_t at = (size_t)a.page_table[(size_t)a.seq[b] * a.pt_stride + lp] * Q38_WEIGHTS_PAGE + j * Q38_WEIGHTS_HEAD + t;
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

/* Inclusive sum over the wave's lanes: within each row of 16, then a row's last
 * lane to the row after it, then the lower half's last to the upper half. */
template <int CTRL, int ROWS>
Q38_DEV uint32_t moved(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false);
}
Q38_DEV uint32_t wave_sum_to(uint32_t x) {
    x += moved<0x111, 0xF>(x); /* row_shr 1, 2, 4, 8 */
    x += moved<0x112, 0xF>(x);
    x += moved<0x114, 0xF>(x);
    x += moved<0x118, 0xF>(x);
    x += moved<0x142, 0xA>(x); /* row_bcast 15, 31 */
    return x + moved<0x143, 0xC>(x);
}
/* Exclusive sum over the workgroup's threads. */
Q38_DEV uint32_t scan(uint32_t x, uint32_t *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t sum = wave_sum_to(x);
    __syncthreads(); /* lds may still be read from the call before */
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) before += w < wave ? lds[w] : 0;
    return before + sum - x;
}

/* The same for kRounds values of each thread, all of a round before the next's:
 * x becomes the exclusive sums, and the total is returned.  (rounds: those that hold
 * anything but 0.) */
constexpr int kRounds = 8;
Q38_DEV uint32_t scan_rounds(uint32_t (&x)[kRounds], int rounds, uint32_t *lds) {
    static_assert(kRounds * kWaves == 128, "two a lane");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t sum[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) sum[r] = r < rounds ? wave_sum_to(x[r]) : 0;
    __syncthreads();
    if (lane == 63)
#pragma unroll
        for (int r = 0; r < kRounds; ++r) lds[r * kWaves + wave] = sum[r];
    __syncthreads();
    if (wave == 0) {
        const uint32_t a = lds[2 * lane], b = lds[2 * lane + 1], to = wave_sum_to(a + b);
        lds[2 * lane] = to - a - b;
        lds[2 * lane + 1] = to - b;
        if (lane == 63) lds[128] = to;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) x[r] = lds[r * kWaves + wave] + sum[r] - x[r];
    return lds[128];
}

/* The n_keep ranks that stay of n: the n_keep-th largest found digit by digit
 * (11, 11 and 10 bits, so that weights of one size spread over the bins), then in
 * one more pass which tokens those are -- all above it, and of those that equal it
 * the first -- and where the holes below n_keep and the tokens that fill them lie.
 * A block of 32768 tokens at a time, kRounds of four tokens to a thread (a page to
 * four of them: a thread a page read a line each, 64 to an instruction, and took
 * 32 us of 32K tokens where this takes 22); the first block's ranks stay in registers, a longer
 * context's others are formed again for each pass.  After the first digit few ranks
 * are left as a rule: up to kList of them are put together in LDS for the other two.
 * Tokens past the last one have rank 0, which none is below, and come after every
 * other of rank 0. */
constexpr int kBins = 2048, kList = 8192, kBlock = 4 * kRounds * kThreads;
typedef uint32_t Ranks[kRounds][4];
Q38_DEV void select(const q38_evict_args &a) {
    __shared__ uint32_t hist[kBins], list[kList];
    __shared__ uint32_t lds[kRounds * kWaves + 1], found[4], listed;
    const int x = blockIdx.x, b = blockIdx.y, slot = x >> 2, j = x & 3, tid = threadIdx.x;
    const int n = a.n_tokens[b], keep = a.n_keep[b], recent = a.first_recent[b], pages = (n + 15) >> 4;
    if (keep >= n || keep == 0) {
        if (tid == 0) a.counts[(size_t)b * gridDim.x + x] = 0;
        return;
    }
    const int32_t *pt = a.page_table + (size_t)a.seq[b] * a.pt_stride;
    const float *weights = a.weights + (size_t)slot * a.slot_weights + j * Q38_WEIGHTS_HEAD;
    const int32_t *tokens = a.tokens + (size_t)slot * a.slot_weights + j * Q38_WEIGHTS_HEAD;
    auto first_of = [&](int block, int r) { return block * kBlock + 4 * (r * kThreads + tid); }; /* a thread's four tokens */
    auto rounds_of = [&](int block) { return min((n - block * kBlock + 4 * kThreads - 1) / (4 * kThreads), kRounds); };
    auto load = [&](int block, Ranks &rank) {
        size_t at[kRounds];
        const int rounds = rounds_of(block);
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int t = first_of(block, r);
            if (r < rounds) at[r] = (size_t)pt[min(t >> 4, pages - 1)] * Q38_WEIGHTS_PAGE + (t & 15);
        }
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            if (r >= rounds) {
#pragma unroll
                for (int e = 0; e < 4; ++e) rank[r][e] = 0;
                continue;
            }
            const f32x4 w = q38_ld4(weights + at[r]);
            const q38_i32x4 own = *reinterpret_cast<const q38_i32x4 *>(tokens + at[r]);
#pragma unroll
            for (int e = 0; e < 4; ++e) rank[r][e] = first_of(block, r) + e < n ? rank_of(w[e], own[e], recent) : 0;
        }
    };
    Ranks held;
    load(0, held);
    auto each = [&](auto use) {
        use(0, held);
        for (int block = 1; block * kBlock < n; ++block) {
            Ranks rank;
            load(block, rank);
            use(block, rank);
        }
    };
    uint32_t prefix = 0, left = (uint32_t)keep; /* the largest digits so far, and ranks to take among those that share them */
    uint32_t known = 0;                         /* their bits */
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digit = pass == 2 ? 1023u : 2047u;
        for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
        if (pass == 1 && tid == 0) listed = 0;
        __syncthreads();
        /* every rank that has a token, and that shares the digits known so far */
        auto ranks = [&](auto use) {
            each([&](int block, const Ranks &rank) {
#pragma unroll
                for (int r = 0; r < kRounds; ++r)
                    if (first_of(block, r) < n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (pass == 0 || (rank[r][e] & known) == prefix) use(rank[r][e]);
            });
        };
        if (pass == 0 || found[2] > kList) {
            ranks([&](uint32_t rank) { atomicAdd(&hist[(rank >> shift) & digit], 1u); });
        } else {
            if (pass == 1) {
                /* a wave's at once (one by one took 2.5 us longer) */
                uint32_t mine = 0;
                ranks([&](uint32_t) { ++mine; });
                const uint32_t to = wave_sum_to(mine);
                uint32_t at = 0;
                if ((tid & 63) == 63) at = atomicAdd(&listed, to);
                at = __builtin_amdgcn_readlane(at, 63) + to - mine;
                ranks([&](uint32_t rank) { list[at++] = rank; });
                __syncthreads();
            }
            for (uint32_t i = tid; i < listed; i += kThreads)
                if ((list[i] & known) == prefix) atomicAdd(&hist[(list[i] >> shift) & digit], 1u);
        }
        __syncthreads();
        /* thread t: the bins kBins - 1 - 2 t and the one below it */
        const uint32_t c0 = hist[kBins - 1 - 2 * tid], c1 = hist[kBins - 2 - 2 * tid];
        const uint32_t above = scan(c0 + c1, lds);
        if (above < left && above + c0 + c1 >= left) {
            const bool upper = above + c0 >= left;
            found[0] = kBins - (upper ? 1 : 2) - 2 * tid;
            found[1] = left - above - (upper ? 0 : c0);
            if (pass == 0) found[2] = upper ? c0 : c1; /* ranks that share the first digit, */
            if (pass == 2) found[3] = upper ? c0 : c1; /* and all */
        }
        __syncthreads();
        prefix |= found[0] << shift;
        known |= digit << shift;
        left = found[1];
    }
    /* prefix: the smallest rank that stays; left of those that equal it do */
    int32_t *holes = a.moves + ((size_t)b * gridDim.x + x) * 2 * a.max_moves, *sources = holes + a.max_moves;
    const bool some = left < found[3];
    uint32_t equal_before = 0, holes_before = 0, sources_before = 0;
    each([&](int block, const Ranks &rank) {
        uint32_t stays[kRounds], count[kRounds];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            stays[r] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) stays[r] |= (rank[r][e] >= prefix ? 1u : 0u) << e;
        }
        if (some) { /* not all that equal it stay: the first ones do */
            uint32_t equal[kRounds];
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                equal[r] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) equal[r] |= (rank[r][e] == prefix ? 1u : 0u) << e;
                count[r] = __popc(equal[r]);
            }
            const uint32_t total = scan_rounds(count, rounds_of(block), lds);
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                uint32_t at = equal_before + count[r];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (equal[r] >> e & 1u) {
                        if (at >= left) stays[r] &= ~(1u << e);
                        ++at;
                    }
            }
            equal_before += total;
        }
        /* holes below n_keep and tokens that stay from there on, 32768 of either at most */
        uint32_t holes_of[kRounds];
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int t = first_of(block, r);
            const uint32_t low = (1u << min(max(keep - t, 0), 4)) - 1u, in = (1u << min(max(n - t, 0), 4)) - 1u;
            holes_of[r] = ~stays[r] & low;
            stays[r] &= in & ~low;
            count[r] = __popc(holes_of[r]) | __popc(stays[r]) << 16;
        }
        const uint32_t total = scan_rounds(count, rounds_of(block), lds);
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            /* a token is in the one list or in the other, by its side of n_keep: four are on one side but where
             * n_keep lies among them */
            const int t = first_of(block, r);
            int32_t *h = holes + holes_before + (count[r] & 0xFFFFu), *f = sources + sources_before + (count[r] >> 16);
            int32_t *out = t < keep ? h : f;
            const uint32_t listed_here = holes_of[r] | stays[r];
            if (__ballot(listed_here != 0) == 0) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (t + e == keep) out = f;
                if (listed_here >> e & 1u) *out++ = t + e;
            }
        }
        holes_before += total & 0xFFFFu;
        sources_before += total >> 16;
    });
    if (tid == 0) a.counts[(size_t)b * gridDim.x + x] = (int32_t)holes_before;
}

/* A row of one kv head on its way: what a wave's lane holds of it.  K goes in its
 * 16-byte pieces, V in the units that hold one token's values alone. */
template <int T>
struct Row {
    static constexpr int kPieces = T == Q38_KV_MX4 ? 8 : T == Q38_KV_Q8 ? 16 : 32;
    static constexpr int kUnits = T == Q38_KV_MX4 ? 2 : 4; /* of V, a lane */
    typedef std::conditional_t<T == Q38_KV_F16 || T == Q38_KV_BF16, uint16_t, uint8_t> Unit;
    q38_u32x4 k;
    Unit v[kUnits];
    uint32_t scale; /* lane 0 K's and lane 1 V's of 8-bit rows; of 4-bit ones lanes 0 .. 7 and 8 .. 15 */

    static Q38_DEV int unit(int i, int t, int lane) {
        if (T == Q38_KV_MX4) {
            const int u = 64 * i + lane;
            return q38_v_index<T>(t, (u >> 4) * 32 + (u & 15)) >> 1;
        }
        return q38_v_index<T>(t, 64 * i + lane);
    }
    Q38_DEV void load(char *kb, char *vb, int t, int head, int lane) {
        k = reinterpret_cast<const q38_u32x4 *>(kb)[min(lane, kPieces - 1) * 16 + t];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) v[i] = reinterpret_cast<const Unit *>(vb)[unit(i, t, lane)];
        if constexpr (T == Q38_KV_Q8) scale = __float_as_uint(q38_kv_scales(lane & 1 ? vb : kb, head)[t]);
        if constexpr (T == Q38_KV_MX4)
            scale = lane & 8 ? q38_mx4_scales(vb, head)[q38_mx4_v_scale(t, 32 * (lane & 7))] : q38_mx4_scales(kb, head)[q38_mx4_k_scale(t, 32 * (lane & 7))];
    }
    Q38_DEV void store(char *kb, char *vb, int t, int head, int lane) const {
        if (lane < kPieces) reinterpret_cast<q38_u32x4 *>(kb)[lane * 16 + t] = k;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) reinterpret_cast<Unit *>(vb)[unit(i, t, lane)] = v[i];
        if constexpr (T == Q38_KV_Q8) {
            if (lane < 2) q38_kv_scales(lane & 1 ? vb : kb, head)[t] = __uint_as_float(scale);
        }
        if constexpr (T == Q38_KV_MX4) {
            if (lane < 8) q38_mx4_scales(kb, head)[q38_mx4_k_scale(t, 32 * lane)] = (uint8_t)scale;
            else if (lane < 16) q38_mx4_scales(vb, head)[q38_mx4_v_scale(t, 32 * (lane & 7))] = (uint8_t)scale;
        }
    }
};

/* Holes lie below n_keep and the rows that fill them from there on: no row is read
 * that another move writes, so the moves run in any order, in place.  A wave a move,
 * of 4-bit rows two: a wave's chain is count - move - pages - rows, and 4-bit ones are too few
 * bytes to fill it (16 layers of 32K tokens to 8K: one / two / four / eight a wave 195 /
 * 158 / 165 / 177 us, to 24K 209 / 164 / 195 / 202; of bf16 462 / 488 / - / -, 691 /
 * 704, Q8_K 265 / 271, 354 / 366).  A row's elements lie
 * among its page's (q38_kv_layout.h), so a line comes in for each sixteenth of a key
 * and each 64 bytes of a value that move; an XCD takes an eighth of a list in one
 * piece, so that neighbours find their lines in its L2 (one layer of bf16 reads 81 MB and
 * writes 35 against 91 and 39, of which a quarter as many requests for parts of 64 bytes; 16
 * layers 462 us against 487, 691 against 753, Q8_K 265 against 278, 354 against 370). */
template <int T>
constexpr int kRowsOf = T == Q38_KV_MX4 ? Q38_EVICT_MX4 : 1;
template <int T>
Q38_DEV void move_rows(const q38_evict_args &a) {
    const int x = blockIdx.y, b = blockIdx.z, slot = x >> 2, j = x & 3;
    const int tid = threadIdx.x, lane = tid & 63;
    constexpr int kRows = kRowsOf<T>, kAll = Q38_EVICT_WAVES * kRows;
    const int n = a.counts[(size_t)b * gridDim.y + x], each = (n + 8 * kAll - 1) / (8 * kAll), u = blockIdx.x >> 3;
    const int i = ((blockIdx.x & 7) * each + u) * kAll + __builtin_amdgcn_readfirstlane(tid >> 6) * kRows;
    if (u >= each || i >= n) return;
    const int32_t *holes = a.moves + ((size_t)b * gridDim.y + x) * 2 * a.max_moves, *sources = holes + a.max_moves;
    const int32_t *pt = a.page_table + (size_t)a.seq[b] * a.pt_stride;
    char *k = a.kpool + (size_t)slot * a.slot_bytes, *v = a.vpool + (size_t)slot * a.slot_bytes;
    Row<T> row[kRows];
    int page1[kRows], page0[kRows], t1[kRows], t0[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) { /* (past the last: that one again, read but not stored) */
        const int at = min(i + r, n - 1), to = holes[at], from = sources[at];
        page1[r] = pt[to >> 4];
        page0[r] = pt[from >> 4];
        t1[r] = to & 15;
        t0[r] = from & 15;
    }
    const size_t first = (size_t)slot * a.slot_weights + j * Q38_WEIGHTS_HEAD;
    float weight[kRows];
    int32_t token[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        row[r].load(q38_kv_block<T>(k, page0[r], j), q38_kv_block<T>(v, page0[r], j), t0[r], j, lane);
        const size_t source = first + (size_t)page0[r] * Q38_WEIGHTS_PAGE + t0[r];
        weight[r] = a.weights[source];
        token[r] = a.tokens[source];
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (i + r >= n) return;
        row[r].store(q38_kv_block<T>(k, page1[r], j), q38_kv_block<T>(v, page1[r], j), t1[r], j, lane);
        if (lane == 0) {
            const size_t hole = first + (size_t)page1[r] * Q38_WEIGHTS_PAGE + t1[r];
            a.weights[hole] = weight[r];
            a.tokens[hole] = token[r];
        }
    }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void q38_kv_weights_copy(q38_kv_weights_args a) { copy_weights(a); }
extern "C" __global__ __launch_bounds__(kThreads) void q38_kv_evict_select(q38_evict_args a) { select(a); }
extern "C" __global__ __launch_bounds__(64 * Q38_EVICT_WAVES) void q38_kv_evict_move_f16(q38_evict_args a) { move_rows<Q38_KV_F16>(a); }
extern "C" __global__ __launch_bounds__(64 * Q38_EVICT_WAVES) void q38_kv_evict_move_bf16(q38_evict_args a) { move_rows<Q38_KV_BF16>(a); }
extern "C" __global__ __launch_bounds__(64 * Q38_EVICT_WAVES) void q38_kv_evict_move_q8k(q38_evict_args a) { move_rows<Q38_KV_Q8>(a); }
extern "C" __global__ __launch_bounds__(64 * Q38_EVICT_WAVES) void q38_kv_evict_move_mxfp4(q38_evict_args a) { move_rows<Q38_KV_MX4>(a); }
