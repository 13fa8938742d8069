// Host-side check of 4-bit pages and of the calls on sums of attention weights
// (q38_kv_track_weights, q38_kv_weights_put / get, q38_attn_observe, q38_kv_evict,
// and decode on a tracking cache), on the CPU: the library's source compiled into
// this program, its launches answered here.  Every launch's arguments are walked
// as the kernels walk them, each access inside what was allocated; refused calls
// launch nothing and leave pages, sequences and evicted counts as they were.
#include <hip/hip_runtime_api.h>

#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>
#include <string>
#include <vector>

#include "q38_kv_layout.h"

struct Launch {
    hipFunction_t f;
    unsigned gx, gy, gz, block;
    std::vector<std::vector<char>> args;
};
static std::vector<Launch> g_launches;
static size_t (*g_arg_bytes)(hipFunction_t, int);
static hipError_t check_launch(hipFunction_t f, unsigned gx, unsigned gy, unsigned gz, unsigned block, unsigned, unsigned, unsigned,
                               hipStream_t, void **params, void **) {
    Launch l{f, gx, gy, gz, block, {}};
    for (int i = 0; i < 2; ++i)
        if (const size_t n = g_arg_bytes(f, i)) l.args.emplace_back((char *)params[i], (char *)params[i] + n);
    g_launches.push_back(l);
    return hipSuccess;
}
static uintptr_t g_next = 0x100000000000ull;
static std::vector<std::pair<uintptr_t, size_t>> g_allocated;
template <typename T>
static hipError_t check_malloc(T **p, size_t bytes) {
    *p = reinterpret_cast<T *>(g_next);
    g_allocated.push_back({g_next, bytes});
    g_next += (bytes + 0xFFFFFFF) & ~(size_t)0xFFFFFFF;
    return hipSuccess;
}
static hipError_t check_free(void *) { return hipSuccess; }
static hipError_t check_copy(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
static hipError_t check_set(void *, int, size_t, hipStream_t) { return hipSuccess; }
static hipError_t check_sync(hipStream_t) { return hipSuccess; }
static hipStreamCaptureStatus g_capture = hipStreamCaptureStatusNone;
static hipError_t check_capturing(hipStream_t, hipStreamCaptureStatus *status) {
    *status = g_capture;
    return hipSuccess;
}
#define hipMalloc check_malloc
#define hipFree check_free
#define hipMemsetAsync check_set
#define hipStreamIsCapturing check_capturing
#define hipModuleLaunchKernel check_launch
#define hipMemcpyAsync check_copy
#define hipStreamSynchronize check_sync
#include "../../qwen3.8_27b_in_rust_amd/csrc/host/q38_attn.cpp"

int q38_scratch_address(int, void **ptr) {
    *ptr = nullptr;
    return -1;
}

#define REQUIRE(c)                                                                               \
    do {                                                                                         \
        if (!(c)) { printf("line %d: %s (%s)\n", __LINE__, #c, q38_last_error()); exit(1); }     \
    } while (0)

static hipFunction_t const kCopy = (hipFunction_t)0x1000, kSelect = (hipFunction_t)0x2000, kMove = (hipFunction_t)0x3000,
                           kStats = (hipFunction_t)0x4000, kSums = (hipFunction_t)0x5000, kWeigh = (hipFunction_t)0x6000,
                           kWeighMerge = (hipFunction_t)0x7000, kRows = (hipFunction_t)0x8000, kAdd = (hipFunction_t)0x9000;
static size_t arg_bytes(hipFunction_t f, int i) {
    if (f == kWeigh) return i ? sizeof(q38_weigh_args) : sizeof(q38_decode_typed_args);
    if (f == kWeighMerge) return i ? sizeof(q38_weigh_merge_args) : sizeof(q38_merge_args);
    if (i) return 0;
    if (f == kCopy) return sizeof(q38_kv_weights_args);
    if (f == kSelect || f == kMove) return sizeof(q38_evict_args);
    if (f == kStats || f == kSums || f == kAdd) return sizeof(q38_observe_args);
    return 0;
}
template <typename T>
static T arg(const Launch &l, int i = 0) {
    T a;
    REQUIRE(l.args.at(i).size() == sizeof(T));
    memcpy(&a, l.args[i].data(), sizeof(T));
    return a;
}
static bool inside(const void *p, size_t bytes) {
    for (auto &a : g_allocated)
        if ((uintptr_t)p >= a.first && (uintptr_t)p + bytes <= a.first + a.second) return true;
    return false;
}

static void check_layout() {
    constexpr int T = Q38_KV_MX4;
    std::set<int> k, v, ks, vs;
    for (int t = 0; t < 16; ++t)
        for (int d = 0; d < 256; ++d) {
            k.insert(q38_k_index<T>(t, d));
            v.insert(q38_v_index<T>(t, d));
            ks.insert(q38_mx4_k_scale(t, d));
            vs.insert(q38_mx4_v_scale(t, d));
            /* four dims of a key in order in 16 bits; a value and its partner 16 dims on in a byte */
            if (d % 4 == 0) REQUIRE(q38_k_index<T>(t, d) % 4 == 0 && q38_k_index<T>(t, d + 3) == q38_k_index<T>(t, d) + 3);
            if (d % 32 < 16) REQUIRE(q38_v_index<T>(t, d) % 2 == 0 && q38_v_index<T>(t, d + 16) == q38_v_index<T>(t, d) + 1);
            /* the byte of token t of a word of values is the byte of its scale's word */
            REQUIRE((q38_v_index<T>(t, d) / 2) % 4 == q38_mx4_v_scale(t, d) % 4);
        }
    REQUIRE(k.size() == 4096 && *k.rbegin() == 4095 && v.size() == 4096 && *v.rbegin() == 4095);
    REQUIRE(ks.size() == 128 && *ks.rbegin() == 127 && vs.size() == 128 && *vs.rbegin() == 127);
    REQUIRE(q38_kv_block_bytes<T>() == 2048 && q38_kv_page_bytes<T>() == Q38_KV_PAGE_MX4 && Q38_KV_PAGE_MX4 == 4 * (2048 + 128));
    for (int head = 0; head < 4; ++head) /* past the four blocks, inside the page */
        REQUIRE(head * 2048 + q38_mx4_scales_offset(head) == 4 * 2048 + 128 * head);
}

struct Cache {
    q38_ctx ctx;
    q38_kv *kv = nullptr;
    std::vector<int32_t> staging;
    Cache(int type, int slots, int pages, int seqs, int tokens) {
        ctx.cu_count = 256;
        ctx.f_weights_copy = kCopy;
        ctx.f_evict_select = kSelect;
        ctx.f_weigh_merge = kWeighMerge;
        ctx.f_observe_add = kAdd;
        for (int i = 0; i < kKvTypeCount; ++i) {
            ctx.f_evict_move[i] = kMove;
            for (int v = 0; v < 2; ++v) {
                ctx.f_observe_stats[i][v][0] = ctx.f_observe_stats[i][v][1] = kStats;
                ctx.f_observe_sums[i][v] = kSums;
                ctx.f_weigh[i][v] = kWeigh;
            }
            for (q38_ctx::RowsKernel *k : {&ctx.f_kv_append[i], &ctx.f_kv_gather[i]}) k->many = k->few = kRows;
        }
        kv = new q38_kv;
        kv->ctx = &ctx;
        kv->type = type;
        kv->n_slots = slots;
        kv->max_pages = pages;
        kv->max_seqs = seqs;
        kv->pt_stride = (tokens + 15) / 16;
        check_malloc(&kv->kpool, slots * kv->slot_bytes());
        check_malloc(&kv->vpool, slots * kv->slot_bytes());
        check_malloc(&kv->d_page_table, (size_t)seqs * kv->pt_stride * 4);
        kv->page_table.assign((size_t)seqs * kv->pt_stride, -1);
        for (int p = pages - 1; p >= 0; --p) kv->free_pages.push_back(p);
        kv->seq_live.assign(seqs, 0);
        kv->seq_pages.assign(seqs, 0);
        kv->images.assign((size_t)seqs * slots, q38_kv::Images());
        staging.resize(1 << 20);
        kv->staging = staging.data();
        kv->staging_len = staging.size();
    }
    std::vector<int32_t> snapshot() const {
        std::vector<int32_t> s = kv->page_table;
        s.insert(s.end(), kv->free_pages.begin(), kv->free_pages.end());
        s.insert(s.end(), kv->seq_pages.begin(), kv->seq_pages.end());
        for (auto &e : kv->evicted) s.push_back(e.tokens), s.push_back(e.kept);
        s.push_back(kv->tracks);
        return s;
    }
    /* the sum of (position, head) of a sequence in a slot */
    const float *sum_at(int slot, int seq, int p, int j) const {
        const int page = kv->page_table[(size_t)seq * kv->pt_stride + p / 16];
        REQUIRE(page >= 0 && page < kv->max_pages);
        return kv->weights + (size_t)slot * kv->slot_sums() + (size_t)page * Q38_WEIGHTS_PAGE + j * Q38_WEIGHTS_HEAD + p % 16;
    }
};

/* A copy's launches walked as the kernel does: every row once, in order. */
static void walk_copy(const Cache &c, size_t from, int slot, const std::vector<int32_t> &seq, const std::vector<int32_t> &pos,
                      const std::vector<int32_t> &cnt, const float *d_w, const int32_t *d_t, bool to_pages) {
    std::vector<std::pair<int, int>> want;
    for (size_t b = 0; b < seq.size(); ++b)
        for (int i = 0; i < cnt[b]; ++i) want.push_back({seq[b], pos[b] + i});
    std::vector<int> moved(want.size(), 0);
    size_t before = 0;
    for (size_t l = from; l < g_launches.size(); ++l) {
        REQUIRE(g_launches[l].f == kCopy && g_launches[l].block == 256 && g_launches[l].gy == 1);
        const auto a = arg<q38_kv_weights_args>(g_launches[l]);
        REQUIRE(a.to_pages == (to_pages ? 1 : 0) && a.n_seq >= 1 && a.n_seq <= Q38_MAX_BATCH);
        REQUIRE(a.weight_rows == (d_w ? d_w + before * 4 : nullptr) && a.token_rows == (d_t ? d_t + before * 4 : nullptr));
        REQUIRE(a.weights == c.kv->weights_of(slot) && (float *)a.tokens == a.weights + 16);
        for (int x = 0; x < (int)g_launches[l].gx * 4; ++x) {
            if (x >= a.page_base[a.n_seq]) continue;
            int b = 0;
            for (int i0 = 1; i0 < a.n_seq; i0 += 8)
                for (int i = 0; i < 8; ++i) b += a.page_base[i0 + i] <= x ? 1 : 0;
            REQUIRE(b < a.n_seq);
            const int first = a.pos0[b], n = a.row_base[b + 1] - a.row_base[b], lp = (first >> 4) + x - a.page_base[b];
            for (int t = 0; t < 16; ++t) {
                const int p = lp * 16 + t;
                if (p < first || p >= first + n) continue;
                const size_t row = before + a.row_base[b] + p - first;
                REQUIRE(row < want.size() && want[row].first == a.seq[b] && want[row].second == p);
                REQUIRE(a.evicted[b] == c.kv->evicted_of(a.seq[b]));
                for (int j = 0; j < 4; ++j) REQUIRE(inside(c.sum_at(slot, a.seq[b], p, j), 4) && inside(c.sum_at(slot, a.seq[b], p, j) + 16, 4));
                ++moved[row];
            }
        }
        before += a.row_base[a.n_seq];
    }
    for (int m : moved) REQUIRE(m == 1);
}

int main() {
    g_arg_bytes = arg_bytes;
    check_layout();
    srand(11);
    float *d_w = reinterpret_cast<float *>(0x50000000000ull);
    int32_t *d_t = reinterpret_cast<int32_t *>(0x60000000000ull);
    for (int type = 1; type < kKvTypeCount; ++type) {
        Cache c(type, 2, 8000, 150, 25000);
        q38_kv *kv = c.kv;
        std::vector<int> ids;
        for (int i = 0; i < 150; ++i) {
            int s;
            REQUIRE(q38_seq_create(kv, &s) == 0 && q38_seq_reserve(kv, s, 16 + rand() % 380) == 0);
            ids.push_back(s);
        }
        int n_out = -1;
        REQUIRE(q38_seq_evicted(kv, ids[0], &n_out) == 0 && n_out == 0);
        const int32_t one = ids[0], zero = 0, three = 3;
        REQUIRE(q38_kv_weights_get(kv, 3, 1, &one, &zero, &three, d_w, d_t) == -1 && strstr(q38_last_error(), "does not track"));
        /* tracking on: what is held gets its positions, in every slot */
        g_launches.clear();
        REQUIRE(q38_kv_track_weights(kv, 1) == 0 && g_launches.size() == 300);
        REQUIRE(q38_kv_track_weights(kv, 1) == 0 && g_launches.size() == 300);
        for (int it = 0; it < 40; ++it) {
            std::vector<int32_t> seq(ids.begin(), ids.end()), pos, cnt;
            for (size_t i = seq.size() - 1; i > 0; --i) std::swap(seq[i], seq[rand() % (i + 1)]);
            seq.resize(1 + rand() % (it % 3 == 0 ? 12 : seq.size()));
            for (int s : seq) {
                const int held = kv->seq_pages[s] * 16;
                pos.push_back(rand() % held);
                cnt.push_back(rand() % 4 ? rand() % (held - pos.back() + 1) : 0);
            }
            const bool to = it & 1;
            g_launches.clear();
            const int rc = to ? q38_kv_weights_put(kv, 7, (int)seq.size(), seq.data(), pos.data(), cnt.data(), it % 4 == 1 ? nullptr : d_w, it % 8 > 3 ? nullptr : d_t)
                              : q38_kv_weights_get(kv, 7, (int)seq.size(), seq.data(), pos.data(), cnt.data(), d_w, it % 8 > 3 ? nullptr : d_t);
            REQUIRE(rc == 0);
            walk_copy(c, 0, 1, seq, pos, cnt, to && it % 4 == 1 ? nullptr : d_w, it % 8 > 3 ? nullptr : d_t, to);
        }
        /* a decode step: the launch and its merge over more sequences than one takes */
        for (int split : {0, 16, 512}) {
            c.ctx.split_tokens = split;
            std::vector<int32_t> seq(ids.begin(), ids.begin() + 70), pos;
            for (int s : seq) pos.push_back(rand() % (kv->seq_pages[s] * 16));
            g_launches.clear();
            const float *q = reinterpret_cast<float *>(0x70000000000ull);
            REQUIRE(q38_attn_decode(kv, 3, 70, seq.data(), pos.data(), q, nullptr, nullptr, nullptr, const_cast<float *>(q)) == 0);
            size_t l = 0;
            for (int b0 = 0; b0 < 70; b0 += Q38_MAX_BATCH) {
                REQUIRE(l < g_launches.size() && g_launches[l].f == kWeigh);
                const auto a = arg<q38_decode_typed_args>(g_launches[l]);
                const auto w = arg<q38_weigh_args>(g_launches[l], 1);
                REQUIRE(a.n_seq == std::min(70 - b0, Q38_MAX_BATCH) && w.weights == kv->weights_of(0) && w.tokens == kv->tokens_of(0));
                /* sequences of one split add their weights themselves */
                if (a.total_splits == a.n_seq) {
                    ++l;
                    REQUIRE(inside(w.scores, (size_t)a.total_splits * (a.split_tokens / 16) * 4 * Q38_SCORES_PAGE * 4));
                    continue;
                }
                REQUIRE(l + 1 < g_launches.size());
                const auto m = arg<q38_merge_args>(g_launches[l + 1]);
                const auto mw = arg<q38_weigh_merge_args>(g_launches[l + 1], 1);
                REQUIRE(g_launches[l].f == kWeigh && g_launches[l].gx == (unsigned)a.total_splits && g_launches[l].block == 512);
                REQUIRE(g_launches[l + 1].f == kWeighMerge && g_launches[l + 1].gx == (unsigned)(96 * a.n_seq + 4 * a.total_splits));
                REQUIRE(w.scores == mw.scores && mw.split_tokens == a.split_tokens && m.n_seq == a.n_seq && mw.appended == 0);
                REQUIRE(m.part_ml == a.part_ml && m.split_base[m.n_seq] == a.total_splits);
                /* the partials, then the scores of every split's pages, inside the workspace and apart */
                const size_t parts = (size_t)a.total_splits * 24 * 258 * 4, pages = (size_t)a.total_splits * (a.split_tokens / 16);
                REQUIRE((char *)w.scores == (char *)a.part_o + parts && (char *)a.part_ml == (char *)a.part_o + (size_t)a.total_splits * 24 * 256 * 4);
                REQUIRE(inside(a.part_o, parts + pages * 4 * Q38_SCORES_PAGE * 4));
                for (int b = 0; b < a.n_seq; ++b) {
                    REQUIRE(mw.seq[b] == a.seq[b] && mw.pos[b] == a.pos[b] && a.pos[b] / 16 < kv->seq_pages[a.seq[b]]);
                    REQUIRE(m.split_base[b] == a.split_base[b]);
                    REQUIRE((a.split_base[b + 1] - a.split_base[b]) == (a.pos[b] + a.split_tokens) / a.split_tokens);
                }
                l += 2;
            }
            REQUIRE(l == g_launches.size());
        }
        c.ctx.split_tokens = 0;
        /* a prompt's queries: every page of every group in one split of either launch, statistics inside the workspace */
        int big;
        REQUIRE(q38_seq_free(kv, ids.back()) == 0 && q38_seq_create(kv, &big) == 0);
        for (int held : {16, 200, 4096, 24576, 24577}) {
            REQUIRE(q38_seq_reset(kv, big) == 0 && q38_seq_reserve(kv, big, held) == 0);
            for (int n : {1, 16, 17, 160, 4096}) {
                if (n > held) continue;
                const float *q = reinterpret_cast<float *>(0x70000000000ull);
                g_launches.clear();
                REQUIRE(q38_attn_observe(kv, 3, big, held - n, n, q) == 0 && g_launches.size() >= 2);
                const auto a = arg<q38_observe_args>(g_launches[0]), s = arg<q38_observe_args>(g_launches[1]);
                const int pages = (held + 15) / 16, groups = (n + 15) / 16;
                if (g_launches[1].f == kAdd) {
                    /* scores kept: every group in one batch, its statistics and scores inside the workspace */
                    int next = 0;
                    for (size_t l = 0; l < g_launches.size(); l += 2) {
                        const auto x = arg<q38_observe_args>(g_launches[l]), y = arg<q38_observe_args>(g_launches[l + 1]);
                        REQUIRE(!memcmp(&x, &y, sizeof(x)) && x.group0 == next && x.n_groups > 0 && x.n_tokens == n && x.base_pos == held - n);
                        next += x.n_groups;
                        REQUIRE(g_launches[l].f == kStats && g_launches[l].gy == 4 && (int)g_launches[l].gz == x.n_groups && (int)g_launches[l].gx == x.n_splits);
                        REQUIRE(x.n_splits <= 64 && (x.n_splits - 1) * x.split_pages < pages && x.n_splits * x.split_pages >= pages);
                        REQUIRE(g_launches[l + 1].f == kAdd && (int)g_launches[l + 1].gx == (pages + 7) / 8 && g_launches[l + 1].gy == 4 && g_launches[l + 1].gz == 1);
                        const size_t stats = (size_t)x.n_groups * 4 * Q38_OBSERVE_COLS * x.n_splits * 8;
                        REQUIRE(inside(x.part_ml, stats) && (char *)x.scores >= (char *)x.part_ml + stats && (uintptr_t)x.scores % 16 == 0);
                        REQUIRE(inside(x.scores, (size_t)x.n_groups * 4 * pages * Q38_OBSERVE_COLS * 16 * 4));
                        REQUIRE(x.page_row == kv->d_page_table + (size_t)big * kv->pt_stride && x.weights == kv->weights_of(0));
                    }
                    REQUIRE(next == groups);
                    continue;
                }
                REQUIRE(g_launches[0].f == kStats && g_launches[0].gy == 4 && (int)g_launches[0].gz == groups && a.n_groups == groups);
                REQUIRE((int)g_launches[0].gx == a.n_splits && a.n_splits <= 64 && (a.n_splits - 1) * a.split_pages < pages && a.n_splits * a.split_pages >= pages);
                REQUIRE(g_launches[1].f == kSums && g_launches[1].gy == 4 && g_launches[1].gz == 1 && s.n_splits == a.n_splits);
                REQUIRE(((int)g_launches[1].gx - 1) * s.split_pages < pages && (int)g_launches[1].gx * s.split_pages >= pages);
                REQUIRE(inside(a.part_ml, (size_t)groups * 4 * Q38_OBSERVE_COLS * a.n_splits * 8) && s.part_ml == a.part_ml);
                REQUIRE(a.page_row == kv->d_page_table + (size_t)big * kv->pt_stride && a.weights == kv->weights_of(0));
            }
        }
        /* eviction: the moves' lists and counts inside the workspace, of every sequence and slot */
        {
            std::vector<int32_t> seq(ids.begin(), ids.begin() + 70), n, keep, recent;
            for (int s : seq) {
                n.push_back(rand() % (kv->seq_pages[s] * 16 + 1));
                keep.push_back(n.back() ? rand() % (n.back() + 1) : 0);
                recent.push_back(keep.back() ? rand() % (keep.back() + 1) : 0);
            }
            const auto pages = kv->seq_pages;
            g_launches.clear();
            REQUIRE(q38_kv_evict(kv, 70, seq.data(), n.data(), keep.data(), recent.data()) == 0);
            REQUIRE(g_launches.size() == 4);
            int b = 0;
            for (int l = 0; l < 4; l += 2) {
                const auto a = arg<q38_evict_args>(g_launches[l]), m = arg<q38_evict_args>(g_launches[l + 1]);
                REQUIRE(!memcmp(&a, &m, sizeof(a)) && g_launches[l].f == kSelect && g_launches[l].block == 1024 && g_launches[l].gx == 8);
                REQUIRE(g_launches[l + 1].f == kMove && g_launches[l + 1].gy == 8 && g_launches[l + 1].gz == g_launches[l].gy);
                /* (an eighth of a list's workgroups to each XCD) */
                const int rows = Q38_EVICT_WAVES * (kKvTypes[kv->type].ggml_type == Q38_GGML_MXFP4 ? Q38_EVICT_MX4 : 1);
                REQUIRE((int)g_launches[l + 1].gx * rows >= a.max_moves && g_launches[l + 1].gx % 8 == 0);
                const size_t lists = (size_t)g_launches[l].gy * 8;
                REQUIRE(inside(a.counts, lists * 4) && inside(a.moves, lists * 2 * a.max_moves * 4));
                REQUIRE((char *)a.moves >= (char *)a.counts + lists * 4);
                for (int i = 0; i < (int)g_launches[l].gy; ++i, ++b) {
                    REQUIRE(a.seq[i] == seq[b] && a.n_tokens[i] == n[b] && a.n_keep[i] == keep[b]);
                    REQUIRE(a.first_recent[i] == n[b] - recent[b]); /* none evicted before */
                    REQUIRE(std::min(keep[b], n[b] - keep[b]) <= a.max_moves && (n[b] + 15) / 16 <= pages[seq[b]]);
                }
            }
            REQUIRE(b == 70);
            for (b = 0; b < 70; ++b) {
                REQUIRE(kv->seq_pages[seq[b]] == std::min(pages[seq[b]], (keep[b] + 15) / 16));
                REQUIRE(q38_seq_evicted(kv, seq[b], &n_out) == 0 && n_out == n[b] - keep[b]);
            }
        }
        /* refusals: nothing launched, nothing changed */
        const int a = ids[75], e = ids[76];
        REQUIRE(q38_seq_reset(kv, a) == 0 && q38_seq_reserve(kv, a, 100) == 0 && q38_seq_reset(kv, e) == 0 && q38_seq_reserve(kv, e, 100) == 0);
        {
            const int32_t s = e, n = 100, k = 40, r = 7;
            REQUIRE(q38_kv_evict(kv, 1, &s, &n, &k, &r) == 0);
        }
        const auto before = c.snapshot();
        const size_t launches = g_launches.size();
        auto refused = [&](int rc, const char *why) {
            REQUIRE(rc == -1);
            if (std::string(q38_last_error()).find(why) == std::string::npos) {
                printf("expected '%s', got '%s'\n", why, q38_last_error());
                exit(1);
            }
            REQUIRE(c.snapshot() == before && g_launches.size() == launches);
        };
        int32_t s2[2] = {a, ids[77]}, twice[2] = {a, a}, none[2] = {a, 999}, p[2] = {0, 5}, cnt[2] = {3, 7}, far[2] = {110, 0}, neg[2] = {-1, 0};
        const float *f = d_w;
        refused(q38_kv_weights_put(nullptr, 3, 2, s2, p, cnt, f, d_t), "kv is NULL");
        refused(q38_kv_weights_put(kv, 4, 2, s2, p, cnt, f, d_t), "not a full-attention layer");
        refused(q38_kv_weights_put(kv, 11, 2, s2, p, cnt, f, d_t), "needs slot 2");
        refused(q38_kv_weights_put(kv, 3, 2, twice, p, cnt, f, d_t), "appears twice");
        refused(q38_kv_weights_put(kv, 3, 2, none, p, cnt, f, d_t), "does not exist");
        refused(q38_kv_weights_put(kv, 3, 2, s2, far, cnt, f, d_t), "not reserved");
        refused(q38_kv_weights_put(kv, 3, 2, s2, neg, cnt, f, d_t), "negative");
        refused(q38_kv_weights_put(kv, 3, 2, nullptr, p, cnt, f, d_t), "NULL");
        refused(q38_kv_weights_get(kv, 3, 2, s2, far, cnt, d_w, d_t), "not reserved");
        refused(q38_kv_weights_get(kv, 3, 2, s2, p, cnt, nullptr, nullptr), "no output");
        refused(q38_kv_weights_get(kv, 3, 2, s2, p, cnt, d_w, (int32_t *)d_w + 39), "overlaps");
        refused(q38_attn_observe(nullptr, 3, a, 0, 3, f), "kv is NULL");
        refused(q38_attn_observe(kv, 3, 999, 0, 3, f), "does not exist");
        refused(q38_attn_observe(kv, 4, a, 0, 3, f), "not a full-attention layer");
        refused(q38_attn_observe(kv, 3, a, -1, 3, f), "negative");
        refused(q38_attn_observe(kv, 3, a, 0, -3, f), "negative");
        refused(q38_attn_observe(kv, 3, a, 110, 3, f), "not reserved");
        refused(q38_attn_observe(kv, 3, a, 2147483647, 2147483647, f), "not reserved");
        refused(q38_attn_observe(kv, 3, a, 0, 3, nullptr), "NULL argument");
        refused(q38_attn_observe(kv, 3, a, 0, 3, f + 1), "16-byte aligned");
        int32_t n[2] = {100, 9}, k[2] = {50, 9}, r[2] = {10, 9}, more[2] = {113, 9}, above[2] = {101, 9}, most[2] = {51, 9}, mine[2] = {-5, 9};
        refused(q38_kv_evict(nullptr, 2, s2, n, k, r), "kv is NULL");
        refused(q38_kv_evict(kv, -1, s2, n, k, r), "negative n_seq");
        refused(q38_kv_evict(kv, 2, nullptr, n, k, r), "NULL argument");
        refused(q38_kv_evict(kv, 2, s2, nullptr, k, r), "NULL argument");
        refused(q38_kv_evict(kv, 2, s2, n, nullptr, r), "NULL argument");
        refused(q38_kv_evict(kv, 2, s2, n, k, nullptr), "NULL argument");
        refused(q38_kv_evict(kv, 2, twice, n, k, r), "appears twice");
        refused(q38_kv_evict(kv, 2, none, n, k, r), "does not exist");
        refused(q38_kv_evict(kv, 2, s2, more, k, r), "not reserved");
        refused(q38_kv_evict(kv, 2, s2, n, above, r), "to keep of");
        refused(q38_kv_evict(kv, 2, s2, n, k, most), "recent tokens");
        refused(q38_kv_evict(kv, 2, s2, mine, k, r), "negative count");
        refused(q38_kv_evict(kv, 2, s2, n, mine, r), "negative count");
        refused(q38_kv_evict(kv, 2, s2, n, k, mine), "negative count");
        int32_t es[1] = {e}, e39[1] = {39}, e3[1] = {3};
        refused(q38_kv_evict(kv, 1, es, e39, e3, e3), "since its last eviction");
        g_capture = hipStreamCaptureStatusActive;
        refused(q38_kv_evict(kv, 2, s2, n, k, r), "cannot be captured");
        refused(q38_kv_track_weights(kv, 0), "cannot be captured");
        refused(q38_attn_observe(kv, 3, a, 0, 3, f), "cannot be captured");
        g_capture = hipStreamCaptureStatusNone;
        refused(q38_kv_track_weights(kv, 0), "has evicted tokens");
        refused(q38_seq_truncate(kv, e, 39), "in no order");
        refused(q38_kv_write(kv, 3, e, 39, 4, f, f), "in no order");
        refused(q38_attn_prefill(kv, 3, e, 39, 4, f, f, f, nullptr, d_w), "in no order");
        int32_t e0[1] = {39}, e40[1] = {40}, e2[1] = {2};
        refused(q38_attn_decode(kv, 3, 1, es, e0, f, f, f, nullptr, d_w), "in no order");
        refused(q38_full_core(kv, 3, 1, es, e0, f, f, f, f, f, d_w), "in no order");
        refused(q38_kv_append(kv, 3, 1, es, e40, e2, f, f, f), "has evicted tokens");
        int32_t at[2] = {0, 0};
        refused(q38_attn_decode(kv, 3, 2, twice, at, f, nullptr, nullptr, nullptr, d_w), "appears twice");
        refused(q38_seq_evicted(kv, 999, &n_out), "does not exist");
        refused(q38_seq_evicted(kv, e, nullptr), "NULL argument");
        /* nothing to do is no failure */
        int32_t zeros[2] = {0, 0};
        REQUIRE(q38_kv_weights_put(kv, 3, 2, s2, p, zeros, nullptr, nullptr) == 0);
        REQUIRE(q38_kv_weights_get(kv, 3, 2, s2, p, zeros, nullptr, nullptr) == 0);
        REQUIRE(q38_attn_observe(kv, 3, a, 5, 0, nullptr) == 0 && q38_kv_evict(kv, 0, nullptr, nullptr, nullptr, nullptr) == 0);
        REQUIRE(c.snapshot() == before && g_launches.size() == launches);
        /* an eviction of nothing moves nothing, of everything too; what is left begins anew at 0 */
        int32_t ae[2] = {a, e}, same[2] = {100, 40}, all[2] = {0, 0};
        REQUIRE(q38_kv_evict(kv, 2, ae, same, same, zeros) == 0 && g_launches.size() == launches);
        REQUIRE(q38_kv_evict(kv, 2, ae, same, all, zeros) == 0 && g_launches.size() == launches);
        REQUIRE(q38_seq_evicted(kv, a, &n_out) == 0 && n_out == 100 && kv->seq_pages[a] == 0);
        REQUIRE(q38_seq_evicted(kv, e, &n_out) == 0 && n_out == 100);
        REQUIRE(q38_seq_truncate(kv, e, 0) == 0 && q38_seq_reset(kv, a) == 0);
        REQUIRE(q38_seq_evicted(kv, e, &n_out) == 0 && n_out == 0);
        REQUIRE(q38_seq_evicted(kv, a, &n_out) == 0 && n_out == 0);
    }
    /* f32 rows */
    Cache c(0, 1, 10, 2, 64);
    REQUIRE(q38_kv_track_weights(c.kv, 1) == -1 && strstr(q38_last_error(), "F32 rows"));
    REQUIRE(q38_kv_track_weights(nullptr, 1) == -1);
    /* a long context's lists, a few sequences a launch */
    Cache l(4, 17, 80000, 6, 200000);
    REQUIRE(q38_kv_track_weights(l.kv, 1) == 0);
    std::vector<int32_t> seq, n, keep, recent;
    for (int i = 0; i < 6; ++i) {
        int s;
        REQUIRE(q38_seq_create(l.kv, &s) == 0 && q38_seq_reserve(l.kv, s, 200000) == 0);
        seq.push_back(s), n.push_back(200000 - i), keep.push_back(100000), recent.push_back(0);
    }
    g_launches.clear();
    REQUIRE(q38_kv_evict(l.kv, 6, seq.data(), n.data(), keep.data(), recent.data()) == 0);
    int done = 0;
    for (size_t i = 0; i < g_launches.size(); i += 2) {
        const auto a = arg<q38_evict_args>(g_launches[i]);
        REQUIRE(inside(a.moves, (size_t)g_launches[i].gy * 68 * 2 * a.max_moves * 4) && (size_t)g_launches[i].gy * 68 * 2 * a.max_moves * 4 <= (256u << 20));
        for (unsigned b = 0; b < g_launches[i].gy; ++b) REQUIRE(a.seq[b] == seq[done++]);
    }
    REQUIRE(done == 6 && g_launches.size() == 4);
    printf("weights ok\n");
    return 0;
}
