// Host-side check of the typed cache's row calls (q38_kv_append,
// q38_kv_gather, q38_kv_write, q38_kv_read) and of the page layouts, on the
// CPU: the library's source compiled into this program, its launches answered
// here.  Every launch's arguments are walked as the kernel walks them -- which
// page of which sequence a workgroup serves, which rows -- and each access has
// to lie inside the pool, the page table and the caller's rows, every row
// moved once, in order.  Refused calls launch nothing and leave pages and
// sequences as they were.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <cstddef>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "q38_kv_layout.h"

static int g_launches = 0;
static std::vector<std::vector<char>> g_args;
static std::vector<unsigned> g_grid;
/* the functions that a launch names: one handle for each argument block */
static hipFunction_t const kMany = (hipFunction_t)0x1000, kFew = (hipFunction_t)0x2000, kFewGather = (hipFunction_t)0x3000;
static int g_pt_stride; /* of the cache at hand */
static hipError_t check_launch(hipFunction_t f, unsigned gx, unsigned gy, unsigned, unsigned block, unsigned, unsigned,
                               unsigned, hipStream_t, void **params, void **) {
    ++g_launches;
    if (gy != 2 || block != Q38_KV_ROWS_THREADS) { printf("unexpected grid\n"); exit(1); }
    q38_kv_rows_args a;
    if (f == kFew || f == kFewGather) {
        /* the arguments in the kernels' order */
        q38_kv_rows_few_args w;
        void **p = params;
        auto take = [&](auto &x) { memcpy(&x, *p++, sizeof(x)); };
        memset(&w, 0xAB, sizeof(w));
        if (f == kFewGather) {
            q38_kv_gather_few_rest rest;
            take(w.table), take(w.pos0), take(w.n_tokens), take(w.head.page_table), take(rest);
            w.head.k_rows = rest.k_rows, w.head.v_rows = rest.v_rows;
            w.head.kpool = rest.kpool, w.head.vpool = rest.vpool;
        } else {
            take(w);
        }
        memset(&a, 0xAB, sizeof(a)); /* what the kernel does not get */
        a.head = w.head;
        /* the bases as the kernel finds them from the counts, 0 past the last sequence */
        a.n_seq = 0;
        a.row_base[0] = a.page_base[0] = 0;
        for (int i = 0; i < Q38_KV_ROWS_FEW; ++i) {
            if (w.table[i] % g_pt_stride != 0) { printf("a table that is no sequence's\n"); exit(1); }
            a.seq[i] = w.table[i] / g_pt_stride;
            a.pos0[i] = w.pos0[i];
            const int pages = ((w.pos0[i] + w.n_tokens[i] - 1) >> 4) - (w.pos0[i] >> 4) + 1;
            if ((pages > 0) != (w.n_tokens[i] > 0) || (pages > 0 && a.n_seq != i)) { printf("counts with a gap\n"); exit(1); }
            a.n_seq += pages > 0;
            a.row_base[i + 1] = a.row_base[i] + w.n_tokens[i];
            a.page_base[i + 1] = a.page_base[i] + pages;
        }
        for (int i = a.n_seq + 1; i < Q38_MAX_BATCH + 8; ++i) a.page_base[i] = INT_MAX;
    } else {
        a = *static_cast<const q38_kv_rows_args *>(params[0]);
    }
    const char *p = reinterpret_cast<const char *>(&a);
    g_args.emplace_back(p, p + sizeof(a));
    if (gx % Q38_KV_ROWS_PARTS != 0) { printf("a page in part\n"); exit(1); }
    g_grid.push_back(gx / Q38_KV_ROWS_PARTS); /* pages */
    return hipSuccess;
}
static hipError_t check_copy(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
static hipError_t check_sync(hipStream_t) { return hipSuccess; }
static hipError_t check_capturing(hipStream_t, hipStreamCaptureStatus *status) {
    *status = hipStreamCaptureStatusNone;
    return hipSuccess;
}
#define hipStreamIsCapturing check_capturing
#define hipModuleLaunchKernel check_launch
#define hipMemcpyAsync check_copy
#define hipStreamSynchronize check_sync
#include "../../qwen3.8_27b_in_rust_amd/csrc/host/q38_attn.cpp"

int q38_scratch_address(int, void **ptr) {
    *ptr = nullptr;
    return -1;
}

#define REQUIRE(c)                                                                        \
    do {                                                                                  \
        if (!(c)) { printf("line %d: %s (%s)\n", __LINE__, #c, q38_last_error()); exit(1); } \
    } while (0)

template <int T>
static void check_layout() {
    std::set<int> k, v;
    const int size = T == Q38_KV_Q8 ? 1 : T == Q38_KV_F32 ? 4 : 2;
    for (int t = 0; t < 16; ++t)
        for (int d = 0; d < 256; ++d) {
            k.insert(q38_k_index<T>(t, d));
            v.insert(q38_v_index<T>(t, d));
        }
    REQUIRE(k.size() == 4096 && *k.begin() == 0 && *k.rbegin() == 4095);
    REQUIRE(v.size() == 4096 && *v.begin() == 0 && *v.rbegin() == 4095);
    REQUIRE(q38_kv_block_bytes<T>() == 4096 * size && q38_kv_page_bytes<T>() % 128 == 0);
    REQUIRE(q38_kv_page_bytes<T>() == 4 * q38_kv_block_bytes<T>() + (T == Q38_KV_Q8 ? 4 * 64 : 0));
    for (int head = 0; head < 4; ++head) /* past the four blocks, a line apart, inside the page */
        REQUIRE(head * 4096 + q38_kv_scales_offset(head) == 4 * 4096 + 64 * head);
}

struct Cache {
    q38_ctx ctx;
    q38_kv kv;
    std::vector<int32_t> staging;
    Cache(int type, int slots, int pages, int seqs, int tokens) {
        for (int i = 0; i < kKvTypeCount; ++i)
            for (q38_ctx::RowsKernel *k : {&ctx.f_kv_append[i], &ctx.f_kv_gather[i], &ctx.f_kv_gather_16}) {
                k->many = kMany;
                k->gathers = k != &ctx.f_kv_append[i];
                k->few = k->gathers ? kFewGather : kFew;
            }
        kv.ctx = &ctx;
        kv.type = type;
        kv.n_slots = slots;
        kv.max_pages = pages;
        kv.max_seqs = seqs;
        kv.pt_stride = g_pt_stride = (tokens + 15) / 16;
        kv.kpool = reinterpret_cast<float *>(0x100000000000ull);
        kv.vpool = reinterpret_cast<float *>(0x200000000000ull);
        kv.d_page_table = reinterpret_cast<int32_t *>(0x300000000000ull);
        kv.page_table.assign((size_t)seqs * kv.pt_stride, -1);
        for (int p = pages - 1; p >= 0; --p) kv.free_pages.push_back(p);
        kv.seq_live.assign(seqs, 0);
        kv.seq_pages.assign(seqs, 0);
        kv.images.assign((size_t)seqs * slots, q38_kv::Images());
        staging.resize(1 << 20);
        kv.staging = staging.data();
        kv.staging_len = staging.size();
    }
    std::vector<int32_t> snapshot() const {
        std::vector<int32_t> s = kv.page_table;
        s.insert(s.end(), kv.free_pages.begin(), kv.free_pages.end());
        s.insert(s.end(), kv.seq_pages.begin(), kv.seq_pages.end());
        return s;
    }
};

/* The batch's launches walked as the kernel does. */
static void walk(const Cache &c, int slot, const std::vector<int32_t> &seq, const std::vector<int32_t> &pos,
                 const std::vector<int32_t> &cnt, char *d_k, char *d_v, size_t elem) {
    std::vector<std::pair<int, int>> want; /* (seq, position) of each row */
    for (size_t b = 0; b < seq.size(); ++b)
        for (int i = 0; i < cnt[b]; ++i) want.push_back({seq[b], pos[b] + i});
    std::vector<int> moved(want.size(), 0);
    for (size_t l = 0; l < g_args.size(); ++l) {
        q38_kv_rows_args a;
        memcpy(&a, g_args[l].data(), sizeof(a));
        REQUIRE(a.head.kpool == c.kv.kslot(slot) && a.head.vpool == c.kv.vslot(slot));
        REQUIRE(a.n_seq >= 1 && a.n_seq <= Q38_MAX_BATCH && (unsigned)a.page_base[a.n_seq] == g_grid[l]);
        const size_t row_off = (static_cast<char *>(a.head.k_rows) - d_k) / (1024 * elem);
        REQUIRE(row_off == (size_t)(static_cast<char *>(a.head.v_rows) - d_v) / (1024 * elem));
        for (unsigned x = 0; x < g_grid[l]; ++x) {
            int b = 0;
            for (int i0 = 1; i0 < a.n_seq; i0 += 8)
                for (int i = 0; i < 8; ++i) b += a.page_base[i0 + i] <= (int)x ? 1 : 0;
            REQUIRE(((a.n_seq - 2) / 8) * 8 + 8 < Q38_MAX_BATCH + 8);
            REQUIRE(b < a.n_seq && a.page_base[b] <= (int)x && (int)x < a.page_base[b + 1]);
            const int first = a.pos0[b], n = a.row_base[b + 1] - a.row_base[b];
            const int lp = (first >> 4) + (int)x - a.page_base[b];
            const int p0 = std::max(first, lp * 16), p1 = std::min(first + n, (lp + 1) * 16);
            REQUIRE(p1 > p0 && lp < c.kv.seq_pages[a.seq[b]]);
            const int page = c.kv.page_table[(size_t)a.seq[b] * c.kv.pt_stride + lp];
            REQUIRE(page >= 0 && page < c.kv.max_pages);
            for (int p = p0; p < p1; ++p) {
                const size_t row = row_off + a.row_base[b] + p - first;
                REQUIRE(row < want.size() && want[row].first == a.seq[b] && want[row].second == p);
                ++moved[row];
            }
        }
    }
    for (int m : moved) REQUIRE(m == 1);
}

int main() {
    check_layout<Q38_KV_F32>();
    check_layout<Q38_KV_F16>();
    check_layout<Q38_KV_BF16>();
    check_layout<Q38_KV_Q8>();
    srand(7);
    float *w = reinterpret_cast<float *>(0x400000000000ull), *k = reinterpret_cast<float *>(0x500000000000ull),
          *v = reinterpret_cast<float *>(0x600000000000ull);
    int calls = 0;
    for (int type = 0; type < 4; ++type) {
        Cache c(type, 2, 4000, 150, 4096);
        std::vector<int> ids;
        for (int i = 0; i < 150; ++i) {
            int s;
            REQUIRE(q38_seq_create(&c.kv, &s) == 0);
            ids.push_back(s);
        }
        for (int it = 0; it < 60; ++it) {
            /* distinct sequences in a random order, 1 .. 150 of them, pieces of 0 .. 70 tokens */
            std::vector<int32_t> seq(ids.begin(), ids.end()), pos, cnt;
            for (size_t i = seq.size() - 1; i > 0; --i) std::swap(seq[i], seq[rand() % (i + 1)]);
            seq.resize(1 + rand() % (it % 3 == 0 ? 12 : seq.size()));
            for (size_t i = 0; i < seq.size(); ++i) pos.push_back(rand() % 300), cnt.push_back(rand() % 4 ? rand() % 71 : 0);
            g_args.clear(), g_grid.clear();
            REQUIRE(q38_kv_append(&c.kv, 7, (int)seq.size(), seq.data(), pos.data(), cnt.data(), w, k, v) == 0);
            walk(c, 1, seq, pos, cnt, (char *)k, (char *)v, 4);
            g_args.clear(), g_grid.clear();
            REQUIRE(q38_kv_gather(&c.kv, 3, (int)seq.size(), seq.data(), pos.data(), cnt.data(), 0, k, v) == 0);
            walk(c, 0, seq, pos, cnt, (char *)k, (char *)v, 4);
            if (type == 1 || type == 2) {
                g_args.clear(), g_grid.clear();
                REQUIRE(q38_kv_gather(&c.kv, 3, (int)seq.size(), seq.data(), pos.data(), cnt.data(),
                                      kKvTypes[type].ggml_type, k, v) == 0);
                walk(c, 0, seq, pos, cnt, (char *)k, (char *)v, 2);
            }
            ++calls;
        }
        /* refusals: nothing launched, nothing changed */
        const auto before = c.snapshot();
        const int launches = g_launches;
        int32_t s2[2] = {ids[0], ids[1]}, twice[2] = {ids[0], ids[0]}, none[2] = {ids[0], 999}, p[2] = {0, 5},
                far[2] = {0, 4090}, neg[2] = {-1, 0}, big[2] = {2147483647, 2147483647}, n[2] = {3, 7}, nn[2] = {3, -1},
                full[2] = {4097, 4096};
        auto refused = [&](int rc, const char *why) {
            REQUIRE(rc == -1);
            if (std::string(q38_last_error()).find(why) == std::string::npos) {
                printf("expected '%s', got '%s'\n", why, q38_last_error());
                exit(1);
            }
            REQUIRE(c.snapshot() == before && g_launches == launches);
        };
        refused(q38_kv_append(nullptr, 3, 2, s2, p, n, w, k, v), "kv is NULL");
        refused(q38_kv_append(&c.kv, 4, 2, s2, p, n, w, k, v), "not a full-attention layer");
        refused(q38_kv_append(&c.kv, 11, 2, s2, p, n, w, k, v), "needs slot 2");
        refused(q38_kv_append(&c.kv, 3, -1, s2, p, n, w, k, v), "negative n_seq");
        refused(q38_kv_append(&c.kv, 3, 2, nullptr, p, n, w, k, v), "NULL seq_ids");
        refused(q38_kv_append(&c.kv, 3, 2, s2, nullptr, n, w, k, v), "NULL seq_ids");
        refused(q38_kv_append(&c.kv, 3, 2, s2, p, nullptr, w, k, v), "NULL seq_ids");
        refused(q38_kv_append(&c.kv, 3, 2, twice, p, n, w, k, v), "appears twice");
        refused(q38_kv_append(&c.kv, 3, 2, none, p, n, w, k, v), "does not exist");
        refused(q38_kv_append(&c.kv, 3, 2, s2, neg, n, w, k, v), "negative position");
        refused(q38_kv_append(&c.kv, 3, 2, s2, p, nn, w, k, v), "negative position or count");
        refused(q38_kv_append(&c.kv, 3, 2, s2, far, n, w, k, v), "past the context limit");
        refused(q38_kv_append(&c.kv, 3, 2, s2, big, n, w, k, v), "past the context limit");
        refused(q38_kv_append(&c.kv, 3, 2, s2, p, n, nullptr, k, v), "NULL argument");
        refused(q38_kv_append(&c.kv, 3, 2, s2, p, n, w, nullptr, v), "NULL argument");
        refused(q38_kv_append(&c.kv, 3, 2, s2, p, n, w, k, nullptr), "NULL argument");
        refused(q38_kv_append(&c.kv, 3, 2, s2, p, n, w, k + 1, v), "16-byte aligned");
        {
            std::vector<int32_t> all(ids.begin(), ids.end()), zero(150, 0), most(150, 4096);
            refused(q38_kv_append(&c.kv, 3, 150, all.data(), zero.data(), most.data(), w, k, v), "KV pool exhausted");
        }
        refused(q38_kv_gather(&c.kv, 3, 2, s2, p, full, 0, k, v), "past the context limit");
        int32_t held[2] = {4000, 4000};
        refused(q38_kv_gather(&c.kv, 3, 2, s2, held, n, 0, k, v), "not reserved");
        refused(q38_kv_gather(&c.kv, 3, 1, s2, p, n, 12, k, v), "not as type 12");
        refused(q38_kv_gather(&c.kv, 3, 1, s2, p, n, type == 1 ? 30 : 1, k, v), "not as type");
        refused(q38_kv_gather(&c.kv, 3, 1, s2, p, n, 15, k, v), "not as type 15");
        refused(q38_kv_gather(&c.kv, 3, 1, s2, p, n, 0, nullptr, v), "NULL argument");
        refused(q38_kv_gather(&c.kv, 3, 1, s2, p, n, 0, k, reinterpret_cast<char *>(v) + 8), "16-byte aligned");
        refused(q38_attn_prefill(&c.kv, 3, ids[0], 0, 4, w, k, nullptr, nullptr, v), "go together");
        refused(q38_attn_prefill(&c.kv, 3, ids[0], 4000, 4, w, nullptr, nullptr, nullptr, v), "not reserved");
        /* nothing to move is no failure */
        int32_t zeros[2] = {0, 0};
        REQUIRE(q38_kv_append(&c.kv, 3, 2, s2, p, zeros, nullptr, nullptr, nullptr) == 0);
        REQUIRE(q38_kv_append(&c.kv, 3, 0, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) == 0);
        REQUIRE(q38_kv_gather(&c.kv, 3, 2, s2, p, zeros, 0, nullptr, nullptr) == 0);
        REQUIRE(c.snapshot() == before && g_launches == launches);
    }
    /* a cache's type */
    q38_ctx ctx;
    q38_kv *out = nullptr;
    for (int ty : {-1, 2, 8, 12, 24, 31}) {
        REQUIRE(q38_kv_create_typed(&ctx, ty, 1, 1, 1, 16, &out) == -1 && out == nullptr);
        REQUIRE(std::string(q38_last_error()).find("a KV cache holds") == 0);
    }
    /* the norm's refusals */
    auto norm_refused = [&](int rc, const char *why) {
        REQUIRE(rc == -1);
        REQUIRE(std::string(q38_last_error()).find(why) != std::string::npos);
    };
    const int launches = g_launches;
    norm_refused(q38_add_rms_norm(nullptr, 1, 256, k, v, w, k, nullptr, nullptr), "ctx is NULL");
    norm_refused(q38_add_rms_norm(&ctx, -1, 256, k, v, w, k, nullptr, nullptr), "negative");
    norm_refused(q38_add_rms_norm(&ctx, 1, 0, k, v, w, k, nullptr, nullptr), "not positive");
    norm_refused(q38_add_rms_norm(&ctx, 1, 300, k, v, w, nullptr, nullptr, v + (1 << 20)), "multiple of 256");
    norm_refused(q38_add_rms_norm(&ctx, 1, 256, nullptr, v, w, k, nullptr, nullptr), "NULL argument");
    norm_refused(q38_add_rms_norm(&ctx, 1, 256, k, v, nullptr, k, nullptr, nullptr), "NULL argument");
    norm_refused(q38_add_rms_norm(&ctx, 1, 256, k, v, w, nullptr, nullptr, nullptr), "no output");
    norm_refused(q38_add_rms_norm(&ctx, 1, 256, k, v, w, nullptr, nullptr, reinterpret_cast<char *>(w) + 4104), "16-byte");
    norm_refused(q38_add_rms_norm(&ctx, 2, 256, k, v, w, k + 256, nullptr, nullptr), "in part");
    norm_refused(q38_add_rms_norm(&ctx, 2, 256, k, v, w, nullptr, v - 4, nullptr), "in part");
    norm_refused(q38_add_rms_norm(&ctx, 2, 256, k, v, w, w, nullptr, nullptr), "overlaps the weight");
    norm_refused(q38_add_rms_norm(&ctx, 2, 256, k, v, w, k, k, nullptr), "outputs overlap");
    norm_refused(q38_add_rms_norm(&ctx, 2, 256, k, v, w, nullptr, nullptr, k), "overlaps an input");
    norm_refused(q38_add_rms_norm(&ctx, 2, 256, k, v, w, w + 4096, nullptr, w + 4096), "outputs overlap");
    norm_refused(q38_dequantize_q8_k(nullptr, 1, 256, k, v), "ctx is NULL");
    norm_refused(q38_dequantize_q8_k(&ctx, 1, 255, k, v), "multiple of 256");
    norm_refused(q38_dequantize_q8_k(&ctx, -1, 256, k, v), "negative");
    norm_refused(q38_dequantize_q8_k(&ctx, 1, 256, nullptr, v), "NULL argument");
    norm_refused(q38_dequantize_q8_k(&ctx, 1, 256, k, v + 1), "16-byte aligned");
    REQUIRE(q38_add_rms_norm(&ctx, 0, 256, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) == 0);
    REQUIRE(g_launches == launches);
    printf("%d row batches ok\n", calls);
    return 0;
}
