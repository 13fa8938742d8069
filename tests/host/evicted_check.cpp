// Host-side check of sequences that have evicted tokens, on the CPU: the library's
// source compiled into this program, its launches and graphs answered here.
#include <hip/hip_runtime_api.h>

#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "q38_kv_layout.h"

static std::vector<hipFunction_t> g_launches;
static int g_replays = 0;
static uintptr_t g_next = 0x100000000000ull;
static hipStreamCaptureStatus g_capture = hipStreamCaptureStatusNone;
static hipError_t check_launch(hipFunction_t f, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, hipStream_t, void **, void **) {
    g_launches.push_back(f);
    return hipSuccess;
}
static int g_device = 0;
static std::vector<int> g_malloc_devices; /* that were current at each allocation */
static hipError_t check_get_device(int *device) {
    *device = g_device;
    return hipSuccess;
}
static hipError_t check_set_device(int device) {
    g_device = device;
    return hipSuccess;
}
template <typename T>
static hipError_t check_malloc(T **p, size_t bytes) {
    g_malloc_devices.push_back(g_device);
    *p = reinterpret_cast<T *>(g_next);
    g_next += (bytes + 0xFFFFFFF) & ~(size_t)0xFFFFFFF;
    return hipSuccess;
}
static hipError_t check_free(void *) { return hipSuccess; }
static hipError_t check_copy(void *, const void *, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
static hipError_t check_set(void *, int, size_t, hipStream_t) { return hipSuccess; }
static hipError_t check_sync(hipStream_t) { return hipSuccess; }
static hipError_t check_capturing(hipStream_t, hipStreamCaptureStatus *status) {
    *status = g_capture;
    return hipSuccess;
}
static hipError_t check_graph_create(hipGraph_t *g, unsigned) {
    *g = reinterpret_cast<hipGraph_t>(g_next);
    return hipSuccess;
}
static hipError_t check_add_node(hipGraphNode_t *n, hipGraph_t, const hipGraphNode_t *, size_t, const hipKernelNodeParams *) {
    *n = reinterpret_cast<hipGraphNode_t>(g_next);
    return hipSuccess;
}
static hipError_t check_node_params(hipGraphNode_t, const hipKernelNodeParams *) { return hipSuccess; }
static hipError_t check_exec_params(hipGraphExec_t, hipGraphNode_t, const hipKernelNodeParams *) { return hipSuccess; }
static hipError_t check_instantiate(hipGraphExec_t *e, hipGraph_t, hipGraphNode_t *, char *, size_t) {
    *e = reinterpret_cast<hipGraphExec_t>(g_next);
    return hipSuccess;
}
static hipError_t check_graph_launch(hipGraphExec_t, hipStream_t) {
    ++g_replays;
    return hipSuccess;
}
static hipError_t check_graph_destroy(hipGraph_t) { return hipSuccess; }
static hipError_t check_exec_destroy(hipGraphExec_t) { return hipSuccess; }
#define hipMalloc check_malloc
#define hipGetDevice check_get_device
#define hipSetDevice check_set_device
#define hipFree check_free
#define hipMemsetAsync check_set
#define hipStreamIsCapturing check_capturing
#define hipModuleLaunchKernel check_launch
#define hipMemcpyAsync check_copy
#define hipStreamSynchronize check_sync
#define hipGraphCreate check_graph_create
#define hipGraphAddKernelNode check_add_node
#define hipGraphKernelNodeSetParams check_node_params
#define hipGraphExecKernelNodeSetParams check_exec_params
#define hipGraphInstantiate check_instantiate
#define hipGraphLaunch check_graph_launch
#define hipGraphDestroy check_graph_destroy
#define hipGraphExecDestroy check_exec_destroy
#include "../../qwen3.8_27b_in_rust_amd/csrc/host/q38_attn.cpp"

int q38_scratch_address(int, void **ptr) {
    *ptr = nullptr;
    return -1;
}

#define REQUIRE(c)                                                                           \
    do {                                                                                     \
        if (!(c)) { printf("line %d: %s (%s)\n", __LINE__, #c, q38_last_error()); exit(1); } \
    } while (0)

/* a device pointer that nothing reads */
static float *const d = reinterpret_cast<float *>(0x70000000000ull);

struct Cache {
    q38_ctx ctx;
    q38_kv *kv = new q38_kv;
    std::vector<int32_t> staging = std::vector<int32_t>(1 << 16);
    explicit Cache(int type, int slots = 2, int pages = 64, int seqs = 4, int tokens = 512) {
        ctx.cu_count = 256;
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
        kv->staging = staging.data();
        kv->staging_len = staging.size();
    }
    int seq(int tokens) {
        int s;
        REQUIRE(q38_seq_create(kv, &s) == 0 && q38_seq_reserve(kv, s, tokens) == 0);
        return s;
    }
    void evict(int32_t s, int32_t n, int32_t keep, int32_t recent = 0) { REQUIRE(q38_kv_evict(kv, 1, &s, &n, &keep, &recent) == 0); }
    int gone(int s) {
        int n;
        REQUIRE(q38_seq_evicted(kv, s, &n) == 0);
        return n;
    }
    /* A call that fails as `why` says, launches nothing and leaves pages, sequences and evicted counts as they were. */
    template <typename Call>
    void refused(Call call, const char *why) {
        auto state = [&] {
            std::vector<int32_t> s = kv->page_table;
            s.insert(s.end(), kv->free_pages.begin(), kv->free_pages.end());
            s.insert(s.end(), kv->seq_pages.begin(), kv->seq_pages.end());
            for (auto &e : kv->evicted) s.push_back(e.tokens), s.push_back(e.kept);
            s.push_back((int)g_launches.size());
            s.push_back(g_replays);
            return s;
        };
        const auto before = state();
        REQUIRE(call() == -1);
        if (strstr(q38_last_error(), why) == nullptr) {
            printf("expected '%s', got '%s'\n", why, q38_last_error());
            exit(1);
        }
        REQUIRE(state() == before);
    }
};

/* The count and order of a sequence that comes from another cache. */
static void handed_on(int type) {
    Cache c(type);
    const int a = c.seq(100);
    c.refused([&] { return q38_seq_set_evicted(nullptr, a, 60, 40); }, "kv is NULL");
    c.refused([&] { return q38_seq_set_evicted(c.kv, a, 60, 40); }, "does not track");
    REQUIRE(q38_kv_track_weights(c.kv, 1) == 0);
    c.refused([&] { return q38_seq_set_evicted(c.kv, 3, 60, 40); }, "does not exist");
    c.refused([&] { return q38_seq_set_evicted(c.kv, -1, 60, 40); }, "does not exist");
    c.refused([&] { return q38_seq_set_evicted(c.kv, a, -1, 40); }, "negative");
    c.refused([&] { return q38_seq_set_evicted(c.kv, a, 60, -1); }, "negative");
    c.refused([&] { return q38_seq_set_evicted(c.kv, a, 0, 1); }, "keeps 1 of them");
    c.refused([&] { return q38_seq_set_evicted(c.kv, a, 60, 113); }, "not reserved");
    c.refused([&] { return q38_seq_set_evicted(c.kv, a, INT_MAX, 40); }, "2^30");
    REQUIRE(q38_seq_set_evicted(c.kv, a, 0, 0) == 0 && c.gone(a) == 0);
    REQUIRE(q38_seq_set_evicted(c.kv, a, 60, 40) == 0 && c.gone(a) == 60);
    /* as after an eviction here */
    c.refused([&] { return q38_seq_set_evicted(c.kv, a, 61, 40); }, "has evicted tokens");
    c.refused([&] { return q38_seq_truncate(c.kv, a, 39); }, "in no order");
    c.refused([&] { return q38_kv_write(c.kv, 3, a, 39, 4, d, d); }, "in no order");
    c.refused([&] { return q38_kv_track_weights(c.kv, 0); }, "has evicted tokens");
    const int32_t s = a, at = 40, two = 2;
    c.refused([&] { return q38_kv_append(c.kv, 3, 1, &s, &at, &two, d, d, d); }, "has evicted tokens");
    REQUIRE(q38_kv_write(c.kv, 3, a, 40, 4, d, d) == 0);
    c.evict(a, 100, 50);
    REQUIRE(c.gone(a) == 110);
    /* a new beginning, and another sequence in its place */
    REQUIRE(q38_seq_truncate(c.kv, a, 0) == 0 && c.gone(a) == 0 && q38_seq_reserve(c.kv, a, 50) == 0);
    REQUIRE(q38_seq_set_evicted(c.kv, a, 7, 0) == 0 && c.gone(a) == 7);
    REQUIRE(q38_seq_free(c.kv, a) == 0 && c.seq(10) == a && c.gone(a) == 0);
}

/* Positions below what the last eviction kept: nothing is attended to by place there. */
static void reads_in_no_order(int type) {
    Cache c(type);
    REQUIRE(q38_kv_track_weights(c.kv, 1) == 0);
    const int a = c.seq(100), b = c.seq(100);
    c.evict(a, 100, 40);
    const int32_t both[2] = {b, a}, at[2] = {5, 38}, last[2] = {5, 39};
    c.refused([&] { return q38_attn_decode(c.kv, 3, 2, both, at, d, nullptr, nullptr, nullptr, d); }, "before 40 have been in no order");
    c.refused([&] { return q38_attn_prefill(c.kv, 3, a, 38, 1, d, nullptr, nullptr, nullptr, d); }, "before 40 have been in no order");
    c.refused([&] { return q38_attn_prefill(c.kv, 3, a, 0, 45, d, nullptr, nullptr, nullptr, d); }, "in no order");
    /* all that were kept are an order's end */
    REQUIRE(q38_attn_decode(c.kv, 3, 2, both, last, d, nullptr, nullptr, nullptr, d) == 0);
    REQUIRE(q38_attn_prefill(c.kv, 3, a, 39, 5, d, nullptr, nullptr, nullptr, d) == 0);
    q38_decode_call call = {};
    call.layer = 3;
    call.d_q = d;
    call.d_out = d;
    q38_decode_graph *g = nullptr;
    c.refused([&] { return q38_decode_graph_create(c.kv, 2, both, at, 1, &call, &g); }, "in no order");
    REQUIRE(q38_decode_graph_create(c.kv, 2, both, last, 1, &call, &g) == 0);
    c.refused([&] { return q38_decode_graph_set_positions(g, at); }, "in no order");
    REQUIRE(q38_decode_graph_launch(g) == 0 && g_replays > 0);
    REQUIRE(q38_decode_graph_destroy(g) == 0);
    /* a cache that tracks nothing has an order everywhere */
    REQUIRE(q38_seq_reset(c.kv, a) == 0 && q38_seq_reserve(c.kv, a, 100) == 0);
    REQUIRE(q38_attn_decode(c.kv, 3, 2, both, at, d, nullptr, nullptr, nullptr, d) == 0);
}

/* Sums put back without own positions: those of positions in no order are nothing that a place tells. */
static void sums_in_no_order(int type) {
    Cache c(type);
    REQUIRE(q38_kv_track_weights(c.kv, 1) == 0);
    const int a = c.seq(100), b = c.seq(100);
    c.evict(a, 100, 40);
    REQUIRE(q38_seq_reserve(c.kv, a, 60) == 0);
    const int32_t both[2] = {b, a}, at[2] = {0, 39}, next[2] = {0, 40}, n[2] = {30, 3}, one[2] = {30, 0};
    int32_t *own = reinterpret_cast<int32_t *>(d);
    for (const float *sums : {(const float *)nullptr, (const float *)d})
        c.refused([&] { return q38_kv_weights_put(c.kv, 3, 2, both, at, n, sums, nullptr); }, "before 40 have been in no order");
    /* with them, past them, and none of them */
    REQUIRE(q38_kv_weights_put(c.kv, 3, 2, both, at, n, nullptr, own) == 0);
    REQUIRE(q38_kv_weights_put(c.kv, 3, 2, both, at, n, d, own) == 0);
    REQUIRE(q38_kv_weights_put(c.kv, 3, 2, both, next, n, d, nullptr) == 0);
    REQUIRE(q38_kv_weights_put(c.kv, 3, 2, both, at, one, d, nullptr) == 0);
}

/* Graphs whose positions an eviction, or what came after it, has taken away. */
static void graphs_of_positions_gone(int type) {
    Cache c(type);
    REQUIRE(q38_kv_track_weights(c.kv, 1) == 0);
    const int32_t a = c.seq(100);
    q38_decode_call call = {};
    call.layer = 3;
    call.d_q = call.d_k_new = call.d_v_new = d;
    call.d_out = d;
    q38_decode_graph *g = nullptr;
    auto launch = [&] { return q38_decode_graph_launch(g); };
    /* an eviction of nothing gives back the page that the graph's next token is for */
    int32_t at = 112;
    REQUIRE(q38_decode_graph_create(c.kv, 1, &a, &at, 1, &call, &g) == 0 && launch() == 0);
    c.evict(a, 112, 112);
    REQUIRE(c.gone(a) == 0);
    c.refused(launch, "position 112 is not reserved any more");
    REQUIRE(q38_decode_graph_set_positions(g, &at) == 0 && launch() == 0);
    /* as many evicted as before, of which more were kept */
    at = 40;
    c.evict(a, 100, 40);
    c.refused(launch, "evicted tokens since");
    REQUIRE(q38_decode_graph_set_positions(g, &at) == 0 && launch() == 0);
    REQUIRE(q38_seq_reset(c.kv, a) == 0 && q38_seq_reserve(c.kv, a, 120) == 0);
    c.refused(launch, "evicted tokens since");
    c.evict(a, 120, 60);
    REQUIRE(c.gone(a) == 60);
    c.refused(launch, "before 60 have been in no order");
    at = 60;
    REQUIRE(q38_decode_graph_set_positions(g, &at) == 0 && launch() == 0);
    /* a sequence that is no more, and another in its place */
    REQUIRE(q38_seq_free(c.kv, a) == 0);
    c.refused(launch, "does not exist");
    REQUIRE(c.seq(16) == a);
    c.refused(launch, "evicted tokens since");
    REQUIRE(q38_decode_graph_destroy(g) == 0);
    /* calls without a new row */
    call.d_k_new = call.d_v_new = nullptr;
    REQUIRE(q38_seq_reserve(c.kv, a, 100) == 0);
    at = 30;
    REQUIRE(q38_decode_graph_create(c.kv, 1, &a, &at, 1, &call, &g) == 0 && launch() == 0);
    REQUIRE(q38_seq_truncate(c.kv, a, 16) == 0);
    c.refused(launch, "position 30 is not reserved any more");
    REQUIRE(q38_decode_graph_destroy(g) == 0);
    /* a graph without decode calls has no positions */
    q38_linear_weights w = {d, d, d, d};
    REQUIRE(q38_seq_reserve(c.kv, a, 100) == 0 && q38_decode_graph_begin(c.kv, 1, &a, &at, &g) == 0);
    REQUIRE(q38_decode_graph_add_linear_core(g, 1, &w, d, d, d, d, d, d, d) == 0 && q38_decode_graph_end(g) == 0);
    c.evict(a, 100, 10);
    REQUIRE(launch() == 0 && q38_decode_graph_destroy(g) == 0);
}

/* A context of one device while another is current: what its calls allocate is its own. */
static void two_devices(int type) {
    Cache c(type);
    c.ctx.device = 1;
    auto own = [&](auto call) {
        const size_t before = g_malloc_devices.size();
        REQUIRE(call() == 0 && g_malloc_devices.size() > before && g_device == 0);
        for (size_t i = before; i < g_malloc_devices.size(); ++i) REQUIRE(g_malloc_devices[i] == 1);
    };
    void *p = nullptr;
    own([&] { return q38_alloc(&c.ctx, 100, &p); });
    own([&] { return q38_kv_track_weights(c.kv, 1); });
    const int32_t a = c.seq(500), at = 499, n = 500, keep = 250, none = 0;
    auto fresh = [&] { c.ctx.work = nullptr, c.ctx.work_bytes = 0; };
    own([&] { return q38_attn_decode(c.kv, 3, 1, &a, &at, d, nullptr, nullptr, nullptr, d); });
    fresh();
    own([&] { return q38_attn_observe(c.kv, 3, a, 480, 20, d); });
    fresh();
    own([&] { return q38_attn_prefill(c.kv, 3, a, 480, 20, d, nullptr, nullptr, nullptr, d); });
    fresh();
    own([&] { return q38_kv_evict(c.kv, 1, &a, &n, &keep, &none); });
    q38_decode_call call = {};
    call.layer = 3;
    call.d_q = call.d_k_new = call.d_v_new = d;
    call.d_out = d;
    q38_decode_graph *g = nullptr;
    own([&] { return q38_decode_graph_create(c.kv, 1, &a, &keep, 1, &call, &g); });
    REQUIRE(q38_decode_graph_destroy(g) == 0);
}

int main() {
    for (int type : {1, 4}) {
        two_devices(type);
        graphs_of_positions_gone(type);
        sums_in_no_order(type);
        handed_on(type);
        reads_in_no_order(type);
    }
    printf("evicted ok\n");
    return 0;
}
