// Host-side check of the calls whose buffers must lie apart, on the CPU: calls
// on overlapping ones are refused before a launch.  The library's source and the
// launches' stand-in come with
// kv_rows_check.cpp.
#define main kv_rows_main
#include "kv_rows_check.cpp"
#undef main

static void refused(int rc, const char *why) {
    REQUIRE(rc == -1);
    REQUIRE(std::string(q38_last_error()).find(why) != std::string::npos);
}

int main() {
    const int launches = g_launches;
    /* 3 rows of 512: 1536 quants, 96 sums of 16 and 6 scales take 1752 bytes, the values 6144 */
    q38_ctx ctx;
    char *base = reinterpret_cast<char *>(0x300000000000ull);
    for (long at : {0l, 16l, 1744l, -16l, -6128l})
        refused(q38_dequantize_q8_k(&ctx, 3, 512, base, reinterpret_cast<float *>(base + at)), "overlaps");
    REQUIRE(q38_dequantize_q8_k(&ctx, 0, 512, base, reinterpret_cast<float *>(base)) == 0);
    REQUIRE(g_launches == launches);
    REQUIRE(Q38_Q8K_BYTES(3, 512) == 1752);

    /* 40 rows of two sequences: 4096 bytes a row, 2048 as stored */
    for (int type : {0, 2}) {
        Cache c(type, 1, 64, 4, 512);
        int32_t s[2], p[2] = {3, 0}, n[2] = {33, 7};
        for (int i = 0; i < 2; ++i) {
            REQUIRE(q38_seq_create(&c.kv, &s[i]) == 0);
            REQUIRE(q38_seq_reserve(&c.kv, s[i], 64) == 0);
        }
        const int own = kKvTypes[type].ggml_type;
        const long bytes = 40l * 1024 * (type == 0 ? 4 : 2);
        const int before = g_launches;
        for (long at : {0l, 16l, bytes - 16, -16l, 16 - bytes})
            refused(q38_kv_gather(&c.kv, 3, 2, s, p, n, own, base, base + at), "overlaps");
        REQUIRE(g_launches == before);
        for (long at : {bytes, -bytes}) REQUIRE(q38_kv_gather(&c.kv, 3, 2, s, p, n, own, base, base + at) == 0);
        REQUIRE(g_launches == before + 2);
    }
    printf("row buffers ok\n");
    return 0;
}
