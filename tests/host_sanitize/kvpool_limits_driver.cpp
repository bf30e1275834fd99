// Limits of the host side of the operators on a cache in pages and of sampling whose products pass 64 or 32 bits, with the stand-ins of kvpool_driver.cpp.  Built and
// run by tests/test_kvpool_limits.py; prints "ok" and returns 0.
#define main kvpool_driver_main
#include "kvpool_driver.cpp"
#undef main

// Layers times rows of exactly 2^64, of a little more, and of the most that is taken.
static void pools_past_64_bits() {
    l2_kvpool *p = nullptr;
    const int sizes[][5] = {{1 << 21, 1 << 28, 256, 128, 64}, {(1 << 21) + 1, 1 << 28, 256, 128, 64}, {0x7FFFFFFF, 1 << 27, 256, 512, 128}, {2, 1 << 27, 256, 256, 128}, {1 << 20, 1 << 12, 256, 16, 64}};
    for (const auto &s : sizes)
        for (int t : {L2_KV_I8, L2_KV_E4M3, L2_KV_F16, L2_KV_BF16}) {
            p = (l2_kvpool *)1;
            REFUSED(L2_ERR_RANGE, l2_kvpool_create(s[0], s[1], s[2], s[3], s[4], t, &p));
            REQUIRE(!p);
        }
    no_memory = true; // one row fewer is a matter of memory
    REFUSED(L2_ERR_HIP, l2_kvpool_create((1 << 20) - 1, 1 << 12, 256, 16, 64, L2_KV_I8, &p));
    no_memory = false;
}

// Rows of logits, a block of 1024 threads each: a launch takes fewer than 2^32.
static void rows_past_32_bits() {
    float x[1] = {};
    int32_t ids[1];
    const l2_sampling s{nullptr, nullptr, nullptr, nullptr, x};
    for (int rows : {(1 << 21) + 1, 1 << 22, 0x7FFFFFFF}) REFUSED(L2_ERR_RANGE, l2_sample_device((void *)64, L2_F32, rows, 1, 0, &s, ids, nullptr));
    REQUIRE(l2_sample_device((void *)64, L2_F32, 1 << 21, 1, 0, &s, ids, nullptr) == L2_OK);
}

int main() {
    pools_past_64_bits();
    rows_past_32_bits();
    puts("ok");
    return 0;
}
