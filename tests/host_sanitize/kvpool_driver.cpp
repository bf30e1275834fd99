// The host side of the operators on a cache in pages and of sampling, under the sanitizers and without a GPU: the runtime's calls and the kernels' launches are
// stand-ins, which count what reaches them.  Every call that is refused must reach none.  Built and run by tests/test_kvpool_host.py; prints "ok" and returns 0.
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <thread>
#include <vector>

#include "../../llama2.rs_amd/csrc/host_kvpool.cpp"

static thread_local int launches = 0, current = 0;
static int devices = 2, stream_device = 0;
static bool no_memory = false;
static thread_local KvLayer layer_seen;
static thread_local KvRows rows_seen;
static thread_local KvAttention attention_seen;
static thread_local SampleSettings settings_seen;

int l2_fail(int code, const char *fmt, ...) {
    char text[512];
    va_list args;
    va_start(args, fmt);
    const int n = vsnprintf(text, sizeof text, fmt, args);
    va_end(args);
    return n > 0 ? code : 0;
}
void l2_pass_by(int) {}
int kv_rows_warm_up() { return L2_OK; }
int kv_attention_warm_up() { return L2_OK; }
int sample_warm_up() { return L2_OK; }
int kv_write_launch(const KvLayer &l, int, const l2_kvbatch &, const KvRows &rows, hipStream_t) { return launches++, layer_seen = l, rows_seen = rows, L2_OK; }
int kv_read_launch(const KvLayer &l, int, const l2_kvbatch &, const KvRows &rows, hipStream_t) { return launches++, layer_seen = l, rows_seen = rows, L2_OK; }
void kv_attention_plan(const KvLayer &, int, const l2_kvbatch &, const KvAttention &, KvAttnPlan *plan) { plan->workspace = 1000; }
int kv_attention_launch(const KvLayer &l, int, const l2_kvbatch &, const KvAttention &a, const KvAttnPlan &, void *, hipStream_t) {
    return launches++, layer_seen = l, attention_seen = a, L2_OK;
}
int sample_launch(const void *, int, int, int, int64_t stride, const SampleSettings &s, int32_t *, hipStream_t) {
    return launches++, settings_seen = s, rows_seen.k_stride = stride, L2_OK;
}
extern "C" {
hipError_t hipGetDeviceCount(int *n) { return *n = devices, devices ? hipSuccess : hipErrorNoDevice; }
hipError_t hipGetDevice(int *d) { return *d = current, hipSuccess; }
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t *d) { return *d = stream_device, hipSuccess; }
hipError_t hipMalloc(void **p, size_t n) { return *p = no_memory ? nullptr : malloc(n), *p ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipMemset(void *p, int v, size_t n) { return memset(p, v, n), hipSuccess; }
hipError_t hipFree(void *p) { return free(p), hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char *hipGetErrorString(hipError_t) { return "an error"; }
}

#define REQUIRE(cond)                                                     \
    do {                                                                  \
        if (!(cond)) {                                                    \
            fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #cond);    \
            exit(1);                                                      \
        }                                                                 \
    } while (0)
#define REFUSED(code, call)         \
    do {                            \
        const int before = launches; \
        REQUIRE((call) == (code));  \
        REQUIRE(launches == before); \
    } while (0)

static void pools() {
    l2_kvpool *p = (l2_kvpool *)1;
    const int big = 0x7FFFFFFF;
    REFUSED(L2_ERR_ARG, l2_kvpool_create(1, 1, 16, 1, 64, L2_KV_I8, nullptr));
    const int bad[][6] = {{0, 1, 16, 1, 64, 0}, {1, 0, 16, 1, 64, 0}, {1, 1, 8, 1, 64, 0},  {1, 1, 512, 1, 64, 0},    {1, 1, 48, 1, 64, 0}, {1, 1, 0, 1, 64, 0},
                          {1, 1, -16, 1, 64, 0}, {1, 1, 16, 0, 64, 0}, {1, 1, 16, 65536, 64, 0}, {1, 1, 16, 1, 96, 0}, {1, 1, 16, 1, 64, 4}, {1, 1, 16, 1, 64, -1}};
    for (const auto &b : bad) {
        p = (l2_kvpool *)1;
        REFUSED(L2_ERR_ARG, l2_kvpool_create(b[0], b[1], b[2], b[3], b[4], b[5], &p));
        REQUIRE(!p);
    }
    REFUSED(L2_ERR_RANGE, l2_kvpool_create(big, big, 256, 65535, 128, L2_KV_F16, &p));
    REFUSED(L2_ERR_RANGE, l2_kvpool_create(big, 16, 256, 1024, 128, L2_KV_F16, &p));
    no_memory = true;
    REFUSED(L2_ERR_HIP, l2_kvpool_create(1, 1, 16, 1, 64, L2_KV_I8, &p));
    no_memory = false;
    devices = 0;
    REFUSED(L2_ERR_HIP, l2_kvpool_create(1, 1, 16, 1, 64, L2_KV_I8, &p));
    devices = 2;
    REQUIRE(!p);
    l2_kvpool_free(nullptr);
    REQUIRE(l2_kvpool_bytes(nullptr) == 0);
}

// One pool from its making to its end, every call once as it should be and in all the ways in which it should not.
static void calls(int kv_type) {
    l2_kvpool *p = nullptr;
    const int layers = 3, pages = 5, size = 32, heads = 2, d = 64;
    REQUIRE(l2_kvpool_create(layers, pages, size, heads, d, kv_type, &p) == L2_OK && p);
    const size_t cells = (size_t)pages * size * heads * d * (kv_type <= L2_KV_E4M3 ? 1 : 2), scales = kv_type <= L2_KV_E4M3 ? (size_t)pages * size * heads * 4 : 0;
    REQUIRE(l2_kvpool_bytes(p) == 2 * layers * (cells + scales));
    std::vector<int32_t> starts(4), lengths(3), table(3 * 4);
    std::vector<float> k(64), v(64);
    const l2_kvbatch good{starts.data(), lengths.data(), table.data(), 3, 4, 10, 5, 128};
    const hipStream_t st = (hipStream_t)0x1000;
    auto write = [&](const l2_kvbatch *b, int layer = 0, const void *kk = (void *)64, const void *vv = (void *)64, int type = L2_F32, int64_t ks = 0, int64_t vs = 0) {
        return l2_kvpool_write(p, layer, b, kk, vv, type, ks, vs, st);
    };
    // as it should be; the layer's arrays lie behind one another inside the pool
    const char *last = nullptr;
    for (int layer = 0; layer < layers; layer++) {
        REQUIRE(write(&good, layer) == L2_OK && launches);
        REQUIRE(rows_seen.k_stride == heads * d && rows_seen.v_stride == heads * d);
        REQUIRE(!last || layer_seen.k == last);
        REQUIRE((char *)layer_seen.v == (char *)layer_seen.k + cells && layer_seen.page_shift == 5);
        last = (char *)layer_seen.k + 2 * (cells + scales);
        if (scales) REQUIRE((char *)layer_seen.v_scale + scales == last && (char *)layer_seen.k_scale + scales == (char *)layer_seen.v_scale);
    }
    REQUIRE(l2_kvpool_read(p, 1, &good, (void *)2, (void *)6, L2_BF16, 130, 0, nullptr) == L2_OK && rows_seen.k_stride == 130);
    // batches
    for (int w = 0; w < 13; w++) {
        l2_kvbatch b = good;
        switch (w) {
        case 0: b.n_seqs = -1; break;
        case 1: b.n_seqs = 65536; break;
        case 2: b.max_pages = -1; break;
        case 3: b.n_rows = -1; break;
        case 4: b.max_rows = -1; break;
        case 5: b.max_length = -1; break;
        case 6: b.max_length = 4 * size + 1; break;
        case 7: b.starts = nullptr; break;
        case 8: b.lengths = nullptr; break;
        case 9: b.pages = nullptr; break;
        case 10: b.starts = (int32_t *)((char *)starts.data() + 1); break;
        case 11: b.lengths = (int32_t *)((char *)lengths.data() + 2); break;
        case 12: b.pages = (int32_t *)((char *)table.data() + 3); break;
        }
        l2_attention a{heads, L2_F32, 0.f, 0, 0, 0, 0};
        size_t n = 0;
        REFUSED(L2_ERR_ARG, write(&b));
        REFUSED(L2_ERR_ARG, l2_kvpool_read(p, 0, &b, (void *)64, (void *)64, L2_F32, 0, 0, st));
        REFUSED(L2_ERR_ARG, l2_kvpool_attention_workspace(p, &b, &a, &n));
        REFUSED(L2_ERR_ARG, l2_kvpool_attention(p, 0, &b, &a, (void *)64, (void *)64, (void *)64, 1000, st));
    }
    l2_kvbatch many = good;
    many.n_rows = (1 << 22) + 1;
    REFUSED(L2_ERR_RANGE, write(&many));
    many = good;
    many.max_pages = 1 << 26, many.max_length = (1 << 30) + 1;
    REFUSED(L2_ERR_RANGE, write(&many));
    many = good;
    many.n_rows = 1 << 22;
    const l2_attention wide{257 * heads, L2_F32, 0.f, 0, 0, 0, 0};
    REFUSED(L2_ERR_RANGE, l2_kvpool_attention(p, 0, &many, &wide, (void *)64, (void *)128, (void *)64, 1000, st));
    REFUSED(L2_ERR_ARG, write(nullptr));
    REFUSED(L2_ERR_ARG, l2_kvpool_write(nullptr, 0, &good, (void *)64, (void *)64, L2_F32, 0, 0, st));
    // layers, types, addresses, strides
    REFUSED(L2_ERR_RANGE, write(&good, -1));
    REFUSED(L2_ERR_RANGE, write(&good, layers));
    REFUSED(L2_ERR_ARG, write(&good, 0, nullptr));
    REFUSED(L2_ERR_ARG, write(&good, 0, (void *)64, nullptr));
    REFUSED(L2_ERR_ARG, write(&good, 0, (void *)66));
    REFUSED(L2_ERR_ARG, write(&good, 0, (void *)64, (void *)65, L2_F16));
    REFUSED(L2_ERR_ARG, write(&good, 0, (void *)64, (void *)64, 3));
    REFUSED(L2_ERR_ARG, write(&good, 0, (void *)64, (void *)64, -1));
    for (int64_t bad : {(int64_t)heads * d - 1, (int64_t)-1, (int64_t)-heads * d, ((int64_t)1 << 40) + 1}) {
        REFUSED(L2_ERR_ARG, write(&good, 0, (void *)64, (void *)64, L2_F32, bad));
        REFUSED(L2_ERR_ARG, write(&good, 0, (void *)64, (void *)64, L2_F32, 0, bad));
    }
    // nothing to do
    for (int w = 0; w < 3; w++) {
        l2_kvbatch b = good;
        (w == 0 ? b.n_seqs : w == 1 ? b.n_rows : b.max_rows) = 0;
        l2_attention a{heads, L2_F32, 0.f, 0, 0, 0, 0};
        REFUSED(L2_OK, write(&b, 0, nullptr, nullptr));
        REFUSED(L2_OK, l2_kvpool_attention(p, 0, &b, &a, nullptr, nullptr, nullptr, 0, st));
    }
    // other devices
    current = 1;
    REFUSED(L2_ERR_ARG, write(&good));
    current = 0;
    // attention
    auto attend = [&](l2_attention a, void *out = (void *)128, void *ws = (void *)64, size_t bytes = 1000, int layer = 0) {
        return l2_kvpool_attention(p, layer, &good, &a, (void *)64, out, ws, bytes, st);
    };
    const l2_attention fine{3 * heads, L2_F16, 0.f, 7, 2, 0, 0};
    REQUIRE(attend(fine) == L2_OK && attention_seen.scale == 0.125f && attention_seen.q_stride == 3 * heads * d && attention_seen.window == 7 && attention_seen.sinks == 2);
    REQUIRE(attend({heads, L2_F32, 2.f, 0, 0, 200, 300}) == L2_OK && attention_seen.scale == 2.f && attention_seen.q_stride == 200 && attention_seen.out_stride == 300);
    REQUIRE(attend({heads, L2_F32, 2.f, 0, 0, 200, 200}, (void *)64) == L2_OK);
    const l2_attention not_fine[] = {{0, L2_F32, 0.f, 0, 0, 0, 0},      {-2, L2_F32, 0.f, 0, 0, 0, 0},      {3, L2_F32, 0.f, 0, 0, 0, 0},       {65536, L2_F32, 0.f, 0, 0, 0, 0},
                                     {2, 3, 0.f, 0, 0, 0, 0},           {2, L2_F32, -1.f, 0, 0, 0, 0},      {2, L2_F32, INFINITY, 0, 0, 0, 0},  {2, L2_F32, NAN, 0, 0, 0, 0},
                                     {2, L2_F32, 0.f, -1, 0, 0, 0},     {2, L2_F32, 0.f, 0, -1, 0, 0},      {2, L2_F32, 0.f, 0, 0, 127, 0},     {2, L2_F32, 0.f, 0, 0, 0, 127},
                                     {2, L2_F32, 0.f, 0, 0, -128, 0}};
    for (const l2_attention &a : not_fine) {
        size_t n = 0;
        REFUSED(L2_ERR_ARG, attend(a));
        REFUSED(L2_ERR_ARG, l2_kvpool_attention_workspace(p, &good, &a, &n));
    }
    size_t n = 0;
    REQUIRE(l2_kvpool_attention_workspace(p, &good, &fine, &n) == L2_OK && n == 1000);
    REFUSED(L2_ERR_ARG, l2_kvpool_attention_workspace(p, &good, &fine, nullptr));
    REFUSED(L2_ERR_ARG, l2_kvpool_attention_workspace(p, &good, nullptr, &n));
    REFUSED(L2_ERR_ARG, attend(fine, nullptr));
    REFUSED(L2_ERR_ARG, attend(fine, (void *)65));
    REFUSED(L2_ERR_ARG, attend(fine, (void *)128, nullptr));
    REFUSED(L2_ERR_ARG, attend(fine, (void *)128, (void *)72));
    REFUSED(L2_ERR_ARG, attend(fine, (void *)128, (void *)64, 999));
    REFUSED(L2_ERR_RANGE, attend(fine, (void *)128, (void *)64, 1000, layers));
    REFUSED(L2_ERR_ARG, attend({heads, L2_F32, 0.f, 0, 0, 200, 0}, (void *)64)); // in place with two strides
    l2_kvpool_free(p);
}

static void sampling() {
    float x[4] = {};
    int32_t ids[4], k[4];
    const l2_sampling s{x, k, x, x, x}, only_u{nullptr, nullptr, nullptr, nullptr, x};
    auto call = [&](const l2_sampling *how, int rows = 2, int vocab = 100, int type = L2_F32, int64_t stride = 0, const void *at = (void *)64, void *to = nullptr) {
        return l2_sample_device(at, type, rows, vocab, stride, how, to ? (int32_t *)to : ids, nullptr);
    };
    REQUIRE(call(&s) == L2_OK && launches && settings_seen.temperature == x && settings_seen.top_k == k && rows_seen.k_stride == 100);
    REQUIRE(call(&only_u, 2, 100, L2_F16, 101, (void *)2) == L2_OK && !settings_seen.top_p && settings_seen.temperature0 == 1.f && settings_seen.top_p0 == 1.f &&
            settings_seen.min_p0 == 0.f && rows_seen.k_stride == 101);
    REFUSED(L2_OK, call(&s, 0, 100, L2_F32, 0, nullptr));
    REFUSED(L2_ERR_ARG, call(nullptr));
    REFUSED(L2_ERR_ARG, call(&s, -1));
    REFUSED(L2_ERR_ARG, call(&s, 2, 0));
    REFUSED(L2_ERR_ARG, call(&s, 2, (1 << 19) + 1));
    REFUSED(L2_ERR_ARG, call(&s, 2, 100, 3));
    REFUSED(L2_ERR_ARG, call(&s, 2, 100, L2_F32, 99));
    REFUSED(L2_ERR_ARG, call(&s, 2, 100, L2_F32, -100));
    REFUSED(L2_ERR_ARG, call(&s, 2, 100, L2_F32, 0, nullptr));
    REFUSED(L2_ERR_ARG, call(&s, 2, 100, L2_F32, 0, (void *)66));
    REFUSED(L2_ERR_ARG, call(&s, 2, 100, L2_F32, 0, (void *)64, (char *)ids + 2));
    for (int w = 0; w < 5; w++) {
        l2_sampling odd = s;
        const void *at = (char *)x + 1;
        w == 0 ? (void)(odd.temperature = (const float *)at) : w == 1 ? (void)(odd.top_k = (const int32_t *)at) : w == 2 ? (void)(odd.top_p = (const float *)at) : w == 3 ? (void)(odd.min_p = (const float *)at) : (void)(odd.u = (const float *)at);
        REFUSED(L2_ERR_ARG, call(&odd));
    }
    l2_sampling none = s;
    none.u = nullptr;
    REFUSED(L2_ERR_ARG, call(&none));
    stream_device = 1;
    REFUSED(L2_ERR_ARG, l2_sample_device((void *)64, L2_F32, 2, 100, 0, &s, ids, (void *)0x1000));
    stream_device = 0;
}

int main() {
    pools();
    for (int t : {L2_KV_I8, L2_KV_E4M3, L2_KV_F16, L2_KV_BF16}) calls(t);
    sampling();
    std::vector<std::thread> all; // nothing is shared between pools
    for (int t = 0; t < 4; t++) all.emplace_back(calls, t);
    for (std::thread &t : all) t.join();
    puts("ok");
    return 0;
}
