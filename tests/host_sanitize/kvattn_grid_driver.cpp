// The launches of attention over pages for any limits that the header allows: what the runtime takes (fewer than 2^32 threads in x, 2^16 blocks in y and z), or a refusal and
// no launch at all.  Without a GPU: launches are counted, not made.  Built and run by tests/test_kvpool_limits.py; prints "ok" and returns 0.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../../llama2.rs_amd/csrc/kernels_kvattn.hip"

static int launches = 0;
static bool fits = true;

int l2_fail(int code, const char *, ...) { return code; }
extern "C" {
const char __hip_fatbin[16] = {}; // there is no device code
void **__hipRegisterFatBinary(const void *) { return nullptr; }
void __hipRegisterFunction(void **, const void *, char *, const char *, unsigned, void *, void *, void *, void *, int *) {}
void __hipUnregisterFatBinary(void **) {}
hipError_t hipLaunchKernel(const void *kernel, dim3 grid, dim3 block, void **, size_t, hipStream_t) {
    launches++;
    fits = fits && kernel && grid.x && grid.y && grid.z && (uint64_t)grid.x * block.x < (1ull << 32) && grid.y < 65536 && grid.z < 65536;
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDevice(int *d) { return *d = 0, hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t *p, int) { return p->multiProcessorCount = 256, hipSuccess; }
}

int main() {
    std::mt19937_64 rng(1);
    auto upto = [&](double most) { // evenly over the logarithm, the ends often
        const double u = std::uniform_real_distribution<double>(-0.1, 1.1)(rng);
        return (int)std::min(most, std::max(1.0, std::pow(most, std::max(u, 0.0))));
    };
    int refused = 0, wide = 0;
    for (int n = 0; n < 300000; n++) {
        l2_kvbatch b{};
        b.n_seqs = upto(65535), b.n_rows = upto(1 << 22), b.max_rows = upto(1 << 22), b.max_length = upto(1 << 30), b.max_pages = b.max_length / 16 + 1;
        KvLayer l{};
        l.n_heads = upto(65535), l.head_size = n % 2 ? 64 : 128, l.page_shift = 4, l.n_pages = 1;
        KvAttention a{};
        a.n_heads = l.n_heads * upto(65535 / l.n_heads), a.type = n % 3, a.scale = 1.f, a.window = n % 5 ? 0 : upto(0x7FFFFFFF), a.sinks = n % 7 ? 0 : upto(0x7FFFFFFF);
        a.q_stride = a.out_stride = (int64_t)a.n_heads * l.head_size;
        if ((int64_t)b.n_rows * (a.n_heads / l.n_heads) > 1 << 30) continue;
        const int kv = n / 2 % 4;
        KvAttnPlan plan{};
        kv_attention_plan(l, kv, b, a, &plan);
        launches = 0;
        const int rc = kv_attention_launch(l, kv, b, a, plan, (void *)64, nullptr);
        if ((rc == L2_OK ? launches == 0 : rc != L2_ERR_RANGE || launches != 0) || !fits) {
            fprintf(stderr, "%d: rc %d, %d launches, fits %d: %d seqs, %d rows, %d at most, %d positions, %d heads on %d\n", n, rc, launches, fits, b.n_seqs, b.n_rows, b.max_rows, b.max_length,
                    a.n_heads, l.n_heads);
            return 1;
        }
        refused += rc != L2_OK, wide += plan.wide;
    }
    if (!refused || !wide || refused > wide / 2) return fprintf(stderr, "%d refused, %d wide\n", refused, wide), 1;
    puts("ok");
    return 0;
}
