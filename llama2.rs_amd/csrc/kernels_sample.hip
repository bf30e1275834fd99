// One token per row of logits: temperature, top-k, top-p, min-p and a given random number.
//
// In falling order of (logit, then id) what every one of the three filters keeps is a prefix, so each is a threshold on that order, the pair
// (logit, id) as one 64-bit number.  A threshold is found by weights (one each, or the tokens' exponentials) summed over bins of falling
// logits, the bin in which the sum reaches its target cut into finer bins, until a bin's tokens are few enough to be set against one another.
// Weights are whole multiples of 2^-44 in 64-bit integers: sums are exact whatever the order atomics come in, so an answer depends on its row
// alone.  Their rounding moves a border between two tokens by 2^-45 of the largest weight.
#include "kvpool.h"

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kFew = 128;
constexpr int kChunk = 4 * kThreads; // logits that a block takes at a time, four to a thread
constexpr int kKept = 8;             // chunks that stay in registers

__device__ __forceinline__ u64 shfl(u64 v, int from) {
    const uint32_t lo = __shfl((uint32_t)v, from), hi = __shfl((uint32_t)(v >> 32), from);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 shfl_xor(u64 v, int m) {
    const uint32_t lo = __shfl_xor((uint32_t)v, m), hi = __shfl_xor((uint32_t)(v >> 32), m);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
    for (int o = 32; o; o >>= 1) v += shfl_xor(v, o);
    return v;
}
// The sum over this lane and those before it.
__device__ __forceinline__ u64 wave_scan(u64 v) {
    const int lane = threadIdx.x & 63;
    for (int o = 1; o < 64; o <<= 1) {
        const u64 w = shfl(v, lane - o < 0 ? lane : lane - o);
        if (lane >= o) v += w;
    }
    return v;
}

__device__ __forceinline__ uint32_t key_of(float x) { // rises with x
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ u64 order_of(float x, int id) { return (u64)key_of(x) << 32 | ~(uint32_t)id; }

struct Shared {
    double exp2[256];   // 2^(i / 256)
    u64 mass[kBins];
    uint32_t count[kBins];
    u64 part[kWaves];
    u64 few_order[kFew], few_mass[kFew];
    u64 lo, hi, before, found;
    uint32_t n;
    int bin;
    u64 pieces[(kMaxVocab + 255) / 256]; // sums over 256 logits
};

// exp((x - top) / temperature) as a multiple of 2^-44.
struct Weights {
    float top;
    double scale; // log2(e) / temperature
    const double *exp2;
    __device__ __forceinline__ u64 operator()(float x) const {
        if (x == top) return 1ull << 44; // equals of an infinite one among them
        const double y = ((double)x - (double)top) * scale;
        if (!(y > -46.0)) return 0;
        const double n = floor(y), f = (y - n) * 256.0;
        const int i = min((int)f, 255); // y - n rounds to 1 just below a whole y
        const double r = (f - (double)i) * (0.693147180559945309417 / 256.0); // below 2.71e-3: r^5 / 120 is 2^-49
        const double p = fma(r, fma(r, fma(r, fma(r, 1.0 / 24.0, 1.0 / 6.0), 0.5), 1.0), 1.0);
        const double w = ldexp(exp2[i] * p, (int)n + 44);
        return (u64)__builtin_bit_cast(long long, w + 0x1p52) & ((1ull << 52) - 1); // nearest whole number
    }
};

template <class T>
__device__ __forceinline__ float logit(const T *p, int i);
template <>
__device__ __forceinline__ float logit(const float *p, int i) { return p[i]; }
template <>
__device__ __forceinline__ float logit(const _Float16 *p, int i) { return (float)p[i]; }
template <>
__device__ __forceinline__ float logit(const uint16_t *p, int i) { return kv::bf16_float(p[i]); }

// A row's logits, four to a thread and chunk: NaN and what is behind the row's end are -infinity, and zero has one sign.
template <class T, bool REGS>
struct Row {
    const T *p;
    int n;
    float v[REGS ? kKept : 1][4];
    __device__ __forceinline__ float at(int i) const {
        const float x = i < n ? logit(p, i) : -__builtin_inff();
        return x == x ? x + 0.f : -__builtin_inff();
    }
    __device__ __forceinline__ void load() {
        if (REGS)
            for (int j = 0; j < kKept; j++)
                for (int e = 0; e < 4; e++) v[j][e] = at(kChunk * j + 4 * (int)threadIdx.x + e);
    }
    __device__ __forceinline__ int chunks() const { return (n + kChunk - 1) / kChunk; }
    // f(logit, id) for this thread's logits of chunk j
    template <class F>
    __device__ __forceinline__ void chunk(int j, F f) const {
        const int i = kChunk * j + 4 * (int)threadIdx.x;
        for (int e = 0; e < 4; e++) f(REGS ? v[j][e] : at(i + e), i + e);
    }
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        if (REGS) {
#pragma unroll
            for (int j = 0; j < kKept; j++)
                if (kChunk * j < n) chunk(j, f);
        } else {
            for (int j = 0; j < chunks(); j++) chunk(j, f);
        }
    }
};

// The place in the order (inclusive) at which the weights of the tokens at `least` and above, summed from the front, reach `target`, which
// they do.  MASS: by weight, otherwise a token counts one.
template <bool MASS, class R>
__device__ u64 reach(Shared &sh, const R &row, const Weights &weight, float bins_per_unit, u64 least, u64 target) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    u64 lo = least, hi = ~0ull, before = 0;
    int shift = -1; // bins of equal width in logits first, then of 2^shift places in the order below hi
    for (;;) {
        for (int i = tid; i < kBins; i += kThreads) sh.mass[i] = 0, sh.count[i] = 0;
        __syncthreads();
        auto bin_of = [&](float x, u64 o) {
            if (shift >= 0) return (int)((hi - o) >> shift);
            if (x == weight.top) return 0;
            const float d = (weight.top - x) * bins_per_unit;
            return d < (float)(kBins - 1) ? (int)d : kBins - 1;
        };
        row.each([&](float x, int id) {
            const u64 o = order_of(x, id);
            if (o < lo || o > hi) return;
            const int bin = bin_of(x, o);
            if (MASS) atomicAdd(&sh.mass[bin], weight(x));
            atomicAdd(&sh.count[bin], 1u);
        });
        __syncthreads();
        // bins 2 tid and 2 tid + 1 of this thread, and what is before them
        const u64 w0 = MASS ? sh.mass[2 * tid] : sh.count[2 * tid], w1 = MASS ? sh.mass[2 * tid + 1] : sh.count[2 * tid + 1];
        u64 upto = wave_scan(w0 + w1);
        if (lane == 63) sh.part[w] = upto;
        __syncthreads();
        upto += before;
        for (int i = 0; i < w; i++) upto += sh.part[i];
        const u64 b0 = upto - w1 - w0, b1 = upto - w1;
        if (b0 < target && upto >= target) { // one thread
            const bool second = b1 < target;
            sh.bin = 2 * tid + second, sh.before = second ? b1 : b0;
            sh.n = sh.count[2 * tid + second];
        }
        __syncthreads();
        const int bin = sh.bin;
        const uint32_t n = sh.n;
        before = sh.before;
        __syncthreads();
        if (n <= kFew) {
            if (tid == 0) sh.n = 0;
            __syncthreads();
            row.each([&](float x, int id) {
                const u64 o = order_of(x, id);
                if (o < lo || o > hi || bin_of(x, o) != bin) return;
                const uint32_t at = atomicAdd(&sh.n, 1u);
                sh.few_order[at] = o, sh.few_mass[at] = MASS ? weight(x) : 1;
            });
            __syncthreads();
            if (tid < (int)n) {
                const u64 o = sh.few_order[tid];
                u64 sum = before;
                for (uint32_t i = 0; i < n; i++) sum += sh.few_order[i] >= o ? sh.few_mass[i] : 0;
                if (sum >= target && sum - sh.few_mass[tid] < target) sh.found = o; // one thread
            }
            __syncthreads();
            return sh.found;
        }
        // the bin's first and last place in the order
        u64 first = 0, last = ~0ull;
        row.each([&](float x, int id) {
            const u64 o = order_of(x, id);
            if (o < lo || o > hi || bin_of(x, o) != bin) return;
            first = o > first ? o : first, last = o < last ? o : last;
        });
        for (int o = 32; o; o >>= 1) {
            const u64 f = shfl_xor(first, o), g = shfl_xor(last, o);
            first = f > first ? f : first, last = g < last ? g : last;
        }
        if (tid == 0) sh.hi = 0, sh.lo = ~0ull;
        __syncthreads();
        if (lane == 0) atomicMax(&sh.hi, first), atomicMin(&sh.lo, last);
        __syncthreads();
        hi = sh.hi, lo = sh.lo;
        shift = max(0, 64 - __builtin_clzll(hi - lo) - 11); // more than kFew places apart
        __syncthreads();
    }
}

template <class T, bool REGS>
__global__ __launch_bounds__(kThreads) void sample_kernel(const T *logits, int vocab, int64_t stride, SampleSettings s, int32_t *ids) {
    __shared__ Shared sh;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    Row<T, REGS> row;
    row.p = logits + r * stride, row.n = vocab;
    row.load();
    float temperature = s.temperature ? s.temperature[r] : s.temperature0;
    const int k = s.top_k ? s.top_k[r] : s.top_k0;
    const float p = s.top_p ? s.top_p[r] : s.top_p0, least_p = s.min_p ? s.min_p[r] : s.min_p0, u = s.u ? s.u[r] : s.u0;
    if (tid < 256) sh.exp2[tid] = exp2((double)tid / 256.0);

    // the first of the order
    u64 first = 0;
    row.each([&](float x, int id) {
        const u64 o = order_of(x, id);
        first = o > first ? o : first;
    });
    for (int o = 32; o; o >>= 1) {
        const u64 f = shfl_xor(first, o);
        first = f > first ? f : first;
    }
    if (lane == 0) sh.part[w] = first;
    __syncthreads();
    for (int i = 0; i < kWaves; i++) first = sh.part[i] > first ? sh.part[i] : first;
    __syncthreads();
    const float top = value_of((uint32_t)(first >> 32));
    const bool none = top == -__builtin_inff();
    if (none || !(temperature > 0.f)) {
        if (tid == 0) ids[r] = none ? -1 : (int32_t)~(uint32_t)first;
        return;
    }
    const Weights weight{top, 1.4426950408889634074 / (double)temperature, sh.exp2};
    const float per_unit = 64.f / temperature; // infinity below 2^-122, where no bin but the first and the last is taken

    u64 least = 0; // tokens of this place and above are kept
    if (k > 0 && k < vocab) least = reach<false>(sh, row, weight, per_unit, 0, (u64)k);
    if (p < 1.f) {
        u64 sum = 0;
        row.each([&](float x, int id) {
            if (order_of(x, id) >= least) sum += weight(x);
        });
        sum = wave_sum(sum);
        if (lane == 0) sh.part[w] = sum;
        __syncthreads();
        sum = 0;
        for (int i = 0; i < kWaves; i++) sum += sh.part[i];
        __syncthreads();
        const double target = ceil((double)p * (double)sum);
        const u64 t = target > 1.0 ? (u64)target : 1ull; // the first is always kept
        least = reach<true>(sh, row, weight, per_unit, least, t < sum ? t : sum);
    }
    const double least_w = (double)fminf(fmaxf(least_p, 0.f), 1.f) * 0x1p44;
    auto kept = [&](float x, int id) -> u64 {
        if (order_of(x, id) < least) return 0;
        const u64 m = weight(x);
        return (double)m >= least_w ? m : 0;
    };
    // sums over 256 logits that follow one another, a wave's of a chunk
    auto piece = [&](int j) {
        u64 sum = 0;
        row.chunk(j, [&](float x, int id) { sum += kept(x, id); });
        sum = wave_sum(sum);
        if (lane == 0) sh.pieces[kWaves * j + w] = sum;
    };
    const int chunks = row.chunks(), pieces = kWaves * chunks;
    if (REGS) {
#pragma unroll
        for (int j = 0; j < kKept; j++)
            if (j < chunks) piece(j);
    } else {
        for (int j = 0; j < chunks; j++) piece(j);
    }
    __syncthreads();
    if (w) return;
    // the piece, then the token, at which the running sum passes u of the whole; at the latest the last one with a weight
    const int each = (pieces + 63) / 64;
    u64 own = 0;
    for (int i = 0; i < each; i++) own += lane * each + i < pieces ? sh.pieces[lane * each + i] : 0;
    const u64 upto = wave_scan(own), sum = shfl(upto, 63);
    const double share = (u > 0.f ? (double)u : 0.0) * (double)sum;
    u64 passed = share < (double)sum ? (u64)share : sum - 1; // the first running sum above this
    passed = passed < sum ? passed : sum - 1;
    const u64 has = __ballot(upto > passed);
    const int at = __builtin_ctzll(has);
    u64 before = shfl(upto - own, at);
    int i = at * each;
    while (before + sh.pieces[i] <= passed) before += sh.pieces[i++];
    const int id = 256 * i + 4 * lane;
    u64 m[4], mine = 0;
    for (int e = 0; e < 4; e++) mine += m[e] = id + e < vocab ? kept(row.at(id + e), id + e) : 0;
    const u64 end = wave_scan(mine) + before;
    const u64 hit = __ballot(end > passed);
    if (lane == __builtin_ctzll(hit)) {
        u64 c = end - mine;
        int e = 0;
        while (e < 3 && c + m[e] <= passed) c += m[e++];
        ids[r] = id + e;
    }
}

template <class T>
void launch(const void *logits, int rows, int vocab, int64_t stride, const SampleSettings &s, int32_t *ids, hipStream_t st) {
    const bool regs = vocab <= kKept * kChunk;
    l2_launch(regs ? sample_kernel<T, true> : sample_kernel<T, false>, dim3(rows), dim3(kThreads), 0, st, (const T *)logits, vocab, stride, s, ids);
}

} // namespace

int sample_launch(const void *logits, int type, int rows, int vocab, int64_t stride, const SampleSettings &s, int32_t *ids, hipStream_t st) {
    if (vocab < 1 || vocab > kMaxVocab) return l2_fail(L2_ERR_ARG, "sampling from %d logits (up to 2^19)", vocab);
    if (type == L2_F32) launch<float>(logits, rows, vocab, stride, s, ids, st);
    else if (type == L2_F16) launch<_Float16>(logits, rows, vocab, stride, s, ids, st);
    else launch<uint16_t>(logits, rows, vocab, stride, s, ids, st);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int sample_warm_up() {
    hipFuncAttributes a;
    for (const void *f : {(const void *)sample_kernel<float, true>, (const void *)sample_kernel<float, false>, (const void *)sample_kernel<_Float16, true>,
                          (const void *)sample_kernel<_Float16, false>, (const void *)sample_kernel<uint16_t, true>, (const void *)sample_kernel<uint16_t, false>})
        L2_HIP(hipFuncGetAttributes(&a, f));
    return L2_OK;
}
