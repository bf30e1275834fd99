// One token per row of logits: temperature, top-k, top-p, min-p and a given random number.
//
// In falling order of (logit, then id) what every one of the three filters keeps is a prefix, so each is a threshold on that order.  Weights are whole multiples
// of 2^-44 in 64-bit integers: sums are exact whatever the order atomics come in, so an answer depends on its row alone.  A weight is off by up to 2^-45 of the largest, so a border
// between two tokens, which is a sum of n of them, by n times that: 2^-30 of 32000 tokens, 2^-26 of the most.  One that rounds to zero is never chosen.
//
// One block of 16 waves per row.  It is bound by the instructions that one CU can issue, not by the 128 KB of a row, so passes are few and short: the largest logit;
// for top-k, how many logits lie in each of 2048 bins, of those not below the bin that k threads' largest reach, and the tokens of the bin that the k-th is in;
// for top-p the same with rounded weights; then one pass with the exact weights, which leaves their sums over 256 logits that the answer is looked up in.  For
// top-p that pass also has the sum of all, the sum in front of the bins in question and the tokens in these, which must contain the border.  What a top-k of some hundred keeps is
// put into the list whole, and the rest happens there.  Where a border
// is not among few tokens (ties, temperatures that put everything into one bin), reach() cuts the order finer until it is.
// 256 rows of 32000 fp32 logits, of memory: a temperature 20 us, top-k 40 and top-p 0.9 23, top-k 200 and top-p 0.9 35, top-p alone 35 (a pass for the rounded weights,
// one with the exact ones for sums in front of the bins); at a large copy's rate the logits are 7.
#include "kvpool.h"
#include "lanes.h"

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048, kList = 512;
constexpr int kChunk = 4 * kThreads; // logits that a block takes at a time, four to a thread

// 2^(i / 1024) * 2^44.
struct Exp2Table {
    double v[1024];
};
constexpr Exp2Table exp2_table() {
    Exp2Table t{};
    for (int i = 0; i < 1024; i++) {
        const double x = i * (0.693147180559945309417 / 1024);
        double sum = 0, term = 1;
        for (int n = 1; n < 24; n++) {
            sum += term;
            term *= x / n;
        }
        t.v[i] = sum * 0x1p44;
    }
    return t;
}
__device__ const Exp2Table kExp2 = exp2_table();

__device__ __forceinline__ u64 shfl(u64 v, int from) {
    const uint32_t lo = __shfl((uint32_t)v, from), hi = __shfl((uint32_t)(v >> 32), from);
    return (u64)hi << 32 | lo;
}
// v of the lane that a row's pattern names.
template <int CTRL>
__device__ __forceinline__ u64 other(u64 v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xF, 0xF, false);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 other_row(u64 v, bool far) { // of the lane 16 (32) away
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    const auto l = far ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false) : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto h = far ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false) : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    return ((u64)h[0] << 32 | l[0]) + ((u64)h[1] << 32 | l[1]) - v; // both in the same order for both lanes
}
template <class F>
__device__ __forceinline__ u64 wave_all(u64 v, F f) {
    v = f(v, other<0xB1>(v)); // lanes 1, then 2 away; the other four, the other eight of a row
    v = f(v, other<0x4E>(v));
    v = f(v, other<0x141>(v));
    v = f(v, other<0x140>(v));
    v = f(v, other_row(v, false));
    return f(v, other_row(v, true));
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true);
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = a[0] + a[1];
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return b[0] + b[1];
}
// Of numbers below 2^48, in halves of 24 bits (30 as sums): an addition takes its operand from another lane itself, one of 64 bits does not.
__device__ __forceinline__ u64 wave_sum48(u64 v) {
    return (u64)wave_sum((uint32_t)v & 0xFFFFFFu) + ((u64)wave_sum((uint32_t)(v >> 24)) << 24);
}
__device__ __forceinline__ u64 wave_sum(u64 v) {
    return wave_all(v, [](u64 a, u64 b) { return a + b; });
}
// The sum over this lane and those before it.
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int o = 1; o < 64; o <<= 1) {
        const V x = __shfl_up(v, o);
        v += lane >= o ? x : 0;
    }
    return v;
}

__device__ __forceinline__ uint32_t key_of(float x) { // rises with x; zero has one sign
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ u64 order_of(float x, int id) { return (u64)key_of(x) << 32 | ~(uint32_t)id; }

// The tokens at a place of the order and before.
struct Cut {
    float x = -__builtin_inff();
    int id = 0x7FFFFFFF;
    Cut() = default;
    __device__ explicit Cut(u64 order) : x(value_of((uint32_t)(order >> 32))), id((int)~(uint32_t)order) {}
    __device__ __forceinline__ bool has(float v, int i) const { return v > x || (v == x && i <= id); }
    __device__ __forceinline__ u64 order() const { return order_of(x, id); }
};

struct Place {
    int bin, bin1;
    u64 before;
};

struct Shared {
    double exp2[1024];
    u64 mass[kBins];
    uint32_t count[kBins];
    u64 part[kWaves];
    struct {
        u64 order, mass;
    } few[kList];
    u64 before, found;
    uint32_t n;
    int bin;
    Place place;
    u64 pieces[kMaxVocab / 256]; // sums over 256 logits
};

// exp((x - top) / temperature) as a multiple of 2^-44.
struct Weights {
    float top;
    double scale; // log2(e) / temperature
    const double *exp2;
    __device__ __forceinline__ u64 operator()(float x) const {
        // 2^y = 2^(k / 1024) 2^r, |r| <= 2^-11: the next term of the series is 2^-50.  k is what an addition rounds y to, in its last bits.
        const double y = fmax(((double)x - (double)top) * scale, -100.0), z = y + 0x1.8p42;
        const int k = (int)__builtin_bit_cast(long long, z);
        const double r = y - (z - 0x1.8p42);
        constexpr double l = 0.693147180559945309417;
        const double p = fma(r, fma(r, fma(r, l * l * l / 6, l * l / 2), l), 1.0);
        const long long e = __builtin_bit_cast(long long, exp2[k & 1023]) + ((long long)(k >> 10) << 52);
        const double w = fma(__builtin_bit_cast(double, e), p, 0x1p52); // the nearest whole number, in its last bits
        return (u64)__builtin_bit_cast(long long, w) & ((1ull << 52) - 1);
    }
};

// A row's logits, four to a thread and chunk of 4096, read again by every pass (from the caches; held in registers, every pass was code fetched for one use, 92 us a
// row).  NaN and what is behind the row's end are -infinity.  infinite: the largest is, and counts as 0, all others as -infinity.
struct Four {
    float v[4];
};
template <class T>
struct Row {
    const T *p;
    int n;
    bool infinite;
    typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    static __device__ __forceinline__ float as_float(T v) {
        if constexpr (std::is_same_v<T, uint16_t>) return kv::bf16_float(v);
        else return (float)v;
    }
    __device__ __forceinline__ float value(T v) const {
        float x = fmaxf(as_float(v), -__builtin_inff());
        if (infinite) x = x == __builtin_inff() ? 0.f : -__builtin_inff();
        return x;
    }
    __device__ __forceinline__ float at(int i) const { return i < n ? value(p[i]) : -__builtin_inff(); }
    __device__ __forceinline__ int chunks() const { return (n + kChunk - 1) / kChunk; }
    __device__ __forceinline__ Four load(int j) const {
        const int i = kChunk * j + 4 * (int)threadIdx.x;
        Four f;
        if (kChunk * (j + 1) <= n) {
            const four v = *(const four *)(p + i);
#pragma unroll
            for (int e = 0; e < 4; e++) f.v[e] = value(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) f.v[e] = at(i + e);
        }
        return f;
    }
    // f(j, four logits, id of the first) for this thread's part of each chunk
    template <class F>
    __device__ __forceinline__ void fours(F f) const {
        Four next = load(0), then = load(1);
#pragma unroll 1
        for (int j = 0; j < chunks(); j++) {
            const Four v = next;
            next = then;
            if (j + 2 < chunks()) then = load(j + 2);
            f(j, v.v, kChunk * j + 4 * (int)threadIdx.x);
        }
    }
    // f(logit, id) for each
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        fours([&](int, const float (&v)[4], int id) {
#pragma unroll
            for (int e = 0; e < 4; e++) f(v[e], id + e);
        });
    }
};

// Bins of equal width in logits, the first from the top.
struct Bins {
    float top, per_unit;
    __device__ __forceinline__ float place(float x) const { return (top - x) * per_unit; }
    __device__ __forceinline__ int operator()(float x) const { return (int)fminf(place(x), (float)(kBins - 1)); } // of NaN (-infinity at no slope) the last
};

// The sum over the threads up to this one, given the wave's.
template <class V>
__device__ __forceinline__ V behind_waves(Shared &sh, V upto) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    V *part = (V *)sh.part;
    if (lane == 63) part[w] = upto;
    __syncthreads();
    V sum = upto;
#pragma unroll
    for (int i = 0; i < kWaves; i++) sum += i < w ? part[i] : 0;
    return sum;
}

// The first bins up to which `of` sums to at least `t0` (`t1`), and what is before the first; kBins - 1 if none.
template <class V>
__device__ __forceinline__ Place first_bins(Shared &sh, const V *of, V t0, V t1) {
    const int tid = threadIdx.x;
    const V a = of[2 * tid], b = of[2 * tid + 1];
    if (tid == 0) sh.place = {kBins - 1, kBins - 1, 0};
    const V upto = behind_waves(sh, wave_scan(a + b)), at = upto - b, under = at - a;
    if (upto >= t0 && (under < t0 || tid == 0)) sh.place.bin = at >= t0 ? 2 * tid : 2 * tid + 1, sh.place.before = at >= t0 ? under : at; // one thread
    if (upto >= t1 && (under < t1 || tid == 0)) sh.place.bin1 = at >= t1 ? 2 * tid : 2 * tid + 1;
    __syncthreads();
    return sh.place;
}

// Of the sh.n <= kList tokens in the list: which brings the sum over those not behind it, and `before`, to `target`.  False if none does, or one before them all does.
// (The waves share the sums out.)
__device__ __forceinline__ bool among_few(Shared &sh, u64 before, u64 target) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = (int)sh.n;
    if (tid < n) sh.mass[tid] = before;
    __syncthreads();
    for (int i = lane; i < n; i += 64) {
        const u64 o = sh.few[i].order;
        u64 sum = 0;
#pragma unroll 2
        for (int j = w; j < n; j += kWaves) sum += sh.few[j].order >= o ? sh.few[j].mass : 0;
        atomicAdd(&sh.mass[i], sum);
    }
    __syncthreads();
    const bool here = tid < n && sh.mass[tid] >= target && sh.mass[tid] - sh.few[tid].mass < target;
    if (here) sh.found = sh.few[tid].order;
    return __syncthreads_or(here) != 0;
}

// The place in the order (inclusive) at which the weights of the tokens of `cut`, summed from the front, reach `target`, which they do.  MASS: by weight, otherwise a
// token counts one.
template <bool MASS, class R>
__device__ __attribute__((noinline)) u64 reach(Shared &sh, const R row, const Weights weight, u64 least, u64 target) {
    const int tid = threadIdx.x;
    u64 lo = least, hi = order_of(weight.top, 0), before = 0;
    for (;;) {
        const int shift = max(0, 64 - __builtin_clzll((hi - lo) | 1) - 11); // bins of 2^shift places in the order below hi
        for (int i = tid; i < kBins; i += kThreads) sh.mass[i] = 0, sh.count[i] = 0;
        __syncthreads();
        row.each([&](float x, int id) {
            const u64 o = order_of(x, id);
            if (o < lo || o > hi) return;
            if (MASS) atomicAdd(&sh.mass[(hi - o) >> shift], weight(x));
            atomicAdd(&sh.count[(hi - o) >> shift], 1u);
        });
        __syncthreads();
        // bins 2 tid and 2 tid + 1 of this thread, and what is before them
        const u64 w0 = MASS ? sh.mass[2 * tid] : sh.count[2 * tid], w1 = MASS ? sh.mass[2 * tid + 1] : sh.count[2 * tid + 1];
        const u64 upto = behind_waves(sh, wave_scan(w0 + w1)) + before;
        const u64 b0 = upto - w1 - w0, b1 = upto - w1;
        if (b0 < target && upto >= target) { // one thread
            const bool second = b1 < target;
            sh.bin = 2 * tid + second, sh.before = second ? b1 : b0;
        }
        __syncthreads();
        const int bin = sh.bin;
        before = sh.before;
        if (tid == 0) sh.n = 0;
        const u64 top = hi - ((u64)bin << shift), under = (1ull << shift) - 1;
        hi = top, lo = top - min(under, top - lo);
        __syncthreads();
        if (sh.count[bin] <= kList) {
            row.each([&](float x, int id) {
                const u64 o = order_of(x, id);
                if (o < lo || o > hi) return;
                const uint32_t at = atomicAdd(&sh.n, 1u);
                sh.few[at] = {o, MASS ? weight(x) : 1};
            });
            __syncthreads();
            among_few(sh, before, target);
            return sh.found;
        }
        __syncthreads();
    }
}

template <class T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const T *logits, int vocab, int64_t stride, SampleSettings s, int32_t *ids) {
    __shared__ Shared sh;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    Row<T> row{logits + r * stride, vocab, false};
    const float temperature = s.temperature ? s.temperature[r] : s.temperature0;
    const int k = s.top_k ? s.top_k[r] : s.top_k0;
    const float p = s.top_p ? s.top_p[r] : s.top_p0, least_p = s.min_p ? s.min_p[r] : s.min_p0, u = s.u ? s.u[r] : s.u0;
    sh.exp2[tid] = kExp2.v[tid];
    for (int i = tid; i < kBins; i += kThreads) sh.count[i] = 0, sh.mass[i] = 0;
    if (tid == 0) sh.n = 0;

    // the first of the order
    float most = -__builtin_inff();
    int most_id = 0; // for the greedy alone
    if (temperature > 0.f) {
        row.fours([&](int, const float (&x)[4], int) { most = fmaxf(most, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))); });
    } else {
        row.each([&](float x, int id) {
            if (x > most) most = x, most_id = id;
        });
    }
    {
        u64 first = wave_all(order_of(most, most_id), [](u64 a, u64 b) { return a > b ? a : b; });
        if (lane == 0) sh.part[w] = first;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; i++) first = sh.part[i] > first ? sh.part[i] : first;
        const float x = value_of((uint32_t)(first >> 32));
        const bool none = x == -__builtin_inff();
        if (none || !(temperature > 0.f)) {
            if (tid == 0) ids[r] = none ? -1 : (int32_t)~(uint32_t)first;
            return;
        }
        row.infinite = x == __builtin_inff();
        if (row.infinite) most = most == x ? 0.f : -__builtin_inff();
        sh.found = first;
        __syncthreads();
    }
    const float top = row.infinite ? 0.f : value_of((uint32_t)(sh.found >> 32));
    const Weights weight{top, 1.4426950408889634074 / (double)temperature, sh.exp2};
    const Bins bins{top, fminf(128.f / temperature, 3e38f)};

    const double least_w = ceil((double)fminf(fmaxf(least_p, 0.f), 1.f) * 0x1p44);
    const u64 least = (u64)least_w;
    auto block_sum = [&](u64 v) {
        v = wave_sum(v);
        if (lane == 0) sh.part[w] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < kWaves; i++) v += sh.part[i];
        __syncthreads();
        return v;
    };
    auto border = [&](u64 all) { // the sum that top_p asks for
        const double share = ceil((double)p * (double)all);
        return min(share > 1.0 ? (u64)share : 1ull, all); // the first is always kept
    };
    auto passed_by = [&](u64 sum) { // the first running sum above this is the answer's, at the latest the last
        const double share = (u > 0.f ? (double)u : 0.0) * (double)sum;
        const u64 passed = share < (double)sum ? (u64)share : sum - 1;
        return passed < sum ? passed : sum - 1;
    };

    Cut cut; // what is kept
    if (k > 0 && k < vocab) {
        int last = kBins - 1;
        if (k <= kThreads) { // as many tokens as threads whose largest logit lies in a bin or before
            atomicAdd(&sh.count[bins(most)], 1u);
            __syncthreads();
            last = first_bins<uint32_t>(sh, sh.count, k, k).bin;
            sh.count[tid] = sh.count[tid + kThreads] = 0;
            __syncthreads();
        }
        const float end = last == kBins - 1 ? __builtin_inff() : (float)(last + 1);
        row.fours([&](int, const float (&x)[4], int) {
            if (__ballot(bins.place(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))) < end))
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (bins.place(x[e]) < end) atomicAdd(&sh.count[bins(x[e])], 1u);
        });
        __syncthreads();
        const Place place = first_bins<uint32_t>(sh, sh.count, k, k);
        const int bin = place.bin;
        const bool few = sh.count[bin] <= kList && bin < kBins - 1;
        const bool all_few = few && place.before + sh.count[bin] <= kList; // all that top-k keeps: the rest is done in the list
        bool found = false;
        if (few) {
            const float from = all_few ? 0.f : (float)bin;
            row.fours([&](int, const float (&x)[4], int id) {
                if (__ballot(bins.place(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))) < (float)(bin + 1)))
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float d = bins.place(x[e]);
                        if (d >= from && d < (float)(bin + 1)) {
                            const uint32_t at = atomicAdd(&sh.n, 1u);
                            if (at < kList) sh.few[at] = {order_of(x[e], id + e), 1};
                        }
                    }
            });
            __syncthreads();
            found = among_few(sh, all_few ? 0 : place.before, (u64)k);
        }
        if (found && all_few) {
            const bool is = tid < (int)sh.n;
            const u64 order = is ? sh.few[tid].order : 0;
            u64 o = sh.found, m = is && order >= o ? weight(value_of((uint32_t)(order >> 32))) : 0;
            if (p < 1.f) {
                if (is) sh.few[tid].mass = m;
                among_few(sh, 0, border(block_sum(m)));
                o = sh.found;
            }
            if (order < o || m < least) m = 0;
            __syncthreads();
            if (is) sh.few[tid] = {(uint32_t)order, m}; // the lower id counts as the later
            among_few(sh, 0, passed_by(block_sum(m)) + 1);
            if (tid == 0) ids[r] = (int32_t)~(uint32_t)sh.found;
            return;
        }
        const u64 o = found ? sh.found : reach<false>(sh, row, weight, 0, (u64)k);
        cut = Cut(o);
        __syncthreads();
        if (tid == 0) sh.n = 0;
        if (p < 1.f)
            for (int i = tid; i < kBins; i += kThreads) sh.mass[i] = 0;
        __syncthreads();
    }
    const int pieces = kWaves * row.chunks();
    // Sums over 256 logits that follow one another, a wave's of a chunk, of the tokens of `cut` in the bins before `first`; the sum of all of its weights and that before
    // the bin; and its tokens in the bins first..last.
    u64 all = 0, front = 0;
    auto exact = [&](auto with_bins, float first, float last) {
        constexpr bool BINS = decltype(with_bins)::value;
        const bool some = cut.id != 0x7FFFFFFF; // not all tokens
        all = front = 0;
        row.fours([&](int j, const float (&x)[4], int id) {
            u64 sum = 0, m[4];
            float d[4];
            const float largest = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            if (__ballot(largest >= cut.x)) {
#pragma unroll
                for (int e = 0; e < 4; e++) m[e] = weight(x[e]); // no branches: the four side by side
                if (some)
#pragma unroll
                    for (int e = 0; e < 4; e++) m[e] = cut.has(x[e], id + e) ? m[e] : 0;
                if constexpr (BINS) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        d[e] = bins.place(x[e]);
                        all += m[e];
                        u64 f = d[e] < first ? m[e] : 0;
                        front += f;
                        if (least) f = f >= least ? f : 0;
                        sum += f;
                    }
                    if (__ballot(bins.place(largest) < last))
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (d[e] >= first && d[e] < last && cut.has(x[e], id + e)) {
                                const uint32_t at = atomicAdd(&sh.n, 1u);
                                if (at < kList) sh.few[at] = {order_of(x[e], id + e), m[e]};
                            }
                } else {
                    if (least)
#pragma unroll
                        for (int e = 0; e < 4; e++) m[e] = m[e] >= least ? m[e] : 0;
                    sum = (m[0] + m[1]) + (m[2] + m[3]);
                }
                sum = wave_sum48(sum);
            }
            if (lane == 0) sh.pieces[kWaves * j + w] = sum;
        });
    };
    bool done = false;
    if (p < 1.f) {
        // weights of fp32 as multiples of 2^-31, and the sum of all as floats have it
        const float slope = -1.44269504f / 128.f;
        const bool some = cut.id != 0x7FFFFFFF;
        float part = 0.f;
        row.fours([&](int, const float (&x)[4], int id) {
            if (!__ballot(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) >= cut.x)) return;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = bins.place(x[e]);
                float m = __builtin_amdgcn_exp2f(fmaxf(d, 0.f) * slope);
                if (some) m = cut.has(x[e], id + e) ? m : 0.f;
                part += m;
                const uint32_t whole = (uint32_t)(m * 0x1p31f);
                if (whole && d < (float)(kBins - 1)) atomicAdd(&sh.mass[(int)d], (u64)whole);
            }
        });
        for (int o = 32; o; o >>= 1) part += __shfl_xor(part, o);
        float *parts = (float *)sh.part;
        if (lane == 0) parts[w] = part;
        __syncthreads();
        part = 0.f;
#pragma unroll
        for (int i = 0; i < kWaves; i++) part += parts[i];
        __syncthreads();
        const float margin = part * 0x1p-16f, near = fmaxf(p, 0.f) * part;
        const Place in_question = first_bins<u64>(sh, sh.mass, (u64)(fmaxf(near - margin, 0.f) * 0x1p31f), (u64)((near + margin) * 0x1p31f));
        exact(std::true_type{}, (float)in_question.bin, in_question.bin1 == kBins - 1 ? __builtin_inff() : (float)(in_question.bin1 + 1));
        all = block_sum(all), front = block_sum(front);
        const u64 target = border(all);
        done = sh.n <= kList && among_few(sh, front, target);
        if (done) {
            const u64 o = sh.found;
            if (tid < (int)sh.n && sh.few[tid].order >= o && sh.few[tid].mass >= least) atomicAdd(&sh.pieces[~(uint32_t)sh.few[tid].order >> 8], sh.few[tid].mass);
            cut = Cut(o);
        } else {
            cut = Cut(reach<true>(sh, row, weight, cut.order(), target));
        }
    }
    if (!done) exact(std::false_type{}, 0.f, 0.f);
    __syncthreads();
    if (w) return;
    // the piece, then the token, at which the running sum passes u of the whole; at the latest the last one with a weight
    const int each = (pieces + 63) / 64;
    u64 own = 0;
    for (int i = 0; i < each; i++) own += lane * each + i < pieces ? sh.pieces[lane * each + i] : 0;
    const u64 upto = wave_scan(own), sum = shfl(upto, 63);
    const u64 passed = passed_by(sum);
    const u64 has = __ballot(upto > passed);
    const int at = __builtin_ctzll(has);
    u64 before = shfl(upto - own, at);
    int i = at * each;
    while (before + sh.pieces[i] <= passed) before += sh.pieces[i++];
    const int id = 256 * i + 4 * lane;
    u64 m[4], mine = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float x = row.at(id + e);
        const u64 v = weight(x);
        mine += m[e] = cut.has(x, id + e) && v >= least ? v : 0;
    }
    const u64 end = wave_scan(mine) + before;
    const u64 hit = __ballot(end > passed);
    if (lane == __builtin_ctzll(hit)) {
        u64 c = end - mine;
        int e = 0;
        for (int f = 0; f < 3; f++)
            if (e == f && c + m[f] <= passed) c += m[f], e = f + 1;
        ids[r] = id + e;
    }
}

template <class T>
void launch(const void *logits, int rows, int vocab, int64_t stride, const SampleSettings &s, int32_t *ids, hipStream_t st) {
    l2_launch(sample_kernel<T>, dim3(rows), dim3(kThreads), 0, st, (const T *)logits, vocab, stride, s, ids);
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
    for (const void *f : {(const void *)sample_kernel<float>, (const void *)sample_kernel<_Float16>, (const void *)sample_kernel<uint16_t>})
        L2_HIP(hipFuncGetAttributes(&a, f));
    return L2_OK;
}
