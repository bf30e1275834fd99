// Attention of new rows over a cache in pages: out = sum over t of softmax(scale q.k_t) v_t, in one pass with a running maximum and sum.
//
// Both products are the matrix cores', transposed: S^T = K q^T and O^T = V^T P^T.  The result of the first has a row of queries in each lane and its
// positions in the lane's registers, which is the second operand of the second product as it stands, once the rows of K are dealt to the lanes in
// the fitting order; maxima and sums are a lane's own but for two exchanges, and the factors between tiles one register.  V lies transposed in the pool, so
// nothing is transposed here.  Codes of 8 bits become 16-bit floats exactly (fp16).  Scales of keys multiply the scores, those of values the weights.
//
// Weights enter the second product in 16 bits, times a factor that cancels in the quotient with their sum: p_t = exp2(s_t - off).  `off` follows the largest s_t + log2 of the
// scale of v_t, so that p_t * (scale of v_t) is what is bounded, by 2^15 for fp16, and the largest of these is 2^7 or more (over bf16 2^-16 and 2^-24, whose small numbers are as good: sums over 2^16 positions are finite, whatever the values): off goes to 7 below it, and
// is left where it is until it lies more than 8 higher, so that sums are seldom rescaled (a tile of 32 rows would have a new maximum among them nearly always).  The largest s
// with the largest scale of a tile, which a product of less weight may have, only says whether that may be so: where it may, the positions are gone over one by one.
// Weights, times scales, are two fp16 numbers each (to within 2^-22, and no less than 2^-32 of the largest) or, over a pool in bf16, two of bf16 (2^-16) for rows of 16 bits and three for
// fp32 rows.  One would be what a result's own rounding is: of rows in fp16 and bf16 over pools in i8 and bf16 they then were off by 1.4 and 1.3 times what fp32 weights leave, 2.9e-4 for
// 2.1e-4 and 2.1e-3 for 1.6e-3.  q is one number where that holds it as it is, as many as a weight for fp32 rows, two for fp16 rows over bf16; for fp16 numbers scaled by a power of two per
// row, so that they hold what bf16 and fp32 rows may contain.
// Values of 16 bits that are not finite would be NaN times the second number of a weight, or times one that is zero, and for rows that do not see them: they are taken out of
// tiles that some row may not see whole, and sums that are not finite behind the last tile, or lack some, are made from the values that are not (repair).
#include <algorithm>

#include "kvpool.h"
#include "lanes.h"

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
using kv::f4;
using kv::f8;
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLeastE = -67.f; // rows whose values are held at all have scales from 2^-67
constexpr float kSlack = 8.f;
constexpr float base_of(int kv_type) { return kv_type == L2_KV_BF16 ? -24.f : 7.f; }

// `off` behind a tile whose largest score times its factor, with the scale of its values, is `top`, and the factor of the sums so far.
template <int KV>
__device__ __forceinline__ bool raises(float off, float top) {
    return top - base_of(KV) > off + kSlack;
}
template <int KV>
__device__ __forceinline__ float follow(float &off, float top) {
    const float to = top - base_of(KV);
    if (!raises<KV>(off, top)) return 1.f; // or nothing is seen
    const float f = __builtin_amdgcn_exp2f(off - to);
    off = to;
    return f;
}
// 2^e above x; x as a power of two.
__device__ __forceinline__ float above(float x) { return x > 0.f ? fmaxf((float)__builtin_amdgcn_frexp_expf(x), kLeastE) : kLeastE; }
__device__ __forceinline__ float log2_of(float x) { return fmaxf(__builtin_amdgcn_logf(x), kLeastE); }

// Of a row of q whose largest number is `top`: times 2^e for fp16, and `c`, the exponent of two per unit of the scores' sums, times scales (of keys) that come as scale_of_key().
// The largest number of q is in [2^14, 2^15), or as far below as it takes for c to be a normal number: a c of zero would make NaN of a score that is not seen, and
// scores that so small a factor goes with are next to zero.  Sums times scales are up to 2^152 of i8, hence the 2^-24.
template <bool EIGHT>
__device__ __forceinline__ int fit_q(float top, float &c) {
    constexpr int kKey = EIGHT ? 24 : 0;
    const int most = 125 + kKey + __builtin_amdgcn_frexp_expf(c);
    const int e = min(top > 0.f && top < kInf ? 15 - __builtin_amdgcn_frexp_expf(top) : 0, most);
    c = fminf(ldexpf(c, kKey - e), 0x1p127f); // at 2^127 scores are far apart or the same
    return e;
}
__device__ __forceinline__ float scale_of_key(float s) { return s * 0x1p-24f; }

// What a pool's cells become for the matrix cores: eight of them, from 8 (16) bytes.
template <int KV>
struct Cells {
    static constexpr bool kEight = KV <= L2_KV_E4M3, kHalf = KV != L2_KV_BF16;
    static constexpr int kSize = kEight ? 1 : 2;
    using Frag = std::conditional_t<kHalf, h8, b8>;
    using One = std::conditional_t<kHalf, _Float16, __bf16>;
    // frag v of 16 bytes: 8 of their 16 codes, or all 8 cells
    static __device__ __forceinline__ Frag frag(const u4 &x, int v) {
        if constexpr (KV == L2_KV_I8) {
            u4 out;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t b = x[2 * v + i] ^ 0x80808080u; // c + 128, and as the last byte of an fp16 number 1024 + c + 128
                const h2 k = {(_Float16)-1152.f, (_Float16)-1152.f};
                out[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + k);
                out[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + k);
            }
            return __builtin_bit_cast(h8, out);
        } else if constexpr (KV == L2_KV_E4M3) {
            u4 out;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                out[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x[2 * v + i], 1.f, false));
                out[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x[2 * v + i], 1.f, true));
            }
            return __builtin_bit_cast(h8, out);
        } else {
            return __builtin_bit_cast(Frag, x);
        }
    }
};

__device__ __forceinline__ f4 mfma16(const h8 &a, const h8 &b, const f4 &c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma16(const b8 &a, const b8 &b, const f4 &c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// x as a sum of NP numbers of 16 bits, each the nearest to what those before it leave.  Two at a time, as one instruction converts them and takes the numbers out of its
// result again; that is a value which the compiler knows nothing of, so that it cannot make a product and its rounding one operation for one of the two places it goes to.
template <class Frag, class One, int NP>
__device__ __forceinline__ void pieces(f8 x, Frag (&out)[NP]) {
    typedef One two __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    float minus = -1.f; // unknown too: a product with a number of 16 bits and a sum are one instruction, a difference from one is two
    if (NP > 1) asm("" : "+s"(minus));
#pragma unroll
    for (int i = 0; i < NP; i++) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x[j], x[j + 1]}, two));
            if (i + 1 < NP) asm("" : "+v"(bits));
            const two n = __builtin_bit_cast(two, bits);
            out[i][j] = n[0], out[i][j + 1] = n[1];
            if (i + 1 < NP) x[j] = fmaf((float)n[0], minus, x[j]), x[j + 1] = fmaf((float)n[1], minus, x[j + 1]);
        }
    }
}

// The positions that the rows of a tile of queries have to do with, in tiles of TT: those of the first tokens that stay visible, then those from the
// first row's window (or from the start) to the last row's own.
struct Range {
    int sinks_end, first, n; // tile i is i below sinks_end, first + i - sinks_end from there on
    __device__ __forceinline__ int tile(int i) const { return i < sinks_end ? i : first + i - sinks_end; }
};
template <int TT>
__device__ __forceinline__ Range range_of(const KvAttention &a, int pos_first, int pos_last) {
    if (pos_last < 0) return {0, 0, 0};
    const int end = pos_last / TT + 1;
    if (!a.window) return {0, 0, end};
    const int from = max(0, max(pos_first, 0) - a.window + 1) / TT;
    const int se = min((int)(((int64_t)a.sinks + TT - 1) / TT), from);
    return {se, from, se + end - from};
}

// What the row of position pos sees: up to pos, from `from` on or below `sinks`.
struct Seen {
    int pos, from, sinks;
    __device__ __forceinline__ Seen(const KvAttention &a, int pos) : pos(pos), from(a.window ? max(pos - a.window + 1, 0) : 0), sinks(a.sinks) {}
    __device__ __forceinline__ bool operator()(int t) const { return (t <= pos) & ((t >= from) | (t < sinks)); }
};

// v with fp16 (bf16) numbers that are not finite as zeros, and whether there are any.
template <int KV>
__device__ __forceinline__ u4 finite(u4 v, bool &odd) {
    constexpr uint32_t ones = KV == L2_KV_F16 ? 0x7C00u : 0x7F80u;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const bool lo = (v[r] & ones) == ones, hi = (v[r] >> 16 & ones) == ones;
        odd |= lo || hi;
        v[r] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
    }
    return v;
}

// The sums of a row over tiles whose values may not be finite: those that are not finite as a number that no sum is, so that a value that the row sees makes it that, or NaN;
// and what is left behind all values.
constexpr float kBroken = 0x1.fffffep127f;
__device__ __forceinline__ float broken(float sum) { return fabsf(sum) < kInf ? sum : kBroken; }
__device__ __forceinline__ float mended(float sum) { return sum == kBroken ? __builtin_nanf("") : sum; }
// A cell that is not finite, or else zero.
template <int KV>
__device__ __forceinline__ float not_finite(uint16_t bits) {
    const float v = KV == L2_KV_F16 ? (float)__builtin_bit_cast(_Float16, bits) : kv::bf16_float(bits);
    return fabsf(v) < kInf ? 0.f : v;
}
// A part's sum times its factor, which may be zero.
__device__ __forceinline__ float times(float sum, float f) { return fabsf(sum) < kInf ? sum * f : sum; }

constexpr int kNarrowRows = 16, kNarrowWaves = 4;

// The numbers that a weight is, of rows whose q is NQ.
constexpr int weight_numbers(int nq) { return nq == 3 ? 3 : 2; }

// How a launch cuts positions: `splits` parts of `per` tiles each, `stride` parts of a row in the workspace; and the query rows per kv head of a sequence up to which
// it is the narrow kernel's.
struct Cut {
    int splits, per, stride, narrow;
};

// A query row's part: what a block found of it.  `off` is common to the weights in acc and sum.
struct Parts {
    float *acc;   // [row][head][split][D]
    float2 *stat; // [row][head][split]: off, sum
};

// Sequences of few query rows per kv head (new tokens x query heads of the group).  A block has 16 rows of one sequence and kv head and part of the positions, its
// four waves tiles of 64 positions (32 of 16-bit cells) in turn, straight from memory into registers: 8 KB of keys and 8 KB of values, the next tile's keys
// asked for once this one's scores are there and its values once this one's are summed.  LDS only joins the waves: a row of V^T or K is read by one wave alone.
// Bound by memory where the launch fills the chip: 32 sequences' next tokens, 64 heads on 8, up to 4096 positions in e4m3, 49 us (29 at the 6.3 TB/s
// of launches that only read); one behind 60001 positions of 32 heads in i8, 103 us (80).  One behind 500 takes 11 us: two launches, and in each two or three trips
// to memory that wait for one another.
template <int KV, int NQ, int D>
__global__ __launch_bounds__(64 * kNarrowWaves, 2) void kv_narrow_kernel(KvLayer l, l2_kvbatch b, KvAttention a, Parts parts, Cut cut) {
    using C = Cells<KV>;
    using Frag = typename C::Frag;
    constexpr int TT = 64 / C::kSize, ST = TT / 16, CH = TT / 4, FR = 2 / C::kSize, KL = D * C::kSize / 64, DT = D / 16, VS = TT / 32, NP = weight_numbers(NQ);
    const int split = blockIdx.x % cut.splits, r0 = kNarrowRows * (blockIdx.x / cut.splits), h = blockIdx.y, i = blockIdx.z;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const kv::Seq s = kv::sequence(b, i);
    const int group = a.n_heads / l.n_heads, rows = s.rows * group;
    if (r0 >= rows || rows > cut.narrow) return;
    const int base = s.length - s.rows; // position of the first row
    const bool real = r0 + m < rows;
    const Seen seen(a, real ? base + (r0 + m) / group : -1);
    const int64_t q_row = s.first + (real ? (r0 + m) / group : 0), head = h * group + (real ? (r0 + m) % group : 0);

    const Range range = range_of<TT>(a, base, s.length - 1);
    const int begin = min(split * cut.per, range.n), end = min(begin + cut.per, range.n);
    const int size = 1 << l.page_shift;
    const char *kb = (const char *)l.k, *vb = (const char *)l.v;

    u4 kr[ST][KL], vr[DT];
    f4 ks[ST], vs[ST];
    int page_k, page_v; // of the tile that is asked for next: of this lane's row of K, and of its positions
    auto pages = [&](int n) {
        const int t0 = range.tile(n) * TT;
        page_k = kv::page_at(b, l.n_pages, i, (t0 + CH * (m >> 2)) >> l.page_shift);
        page_v = kv::page_at(b, l.n_pages, i, (t0 + CH * g) >> l.page_shift);
    };
    auto load_k = [&](int n, int page, int own) {
        const int t0 = range.tile(n) * TT;
        const int64_t ph = (int64_t)max(page, 0) * l.n_heads + h;
        const char *p = kb + ((ph * size + ((t0 + CH * (m >> 2)) & (size - 1)) + (m & 3)) * D * C::kSize + 16 * g);
#pragma unroll
        for (int x = 0; x < ST; x++)
#pragma unroll
            for (int u = 0; u < KL; u++) kr[x][u] = *(const u4 *)(p + 4 * x * D * C::kSize + 64 * u);
        if (C::kEight) {
            const float *sc = l.k_scale + (((int64_t)max(own, 0) * l.n_heads + h) * size + ((t0 + CH * g) & (size - 1)));
#pragma unroll
            for (int x = 0; x < ST; x++) ks[x] = *(const f4 *)(sc + 4 * x);
        }
    };
    auto load_v = [&](int n, int page) {
        const int t0 = range.tile(n) * TT;
        const int64_t ph = (int64_t)max(page, 0) * l.n_heads + h;
        const int slot = (t0 + CH * g) & (size - 1);
        const char *p = vb + ((ph * D + m) * size + slot) * C::kSize;
#pragma unroll
        for (int x = 0; x < DT; x++) vr[x] = *(const u4 *)(p + (int64_t)16 * x * size * C::kSize);
        if (C::kEight) {
            const float *sc = l.v_scale + (ph * size + slot);
#pragma unroll
            for (int x = 0; x < ST; x++) vs[x] = *(const f4 *)(sc + 4 * x);
        }
    };

    // What the first tile waits for is asked for in the order of its waits: pages and q, then keys and values.
    int n = begin + w;
    page_k = page_v = -1;
    if (n < end) pages(n);
    kv::raw8 q_raw[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; k++)
        q_raw[k] = kv::load_raw8(a.q, a.type, q_row * a.q_stride + head * D + (k / FR) * (64 / C::kSize) + (16 / C::kSize) * g + 8 * (k % FR));
    int here = page_v;
    if (n < end) {
        load_k(n, page_k, page_v);
        load_v(n, page_v);
        if (n + kNarrowWaves < end) pages(n + kNarrowWaves);
    }
    // q: this lane's row, the dimensions that lie across from its 16 bytes of a key
    Frag q[D / 32][NQ];
    float c; // exponent of two per unit of the scores' sums
    {
        f8 x[D / 32];
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < D / 32; k++) {
            x[k] = kv::values8(q_raw[k], a.type);
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[k][j]));
        }
        c = a.scale * kLog2e;
        if (C::kHalf) {
            top = lanes::rows_max(top);
            const int e = fit_q<C::kEight>(top, c);
#pragma unroll
            for (int k = 0; k < D / 32; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = ldexpf(x[k][j], e);
        }
#pragma unroll
        for (int k = 0; k < D / 32; k++) pieces<Frag, typename C::One, NQ>(x[k], q[k]);
    }

    f4 acc[DT] = {};
    float off = -kInf, sum = 0.f;
    bool odd = false; // values were taken out
    for (; n < end; n += kNarrowWaves) {
        const int t0 = range.tile(n) * TT;
        const bool more = n + kNarrowWaves < end;
        f4 sc[ST] = {};
#pragma unroll
        for (int k = 0; k < D / 32; k++)
#pragma unroll
            for (int x = 0; x < ST; x++) {
                const Frag f = C::frag(kr[x][k / FR], k % FR);
#pragma unroll
                for (int y = 0; y < NQ; y++) sc[x] = mfma16(f, q[k][y], sc[x]);
            }
        if (C::kEight)
#pragma unroll
            for (int x = 0; x < ST; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) sc[x][r] *= scale_of_key(ks[x][r]);
        const int here_next = page_v;
        if (more) load_k(n + kNarrowWaves, page_k, page_v);

        // positions CH g + 4 x + r of the tile are this lane's
        const bool whole = t0 + TT - 1 <= base && (!a.window || t0 > s.length - 1 - a.window || t0 + TT <= a.sinks) && __ballot(here < 0) == 0;
        if (!whole) {
#pragma unroll
            for (int x = 0; x < ST; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool see = (here >= 0) & seen(t0 + CH * g + 4 * x + r);
                    sc[x][r] = see ? sc[x][r] : -kInf;
                    if (C::kEight) vs[x][r] = see ? vs[x][r] : 0.f;
                }
            if (!C::kEight)
#pragma unroll
                for (int x = 0; x < DT; x++) vr[x] = finite<KV>(vr[x], odd);
        }
        float mx = -kInf;
#pragma unroll
        for (int x = 0; x < ST; x++)
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, sc[x][r]);
        float top = lanes::rows_max(mx) * c;
        if (C::kEight) {
            float mv = 0.f;
#pragma unroll
            for (int x = 0; x < ST; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) mv = fmaxf(mv, vs[x][r]);
            top += above(lanes::rows_max(mv));
            if (__ballot(raises<KV>(off, top))) {
                top = -kInf;
#pragma unroll
                for (int x = 0; x < ST; x++)
#pragma unroll
                    for (int r = 0; r < 4; r++) top = fmaxf(top, fmaf(sc[x][r], c, log2_of(vs[x][r])));
                top = lanes::rows_max(top);
            }
        }
        const float f = follow<KV>(off, top);
        if (__ballot(f != 1.f)) {
#pragma unroll
            for (int x = 0; x < DT; x++) acc[x] *= f;
            sum *= f;
        }
        const float now = off == -kInf ? 0.f : off; // nothing seen yet: every weight is exp2(-inf)
#pragma unroll
        for (int v = 0; v < VS; v++) {
            f8 p;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float t = __builtin_amdgcn_exp2f(fmaf(sc[2 * v + j / 4][j % 4], c, -now));
                sum += t;
                p[j] = C::kEight ? t * vs[2 * v + j / 4][j % 4] : t;
            }
            Frag pf[NP];
            pieces<Frag, typename C::One, NP>(p, pf);
#pragma unroll
            for (int x = 0; x < DT; x++) {
                const Frag fr = C::frag(vr[x], v);
#pragma unroll
                for (int y = 0; y < NP; y++) acc[x] = mfma16(fr, pf[y], acc[x]);
            }
        }
        here = here_next;
        if (more) {
            load_v(n + kNarrowWaves, page_v);
            if (n + 2 * kNarrowWaves < end) pages(n + 2 * kNarrowWaves);
        }
    }
    sum = lanes::rows_sum(sum);
    if constexpr (!C::kEight) {
#pragma unroll
        for (int x = 0; x < DT; x++)
#pragma unroll
            for (int r = 0; r < 4; r++) odd |= !(fabsf(acc[x][r]) < kInf);
        if (__ballot(odd)) { // repair: position by position
#pragma unroll
            for (int x = 0; x < DT; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[x][r] = broken(acc[x][r]);
#pragma unroll 1
            for (int y = TT * (begin + w); y < TT * end; y += y % TT == TT - 1 ? TT * (kNarrowWaves - 1) + 1 : 1) {
                const int t = range.tile(y / TT) * TT + y % TT, page = kv::page_at(b, l.n_pages, i, t >> l.page_shift);
                if (page < 0 || !seen(t)) continue;
                const uint16_t *p = (const uint16_t *)vb + ((((int64_t)page * l.n_heads + h) * D + 4 * g) * size + (t & (size - 1)));
#pragma unroll
                for (int x = 0; x < DT; x++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[x][r] += not_finite<KV>(p[(int64_t)(16 * x + r) * size]);
            }
#pragma unroll
            for (int x = 0; x < DT; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[x][r] = mended(acc[x][r]);
        }
    }

    // the waves' parts together
    constexpr int LD = D + 4;
    __shared__ float sh_acc[kNarrowWaves][kNarrowRows][LD];
    __shared__ float2 sh_stat[kNarrowWaves][kNarrowRows];
#pragma unroll
    for (int x = 0; x < DT; x++) *(f4 *)&sh_acc[w][m][16 * x + 4 * g] = acc[x];
    if (g == 0) sh_stat[w][m] = make_float2(off, sum);
    __syncthreads();
    for (int x = threadIdx.x; x < min(rows - r0, kNarrowRows) * (D / 4); x += 64 * kNarrowWaves) {
        const int r = x / (D / 4), d = 4 * (x % (D / 4));
        float o = -kInf, total = 0.f;
#pragma unroll
        for (int y = 0; y < kNarrowWaves; y++) o = fmaxf(o, sh_stat[y][r].x);
        f4 v = {};
#pragma unroll
        for (int y = 0; y < kNarrowWaves; y++) {
            const float2 st = sh_stat[y][r];
            const float f = st.x == o ? 1.f : __builtin_amdgcn_exp2f(st.x - o);
            if (st.y == 0.f && st.x == -kInf) continue;
            total += st.y * f;
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] += times(sh_acc[y][r][d + j], f);
        }
        const int64_t row = s.first + (r0 + r) / group, hq = h * group + (r0 + r) % group;
        if (cut.splits == 1) {
            const float inv = total == 0.f ? 0.f : 1.f / total;
            for (int j = 0; j < 4; j++) v[j] = total == 0.f ? 0.f : v[j] * inv;
            kv::store4(a.out, a.type, row * a.out_stride + hq * D + d, v);
        } else {
            const int64_t at = (row * a.n_heads + hq) * cut.stride + split;
            *(f4 *)(parts.acc + at * D + d) = v;
            if (d == 0) parts.stat[at] = make_float2(o, total);
        }
    }
}

// What lane M of a row of 16 lanes has, for every lane of the row.
template <int M>
__device__ __forceinline__ float scale_at(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + M, 0xF, 0xF, true));
}
template <class F, int... I>
__device__ __forceinline__ void each_of(const F &f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(const F &f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

__device__ __forceinline__ float row_max(float v) { // of a row of 16 lanes: 1, then 2 away; the other four, the other eight
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true)));
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true)));
    return v;
}
__device__ __forceinline__ float wave_max(float v) { return lanes::rows_max(row_max(v)); }

// Joins the parts of each query row.  Of up to kFewParts parts (FEW) a wave has a row and head to itself, its lanes a part's statistics each; of more the four waves of a
// block share one, parts in turn.  NARROW: block x has row x % most of sequence x / most, most rows at the most; else row x.
constexpr int kJoinWaves = 4, kFewParts = 8;
template <int D, bool NARROW, bool FEW>
__global__ __launch_bounds__(64 * kJoinWaves) void kv_join_kernel(l2_kvbatch b, KvAttention a, Parts parts, int splits, int stride, int group, int most) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, hq = FEW ? kJoinWaves * blockIdx.y + w : blockIdx.y;
    const int i = NARROW ? (int)blockIdx.x / most : kv::sequence_of(b, blockIdx.x);
    if (i >= b.n_seqs) return;
    const kv::Seq s = kv::sequence(b, i);
    const int row = NARROW ? s.first + (int)blockIdx.x % most : blockIdx.x;
    if (row - s.first >= s.rows || (s.rows <= most) != NARROW) return;
    if (FEW && hq >= a.n_heads) return;
    const int64_t at = ((int64_t)row * a.n_heads + hq) * stride;
    auto none = [](float2 st) { return st.y == 0.f && st.x == -kInf; }; // nothing of it is there
    constexpr int E = D / 64;
    float v[E] = {};
    if constexpr (FEW) {
        const float2 st = lane < splits ? parts.stat[at + lane] : make_float2(-kInf, 0.f);
        float part[kFewParts][E] = {};
#pragma unroll
        for (int x = 0; x < kFewParts; x++)
            if (x < splits)
#pragma unroll
                for (int e = 0; e < E; e++) part[x][e] = parts.acc[(at + x) * D + E * lane + e];
        const float o = wave_max(st.x), f = none(st) ? 0.f : st.x == o ? 1.f : __builtin_amdgcn_exp2f(st.x - o), mine = none(st) ? 0.f : st.y * f;
        const int is = !none(st);
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < kFewParts; x++) {
            const float fx = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), x));
            sum += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), x));
            if (__builtin_amdgcn_readlane(is, x))
#pragma unroll
                for (int e = 0; e < E; e++) v[e] += times(part[x][e], fx);
        }
#pragma unroll
        for (int e = 0; e < E; e++) kv::store(a.out, a.type, row * a.out_stride + (int64_t)hq * D + E * lane + e, sum == 0.f ? 0.f : v[e] / sum);
    } else {
        __shared__ float sh_acc[kJoinWaves][D], sh_sum[kJoinWaves];
        float o = -kInf;
        for (int x = lane; x < splits; x += 64) o = fmaxf(o, parts.stat[at + x].x);
        o = wave_max(o);
        float total = 0.f;
#pragma unroll 4
        for (int x = w; x < splits; x += kJoinWaves) {
            const float2 st = parts.stat[at + x];
            float part[E];
#pragma unroll
            for (int e = 0; e < E; e++) part[e] = parts.acc[(at + x) * D + E * lane + e];
            const float f = none(st) ? 0.f : st.x == o ? 1.f : __builtin_amdgcn_exp2f(st.x - o);
            total += none(st) ? 0.f : st.y * f;
#pragma unroll
            for (int e = 0; e < E; e++) v[e] += none(st) ? 0.f : times(part[e], f);
        }
#pragma unroll
        for (int e = 0; e < E; e++) sh_acc[w][E * lane + e] = v[e];
        if (lane == 0) sh_sum[w] = total;
        __syncthreads();
        if (threadIdx.x >= D) return;
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int x = 0; x < kJoinWaves; x++) sum += sh_sum[x], acc += sh_acc[x][threadIdx.x];
        kv::store(a.out, a.type, row * a.out_stride + (int64_t)hq * D + threadIdx.x, sum == 0.f ? 0.f : acc / sum);
    }
}

typedef float f16v __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f16v mfma32(const h8 &a, const h8 &b, const f16v &c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16v mfma32(const b8 &a, const b8 &b, const f16v &c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

constexpr int kWideWaves = 8, kWideRows = 32 * kWideWaves, kWideThreads = 64 * kWideWaves;

// Where 16-byte piece x of row r lies in a tile of rows of 128 (256) bytes: the sixteen rows that a 16-byte LDS read takes together then meet sixteen places.
template <int PER_ROW>
__device__ __forceinline__ int piece_at(int r, int x) {
    return r * PER_ROW + (PER_ROW == 16 ? x ^ (r & 15) : x ^ (r >> 1 & 7));
}

// Values that are the same in every lane, in scalar registers.
__device__ __forceinline__ kv::Seq uniform(const kv::Seq &s) {
    return {__builtin_amdgcn_readfirstlane(s.first), __builtin_amdgcn_readfirstlane(s.rows), __builtin_amdgcn_readfirstlane(s.length)};
}
// From memory (a base that is the same in every lane, and an offset of each) into LDS, lane l's 16 bytes to `lds` + 16 l.  The compiler does not know of
// these loads: wait_lds_loads() before the barrier behind which they are read.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // it need not keep m0
__device__ __forceinline__ void lds_load(uint32_t lds, const char *base, uint32_t off) {
    const uint64_t p = (uint64_t)base;
    const uint64_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)p) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(at) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_lds_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// A barrier that waits for this wave's LDS accesses and for no loads from memory.
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Longer chunks.  A block has 256 query rows of one sequence and kv head, a wave 32 of them; keys and values come in tiles of 64 positions through LDS, in 16
// bits, the next one or two on their way meanwhile: codes of 8 bits into registers, to be converted once for all waves, 16-bit cells straight into LDS.  A tile is four
// runs of 16 positions, each in one page: four waves bring a run of keys each, the other four one of values, so that a wave has one entry of the table to ask for.
//
// The two waves of a SIMD take turns: while the first four waves have the matrix cores (the weighted sum of the tile before, then the scores of this one), the
// last four have the vector ALUs (exponentials), half a tile behind, and the barriers between keep it so.  Left to themselves, waves of
// two blocks had either unit busy for 28 and 52 % of the time, hardly ever together.  In steps of half a tile, 0 the first: the first four do the products of tile i in step 2 i
// and its exponentials in 2 i + 1, the others each a step later.  So keys of tile i are read in steps 2 i and 2 i + 1, its values in 2 i + 2 and 2 i + 3, its scales in 2 i + 1 and 2 i + 2;
// with two places for keys and three for the rest, tile i + 1 may be written from step 2 i on, and is there before 2 i + 2.
//
// Of heads of 128, a wave's products of a tile are 512 clocks of its matrix core per number that q is made of, and as many per number of a weight: 1536 of 16-bit rows.  Each score
// and weight of 8-bit cells is multiplied by a scale, and conversion is the vector ALUs' too.  512 rows of 64 heads on 8 behind 7488 positions in i8: 206 us, 630 TFLOP/s of what
// one number each would take (a large library product in fp16: 1170); two prompts of 4096 and 2542, 32 heads, window 1024, bf16: 204 us, 464 TFLOP/s, of which a quarter is the last of four rounds of
// blocks.  Weights in one number took 171 and 171.  What did not pay: one conversion spread between the products
// (+9 %), the values' wait half a tile later, scales as float4 from LDS (16 reads a tile; they now are two registers, broadcast in rows of lanes).
template <int KV, int NQ, int D>
__global__ __launch_bounds__(kWideThreads, 2) void kv_wide_kernel(KvLayer l, l2_kvbatch b, KvAttention a, Parts parts, Cut cut) {
    using C = Cells<KV>;
    using Frag = typename C::Frag;
    constexpr int TT = 64, PK = D / 8, DT = D / 32, KS = D / 16, NP = weight_numbers(NQ), LOADS = D * C::kSize / 64; // (of 16 bytes per lane: 16 positions)
    __shared__ __align__(16) u4 sh_k[2][TT * PK], sh_v[3][D * 8];
    __shared__ __align__(16) float sh_ks[3][TT], sh_vs[3][TT];
    __shared__ __align__(16) float sh_top[3][4];
    __shared__ uint32_t sh_there[3];
    __shared__ int sh_seq, sh_tile, sh_odd;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, hh = lane >> 5;
    const int group = a.n_heads / l.n_heads;
    const int h = __builtin_amdgcn_readfirstlane(blockIdx.x % l.n_heads), split = __builtin_amdgcn_readfirstlane(blockIdx.x / l.n_heads % cut.splits);

    // which sequence's rows: the tiles of all sequences one behind the other
    {
        int at = blockIdx.x / (l.n_heads * cut.splits);
        if (tid == 0) sh_seq = -1, sh_odd = 0;
        __syncthreads();
        for (int i0 = 0; i0 < b.n_seqs; i0 += 64) {
            int tiles = 0;
            if (i0 + lane < b.n_seqs) {
                const int64_t r = (int64_t)kv::sequence(b, i0 + lane).rows * group;
                tiles = r > cut.narrow ? (int)((r + kWideRows - 1) / kWideRows) : 0;
            }
            int upto = tiles;
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(upto, o);
                if (lane >= o) upto += x;
            }
            if (w == 0 && upto > at && upto - tiles <= at) sh_seq = i0 + lane, sh_tile = tiles - 1 - (at - (upto - tiles)); // the longest first
            const int all = __shfl(upto, 63);
            if (at < all) break;
            at -= all;
        }
        __syncthreads();
    }
    const int i = __builtin_amdgcn_readfirstlane(sh_seq), tile = __builtin_amdgcn_readfirstlane(sh_tile);
    if (i < 0) return;
    const kv::Seq s = uniform(kv::sequence(b, i));
    const int rows = s.rows * group, row0 = tile * kWideRows + 32 * w, base = s.length - s.rows;
    const bool real = row0 + n < rows;
    const int tok = real ? (row0 + n) / group : 0;
    const Seen seen(a, real ? base + tok : -1);
    const int64_t q_row = s.first + tok, head = h * group + (real ? (row0 + n) % group : 0);
    // the positions of the wave's rows and of the block's
    const int w_first = __builtin_amdgcn_readfirstlane(base + min(row0, rows - 1) / group);
    const int w_last = __builtin_amdgcn_readfirstlane(row0 < rows ? base + (min(row0 + 32, rows) - 1) / group : -1);
    const int b_first = __builtin_amdgcn_readfirstlane(base + tile * kWideRows / group);
    const int b_last = __builtin_amdgcn_readfirstlane(base + (min((tile + 1) * kWideRows, rows) - 1) / group);

    Frag q[KS][NQ];
    float c = a.scale * kLog2e;
    {
        kv::raw8 raw[KS];
#pragma unroll
        for (int k = 0; k < KS; k++) raw[k] = kv::load_raw8(a.q, a.type, q_row * a.q_stride + head * D + 16 * k + 8 * hh);
        float top = 0.f;
        int e = 0;
        if (C::kHalf) {
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const f8 x = kv::values8(raw[k], a.type);
#pragma unroll
                for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[j]));
            }
            const lanes::Both t = lanes::both32(top);
            top = fmaxf(t.lo, t.hi);
            e = fit_q<C::kEight>(top, c);
        }
#pragma unroll
        for (int k = 0; k < KS; k++) {
            f8 x = kv::values8(raw[k], a.type);
            if (C::kHalf)
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = ldexpf(x[j], e);
            pieces<Frag, typename C::One, NQ>(x, q[k]);
        }
    }

    const Range range = range_of<TT>(a, b_first, b_last);
    const int begin = min(split * cut.per, range.n), end = min(begin + cut.per, range.n);
    const int size = 1 << l.page_shift;

    // The first four waves have the keys to bring, the others the values: each 16 positions of a tile, a run, which lie in one page.  A run of values is D rows of two
    // pieces; their order in a pair changes so that the rows that an LDS read takes together meet different places.
    const bool late = w >= kWideWaves / 2;
    const int run = w & 3;
    auto v_swap = [](int row) { return (row >> 2 ^ row >> 3) & 1; };
    const uint32_t k_off = lane / PK * (D * 2) + 16 * (lane % PK ^ (PK == 16 ? lane / PK : lane / PK >> 1)); // piece `lane` of a run in LDS
    const uint32_t v_off = lane / 2 * size * 2 + 16 * ((lane & 1) ^ v_swap(lane / 2));
    const uint32_t lds_k = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) u4 *)&sh_k[0][0]) + run * (16 * PK * 16);
    const uint32_t lds_v = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) u4 *)&sh_v[0][0]) + run * (2 * D * 16);

    // Whether every row of those from position `first` to `last` sees all of a tile whose pages are there.
    auto all_visible = [&](int t0, int first, int last) { return t0 + TT - 1 <= first && (!a.window || t0 > last - a.window || t0 + TT <= a.sinks); };

    // The tile at hand, tile x, has place `cur` of three; where tile x + by is.
    int cur = 0;
    auto place = [&](int by) { return cur + by % 3 >= 3 ? cur + by % 3 - 3 : cur + by % 3; };
    u4 raw[C::kEight ? LOADS : 1];
    float scale = 0.f;
    bool there = false; // whether the run that was asked for has a page
    // The entry of the table for the run that is asked for next (not by a scalar load, which the compiler would put off until the entry is needed).  What lies
    // behind the table is behind every position too.
    int entry = -1;
    const int32_t *table = b.pages + (int64_t)i * b.max_pages;
    auto ask_page = [&](int x) { entry = table[min((range.tile(x) * TT + 16 * run) >> l.page_shift, b.max_pages - 1)]; };
    const int64_t page_cells = (int64_t)l.n_heads * size * D * C::kSize; // bytes of a page's K (V)
    const char *from = (const char *)(late ? l.v : l.k) + (int64_t)h * size * D * C::kSize;
    // Asks for this wave's run of tile x + by, whose page has been asked for, and for the page of the tile behind that.
    auto ask = [&](int x, int by) {
        x += by;
        if (x >= end) return;
        const int found = __builtin_amdgcn_readfirstlane(entry);
        there = (uint32_t)found < (uint32_t)l.n_pages;
        const int page = there ? found : 0, slot = (range.tile(x) * TT + 16 * run) & (size - 1);
        const char *at = from + page * page_cells + slot * (late ? C::kSize : D * C::kSize);
        if constexpr (C::kEight) {
            const uint32_t off = late ? lane * size : lane * 16, step = late ? 64 * size : 1024;
#pragma unroll
            for (int y = 0; y < LOADS; y++) raw[y] = *(const u4 *)(at + y * step + off);
            scale = (late ? l.v_scale : l.k_scale)[((int64_t)page * l.n_heads + h) * size + slot + (lane & 15)];
        } else if (late) {
#pragma unroll
            for (int y = 0; y < LOADS; y++) lds_load(lds_v + place(by) * (D * 8 * 16) + y * 1024, at + y * (64 * size), v_off);
        } else {
            const uint32_t to = lds_k + ((x - begin) & 1) * (TT * PK * 16);
#pragma unroll
            for (int y = 0; y < LOADS; y++) lds_load(to + y * 1024, at + y * 1024, k_off ^ 64 * y);
        }
        if (x + 1 < end) ask_page(x + 1);
    };
    // Has this wave's run of tile x + by, asked for before, in LDS.  16-bit cells get there by themselves: where a row may not see all of the tile, values that
    // are not finite are taken out.
    auto put = [&](int x, int by) {
        x += by;
        if (x >= end) return;
        const int kb = (x - begin) & 1, vb = place(by);
        if (!late && lane == 0) ((uint8_t *)&sh_there[vb])[run] = there;
        if constexpr (C::kEight) {
#pragma unroll
            for (int y = 0; y < LOADS; y++) {
                const int p = 64 * y + lane, row = 16 * run + p / (PK / 2), x2 = 2 * (p % (PK / 2));
                const Frag f0 = C::frag(raw[y], 0), f1 = C::frag(raw[y], 1);
                u4 *to = late ? &sh_v[vb][2 * D * run + 2 * p] : &sh_k[kb][0];
                to[late ? v_swap(p) : piece_at<PK>(row, x2)] = __builtin_bit_cast(u4, f0);
                to[late ? v_swap(p) ^ 1 : piece_at<PK>(row, x2 + 1)] = __builtin_bit_cast(u4, f1);
            }
            if (lane < 16) (late ? sh_vs : sh_ks)[vb][16 * run + lane] = scale;
            if (late) {
                const float most = row_max(scale);
                if (lane == 0) sh_top[vb][run] = most;
            }
        } else {
            wait_lds_loads();
            if (!late || (there && all_visible(range.tile(x) * TT, b_first, b_last))) return;
#pragma unroll
            for (int y = 0; y < LOADS; y++) {
                bool odd = false;
                u4 *at = &sh_v[vb][2 * D * run + 64 * y + lane];
                const u4 v = finite<KV>(*at, odd);
                if (odd) *at = v, sh_odd = 1;
            }
        }
    };

    const int kr_row = (n & 0x13) | (n & 4) << 1 | (n & 8) >> 1;
    // (2 k + hh) ^ x is (hh ^ x) ^ 2 k: a piece's address is the first one's but for the bits of k
    const uint32_t k_base = 16 * piece_at<PK>(kr_row, hh), v_base = 16 * (2 * n + (hh ^ v_swap(n)));
    auto k_at = [&](int buf, int k, int y) { return *(const u4 *)((const char *)&sh_k[buf][32 * y * PK] + (k_base ^ (32 * k))); };
    auto v_at = [&](int buf, int y, int v) { return *(const u4 *)((const char *)&sh_v[buf][2 * (D * v + 32 * y)] + v_base); };
    auto run_of = [](int z) { return 32 * (z / 4) + 16 * (z / 2 & 1) + 4 * (z & 1); }; // position of element 4 (z & 3) of sc[z / 4], less 8 hh

    f16v acc[DT] = {}, sc[2];
    Frag pf[4][NP]; // weights of positions 16 v + 8 hh + j
    float off = -kInf, sum = 0.f;
    // The weighted sum of one tile and the scores of the other, 2 x 32 positions.  Each of these products wants 16 bytes of LDS per lane, as long on their way as four
    // products take and no less of LDS's time than of the matrix cores': they are asked for kDeep products ahead.
    auto products = [&](auto with_values, auto with_scores, int vb, int kb) {
        constexpr int V = decltype(with_values)::value ? 4 * DT : 0, K = decltype(with_scores)::value ? 2 * KS : 0, kDeep = NQ == 1 ? 4 : 5 - NP;
        auto at = [&](int z) { return z < V ? v_at(vb, z % DT, z / DT) : k_at(kb, (z - V) / 2, (z - V) % 2); };
        if (K) sc[0] = sc[1] = f16v{};
        u4 ring[kDeep];
#pragma unroll
        for (int z = 0; z < kDeep; z++) ring[z] = at(z);
#pragma unroll
        for (int z = 0; z < V + K; z++) {
            const Frag f = __builtin_bit_cast(Frag, ring[z % kDeep]);
            if (z + kDeep < V + K) ring[z % kDeep] = at(z + kDeep);
            if (z < V) {
#pragma unroll
                for (int y = 0; y < NP; y++) acc[z % DT] = mfma32(f, pf[z / DT][y], acc[z % DT]);
            } else {
#pragma unroll
                for (int y = 0; y < NQ; y++) sc[(z - V) % 2] = mfma32(f, q[(z - V) / 2][y], sc[(z - V) % 2]);
            }
        }
        __builtin_amdgcn_sched_group_barrier(0x100, kDeep, 0);
#pragma unroll
        for (int z = 0; z < V + K; z++) {
            if (z < V) __builtin_amdgcn_sched_group_barrier(0x8, NP, 0);
            else __builtin_amdgcn_sched_group_barrier(0x8, NQ, 0);
            if (z + kDeep < V + K) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    };
    // A tile's scales, of which a lane wants 32 and every lane of its half the same: lane m of a row of 16 has those of elements m of sc[0] and sc[1].
    float ks[2], vs[2];
    auto ask_scales = [&](const float *from, float *to) {
        const float *at = from + (lane & 3) + (lane & 4) + 2 * (lane & 8) + 8 * hh; // run_of(m / 4) + m % 4
        to[0] = at[0];
        to[1] = at[32];
    };
    // What weights() needs of tile x + by, ahead of it.
    uint32_t runs = 0; // which runs have a page, a byte each
    auto look = [&](int by) {
        runs = sh_there[place(by)];
        if (C::kEight) ask_scales(sh_ks[place(by)], ks);
    };
    // Weights of tile x from its scores.
    auto weights = [&](int x) {
        const int vb = cur, t0 = range.tile(x) * TT;
        const uint32_t bits_there = __builtin_amdgcn_readfirstlane(runs);
        const bool whole = bits_there == 0x01010101 && all_visible(t0, w_first, w_last);
        if constexpr (C::kEight) {
            ask_scales(sh_vs[vb], vs);
            ks[0] = scale_of_key(ks[0]), ks[1] = scale_of_key(ks[1]);
            each<32>([&](auto at) { sc[at / 16][at % 16] *= scale_at<at % 16>(ks[at / 16]); });
        }
        if (!whole) {
            each<32>([&](auto at) {
                constexpr int z = at / 4, r = at % 4;
                const int t = run_of(z) + 8 * hh;
                const float v_scale = C::kEight ? scale_at<at % 16>(vs[at / 16]) : 0.f; // (by all lanes of the row)
                const bool here = bits_there >> 8 * (2 * (z / 4) + (z / 2 & 1)) & 1, see = here & seen(t0 + t + r); // run t / 16
                const float score = sc[z / 4][4 * (z & 3) + r];
                sc[z / 4][4 * (z & 3) + r] = see ? C::kEight ? fmaf(v_scale, 0.f, score) : score : -kInf; // NaN where the values are
            });
            if (C::kEight)
#pragma unroll
                for (int z = 0; z < 2; z++) vs[z] = vs[z] == vs[z] ? vs[z] : 0.f; // nothing of a row that is not seen
        }
        float mx = -kInf;
#pragma unroll
        for (int z = 0; z < 8; z++)
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, sc[z / 4][4 * (z & 3) + r]);
        const lanes::Both m2 = lanes::both32(mx);
        float top = fmaxf(m2.lo, m2.hi) * c;
        if constexpr (C::kEight) {
            if (whole) top += above(fmaxf(fmaxf(sh_top[vb][0], sh_top[vb][1]), fmaxf(sh_top[vb][2], sh_top[vb][3])));
            if (!whole || __ballot(raises<KV>(off, top))) {
                const float e[2] = {log2_of(vs[0]), log2_of(vs[1])};
                mx = -kInf;
                each<32>([&](auto at) { mx = fmaxf(mx, fmaf(sc[at / 16][at % 16], c, scale_at<at % 16>(e[at / 16]))); });
                const lanes::Both e2 = lanes::both32(mx);
                top = fmaxf(e2.lo, e2.hi);
            }
        }
        const float f = follow<KV>(off, top);
        if (__ballot(f != 1.f)) {
#pragma unroll
            for (int y = 0; y < DT; y++) acc[y] *= f;
            sum *= f;
        }
        const float now = off == -kInf ? 0.f : off; // nothing seen yet: every weight is exp2(-inf)
        each<4>([&](auto v) { // positions 16 v + 8 hh + j
            f8 p;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(fmaf(sc[v / 2][8 * (v & 1) + j], c, -now));
                sum += p[j];
            }
            if constexpr (C::kEight) each<8>([&](auto j) { p[(int)j] *= scale_at<8 * (v & 1) + j>(vs[v / 2]); });
            pieces<Frag, typename C::One, NP>(p, pf[v]);
        });
        // here, not where the compiler would have them: between the products, which then wait for the first ones
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int y = 0; y < NP; y++) asm volatile("" : "+v"(pf[v][y]));
    };

    if (begin < end) {
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        ask_page(begin);
        ask(begin, 0);
        put(begin, 0);
        if (C::kEight || late) ask(begin, 1);
        barrier();
        if (late) barrier();
        // before the products of tile x + by: what is behind it
        auto behind = [&](int x, int by) {
            if constexpr (C::kEight) {
                put(x, by + 1);
                ask(x, by + 2);
            } else if (!late) {
                ask(x, by + 1);
            }
        };
        behind(begin, 0);
        products(no, yes, 0, 0);
        look(0);
        if (!C::kEight && late) put(begin, 1);
        barrier();
        for (int x = begin; x + 1 < end; x++) { // (left in its middle, the loop has the accumulators in registers twice)
            // the vector ALUs' step
            if (!C::kEight && late) ask(x, 2);
            weights(x);
            if (!C::kEight && !late) put(x, 1);
            barrier();
            // the matrix cores'
            behind(x, 1);
            products(yes, yes, cur, (x + 1 - begin) & 1);
            look(1);
            if (!C::kEight && late) put(x, 2);
            barrier();
            cur = place(1);
        }
        weights(end - 1);
        barrier();
        products(yes, no, cur, 0);
        if (!late) barrier();
    }
    if constexpr (!C::kEight) { // as in the narrow kernel
        bool odd = begin < end && sh_odd;
#pragma unroll
        for (int y = 0; y < DT; y++)
#pragma unroll
            for (int z = 0; z < 16; z++) odd |= !(fabsf(acc[y][z]) < kInf);
        if (__ballot(odd)) {
#pragma unroll
            for (int y = 0; y < DT; y++)
#pragma unroll
                for (int z = 0; z < 16; z++) acc[y][z] = broken(acc[y][z]);
#pragma unroll 1
            for (int x = TT * begin; x < TT * end; x++) {
                const int t = range.tile(x / TT) * TT + x % TT, page = kv::page_at(b, l.n_pages, i, t >> l.page_shift);
                if (page < 0 || !seen(t)) continue;
                const uint16_t *p = (const uint16_t *)l.v + ((((int64_t)page * l.n_heads + h) * D + 4 * hh) * size + (t & (size - 1)));
#pragma unroll
                for (int y = 0; y < DT; y++)
#pragma unroll
                    for (int z = 0; z < 16; z++) acc[y][z] += not_finite<KV>(p[(int64_t)(32 * y + 8 * (z / 4) + z % 4) * size]);
            }
#pragma unroll
            for (int y = 0; y < DT; y++)
#pragma unroll
                for (int z = 0; z < 16; z++) acc[y][z] = mended(acc[y][z]);
        }
    }
    const lanes::Both s2 = lanes::both32(sum);
    sum = s2.lo + s2.hi;
    if (!real) return;
    if (cut.splits == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int y = 0; y < DT; y++)
#pragma unroll
            for (int z = 0; z < 4; z++) {
                const int64_t at = q_row * a.out_stride + head * D + 32 * y + 8 * z + 4 * hh;
                f4 v;
#pragma unroll
                for (int r = 0; r < 4; r++) v[r] = sum == 0.f ? 0.f : acc[y][4 * z + r] * inv;
                kv::store4(a.out, a.type, at, v);
            }
    } else {
        const int64_t at = (q_row * a.n_heads + head) * cut.stride + split;
#pragma unroll
        for (int y = 0; y < DT; y++)
#pragma unroll
            for (int z = 0; z < 4; z++)
                *(f4 *)(parts.acc + at * D + 32 * y + 8 * z + 4 * hh) = f4{acc[y][4 * z], acc[y][4 * z + 1], acc[y][4 * z + 2], acc[y][4 * z + 3]};
        if (hh == 0) parts.stat[at] = make_float2(off, sum);
    }
}

typedef void (*AttnKernel)(KvLayer, l2_kvbatch, KvAttention, Parts, Cut);
#define SIZES(kernel, kv, nq) {kernel<kv, nq, 64>, kernel<kv, nq, 128>}
#define ALL(kernel)                                                                                                                             \
    {{SIZES(kernel, 0, 1), SIZES(kernel, 0, 2), {}}, {SIZES(kernel, 1, 1), SIZES(kernel, 1, 2), {}}, {SIZES(kernel, 2, 1), SIZES(kernel, 2, 2), {}}, \
     {SIZES(kernel, 3, 1), SIZES(kernel, 3, 2), SIZES(kernel, 3, 3)}}
const AttnKernel kNarrow[4][3][2] = ALL(kv_narrow_kernel), kWide[4][3][2] = ALL(kv_wide_kernel);
typedef void (*JoinKernel)(l2_kvbatch, KvAttention, Parts, int, int, int, int);
const JoinKernel kJoin[2][2][2] = {{{kv_join_kernel<64, false, false>, kv_join_kernel<64, false, true>}, {kv_join_kernel<64, true, false>, kv_join_kernel<64, true, true>}},
                                   {{kv_join_kernel<128, false, false>, kv_join_kernel<128, false, true>}, {kv_join_kernel<128, true, false>, kv_join_kernel<128, true, true>}}};

// In how many 16-bit numbers q enters the matrix cores, less one.
int pieces_index(int kv_type, int type) {
    if (kv_type == L2_KV_BF16) return type == L2_BF16 ? 0 : type == L2_F16 ? 1 : 2;
    return type == L2_F32 ? 1 : 0;
}

} // namespace

void kv_attention_plan(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvAttention &a, KvAttnPlan *plan) {
    const int group = a.n_heads / l.n_heads;
    const int64_t rows = std::min(b.max_rows, b.n_rows), seqs = std::max(b.n_seqs, 1);
    auto tiles_seen = [&](int64_t tt, int64_t per_tile) { // of the row tile that sees most
        int64_t seen = b.max_length;
        if (a.window) seen = std::min<int64_t>(seen, (int64_t)a.window + std::min(rows, per_tile) + a.sinks + 2 * tt);
        return (seen + tt - 1) / tt;
    };
    // Parts so that `full` blocks come to be, of `least` tiles or more.  Two narrow blocks per CU: with 3, 4 and 6 the step of 32 sequences above took 55, 52 and 56 us instead
    // of 48.  One wide block, which fills a CU: three parts instead of one, of a batch of twelve, cost 28 us of joining and saved none.
    auto parts_of = [&](int64_t blocks, int64_t full, int64_t tiles, int64_t least, int *splits, int *per) {
        const int64_t parts = std::max<int64_t>(1, std::min<int64_t>((full + blocks - 1) / blocks, tiles / least));
        *per = (int)((tiles + parts - 1) / parts);
        *splits = *per ? (int)((tiles + *per - 1) / *per) : 1;
    };
    // Where no sequence has more than `most` rows the narrow kernel takes all, cells read once for each 16 rows.  us as narrow and wide, 32 sequences of 2048 positions, 64 heads on
    // 8: 24, 48, 64 and 80 rows of bf16 on e4m3 46 / 112, 74 / 106, 86 / 108 and 108 / 111, of fp32 on i8 49 / 125, 79 / 130, 90 / 132 and 112 / 138, of fp32 on bf16, three numbers each, 84 / 206, 131 / 212,
    // 158 / 215 and 198 / 219.  Over other cells of 16 bits, of which a block reads twice the bytes: 24, 32, 48 and 64 of fp16 on fp16 83 / 99, 83 / 105, 132 / 111 and 156 / 112, of fp32
    // 84 / 123, 85 / 123, 132 / 129 and 159 / 132.
    const int most = (kv_type > L2_KV_E4M3 && pieces_index(kv_type, a.type) < 2 ? 32 : 64) / group * group;
    plan->wide = rows * group > most;
    // The one kernel's or the other's alone, where every sequence has that many rows if the call's arrays are full; else they may be some of each.
    if (!plan->wide) plan->narrow_rows = most;
    else plan->narrow_rows = group > kNarrowRows || (b.n_rows - (seqs - 1) * rows) * group > kNarrowRows ? 0 : kNarrowRows / group * group;
    plan->narrow_blocks = (int)std::max<int64_t>((std::min<int64_t>(rows * group, plan->narrow_rows) + kNarrowRows - 1) / kNarrowRows, 1);
    plan->narrow_splits = plan->wide_splits = 1;
    // Beside chunks, parts as for half of the sequences: where 1, a few, half and all but one of 4, 12 and 32 are chunks, counting a quarter, three quarters or all of them made
    // such batches up to 8 % quicker or slower, in no order.
    if (plan->narrow_rows)
        parts_of((plan->wide ? (seqs + 1) / 2 : seqs) * l.n_heads * plan->narrow_blocks, 2 * cu_count(), tiles_seen(kv_type <= L2_KV_E4M3 ? 64 : 32, plan->narrow_rows),
                 kNarrowWaves, &plan->narrow_splits, &plan->narrow_per);
    // row tiles of all sequences, at most: their whole ones, and a last one of each that has more rows than the narrow kernel takes
    const int64_t all = (int64_t)b.n_rows * group;
    const int64_t tile = kWideRows;
    plan->wide_tiles = all / tile + std::min<int64_t>(seqs, all / (plan->narrow_rows + 1));
    if (plan->wide) // (as many tiles as there would be if each sequence's last one were half full)
        parts_of(std::min<int64_t>((all + seqs * (tile / 2) + tile / 2 - 1) / tile, plan->wide_tiles) * l.n_heads, cu_count(), tiles_seen(64, (tile + group - 1) / group), 4, &plan->wide_splits,
                 &plan->wide_per);
    plan->stride = std::max(plan->narrow_splits, plan->wide_splits);
    plan->workspace = plan->stride > 1 ? (size_t)b.n_rows * a.n_heads * plan->stride * (l.head_size * 4 + 8) : 0;
}

int kv_attention_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvAttention &a, const KvAttnPlan &plan, void *workspace, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    const int big = l.head_size == 128, group = a.n_heads / l.n_heads, nq = pieces_index(kv_type, a.type);
    Parts parts{(float *)workspace, nullptr};
    parts.stat = (float2 *)(parts.acc + (size_t)b.n_rows * a.n_heads * plan.stride * l.head_size);
    if (plan.wide && plan.wide_tiles) {
        const int64_t blocks = plan.wide_tiles * l.n_heads * plan.wide_splits;
        if (blocks >= ((int64_t)1 << 32) / kWideThreads) return l2_fail(L2_ERR_RANGE, "%d rows of %d heads", b.n_rows, a.n_heads); // a launch has fewer than 2^32 threads
        l2_launch(kWide[kv_type][nq][big], dim3((unsigned)blocks), dim3(kWideThreads), 0, st, l, b, a, parts,
                  Cut{plan.wide_splits, plan.wide_per, plan.stride, plan.narrow_rows});
    }
    if (plan.narrow_rows)
        l2_launch(kNarrow[kv_type][nq][big], dim3(plan.narrow_splits * plan.narrow_blocks, l.n_heads, b.n_seqs), dim3(64 * kNarrowWaves), 0, st, l, b, a, parts,
                  Cut{plan.narrow_splits, plan.narrow_per, plan.stride, plan.narrow_rows});
    const int most = plan.narrow_rows / group; // rows of a sequence that the narrow kernel takes
    auto join = [&](bool narrow, int blocks, int splits, int most) {
        const bool few = splits <= kFewParts;
        l2_launch(kJoin[big][narrow][few], dim3(blocks, few ? (a.n_heads + kJoinWaves - 1) / kJoinWaves : a.n_heads), dim3(64 * kJoinWaves), 0, st, b, a, parts, splits,
                  plan.stride, group, most);
    };
    if (plan.narrow_rows && plan.narrow_splits > 1) join(true, b.n_seqs * std::min(most, b.max_rows), plan.narrow_splits, std::min(most, b.max_rows));
    if (plan.wide && plan.wide_splits > 1) join(false, b.n_rows, plan.wide_splits, most);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_attention_warm_up() {
    hipFuncAttributes a;
    for (auto &all : {&kNarrow, &kWide})
        for (auto &k : *all)
            for (auto &n : k)
                for (AttnKernel f : n)
                    if (f) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    for (auto &d : kJoin)
        for (auto &k : d)
            for (JoinKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    return L2_OK;
}
