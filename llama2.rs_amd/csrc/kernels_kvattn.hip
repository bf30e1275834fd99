// Attention of new rows over a cache in pages: out = sum over t of softmax(scale q.k_t) v_t, in one pass with a running maximum and sum.
//
// Both products are the matrix cores', transposed: S^T = K q^T and O^T = V^T P^T.  The result of the first has a row of queries in each lane and its
// positions in the lane's registers, which is the second operand of the second product as it stands, once the rows of K are dealt to the lanes in
// the fitting order; maxima and sums are a lane's own but for two exchanges, and the factors between tiles one register.  V lies transposed in the pool, so
// nothing is transposed here.  Codes of 8 bits become 16-bit floats exactly (fp16).  Scales of keys multiply the scores, those of values the weights.
//
// Weights enter the second product in 16 bits, fp16 as 2^15 at most: p_t = exp2(s_t - off) with off = max s + e - 15, where 2^e is the power of two above the largest
// scale of the values seen; then p_t * (scale of v_t) is below 2^15 whatever the scales, and off cancels in the quotient with the sum of the p_t.  fp32 rows have q
// and p in two fp16 numbers (2^-22) or, over a pool in bf16, in three; rows of 16 bits in one where that holds a q as it is.  q is scaled by a power of two per
// row, so that fp16 holds what bf16 and fp32 rows may contain.
#include <algorithm>

#include "kvpool.h"
#include "lanes.h"

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLeastE = -67.f; // rows whose values are held at all have scales from 2^-67

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

// x as a sum of NP numbers of 16 bits, each the nearest to what those before it leave.  The compiler may make a product and its rounding to fp16
// one instruction that rounds once, for one of the two places that the first number goes to: x is a value that it knows nothing of.
template <class Frag, class One, int NP>
__device__ __forceinline__ void pieces(f8 x, Frag (&out)[NP]) {
    if (NP > 1)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float v = x[j];
            asm("" : "+v"(v));
            x[j] = v;
        }
#pragma unroll
    for (int i = 0; i < NP; i++) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            out[i][j] = (One)x[j];
            if (i + 1 < NP) x[j] -= (float)out[i][j];
        }
    }
}

// Eight values of a row of the caller's, aligned as their type is.
__device__ __forceinline__ f8 load8(const void *p, int type, int64_t i) {
    typedef float any __attribute__((ext_vector_type(8), aligned(4)));
    typedef _Float16 anyh __attribute__((ext_vector_type(8), aligned(2)));
    typedef uint16_t anyb __attribute__((ext_vector_type(8), aligned(2)));
    f8 x;
    if (type == L2_F32) {
        const any v = *(const any *)((const float *)p + i);
        for (int j = 0; j < 8; j++) x[j] = v[j];
    } else if (type == L2_F16) {
        const anyh v = *(const anyh *)((const _Float16 *)p + i);
        for (int j = 0; j < 8; j++) x[j] = (float)v[j];
    } else {
        const anyb v = *(const anyb *)((const uint16_t *)p + i);
        for (int j = 0; j < 8; j++) x[j] = kv::bf16_float(v[j]);
    }
    return x;
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

__device__ __forceinline__ bool visible(const KvAttention &a, int t, int pos) {
    return t <= pos && (!a.window || t > pos - a.window || t < a.sinks);
}

constexpr int kNarrowRows = 16, kNarrowWaves = 4;

// A query row's part: what a block found of it.  `off` is common to the weights in acc and sum.
struct Parts {
    float *acc;   // [row][head][split][D]
    float2 *stat; // [row][head][split]: off, sum
};

// Sequences of up to 16 query rows per kv head (new tokens x query heads of the group).  A block has one sequence, kv head and part of the positions, its
// four waves tiles of 64 positions (32 of 16-bit cells) in turn, straight from memory into registers: 8 KB of keys and 8 KB of values, the next tile's keys
// asked for once this one's scores are there and its values once this one's are summed.
template <int KV, int NP, int D>
__global__ __launch_bounds__(64 * kNarrowWaves, 2) void kv_narrow_kernel(KvLayer l, l2_kvbatch b, KvAttention a, Parts parts, int splits) {
    using C = Cells<KV>;
    using Frag = typename C::Frag;
    constexpr int TT = 64 / C::kSize, ST = TT / 16, CH = TT / 4, FR = 2 / C::kSize, KL = D * C::kSize / 64, DT = D / 16, VS = TT / 32;
    const int split = blockIdx.x, h = blockIdx.y, i = blockIdx.z;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
    const kv::Seq s = kv::sequence(b, i);
    const int group = a.n_heads / l.n_heads, rows = s.rows * group;
    if (rows == 0 || rows > kNarrowRows) return;
    const int base = s.length - s.rows; // position of the first row
    const bool real = m < rows;
    const int pos = real ? base + m / group : -1;
    const int64_t q_row = s.first + (real ? m / group : 0), head = h * group + (real ? m % group : 0);

    // q: this lane's row, the dimensions that lie across from its 16 bytes of a key
    Frag q[D / 32][NP];
    float c; // exponent of two per unit of the scores' sums
    {
        f8 x[D / 32];
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < D / 32; k++) {
            const int d = (k / FR) * (64 / C::kSize) + (16 / C::kSize) * g + 8 * (k % FR);
            x[k] = load8(a.q, a.type, q_row * a.q_stride + head * D + d);
#pragma unroll
            for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[k][j]));
        }
        c = a.scale * kLog2e;
        if (C::kHalf) {
            top = lanes::rows_max(top);
            const int e = top > 0.f && top < kInf ? 15 - __builtin_amdgcn_frexp_expf(top) : 0; // the largest in [2^14, 2^15)
#pragma unroll
            for (int k = 0; k < D / 32; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[k][j] = ldexpf(x[k][j], e);
            c = ldexpf(c, -e);
        }
#pragma unroll
        for (int k = 0; k < D / 32; k++) pieces<Frag, typename C::One, NP>(x[k], q[k]);
    }

    const Range range = range_of<TT>(a, base, s.length - 1);
    const int per = (range.n + splits - 1) / splits, begin = min(split * per, range.n), end = min(begin + per, range.n);
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

    f4 acc[DT] = {};
    float top = -kInf, e = kLeastE, off = -kInf, sum = 0.f;
    int n = begin + w;
    if (n < end) {
        pages(n);
        load_k(n, page_k, page_v);
        load_v(n, page_v);
    }
    int here = page_v;
    if (n + kNarrowWaves < end) pages(n + kNarrowWaves);
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
                for (int y = 0; y < NP; y++) sc[x] = mfma16(f, q[k][y], sc[x]);
            }
        if (C::kEight)
#pragma unroll
            for (int x = 0; x < ST; x++) sc[x] *= ks[x];
        const int here_next = page_v;
        if (more) load_k(n + kNarrowWaves, page_k, page_v);

        // positions CH g + 4 x + r of the tile are this lane's
        const bool whole = t0 + TT - 1 <= base && (!a.window || t0 > s.length - 1 - a.window || t0 + TT <= a.sinks) && __ballot(here < 0) == 0;
        bool odd = false; // a value that is not finite where some row may not see it
        if (!whole) {
#pragma unroll
            for (int x = 0; x < ST; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool see = here >= 0 && visible(a, t0 + CH * g + 4 * x + r, pos);
                    sc[x][r] = see ? sc[x][r] : -kInf;
                    if (C::kEight) vs[x][r] = see ? vs[x][r] : 0.f;
                }
            if (!C::kEight) {
                constexpr uint32_t ones = KV == L2_KV_F16 ? 0x7C00u : 0x7F80u;
#pragma unroll
                for (int x = 0; x < DT; x++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t v = vr[x][r];
                        const bool lo = (v & ones) == ones, hi = (v >> 16 & ones) == ones;
                        odd |= lo || hi;
                        vr[x][r] = v & ((lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u));
                    }
            }
        }
        float mx = -kInf;
#pragma unroll
        for (int x = 0; x < ST; x++)
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, sc[x][r]);
        top = fmaxf(top, lanes::rows_max(mx) * c);
        if (C::kEight) {
            float mv = 0.f;
#pragma unroll
            for (int x = 0; x < ST; x++)
#pragma unroll
                for (int r = 0; r < 4; r++) mv = fmaxf(mv, vs[x][r]);
            mv = lanes::rows_max(mv);
            if (mv > 0.f) e = fmaxf(e, (float)__builtin_amdgcn_frexp_expf(mv));
        }
        // nothing seen yet: every weight is exp2(-inf)
        const float now = top == -kInf ? 0.f : C::kEight ? top + (e - 15.f) : C::kHalf ? top - 15.f : top;
        const float f = off == now ? 1.f : __builtin_amdgcn_exp2f(off - now);
        if (__ballot(f != 1.f)) {
#pragma unroll
            for (int x = 0; x < DT; x++) acc[x] *= f;
            sum *= f;
        }
        off = top == -kInf ? -kInf : now;
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
        if (__ballot(odd)) { // added one by one, to the rows that see them
            for (int y = 0; y < TT; y++) {
                const int t = t0 + y, page = kv::page_at(b, l.n_pages, i, t >> l.page_shift);
                if (page < 0 || !visible(a, t, pos)) continue;
                const uint16_t *p = (const uint16_t *)vb + (((int64_t)page * l.n_heads + h) * D * size + (t & (size - 1)));
#pragma unroll
                for (int x = 0; x < DT; x++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint16_t bits = p[(int64_t)(16 * x + 4 * g + r) * size];
                        const float v = KV == L2_KV_F16 ? (float)__builtin_bit_cast(_Float16, bits) : kv::bf16_float(bits);
                        if (!(fabsf(v) < kInf)) acc[x][r] += v;
                    }
            }
        }
        here = here_next;
        if (more) {
            load_v(n + kNarrowWaves, page_v);
            if (n + 2 * kNarrowWaves < end) pages(n + 2 * kNarrowWaves);
        }
    }
    sum = lanes::rows_sum(sum);

    // the waves' parts together
    constexpr int LD = D + 4;
    __shared__ float sh_acc[kNarrowWaves][kNarrowRows][LD];
    __shared__ float2 sh_stat[kNarrowWaves][kNarrowRows];
#pragma unroll
    for (int x = 0; x < DT; x++) *(f4 *)&sh_acc[w][m][16 * x + 4 * g] = acc[x];
    if (g == 0) sh_stat[w][m] = make_float2(off, sum);
    __syncthreads();
    for (int x = threadIdx.x; x < rows * (D / 4); x += 64 * kNarrowWaves) {
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
            v += *(const f4 *)&sh_acc[y][r][d] * f;
        }
        const int64_t row = s.first + r / group, hq = h * group + r % group;
        if (splits == 1) {
            for (int j = 0; j < 4; j++) kv::store(a.out, a.type, row * a.out_stride + hq * D + d + j, total == 0.f ? 0.f : v[j] / total);
        } else {
            const int64_t at = (row * a.n_heads + hq) * splits + split;
            *(f4 *)(parts.acc + at * D + d) = v;
            if (d == 0) parts.stat[at] = make_float2(o, total);
        }
    }
}

// Joins the splits of each query row: one wave per row and head of a sequence that the kernel above takes.
template <int D>
__global__ __launch_bounds__(64) void kv_join_kernel(l2_kvbatch b, KvAttention a, Parts parts, int splits, int group) {
    const int row = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x;
    const int i = kv::sequence_of(b, row);
    if (i >= b.n_seqs) return;
    const kv::Seq s = kv::sequence(b, i);
    if (row - s.first >= s.rows || s.rows * group > kNarrowRows) return;
    const int64_t at = ((int64_t)row * a.n_heads + hq) * splits;
    float o = -kInf, total = 0.f;
    for (int x = 0; x < splits; x++) o = fmaxf(o, parts.stat[at + x].x);
    constexpr int E = D / 64;
    float v[E] = {};
    for (int x = 0; x < splits; x++) {
        const float2 st = parts.stat[at + x];
        if (st.y == 0.f && st.x == -kInf) continue;
        const float f = st.x == o ? 1.f : __builtin_amdgcn_exp2f(st.x - o);
        total += st.y * f;
        for (int e = 0; e < E; e++) v[e] += parts.acc[(at + x) * D + E * lane + e] * f;
    }
    for (int e = 0; e < E; e++) kv::store(a.out, a.type, row * a.out_stride + (int64_t)hq * D + E * lane + e, total == 0.f ? 0.f : v[e] / total);
}

// One block per row and query head; its four waves take positions in turn, each with a running maximum and sum, and are joined at the end.
template <int KV, int D>
__global__ __launch_bounds__(256) void kv_attention_kernel(KvLayer l, l2_kvbatch b, KvAttention a) {
    const int row = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int i = kv::sequence_of(b, row);
    if (i >= b.n_seqs) return;
    const kv::Seq s = kv::sequence(b, i);
    const int at = row - s.first, pos = s.length - s.rows + at;
    if (at >= s.rows || s.rows * (a.n_heads / l.n_heads) <= kNarrowRows) return;
    const int h = hq / (a.n_heads / l.n_heads);
    constexpr int E = D / 64;
    float q[E], acc[E] = {}, m = -__builtin_inff(), sum = 0.f;
    for (int e = 0; e < E; e++) q[e] = kv::load(a.q, a.type, row * a.q_stride + (int64_t)hq * D + 64 * e + lane);
    const int size = 1 << l.page_shift;
    for (int t = w; t <= pos; t += 4) {
        if (a.window && t <= pos - a.window && t >= a.sinks) continue;
        const int page = kv::page_at(b, l.n_pages, i, t >> l.page_shift);
        if (page < 0) continue;
        const int slot = t & (size - 1);
        const int64_t ph = (int64_t)page * l.n_heads + h;
        float kx[E], vx[E], dot = 0.f;
        const float ks = KV <= L2_KV_E4M3 ? l.k_scale[ph * size + slot] : 1.f, vs = KV <= L2_KV_E4M3 ? l.v_scale[ph * size + slot] : 1.f;
        for (int e = 0; e < E; e++) {
            const int64_t ki = (ph * size + slot) * D + 64 * e + lane, vi = (ph * D + 64 * e + lane) * size + slot;
            if (KV == L2_KV_I8) kx[e] = (float)((const int8_t *)l.k)[ki], vx[e] = (float)((const int8_t *)l.v)[vi];
            else if (KV == L2_KV_E4M3) kx[e] = kv::from_e4m3(((const uint8_t *)l.k)[ki]), vx[e] = kv::from_e4m3(((const uint8_t *)l.v)[vi]);
            else if (KV == L2_KV_F16) kx[e] = (float)((const _Float16 *)l.k)[ki], vx[e] = (float)((const _Float16 *)l.v)[vi];
            else kx[e] = kv::bf16_float(((const uint16_t *)l.k)[ki]), vx[e] = kv::bf16_float(((const uint16_t *)l.v)[vi]);
            dot += q[e] * kx[e];
        }
        for (int o = 32; o; o >>= 1) dot += __shfl_xor(dot, o);
        dot *= ks * a.scale;
        const float mm = dot > m || dot != dot ? dot : m, f = m == mm ? 1.f : expf(m - mm), p = dot == mm ? 1.f : expf(dot - mm);
        sum = sum * f + p;
        for (int e = 0; e < E; e++) acc[e] = acc[e] * f + p * (vx[e] * vs);
        m = mm;
    }
    __shared__ float sm[4], ss[4], sa[4][D];
    if (lane == 0) sm[w] = m, ss[w] = sum;
    for (int e = 0; e < E; e++) sa[w][64 * e + lane] = acc[e];
    __syncthreads();
    if (w) return;
    float top = -__builtin_inff(), total = 0.f;
    for (int x = 0; x < 4; x++) top = sm[x] > top || sm[x] != sm[x] ? sm[x] : top;
    float o[E] = {};
    for (int x = 0; x < 4; x++) {
        if (ss[x] == 0.f) continue;
        const float f = sm[x] == top ? 1.f : expf(sm[x] - top);
        total += ss[x] * f;
        for (int e = 0; e < E; e++) o[e] += sa[x][64 * e + lane] * f;
    }
    for (int e = 0; e < E; e++) kv::store(a.out, a.type, row * a.out_stride + (int64_t)hq * D + 64 * e + lane, total == 0.f ? 0.f : o[e] / total);
}

typedef void (*AttnKernel)(KvLayer, l2_kvbatch, KvAttention);
const AttnKernel kAttn[4][2] = {{kv_attention_kernel<0, 64>, kv_attention_kernel<0, 128>}, {kv_attention_kernel<1, 64>, kv_attention_kernel<1, 128>},
                                {kv_attention_kernel<2, 64>, kv_attention_kernel<2, 128>}, {kv_attention_kernel<3, 64>, kv_attention_kernel<3, 128>}};
typedef void (*NarrowKernel)(KvLayer, l2_kvbatch, KvAttention, Parts, int);
#define NARROW(kv, np) {kv_narrow_kernel<kv, np, 64>, kv_narrow_kernel<kv, np, 128>}
const NarrowKernel kNarrow[4][3][2] = {{NARROW(0, 1), NARROW(0, 2), {}}, {NARROW(1, 1), NARROW(1, 2), {}}, {NARROW(2, 1), NARROW(2, 2), {}}, {NARROW(3, 1), NARROW(3, 2), NARROW(3, 3)}};
typedef void (*JoinKernel)(l2_kvbatch, KvAttention, Parts, int, int);
const JoinKernel kJoin[2] = {kv_join_kernel<64>, kv_join_kernel<128>};

// In how many 16-bit numbers q and the weights enter the matrix cores, less one.
int pieces_index(int kv_type, int type) {
    if (kv_type == L2_KV_BF16) return type == L2_BF16 ? 0 : type == L2_F16 ? 1 : 2;
    return type == L2_F32 ? 1 : 0;
}

} // namespace

void kv_attention_plan(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvAttention &a, KvAttnPlan *plan) {
    const int tt = kv_type <= L2_KV_E4M3 ? 64 : 32;
    int64_t seen = b.max_length; // positions of the longest row
    if (a.window) seen = std::min<int64_t>(seen, (int64_t)a.window + b.max_rows + a.sinks + 2 * tt);
    const int64_t tiles = (seen + tt - 1) / tt, blocks = (int64_t)std::max(b.n_seqs, 1) * l.n_heads;
    const int64_t want = (2 * cu_count() + blocks - 1) / blocks;
    plan->splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, tiles / (2 * kNarrowWaves)));
    const size_t cells = (size_t)b.n_rows * a.n_heads * plan->splits;
    plan->workspace = plan->splits > 1 ? cells * (l.head_size * 4 + 8) : 0;
}

int kv_attention_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvAttention &a, const KvAttnPlan &plan, void *workspace, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    const int wide = l.head_size == 128, group = a.n_heads / l.n_heads;
    Parts parts{(float *)workspace, nullptr};
    parts.stat = (float2 *)(parts.acc + (size_t)b.n_rows * a.n_heads * plan.splits * l.head_size);
    if (group <= kNarrowRows) {
        l2_launch(kNarrow[kv_type][pieces_index(kv_type, a.type)][wide], dim3(plan.splits, l.n_heads, b.n_seqs), dim3(64 * kNarrowWaves), 0, st, l, b, a, parts,
                  plan.splits);
        if (plan.splits > 1) l2_launch(kJoin[wide], dim3(b.n_rows, a.n_heads), dim3(64), 0, st, b, a, parts, plan.splits, group);
    }
    if ((int64_t)b.max_rows * group > kNarrowRows)
        l2_launch(kAttn[kv_type][wide], dim3(b.n_rows, a.n_heads), dim3(256), 0, st, l, b, a);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_attention_warm_up() {
    hipFuncAttributes a;
    for (auto &k : kAttn) for (AttnKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    for (auto &k : kNarrow) for (auto &n : k) for (NarrowKernel f : n) if (f) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    for (JoinKernel f : kJoin) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    return L2_OK;
}
