// A cache in pages: rows quantised into their slots, and read back.
#include "kvpool.h"

namespace {

constexpr float kSmallest = 0x1p-60f;

// The whole number nearest to x / s, the tie to even, from the exact quotient: with q near it, x - q s is a float (its last place is no
// finer than half of s's or x's own, and it is at most about s), and says on which side of a half x / s lies.
__device__ __forceinline__ int code_i8(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), half = r + r;
    if (half > s || (half == s && ((int)q & 1))) q += 1.f;
    else if (half < -s || (half == -s && ((int)q & 1))) q -= 1.f;
    return (int)q;
}

// e4m3 nearest to x / s.  The quotient rounded to a float may meet a tie between two codes that the exact one only comes close to: where it is not
// exact, a float of the tie's form (an even last place) is moved off it to the exact one's side.
__device__ __forceinline__ uint8_t code_e4m3(float x, float s) {
    const float y = x / s, r = fmaf(-y, s, x);
    uint32_t b = __builtin_bit_cast(uint32_t, y);
    if (r != 0.f && !(b & 1) && (b << 1)) b += (r > 0.f) == (y > 0.f) ? 1u : ~0u;
    const float z = __builtin_bit_cast(float, b);
    return kv::to_e4m3(fminf(fmaxf(z, -448.f), 448.f));
}

__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// One wave per row and kv head.
template <int KV, int D>
__global__ __launch_bounds__(64) void kv_write_kernel(KvLayer l, l2_kvbatch b, KvRows rows) {
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int i = kv::sequence_of(b, row);
    if (i >= b.n_seqs) return;
    const kv::Seq s = kv::sequence(b, i);
    const int at = row - s.first, pos = s.length - s.rows + at;
    if (at >= s.rows || pos < 0) return;
    const int page = kv::page_at(b, l.n_pages, i, pos >> l.page_shift);
    if (page < 0) return;
    const int slot = pos & ((1 << l.page_shift) - 1);
    const int64_t ph = (int64_t)page * l.n_heads + h, size = 1 << l.page_shift;
    constexpr int E = D / 64;
    for (int x = 0; x < 2; x++) {
        float v[E], a = 0.f;
        for (int e = 0; e < E; e++) {
            v[e] = kv::load(x ? rows.v : rows.k, rows.type, row * (x ? rows.v_stride : rows.k_stride) + (int64_t)h * D + 64 * e + lane);
            a = fmaxf(a, fabsf(v[e]) < __builtin_inff() ? fabsf(v[e]) : __builtin_inff());
        }
        a = wave_max(a);
        const bool fine = a < __builtin_inff(), some = fine && a >= kSmallest;
        const float scale = some ? a / (KV == L2_KV_I8 ? 127.f : 448.f) : 0.f, inv = some ? 1.f / scale : 0.f;
        if (KV <= L2_KV_E4M3 && lane == 0) (x ? l.v_scale : l.k_scale)[ph * size + slot] = fine ? scale : __builtin_nanf("");
        for (int e = 0; e < E; e++) {
            const int d = 64 * e + lane;
            const int64_t to = x ? (ph * D + d) * size + slot : (ph * size + slot) * D + d;
            void *dst = x ? l.v : l.k;
            if (KV == L2_KV_I8) ((int8_t *)dst)[to] = some ? (int8_t)code_i8(v[e], scale, inv) : 0;
            else if (KV == L2_KV_E4M3) ((uint8_t *)dst)[to] = some ? code_e4m3(v[e], scale) : 0;
            else if (KV == L2_KV_F16) ((_Float16 *)dst)[to] = (_Float16)v[e];
            else ((uint16_t *)dst)[to] = kv::float_bf16(v[e]);
        }
    }
}

template <int KV, int D>
__global__ __launch_bounds__(64) void kv_read_kernel(KvLayer l, l2_kvbatch b, KvRows rows) {
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int i = kv::sequence_of(b, row);
    if (i >= b.n_seqs) return;
    const kv::Seq s = kv::sequence(b, i);
    const int at = row - s.first, pos = s.length - s.rows + at;
    if (at >= s.rows) return;
    const int page = pos < 0 ? -1 : kv::page_at(b, l.n_pages, i, pos >> l.page_shift);
    const int slot = pos & ((1 << l.page_shift) - 1);
    const int64_t ph = (int64_t)page * l.n_heads + h, size = 1 << l.page_shift;
    for (int x = 0; x < 2; x++) {
        const float scale = KV <= L2_KV_E4M3 && page >= 0 ? (x ? l.v_scale : l.k_scale)[ph * size + slot] : 0.f;
        for (int d = lane; d < D; d += 64) {
            float v = 0.f;
            if (page >= 0) {
                const int64_t from = x ? (ph * D + d) * size + slot : (ph * size + slot) * D + d;
                const void *src = x ? l.v : l.k;
                if (KV == L2_KV_I8) v = (float)((const int8_t *)src)[from] * scale;
                else if (KV == L2_KV_E4M3) v = kv::from_e4m3(((const uint8_t *)src)[from]) * scale;
                else if (KV == L2_KV_F16) v = (float)((const _Float16 *)src)[from];
                else v = kv::bf16_float(((const uint16_t *)src)[from]);
            }
            kv::store(const_cast<void *>(x ? rows.v : rows.k), rows.type, row * (x ? rows.v_stride : rows.k_stride) + (int64_t)h * D + d, v);
        }
    }
}

typedef void (*RowsKernel)(KvLayer, l2_kvbatch, KvRows);
const RowsKernel kWrite[4][2] = {{kv_write_kernel<0, 64>, kv_write_kernel<0, 128>}, {kv_write_kernel<1, 64>, kv_write_kernel<1, 128>},
                                 {kv_write_kernel<2, 64>, kv_write_kernel<2, 128>}, {kv_write_kernel<3, 64>, kv_write_kernel<3, 128>}};
const RowsKernel kRead[4][2] = {{kv_read_kernel<0, 64>, kv_read_kernel<0, 128>}, {kv_read_kernel<1, 64>, kv_read_kernel<1, 128>},
                                {kv_read_kernel<2, 64>, kv_read_kernel<2, 128>}, {kv_read_kernel<3, 64>, kv_read_kernel<3, 128>}};

} // namespace

int kv_write_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    l2_launch(kWrite[kv_type][l.head_size == 128], dim3(b.n_rows, l.n_heads), dim3(64), 0, st, l, b, rows);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_read_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    l2_launch(kRead[kv_type][l.head_size == 128], dim3(b.n_rows, l.n_heads), dim3(64), 0, st, l, b, rows);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_rows_warm_up() {
    hipFuncAttributes a;
    for (auto &k : kWrite) for (RowsKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    for (auto &k : kRead) for (RowsKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    return L2_OK;
}
