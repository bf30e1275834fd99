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

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64, kThreads = 256; // positions of a block, aligned

// A block's sequence and tile: tile x of sequence i is block starts[i] / 64 + 2 i + x, which leaves every sequence as many as it may need (its rows
// are its last positions, wherever these begin); of single rows, block i.  False: the block has none.
struct Work {
    kv::Seq s;
    int i, base, p0; // base: position of the first row; p0: of the tile
};
__device__ __forceinline__ bool work_of(const l2_kvbatch &b, Work &w) {
    const int j = blockIdx.x;
    if (b.max_rows == 1) {
        w.i = j;
    } else {
        int lo = 0, hi = b.n_seqs; // the last i whose first block is not behind this one
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((min(max(b.starts[mid], 0), b.n_rows) >> 6) + 2 * mid <= j) lo = mid;
            else hi = mid;
        }
        w.i = lo;
    }
    w.s = kv::sequence(b, w.i);
    const int x = b.max_rows == 1 ? 0 : j - (w.s.first >> 6) - 2 * w.i;
    w.base = w.s.length - w.s.rows;
    w.p0 = ((w.base >> 6) + x) * kTile;
    return x >= 0 && w.p0 < w.s.length && w.s.rows > 0;
}

// The largest of a row's lanes.
template <int LANES>
__device__ __forceinline__ float row_max(float v) {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// A block quantises 64 positions of a kv head, eight values of a row to a lane.  Values go through LDS, where they turn, so that 64 positions of each
// dimension are stored side by side (the runs of 16 that are not whole, one by one).  Bound by memory.
template <int KV, int D>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvLayer l, l2_kvbatch b, KvRows rows) {
    constexpr bool kEight = KV <= L2_KV_E4M3;
    using Cell = std::conditional_t<kEight, uint8_t, uint16_t>;
    constexpr int LANES = D / 8, AT_ONCE = kThreads / LANES, PER = 16 / sizeof(Cell), LD = kTile + 4 / sizeof(Cell);
    __shared__ Cell sh[D][LD];
    Work w;
    if (!work_of(b, w)) return;
    const int h = blockIdx.y, tid = threadIdx.x, x = tid % LANES, size = 1 << l.page_shift;
    const int from = max(w.base, 0); // positions from here are written
#pragma unroll
    for (int y = 0; y < kTile / AT_ONCE; y++) {
        const int t = tid / LANES + AT_ONCE * y, pos = w.p0 + t;
        const int page = pos >= from && pos < w.s.length ? kv::page_at(b, l.n_pages, w.i, pos >> l.page_shift) : -1;
        if (page < 0) continue; // all lanes of the row
        const int64_t row = w.s.first + pos - w.base, ph = (int64_t)page * l.n_heads + h, slot = ph * size + (pos & (size - 1));
#pragma unroll
        for (int v = 0; v < 2; v++) {
            const kv::f8 val = kv::load8(v ? rows.v : rows.k, rows.type, row * (v ? rows.v_stride : rows.k_stride) + (int64_t)h * D + 8 * x);
            Cell c[8];
            if constexpr (kEight) {
                float a = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) a = fmaxf(a, fabsf(val[j]) < __builtin_inff() ? fabsf(val[j]) : __builtin_inff());
                a = row_max<LANES>(a);
                const bool fine = a < __builtin_inff(), some = fine && a >= kSmallest;
                const float scale = some ? a / (KV == L2_KV_I8 ? 127.f : 448.f) : 0.f, inv = some ? 1.f / scale : 0.f;
                if (x == 0) (v ? l.v_scale : l.k_scale)[slot] = fine ? scale : __builtin_nanf("");
#pragma unroll
                for (int j = 0; j < 8; j++) c[j] = !some ? 0 : KV == L2_KV_I8 ? (uint8_t)code_i8(val[j], scale, inv) : code_e4m3(val[j], scale);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) c[j] = KV == L2_KV_F16 ? __builtin_bit_cast(uint16_t, (_Float16)val[j]) : kv::float_bf16(val[j]);
            }
            if (v == 0) {
                typedef Cell eight __attribute__((ext_vector_type(8)));
                *(eight *)((Cell *)l.k + (slot * D + 8 * x)) = eight{c[0], c[1], c[2], c[3], c[4], c[5], c[6], c[7]};
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) sh[8 * x + j][t] = c[j];
            }
        }
    }
    __syncthreads();
    constexpr int RUNS = kTile / PER;
    for (int p = tid; p < D * RUNS; p += kThreads) {
        const int d = p / RUNS, t = p % RUNS * PER, pos = w.p0 + t;
        if (pos + PER <= from || pos >= w.s.length) continue;
        const int page = kv::page_at(b, l.n_pages, w.i, pos >> l.page_shift); // pages are whole runs of 16
        if (page < 0) continue;
        Cell *to = (Cell *)l.v + ((((int64_t)page * l.n_heads + h) * D + d) * size + (pos & (size - 1)));
        if (pos >= from && pos + PER <= w.s.length) {
            u4 c;
#pragma unroll
            for (int j = 0; j < 4; j++) c[j] = *(const uint32_t *)&sh[d][t + j * PER / 4];
            *(u4 *)to = c;
        } else {
            for (int j = 0; j < PER; j++)
                if (pos + j >= from && pos + j < w.s.length) to[j] = sh[d][t + j];
        }
    }
}

// The inverse, the same way.
template <int KV, int D>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvLayer l, l2_kvbatch b, KvRows rows) {
    constexpr bool kEight = KV <= L2_KV_E4M3;
    using Cell = std::conditional_t<kEight, uint8_t, uint16_t>;
    constexpr int LANES = D / 8, AT_ONCE = kThreads / LANES, PER = 16 / sizeof(Cell), LD = kTile + 4 / sizeof(Cell), RUNS = kTile / PER;
    __shared__ Cell sh[D][LD];
    Work w;
    if (!work_of(b, w)) return;
    const int h = blockIdx.y, tid = threadIdx.x, x = tid % LANES, size = 1 << l.page_shift;
#pragma unroll
    for (int y = 0; y < D * RUNS / kThreads; y++) {
        const int p = tid + kThreads * y, d = p / RUNS, t = p % RUNS * PER, pos = w.p0 + t;
        if (pos + PER <= w.base || pos < 0 || pos >= w.s.length) continue;
        const int page = kv::page_at(b, l.n_pages, w.i, pos >> l.page_shift);
        if (page < 0) continue;
        const u4 c = *(const u4 *)((const Cell *)l.v + ((((int64_t)page * l.n_heads + h) * D + d) * size + (pos & (size - 1))));
#pragma unroll
        for (int j = 0; j < 4; j++) *(uint32_t *)&sh[d][t + j * PER / 4] = c[j];
    }
    __syncthreads();
#pragma unroll
    for (int y = 0; y < kTile / AT_ONCE; y++) {
        const int t = tid / LANES + AT_ONCE * y, pos = w.p0 + t;
        if (pos < w.base || pos >= w.s.length) continue;
        const int page = pos < 0 ? -1 : kv::page_at(b, l.n_pages, w.i, pos >> l.page_shift);
        const int64_t row = w.s.first + pos - w.base, slot = ((int64_t)page * l.n_heads + h) * size + (pos & (size - 1));
#pragma unroll
        for (int v = 0; v < 2; v++) {
            kv::f8 val = {};
            if (page >= 0) {
                typedef Cell eight __attribute__((ext_vector_type(8)));
                eight c;
                if (v == 0) c = *(const eight *)((const Cell *)l.k + (slot * D + 8 * x));
                else
#pragma unroll
                    for (int j = 0; j < 8; j++) c[j] = sh[8 * x + j][t];
                const float scale = kEight ? (v ? l.v_scale : l.k_scale)[slot] : 1.f;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    val[j] = KV == L2_KV_I8     ? (float)(int8_t)c[j] * scale
                             : KV == L2_KV_E4M3 ? kv::from_e4m3((uint8_t)c[j]) * scale
                             : KV == L2_KV_F16  ? (float)__builtin_bit_cast(_Float16, (uint16_t)c[j])
                                                : kv::bf16_float(c[j]);
            }
            kv::store8(const_cast<void *>(v ? rows.v : rows.k), rows.type, row * (v ? rows.v_stride : rows.k_stride) + (int64_t)h * D + 8 * x, val);
        }
    }
}

typedef void (*RowsKernel)(KvLayer, l2_kvbatch, KvRows);
const RowsKernel kWrite[4][2] = {{kv_write_kernel<0, 64>, kv_write_kernel<0, 128>}, {kv_write_kernel<1, 64>, kv_write_kernel<1, 128>},
                                 {kv_write_kernel<2, 64>, kv_write_kernel<2, 128>}, {kv_write_kernel<3, 64>, kv_write_kernel<3, 128>}};
const RowsKernel kRead[4][2] = {{kv_read_kernel<0, 64>, kv_read_kernel<0, 128>}, {kv_read_kernel<1, 64>, kv_read_kernel<1, 128>},
                                {kv_read_kernel<2, 64>, kv_read_kernel<2, 128>}, {kv_read_kernel<3, 64>, kv_read_kernel<3, 128>}};

dim3 grid(const KvLayer &l, const l2_kvbatch &b) { return dim3(b.max_rows == 1 ? b.n_seqs : b.n_rows / kTile + 2 * b.n_seqs, l.n_heads); }

} // namespace

int kv_write_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    l2_launch(kWrite[kv_type][l.head_size == 128], grid(l, b), dim3(kThreads), 0, st, l, b, rows);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_read_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    l2_launch(kRead[kv_type][l.head_size == 128], grid(l, b), dim3(kThreads), 0, st, l, b, rows);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_rows_warm_up() {
    hipFuncAttributes a;
    for (auto &k : kWrite) for (RowsKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    for (auto &k : kRead) for (RowsKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    return L2_OK;
}
