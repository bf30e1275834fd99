// A cache in pages: rows quantised into their slots, and read back.
#include "kvpool.h"

namespace {

constexpr float kSmallest = 0x1p-60f;

// A float that rounds to a code as x / s does, x >= 0: within a step of the quotient, and where it is not exact an odd one on the exact one's side of any tie
// between two codes (those are even), found from the remainder, which is a float.
__device__ __forceinline__ float odd_quotient(float x, float s, float inv) {
    float y = x * inv;
    y = fmaf(fmaf(-y, s, x), inv, y);
    const float r = fmaf(-y, s, x);
    const uint32_t up = __builtin_bit_cast(uint32_t, r) >> 31; // y is above the quotient
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, y) - up) | (r != 0.f));
}

// E values of a row as cells; some: the row is held at all.
template <int KV, int E, class Cell>
__device__ __forceinline__ void cells_of(const float (&v)[E], bool some, float scale, float inv, Cell (&c)[E]) {
    if constexpr (KV == L2_KV_E4M3) {
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            const int k = j + 1 < E ? j + 1 : j;
            const float y0 = copysignf(odd_quotient(fabsf(v[j]), scale, inv), v[j]), y1 = copysignf(odd_quotient(fabsf(v[k]), scale, inv), v[k]);
            const int two = some ? __builtin_amdgcn_cvt_pk_fp8_f32(y0, y1, 0, false) : 0;
            c[j] = (Cell)two;
            if (k > j) c[k] = (Cell)(two >> 8);
        }
    } else {
#pragma unroll
        for (int j = 0; j < E; j++)
            c[j] = KV == L2_KV_I8    ? some ? (Cell)(int)rintf(copysignf(odd_quotient(fabsf(v[j]), scale, inv), v[j])) : 0
                   : KV == L2_KV_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[j])
                                     : kv::float_bf16(v[j]);
    }
}
template <int KV, class Cell>
__device__ __forceinline__ float value_of(Cell c, float scale) {
    return KV == L2_KV_I8     ? (float)(int8_t)c * scale
           : KV == L2_KV_E4M3 ? kv::from_e4m3((uint8_t)c) * scale
           : KV == L2_KV_F16  ? (float)__builtin_bit_cast(_Float16, (uint16_t)c)
                              : kv::bf16_float(c);
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64, kThreads = 256; // positions of a block, aligned

// A block's sequence and tile: tile x of sequence i is block starts[i] / 64 + 2 i + x, which leaves every sequence as many as it may need (its rows
// are its last positions, wherever these begin).  False: the block has none.
struct Work {
    kv::Seq s;
    int i, base, p0; // base: position of the first row; p0: of the tile
};
__device__ __forceinline__ bool work_of(const l2_kvbatch &b, Work &w) {
    const int j = blockIdx.x;
    // the last i whose first block is not behind this one, 64 at a time
    const int lane = threadIdx.x & 63;
    int lo = 0, n = b.n_seqs;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lo + lane * step;
        const bool fits = lane * step < n && (min(max(b.starts[i], 0), b.n_rows) >> 6) + 2 * i <= j;
        const int behind = max(__popcll(__ballot(fits)) - 1, 0) * step;
        lo += behind, n = min(step, n - behind);
    }
    w.i = lo;
    w.s = kv::sequence(b, w.i);
    const int x = j - (w.s.first >> 6) - 2 * w.i;
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

// Of E values of a row of a kv head, LANES lanes with as many each: the row's scale, its inverse, and whether it is held at all (values that are not finite: as NaN).
struct Scale {
    float s, inv;
    bool some, fine;
};
template <int KV, int LANES, int E>
__device__ __forceinline__ Scale scale_of(const float (&v)[E]) {
    Scale o{0.f, 0.f, true, true};
    if constexpr (KV <= L2_KV_E4M3) {
        float a = 0.f;
#pragma unroll
        for (int j = 0; j < E; j++) a = fmaxf(a, fabsf(v[j]) < __builtin_inff() ? fabsf(v[j]) : __builtin_inff());
        a = row_max<LANES>(a);
        o.fine = a < __builtin_inff();
        o.some = o.fine && a >= kSmallest;
        o.s = o.some ? a / (KV == L2_KV_I8 ? 127.f : 448.f) : 0.f, o.inv = o.some ? 1.f / o.s : 0.f;
    }
    return o;
}

// Few rows: a wave for the key and one for the value of a row's head, two values (one) to a lane, no LDS.  Rows i * max_rows + at, row `at` of sequence i.  Bound by
// the launch and four dependent loads.
template <int KV, int D>
__global__ __launch_bounds__(128) void kv_write_rows_kernel(KvLayer l, l2_kvbatch b, KvRows rows) {
    using Cell = std::conditional_t<KV <= L2_KV_E4M3, uint8_t, uint16_t>;
    constexpr int E = D / 64;
    const int i = blockIdx.x / b.max_rows, at = blockIdx.x % b.max_rows, h = blockIdx.y, lane = threadIdx.x & 63;
    const bool value = threadIdx.x >= 64;
    const kv::Seq s = kv::sequence(b, i);
    const int pos = s.length - s.rows + at, size = 1 << l.page_shift;
    if (at >= s.rows || pos < 0) return;
    const int64_t from = (s.first + at) * (value ? rows.v_stride : rows.k_stride) + (int64_t)h * D + E * lane;
    const int page = kv::page_at(b, l.n_pages, i, pos >> l.page_shift);
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = kv::load(value ? rows.v : rows.k, rows.type, from + e);
    const Scale o = scale_of<KV, 64, E>(v);
    if (page < 0) return;
    const int64_t ph = (int64_t)page * l.n_heads + h, slot = ph * size + (pos & (size - 1));
    if (KV <= L2_KV_E4M3 && lane == 0) (value ? l.v_scale : l.k_scale)[slot] = o.fine ? o.s : __builtin_nanf("");
    Cell c[E];
    cells_of<KV, E, Cell>(v, o.some, o.s, o.inv, c);
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (value) ((Cell *)l.v)[(ph * D + E * lane + e) * size + (pos & (size - 1))] = c[e];
        else ((Cell *)l.k)[slot * D + E * lane + e] = c[e];
    }
}
template <int KV, int D>
__global__ __launch_bounds__(128) void kv_read_rows_kernel(KvLayer l, l2_kvbatch b, KvRows rows) {
    using Cell = std::conditional_t<KV <= L2_KV_E4M3, uint8_t, uint16_t>;
    constexpr int E = D / 64;
    const int i = blockIdx.x / b.max_rows, at = blockIdx.x % b.max_rows, h = blockIdx.y, lane = threadIdx.x & 63;
    const bool value = threadIdx.x >= 64;
    const kv::Seq s = kv::sequence(b, i);
    const int pos = s.length - s.rows + at, size = 1 << l.page_shift;
    if (at >= s.rows) return;
    const int page = pos < 0 ? -1 : kv::page_at(b, l.n_pages, i, pos >> l.page_shift);
    const int64_t ph = (int64_t)page * l.n_heads + h, slot = ph * size + (pos & (size - 1));
    float v[E] = {};
    if (page >= 0) {
        Cell c[E];
#pragma unroll
        for (int e = 0; e < E; e++) c[e] = value ? ((const Cell *)l.v)[(ph * D + E * lane + e) * size + (pos & (size - 1))] : ((const Cell *)l.k)[slot * D + E * lane + e];
        const float scale = KV <= L2_KV_E4M3 ? (value ? l.v_scale : l.k_scale)[slot] : 1.f;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = value_of<KV>(c[e], scale);
    }
    const int64_t to = (s.first + at) * (value ? rows.v_stride : rows.k_stride) + (int64_t)h * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; e++) kv::store(const_cast<void *>(value ? rows.v : rows.k), rows.type, to + e, v[e]);
}

// A block quantises 64 positions of a kv head, eight values of a row to a lane.  Values go through LDS, where they turn, so that 64 positions of each
// dimension are stored side by side (the runs of 16 that are not whole, one by one).  Bound by memory.
template <int KV, int D>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvLayer l, l2_kvbatch b, KvRows rows) {
    constexpr bool kEight = KV <= L2_KV_E4M3;
    using Cell = std::conditional_t<kEight, uint8_t, uint16_t>;
    typedef Cell eight __attribute__((ext_vector_type(8)));
    constexpr int LANES = D / 8, AT_ONCE = kThreads / LANES, PER = 16 / sizeof(Cell), LD = kTile + 4 / sizeof(Cell);
    __shared__ Cell sh[D][LD];
    Work w;
    if (!work_of(b, w)) return;
    const int h = blockIdx.y, tid = threadIdx.x, x = tid % LANES, size = 1 << l.page_shift;
    const int from = max(w.base, 0); // positions from here are written
    auto row_cells = [&](const kv::f8 &val, float *scales, int64_t slot, Cell (&c)[8]) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = val[j];
        const Scale o = scale_of<KV, LANES, 8>(v);
        if (kEight && x == 0) scales[slot] = o.fine ? o.s : __builtin_nanf("");
        cells_of<KV, 8, Cell>(v, o.some, o.s, o.inv, c);
    };
#pragma unroll
    for (int y = 0; y < kTile / AT_ONCE; y++) {
        const int t = tid / LANES + AT_ONCE * y, pos = w.p0 + t;
        const int page = pos >= from && pos < w.s.length ? kv::page_at(b, l.n_pages, w.i, pos >> l.page_shift) : -1;
        if (page < 0) continue; // all lanes of the row
        const int64_t row = w.s.first + pos - w.base, slot = ((int64_t)page * l.n_heads + h) * size + (pos & (size - 1));
        Cell c[8];
        row_cells(kv::load8(rows.k, rows.type, row * rows.k_stride + (int64_t)h * D + 8 * x), l.k_scale, slot, c);
        *(eight *)((Cell *)l.k + (slot * D + 8 * x)) = eight{c[0], c[1], c[2], c[3], c[4], c[5], c[6], c[7]};
        row_cells(kv::load8(rows.v, rows.type, row * rows.v_stride + (int64_t)h * D + 8 * x), l.v_scale, slot, c);
#pragma unroll
        for (int j = 0; j < 8; j++) sh[8 * x + j][t] = c[j];
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
    typedef Cell eight __attribute__((ext_vector_type(8)));
    const int h = blockIdx.y, tid = threadIdx.x, x = tid % LANES, size = 1 << l.page_shift;
#pragma unroll
    for (int y = 0; y < D * RUNS / kThreads; y++) {
        const int p = tid + kThreads * y, d = p / RUNS, t = p % RUNS * PER, pos = w.p0 + t;
        if (pos + PER <= w.base || pos < 0 || pos >= w.s.length) continue;
        const int pv = kv::page_at(b, l.n_pages, w.i, pos >> l.page_shift);
        if (pv < 0) continue;
        const u4 c = *(const u4 *)((const Cell *)l.v + ((((int64_t)pv * l.n_heads + h) * D + d) * size + (pos & (size - 1))));
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
                eight c;
                if (v == 0) c = *(const eight *)((const Cell *)l.k + (slot * D + 8 * x));
                else
#pragma unroll
                    for (int j = 0; j < 8; j++) c[j] = sh[8 * x + j][t];
                const float scale = kEight ? (v ? l.v_scale : l.k_scale)[slot] : 1.f;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    val[j] = value_of<KV>(c[j], scale);
            }
            kv::store8(const_cast<void *>(v ? rows.v : rows.k), rows.type, row * (v ? rows.v_stride : rows.k_stride) + (int64_t)h * D + 8 * x, val);
        }
    }
}

typedef void (*RowsKernel)(KvLayer, l2_kvbatch, KvRows);
#define ALL(kernel) {{kernel<0, 64>, kernel<0, 128>}, {kernel<1, 64>, kernel<1, 128>}, {kernel<2, 64>, kernel<2, 128>}, {kernel<3, 64>, kernel<3, 128>}}
const RowsKernel kWrite[4][2] = ALL(kv_write_kernel), kWriteRows[4][2] = ALL(kv_write_rows_kernel), kRead[4][2] = ALL(kv_read_kernel), kReadRows[4][2] = ALL(kv_read_rows_kernel);

// Rows by themselves where tiles of 64 positions would be nearly empty, or too few to fill the device.  us as rows and as tiles, 8 kv heads, fp32 rows to 8 bits and fp16
// rows to fp16: one row of each of 16, 128, 512 sequences 3.7 / 5.9, 4.6 / 11, 9.7 / 22 and 3.6 / 5.1, 4.1 / 8.8, 9.5 / 20 (3.5 is what a call takes); 200, 400, 800 rows of one
// sequence 4.2 / 10, 6.0 / 9.6, 8.8 / 11 and 4.1 / 6.8, 5.9 / 5.7, 9.0 / 5.9; read back 3.6 / 5.1, 4.1 / 5.4, 5.7 / 5.9.
constexpr int kFewRows = 8, kFew = 2048; // of a sequence; rows times heads

dim3 grid(const KvLayer &l, const l2_kvbatch &b) { return dim3(b.n_rows / kTile + 2 * b.n_seqs, l.n_heads); }

} // namespace

static int launch(const RowsKernel (&tiles)[4][2], const RowsKernel (&few)[4][2], const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    const int big = l.head_size == 128;
    const bool rows_alone = b.max_rows <= kFewRows || (int64_t)b.n_seqs * b.max_rows * l.n_heads <= kFew;
    if (rows_alone) l2_launch(few[kv_type][big], dim3(b.n_seqs * b.max_rows, l.n_heads), dim3(128), 0, st, l, b, rows);
    else l2_launch(tiles[kv_type][big], grid(l, b), dim3(kThreads), 0, st, l, b, rows);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_write_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st) { return launch(kWrite, kWriteRows, l, kv_type, b, rows, st); }
int kv_read_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st) { return launch(kRead, kReadRows, l, kv_type, b, rows, st); }

int kv_rows_warm_up() {
    hipFuncAttributes a;
    for (auto *all : {&kWrite, &kWriteRows, &kRead, &kReadRows})
        for (auto &k : *all)
            for (RowsKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    return L2_OK;
}
