// The pages of a pool and the sequences of a call, as the kernels on them see these (kernels_kvpool.hip, kernels_kvattn.hip).
#pragma once

#include <hip/hip_fp16.h>

#include "l2_internal.h"

// One layer of a pool.  Keys lie as [page][kv head][slot][value] and values as [page][kv head][value][slot]: both are then what the matrix
// instructions of scores and of weighted sums want of their first operand, 16 contiguous bytes of the inner dimension per lane, without a transposition.
// Scales lie as [page][kv head][slot].
struct KvLayer {
    void *k, *v;
    float *k_scale, *v_scale; // 8 bits only
    int n_pages, n_heads, head_size;
    int page_shift; // log2 of the positions of a page
};

struct KvRows { // rows of the caller's: [row][kv head][value]
    const void *k, *v;
    int64_t k_stride, v_stride;
    int type;
};

int kv_write_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st);
int kv_read_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvRows &rows, hipStream_t st);
// Loads what the launches above need, on the current device.
int kv_rows_warm_up();

struct KvAttention {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    int n_heads, type;
    float scale;
    int window, sinks;
};
// How the limits of a call are cut up: a function of them alone.
struct KvAttnPlan {
    size_t workspace;               // bytes
    bool wide;                      // whether there may be sequences of more rows than ..
    int narrow_rows;                // .. the narrow kernel takes, per kv head; 0: it takes none
    int narrow_blocks;              // of 16 rows, of a sequence and kv head
    int narrow_splits, wide_splits; // parts that positions are cut into,
    int narrow_per, wide_per;       // each of so many tiles
    int stride;                     // the larger of both: parts of a row in the workspace
    int64_t wide_tiles;             // tiles of rows of the wide kernel, at most
};
void kv_attention_plan(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvAttention &a, KvAttnPlan *plan);
int kv_attention_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvAttention &a, const KvAttnPlan &plan, void *workspace,
                        hipStream_t st);
int kv_attention_warm_up();
int sample_warm_up();

#if defined(__HIPCC__)
namespace kv {

// What a call's arrays say of a sequence, cut off at the call's limits.
struct Seq {
    int first, rows; // rows of the call's arrays
    int length;      // positions
};
__device__ __forceinline__ Seq sequence(const l2_kvbatch &b, int i) {
    const int s0 = min(max(b.starts[i], 0), b.n_rows), s1 = min(max(b.starts[i + 1], s0), b.n_rows);
    const int most = (int)min((int64_t)b.max_length, (int64_t)b.max_pages << 8);
    return {s0, min(s1 - s0, b.max_rows), min(max(b.lengths[i], 0), most)};
}

// The sequence that a row of the call's arrays belongs to; n_seqs if none.
__device__ __forceinline__ int sequence_of(const l2_kvbatch &b, int row) {
    int lo = 0, hi = b.n_seqs; // the first i with starts[i + 1] > row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (b.starts[mid + 1] > row) hi = mid;
        else lo = mid + 1;
    }
    return lo < b.n_seqs && b.starts[lo] <= row ? lo : b.n_seqs;
}

// The page of a position (in units of pages) of sequence i; -1: none.
__device__ __forceinline__ int page_at(const l2_kvbatch &b, int n_pages, int i, int at) {
    if (at >= b.max_pages) return -1;
    const int p = b.pages[(int64_t)i * b.max_pages + at];
    return (uint32_t)p < (uint32_t)n_pages ? p : -1;
}

// What a code of e4m3 stands for.
__device__ __forceinline__ float from_e4m3(uint8_t c) { return __builtin_amdgcn_cvt_f32_fp8((int)c, 0); }

__device__ __forceinline__ float bf16_float(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
__device__ __forceinline__ uint16_t float_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

__device__ __forceinline__ float load(const void *p, int type, int64_t i) {
    if (type == L2_F32) return ((const float *)p)[i];
    if (type == L2_F16) return (float)((const _Float16 *)p)[i];
    return bf16_float(((const uint16_t *)p)[i]);
}
__device__ __forceinline__ void store(void *p, int type, int64_t i, float v) {
    if (type == L2_F32) ((float *)p)[i] = v;
    else if (type == L2_F16) ((_Float16 *)p)[i] = (_Float16)v;
    else ((uint16_t *)p)[i] = float_bf16(v);
}

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));

// Eight values of a row of the caller's, aligned as their type is; as they lie in memory first, so that several are on their way at once.
typedef uint32_t raw8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ raw8 load_raw8(const void *p, int type, int64_t i) {
    typedef uint32_t any8 __attribute__((ext_vector_type(8), aligned(4)));
    typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
    if (type == L2_F32) {
        const any8 v = *(const any8 *)((const float *)p + i);
        return raw8{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
    }
    const any4 v = *(const any4 *)((const uint16_t *)p + i);
    return raw8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
}
__device__ __forceinline__ f8 values8(const raw8 &v, int type) {
    f8 x;
    if (type == L2_F32) {
        x = __builtin_bit_cast(f8, v);
    } else if (type == L2_F16) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = (float)__builtin_bit_cast(_Float16, (uint16_t)(v[j / 2] >> 16 * (j % 2)));
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = bf16_float((uint16_t)(v[j / 2] >> 16 * (j % 2)));
    }
    return x;
}
__device__ __forceinline__ f8 load8(const void *p, int type, int64_t i) { return values8(load_raw8(p, type, i), type); }

__device__ __forceinline__ void store4(void *p, int type, int64_t i, const f4 &v) {
    typedef _Float16 anyh __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint16_t anyb __attribute__((ext_vector_type(4), aligned(2)));
    if (type == L2_F32) *(float4_any *)((float *)p + i) = float4_any{v[0], v[1], v[2], v[3]};
    else if (type == L2_F16) *(anyh *)((_Float16 *)p + i) = anyh{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    else *(anyb *)((uint16_t *)p + i) = anyb{float_bf16(v[0]), float_bf16(v[1]), float_bf16(v[2]), float_bf16(v[3])};
}

__device__ __forceinline__ void store8(void *p, int type, int64_t i, const f8 &v) {
    if (type != L2_F32) {
        typedef uint16_t any __attribute__((ext_vector_type(8), aligned(2)));
        any c;
        for (int j = 0; j < 8; j++) c[j] = type == L2_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[j]) : float_bf16(v[j]);
        *(any *)((uint16_t *)p + i) = c;
    } else {
        store4(p, type, i, f4{v[0], v[1], v[2], v[3]});
        store4(p, type, i + 4, f4{v[4], v[5], v[6], v[7]});
    }
}

} // namespace kv
#endif
