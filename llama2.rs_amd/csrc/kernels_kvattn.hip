// Attention of new rows over a cache in pages.
#include "kvpool.h"

namespace {

// One block per row and query head; its four waves take positions in turn, each with a running maximum and sum, and are joined at the end.
template <int KV, int D>
__global__ __launch_bounds__(256) void kv_attention_kernel(KvLayer l, l2_kvbatch b, KvAttention a) {
    const int row = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int i = kv::sequence_of(b, row);
    if (i >= b.n_seqs) return;
    const kv::Seq s = kv::sequence(b, i);
    const int at = row - s.first, pos = s.length - s.rows + at;
    if (at >= s.rows) return;
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

} // namespace

void kv_attention_plan(const KvLayer &, int, const l2_kvbatch &, const KvAttention &, KvAttnPlan *plan) { plan->workspace = 0; }

int kv_attention_launch(const KvLayer &l, int kv_type, const l2_kvbatch &b, const KvAttention &a, const KvAttnPlan &, void *, hipStream_t st) {
    if (b.n_rows == 0 || b.n_seqs == 0 || b.max_rows == 0) return L2_OK;
    l2_launch(kAttn[kv_type][l.head_size == 128], dim3(b.n_rows, a.n_heads), dim3(256), 0, st, l, b, a);
    L2_HIP(hipGetLastError());
    return L2_OK;
}

int kv_attention_warm_up() {
    hipFuncAttributes a;
    for (auto &k : kAttn) for (AttnKernel f : k) L2_HIP(hipFuncGetAttributes(&a, (const void *)f));
    return L2_OK;
}
