// Host side of the operators on a cache in pages and of sampling on device memory: handles, checks of arguments, launches.
#include <math.h>

#include <initializer_list>
#include <new>

#include "kvpool.h"

struct l2_kvpool {
    int n_layers = 0, n_pages = 0, page_size = 0, n_kv_heads = 0, head_size = 0, type = 0, device = 0;
    char *base = nullptr;
    size_t cells = 0, scales = 0; // bytes of the keys (as many of the values) of a layer, and of their scales
    size_t bytes() const { return 2 * (size_t)n_layers * (cells + scales); }
    KvLayer layer(int i) const {
        char *at = base + 2 * (size_t)i * (cells + scales);
        KvLayer l{};
        l.k = at, l.v = at + cells;
        l.k_scale = (float *)(at + 2 * cells), l.v_scale = (float *)(at + 2 * cells + scales);
        l.n_pages = n_pages, l.n_heads = n_kv_heads, l.head_size = head_size;
        l.page_shift = __builtin_ctz((unsigned)page_size);
        return l;
    }
};

// The device that work on `stream` goes to is the current one, and the one that memory is on.
static int check_device(int device, void *stream) {
    int now = 0, of = 0;
    L2_HIP(hipGetDevice(&now));
    if (device >= 0 && now != device) return l2_fail(L2_ERR_ARG, "the pool is on device %d, the current one is %d", device, now);
    if (stream) {
        L2_HIP(hipStreamGetDevice((hipStream_t)stream, &of));
        if (of != now) return l2_fail(L2_ERR_ARG, "the stream is on device %d, the current one is %d", of, now);
    }
    l2_pass_by(now);
    return L2_OK;
}

static int check_type(int type) {
    if (type != L2_F32 && type != L2_F16 && type != L2_BF16) return l2_fail(L2_ERR_ARG, "type %d (L2_F32, L2_F16 or L2_BF16)", type);
    return L2_OK;
}
static int type_size(int type) { return type == L2_F32 ? 4 : 2; }

static int check_aligned(const void *p, int type, const char *what) {
    if (reinterpret_cast<uintptr_t>(p) % type_size(type)) return l2_fail(L2_ERR_ARG, "%s is not aligned to %d bytes", what, type_size(type));
    return L2_OK;
}
static int check_words(std::initializer_list<const void *> arrays) { // of 32-bit numbers, or absent
    for (const void *p : arrays)
        if (reinterpret_cast<uintptr_t>(p) % 4) return l2_fail(L2_ERR_ARG, "an array of 32-bit numbers at %p", p);
    return L2_OK;
}

// Rows of `width` values, `*stride` apart.
static int check_stride(int64_t *stride, int64_t width, const char *what) {
    if (*stride == 0) *stride = width;
    if (*stride < width || *stride > (int64_t)1 << 40) return l2_fail(L2_ERR_ARG, "%s %lld, rows have %lld values", what, (long long)*stride, (long long)width);
    return L2_OK;
}

extern "C" int l2_kvpool_create(int n_layers, int n_pages, int page_size, int n_kv_heads, int head_size, int kv_type, l2_kvpool **out) {
    if (!out) return l2_fail(L2_ERR_ARG, "null argument");
    *out = nullptr;
    if (n_layers < 1 || n_pages < 1 || n_kv_heads < 1 || n_kv_heads > 65535)
        return l2_fail(L2_ERR_ARG, "pool of %d layers, %d pages, %d kv heads", n_layers, n_pages, n_kv_heads);
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return l2_fail(L2_ERR_ARG, "page size %d (16, 32, 64, 128 or 256)", page_size);
    if (head_size != 64 && head_size != 128) return l2_fail(L2_ERR_ARG, "head size %d (64 or 128)", head_size);
    if (kv_type < L2_KV_I8 || kv_type > L2_KV_BF16) return l2_fail(L2_ERR_ARG, "kv type %d", kv_type);
    const bool eight = kv_type <= L2_KV_E4M3;
    const size_t rows = (size_t)n_pages * page_size * n_kv_heads; // below 2^31 * 2^8 * 2^16
    constexpr size_t kMost = ((size_t)1 << 44) - 1;
    if (rows > kMost || (size_t)n_layers > kMost / rows) return l2_fail(L2_ERR_RANGE, "a pool of more than 2^44 rows");
    int n = 0;
    const hipError_t e = hipGetDeviceCount(&n);
    if (e != hipSuccess || n < 1) {
        (void)hipGetLastError();
        return l2_fail(L2_ERR_HIP, "no HIP device available (%s)", e == hipSuccess ? "count is 0" : hipGetErrorString(e));
    }
    L2_TRY(kv_rows_warm_up());
    L2_TRY(kv_attention_warm_up());
    L2_TRY(sample_warm_up());
    l2_kvpool *p = new (std::nothrow) l2_kvpool();
    if (!p) return l2_fail(L2_ERR_HIP, "out of host memory");
    p->n_layers = n_layers, p->n_pages = n_pages, p->page_size = page_size, p->n_kv_heads = n_kv_heads, p->head_size = head_size, p->type = kv_type;
    p->cells = rows * head_size * (eight ? 1 : 2);
    p->scales = eight ? rows * 4 : 0;
    hipError_t err = hipGetDevice(&p->device);
    void *base = nullptr;
    if (err == hipSuccess) err = hipMalloc(&base, p->bytes());
    p->base = (char *)base;
    if (err == hipSuccess) err = hipMemset(base, 0, p->bytes());
    if (err == hipSuccess) err = hipDeviceSynchronize();
    if (err != hipSuccess) {
        const size_t bytes = p->bytes();
        if (base) (void)hipFree(base);
        delete p;
        (void)hipGetLastError();
        return l2_fail(L2_ERR_HIP, "pool of %zu bytes: %s", bytes, hipGetErrorString(err));
    }
    *out = p;
    return L2_OK;
}

extern "C" void l2_kvpool_free(l2_kvpool *p) {
    if (!p) return;
    if (p->base) (void)hipFree(p->base); // waits for the device
    delete p;
}

extern "C" size_t l2_kvpool_bytes(const l2_kvpool *p) { return p ? p->bytes() : 0; }

static int check_batch(const l2_kvpool *p, const l2_kvbatch *b) {
    if (!p || !b) return l2_fail(L2_ERR_ARG, "null argument");
    if (b->n_seqs < 0 || b->n_seqs > 65535 || b->max_pages < 0 || b->n_rows < 0 || b->max_rows < 0 || b->max_length < 0)
        return l2_fail(L2_ERR_ARG, "batch of %d sequences (up to 65535), %d rows, limits %d pages, %d rows, %d positions", b->n_seqs, b->n_rows, b->max_pages,
                       b->max_rows, b->max_length);
    if (b->n_rows > 1 << 22) return l2_fail(L2_ERR_RANGE, "%d rows (up to 2^22)", b->n_rows);
    if (b->max_length > 1 << 30) return l2_fail(L2_ERR_RANGE, "%d positions (up to 2^30)", b->max_length);
    if ((int64_t)b->max_length > (int64_t)b->max_pages * p->page_size)
        return l2_fail(L2_ERR_ARG, "%d positions do not fit %d pages of %d", b->max_length, b->max_pages, p->page_size);
    if (b->n_seqs && (!b->starts || !b->lengths || (b->max_pages && !b->pages))) return l2_fail(L2_ERR_ARG, "null argument");
    return check_words({b->starts, b->lengths, b->pages});
}

static int check_layer(const l2_kvpool *p, int layer) {
    if (layer < 0 || layer >= p->n_layers) return l2_fail(L2_ERR_RANGE, "layer %d of %d", layer, p->n_layers);
    return L2_OK;
}

static int rows_call(l2_kvpool *p, int layer, const l2_kvbatch *batch, const void *k, const void *v, int type, int64_t k_stride, int64_t v_stride,
                     void *stream, bool write) {
    L2_TRY(check_batch(p, batch));
    L2_TRY(check_layer(p, layer));
    L2_TRY(check_type(type));
    const int64_t width = (int64_t)p->n_kv_heads * p->head_size;
    KvRows rows{k, v, k_stride, v_stride, type};
    L2_TRY(check_stride(&rows.k_stride, width, "k_stride"));
    L2_TRY(check_stride(&rows.v_stride, width, "v_stride"));
    if (batch->n_seqs == 0 || batch->n_rows == 0 || batch->max_rows == 0) return L2_OK;
    if (!k || !v) return l2_fail(L2_ERR_ARG, "null argument");
    L2_TRY(check_aligned(k, type, "k"));
    L2_TRY(check_aligned(v, type, "v"));
    L2_TRY(check_device(p->device, stream));
    return (write ? kv_write_launch : kv_read_launch)(p->layer(layer), p->type, *batch, rows, (hipStream_t)stream);
}

extern "C" int l2_kvpool_write(l2_kvpool *p, int layer, const l2_kvbatch *batch, const void *k_dev, const void *v_dev, int type, int64_t k_stride,
                               int64_t v_stride, void *hip_stream) {
    return rows_call(p, layer, batch, k_dev, v_dev, type, k_stride, v_stride, hip_stream, true);
}

extern "C" int l2_kvpool_read(l2_kvpool *p, int layer, const l2_kvbatch *batch, void *k_dev, void *v_dev, int type, int64_t k_stride,
                              int64_t v_stride, void *hip_stream) {
    return rows_call(p, layer, batch, k_dev, v_dev, type, k_stride, v_stride, hip_stream, false);
}

static int check_attention(const l2_kvpool *p, const l2_kvbatch *batch, const l2_attention *a, KvAttention *out, KvAttnPlan *plan) {
    L2_TRY(check_batch(p, batch));
    if (!a) return l2_fail(L2_ERR_ARG, "null argument");
    L2_TRY(check_type(a->type));
    if (a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % p->n_kv_heads)
        return l2_fail(L2_ERR_ARG, "%d query heads over %d kv heads", a->n_heads, p->n_kv_heads);
    if ((int64_t)batch->n_rows * (a->n_heads / p->n_kv_heads) > 1 << 30)
        return l2_fail(L2_ERR_RANGE, "%d rows of %d query heads to a kv head (up to 2^30 together)", batch->n_rows, a->n_heads / p->n_kv_heads);
    if (!(a->scale >= 0.f && a->scale < INFINITY)) return l2_fail(L2_ERR_ARG, "scale %g", (double)a->scale);
    if (a->window < 0 || a->sinks < 0) return l2_fail(L2_ERR_ARG, "window %d, sinks %d", a->window, a->sinks);
    *out = KvAttention{};
    out->n_heads = a->n_heads, out->type = a->type, out->window = a->window, out->sinks = a->sinks;
    out->scale = a->scale > 0.f ? a->scale : 1.f / sqrtf((float)p->head_size);
    out->q_stride = a->q_stride, out->out_stride = a->out_stride;
    const int64_t width = (int64_t)a->n_heads * p->head_size;
    L2_TRY(check_stride(&out->q_stride, width, "q_stride"));
    L2_TRY(check_stride(&out->out_stride, width, "out_stride"));
    kv_attention_plan(p->layer(0), p->type, *batch, *out, plan);
    return L2_OK;
}

extern "C" int l2_kvpool_attention_workspace(const l2_kvpool *p, const l2_kvbatch *batch, const l2_attention *a, size_t *bytes) {
    if (!bytes) return l2_fail(L2_ERR_ARG, "null argument");
    KvAttention at;
    KvAttnPlan plan{};
    L2_TRY(check_attention(p, batch, a, &at, &plan));
    *bytes = plan.workspace;
    return L2_OK;
}

extern "C" int l2_kvpool_attention(l2_kvpool *p, int layer, const l2_kvbatch *batch, const l2_attention *a, const void *q_dev, void *out_dev,
                                   void *workspace_dev, size_t workspace_bytes, void *hip_stream) {
    KvAttention at;
    KvAttnPlan plan{};
    L2_TRY(check_attention(p, batch, a, &at, &plan));
    L2_TRY(check_layer(p, layer));
    if (batch->n_seqs == 0 || batch->n_rows == 0 || batch->max_rows == 0) return L2_OK;
    if (!q_dev || !out_dev) return l2_fail(L2_ERR_ARG, "null argument");
    L2_TRY(check_aligned(q_dev, a->type, "q"));
    L2_TRY(check_aligned(out_dev, a->type, "out"));
    if (q_dev == out_dev && at.q_stride != at.out_stride)
        return l2_fail(L2_ERR_ARG, "out is q, %lld and %lld from row to row", (long long)at.out_stride, (long long)at.q_stride);
    if (plan.workspace && (!workspace_dev || workspace_bytes < plan.workspace || reinterpret_cast<uintptr_t>(workspace_dev) % 16))
        return l2_fail(L2_ERR_ARG, "workspace of %zu bytes at %p (%zu wanted, aligned to 16)", workspace_bytes, workspace_dev, plan.workspace);
    L2_TRY(check_device(p->device, hip_stream));
    at.q = q_dev, at.out = out_dev;
    return kv_attention_launch(p->layer(layer), p->type, *batch, at, plan, workspace_dev, (hipStream_t)hip_stream);
}

extern "C" int l2_sample_device(const void *logits_dev, int type, int rows, int vocab, int64_t stride, const l2_sampling *s, int32_t *ids_dev,
                                void *hip_stream) {
    if (!s) return l2_fail(L2_ERR_ARG, "null argument");
    L2_TRY(check_type(type));
    if (rows < 0 || vocab < 1 || vocab > kMaxVocab) return l2_fail(L2_ERR_ARG, "%d rows of %d logits (up to 2^19)", rows, vocab);
    if (rows > 1 << 21) return l2_fail(L2_ERR_RANGE, "%d rows (up to 2^21)", rows); // blocks of 2^10 threads, of which a launch has fewer than 2^32
    L2_TRY(check_stride(&stride, vocab, "stride"));
    if (rows == 0) return L2_OK;
    if (!logits_dev || !ids_dev || !s->u) return l2_fail(L2_ERR_ARG, "null argument");
    L2_TRY(check_aligned(logits_dev, type, "logits"));
    L2_TRY(check_words({s->temperature, s->top_k, s->top_p, s->min_p, s->u, ids_dev}));
    L2_TRY(check_device(-1, hip_stream));
    SampleSettings how{};
    how.temperature = s->temperature, how.top_k = s->top_k, how.top_p = s->top_p, how.min_p = s->min_p, how.u = s->u;
    how.temperature0 = 1.f, how.top_p0 = 1.f;
    return sample_launch(logits_dev, type, rows, vocab, stride, how, ids_dev, (hipStream_t)hip_stream);
}
