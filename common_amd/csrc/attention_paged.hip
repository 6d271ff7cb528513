// Causal attention of chunks of new tokens over a paged cache (include/ar_pages.h).
#include <cmath>

#include "page_common.h"

namespace {

struct PagedParams {
    const void* q;
    void* out;
    const char *kp, *vp;  // pools at the call's layer
    const int *table, *seq, *start, *at;
    int heads, kv_heads, seqs, max_pages, pages, shift, n, rows;
    float scale;          // log2(e) / sqrt(head_dim)
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float* p, float v) { *p = v; }
__device__ __forceinline__ void from_f(__hip_bfloat16* p, float v) {
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)bf16_rne_bits(v);
}

// One wavefront per (row, head): a lane takes a key of 64 for the scores and hd / 64 dims for the products.
template <int HD, typename QT, typename KT>
__global__ __launch_bounds__(256) void attention_paged_kernel(PagedParams p) {
    __shared__ float s_q[4][HD], s_p[4][64];
    __shared__ int s_page[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int head = blockIdx.y * 4 + wave, row = blockIdx.x;
    const int chunk = chunk_of_row(p.start, p.n, p.rows, row);
    if (chunk < 0 || head >= p.heads) return;
    int first, count;
    chunk_rows(p.start, chunk, p.rows, &first, &count);
    const int seq = p.seq ? p.seq[chunk] : chunk, pos = cache_row(p.at[chunk], row - first);
    const int kvh = head / (p.heads / p.kv_heads);
    const QT* q = (const QT*)p.q + ((size_t)row * p.heads + head) * HD;
    for (int d = lane; d < HD; d += 64) s_q[wave][d] = to_f(q[d]) * p.scale;
    float m = -INFINITY, l = 0.f, o[HD / 64] = {};
    const int end = min(pos + 1LL, (long long)p.max_pages << p.shift);
    for (int k0 = 0; k0 < end; k0 += 64) {
        const int key = k0 + lane;
        const int page = key < end ? page_of_row(p.table, p.seqs, p.max_pages, p.pages, p.shift, seq, key) : -1;
        float s = -INFINITY;
        if (page >= 0) {
            const KT* k = (const KT*)p.kp + ((((size_t)page * p.kv_heads + kvh) << p.shift) + (key & ((1 << p.shift) - 1))) * HD;
            s = 0.f;
            for (int d = 0; d < HD; d++) s = fmaf(s_q[wave][d], to_f(k[d]), s);
        }
        float mx = s;
        for (int d = 32; d; d /= 2) mx = fmaxf(mx, __shfl_xor(mx, d));
        const float mn = fmaxf(m, mx), a = m == mn ? 1.f : m == -INFINITY ? 0.f : exp2f(m - mn);
        const float w = page < 0 ? 0.f : exp2f(s - mn);
        float sum = w;
        for (int d = 32; d; d /= 2) sum += __shfl_xor(sum, d);
        l = l * a + sum;
        m = mn;
        s_p[wave][lane] = w;
        s_page[wave][lane] = page;
        for (int i = 0; i < HD / 64; i++) o[i] *= a;
        for (int j = 0; j < 64; j++) {
            const int pg = s_page[wave][j];
            if (pg < 0) continue;
            const KT* v = (const KT*)p.vp + ((((size_t)pg * p.kv_heads + kvh) << p.shift) + ((k0 + j) & ((1 << p.shift) - 1))) * HD;
            for (int i = 0; i < HD / 64; i++) o[i] = fmaf(s_p[wave][j], to_f(v[lane + 64 * i]), o[i]);
        }
    }
    QT* out = (QT*)p.out + ((size_t)row * p.heads + head) * HD;
    for (int i = 0; i < HD / 64; i++) from_f(out + lane + 64 * i, l > 0.f || l != l ? o[i] / l : 0.f);
}

template <int HD, typename QT>
void launch_kt(int dtype, const PagedParams& p, hipStream_t st) {
    const dim3 grid(p.rows, (p.heads + 3) / 4), block(256);
    if (dtype == AR_DTYPE_F32) hipLaunchKernelGGL((attention_paged_kernel<HD, QT, float>), grid, block, 0, st, p);
    else if (dtype == AR_DTYPE_F16) hipLaunchKernelGGL((attention_paged_kernel<HD, QT, _Float16>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((attention_paged_kernel<HD, QT, __hip_bfloat16>), grid, block, 0, st, p);
}

int check_attention(const ar_pages* pages, const ar_chunks* chunks, int heads, const char* what) {
    AR_TRY(page_check(pages, true, what));
    AR_TRY(page_check_chunks(pages, chunks, what));
    AR_CHECK_ARG(heads > 0 && heads <= 1 << 16 && heads % pages->kv_heads == 0, "%s: bad head counts %d/%d", what, heads,
                 pages->kv_heads);
    return AR_HIP_OK;
}
}  // namespace

extern "C" int ar_hip_attention_paged_work(ar_hip_ctx* ctx, const ar_pages* pages, const ar_chunks* chunks, int heads,
                                           size_t* bytes) {
    AR_TRY(check_attention(pages, chunks, heads, "paged attention work"));
    AR_CHECK_ARG(bytes, "paged attention work: bytes is null");
    AR_CHECK_ARG(ctx, "ctx is null");
    *bytes = 16;
    return AR_HIP_OK;
}

extern "C" int ar_hip_attention_paged(ar_hip_ctx* ctx, const ar_pages* pages, int layer, const ar_chunks* chunks,
                                      const void* q, int act_dtype, int heads, void* out, void* work,
                                      size_t work_bytes) {
    const char* what = "paged attention";
    AR_TRY(check_attention(pages, chunks, heads, what));
    AR_CHECK_ARG(layer >= 0 && layer < pages->layers, "%s: layer %d of %d", what, layer, pages->layers);
    AR_CHECK_ARG(q && out, "%s: null queries or output", what);
    AR_CHECK_ARG(act_dtype == AR_DTYPE_F32 || act_dtype == AR_DTYPE_BF16, "%s: unknown activation dtype %d", what, act_dtype);
    AR_CHECK_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15) == 0, "%s: pointers must be 16-byte aligned", what);
    AR_CHECK_ARG(ctx, "ctx is null");
    if (chunks->rows == 0) return AR_HIP_OK;
    const int hd = pages->head_dim;
    const size_t act = act_dtype == AR_DTYPE_F32 ? 4 : 2, bytes = (size_t)chunks->rows * heads * hd * act;
    if (ar_check_ptrs_enabled()) {
        AR_TRY(page_check_ranges(pages, what));
        AR_TRY(page_check_chunk_ranges(chunks, what));
        AR_TRY(ar_check_range(q, bytes, what, "queries"));
        AR_TRY(ar_check_range(out, bytes, what, "output"));
    }
    const size_t layer_bytes = (size_t)pages->pages * pages->kv_heads * hd * pages->page_rows * page_elem_bytes(pages->dtype);
    PagedParams p;
    p.q = q; p.out = out;
    p.kp = (const char*)pages->k + layer * layer_bytes;
    p.vp = (const char*)pages->v + layer * layer_bytes;
    p.table = pages->table; p.seq = chunks->seq; p.start = chunks->start; p.at = chunks->at; p.heads = heads;
    p.kv_heads = pages->kv_heads; p.seqs = pages->seqs; p.max_pages = pages->max_pages; p.pages = pages->pages;
    p.shift = page_shift_of(pages); p.n = chunks->n; p.rows = chunks->rows;
    p.scale = (float)(1.4426950408889634 / std::sqrt((double)hd));
    if (hd == 128) {
        if (act == 4) launch_kt<128, float>(pages->dtype, p, ctx->stream);
        else launch_kt<128, __hip_bfloat16>(pages->dtype, p, ctx->stream);
    } else {
        if (act == 4) launch_kt<64, float>(pages->dtype, p, ctx->stream);
        else launch_kt<64, __hip_bfloat16>(pages->dtype, p, ctx->stream);
    }
    AR_LAUNCH_CHECK();
    return AR_HIP_OK;
}
