// Rows of new tokens on their way into a paged cache: QK-norm, rotary positions, page stores (include/ar_pages.h).
//
//   y = g * x / sqrt(mean(x^2) + eps)                 over each head, or over all heads of a row
//   z[f]          = y[f] cos a - y[f + hd/2] sin a     a = position[axis(f)] * theta^(-2f/hd)
//   z[f + hd/2]   = y[f] sin a + y[f + hd/2] cos a
//
// Bound by HBM: a row is read once (fp32) and its queries, keys and values are written once.  One block per row; a
// thread holds the dims f .. f+3 and f + hd/2 .. +3 of a head, so a 16-byte load each feeds its four rotations, a head
// is hd / 8 lanes of one wavefront, and its norm is a reduction within them.  Angles: hd / 2 per row and not per head,
// computed by the block's first threads in double (a position times a frequency, less whole turns) and shared in LDS.
// Measured: 6,958 rows of 16 / 8 heads of 128 to bf16 (171 MB) 31 us, 5.5 TB/s; a decode step of 8 rows 5 us, a launch
// and its chain of loads (chunk, page, angles).
#include <cmath>

#include "page_common.h"

namespace {

struct WriteParams {
    const float *q, *k, *v;
    const float *q_norm, *k_norm;
    void *q_out, *kp, *vp;   // pools at the call's layer
    const int *table, *seq, *start, *at, *positions;
    int q_stride, kv_stride, heads, kv_heads;
    int seqs, max_pages, pages, shift, n, rows;
    int axes;
    float eps;
    int per_head;
    unsigned char axis[64];  // of each frequency
    double inv[64];          // theta^(-2f/hd)
};

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v);
template <>
__device__ __forceinline__ void store4<float>(float* p, float4 v) {
    *reinterpret_cast<float4*>(p) = v;
}
template <>
__device__ __forceinline__ void store4<__hip_bfloat16>(__hip_bfloat16* p, float4 v) {
    const uint2 u = make_uint2(bf16_rne_bits(v.x) | bf16_rne_bits(v.y) << 16, bf16_rne_bits(v.z) | bf16_rne_bits(v.w) << 16);
    *reinterpret_cast<uint2*>(p) = u;
}
template <>
__device__ __forceinline__ void store4<_Float16>(_Float16* p, float4 v) {
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    half4 h = {(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w};
    *reinterpret_cast<half4*>(p) = h;
}

// sum over the LPH (8 or 16) lanes that hold a head
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
    v += dpp_mov<0xB1, 0xF>(v);
    v += dpp_mov<0x4E, 0xF>(v);
    v += dpp_mov<0x141, 0xF>(v);  // the other quad of the half row
    if (LPH == 16) v += dpp_mov<0x140, 0xF>(v);
    return v;
}

__device__ __forceinline__ float sum4(float4 a) { return (a.x * a.x + a.y * a.y) + (a.z * a.z + a.w * a.w); }

constexpr int kWriteThreads = 256;

template <int HD, typename QT, typename KT>
__global__ __launch_bounds__(kWriteThreads) void write_rows_kernel(WriteParams p) {
    constexpr int LPH = HD / 8;                  // lanes of a head
    constexpr int HPB = kWriteThreads / LPH;     // heads a block holds at once
    constexpr int HALF = HD / 2;
    __shared__ float s_cos[HALF], s_sin[HALF], s_sum[2][kWriteThreads / 64];
    const int row = blockIdx.x, tid = threadIdx.x;
    const int chunk = chunk_of_row(p.start, p.n, p.rows, row);
    if (chunk < 0) return;
    int first, count;
    chunk_rows(p.start, chunk, p.rows, &first, &count);
    const int seq = p.seq ? p.seq[chunk] : chunk;
    const int at = cache_row(p.at[chunk], row - first);
    int page = page_of_row(p.table, p.seqs, p.max_pages, p.pages, p.shift, seq, at);
    if (p.seq) {
        bool before = false;
        for (int j = tid; j < chunk; j += kWriteThreads) before |= p.seq[j] == seq;
        if (__syncthreads_or(before)) page = -1;
    }
    if (page < 0 && !p.q) return;

    for (int f = tid; f < HALF; f += kWriteThreads) {
        const int pos = p.positions ? p.positions[(size_t)p.axis[f] * p.rows + row] : at < 0 ? 0 : at;
        const double a = pos * p.inv[f];
        // less whole turns, 2 pi in two parts: the angle's own rounding is all that is lost
        const double turns = rint(a * 0.15915494309189535);
        const float r = (float)fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, a));
        s_cos[f] = cosf(r);
        s_sin[f] = sinf(r);
    }

    const int lh = tid % LPH, hb = tid / LPH, f0 = 4 * lh;
    float qs = 0.f, ks = 0.f;
    if (!p.per_head) {  // whole-vector sums ahead of the rotations
        if (p.q_norm && p.q)
            for (int h = hb; h < p.heads; h += HPB) {
                const float* x = p.q + (size_t)row * p.q_stride + h * HD + f0;
                qs += sum4(*reinterpret_cast<const float4*>(x)) + sum4(*reinterpret_cast<const float4*>(x + HALF));
            }
        if (p.k_norm)
            for (int h = hb; h < p.kv_heads; h += HPB) {
                const float* x = p.k + (size_t)row * p.kv_stride + h * HD + f0;
                ks += sum4(*reinterpret_cast<const float4*>(x)) + sum4(*reinterpret_cast<const float4*>(x + HALF));
            }
        qs = wave_sum_lane63(qs);
        ks = wave_sum_lane63(ks);
        if ((tid & 63) == 63) {
            s_sum[0][tid >> 6] = qs;
            s_sum[1][tid >> 6] = ks;
        }
    }
    __syncthreads();
    if (!p.per_head) {
        qs = (s_sum[0][0] + s_sum[0][1]) + (s_sum[0][2] + s_sum[0][3]);
        ks = (s_sum[1][0] + s_sum[1][1]) + (s_sum[1][2] + s_sum[1][3]);
        qs = 1.f / sqrtf(qs / (p.heads * HD) + p.eps);
        ks = 1.f / sqrtf(ks / (p.kv_heads * HD) + p.eps);
    }
    const float4 c = *reinterpret_cast<const float4*>(&s_cos[f0]), s = *reinterpret_cast<const float4*>(&s_sin[f0]);

    auto turned = [&](const float* x, const float* g, float scale, float4* lo, float4* hi) __attribute__((always_inline)) {
        float4 a = *reinterpret_cast<const float4*>(x), b = *reinterpret_cast<const float4*>(x + HALF);
        if (g) {
            if (p.per_head) scale = 1.f / sqrtf(head_sum<LPH>(sum4(a) + sum4(b)) / HD + p.eps);
            const float4 ga = *reinterpret_cast<const float4*>(g), gb = *reinterpret_cast<const float4*>(g + HALF);
            a = make_float4(ga.x * a.x * scale, ga.y * a.y * scale, ga.z * a.z * scale, ga.w * a.w * scale);
            b = make_float4(gb.x * b.x * scale, gb.y * b.y * scale, gb.z * b.z * scale, gb.w * b.w * scale);
        }
        *lo = make_float4(a.x * c.x - b.x * s.x, a.y * c.y - b.y * s.y, a.z * c.z - b.z * s.z, a.w * c.w - b.w * s.w);
        *hi = make_float4(a.x * s.x + b.x * c.x, a.y * s.y + b.y * c.y, a.z * s.z + b.z * c.z, a.w * s.w + b.w * c.w);
    };
    if (p.q)
        for (int h = hb; h < p.heads; h += HPB) {
            float4 lo, hi;
            turned(p.q + (size_t)row * p.q_stride + h * HD + f0, p.q_norm ? p.q_norm + h * HD + f0 : nullptr, qs, &lo, &hi);
            QT* o = (QT*)p.q_out + ((size_t)row * p.heads + h) * HD + f0;
            store4<QT>(o, lo);
            store4<QT>(o + HALF, hi);
        }
    if (page < 0) return;
    const int in_page = at & ((1 << p.shift) - 1);
    for (int h = hb; h < p.kv_heads; h += HPB) {
        float4 lo, hi;
        turned(p.k + (size_t)row * p.kv_stride + h * HD + f0, p.k_norm ? p.k_norm + h * HD + f0 : nullptr, ks, &lo, &hi);
        const float* x = p.v + (size_t)row * p.kv_stride + h * HD + f0;
        const size_t cell = ((((size_t)page * p.kv_heads + h) << p.shift) + in_page) * HD + f0;
        KT *ko = (KT*)p.kp + cell, *vo = (KT*)p.vp + cell;
        store4<KT>(ko, lo);
        store4<KT>(ko + HALF, hi);
        store4<KT>(vo, *reinterpret_cast<const float4*>(x));
        store4<KT>(vo + HALF, *reinterpret_cast<const float4*>(x + HALF));
    }
}

template <int HD, typename QT>
void launch_kt(int dtype, const WriteParams& p, hipStream_t st) {
    const dim3 grid(p.rows), block(kWriteThreads);
    if (dtype == AR_DTYPE_F32) hipLaunchKernelGGL((write_rows_kernel<HD, QT, float>), grid, block, 0, st, p);
    else if (dtype == AR_DTYPE_F16) hipLaunchKernelGGL((write_rows_kernel<HD, QT, _Float16>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((write_rows_kernel<HD, QT, __hip_bfloat16>), grid, block, 0, st, p);
}
}  // namespace

extern "C" int ar_hip_pages_write(ar_hip_ctx* ctx, const ar_pages* pages, int layer, const ar_chunks* chunks,
                                  const float* q, const float* k, const float* v, int q_stride, int kv_stride, int heads,
                                  const float* q_norm, const float* k_norm, float qk_eps, int qk_norm_mode,
                                  const ar_rotary* rotary, void* q_out, int act_dtype) {
    const char* what = "pages write";
    AR_TRY(page_check(pages, true, what));
    AR_TRY(page_check_chunks(pages, chunks, what));
    AR_CHECK_ARG(layer >= 0 && layer < pages->layers, "%s: layer %d of %d", what, layer, pages->layers);
    AR_CHECK_ARG(k && v, "%s: null keys or values", what);
    AR_CHECK_ARG(!q == !q_out, "%s: queries need both q and q_out", what);
    AR_CHECK_ARG(act_dtype == AR_DTYPE_F32 || act_dtype == AR_DTYPE_BF16, "%s: unknown activation dtype %d", what, act_dtype);
    AR_CHECK_ARG(heads > 0 && heads <= 1 << 16 && heads % pages->kv_heads == 0, "%s: bad head counts %d/%d", what, heads,
                 pages->kv_heads);
    AR_CHECK_ARG(qk_norm_mode == AR_QK_NORM_WHOLE || qk_norm_mode == AR_QK_NORM_PER_HEAD, "%s: bad qk-norm mode", what);
    const int hd = pages->head_dim, kv = pages->kv_heads * hd;
    AR_CHECK_ARG(kv_stride >= kv && kv_stride % 4 == 0, "%s: kv_stride %d is below %d or no multiple of 4", what, kv_stride, kv);
    AR_CHECK_ARG(!q || (q_stride >= heads * hd && q_stride % 4 == 0), "%s: q_stride %d is below %d or no multiple of 4",
                 what, q_stride, heads * hd);
    AR_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)q_out) & 15) == 0,
                 "%s: pointers must be 16-byte aligned", what);
    AR_CHECK_ARG(!q || (const void*)q != q_out || (act_dtype == AR_DTYPE_F32 && q_stride == heads * hd),
                 "%s: queries in place need fp32 rows of heads * head_dim", what);
    AR_CHECK_ARG(rotary && rotary->axes >= 1 && rotary->axes <= 4, "%s: 1 to 4 rotary axes", what);
    AR_CHECK_ARG(rotary->theta > 0 && std::isfinite(rotary->theta), "%s: theta must be positive", what);
    AR_CHECK_ARG(rotary->layout == AR_ROPE_SECTIONS || rotary->layout == AR_ROPE_INTERLEAVED, "%s: unknown rotary layout %d",
                 what, rotary->layout);
    WriteParams p{};
    int sum = 0;
    for (int a = 0; a < rotary->axes; a++) {
        const int have = rotary->section[a];
        AR_CHECK_ARG(have >= 0 && have <= hd / 2, "%s: rotary section %d of %d frequencies", what, a, have);
        AR_CHECK_ARG(rotary->layout == AR_ROPE_SECTIONS || a == 0 || have <= (hd / 2 - a + rotary->axes - 1) / rotary->axes,
                     "%s: rotary section %d of %d frequencies does not fit its interleaving", what, a, have);
        sum += have;
    }
    AR_CHECK_ARG(sum == hd / 2, "%s: rotary sections add up to %d, not %d", what, sum, hd / 2);
    for (int f = 0, a = 0, left = rotary->section[0]; f < hd / 2; f++) {
        if (rotary->layout == AR_ROPE_INTERLEAVED) {
            const int own = f % rotary->axes;
            p.axis[f] = f / rotary->axes < rotary->section[own] ? own : 0;
        } else {
            while (left == 0) left = rotary->section[++a];
            p.axis[f] = a;
            left--;
        }
        p.inv[f] = std::pow(rotary->theta, -2.0 * f / hd);
    }
    AR_CHECK_ARG(ctx, "ctx is null");
    if (chunks->rows == 0) return AR_HIP_OK;
    const size_t R = chunks->rows, act = act_dtype == AR_DTYPE_F32 ? 4 : 2;
    if (ar_check_ptrs_enabled()) {
        AR_TRY(page_check_ranges(pages, what));
        AR_TRY(page_check_chunk_ranges(chunks, what));
        if (q) AR_TRY(ar_check_range(q, ((R - 1) * q_stride + (size_t)heads * hd) * 4, what, "q rows"));
        AR_TRY(ar_check_range(k, ((R - 1) * kv_stride + kv) * 4, what, "k rows"));
        AR_TRY(ar_check_range(v, ((R - 1) * kv_stride + kv) * 4, what, "v rows"));
        AR_TRY(ar_check_range(q_norm, (size_t)heads * hd * 4, what, "q norm gain"));
        AR_TRY(ar_check_range(k_norm, (size_t)kv * 4, what, "k norm gain"));
        AR_TRY(ar_check_range(rotary->positions, R * rotary->axes * 4, what, "positions"));
        AR_TRY(ar_check_range(q_out, R * heads * hd * act, what, "query output"));
    }
    const size_t layer_bytes = (size_t)pages->pages * kv * pages->page_rows * page_elem_bytes(pages->dtype);
    p.q = q; p.k = k; p.v = v; p.q_norm = q_norm; p.k_norm = k_norm; p.q_out = q_out;
    p.kp = (char*)pages->k + layer * layer_bytes;
    p.vp = (char*)pages->v + layer * layer_bytes;
    p.table = pages->table; p.seq = chunks->seq; p.start = chunks->start; p.at = chunks->at;
    p.positions = rotary->positions; p.q_stride = q_stride; p.kv_stride = kv_stride; p.heads = heads;
    p.kv_heads = pages->kv_heads; p.seqs = pages->seqs; p.max_pages = pages->max_pages; p.pages = pages->pages;
    p.shift = page_shift_of(pages); p.n = chunks->n; p.rows = chunks->rows; p.axes = rotary->axes; p.eps = qk_eps;
    p.per_head = qk_norm_mode == AR_QK_NORM_PER_HEAD;
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
