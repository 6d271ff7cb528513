// Rows in 8 bits: floats to 8 bits, the residual's norm on its way there, and back.
#include "i8_common.h"

namespace {

constexpr float kTiny = 0x1p-100f;  // rows below it become zeros (127 / m stays finite above)
constexpr int kLaunchRows = 1 << 20;  // rows of a launch, so that its threads are fewer than 2^32

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
__device__ inline unsigned wave_max_u32(unsigned v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const unsigned o = __shfl_xor(v, off, 64);
        v = o > v ? o : v;
    }
    return v;
}

// Sum / maximum over the wavefronts of a row, in all their threads: `red` has a place for each of them and is free again
// behind the next barrier.  One wavefront needs neither.
__device__ inline double row_sum(double v, double* red, int waves) {
    v = wave_sum_f64(v);
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < waves; i++) t += red[i];
    return t;
}
__device__ inline unsigned row_max(unsigned v, unsigned* red, int waves) {
    v = wave_max_u32(v);
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned t = 0u;
    for (int i = 0; i < waves; i++) t = red[i] > t ? red[i] : t;
    return t;
}

// 1 / sqrt(mean of squares + eps) of a row whose squares' sum is ss.  Past 2^126 that is no normal number and short of bits:
// `pre` (else 1) takes the values 2^64 times smaller first, which costs none that its product does not lose.
__device__ inline float reciprocal_root(double ss, int n, float eps, float* pre) {
    const double root = sqrt(ss / (double)n + (double)eps);
    *pre = root > 0x1p126 ? 0x1p-64f : 1.f;
    return (float)((root > 0x1p126 ? 0x1p64 : 1.0) / root);
}

// The magnitude's bits: ordered as the magnitudes are, infinities and NaN above every number.
__device__ inline unsigned magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// scale and 127 / m of a row whose largest magnitude has the bits m
__device__ inline void steps(unsigned m, float* scale, float* inv) {
    const float top = __uint_as_float(m);
    const bool finite = m < 0x7F800000u, some = top >= kTiny;
    *scale = !finite ? __uint_as_float(0x7FC00000u) : some ? top / 127.f : 0.f;
    *inv = finite && some ? 127.f / top : 0.f;
}
__device__ inline int8_t eight(float v, float inv) { return inv > 0.f ? (int8_t)(int)rintf(v * inv) : (int8_t)0; }

struct RowParams {
    void* h;          // [rows][h_stride], or null (x alone)
    const void* x;    // [rows][x_stride], or null
    void* y;          // float output, or null
    int8_t* q;        // 8-bit output, or null
    float* scale;
    const float* w;   // gain, or null (no norm)
    int64_t h_stride, x_stride, y_stride, q_stride;
    int n;
    float eps;
};

// Wide accesses to values that are aligned to their type only, which global memory allows.
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4), aligned(2)));

// Eight values from p on; of the last ones of a row (left < 8) those behind its end are zero.
template <class T>
__device__ inline void load8(const T* p, int left, float (&v)[8]) {
    if (left >= 8) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[i] = a[i];
                v[4 + i] = b[i];
            }
        } else {
            const u32x4 a = *(const u32x4*)p;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[2 * i] = __uint_as_float(a[i] << 16);
                v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < left ? to_float<T>(p[i]) : 0.f;
    }
}
template <class T>
__device__ inline void store8(T* p, int left, const float (&v)[8]) {
    if (left >= 8) {
        if constexpr (sizeof(T) == 4) {
            *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
            *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = from_float<uint16_t>(v[2 * i]) | (unsigned)from_float<uint16_t>(v[2 * i + 1]) << 16;
            *(u32x4*)p = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < left) p[i] = from_float<T>(v[i]);
    }
}
__device__ inline unsigned four(float a, float b, float c, float d, float inv) {
    return (unsigned)(uint8_t)eight(a, inv) | (unsigned)(uint8_t)eight(b, inv) << 8 | (unsigned)(uint8_t)eight(c, inv) << 16 |
           (unsigned)(uint8_t)eight(d, inv) << 24;
}

// Rows of up to 32,768 values, each read once and held in registers: threadIdx.y is the row of the block, its blockDim.x threads
// hold CHUNKS runs of eight values each.  Bound by memory: the squares' sum in double and the rounding hide behind it.
template <class HT, class XT, class YT, bool NORM, bool I8, int CHUNKS>
__global__ __launch_bounds__(1024) void held_rows_kernel(RowParams p, int row0, int rows) {
    __shared__ double red_sum[16];
    __shared__ unsigned red_max[16];
    const int r = row0 + blockIdx.x * blockDim.y + threadIdx.y, waves = blockDim.x >> 6;
    if (r >= rows) return;  // (where a block has several rows, each is one wavefront's, without barriers)
    HT* const h = NORM ? (HT*)p.h + (size_t)r * p.h_stride : nullptr;
    const XT* const x = p.x ? (const XT*)p.x + (size_t)r * p.x_stride : nullptr;
    float v[CHUNKS][8];
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
        const int i = (c * blockDim.x + threadIdx.x) * 8, left = p.n - i;
        if constexpr (NORM) {
            load8<HT>(h + i, left, v[c]);
            if (x) {
                float add[8];
                load8<XT>(x + i, left, add);
#pragma unroll
                for (int j = 0; j < 8; j++) v[c][j] += add[j];
                store8<HT>(h + i, left, v[c]);
            }
        } else {
            load8<XT>(x + i, left, v[c]);
        }
    }
    if constexpr (NORM) {
        double ss = 0.0;
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) ss = fma((double)v[c][j], (double)v[c][j], ss);
        float pre;
        const float rs = reciprocal_root(row_sum(ss, red_sum, waves), p.n, p.eps, &pre);
        if (pre != 1.f) {
#pragma unroll
            for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                for (int j = 0; j < 8; j++) v[c][j] *= pre;
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            const int i = (c * blockDim.x + threadIdx.x) * 8, left = p.n - i;
            float w[8];
            load8<float>(p.w + i, left, w);
#pragma unroll
            for (int j = 0; j < 8; j++) v[c][j] = v[c][j] * rs * w[j];
            if constexpr (!I8) store8<YT>((YT*)p.y + (size_t)r * p.y_stride + i, left, v[c]);
        }
    }
    if constexpr (I8) {
        unsigned m = 0u;
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // (a row's last runs hold zeros, which 0 / sqrt(0) makes NaN of: their magnitudes do not count)
                const unsigned a = magnitude(v[c][j]);
                const bool in = (int)((c * blockDim.x + threadIdx.x) * 8) + j < p.n;
                m = in && a > m ? a : m;
            }
        m = row_max(m, red_max, waves);
        float scale, inv;
        steps(m, &scale, &inv);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++) {
            const int i = (c * blockDim.x + threadIdx.x) * 8;
            if (i >= (p.n + 15) / 16 * 16) continue;
            const float(&u)[8] = v[c];
            *(uint2*)(p.q + (size_t)r * p.q_stride + i) =
                make_uint2(four(u[0], u[1], u[2], u[3], inv), four(u[4], u[5], u[6], u[7], inv));
        }
        if (threadIdx.x == 0) p.scale[r] = scale;
    }
}

// Longer rows, a block each: the row is read again for each of its passes (sum of squares, largest magnitude, output).
template <class HT, class XT, class YT, bool NORM, bool I8>
__global__ __launch_bounds__(256) void rows_kernel(RowParams p, int row0) {
    __shared__ double red_sum[16];
    __shared__ unsigned red_max[16];
    const size_t r = row0 + blockIdx.x;
    HT* const h = p.h ? (HT*)p.h + r * p.h_stride : nullptr;
    const XT* const x = p.x ? (const XT*)p.x + r * p.x_stride : nullptr;
    auto value = [&](int i) {
        if constexpr (!NORM) return to_float<XT>(x[i]);
        const float a = to_float<HT>(h[i]);
        return x ? a + to_float<XT>(x[i]) : a;
    };
    float rs = 1.f, pre = 1.f;
    if constexpr (NORM) {
        double ss = 0.0;
        for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float v = value(i);
            ss += (double)v * (double)v;
        }
        rs = reciprocal_root(row_sum(ss, red_sum, blockDim.x >> 6), p.n, p.eps, &pre);
    }
    auto normed = [&](int i) {
        const float v = value(i);
        return NORM ? v * pre * rs * p.w[i] : v;
    };
    if constexpr (I8) {
        unsigned m = 0u;
        for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
            const unsigned a = magnitude(normed(i));
            m = a > m ? a : m;
        }
        m = row_max(m, red_max, blockDim.x >> 6);
        float scale, inv;
        steps(m, &scale, &inv);
        int8_t* const q = p.q + r * p.q_stride;
        const int padded = (p.n + 15) / 16 * 16;
        for (int i = threadIdx.x; i < padded; i += blockDim.x) q[i] = i < p.n ? eight(normed(i), inv) : (int8_t)0;
        if (threadIdx.x == 0) p.scale[r] = scale;
    } else {
        // (y may be x: each thread reads an element of x and h before it writes there)
        YT* const y = (YT*)p.y + r * p.y_stride;
        for (int i = threadIdx.x; i < p.n; i += blockDim.x) {
            const float v = value(i), o = v * pre * rs * p.w[i];
            if (x) h[i] = from_float<HT>(v);
            y[i] = from_float<YT>(o);
        }
        return;
    }
    if constexpr (NORM) {
        if (x)
            for (int i = threadIdx.x; i < p.n; i += blockDim.x) h[i] = from_float<HT>(value(i));
    }
}

// Rows of a table by token, 16 bytes of output a thread and turn, so that a wavefront's stores lie side by side.  Bound by the
// outputs' way to memory: 8,192 rows of 2,560 to fp32 18.7 us (5.6 TB/s; by eight values a thread 27.9: two stores with gaps).
// PAST: stores past the caches, which outputs larger than them would only empty (the same by eight values 20.1 us instead of
// 27.9).
template <class YT, bool PAST>
__global__ __launch_bounds__(1024) void embed_kernel(const int8_t* q, const float* scale, int64_t stride, int table, int n,
                                                     const int32_t* tokens, int row0, int count, YT* y, int64_t y_stride) {
    constexpr int V = 16 / sizeof(YT);
    const int r = row0 + blockIdx.x * blockDim.y + threadIdx.y;
    if (r >= count) return;
    const int t = tokens ? tokens[r] : r;
    const bool in = t >= 0 && t < table;
    const float s = in ? scale[t] : 0.f;
    const int8_t* const row = q + (size_t)(in ? t : 0) * stride;
    YT* const to = y + (size_t)r * y_stride;
    for (int i = threadIdx.x * V; i < n; i += blockDim.x * V) {
        unsigned b[2] = {0u, 0u};
        if (in) {  // (rows go on to a multiple of 16)
            if constexpr (V == 4) {
                b[0] = *(const unsigned*)(row + i);
            } else {
                const uint2 w = *(const uint2*)(row + i);
                b[0] = w.x;
                b[1] = w.y;
            }
        }
        YT v[V];
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = from_float<YT>(in ? (float)(int8_t)(b[j / 4] >> (j % 4) * 8) * s : 0.f);
        if (i + V <= n) {
            u32x4 o;
            __builtin_memcpy(&o, v, 16);
            if constexpr (PAST) __builtin_nontemporal_store(o, (u32x4*)(to + i));
            else *(u32x4*)(to + i) = o;
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (i + j < n) to[i + j] = v[j];
        }
    }
}

// Threads of a row and rows of a block for rows of n values, eight a thread and run: more runs where one would take more than
// 512 threads, and four rows a block where one wavefront holds a row.  Rows of 16-bit values alone have two runs from 1,024
// values on, for as many bytes on their way as fp32 rows have (19,456 x 2,560 bf16 to 8 bits 32 us, with one run 38, four 33;
// 4,093 x 2,560 norms of bf16 16.8, 17.8 and 19.6; but 16,384 x 2,048 norms of fp32 rows 85, 74 and 87).
struct RowShape {
    int runs;
    dim3 block;
};
RowShape row_shape(int n, bool half) {
    const int eights = (n + 15) / 16 * 2;
    int runs = half && n >= 1024 ? 2 : 1;
    while (runs < 4 && (eights + runs - 1) / runs > 512) runs *= 2;
    const int threads = ((eights + runs - 1) / runs + 63) / 64 * 64;
    return RowShape{runs, dim3(threads, threads == 64 ? 4 : 1)};
}

template <class HT, class XT, class YT, bool NORM, bool I8>
int launch_rows(const RowParams& p, int rows, hipStream_t st) {
    const RowShape s = row_shape(p.n, sizeof(XT) == 2 && (!NORM || sizeof(HT) == 2));
    for (int row0 = 0; row0 < rows; row0 += kLaunchRows) {
        const int end = rows - row0 < kLaunchRows ? rows : row0 + kLaunchRows;
        const dim3 grid((end - row0 + s.block.y - 1) / s.block.y);
        if (s.block.x > 1024) {
            hipLaunchKernelGGL((rows_kernel<HT, XT, YT, NORM, I8>), dim3(end - row0), dim3(256), 0, st, p, row0);
        } else if (s.runs == 1) {
            hipLaunchKernelGGL((held_rows_kernel<HT, XT, YT, NORM, I8, 1>), grid, s.block, 0, st, p, row0, end);
        } else if (s.runs == 2) {
            hipLaunchKernelGGL((held_rows_kernel<HT, XT, YT, NORM, I8, 2>), grid, s.block, 0, st, p, row0, end);
        } else {
            hipLaunchKernelGGL((held_rows_kernel<HT, XT, YT, NORM, I8, 4>), grid, s.block, 0, st, p, row0, end);
        }
        AR_LAUNCH_CHECK();
    }
    return AR_HIP_OK;
}

template <class YT>
int launch_embed(const ar_rows_i8* table, const int32_t* tokens, int count, void* y, int64_t y_stride, hipStream_t st) {
    const int threads = ((table->n * (int)sizeof(YT) + 15) / 16 + 63) / 64 * 64;
    const dim3 block(threads < 1024 ? threads : 1024, threads == 64 ? 4 : 1);
    const bool past = (double)count * table->n * sizeof(YT) > 32e6;  // (eight XCDs' L2s hold 32 MB)
    const auto kernel = past ? embed_kernel<YT, true> : embed_kernel<YT, false>;
    for (int row0 = 0; row0 < count; row0 += kLaunchRows) {
        const int end = count - row0 < kLaunchRows ? count : row0 + kLaunchRows;
        hipLaunchKernelGGL(kernel, dim3((end - row0 + block.y - 1) / block.y), block, 0, st, table->q, table->scale,
                           table->stride, table->rows, table->n, tokens, row0, end, (YT*)y, y_stride);
        AR_LAUNCH_CHECK();
    }
    return AR_HIP_OK;
}

template <class HT, class XT>
int launch_norm(const RowParams& p, int y_dtype, int rows, hipStream_t st) {
    if (p.q) return launch_rows<HT, XT, float, true, true>(p, rows, st);
    return y_dtype == AR_DTYPE_F32 ? launch_rows<HT, XT, float, true, false>(p, rows, st)
                                   : launch_rows<HT, XT, uint16_t, true, false>(p, rows, st);
}

int launch_norm_types(const RowParams& p, int h_dtype, int x_dtype, int y_dtype, int rows, hipStream_t st) {
    const bool h32 = h_dtype == AR_DTYPE_F32, x32 = x_dtype == AR_DTYPE_F32;
    if (h32) return x32 ? launch_norm<float, float>(p, y_dtype, rows, st) : launch_norm<float, uint16_t>(p, y_dtype, rows, st);
    return x32 ? launch_norm<uint16_t, float>(p, y_dtype, rows, st) : launch_norm<uint16_t, uint16_t>(p, y_dtype, rows, st);
}

// Checks of the arguments that both norms have.
int norm_check(const void* h, int h_dtype, int h_stride, const void* x, int x_dtype, int x_stride, const float* w,
               float eps, int rows, int n, const char* what) {
    AR_TRY(float_rows_check(h, h_dtype, h_stride, rows, n, what, "h"));
    if (x) AR_TRY(float_rows_check(x, x_dtype, x_stride, rows, n, what, "x"));
    AR_CHECK_ARG(w, "%s: the gain is null", what);
    AR_CHECK_ARG(aligned_to(w, 4), "%s: the gain is not aligned to its type", what);
    AR_CHECK_ARG(eps >= 0.f && eps < INFINITY, "%s: eps %g", what, eps);
    return AR_HIP_OK;
}

int norm_ranges(const void* h, int h_dtype, int h_stride, const void* x, int x_dtype, int x_stride, const float* w,
                int rows, int n, const char* what) {
    AR_TRY(float_rows_ranges(h, h_dtype, h_stride, rows, n, what, "h"));
    if (x) AR_TRY(float_rows_ranges(x, x_dtype, x_stride, rows, n, what, "x"));
    return ar_check_range(w, (size_t)n * 4, what, "gain");
}

}  // namespace

extern "C" int ar_hip_quantize_i8(ar_hip_ctx* ctx, const void* x, int x_dtype, int x_stride, const ar_rows_i8* out) {
    const char* what = "quantize i8";
    AR_TRY(i8_check(out, what, "out"));
    AR_TRY(float_rows_check(x, x_dtype, x_stride, out->rows, out->n, what, "x"));
    AR_CHECK_ARG(ctx, "ctx is null");
    if (out->rows == 0) return AR_HIP_OK;
    AR_TRY(float_rows_ranges(x, x_dtype, x_stride, out->rows, out->n, what, "x"));
    AR_TRY(i8_check_ranges(out, what, "out"));
    RowParams p{};
    p.x = x; p.x_stride = x_stride; p.q = out->q; p.scale = out->scale; p.q_stride = out->stride; p.n = out->n;
    return x_dtype == AR_DTYPE_F32 ? launch_rows<float, float, float, false, true>(p, out->rows, ctx->stream)
                                   : launch_rows<float, uint16_t, float, false, true>(p, out->rows, ctx->stream);
}

extern "C" int ar_hip_add_rmsnorm(ar_hip_ctx* ctx, void* h, int h_dtype, int h_stride, const void* x, int x_dtype,
                                  int x_stride, const float* w, float eps, int rows, int n, void* y, int y_dtype,
                                  int y_stride) {
    const char* what = "add rmsnorm";
    AR_CHECK_ARG(rows >= 0 && rows <= kI8MaxRows, "%s: %d rows", what, rows);
    AR_CHECK_ARG(n >= 1 && n <= kI8MaxN, "%s: %d values a row (1 .. %d)", what, n, kI8MaxN);
    AR_TRY(norm_check(h, h_dtype, h_stride, x, x_dtype, x_stride, w, eps, rows, n, what));
    AR_TRY(float_rows_check(y, y_dtype, y_stride, rows, n, what, "y"));
    AR_CHECK_ARG(rows == 0 || y != h, "%s: y is h", what);
    AR_CHECK_ARG(rows == 0 || y != x || (y_dtype == x_dtype && y_stride == x_stride),
                 "%s: y is x, but of another type or stride", what);
    AR_CHECK_ARG(ctx, "ctx is null");
    if (rows == 0) return AR_HIP_OK;
    AR_TRY(norm_ranges(h, h_dtype, h_stride, x, x_dtype, x_stride, w, rows, n, what));
    AR_TRY(float_rows_ranges(y, y_dtype, y_stride, rows, n, what, "y"));
    RowParams p{};
    p.h = h; p.h_stride = h_stride; p.x = x; p.x_stride = x_stride; p.w = w; p.eps = eps; p.n = n; p.y = y;
    p.y_stride = y_stride;
    return launch_norm_types(p, h_dtype, x ? x_dtype : h_dtype, y_dtype, rows, ctx->stream);
}

extern "C" int ar_hip_add_rmsnorm_i8(ar_hip_ctx* ctx, void* h, int h_dtype, int h_stride, const void* x, int x_dtype,
                                     int x_stride, const float* w, float eps, const ar_rows_i8* out) {
    const char* what = "add rmsnorm i8";
    AR_TRY(i8_check(out, what, "out"));
    AR_TRY(norm_check(h, h_dtype, h_stride, x, x_dtype, x_stride, w, eps, out->rows, out->n, what));
    AR_CHECK_ARG(ctx, "ctx is null");
    if (out->rows == 0) return AR_HIP_OK;
    AR_TRY(norm_ranges(h, h_dtype, h_stride, x, x_dtype, x_stride, w, out->rows, out->n, what));
    AR_TRY(i8_check_ranges(out, what, "out"));
    RowParams p{};
    p.h = h; p.h_stride = h_stride; p.x = x; p.x_stride = x_stride; p.w = w; p.eps = eps; p.n = out->n; p.q = out->q;
    p.scale = out->scale; p.q_stride = out->stride;
    return launch_norm_types(p, h_dtype, x ? x_dtype : h_dtype, AR_DTYPE_F32, out->rows, ctx->stream);
}

extern "C" int ar_hip_embed_i8(ar_hip_ctx* ctx, const ar_rows_i8* table, const int32_t* tokens, int count, void* y,
                               int y_dtype, int y_stride) {
    const char* what = "embed i8";
    AR_TRY(i8_check(table, what, "table"));
    AR_CHECK_ARG(count >= 0 && count <= kI8MaxRows, "%s: %d rows", what, count);
    AR_CHECK_ARG(tokens || count <= table->rows, "%s: %d rows of a table of %d", what, count, table->rows);
    AR_CHECK_ARG(aligned_to(tokens, 4), "%s: tokens are not aligned to their type", what);
    AR_TRY(float_rows_check(y, y_dtype, y_stride, count, table->n, what, "y"));
    AR_CHECK_ARG(ctx, "ctx is null");
    if (count == 0) return AR_HIP_OK;
    AR_TRY(i8_check_ranges(table, what, "table"));
    if (tokens) AR_TRY(ar_check_range(tokens, (size_t)count * 4, what, "tokens"));
    AR_TRY(float_rows_ranges(y, y_dtype, y_stride, count, table->n, what, "y"));
    return y_dtype == AR_DTYPE_F32 ? launch_embed<float>(table, tokens, count, y, y_stride, ctx->stream)
                                   : launch_embed<uint16_t>(table, tokens, count, y, y_stride, ctx->stream);
}
