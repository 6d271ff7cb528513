// Products of rows in 8 bits: C[m][n] = scaleA[m] scaleW[n] sum_k A[m][k] W[n][k], sums in 32-bit whole numbers.
//
// Both operands lie along k, as the matrix instructions take them.  Where a token has few weights to meet, they come straight
// from memory (v_mfma_i32_16x16x64_i8: lane l supplies row l % 16 and the 16 bytes from (l / 16) * 16 of a 64-wide slice;
// register i of lane l is output 4 (l / 16) + i of token l % 16); otherwise through LDS in tiles.
#include <atomic>
#include <type_traits>

#include "i8_common.h"
#include "i8_plan.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct I8Params {
    const int8_t *a, *w, *w2;
    const float *sa, *sw, *sw2;
    int64_t lda, ldw;
    int M, N, K;       // K: rounded up to 16
    const float* bias;
    void* c;
    int64_t ldc;
};

// up * silu(gate) for gates from kFarGate on, and NaN.  EXACT (fp32 outputs): from e = exp(-|gate|), which does not overflow:
// silu = gate / (1 + e), times e for gates below 0; e is the square of 2^(t/2), t = -|gate| log2(e), which reaches twice as far
// down as the hardware's 2^t, corrected by the rounding error of t, and the quotient is corrected by one step: to about 2^-23.
// bf16 outputs: the bare reciprocal of 1 + 2^t, t = -gate log2(e), some |gate| 2^-23 off, far below half a step of bf16.
constexpr float kFarGate = -87.f;
template <bool EXACT>
__device__ inline float gated(float g, float u) {
#pragma clang fp contract(off)
    if constexpr (EXACT) {
        const float a = fminf(fabsf(g), 128.f), t = a * -1.44269502f;
        const float s = __builtin_amdgcn_exp2f(0.5f * t);
        const float d = fmaf(t, 1.90465421e-9f, fmaf(t, -0.693147182f, -a));  // ln 2 = 0.693147182 - 1.904654e-9
        const float tail = fmaf(s, d, s);                                     // e = s * tail
        const float num = g >= 0.f ? g : g * s * tail, den = fmaf(s, tail, 1.f);
        const float r = __builtin_amdgcn_rcpf(den), q = num * r;
        return u * (q < INFINITY ? fmaf(fmaf(-den, q, num), r, q) : q);
    } else {
        return u * (g * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269502f)));
    }
}

// ... and for gates below kFarGate, whose silu = gate * e, e = exp(gate), need not be a normal number where its product with
// `up` is one: e is the fourth power of 2^(t/4), two of which go to the gate and two to `up`, corrected as above.  Gates below
// -300, minus infinity among them, count as that, where two are 0.
__device__ inline float gated_far(float g, float u) {
#pragma clang fp contract(off)
    g = fmaxf(g, -300.f);
    const float t = g * 1.44269502f, s = __builtin_amdgcn_exp2f(0.25f * t);
    const float d = fmaf(t, 1.90465421e-9f, fmaf(t, -0.693147182f, g)), v = u * s * s * (g * s * s);
    return fmaf(v, d, v);
}

// sa * sw * sum (+ more).  sa * sum may be past fp32 where the product is not, from token scales of kFarScale on (sums are below
// 2^31 in magnitude): FAR takes it 2^64 times smaller then, which is the same to the last bit but for what fp32 cannot hold.
constexpr float kFarScale = 0x1p96f;
template <bool FAR, bool ADD>
__device__ inline float scaled(int sum, float sa, float sw, float more) {
#pragma clang fp contract(off)
    const float v = (float)sum * sa, near = ADD ? fmaf(v, sw, more) : v * sw;
    if constexpr (!FAR) return near;
    const float less = (float)sum * (sa * 0x1p-64f) * sw;
    return fabsf(v) < INFINITY ? near : ADD ? fmaf(less, 0x1p64f, more) : less * 0x1p64f;
}

// One output from the sums over W (and W2).  Every kernel ends in these operations and no others, so that a row's bits do
// not depend on the batch.  FAR: token scales may be above kFarScale, gates below kFarGate.
template <int EPI, class CT, bool FAR>
__device__ inline float finished(float sa, float sw, float sw2, float more, int g, int u) {
    if constexpr (EPI == GEMV_EPI_SWIGLU) {
        const float gate = scaled<FAR, false>(g, sa, sw, 0.f), up = scaled<FAR, false>(u, sa, sw2, 0.f);
        const float near = gated<sizeof(CT) == 4>(gate, up);
        if constexpr (!FAR) return near;
        return gate < kFarGate ? gated_far(gate, up) : near;
    } else {
        return scaled<FAR, true>(g, sa, sw, more);  // more: the bias, the residual or nothing
    }
}

// ---- few tokens, few outputs: weights straight from memory -----------------------------------
//
// The 8 wavefronts of a block take 16 outputs (gated: of both matrices) of up to 16 tokens, each over every eighth 128 bytes
// of k, and add their sums up in LDS.  Both halves of a line are read by one wavefront, UNITS lines of a row ahead; the
// tokens' rows come from the caches.  Bound by the latency of memory: one token x 2,560 over 9,728 7.9 us (25 MB, 3.1 TB/s).
template <int EPI, class CT>
__global__ __launch_bounds__(512) void gemm_i8_rows_kernel(I8Params p) {
    constexpr int NW = EPI == GEMV_EPI_SWIGLU ? 2 : 1, WAVES = 8, UNITS = 4 / NW;
    __shared__ i32x4 sums[WAVES][NW][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, r = lane & 15, at = (lane >> 4) * 16;
    const int8_t* const a = p.a + (size_t)min(r, p.M - 1) * p.lda + at;
    const size_t row = (size_t)min(n0 + r, p.N - 1) * p.ldw + at;
    const int8_t* const w[2] = {p.w + row, NW == 2 ? p.w2 + row : nullptr};
    i32x4 acc[NW];
#pragma unroll
    for (int v = 0; v < NW; v++) acc[v] = i32x4{0, 0, 0, 0};
    auto lines = [&](int k, auto whole) {  // of the last ones those behind the end become zeros
        i32x4 x[UNITS][2], y[UNITS][2][NW];
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int from = k + u * WAVES * 128 + h * 64;
                const bool in = whole.value || from + at < p.K;
                const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
                for (int v = 0; v < NW; v++) y[u][h][v] = in ? *(const i32x4*)(w[v] + from) : zero;
                x[u][h] = in ? *(const i32x4*)(a + from) : zero;
            }
#pragma unroll
        for (int u = 0; u < UNITS; u++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int v = 0; v < NW; v++)
                    acc[v] = __builtin_amdgcn_mfma_i32_16x16x64_i8(y[u][h][v], x[u][h], acc[v], 0, 0, 0);
    };
    int k = wave * 128;
    for (; k + (UNITS - 1) * WAVES * 128 + 128 <= p.K; k += UNITS * WAVES * 128) lines(k, std::true_type{});
    if (k < p.K) lines(k, std::false_type{});
#pragma unroll
    for (int v = 0; v < NW; v++) sums[wave][v][lane] = acc[v];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int v = 0; v < NW; v++)
#pragma unroll
        for (int q = 1; q < WAVES; q++) acc[v] += sums[q][v][lane];
    const int n = n0 + (lane >> 4) * 4, last = p.N - 1 - n;
    if (r >= p.M || last < 0) return;
    CT* const c = (CT*)p.c + (size_t)r * p.ldc + n;
    const float sa = p.sa[r];
    float out[4], sw[4], sw2[4], more[4], least = 0.f;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int i = min(q, last);
        sw[q] = p.sw[n + i];
        sw2[q] = NW == 2 ? p.sw2[n + i] : 0.f;
        more[q] = 0.f;
        if constexpr (EPI == GEMV_EPI_STORE) more[q] = p.bias ? p.bias[n + i] : 0.f;
        if constexpr (EPI == GEMV_EPI_RESIDUAL) more[q] = to_float<CT>(c[i]);
    }
#pragma unroll
    for (int q = 0; q < 4; q++) {
        out[q] = finished<EPI, CT, false>(sa, sw[q], sw2[q], more[q], acc[0][q], acc[NW - 1][q]);
        if constexpr (NW == 2) least = fminf(least, scaled<false, false>(acc[0][q], sa, sw[q], 0.f));
    }
    if (fabsf(sa) > kFarScale || least < kFarGate) {
#pragma unroll
        for (int q = 0; q < 4; q++)
            out[q] = finished<EPI, CT, true>(sa, sw[q], sw2[q], more[q], acc[0][q], acc[NW - 1][q]);
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
        if (q <= last) c[q] = from_float<CT>(out[q]);
}

// ---- more tokens: tiles fed by direct global -> LDS copies -----------------------------------
//
// A block of WAVES wavefronts owns BM tokens by BN weight rows (gated: BN / 2 gate rows and their up rows), a wavefront
// (BM / GM) x (BN / GN) of them in accumulators of v_mfma_i32_32x32x32_i8: lane l supplies row l % 32 and the 16 bytes from
// (l / 32) * 16 of a 32-wide k-step; register i holds token 8 (i / 4) + 4 (l / 32) + i % 4, output l % 32.
// k is walked in steps of BK bytes through STAGES LDS buffers.  The rows of a buffer lie one behind the other; chunk c (16
// bytes) of row r sits in slot c ^ swizzle(r), so that the eight lanes of an LDS cycle meet eight different groups of banks.
// A block takes tile after tile, and the copies run ahead across them: the first buffers of the next tile are on their way
// while this one is finished and stored.
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) unsigned char lds_byte;

#ifdef __HIP_DEVICE_COMPILE__
// Memory from p on as a buffer: offsets below 2^31, which a block's rows keep (256 rows of at most 2^22 bytes).
__device__ inline __amdgpu_buffer_rsrc_t buffer_of(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x80000000u, 0x00020000);
}
#endif

constexpr int kNoOffset = (int)0x80000000;  // past the end of buffer_of's buffers
// s_waitcnt for at most v outstanding loads, LDS reads awaited too where lgkm is 0
constexpr int wait_imm(int v, int lgkm) { return (v & 15) | ((v >> 4) << 14) | (7 << 4) | (lgkm << 8); }

template <int EPI_, class CT_, int BM_, int BN_, int GM_, int GN_, int BK_, int STAGES_, int PER_CU_>
struct Tile {
    static constexpr int EPI = EPI_, BM = BM_, BN = BN_, GM = GM_, GN = GN_, BK = BK_, STAGES = STAGES_, PER_CU = PER_CU_;
    using CT = CT_;
    static constexpr int WAVES = GM * GN, NW = EPI == GEMV_EPI_SWIGLU ? 2 : 1, BNO = BN / NW;
    static constexpr int WM = BM / GM, WN = BNO / GN, FM = WM / 32, FN = WN / 32, KS = BK / 32, CH = BK / 16;
    static constexpr int TILE_A = BM * BK, STAGE = (BM + BN) * BK, LDS = STAGES * STAGE;
    static constexpr int COPY_A = TILE_A / 1024 / WAVES, COPY_W = BN * BK / 1024 / WAVES, COPIES = COPY_A + COPY_W;
    static constexpr int ROWS = 1024 / BK;  // rows of a copy
    static_assert(WM % 32 == 0 && WN % 32 == 0 && TILE_A % (1024 * WAVES) == 0 && BNO * BK % (1024 * WAVES) == 0, "");
    static_assert(ROWS * WAVES % 16 == 0, "a wavefront's copies have the swizzle's phase in common");
    static_assert(LDS * PER_CU <= 160 * 1024, "");
    static __device__ inline int slot(int r, int c) { return c ^ ((r >> 1) & (CH - 1)); }
};

// How a product is cut: mt x nt tiles, each in `splits` parts of k (then `part` takes the sums).
struct Cut {
    int mt, nt, splits;
    int* part;  // [splits][tiles][wavefront][matrix, i, j][4][lane][4]
};

// Task t of a block -> tile and part of k.  Blocks are dealt round-robin over 8 XCDs, so t % 8 is the XCD; each takes a run
// of consecutive tasks, which walk groups of 8 token tiles column by column, so that what an XCD runs at a time shares rows of
// both operands in its L2.
__device__ inline void task_at(int t, const Cut& cut, int* mi, int* ni, int* part) {
    const int tiles = cut.mt * cut.nt, all = tiles * cut.splits, q = all >> 3, rest = all & 7, x = t & 7;
    const int u = x * q + min(x, rest) + (t >> 3);  // XCD x has q tasks, the first `rest` one more
    *part = u / tiles;
    const int v = u - *part * tiles;
    constexpr int G = 8;
    const int group = v / (G * cut.nt), first = group * G, size = min(cut.mt - first, G), r = v - group * G * cut.nt;
    *ni = r / size;
    *mi = first + r - *ni * size;
}

#ifdef __HIP_DEVICE_COMPILE__
// A lane's place in 32 x 32 outputs: register r is token 4 (lane / 32) + token_of(r), output lane % 32.
__device__ constexpr int token_of(int r) { return (r >> 2) * 8 + (r & 3); }

// 32 x 32 outputs of a wavefront, from (m0, n0) on, from their sums.  They are addressed as a buffer from (m0, n0) on, the
// lane's place as its offset and the register's token as the scalar one (32 rows of at most 2^24 values: below 2^31 bytes);
// outputs that do not exist get an offset past the buffer's end, where loads give zero and stores do nothing.  Without
// branches: a load that some path does not use makes the compiler wait for all loads, the copies among them, wherever its
// register is used next, which was in the loop over k (1,024 x 2,560 over 4,096 25 us instead of 19).
// pair: all outputs exist and two bf16 ones fit a 4-byte store.  far: one of the tokens' scales is above kFarScale.
template <int EPI, class CT, class Sums>
__device__ inline void store_32x32(const I8Params& p, int m0, int n0, bool pair, bool far, const float (&sa)[16], float sw,
                                   float sw2, float bias, const Sums& g, const Sums& u) {
    const __amdgpu_buffer_rsrc_t c = buffer_of((CT*)p.c + (size_t)m0 * p.ldc + n0);
    const int lane = threadIdx.x & 63, first = (lane >> 5) * 4, bytes = (int)p.ldc * (int)sizeof(CT);
    const int at = first * bytes + (lane & 31) * (int)sizeof(CT);
    const int tokens = n0 + (lane & 31) < p.N ? p.M - m0 - first : 0;  // that the lane's output has
    auto place = [&](int r, int tokens, int at) { return token_of(r) < tokens ? at : kNoOffset; };
    auto more = [&](int r, int tokens, int at) {
        if constexpr (EPI != GEMV_EPI_RESIDUAL) return bias;
        else if constexpr (sizeof(CT) == 4)
            return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(c, place(r, tokens, at), token_of(r) * bytes, 0));
        else
            return to_float<CT>(__builtin_amdgcn_raw_buffer_load_b16(c, place(r, tokens, at), token_of(r) * bytes, 0));
    };
    float out[16];
#pragma unroll
    for (int r = 0; r < 16; r++) out[r] = more(r, tokens, at);
#pragma unroll
    for (int r = 0; r < 16; r++) out[r] = finished<EPI, CT, false>(sa[r], sw, sw2, out[r], g[r], u[r]);
    if constexpr (EPI == GEMV_EPI_SWIGLU) {
        float least = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r++) least = fminf(least, scaled<false, false>(g[r], sa[r], sw, 0.f));
        far = far || __builtin_amdgcn_ballot_w64(least < kFarGate) != 0;
    }
    if (far) {
#pragma unroll
        for (int r = 0; r < 16; r++) {
            // (hidden, or what both have in common would be computed, and held, ahead of the branch)
            int sum = g[r], sum2 = u[r], left = tokens, first_at = at;
            asm volatile("" : "+v"(sum), "+v"(sum2), "+v"(left), "+v"(first_at)::"memory");
            __builtin_amdgcn_sched_barrier(0);
            out[r] = finished<EPI, CT, true>(sa[r], sw, sw2, more(r, left, first_at), sum, sum2);
        }
    }
    if constexpr (sizeof(CT) == 2) {
        if (pair) {  // neighbouring lanes swap one of two tokens' values: each stores two outputs of one token
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            const bool odd = lane & 1;
            const int mine = at + (odd ? bytes - 2 : 0);
            const unsigned pick = odd ? 0x03020706u : 0x05040100u;  // (neighbour's upper, own upper : own lower, neighbour's)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const bf16x2 both = __builtin_convertvector(f32x2{out[r], out[r + 1]}, bf16x2);
                const unsigned own = __builtin_bit_cast(unsigned, both);
                const unsigned other = __builtin_amdgcn_update_dpp(0u, own, 0xB1, 0xF, 0xF, true);
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_amdgcn_perm(other, own, pick), c, mine, token_of(r) * bytes, 0);
            }
            return;
        }
    }
    int from = at;
    if constexpr (sizeof(CT) == 2) asm volatile("" : "+v"(from));  // (places anew, instead of 16 registers for the loads' ones)
#pragma unroll
    for (int r = 0; r < 16; r++) {
        if constexpr (sizeof(CT) == 4)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(out[r]), c, place(r, tokens, from), token_of(r) * bytes, 0);
        else
            __builtin_amdgcn_raw_buffer_store_b16(from_float<CT>(out[r]), c, place(r, tokens, from), token_of(r) * bytes, 0);
    }
}
template <class CT>
__device__ inline bool pairs_fit(const I8Params& p) {
    return (reinterpret_cast<uintptr_t>(p.c) & 3) == 0 && p.ldc % 2 == 0;
}
// The scales of a lane's 16 tokens from m0 on; true where one of the wavefront's 32 is above kFarScale.
__device__ inline bool token_scales(const I8Params& p, int m0, float (&sa)[16]) {
    typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
    const int lane = threadIdx.x & 63, first = lane >> 5 << 2;
    const float one = p.sa[min(m0 + (lane & 31), p.M - 1)];  // (a token a lane: one comparison looks at all of them)
    if (m0 + 32 <= p.M) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const f32x4 v = *(const f32x4*)(p.sa + m0 + first + q * 8);
#pragma unroll
            for (int i = 0; i < 4; i++) sa[4 * q + i] = v[i];
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; r++) sa[r] = p.sa[min(m0 + first + token_of(r), p.M - 1)];
    }
    return __builtin_amdgcn_ballot_w64(fabsf(one) > kFarScale) != 0;
}
#endif

template <class T, bool SPLIT>
__global__ __launch_bounds__(T::WAVES * 64, T::PER_CU * T::WAVES / 4) void gemm_i8_tile_kernel(I8Params p, Cut cut) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass does not know the buffer builtins)
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / T::GN, wn = wave % T::GN;
    const int tasks = cut.mt * cut.nt * (SPLIT ? cut.splits : 1), steps = (p.K + T::BK - 1) / T::BK;
    auto first_step = [&](int part) { return SPLIT ? (int)((long long)steps * part / cut.splits) : steps * part; };

    // The copies' side.  Copy i of wavefront w fills 1 KB, the rows ROWS j .. ROWS j + ROWS - 1 (j = WAVES i + w) of a buffer;
    // lane l slot l % CH of row ROWS j + l / CH.  The tile's first rows are the bases of buffers (rows past the last are read
    // from the last), a lane's offsets in them stay along k, and k goes into the scalar offset: a copy is one instruction.
    // (Loads through flat addresses would also make the compiler wait for every outstanding LDS read where it needs one.)
    // Each XCD begins an eighth of k further on and comes round to it (sums in whole numbers have no order), so that not all
    // ask the same channels of memory at a time: 2,048 x 6,144 over 2,560 40.4 us, in step 43.3; 8,192 x 9,728 gated over 2,560
    // 374 and 388.  copy_step counts, copy_k is where the copies are; a cut step comes last.
    __amdgpu_buffer_rsrc_t bufA, bufW, bufW2;
    unsigned offA[T::COPY_A], offW[T::COPY_W];
    const int at = T::ROWS * wave + lane / T::CH, chunk = T::slot(at, lane % T::CH) * 16;
    int copy_task = blockIdx.x, copy_step = 0, copy_stop = 0, copy_end = 0, copy_k = 0, first_k = 0, end_k = 0;
    // Ahead of the last step of k, if it is not a whole one: chunks behind the end become zeros (as all past a buffer's end does).
    auto cut_step = [&]() {
        const unsigned past = copy_step * T::BK + chunk < p.K ? 0u : (unsigned)kNoOffset;
#pragma unroll
        for (int i = 0; i < T::COPY_A; i++) offA[i] |= past;
#pragma unroll
        for (int i = 0; i < T::COPY_W; i++) offW[i] |= past;
        copy_stop = copy_end;
        copy_k = copy_step * T::BK;
    };
    auto aim = [&](int t) {
        int mi, ni, part;
        task_at(t, cut, &mi, &ni, &part);
        const int m0 = mi * T::BM, n0 = ni * T::BNO;
        copy_step = first_step(part);
        copy_end = first_step(part + 1);
        bufA = buffer_of(p.a + (size_t)m0 * p.lda);
        bufW = buffer_of(p.w + (size_t)n0 * p.ldw);
        if constexpr (T::NW == 2) bufW2 = buffer_of(p.w2 + (size_t)n0 * p.ldw);
#pragma unroll
        for (int i = 0; i < T::COPY_A; i++)
            offA[i] = (unsigned)min(T::ROWS * T::WAVES * i + at, p.M - 1 - m0) * (unsigned)p.lda + chunk;
#pragma unroll
        for (int i = 0; i < T::COPY_W; i++)
            offW[i] = (unsigned)min((T::ROWS * T::WAVES * i + at) % T::BNO, p.N - 1 - n0) * (unsigned)p.ldw + chunk;
        copy_stop = min(copy_end, p.K / T::BK);  // (whole steps)
        first_k = copy_step * T::BK;
        end_k = copy_stop * T::BK;
        copy_k = first_k + ((copy_stop - copy_step) * (t & 7) >> 3) * T::BK;
        if (copy_step >= copy_stop) cut_step();
    };
    lds_byte* const lds_base = (lds_byte*)lds + wave * 1024;
    auto copy = [&](int buffer, int lo, int hi) {  // copies lo .. hi - 1 of the step that is next
        lds_byte* const st = lds_base + buffer * T::STAGE;
#pragma unroll
        for (int i = 0; i < T::COPIES; i++) {
            if (i < lo || i >= hi) continue;
            const bool isA = i < T::COPY_A;
            const int j = isA ? i : i - T::COPY_A;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(isA ? bufA : T::NW == 2 && j >= T::COPY_W / 2 ? bufW2 : bufW,
                                                     (lds_void*)(st + (isA ? 0 : T::TILE_A) + T::WAVES * j * 1024), 16,
                                                     isA ? offA[j] : offW[j], copy_k, 0, 0);
        }
    };
    // Past the last task its last step is copied again, so that the number of outstanding copies is always the same.
    auto advance = [&]() {
        const int before = copy_k;
        copy_k = copy_k + T::BK == end_k ? first_k : copy_k + T::BK;
        if (++copy_step < copy_stop) return;
        if (copy_step < copy_end) {
            cut_step();
        } else if (copy_task + (int)gridDim.x < tasks) {
            copy_task += gridDim.x;
            aim(copy_task);
        } else {
            copy_step = copy_end - 1;
            copy_k = before;
        }
    };

    i32x16 acc[T::NW][T::FM][T::FN];
    i32x4 fa[2][T::FM], fw[2][T::NW][T::FN];
    auto read = [&](int set, const unsigned char* st, int ks) {
        const int c = ks * 2 + (lane >> 5);
#pragma unroll
        for (int i = 0; i < T::FM; i++) {
            const int r = wm * T::WM + i * 32 + (lane & 31);
            fa[set][i] = *(const i32x4*)(st + r * T::BK + T::slot(r, c) * 16);
        }
#pragma unroll
        for (int w = 0; w < T::NW; w++)
#pragma unroll
            for (int j = 0; j < T::FN; j++) {
                const int r = w * T::BNO + wn * T::WN + j * 32 + (lane & 31);
                fw[set][w][j] = *(const i32x4*)(st + T::TILE_A + r * T::BK + T::slot(r, c) * 16);
            }
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int w = 0; w < T::NW; w++)
#pragma unroll
            for (int i = 0; i < T::FM; i++)
#pragma unroll
                for (int j = 0; j < T::FN; j++)
                    acc[w][i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[set][i], fw[set][w][j], acc[w][i][j], 0, 0, 0);
    };

    int buffer = 0;
    aim(copy_task);
#pragma unroll
    for (int s = 0; s + 1 < T::STAGES; s++) {
        copy(s, 0, T::COPIES);
        advance();
    }
    copy(T::STAGES - 1, 0, T::COPIES / 2);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_imm(T::COPIES * (T::STAGES - 2) + T::COPIES / 2, 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, lds, 0);
    for (int t = blockIdx.x; t < tasks; t += gridDim.x) {
        int mi, ni, part;
        task_at(t, cut, &mi, &ni, &part);
        const int m0 = mi * T::BM, n0 = ni * T::BNO, count = first_step(part + 1) - first_step(part);
#pragma unroll
        for (int w = 0; w < T::NW; w++)
#pragma unroll
            for (int i = 0; i < T::FM; i++)
#pragma unroll
                for (int j = 0; j < T::FN; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[w][i][j][r] = 0;
        // A buffer is free for the step STAGES later as soon as every wavefront holds its last fragments, one k-step before
        // the step's end: there is the one barrier of a step, and behind it the first fragments of the next step are read
        // while the last k-step is multiplied.  The copies of a step go out in two halves, here and behind the next step's
        // first reads (all at once they hold up the wavefronts at issue: 8,192^3 1,942 x 10^12 operations a second in
        // halves, 1,873 at once, both with loads through flat addresses).
        for (int n = 0; n < count; n++) {
            const unsigned char* const st = lds + buffer * T::STAGE;
            const int next = buffer + 1 == T::STAGES ? 0 : buffer + 1, before = buffer == 0 ? T::STAGES - 1 : buffer - 1;
#pragma unroll
            for (int ks = 0; ks + 1 < T::KS; ks++) {
                read((ks + 1) & 1, st, ks + 1);
                if (ks == 0) copy(before, T::COPIES / 2, T::COPIES);
                __builtin_amdgcn_sched_barrier(0);
                multiply(ks & 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" ::: "memory");  // (keeps the last reads ahead of the branches: 509 x 2,560 over 9,728 24.6 us, else 28.8)
            advance();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(wait_imm(T::COPIES * (T::STAGES - 2), 0));
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            copy(buffer, 0, T::COPIES / 2);
            read(0, lds + next * T::STAGE, 0);
            __builtin_amdgcn_sched_barrier(0);
            multiply((T::KS - 1) & 1);
            __builtin_amdgcn_sched_barrier(0);
            buffer = next;
        }
        if constexpr (SPLIT) {
            i32x4* const to = (i32x4*)cut.part +
                              ((size_t)(part * cut.mt * cut.nt + mi * cut.nt + ni) * T::WAVES + wave) * (T::NW * T::FM * T::FN * 256) + lane;
#pragma unroll
            for (int w = 0; w < T::NW; w++)
#pragma unroll
                for (int i = 0; i < T::FM; i++) {
                    if (m0 + wm * T::WM + i * 32 >= p.M) continue;
#pragma unroll
                    for (int j = 0; j < T::FN; j++)
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            to[((w * T::FM + i) * T::FN + j) * 256 + q * 64] =
                                i32x4{acc[w][i][j][4 * q], acc[w][i][j][4 * q + 1], acc[w][i][j][4 * q + 2], acc[w][i][j][4 * q + 3]};
                }
        } else {
            using CT = typename T::CT;
            const bool pair = sizeof(CT) == 2 && m0 + T::BM <= p.M && n0 + T::BNO <= p.N && pairs_fit<CT>(p);
            const int mw = m0 + wm * T::WM, nw = n0 + wn * T::WN;
            float sw[T::FN], sw2[T::FN], bias[T::FN];
#pragma unroll
            for (int j = 0; j < T::FN; j++) {
                const int n = min(nw + j * 32 + (lane & 31), p.N - 1);
                sw[j] = p.sw[n];
                sw2[j] = T::NW == 2 ? p.sw2[n] : 0.f;
                bias[j] = T::EPI == GEMV_EPI_STORE && p.bias ? p.bias[n] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < T::FM; i++) {
                float sa[16];
                const bool far = token_scales(p, mw + i * 32, sa);
#pragma unroll
                for (int j = 0; j < T::FN; j++) {
                    store_32x32<T::EPI, CT>(p, mw + i * 32, nw + j * 32, pair, far, sa, sw[j], sw2[j], bias[j],
                                            acc[0][i][j], acc[T::NW - 1][i][j]);
                    __builtin_amdgcn_sched_barrier(0);  // (what all 32 x 32 read would not fit the registers at once)
                }
            }
        }
    }
    __builtin_amdgcn_s_waitcnt(0);  // no copy in flight when the block ends
#endif
}

// The parts' sums, added up and finished: a wavefront takes 32 x 32 outputs.
template <class T>
__global__ __launch_bounds__(256) void gemm_i8_sum_kernel(I8Params p, Cut cut) {
#ifdef __HIP_DEVICE_COMPILE__
    using CT = typename T::CT;
    const int lane = threadIdx.x & 63, tiles = cut.mt * cut.nt;
    const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int sub = id % (T::FM * T::FN), wave = id / (T::FM * T::FN) % T::WAVES, tile = id / (T::FM * T::FN * T::WAVES);
    if (tile >= tiles) return;
    const int m0 = tile / cut.nt * T::BM + wave / T::GN * T::WM + sub / T::FN * 32;
    const int n0 = tile % cut.nt * T::BNO + wave % T::GN * T::WN + sub % T::FN * 32;
    if (m0 >= p.M || n0 >= p.N) return;
    const size_t stride = (size_t)tiles * T::WAVES * (T::NW * T::FM * T::FN * 256);
    const i32x4* const from = (const i32x4*)cut.part + ((size_t)tile * T::WAVES + wave) * (T::NW * T::FM * T::FN * 256) +
                              sub * 256 + lane;
    i32x16 sum[T::NW];
#pragma unroll
    for (int w = 0; w < T::NW; w++) {
#pragma unroll
        for (int r = 0; r < 16; r++) sum[w][r] = 0;
#pragma unroll 4
        for (int s = 0; s < cut.splits; s++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const i32x4 v = from[s * stride + w * (T::FM * T::FN * 256) + q * 64];
#pragma unroll
                for (int r = 0; r < 4; r++) sum[w][4 * q + r] += v[r];
            }
    }
    const int n = min(n0 + (lane & 31), p.N - 1);
    float sa[16];
    const bool far = token_scales(p, m0, sa);
    store_32x32<T::EPI, CT>(p, m0, n0, m0 + 32 <= p.M && n0 + 32 <= p.N && pairs_fit<CT>(p), far, sa, p.sw[n],
                            T::NW == 2 ? p.sw2[n] : 0.f, T::EPI == GEMV_EPI_STORE && p.bias ? p.bias[n] : 0.f, sum[0],
                            sum[T::NW - 1]);
#endif
}

template <class T, bool SPLIT>
int launch_tile(const I8Params& p, const Cut& cut, int cus, hipStream_t st) {
    // more than 64 KB of dynamic LDS needs the per-kernel opt-in, once per device
    static std::atomic<bool> set[kMaxDevices];
    const int slot = ar_device_slot(st);
    if (slot < 0 || !set[slot].load(std::memory_order_relaxed)) {
        int current = slot;  // (of the stream's device, whichever is current)
        if (slot >= 0) AR_HIP_TRY(hipGetDevice(&current));
        if (current != slot) AR_HIP_TRY(hipSetDevice(slot));
        const hipError_t e = hipFuncSetAttribute((const void*)gemm_i8_tile_kernel<T, SPLIT>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if (current != slot) AR_HIP_TRY(hipSetDevice(current));
        AR_HIP_TRY(e);
        if (slot >= 0) set[slot].store(true, std::memory_order_relaxed);
    }
    // (a multiple of 8 blocks, or all the tasks: a block's tasks stay on its XCD)
    const long long tasks = (long long)cut.mt * cut.nt * cut.splits;
    const int blocks = (int)(tasks < (long long)cus * T::PER_CU ? tasks : (long long)(cus * T::PER_CU) & ~7LL);
    hipLaunchKernelGGL((gemm_i8_tile_kernel<T, SPLIT>), dim3(blocks), dim3(T::WAVES * 64), T::LDS, st, p, cut);
    AR_LAUNCH_CHECK();
    if constexpr (SPLIT) {
        const long long waves = (long long)cut.mt * cut.nt * T::WAVES * T::FM * T::FN;
        hipLaunchKernelGGL(gemm_i8_sum_kernel<T>, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, p, cut);
        AR_LAUNCH_CHECK();
    }
    return AR_HIP_OK;
}

template <int EPI, class CT>
int launch_rows(const I8Params& p, hipStream_t st) {
    hipLaunchKernelGGL((gemm_i8_rows_kernel<EPI, CT>), dim3((p.N + 15) / 16), dim3(512), 0, st, p);
    AR_LAUNCH_CHECK();
    return AR_HIP_OK;
}

template <int KIND, int GM, int GN, int EPI, class CT>
int launch_kind(const I8Params& p, const I8Plan& plan, void* work, int cus, hipStream_t st) {
    constexpr auto t = kTileSize[KIND];
    constexpr bool GATED = EPI == GEMV_EPI_SWIGLU;
    using T = Tile<EPI, CT, t.bm, GATED ? t.gated_bn : t.bn, GM, GN, 128, GATED ? t.gated_buffers : t.buffers, t.per_cu>;
    const Cut cut{(p.M + T::BM - 1) / T::BM, (p.N + T::BNO - 1) / T::BNO, plan.splits, (int*)work};
    if constexpr (t.split)
        if (plan.splits > 1) return launch_tile<T, true>(p, cut, cus, st);
    return launch_tile<T, false>(p, cut, cus, st);
}

template <int EPI, class CT>
int launch_product(const I8Params& p, void* work, int cus, hipStream_t st) {
    constexpr bool GATED = EPI == GEMV_EPI_SWIGLU;
    const I8Plan plan = i8_plan(p.M, p.N, p.K, GATED, cus);
    switch (plan.kind) {
        case kRows: return launch_rows<EPI, CT>(p, st);
        case kTile32: return launch_kind<kTile32, 1, GATED ? 2 : 4, EPI, CT>(p, plan, work, cus, st);
        case kTile64: return launch_kind<kTile64, 2, 2, EPI, CT>(p, plan, work, cus, st);
        case kTile128: return launch_kind<kTile128, 4, 2, EPI, CT>(p, plan, work, cus, st);
        case kTile128x256: return launch_kind<kTile128x256, 2, 4, EPI, CT>(p, plan, work, cus, st);
        case kTile256: return launch_kind<kTile256, 2, 4, EPI, CT>(p, plan, work, cus, st);
        default: break;
    }
    if constexpr (!GATED) {  // (two weight tiles of these widths do not split over the wavefronts)
        if (plan.kind == kTile64x128) return launch_kind<kTile64x128, 2, 4, EPI, CT>(p, plan, work, cus, st);
        if (plan.kind == kTile256x192) return launch_kind<kTile256x192, 4, 2, EPI, CT>(p, plan, work, cus, st);
    }
    ar_set_error("GEMM i8: no kernel for plan %d", (int)plan.kind);
    return AR_HIP_ERR_STATE;
}

template <int EPI>
int launch_types(const I8Params& p, int c_dtype, void* work, const ar_hip_ctx* ctx) {
    return c_dtype == AR_DTYPE_F32 ? launch_product<EPI, float>(p, work, ctx->num_cus, ctx->stream)
                                   : launch_product<EPI, uint16_t>(p, work, ctx->num_cus, ctx->stream);
}

int check_shape(int M, int N, int K, int epilogue, const char* what) {
    AR_CHECK_ARG(M >= 0 && M <= kI8MaxRows && N >= 0 && N <= kI8MaxRows && K >= 1 && K <= kI8MaxN,
                 "%s: product of %d x %d over %d", what, M, N, K);
    AR_CHECK_ARG((long long)M * N <= 1LL << 40, "%s: %d x %d outputs (at most 2^40)", what, M, N);
    AR_CHECK_ARG(epilogue == AR_GEMM_STORE || epilogue == AR_GEMM_RESIDUAL || epilogue == AR_GEMM_SWIGLU,
                 "%s: unknown epilogue %d", what, epilogue);
    return AR_HIP_OK;
}

}  // namespace

extern "C" int ar_hip_gemm_i8_work(ar_hip_ctx* ctx, int M, int N, int K, int epilogue, size_t* bytes) {
    const char* what = "GEMM i8";
    AR_CHECK_ARG(bytes, "%s: bytes is null", what);
    AR_TRY(check_shape(M, N, K, epilogue, what));
    AR_CHECK_ARG(ctx, "ctx is null");
    *bytes = i8_work_bytes(M, N, (K + 15) / 16 * 16, epilogue == AR_GEMM_SWIGLU, ctx->num_cus);
    return AR_HIP_OK;
}

extern "C" int ar_hip_gemm_i8(ar_hip_ctx* ctx, const ar_rows_i8* A, const ar_rows_i8* W, const ar_rows_i8* W2,
                              const float* bias, void* C, int c_dtype, int ldc, int epilogue, void* work,
                              size_t work_bytes) {
    const char* what = "GEMM i8";
    AR_TRY(i8_check(A, what, "A"));
    AR_TRY(i8_check(W, what, "W"));
    AR_TRY(check_shape(A->rows, W->rows, A->n, epilogue, what));
    AR_CHECK_ARG(W->n == A->n, "%s: rows of %d values times rows of %d", what, A->n, W->n);
    AR_CHECK_ARG((epilogue == AR_GEMM_SWIGLU) == (W2 != nullptr), "%s: W2 goes with the SwiGLU epilogue", what);
    if (W2) {
        AR_TRY(i8_check(W2, what, "W2"));
        AR_CHECK_ARG(W2->n == W->n && W2->rows == W->rows && W2->stride == W->stride, "%s: W2 is not of W's sizes", what);
    }
    AR_CHECK_ARG(!bias || epilogue == AR_GEMM_STORE, "%s: a bias goes with the store epilogue", what);
    AR_CHECK_ARG(aligned_to(bias, 4), "%s: the bias is not aligned to its type", what);
    AR_CHECK_ARG(is_float_dtype(c_dtype), "%s: unknown dtype %d of C", what, c_dtype);
    AR_CHECK_ARG(ldc >= W->rows && ldc <= kI8MaxRows, "%s: stride of %d values of C (%d .. %d)", what, ldc, W->rows,
                 kI8MaxRows);
    const bool empty = A->rows == 0 || W->rows == 0;
    AR_CHECK_ARG(empty || C, "%s: C is null", what);
    AR_CHECK_ARG(aligned_to(C, float_bytes(c_dtype)), "%s: C is not aligned to its type", what);
    AR_CHECK_ARG(ctx, "ctx is null");
    if (empty) return AR_HIP_OK;
    const int K = (A->n + 15) / 16 * 16;
    const size_t need = i8_work_bytes(A->rows, W->rows, K, epilogue == AR_GEMM_SWIGLU, ctx->num_cus);
    AR_CHECK_ARG(need == 0 || (work && work_bytes >= need), "%s: work space of %zu bytes, needs %zu", what,
                 work ? work_bytes : (size_t)0, need);
    AR_CHECK_ARG(aligned_to(work, 16), "%s: the work space must be 16-byte aligned", what);
    if (ar_check_ptrs_enabled()) {
        AR_TRY(i8_check_ranges(A, what, "A"));
        AR_TRY(i8_check_ranges(W, what, "W"));
        if (W2) AR_TRY(i8_check_ranges(W2, what, "W2"));
        if (bias) AR_TRY(ar_check_range(bias, (size_t)W->rows * 4, what, "bias"));
        AR_TRY(float_rows_ranges(C, c_dtype, ldc, A->rows, W->rows, what, "C"));
        if (need) AR_TRY(ar_check_range(work, need, what, "work space"));
    }
    I8Params p{};
    p.a = A->q; p.sa = A->scale; p.lda = A->stride; p.w = W->q; p.sw = W->scale; p.ldw = W->stride;
    if (W2) { p.w2 = W2->q; p.sw2 = W2->scale; }
    p.M = A->rows; p.N = W->rows; p.K = K; p.bias = bias; p.c = C; p.ldc = ldc;
    switch (epilogue) {
        case AR_GEMM_STORE: return launch_types<GEMV_EPI_STORE>(p, c_dtype, work, ctx);
        case AR_GEMM_RESIDUAL: return launch_types<GEMV_EPI_RESIDUAL>(p, c_dtype, work, ctx);
        default: return launch_types<GEMV_EPI_SWIGLU>(p, c_dtype, work, ctx);
    }
}
