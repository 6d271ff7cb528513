// Causal attention of chunks of new tokens over a paged cache (include/ar_pages.h).
//
//   out_r = sum_j w_rj v_j / sum_j w_rj,   w_rj = exp(q_r k_j / sqrt(hd) - m_r),   j <= position of r, j on a page
//
// in one pass over the keys with a running maximum m and sum l.  The rows of a chunk's query heads that share a KV head
// are packed (row t * G + g: token t, head g of the group), so that a tile of 32 rows uses every key G times more often,
// and both products run on the matrix units, transposed, so that a lane owns one row and the weights feed the second
// product from the registers the first one left them in:
//   S^T (32 keys x 32 rows) = K Q^T    A: lane l has key l % 32, dims 16 s + 8 (l / 32) .. + 7 of step s
//   O^T (hd x 32 rows)     += V^T P^T  A: lane l has dim l % 32, keys 4 (l / 32) + 0..3 and 8 + those of each 16, the
//                                      order in which S^T leaves them; read transposed from V's rows in LDS
// 16-bit matrix units, more precise where the types are: a value of more bits is a sum of 16-bit planes, and products
// of planes whose sum of indexes stays below `depth` are added up (fp32 activations: 3 bf16 planes hold 24 bits; over
// an fp16 cache 2 fp16 planes of the query scaled into fp16's range hold 22, its weights scaled by 2^14 likewise).
#include <cmath>

#include "page_common.h"

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

struct PagedParams {
    const void* q;
    void* out;
    const char *kp, *vp;  // pools at the call's layer
    const int *table, *seq, *start, *at;
    int heads, kv_heads, group, seqs, max_pages, pages, shift, n, rows;
    float scale;          // log2(e) / sqrt(head_dim)
    int small_rows;       // chunks of at most this many packed rows are the few-row kernel's
    int slots, splits;
    float* part;          // [slots][kv_heads][splits][tile rows][hd] unnormalised outputs, then (m, l) of each
    float2* part_ml;
};

// 16-bit element of the matrix units: bf16, or fp16 for fp16 caches.
template <bool F16>
struct Elem;
template <>
struct Elem<false> {
    static __device__ __forceinline__ floatx16 mac(uint4 a, uint4 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    // two values rounded to nearest even, and what they stand for
    static __device__ __forceinline__ unsigned pack(float x, float y) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        const b2 v = {(__bf16)x, (__bf16)y};
        return __builtin_bit_cast(unsigned, v);
    }
    static __device__ __forceinline__ float low(unsigned u) { return __uint_as_float(u << 16); }
    static __device__ __forceinline__ float high(unsigned u) { return __uint_as_float(u & 0xFFFF0000u); }
    static constexpr unsigned kExponent = 0x7F80;
};
template <>
struct Elem<true> {
    static __device__ __forceinline__ floatx16 mac(uint4 a, uint4 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pack(float x, float y) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 v = {(_Float16)x, (_Float16)y};
        return __builtin_bit_cast(unsigned, v);
    }
    static __device__ __forceinline__ float low(unsigned u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)u); }
    static __device__ __forceinline__ float high(unsigned u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16)); }
    static constexpr unsigned kExponent = 0x7C00;
};

// N planes of two values: v = plane 0 + plane 1 + ...  (an infinity or NaN is in plane 0 alone)
template <bool F16, int N>
__device__ __forceinline__ void split2(float x, float y, unsigned* out) {
    typedef Elem<F16> E;
    out[0] = E::pack(x, y);
    if constexpr (N > 1) {
        x = fabsf(x) < INFINITY ? x - E::low(out[0]) : 0.f;
        y = fabsf(y) < INFINITY ? y - E::high(out[0]) : 0.f;
        out[1] = E::pack(x, y);
    }
    if constexpr (N > 2) out[2] = E::pack(x - E::low(out[1]), y - E::high(out[1]));
}

template <typename T>
struct Kind;
template <>
struct Kind<float> { static constexpr int id = AR_DTYPE_F32; };
template <>
struct Kind<__hip_bfloat16> { static constexpr int id = AR_DTYPE_BF16; };
template <>
struct Kind<_Float16> { static constexpr int id = AR_DTYPE_F16; };

constexpr int kThreads = 256, kWaves = 4;

// SMALL: a block takes 32 packed rows, and its wavefronts take key tiles in turn, each in an LDS space of its own.
// Otherwise it takes 128 rows, 32 a wavefront, and the wavefronts share each key tile.
template <int HD, typename QT, typename KT, bool SMALL>
struct Shape {
    static constexpr bool F16 = Kind<KT>::id == AR_DTYPE_F16, QF = Kind<QT>::id == AR_DTYPE_F32, KF = Kind<KT>::id == AR_DTYPE_F32;
    static constexpr int NQ = !QF ? 1 : F16 ? 2 : 3;      // planes of queries and of weights
    static constexpr int NK = !KF ? 1 : QF ? 3 : 2;       // planes of keys and values
    static constexpr int DEPTH = NQ > NK ? NQ : NK;       // plane pairs (i, j) with i + j < DEPTH are multiplied
    static constexpr int BK = SMALL || KF || NQ == 3 ? 32 : 64;  // keys of a tile
    static constexpr int ROWS = SMALL ? 32 : 128;         // packed rows of a block
    static constexpr int NT = SMALL ? 64 : kThreads;      // threads that share a key tile
    static constexpr int CPR = HD / 8;                    // 8-value pieces of a row
    static constexpr int UNITS = BK * CPR / NT;           // pieces of a tile per thread
    static constexpr int PLANE = BK * HD * 2;             // bytes of a plane of a tile
    static constexpr int TILE = NK * PLANE;
    static constexpr int SETS = SMALL ? kWaves : 2;       // SMALL: a space per wavefront; else one for K, one for V
    static constexpr int MERGE = SMALL ? 2 * 32 * HD * 4 : 0;  // two wavefronts' outputs
    static constexpr int LDS = SETS * TILE > MERGE ? SETS * TILE : MERGE;
    static constexpr int BLOCKS = SMALL && KF ? 1 : 2;   // of a CU, by registers and LDS
    static constexpr float BIAS = F16 ? 14.f : 0.f;       // weights scaled by 2^14 in fp16: their small ones keep bits
};

// What a block works on.
struct Task {
    int seq, first, count;  // chunk
    long long at;           // cache row of its first token
    int r0, rows;           // packed rows: first, and how many there are
    int units, per, active; // key tiles in all, in a split, splits that have any
};

// Slot, split -> task, by one wavefront (every wavefront of a block computes it for itself).
template <int ROWS, int BKS>
__device__ __forceinline__ bool find_task(const PagedParams& p, int slot, Task* t) {
    const int lane = threadIdx.x & 63;
    int chunk;
    if (!p.start) {
        const int tiles = (p.group + ROWS - 1) / ROWS;
        chunk = slot / tiles;
        t->r0 = (slot - chunk * tiles) * ROWS;
    } else if (ROWS == 32 && p.small_rows == 32) {  // chunks of one tile: a slot each
        chunk = slot;
    } else {
        chunk = chunk_search(p.n, 64, [&](int i, int k, int len) {
            const bool below = (long long)lane * k < len && chunk_slot(p.start[i + lane * k], i + lane * k, p.group, ROWS) <= slot;
            const unsigned long long m = __ballot(below);
            return m == ~0ull ? 64 : __builtin_ctzll(~m);
        });
        chunk = __builtin_amdgcn_readfirstlane(chunk);
    }
    if (chunk >= p.n) return false;
    chunk_rows(p.start, chunk, p.rows, &t->first, &t->count);
    if (p.start) {
        if (t->count == 0) return false;
        const long long tile = ROWS == 32 && p.small_rows == 32 ? 0 : slot - chunk_slot(t->first, chunk, p.group, ROWS);
        if (tile < 0 || tile * ROWS >= (long long)t->count * p.group) return false;
        t->r0 = (int)(tile * ROWS);
    }
    const long long packed = (long long)t->count * p.group;
    if (t->count == 0 || t->r0 >= packed) return false;
    if (ROWS == 128 ? packed <= p.small_rows : packed > p.small_rows) return false;
    t->rows = (int)(packed - t->r0 < ROWS ? packed - t->r0 : ROWS);
    t->seq = p.seq ? p.seq[chunk] : chunk;
    t->at = p.at[chunk];
    // keys that the last row sees
    const long long cap = (long long)p.max_pages << p.shift;
    long long end = t->at + (t->r0 + t->rows - 1) / p.group + 1;
    if (end > cap) end = cap;
    if (t->at < 0 || t->seq < 0 || t->seq >= p.seqs) end = 0;
    t->units = (int)((end + BKS - 1) / BKS);
    t->per = (t->units + p.splits - 1) / p.splits;
    if (t->per < 1) t->per = 1;
    t->active = (t->units + t->per - 1) / t->per;
    return true;
}

template <typename QT>
__device__ __forceinline__ void load8(const QT* p, float* v);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* v) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__hip_bfloat16>(const __hip_bfloat16* p, float* v) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const unsigned u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_float(__hip_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
__device__ __forceinline__ void store4(__hip_bfloat16* p, float a, float b, float c, float d) {
    *reinterpret_cast<uint2*>(p) = make_uint2(Elem<false>::pack(a, b), Elem<false>::pack(c, d));
}

template <int HD, typename QT, typename KT, bool SMALL>
__global__ __launch_bounds__(kThreads, (Shape<HD, QT, KT, SMALL>::BLOCKS)) void paged_tiles_kernel(PagedParams p) {
    typedef Shape<HD, QT, KT, SMALL> C;
    typedef Elem<C::F16> E;
    constexpr int NQ = C::NQ, NK = C::NK, BK = C::BK, KT32 = BK / 32, NJ = HD / 32, KS = HD / 16;
    __shared__ __attribute__((aligned(16))) char lds[C::LDS];
    __shared__ float s_m[kWaves][32], s_l[kWaves][32];
    __shared__ int s_bad;

    const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // KV head fastest (8 of them: one to an XCD, whose L2 then holds that head's rows), later rows, with more keys, first
    int b = blockIdx.x;
    const int kvh = b % p.kv_heads;
    b /= p.kv_heads;
    const int split = b % p.splits, slot = p.slots - 1 - b / p.splits;
    Task t;
    if (!find_task<C::ROWS, SMALL ? 4 * BK : BK>(p, slot, &t)) return;
    if (split >= (t.active > 0 ? t.active : 1)) return;

    const int row = t.r0 + (SMALL ? 0 : 32 * wave) + lq, packed = t.r0 + t.rows;  // row: packed, in the chunk
    const bool mine = row < packed;
    const int tok = mine ? row / p.group : 0, head = kvh * p.group + (mine ? row - tok * p.group : 0);
    const size_t qrow = ((size_t)(t.first + tok) * p.heads + head) * HD;
    const long long cap = (long long)p.max_pages << p.shift;
    const bool present = t.units > 0;
    // the last key a row sees; the block's and the wavefront's first and last rows'
    const int lim = !mine || !present ? -1 : (int)(t.at + tok < cap ? t.at + tok : cap - 1);
    const int w0 = t.r0 + (SMALL ? 0 : 32 * wave), w1 = (w0 + 31 < packed ? w0 + 31 : packed - 1);
    const bool idle = w0 >= packed;
    const int lim0 = idle || !present ? -1 : (int)(t.at + w0 / p.group < cap ? t.at + w0 / p.group : cap - 1);
    const int lim1 = idle || !present ? -1 : (int)(t.at + w1 / p.group < cap ? t.at + w1 / p.group : cap - 1);
    const int blim0 = !present ? -1 : (int)(t.at + t.r0 / p.group < cap ? t.at + t.r0 / p.group : cap - 1);
    const int kend = !present ? 0 : (int)(t.at + (packed - 1) / p.group < cap ? t.at + (packed - 1) / p.group : cap - 1) + 1;

    // queries: planes in registers, rows of an fp16 cache's scaled into its range
    uint4 qf[NQ][KS];
    float c = p.scale;
    {
        const QT* q = (const QT*)p.q + qrow;
        float v[KS][8];
#pragma unroll
        for (int s = 0; s < KS; s++) {
            if (mine) load8<QT>(q + 16 * s + 8 * h, v[s]);
            else
#pragma unroll
                for (int i = 0; i < 8; i++) v[s][i] = 0.f;
        }
        if constexpr (C::F16) {
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[s][i]));
            top = max_xor32(top);
            int e = 0;
            if (top > 0.f && top < INFINITY) e = min(14 - ilogbf(top), 100);  // the largest in [2^14, 2^15)
            c = ldexpf(c, -e);
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) v[s][i] = ldexpf(v[s][i], e);
        }
#pragma unroll
        for (int s = 0; s < KS; s++) {
            unsigned u[4][NQ];
#pragma unroll
            for (int i = 0; i < 4; i++) split2<C::F16, NQ>(v[s][2 * i], v[s][2 * i + 1], u[i]);
#pragma unroll
            for (int n = 0; n < NQ; n++) qf[n][s] = make_uint4(u[0][n], u[1][n], u[2][n], u[3][n]);
        }
    }

    floatx16 o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[j][r] = 0.f;
    float m = -INFINITY, l = 0.f;

    // key tiles of this split (SMALL: of this wavefront)
    const int step = SMALL ? kWaves : 1;
    const int t0 = SMALL ? split * t.per * kWaves + wave : split * t.per;
    const int t1 = min((split + 1) * t.per * step, (kend + BK - 1) / BK);
    const int* table = p.table + (size_t)(t.seq < 0 ? 0 : t.seq) * p.max_pages;
    const int pmask = (1 << p.shift) - 1;

    char* const kbuf = lds + (SMALL ? wave * C::TILE : 0);
    char* const vbuf = SMALL ? kbuf : lds + C::TILE;
    const int stid = SMALL ? lane : tid;
    // swizzles of 16-byte pieces in a row: K, 16 rows of one column over all banks; V, 4 rows of 4 columns
    const int kx = HD == 128 ? lq & 15 : (lq >> 1) & 7;
    const unsigned kaddr = lq * (HD * 2) + ((h ^ kx) * 16);
    const int i16 = lane & 15, vrow = 4 * h + (i16 >> 2);
    const int vx = HD == 128 ? (vrow & 3) << 2 : ((vrow >> 1) & 1) << 2;
    const unsigned vaddr = vrow * (HD * 2) + (((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ vx) * 16) + (i16 & 1) * 8;

    // A wavefront's 64 pieces of a load lie in 64 / CPR rows of one page (its first row is a multiple of that, and pages
    // are longer), so that all but a fixed offset of each lane's address is the same for the wavefront.
    constexpr int ROW = HD * (int)sizeof(KT);
    uint4 st[C::UNITS * (C::KF ? 2 : 1)];
    const unsigned lane_at = (lane / C::CPR) * ROW + (lane % C::CPR) * (8 * (int)sizeof(KT));
    int pg0 = -1, pg1 = -1, pg2 = -1, pg3 = -1;
    auto page_at = [&](int k0, int i) __attribute__((always_inline)) {
        const int key = k0 + (i << p.shift);
        int g = -1;
        if ((i << p.shift) < BK && key < kend) g = table[key >> p.shift];
        return g >= 0 && g < p.pages ? g : -1;
    };
    auto load_pages = [&](int tile) __attribute__((always_inline)) {
        const int k0 = tile * BK;
        pg0 = page_at(k0, 0);
        pg1 = page_at(k0, 1);
        if constexpr (BK > 32) {
            pg2 = page_at(k0, 2);
            pg3 = page_at(k0, 3);
        }
    };
    // (a row on no page: some row of the pool in its place; keys are hidden by their scores, values zeroed below)
    auto stage_load = [&](int tile, const char* pool) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < C::UNITS; u++) {
            const int row0 = (u * C::NT + (SMALL ? 0 : wave * 64)) / C::CPR, i = row0 >> p.shift;
            int page = i == 0 ? pg0 : i == 1 ? pg1 : i == 2 ? pg2 : pg3;
            page = page < 0 ? 0 : page;
            const char* src = pool + ((((size_t)page * p.kv_heads + kvh) << p.shift) + ((tile * BK + row0) & pmask)) * ROW;
            if constexpr (C::KF) {
                st[2 * u] = *reinterpret_cast<const uint4*>(src + lane_at);
                st[2 * u + 1] = *reinterpret_cast<const uint4*>(src + lane_at + 16);
            } else {
                st[u] = *reinterpret_cast<const uint4*>(src + lane_at);
            }
        }
    };
    auto stage_store = [&](char* buf, bool values) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < C::UNITS; u++) {
            const int piece = u * C::NT + stid, key = piece / C::CPR, col = piece % C::CPR;
            const int x = values ? (HD == 128 ? (key & 3) << 2 : ((key >> 1) & 1) << 2) : (HD == 128 ? key & 15 : (key >> 1) & 7);
            char* dst = buf + key * (HD * 2) + ((col ^ x) * 16);
            if constexpr (C::KF) {
                const uint4 a = st[2 * u], d = st[2 * u + 1];
                const unsigned w[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
                unsigned pl[4][NK];
#pragma unroll
                for (int i = 0; i < 4; i++) split2<false, NK>(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), pl[i]);
#pragma unroll
                for (int n = 0; n < NK; n++)
                    *reinterpret_cast<uint4*>(dst + n * C::PLANE) = make_uint4(pl[0][n], pl[1][n], pl[2][n], pl[3][n]);
            } else {
                *reinterpret_cast<uint4*>(dst) = st[u];
            }
        }
    };
    // Zeros the staged values of rows on no page or behind the last key, and leaves infinities and NaN out of the others;
    // whether there were any.  A hidden key's weight of 0 times one of them would reach rows that do not see it.
    auto leave_out = [&](int k0, unsigned long long miss) __attribute__((always_inline)) {
        unsigned bad = 0;
#pragma unroll
        for (int u = 0; u < C::UNITS; u++) {
            const int key = (u * C::NT + (SMALL ? 0 : wave * 64)) / C::CPR + lane / C::CPR;
            if (k0 + key >= kend || (miss >> key & 1)) {
                st[C::KF ? 2 * u : u] = make_uint4(0, 0, 0, 0);
                if constexpr (C::KF) st[2 * u + 1] = make_uint4(0, 0, 0, 0);
            }
        }
        auto clean = [&](unsigned& w) __attribute__((always_inline)) {
            unsigned gone;
            if constexpr (C::KF) gone = (w & 0x7F800000u) == 0x7F800000u ? ~0u : 0u;
            else gone = ((w & E::kExponent) == E::kExponent ? 0xFFFFu : 0u) | ((w >> 16 & E::kExponent) == E::kExponent ? 0xFFFF0000u : 0u);
            w &= ~gone;
            bad |= gone;
        };
#pragma unroll
        for (int u = 0; u < C::UNITS * (C::KF ? 2 : 1); u++) {
            clean(st[u].x);
            clean(st[u].y);
            clean(st[u].z);
            clean(st[u].w);
        }
        return bad != 0;
    };
    auto tile_sync = [&]() __attribute__((always_inline)) {
        if constexpr (SMALL) {
            // one wavefront's own LDS space: its accesses are served in order
            asm volatile("" ::: "memory");
            __builtin_amdgcn_wave_barrier();
        } else {
            __syncthreads();
        }
    };

    if constexpr (!SMALL) {
        if (tid == 0) s_bad = -1;
    }
    if (t0 < t1) {
        load_pages(t0);
        stage_load(t0, p.kp);
    }
    for (int tile = t0; tile < t1; tile += step) {
        const int k0 = tile * BK;
        unsigned long long miss = 0;  // keys of the tile that lie on no page
        const unsigned long long page_keys = p.shift >= 6 ? ~0ull : (1ull << (1 << p.shift)) - 1;
        if (pg0 < 0) miss |= page_keys;
        if (pg1 < 0 && (1 << p.shift) < BK) miss |= page_keys << ((1 << p.shift) & 63);
        if (pg2 < 0 && (2 << p.shift) < BK) miss |= page_keys << ((2 << p.shift) & 63);
        if (pg3 < 0 && (3 << p.shift) < BK) miss |= page_keys << ((3 << p.shift) & 63);
        const bool masked = miss != 0 || k0 + BK - 1 > blim0;  // some row of the block does not see all of it
        stage_store(kbuf, false);
        stage_load(tile, p.vp);
        load_pages(tile + step);  // (past the split's end: not used)
        tile_sync();

        const bool work = k0 <= lim1;
        floatx16 s[KT32];
        if (work) {
#pragma unroll
            for (int kt = 0; kt < KT32; kt++) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[kt][r] = 0.f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
#pragma unroll
                    for (int j = 0; j < NK; j++) {
                        const uint4 kf = *reinterpret_cast<const uint4*>(kbuf + j * C::PLANE + kt * 32 * HD * 2 + (kaddr ^ (ks * 32)));
#pragma unroll
                        for (int i = 0; i < NQ; i++)
                            if (i + j < C::DEPTH) s[kt] = E::mac(kf, qf[i][ks], s[kt]);
                    }
                }
            }
            if (k0 + BK - 1 > lim0) {  // (the lane's keys are 32 kt + 8 (r / 4) + r % 4, and 4 h)
                const int last = lim - k0 - 4 * h;
#pragma unroll
                for (int kt = 0; kt < KT32; kt++)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (32 * kt + 8 * (r >> 2) + (r & 3) > last) s[kt][r] = -INFINITY;
            }
            if (miss != 0) {
#pragma unroll
                for (int kt = 0; kt < KT32; kt++) {
                    const unsigned gone = (unsigned)(miss >> (32 * kt)) >> (4 * h);
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (gone >> (8 * (r >> 2) + (r & 3)) & 1) s[kt][r] = -INFINITY;
                }
            }
            float mx = s[0][0];
#pragma unroll
            for (int kt = 0; kt < KT32; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[kt][r]);
            mx = max_xor32(mx) * c;
            if (__ballot(mx > m)) {
                const float mn = fmaxf(m, mx);
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
                l *= alpha;
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[j][r] *= alpha;
                m = mn;
            }
            // (a row that has seen no key yet keeps m = -inf: weights 0)
            const float mu = m == -INFINITY ? 0.f : m - C::BIAS;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kt = 0; kt < KT32; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[kt][r] = __builtin_amdgcn_exp2f(fmaf(s[kt][r], c, -mu));
                    sum[r & 3] += s[kt][r];
                }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);  // this lane's half of the keys
        }
        bool bad = false;
        if (masked) {
            bad = leave_out(k0, miss);
            if constexpr (SMALL) bad = __ballot(bad) != 0;
            else if (bad) s_bad = tile;
        }
        stage_store(vbuf, true);
        const int next = tile + step;
        if (next < t1) stage_load(next, p.kp);
        tile_sync();
        if constexpr (!SMALL) bad = masked && s_bad == tile;
        if (work) {
#pragma unroll
            for (int kt = 0; kt < KT32; kt++)
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) {
                    if (NQ > 1) __builtin_amdgcn_sched_barrier(0);  // one step's planes at a time: registers
                    unsigned u[4][NQ];
#pragma unroll
                    for (int i = 0; i < 4; i++) split2<C::F16, NQ>(s[kt][8 * k2 + 2 * i], s[kt][8 * k2 + 2 * i + 1], u[i]);
                    uint4 pf[NQ];
#pragma unroll
                    for (int n = 0; n < NQ; n++) pf[n] = make_uint4(u[0][n], u[1][n], u[2][n], u[3][n]);
#pragma unroll
                    for (int jt = 0; jt < NJ; jt++)
#pragma unroll
                        for (int j = 0; j < NK; j++) {
                            const char* a = vbuf + j * C::PLANE + (vaddr ^ (jt * 64)) + (32 * kt + 16 * k2) * (HD * 2);
                            typedef __attribute__((address_space(3))) shortx4 lds4;
                            const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)a);
                            const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(a + 8 * HD * 2));
                            const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
                            const uint4 vf = make_uint4(x.x, x.y, y.x, y.y);
#pragma unroll
                            for (int i = 0; i < NQ; i++)
                                if (i + j < C::DEPTH) o[jt] = E::mac(vf, pf[i], o[jt]);
                        }
                }
            if (__builtin_expect(bad, 0)) {
                // the values that were left out: their weights are positive, so that each is its own contribution
#pragma unroll 1
                for (int key = 0; key < BK && k0 + key < kend; key++) {
                    const int page = __builtin_amdgcn_readfirstlane(page_of_row(p.table, p.seqs, p.max_pages, p.pages, p.shift, t.seq, k0 + key));
                    if (page < 0) continue;
                    const KT* v = (const KT*)p.vp + ((((size_t)page * p.kv_heads + kvh) << p.shift) + ((k0 + key) & pmask)) * HD + 4 * h;
                    const bool seen = k0 + key <= lim;
#pragma unroll
                    for (int j = 0; j < NJ; j++)
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const float x = to_float(v[32 * j + 8 * (r >> 2) + (r & 3)]);
                            if (seen && !(fabsf(x) < INFINITY)) o[j][r] += x;
                            if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // few loads at a time: registers
                        }
                }
            }
        }
        if constexpr (SMALL) tile_sync();
    }
    l = sum_xor32(l);

    if constexpr (SMALL) {  // the wavefronts' states: a common maximum, then the sums of 2 + 3 into 0 + 1, of 1 into 0
        if (h == 0) s_m[wave][lq] = m;
        __syncthreads();
        float mm = s_m[0][lq];
#pragma unroll
        for (int w = 1; w < kWaves; w++) mm = fmaxf(mm, s_m[w][lq]);
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mm);
        l *= f;
        m = mm;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[j][r] *= f;
        if (h == 0) s_l[wave][lq] = l;
        float* const mine_o = reinterpret_cast<float*>(lds) + lane;
#pragma unroll
        for (int half = 2; half > 0; half /= 2) {
            __syncthreads();
            if (wave >= half && wave < 2 * half)
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) mine_o[(((wave - half) * NJ + j) * 16 + r) * 64] = o[j][r];
            __syncthreads();
            if (wave < half)
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[j][r] += mine_o[((wave * NJ + j) * 16 + r) * 64];
        }
        if (wave > 0) return;
        l = (s_l[0][lq] + s_l[1][lq]) + (s_l[2][lq] + s_l[3][lq]);
    }
    if (!mine) return;
    if (t.active <= 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        QT* out = (QT*)p.out + qrow;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                store4(out + 32 * j + 2 * r + 4 * h, o[j][r] * inv, o[j][r + 1] * inv, o[j][r + 2] * inv, o[j][r + 3] * inv);
    } else {
        const size_t at = (((size_t)slot * p.kv_heads + kvh) * p.splits + split) * C::ROWS + (row - t.r0);
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                store4(p.part + at * HD + 32 * j + 2 * r + 4 * h, o[j][r], o[j][r + 1], o[j][r + 2], o[j][r + 3]);
        if (h == 0) p.part_ml[at] = make_float2(m, l);
    }
}

// The splits of a row, in their order.  A block takes four rows of a task.
template <int HD, typename QT, int ROWS, int BKS>
__global__ __launch_bounds__(4 * HD) void paged_merge_kernel(PagedParams p) {
    int b = blockIdx.x;
    const int kvh = b % p.kv_heads;
    b /= p.kv_heads;
    const int quad = b % (ROWS / 4), slot = b / (ROWS / 4);
    Task t;
    if (!find_task<ROWS, BKS>(p, slot, &t) || t.active <= 1) return;
    const int r = 4 * quad + threadIdx.x / HD, d = threadIdx.x % HD;
    if (r >= t.rows) return;
    const size_t at = (((size_t)slot * p.kv_heads + kvh) * p.splits) * ROWS + r;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int s = 0; s < t.active; s++) m = fmaxf(m, p.part_ml[at + (size_t)s * ROWS].x);
    for (int s = 0; s < t.active; s++) {
        const float2 ml = p.part_ml[at + (size_t)s * ROWS];
        const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m);
        l = fmaf(ml.y, f, l);
        // (a split without a visible key holds zeros)
        o = fmaf(p.part[(at + (size_t)s * ROWS) * HD + d], f, o);
    }
    const int row = t.r0 + r, tok = row / p.group, head = kvh * p.group + row - tok * p.group;
    const float v = l == 0.f ? 0.f : o / l;
    QT* out = (QT*)p.out + ((size_t)(t.first + tok) * p.heads + head) * HD + d;
    if constexpr (sizeof(QT) == 4) *reinterpret_cast<float*>(out) = v;
    else *reinterpret_cast<uint16_t*>(out) = (uint16_t)bf16_rne_bits(v);
}

// ---- host side ----------------------------------------------------------------------------------------------

// The launches of a call.  Chunks of few packed rows go to the few-row kernel, which splits a chunk's keys over the
// wavefronts of a block too; where the call's rows are few for its chunks, all of them do.
struct Plan {
    bool small = false, big = false;
    int small_rows = 0;                 // the few-row kernel's chunks
    int small_slots = 0, small_splits = 1, big_slots = 0, big_splits = 1;
    size_t bytes = 16;
};

size_t part_bytes(const ar_pages* p, int slots, int splits, int rows) {
    return splits <= 1 ? 0 : (size_t)slots * p->kv_heads * splits * rows * ((size_t)p->head_dim * 4 + 8);
}

int splits_for(const ar_pages* p, int slots, int per_cu, int cus, int keys) {
    const long long cap = (long long)p->max_pages * p->page_rows, most = (cap + keys - 1) / keys;
    const long long want = ((long long)per_cu * cus + (long long)slots * p->kv_heads - 1) / ((long long)slots * p->kv_heads);
    return (int)std::max(1LL, std::min(std::min(want, most), 64LL));
}

int plan_of(const ar_hip_ctx* ctx, const ar_pages* p, const ar_chunks* c, int heads, Plan* out) {
    const long long group = heads / p->kv_heads, packed = (long long)c->rows * group;
    Plan a;
    AR_CHECK_ARG(packed <= 1 << 30, "paged attention: %d rows of %lld heads per KV head are too many", c->rows, group);
    if (!c->start || packed <= 32LL * c->n) {
        a.small = true;
        a.small_rows = 0x7fffffff;
        const long long slots = !c->start ? (long long)c->n * ((group + 31) / 32) : packed / 32 + c->n;
        AR_CHECK_ARG(slots * p->kv_heads <= 0x7fffffffLL / 64, "paged attention: %d rows of %d heads are too many", c->rows,
                     heads);
        a.small_slots = (int)slots;
    } else {
        a.big = true;
        const long long slots = packed / 128 + c->n;
        AR_CHECK_ARG(slots * p->kv_heads <= 0x7fffffffLL / 64, "paged attention: %d rows of %d heads are too many", c->rows,
                     heads);
        a.big_slots = (int)slots;
        if (c->n > 1) {
            a.small = true;
            a.small_rows = 32;
            a.small_slots = c->n;
        }
    }
    if (a.small) a.small_splits = splits_for(p, std::min(a.small_slots, c->n * (int)((group + 31) / 32)), 2, ctx->num_cus, 128);
    if (a.big) a.big_splits = splits_for(p, a.big_slots, 2, ctx->num_cus, 128);
    a.bytes = std::max<size_t>(16, part_bytes(p, a.small_slots, a.small_splits, 32) + part_bytes(p, a.big_slots, a.big_splits, 128));
    *out = a;
    return AR_HIP_OK;
}

template <int HD, typename QT, typename KT, bool SMALL>
int launch_tiles(PagedParams p, int slots, int splits, char* work, hipStream_t st) {
    typedef Shape<HD, QT, KT, SMALL> C;
    p.slots = slots;
    p.splits = splits;
    const size_t rows = (size_t)slots * p.kv_heads * splits * C::ROWS;
    p.part = (float*)work;
    p.part_ml = (float2*)(work + rows * HD * 4);
    hipLaunchKernelGGL((paged_tiles_kernel<HD, QT, KT, SMALL>), dim3((unsigned)((long long)slots * p.kv_heads * splits)),
                       dim3(kThreads), 0, st, p);
    AR_LAUNCH_CHECK();
    if (splits > 1) {
        hipLaunchKernelGGL((paged_merge_kernel<HD, QT, C::ROWS, SMALL ? 4 * C::BK : C::BK>),
                           dim3((unsigned)((long long)slots * p.kv_heads * (C::ROWS / 4))), dim3(4 * HD), 0, st, p);
        AR_LAUNCH_CHECK();
    }
    return AR_HIP_OK;
}

template <int HD, typename QT, typename KT>
int launch_plan(const Plan& a, const PagedParams& p, char* work, size_t big_at, hipStream_t st) {
    if (a.big) AR_TRY((launch_tiles<HD, QT, KT, false>(p, a.big_slots, a.big_splits, work + big_at, st)));
    if (a.small) AR_TRY((launch_tiles<HD, QT, KT, true>(p, a.small_slots, a.small_splits, work, st)));
    return AR_HIP_OK;
}

template <int HD, typename QT>
int launch_kt(int dtype, const Plan& a, const PagedParams& p, char* work, size_t big_at, hipStream_t st) {
    if (dtype == AR_DTYPE_F32) return launch_plan<HD, QT, float>(a, p, work, big_at, st);
    if (dtype == AR_DTYPE_F16) return launch_plan<HD, QT, _Float16>(a, p, work, big_at, st);
    return launch_plan<HD, QT, __hip_bfloat16>(a, p, work, big_at, st);
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
    Plan a;
    AR_TRY(plan_of(ctx, pages, chunks, heads, &a));
    *bytes = a.bytes;
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
    Plan a;
    AR_TRY(plan_of(ctx, pages, chunks, heads, &a));
    AR_CHECK_ARG(work && work_bytes >= a.bytes, "%s: %zu bytes of work space given, %zu needed", what, work ? work_bytes : 0, a.bytes);
    const int hd = pages->head_dim;
    const size_t act = act_dtype == AR_DTYPE_F32 ? 4 : 2, bytes = (size_t)chunks->rows * heads * hd * act;
    if (ar_check_ptrs_enabled()) {
        AR_TRY(page_check_ranges(pages, what));
        AR_TRY(page_check_chunk_ranges(chunks, what));
        AR_TRY(ar_check_range(q, bytes, what, "queries"));
        AR_TRY(ar_check_range(out, bytes, what, "output"));
        AR_TRY(ar_check_range(work, a.bytes, what, "work space"));
    }
    const size_t layer_bytes = (size_t)pages->pages * pages->kv_heads * hd * pages->page_rows * page_elem_bytes(pages->dtype);
    PagedParams p{};
    p.q = q; p.out = out;
    p.kp = (const char*)pages->k + layer * layer_bytes;
    p.vp = (const char*)pages->v + layer * layer_bytes;
    p.table = pages->table; p.seq = chunks->seq; p.start = chunks->start; p.at = chunks->at; p.heads = heads;
    p.kv_heads = pages->kv_heads; p.group = heads / pages->kv_heads; p.seqs = pages->seqs;
    p.max_pages = pages->max_pages; p.pages = pages->pages; p.shift = page_shift_of(pages); p.n = chunks->n;
    p.rows = chunks->rows; p.small_rows = a.small_rows;
    p.scale = (float)(1.4426950408889634 / std::sqrt((double)hd));
    const size_t big_at = part_bytes(pages, a.small_slots, a.small_splits, 32);
    char* const w = (char*)work;
    if (hd == 128)
        return act == 4 ? launch_kt<128, float>(pages->dtype, a, p, w, big_at, ctx->stream)
                        : launch_kt<128, __hip_bfloat16>(pages->dtype, a, p, w, big_at, ctx->stream);
    return act == 4 ? launch_kt<64, float>(pages->dtype, a, p, w, big_at, ctx->stream)
                    : launch_kt<64, __hip_bfloat16>(pages->dtype, a, p, w, big_at, ctx->stream);
}
