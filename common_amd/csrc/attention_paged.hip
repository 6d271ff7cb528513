// Causal attention of chunks of new tokens over a paged cache (include/ar_pages.h).
//
//   out_r = sum_j w_rj v_j / sum_j w_rj,   w_rj = exp(q_r k_j / sqrt(hd) - m_r),   j <= position of r, j on a page
//
// in one pass over the keys with a running maximum m and sum l.  The rows of a chunk's query heads that share a KV head
// are packed (row t * G + g: token t, head g of the group), so that a tile of rows uses every key G times more often.
// Two kernels share the work by a chunk's packed rows: the tile kernel (many rows, bound by the matrix units and by the
// softmax's vector instructions) and the few-row kernel (decode steps, bound by HBM); where the keys are cut among
// blocks, a merge kernel adds the parts up in a fixed order.
//
// Both products run on the matrix units, transposed, so that a lane owns one row and the weights feed the second
// product from the registers the first one left them in:
//   S^T (32 keys x 32 rows) = K Q^T    A: lane l has key l % 32, dims 16 s + 8 (l / 32) .. + 7 of step s
//   O^T (hd x 32 rows)     += V^T P^T  A: lane l has dim l % 32, keys 4 (l / 32) + 0..3 and 8 + those of each 16, the
//                                      order in which S^T leaves them; read transposed from V's rows in LDS
// 16-bit matrix units, more precise where the types are: a value of more bits is a sum of 16-bit planes, and products
// of planes whose sum of indexes stays below `depth` are added up.
//   bf16 activations:           one plane of the query (scaled into fp16's range over fp16 and fp32 caches) and one of
//                               the weights: rounded to 8 or 11 bits, no more than the output's own rounding
//   fp32 over a bf16 cache:     3 bf16 planes of the query and the weights hold 24 bits
//   fp32 over an fp16 cache:    2 fp16 planes hold 22; the query is scaled by a power of two so that its largest value
//                               is near 2^14, the weights by 2^6 (and 2^kSlack while the maximum lags): what is below
//                               2^-24 of fp16's scale is lost, 2^-30 of a row's largest weight
//   fp32 caches (tile kernel):  2 fp16 planes of keys and values, too, each row with its own power of two
//   fp32 caches (few rows):     fp32 matrix instructions; HBM bounds them all the same
// Three plane products at 1,100 TFLOP/s beat one at the fp32 units' 154.
#include <cmath>

#include "page_common.h"
#include "page_tasks.h"

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));  // (staged values stay in registers)
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x4 quad(unsigned a, unsigned b, unsigned c, unsigned d) { return u32x4{a, b, c, d}; }

// One kernel's share of a call.
struct PartArgs {
    int tiles, tasks;     // at most
    int target, blocks;   // how many tasks to cut the keys for (0: a tile is a task), and how many they may become
    float* part;          // [tasks][kv_heads][tile rows][hd] unnormalised outputs of splits, and (m, l) of each
    float2* part_ml;
};

struct PagedParams {
    const void* q;
    void* out;
    const char *kp, *vp;  // pools at the call's layer
    const int *table, *seq, *start, *at;
    int heads, kv_heads, group, seqs, max_pages, pages, shift, n, rows;
    float scale;          // log2(e) / sqrt(head_dim)
    int few_rows;         // chunks of at most this many packed rows are the few-row kernel's
    int merge_rows;       // of a tile, that a merging block takes
    PartArgs few, tile;
};

// 16-bit element of the matrix units: bf16, or fp16 for fp16 caches.
template <bool F16>
struct Elem;
template <>
struct Elem<false> {
    static __device__ __forceinline__ floatx16 mac(u32x4 a, u32x4 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx4 mac16(u32x4 a, u32x4 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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
    static __device__ __forceinline__ floatx16 mac(u32x4 a, u32x4 b, floatx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ floatx4 mac16(u32x4 a, u32x4 b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
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

// N planes of two values: v = plane 0 + plane 1 + ...  (SPECIAL: an infinity or NaN is in plane 0 alone)
template <bool F16, int N, bool SPECIAL>
__device__ __forceinline__ void split2(float x, float y, unsigned* out) {
    typedef Elem<F16> E;
    out[0] = E::pack(x, y);
    if constexpr (N > 1) {
        const bool fx = !SPECIAL || fabsf(x) < INFINITY, fy = !SPECIAL || fabsf(y) < INFINITY;
        x = fx ? x - E::low(out[0]) : 0.f;
        y = fy ? y - E::high(out[0]) : 0.f;
        out[1] = E::pack(x, y);
    }
    if constexpr (N > 2) out[2] = E::pack(x - E::low(out[1]), y - E::high(out[1]));
}

// Two fp16 planes of a value times a power of two, each in one mixed-precision multiply-add per value.
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split2_scaled(float x, float y, float scale, unsigned* out) {
    const halfx2 a = {(_Float16)fmaf(x, scale, 0.f), (_Float16)fmaf(y, scale, 0.f)};
    const halfx2 b = {(_Float16)fmaf(x, scale, -(float)a.x), (_Float16)fmaf(y, scale, -(float)a.y)};
    out[0] = __builtin_bit_cast(unsigned, a);
    out[1] = __builtin_bit_cast(unsigned, b);
}

// The same of the values themselves; `one` is 1, and the compiler not to know it.
__device__ __forceinline__ void split2_mixed(float x, float y, float one, unsigned* out) {
    const halfx2 a = {(_Float16)x, (_Float16)y};
    out[0] = __builtin_bit_cast(unsigned, a);
    asm("" : "+v"(out[0]));  // (not converted a second time for the difference)
    const halfx2 c = __builtin_bit_cast(halfx2, out[0]);
    const halfx2 b = {(_Float16)fmaf(x, one, -(float)c.x), (_Float16)fmaf(y, one, -(float)c.y)};
    out[1] = __builtin_bit_cast(unsigned, b);
}

// fp32 products: a (bits) x b, 16 x 16 x 4
__device__ __forceinline__ floatx4 mac4f(unsigned a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a), b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mac4(unsigned a, unsigned b, floatx4 c) { return mac4f(a, __uint_as_float(b), c); }

// Power of two that brings a row whose largest finite value is `top` into fp16's range, its largest to [2^14, 2^15); at
// most 2^122, also for a row of zeros (a row of values below 2^-108 to less, one below 2^-122 with fewer bits; and a
// score's scale times its inverse is still a normal number).
__device__ __forceinline__ int fp16_shift(float top) { return min(141 - (int)(__float_as_uint(top) >> 23), 122); }

// maximum over the LANES (8 or 16) lanes that hold a row; of values >= 0, as their bits (which need no canonical form)
template <int LANES>
__device__ __forceinline__ float row_max(float value) {
    unsigned v = __float_as_uint(value);
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));   // quad_perm 1,0,3,2
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));   // quad_perm 2,3,0,1
    v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));  // row_half_mirror
    if (LANES == 16) v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));  // row_mirror
    return __uint_as_float(v);
}

// A piece of values (of fp32 or 16-bit ones) with zeros for infinities and NaN, which a hidden key's weight of 0 would
// carry into rows that do not see them; *any becomes nonzero if there were some.
template <bool KF, bool F16>
__device__ __forceinline__ u32x4 drop_special(u32x4 v, unsigned* any) {
    constexpr unsigned x = Elem<F16>::kExponent;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned gone;
        if constexpr (KF) gone = (v[i] & 0x7F800000u) == 0x7F800000u ? ~0u : 0u;
        else gone = ((v[i] & x) == x ? 0xFFFFu : 0u) | ((v[i] >> 16 & x) == x ? 0xFFFF0000u : 0u);
        v[i] &= ~gone;
        *any |= gone;
    }
    return v;
}
// The same for a piece in LDS, all of it where `out`.
template <bool F16>
__device__ __forceinline__ unsigned leave_out(u32x4* at, bool out) {
    unsigned gone = 0;
    const u32x4 v = drop_special<false, F16>(*at, &gone);
    if (out || gone) *at = out ? quad(0, 0, 0, 0) : v;
    return out ? 0u : gone;
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
// The tile kernel's maximum of a row may lag behind by this power of two: weights up to 2^kSlack (fp16: 2^14); what a
// lane's weights of a tile may add up to without a look at their maximum.
constexpr float kSlack = 8.f, kBound = 16384.f;

// Planes and sizes of a (head size, activation, cache) combination.
template <int HD, typename QT, typename KT>
struct Shape {
    static constexpr bool QF = Kind<QT>::id == AR_DTYPE_F32, KF = Kind<KT>::id == AR_DTYPE_F32;
    static constexpr bool F16 = Kind<KT>::id != AR_DTYPE_BF16;
    static constexpr int NQ = !QF ? 1 : F16 ? 2 : 3;      // planes of queries and of weights
    static constexpr int NK = KF ? 2 : 1;                 // planes of keys and values
    static constexpr int DEPTH = NQ > NK ? NQ : NK;       // plane pairs (i, j) with i + j < DEPTH are multiplied
    static constexpr int CPR = HD / 8;                    // 8-value pieces of a row
    // the tile kernel: 128 packed rows a block, 32 a wavefront, key tiles of BK shared by the block
    static constexpr int ROWS = 128;
    static constexpr int BK = KF || NQ == 3 ? 32 : 64;
    static constexpr int UNITS = BK * CPR / kThreads;     // pieces of a tile per thread
    static constexpr int PLANE = BK * HD * 2;             // bytes of a plane of a tile
    static constexpr int TILE = NK * PLANE;
    static constexpr float BIAS = F16 ? 6.f : 0.f;  // weights scaled by 2^6 in fp16, and kSlack more: their small ones keep bits
};

// ---- what a block works on (page_tasks.h) -----------------------------------------------------------------------
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// The table is read with scalar loads: nothing writes it while these kernels run.
typedef const __attribute__((address_space(4))) int* TableRow;
__device__ __forceinline__ TableRow table_row(const PagedParams& p, int seq) {
    return (TableRow)(uintptr_t)(p.table + (size_t)(seq < 0 || seq >= p.seqs ? 0 : seq) * p.max_pages);
}

// Chunk i's rows, sequence and place; the number of its tiles (0: not this kernel's, or i past the last chunk).
template <int ROWS>
__device__ __forceinline__ int chunk_tiles(const PagedParams& p, int i, Task* t) {
    const int j = min(i, p.n - 1);
    // (all loads at once)
    const int a = p.start ? p.start[j] : j, b = p.start ? p.start[j + 1] : j + 1;
    const int at = p.at[j], seq = p.seq ? p.seq[j] : j;
    return tiles_of_chunk<ROWS>(p, a, i < p.n ? b : a, at, seq, t);
}

// Sum over the lanes up to and with this one (row shifts, then row broadcasts).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Task `index` (MERGE: tile `index` and its first task) -> *t, by one wavefront; every wavefront of a block computes it
// for itself, without LDS: it is the first thing that a block waits for.
template <int ROWS, bool MERGE>
__device__ __forceinline__ bool find_task(const PagedParams& p, int index, Task* t) {
    const int target = ROWS == 16 ? p.few.target : p.tile.target;
    const int lane = threadIdx.x & 63;
    int tile = 0;
    if (target == 0) {
        const int per_chunk = (p.group + ROWS - 1) / ROWS;
        const int chunk = !p.start ? index / per_chunk : chunk_search(p.n, 64, [&](int i, int k, int len) {
            const bool below = (long long)lane * k < len && chunk_slot(p.start[i + lane * k], i + lane * k, p.group, ROWS) <= index;
            const unsigned long long m = __ballot(below);
            return m == ~0ull ? 64 : __builtin_ctzll(~m);
        });
        const int tiles = chunk_tiles<ROWS>(p, chunk, t);
        const long long at = !p.start ? index % per_chunk : index - chunk_slot(t->first, chunk, p.group, ROWS);
        if (at < 0 || at >= tiles) return false;
        tile = (int)at;
        t->per = t->units > 0 ? t->units : 1;
        t->splits = 1;
        t->split = 0;
        t->base = index;
    } else {
        // (of up to 64 chunks each lane keeps its own)
        Task c;
        int n = chunk_tiles<ROWS>(p, lane, &c);
        float keys = keys_of_chunk<ROWS>(p, c, n);
        for (int i = lane + 64; i < p.n; i += 64) {
            Task d;
            const int k = chunk_tiles<ROWS>(p, i, &d);
            keys += keys_of_chunk<ROWS>(p, d, k);
        }
        keys = __int_as_float(lane_value(__float_as_int(wave_sum_lane63(keys)), 63));
        const float share = even_share<ROWS>(keys, target);
        const double inv = 1. / ((double)share * kUnit<ROWS>);
        int per = (int)fminf(share, kMostUnits);
        // That many units in a split are surely few enough tasks, with one more a tile.  Few rows, where the lanes hold
        // the units of all tiles: the fewest units whose tasks are all resident at once (16 sequences of 8,192 rows: 78 us
        // instead of 82, 40 of 2,000: 59 instead of 68).
        if (ROWS == 16 && p.n <= 64 && __ballot(n > 1) == 0) {
            const int most = min(p.few.blocks, p.few.tasks);
            per = fewest_units(least_share<ROWS>(keys, most, per), per, [&](int units) {
                return lane_value(wave_scan(n == 0 ? 0 : splits_of(c.units, units)), 63) <= most;
            });
        }
        int tasks = 0, tiles = 0;  // before these 64 chunks
        bool found = false;
        for (int i0 = 0; i0 < p.n && !found; i0 += 64) {
            if (i0) n = chunk_tiles<ROWS>(p, i0 + lane, &c);
            const int mine = tasks_of_chunk<ROWS>(p, c, n, per, inv);
            const int a = wave_scan(mine), b = wave_scan(n);  // with this lane's chunk
            const unsigned long long m = __ballot((MERGE ? tiles + b : tasks + a) > index);
            if (m) {
                const int l = __builtin_ctzll(m);
                t->first = lane_value(c.first, l);
                t->count = lane_value(c.count, l);
                t->seq = lane_value(c.seq, l);
                t->at = lane_value(c.at, l);
                t->units = lane_value(c.units, l);
                const int all = lane_value(n, l), a0 = tasks + lane_value(a, l) - lane_value(mine, l), b0 = tiles + lane_value(b, l) - all;
                const int q = index - (MERGE ? b0 : a0);
                tile = MERGE ? q : tile_of_task<ROWS>(p, *t, all, q, inv);
                const int begin = tile_begin<ROWS>(p, *t, all, tile, inv);
                t->splits = tile_splits<ROWS>(p, *t, tile, per);
                t->split = MERGE ? 0 : q - begin;
                t->base = a0 + begin;
                found = true;
            }
            tasks += lane_value(a, 63);
            tiles += lane_value(b, 63);
        }
        if (!found || t->split >= t->splits) return false;
        t->per = per;
    }
    t->r0 = tile * ROWS;
    t->rows = min(t->count * p.group - t->r0, ROWS);
    return true;
}

// Says that a found task is the same in every lane: its fields go into scalar registers, and so does what follows from
// them (behind the branch on whether there is one: values that meet behind it count as different).
__device__ __forceinline__ Task settled(Task t) {
    t.seq = uniform(t.seq);
    t.first = uniform(t.first);
    t.count = uniform(t.count);
    t.at = uniform(t.at);
    t.r0 = uniform(t.r0);
    t.rows = uniform(t.rows);
    t.units = uniform(t.units);
    t.per = uniform(t.per);
    t.splits = uniform(t.splits);
    t.split = uniform(t.split);
    t.base = uniform(t.base);
    return t;
}

// The last key that packed row r of the task's chunk sees, -1: none.
__device__ __forceinline__ int last_key(const PagedParams& p, const Task& t, int r) {
    const int cap = p.max_pages << p.shift;
    return t.units == 0 ? -1 : t.at >= cap ? cap - 1 : min(t.at + r / p.group, cap - 1);
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
    const u32x4 a = *reinterpret_cast<const u32x4*>(p);
    const unsigned u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ u32x4 load4(const float* p) { return *reinterpret_cast<const u32x4*>(p); }
__device__ __forceinline__ u32x4 load4(const __hip_bfloat16* p) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    return quad(a.x << 16, a.x & 0xFFFF0000u, a.y << 16, a.y & 0xFFFF0000u);
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

// A barrier over LDS only: loads from memory stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ---- the tile kernel ---------------------------------------------------------------------------------------------
// 128 packed rows a block, 32 a wavefront; keys and values of a tile (64 keys; 32 of fp32 rows or three planes) in LDS, twice, so
// that one barrier a tile is enough: 66 KB, two blocks a CU, whose matrix and vector instructions fill each other's
// gaps.  (Tiles of 32 keys and three blocks a CU: 795 us against 709, at the same state of the rest.)  The staged loads
// of the tile after the next are in flight across the barrier.  The maximum may lag by 2^kSlack, so that most tiles
// rescale nothing.  (The second half's weights under the first one's matrix instructions: the same time.)
// Measured, 32 / 8 heads of 128: bf16, three chunks of 2,048 tokens over 8,192 rows: 657 us, 910 TFLOP/s (a library
// product of 8192^3: 1,144); matrix units busy for 40% of the time, vector units for 36%, little of it at once:
// wavefronts wait to issue for 36%.  fp32 over fp16, three chunks of 1,024 tokens: 597 us, 457 TFLOP/s of the formula,
// twice that of planes.  fp32 rows, 16 / 8 heads, 509 tokens over 1,530 rows: 45 us, of which the parts' way through
// memory and their merge take a third; over 8,698 rows 149 us, 3.7 us a tile of 32 keys and pair of blocks.
template <int HD, typename QT, typename KT>
struct TileSpace {
    typedef Shape<HD, QT, KT> C;
    char lds[4 * C::TILE];      // keys and values of a tile and of the next
    int s_exp[2][2][C::BK];     // fp32 caches: powers of two that they carry
    int s_bad[2];
};

template <int HD, typename QT, typename KT>
__device__ __forceinline__ void tile_block(const PagedParams& p, int index, int kvh, TileSpace<HD, QT, KT>& space) {
    typedef Shape<HD, QT, KT> C;
    typedef Elem<C::F16> E;
    constexpr int NQ = C::NQ, NK = C::NK, BK = C::BK, KT32 = BK / 32, NJ = HD / 32, KS = HD / 16;
    char* const lds = space.lds;
    int (*const s_exp)[2][BK] = space.s_exp;
    int* const s_bad = space.s_bad;

    const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Task found;
    if (!find_task<C::ROWS, false>(p, index, &found)) return;
    const Task t = settled(found);

    const int row = t.r0 + 32 * wave + lq, packed = t.r0 + t.rows;  // row: packed, in the chunk
    const bool mine = row < packed;
    const int tok = mine ? row / p.group : 0, head = kvh * p.group + (mine ? row - tok * p.group : 0);
    const size_t qrow = ((size_t)(t.first + tok) * p.heads + head) * HD;
    // the last key a row sees; the wavefront's first and last rows', the block's
    const int w0 = t.r0 + 32 * wave;
    const int lim = mine ? last_key(p, t, row) : -1, lim0 = uniform(w0 < packed ? last_key(p, t, w0) : -1);
    const int lim1 = uniform(w0 < packed ? last_key(p, t, min(w0 + 31, packed - 1)) : -1);
    const int blim0 = uniform(last_key(p, t, t.r0)), kend = uniform(last_key(p, t, packed - 1)) + 1;

    floatx16 o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[j][r] = 0.f;
    float m = -INFINITY, l = 0.f;
    float wm = 0.f;  // (fp32 caches) the largest weight, times its value row's power of two; the outputs are times 2^ve
    int ve = 120;

    const int t0 = t.split * t.per * (kUnit<128> / BK), t1 = min(t0 + t.per * (kUnit<128> / BK), (kend + BK - 1) / BK);
    const TableRow table = table_row(p, t.seq);
    const int kmax = max(kend - 1, 0);
    const int pmask = (1 << p.shift) - 1;

    // swizzles of 16-byte pieces in a row: K, 16 rows of one column over all banks; V, 4 rows of 4 columns
    const int kx = HD == 128 ? lq & 15 : (lq >> 1) & 7;
    const unsigned kaddr = lq * (HD * 2) + ((h ^ kx) * 16);
    const int i16 = lane & 15, vrow = 4 * h + (i16 >> 2);
    auto value_swizzle = [](int key) { return HD == 128 ? (key & 3) << 2 : ((key >> 1) & 1) << 2; };
    const unsigned vaddr = vrow * (HD * 2) + (((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ value_swizzle(vrow)) * 16) + (i16 & 1) * 8;

    // A wavefront's 64 pieces of a load lie in 64 / CPR rows of one page (its first row is a multiple of that, and pages
    // are longer), so that all but a fixed offset of each lane's address is the same for the wavefront.
    constexpr int ROW = HD * (int)sizeof(KT);
    typedef u32x4 Staged[C::UNITS * (C::KF ? 2 : 1)];
    Staged sk, sv;  // the next tile's keys and values, on their way
    const unsigned lane_at = (lane / C::CPR) * ROW + (lane % C::CPR) * (8 * (int)sizeof(KT));
    int pg0 = -1, pg1 = -1, pg2 = -1, pg3 = -1;
    auto page_at = [&](int k0, int i) __attribute__((always_inline)) {
        const int key = k0 + (i << p.shift), n = table[min(key, kmax) >> p.shift];
        return (i << p.shift) < BK && key < kend && n >= 0 && n < p.pages ? n : -1;
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
    auto stage_load = [&](Staged& st, int tile, const char* pool, int a0, int a1, int a2, int a3) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < C::UNITS; u++) {
            const int row0 = (u * kThreads + wave * 64) / C::CPR, i = row0 >> p.shift;
            int page = i >= 1 ? a1 : a0;
            page = i >= 2 ? a2 : page;
            page = i >= 3 ? a3 : page;
            page = page < 0 ? 0 : page;
            const char* src = pool + ((((size_t)page * p.kv_heads + kvh) << p.shift) + ((tile * BK + row0) & pmask)) * ROW;
            if constexpr (C::KF) {
                st[2 * u] = *reinterpret_cast<const u32x4*>(src + lane_at);
                st[2 * u + 1] = *reinterpret_cast<const u32x4*>(src + lane_at + 16);
            } else {
                st[u] = *reinterpret_cast<const u32x4*>(src + lane_at);
            }
        }
    };
    auto staged_at = [&](int u, int odd, int values) __attribute__((always_inline)) {
        const int piece = u * kThreads + tid, key = piece / C::CPR, col = piece % C::CPR;
        const int x = values ? value_swizzle(key) : HD == 128 ? key & 15 : (key >> 1) & 7;
        return lds + (2 * odd + values) * C::TILE + key * (HD * 2) + ((col ^ x) * 16);
    };
    // Staged rows into LDS.  fp32 ones become two fp16 planes and a power of two, in kSteps steps a piece, each short
    // enough to run under one matrix instruction, and free of branches: `special` becomes nonzero if one holds an
    // infinity or NaN (then stage_special does the work again).
    constexpr int kSteps = 6;
    float p_scale = 0.f;
    unsigned p_plane[4][2], special = 0;
    halfx2 p_zero = {0, 0};
    auto stage_step = [&](const Staged& st, int u, int part, int odd, int values) __attribute__((always_inline)) {
        auto value = [&](int i) __attribute__((always_inline)) { return __uint_as_float(st[2 * u + i / 4][i % 4]); };
        if (part == 0) {
            p_scale = fabsf(value(0));
#pragma unroll
            for (int i = 1; i < 8; i++) p_scale = fmaxf(p_scale, fabsf(value(i)));
            p_zero = halfx2{0, 0};
        } else if (part == 1) {
            const int e = fp16_shift(row_max<C::CPR>(p_scale));
            p_scale = __uint_as_float((unsigned)(e + 127) << 23);
            s_exp[odd][values][(u * kThreads + tid) / C::CPR] = -e;  // (by all of the row's lanes)
        } else {
            const int i = part - 2;
            split2_scaled(value(2 * i), value(2 * i + 1), p_scale, p_plane[i]);
            p_zero = __builtin_elementwise_fma(__builtin_bit_cast(halfx2, p_plane[i][0]), halfx2{0, 0}, p_zero);  // (NaN)
            if (i == 3) {
                special |= __builtin_bit_cast(unsigned, p_zero);
#pragma unroll
                for (int n = 0; n < 2; n++)
                    *reinterpret_cast<u32x4*>(staged_at(u, odd, values) + n * C::PLANE) =
                        quad(p_plane[0][n], p_plane[1][n], p_plane[2][n], p_plane[3][n]);
            }
        }
    };
    // step n of a tile's: its keys' pieces, then its values'
    auto stage_nth = [&](int n, int odd) __attribute__((always_inline)) {
        const int piece = n / kSteps;
        if (piece < C::UNITS) stage_step(sk, piece, n % kSteps, odd, 0);
        else stage_step(sv, piece - C::UNITS, n % kSteps, odd, 1);
    };
    auto stage_store = [&](int odd) __attribute__((always_inline)) {
        if constexpr (C::KF) {
#pragma unroll
            for (int n = 0; n < 2 * C::UNITS * kSteps; n++) stage_nth(n, odd);
        } else {
#pragma unroll
            for (int u = 0; u < C::UNITS; u++) *reinterpret_cast<u32x4*>(staged_at(u, odd, 0)) = sk[u];
#pragma unroll
            for (int u = 0; u < C::UNITS; u++) *reinterpret_cast<u32x4*>(staged_at(u, odd, 1)) = sv[u];
        }
    };
    auto stage_special = [&](const Staged& st, int odd, int values) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < C::UNITS; u++) {
            char* dst = staged_at(u, odd, values);
            float v[8], top = 0.f;  // the largest finite value of the row
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] = __uint_as_float(st[2 * u + i / 4][i % 4]);
                top = fmaxf(top, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.f);
            }
            const int e = fp16_shift(row_max<C::CPR>(top));
            const float scale = __uint_as_float((unsigned)(e + 127) << 23);
            unsigned pl[4][2];
#pragma unroll
            for (int i = 0; i < 4; i++) split2<true, 2, true>(v[2 * i] * scale, v[2 * i + 1] * scale, pl[i]);
#pragma unroll
            for (int n = 0; n < 2; n++)
                *reinterpret_cast<u32x4*>(dst + n * C::PLANE) = quad(pl[0][n], pl[1][n], pl[2][n], pl[3][n]);
            s_exp[odd][values][(u * kThreads + tid) / C::CPR] = -e;  // (by all of the row's lanes)
        }
    };
    // Zeros this thread's pieces of values that are not there, infinities and NaN, in LDS; whether there were any of
    // these.  (Few tiles need it: a loop, and in LDS, for the sake of the others' registers.)
    auto clean = [&](int odd, int k0, unsigned long long miss) __attribute__((always_inline)) {
        unsigned any = 0;
#pragma unroll 1
        for (int u = 0; u < C::UNITS * NK; u++) {
            const int piece = u / NK * kThreads + tid, key = piece / C::CPR, col = piece % C::CPR;
            u32x4* const at = reinterpret_cast<u32x4*>(lds + (2 * odd + 1) * C::TILE + u % NK * C::PLANE + key * (HD * 2) +
                                                    ((col ^ value_swizzle(key)) * 16));
            const bool out = k0 + key >= kend || (miss >> key & 1);
            any |= leave_out<C::F16>(at, out);
        }
        return any != 0;
    };

    // keys of a tile that lie on no page (or behind the last key), by its pages
    auto missing = [&]() __attribute__((always_inline)) {
        const unsigned long long page_keys = p.shift >= 6 ? ~0ull : (1ull << (1 << p.shift)) - 1;
        unsigned long long miss = 0;
        if (pg0 < 0) miss |= page_keys;
        if (pg1 < 0 && (1 << p.shift) < BK) miss |= page_keys << ((1 << p.shift) & 63);
        if (pg2 < 0 && (2 << p.shift) < BK) miss |= page_keys << ((2 << p.shift) & 63);
        if (pg3 < 0 && (3 << p.shift) < BK) miss |= page_keys << ((3 << p.shift) & 63);
        return miss;
    };
    // What the staged tile needs besides; where some row of the block does not see all of it, its values are cleaned.
    auto stage_rest = [&](int tile, unsigned long long miss) __attribute__((always_inline)) {
        const int odd = tile & 1;
        if constexpr (C::KF) {
            if (__builtin_expect(__ballot(special != 0) != 0, 0)) {
                stage_special(sk, odd, 0);
                stage_special(sv, odd, 1);
                special = 0;
            }
        }
        if (tile < t1 && (miss != 0 || tile * BK + BK - 1 > blim0) && clean(odd, tile * BK, miss)) s_bad[odd] = tile;
    };

    if (tid < 2) s_bad[tid] = -1;
    __syncthreads();
    load_pages(t0);
    unsigned long long miss = missing();
    if (t0 < t1) {
        stage_load(sk, t0, p.kp, pg0, pg1, pg2, pg3);
        stage_load(sv, t0, p.vp, pg0, pg1, pg2, pg3);
    }

    // queries: planes in registers, rows of an fp16 cache's scaled into its range
    u32x4 qf[NQ][KS];
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
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[s][i]) < INFINITY ? fabsf(v[s][i]) : 0.f);
            top = max_xor32(top);
            const int e = fp16_shift(top);
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
            for (int i = 0; i < 4; i++) split2<C::F16, NQ, true>(v[s][2 * i], v[s][2 * i + 1], u[i]);
#pragma unroll
            for (int n = 0; n < NQ; n++) qf[n][s] = quad(u[0][n], u[1][n], u[2][n], u[3][n]);
        }
    }

    float one = 1.f;
    asm volatile("" : "+s"(one));
    unsigned long long miss_next = 0;
    if (t0 < t1) {
        load_pages(t0 + 1);
        stage_store(t0 & 1);
        stage_rest(t0, miss);
        miss_next = missing();
        stage_load(sk, t0 + 1, p.kp, pg0, pg1, pg2, pg3);
        stage_load(sv, t0 + 1, p.vp, pg0, pg1, pg2, pg3);
        load_pages(t0 + 2);
    }

    // One barrier a tile: behind it the tile is in LDS, and the one before it is done with; the next one goes from the
    // registers into its place, and the loads of the one after that are issued, with a whole tile's time to arrive
    // (past the split's end: rows that are not used).
    for (int tile = t0; tile < t1; tile++) {
        const int k0 = tile * BK, odd = tile & 1;
        lds_barrier();
        const bool bad = s_bad[odd] == tile;
        const char* const kbuf = lds + 2 * odd * C::TILE;
        const char* const vbuf = kbuf + C::TILE;
        floatx16 s[KT32];
        // LDS reads run ahead of the matrix instructions that take them, by several where one takes 32 cycles (three
        // chunks of 1,024 tokens, bf16: 425 us one ahead, 406 so; several planes: 625 us, more ahead 643, registers).
        // kPinned: both keep their order across a step, all else may move.
        constexpr int kPinned = 0x406, kAhead = NQ == 1 ? 4 : 1, kAheadV = NQ == 1 ? 2 : 1;
        auto scores = [&]() __attribute__((always_inline)) {  // (caches of one plane)
            u32x4 kf[kAhead];
            auto load = [&](int n) __attribute__((always_inline)) {
                kf[n % kAhead] = *reinterpret_cast<const u32x4*>(kbuf + n / KS * 32 * HD * 2 + (kaddr ^ (n % KS * 32)));
            };
#pragma unroll
            for (int n = 0; n < kAhead; n++) load(n);
#pragma unroll
            for (int n = 0; n < KT32 * KS; n++) {
                if (n % KS == 0)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[n / KS][r] = 0.f;
#pragma unroll
                for (int i = 0; i < NQ; i++) s[n / KS] = E::mac(kf[n % kAhead], qf[i][n % KS], s[n / KS]);
                if (n + kAhead < KT32 * KS) load(n + kAhead);
                __builtin_amdgcn_sched_barrier(kPinned);
            }
        };
        if constexpr (C::KF) {
            // the next tile's planes are made under this one's matrix instructions
            constexpr int kSteps0 = 2 * C::UNITS * kSteps, kMacs = KS * (NQ == 1 ? 2 : 3);
            u32x4 kf[2][NK];
            auto key_load = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < NK; j++) kf[ks & 1][j] = *reinterpret_cast<const u32x4*>(kbuf + j * C::PLANE + (kaddr ^ (ks * 32)));
            };
            key_load(0);
#pragma unroll
            for (int r = 0; r < 16; r++) s[0][r] = 0.f;
            int n = 0;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                if (ks + 1 < KS) key_load(ks + 1);
#pragma unroll
                for (int j = 0; j < NK; j++)
#pragma unroll
                    for (int i = 0; i < NQ; i++)
                        if (i + j < C::DEPTH) {
                            s[0] = E::mac(kf[ks & 1][j], qf[i][ks], s[0]);
#pragma unroll
                            for (int x = n * kSteps0 / kMacs; x < (n + 1) * kSteps0 / kMacs; x++) stage_nth(x, 1 - odd);
                            n++;
                            __builtin_amdgcn_sched_barrier(0);
                        }
            }
        } else {
            stage_store(1 - odd);
        }
        stage_rest(tile + 1, miss_next);
        stage_load(sk, tile + 2, p.kp, pg0, pg1, pg2, pg3);
        stage_load(sv, tile + 2, p.vp, pg0, pg1, pg2, pg3);
        const unsigned long long miss_here = miss;
        miss = miss_next;
        miss_next = missing();
        load_pages(tile + 3);

        auto largest = [&](int kt) __attribute__((always_inline)) {
            float mx = s[kt][0];
#pragma unroll
            for (int r = 1; r < 16; r++) mx = fmaxf(mx, s[kt][r]);
            return mx;
        };
        // scores to weights; their sum, of this lane's half of the keys
        auto weights = [&](int kt, float mu) __attribute__((always_inline)) {
            float sum[4];
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[kt][r] = __builtin_amdgcn_exp2f(fmaf(s[kt][r], c, -mu));
                sum[r & 3] = r < 4 ? s[kt][r] : sum[r & 3] + s[kt][r];
            }
            return (sum[0] + sum[1]) + (sum[2] + sum[3]);
        };
        auto products = [&](int kt, float scale) __attribute__((always_inline)) {  // (scale: of fp32 caches)
            constexpr int N = 2 * NJ * NK;
            u32x4 vf[kAheadV];
            auto load = [&](int n) __attribute__((always_inline)) {
                const int k2 = n / (NJ * NK), jt = n / NK % NJ, j = n % NK;
                const char* a = vbuf + j * C::PLANE + (vaddr ^ (jt * 64)) + (32 * kt + 16 * k2) * (HD * 2);
                typedef __attribute__((address_space(3))) shortx4 lds4;
                const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)a));
                const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(a + 8 * HD * 2)));
                vf[n % kAheadV] = quad(x.x, x.y, y.x, y.y);
            };
#pragma unroll
            for (int n = 0; n < kAheadV; n++) load(n);
            u32x4 pf[NQ];
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int k2 = n / (NJ * NK), jt = n / NK % NJ, j = n % NK;
                if (n % (NJ * NK) == 0) {
                    if (NQ > 1 && n) __builtin_amdgcn_sched_barrier(0);  // one step's planes at a time: registers
                    unsigned u[4][NQ];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = s[kt][8 * k2 + 2 * i], y = s[kt][8 * k2 + 2 * i + 1];
                        if constexpr (!C::KF && C::F16 && NQ == 2) split2_mixed(x, y, one, u[i]);
                        else if constexpr (!C::KF) split2<C::F16, NQ, false>(x, y, u[i]);
                        else if constexpr (NQ == 1) split2<true, 1, false>(x * scale, y * scale, u[i]);
                        else split2_scaled(x, y, scale, u[i]);
                    }
#pragma unroll
                    for (int q = 0; q < NQ; q++) pf[q] = quad(u[0][q], u[1][q], u[2][q], u[3][q]);
                }
#pragma unroll
                for (int i = 0; i < NQ; i++)
                    if (i + j < C::DEPTH) o[jt] = E::mac(vf[n % kAheadV], pf[i], o[jt]);
                if (n + kAheadV < N) load(n + kAheadV);
                __builtin_amdgcn_sched_barrier(kPinned);
            }
        };

        if (k0 > lim1) continue;
        // Tiles that every row sees in full, while no row's weights pass a bound (most of them): their sum, which every
        // weight is below, is all that is looked at.  (No key seen before: infinity; NaN passes no bound.)
        float slack = kSlack;
        if constexpr (!C::KF) {
            if (miss_here == 0 && k0 + BK - 1 <= lim0 && !bad) {
                if (NQ > 1) __builtin_amdgcn_s_setprio(1);  // (several planes: matrix instructions first)
                scores();
                if (NQ > 1) __builtin_amdgcn_s_setprio(0);
                float sum = 0.f;
#pragma unroll
                for (int kt = 0; kt < KT32; kt++) sum += weights(kt, m - C::BIAS);
                if (!__ballot(!(sum <= kBound))) {
                    l += sum;
                    if (NQ > 1) __builtin_amdgcn_s_setprio(1);
                    products(0, 1.f);
                    if (NQ > 1) __builtin_amdgcn_s_setprio(0);
                    if constexpr (KT32 > 1) products(1, 1.f);
                    continue;
                }
                slack = 0.f;
            }
        }
        if constexpr (!C::KF) {
            scores();
        } else {
#pragma unroll
            for (int kt = 0; kt < KT32; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[kt][r] = ldexpf(s[kt][r], s_exp[odd][0][32 * kt + 8 * (r >> 2) + 4 * h + (r & 3)]);
        }
        if (k0 + BK - 1 > lim0) {  // (the lane's keys are 32 kt + 8 (r / 4) + r % 4, and 4 h)
            asm volatile("");      // (a branch: few tiles have hidden keys)
            const int last = lim - k0 - 4 * h;
#pragma unroll
            for (int kt = 0; kt < KT32; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (32 * kt + 8 * (r >> 2) + (r & 3) > last) s[kt][r] = -INFINITY;
        }
        if (miss_here != 0) {
            asm volatile("");
#pragma unroll
            for (int kt = 0; kt < KT32; kt++) {
                const unsigned gone = (unsigned)(miss_here >> (32 * kt)) >> (4 * h);
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (gone >> (8 * (r >> 2) + (r & 3)) & 1) s[kt][r] = -INFINITY;
            }
        }
        float mx = largest(0);
        if constexpr (KT32 > 1) mx = fmaxf(mx, largest(1));
        mx = max_xor32(mx) * c;
        if (__ballot(mx - m > slack)) {  // (no key seen before: infinity; none yet: NaN)
            const float mn = fmaxf(m, mx);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
            if (C::KF) wm *= alpha;
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[j][r] *= alpha;
            m = mn;
        }
        // (a row that has seen no key yet keeps m = -inf: weights 0)
        const float mu = m == -INFINITY ? 0.f : m - C::BIAS;
#pragma unroll
        for (int kt = 0; kt < KT32; kt++) l += weights(kt, mu);
        float scale = 1.f;
        if constexpr (C::KF) {
            // weights take over the values' powers of two, and a power of the row's that brings the largest so far
            // into [2^3, 2^15]: bits are lost relative to the largest contribution, not to the largest value
            float top = 0.f;
#pragma unroll
            for (int kt = 0; kt < KT32; kt++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[kt][r] = ldexpf(s[kt][r], s_exp[odd][1][32 * kt + 8 * (r >> 2) + 4 * h + (r & 3)]);
                    top = fmaxf(top, s[kt][r]);
                }
            wm = fmaxf(wm, max_xor32(top));
            const float x = ldexpf(wm, ve);
            if (__ballot(x > 32768.f || (x < 8.f && ve < 120))) {
                const int to = min(137 - (int)(__float_as_uint(wm) >> 23), 120);  // the largest to [2^10, 2^11)
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[j][r] = ldexpf(o[j][r], to - ve);
                ve = to;
            }
            scale = __uint_as_float((unsigned)(ve + 127) << 23);
        }
#pragma unroll
        for (int kt = 0; kt < KT32; kt++) products(kt, scale);
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
    l = sum_xor32(l);

    if (!mine) return;
    if constexpr (C::KF) {
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[j][r] = ldexpf(o[j][r], -ve);
    }
    if (t.splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        QT* out = (QT*)p.out + qrow;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                store4(out + 32 * j + 2 * r + 4 * h, o[j][r] * inv, o[j][r + 1] * inv, o[j][r + 2] * inv, o[j][r + 3] * inv);
    } else {
        const size_t at = ((size_t)(t.base + t.split) * p.kv_heads + kvh) * C::ROWS + (row - t.r0);
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                store4(p.tile.part + at * HD + 32 * j + 2 * r + 4 * h, o[j][r], o[j][r + 1], o[j][r + 2], o[j][r + 3]);
        if (h == 0) p.tile.part_ml[at] = make_float2(m, l);
    }
}

// ---- few rows: one token of a sequence, or some ----------------------------------------------------------------------
// A block takes 16 packed rows and its four wavefronts take key tiles of 32 in turn, so that a decode step streams its
// keys and values from as many places as there are wavefronts, with no barrier between them.  16 x 16 matrix
// instructions: S^T (16 keys x 16 rows) twice, lane l has row l % 16 and keys 4 (l / 16) + 0..3; O^T (16 dims x 16 rows)
// from 32 keys at a time.  Keys go from memory straight into the operands (a lane's 16 bytes lie beside its three
// neighbours' in the row).  16-bit values take the way over the wavefront's own LDS space, for the transposed reads;
// fp32 ones do not: v_mfma_f32_16x16x4_f32 wants one value of a key per lane, and output row i of tile (a, j) is dim
// 64 a + 4 i + j, so that 16 bytes of a value row feed four tiles.  Of the next tile, keys are loaded when this one's
// scores are done and values when its own are in LDS (or used).
// HBM bounds it.  Measured, head size 128: 16 sequences of up to 8,192 rows (386 MB, fp16): 78 us, 4.95 TB/s, what a
// large copy reaches; 8 of 4,000 fp32 rows (194 MB): 46 us, 4.2 TB/s; one of 4,096 rows (17 MB): 14 us, of which two
// launches and the wait for the first keys are 10; one token over 100 rows: 7 us, a launch and its dependent loads.
template <int HD>
struct FewSpace {
    char lds[kWaves * 32 * HD * 2];  // values, later the wavefronts' outputs
    float s_m[kWaves][16], s_l[kWaves][16];
};

template <int HD, typename QT, typename KT>
__device__ __forceinline__ void few_block(const PagedParams& p, int index, int kvh, FewSpace<HD>& space) {
    typedef Shape<HD, QT, KT> C;
    typedef Elem<C::F16> E;
    constexpr bool KF = C::KF;
    constexpr int NQ = C::NQ, NJ = HD / 16, KS = HD / 32, QC = HD / 16, JJ = HD / 64;
    constexpr int ROW = HD * (int)sizeof(KT), UNITS = 32 * C::CPR / 64, VBYTES = 32 * HD * 2;
    char* const lds = space.lds;
    float (*const s_m)[16] = space.s_m;
    float (*const s_l)[16] = space.s_l;

    const int tid = threadIdx.x, lane = tid & 63, lq = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Task found;
    if (!find_task<16, false>(p, index, &found)) return;
    const Task t = settled(found);
    const int row = t.r0 + lq, packed = t.r0 + t.rows;
    const bool mine = row < packed;
    const int tok = mine ? row / p.group : 0, head = kvh * p.group + (mine ? row - tok * p.group : 0);
    const size_t qrow = ((size_t)(t.first + tok) * p.heads + head) * HD;
    const int lim = mine ? last_key(p, t, row) : -1;
    const int lim0 = uniform(last_key(p, t, t.r0)), kend = uniform(last_key(p, t, packed - 1)) + 1;
    const int t0 = t.split * t.per * 4 + wave, t1 = min((t.split + 1) * t.per * 4, (kend + 31) / 32);

    const TableRow table = table_row(p, t.seq);
    const int kmax = max(kend - 1, 0);
    const int pmask = (1 << p.shift) - 1;
    auto page_at = [&](int tile, int i) __attribute__((always_inline)) {  // page of the tile's keys 16 i on
        const int key = 32 * tile + 16 * i, n = table[min(key, kmax) >> p.shift];
        return key < kend && n >= 0 && n < p.pages ? n : -1;
    };
    // start of the pool row of key 16 i of a tile (a row on no page: some row of the pool in its place)
    auto row_at = [&](const char* pool, int tile, int page, int key) __attribute__((always_inline)) {
        return pool + ((((size_t)(page < 0 ? 0 : page) * p.kv_heads + kvh) << p.shift) + ((32 * tile + key) & pmask)) * ROW;
    };
    u32x4 kf[2][KF ? QC : KS], vf[KF ? 2 * 4 * JJ : UNITS];
    const unsigned k_at = lq * ROW + g * 16;
    const unsigned v_at = KF ? 4 * g * ROW + lq * 16 : (lane / C::CPR) * ROW + (lane % C::CPR) * 16;
    int pg0 = page_at(t0, 0), pg1 = page_at(t0, 1);
    auto load_k = [&](int tile, int a0, int a1) __attribute__((always_inline)) {
#pragma unroll
        for (int a = 0; a < 2; a++) {
            const char* src = row_at(p.kp, tile, a ? a1 : a0, 16 * a) + k_at;
#pragma unroll
            for (int s = 0; s < (KF ? QC : KS); s++) kf[a][s] = *reinterpret_cast<const u32x4*>(src + 64 * s);
        }
    };
    auto load_v = [&](int tile, int a0, int a1) __attribute__((always_inline)) {
        if constexpr (KF) {
#pragma unroll
            for (int a = 0; a < 2; a++) {
                const char* src = row_at(p.vp, tile, a ? a1 : a0, 16 * a) + v_at;
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int j = 0; j < JJ; j++) vf[(4 * a + r) * JJ + j] = *reinterpret_cast<const u32x4*>(src + r * ROW + 256 * j);
            }
        } else {
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                const int key = u * 64 / C::CPR;
                vf[u] = *reinterpret_cast<const u32x4*>(row_at(p.vp, tile, key >= 16 ? a1 : a0, key) + v_at);
            }
        }
    };
    if (t0 < t1) {
        load_k(t0, pg0, pg1);
        load_v(t0, pg0, pg1);
    }
    int pn0 = page_at(t0 + kWaves, 0), pn1 = page_at(t0 + kWaves, 1);

    // queries
    u32x4 qf[KF ? 1 : NQ][KF ? QC : KS];
    float c = p.scale;
    if constexpr (KF) {
#pragma unroll
        for (int s = 0; s < QC; s++) qf[0][s] = mine ? load4((const QT*)p.q + qrow + 16 * s + 4 * g) : quad(0, 0, 0, 0);
    } else {
        float v[KS][8];
#pragma unroll
        for (int s = 0; s < KS; s++) {
            if (mine) load8<QT>((const QT*)p.q + qrow + 32 * s + 8 * g, v[s]);
            else
#pragma unroll
                for (int i = 0; i < 8; i++) v[s][i] = 0.f;
        }
        if constexpr (C::F16) {
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[s][i]) < INFINITY ? fabsf(v[s][i]) : 0.f);
            top = max_xor32(fmaxf(top, xor16(top, lane)));
            const int e = fp16_shift(top);
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
            for (int i = 0; i < 4; i++) split2<C::F16, NQ, true>(v[s][2 * i], v[s][2 * i + 1], u[i]);
#pragma unroll
            for (int n = 0; n < NQ; n++) qf[n][s] = quad(u[0][n], u[1][n], u[2][n], u[3][n]);
        }
    }

    floatx4 o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) o[j] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // values in LDS: swizzled so that 8 rows of two 16-byte pieces lie over all banks (transposed reads)
    char* const vbuf = lds + wave * VBYTES;
    auto swizzle = [](int key) { return HD == 128 ? (key & 3) << 2 | (key >> 2 & 1) << 1 : (key >> 1 & 3) << 1; };
    const int vrow = 4 * g + (lq >> 2);
    const unsigned vaddr = vrow * (HD * 2) + ((((lq & 3) >> 1) ^ swizzle(vrow)) * 16) + (lq & 1) * 8;

    for (int tile = t0; tile < t1; tile += kWaves) {
        const int k0 = 32 * tile;
        const unsigned miss = (pg0 < 0 ? 0xFFFFu : 0u) | (pg1 < 0 ? 0xFFFF0000u : 0u);  // keys on no page (or past the end)
        const bool masked = miss != 0 || k0 + 31 > lim0;
        floatx4 s[2];
#pragma unroll
        for (int a = 0; a < 2; a++) {
            s[a] = floatx4{0.f, 0.f, 0.f, 0.f};
            if constexpr (KF) {
                floatx4 s1 = s[a];
#pragma unroll
                for (int q = 0; q < QC; q++) {
                    floatx4& x = q & 1 ? s1 : s[a];
                    x = mac4(kf[a][q].x, qf[0][q].x, x);
                    x = mac4(kf[a][q].y, qf[0][q].y, x);
                    x = mac4(kf[a][q].z, qf[0][q].z, x);
                    x = mac4(kf[a][q].w, qf[0][q].w, x);
                }
                s[a] += s1;
            } else {
#pragma unroll
                for (int q = 0; q < KS; q++)
#pragma unroll
                    for (int i = 0; i < NQ; i++) s[a] = E::mac16(kf[a][q], qf[i][q], s[a]);
            }
        }
        const int next = tile + kWaves;
        load_k(next, pn0, pn1);  // (past the end: rows of no page, not used)
        if (masked) {
            asm volatile("");  // (a branch: few tiles have hidden keys)
            const int last = lim - k0 - 4 * g;
            const unsigned gone = miss >> (4 * g);
#pragma unroll
            for (int a = 0; a < 2; a++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (16 * a + r > last || (gone >> (16 * a + r) & 1)) s[a][r] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_xor32(fmaxf(mx, xor16(mx, lane))) * c;
        if (__ballot(mx > m)) {
            const float mn = fmaxf(m, mx);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= alpha;
#pragma unroll
            for (int j = 0; j < NJ; j++) o[j] *= alpha;
            m = mn;
        }
        const float mu = m == -INFINITY ? 0.f : m - C::BIAS;  // (no key seen yet: weights 0)
#pragma unroll
        for (int a = 0; a < 2; a++)
#pragma unroll
            for (int r = 0; r < 4; r++) s[a][r] = __builtin_amdgcn_exp2f(fmaf(s[a][r], c, -mu));
        l += ((s[0][0] + s[0][1]) + (s[0][2] + s[0][3])) + ((s[1][0] + s[1][1]) + (s[1][2] + s[1][3]));
        // (as in the tile kernel: values of rows that are not there, infinities and NaN are left out)
        bool bad = false;
        if constexpr (KF) {
            if (masked) {
                unsigned any = 0;
#pragma unroll
                for (int u = 0; u < 2 * 4 * JJ; u++) {
                    const int key = 16 * (u / (4 * JJ)) + 4 * g + u / JJ % 4;
                    if (k0 + key >= kend || (miss >> key & 1)) vf[u] = quad(0, 0, 0, 0);
                    vf[u] = drop_special<true, false>(vf[u], &any);
                    __builtin_amdgcn_sched_barrier(0);  // one piece at a time: registers
                }
                bad = __ballot(any != 0) != 0;
            }
        }
        if constexpr (KF) {
#pragma unroll
            for (int a = 0; a < 2; a++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int j = 0; j < JJ; j++) {
                        const u32x4 v = vf[(4 * a + r) * JJ + j];
                        o[4 * j] = mac4f(v.x, s[a][r], o[4 * j]);
                        o[4 * j + 1] = mac4f(v.y, s[a][r], o[4 * j + 1]);
                        o[4 * j + 2] = mac4f(v.z, s[a][r], o[4 * j + 2]);
                        o[4 * j + 3] = mac4f(v.w, s[a][r], o[4 * j + 3]);
                    }
            load_v(next, pn0, pn1);
        } else {
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                const int key = u * 64 / C::CPR + lane / C::CPR, col = lane % C::CPR;
                *reinterpret_cast<u32x4*>(vbuf + key * (HD * 2) + ((col ^ swizzle(key)) * 16)) = vf[u];
            }
            load_v(next, pn0, pn1);
            if (masked) {
                unsigned any = 0;
#pragma unroll 1
                for (int u = 0; u < UNITS; u++) {
                    const int key = u * 64 / C::CPR + lane / C::CPR, col = lane % C::CPR;
                    any |= leave_out<C::F16>(reinterpret_cast<u32x4*>(vbuf + key * (HD * 2) + ((col ^ swizzle(key)) * 16)),
                                             k0 + key >= kend || (miss >> key & 1));
                }
                bad = __ballot(any != 0) != 0;
            }
            asm volatile("" ::: "memory");  // (one wavefront's LDS accesses are served in order)
            __builtin_amdgcn_wave_barrier();
            u32x4 pf[NQ];
            {
                unsigned u[4][NQ];
#pragma unroll
                for (int i = 0; i < 4; i++) split2<C::F16, NQ, false>(s[i >> 1][2 * (i & 1)], s[i >> 1][2 * (i & 1) + 1], u[i]);
#pragma unroll
                for (int n = 0; n < NQ; n++) pf[n] = quad(u[0][n], u[1][n], u[2][n], u[3][n]);
            }
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                typedef __attribute__((address_space(3))) shortx4 lds4;
                const char* a = vbuf + (vaddr ^ (j * 32));
                const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)a));
                const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(a + 16 * HD * 2)));
#pragma unroll
                for (int i = 0; i < NQ; i++) o[j] = E::mac16(quad(x.x, x.y, y.x, y.y), pf[i], o[j]);
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_wave_barrier();
        }
        if (__builtin_expect(bad, 0)) {
#pragma unroll 1
            for (int key = 0; key < 32 && k0 + key < kend; key++) {
                const int page = key >= 16 ? pg1 : pg0;
                if (page < 0) continue;
                const KT* v = (const KT*)row_at(p.vp, tile, page, key);
                const bool seen = k0 + key <= lim;
#pragma unroll
                for (int j = 0; j < NJ; j++) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float x = to_float(v[KF ? 64 * (j / 4) + 4 * (4 * g + r) + j % 4 : 16 * j + 4 * g + r]);
                        if (seen && !(fabsf(x) < INFINITY)) o[j][r] += x;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        pg0 = pn0;
        pg1 = pn1;
        pn0 = page_at(next + kWaves, 0);
        pn1 = page_at(next + kWaves, 1);
    }

    // the wavefronts' states at a common maximum; each adds up a quarter of the outputs
    l += xor16(l, lane);
    l = sum_xor32(l);
    if (g == 0) s_m[wave][lq] = m;
    __syncthreads();  // (values in LDS are done with, too)
    float mm = s_m[0][lq];
#pragma unroll
    for (int w = 1; w < kWaves; w++) mm = fmaxf(mm, s_m[w][lq]);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mm);
    if (g == 0) s_l[wave][lq] = l * f;
    float* const st = reinterpret_cast<float*>(lds) + lane;  // [wavefront][tile][register][lane]
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) st[((wave * NJ + j) * 4 + r) * 64] = o[j][r] * f;
    __syncthreads();
    if (!mine) return;
    l = (s_l[0][lq] + s_l[1][lq]) + (s_l[2][lq] + s_l[3][lq]);
    const size_t at = ((size_t)(t.base + t.split) * p.kv_heads + kvh) * 16 + lq;
    const float inv = t.splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int q = 0; q < NJ / 4; q++) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // 16-bit caches: tile q + NJ / 4 * wave, register i; fp32: tiles 4 q + i, register `wave`
            const float* a = st + (KF ? (4 * q + i) * 4 + wave : (q + NJ / 4 * wave) * 4 + i) * 64;
            v[i] = ((a[0] + a[NJ * 256]) + (a[2 * NJ * 256] + a[3 * NJ * 256])) * inv;
        }
        const int d = KF ? 64 * q + 4 * (4 * g + wave) : 16 * (q + NJ / 4 * wave) + 4 * g;
        if (t.splits > 1) store4(p.few.part + at * HD + d, v[0], v[1], v[2], v[3]);
        else store4((QT*)p.out + qrow + d, v[0], v[1], v[2], v[3]);
    }
    if (t.splits > 1 && wave == 0 && g == 0) p.few.part_ml[at] = make_float2(mm, l);
}

// ---- both in one launch -------------------------------------------------------------------------------------------
// PARTS: 1 few rows, 2 tiles, 3 both (blocks of tiles first).  KV head fastest (8 of them: one to an XCD, whose L2 then
// holds that head's rows); tiles from the last, with the most keys, on.
template <int HD, typename QT, typename KT, int PARTS>
__global__ __launch_bounds__(kThreads, 2) void paged_attention_kernel(PagedParams p) {
    union Space {
        TileSpace<HD, QT, KT> tile;
        FewSpace<HD> few;
    };
    __shared__ __attribute__((aligned(16))) char space[PARTS == 1 ? sizeof(FewSpace<HD>) : sizeof(Space)];
    const int kvh = blockIdx.x % p.kv_heads, b = blockIdx.x / p.kv_heads;
    if (PARTS == 2 || (PARTS == 3 && b < p.tile.tasks))
        tile_block<HD, QT, KT>(p, p.tile.tasks - 1 - b, kvh, *reinterpret_cast<TileSpace<HD, QT, KT>*>(space));
    else if (PARTS & 1)
        few_block<HD, QT, KT>(p, b - (PARTS == 3 ? p.tile.tasks : 0), kvh, *reinterpret_cast<FewSpace<HD>*>(space));
}

// ---- the splits of a row, in a fixed order ------------------------------------------------------------------------
// A block takes 16 rows of a tile, or twice 16 where that many blocks would not be resident at once (16 chunks of 64
// tokens in bf16: 62.4 us, 64.6 with 16; 509 fp32 tokens of one chunk: 48.3 and 47.5); where there are fewer rows, several
// groups of HD / 4 lanes share a row's splits.  Bound by memory (the parts come out of L2 and the cache behind it) and by
// the way to its task: 5.4 us after the decode step above, 8.6 us for the 29 MB of the fp32 chunk's.
template <int HD, typename QT, int ROWS>
__device__ __forceinline__ void merge_block(const PagedParams& p, int b, int kvh, float (*s_o)[HD], float* s_l) {
    constexpr int LPR = HD / 4, NG = 512 / LPR;
    const int per_block = ROWS == 16 ? 16 : p.merge_rows, blocks = ROWS / per_block;
    const PartArgs& a = ROWS == 16 ? p.few : p.tile;
    Task found;
    if (!find_task<ROWS, true>(p, b / blocks, &found)) return;
    const Task t = settled(found);
    // (chunks whose starts are not in order may have more tasks than there is space for: they are not all computed)
    if (t.splits == 1 || t.base < 0 || t.base + t.splits > a.tasks) return;
    const int group = threadIdx.x / LPR, col = threadIdx.x % LPR;
    const size_t step = (size_t)p.kv_heads * ROWS;
    const int first = per_block * (b % blocks), last = min(t.rows, first + per_block);
    for (int r0 = first; r0 < last; r0 += 16) {
        const int rows = min(last - r0, 16);
        int share = 1;  // groups of a row
        while (2 * share * rows <= NG) share *= 2;
        const int r = group / share, sub = group % share;
        const size_t at = ((size_t)t.base * p.kv_heads + kvh) * ROWS + r0 + min(r, rows - 1);
        float m = -INFINITY, l = 0.f;
        for (int s = col; s < t.splits; s += LPR) m = fmaxf(m, a.part_ml[at + s * step].x);
#pragma unroll
        for (int d = 1; d < LPR; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = sub; s < t.splits; s += share) {
            const float2 ml = a.part_ml[at + s * step];
            const float4 v = *reinterpret_cast<const float4*>(a.part + (at + s * step) * HD + 4 * col);
            const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m);  // (no key seen: zeros)
            l = fmaf(ml.y, f, l);
            o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
        }
        if (share > 1) {
            if (r0 > first) __syncthreads();  // (the rows before have been read)
            *reinterpret_cast<float4*>(&s_o[group][4 * col]) = o;
            if (col == 0) s_l[group] = l;
            __syncthreads();
        }
        if (sub != 0 || r >= rows) continue;
        for (int k = 1; k < share; k++) {
            const float4 v = *reinterpret_cast<const float4*>(&s_o[group + k][4 * col]);
            o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
            l += s_l[group + k];
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int row = t.r0 + r0 + r, tok = row / p.group, head = kvh * p.group + row - tok * p.group;
        store4((QT*)p.out + ((size_t)(t.first + tok) * p.heads + head) * HD + 4 * col, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
}

template <int HD, typename QT>
__global__ __launch_bounds__(512) void paged_merge_kernel(PagedParams p) {
    __shared__ __attribute__((aligned(16))) float s_o[512 / (HD / 4)][HD];
    __shared__ float s_l[512 / (HD / 4)];
    const int kvh = blockIdx.x % p.kv_heads, b = blockIdx.x / p.kv_heads;
    const int tiles = p.tile.target ? 128 / p.merge_rows * p.tile.tiles : 0;
    if (b < tiles) merge_block<HD, QT, 128>(p, b, kvh, s_o, s_l);
    else merge_block<HD, QT, 16>(p, b - tiles, kvh, s_o, s_l);
}

// ---- host side ----------------------------------------------------------------------------------------------

size_t part_bytes(const ar_pages* p, const Part& a, int rows) {
    return a.target ? (size_t)a.tasks() * p->kv_heads * rows * ((size_t)p->head_dim * 4 + 8) : 0;
}

int plan_of(const ar_hip_ctx* ctx, const ar_pages* p, const ar_chunks* c, int heads, Plan* out) {
    const long long group = heads / p->kv_heads, packed = (long long)c->rows * group;
    AR_CHECK_ARG(packed <= 1 << 30 && (packed / 16 + c->n) * p->kv_heads < 1 << 23, "paged attention: %d rows of %d heads are too many",
                 c->rows, heads);
    *out = plan_tasks(ctx->num_cus, p->kv_heads, p->dtype == AR_DTYPE_F32, (long long)p->max_pages * p->page_rows, c->start != nullptr,
                      c->n, c->rows, (int)group);
    return AR_HIP_OK;
}

size_t plan_bytes(const ar_pages* p, const Plan& a) { return std::max<size_t>(16, part_bytes(p, a.few, 16) + part_bytes(p, a.tile, 128)); }

template <int HD, typename QT, typename KT>
int launch_plan(const ar_pages* pages, const Plan& a, PagedParams p, char* work, hipStream_t st) {
    auto part = [&](const Part& x, int rows, char* at) {
        return PartArgs{x.tiles, x.tasks(), x.target, x.blocks, (float*)at, (float2*)(at + (size_t)x.tasks() * p.kv_heads * rows * HD * 4)};
    };
    p.few = part(a.few, 16, work);
    p.tile = part(a.tile, 128, work + part_bytes(pages, a.few, 16));
    const dim3 grid((unsigned)(p.few.tasks + p.tile.tasks) * p.kv_heads), block(kThreads);
    if (!p.tile.tasks) hipLaunchKernelGGL((paged_attention_kernel<HD, QT, KT, 1>), grid, block, 0, st, p);
    else if (!p.few.tasks) hipLaunchKernelGGL((paged_attention_kernel<HD, QT, KT, 2>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((paged_attention_kernel<HD, QT, KT, 3>), grid, block, 0, st, p);
    AR_LAUNCH_CHECK();
    const int merges = (p.tile.target ? 128 / p.merge_rows * p.tile.tiles : 0) + (p.few.target ? p.few.tiles : 0);
    if (merges) {
        hipLaunchKernelGGL((paged_merge_kernel<HD, QT>), dim3((unsigned)merges * p.kv_heads), dim3(512), 0, st, p);
        AR_LAUNCH_CHECK();
    }
    return AR_HIP_OK;
}

template <int HD, typename QT>
int launch_kt(const ar_pages* pages, const Plan& a, const PagedParams& p, char* work, hipStream_t st) {
    if (pages->dtype == AR_DTYPE_F32) return launch_plan<HD, QT, float>(pages, a, p, work, st);
    if (pages->dtype == AR_DTYPE_F16) return launch_plan<HD, QT, _Float16>(pages, a, p, work, st);
    return launch_plan<HD, QT, __hip_bfloat16>(pages, a, p, work, st);
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
    *bytes = plan_bytes(pages, a);
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
    const size_t need = plan_bytes(pages, a);
    AR_CHECK_ARG(work && work_bytes >= need, "%s: %zu bytes of work space given, %zu needed", what, work ? work_bytes : 0, need);
    const int hd = pages->head_dim;
    const size_t act = act_dtype == AR_DTYPE_F32 ? 4 : 2, bytes = (size_t)chunks->rows * heads * hd * act;
    if (ar_check_ptrs_enabled()) {
        AR_TRY(page_check_ranges(pages, what));
        AR_TRY(page_check_chunk_ranges(chunks, what));
        AR_TRY(ar_check_range(q, bytes, what, "queries"));
        AR_TRY(ar_check_range(out, bytes, what, "output"));
        AR_TRY(ar_check_range(work, need, what, "work space"));
    }
    const size_t layer_bytes = (size_t)pages->pages * pages->kv_heads * hd * pages->page_rows * page_elem_bytes(pages->dtype);
    PagedParams p{};
    p.q = q; p.out = out;
    p.kp = (const char*)pages->k + layer * layer_bytes;
    p.vp = (const char*)pages->v + layer * layer_bytes;
    p.table = pages->table; p.seq = chunks->seq; p.start = chunks->start; p.at = chunks->at; p.heads = heads;
    p.kv_heads = pages->kv_heads; p.group = heads / pages->kv_heads; p.seqs = pages->seqs;
    p.max_pages = pages->max_pages; p.pages = pages->pages; p.shift = page_shift_of(pages); p.n = chunks->n;
    p.rows = chunks->rows; p.few_rows = a.few_rows;
    p.merge_rows = 8LL * a.tile.tiles * p.kv_heads > 4LL * ctx->num_cus ? 32 : 16;
    p.scale = (float)(1.4426950408889634 / std::sqrt((double)hd));
    char* const w = (char*)work;
    if (hd == 128)
        return act == 4 ? launch_kt<128, float>(pages, a, p, w, ctx->stream)
                        : launch_kt<128, __hip_bfloat16>(pages, a, p, w, ctx->stream);
    return act == 4 ? launch_kt<64, float>(pages, a, p, w, ctx->stream)
                    : launch_kt<64, __hip_bfloat16>(pages, a, p, w, ctx->stream);
}
