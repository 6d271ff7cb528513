// Paged KV cache: page copies, and the calls that share, take, give back and move pages (include/ar_pages.h).
// Tables and counts stay on the device, so that a token loop need not wait for the host to learn a page number.
#include "page_common.h"

namespace {

constexpr int kMaxEntries = 4096;  // chunks / entries of one table call: their state lies in one block's LDS

// ---- page copies -----------------------------------------------------------------------------------
// Bound by HBM, each byte read and written once.  A block moves pieces of 16 KB: 256 threads x four 16-byte loads in
// flight before their stores, so 8 blocks on a CU keep 128 KB in flight.  Measured: 255 pages of 28 layers (1.87 GB read
// and written) 371 us, 5.0 TB/s, what one large copy reaches; 16 of them 25 us; 9 small pages 5 us, a launch.  Pieces of 4
// and 8 KB: 389 and 380 us (16 KB: 381).  Loads and stores that leave the caches to others: 381 -> 371 us, 64 forks'
// last pages 211 -> 202.
constexpr int kCopyThreads = 256, kCopyUnroll = 4, kPieceBytes = 16384;

struct CopyParams {
    const char *sk, *sv;
    char *dk, *dv;
    size_t s_layer, d_layer;  // bytes of a layer in each pool
    unsigned page_bytes;
    int layers, pieces;
    // what to copy: pairs[i] = {source, target} for i < *count (or slots where count is null; source -1: none)
    const int2* pairs;
    const int* count;
    int slots;
    // or page numbers of the caller's
    const int *src, *dst;
    int s_pages, d_pages, same_pool;
    // a table whose entries move with the pages (null: none): page g becomes to[g]
    int* table;
    const int* to;
    size_t cells;
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));  // (an array of structures goes to LDS: 17 us for 4)

__device__ __forceinline__ void copy_run(const char* s, char* d, unsigned bytes) {
    const unsigned units = bytes / 16, step = kCopyThreads * kCopyUnroll;
    const u32x4* a = reinterpret_cast<const u32x4*>(s);
    u32x4* b = reinterpret_cast<u32x4*>(d);
    unsigned i = threadIdx.x;
    for (; i + step - kCopyThreads < units; i += step) {
        u32x4 t[kCopyUnroll];
#pragma unroll
        for (int u = 0; u < kCopyUnroll; u++) t[u] = __builtin_nontemporal_load(a + i + u * kCopyThreads);
#pragma unroll
        for (int u = 0; u < kCopyUnroll; u++) __builtin_nontemporal_store(t[u], b + i + u * kCopyThreads);
    }
    for (; i < units; i += kCopyThreads) b[i] = a[i];
}

__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(CopyParams p) {
    if (p.table) {
        const size_t step = (size_t)gridDim.x * gridDim.y * kCopyThreads;
        for (size_t i = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * kCopyThreads + threadIdx.x; i < p.cells; i += step) {
            const int page = p.table[i];
            if (page < 0 || page >= p.s_pages) continue;
            const int to = p.to[page];
            if (to != page) p.table[i] = to;
        }
    }
    const int slots = p.count ? min(*p.count, p.slots) : p.slots;
    for (int slot = blockIdx.y; slot < slots; slot += gridDim.y) {
        int s, d;
        if (p.pairs) {
            const int2 e = p.pairs[slot];
            s = e.x;
            d = e.y;
        } else {
            s = p.src[slot];
            d = p.dst[slot];
            bool out = (unsigned)s >= (unsigned)p.s_pages || (unsigned)d >= (unsigned)p.d_pages;
            if (!out)  // an earlier entry with this target, or (one pool) an entry that reads it
                for (int j = threadIdx.x; j < slots; j += kCopyThreads) {
                    const int sj = p.src[j], dj = p.dst[j];
                    if ((unsigned)sj >= (unsigned)p.s_pages || (unsigned)dj >= (unsigned)p.d_pages) continue;
                    out |= (j < slot && dj == d) || (p.same_pool && sj == d);
                }
            if (__syncthreads_or(out)) continue;
        }
        if (s < 0) continue;
        for (int item = blockIdx.x; item < 2 * p.layers * p.pieces; item += gridDim.x) {
            const int piece = item % p.pieces, part = item / p.pieces, layer = part >> 1;
            const size_t so = layer * p.s_layer + (size_t)s * p.page_bytes, dof = layer * p.d_layer + (size_t)d * p.page_bytes;
            const char* from = (part & 1 ? p.sv : p.sk) + so;
            char* to = (part & 1 ? p.dv : p.dk) + dof;
            const unsigned at = (unsigned)piece * kPieceBytes;
            copy_run(from + at, to + at, min((unsigned)kPieceBytes, p.page_bytes - at));
        }
    }
}

CopyParams copy_params(const ar_pages* from, const ar_pages* to) {
    CopyParams p{};
    p.sk = (const char*)from->k;
    p.sv = (const char*)from->v;
    p.dk = (char*)to->k;
    p.dv = (char*)to->v;
    p.page_bytes = (unsigned)((size_t)from->head_dim * page_elem_bytes(from->dtype) * from->page_rows * from->kv_heads);
    p.s_layer = (size_t)p.page_bytes * from->pages;
    p.d_layer = (size_t)p.page_bytes * to->pages;
    p.layers = from->layers;
    p.pieces = (int)((p.page_bytes + kPieceBytes - 1) / kPieceBytes);
    p.s_pages = from->pages;
    p.d_pages = to->pages;
    return p;
}

int launch_copy(const ar_hip_ctx* ctx, const CopyParams& p) {
    // about 16 blocks per CU over all slots, so that they finish together
    const long long items = 2LL * p.layers * p.pieces, want = 16LL * ctx->num_cus;
    const int y = std::min(p.slots, 32768);
    const int x = (int)std::max(1LL, std::min(items, (want + y - 1) / y));
    hipLaunchKernelGGL(copy_pages_kernel, dim3(x, y), dim3(kCopyThreads), 0, ctx->stream, p);
    AR_LAUNCH_CHECK();
    return AR_HIP_OK;
}

// ---- block-wide helpers ------------------------------------------------------------------------------

// Exclusive prefix sum over a block of NT threads (a multiple of 64); *total receives the sum.  `part`: NT / 64 ints
// of LDS, free for reuse after the next barrier.
template <int NT>
__device__ __forceinline__ int block_prefix(int v, int* part, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        const int t = part[w];
        before += w < wave ? t : 0;
        sum += t;
    }
    *total = sum;
    __syncthreads();
    return before + x - v;
}

// ---- taking pages --------------------------------------------------------------------------------------
// One block: the chunks' needs, their prefix sum, the free pages in ascending order, then table and counts.  The
// work is small (a few words per chunk and page); what bounds it is the chain of dependent loads: 6 us for 4 chunks, 9
// for 128.  (Several blocks would need a launch between the steps, 3 us each.)
struct GrowParams {
    int *table, *rows, *refs;
    int seqs, max_pages, pages, shift;
    const int *seq, *start;
    int* at;
    int n, total;
    int* missing;
    int2* pairs;  // [n]: a last page to copy {source, target}, source -1: none
    int* found;   // [pages]: the free pages
};

constexpr int kGrowThreads = 1024;

__global__ __launch_bounds__(kGrowThreads) void grow_kernel(GrowParams p) {
    __shared__ int s_seq[kMaxEntries], s_last[kMaxEntries], s_end[kMaxEntries + 1], s_part[kGrowThreads / 64], s_fail;
    const int tid = threadIdx.x, mask = (1 << p.shift) - 1;
    const long long cap = (long long)p.max_pages << p.shift;
    for (int i = tid; i < p.n; i += kGrowThreads) {
        const int s = p.seq ? p.seq[i] : i;
        s_seq[i] = s >= 0 && s < p.seqs ? s : -1;
    }
    if (tid == 0) s_fail = p.n;
    __syncthreads();
    for (int i = tid; i < p.n; i += kGrowThreads) {
        const int s = s_seq[i];
        int first, count, last = -1, old = -1;
        chunk_rows(p.start, i, p.total, &first, &count);
        bool ok = s >= 0;
        if (ok && p.seq)
            for (int j = 0; j < i; j++) ok &= s_seq[j] != s;
        if (ok) {
            old = p.rows[s];
            ok = old >= 0 && old + (long long)count <= cap;
        }
        if (ok && count > 0 && (old & mask)) {
            last = p.table[(size_t)s * p.max_pages + (old >> p.shift)];
            if (last < 0 || last >= p.pages) last = -1;
        }
        s_last[i] = ok ? last : -1;
        p.at[i] = ok ? old : -1;
    }
    __syncthreads();
    // need of each chunk; s_end: pages up to and with it
    int base = 0;
    for (int i0 = 0; i0 < p.n; i0 += kGrowThreads) {
        const int i = i0 + tid;
        int need = 0;
        if (i < p.n && p.at[i] >= 0) {
            int first, count;
            chunk_rows(p.start, i, p.total, &first, &count);
            const int old = p.at[i], last = s_last[i];
            if (count > 0) {
                need = (int)((((unsigned)old + count + mask) >> p.shift) - (((unsigned)old + mask) >> p.shift));
                if (last >= 0) {
                    int rank = 0;
                    for (int j = 0; j < i; j++) rank += s_last[j] == last;
                    if (rank < p.refs[last] - 1) need++;
                    else s_seq[i] |= 1 << 30;  // alone with it: keeps it
                }
            }
        }
        int sum;
        const int before = block_prefix<kGrowThreads>(need, s_part, &sum);
        if (i < p.n) s_end[i + 1] = base + before + need;
        base += sum;
    }
    if (tid == 0) s_end[0] = 0;
    // the lowest free pages, as many as are wanted
    int avail = 0;
    for (int g0 = 0; g0 < p.pages && avail < base; g0 += 4 * kGrowThreads) {
        const int g = g0 + 4 * tid;
        int free4[4], c = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            free4[u] = g + u < p.pages && p.refs[g + u] == 0;
            c += free4[u];
        }
        int sum;
        int k = avail + block_prefix<kGrowThreads>(c, s_part, &sum);
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (free4[u]) p.found[k++] = g + u;
        avail += sum;
    }
    if (avail > base) avail = base;
    __syncthreads();
    // chunks past the free pages; and a chunk that counted on an earlier one to leave their page
    for (int i = tid; i < p.n; i += kGrowThreads)
        if (s_end[i + 1] > avail && s_end[i + 1] > s_end[i]) atomicMin(&s_fail, i);
    __syncthreads();
    const int fail = s_fail;
    for (int i = tid; i < p.n; i += kGrowThreads) {
        const int old = p.at[i], last = s_last[i], s = s_seq[i] & ~(1 << 30);
        int2 pair = make_int2(-1, -1);
        if (old >= 0) {
            int first, count;
            chunk_rows(p.start, i, p.total, &first, &count);
            const int need = s_end[i + 1] - s_end[i];
            bool ok = s_end[i + 1] <= avail || need == 0;
            if (i > fail && last >= 0 && need == 0)
                for (int j = fail; j < i; j++) ok &= s_last[j] != last;
            const bool copies = last >= 0 && !(s_seq[i] & (1 << 30));
            if (ok) {
                int col = (old >> p.shift) + ((old & mask) && !copies ? 1 : 0);
                for (int k = s_end[i]; k < s_end[i + 1]; k++, col++) {
                    const int page = p.found[k];
                    p.table[(size_t)s * p.max_pages + col] = page;
                    p.refs[page] = 1;
                    if (copies && k == s_end[i]) {
                        pair = make_int2(last, page);
                        atomicSub(&p.refs[last], 1);
                    }
                }
                p.rows[s] = old + count;
            } else {
                p.at[i] = -1;
            }
        }
        p.pairs[i] = pair;
    }
    if (tid == 0 && p.missing) *p.missing = base - avail;
}

// ---- giving pages back -----------------------------------------------------------------------------------
// A block per entry (2 to 5 us, a launch and a chain of three loads).  Whether an earlier entry names the same sequence
// is looked up by all threads.
__device__ __forceinline__ bool named_before(const int* list, int i, int value) {
    bool found = false;
    if (list)
        for (int j = threadIdx.x; j < i; j += blockDim.x) found |= list[j] == value;
    return __syncthreads_or(found);
}

struct TrimParams {
    int *table, *rows, *refs;
    int seqs, max_pages, pages, shift;
    const int *seq, *keep;
};

__global__ __launch_bounds__(256) void trim_kernel(TrimParams p) {
    const int i = blockIdx.x, s = p.seq ? p.seq[i] : i;
    if (s < 0 || s >= p.seqs || named_before(p.seq, i, s)) return;
    const int have = p.rows[s], keep = p.keep ? max(p.keep[i], 0) : 0;
    if (keep >= have) return;
    const int mask = (1 << p.shift) - 1;
    const int end = min((int)(((long long)have + mask) >> p.shift), p.max_pages);
    for (int c = (int)(((long long)keep + mask) >> p.shift) + threadIdx.x; c < end; c += blockDim.x) {
        int* cell = &p.table[(size_t)s * p.max_pages + c];
        const int page = *cell;
        *cell = -1;
        if (page >= 0 && page < p.pages) atomicSub(&p.refs[page], 1);
    }
    __syncthreads();  // every thread has read the count
    if (threadIdx.x == 0) p.rows[s] = keep;
}

// ---- forking ---------------------------------------------------------------------------------------------
// Two launches (3 to 5 us each): the sources' table rows are set aside and counted, then the targets let go of theirs
// and take them.  Counts are added up with integer atomics, whose order does not show.
struct ForkParams {
    int *table, *rows, *refs;
    int seqs, max_pages, pages, shift;
    const int *src, *dst;
    int* kept;  // [n][1 + max_pages]: rows, then pages
};

__device__ __forceinline__ bool fork_entry(const ForkParams& p, int i, int* s, int* d) {
    *s = p.src[i];
    *d = p.dst[i];
    // (an earlier entry with an unknown source is passed over and does not stand in the way)
    bool out = *s < 0 || *s >= p.seqs || *d < 0 || *d >= p.seqs;
    if (!out)
        for (int j = threadIdx.x; j < i; j += blockDim.x) out |= p.dst[j] == *d && p.src[j] >= 0 && p.src[j] < p.seqs;
    return !__syncthreads_or(out) && *s != *d;
}

__device__ __forceinline__ int columns_of(const ForkParams& p, int rows) {
    if (rows <= 0) return 0;
    return min((int)(((long long)rows + (1 << p.shift) - 1) >> p.shift), p.max_pages);
}

__global__ __launch_bounds__(256) void fork_read_kernel(ForkParams p) {
    int s, d;
    if (!fork_entry(p, blockIdx.x, &s, &d)) return;
    int* kept = p.kept + (size_t)blockIdx.x * (1 + p.max_pages);
    const int rows = p.rows[s], cols = columns_of(p, rows);
    if (threadIdx.x == 0) kept[0] = rows;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
        const int page = p.table[(size_t)s * p.max_pages + c];
        kept[1 + c] = page;
        if (page >= 0 && page < p.pages) atomicAdd(&p.refs[page], 1);
    }
}

__global__ __launch_bounds__(256) void fork_write_kernel(ForkParams p) {
    int s, d;
    if (!fork_entry(p, blockIdx.x, &s, &d)) return;
    const int* kept = p.kept + (size_t)blockIdx.x * (1 + p.max_pages);
    const int rows = kept[0], cols = columns_of(p, rows), had = columns_of(p, p.rows[d]);
    for (int c = threadIdx.x; c < max(cols, had); c += blockDim.x) {
        int* cell = &p.table[(size_t)d * p.max_pages + c];
        if (c < had) {
            const int page = *cell;
            if (page >= 0 && page < p.pages) atomicSub(&p.refs[page], 1);
        }
        *cell = c < cols ? kept[1 + c] : -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) p.rows[d] = rows;
}

// ---- compacting --------------------------------------------------------------------------------------------
// One block ranks holes and movers (5 to 6 us), then the copies' blocks rewrite the table and move the pages: sources and
// targets are disjoint.  48 sequences of 1,100 rows, a third of them gone: 600 us for 3.1 GB, the copies' rate.
struct CompactParams {
    int* refs;
    int pages;
    int* live;
    int2* pairs;  // [pages / 2]: moves
    int* count;   // moves
    int* to;      // [pages]: where a page goes
};

__global__ __launch_bounds__(1024) void compact_plan_kernel(CompactParams p) {
    __shared__ int s_part[16];
    const int tid = threadIdx.x;
    int live = 0;
    for (int g0 = 0; g0 < p.pages; g0 += 4096) {
        int c = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) c += g0 + 4 * tid + u < p.pages && p.refs[g0 + 4 * tid + u] > 0;
        int sum;
        block_prefix<1024>(c, s_part, &sum);
        live += sum;
    }
    // holes before `live` and used pages from it on: as many of either
    int holes = 0, movers = 0;
    for (int g0 = 0; g0 < p.pages; g0 += 4096) {
        int used[4], h = 0, m = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int g = g0 + 4 * tid + u;
            used[u] = g < p.pages && p.refs[g] > 0;
            h += g < live && !used[u];
            m += g >= live && used[u];
        }
        int hs, ms;
        int kh = holes + block_prefix<1024>(h, s_part, &hs), km = movers + block_prefix<1024>(m, s_part, &ms);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int g = g0 + 4 * tid + u;
            if (g < live && !used[u]) p.pairs[kh++].y = g;
            if (g >= live && used[u]) p.pairs[km++].x = g;
            if (g < p.pages && (g < live || !used[u])) p.to[g] = g;
        }
        holes += hs;
        movers += ms;
    }
    __syncthreads();
    for (int k = tid; k < movers; k += 1024) {
        const int from = p.pairs[k].x, to = p.pairs[k].y;
        p.to[from] = to;
        p.refs[to] = p.refs[from];
        p.refs[from] = 0;
    }
    if (tid == 0) {
        *p.count = movers;
        if (p.live) *p.live = live;
    }
}

// ---- host side ----------------------------------------------------------------------------------------------

int check_counts(const ar_pages* p, const char* what) {
    AR_CHECK_ARG(p->rows && p->refs, "%s: the pool has no row counts or page counts", what);
    AR_CHECK_ARG(p->seqs > 0, "%s: the pool has no sequences", what);
    return AR_HIP_OK;
}

int check_entries(int n, const char* what) {
    AR_CHECK_ARG(n >= 0 && n <= kMaxEntries, "%s: %d entries not in [0,%d]", what, n, kMaxEntries);
    return AR_HIP_OK;
}

size_t work_bytes_of(const ar_pages* p, int n) {
    const size_t grow = (size_t)n * sizeof(int2) + (size_t)p->pages * 4;
    const size_t fork = (size_t)n * (1 + (size_t)p->max_pages) * 4;
    const size_t compact = 16 + (size_t)(p->pages / 2) * sizeof(int2) + (size_t)p->pages * 4;
    return std::max(std::max(grow, fork), std::max(compact, (size_t)16));
}

int check_work(const ar_pages* p, int n, const void* work, size_t have, const char* what) {
    const size_t need = work_bytes_of(p, n);
    AR_CHECK_ARG(work && have >= need, "%s: %zu bytes of work space given, %zu needed", what, work ? have : 0, need);
    AR_CHECK_ARG(((uintptr_t)work & 15) == 0, "%s: work space must be 16-byte aligned", what);
    return AR_HIP_OK;
}

int check_ranges(const ar_pages* p, const char* what) {
    if (!ar_check_ptrs_enabled()) return AR_HIP_OK;
    AR_TRY(page_check_ranges(p, what));
    AR_TRY(ar_check_range(p->rows, (size_t)p->seqs * 4, what, "row counts"));
    return ar_check_range(p->refs, (size_t)p->pages * 4, what, "page counts");
}
}  // namespace

int page_check(const ar_pages* p, bool table, const char* what) {
    AR_CHECK_ARG(p, "%s: pages is null", what);
    AR_CHECK_ARG(p->k && p->v, "%s: the pool has no keys or values", what);
    AR_CHECK_ARG((((uintptr_t)p->k | (uintptr_t)p->v) & 15) == 0, "%s: pools must be 16-byte aligned", what);
    AR_CHECK_ARG(p->dtype == AR_DTYPE_F32 || p->dtype == AR_DTYPE_BF16 || p->dtype == AR_DTYPE_F16,
                 "%s: unknown pool dtype %d", what, p->dtype);
    AR_CHECK_ARG(p->head_dim == 64 || p->head_dim == 128, "%s: head_dim %d not supported (64, 128)", what, p->head_dim);
    AR_CHECK_ARG(p->page_rows >= 16 && p->page_rows <= 256 && (p->page_rows & (p->page_rows - 1)) == 0,
                 "%s: page_rows %d is not a power of two in [16,256]", what, p->page_rows);
    AR_CHECK_ARG(p->layers > 0 && p->pages > 0 && p->kv_heads > 0, "%s: an empty pool", what);
    AR_CHECK_ARG(p->layers <= 4096 && p->kv_heads <= 4096 && p->pages <= 1 << 28,
                 "%s: more than 4096 layers, 4096 KV heads or 2^28 pages", what);
    AR_CHECK_ARG(p->seqs >= 0 && p->seqs < 1 << 30 && p->max_pages >= 0, "%s: table of %d sequences, %d pages each", what,
                 p->seqs, p->max_pages);
    AR_CHECK_ARG((long long)p->max_pages * p->page_rows <= 1LL << 30, "%s: table rows of %d pages of %d rows pass 2^30",
                 what, p->max_pages, p->page_rows);
    AR_CHECK_ARG(!table || (p->table && p->seqs > 0 && p->max_pages > 0), "%s: the pool has no table", what);
    return AR_HIP_OK;
}

int page_check_chunks(const ar_pages* p, const ar_chunks* c, const char* what) {
    AR_CHECK_ARG(c, "%s: chunks is null", what);
    AR_CHECK_ARG(c->at, "%s: chunks have no cache rows (at)", what);
    AR_CHECK_ARG(c->n > 0 && c->n <= 1 << 20, "%s: %d chunks not in [1,2^20]", what, c->n);
    AR_CHECK_ARG(c->rows >= 0, "%s: negative row count", what);
    AR_CHECK_ARG(c->rows <= 1 << 22, "%s: %d rows are more than 2^22", what, c->rows);
    AR_CHECK_ARG(c->start || c->rows >= c->n, "%s: %d rows for %d chunks of one row", what, c->rows, c->n);
    AR_CHECK_ARG(c->seq || c->n <= p->seqs, "%s: %d chunks for %d sequences", what, c->n, p->seqs);
    return AR_HIP_OK;
}

int page_check_ranges(const ar_pages* p, const char* what) {
    if (!ar_check_ptrs_enabled()) return AR_HIP_OK;
    const size_t pool = (size_t)p->layers * p->pages * p->kv_heads * p->page_rows * p->head_dim * page_elem_bytes(p->dtype);
    AR_TRY(ar_check_range(p->k, pool, what, "key pool"));
    AR_TRY(ar_check_range(p->v, pool, what, "value pool"));
    return ar_check_range(p->table, (size_t)p->seqs * p->max_pages * 4, what, "page table");
}

int page_check_chunk_ranges(const ar_chunks* c, const char* what) {
    if (!ar_check_ptrs_enabled()) return AR_HIP_OK;
    AR_TRY(ar_check_range(c->seq, (size_t)c->n * 4, what, "chunk sequences"));
    AR_TRY(ar_check_range(c->start, ((size_t)c->n + 1) * 4, what, "chunk starts"));
    return ar_check_range(c->at, (size_t)c->n * 4, what, "chunk cache rows");
}

extern "C" int ar_hip_pages_work(const ar_pages* pages, int n, size_t* bytes) {
    AR_TRY(page_check(pages, false, "pages work"));
    AR_TRY(check_entries(n, "pages work"));
    AR_CHECK_ARG(bytes, "pages work: bytes is null");
    *bytes = work_bytes_of(pages, n);
    return AR_HIP_OK;
}

extern "C" int ar_hip_pages_grow(ar_hip_ctx* ctx, const ar_pages* pages, const ar_chunks* chunks, int32_t* missing,
                                 void* work, size_t work_bytes) {
    const char* what = "pages grow";
    AR_TRY(page_check(pages, true, what));
    AR_TRY(check_counts(pages, what));
    AR_TRY(page_check_chunks(pages, chunks, what));
    AR_TRY(check_entries(chunks->n, what));
    AR_TRY(check_work(pages, chunks->n, work, work_bytes, what));
    AR_CHECK_ARG(ctx, "ctx is null");
    AR_TRY(check_ranges(pages, what));
    AR_TRY(page_check_chunk_ranges(chunks, what));
    AR_TRY(ar_check_range(missing, 4, what, "missing pages"));
    AR_TRY(ar_check_range(work, work_bytes_of(pages, chunks->n), what, "work space"));
    GrowParams g;
    g.table = pages->table; g.rows = pages->rows; g.refs = pages->refs; g.seqs = pages->seqs;
    g.max_pages = pages->max_pages; g.pages = pages->pages; g.shift = page_shift_of(pages);
    g.seq = chunks->seq; g.start = chunks->start; g.at = chunks->at; g.n = chunks->n; g.total = chunks->rows;
    g.missing = missing; g.pairs = (int2*)work; g.found = (int*)(g.pairs + chunks->n);
    hipLaunchKernelGGL(grow_kernel, dim3(1), dim3(kGrowThreads), 0, ctx->stream, g);
    AR_LAUNCH_CHECK();
    CopyParams c = copy_params(pages, pages);
    c.pairs = g.pairs;
    c.slots = chunks->n;
    return launch_copy(ctx, c);
}

extern "C" int ar_hip_pages_trim(ar_hip_ctx* ctx, const ar_pages* pages, const int32_t* seq, const int32_t* keep, int n) {
    const char* what = "pages trim";
    AR_TRY(page_check(pages, true, what));
    AR_TRY(check_counts(pages, what));
    AR_TRY(check_entries(n, what));
    AR_CHECK_ARG(seq || n <= pages->seqs, "%s: %d entries for %d sequences", what, n, pages->seqs);
    AR_CHECK_ARG(ctx, "ctx is null");
    if (n == 0) return AR_HIP_OK;
    AR_TRY(check_ranges(pages, what));
    AR_TRY(ar_check_range(seq, (size_t)n * 4, what, "sequences"));
    AR_TRY(ar_check_range(keep, (size_t)n * 4, what, "kept rows"));
    TrimParams t;
    t.table = pages->table; t.rows = pages->rows; t.refs = pages->refs; t.seqs = pages->seqs;
    t.max_pages = pages->max_pages; t.pages = pages->pages; t.shift = page_shift_of(pages); t.seq = seq; t.keep = keep;
    hipLaunchKernelGGL(trim_kernel, dim3(n), dim3(256), 0, ctx->stream, t);
    AR_LAUNCH_CHECK();
    return AR_HIP_OK;
}

extern "C" int ar_hip_pages_fork(ar_hip_ctx* ctx, const ar_pages* pages, const int32_t* src, const int32_t* dst, int n,
                                 void* work, size_t work_bytes) {
    const char* what = "pages fork";
    AR_TRY(page_check(pages, true, what));
    AR_TRY(check_counts(pages, what));
    AR_TRY(check_entries(n, what));
    AR_CHECK_ARG(src && dst, "%s: null sequence list", what);
    AR_TRY(check_work(pages, n, work, work_bytes, what));
    AR_CHECK_ARG(ctx, "ctx is null");
    if (n == 0) return AR_HIP_OK;
    AR_TRY(check_ranges(pages, what));
    AR_TRY(ar_check_range(src, (size_t)n * 4, what, "sources"));
    AR_TRY(ar_check_range(dst, (size_t)n * 4, what, "targets"));
    AR_TRY(ar_check_range(work, work_bytes_of(pages, n), what, "work space"));
    ForkParams f;
    f.table = pages->table; f.rows = pages->rows; f.refs = pages->refs; f.seqs = pages->seqs;
    f.max_pages = pages->max_pages; f.pages = pages->pages; f.shift = page_shift_of(pages); f.src = src; f.dst = dst;
    f.kept = (int*)work;
    hipLaunchKernelGGL(fork_read_kernel, dim3(n), dim3(256), 0, ctx->stream, f);
    AR_LAUNCH_CHECK();
    hipLaunchKernelGGL(fork_write_kernel, dim3(n), dim3(256), 0, ctx->stream, f);
    AR_LAUNCH_CHECK();
    return AR_HIP_OK;
}

extern "C" int ar_hip_pages_compact(ar_hip_ctx* ctx, const ar_pages* pages, int32_t* live, void* work,
                                    size_t work_bytes) {
    const char* what = "pages compact";
    AR_TRY(page_check(pages, true, what));
    AR_CHECK_ARG(pages->refs, "%s: the pool has no page counts", what);
    AR_TRY(check_work(pages, 0, work, work_bytes, what));
    AR_CHECK_ARG(ctx, "ctx is null");
    if (ar_check_ptrs_enabled()) {
        AR_TRY(page_check_ranges(pages, what));
        AR_TRY(ar_check_range(pages->refs, (size_t)pages->pages * 4, what, "page counts"));
        AR_TRY(ar_check_range(live, 4, what, "live pages"));
        AR_TRY(ar_check_range(work, work_bytes_of(pages, 0), what, "work space"));
    }
    CompactParams c;
    c.refs = pages->refs; c.pages = pages->pages; c.live = live; c.count = (int*)work; c.pairs = (int2*)((char*)work + 16);
    c.to = (int*)(c.pairs + pages->pages / 2);
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(1024), 0, ctx->stream, c);
    AR_LAUNCH_CHECK();
    if (pages->pages < 2) return AR_HIP_OK;  // (nothing can move)
    CopyParams m = copy_params(pages, pages);
    m.pairs = c.pairs;
    m.count = c.count;
    m.slots = pages->pages / 2;
    m.table = pages->table;
    m.to = c.to;
    m.cells = (size_t)pages->seqs * pages->max_pages;
    return launch_copy(ctx, m);
}

extern "C" int ar_hip_pages_copy(ar_hip_ctx* ctx, const ar_pages* from, const ar_pages* to, const int32_t* src,
                                 const int32_t* dst, int n) {
    const char* what = "pages copy";
    AR_TRY(page_check(from, false, what));
    AR_TRY(page_check(to, false, what));
    AR_CHECK_ARG(from->dtype == to->dtype && from->layers == to->layers && from->kv_heads == to->kv_heads &&
                     from->page_rows == to->page_rows && from->head_dim == to->head_dim,
                 "%s: the pools differ in dtype, layers, kv_heads, page_rows or head_dim", what);
    const bool same = from->k == to->k && from->v == to->v;
    AR_CHECK_ARG(!same || from->pages == to->pages, "%s: one pool with two page counts", what);
    const size_t page = (size_t)from->layers * from->kv_heads * from->page_rows * from->head_dim * page_elem_bytes(from->dtype);
    auto overlap = [&](const void* a, int na, const void* b, int nb) {
        const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
        return x < y + page * nb && y < x + page * na;
    };
    AR_CHECK_ARG(same || !(overlap(from->k, from->pages, to->k, to->pages) || overlap(from->v, from->pages, to->v, to->pages) ||
                           overlap(from->k, from->pages, to->v, to->pages) || overlap(from->v, from->pages, to->k, to->pages)),
                 "%s: the pools share part of their memory", what);
    AR_TRY(check_entries(n, what));
    AR_CHECK_ARG(src && dst, "%s: null page list", what);
    AR_CHECK_ARG(ctx, "ctx is null");
    if (n == 0) return AR_HIP_OK;
    AR_TRY(page_check_ranges(from, what));
    AR_TRY(page_check_ranges(to, what));
    AR_TRY(ar_check_range(src, (size_t)n * 4, what, "sources"));
    AR_TRY(ar_check_range(dst, (size_t)n * 4, what, "targets"));
    CopyParams c = copy_params(from, to);
    c.src = src;
    c.dst = dst;
    c.slots = n;
    c.same_pool = same;
    return launch_copy(ctx, c);
}
