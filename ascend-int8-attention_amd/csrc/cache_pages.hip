// MI355X (gfx950) operations on the pages of an INT8 cache pool: accepted
// paths of drafted tokens, forked and freed rows of a block table, compaction.
// The argument blocks and their rules are in sharedkv_hip.h.
//
// None of these computes; each is bound by the bytes it moves (whole pages and
// rows, 16 bytes a lane) and, where these are few, by its chain of dependent
// reads.  Which page goes where follows from counts: the k-th free or moving
// page in index order, found with prefix sums over chunks of the reference
// counts, so the result does not depend on the order in which work-groups run.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sharedkv_hip.h"

namespace {

constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;
constexpr int PER_THREAD = 8;
constexpr int CHUNK = THREADS * PER_THREAD;     // pages whose counts one work-group takes
constexpr int MAX_CHUNKS = 2048;
constexpr int64_t MAX_PAGES = (int64_t)CHUNK * MAX_CHUNKS;
constexpr int PATH = 64;                        // path entries that are resident at once
constexpr int64_t SLICE = 65536;                // bytes of a page that one work-group copies
// Chunks up to which compact_plan counts the pool itself, in every work-group, where a launch before it would (16 KiB
// pages, half of them in use, microseconds counted by itself and before: 3000 pages 15.5 and 16.9, 4096 17.0 and 18.2,
// 6000 25.5 and 22.2, 16000 46.4 and 31.9).
constexpr uint32_t FEW_CHUNKS = 2;
// Pools above this size do not fit the memory-side cache: compaction copies past it (1536 pages of 608 KiB with 380
// moves: 88.6 us, 96.4 with ordinary copies).  Forked tails are read again soon and stay (64 beams: 11.5 us, 13.1 past it).
constexpr uint64_t STREAMED_POOL = 256ull << 20;
constexpr int COPY = 8;                          // 16-byte units of a thread that are under way at once
constexpr int WANTED = -2;                      // a staged entry that gets a free page
// Work-groups of a launch: their threads are counted in 32 bits.  Checked before the first of a call's launches, so
// that a refused call leaves the workspace as it was.
constexpr uint64_t MAX_GROUPS = 0xffffffffull / THREADS;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ const __attribute__((address_space(1))) T *gptr(uint64_t a)
{
    return reinterpret_cast<const __attribute__((address_space(1))) T *>(a);
}
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T *gout(uint64_t a)
{
    return reinterpret_cast<__attribute__((address_space(1))) T *>(a);
}

// Eight words from `at` on of an array of `count`, `other` past its end; in two loads where they may be.
__device__ __forceinline__ void load_words(int (&v)[PER_THREAD], uint64_t array, int64_t at, int64_t count, int other)
{
    if (at + PER_THREAD <= count && !(array & 15)) {
        const u32x4 a = gptr<u32x4>(array)[at / 4], b = gptr<u32x4>(array)[at / 4 + 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (int)a[i], v[4 + i] = (int)b[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) v[i] = at + i < count ? gptr<int32_t>(array)[at + i] : other;
}

// Sum over the work-group, in every thread.
__device__ __forceinline__ int block_sum(int v)
{
    __shared__ int part[WAVES];
#pragma unroll
    for (int step = 32; step; step /= 2) v += __shfl_xor(v, step);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += part[w];
    return total;
}

// Sum over the threads before this one; `total` gets the whole.
__device__ __forceinline__ int block_before(int v, int &total)
{
    __shared__ int part[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto = v;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int other = __shfl_up(upto, step);
        if (lane >= step) upto += other;
    }
    __syncthreads();
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    total = 0;
    int before = upto - v;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before;
}

__device__ __forceinline__ CacheSpan span_at(uint64_t caches, uint32_t c)
{
    const auto *from = gptr<CacheSpan>(caches) + c;
    CacheSpan span;
    span.base = from->base, span.pageStride = from->pageStride, span.rowStride = from->rowStride, span.bytes = from->bytes;
    return span;
}

// Bytes [first, last) of page `from` to page `to`, over the caches one after
// another (all multiples of 16); `span` is the first cache.
template <bool STREAM = false>
__device__ __forceinline__ void copy_page(uint64_t caches, uint32_t count, CacheSpan span, int64_t from, int64_t to,
                                          int64_t first, int64_t last)
{
    int64_t at = 0;
    for (uint32_t c = 0; c < count && at < last; ++c) {
        if (c) span = span_at(caches, c);
        const int64_t bytes = (int64_t)span.bytes;
        const int64_t lo = first > at ? first - at : 0, hi = last - at < bytes ? last - at : bytes;
        if (lo < hi) {
            const auto *src = gptr<u32x4>(span.base + (uint64_t)from * span.pageStride);
            auto *dst = gout<u32x4>(span.base + (uint64_t)to * span.pageStride);
            const int64_t end = hi / 16;
            int64_t i = lo / 16 + threadIdx.x;
            for (; i + (COPY - 1) * THREADS < end; i += COPY * THREADS) {
                u32x4 v[COPY];
#pragma unroll
                for (int k = 0; k < COPY; ++k)
                    v[k] = STREAM ? __builtin_nontemporal_load(&src[i + k * THREADS]) : src[i + k * THREADS];
#pragma unroll
                for (int k = 0; k < COPY; ++k)
                    if (STREAM) __builtin_nontemporal_store(v[k], &dst[i + k * THREADS]);
                    else dst[i + k * THREADS] = v[k];
            }
            for (; i < end; i += THREADS) dst[i] = src[i];
        }
        at += bytes;
    }
}

// ------------------------------------------------------------ accepted paths

// One work-group moves a 16-byte column per thread through a request's path:
// a thread reads a few entries ahead of its writes, which never reach a row
// that it still has to read (paths[k] >= k and rises).  Few rows move, so this is
// a launch and its two round trips (lengths and path, then the table): 4.1 us for
// one request, 5.2 for 64 with paths of a few tokens in every layer (11 MB, 2.2
// TB/s).
constexpr int AHEAD = 8;
__global__ void __launch_bounds__(THREADS) path_commit(const PathCommitArgs p)
{
    __shared__ int32_t place[PATH][4];           // page (-1: no move) and row of source and target
    __shared__ int kept;
    const int tid = threadIdx.x, b = (int)blockIdx.x;
    const int tokens = (int)p.tokens;
    const int first = min(max(gptr<int32_t>(p.cuQ)[b], 0), tokens);
    const int nodes = min(max(gptr<int32_t>(p.cuQ)[b + 1], first), tokens) - first;
    const int length = gptr<int32_t>(p.seqLens)[b];
    const int most = length > 0 ? min(max(gptr<int32_t>(p.pathLens)[b], 0), (int)p.depth) : 0;
    const int committed = max(0, length - nodes);
    const uint32_t columns = p.rowBytes / 16, item = blockIdx.y * THREADS + tid;
    const uint32_t cache = item / columns, column = item % columns;
    CacheSpan span = {};
    if (cache < p.cacheCount) span = span_at(p.caches, cache);
    const bool mine = cache < p.cacheCount && column * 16 < span.bytes;
    const auto *path = gptr<int32_t>(p.paths) + (int64_t)b * p.depth;
    int done = 0;
    for (int at = 0; at < most; at += PATH) {
        __syncthreads();
        if (tid < 64) {
            const int k = at + tid;
            const int node = k < most ? path[k] : -1, before = k > 0 && k < most ? path[k - 1] : -1;
            const bool good = k < most && node > before && node < nodes;
            const uint64_t bad = __ballot(!good);
            const int n = bad ? __builtin_ctzll(bad) : 64;
            if (tid == 0) kept = n;
            int32_t page[2] = {-1, -1}, row[2] = {0, 0};
            if (tid < n && node != k) {
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    const int64_t at_row = (int64_t)committed + (side ? k : node);
                    const int64_t e = at_row / p.pageRows;
                    page[side] = e < p.tableWidth ? gptr<int32_t>(p.table)[(int64_t)b * p.tableWidth + e] : -1;
                    row[side] = (int32_t)(at_row % p.pageRows);
                }
            }
            const bool moves = (uint32_t)page[0] < p.pages && (uint32_t)page[1] < p.pages;
            place[tid][0] = moves ? page[0] : -1;
            place[tid][1] = row[0];
            place[tid][2] = page[1];
            place[tid][3] = row[1];
        }
        __syncthreads();
        const int n = kept;
        done += n;
        if (mine) {
            for (int k = 0; k < n; k += AHEAD) {
                u32x4 v[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    if (k + i < n && place[k + i][0] >= 0)
                        v[i] = gptr<u32x4>(span.base + (uint64_t)place[k + i][0] * span.pageStride +
                                           (uint64_t)place[k + i][1] * span.rowStride)[column];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i)
                    if (k + i < n && place[k + i][0] >= 0)
                        gout<u32x4>(span.base + (uint64_t)place[k + i][2] * span.pageStride +
                                    (uint64_t)place[k + i][3] * span.rowStride)[column] = v[i];
            }
        }
        if (n < PATH) break;
    }
    if (blockIdx.y == 0 && tid == 0)
        reinterpret_cast<int32_t *>(p.lengths)[b] = length > 0 ? committed + done : 0;
}

// ------------------------------------------------------------ fork

struct ForkSpace {
    int32_t *staged;       // [children][width] new entries, WANTED where a free page comes
    int32_t *source;       // [children] page of the parent's partly filled entry
    int32_t *need;         // [children] free pages wanted
    int32_t *length;       // [children] the parent's length
    int32_t *tail;         // [children] the staged entry of the partly filled page
    int32_t *freed;        // [chunks][CHUNK] the chunk's free pages, in order
    int32_t *count;        // [chunks] how many there are
    int32_t *delta;        // [pages] change of the reference counts; zero between launches
};
__host__ __device__ inline uint32_t chunks_of(uint32_t pages) { return (pages + CHUNK - 1) / CHUNK; }
__host__ __device__ inline uint64_t fork_words(uint32_t children, uint32_t width, uint32_t pages)
{
    const uint64_t chunks = chunks_of(pages);
    return (uint64_t)pages + (uint64_t)children * (width + 4) + chunks * (CHUNK + 1);
}
__device__ __forceinline__ ForkSpace fork_space(const PageForkArgs &p)
{
    ForkSpace w;
    w.delta = reinterpret_cast<int32_t *>(p.workspace);
    w.staged = w.delta + p.pages;
    w.source = w.staged + (int64_t)p.children * p.width;
    w.need = w.source + p.children;
    w.length = w.need + p.children;
    w.tail = w.length + p.children;
    w.count = w.tail + p.children;
    w.freed = w.count + chunks_of(p.pages);
    return w;
}

// A row's length and what follows from it: whole pages, pages with room.
struct Extent {
    int32_t length, whole, needed;
};
__device__ __forceinline__ Extent extent_of(const PageForkArgs &p, int seq_len)
{
    const int64_t most = (int64_t)p.width * p.pageRows;
    const int64_t length = min(max((int64_t)seq_len, (int64_t)0), min(most, (int64_t)0x7fffffff));
    Extent x;
    x.length = (int32_t)length;
    x.whole = (int32_t)((uint32_t)x.length / p.pageRows);
    x.needed = (int32_t)min((int64_t)p.width, (length + p.room + p.pageRows - 1) / p.pageRows);
    return x;
}

// Work-groups: the new rows (staged entries, free pages wanted), the old rows
// (reference counts), the chunks of pages (free pages).  Bound by the chain of
// reads parent -> row and length -> counts, so whatever does not depend on the
// last read is requested with it.  Two launches, since free pages are handed out
// in the order of all rows before any is written: 7.6 us where one request goes
// on as four, 9.1 for 256 rows of a one-layer pool, and 10.8 where 64 tails of all
// layers are copied (29 MB, 2.7 TB/s).
__global__ void __launch_bounds__(THREADS) fork_plan(const PageForkArgs p)
{
    const ForkSpace w = fork_space(p);
    const int tid = threadIdx.x, width = (int)p.width;
    const auto *refs = gptr<int32_t>(p.refs), *table = gptr<int32_t>(p.table), *parents = gptr<int32_t>(p.parents);
    uint32_t at = blockIdx.x;
    if (at < p.children) {
        const int parent = parents[at];
        int others = tid < (int)at ? parents[tid] : -1;          // children before this one
        const bool alive = (uint32_t)parent < p.rows;
        const int64_t row = alive ? (int64_t)parent * width : 0;
        const int length = gptr<int32_t>(p.seqLens)[alive ? parent : 0];
        int old = tid < width ? table[row + tid] : -1;
        int same = others == parent;
        for (int i = tid + THREADS; i < (int)at; i += THREADS) same += parents[i] == parent;
        Extent x = {};
        if (alive) x = extent_of(p, length);
        const bool first = block_sum(same) == 0;
        int wanted = 0;
        for (int e = tid; e < width; e += THREADS) {
            if (e >= THREADS) old = e < x.needed ? table[row + e] : -1;
            const bool good = (uint32_t)old < p.pages;
            int entry = -1;
            if (e < x.whole) entry = good ? old : -1;
            else if (e < x.needed) {
                entry = first && good && refs[old] == 1 ? old : WANTED;
                wanted += entry == WANTED;
            }
            w.staged[(int64_t)at * width + e] = entry;
            if (e == x.whole) w.source[at] = alive && good ? old : -1, w.tail[at] = entry;
        }
        wanted = block_sum(wanted);
        if (tid == 0) w.need[at] = wanted, w.length[at] = x.length;
        return;
    }
    at -= p.children;
    if (at < p.rows) {
        int old = tid < width ? table[(int64_t)at * width + tid] : -1;
        const Extent x = extent_of(p, gptr<int32_t>(p.seqLens)[at]);
        int children = 0;
        for (int i = tid; i < (int)p.children; i += THREADS) children += parents[i] == (int)at;
        children = block_sum(children);
        for (int e = tid; e < width; e += THREADS) {
            if (e >= THREADS) old = table[(int64_t)at * width + e];
            if ((uint32_t)old >= p.pages) continue;
            const int held = e < x.whole ? children : children && e < x.needed && refs[old] == 1 ? 1 : 0;
            if (held != 1) atomicAdd(&w.delta[old], held - 1);
        }
        return;
    }
    at -= p.rows;
    const int64_t page = (int64_t)at * CHUNK + tid * PER_THREAD;
    int held[PER_THREAD], mine = 0;
    load_words(held, p.refs, page, p.pages, 1);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) mine += held[i] == 0;
    int total, rank = block_before(mine, total);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i)
        if (held[i] == 0) w.freed[(int64_t)at * CHUNK + rank++] = (int32_t)(page + i);
    if (tid == 0) w.count[at] = total;
}

// Work-groups: slices of the new rows (the first writes the row, all copy its
// partly filled page), then the chunks of pages (reference counts).  The old
// table, lengths and counts may be the new ones: rows come from the workspace
// and a page's count is read by the thread that writes it.
__global__ void __launch_bounds__(THREADS) fork_apply(const PageForkArgs p, uint32_t slices)
{
    __shared__ int32_t upto[MAX_CHUNKS];         // free pages up to and with each chunk
    const ForkSpace w = fork_space(p);
    const int tid = threadIdx.x;
    const int chunks = (int)chunks_of(p.pages);
    uint32_t at = blockIdx.x;
    if (at < p.children * slices) {
        const int row = (int)(at / slices), slice = (int)(at % slices), width = (int)p.width;
        // One round trip: the row's own words, the needs of those before it, the counts, the row and the first cache.
        const int wanted = w.need[row], length = w.length[row], source_page = w.source[row];
        const int staged_tail = w.tail[row];
        const int first_entry = slice == 0 && tid < width ? w.staged[(int64_t)row * width + tid] : -1;
        const CacheSpan span = span_at(p.caches, 0);
        int count = tid < chunks ? w.count[tid] : 0;
        int before = 0;
        for (int i = tid; i < row; i += THREADS) before += w.need[i];
        before = block_sum(before);
        int free_pages = 0;
        for (int c = 0; c < chunks; c += THREADS) {
            if (c) count = c + tid < chunks ? w.count[c + tid] : 0;
            int total;
            const int ahead = block_before(count, total);
            if (c + tid < chunks) upto[c + tid] = free_pages + ahead + count;
            free_pages += total;
        }
        __syncthreads();
        auto fresh = [&](int rank) {
            if (rank >= free_pages) return -1;
            int lo = 0, hi = chunks - 1;         // the first chunk with more than `rank` up to its end
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (upto[mid] > rank) hi = mid;
                else lo = mid + 1;
            }
            return w.freed[(int64_t)lo * CHUNK + rank - (lo ? upto[lo - 1] : 0)];
        };
        const int whole = (int)((uint32_t)length / p.pageRows);
        const bool partly = (uint32_t)length % p.pageRows != 0;
        const int tail = partly ? staged_tail : -1;
        const int target = tail == WANTED ? fresh(before) : tail;
        const int source = partly && tail == WANTED ? source_page : -1;
        if (slice == 0) {
            int rank = before;
            for (int e0 = 0; e0 < width; e0 += THREADS) {
                const int e = e0 + tid;
                int entry = e0 == 0 ? first_entry : e < width ? w.staged[(int64_t)row * width + e] : -1;
                int total = 0, ahead = 0;
                if (wanted) ahead = block_before(entry == WANTED, total);
                if (entry == WANTED) entry = fresh(rank + ahead);
                rank += total;
                if (e < width) gout<int32_t>(p.newTable)[(int64_t)row * width + e] = entry;
            }
            if (tid == 0) gout<int32_t>(p.newLens)[row] = partly && target < 0 ? whole * (int)p.pageRows : length;
        }
        if (source >= 0 && target >= 0)
            copy_page(p.caches, p.cacheCount, span, source, target, slice * SLICE, (slice + 1) * SLICE);
        return;
    }
    at -= p.children * slices;
    const int64_t page = (int64_t)at * CHUNK + tid * PER_THREAD;
    int held[PER_THREAD], change[PER_THREAD], mine = 0;
    load_words(held, p.refs, page, p.pages, 1);
    load_words(change, (uint64_t)(uintptr_t)w.delta, page, p.pages, 0);
    int needed = 0, before = 0, free_pages = 0;
    for (int i = tid; i < (int)p.children; i += THREADS) needed += w.need[i];
    for (int c = tid; c < chunks; c += THREADS) {
        free_pages += w.count[c];
        if (c < (int)at) before += w.count[c];
    }
    needed = block_sum(needed);
    before = block_sum(before);
    if (at == 0) {
        free_pages = block_sum(free_pages);
        if (tid == 0) gout<int32_t>(p.missing)[0] = max(0, needed - free_pages);
    }
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) mine += held[i] == 0;
    int total, rank = before + block_before(mine, total);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i)
        if (page + i < p.pages) {
            if (change[i]) w.delta[page + i] = 0;
            const int given = held[i] == 0 && rank++ < needed;
            gout<int32_t>(p.newRefs)[page + i] = held[i] + change[i] + given;
        }
}

// ------------------------------------------------------------ compaction

struct CompactSpace {
    int32_t *count;        // [chunks] pages in use
    int32_t *moves;        // [1]
    int32_t *place;        // [pages] a page's own number, -1, or -2 - k: the k-th that moves
    int32_t *target;       // [pages] free pages below L
    int32_t *source;       // [pages] pages that move
    int32_t *refs;         // [pages] their reference counts
};
__host__ __device__ inline uint64_t compact_words(uint32_t pages) { return (uint64_t)chunks_of(pages) + 1 + 4ull * pages; }
__device__ __forceinline__ CompactSpace compact_space(const PageCompactArgs &p)
{
    CompactSpace w;
    w.count = reinterpret_cast<int32_t *>(p.workspace);
    w.moves = w.count + chunks_of(p.pages);
    w.place = w.moves + 1;
    w.target = w.place + p.pages;
    w.source = w.target + p.pages;
    w.refs = w.source + p.pages;
    return w;
}

__global__ void __launch_bounds__(THREADS) compact_count(const PageCompactArgs p)
{
    const CompactSpace w = compact_space(p);
    const int64_t page = (int64_t)blockIdx.x * CHUNK + threadIdx.x * PER_THREAD;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) mine += page + i < p.pages && gptr<int32_t>(p.refs)[page + i] > 0;
    const int total = block_sum(mine);
    if (threadIdx.x == 0) w.count[blockIdx.x] = total;
}

__global__ void __launch_bounds__(THREADS) compact_plan(const PageCompactArgs p)
{
    const CompactSpace w = compact_space(p);
    const int tid = threadIdx.x, chunks = (int)chunks_of(p.pages), chunk = (int)blockIdx.x;
    const auto *refs = gptr<int32_t>(p.refs);
    const bool few = chunks <= (int)FEW_CHUNKS;
    int before = 0, live = 0, below = 0;
    if (few)                                     // compact_count has not run
        for (int c = 0; c < chunks; ++c) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < PER_THREAD; ++i) {
                const int64_t page = (int64_t)c * CHUNK + i * THREADS + tid;
                n += page < p.pages && refs[page] > 0;
            }
            live += n;
            if (c < chunk) before += n;
        }
    else
        for (int c = tid; c < chunks; c += THREADS) {
            live += w.count[c];
            if (c < chunk) before += w.count[c];
        }
    before = block_sum(before);
    live = block_sum(live);
    // Pages in use below L: whole chunks, then a part of L's chunk.
    const int last = few ? 0 : live / CHUNK;
    for (int c = tid; c < min(last, chunks); c += THREADS) below += w.count[c];
    for (int64_t i = (int64_t)last * CHUNK + tid; i < live; i += THREADS) below += refs[i] > 0;
    below = block_sum(below);
    if (chunk == 0 && tid == 0) {
        w.moves[0] = live - below;
        gout<int32_t>(p.live)[0] = live;
    }
    const int64_t page = (int64_t)chunk * CHUNK + tid * PER_THREAD;
    int held[PER_THREAD], mine = 0;
    load_words(held, p.refs, page, p.pages, 0);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) mine += held[i] > 0;
    int total, rank = before + block_before(mine, total);
    if (few && tid == 0) w.count[chunk] = total;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int64_t at = page + i;
        if (at >= p.pages) break;
        int place = -1;
        if (held[i] > 0) {
            place = (int)at;
            if (at >= live) {
                const int k = rank - below;
                place = -2 - k;
                w.source[k] = (int)at;
                w.refs[k] = held[i];
            }
            ++rank;
        } else if (at < live)
            w.target[at - rank] = (int)at;
        w.place[at] = place;
    }
}

// Work-groups: copies, chunks of table entries, chunks of pages.
template <bool STREAM>
__global__ void __launch_bounds__(THREADS) compact_apply(const PageCompactArgs p, uint32_t table_groups, uint32_t copies,
                                                         uint32_t slices)
{
    const CompactSpace w = compact_space(p);
    const int tid = threadIdx.x;
    uint32_t at = blockIdx.x;
    auto settle = [&](int place) { return place <= -2 ? w.target[-2 - place] : place; };
    if (at < copies) {
        const int64_t items = (int64_t)w.moves[0] * slices;
        const CacheSpan span = span_at(p.caches, 0);
        for (int64_t i = at; i < items; i += copies) {
            const int k = (int)(i / slices);
            const int64_t slice = i % slices;
            copy_page<STREAM>(p.caches, p.cacheCount, span, w.source[k], w.target[k], slice * SLICE, (slice + 1) * SLICE);
        }
        return;
    }
    at -= copies;
    if (at < table_groups) {
        const int64_t first = (int64_t)at * CHUNK, end = min(first + CHUNK, (int64_t)p.rows * p.width);
        for (int64_t i = first + tid; i < end; i += THREADS) {
            const int page = gptr<int32_t>(p.table)[i];
            gout<int32_t>(p.newTable)[i] = (uint32_t)page < p.pages ? settle(w.place[page]) : -1;
        }
        return;
    }
    at -= table_groups;
    const int live = gptr<int32_t>(p.live)[0];
    const int64_t page = (int64_t)at * CHUNK + tid * PER_THREAD;
    int held[PER_THREAD];
    load_words(held, p.refs, page, p.pages, 0);
    // Free pages of the chunk below L take the pages that move, in order: their rank is what is left of their index.
    int spare = 0;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) spare += page + i < live && held[i] <= 0;
    int total, rank = block_before(spare, total);
    int before = 0;
    for (int c = tid; c < (int)at; c += THREADS) before += CHUNK - w.count[c];
    rank += block_sum(before);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        if (page + i >= p.pages) break;
        const bool inside = page + i < live;
        int count = 0;
        if (inside) count = held[i] > 0 ? held[i] : w.refs[rank++];
        gout<int32_t>(p.newRefs)[page + i] = count;
        gout<int32_t>(p.moved)[page + i] = settle(w.place[page + i]);
    }
}

// Compaction of a pool of one chunk in one launch, where no output is an
// input: every work-group counts the pages for itself, in LDS, instead of
// reading what two launches before it have counted (509 pages with 41 moves of
// 16 KiB: 4.9 us, 12.8 in three launches; 1536 pages of 608 KiB with 380 moves:
// 89.5 us, 5.3 TB/s, as a plain copy of that size).
template <bool STREAM>
__global__ void __launch_bounds__(THREADS) compact_small(const PageCompactArgs p, uint32_t table_groups, uint32_t copies,
                                                         uint32_t slices)
{
    __shared__ int32_t place[CHUNK], target[CHUNK], source[CHUNK];
    const int tid = threadIdx.x;
    uint32_t at = blockIdx.x;
    const CacheSpan span = span_at(p.caches, 0);
    // This work-group's first table entry is on its way meanwhile.
    const int64_t first = ((int64_t)at - copies) * THREADS + tid, entries = (int64_t)p.rows * p.width;
    const bool has_entry = at >= copies && at < copies + table_groups && first < entries;
    const int entry = has_entry ? gptr<int32_t>(p.table)[first] : -1;
    int held[PER_THREAD], mine = 0;
    load_words(held, p.refs, tid * PER_THREAD, p.pages, 0);
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) mine += held[i] > 0;
    int live, rank = block_before(mine, live), inside = 0;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) inside += held[i] > 0 && tid * PER_THREAD + i < live;
    const int below = block_sum(inside), moves = live - below;
    int its_rank = rank;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int page = tid * PER_THREAD + i;
        int its = -1;
        if (held[i] > 0) {
            its = page;
            if (page >= live) its = -2 - (its_rank - below), source[its_rank - below] = page;
            ++its_rank;
        } else if (page < live)
            target[page - its_rank] = page;
        place[page] = its;
    }
    __syncthreads();
    auto settle = [&](int its) { return its <= -2 ? target[-2 - its] : its; };
    if (at < copies) {
        for (int64_t i = at; i < (int64_t)moves * slices; i += copies) {
            const int k = (int)(i / slices);
            const int64_t slice = i % slices;
            copy_page<STREAM>(p.caches, p.cacheCount, span, source[k], target[k], slice * SLICE, (slice + 1) * SLICE);
        }
        return;
    }
    if (at < copies + table_groups) {
        if (has_entry) gout<int32_t>(p.newTable)[first] = (uint32_t)entry < p.pages ? settle(place[entry]) : -1;
        return;
    }
    // A page below L that was free takes the count of the page that moves there.
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
        const int page = tid * PER_THREAD + i;
        if (page >= (int)p.pages) break;
        int count = 0;
        if (page < live) count = held[i] > 0 ? held[i] : gptr<int32_t>(p.refs)[source[page - rank]];
        rank += held[i] > 0;
        gout<int32_t>(p.newRefs)[page] = count;
        gout<int32_t>(p.moved)[page] = settle(place[page]);
    }
    if (tid == 0) gout<int32_t>(p.live)[0] = live;
}

}  // namespace

extern "C" {

int launch_sharedkv_path_commit(void *stream, const PathCommitArgs *a)
{
    if (!a || !a->caches || !a->table || !a->cuQ || !a->seqLens || !a->paths || !a->pathLens || !a->lengths)
        return (int)hipErrorInvalidValue;
    if (!a->cacheCount || !a->tableWidth || !a->pages || !a->pageRows || !a->rowBytes || (a->rowBytes & 15) || !a->depth)
        return (int)hipErrorInvalidValue;
    if (a->pages > 0x7fffffffu || a->tokens > 0x7fffffffu || a->depth > 0x3fffffffu) return (int)hipErrorInvalidValue;
    if (!a->batch) return (int)hipSuccess;
    const uint64_t groups = ((uint64_t)a->cacheCount * (a->rowBytes / 16) + THREADS - 1) / THREADS;
    if (groups > 65535 || a->batch > MAX_GROUPS) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(path_commit, dim3(a->batch, (uint32_t)groups), dim3(THREADS), 0, static_cast<hipStream_t>(stream), *a);
    return (int)hipGetLastError();
}

int launch_sharedkv_page_fork(void *stream, const PageForkArgs *a)
{
    if (!a || !a->caches || !a->table || !a->seqLens || !a->refs || !a->parents || !a->newTable || !a->newLens ||
        !a->newRefs || !a->missing || !a->workspace)
        return (int)hipErrorInvalidValue;
    if (!a->cacheCount || !a->rows || !a->children || !a->width || !a->pages || !a->pageRows || !a->pageBytes)
        return (int)hipErrorInvalidValue;
    const uint64_t slices = (a->pageBytes + SLICE - 1) / SLICE;
    if (a->pages > MAX_PAGES || a->rows > 0xfffffu || a->children > 0xfffffu || a->width > 0xffffffu ||
        a->pageRows > 0xffffffu || a->room > 0x3fffffffu)
        return (int)hipErrorInvalidValue;
    const uint32_t chunks = chunks_of(a->pages);
    if (slices > MAX_GROUPS || slices * a->children + chunks > MAX_GROUPS) return (int)hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(fork_plan, dim3(a->children + a->rows + chunks), dim3(THREADS), 0, s, *a);
    hipLaunchKernelGGL(fork_apply, dim3((uint32_t)slices * a->children + chunks), dim3(THREADS), 0, s, *a, (uint32_t)slices);
    return (int)hipGetLastError();
}

int launch_sharedkv_page_compact(void *stream, const PageCompactArgs *a)
{
    if (!a || !a->caches || !a->table || !a->refs || !a->newTable || !a->newRefs || !a->moved || !a->live || !a->workspace)
        return (int)hipErrorInvalidValue;
    if (!a->cacheCount || !a->pages || !a->pageBytes || a->pages > MAX_PAGES) return (int)hipErrorInvalidValue;
    const uint64_t slices = (a->pageBytes + SLICE - 1) / SLICE, entries = (uint64_t)a->rows * a->width;
    if (slices > 0xfffffu || entries > 0xffffffffull) return (int)hipErrorInvalidValue;
    const uint32_t chunks = chunks_of(a->pages), table_groups = (uint32_t)((entries + CHUNK - 1) / CHUNK);
    // At most half of the pages move; eight work-groups per CU fill the chip.
    const uint64_t most = slices * (a->pages / 2);
    const uint32_t copies = (uint32_t)(most < 2048 ? most : 2048);
    const bool streamed = a->pageBytes * a->pages > STREAMED_POOL;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (a->pages <= (uint32_t)CHUNK && a->newTable != a->table && a->newRefs != a->refs) {
        const uint32_t groups = (uint32_t)((entries + THREADS - 1) / THREADS);
        if (copies + (uint64_t)groups + 1 > MAX_GROUPS) return (int)hipErrorInvalidValue;
        hipLaunchKernelGGL((streamed ? &compact_small<true> : &compact_small<false>), dim3(copies + groups + 1), dim3(THREADS), 0, s, *a, groups, copies,
                           (uint32_t)slices);
        return (int)hipGetLastError();
    }
    if (chunks > FEW_CHUNKS) hipLaunchKernelGGL(compact_count, dim3(chunks), dim3(THREADS), 0, s, *a);
    hipLaunchKernelGGL(compact_plan, dim3(chunks), dim3(THREADS), 0, s, *a);
    hipLaunchKernelGGL((streamed ? &compact_apply<true> : &compact_apply<false>), dim3(copies + table_groups + chunks),
                       dim3(THREADS), 0, s, *a, table_groups, copies, (uint32_t)slices);
    return (int)hipGetLastError();
}

uint64_t sharedkv_page_fork_workspace(uint32_t children, uint32_t width, uint32_t pages)
{
    return 4 * fork_words(children, width, pages);
}
uint64_t sharedkv_page_compact_workspace(uint32_t pages) { return 4 * compact_words(pages); }

uint32_t sharedkv_path_commit_args_size(void) { return (uint32_t)sizeof(PathCommitArgs); }
uint32_t sharedkv_page_fork_args_size(void) { return (uint32_t)sizeof(PageForkArgs); }
uint32_t sharedkv_page_compact_args_size(void) { return (uint32_t)sizeof(PageCompactArgs); }

}  // extern "C"
