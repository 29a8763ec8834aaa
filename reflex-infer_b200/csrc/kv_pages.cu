// Page bookkeeping of a paged KV pool on the device: fork (share a request's pages with its children), free,
// compact (move the live pages to the front), and the copies that fork and compact ask for.
//
// The state is one int32 count of owners per page (0 = free); pages are handed out lowest first, so every
// result follows from the inputs alone, whatever the order in which threads run. Fork and compact only do
// the bookkeeping and leave a list of copies: the layers of a model share one table, and kv_copy_pages
// takes the caches of all of them in one launch.
//
// Every kernel here waits for what is ahead of it before it touches memory, and lets the kernel behind it start
// only after that. The last kernel of a fork, a free or a compaction does not let it start early at all: it writes 32-bit
// words (positions to copy, counts of owners) that a caller may give to attention as context lengths, and the plan kernel
// (plan.cu) reads those before its own wait.
//
// Algorithmic bytes: 4 per page (counts) and 8 per table entry read and written; copies 2 * moved bytes.
#include <cooperative_groups.h>

#include "common.cuh"
#include "ptx.cuh"

namespace rfx {
namespace {

// ---- block-wide helpers -----------------------------------------------------------------------------
// Exclusive sum over the CTA's threads; `total` is the sum. `part` holds one int per warp.
template <int THREADS> __device__ __forceinline__ int block_scan(int v, int* part, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int WARPS = THREADS / 32;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // `part` may still be read by the call before
    if (lane == 31) part[warp] = x;
    __syncthreads();
    int before = 0;
    total = 0;
    // every warp sums the warps' totals for itself: one value per lane
    int p = lane < WARPS ? part[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, p, o);
        if (lane >= o) p += y;
    }
    total = __shfl_sync(0xffffffffu, p, WARPS - 1);
    before = warp ? __shfl_sync(0xffffffffu, p, warp - 1) : 0;
    return before + x - v;
}

// Bit j set: page base + j is free (count 0). Pages outside [from, num) count as taken.
template <int PAGES> __device__ __forceinline__ uint32_t free_mask(const int32_t* counts, int64_t base, int64_t from,
                                                                   int64_t num, bool aligned) {
    uint32_t m = 0;
    if (aligned && base >= from && base + PAGES <= num) {
        int4 v[PAGES / 4];
#pragma unroll
        for (int k = 0; k < PAGES / 4; ++k) v[k] = reinterpret_cast<const int4*>(counts + base)[k];
#pragma unroll
        for (int k = 0; k < PAGES / 4; ++k)
            m |= (uint32_t)((v[k].x <= 0) | (v[k].y <= 0) << 1 | (v[k].z <= 0) << 2 | (v[k].w <= 0) << 3) << (4 * k);
    } else {
        for (int j = 0; j < PAGES; ++j)
            if (base + j >= from && base + j < num && counts[base + j] <= 0) m |= 1u << j;
    }
    return m;
}

// ---- fork -------------------------------------------------------------------------------------------
struct ForkParams {
    const int64_t* table;
    const int32_t *lens, *parents;
    int32_t* counts;
    int64_t *child, *src, *dst;
    int32_t* rows;
    int64_t n, batch, max_blocks, bt_s, num_blocks;
    int block_size;
};

struct Child {
    int64_t parent;   // -1: no such row
    int64_t full;     // whole pages, shared
    int rest;         // filled positions of the page behind them
    int64_t page;     // that page, -1 if there is none in the pool
};

__device__ __forceinline__ Child child_of(const ForkParams& P, int64_t i) {
    Child c = {-1, 0, 0, -1};
    const int64_t p = P.parents[i];
    if (p < 0 || p >= P.batch) return c;
    c.parent = p;
    const int64_t most = P.max_blocks * P.block_size;
    int64_t len = P.lens[p];
    len = len < 0 ? 0 : (len > most ? most : len);
    c.full = len / P.block_size;
    c.rest = (int)(len - c.full * P.block_size);
    if (c.rest) {
        const int64_t page = P.table[p * P.bt_s + c.full];
        if (page >= 0 && page < P.num_blocks) c.page = page;
    }
    return c;
}

// One CTA hands out the pages: children in order, 1024 at a time, each group's pages from one walk over the
// counts that stops where the last one was found and goes on there for the next group: first four pages a thread, as
// free pages are often near, then 32.
constexpr int kForkThreads = 1024, kForkPages = 32, kForkFirst = 4;
__device__ __forceinline__ void fork_take(const ForkParams& P) {
    __shared__ int part[32];
    __shared__ int fresh[kForkThreads];
    __shared__ int64_t next_from;
    const bool aligned = ((uintptr_t)P.counts & 15) == 0;
    int64_t from = 0;
    // No page that a child copies from is handed out, even if its count says that it is free: the copies run side by side. (Whole
    // pages that are shared are not looked at here; that they count 1 at least is the caller's part.)
    Child mine_first = {-1, 0, 0, -1};
    for (int64_t i = threadIdx.x; i < P.n; i += kForkThreads) {
        const Child c = child_of(P, i);
        if (c.page >= 0 && P.counts[c.page] <= 0) P.counts[c.page] = 1;
        if (i < kForkThreads) mine_first = c;
    }
    __syncthreads();
    for (int64_t c0 = 0; c0 < P.n; c0 += kForkThreads) {
        const int64_t i = c0 + threadIdx.x;
        Child c = mine_first;
        if (c0 > 0) {
            c = {-1, 0, 0, -1};
            if (i < P.n) c = child_of(P, i);
        }
        const bool need = c.page >= 0;
        int wanted;
        const int rank = block_scan<kForkThreads>(need ? 1 : 0, part, wanted);
        int found = 0;
        if (threadIdx.x == 0) next_from = wanted ? P.num_blocks : from;
        int per = kForkFirst;
        for (int64_t base = from & ~(int64_t)(kForkPages - 1); base < P.num_blocks && found < wanted; base += (int64_t)kForkThreads * per) {
            if (base != (from & ~(int64_t)(kForkPages - 1))) per = kForkPages;
            const int64_t mine = base + (int64_t)threadIdx.x * per;
            uint32_t m = per == kForkPages ? free_mask<kForkPages>(P.counts, mine, from, P.num_blocks, aligned)
                                           : free_mask<kForkFirst>(P.counts, mine, from, P.num_blocks, aligned);
            int total;
            int at = found + block_scan<kForkThreads>(__popc(m), part, total);
            while (m && at < wanted) {
                const int j = __ffs(m) - 1;
                m &= m - 1;
                fresh[at] = (int)(mine + j);
                if (++at == wanted) next_from = mine + j + 1;
            }
            found += total;
        }
        __syncthreads();
        const int64_t page = need && rank < found ? (int64_t)fresh[rank] : -1;
        from = next_from;
        if (page >= 0) P.counts[page] = 1;
        if (i < P.n) {
            P.src[i] = need ? c.page : -1;
            P.dst[i] = page;
            P.rows[i] = need ? c.rest : 0;
        }
        __syncthreads();  // fresh, next_from
    }
}

constexpr int kForkEntries = 8;
// Entries j0, j0 + step, ... (kForkEntries of them) of child i: the loads first, so that they are under way together.
__device__ __forceinline__ void fork_entries(const ForkParams& P, const Child& c, int64_t own, int64_t i, int64_t j0, int step) {
    const bool dropped = c.parent < 0 || (c.page >= 0 && own < 0);  // no parent, or no page was left
    const int64_t* row = P.table + (c.parent < 0 ? 0 : c.parent) * P.bt_s;
    const int64_t shared = dropped ? 0 : c.full, last = dropped || !c.rest ? -1 : c.full;
    int64_t e[kForkEntries];
#pragma unroll
    for (int x = 0; x < kForkEntries; ++x) {
        const int64_t j = j0 + x * step;
        e[x] = -1;
        if (j < shared || (j == last && c.page < 0)) e[x] = row[j];
        else if (j == last) e[x] = own;
    }
#pragma unroll
    for (int x = 0; x < kForkEntries; ++x) {
        const int64_t j = j0 + x * step;
        if (j >= P.max_blocks) break;
        if (j < shared && e[x] >= 0 && e[x] < P.num_blocks) atomicAdd(P.counts + e[x], 1);
        P.child[i * P.max_blocks + j] = e[x];
    }
}

// Small forks in one launch: a cluster whose first CTA hands out the pages and whose warps then take the children in turn.
// (Two launches cost the host 4 us more, which is what a small fork takes.)
constexpr int kForkCluster = 8;
__global__ void __cluster_dims__(kForkCluster, 1, 1) __launch_bounds__(kForkThreads) kv_fork_small_kernel(const ForkParams P) {
    ptx::pdl_wait();
    const int lane = threadIdx.x & 31, warps = kForkCluster * kForkThreads / 32;
    const int64_t first = blockIdx.x * (kForkThreads / 32) + (threadIdx.x >> 5);
    Child c = {-1, 0, 0, -1};
    if (first < P.n) c = child_of(P, first);
    if (blockIdx.x == 0) fork_take(P);
    cooperative_groups::this_cluster().sync();  // also makes the pages visible to the other CTAs
    for (int64_t i = first; i < P.n; i += warps) {
        if (i != first) c = child_of(P, i);
        const int64_t own = *(volatile int64_t*)(P.dst + i);
        for (int64_t j = lane; j < P.max_blocks; j += 32 * kForkEntries) fork_entries(P, c, own, i, j, 32);
    }
}
// Large ones in two.
__global__ void __launch_bounds__(kForkThreads) kv_fork_take_kernel(const ForkParams P) {
    ptx::pdl_wait();
    ptx::pdl_trigger();
    fork_take(P);
}
__global__ void __launch_bounds__(256) kv_fork_table_kernel(const ForkParams P) {
    ptx::pdl_wait();
    const int64_t i = blockIdx.x;
    const Child c = child_of(P, i);
    constexpr int kStep = 256 * kForkEntries;
    for (int64_t j = blockIdx.y * kStep + threadIdx.x; j < P.max_blocks; j += (int64_t)gridDim.y * kStep) fork_entries(P, c, P.dst[i], i, j, 256);
}

// ---- free -------------------------------------------------------------------------------------------
// An entry is taken out of the table before its page is given up, so a row named twice gives up its pages
// once. A count that is zero already stays zero.
__global__ void __launch_bounds__(256) kv_free_kernel(int64_t* table, int64_t bt_s, const int32_t* rows, int64_t batch,
                                                      int64_t max_blocks, int64_t num_blocks, int32_t* counts) {
    ptx::pdl_wait();
    const int64_t r = rows[blockIdx.x];
    if (r < 0 || r >= batch) return;
    for (int64_t j = blockIdx.y * 256 + threadIdx.x; j < max_blocks; j += (int64_t)gridDim.y * 256) {
        unsigned long long* e = (unsigned long long*)(table + r * bt_s + j);
        if ((int64_t)*(volatile unsigned long long*)e == -1) continue;
        const int64_t page = (int64_t)atomicExch(e, ~0ull);
        if (page < 0 || page >= num_blocks) continue;
        if (atomicSub(counts + page, 1) <= 0) atomicAdd(counts + page, 1);
    }
}

// ---- compact ----------------------------------------------------------------------------------------
// With L(i) live pages below i and `live` of them in all: a live page i >= live moves, as number
// live - 1 - L(i) counted from the last; a free page i < live is hole number i - L(i). There are as many of
// one as of the other, and the last live page goes to the first hole.
constexpr int kCompactThreads = 256, kCompactPages = 16, kCompactChunk = kCompactThreads * kCompactPages;

struct CompactParams {
    int32_t* counts;
    int64_t num;
    int32_t* chunk;   // live pages of every kCompactChunk pages
    int64_t *map, *src, *dst;
    int32_t* n_moves;
    int64_t* table;
    int64_t bt_s, batch, max_blocks;
    int chunks;
};

__device__ __forceinline__ void compact_count(const CompactParams& P, int g) {
    __shared__ int part[32];
    const int64_t base = g * (int64_t)kCompactChunk + threadIdx.x * kCompactPages;
    const int in = (int)(base >= P.num ? 0 : (P.num - base < kCompactPages ? P.num - base : kCompactPages));
    const uint32_t m = free_mask<kCompactPages>(P.counts, base, 0, P.num, ((uintptr_t)P.counts & 15) == 0);
    int total;
    block_scan<kCompactThreads>(in - __popc(m), part, total);
    if (threadIdx.x == 0) P.chunk[g] = total;
}

__device__ __forceinline__ void compact_place(const CompactParams& P, int g) {
    __shared__ int part[32];
    const int64_t base = g * (int64_t)kCompactChunk + threadIdx.x * kCompactPages;
    const int in = (int)(base >= P.num ? 0 : (P.num - base < kCompactPages ? P.num - base : kCompactPages));
    const uint32_t m = free_mask<kCompactPages>(P.counts, base, 0, P.num, ((uintptr_t)P.counts & 15) == 0);
    int all = 0, below = 0, unused;
    for (int x = threadIdx.x; x < P.chunks; x += kCompactThreads) {
        const int c = *(volatile int32_t*)(P.chunk + x);
        all += c;
        if (x < g) below += c;
    }
    int live, before;
    block_scan<kCompactThreads>(all, part, live);
    block_scan<kCompactThreads>(below, part, before);
    int64_t L = before + block_scan<kCompactThreads>(in - __popc(m), part, unused);
    for (int j = 0; j < in; ++j) {
        const int64_t i = base + j;
        if (i == live) *P.n_moves = (int)(live - L);
        if (m >> j & 1) {
            P.map[i] = -1;
            if (i < live) P.dst[i - L] = i;
        } else {
            const int64_t rank = live - 1 - L;
            P.map[i] = i < live ? i : -2 - rank;  // the hole's number, until its page is put there
            if (i >= live) P.src[rank] = i;
            ++L;
        }
    }
    if (live == P.num && g == 0 && threadIdx.x == 0) *P.n_moves = 0;
}

__device__ __forceinline__ void compact_apply(const CompactParams& P, int64_t first, int64_t step) {
    const int64_t moves = *(volatile int32_t*)P.n_moves;
    for (int64_t r = first; r < moves; r += step) {
        const int64_t s = *(volatile int64_t*)(P.src + r), d = *(volatile int64_t*)(P.dst + r);
        P.counts[d] = P.counts[s];
        P.counts[s] = 0;
        *(volatile int64_t*)(P.map + s) = d;
    }
    for (int64_t x = first; x < P.batch * P.max_blocks; x += step) {
        const int64_t b = x / P.max_blocks;
        int64_t* e = P.table + b * P.bt_s + (x - b * P.max_blocks);
        const int64_t page = *e;
        if (page < 0 || page >= P.num) continue;
        const int64_t to = *(volatile int64_t*)(P.map + page);  // either form of a moved page's entry will do
        *e = to < -1 ? *(volatile int64_t*)(P.dst - 2 - to) : to;
    }
}

// Small pools in one launch of one cluster; large ones in three.
constexpr int kCompactCluster = 8;
constexpr int64_t kSmallCompact = 1 << 15;  // pages, and table entries
__global__ void __cluster_dims__(kCompactCluster, 1, 1) __launch_bounds__(kCompactThreads) kv_compact_small_kernel(const CompactParams P) {
    ptx::pdl_wait();
    for (int g = blockIdx.x; g < P.chunks; g += kCompactCluster) compact_count(P, g);
    cooperative_groups::this_cluster().sync();
    for (int g = blockIdx.x; g < P.chunks; g += kCompactCluster) compact_place(P, g);
    cooperative_groups::this_cluster().sync();
    compact_apply(P, blockIdx.x * (int64_t)kCompactThreads + threadIdx.x, kCompactCluster * kCompactThreads);
}
__global__ void __launch_bounds__(kCompactThreads) kv_compact_count_kernel(const CompactParams P) {
    ptx::pdl_wait();
    ptx::pdl_trigger();
    compact_count(P, blockIdx.x);
}
__global__ void __launch_bounds__(kCompactThreads) kv_compact_place_kernel(const CompactParams P) {
    ptx::pdl_wait();
    ptx::pdl_trigger();
    compact_place(P, blockIdx.x);
}
__global__ void __launch_bounds__(kCompactThreads) kv_compact_apply_kernel(const CompactParams P) {
    ptx::pdl_wait();
    compact_apply(P, blockIdx.x * (int64_t)kCompactThreads + threadIdx.x, (int64_t)gridDim.x * kCompactThreads);
}

// ---- copies -----------------------------------------------------------------------------------------
constexpr int kCopyLayers = 64;  // cache pairs of one launch: their addresses travel as kernel arguments
struct Scales { float* of[2 * kCopyLayers]; };
struct NoScales {};
template <typename S> struct CopyParams {
    void* cache[2 * kCopyLayers];
    S scales;
    const int64_t *src, *dst;
    const int32_t *rows, *n_moves;
    int64_t n_pairs, num_blocks;
    int64_t sblk, sh, spos;  // in vectors
    int tensors, heads, vpr, block_size, strips;
    bool linear;             // a head's positions follow one another without a gap
};

// A warp copies a strip of 32*PER vectors of one head's positions of one page: every lane has all its loads
// under way before the first store.
template <typename VEC, int PER, typename S>
__global__ void __launch_bounds__(256) kv_copy_pages_kernel(const CopyParams<S> P) {
    ptx::pdl_wait();
    ptx::pdl_trigger();
    const int lane = threadIdx.x & 31;
    int64_t pairs = P.n_pairs;
    if (P.n_moves) {
        const int64_t m = *P.n_moves;
        pairs = m < pairs ? (m < 0 ? 0 : m) : pairs;
    }
    const int64_t per_pair = (int64_t)P.heads * P.strips;
    const int64_t total = pairs * per_pair * P.tensors;
    const int64_t warps = ((int64_t)gridDim.x * blockDim.x) >> 5;
    for (int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; w < total; w += warps) {
        int64_t pair, rest;
        int t, h, strip;
        if (total < (1ll << 31)) {  // 32-bit divisions where they do
            uint32_t x = (uint32_t)w;
            strip = (int)(x % (uint32_t)P.strips); x /= (uint32_t)P.strips;
            h = (int)(x % (uint32_t)P.heads); x /= (uint32_t)P.heads;
            pair = x % (uint32_t)pairs;
            t = (int)(x / (uint32_t)pairs);
        } else {
            rest = w;
            strip = (int)(rest % P.strips); rest /= P.strips;
            h = (int)(rest % P.heads); rest /= P.heads;
            pair = rest % pairs;
            t = (int)(rest / pairs);
        }
        const int64_t src = P.src[pair], dst = P.dst[pair];
        if (src < 0 || src >= P.num_blocks || dst < 0 || dst >= P.num_blocks || src == dst) continue;
        int rows = P.block_size;
        if (P.rows) { const int r = P.rows[pair]; rows = r < rows ? (r < 0 ? 0 : r) : rows; }
        const VEC* from = (const VEC*)P.cache[t] + src * P.sblk + h * P.sh;
        VEC* to = (VEC*)P.cache[t] + dst * P.sblk + h * P.sh;
        const int64_t end = (int64_t)rows * P.vpr;
        const int64_t v0 = (int64_t)strip * (32 * PER) + lane;
        VEC x[PER];
        if (P.linear) {
#pragma unroll
            for (int k = 0; k < PER; ++k) if (v0 + 32 * k < end) x[k] = from[v0 + 32 * k];
#pragma unroll
            for (int k = 0; k < PER; ++k) if (v0 + 32 * k < end) to[v0 + 32 * k] = x[k];
        } else {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int64_t v = v0 + 32 * k;
                if (v < end) { const int64_t at = v / P.vpr; x[k] = from[at * P.spos + (v - at * P.vpr)]; }
            }
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int64_t v = v0 + 32 * k;
                if (v < end) { const int64_t at = v / P.vpr; to[at * P.spos + (v - at * P.vpr)] = x[k]; }
            }
        }
        if constexpr (sizeof(S) == sizeof(Scales)) {
            float* sc = P.scales.of[t];
            if (strip == 0)
                for (int r = lane; r < rows; r += 32)
                    sc[(dst * P.heads + h) * P.block_size + r] = sc[(src * P.heads + h) * P.block_size + r];
        }
    }
}

int done(cudaError_t e, const char* name) {
    if (e != cudaSuccess) { cudaGetLastError(); return fail(RFX_CUDA_ERROR, "%s: %s", name, cudaGetErrorString(e)); }
    return check_launch(name);
}


template <typename S> int copy_impl(const RfxKvCopyArgs* a, size_t vec, size_t e, const char* name) {
    const int64_t per = (int64_t)(vec / e);
    CopyParams<S> P;
    P.src = a->src_pages; P.dst = a->dst_pages; P.rows = a->copy_rows; P.n_moves = a->n_moves;
    P.n_pairs = a->n_pairs; P.num_blocks = a->num_blocks;
    P.sblk = a->cache_stride_blk / per; P.sh = a->cache_stride_h / per; P.spos = a->cache_stride_pos / per;
    P.heads = (int)a->num_kv_heads; P.vpr = (int)((size_t)a->head_dim * e / vec); P.block_size = (int)a->block_size;
    P.linear = P.spos == P.vpr;
    constexpr int PER = 8;
    const int64_t strips = ceil_div<int64_t>((int64_t)P.vpr * P.block_size, 32 * PER);
    RFX_REQUIRE(strips < (1ll << 31), "%s: a page of %lld positions x %lld elements is too large", name,
                (long long)a->block_size, (long long)a->head_dim);
    P.strips = (int)strips;
    cudaStream_t s = as_stream(a->stream);
    for (int64_t l0 = 0; l0 < a->n_layers; l0 += kCopyLayers) {
        const int m = (int)(a->n_layers - l0 < kCopyLayers ? a->n_layers - l0 : kCopyLayers);
        P.tensors = 2 * m;
        for (int l = 0; l < m; ++l) {
            P.cache[2 * l] = a->k_caches[l0 + l];
            P.cache[2 * l + 1] = a->v_caches[l0 + l];
            if constexpr (sizeof(S) == sizeof(Scales)) {
                P.scales.of[2 * l] = a->k_scales[l0 + l];
                P.scales.of[2 * l + 1] = a->v_scales[l0 + l];
            }
        }
        const int64_t items = P.n_pairs * P.tensors * (int64_t)P.heads * P.strips;
        int64_t blocks = ceil_div<int64_t>(items, 8);
        if (blocks > (int64_t)sm_count() * 8) blocks = (int64_t)sm_count() * 8;
        cudaError_t le;
        switch (vec) {
            case 16: le = launch_pdl(kv_copy_pages_kernel<uint4, PER, S>, dim3((unsigned)blocks), dim3(256), 0, s, P); break;
            case 8: le = launch_pdl(kv_copy_pages_kernel<uint2, PER, S>, dim3((unsigned)blocks), dim3(256), 0, s, P); break;
            case 4: le = launch_pdl(kv_copy_pages_kernel<uint32_t, PER, S>, dim3((unsigned)blocks), dim3(256), 0, s, P); break;
            case 2: le = launch_pdl(kv_copy_pages_kernel<uint16_t, PER, S>, dim3((unsigned)blocks), dim3(256), 0, s, P); break;
            default: le = launch_pdl(kv_copy_pages_kernel<uint8_t, PER, S>, dim3((unsigned)blocks), dim3(256), 0, s, P); break;
        }
        if (le != cudaSuccess) return done(le, name);
    }
    return check_launch(name);
}

}  // namespace
}  // namespace rfx

extern "C" int rfx_kv_fork(const RfxKvForkArgs* a) {
    using namespace rfx;
    const char* name = "rfx_kv_fork";
    if (!a) return fail(RFX_INVALID_ARGUMENT, "%s: null args", name);
    RFX_REQUIRE(a->n_children >= 0 && a->n_children < (1ll << 31) && a->batch >= 0 && a->max_blocks >= 0 &&
                    a->num_blocks > 0 && a->num_blocks < (1ll << 31) && a->block_size > 0 && a->block_size < (1ll << 31),
                "%s: bad sizes children=%lld rows=%lld entries=%lld blocks=%lld bs=%lld", name, (long long)a->n_children,
                (long long)a->batch, (long long)a->max_blocks, (long long)a->num_blocks, (long long)a->block_size);
    if (a->n_children == 0) return RFX_SUCCESS;
    RFX_REQUIRE(a->parents && a->ref_counts && a->src_pages && a->dst_pages && a->copy_rows, "%s: null pointer", name);
    RFX_REQUIRE(a->batch == 0 || a->context_lens, "%s: null pointer", name);
    RFX_REQUIRE(a->max_blocks == 0 || a->batch == 0 || a->block_table, "%s: null block_table", name);
    RFX_REQUIRE(a->max_blocks == 0 || a->child_table, "%s: null child_table", name);
    int st = check_device();
    if (st != RFX_SUCCESS) return st;
    ForkParams P = {a->block_table, a->context_lens, a->parents, a->ref_counts, a->child_table, a->src_pages, a->dst_pages,
                    a->copy_rows, a->n_children, a->batch, a->max_blocks, a->bt_stride_b, a->num_blocks, (int)a->block_size};
    cudaStream_t s = as_stream(a->stream);
    // One launch up to 32 K table entries; behind that the eight SMs of a cluster are too few (131 K entries with 65 K pages shared:
    // 21 us, two launches 12).
    if (a->n_children * a->max_blocks <= (1ll << 15))
        return done(launch_pdl(kv_fork_small_kernel, dim3(kForkCluster), dim3(kForkThreads), 0, s, P), name);
    cudaError_t e = launch_pdl(kv_fork_take_kernel, dim3(1), dim3(kForkThreads), 0, s, P);
    if (e != cudaSuccess) return done(e, name);
    if (a->max_blocks > 0) {
        int64_t y = ceil_div<int64_t>(a->max_blocks, 256 * kForkEntries);
        if (y > 64) y = 64;
        e = launch_pdl(kv_fork_table_kernel, dim3((unsigned)a->n_children, (unsigned)y), dim3(256), 0, s, P);
    }
    return done(e, name);
}

extern "C" int rfx_kv_free(const RfxKvFreeArgs* a) {
    using namespace rfx;
    const char* name = "rfx_kv_free";
    if (!a) return fail(RFX_INVALID_ARGUMENT, "%s: null args", name);
    RFX_REQUIRE(a->n_rows >= 0 && a->n_rows < (1ll << 31) && a->batch >= 0 && a->max_blocks >= 0 && a->num_blocks > 0,
                "%s: bad sizes", name);
    if (a->n_rows == 0 || a->max_blocks == 0 || a->batch == 0) return RFX_SUCCESS;
    RFX_REQUIRE(a->block_table && a->rows && a->ref_counts, "%s: null pointer", name);
    int st = check_device();
    if (st != RFX_SUCCESS) return st;
    int64_t y = ceil_div<int64_t>(a->max_blocks, 256);
    if (y > 64) y = 64;
    return done(launch_pdl(kv_free_kernel, dim3((unsigned)a->n_rows, (unsigned)y), dim3(256), 0, as_stream(a->stream),
                           a->block_table, a->bt_stride_b, a->rows, a->batch, a->max_blocks, a->num_blocks, a->ref_counts),
                name);
}

extern "C" size_t rfx_kv_compact_workspace_bytes(int64_t num_blocks) {
    if (num_blocks <= 0 || num_blocks >= (1ll << 31)) return 0;
    return (size_t)rfx::round_up<int64_t>(rfx::ceil_div<int64_t>(num_blocks, rfx::kCompactChunk) * 4, 256);
}

extern "C" int rfx_kv_compact(const RfxKvCompactArgs* a) {
    using namespace rfx;
    const char* name = "rfx_kv_compact";
    if (!a) return fail(RFX_INVALID_ARGUMENT, "%s: null args", name);
    RFX_REQUIRE(a->num_blocks > 0 && a->num_blocks < (1ll << 31) && a->batch >= 0 && a->max_blocks >= 0, "%s: bad sizes", name);
    RFX_REQUIRE(a->ref_counts && a->page_map && a->src_pages && a->dst_pages && a->n_moves, "%s: null pointer", name);
    RFX_REQUIRE(a->batch * a->max_blocks == 0 || a->block_table, "%s: null block_table", name);
    const size_t need = rfx_kv_compact_workspace_bytes(a->num_blocks);
    if (!a->workspace || a->workspace_bytes < need)
        return fail(RFX_WORKSPACE_TOO_SMALL, "%s: needs a workspace of %zu bytes, got %zu", name, need, a->workspace_bytes);
    int st = check_device();
    if (st != RFX_SUCCESS) return st;
    cudaStream_t s = as_stream(a->stream);
    const int64_t g = ceil_div<int64_t>(a->num_blocks, kCompactChunk), entries = a->batch * a->max_blocks;
    const CompactParams P = {a->ref_counts, a->num_blocks, (int32_t*)a->workspace, a->page_map, a->src_pages, a->dst_pages, a->n_moves,
                             a->block_table, a->bt_stride_b, a->batch, a->max_blocks, (int)g};
    if (a->num_blocks <= kSmallCompact && entries <= kSmallCompact)
        return done(launch_pdl(kv_compact_small_kernel, dim3(kCompactCluster), dim3(kCompactThreads), 0, s, P), name);
    cudaError_t e = launch_pdl(kv_compact_count_kernel, dim3((unsigned)g), dim3(kCompactThreads), 0, s, P);
    if (e != cudaSuccess) return done(e, name);
    e = launch_pdl(kv_compact_place_kernel, dim3((unsigned)g), dim3(kCompactThreads), 0, s, P);
    if (e != cudaSuccess) return done(e, name);
    const int64_t most = entries > a->num_blocks / 2 ? entries : a->num_blocks / 2;
    int64_t blocks = ceil_div<int64_t>(most < 1 ? 1 : most, kCompactThreads);
    if (blocks > (int64_t)sm_count() * 8) blocks = (int64_t)sm_count() * 8;
    e = launch_pdl(kv_compact_apply_kernel, dim3((unsigned)blocks), dim3(kCompactThreads), 0, s, P);
    return done(e, name);
}

extern "C" int rfx_kv_copy_pages(const RfxKvCopyArgs* a) {
    using namespace rfx;
    const char* name = "rfx_kv_copy_pages";
    if (!a) return fail(RFX_INVALID_ARGUMENT, "%s: null args", name);
    RFX_REQUIRE(a->kv_int8 || dtype_ok(a->dtype), "%s: unknown dtype %d", name, a->dtype);
    RFX_REQUIRE(a->n_layers >= 0 && a->n_pairs >= 0 && a->num_kv_heads > 0 && a->num_kv_heads < (1 << 20) && a->head_dim > 0 &&
                    a->num_blocks > 0 && a->block_size > 0 && a->block_size < (1ll << 31) && a->head_dim < (1 << 20),
                "%s: bad sizes layers=%lld pairs=%lld H=%lld D=%lld blocks=%lld bs=%lld", name, (long long)a->n_layers,
                (long long)a->n_pairs, (long long)a->num_kv_heads, (long long)a->head_dim, (long long)a->num_blocks,
                (long long)a->block_size);
    if (a->n_pairs == 0 || a->n_layers == 0) return RFX_SUCCESS;
    RFX_REQUIRE(a->k_caches && a->v_caches && a->src_pages && a->dst_pages, "%s: null pointer", name);
    RFX_REQUIRE(!a->kv_int8 || (a->k_scales && a->v_scales), "%s: an int8 pool needs k_scales and v_scales", name);
    for (int64_t l = 0; l < a->n_layers; ++l)
        RFX_REQUIRE(a->k_caches[l] && a->v_caches[l] && (!a->kv_int8 || (a->k_scales[l] && a->v_scales[l])),
                    "%s: null cache pointer of layer %lld", name, (long long)l);
    int st = check_device();
    if (st != RFX_SUCCESS) return st;

    const size_t e = a->kv_int8 ? 1 : dtype_size(a->dtype);
    const size_t row = (size_t)a->head_dim * e;
    size_t vec = 16;
    auto fits = [&](size_t v) {
        if (row % v) return false;
        for (int64_t s : {a->cache_stride_blk, a->cache_stride_h, a->cache_stride_pos})
            if (((size_t)s * e) % v) return false;
        for (int64_t l = 0; l < a->n_layers; ++l)
            if ((uintptr_t)a->k_caches[l] % v || (uintptr_t)a->v_caches[l] % v) return false;
        return true;
    };
    while (vec > e && !fits(vec)) vec /= 2;
    if (a->kv_int8) return copy_impl<Scales>(a, vec, e, name);
    return copy_impl<NoScales>(a, vec, e, name);
}
