// Sampling one token per row from logits with temperature, top-k, top-p and min-p and a given uniform number.
//
//   z_i = (l_i - max) / T;  top-k keeps the k largest (ties: lowest index);  w_i = exp(z_i) over those;
//   top-p keeps, in falling order (ties: lowest index), while the mass before is < p * total;
//   min-p keeps w_i >= min_p (the largest weight is 1);
//   the token is the lowest index whose running sum of kept weights, in index order, exceeds u * their sum.
//
// The answer hangs on which side of a border a sum lies, so sums must not depend on the order in which
// threads or CTAs run: a weight is exp() in 64 bits, rounded to a whole multiple of 2^-S with
// S = min(50, 62 - log2 V), and added up as a 64-bit integer. Such sums are exact in any order; what a weight
// loses (2^-S-1 of the largest, 2^-46 at 131072 tokens) is far below the distance of two borders.
//
// A cluster of up to 8 CTAs takes a row, each a slice of it, which stays in shared memory: the logits are read
// from HBM once (algorithmic bytes: V*e a row). Two ways to the answer:
//   list     (top-k up to 512 a CTA) every thread's largest logit is known from the load; the ceil(k/C)-th largest of
//            those, lowest over the CTAs, bounds the k-th largest logit from below. What lies above it (about 1.4 k
//            logits) is sorted by one CTA, which then has the whole kept set in hand.
//   general  a histogram over max - l (counts for top-k, masses for top-p) names the bin with the border,
//            the logits of that bin are sorted, and a pass in index order adds up what is kept. Without
//            top-k and top-p only that pass is left.
// A list that overflows (thousands of equal logits) is replaced by a search over the bits of the border's
// key and index: slower, and right for every input.
#include <cooperative_groups.h>

#include "common.cuh"
#include "ptx.cuh"

namespace rfx {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kCap = 2048;   // logits that one CTA sorts
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr size_t kStageTwo = 78 * 1024;   // slice that lets two CTAs share an SM
constexpr size_t kStageMax = 188 * 1024;  // largest slice kept in shared memory

struct SampleParams {
    const void* logits;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int64_t* tokens;
    int64_t row_stride;
    float temperature0, top_p0, min_p0;
    int32_t top_k0;
    int vocab, slice;  // slice: logits per CTA, a multiple of 8
    int shift;         // S: weights are multiples of 2^-S
};

struct Shared {
    u64 list[kCap];
    union {
        struct { uint32_t lo[kBins], hi[kBins]; } hist;
        u64 weight[kCap];  // of the sorted list
    };
    u64 part[kWarps];
    u64 slot[2];
    u64 found[2];  // what rank 0 tells the others
    int n;         // entries that want to be in `list`
};

__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <typename T> struct Chunk {  // 16 bytes of logits
    static constexpr int N = 16 / sizeof(T);
    union { uint4 raw; T v[N]; };
    __device__ Chunk() {}
    __device__ __forceinline__ float at(int e) const {
        const float f = Num<T>::to_f(v[e]) + 0.f;  // -0 and +0 are one value
        return f == f ? f : -INFINITY;             // NaN counts as masked
    }
};

// One CTA's view of its row.
template <typename T, bool STAGED> struct Row {
    static constexpr int N = Chunk<T>::N;
    const T* row;    // the row's logits
    T* stage;        // the slice in shared memory, at the 16-byte phase it has in global memory
    int lo, hi;      // the CTA's logits [lo, hi)
    int base, nvec;  // 16-byte chunks from index `base` (lo rounded down to the boundary)
    Shared& s;
    int rank, ranks, parity;
    float top;            // the row's largest logit
    double scale;         // log-weight per unit: 1 / T
    double unit;          // 2^S
    float bins;           // histogram bins per unit
    int vocab;
    uint32_t cut_key;     // kept: key > cut_key, or key == cut_key and index <= cut_index
    int cut_index;

    __device__ __forceinline__ Chunk<T> load_global(int j) const {
        Chunk<T> c;
        const int i0 = base + j * N;
        if (i0 >= lo && i0 + N <= hi) {
            c.raw = __ldg(reinterpret_cast<const uint4*>(row + i0));
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) c.v[e] = i0 + e >= lo && i0 + e < hi ? row[i0 + e] : Num<T>::from_f(-INFINITY);
        }
        return c;
    }
    __device__ __forceinline__ Chunk<T> load(int j) const {
        if (!STAGED) return load_global(j);
        Chunk<T> c;
        c.raw = reinterpret_cast<const uint4*>(stage)[j];
        return c;
    }
    // f(value, index) for the slice; what lies outside it reads as -inf
    template <typename F> __device__ __forceinline__ void each(F f) const {
        for (int j = threadIdx.x; j < nvec; j += kThreads) {
            const Chunk<T> c = load(j);
#pragma unroll
            for (int e = 0; e < N; ++e) f(c.at(e), base + j * N + e);
        }
    }
    __device__ __forceinline__ double weight(float v) const {
        return v == top ? 1.0 : exp(((double)v - (double)top) * scale);
    }
    __device__ __forceinline__ u64 fixed(double w) const { return (u64)__double2ll_rn(w * unit); }
    __device__ __forceinline__ bool kept(float v, int i) const {
        const uint32_t k = key_of(v);
        return v > -INFINITY && (k > cut_key || (k == cut_key && i <= cut_index));
    }
    // Histogram bin, kBins and more: weight zero. Never rises with v.
    __device__ __forceinline__ int bin_of(float v) const {
        const float x = v == top ? 0.f : fminf(top - v, 3.4e38f) * bins;
        return x < (float)kBins ? (int)x : kBins;
    }

    __device__ __forceinline__ u64 block_sum(u64 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = v;
        __syncthreads();
        u64 t = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) t += s.part[w];
        return t;
    }
    // Exclusive prefix over the CTA's threads.
    __device__ __forceinline__ u64 block_scan(u64 v, u64& total) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        u64 x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 31) s.part[warp] = x;
        __syncthreads();
        u64 before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s.part[w];
            total += s.part[w];
        }
        return before + x - v;
    }
    // Every CTA's word, seen by all: word(r) after the call. Two slots in turn: a CTA writes a slot again only
    // after the next exchange, which the readers of this one have reached by then.
    __device__ __forceinline__ u64* exchange(u64 mine) {
        parity ^= 1;
        if (threadIdx.x == 0) s.slot[parity] = mine;
        cg::this_cluster().sync();
        return &s.slot[parity];
    }
    __device__ __forceinline__ u64 word(u64* slot, int r) const { return *cg::this_cluster().map_shared_rank(slot, r); }
    __device__ __forceinline__ u64 cluster_sum(u64 v) {
        u64* slot = exchange(block_sum(v));
        u64 t = 0;
        for (int r = 0; r < ranks; ++r) t += word(slot, r);
        return t;
    }
    // Two words from rank 0 to everyone.
    __device__ __forceinline__ void tell(u64& a, u64& b) {
        if (rank == 0 && threadIdx.x == 0) { s.found[0] = a; s.found[1] = b; }
        cg::this_cluster().sync();
        const u64* f = cg::this_cluster().map_shared_rank(s.found, 0);
        a = f[0];
        b = f[1];
        cg::this_cluster().sync();
    }

    // Puts the logits that `want` takes into rank 0's list; returns their number (the list holds them all
    // only up to kCap).
    template <typename F> __device__ __forceinline__ int gather(F want) {
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        each([&](float v, int i) {
            if (!want(v, i)) return;
            const int at = atomicAdd(&s.n, 1);
            if (at < kCap) s.list[at] = (u64)key_of(v) << 32 | (0xffffffffu - (uint32_t)i);
        });
        __syncthreads();
        u64* slot = exchange((u64)(unsigned)s.n);
        int total = 0;
        for (int r = 0; r < ranks; ++r) total += (int)word(slot, r);
        if (rank == 0 && total <= kCap) {
            int at = s.n;
            for (int r = 1; r < ranks; ++r) {
                const int n = (int)word(slot, r);
                const u64* from = cg::this_cluster().map_shared_rank(s.list, r);
                for (int x = threadIdx.x; x < n; x += kThreads) s.list[at + x] = from[x];
                at += n;
            }
            __syncthreads();
        }
        return total;
    }
    // Bitonic sort of list[0, n), falling. A stage whose pairs stay inside a warp's 64 entries needs no block barrier.
    __device__ void sort(int n) {
        int n2 = 64;
        while (n2 < n) n2 *= 2;
        __syncthreads();
        for (int i = n + threadIdx.x; i < n2; i += kThreads) s.list[i] = 0;
        __syncthreads();
        for (int size = 2; size <= n2; size *= 2) {
            for (int stride = size / 2; stride > 0; stride /= 2) {
                for (int t = threadIdx.x; t < n2 / 2; t += kThreads) {
                    const int i = 2 * t - (t & (stride - 1));
                    const u64 a = s.list[i], b = s.list[i + stride];
                    if ((a < b) == ((i & size) == 0)) { s.list[i] = b; s.list[i + stride] = a; }
                }
                if (stride > 32 || (stride == 1 && size >= 64)) __syncthreads(); else __syncwarp();
            }
        }
        __syncthreads();
    }

    // The border of a sum over the kept logits in falling order: count (top-k) or mass (top-p) up to and
    // including the border first reaches the target. Moves the cut there.
    template <bool MASS> __device__ void cut(int k, float p) {
        for (int b = threadIdx.x; b < kBins; b += kThreads) s.hist.lo[b] = s.hist.hi[b] = 0;
        __syncthreads();
        each([&](float v, int i) {
            if (!kept(v, i)) return;
            const int b = bin_of(v);
            if (b >= kBins) return;
            if (MASS) {  // 64 bits as two words: the one that overflows the low word carries
                const u64 w = fixed(weight(v));
                const uint32_t low = (uint32_t)w, old = atomicAdd(&s.hist.lo[b], low);
                const uint32_t high = (uint32_t)(w >> 32) + (old + low < old ? 1u : 0u);
                if (high) atomicAdd(&s.hist.hi[b], high);
            } else {
                atomicAdd(&s.hist.lo[b], 1u);
            }
        });
        cg::this_cluster().sync();
        u64 at = ~0ull, above = 0, target = (u64)k;
        if (rank == 0) {
            constexpr int PER = kBins / kThreads;
            u64 m[PER], sum = 0, total;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = threadIdx.x * PER + j;
                m[j] = 0;
                for (int r = 0; r < ranks; ++r) {
                    m[j] += (u64)*cg::this_cluster().map_shared_rank(&s.hist.hi[b], r) << 32;
                    m[j] += *cg::this_cluster().map_shared_rank(&s.hist.lo[b], r);
                }
                sum += m[j];
            }
            u64 before = block_scan(sum, total);
            if (MASS) target = target_of(p, total);
            if (threadIdx.x == 0) { s.found[0] = ~0ull; s.found[1] = 0; }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (before < target && before + m[j] >= target && total > target - (MASS ? 1 : 0)) {
                    s.found[0] = (u64)(threadIdx.x * PER + j);
                    s.found[1] = before;
                    s.slot[parity ^ 1] = target;  // free until the next exchange
                }
                before += m[j];
            }
            __syncthreads();
        }
        cg::this_cluster().sync();
        at = *cg::this_cluster().map_shared_rank(&s.found[0], 0);
        above = *cg::this_cluster().map_shared_rank(&s.found[1], 0);
        target = *cg::this_cluster().map_shared_rank(&s.slot[parity ^ 1], 0);
        cg::this_cluster().sync();
        if (at == ~0ull) return;  // the border lies behind the last logit that weighs anything
        const int bin = (int)at;
        const int n = gather([&](float v, int i) { return kept(v, i) && bin_of(v) == bin; });
        if (n <= kCap) {
            u64 key = 0, index = 0;
            if (rank == 0) {
                sort(n);
                constexpr int PER = kCap / kThreads;
                u64 m[PER], sum = 0, total;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const int i = threadIdx.x * PER + j;
                    m[j] = i < n ? (MASS ? fixed(weight(value_of((uint32_t)(s.list[i] >> 32)))) : 1) : 0;
                    sum += m[j];
                }
                u64 before = above + block_scan(sum, total);
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    if (before < target && before + m[j] >= target) s.found[0] = s.list[threadIdx.x * PER + j];
                    before += m[j];
                }
                __syncthreads();
                key = s.found[0];
                __syncthreads();
            }
            tell(key, index);
            cut_key = (uint32_t)(key >> 32);
            cut_index = (int)(0xffffffffu - (uint32_t)key);
            return;
        }
        // thousands of logits in one bin: the border's key, bit by bit, then its index
        auto sum_from = [&](uint32_t from) {  // over the bin's logits with keys >= from
            u64 t = 0;
            each([&](float v, int i) {
                if (kept(v, i) && bin_of(v) == bin && key_of(v) >= from) t += MASS ? fixed(weight(v)) : 1;
            });
            return above + cluster_sum(t);
        };
        uint32_t key = 0;
        for (int bit = 31; bit >= 0; --bit)
            if (sum_from(key | 1u << bit) >= target) key |= 1u << bit;
        const u64 over = key == 0xffffffffu ? above : sum_from(key + 1);
        const u64 each_w = MASS ? fixed(weight(value_of(key))) : 1;
        const u64 ties = (target - over + each_w - 1) / each_w;  // equal logits that stay
        const uint32_t old_key = cut_key;
        const int old_index = cut_index;
        int index = -1;  // largest index with fewer than `ties` equal ones up to it, then the next
        for (int bit = 24; bit >= 0; --bit) {
            const int to = index + (1 << bit);
            if (to >= vocab) continue;
            u64 t = 0;
            each([&](float v, int i) {
                if (v > -INFINITY && key_of(v) == key && (key > old_key || i <= old_index) && i <= to) ++t;
            });
            if (cluster_sum(t) < ties) index = to;
        }
        cut_key = key;
        cut_index = index + 1;
    }
    // Sums below p of the total; the first logit always stays.
    __device__ __forceinline__ u64 target_of(float p, u64 total) const {
        const double t = ceil((double)p * (double)total);
        return t < 1.0 ? 1 : (u64)t;
    }
    __device__ __forceinline__ u64 drawn(float u, u64 total) const {
        const double t = (double)u * (double)total;
        const u64 x = t > 0.0 ? (u64)t : 0;  // a NaN draws the first
        return x < total ? x : total - 1;
    }

    // The draw over everything kept: sums per warp over neighbouring logits, then one warp looks closer.
    __device__ void draw(float u, float min_p, int64_t* token) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int per = (nvec + kWarps - 1) / kWarps, from = warp * per, to = min(nvec, from + per);
        const double least = (min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0);
        auto of = [&](float v, int i) -> u64 {
            if (!kept(v, i)) return 0;
            const double w = weight(v);
            return w >= least ? fixed(w) : 0;
        };
        u64 sum = 0;
        for (int j = from + lane; j < to; j += 32) {
            const Chunk<T> c = load(j);
#pragma unroll
            for (int e = 0; e < N; ++e) sum += of(c.at(e), base + j * N + e);
        }
        u64 all = sum;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        __syncthreads();
        if (lane == 0) s.part[warp] = all;
        __syncthreads();
        u64 mine = 0, before = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s.part[w];
            mine += s.part[w];
        }
        u64* slot = exchange(mine);
        u64 total = 0;
        for (int r = 0; r < ranks; ++r) {
            const u64 x = word(slot, r);
            if (r < rank) before += x;
            total += x;
        }
        const u64 target = drawn(u, total);
        if (target < before || target >= before + all) return;  // whole warps
        for (int j0 = from; j0 < to; j0 += 32) {
            u64 m[N], own = 0;
            const int j = j0 + lane;
#pragma unroll
            for (int e = 0; e < N; ++e) m[e] = 0;
            if (j < to) {
                const Chunk<T> c = load(j);
#pragma unroll
                for (int e = 0; e < N; ++e) { m[e] = of(c.at(e), base + j * N + e); own += m[e]; }
            }
            u64 x = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const u64 group = __shfl_sync(0xffffffffu, x, 31);
            if (target < before + group) {
                u64 at = before + x - own;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (target >= at && target < at + m[e]) *token = base + j * N + e;
                    at += m[e];
                }
                return;
            }
            before += group;
        }
    }

    // rank 0, with the largest logits in list[0, n): everything that is left to do
    __device__ void finish_list(int n, int k, float p, float min_p, float u, int64_t* token) {
        sort(n);
        if (k < n) n = k;
        constexpr int PER = kCap / kThreads;
        u64 m[PER], sum = 0, total, unused;
        double w[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x * PER + j;
            w[j] = i < n ? weight(value_of((uint32_t)(s.list[i] >> 32))) : -1.0;
            m[j] = i < n ? fixed(w[j]) : 0;
            sum += m[j];
        }
        u64 before = block_scan(sum, total);
        const u64 target = p < 1.f ? target_of(p, total) : ~0ull;
        const double least = (min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0);
        int stay = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool in = w[j] >= 0.0 && before < target && w[j] >= least;
            before += m[j];
            if (!in) m[j] = 0;
            stay += in;
        }
        const int kept_n = (int)block_sum((u64)stay);  // a prefix of the list: weights only fall
        // in index order: entries (index, place), with their weights beside them
        u64 e[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x * PER + j;
            e[j] = i < kept_n ? (s.list[i] << 32 | (u64)i) : 0;  // low word: ~index, so falling is rising in index
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x * PER + j;
            if (i < kept_n) { s.list[i] = e[j]; s.weight[i] = m[j]; }
        }
        sort(kept_n);
        sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x * PER + j;
            e[j] = i < kept_n ? s.list[i] : 0;
            m[j] = i < kept_n ? s.weight[(uint32_t)e[j]] : 0;
            sum += m[j];
        }
        u64 at = block_scan(sum, unused);
        const u64 x = drawn(u, unused);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (x >= at && x < at + m[j]) *token = (int64_t)(0xffffffffu - (uint32_t)(e[j] >> 32));
            at += m[j];
        }
    }
};

template <typename T, bool STAGED>
__global__ void __launch_bounds__(kThreads, STAGED ? 2 : 1) sample_kernel(const SampleParams P) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    extern __shared__ __align__(16) unsigned char stage[];
    __shared__ Shared shared;
    auto cluster = cg::this_cluster();
    using R = Row<T, STAGED>;
    constexpr int N = R::N;
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int64_t b = blockIdx.x / ranks;
    const T* row = (const T*)P.logits + b * P.row_stride;
    const int lo = min(P.vocab, rank * P.slice), hi = min(P.vocab, lo + P.slice);
    const int phase = (int)(((uintptr_t)(row + lo) & 15) / sizeof(T));
    R r{row, (T*)stage, lo, hi, lo - phase, lo < hi ? (hi - lo + phase + N - 1) / N : 0, shared, rank, ranks, 0};
    r.vocab = P.vocab;

    const float temperature = P.temperature ? P.temperature[b] : P.temperature0;
    const float p = P.top_p ? P.top_p[b] : P.top_p0, min_p = P.min_p ? P.min_p[b] : P.min_p0;
    int k = P.top_k ? P.top_k[b] : P.top_k0;
    if (k <= 0 || k > P.vocab) k = P.vocab;
    const float u = P.u[b];
    int64_t* token = P.tokens + b;

    // the slice into shared memory; the thread's largest logit on the way
    uint32_t most = 0;
    for (int j0 = threadIdx.x; j0 < r.nvec; j0 += 4 * kThreads) {
        Chunk<T> c[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (j0 + x * kThreads < r.nvec) c[x] = r.load_global(j0 + x * kThreads);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int j = j0 + x * kThreads;
            if (j >= r.nvec) continue;
            if (STAGED) reinterpret_cast<uint4*>(stage)[j] = c[x].raw;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = r.base + j * N + e;
                if (i >= lo && i < hi) most = max(most, key_of(c[x].at(e)));
            }
        }
    }
    const bool greedy = !(temperature > 0.f);
    const int local = (k + ranks - 1) / ranks;
    const bool by_list = !greedy && k < P.vocab && local <= kThreads;
    uint32_t bound = 0;  // at least `local` threads hold a logit with a key from here on
    if (by_list) {
        for (int bit = 31; bit >= 10; --bit)
            if (__syncthreads_count(most >= (bound | 1u << bit)) >= local) bound |= 1u << bit;
    }
    __syncthreads();
    {
        uint32_t top = most;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((threadIdx.x & 31) == 0) shared.part[threadIdx.x >> 5] = top;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) top = max(top, (uint32_t)shared.part[w]);
        u64* slot = r.exchange((u64)top << 32 | bound);
        for (int x = 0; x < ranks; ++x) {
            const u64 o = r.word(slot, x);
            top = max(top, (uint32_t)(o >> 32));
            bound = min(bound, (uint32_t)o);
        }
        r.top = value_of(top);
    }
    r.scale = fmax(1.0 / (double)temperature, 1e-300);  // at T = inf every finite logit weighs 1
    r.unit = (double)(1ull << P.shift);
    r.bins = (float)((double)kBins / (((double)P.shift + 2.0) * 0.6931471805599453 * (double)temperature));
    r.cut_key = 0;
    r.cut_index = 0;

    if (r.top == -INFINITY) {  // nothing to draw from
        if (rank == 0 && threadIdx.x == 0) *token = -1;
    } else if (greedy) {
        int first = 0x7fffffff;
        r.each([&](float v, int i) { if (v == r.top) first = min(first, i); });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) shared.part[threadIdx.x >> 5] = (u64)first;
        __syncthreads();
        u64 least = shared.part[0];
        for (int w = 1; w < kWarps; ++w) least = least < shared.part[w] ? least : shared.part[w];
        u64* slot = r.exchange(least);
        if (rank == 0 && threadIdx.x == 0) {
            for (int x = 1; x < ranks; ++x) { const u64 o = r.word(slot, x); least = least < o ? least : o; }
            *token = (int64_t)least;
        }
    } else {
        bool done = false;
        if (by_list) {
            const uint32_t from = bound;
            const int n = r.gather([&](float v, int) { return v > -INFINITY && key_of(v) >= from; });
            if (n <= kCap) {
                done = true;
                if (rank == 0) r.finish_list(n, k, p, min_p, u, token);
            }
        }
        if (!done) {
            if (k < P.vocab) r.template cut<false>(k, 0.f);
            if (p < 1.f) r.template cut<true>(0, p);
            r.draw(u, min_p, token);
        }
    }
    cluster.sync();  // nobody leaves while its shared memory may still be read
}

}  // namespace
}  // namespace rfx

extern "C" int rfx_sample_tokens(const RfxSampleArgs* a) {
    using namespace rfx;
    const char* name = "rfx_sample_tokens";
    if (!a) return fail(RFX_INVALID_ARGUMENT, "%s: null args", name);
    RFX_REQUIRE(dtype_ok(a->dtype), "%s: unknown dtype %d", name, a->dtype);
    RFX_REQUIRE(a->batch >= 0 && a->batch < (1ll << 28) && a->vocab >= 0 && a->vocab <= (1ll << 24),
                "%s: bad sizes rows=%lld vocab=%lld (at most 2^24)", name, (long long)a->batch, (long long)a->vocab);
    if (a->batch == 0) return RFX_SUCCESS;
    RFX_REQUIRE(a->vocab > 0, "%s: vocab is 0", name);
    RFX_REQUIRE(a->logits && a->uniform && a->tokens, "%s: null pointer", name);
    const size_t e = dtype_size(a->dtype);
    RFX_REQUIRE(((uintptr_t)a->logits % e) == 0, "%s: logits are not aligned to their type", name);
    int st = check_device();
    if (st != RFX_SUCCESS) return st;

    // CTAs of a row: as many as its slice needs to leave room for a second CTA on the SM, and more while SMs would
    // stand idle and a CTA keeps 8 logits or more a thread.
    int C = 1;
    auto slice_of = [&](int c) { return round_up<int64_t>(ceil_div<int64_t>(a->vocab, c), 8); };
    while (C < kMaxCluster && ((slice_of(C) + 8) * e > kStageTwo || (a->batch * C < sm_count() && slice_of(C) > 8 * kThreads)))
        C *= 2;
    const int64_t slice = slice_of(C);
    const size_t bytes = round_up<size_t>((size_t)(slice + 8) * e, 16);
    const bool staged = bytes <= kStageMax;
    SampleParams P = {};
    P.logits = a->logits; P.u = a->uniform; P.temperature = a->temperature; P.top_p = a->top_p; P.min_p = a->min_p;
    P.top_k = a->top_k; P.tokens = a->tokens; P.row_stride = a->row_stride;
    P.temperature0 = a->temperature_all; P.top_p0 = a->top_p_all; P.min_p0 = a->min_p_all; P.top_k0 = a->top_k_all;
    P.vocab = (int)a->vocab; P.slice = (int)slice;
    int log2v = 0;
    while ((1ll << log2v) < a->vocab) ++log2v;
    P.shift = 62 - log2v < 50 ? 62 - log2v : 50;

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a->batch * C));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = staged ? bytes : 0;
    cfg.stream = as_stream(a->stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t le = cudaSuccess;
    auto launch = [&](auto kern, PerDeviceOnce& once) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (staged && !once.done(dev)) {
            le = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kStageMax);
            if (le != cudaSuccess) return;
            once.mark(dev);
        }
        le = cudaLaunchKernelEx(&cfg, kern, P);
    };
    RFX_DISPATCH_DTYPE(a->dtype, T, {
        static PerDeviceOnce once;
        if (staged) launch(sample_kernel<T, true>, once);
        else launch(sample_kernel<T, false>, once);
    });
    if (le != cudaSuccess) { cudaGetLastError(); return fail(RFX_CUDA_ERROR, "%s: %s", name, cudaGetErrorString(le)); }
    return check_launch(name);
}
