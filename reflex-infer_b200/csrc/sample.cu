// Sampling one token per row from logits with temperature, top-k, top-p and min-p and a given uniform number.
//
//   z_i = (l_i - max) / T;  top-k keeps the k largest (ties: lowest index);  w_i = exp(z_i) over those;
//   top-p keeps, in falling order (ties: lowest index), while the mass before is < p * total;
//   min-p keeps w_i >= min_p (the largest weight is 1);
//   the token is the lowest index whose running sum of kept weights, in index order, exceeds u * their sum.
//
// The answer hangs on which side of a border a sum lies, so sums must not depend on the order in which
// threads or CTAs run: a weight is computed in 64 bits to 2^-39 of itself, rounded to a whole multiple of 2^-S of the
// largest, and added up as a 64-bit integer. Such sums are exact in any order. With M logits that can weigh anything (M = top-k, or
// V) all of them may weigh the same, so S = min(50, 63 - log2 M), log2 rounded up, keeps any sum below 2^63. Equal logits all
// round the same way, so a sum may be off by M 2^-(S+1) of the largest weight: 2^-38 up to M = 2^13, 2^-30 at 2^17, 2^-28
// at 2^18. Beyond that such a bound would reach the 2^-24 between two uniform numbers (2^24 logits, all but one 27 below that
// one: a mass of 3e-5 would be lost). There a pass adds up the row at that S first, and S is raised as far as this sum allows
// (see sharpen()): then a sum is off by 2^-27 of the total at most.
//
// A cluster of up to 8 CTAs takes a row, each a slice of it (one CTA a row in large batches). Two ways to the
// answer, by the row's settings:
//   list     (top-k up to 512) The logits stream through registers once. Every thread keeps the largest of two groups
//            of its own; the k-th largest of the CTA's 1024 group maxima bounds the k-th largest logit from below, and
//            what reaches the bound, renewed whenever four times as many logits have been seen (twice as many
//            where k is above 227), goes to a list in shared memory. About 1.3 k logits are left in the end; one CTA
//            ranks them, and has the kept set in hand.
//   general  The slice stays in shared memory (or is read again from L2). A histogram over max - l (counts for top-k,
//            masses for top-p) names the bin with the border, the logits of that bin are ranked, and a pass in index
//            order adds up what is kept. Without top-k and top-p only that pass is left.
// A list that overflows leaves the row to the general way: thousands of equal logits, or several CTAs a row of one batch of loads
// each, of which one has nothing but masked logits and so no bound to offer (8 x 128000 bf16, top-k 50: 9 us, with the last seven
// eighths masked 42). A bin of more than kCap logits is searched bit by bit over the border's key and index: right for every input,
// and some 58 passes over the row (64 x 131072 bf16, top-p 0.9: 52 us, with 20 added to all logits 596).
//
// Algorithmic bytes: V*e a row, read once. List rows are bound by HBM in large batches and by the dozen barriers and
// three cluster barriers of a row in small ones; general rows by the 64-bit exponentials, one a logit.
#include <cooperative_groups.h>

#include <math.h>
#include <string.h>

#include <type_traits>
#include <utility>

#include "common.cuh"
#include "ptx.cuh"

namespace rfx {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kCap = 2048;     // logits that one CTA ranks
constexpr int kPairs = 128;     // a list up to here is ranked by comparing all pairs, a longer one sorted (300: 10 and 4 us) or narrowed
                                // down (32 x 50257 bf16, top-p, some 130 to 260 logits in the border's bin: 25.5 us; with 256 here 26.5, 0: 26.9)
constexpr int kBins = 2048;   // more than 32 * (S + 2), the steps to a weight of zero
constexpr int kMaxCluster = 8;
constexpr int kGroups = 2 * kThreads;     // groups whose maxima bound the k-th largest logit
constexpr int kListK = kGroups / 2;       // with k near kGroups the bound sinks to the smallest of the maxima
constexpr int kBatch = 4;                 // 16-byte chunks a thread has under way
constexpr size_t kStageTwo = 72 * 1024;   // slice that lets two CTAs share an SM
constexpr size_t kStageMax = 180 * 1024;  // largest slice kept in shared memory
constexpr int kParts = 8;                 // of a warp's range in the draw
constexpr int kShift = 50;                // the largest S: a weight and 2^52 have to fit a double
constexpr int kFewWeights = 1 << 18;      // logits that can weigh anything, up to which S follows from their number alone
constexpr float kLowest = -3.402823466e38f;

enum { kAllRows = 0, kListRows = 1, kOtherRows = 2 };
struct SampleParams {
    const void* logits;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t* top_k;
    int64_t* tokens;
    int64_t row_stride;
    float temperature0, top_p0, min_p0;
    int32_t top_k0;
    int vocab, slice;  // slice: logits per CTA, a multiple of 8
    double power[32];  // 2^(kShift + i/32), with i * 2^15 taken off the upper word
    int staged;        // general rows keep their slice in shared memory
    int rows;          // which rows this launch takes
};

struct __align__(16) Entry { u64 key, mass; };  // key: the logit's ordered bits, then ~index

struct __align__(16) Shared {
    u64 list[kCap];
    union {
        struct { uint32_t lo[kBins], hi[kBins]; } hist;
        u64 weight[kCap];       // of the sorted list
        Entry pair[kPairs];  // of the list where all pairs are compared
        uint32_t group[kGroups];
    };
    u64 part[kWarps];
    u64 slot[2][kMaxCluster];  // words of the other CTAs, written by them
    u64 shares[2][kMaxCluster][kMaxCluster];  // [top-k, top-p][CTA][share of the bins]: what that CTA's logits add to it
    u64 found[3];              // a bin and the sum before it; what one CTA tells all, a cut
    double power[32];          // as in SampleParams, for the row's S
    uint32_t picked[3];        // of select(): the bound, the largest key, n before it
    int n;                     // entries that want to be in `list`
};

__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);  // -0 and +0 are one value
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// The smallest finite value that a key, or any bits below those of -inf, lets through: never -inf or NaN.
__device__ __forceinline__ float bound_of(uint32_t k) { return k <= 0x00800000u ? kLowest : value_of(k); }

template <typename T> struct Chunk {  // 16 bytes of logits
    static constexpr int N = 16 / sizeof(T);
    union { uint4 raw; T v[N]; };
    __device__ Chunk() {}
    __device__ __forceinline__ float at(int e) const {
        const float f = Num<T>::to_f(v[e]) + 0.f;
        return f == f ? f : -INFINITY;  // NaN counts as masked
    }
    __device__ __forceinline__ float raw_at(int e) const { return Num<T>::to_f(v[e]); }
    // The largest that is no NaN; NaN if all are.
    __device__ __forceinline__ float most() const {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        } else {
            using W = typename Pair16<T>::P;
            const W* w = reinterpret_cast<const W*>(v);
            const float2 f = Pair16<T>::widen(__hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3])));
            return fmaxf(f.x, f.y);
        }
    }
};

// Bitonic sort of list[0, n), falling. A stage whose pairs stay inside a warp's 64 entries needs no block barrier.
__device__ __noinline__ void sort_list(u64* list, int n) {
    int n2 = 64;
    while (n2 < n) n2 *= 2;
    __syncthreads();
    for (int i = n + threadIdx.x; i < n2; i += kThreads) list[i] = 0;
    __syncthreads();
    for (int size = 2; size <= n2; size *= 2) {
        for (int stride = size / 2; stride > 0; stride /= 2) {
            for (int t = threadIdx.x; t < n2 / 2; t += kThreads) {
                const int i = 2 * t - (t & (stride - 1));
                const u64 a = list[i], b = list[i + stride];
                if ((a < b) == ((i & size) == 0)) { list[i] = b; list[i + stride] = a; }
            }
            if (stride > 32 || (stride == 1 && size >= 64)) __syncthreads(); else __syncwarp();
        }
    }
    __syncthreads();
}

// Sorts list[0, n), falling, by bins: bin(entry) in [0, kBins) never falls while entries fall. An entry's place is its
// bin's first place and the number of larger entries in the bin, so the cost is a dozen barriers and a few steps per
// entry (300 entries: 1 us; the bitonic network's 45 stages 3 us). A bin of more than 64 entries leaves it to the network.
template <typename F> __device__ __forceinline__ void sort_by_bins(Shared& s, int n, F bin) {
    constexpr int PER = kCap / kThreads;
    __syncthreads();
    reinterpret_cast<uint4*>(s.hist.lo)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    u64 e[PER];
    int b[PER], at[PER];
    bool crowded = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int i = threadIdx.x + j * kThreads;
        e[j] = 0;
        if (i >= n) continue;
        e[j] = s.list[i];
        b[j] = bin(e[j]);
        at[j] = (int)atomicAdd(&s.hist.lo[b[j]], 1u);
        crowded |= at[j] >= 64;
    }
    if (__syncthreads_or(crowded)) return sort_list(s.list, n);
    const uint4 m = reinterpret_cast<const uint4*>(s.hist.lo)[threadIdx.x];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t own = m.x + m.y + m.z + m.w;
    uint32_t x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s.part[warp] = x;
    __syncthreads();
    const uint32_t ahead = __reduce_add_sync(0xffffffffu, lane < warp ? (uint32_t)s.part[lane & (kWarps - 1)] : 0u);
    uint4 first;
    first.x = ahead + x - own; first.y = first.x + m.x; first.z = first.y + m.y; first.w = first.z + m.z;
    reinterpret_cast<uint4*>(s.hist.lo)[threadIdx.x] = first;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (e[j]) s.list[s.hist.lo[b[j]] + at[j]] = e[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (!e[j]) continue;
        const int from = (int)s.hist.lo[b[j]], to = (int)(b[j] + 1 < kBins ? s.hist.lo[b[j] + 1] : (uint32_t)n);
        int place = from;
        for (int i = from; i < to; ++i) place += s.list[i] > e[j];
        at[j] = place;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (e[j]) s.list[at[j]] = e[j];
    __syncthreads();
}

// A key that at least `count` <= kGroups of the CTA's group maxima reach, or below which no logit weighs anything, whichever is
// larger; a little below the count-th largest. Leaves it, the largest key and s.n in s.picked. One histogram of 1024 bins
// over the maxima between the largest and `range` below it (where weights end: a bin over the bits of their keys is
// coarse when some are negative or masked) and a scan: four barriers. (One warp that searched bit by bit took 2 us.)
__device__ __forceinline__ void select(Shared& s, float most0, float most1, int count, float range) {
    static_assert(kGroups == 1024 && kThreads == 512, "two bins a thread");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t k0 = key_of(most0), k1 = key_of(most1);
    reinterpret_cast<uint2*>(s.group)[threadIdx.x] = make_uint2(0, 0);
    const uint32_t h = __reduce_max_sync(0xffffffffu, max(k0, k1)), l = __reduce_min_sync(0xffffffffu, min(k0, k1));
    if (lane == 0) s.part[warp] = (u64)h << 32 | l;
    __syncthreads();
    const u64 hl = s.part[lane & (kWarps - 1)];
    const uint32_t high_key = __reduce_max_sync(0xffffffffu, (uint32_t)(hl >> 32));
    const float high = value_of(high_key), low = fmaxf(fmaxf(value_of(__reduce_min_sync(0xffffffffu, (uint32_t)hl)), high - range), kLowest);
    const float width = fminf(high - low, -kLowest), scale = width > 1e-30f ? 1023.f / width : 0.f;
    // (an infinite maximum: nothing else weighs; none at all: low is above it, and no bin is filled)
    if (most0 >= low && high < INFINITY) atomicAdd(&s.group[min(1023, (int)(fminf(high - most0, -kLowest) * scale))], 1u);
    if (most1 >= low && high < INFINITY) atomicAdd(&s.group[min(1023, (int)(fminf(high - most1, -kLowest) * scale))], 1u);
    if (threadIdx.x == 0) {
        s.picked[0] = high < INFINITY ? key_of(low) : high_key;
        s.picked[1] = high_key;
        s.picked[2] = (uint32_t)s.n;
    }
    __syncthreads();
    const uint2 m = reinterpret_cast<const uint2*>(s.group)[threadIdx.x];
    const int own = (int)(m.x + m.y);
    int x = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s.part[warp] = (u64)x;
    __syncthreads();
    const int ahead = __reduce_add_sync(0xffffffffu, lane < warp ? (int)s.part[lane & (kWarps - 1)] : 0);
    const int before = ahead + x - own;
    if (before < count && before + own >= count) {
        const int bin = 2 * threadIdx.x + (before + (int)m.x >= count ? 0 : 1);
        // the bin's lower end, further down than any rounding
        const float end = high - (float)(bin + 1) / scale - 1e-6f * (fabsf(high) + width);
        if (scale > 0.f && end > low) s.picked[0] = key_of(end);
    }
    __syncthreads();
}

// (ln 2 / 32)^k / k! for k = 1 .. 4
__device__ constexpr double kTerm[4] = {0.02166084939249829, 0.00023459619820224677, 1.6938509724371819e-06, 9.172562701824643e-09};

// One CTA's view of its row.
template <typename T> struct Row {
    static constexpr int N = Chunk<T>::N;
    const T* row;    // the row's logits
    T* stage;        // the slice in shared memory, at the 16-byte phase it has in global memory
    int lo, hi;      // the CTA's logits [lo, hi)
    int base, nvec;  // 16-byte chunks from index `base` (lo rounded down to the boundary)
    Shared& s;
    int rank, ranks, parity;
    int vocab;
    int shift;            // S
    bool staged;
    float top;            // the row's largest logit
    double top_wide;      // the same, at most the largest finite float
    double scale;         // 32 log2 of a weight is (v - top_wide) * scale
    float zero_below;     // logits below weigh less than 2^-S-1: nothing
    float cut_value;      // kept: v > cut_value, or v == cut_value and index <= cut_index
    int cut_index;
    float cut_next;       // the value above cut_value

    __device__ __forceinline__ void set_top(float v) {
        top = v;
        top_wide = (double)fminf(v, -kLowest);
        zero_below = v == INFINITY ? INFINITY : fmaxf(kLowest, __double2float_ru(top_wide - 32.0 * (shift + 2) / scale));
        cut_value = zero_below;
    }
    // S of a row, see the head of this file. `some`: logits that can weigh anything
    __device__ __forceinline__ static int shift_of(int some) { return min(kShift, 63 - (32 - __clz(some - 1))); }
    // Raises S by the steps that the sum of the row's masses leaves room for. With x that sum and one more per logit (rounding takes half
    // a unit at most), the sum at S + d is at most x 2^d; d = clz(x) - 1 keeps that below 2^63. The sum is over the whole row, before any cut, so
    // what is kept later has room too.
    __device__ __forceinline__ void sharpen() {
        u64 sum = 0;
        each_chunk([&](const Chunk<T>& c, int) {
            if (!(c.most() >= zero_below)) return;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                int unused;
                const double w = mass_of(c.raw_at(e), unused);
                sum += c.raw_at(e) >= zero_below ? low52(w) : 0;
            }
        });
        sum = cluster_sum(sum);
        const int more = min(kShift - shift, max(0, __clzll((long long)(sum + (u64)vocab)) - 1));
        if (threadIdx.x < 32)  // (nobody looks for a weight between the barriers of the sum and this one)
            s.power[threadIdx.x] = __hiloint2double(__double2hiint(s.power[threadIdx.x]) + (more << 20), __double2loint(s.power[threadIdx.x]));
        __syncthreads();
        shift += more;
        set_top(top);
    }
    // A chunk that reaches over an end of the slice (the first or the last one), element by element.
    __device__ __forceinline__ Chunk<T> load_edge(int j) const {
        Chunk<T> c;
        const int i0 = base + j * N;
#pragma unroll
        for (int e = 0; e < N; ++e) c.v[e] = i0 + e >= lo && i0 + e < hi ? row[i0 + e] : Num<T>::from_f(-INFINITY);
        return c;
    }
    __device__ __forceinline__ bool whole(int j) const { return base + j * N >= lo && base + j * N + N <= hi; }
    __device__ __forceinline__ Chunk<T> load_global(int j) const {
        Chunk<T> c;
        if (!whole(j)) return load_edge(j);
        c.raw = __ldg(reinterpret_cast<const uint4*>(row + base + j * N));
        return c;
    }
    // Whether the kBatch * kThreads chunks from j on are all whole.
    __device__ __forceinline__ bool inside(int j) const { return whole(j) && j + kBatch * kThreads <= nvec && whole(j + kBatch * kThreads - 1); }
    // Chunks j0, j0 + kThreads, ...: all loads go out before anything waits for one of them. A branch around each
    // (the ends of the slice) made them wait for one another, so where a batch is not inside the slice they are
    // loaded from the nearest whole chunk first and replaced afterwards. Chunks behind the last hold anything.
    template <bool INSIDE> __device__ __forceinline__ void fetch(Chunk<T> (&to)[kBatch], int j0) const {
        const uint4* from = reinterpret_cast<const uint4*>(row + base);
        if (INSIDE) {
#pragma unroll
            for (int x = 0; x < kBatch; ++x) to[x].raw = __ldg(from + j0 + x * kThreads);
            return;
        }
        const int first = whole(0) ? 0 : 1, last = whole(nvec - 1) ? nvec - 1 : nvec - 2;
        if (first <= last) {
#pragma unroll
            for (int x = 0; x < kBatch; ++x) to[x].raw = __ldg(from + max(first, min(last, j0 + x * kThreads)));
        }
#pragma unroll
        for (int x = 0; x < kBatch; ++x) {
            const int j = j0 + x * kThreads;
            if (j < nvec && (j < first || j > last)) to[x] = load_edge(j);
        }
    }
    // The same from shared memory where the slice is there.
    __device__ __forceinline__ void fetch_any(Chunk<T> (&to)[kBatch], int j0) const {
        if (staged) {
#pragma unroll
            for (int x = 0; x < kBatch; ++x) to[x].raw = reinterpret_cast<const uint4*>(stage)[min(j0 + x * kThreads, nvec - 1)];
        } else if (inside(j0 - threadIdx.x)) {
            fetch<true>(to, j0);
        } else {
            fetch<false>(to, j0);
        }
    }
    __device__ __forceinline__ Chunk<T> load(int j) const {
        if (!staged) return load_global(j);
        Chunk<T> c;
        c.raw = reinterpret_cast<const uint4*>(stage)[j];
        return c;
    }
    // f(chunk, its number) for chunks from, from + step, ... below `to`; what lies outside the slice reads as -inf. The next
    // chunk is on its way while one is worked on: where the slice is not staged it comes from L2.
    template <typename F> __device__ __forceinline__ void chunks(int from, int to, int step, F f) const {
        if (from >= to) return;
        Chunk<T> c = load(from);
        for (int j = from; j < to; j += step) {
            Chunk<T> next;
            if (j + step < to) next = load(j + step);
            f(c, j);
            c.raw = next.raw;
        }
    }
    template <typename F> __device__ __forceinline__ void each_chunk(F f) const {
        chunks(threadIdx.x, nvec, kThreads, [&](const Chunk<T>& c, int j) { f(c, base + j * N); });
    }
    // f(value, index) for the slice
    template <typename F> __device__ __forceinline__ void each(F f) const {
        each_chunk([&](const Chunk<T>& c, int i0) {
#pragma unroll
            for (int e = 0; e < N; ++e) f(c.at(e), i0 + e);
        });
    }
    // The weight exp((v - top) / T) as a multiple of 2^-S, rounded to a whole number, for zero_below <= v <= top; and its
    // bin, the weight's distance from 1 in steps of 1/32 of a power of two. With 32 log2 of the weight = n + f, n whole and
    // |f| <= 1/2: 2^(n/32) comes from a table of 32 and a shift, 2^(f/32) = sum (f ln 2 / 32)^k / k! to k = 4 (the first term left out
    // is 2^-39 of the weight); adding 2^52 rounds, and leaves the whole number in the low bits.
    // A pass over weights is bound by the integer and compare instructions (half rate) and the nine 64-bit operations. So
    // n is rounded in 64 bits too, the float is widened by the conversion unit, and the table's entries have their
    // place in the table taken off the exponent's field: n * 2^15 added to the upper word is the whole shift.
    __device__ __forceinline__ double mass_of(float v, int& bin) const {
        constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
        const double d = (double)fminf(v, -kLowest) - top_wide;
        const double t = fma(d, scale, kMagic);
        const double f = fma(d, scale, kMagic - t);
        const int n = __double2loint(t);
        bin = -n;
        double p = fma(kTerm[3], f, kTerm[2]);
        p = fma(p, f, kTerm[1]);
        p = fma(p, f, kTerm[0]);
        p = fma(p, f, 1.0);
        const double w = s.power[n & 31];
        return fma(p, __hiloint2double(__double2hiint(w) + n * 32768, __double2loint(w)), kWhole);
    }
    static constexpr double kWhole = 4503599627370496.0;  // 2^52: a mass, added to it, is the low 52 bits
    __device__ __forceinline__ static u64 low52(double m) { return (u64)__double_as_longlong(m) & 0xfffffffffffffull; }
    __device__ __forceinline__ int bin_of(float v) const {
        return -__double2loint(fma((double)fminf(v, -kLowest) - top_wide, scale, 6755399441055744.0));
    }
    __device__ __forceinline__ u64 mass(uint32_t key) const {
        int unused;
        return value_of(key) >= zero_below ? low52(mass_of(value_of(key), unused)) : 0;
    }
    __device__ __forceinline__ bool kept(float v, int i) const { return v >= cut_value && (v > cut_value || i <= cut_index); }
    // The logits of the chunk from index i0 on that are kept are those from the returned value on: the cut, or the next value above
    // it behind the last index that stays. The one chunk with that index inside loses the others at the cut.
    __device__ __forceinline__ float cut_of(Chunk<T>& c, int i0) const {
        if (i0 + N - 1 > cut_index) {
            if (i0 > cut_index) return cut_next;
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (!kept(c.raw_at(e), i0 + e)) c.v[e] = Num<T>::from_f(-INFINITY);
        }
        return cut_value;
    }
    __device__ __forceinline__ static u64 warp_total(u64 v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    __device__ __forceinline__ u64 block_sum(u64 v) {
        v = warp_total(v);
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
    // Every CTA's word: CTA r's in lane r, 0 behind the last. A CTA writes its word into the others' shared memory, so
    // that after the barrier everyone reads its own. Two sets of slots in turn: one is written again only after the
    // next exchange, which the readers of this one have reached by then. Thread 0's word counts; every CTA of the
    // cluster must have started (see the kernel).
    __device__ __forceinline__ u64 exchange(u64 mine) {
        parity ^= 1;
        const int lane = threadIdx.x & 31;
        if (threadIdx.x < 32) {
            mine = __shfl_sync(0xffffffffu, mine, 0);
            if (lane < ranks) *cg::this_cluster().map_shared_rank(&s.slot[parity][rank], lane) = mine;
        }
        cg::this_cluster().sync();
        return lane < ranks ? s.slot[parity][lane] : 0;
    }
    __device__ __forceinline__ u64 cluster_sum(u64 v) { return warp_total(exchange(block_sum(v))); }
    // A word of rank 0's thread 0 to everyone.
    __device__ __forceinline__ u64 tell(u64 word) {
        if (rank == 0 && threadIdx.x == 0)
            for (int r = 0; r < ranks; ++r) *cg::this_cluster().map_shared_rank(&s.found[2], r) = word;
        cg::this_cluster().sync();
        return s.found[2];
    }

    __device__ __forceinline__ void put(float v, int i) {
        const int at = atomicAdd(&s.n, 1);
        if (at < kCap) s.list[at] = (u64)key_of(v) << 32 | (0xffffffffu - (uint32_t)i);
    }
    // Rank 0 collects the CTAs' lists; returns the entries of all of them (the list holds them only up to kCap).
    __device__ __forceinline__ int collect() {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        __syncthreads();
        const int n = (int)exchange((u64)(unsigned)s.n);
        const int total = (int)warp_total((u64)n);
        if (rank == 0 && total <= kCap && ranks > 1) {
            // a CTA's list is pulled by the kWarps / kMaxCluster warps of its number
            const int r = warp % kMaxCluster;
            const int at = __reduce_add_sync(0xffffffffu, lane < r ? n : 0);
            const int mine = __shfl_sync(0xffffffffu, n, r);
            if (r > 0 && r < ranks) {
                const u64* from = cg::this_cluster().map_shared_rank(s.list, r);
                for (int x = warp / kMaxCluster * 32 + lane; x < mine; x += kWarps / kMaxCluster * 32) s.list[at + x] = from[x];
            }
        }
        __syncthreads();
        return total;
    }
    // The border of a sum over the kept logits in falling order: count (top-k) or mass (top-p) up to and
    // including the border first reaches the target. Moves the cut there.
    template <bool MASS> __device__ __forceinline__ void cut(int k, float p) {
        reinterpret_cast<uint4*>(s.hist.lo)[threadIdx.x] = reinterpret_cast<uint4*>(s.hist.hi)[threadIdx.x] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        each_chunk([&](Chunk<T> c, int i0) {
            const float from = cut_of(c, i0);
            if (!(c.most() >= from)) return;
            int bin[N];
            double w[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if (MASS) w[e] = mass_of(c.raw_at(e), bin[e]);
                else bin[e] = bin_of(c.raw_at(e));
            }
            uint32_t old[N];
#pragma unroll
            for (int e = 0; e < N; ++e)
                old[e] = c.raw_at(e) >= from ? atomicAdd(&s.hist.lo[bin[e]], MASS ? (uint32_t)__double2loint(w[e]) : 1u) : 0u;
            if (!MASS) return;
#pragma unroll
            for (int e = 0; e < N; ++e) {  // 64 bits as two words: the one that overflows the low word carries
                const uint32_t low = (uint32_t)__double2loint(w[e]);
                const uint32_t high = ((uint32_t)__double2hiint(w[e]) & 0xfffffu) + (old[e] + low < low ? 1u : 0u);
                if (c.raw_at(e) >= from && high) atomicAdd(&s.hist.hi[bin[e]], high);
            }
        });
        // The bins are cut into one share per CTA. Everyone tells everyone what its own logits add to each share, so after one
        // barrier all know in whose share the border lies, and add up that share's bins over the cluster, each for itself (one CTA for
        // all would take another cluster barrier). The histograms stay as they are until the exchange in collect().
        __syncthreads();
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = kBins / ranks;
        {
            static_assert(kBins == 4 * kThreads && kWarps >= 2 * kMaxCluster, "a warp's bins lie in one share");
            const uint4 l = reinterpret_cast<const uint4*>(s.hist.lo)[threadIdx.x];
            u64 m = (u64)l.x + l.y + l.z + l.w;
            if (MASS) {
                const uint4 h = reinterpret_cast<const uint4*>(s.hist.hi)[threadIdx.x];
                m += (u64)h.x + h.y + h.z + h.w << 32;
            }
            m = warp_total(m);
            if (lane == 0) s.part[warp] = m;
            __syncthreads();
            if (threadIdx.x < ranks) {
                const int per = kWarps / ranks;
                m = 0;
                for (int w = 0; w < per; ++w) m += s.part[threadIdx.x * per + w];
                for (int r = 0; r < ranks; ++r) *cg::this_cluster().map_shared_rank(&s.shares[MASS][rank][threadIdx.x], r) = m;
            }
        }
        cg::this_cluster().sync();
        u64 in_share = 0;
        if (lane < ranks)
            for (int r = 0; r < ranks; ++r) in_share += s.shares[MASS][r][lane];
        u64 total = warp_total(in_share);
        if (!MASS && total <= (u64)k) return;  // the border lies behind the last logit that weighs anything
        const u64 target = MASS ? target_of(p, total) : (u64)k;
        u64 upto = in_share;
#pragma unroll
        for (int o = 1; o < kMaxCluster; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const int of = __ffs(__ballot_sync(0xffffffffu, upto >= target)) - 1;
        u64 before = __shfl_sync(0xffffffffu, upto - in_share, of);
        const int per = max(1, share / kThreads), first = (int)threadIdx.x * per;
        u64 m[kBins / kThreads], sum = 0, unused;
#pragma unroll
        for (int j = 0; j < kBins / kThreads; ++j) {
            m[j] = 0;
            if (j >= per || first >= share) continue;
            const int b = of * share + first + j;
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) {  // all reads under way together
                if (r >= ranks) continue;
                m[j] += *cg::this_cluster().map_shared_rank(&s.hist.lo[b], r);
                if (MASS) m[j] += (u64)*cg::this_cluster().map_shared_rank(&s.hist.hi[b], r) << 32;
            }
            sum += m[j];
        }
        before += block_scan(sum, unused);
#pragma unroll
        for (int j = 0; j < kBins / kThreads; ++j) {
            if (before < target && before + m[j] >= target) { s.found[0] = (u64)(of * share + first + j); s.found[1] = before; }
            before += m[j];
        }
        __syncthreads();
        const int bin = (int)s.found[0];
        const u64 above = s.found[1];
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        // a window around the bin, wider than any rounding, spares most logits the exact question
        const float width = (float)(1.0 / scale), slack = 1e-5f * (fabsf(top) + (float)(bin + 2) * width);
        const bool windowed = top < INFINITY && width < 1e30f && slack < 1e30f;
        const float from = windowed ? top - ((float)bin + 0.5f) * width - slack : kLowest;
        const float to = windowed ? top - ((float)bin - 0.5f) * width + slack : INFINITY;
        for (int j0 = threadIdx.x; j0 < nvec; j0 += kBatch * kThreads) {
            Chunk<T> c[kBatch];
            fetch_any(c, j0);
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                if (j0 + x * kThreads >= nvec || !(c[x].most() >= from)) continue;
                const int i0 = base + (j0 + x * kThreads) * N;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float v = c[x].raw_at(e);
                    if (v >= from && v <= to && kept(v, i0 + e) && bin_of(v) == bin) put(v, i0 + e);
                }
            }
        }
        const int n = collect();
        if (n <= kCap) {
            u64 key = 0;
            if (rank == 0) {
                if (n <= kPairs) {
                    rank_pairs<MASS>(n, [&](u64 e, int, u64 before, u64 m) {
                        before += above;
                        if (before < target && before + m >= target) s.found[0] = e;
                    });
                    __syncthreads();
                    key = s.found[0];
                } else {
                    key = border<MASS>(n, above, target, dense_of((u64)key_of(from) << 32), dense_of((u64)key_of(to) << 32 | 0xffffffffu));
                }
            }
            key = tell(key);
            cut_value = value_of((uint32_t)(key >> 32));
            cut_next = value_of((uint32_t)(key >> 32) + 1u);
            cut_index = (int)(0xffffffffu - (uint32_t)key);
            return;
        }
        // thousands of logits in one bin: the border's key, bit by bit, then its index
        auto sum_from = [&](uint32_t from) {  // over the bin's logits with keys >= from
            u64 t = 0;
            each([&](float v, int i) {
                if (kept(v, i) && bin_of(v) == bin && key_of(v) >= from) t += MASS ? mass(key_of(v)) : 1;
            });
            return above + cluster_sum(t);
        };
        uint32_t key = 0;
        for (int bit = 31; bit >= 0; --bit)
            if (sum_from(key | 1u << bit) >= target) key |= 1u << bit;
        const u64 over = key == 0xffffffffu ? above : sum_from(key + 1);
        const u64 each_one = MASS ? mass(key) : 1;
        const u64 ties = (target - over + each_one - 1) / each_one;  // equal logits that stay
        int index = -1;  // largest index with fewer than `ties` equal ones up to it
        for (int bit = 24; bit >= 0; --bit) {
            const int to = index + (1 << bit);
            if (to >= vocab) continue;
            u64 t = 0;
            each([&](float v, int i) {
                if (i <= to && key_of(v) == key && kept(v, i)) ++t;
            });
            if (cluster_sum(t) < ties) index = to;
        }
        cut_value = value_of(key);
        cut_next = value_of(key + 1u);
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
    // The smallest mass that stays: min_p of the largest.
    __device__ __forceinline__ u64 least_of(float min_p) const {
        return min_p > 0.f ? (u64)ceil(fmin((double)min_p, 1.0) * (double)mass(key_of(top))) : 0;
    }

    // The draw over everything kept: sums per warp over neighbouring logits, then one warp looks closer.
    __device__ __forceinline__ void draw(float u, float min_p, int64_t* token) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int per = (nvec + kWarps - 1) / kWarps, from = warp * per, to = min(nvec, from + per);
        const u64 least = least_of(min_p);
        const double least_whole = kWhole + (double)least;
        // the masses of a chunk's logits that stay; their sum
        auto masses = [&](Chunk<T> c, int j, u64 (&m)[N]) {
            u64 sum = 0;
            const float cut = cut_of(c, base + j * N);
            if (!(c.most() >= cut)) {
#pragma unroll
                for (int e = 0; e < N; ++e) m[e] = 0;
                return sum;
            }
#pragma unroll
            for (int e = 0; e < N; ++e) {
                int unused;
                const double w = mass_of(c.raw_at(e), unused);
                m[e] = c.raw_at(e) >= cut && w >= least_whole ? low52(w) : 0;
                sum += m[e];
            }
            return sum;
        };
        // The lanes' sums over each part of the warp's range stay in shared memory: the warp with the token looks into one
        // part alone (through a whole range of 131072 / 16 logits it took up to 27 us).
        static_assert(kParts == 8 && 4 * kThreads == kCap, "four parts in the list's place, four in the weights'");
        const int span = 32 * max(4, (per + 32 * kParts - 1) / (32 * kParts));
        auto part_sum = [&](int part) -> u64& { return (part < 4 ? s.list : s.weight)[(part & 3) * kThreads + threadIdx.x]; };
        u64 all = 0;
        for (int start = from, part = 0; start < to; start += span, ++part) {
            u64 sum = 0;
            chunks(start + lane, min(to, start + span), 32, [&](const Chunk<T>& c, int j) {
                u64 m[N];
                sum += masses(c, j, m);
            });
            part_sum(part) = sum;
            all += sum;
        }
        all = warp_total(all);
        __syncthreads();
        if (lane == 0) s.part[warp] = all;
        __syncthreads();
        u64 mine = 0, before = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s.part[w];
            mine += s.part[w];
        }
        const u64 each_cta = exchange(mine);
        const u64 total = warp_total(each_cta);
        before += warp_total(lane < rank ? each_cta : 0);
        const u64 target = drawn(u, total);
        if (target < before || target >= before + all) return;  // whole warps
        int start = from;
        for (int part = 0; start + span < to; start += span, ++part) {
            const u64 sum = warp_total(part_sum(part));
            if (target < before + sum) break;
            before += sum;
        }
        for (int j0 = start; j0 < to; j0 += 32) {
            u64 m[N], own = 0;
            const int j = j0 + lane;
#pragma unroll
            for (int e = 0; e < N; ++e) m[e] = 0;
            if (j < to) own = masses(load(j), j, m);
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

    // An entry's rank as a number without gaps: value (without the bits that T does not have), then index.
    __device__ __forceinline__ u64 dense_of(u64 entry) const {
        const int bits = 32 - __clz(vocab - 1);  // of an index
        constexpr int kEmpty = std::is_same_v<T, __nv_bfloat16> ? 16 : std::is_same_v<T, __half> ? 13 : 0;
        return (u64)((uint32_t)(entry >> 32) >> kEmpty) << bits | ((uint32_t)entry & ((1u << bits) - 1));
    }
    // The entry of list[0, n) at which the sum of masses (or 1 each) over falling entries, with `above` before the first, first
    // reaches the target; all dense numbers lie in [low, high]. A histogram of 1024 steps over [low, high], again over the
    // step with the border while that holds more than a warp can rank: one round for as good as every row, for equal
    // logits too (then the steps part their indexes).
    template <bool MASS> __device__ __forceinline__ u64 border(int n, u64 above, u64 target, u64 low, u64 high) {
        constexpr int PER = kCap / kThreads;
        const int lane = threadIdx.x & 31;
        u64 e[PER], m[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * kThreads;
            e[j] = i < n ? s.list[i] : 0;  // 0: out
            m[j] = i < n ? (MASS ? mass((uint32_t)(e[j] >> 32)) : 1) : 0;
        }
        for (;;) {
            const int shift = max(0, 54 - __clzll((long long)(high - low | 1)));
            __syncthreads();
            reinterpret_cast<uint2*>(s.hist.lo)[threadIdx.x] = reinterpret_cast<uint2*>(s.hist.hi)[threadIdx.x] = make_uint2(0, 0);
            if (threadIdx.x == 0) s.n = 0;
            __syncthreads();
            int at[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (!e[j]) continue;
                at[j] = (int)((high - dense_of(e[j])) >> shift);  // the largest in front
                const uint32_t add = (uint32_t)m[j], old = atomicAdd(&s.hist.lo[at[j]], add);
                const uint32_t up = (uint32_t)(m[j] >> 32) + (old + add < old ? 1u : 0u);
                if (up) atomicAdd(&s.hist.hi[at[j]], up);
            }
            __syncthreads();
            const uint2 l = reinterpret_cast<const uint2*>(s.hist.lo)[threadIdx.x], h = reinterpret_cast<const uint2*>(s.hist.hi)[threadIdx.x];
            const u64 m0 = (u64)h.x << 32 | l.x, m1 = (u64)h.y << 32 | l.y;
            u64 unused;
            const u64 before = above + block_scan(m0 + m1, unused);
            if (before < target && before + m0 + m1 >= target) {
                const bool second = before + m0 < target;
                s.found[0] = 2 * threadIdx.x + (second ? 1 : 0);
                s.found[1] = before + (second ? m0 : 0);
            }
            __syncthreads();
            const int step = (int)s.found[0];
            above = s.found[1];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (!e[j]) continue;
                if (at[j] != step) { e[j] = 0; continue; }
                const int x = atomicAdd(&s.n, 1);
                if (x < 32) s.pair[x] = Entry{e[j], m[j]};
            }
            __syncthreads();
            const int left = s.n;
            if (left <= 32 || shift == 0) {  // (a step of one dense number holds one entry)
                const Entry mine = s.pair[lane < left ? lane : 0];
                u64 sum = above;
                for (int j = 0; j < left; ++j) {
                    const Entry o = s.pair[j];
                    if (o.key > mine.key) sum += o.mass;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, lane < left && sum < target && sum + mine.mass >= target);
                return __shfl_sync(0xffffffffu, mine.key, __ffs(hit) - 1);
            }
            high -= (u64)step << shift;
            low = max(low, high - ((1ull << shift) - 1));
        }
    }

    // f(entry, its place, the sum before it, its own mass or 1) for list[0, n), n <= kPairs, all in falling order,
    // without sorting: a thread compares its entry with every other.
    template <bool MASS, typename F> __device__ __forceinline__ void rank_pairs(int n, F f) {
        const int i = threadIdx.x;
        Entry mine = {0, 0};
        if (i < n) {
            mine.key = s.list[i];
            mine.mass = MASS ? mass((uint32_t)(mine.key >> 32)) : 1;
            s.pair[i] = mine;
        }
        __syncthreads();
        if (i >= n) return;
        int place = 0;
        u64 before = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const Entry o = s.pair[j];
            if (o.key > mine.key) { ++place; before += o.mass; }
        }
        f(mine.key, place, before, mine.mass);
    }

    // rank 0, with the largest logits in list[0, n): everything that is left to do
    __device__ __forceinline__ void finish_list(int n, int k, float p, float min_p, float u, int64_t* token) {
        const u64 least = least_of(min_p);
        if (n <= kPairs) {
            u64 key = 0, before = 0, m = 0;
            bool in = false;
            rank_pairs<true>(n, [&](u64 e, int place, u64 b, u64 w) { key = e; before = b; m = w; in = place < k; });
            const u64 total = block_sum(in ? m : 0);  // (its barrier also ends the reading of s.pair)
            if (p < 1.f) in = in && before < target_of(p, total);
            in = in && m >= least;
            if (threadIdx.x < n) s.pair[threadIdx.x] = Entry{key << 32, in ? m : 0};  // falling in ~index: rising in index
            __syncthreads();
            return draw_pairs(n, u, token);
        }
        // falling from the largest to the smallest listed
        const float low = value_of(lowest_key(n));
        const float per_unit = top - low > 0.f ? (float)(kBins - 1) / fminf(top - low, 3.4e38f) : 0.f;
        sort_by_bins(s, n, [&](u64 e) {
            const float d = top - value_of((uint32_t)(e >> 32));
            return d > 0.f ? min(kBins - 1, (int)(fminf(d, 3.4e38f) * per_unit)) : 0;
        });
        finish_sorted(min(n, k), p, least, u, token);
    }
    // The smallest key of list[0, n), over the whole CTA, in every lane.
    __device__ __forceinline__ uint32_t lowest_key(int n) {
        uint32_t low = 0xffffffffu;
        for (int i = threadIdx.x; i < n; i += kThreads) low = min(low, (uint32_t)(s.list[i] >> 32));
        low = __reduce_min_sync(0xffffffffu, low);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = low;
        __syncthreads();
        return __reduce_min_sync(0xffffffffu, (uint32_t)s.part[threadIdx.x & (kWarps - 1)]);
    }
    // The rest over the first n <= kListK entries of a sorted list, one a thread.
    __device__ __forceinline__ void finish_sorted(int n, float p, u64 least, float u, int64_t* token) {
        static_assert(kListK <= kThreads, "an entry a thread");
        const int i = threadIdx.x;
        u64 total, e = i < n ? s.list[i] : 0, m = i < n ? mass((uint32_t)(e >> 32)) : 0;
        const u64 before = block_scan(m, total);
        const bool in = e && before < (p < 1.f ? target_of(p, total) : ~0ull) && m >= least;
        if (!in) m = 0;
        const int kept_n = (int)block_sum((u64)in);  // a prefix of the list: weights only fall
        if (kept_n <= kPairs) {
            if (i < kept_n) s.pair[i] = Entry{e << 32, m};  // falling in ~index: rising in index
            __syncthreads();
            return draw_pairs(kept_n, u, token);
        }
        // in index order: entries (index, place), with their weights beside them
        __syncthreads();
        if (i < kept_n) s.list[i] = e << 32 | (u64)i;
        const float per_index = (float)(kBins - 1) / (float)vocab;
        sort_by_bins(s, kept_n, [&](u64 x) { return (int)((float)(0xffffffffu - (uint32_t)(x >> 32)) * per_index); });
        if (i < kept_n) s.weight[i] = m;
        __syncthreads();
        e = i < kept_n ? s.list[i] : 0;
        m = i < kept_n ? s.weight[(uint32_t)e] : 0;
        const u64 at = block_scan(m, total), x = drawn(u, total);
        if (x >= at && x < at + m) *token = (int64_t)(0xffffffffu - (uint32_t)(e >> 32));
    }
    // The draw among pair[0, n): keys that fall as the index rises, and masses. Entry i belongs to thread i.
    __device__ __forceinline__ void draw_pairs(int n, float u, int64_t* token) {
        if (threadIdx.x >= n) return;
        const Entry mine = s.pair[threadIdx.x];
        u64 at = 0, sum = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const Entry o = s.pair[j];
            if (o.key > mine.key) at += o.mass;
            sum += o.mass;
        }
        const u64 x = drawn(u, sum);
        if (x >= at && x < at + mine.mass) *token = (int64_t)(0xffffffffu - (uint32_t)(mine.key >> 32));
    }

    // The logits of a thread's chunks j0, j0 + kThreads, ... that reach the bound, into the list. Few threads have one, so
    // which they are is found first, then one atomic makes room for them and they are read once more (from L1).
    template <bool INSIDE> __device__ __forceinline__ void take(const Chunk<T> (&c)[kBatch], int j0, float bound) {
        uint32_t in = 0;
#pragma unroll
        for (int x = 0; x < kBatch; ++x) {
            if (!(c[x].most() >= bound)) continue;
            if (!INSIDE && j0 + x * kThreads >= nvec) continue;
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c[x].raw_at(e) >= bound) in |= 1u << (x * N + e);
        }
        if (!in) return;
        int at = atomicAdd(&s.n, __popc(in));
        do {
            const int bit = __ffs(in) - 1;
            in &= in - 1;
            const int i = base + (j0 + bit / N * kThreads) * N + bit % N;
            if (at < kCap) s.list[at] = (u64)key_of(Num<T>::to_f(row[i])) << 32 | (0xffffffffu - (uint32_t)i);
            ++at;
        } while (in);
    }
    // Drops the list's entries below a key. Not for a list that has overflowed.
    __device__ __forceinline__ void drop_below(uint32_t key) {
        constexpr int PER = kCap / kThreads;
        u64 e[PER];
        __syncthreads();
        const int n = s.n;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * kThreads;
            e[j] = i < n ? s.list[i] : 0;
        }
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (e[j] && (uint32_t)(e[j] >> 32) >= key) s.list[atomicAdd(&s.n, 1)] = e[j];
        __syncthreads();
    }

    // Streams the slice and leaves every logit that can be among the row's k largest in the CTAs' lists (or more than
    // kCap in one, which says that the list will not do). Sets `top`.
    __device__ __forceinline__ void stream(int k, float range) {
        const int share = (k + ranks - 1) / ranks;  // so many of every CTA together are k
        float most[2] = {-INFINITY, -INFINITY};
        uint32_t own = 0;
        if (threadIdx.x == 0) s.n = 0;
        Chunk<T> c[kBatch];
        constexpr int kStep = kBatch * kThreads;
        auto look = [&](const Chunk<T> (&c)[kBatch], int j0, auto inside) {
#pragma unroll
            for (int x = 0; x < kBatch; ++x)
                if (inside || j0 + x * kThreads < nvec) most[x & 1] = fmaxf(most[x & 1], c[x].most());
        };
        const std::integral_constant<bool, false> ends;
        const std::integral_constant<bool, true> whole_batch;
        const bool one = nvec <= kStep;
        if (one) {
            fetch<false>(c, threadIdx.x);
            look(c, threadIdx.x, ends);
        } else {
            float bound = kLowest;
            int j0 = threadIdx.x, seen = kStep, renew = kStep;  // renew: chunks seen when the bound is renewed next
            // A renewal costs the CTA a microsecond without work. About 1.1 k logits come in between two of them at a
            // doubling, three times as many at a fourfold count: small lists take that.
            const int grow = k <= kCap / 9 ? 4 : 2;
            bool here = inside(0);
            if (here) fetch<true>(c, j0); else fetch<false>(c, j0);
            auto batch = [&](const Chunk<T> (&c)[kBatch], Chunk<T> (&next)[kBatch]) {
                const bool there = seen < nvec && inside(seen);
                if (there) fetch<true>(next, j0 + kStep);
                else if (seen < nvec) fetch<false>(next, j0 + kStep);
                if (here) look(c, j0, whole_batch); else look(c, j0, ends);
                if (seen >= renew || seen >= nvec) {
                    select(s, most[0], most[1], k, range);
                    own = s.picked[0];
                    bound = bound_of(own);
                    renew = grow * seen;
                    const int n = (int)s.picked[2];  // s.n itself is on the move again
                    if (n > kCap / 2 && n <= kCap) drop_below(own);
                }
                if (here) take<true>(c, j0, bound); else take<false>(c, j0, bound);
                if (seen >= nvec) return false;
                here = there;
                j0 += kStep;
                seen += kStep;
                return true;
            };
            Chunk<T> other[kBatch];
            while (batch(c, other) && batch(other, c)) {}
            __syncthreads();
        }
        if (one || ranks > 1) select(s, most[0], most[1], share, range);
        uint32_t bound = s.picked[0];
        const u64 o = exchange((u64)s.picked[1] << 32 | bound);
        const bool lane_in = (threadIdx.x & 31) < ranks;
        set_top(value_of(__reduce_max_sync(0xffffffffu, (uint32_t)(o >> 32))));
        bound = max(own, __reduce_min_sync(0xffffffffu, lane_in ? (uint32_t)o : 0xffffffffu));
        if (one) take<false>(c, threadIdx.x, bound_of(bound));
        else if (s.n <= kCap) drop_below(bound);
    }

    // Reads the slice for the general way (and keeps it in shared memory, if it fits). Sets `top`.
    __device__ __forceinline__ void read_slice() {
        float most = -INFINITY;
        for (int j0 = threadIdx.x; j0 < nvec; j0 += kBatch * kThreads) {
            Chunk<T> c[kBatch];
            if (inside(j0 - threadIdx.x)) fetch<true>(c, j0); else fetch<false>(c, j0);
#pragma unroll
            for (int x = 0; x < kBatch; ++x) {
                if (j0 + x * kThreads >= nvec) continue;
                if (staged) reinterpret_cast<uint4*>(stage)[j0 + x * kThreads] = c[x].raw;
                most = fmaxf(most, c[x].most());
            }
        }
        uint32_t key = __reduce_max_sync(0xffffffffu, key_of(most));
        if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = key;
        __syncthreads();
        key = __reduce_max_sync(0xffffffffu, (uint32_t)s.part[threadIdx.x & (kWarps - 1)]);
        set_top(value_of(__reduce_max_sync(0xffffffffu, (uint32_t)exchange(key))));
    }

    __device__ __forceinline__ void greedy(int64_t* token) {
        uint32_t first = 0x7fffffffu;
        each([&](float v, int i) { if (v == top) first = min(first, (uint32_t)i); });
        first = __reduce_min_sync(0xffffffffu, first);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s.part[threadIdx.x >> 5] = first;
        __syncthreads();
        first = __reduce_min_sync(0xffffffffu, (uint32_t)s.part[threadIdx.x & (kWarps - 1)]);
        const uint32_t o = (uint32_t)exchange(first);
        first = __reduce_min_sync(0xffffffffu, (threadIdx.x & 31) < ranks ? o : 0xffffffffu);
        if (rank == 0 && threadIdx.x == 0) *token = (int64_t)first;
    }
};

// LONG: rows of more than kFewWeights logits. A kernel of its own: with the pass that they need in it the others took up to 4 %
// longer (256 x 131072 fp32: no cut 88.6 us and 85.4, top-p 191 and 187).
template <typename T, bool LONG>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams P) {
    ptx::pdl_wait();
    ptx::pdl_trigger();
    extern __shared__ __align__(16) unsigned char stage[];
    __shared__ Shared shared;
    auto cluster = cg::this_cluster();
    using R = Row<T>;
    constexpr int N = R::N;
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    auto started = cluster.barrier_arrive();  // the first exchange writes to CTAs that must have started
    const int64_t b = blockIdx.x / ranks;
    const T* row = (const T*)P.logits + b * P.row_stride;
    const int lo = min(P.vocab, rank * P.slice), hi = min(P.vocab, lo + P.slice);
    const int phase = (int)(((uintptr_t)(row + lo) & 15) / sizeof(T));
    R r{row, (T*)stage, lo, hi, lo - phase, lo < hi ? (hi - lo + phase + N - 1) / N : 0, shared, rank, ranks, 0, P.vocab, 0, false};

    const float temperature = P.temperature ? P.temperature[b] : P.temperature0;
    const float p = P.top_p ? P.top_p[b] : P.top_p0, min_p = P.min_p ? P.min_p[b] : P.min_p0;
    int k = P.top_k ? P.top_k[b] : P.top_k0;
    if (k <= 0 || k > P.vocab) k = P.vocab;
    const float u = P.u[b];
    int64_t* token = P.tokens + b;
    const bool greedy = !(temperature > 0.f), by_list = !greedy && k < P.vocab && k <= kListK;

    if (P.rows != kAllRows && by_list != (P.rows == kListRows)) {  // the other launch's
        cluster.barrier_wait(std::move(started));
        return;
    }

    const double t = fmax((double)temperature, 1e-20);
    r.scale = fmax(32.0 * 1.4426950408889634 / t, 1e-300);  // at T = inf every finite logit weighs 1
    r.cut_index = 0x7fffffff;
    const bool few = !LONG || k <= kFewWeights;
    r.shift = R::shift_of(few ? k : P.vocab);
    if (threadIdx.x < 32) {
        const double w = P.power[threadIdx.x];
        shared.power[threadIdx.x] = __hiloint2double(__double2hiint(w) - ((kShift - r.shift) << 20), __double2loint(w));
    }
    cluster.barrier_wait(std::move(started));

    if (by_list) {
        r.stream(k, (float)((r.shift + 2) * 0.6931471805599454 * t));  // weights end before that far below the largest
        const int n = r.top == -INFINITY ? 0 : r.collect();
        if (r.top > -INFINITY && n <= kCap) {
            // rank 0 has pulled the lists: the others may leave
            auto pulled = cluster.barrier_arrive();
            if (rank == 0) r.finish_list(n, k, p, min_p, u, token);
            cluster.barrier_wait(std::move(pulled));
            return;
        }
    } else {
        r.staged = P.staged != 0;
        r.read_slice();
    }
    if (r.top == -INFINITY) {  // nothing to draw from
        if (rank == 0 && threadIdx.x == 0) *token = -1;
        return;
    }
    if (greedy) return r.greedy(token);
    if (!few) r.sharpen();
    if (k < P.vocab) r.template cut<false>(k, 0.f);
    if (p < 1.f) r.template cut<true>(0, p);
    r.draw(u, min_p, token);
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

    // CTAs of a row. List rows: as many as leave no more than one SM in six without any, at most one an SM while a CTA keeps fewer
    // than 64 logits a thread, and 8 of those (32 x 50257 bf16: 10 us with four a row, 15.6 with eight; 64 x 131072: 13.3
    // with two, 15.5 with four; 120 x 131072 fp32: 27.7 with one, 23.2 with two; 256 x 131072: 34 and 44).
    // General rows, bound by instructions, give every SM one, and fill both its places while a CTA keeps 64 logits a thread (64 x 131072
    // bf16, top-p: 58 us with two a row, 51 with four, 62 with eight; 256 x 131072 fp32: 193 with one, 182 with two, 198 with
    // four; 512 x 50257: 149, 166, 198). Settings given row by row give rows of unequal work: twice as many (64 x 131072 bf16
    // mixed: 44 us with four, 39 with eight; 256 x 131072 fp32: 166, 110, 105 with one, two, four).
    const bool unequal = a->temperature || a->top_k || a->top_p || a->min_p, all_lists = !a->top_k && a->top_k_all > 0 && a->top_k_all <= kListK;
    const int64_t sms = sm_count();
    constexpr int64_t kFew = 8 * kThreads, kMany = 64 * kThreads;
    auto slice_of = [&](int c) { return round_up<int64_t>(ceil_div<int64_t>(a->vocab, c), 8); };
    auto grow = [&](int c, int64_t ctas, int64_t logits) {
        while (c < kMaxCluster && a->batch * c < ctas && slice_of(c) > logits) c *= 2;
        return c;
    };
    const int C_lists = grow(grow(1, sms / 2 + 1, kFew), sms * 5 / 6, kMany);
    const int C_others = grow(grow(1, unequal && a->batch < sms ? 2 * sms : sms, kFew), (unequal ? 4 : 2) * sms, kMany);
    SampleParams P = {};
    P.logits = a->logits; P.u = a->uniform; P.temperature = a->temperature; P.top_p = a->top_p; P.min_p = a->min_p;
    P.top_k = a->top_k; P.tokens = a->tokens; P.row_stride = a->row_stride;
    P.temperature0 = a->temperature_all; P.top_p0 = a->top_p_all; P.min_p0 = a->min_p_all; P.top_k0 = a->top_k_all;
    P.vocab = (int)a->vocab;
    for (int i = 0; i < 32; ++i) {
        const double w = ldexp(exp2(i / 32.0), kShift);
        uint64_t bits;
        memcpy(&bits, &w, 8);
        bits -= (uint64_t)i << 47;
        memcpy(&P.power[i], &bits, 8);
    }

    cudaError_t le = cudaSuccess;
    auto launch = [&](auto kern, PerDeviceOnce& once, int C, int rows) {
        P.slice = (int)slice_of(C);
        P.rows = rows;
        const size_t bytes = round_up<size_t>((size_t)(P.slice + 8) * e, 16);
        P.staged = rows != kListRows && bytes <= (a->batch * C > sm_count() ? kStageTwo : kStageMax) ? 1 : 0;
        int dev = 0;
        cudaGetDevice(&dev);
        if (P.staged && !once.done(dev)) {
            le = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kStageMax);
            if (le != cudaSuccess) return;
            once.mark(dev);
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(a->batch * C));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = P.staged ? bytes : 0;
        cfg.stream = as_stream(a->stream);
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)C;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        le = cudaLaunchKernelEx(&cfg, kern, P);
    };
    auto launch_all = [&](auto kern, PerDeviceOnce& once) {
        // Where top-k is given row by row, in batches that fill the GPU with one CTA a row, list rows want one CTA and the others
        // several: a launch for each kind (256 x 131072 fp32, lists alone: 39 us, in one launch of one CTA a row 34, of
        // four 60; mixed: 122, 166 and 105).
        if (a->top_k && a->batch >= sms && C_others > 1) {
            launch(kern, once, C_lists, kListRows);
            if (le == cudaSuccess) launch(kern, once, C_others, kOtherRows);
        } else {
            launch(kern, once, all_lists ? C_lists : C_others, kAllRows);
        }
    };
    RFX_DISPATCH_DTYPE(a->dtype, T, {
        static PerDeviceOnce once, once_long;
        if (a->vocab > kFewWeights) launch_all(sample_kernel<T, true>, once_long);
        else launch_all(sample_kernel<T, false>, once);
    });
    if (le != cudaSuccess) { cudaGetLastError(); return fail(RFX_CUDA_ERROR, "%s: %s", name, cudaGetErrorString(le)); }
    return check_launch(name);
}
