// RMS norm of every query and key head with the position rotation in the same pass, to dense rows or
// (with V) straight into the paged pool:
//   r = 1 / sqrt(mean_d x_d^2 + eps),  n_d = x_d * r * w_d,
//   y_i = n_i c_i - n_j s_i,  y_j = n_i s_i + n_j c_i   for the pairs (i, j = i + D/2) or (2i, 2i + 1).
// Everything is fp32 and the result is rounded once (rope.cu rounds every step, because the reference's
// rotation does; there is no such composition to match bit for bit here).
//
// Algorithmic bytes: 2*N*(H_q + 2*H_kv)*D*e plus a table row per token; about 7 fp32 operations per
// element, so HBM-bound at every size that is not bound by the launch.
#include "common.cuh"
#include "ptx.cuh"

namespace rfx {
namespace {

enum QkNormMode { kDense = 0, kPool = 1, kPool8 = 2 };

struct QkNormParams {
    const void *q, *k, *v, *cos, *sin, *wq, *wk;
    void *q_out, *k_out, *k_cache, *v_cache;
    float *k_scales, *v_scales;
    const int64_t* slots;
    const int32_t* positions;
    int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, qo_sn, qo_sh, ko_sn, ko_sh;
    int64_t c_sblk, c_sh, c_spos, t_s;
    int64_t n_tokens, num_slots, table_rows;
    int hq, hkv, D, block_size;
    int lanes;      // lanes of a row, a power of two
    int splits;     // warps that share the rows of a token
    float eps, inv_d;
};

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };

template <typename T, int V> __device__ __forceinline__ void load_f(const T* p, float (&f)[V]) {
    constexpr int W = 16 / sizeof(T) < V ? 16 / sizeof(T) : V;  // at most 16 bytes an access
#pragma unroll
    for (int o = 0; o < V; o += W) {
        const Vec<T, W> x = *reinterpret_cast<const Vec<T, W>*>(p + o);
#pragma unroll
        for (int j = 0; j < W; ++j) f[o + j] = Num<T>::to_f(x.v[j]);
    }
}

template <typename T, int V> __device__ __forceinline__ void store_f(T* p, const float (&f)[V]) {
    Vec<T, V> x;
#pragma unroll
    for (int j = 0; j < V; ++j) x.v[j] = Num<T>::from_f(f[j]);
    *reinterpret_cast<Vec<T, V>*>(p) = x;
}

template <int V> __device__ __forceinline__ void store_q8(int8_t* p, const float (&f)[V], float scale) {
    Vec<int8_t, V> x;
#pragma unroll
    for (int j = 0; j < V; ++j) x.v[j] = (int8_t)fminf(127.f, fmaxf(-127.f, rintf(__fdiv_rn(f[j], scale))));
    *reinterpret_cast<Vec<int8_t, V>*>(p) = x;
}

// A row is cut into pieces of two V-vectors that hold V whole pairs: elements [pV, pV+V) and their
// partners D/2 further on, or 2V neighbours. `lanes` lanes take a row (NP pieces each), a warp
// 32/lanes rows at a time; the sum of squares needs no shared memory. A lane keeps its piece for every
// row of its token, so the table's factors are loaded once per token and lane.
template <typename T, typename TT, int V, int NP, bool INTER, int MODE>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkNormParams P) {
    ptx::pdl_trigger();  // the kernel behind this one waits for this one's end before it reads anything
    ptx::pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int64_t n = warp / P.splits;
    if (n >= P.n_tokens) return;  // whole warps
    const int sub = lane & (P.lanes - 1), group = lane / P.lanes, groups = 32 / P.lanes;
    const int D = P.D, half = D >> 1;
    const int rows = P.hq + (MODE == kDense ? 1 : 2) * P.hkv;

    const int64_t pos = P.positions ? (int64_t)P.positions[n] : n;
    const bool known = pos >= 0 && pos < P.table_rows;
    int64_t at = -1;  // offset of the token's row for kv head 0 in the pool
    int64_t scale_at = 0;
    if (MODE != kDense) {
        const int64_t slot = P.slots[n];
        if (known && slot >= 0 && slot < P.num_slots) {
            const int64_t page = slot / P.block_size;
            const int in = (int)(slot - page * P.block_size);
            at = page * P.c_sblk + in * P.c_spos;
            scale_at = page * P.hkv * P.block_size + in;
        }
    }

    int off1[NP], off2[NP];
    bool mine[NP];
    float c[NP][V], s[NP][V];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int p = sub + k * P.lanes;
        mine[k] = p * V < half;
        off1[k] = mine[k] ? (INTER ? 2 * V * p : V * p) : 0;
        off2[k] = off1[k] + (INTER ? V : half);
        if (!known || !mine[k]) continue;
        const TT* cr = (const TT*)P.cos + pos * P.t_s + off1[k];
        const TT* sr = (const TT*)P.sin + pos * P.t_s + off1[k];
        if constexpr (INTER) {  // the factors of a pair stand at its even entry
            float a[2 * V], b[2 * V];
            load_f<TT, 2 * V>(cr, a);
            load_f<TT, 2 * V>(sr, b);
#pragma unroll
            for (int j = 0; j < V; ++j) { c[k][j] = a[2 * j]; s[k][j] = b[2 * j]; }
        } else {
            load_f<TT, V>(cr, c[k]);
            load_f<TT, V>(sr, s[k]);
        }
    }

    const int step = P.splits * groups;
    for (int base = (int)(warp - n * P.splits) * groups; base < rows; base += step) {
        const int row = base + group;
        const bool in = row < rows;
        const bool is_q = row < P.hq;
        const bool is_v = MODE != kDense && row >= P.hq + P.hkv;
        const int h = is_q ? row : (is_v ? row - P.hq - P.hkv : row - P.hq);
        // a token without a table row, or (K and V) without a slot, writes nothing
        const bool live = in && known && (MODE == kDense || is_q || at >= 0);
        const T* x = is_q ? (const T*)P.q + n * P.q_sn + h * P.q_sh
                          : (is_v ? (const T*)P.v + n * P.v_sn + h * P.v_sh : (const T*)P.k + n * P.k_sn + h * P.k_sh);
        float a[NP][V], b[NP][V];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) a[k][j] = b[k][j] = 0.f;
            if (!live || !mine[k]) continue;
            load_f<T, V>(x + off1[k], a[k]);
            load_f<T, V>(x + off2[k], b[k]);
#pragma unroll
            for (int j = 0; j < V; ++j) sum += a[k][j] * a[k][j] + b[k][j] * b[k][j];
        }
        for (int o = P.lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (!is_v) {
            const float r = 1.f / sqrtf(sum * P.inv_d + P.eps);
            const T* w = (const T*)(is_q ? P.wq : P.wk);
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if (!live || !mine[k]) continue;
                float w1[V], w2[V];
                load_f<T, V>(w + off1[k], w1);
                load_f<T, V>(w + off2[k], w2);
                if constexpr (INTER) {
                    // the piece's 2V neighbours: pair j is (z[2j], z[2j+1])
                    float z[2 * V];
#pragma unroll
                    for (int j = 0; j < V; ++j) { z[j] = a[k][j] * r * w1[j]; z[V + j] = b[k][j] * r * w2[j]; }
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float u = z[2 * j], t = z[2 * j + 1];
                        z[2 * j] = u * c[k][j] - t * s[k][j];
                        z[2 * j + 1] = u * s[k][j] + t * c[k][j];
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) { a[k][j] = z[j]; b[k][j] = z[V + j]; }
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float u = a[k][j] * r * w1[j], t = b[k][j] * r * w2[j];
                        a[k][j] = u * c[k][j] - t * s[k][j];
                        b[k][j] = u * s[k][j] + t * c[k][j];
                    }
                }
            }
        }
        if (MODE == kPool8) {  // the row's scale: max |y| / 127 over its lanes (1 for a row of zeros)
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < NP; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) top = fmaxf(top, fmaxf(fabsf(a[k][j]), fabsf(b[k][j])));
            for (int o = P.lanes >> 1; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (!is_q && live) {
                const float scale = top > 0.f ? __fdiv_rn(top, 127.f) : 1.f;
                int8_t* y = (int8_t*)(is_v ? P.v_cache : P.k_cache) + at + h * P.c_sh;
                if (sub == 0) (is_v ? P.v_scales : P.k_scales)[scale_at + (int64_t)h * P.block_size] = scale;
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    if (!mine[k]) continue;
                    store_q8<V>(y + off1[k], a[k], scale);
                    store_q8<V>(y + off2[k], b[k], scale);
                }
                continue;
            }
        }
        T* y;
        if (is_q) y = (T*)P.q_out + n * P.qo_sn + h * P.qo_sh;
        else if (MODE == kDense) y = (T*)P.k_out + n * P.ko_sn + h * P.ko_sh;
        else y = (T*)(is_v ? P.v_cache : P.k_cache) + at + h * P.c_sh;
        // a dense row of a token without a table row is left as it is where it is rotated in place, else zero
        const bool zero = in && !known && (is_q || MODE == kDense) && y != x;
        if (!live && !zero) continue;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            if (!mine[k]) continue;
            store_f<T, V>(y + off1[k], a[k]);
            store_f<T, V>(y + off2[k], b[k]);
        }
    }
}

int qk_norm_impl(const RfxQkNormRopeArgs* a, bool append, const char* name) {
    if (!a) return fail(RFX_INVALID_ARGUMENT, "%s: null args", name);
    RFX_REQUIRE(dtype_ok(a->dtype), "%s: unknown dtype %d", name, a->dtype);
    RFX_REQUIRE(a->head_dim > 0 && a->head_dim % 2 == 0, "head_dim must be even for RoPE");
    RFX_REQUIRE(a->head_dim <= 512, "%s: head_dim %lld > 512", name, (long long)a->head_dim);
    RFX_REQUIRE(a->n_tokens >= 0 && a->num_q_heads >= 0 && a->num_kv_heads >= 0 && a->table_rows >= 0 &&
                    a->num_q_heads < (1 << 20) && a->num_kv_heads < (1 << 20) && a->n_tokens < (1ll << 40),
                "%s: bad sizes N=%lld Hq=%lld Hkv=%lld rows=%lld", name, (long long)a->n_tokens,
                (long long)a->num_q_heads, (long long)a->num_kv_heads, (long long)a->table_rows);
    RFX_REQUIRE(a->eps >= 0.f, "%s: eps must not be negative", name);
    const bool q8 = append && a->kv_int8;
    if (append)
        RFX_REQUIRE(a->num_kv_heads > 0 && a->num_blocks > 0 && a->block_size > 0 && a->block_size < (1ll << 31),
                    "%s: bad pool sizes blocks=%lld bs=%lld", name, (long long)a->num_blocks, (long long)a->block_size);
    if (a->n_tokens == 0 || a->num_q_heads + a->num_kv_heads == 0) return RFX_SUCCESS;
    RFX_REQUIRE(a->cos && a->sin && a->q_weight && a->k_weight, "%s: null pointer", name);
    RFX_REQUIRE(a->num_q_heads == 0 || (a->q && a->q_out), "%s: null q or q_out", name);
    if (append) {
        RFX_REQUIRE(a->k && a->v && a->k_cache && a->v_cache && a->slot_mapping && a->positions, "%s: null pointer", name);
        RFX_REQUIRE(!q8 || (a->k_scales && a->v_scales), "%s: an int8 pool needs k_scales and v_scales", name);
    } else {
        RFX_REQUIRE(a->num_kv_heads == 0 || (a->k && a->k_out), "%s: null k or k_out", name);
    }
    int st = check_device();
    if (st != RFX_SUCCESS) return st;

    const size_t e = dtype_size(a->dtype), te = a->tables_f32 ? 4 : e;
    const int D = (int)a->head_dim, half = D / 2;
    const bool inter = a->interleaved != 0;
    const int vmax = (int)(16 / e);
    QkNormParams P = {};
    P.q = a->q; P.k = a->k; P.v = a->v; P.cos = a->cos; P.sin = a->sin; P.wq = a->q_weight; P.wk = a->k_weight;
    P.q_out = a->q_out; P.k_out = a->k_out; P.k_cache = a->k_cache; P.v_cache = a->v_cache;
    P.k_scales = a->k_scales; P.v_scales = a->v_scales; P.slots = a->slot_mapping; P.positions = a->positions;
    P.q_sn = a->q_stride_n; P.q_sh = a->q_stride_h; P.k_sn = a->k_stride_n; P.k_sh = a->k_stride_h;
    P.v_sn = a->v_stride_n; P.v_sh = a->v_stride_h;
    P.qo_sn = a->q_out_stride_n; P.qo_sh = a->q_out_stride_h; P.ko_sn = a->k_out_stride_n; P.ko_sh = a->k_out_stride_h;
    P.c_sblk = a->cache_stride_blk; P.c_sh = a->cache_stride_h; P.c_spos = a->cache_stride_pos; P.t_s = a->table_stride;
    if (q8) { P.c_spos = D; P.c_sh = a->block_size * D; P.c_sblk = a->num_kv_heads * P.c_sh; }
    P.n_tokens = a->n_tokens; P.num_slots = a->num_blocks * a->block_size; P.table_rows = a->table_rows;
    P.hq = (int)a->num_q_heads; P.hkv = (int)a->num_kv_heads; P.D = D; P.block_size = (int)a->block_size;
    P.eps = a->eps; P.inv_d = 1.f / (float)D;

    // 16-byte vectors where every row they touch starts on a 16-byte boundary and half a head divides
    // into them, else single elements.
    bool wide = half % vmax == 0;
    auto fits = [&](const void* p, size_t align) { wide = wide && ((uintptr_t)p % align) == 0; };
    auto fits_stride = [&](int64_t s, size_t size, size_t align) { wide = wide && ((size_t)s * size) % align == 0; };
    if (P.hq) {
        fits(P.q, 16); fits(P.q_out, 16);
        fits_stride(P.q_sn, e, 16); fits_stride(P.q_sh, e, 16); fits_stride(P.qo_sn, e, 16); fits_stride(P.qo_sh, e, 16);
    }
    if (P.hkv) { fits(P.k, 16); fits_stride(P.k_sn, e, 16); fits_stride(P.k_sh, e, 16); }
    if (!append && P.hkv) { fits(P.k_out, 16); fits_stride(P.ko_sn, e, 16); fits_stride(P.ko_sh, e, 16); }
    if (append) {
        fits(P.v, 16); fits_stride(P.v_sn, e, 16); fits_stride(P.v_sh, e, 16);
        const size_t ce = q8 ? 1 : e, ca = q8 ? (size_t)vmax : 16;
        fits(P.k_cache, ca); fits(P.v_cache, ca);
        fits_stride(P.c_sblk, ce, ca); fits_stride(P.c_sh, ce, ca); fits_stride(P.c_spos, ce, ca);
    }
    fits(P.cos, 16); fits(P.sin, 16); fits_stride(P.t_s, te, 16);
    fits(P.wq, 16); fits(P.wk, 16);

    const int pieces = wide ? half / vmax : half;
    const int np = pieces <= 32 ? 1 : (wide ? 2 : 8);  // 512 / 2 elements: 64 fp32 vectors, 256 single elements
    int lanes = 1;
    while (lanes < 32 && lanes < pieces) lanes *= 2;
    P.lanes = lanes;
    const int rows = P.hq + (append ? 2 : 1) * P.hkv;
    const int64_t trips = ceil_div<int64_t>(rows, 32 / lanes);  // a warp's passes over the rows of a token
    // One warp per token reads the table once but is a long chain of loads; a warp for every pass reads it
    // `trips` times (from L1 or L2). Small batches want the warps.
    int64_t splits = trips;
    P.splits = (int)splits;
    const int64_t blocks = ceil_div<int64_t>(P.n_tokens * splits * 32, 256);
    RFX_REQUIRE(blocks < (1ll << 31), "%s: too many tokens (%lld)", name, (long long)a->n_tokens);
    cudaStream_t stream = as_stream(a->stream);
    const int mode = append ? (q8 ? kPool8 : kPool) : kDense;
    cudaError_t le = cudaSuccess;
#define RFX_QKN(T, TT, V, NP, II, MM) \
    le = launch_pdl(qk_norm_rope_kernel<T, TT, V, NP, II, MM>, dim3((unsigned)blocks), dim3(256), 0, stream, P)
#define RFX_QKN_MODE(T, TT, V, NP, II)                                   \
    do {                                                                 \
        if (mode == kDense) RFX_QKN(T, TT, V, NP, II, kDense);           \
        else if (mode == kPool) RFX_QKN(T, TT, V, NP, II, kPool);        \
        else RFX_QKN(T, TT, V, NP, II, kPool8);                          \
    } while (0)
#define RFX_QKN_V(T, TT, II)                                                            \
    do {                                                                                \
        constexpr int VM = 16 / (int)sizeof(T);                                         \
        if (wide && np == 1) RFX_QKN_MODE(T, TT, VM, 1, II);                            \
        else if (wide) RFX_QKN_MODE(T, TT, VM, (sizeof(T) == 4 ? 2 : 1), II);           \
        else if (np == 1) RFX_QKN_MODE(T, TT, 1, 1, II);                                \
        else RFX_QKN_MODE(T, TT, 1, 8, II);                                             \
    } while (0)
    RFX_DISPATCH_DTYPE(a->dtype, T, {
        if (a->tables_f32) { if (inter) RFX_QKN_V(T, float, true); else RFX_QKN_V(T, float, false); }
        else { if (inter) RFX_QKN_V(T, T, true); else RFX_QKN_V(T, T, false); }
    });
#undef RFX_QKN_V
#undef RFX_QKN_MODE
#undef RFX_QKN
    if (le != cudaSuccess) { cudaGetLastError(); return fail(RFX_CUDA_ERROR, "%s: %s", name, cudaGetErrorString(le)); }
    return check_launch(name);
}

}  // namespace
}  // namespace rfx

extern "C" int rfx_qk_norm_rope(const RfxQkNormRopeArgs* a) { return rfx::qk_norm_impl(a, false, "rfx_qk_norm_rope"); }

extern "C" int rfx_qk_norm_rope_append(const RfxQkNormRopeArgs* a) {
    return rfx::qk_norm_impl(a, true, "rfx_qk_norm_rope_append");
}
