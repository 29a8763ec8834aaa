// RMS norm of every query and key head with the position rotation in the same pass, to dense rows or
// (with V) straight into the paged pool:
//   r = 1 / sqrt(mean_d x_d^2 + eps),  n_d = x_d * r * w_d,
//   y_i = n_i c_i - n_j s_i,  y_j = n_i s_i + n_j c_i   for the pairs (i, j = i + D/2) or (2i, 2i + 1).
// Everything is fp32 and the result is rounded once (rope.cu rounds every step, because the reference's
// rotation does; there is no such composition to match bit for bit here).
//
// Algorithmic bytes: 2*N*(H_q + 2*H_kv)*D*e plus a table row per token; about 7 fp32 operations per
// element, so HBM-bound at every size that is not bound by the launch.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace rfx {
namespace qkn {

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

constexpr int kAhead = 4;  // passes under way and at work; two: 76 us where four take 68 (16384 tokens of 32 / 8 heads of 128)

template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };

// V elements as they lie in memory, at most 16 bytes an access.
template <typename T, int V> __device__ __forceinline__ void load_f(const T* p, float (&f)[V]) {
    constexpr int W = 16 / (int)sizeof(T) < V ? 16 / (int)sizeof(T) : V;
#pragma unroll
    for (int o = 0; o < V; o += W) {
        const Vec<T, W> x = *reinterpret_cast<const Vec<T, W>*>(p + o);
#pragma unroll
        for (int j = 0; j < W; ++j) f[o + j] = Num<T>::to_f(x.v[j]);
    }
}
template <typename T, int V> __device__ __forceinline__ void store_f(T* p, const float (&f)[V]) {
    Vec<T, V> x;
    if constexpr (sizeof(T) == 2 && V >= 2) {
        using W = typename Pair16<T>::P;
#pragma unroll
        for (int j = 0; j < V; j += 2) reinterpret_cast<W*>(x.v)[j / 2] = Pair16<T>::round(f[j], f[j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x.v[j] = Num<T>::from_f(f[j]);
    }
    *reinterpret_cast<Vec<T, V>*>(p) = x;
}
template <int V> __device__ __forceinline__ void store_q8(int8_t* p, const float (&f)[V], float scale) {
    Vec<int8_t, V> x;
#pragma unroll
    for (int j = 0; j < V; ++j) x.v[j] = (int8_t)fminf(127.f, fmaxf(-127.f, rintf(__fdiv_rn(f[j], scale))));
    *reinterpret_cast<Vec<int8_t, V>*>(p) = x;
}

// A piece of a row: the V pairs (a_j, b_j). In memory they are two V-vectors: the a's and, D/2 further on, the b's; or
// (INTER) 2V neighbours a_0 b_0 a_1 b_1 ...
template <typename T, int V, bool INTER> __device__ __forceinline__ void load_pairs(const T* p1, const T* p2, float (&a)[V], float (&b)[V]) {
    load_f<T, V>(p1, a);
    load_f<T, V>(p2, b);
    if constexpr (INTER && V > 1) {
        float z[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) { z[j] = a[j]; z[V + j] = b[j]; }
#pragma unroll
        for (int j = 0; j < V; ++j) { a[j] = z[2 * j]; b[j] = z[2 * j + 1]; }
    }
}
// Back to memory's order.
template <int V, bool INTER> __device__ __forceinline__ void order(float (&a)[V], float (&b)[V]) {
    if constexpr (INTER && V > 1) {
        float z[2 * V];
#pragma unroll
        for (int j = 0; j < V; ++j) { z[2 * j] = a[j]; z[2 * j + 1] = b[j]; }
#pragma unroll
        for (int j = 0; j < V; ++j) { a[j] = z[j]; b[j] = z[V + j]; }
    }
}

// x * y + z (or - z), two lanes an instruction where V allows.
template <int V> __device__ __forceinline__ void fma_v(const float (&x)[V], const float (&y)[V], float (&z)[V]) {
    if constexpr (V >= 2) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const float2 r = __ffma2_rn(make_float2(x[j], x[j + 1]), make_float2(y[j], y[j + 1]), make_float2(z[j], z[j + 1]));
            z[j] = r.x; z[j + 1] = r.y;
        }
    } else {
        z[0] = fmaf(x[0], y[0], z[0]);
    }
}
template <int V> __device__ __forceinline__ void mul_v(const float (&x)[V], const float (&y)[V], float (&z)[V]) {
    if constexpr (V >= 2) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const float2 r = __fmul2_rn(make_float2(x[j], x[j + 1]), make_float2(y[j], y[j + 1]));
            z[j] = r.x; z[j + 1] = r.y;
        }
    } else {
        z[0] = x[0] * y[0];
    }
}

// A row is cut into pieces of V pairs. `lanes` lanes take a row (NP pieces each), a warp 32/lanes rows at a time; the sum of
// squares needs no shared memory. A lane keeps its piece for every row of its token, so it holds the four factors of the rotation
// with the norm's weight in them,
//   y_i = r (x_i (w_i c_i) - x_j (w_j s_i)),  y_j = r (x_i (w_i s_i) + x_j (w_j c_i)),
// and makes them once for the query rows and once for the key rows it passes. Two fp32 lanes an instruction. (With the
// weights loaded and every product on its own for each row the kernel was bound by its instructions: 300 a pass, 85 us
// for 16384 tokens of 32 / 8 heads of 128.)
// LANES: the lanes of a row where a row is exactly that many pieces, 0 where lanes stay idle or take several.
template <typename T, typename TT, int V, int NP, int LANES, bool INTER, int MODE>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkNormParams P) {
    ptx::pdl_wait();
    ptx::pdl_trigger();  // behind the wait: what starts now finds everything ahead of this kernel complete
    const int lane = threadIdx.x & 31;
    const int64_t warp = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
    const int64_t n = warp / P.splits;
    if (n >= P.n_tokens) return;  // whole warps
    const int lanes = LANES ? LANES : P.lanes;
    const int sub = lane & (lanes - 1), group = lane / lanes, groups = 32 / lanes;
    const int half = LANES ? LANES * V : P.D >> 1;

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
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        const int p = sub + k * lanes;
        mine[k] = LANES || p * V < half;
        off1[k] = mine[k] ? (INTER ? 2 * V * p : V * p) : 0;
        off2[k] = off1[k] + (INTER ? V : half);
    }

    // Passes over the token: its query rows, its key rows, its value rows, `groups` rows each. A pass is of one kind. A
    // token without a table row has none, one without a slot only those of its queries.
    const int pq = (P.hq + groups - 1) / groups, pk = (P.hkv + groups - 1) / groups;
    const int passes = !known ? 0 : MODE == kDense ? pq + pk : at >= 0 ? pq + 2 * pk : pq;
    const int first = (int)(warp - n * P.splits);
    if (!known) {  // its dense rows become zero, or stay as they are where they are rotated in place
        float zero[V];
#pragma unroll
        for (int j = 0; j < V; ++j) zero[j] = 0.f;
        const int end = pq + (MODE == kDense ? pk : 0);
        for (int p = first; p < end; p += P.splits) {
            const bool is_q = p < pq;
            const int h = (is_q ? p : p - pq) * groups + group;
            if (h >= (is_q ? P.hq : P.hkv)) continue;
            const T* x = is_q ? (const T*)P.q + n * P.q_sn + h * P.q_sh : (const T*)P.k + n * P.k_sn + h * P.k_sh;
            T* y = is_q ? (T*)P.q_out + n * P.qo_sn + h * P.qo_sh : (T*)P.k_out + n * P.ko_sn + h * P.ko_sh;
            if (y == x) continue;
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if (!mine[k]) continue;
                store_f<T, V>(y + off1[k], zero);
                store_f<T, V>(y + off2[k], zero);
            }
        }
    }

    // w_i c, -w_j s, w_i s, w_j c; the table's factors stand at a pair's first element (its first half, its even entries)
    float f1[NP][V], f2[NP][V], f3[NP][V], f4[NP][V];
    auto factors = [&](const T* w) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            // (lanes behind the row's end take its first piece: their values go nowhere)
            const TT* cr = (const TT*)P.cos + pos * P.t_s + off1[k];
            const TT* sr = (const TT*)P.sin + pos * P.t_s + off1[k];
            float c[V], s[V], w1[V], w2[V];
            if constexpr (INTER) {
                float unused[V];
                load_pairs<TT, V, true>(cr, cr + V, c, unused);
                load_pairs<TT, V, true>(sr, sr + V, s, unused);
            } else {
                load_f<TT, V>(cr, c);
                load_f<TT, V>(sr, s);
            }
            load_pairs<T, V, INTER>(w + off1[k], w + off2[k], w1, w2);
            mul_v<V>(w1, c, f1[k]);
#pragma unroll
            for (int j = 0; j < V; ++j) f2[k][j] = -w2[j] * s[j];
            mul_v<V>(w1, s, f3[k]);
            mul_v<V>(w2, c, f4[k]);
        }
    };

    // Where a row lies, from pass to pass by an addition (64-bit products and the choice between the tensors for every
    // pass were half of the kernel's instructions); only the change from queries to keys to values looks it up anew.
    struct Cursor {
        int p, stop, h, limit;
        char* x;
        int64_t step;
    };
    const int h_step = P.splits * groups;
    auto set = [&](Cursor& c, auto* q, int64_t q_sh, auto* k, int64_t k_sh, auto* v, int64_t v_sh) {
        using E = std::remove_reference_t<decltype(*k)>;
        const bool is_q = c.p < pq, is_k = !is_q && c.p < pq + pk;
        c.stop = is_q ? pq : is_k ? pq + pk : 0x7fffffff;
        c.limit = is_q ? P.hq : P.hkv;
        c.h = (c.p - (is_q ? 0 : is_k ? pq : pq + pk)) * groups + group;
        const int64_t sh = is_q ? q_sh * (int64_t)sizeof(*q) : (is_k ? k_sh : v_sh) * (int64_t)sizeof(E);
        c.x = (is_q ? (char*)q : is_k ? (char*)k : (char*)v) + c.h * sh;
        c.step = h_step * sh;
    };
    const T* q_from = (const T*)P.q + n * P.q_sn;
    const T* k_from = (const T*)P.k + n * P.k_sn;
    const T* v_from = (const T*)P.v + n * P.v_sn;
    using Y = std::conditional_t<MODE == kPool8, int8_t, T>;
    T* q_to = (T*)P.q_out + n * P.qo_sn;
    Y* k_to = MODE == kDense ? (Y*)P.k_out + n * P.ko_sn : (Y*)P.k_cache + at;
    Y* v_to = (Y*)P.v_cache + at;
    const int64_t k_to_sh = MODE == kDense ? P.ko_sh : P.c_sh;
    auto set_from = [&](Cursor& c) { set(c, q_from, P.q_sh, k_from, P.k_sh, v_from, P.v_sh); };
    auto set_to = [&](Cursor& c) { set(c, q_to, P.qo_sh, k_to, k_to_sh, v_to, P.c_sh); };
    auto move = [&](Cursor& c) {
        c.p += P.splits;
        c.h += h_step;
        c.x += c.step;
        return c.p >= c.stop;
    };

    // Rows come through shared memory, kDepth - 1 passes ahead, every lane's own 16-byte words into its own place: bytes
    // under way without registers to hold them, and no barrier.
    constexpr bool kAsync = V * sizeof(T) == 16;
    constexpr int kDepth = !kAsync ? 1 : NP == 1 ? kAhead : kAhead / 2;
    __shared__ uint4 stage[kAsync ? kDepth * NP * 2 : 1][kAsync ? 256 : 1];
    Cursor from = {first}, to = {first};
    set_from(from);
    set_to(to);
    auto ahead = [&](int slot) {
        if constexpr (kAsync) {
            if (from.p < passes) {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    if (from.h >= from.limit || !mine[k]) continue;
                    ptx::cp_async16(&stage[(slot * NP + k) * 2][threadIdx.x], (const T*)from.x + off1[k]);
                    ptx::cp_async16(&stage[(slot * NP + k) * 2 + 1][threadIdx.x], (const T*)from.x + off2[k]);
                }
                if (move(from)) set_from(from);
            }
            ptx::cp_async_commit();
        }
    };
#pragma unroll
    for (int d = 0; d + 1 < kDepth; ++d) ahead(d);
    int made = 0, slot = 0;  // made: factors at hand, 1 for queries, 2 for keys
    while (to.p < passes) {
        const bool is_q = to.p < pq, is_v = MODE != kDense && to.p >= pq + pk;
        ahead(slot == 0 ? kDepth - 1 : slot - 1);
        if (!is_v && made != (is_q ? 1 : 2)) {
            made = is_q ? 1 : 2;
            factors((const T*)(is_q ? P.wq : P.wk));
        }
        if constexpr (kAsync) ptx::cp_async_wait<kDepth - 1>();
        const bool live = to.h < to.limit;
        float a[NP][V], b[NP][V];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            if constexpr (kAsync) {
                if (LANES || mine[k]) {  // what a lane without a row finds goes nowhere
                    load_pairs<T, V, INTER>((const T*)&stage[(slot * NP + k) * 2][threadIdx.x],
                                            (const T*)&stage[(slot * NP + k) * 2 + 1][threadIdx.x], a[k], b[k]);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) a[k][j] = b[k][j] = 0.f;
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) a[k][j] = b[k][j] = 0.f;
                if (live && mine[k]) load_pairs<T, V, INTER>((const T*)from.x + off1[k], (const T*)from.x + off2[k], a[k], b[k]);
            }
        }
        if (!kAsync && move(from)) set_from(from);
        slot = slot + 1 == kDepth ? 0 : slot + 1;
        if (!is_v) {
            float sq[V], sum = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) sq[j] = 0.f;
#pragma unroll
            for (int k = 0; k < NP; ++k) { fma_v<V>(a[k], a[k], sq); fma_v<V>(b[k], b[k], sq); }
#pragma unroll
            for (int j = 0; j < V; ++j) sum += sq[j];
#pragma unroll
            for (int o = (LANES ? LANES : 32) >> 1; o > 0; o >>= 1)
                if (LANES || o < lanes) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float r = rsqrtf(sum * P.inv_d + P.eps);
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                float u[V], t[V], rr[V];
#pragma unroll
                for (int j = 0; j < V; ++j) rr[j] = r;
                mul_v<V>(b[k], f2[k], u);
                fma_v<V>(a[k], f1[k], u);
                mul_v<V>(b[k], f4[k], t);
                fma_v<V>(a[k], f3[k], t);
                mul_v<V>(u, rr, a[k]);
                mul_v<V>(t, rr, b[k]);
            }
        }
        if (MODE == kPool8 && !is_q) {  // the row's scale: max |y| / 127 over its lanes (1 for a row of zeros)
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < NP; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (mine[k]) top = fmaxf(top, fmaxf(fabsf(a[k][j]), fabsf(b[k][j])));
#pragma unroll
            for (int o = (LANES ? LANES : 32) >> 1; o > 0; o >>= 1)
                if (LANES || o < lanes) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float scale = top > 0.f ? __fdiv_rn(top, 127.f) : 1.f;
            if (live && sub == 0) (is_v ? P.v_scales : P.k_scales)[scale_at + (int64_t)to.h * P.block_size] = scale;
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if (!live || !mine[k]) continue;
                order<V, INTER>(a[k], b[k]);
                store_q8<V>((int8_t*)to.x + off1[k], a[k], scale);
                store_q8<V>((int8_t*)to.x + off2[k], b[k], scale);
            }
        } else {
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if (!live || !mine[k]) continue;
                order<V, INTER>(a[k], b[k]);
                store_f<T, V>((T*)to.x + off1[k], a[k]);
                store_f<T, V>((T*)to.x + off2[k], b[k]);
            }
        }
        if (move(to)) set_to(to);
    }
}

// What the host has chosen for a launch.
struct Shape {
    bool wide;           // 16-byte vectors
    int pieces, np;      // of a row; of a lane
    bool tables_f32, inter;
    int mode;
    unsigned blocks;
};
cudaError_t launch_f32(const QkNormParams& P, const Shape& s, cudaStream_t stream);
cudaError_t launch_bf16(const QkNormParams& P, const Shape& s, cudaStream_t stream);
cudaError_t launch_f16(const QkNormParams& P, const Shape& s, cudaStream_t stream);

// The kernels of one type; each type has a file of its own, so that they compile side by side.
template <typename T, typename TT, bool INTER> cudaError_t launch_tables(const QkNormParams& P, const Shape& s, cudaStream_t stream) {
    constexpr int VM = 16 / (int)sizeof(T);
    auto go = [&](auto dense, auto pool, auto pool8) {
        return launch_pdl(s.mode == kDense ? dense : s.mode == kPool ? pool : pool8, dim3(s.blocks), dim3(256), 0, stream, P);
    };
#define RFX_QKN(V, NP, LANES)                                                                               \
    go(qk_norm_rope_kernel<T, TT, V, NP, LANES, INTER, kDense>, qk_norm_rope_kernel<T, TT, V, NP, LANES, INTER, kPool>, \
       qk_norm_rope_kernel<T, TT, V, NP, LANES, INTER, kPool8>)
    if (s.wide && s.pieces == 4) return RFX_QKN(VM, 1, 4);
    if (s.wide && s.pieces == 8) return RFX_QKN(VM, 1, 8);
    if (s.wide && s.np == 1) return RFX_QKN(VM, 1, 0);
    if constexpr (sizeof(T) == 4)
        if (s.wide) return RFX_QKN(VM, 2, 0);
    if (s.np == 1) return RFX_QKN(1, 1, 0);
    return RFX_QKN(1, 8, 0);
#undef RFX_QKN
}
template <typename T> cudaError_t launch_type(const QkNormParams& P, const Shape& s, cudaStream_t stream) {
    if (s.tables_f32) return s.inter ? launch_tables<T, float, true>(P, s, stream) : launch_tables<T, float, false>(P, s, stream);
    if constexpr (sizeof(T) == 2)
        return s.inter ? launch_tables<T, T, true>(P, s, stream) : launch_tables<T, T, false>(P, s, stream);
    return cudaErrorInvalidValue;  // fp32 tables are tables_f32
}

}  // namespace qkn
}  // namespace rfx
