// Entry points of the norm + rotation of query and key heads: checks, the choice of the kernel, the launch.
#include "qk_norm.cuh"

namespace rfx {
namespace qkn {

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
    const int groups = 32 / lanes;  // rows of a warp's pass; a pass is of queries, keys or values
    const int64_t trips = ceil_div(P.hq, groups) + (append ? 2 : 1) * ceil_div(P.hkv, groups);
    // A warp takes several passes of a token, so that the table row, the slot and the weights are looked up once for them, as
    // long as there are ten warps an SM (2047 tokens of 28 / 4 heads: 7.6 us, with twice the warps 9.3; 256 tokens of 64 / 8: 4.2,
    // with half of them 5.6).
    int64_t splits = ceil_div<int64_t>((int64_t)sm_count() * 10, P.n_tokens);
    if (splits > trips) splits = trips;
    P.splits = (int)splits;
    const int64_t blocks = ceil_div<int64_t>(P.n_tokens * splits * 32, 256);
    RFX_REQUIRE(blocks < (1ll << 31), "%s: too many tokens (%lld)", name, (long long)a->n_tokens);
    cudaStream_t stream = as_stream(a->stream);
    const int mode = append ? (q8 ? kPool8 : kPool) : kDense;
    const Shape shape = {wide, pieces, np, a->tables_f32 || a->dtype == RFX_F32, inter, mode, (unsigned)blocks};
    cudaError_t le;
    if (a->dtype == RFX_F32) le = launch_f32(P, shape, stream);
    else if (a->dtype == RFX_BF16) le = launch_bf16(P, shape, stream);
    else le = launch_f16(P, shape, stream);
    if (le != cudaSuccess) { cudaGetLastError(); return fail(RFX_CUDA_ERROR, "%s: %s", name, cudaGetErrorString(le)); }
    return check_launch(name);
}

}  // namespace qkn
}  // namespace rfx

extern "C" int rfx_qk_norm_rope(const RfxQkNormRopeArgs* a) { return rfx::qkn::qk_norm_impl(a, false, "rfx_qk_norm_rope"); }

extern "C" int rfx_qk_norm_rope_append(const RfxQkNormRopeArgs* a) {
    return rfx::qkn::qk_norm_impl(a, true, "rfx_qk_norm_rope_append");
}
