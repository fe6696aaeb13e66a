// C entry of the attention over a latent cache: argument checks, kernel selection and launch.  See include/intfa.h.
#include "intfa_latent_host.h"
#include "intfa_latent_expanded_host.h"

using namespace intfa;

namespace {

bool rows16(const void* p, int64_t a, int64_t b, int64_t c) { return aligned_to(p, 16) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }

int check(const intfa_latent_attn_params* p) {
    if (p == nullptr || p->q_latent == nullptr || p->q_rope == nullptr || p->out == nullptr || p->seqlens_k == nullptr) return INTFA_ERR_NULL;
    const int rc = latent_cache_check(&p->cache);
    if (rc != INTFA_OK) return rc;
    if (p->batch <= 0 || p->heads <= 0) return INTFA_ERR_SHAPE;
    if (p->seqlen <= 0) return INTFA_ERR_SEQLEN;
    if (p->dtype != INTFA_F16 && p->dtype != INTFA_BF16) return INTFA_ERR_DTYPE;
    if (p->rope.freqs != nullptr && !rope_valid(&p->rope, p->cache.rope_dim)) return INTFA_ERR_ROPE;
    if (!rows16(p->q_latent, p->ql_stride_b, p->ql_stride_h, p->ql_stride_n) || !rows16(p->q_rope, p->qr_stride_b, p->qr_stride_h, p->qr_stride_n) ||
        !rows16(p->out, p->o_stride_b, p->o_stride_h, p->o_stride_n) || !aligned_to(p->lse, 4) || !aligned_to(p->seqlens_k, 4) || !aligned_to(p->seqlens_q, 4) ||
        !aligned_to(p->rope.freqs, 8)) return INTFA_ERR_ALIGN;
    if (size_product((int64_t)p->batch * p->heads, p->seqlen) >= 1ll << 30) return INTFA_ERR_SHAPE;
    return INTFA_OK;
}

// How a call is dealt: rows of a tile, keys of a unit, workgroups (one a compute unit: the ring of stages takes its LDS); and the layout of its workspace.
struct Plan { int rows, tiles, unit_log2, lead, grid; size_t stats_at, items_at, bytes; };
Plan make_plan(const intfa_latent_attn_params* p) {
    Plan a{};
    const int rows = p->heads * p->seqlen;
    const int64_t keys = (int64_t)p->cache.table_width * p->cache.page_size;
    // Tiles of 64 rows take a block of keys in 1.6 times the time of 32 rows, and twice as long until their first and from their last one: with few blocks a compute unit tiles of 32 are
    // faster (128 heads of one request over 8192 tokens 35 -> 27 us, 64 heads of 16 over 2048 34 -> 28; 128 heads of 32 over 2048, eight blocks a unit, 48 both; over 4096 65 -> 75).
    // (The keys that the table has room for; the lengths are on the device.)
    a.rows = rows <= 32 || size_product((int64_t)p->batch * ((rows + 63) / 64), (keys + 63) / 64) <= 8 * kComputeUnits ? 32 : 64;
    a.tiles = (rows + a.rows - 1) / a.rows;
    a.lead = 2;
    a.unit_log2 = 6;
    const int64_t items = (int64_t)p->batch * a.tiles;
    auto units = [&] { return items * (a.lead + ((keys + (1ll << a.unit_log2) - 1) >> a.unit_log2)); };
    a.grid = (int)(units() < kComputeUnits ? units() : kComputeUnits);
    while (units() * a.grid >= 1ll << 32 && a.unit_log2 < 30) ++a.unit_log2;      // (units are numbered in 32 bits, times the workgroups)
    if (units() * a.grid >= 1ll << 32) a.grid = (int)(((1ll << 32) - 1) / units());
    const size_t slot_rows = (size_t)a.grid * 2 * a.rows;
    a.stats_at = slot_rows * p->cache.latent_dim * sizeof(float);
    a.items_at = a.stats_at + slot_rows * 2 * sizeof(float);
    a.bytes = a.items_at + (size_t)a.grid * 16;
    return a;
}

}  // namespace

extern "C" {

size_t intfa_latent_attn_workspace_bytes(const intfa_latent_attn_params* p) { return check(p) == INTFA_OK ? make_plan(p).bytes : 0; }

int intfa_latent_attn_int8(const intfa_latent_attn_params* p, void* stream) {
    const int rc = check(p);
    if (rc != INTFA_OK) return rc;
    const intfa_latent_cache& c = p->cache;
    const Plan a = make_plan(p);
    if (p->workspace == nullptr || p->workspace_bytes < a.bytes || !aligned_to(p->workspace, 16)) return INTFA_ERR_WORKSPACE;
    LatentParams lp{};
    PagedParams& kp = lp.deal;
    kp.q = (const char*)p->q_latent; kp.out = (char*)p->out; kp.lse = p->lse;
    kp.k = (const char*)c.rows; kp.k_scale = c.scale;
    kp.table = c.block_table; kp.seqlens_k = p->seqlens_k; kp.seqlens_q = p->seqlens_q;
    kp.q_sb = p->ql_stride_b * 2; kp.q_sh = p->ql_stride_h * 2; kp.q_sn = p->ql_stride_n * 2;
    kp.o_sb = p->o_stride_b * 2; kp.o_sh = p->o_stride_h * 2; kp.o_sn = p->o_stride_n * 2;
    kp.k_sp = c.r_stride_p; kp.k_sn = (int)c.r_stride_n; kp.ks_sp = c.s_stride_p; kp.ks_sh = c.s_stride_n; kp.bt_sb = c.bt_stride_b;
    kp.batch = p->batch; kp.heads = p->heads; kp.heads_kv = 1; kp.group = p->heads;
    kp.seqlen = p->seqlen; kp.rows = p->heads * p->seqlen;
    kp.page_log2 = __builtin_ctz((unsigned)c.page_size); kp.num_pages = c.num_pages; kp.table_width = c.table_width;
    kp.causal = p->causal != 0;
    kp.qk_scale_log2 = p->sm_scale * 1.4426950408889634f;
    kp.rope = {p->rope.freqs, p->rope.pairs, p->rope.interleaved, p->rope.magnitude};
    kp.tiles = a.tiles; kp.unit_log2 = a.unit_log2; kp.grid = a.grid; kp.lead = a.lead;
    kp.parts = (float*)p->workspace;
    kp.part_stats = (float*)((char*)p->workspace + a.stats_at);
    kp.d_group = make_fast_div(kp.group); kp.d_tiles = make_fast_div(kp.tiles); kp.d_pairs = make_fast_div(kp.rope.freqs != nullptr ? kp.rope.pairs : 1);
    lp.q_rope = (const char*)p->q_rope; lp.qr_sb = p->qr_stride_b * 2; lp.qr_sh = p->qr_stride_h * 2; lp.qr_sn = p->qr_stride_n * 2;
    lp.open_items = (v4i*)((char*)p->workspace + a.items_at);
    hipStream_t st = (hipStream_t)stream;
#define INTFA_CALL(name) (p->dtype == INTFA_BF16 ? name##_bf16(lp, a.rows, st) : name##_f16(lp, a.rows, st))
    if (c.latent_dim == 128) return c.rope_dim == 32 ? INTFA_CALL(launch_latent_c128_r32) : INTFA_CALL(launch_latent_c128_r64);
    if (c.latent_dim == 256) return c.rope_dim == 32 ? INTFA_CALL(launch_latent_c256_r32) : INTFA_CALL(launch_latent_c256_r64);
    return c.rope_dim == 32 ? INTFA_CALL(launch_latent_c512_r32) : INTFA_CALL(launch_latent_c512_r64);
#undef INTFA_CALL
}

int intfa_latent_expanded(const intfa_latent_expanded_params* p, void* stream) {
    if (p == nullptr || p->q_nope == nullptr || p->q_rope == nullptr || p->k_nope == nullptr || p->k_rope == nullptr || p->v == nullptr || p->out == nullptr)
        return INTFA_ERR_NULL;
    if (p->batch <= 0 || p->heads <= 0) return INTFA_ERR_SHAPE;
    if (p->seqlen <= 0 || p->seqlen_k < 0) return INTFA_ERR_SEQLEN;
    const bool wide = p->nope_dim == 128 && p->rope_dim == 64 && p->v_dim == 128;
    if (!wide && !(p->nope_dim == 64 && p->rope_dim == 32 && p->v_dim == 64)) return INTFA_ERR_HEAD_DIM;
    if (p->dtype != INTFA_F16 && p->dtype != INTFA_BF16) return INTFA_ERR_DTYPE;
    if (!rows16(p->q_nope, p->qn_stride_b, p->qn_stride_h, p->qn_stride_n) || !rows16(p->q_rope, p->qr_stride_b, p->qr_stride_h, p->qr_stride_n) ||
        !rows16(p->k_nope, p->kn_stride_b, p->kn_stride_h, p->kn_stride_n) || !rows16(p->k_rope, p->kr_stride_b, 0, p->kr_stride_n) ||
        !rows16(p->v, p->v_stride_b, p->v_stride_h, p->v_stride_n) || !rows16(p->out, p->o_stride_b, p->o_stride_h, p->o_stride_n) || !aligned_to(p->lse, 4) ||
        !aligned_to(p->seqlens_q, 4) || !aligned_to(p->seqlens_k, 4)) return INTFA_ERR_ALIGN;
    // a block of 128 keys spans less than 2^32 bytes
    auto fits = [&](int64_t row, int64_t dim) { return row >= dim && row < 1 << 24; };
    if (!fits(p->kn_stride_n, p->nope_dim) || !fits(p->kr_stride_n, p->rope_dim) || !fits(p->v_stride_n, p->v_dim)) return INTFA_ERR_SHAPE;
    if (p->seqlen > 1 << 30 || p->seqlen_k >= 1 << 25) return INTFA_ERR_SHAPE;
    ExpandedParams ep{};
    // those of a (sequence, head) together, and of the block behind the last one, may span more
    auto far = [&](int64_t row) { return size_product((int64_t)p->seqlen_k + 128, row) >= 1ll << 31; };
    ep.far = far(p->kn_stride_n) || far(p->kr_stride_n) || far(p->v_stride_n);
    ep.tiles = (p->seqlen + 127) / 128;
    const int64_t units = size_product(p->batch, p->heads);
    ep.split = size_product(units, ep.tiles) <= kComputeUnits;
    ep.pairs = ep.split ? ep.tiles : (ep.tiles + 1) / 2;
    const int64_t groups = size_product(units, ep.pairs);
    if (groups * 512 >= 1ll << 32 || groups >= 1ll << 31) return INTFA_ERR_SHAPE;
    ep.qn = (const char*)p->q_nope; ep.qr = (const char*)p->q_rope; ep.kn = (const char*)p->k_nope; ep.kr = (const char*)p->k_rope; ep.v = (const char*)p->v;
    ep.out = (char*)p->out; ep.lse = p->lse; ep.seqlens_q = p->seqlens_q; ep.seqlens_k = p->seqlens_k;
    ep.qn_sb = p->qn_stride_b * 2; ep.qn_sh = p->qn_stride_h * 2; ep.qn_sn = p->qn_stride_n * 2;
    ep.qr_sb = p->qr_stride_b * 2; ep.qr_sh = p->qr_stride_h * 2; ep.qr_sn = p->qr_stride_n * 2;
    ep.kn_sb = p->kn_stride_b * 2; ep.kn_sh = p->kn_stride_h * 2; ep.kn_sn = (uint32_t)(p->kn_stride_n * 2);
    ep.kr_sb = p->kr_stride_b * 2; ep.kr_sn = (uint32_t)(p->kr_stride_n * 2);
    ep.v_sb = p->v_stride_b * 2; ep.v_sh = p->v_stride_h * 2; ep.v_sn = (uint32_t)(p->v_stride_n * 2);
    ep.o_sb = p->o_stride_b * 2; ep.o_sh = p->o_stride_h * 2; ep.o_sn = p->o_stride_n * 2;
    ep.batch = p->batch; ep.heads = p->heads; ep.seqlen = p->seqlen; ep.seqlen_k = p->seqlen_k;
    ep.whole = (int)(units / kXcds) * kXcds * ep.pairs;
    ep.qk_scale_log2 = p->sm_scale * 1.4426950408889634f;
    ep.d_pairs = make_fast_div(ep.pairs); ep.d_heads = make_fast_div(p->heads);
    hipStream_t st = (hipStream_t)stream;
    const bool causal = p->causal != 0;
    if (wide) return p->dtype == INTFA_BF16 ? launch_expanded_n128_bf16(ep, causal, st) : launch_expanded_n128_f16(ep, causal, st);
    return p->dtype == INTFA_BF16 ? launch_expanded_n64_bf16(ep, causal, st) : launch_expanded_n64_f16(ep, causal, st);
}

}  // extern "C"
