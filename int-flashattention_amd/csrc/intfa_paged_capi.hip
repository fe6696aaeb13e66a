// C entry of the attention over a paged int8 cache: argument checks, kernel selection and launch.  See include/intfa.h.
#include "intfa_paged_host.h"

using namespace intfa;

namespace {

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) == 0; }
bool rows16(const void* p, int64_t a, int64_t b, int64_t c) { return aligned(p, 16) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }

int check(const intfa_paged_attn_params* p) {
    if (p == nullptr || p->q == nullptr || p->out == nullptr || p->seqlens_k == nullptr) return INTFA_ERR_NULL;
    const intfa_paged_cache& c = p->cache;
    const int rc = paged_cache_check(&c);
    if (rc != INTFA_OK) return rc;
    if (p->batch <= 0 || p->heads <= 0 || p->heads % c.heads_kv != 0) return INTFA_ERR_SHAPE;
    if (p->seqlen <= 0) return INTFA_ERR_SEQLEN;
    if (p->dtype != INTFA_F16 && p->dtype != INTFA_BF16) return INTFA_ERR_DTYPE;
    if (p->rope.freqs != nullptr && !rope_valid(&p->rope, c.head_dim)) return INTFA_ERR_ROPE;
    if (!rows16(p->q, p->q_stride_b, p->q_stride_h, p->q_stride_n) || !rows16(p->out, p->o_stride_b, p->o_stride_h, p->o_stride_n) ||
        !aligned(p->lse, 4) || !aligned(p->seqlens_k, 4) || !aligned(p->seqlens_q, 4) || !aligned(p->rope.freqs, 8)) return INTFA_ERR_ALIGN;
    if ((int64_t)p->batch * p->heads * p->seqlen >= 1ll << 30) return INTFA_ERR_SHAPE;
    return INTFA_OK;
}

}  // namespace

extern "C" {

size_t intfa_paged_attn_workspace_bytes(const intfa_paged_attn_params* p) { return 0; }

int intfa_paged_attn_int8(const intfa_paged_attn_params* p, void* stream) {
    const int rc = check(p);
    if (rc != INTFA_OK) return rc;
    const intfa_paged_cache& c = p->cache;
    PagedParams kp{};
    kp.q = (const char*)p->q; kp.out = (char*)p->out; kp.lse = p->lse;
    kp.k = (const char*)c.k; kp.v = (const char*)c.v; kp.k_scale = c.k_scale; kp.v_scale = c.v_scale;
    kp.table = c.block_table; kp.seqlens_k = p->seqlens_k; kp.seqlens_q = p->seqlens_q;
    kp.q_sb = p->q_stride_b * 2; kp.q_sh = p->q_stride_h * 2; kp.q_sn = p->q_stride_n * 2;
    kp.o_sb = p->o_stride_b * 2; kp.o_sh = p->o_stride_h * 2; kp.o_sn = p->o_stride_n * 2;
    kp.k_sp = c.k_stride_p; kp.k_sh = c.k_stride_h; kp.v_sp = c.v_stride_p; kp.v_sh = c.v_stride_h;
    kp.ks_sp = c.ks_stride_p; kp.ks_sh = c.ks_stride_h; kp.vs_sp = c.vs_stride_p; kp.vs_sh = c.vs_stride_h; kp.bt_sb = c.bt_stride_b;
    kp.k_sn = (int)c.k_stride_n; kp.v_sn = (int)c.v_stride_n;
    kp.batch = p->batch; kp.heads = p->heads; kp.heads_kv = c.heads_kv; kp.group = p->heads / c.heads_kv;
    kp.seqlen = p->seqlen; kp.rows = kp.group * p->seqlen;
    kp.page_log2 = __builtin_ctz((unsigned)c.page_size); kp.num_pages = c.num_pages; kp.table_width = c.table_width;
    kp.causal = p->causal != 0;
    kp.qk_scale_log2 = p->sm_scale * 1.4426950408889634f;
    kp.rope = {p->rope.freqs, p->rope.pairs, p->rope.interleaved, p->rope.magnitude};
    PagedSel sel{c.head_dim, p->dtype == INTFA_BF16 ? 1 : 0, kp.rows <= 16 ? 1 : 2};
    kp.tiles = (kp.rows + 16 * sel.row_tiles - 1) / (16 * sel.row_tiles);
    kp.d_group = make_fast_div(kp.group); kp.d_tiles = make_fast_div(kp.tiles); kp.d_heads_kv = make_fast_div(kp.heads_kv);
    hipStream_t st = (hipStream_t)stream;
    return c.head_dim == 64 ? launch_paged_d64(kp, sel, st) : c.head_dim == 128 ? launch_paged_d128(kp, sel, st) : launch_paged_d256(kp, sel, st);
}

}  // extern "C"
