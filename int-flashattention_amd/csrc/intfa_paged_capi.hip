// C entry of the attention over a paged int8 cache: argument checks, kernel selection and launch.  See include/intfa.h.
#include "intfa_paged_host.h"
#include "intfa_splitkv.h"

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
    if (size_product((int64_t)p->batch * p->heads, p->seqlen) >= 1ll << 30) return INTFA_ERR_SHAPE;
    return INTFA_OK;
}

// How a call is dealt: rows per tile, keys per unit, workgroups; and the layout of its workspace.
struct Plan { PagedSel sel; int rows, tiles, unit_log2, lead, grid, slot_rows; size_t stats_at, tickets_at, bytes; };
Plan make_plan(const intfa_paged_attn_params* p) {
    const intfa_paged_cache& c = p->cache;
    Plan a{};
    a.rows = p->heads / c.heads_kv * p->seqlen;
    // Rows of 16 x 8 heads over 8192 keys, us, as tiles of 32 in the decode kernel / in the one for many rows: 64 rows d64 68 / 68, d128 92 / 151, d256 210 / 315;
    // 72 rows 108 / 68, 155 / 151, 360 / 315; 128 rows 133 / 70, 184 / 156, 416 / 319.  Rotated fp16 queries take a second product there (PagedQueries::stage), which
    // puts head_dim 128 behind until 128 rows (72 rows 172 / 204, 128 rows 205 / 209, 160 rows 290 / 215) and has no room in head_dim 256's registers: those
    // stay in tiles of 32 (2 x 512 tokens of 32 heads over 7680 keys 975 us, there 1512 with 740 registers spilled).
    const bool two_products = p->dtype == INTFA_F16 && p->rope.freqs != nullptr;
    const bool prefill = a.rows > (two_products && c.head_dim == 128 ? 128 : 64) && !(two_products && c.head_dim == 256);
    a.sel = {c.head_dim, p->dtype == INTFA_BF16 ? 1 : 0, prefill ? 0 : a.rows <= 16 ? 1 : 2, c.page_size >= (!prefill && c.head_dim == 256 ? 32 : 64)};
    a.slot_rows = prefill ? paged_prefill_rows(c.head_dim) : 16 * a.sel.row_tiles;
    a.tiles = (a.rows + a.slot_rows - 1) / a.slot_rows;
    // (many rows, units of 256 keys with a lead of two -> of 64 with a lead of four, which is what beginning a part takes: two ragged chunks of 512 122.0 -> 118.4 us,
    // sixteen chunks of 512 tokens of which fifteen have three 207 -> 172, a prompt of 2048 73.9 -> 72.8; a lead of three 121.2, 170, 77.5, of five 119.6, 177, 70.8)
    a.lead = prefill ? 4 : 2;
    a.unit_log2 = prefill ? 6 : c.head_dim == 256 ? 7 : 8;
    const int64_t items = (int64_t)p->batch * c.heads_kv * a.tiles, keys = (int64_t)c.table_width * c.page_size;
    const int slots = kComputeUnits * (prefill ? paged_prefill_wgs(c.head_dim) : c.head_dim == 256 || a.sel.row_tiles > 1 ? 1 : 2);
    auto units = [&] { return items * (a.lead + ((keys + (1ll << a.unit_log2) - 1) >> a.unit_log2)); };
    a.grid = (int)(units() < slots ? units() : slots);
    while (units() * a.grid >= 1ll << 32 && a.unit_log2 < 30) ++a.unit_log2;      // (units are numbered in 32 bits, times the workgroups)
    if (units() * a.grid >= 1ll << 32) a.grid = (int)(((1ll << 32) - 1) / units());
    const size_t slot_rows = (size_t)a.grid * 2 * a.slot_rows;
    a.stats_at = slot_rows * c.head_dim * sizeof(float);
    a.tickets_at = a.stats_at + slot_rows * 2 * sizeof(float);
    a.bytes = a.tickets_at + (size_t)items * kTicketStride * sizeof(uint64_t);
    return a;
}

}  // namespace

extern "C" {

size_t intfa_paged_attn_workspace_bytes(const intfa_paged_attn_params* p) { return check(p) == INTFA_OK ? make_plan(p).bytes : 0; }

int intfa_paged_attn_int8(const intfa_paged_attn_params* p, void* stream) {
    const int rc = check(p);
    if (rc != INTFA_OK) return rc;
    const intfa_paged_cache& c = p->cache;
    const Plan a = make_plan(p);
    if (p->workspace == nullptr || p->workspace_bytes < a.bytes || !aligned(p->workspace, 16)) return INTFA_ERR_WORKSPACE;
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
    kp.tiles = a.tiles; kp.unit_log2 = a.unit_log2; kp.grid = a.grid; kp.lead = a.lead;
    kp.parts = (float*)p->workspace;
    kp.part_stats = (float*)((char*)p->workspace + a.stats_at);
    kp.ticket = (uint64_t*)((char*)p->workspace + a.tickets_at);
    kp.epoch = next_epoch() << 8;
    kp.d_group = make_fast_div(kp.group); kp.d_tiles = make_fast_div(kp.tiles); kp.d_pairs = make_fast_div(kp.rope.freqs != nullptr ? kp.rope.pairs : 1);
    const PagedSel& sel = a.sel;
    hipStream_t st = (hipStream_t)stream;
    if (sel.row_tiles == 0)
        return c.head_dim == 64 ? launch_paged_prefill_d64(kp, sel, st) : c.head_dim == 128 ? launch_paged_prefill_d128(kp, sel, st) : launch_paged_prefill_d256(kp, sel, st);
    return c.head_dim == 64 ? launch_paged_d64(kp, sel, st) : c.head_dim == 128 ? launch_paged_d128(kp, sel, st) : launch_paged_d256(kp, sel, st);
}

}  // extern "C"
