// Host-side checks that the entry points of rotary positions and of the paged cache share, and the kernel-side block of the attention.
#pragma once
#include "../../include/intfa.h"
#include "intfa_launch.h"
#include "intfa_rope.h"

namespace intfa {

// a * b of sizes that are not negative, the largest number where it does not fit
inline int64_t size_product(int64_t a, int64_t b) {
    int64_t c;
    return __builtin_mul_overflow(a, b, &c) ? INT64_MAX : c;
}

inline bool rope_valid(const intfa_rope* r, int head_dim) {
    return r->pairs > 0 && r->pairs % 8 == 0 && 2 * (int64_t)r->pairs <= head_dim && r->magnitude > 0.f && r->magnitude <= 3.402823466e38f;
}

inline int paged_cache_check(const intfa_paged_cache* c) {
    if (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr || c->block_table == nullptr) return INTFA_ERR_NULL;
    if (c->heads_kv <= 0) return INTFA_ERR_SHAPE;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return INTFA_ERR_HEAD_DIM;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) || c->num_pages <= 0 || c->table_width <= 0)
        return INTFA_ERR_PAGE;
    if ((int64_t)c->table_width * c->page_size >= 1ll << 30) return INTFA_ERR_SHAPE;      // positions of keys are 32-bit numbers
    auto bad = [](const void* p, int64_t a, int64_t b, int64_t n) { return (reinterpret_cast<uintptr_t>(p) & 15u) || a % 16 || b % 16 || n % 16; };
    if (bad(c->k, c->k_stride_p, c->k_stride_h, c->k_stride_n) || bad(c->v, c->v_stride_p, c->v_stride_h, c->v_stride_n) ||
        (reinterpret_cast<uintptr_t>(c->k_scale) & 3u) || (reinterpret_cast<uintptr_t>(c->v_scale) & 3u) ||
        (reinterpret_cast<uintptr_t>(c->block_table) & 3u)) return INTFA_ERR_ALIGN;
    // rows of a page follow each other, and their offsets inside it are 32-bit numbers
    if (c->k_stride_n < c->head_dim || c->v_stride_n < c->head_dim || c->k_stride_n >= 1 << 22 || c->v_stride_n >= 1 << 22) return INTFA_ERR_SHAPE;
    return INTFA_OK;
}

struct PagedParams {
    const char* q; char* out; float* lse;
    const char* k; const char* v; const float* k_scale; const float* v_scale;
    const int32_t* table; const int32_t* seqlens_k; const int32_t* seqlens_q;
    int64_t q_sb, q_sh, q_sn, o_sb, o_sh, o_sn;      // bytes
    int64_t k_sp, k_sh, v_sp, v_sh;                  // bytes
    int64_t ks_sp, ks_sh, vs_sp, vs_sh, bt_sb;       // elements
    int32_t k_sn, v_sn;                              // bytes
    int32_t batch, heads, heads_kv, group, seqlen, rows;      // group: query heads per K/V head; rows = group * seqlen
    int32_t page_log2, num_pages, table_width, causal;
    int32_t tiles;                                   // row tiles of a K/V head
    int32_t unit_log2;                               // keys that are dealt together
    int32_t grid;                                    // workgroups of the launch
    int32_t lead;                                    // units ahead of an item's keys (intfa_paged_device.h)
    float qk_scale_log2;
    RopeArgs rope;
    float* parts; float* part_stats;                 // partial results: two slots per workgroup (intfa_paged_decode.h)
    uint64_t* ticket; uint64_t epoch;
    FastDiv d_group, d_tiles, d_pairs;
};

struct PagedSel { int head_dim, io_dt, row_tiles; bool one_page; };      // row_tiles: of 16 rows, 0 for the prefill kernel; one_page: a page holds the keys that are taken at a time
#define INTFA_DECL_PAGED(name) int name(const PagedParams& p, const PagedSel& sel, hipStream_t stream)
INTFA_DECL_PAGED(launch_paged_d64);
INTFA_DECL_PAGED(launch_paged_d128);
INTFA_DECL_PAGED(launch_paged_d256);
INTFA_DECL_PAGED(launch_paged_prefill_d64);
INTFA_DECL_PAGED(launch_paged_prefill_d128);
INTFA_DECL_PAGED(launch_paged_prefill_d256);
// rows of a tile and workgroups per compute unit of the prefill kernel (intfa_paged_prefill.h)
inline int paged_prefill_rows(int head_dim) { return head_dim == 128 ? 256 : 128; }
inline int paged_prefill_wgs(int head_dim) { return head_dim == 64 ? 2 : 1; }

}  // namespace intfa
