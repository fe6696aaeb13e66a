// Host-side checks that the entry points of the latent cache share.
#pragma once
#include "intfa_paged_host.h"

namespace intfa {

inline bool aligned_to(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) == 0; }

inline int latent_cache_check(const intfa_latent_cache* c) {
    if (c->rows == nullptr || c->scale == nullptr || c->block_table == nullptr) return INTFA_ERR_NULL;
    if ((c->latent_dim != 128 && c->latent_dim != 256 && c->latent_dim != 512) || (c->rope_dim != 32 && c->rope_dim != 64)) return INTFA_ERR_HEAD_DIM;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) || c->num_pages <= 0 || c->table_width <= 0) return INTFA_ERR_PAGE;
    if ((int64_t)c->table_width * c->page_size >= 1ll << 30) return INTFA_ERR_SHAPE;      // positions of keys are 32-bit numbers
    if (!aligned_to(c->rows, 16) || c->r_stride_p % 16 || c->r_stride_n % 16 || !aligned_to(c->scale, 8) || c->s_stride_p % 2 || c->s_stride_n % 2 ||
        !aligned_to(c->block_table, 4)) return INTFA_ERR_ALIGN;
    // rows of a page follow each other, and their offsets inside it are 32-bit numbers
    if (c->r_stride_n < c->latent_dim + c->rope_dim || c->r_stride_n >= 1 << 22 || c->s_stride_n < 2 || c->s_stride_n >= 1 << 20) return INTFA_ERR_SHAPE;
    return INTFA_OK;
}

struct LatentParams {
    PagedParams deal;                          // (k: the rows, k_scale: their scales, ks_sh: elements from token to token; one head)
    const char* q_rope; int64_t qr_sb, qr_sh, qr_sn;      // bytes
    v4i* open_items;                           // [workgroups]: the item that begins in a workgroup's piece and goes on in others (pieces, sequence, tile, its slot there); pieces 0: none
};

#define INTFA_DECL_LATENT(name) int name(const LatentParams& p, int rows, hipStream_t stream)
INTFA_DECL_LATENT(launch_latent_c128_r32_f16); INTFA_DECL_LATENT(launch_latent_c128_r32_bf16); INTFA_DECL_LATENT(launch_latent_c128_r64_f16); INTFA_DECL_LATENT(launch_latent_c128_r64_bf16);
INTFA_DECL_LATENT(launch_latent_c256_r32_f16); INTFA_DECL_LATENT(launch_latent_c256_r32_bf16); INTFA_DECL_LATENT(launch_latent_c256_r64_f16); INTFA_DECL_LATENT(launch_latent_c256_r64_bf16);
INTFA_DECL_LATENT(launch_latent_c512_r32_f16); INTFA_DECL_LATENT(launch_latent_c512_r32_bf16); INTFA_DECL_LATENT(launch_latent_c512_r64_f16); INTFA_DECL_LATENT(launch_latent_c512_r64_bf16);

}  // namespace intfa
