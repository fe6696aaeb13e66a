// Kernel-side block and launch functions of the expanded form of latent attention.
#pragma once
#include "intfa_launch.h"

namespace intfa {

struct ExpandedParams {
    const char* qn; const char* qr; const char* kn; const char* kr; const char* v; char* out; float* lse;
    const int32_t* seqlens_q; const int32_t* seqlens_k;
    int64_t qn_sb, qn_sh, qn_sn, qr_sb, qr_sh, qr_sn, kn_sb, kn_sh, kr_sb, v_sb, v_sh, o_sb, o_sh, o_sn;      // bytes
    uint32_t kn_sn, kr_sn, v_sn;                     // bytes
    int32_t batch, heads, seqlen, seqlen_k, tiles, pairs, whole;      // tiles of a head, pairs of them (split: the tiles again); workgroups of the (sequence, head)s that are dealt whole to the XCDs
    bool split;                                      // a workgroup has one tile, each half of it half of the keys
    bool far;                                        // keys or values of a head span more than 32 bits
    float qk_scale_log2;
    FastDiv d_pairs, d_heads;
};
#define INTFA_DECL_EXPANDED(name) int name(const ExpandedParams& p, bool causal, hipStream_t stream)
INTFA_DECL_EXPANDED(launch_expanded_n128_f16);
INTFA_DECL_EXPANDED(launch_expanded_n128_bf16);
INTFA_DECL_EXPANDED(launch_expanded_n64_f16);
INTFA_DECL_EXPANDED(launch_expanded_n64_bf16);

}  // namespace intfa
