// Attention of prompts whose keys and values are expanded from latent vectors: q and k of DN + DR elements, the last DR of a key shared by all heads, values of DV.
//
// A workgroup of eight waves takes two tiles of 128 query rows of a head, four waves each, 32 rows a wave; both walk the same blocks of 64 keys, which asynchronous copies bring into two
// stages of LDS.  With a causal mask the tiles are the n-th from the end and the n-th from the start, so that all workgroups have the same work.
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16 in the inputs' type, a row in one lane and its pair (l ^ 32), so that P goes from accumulator to operand in its lane.
// Where the tiles are no more than the compute units, a workgroup has one, and each half of it half of the keys - of every block, or (small heads) every second block; the halves' rows are joined in the end
// (SPLIT: 10 heads of 64 + 32, 3 x 777 rows over up to 1555 keys 32 -> 24 us, 16 heads of 128 + 64 over 2048 unmasked tokens 65 -> 47; with twice the tiles, 4096 causal tokens, it would be 106 for 97).
// A third stage of LDS, requested two steps ahead, changed nothing (47 -> 48 us).
// The blocks run as a software pipeline: each product of block n + 1's scores and of block n - 1's values is followed by its share of block n's softmax.
#pragma once
#include "intfa_latent_expanded_host.h"
#include "intfa_splitkv.h"

namespace intfa {

constexpr float kExpandedSlack = 8.f;                // a row's frame follows its maximum where that grows by more
constexpr float kExpandedFar = 0x1p20f;              // a frame of this size: scores become differences from it in a step of their own (its last place is 1/8 there)

// A tile of 64 rows of ROW bytes in LDS.  A copy instruction writes 1 KB side by side: the rows i, i + NI, i + 2 NI .. of instruction i, and PAD bytes lie between two instructions'
// rows.  Neighbouring rows are thereby in different banks without any permutation, and all of a wave's reads are one lane address and constants.  PAD: 16 where sixteen
// neighbouring rows are read in one unit of sixteen bytes (keys), 64 where four are in 64 bytes (values).
template <int ROW, int PAD> struct PaddedTile {
    static constexpr int RPI = 1024 / ROW, NI = 64 / RPI, INST = 1024 + PAD, BYTES = NI * INST;
    static __device__ __forceinline__ uint32_t at(int row) { return (uint32_t)((row % NI) * INST + (row / NI) * ROW); }      // (row: below NI, or a multiple of it: at() adds up)
    // a lane's source: row and byte
    static __device__ __forceinline__ uint32_t source(int inst, int lane, uint32_t stride) { return (uint32_t)(inst + lane / (ROW / 16) * NI) * stride + 16u * (uint32_t)(lane % (ROW / 16)); }
};

template <int DN, int DR, int DV, bool SPLIT> struct ExpandedShape {
    // split: of the small heads a step takes two tiles of keys, one for each half; of the large ones half of a tile for each (two of them twice over have no room)
    static constexpr int PER_STEP = SPLIT && DN == 64 ? 2 : 1, KEYS = 64 * PER_STEP, ROWS = 128;      // of a half of the workgroup
    static constexpr int NROW = 2 * DN, RROW = 2 * DR, VROW = 2 * DV;
    typedef PaddedTile<NROW, 16> N;
    typedef PaddedTile<RROW, 16> R;
    typedef PaddedTile<VROW, 64> V;
    static constexpr int OFF_N = 0, OFF_R = 2 * PER_STEP * N::BYTES, OFF_V = OFF_R + 2 * PER_STEP * R::BYTES, TILES = OFF_V + 2 * PER_STEP * V::BYTES;
    static constexpr int LDS = TILES > 8 * OutStage<DV>::BYTES ? TILES : 8 * OutStage<DV>::BYTES;
    static constexpr int KN = DN / 16, KS = (DN + DR) / 16, DT = DV / 32;
};

// LONG: keys or values of a head span more than 32 bits (slices of a projection of 128 heads from 65408 keys on).  A tile has a resource of its own then, whose address goes on from
// block to block; else one resource has them all, and a tile is an offset from it in a scalar register (4096 causal tokens of 16 heads 88.0 us, and 88.7 with one for each).  Either
// ends with the last key, the offset counted: rows behind it come as zeros, also of a tile that begins there.
template <int DN, int DR, int DV, int DT_, bool CAUSAL, bool SPLIT, bool LONG>
__global__ void __launch_bounds__(512, 2) latent_expanded_kernel(const ExpandedParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef ExpandedShape<DN, DR, DV, SPLIT> S;
    constexpr int KEYS = S::KEYS, KN = S::KN, KS = S::KS, DT = S::DT, TILES = S::PER_STEP, NST = SPLIT && TILES == 1 ? 1 : 2, OWN = 32 * NST, PER = 16 * NST;      // keys of a block that a half has, and a lane's of them
    // P = 2^(x - frame) times this: fp16 keeps its 11 bits down to 2^-21 of the frame's; bf16 has the range, and leaves room for sums of 2^12 of its largest values
    constexpr float kShift = DT_ == 0 ? 7.f : -20.f;
    __shared__ __align__(1024) char lds[S::LDS];
    const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, lh = lane >> 5;
    const int all_wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = all_wave >> 2, wave = all_wave & 3;
    // ---- the workgroup's (sequence, head) and pair of tiles: an XCD's workgroups have whole heads
    int unit, pair;
    if ((int)blockIdx.x < p.whole) {
        const int slot = (int)blockIdx.x >> 3, q = fast_div(slot, p.d_pairs);
        unit = q * 8 + ((int)blockIdx.x & 7);
        pair = slot - q * p.pairs;
    } else {
        unit = fast_div((int)blockIdx.x, p.d_pairs);
        pair = (int)blockIdx.x - unit * p.pairs;
    }
    const int z = fast_div(unit, p.d_heads), head = unit - z * p.heads;
    // (split: the last tiles, which see the most keys, first)
    const int tile = SPLIT ? p.tiles - 1 - pair : CAUSAL ? (half == 0 ? p.tiles - 1 - pair : pair) : 2 * pair + half;
    const bool mine = SPLIT || (CAUSAL ? half == 0 || pair != p.tiles - 1 - pair : tile < p.tiles);
    const int key0 = SPLIT ? OWN * half : 0;   // of the half's keys in a block
    const int own_tile = TILES == 2 ? half : 0, own_row = TILES == 2 ? 0 : key0;
    auto length = [&](const int32_t* lens, int most) __attribute__((always_inline)) {
        if (lens == nullptr) return most;
        const int n = lens[z];
        return n < 0 ? 0 : n < most ? n : most;
    };
    const int m_rows = length(p.seqlens_q, p.seqlen), n_keys = length(p.seqlens_k, p.seqlen_k), off = n_keys - m_rows;
    auto blocks_of = [&](int t) __attribute__((always_inline)) {
        if (t >= p.tiles || t * S::ROWS >= m_rows) return 0;
        const int last = t * S::ROWS + S::ROWS < m_rows ? t * S::ROWS + S::ROWS : m_rows, seen = CAUSAL ? last + off : n_keys;
        return seen <= 0 ? 0 : ((seen < n_keys ? seen : n_keys) + KEYS - 1) / KEYS;
    };
    const int blocks = mine ? blocks_of(tile) : 0;
    const int first = blocks_of(SPLIT ? tile : CAUSAL ? p.tiles - 1 - pair : 2 * pair), second = blocks_of(SPLIT ? tile : CAUSAL ? pair : 2 * pair + 1);
    const int all_blocks = first > second ? first : second;
    const int row = tile * S::ROWS + 32 * wave + lq, row_ld = row < p.seqlen ? row : p.seqlen - 1;
    // ---- copies: a wave's share of a block
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const uint32_t keys_1 = (uint32_t)(n_keys > 0 ? n_keys - 1 : 0);
    struct Rows { v4i all; uint64_t at; uint32_t stride; };
    auto rows_of = [&](const char* first, uint32_t stride, uint32_t row) __attribute__((always_inline)) {
        const v4i all = make_rsrc(first, n_keys > 0 ? keys_1 * stride + row : 0);
        return Rows{all, (uint64_t)(uint32_t)all[1] << 32 | (uint32_t)all[0], stride};
    };
    Rows n_rows = rows_of(p.kn + z * p.kn_sb + head * p.kn_sh, p.kn_sn, S::NROW), r_rows = rows_of(p.kr + z * p.kr_sb, p.kr_sn, S::RROW),
         v_rows = rows_of(p.v + z * p.v_sb + head * p.v_sh, p.v_sn, S::VROW);
    struct TileAt { v4i rsrc; uint32_t off; };
    auto tile_at = [&](const Rows& t, int block, int i) __attribute__((always_inline)) {      // the i-th of a block
        const int key = __builtin_amdgcn_readfirstlane(block * KEYS + 64 * i);
        if (!LONG) return TileAt{t.all, (uint32_t)key * t.stride};
        int keys = __builtin_amdgcn_readfirstlane(n_keys) - key;
        keys = keys < 64 ? keys : 64;
        keys = keys > 0 ? keys : 0;
        return TileAt{make_rsrc((const void*)(t.at + (uint64_t)((uint32_t)i * 64 * t.stride)), (uint32_t)keys * t.stride), 0u};
    };
    auto go_on = [&](Rows& t) __attribute__((always_inline)) { if (LONG) t.at += KEYS * t.stride; };      // (a block's rows span less than 2^32 bytes)
    constexpr int NE = (S::N::NI + 7) / 8, VE = (S::V::NI + 7) / 8;      // instructions of a wave (all eight have as many; those of the rotary part: one of some waves)
    uint32_t n_off[NE], v_off[VE];
#pragma unroll
    for (int i = 0; i < NE; ++i) n_off[i] = S::N::source(all_wave + 8 * i, lane, p.kn_sn);
#pragma unroll
    for (int i = 0; i < VE; ++i) v_off[i] = S::V::source(all_wave + 8 * i, lane, p.v_sn);
    const uint32_t r_off = S::R::source(all_wave % S::R::NI, lane, p.kr_sn);
    static_assert(S::N::NI % 8 == 0 && S::V::NI % 8 == 0 && S::R::NI <= 8, "");
    auto copy_k = [&](int block, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const TileAt n = tile_at(n_rows, block, t);
#pragma unroll
            for (int i = 0; i < NE; ++i) issue_copy_1k<false>(n.rsrc, n_off[i], n.off, lds0 + S::OFF_N + (buf * TILES + t) * S::N::BYTES + S::N::INST * (all_wave + 8 * i));
            const TileAt r = tile_at(r_rows, block, t);
            if (all_wave < S::R::NI) issue_copy_1k<false>(r.rsrc, r_off, r.off, lds0 + S::OFF_R + (buf * TILES + t) * S::R::BYTES + S::R::INST * all_wave);
        }
        go_on(n_rows);
        go_on(r_rows);
    };
    auto copy_v = [&](int block, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const TileAt v = tile_at(v_rows, block, t);
#pragma unroll
            for (int i = 0; i < VE; ++i) issue_copy_1k<false>(v.rsrc, v_off[i], v.off, lds0 + S::OFF_V + (buf * TILES + t) * S::V::BYTES + S::V::INST * (all_wave + 8 * i));
        }
        go_on(v_rows);
    };
    if (all_blocks > 0) copy_k(0, 0);
    // ---- queries (B operand of S^T): sixteen bytes a step; a negative scale of scores turns them
    v4i q[KS];
    {
        const char* const a = p.qn + z * p.qn_sb + head * p.qn_sh + (int64_t)row_ld * p.qn_sn + 16 * lh;
        const char* const b = p.qr + z * p.qr_sb + head * p.qr_sh + (int64_t)row_ld * p.qr_sn + 16 * lh;
        const int flip = p.qk_scale_log2 < 0.f ? (int)0x80008000u : 0;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            q[k] = *(const v4i*)(k < KN ? a + 32 * k : b + 32 * (k - KN));
#pragma unroll
            for (int i = 0; i < 4; ++i) q[k][i] ^= flip;
        }
    }
    const float scale = fmaxf(fabsf(p.qk_scale_log2), 0x1p-126f);      // (never zero: hidden keys are -infinity times it)
    // ---- a lane's places in the tiles
    const uint32_t n_lane = S::OFF_N + own_tile * S::N::BYTES + S::N::at(own_row) + S::N::at(lq) + 16 * lh;
    const uint32_t r_lane = S::OFF_R + own_tile * S::R::BYTES + S::R::at(own_row) + S::R::at(lq) + 16 * lh;
    const uint32_t v_lane = S::OFF_V + own_tile * S::V::BYTES + S::V::at(own_row) + S::V::at(4 * lh + ((lane & 15) >> 2)) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto product = [&](v4i a, v4i b, v16f c) __attribute__((always_inline)) -> v16f {
        if (DT_ == 0) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    };
    uint32_t n_now, r_now, v_now;              // the same in the stage that a step reads
    auto key_fragment = [&](int i) __attribute__((always_inline)) -> v4i {      // of product i: keys 32 (i / KS) .., step i % KS
        const int k = i % KS, st = i / KS;
        return k < KN ? *(const v4i*)(lds + n_now + S::N::at(32 * st) + 32 * k) : *(const v4i*)(lds + r_now + S::R::at(32 * st) + 32 * (k - KN));
    };
    auto value_fragment = [&](int i) __attribute__((always_inline)) -> v4i {    // of product i: output tile i % DT, keys 16 (i / DT) ..
        const uint32_t a = v_now + S::V::at(16 * (i / DT)) + 64 * (i % DT);
        const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)INTFA_LDS(lds + a)));
        const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)INTFA_LDS(lds + a + S::V::at(8))));
        return (v4i){lo[0], lo[1], hi[0], hi[1]};
    };
    // ---- state, by the parity of the block
    constexpr int NQ = NST * KS, NP = 2 * NST * DT, AHEAD = 4;      // products of scores and of values in a block; operands are requested AHEAD products ahead
    v16f s[2][NST], acc[DT];
    v4i pf[2][NST][2];
    float m = -INFINITY, l = 0.f, mx = -INFINITY;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
    // One step: P of block n from s[PAR] (E), scores of block n + 1 into s[PAR ^ 1] (QK), values of block n - 1 (PV).  Returns the sum of P.
    auto step = [&](auto par_tag, auto qk_tag, auto e_tag, auto pv_tag, float factor, float frame) __attribute__((always_inline)) -> float {
        constexpr int PAR = decltype(par_tag)::value ? 1 : 0;
        constexpr bool QK = decltype(qk_tag)::value, E = decltype(e_tag)::value, PV = decltype(pv_tag)::value;
        constexpr int NQS = QK ? NQ : 0, NM = NQS + (PV ? NP : 0);
        v4i fr[AHEAD];
        float x[PER], e[PER], sum = 0.f;
        auto fetch = [&](int i) __attribute__((always_inline)) {
            if (i < NQS) fr[i % AHEAD] = key_fragment(i);
            else if (i < NM) fr[i % AHEAD] = value_fragment(i - NQS);
        };
        // element j of P: its argument two elements ahead, the exponential one ahead, then sum and conversion, so that none waits for the one before it
        auto argument = [&](int j) __attribute__((always_inline)) {
            if (j < PER) {
                x[j] = fmaf(s[PAR][j / 16][j % 16], factor, -frame);
                asm volatile("" : "+v"(x[j]));
            }
        };
        auto element = [&](int j) __attribute__((always_inline)) {
            argument(j + 2);
            if (j + 1 < PER) {
                e[j + 1] = fast_exp2(x[j + 1]);
                asm volatile("" : "+v"(e[j + 1]));
            }
            sum = j == 0 ? e[j] : sum + e[j];
            if (j & 1) {
                const v2f two = {e[j - 1], e[j]};
                int to = DT_ == 0 ? __builtin_bit_cast(int, __builtin_convertvector(two, v2h)) : __builtin_bit_cast(int, __builtin_convertvector(two, v2bf));
                asm volatile("" : "+v"(to), "+v"(sum));
                pf[PAR][j / 16][(j % 16) / 8][(j % 8) / 2] = to;
            }
        };
        auto maximum = [&](int j) __attribute__((always_inline)) {      // of elements 2 j, 2 j + 1 of the next block
            mx = fmaxf(fmaxf(mx, s[PAR ^ 1][j / 8][2 * (j % 8)]), s[PAR ^ 1][j / 8][2 * (j % 8) + 1]);
            asm volatile("" : "+v"(mx));
        };
        if (QK) mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fetch(i);
        if (E) {
            argument(0);
            argument(1);
            e[0] = fast_exp2(x[0]);
        }
        __builtin_amdgcn_sched_barrier(0);
        constexpr int C0 = NQS + 2;            // (the last score is there two products later)
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            if (i < NQS) {
                const int k = i % KS, st = i / KS;
                s[PAR ^ 1][st] = product(fr[i % AHEAD], q[k], k ? s[PAR ^ 1][st] : (v16f){0});
            } else {
                const int k = i - NQS;
                acc[k % DT] = product(fr[i % AHEAD], pf[PAR ^ 1][k / DT / 2][k / DT % 2], acc[k % DT]);
            }
            fetch(i + AHEAD);
            if (E) {
#pragma unroll
                for (int j = i * PER / (NM + !NM); j < (i + 1) * PER / (NM + !NM); ++j) element(j);
            }
            if (QK && PV && i >= C0) {
#pragma unroll
                for (int j = (i - C0) * (PER / 2) / (NM - C0); j < (i + 1 - C0) * (PER / 2) / (NM - C0); ++j) maximum(j);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (E && NM == 0) {
#pragma unroll
            for (int j = 0; j < PER; ++j) element(j);
        }
        if (QK && !PV) {
#pragma unroll
            for (int st = 0; st < NST; ++st) wait_for_product(s[PAR ^ 1][st]);
#pragma unroll
            for (int j = 0; j < PER / 2; ++j) maximum(j);
        }
        return sum;
    };
    // first block with a key that is hidden from a row of the wave: the diagonal's, or the ragged last one
    const int lowest = (CAUSAL ? tile * S::ROWS + 32 * wave + off : n_keys - 1);      // the last key that the wave's first row sees
    // Step n of the half's blocks.  The copies that it needs have been waited for; those of the next are requested.
    auto block = [&](auto par_tag, auto qk_tag, auto pv_tag, int n) __attribute__((always_inline)) {
        constexpr int PAR = decltype(par_tag)::value ? 1 : 0;
        const int at = n * KEYS + key0, lim = lowest - at;
        const bool masked = lim < OWN - 1 || at + OWN > n_keys;
        if (masked) {
            int last = CAUSAL ? lim + lq : lim;
            const int end = n_keys - 1 - at;
            last = (last < end ? last : end) - 4 * lh;
            mx = -INFINITY;
#pragma unroll
            for (int st = 0; st < NST; ++st) {
                const uint32_t hidden = hidden_past(last - 32 * st);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[PAR][st][r] = hide(s[PAR][st][r], hidden, 8 * (r >> 2) + (r & 3));
                    mx = fmaxf(mx, s[PAR][st][r]);
                }
            }
        }
        const float top = half_pair_max(mx) * scale;
        const bool grows = top - m > kExpandedSlack, move = __builtin_amdgcn_ballot_w64(grows) != 0;
        float alpha = 1.f;
        if (__builtin_expect(move, 0)) {       // (rows that do not need it stay: what a row gets does not depend on the others)
            alpha = grows ? fast_exp2(m - top) : 1.f;
            m = grows ? top : m;
        }
        const float base = m == -INFINITY ? 0.f : m;
        // The exponent is one multiply-add of the score.  Far from zero its rounding, and that of the products which the maximum was taken of, would grow past
        // what fp16 has room for: there the scores become differences from the frame first, by the same products.
        const bool far = fabsf(base) > kExpandedFar;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(far) != 0, 0)) {
#pragma clang fp contract(off)
#pragma unroll
            for (int st = 0; st < NST; ++st)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[PAR][st][r] = far ? s[PAR][st][r] * scale - base : s[PAR][st][r];
        }
        const float sum = step(par_tag, qk_tag, BoolTag<true>{}, pv_tag, far ? 1.f : scale, (far ? 0.f : base) - kShift);
        if (__builtin_expect(move, 0)) {       // (the block before was still added in the old frame)
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[dt][r] *= alpha;
        }
        l += sum;
    };
    constexpr BoolTag<false> F{};
    constexpr BoolTag<true> T{};
    // Step n of the workgroup (from -1): scores of block n + 1, softmax of block n, values of block n - 1.  All waves wait and copy alike, and do what their half has.  Blocks lie in the
    // stages by their parity; registers are counted from a half's last block, which is an odd one.
    int n = -1;
    auto sync = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int buf = n & 1;
        if (n + 2 < all_blocks) copy_k(n + 2, buf);
        if (n >= 0 && n < all_blocks) copy_v(n, buf);
        n_now = n_lane + (uint32_t)((buf ^ 1) * TILES * S::N::BYTES);
        r_now = r_lane + (uint32_t)((buf ^ 1) * TILES * S::R::BYTES);
        v_now = v_lane + (uint32_t)((buf ^ 1) * TILES * S::V::BYTES);
    };
    auto next = [&](auto par_tag, auto qk_tag, auto pv_tag) __attribute__((always_inline)) {
        sync();
        block(par_tag, qk_tag, pv_tag, n);
        ++n;
    };
    if (blocks > 0) {
        q_has_arrived(q);
        sync();
        if (blocks & 1) {
            step(F, T, F, F, 0.f, 0.f);
            ++n;
            if (blocks > 1) {
                next(T, T, F);
                next(F, T, T);
            }
        } else {
            step(T, T, F, F, 0.f, 0.f);
            ++n;
            next(F, T, F);
        }
#pragma clang loop unroll(disable)
        while (n + 1 < blocks) {
            next(T, T, T);
            next(F, T, T);
        }
        if (blocks > 1) next(T, F, T); else next(T, F, F);
        sync();
        step(F, F, F, T, 0.f, 0.f);
        ++n;
    }
    for (; n <= all_blocks; ++n) sync();
    // ---- the rows
    l = half_pair_sum(l);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) wait_for_product(acc[dt]);
    if (SPLIT) {                               // the second half's rows to the first
        char* const acc_lds = lds + (wave * DT * 4 * 64 + lane) * 16;
        v2f* const stats = (v2f*)(lds + 4 * DT * 4096) + wave * 64 + lane;
        static_assert(4 * DT * 4096 + 2048 <= S::LDS, "");
        if (half == 1) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int k = 0; k < 4; ++k) *(v4f*)(acc_lds + (dt * 4 + k) * 1024) = (v4f){acc[dt][4 * k], acc[dt][4 * k + 1], acc[dt][4 * k + 2], acc[dt][4 * k + 3]};
            *stats = (v2f){m, l};
        }
        __syncthreads();
        if (half == 0) {
            const v2f other = *stats;
            const float top = fmaxf(m, other[0]), base = top == -INFINITY ? 0.f : top, a = fast_exp2(m - base), b = fast_exp2(other[0] - base);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const v4f o = *(const v4f*)(acc_lds + (dt * 4 + k) * 1024);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[dt][4 * k + i] = acc[dt][4 * k + i] * a + o[i] * b;
                }
            l = l * a + other[1] * b;
            m = top;
        }
        __syncthreads();
        if (half == 1) return;
    }
    if (!mine) return;
    const bool padding = row >= m_rows, empty = padding || m == -INFINITY, zeros = padding || l == 0.f;      // (a row without a key: its products may hold 0 times an infinite value)
    const float inv = empty ? 0.f : 1.f / l;
    if (p.lse != nullptr && lh == 0 && row < p.seqlen)
        p.lse[((int64_t)z * p.heads + head) * p.seqlen + row] = padding ? -INFINITY : (m == -INFINITY ? 0.f : m) - kShift + __builtin_log2f(l);
    char* const stage = lds + all_wave * OutStage<DV>::BYTES;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v4f o = {acc[dt][4 * k], acc[dt][4 * k + 1], acc[dt][4 * k + 2], acc[dt][4 * k + 3]};
            o *= inv;
            if (zeros) o = (v4f){0.f, 0.f, 0.f, 0.f};
            v2i bits;
            store_out4<DT_>((char*)&bits, o);
            out_stage_put<DV>(stage, lq, 32 * dt + 8 * k + 4 * lh, bits);
        }
    const int row0 = tile * S::ROWS + 32 * wave, valid = p.seqlen - row0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    out_stage_flush<DV>(stage, p.out + z * p.o_sb + head * p.o_sh + (int64_t)row0 * p.o_sn, p.o_sn, valid < 32 ? valid : 32, lane);
#endif  // __HIP_DEVICE_COMPILE__
}

template <int DN, int DR, int DV, int DT_, bool LONG> int launch_expanded_span(const ExpandedParams& p, bool causal, hipStream_t stream) {
    const dim3 grid((unsigned)(p.batch * p.heads * p.pairs));
    if (p.split) {
        if (causal) hipLaunchKernelGGL((latent_expanded_kernel<DN, DR, DV, DT_, true, true, LONG>), grid, dim3(512), 0, stream, p);
        else hipLaunchKernelGGL((latent_expanded_kernel<DN, DR, DV, DT_, false, true, LONG>), grid, dim3(512), 0, stream, p);
    } else if (causal) hipLaunchKernelGGL((latent_expanded_kernel<DN, DR, DV, DT_, true, false, LONG>), grid, dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((latent_expanded_kernel<DN, DR, DV, DT_, false, false, LONG>), grid, dim3(512), 0, stream, p);
    return (int)hipGetLastError();
}
template <int DN, int DR, int DV, int DT_> int launch_expanded(const ExpandedParams& p, bool causal, hipStream_t stream) {
    return p.far ? launch_expanded_span<DN, DR, DV, DT_, true>(p, causal, stream) : launch_expanded_span<DN, DR, DV, DT_, false>(p, causal, stream);
}

}  // namespace intfa
