// Attention of a few query rows over a paged int8 cache.
//
// The rows of a K/V head (its group of query heads times the new tokens, tokens outermost) are taken in tiles of sixteen.  S^T = K Q^T
// and O^T = V^T P^T run on v_mfma_f32_16x16x32_f16.  The cache goes from memory into registers in the layouts that the two products want,
// without LDS:
//   K   lane (m = l % 16, c = l / 16) loads bytes 64 j + 16 c .. + 15 of key row m: sixteen elements of the row, eight each for products
//       2 j and 2 j + 1.  Which elements a product takes together is free as long as Q's fragments are laid out the same.
//   P   leaves the first product with keys 4 c + i of each 16-key granule in lane (query n = l % 16, c), and the granules 2 t and 2 t + 1 are
//       the eight slots of lane c in the second one: P goes from accumulator to operand in its lane.
//   V   lane (x = l % 16, c) therefore loads D / 16 bytes, x * D / 16 onward, of key rows 4 c + i of each granule: whole rows, and element j of
//       each is what tile j of V^T (row x: column x * D / 16 + j of V) takes.  The transposition is a byte select inside the lane.
// int8 to fp16 is exact: byte ^ 0x80 under the exponent of 1024 is 1152 + value.
#pragma once
#include "intfa_paged_device.h"

namespace intfa {

constexpr int kPagedWaves = 4;
// P is held as 2^14 p: fp16 keeps its 11 bits down to p = 2^-28, times the ratio of two pages' scales.  The factor goes in with that ratio, p itself being
// 2^(s - m) by a subtraction of its own: taken from m beforehand it would be lost to m's rounding, and p past fp16's range, from |m| = 2^25 on.
constexpr float kPUnit = 0x1p14f;
// Sums of p v are held as 2^-12 of themselves, so that those of 2^12 values fit fp32 wherever the values do, and the least scale that an append leaves
// (2^-100) times all of that is a normal number.  Scales under it count as parts of it in P.
constexpr float kSumUnit = 0x1p-12f, kLeastTop = 0x1p-100f;

// Merges the rows of an item from its pieces: those of workgroups `one` onward, all of them first items of theirs but the one that the item begins in
// the middle of (first_is_first: it begins at that workgroup's first unit).
template <int D, int DT, int R, int THREADS>
__device__ __forceinline__ void paged_merge(PagedArgs p, const PagedItem& t, int row0, int one, int pieces, bool first_is_first, float* lds) {
    constexpr int LPR = D / 4, GROUPS = THREADS / LPR;      // lanes per row; rows, or shares of a row's pieces, side by side
    const int nrows = p->rows - row0 < R ? p->rows - row0 : R;
    const int col = ((int)threadIdx.x % LPR) * 4, group = (int)threadIdx.x / LPR;
    int shares = 1;                                         // of a row's pieces
    while (shares * 2 * nrows <= GROUPS) shares *= 2;
    const int side = GROUPS / shares, share = group / side;
    const BufferRsrc o = __builtin_amdgcn_make_buffer_rsrc(p->parts + (int64_t)one * 2 * R * D, 0, -1, 0x00020000);
    const BufferRsrc s = __builtin_amdgcn_make_buffer_rsrc(p->part_stats + (int64_t)one * 2 * R * 2, 0, -1, 0x00020000);
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    auto slot_of = [&](int i) __attribute__((always_inline)) { return (uint32_t)(2 * i + (i == 0 && !first_is_first)); };
    for (int r0 = 0; r0 < nrows; r0 += side) {
        const int r = r0 + group % side, rr = r < nrows ? r : nrows - 1;
        v4f acc = {0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        auto add = [&](auto many) __attribute__((always_inline)) {
            constexpr int U = decltype(many)::value;
            for (int i0 = share; i0 < pieces; i0 += U * shares) {      // (U loads under way together: each takes a microsecond)
                v4f x[U];
                float ms[U], ls[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * shares < pieces ? i0 + u * shares : i0;
                    const uint32_t row = slot_of(i) * R + (uint32_t)rr;
                    const v2u st = __builtin_amdgcn_raw_buffer_load_b64(s, row * 8u, 0, kSplitAux);
                    x[u] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(o, (row * (uint32_t)D + (uint32_t)col) * 4u, 0, kSplitAux));
                    ms[u] = i0 + u * shares < pieces ? __builtin_bit_cast(float, (unsigned)st[0]) : -INFINITY;
                    ls[u] = __builtin_bit_cast(float, (unsigned)st[1]);
                }
                float top = m;
#pragma unroll
                for (int u = 0; u < U; ++u) top = fmaxf(top, ms[u]);
                const float frame = top == -INFINITY ? 0.f : top;
                const float a = fast_exp2(m - frame);
                acc *= a;
                l *= a;
                m = top;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float w = fast_exp2(ms[u] - frame);
                    acc += w * x[u];
                    l += w * ls[u];
                }
            }
        };
        if (pieces <= 4 * shares) add(IntTag<4>{}); else add(IntTag<16>{});
        if (shares > 1) {                                   // (one row per group then: every thread comes here once)
            __syncthreads();
            float* const mine = lds + threadIdx.x * 6;
            mine[0] = acc[0]; mine[1] = acc[1]; mine[2] = acc[2]; mine[3] = acc[3]; mine[4] = m; mine[5] = l;
            __syncthreads();
            if (share > 0) return;
            for (int k = 1; k < shares; ++k) {
                const float* const other = lds + ((group + k * side) * LPR + (int)threadIdx.x % LPR) * 6;
                const float top = fmaxf(m, other[4]), frame = top == -INFINITY ? 0.f : top, a = fast_exp2(m - frame), w = fast_exp2(other[4] - frame);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = a * acc[j] + w * other[j];
                l = a * l + w * other[5];
                m = top;
            }
        }
        if (r >= nrows) continue;
        const int row = row0 + r, token = paged_div(row, p->d_group), head = t.hk * p->group + row - token * p->group;
        const bool empty = m == -INFINITY || token >= t.m;
        if (token >= t.m) acc = (v4f){0.f, 0.f, 0.f, 0.f};
        store_out4<DT>(p->out + t.z * p->o_sb + head * p->o_sh + token * p->o_sn + col * 2, acc * (empty ? 0.f : 1.f / (kSumUnit * l)));
        if (p->lse != nullptr && col == 0)
            p->lse[((int64_t)t.z * p->heads + head) * p->seqlen + token] = token >= t.m ? -INFINITY : m + __builtin_log2f(l);
    }
}

// Keys that a wave takes at a time, as they come from memory.
template <int D> struct PagedStep {
    static constexpr int KEYS = D == 256 ? 32 : 64, G = KEYS / 16, KJ = D / 64, VB = D / 16, VD = VB / 4;
    typedef uint32_t VRow __attribute__((ext_vector_type(VD)));
    v4i k[G][KJ];
    VRow v[G][4];
    float ks[G], vs[G];
    bool has[G];                  // the granule has a key that some row sees, and the table names its page
};
// Where they come from.  K's registers are refilled once the scores are formed, V's once their products are, so that one of the two is on its way
// under everything that a step does.  The table's entries, which the addresses wait for, are requested a step ahead of that.
// (Two sets of registers, with everything requested a whole step ahead, leave room for one wave per SIMD: 32 x 32 heads of 4096 keys 171 -> 185 us.)
// ONE: a page holds a step's keys (page_size at least KEYS), which takes a quarter of the scalar work.
template <int D, bool ONE> struct PagedStream {
    typedef PagedStep<D> Step;
    static constexpr int G = Step::G, IDS = ONE ? 1 : G;
    const char* k_head; const char* v_head;
    PagedInts table;
    PagedFloats k_scale, v_scale;
    int64_t k_sp, v_sp, ks_sp, vs_sp;
    int k_sn, v_sn, page_log2, num_pages, last_column;
    int most;                     // keys past `most` are not this workgroup's
    uint32_t k_lane, v_lane;
    int id[IDS];
    __device__ __forceinline__ PagedStream(PagedArgs p, const PagedItem& t, int most_, int x, int c)
        : k_head(p->k + t.hk * p->k_sh), v_head(p->v + t.hk * p->v_sh), table((PagedInts)(p->table + t.z * p->bt_sb)),
          k_scale((PagedFloats)(p->k_scale + t.hk * p->ks_sh)), v_scale((PagedFloats)(p->v_scale + t.hk * p->vs_sh)), k_sp(p->k_sp), v_sp(p->v_sp), ks_sp(p->ks_sp),
          vs_sp(p->vs_sp), k_sn(p->k_sn), v_sn(p->v_sn), page_log2(p->page_log2), num_pages(p->num_pages), last_column(p->table_width - 1), most(most_),
          k_lane((uint32_t)(x * p->k_sn + 16 * c)), v_lane((uint32_t)(4 * c * p->v_sn + x * Step::VB)) {}
    __device__ __forceinline__ void look(int key0) {
#pragma unroll
        for (int g = 0; g < IDS; ++g) {
            const int column = (key0 + 16 * g) >> page_log2;
            id[g] = table[column < last_column ? column : last_column];      // (behind the last key the table may hold anything)
        }
    }
    __device__ __forceinline__ bool named(int g) const { return (unsigned)id[g] < (unsigned)num_pages; }
    __device__ __forceinline__ void load_k(int key0, Step& s) const {
        const char* kp[IDS];
#pragma unroll
        for (int g = 0; g < IDS; ++g) kp[g] = k_head + (named(g) ? id[g] : 0) * k_sp + ((key0 + 16 * g) & ((1 << page_log2) - 1)) * k_sn;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < Step::KJ; ++j)
                s.k[g][j] = __builtin_nontemporal_load((const v4i*)((ONE ? kp[0] + 16 * g * k_sn : kp[ONE ? 0 : g]) + k_lane + 64 * j));
    }
    __device__ __forceinline__ void load_v(int key0, Step& s) const {
        const char* vp[IDS];
#pragma unroll
        for (int g = 0; g < IDS; ++g) {
            const int at = named(g) ? id[g] : 0;
            vp[g] = v_head + at * v_sp + ((key0 + 16 * g) & ((1 << page_log2) - 1)) * v_sn;
            s.ks[g] = k_scale[at * ks_sp];
            s.vs[g] = v_scale[at * vs_sp];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            s.has[g] = named(ONE ? 0 : g) && key0 + 16 * g < most;
            if (ONE) {
                s.ks[g] = s.ks[0];
                s.vs[g] = s.vs[0];
            }
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s.v[g][i] = __builtin_nontemporal_load((const typename Step::VRow*)((ONE ? vp[0] + (16 * g + i) * v_sn : vp[ONE ? 0 : g] + i * v_sn) + v_lane));
    }
};

template <int D, int DT, int RT, bool ONE>
__global__ void __launch_bounds__(64 * kPagedWaves, RT == 1 && D < 256 ? 2 : 1) paged_decode_kernel(const PagedParams) {
    constexpr int R = 16 * RT, STEP = PagedStep<D>::KEYS, G = STEP / 16, KJ = D / 64, DT16 = D / 16;
    constexpr int W = kPagedWaves, THREADS = 64 * W, STRIDE = W * STEP;
    typedef PagedQueries<D, DT, R, THREADS> Queries;
    constexpr int O_ROW = D + 4;                           // floats (4 more: the banks)
    __shared__ __align__(16) char q_lds[R * Queries::ROW];
    __shared__ __align__(16) char q_rest[R * Queries::ROW];
    __shared__ float factor_lds[R];
    __shared__ __align__(16) float o_lds[W * 16 * O_ROW];
    static_assert(R * (D / 2) * 8 <= W * 16 * O_ROW * 4 && THREADS * 6 <= W * 16 * O_ROW, "the angles lie there first, and a merge's sums last");
    __shared__ float m_lds[W * R], l_lds[W * R];
    __shared__ uint32_t arrival_lds;
    __shared__ double freq_lds[D / 2];
    PagedArgs p = paged_args_first();
    PagedItem t;
    const double freq = paged_frequency(p);
    PagedPiece piece = paged_find(p, R, t);
    if ((int)threadIdx.x < D / 2) freq_lds[threadIdx.x] = freq;
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), x = lane & 15, c = lane >> 4;
  while (piece.start < piece.end) {
    const int row0 = t.tile * R;
    const PagedPart part = paged_part(p, t, piece);
    if (part.none) break;
    uint64_t ticket_seen = 0;
    if (!part.whole && threadIdx.x == 0) ticket_seen = __hip_atomic_load(paged_ticket(p, t), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    Queries queries;
    queries.request(p, t, row0);
    const bool rope = queries.rope;
    // (a row past the last one or a token past the sequence's new ones counts like the others here; what it gives is not used)
    const int most = part.key_end, least = paged_token_keys(p, t, t.first_token);
    // the first keys are on their way while the queries are staged
    PagedStream<D, ONE> stream(p, t, most, x, c);
    PagedStep<D> now;
    int key0 = part.key_first + wave * STEP;
    if (key0 < most) {
        stream.look(key0);
        stream.load_k(key0, now);
        stream.load_v(key0, now);
        stream.look(key0 + STRIDE);
    }
    int seen[RT];
    float factor[RT], m[RT], l[RT];
    v4f o[RT][DT16];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        seen[rt] = paged_token_keys(p, t, paged_div(row0 + 16 * rt + x, p->d_group));
        m[rt] = -INFINITY;
        l[rt] = 0.f;
#pragma unroll
        for (int j = 0; j < DT16; ++j) o[rt][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    }
    if (rope) {
        queries.turn_angles(p, t, freq_lds, (v2f*)o_lds);
        __syncthreads();
    }
    queries.template stage<true>(p, row0, (const v2f*)o_lds, q_lds, q_rest, factor_lds);
    if (!part.whole) paged_open_ticket(p, paged_ticket(p, t), ticket_seen);
    __syncthreads();
    const char* const q_lane = q_lds + x * Queries::ROW + 32 * c;
    const char* const q_rest_lane = q_rest + x * Queries::ROW + 32 * c;
    v8h q_first[2 * KJ];                                   // (one row tile: in registers)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) factor[rt] = factor_lds[16 * rt + x];
    if (RT == 1) {
#pragma unroll
        for (int j = 0; j < 2 * KJ; ++j) q_first[j] = *(const v8h*)(q_lane + 128 * (j / 2) + 16 * (j & 1));
    }
    for (; key0 < most; key0 += STRIDE) {
        const bool more = key0 + STRIDE < most;
        bool masked = key0 + STEP > least;
#pragma unroll
        for (int g = 0; g < G; ++g) masked = masked || !now.has[g];
        // V's scales relative to the largest of the step's go into P, that one into the sum
        float v_top = kLeastTop;
#pragma unroll
        for (int g = 0; g < G; ++g) v_top = fmaxf(v_top, now.has[g] ? fabsf(now.vs[g]) : 0.f);
        const float v_unit = v_top * (kSumUnit / kPUnit), v_inv = kSumUnit * __builtin_amdgcn_rcpf(v_unit);      // = kPUnit / v_top
        float v_rel[G];
#pragma unroll
        for (int g = 0; g < G; ++g) v_rel[g] = now.has[g] ? now.vs[g] * v_inv : 0.f;
        v4f scores[RT][G];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int g = 0; g < G; ++g) scores[rt][g] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
            v8h kf[G][2];
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t w[4];
                    i8x4_to_f16((uint32_t)now.k[g][j][2 * u], w[0], w[1]);
                    i8x4_to_f16((uint32_t)now.k[g][j][2 * u + 1], w[2], w[3]);
                    kf[g][u] = __builtin_bit_cast(v8h, (v4i){(int)w[0], (int)w[1], (int)w[2], (int)w[3]});
                }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const v8h qf = RT == 1 ? q_first[2 * j + u] : *(const v8h*)(q_lane + 16 * rt * Queries::ROW + 128 * j + 16 * u);
#pragma unroll
                    for (int g = 0; g < G; ++g) scores[rt][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[g][u], qf, scores[rt][g], 0, 0, 0);
                }
                if (rope) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const v8h qf = *(const v8h*)(q_rest_lane + 16 * rt * Queries::ROW + 128 * j + 16 * u);
#pragma unroll
                        for (int g = 0; g < G; ++g) scores[rt][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[g][u], qf, scores[rt][g], 0, 0, 0);
                    }
                }
            }
        }
        if (more) stream.load_k(key0 + STRIDE, now);
        v8h pf[RT][G / 2];
        float alpha[RT];
        bool rescale = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma clang fp contract(off)                               // (what the maximum is taken from is what it was taken of)
            v4f (&s)[G] = scores[rt];
            float top = -INFINITY;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const float f = factor[rt] * now.ks[g];
#pragma unroll
                for (int i = 0; i < 4; ++i) s[g][i] *= f;
            }
            if (masked) {
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int last = now.has[g] ? seen[rt] - (key0 + 16 * g + 4 * c) : 0;      // of the lane's four keys
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[g][i] = i < last ? s[g][i] : -INFINITY;
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, s[g][i]);
            top = reduce_row_lanes(top, [](float a, float b) { return fmaxf(a, b); });
            const float m_new = fmaxf(m[rt], top), frame = m_new == -INFINITY ? 0.f : m_new;
            alpha[rt] = m_new == -INFINITY ? 1.f : fast_exp2(m[rt] - m_new);
            m[rt] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[g][i] = fast_exp2(s[g][i] - frame);      // (a score of the row's is the maximum, bit for bit: p is at most one)
                    sum += s[g][i];
                    s[g][i] *= v_rel[g];
                }
            l[rt] = fmaf(l[rt], alpha[rt], sum);
#pragma unroll
            for (int h = 0; h < G / 2; ++h) {
                v8h f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    f[i] = (_Float16)s[2 * h][i];
                    f[4 + i] = (_Float16)s[2 * h + 1][i];
                }
                pf[rt][h] = f;
            }
            rescale = rescale || alpha[rt] != 1.f;
        }
        if (__any(rescale)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < DT16; ++j) o[rt][j] *= alpha[rt];
        }
        auto tile = [&](auto jt) __attribute__((always_inline)) {
            constexpr int j = decltype(jt)::value;
            v8h vf[G / 2];
#pragma unroll
            for (int h = 0; h < G / 2; ++h) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = i8_pair_to_f16<j % 4>(now.v[2 * h + i / 2][2 * (i & 1)][j / 4], now.v[2 * h + i / 2][2 * (i & 1) + 1][j / 4]);
                vf[h] = __builtin_bit_cast(v8h, (v4i){(int)w[0], (int)w[1], (int)w[2], (int)w[3]});
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                v4f a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < G / 2; ++h) a = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[h], pf[rt][h], a, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[rt][j][i] = fmaf(a[i], v_unit, o[rt][j][i]);
            }
        };
        static_for<DT16>(tile);
        if (more) {
            stream.load_v(key0 + STRIDE, now);
            stream.look(key0 + 2 * STRIDE);
        }
    }
    p = paged_args();
    // ---- the waves' parts of a row meet in LDS
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = reduce_row_lanes(l[rt], [](float a, float b) { return a + b; });
        if (c == 0) {
            m_lds[wave * R + 16 * rt + x] = m[rt];
            l_lds[wave * R + 16 * rt + x] = l[rt];
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (rt > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < DT16; ++j) o_lds[(wave * 16 + x) * O_ROW + (4 * c + i) * DT16 + j] = o[rt][j][i];
        __syncthreads();
        const int r = (int)threadIdx.x / 16, cols = (int)threadIdx.x % 16, row = row0 + 16 * rt + r;      // D / 16 columns of one row
        static_assert(THREADS == 256, "a thread per row and sixteenth of it");
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, m_lds[w * R + 16 * rt + r]);
        const int token = paged_div(row, p->d_group);
        const bool empty = top == -INFINITY || (part.whole && token >= t.m);
        float sum = 0.f, weight[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            weight[w] = empty ? 0.f : fast_exp2(m_lds[w * R + 16 * rt + r] - top);
            sum += weight[w] * l_lds[w * R + 16 * rt + r];
        }
        const int head = t.hk * p->group + row - token * p->group;
        if (row < p->rows) {
            if (part.whole) {
                const float inv = empty ? 0.f : 1.f / (kSumUnit * sum);
                char* const dst = p->out + t.z * p->o_sb + head * p->o_sh + token * p->o_sn + cols * DT16 * 2;
#pragma unroll
                for (int j = 0; j < DT16; j += 4) {
                    v4f a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < W; ++w) a += weight[w] * *(const v4f*)(o_lds + (w * 16 + r) * O_ROW + cols * DT16 + j);
                    if (token >= t.m) a = (v4f){0.f, 0.f, 0.f, 0.f};      // (whatever the row holds: zero times what is not a number is none)
                    store_out4<DT>(dst + j * 2, a * inv);
                }
                if (p->lse != nullptr && cols == 0)
                    p->lse[((int64_t)t.z * p->heads + head) * p->seqlen + token] = token >= t.m ? -INFINITY : top + __builtin_log2f(sum);      // (no key: -infinity twice; no number in the row: the sum is none either)
            } else {
                const PagedParts mine(p, R, D, (int)part.slot);
#pragma unroll
                for (int j = 0; j < DT16; j += 4) {
                    v4f a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < W; ++w) a += weight[w] * *(const v4f*)(o_lds + (w * 16 + r) * O_ROW + cols * DT16 + j);
                    mine.put((uint32_t)(16 * rt + r), D, cols * DT16 + j, a);
                }
                if (cols == 0) mine.put_stats((uint32_t)(16 * rt + r), top, sum);
            }
        }
    }
    if (!part.whole && paged_last_arrival(p, paged_ticket(p, t), &arrival_lds, part.pieces))
        paged_merge<D, DT, R, THREADS>(p, t, row0, part.one, part.pieces, part.first_is_first, o_lds);
    if (!paged_next(p, R, t, piece)) break;
    __syncthreads();
  }
}

template <int D> int launch_paged(const PagedParams& p, const PagedSel& sel, hipStream_t stream) {
    const dim3 grid((unsigned)p.grid);
#define INTFA_CALL(DT, RT) do { \
        if (sel.one_page) hipLaunchKernelGGL((paged_decode_kernel<D, DT, RT, true>), grid, dim3(64 * kPagedWaves), 0, stream, p); \
        else hipLaunchKernelGGL((paged_decode_kernel<D, DT, RT, false>), grid, dim3(64 * kPagedWaves), 0, stream, p); } while (0)
    if (sel.io_dt == 0) {
        if (sel.row_tiles == 1) INTFA_CALL(0, 1); else INTFA_CALL(0, 2);
    } else {
        if (sel.row_tiles == 1) INTFA_CALL(1, 1); else INTFA_CALL(1, 2);
    }
#undef INTFA_CALL
    return (int)hipGetLastError();
}

}  // namespace intfa
