// Attention of many query rows (a chunk of a prompt, or a whole one) over a paged int8 cache.
//
// A wave owns 32 rows of a tile and all waves walk the same key blocks of 64.  S^T = K Q^T and O^T = V^T P^T run on v_mfma_f32_32x32x16_f16 with the
// rows as columns, so that the statistics of a row are one lane's (and its pair's, l ^ 32) and P goes from accumulator to operand in its lane.  The products
// take fp16, and what a block needs of it is made once for all waves: the threads fetch the block's bytes two blocks ahead, turn them into fp16 (exactly:
// intfa_paged_device.h) and store them to LDS, K by rows of keys, V transposed.
//   V^T  a thread takes four consecutive keys by four columns: a word each of four rows, whose bytes it selects into four pairs of pairs.  A row of V^T
//        holds the keys in the order in which P's lanes have them: 16 t + 8 j + 4 h + i at 32 t + 16 h + 8 j + 2 i bytes (h: the lane's half).  Column
//        4 q + b is row b D / 4 + q: neighbouring threads (q) then store to neighbouring rows, in different banks, and a lane's accumulators of the
//        tiles are four neighbouring columns.
// A row's scale of scores and a page's go into one multiplier of the exponent's fused multiply-add (a page's scale is not negative: the maximum of the
// products is that of the scores).  V's scale goes there too, as log2(scale / reference), the reference being the unit of the accumulators: it follows the
// page's scale where that leaves 2^-4 .. 2 of it.  A row's maximum is followed where it grows by more than 2^6, so that most blocks rescale nothing.
//
// What bounds it (2 x 32 x 512 bf16 rows of 128 over up to 30720 keys: 534 - 560 us by card, 910 - 955 TFLOP/s of the 1200 that a matrix product of 8192^3 reaches): per
// block and SIMD 2050 clocks of products and 2400 of other vector work, two thirds of it the softmax, which hardly run beside each other - 4600 clocks
// pass at 2.2 GHz.  P V under the exponentials of the granule behind (1 - 2 % and a fifth slower at head_dim 256), the next block's conversion under Q K,
// a barrier every second block, scales by vector loads and 64 rows a wave changed nothing or spilled.  Short calls pay beginning and end besides: 13 us to
// the first product (of which the queries take 9), 4 to 10 for the partial results and their merge.  (Ragged pair of chunks of 512 over 7680 keys: 116 - 127 us, by card.)
#pragma once
#include "intfa_paged_device.h"

namespace intfa {

constexpr float kPrefillShift = 8.f, kPrefillSlack = 6.f;      // P is held as up to 2^(8 + 6 + 1) p, within fp16
constexpr float kPartUnit = 0x1p-26f;       // partial rows are held as so much of the sums, whose factor is 2^8 to 2^14: those of 2^12 values fit fp32 wherever the values do
constexpr float kPrefillFar = 0x1p20f;      // a maximum of this size: scores are taken from it in a step of their own (its last place is 1/8 there)

template <int D> struct PrefillShape {
    static constexpr int WAVES = D == 128 ? 8 : 4, ROWS = 32 * WAVES, THREADS = 64 * WAVES, KEYS = 64;
    static constexpr int WGS = D == 64 ? 2 : 1;            // workgroups per compute unit
    static constexpr int K_ROW = 2 * D + 16, V_ROW = 2 * KEYS + 16;      // bytes in LDS (16 more: the banks)
    static constexpr int K_BYTES = KEYS * K_ROW, V_BYTES = D * V_ROW, BLOCK = K_BYTES + V_BYTES;
    static constexpr int UNITS = KEYS * D / 16 / THREADS;  // of sixteen bytes, for K and for V, per thread and block
    static constexpr int PASS = D == 256 ? 32 : 64;        // rows whose queries are staged at a time
    static_assert(UNITS >= 1 && UNITS * THREADS * 16 == KEYS * D, "");
};

// A block's bytes on their way, of one thread
template <int D> struct PrefillBytes {
    v4i k[PrefillShape<D>::UNITS];
    uint32_t v[PrefillShape<D>::UNITS][4];
};

// REST: rotated fp16 queries, whose scores take a second product (PagedQueries::stage).  Rotated bf16 queries stay rounded to 11 bits here, three more than
// they came with: a second product doubles Q K, which is half more matrix work, and its fragments have no room in the registers (head_dim 128: 73 spilled, or 59
// with small pages; 2 x 512 tokens over 30720 keys 554 us without it, 742 with it.  head_dim 256: make_plan).  ONE: a page holds a block's keys.
template <int D, int DT, bool REST, bool ONE>
__global__ void __launch_bounds__(PrefillShape<D>::THREADS, PrefillShape<D>::WGS * PrefillShape<D>::WAVES / 4) paged_prefill_kernel(const PagedParams) {
    typedef PrefillShape<D> S;
    constexpr int THREADS = S::THREADS, R = S::ROWS, KS = D / 16, DTILES = D / 32, G = 4, UNITS = S::UNITS, NB = D / 4;
    typedef PagedQueries<D, DT, S::PASS, THREADS> Queries;
    constexpr int ANGLES_AT = 2 * S::PASS * Queries::ROW;
    static_assert(ANGLES_AT + S::PASS * (D / 2) * 8 <= 2 * S::BLOCK, "the queries and their angles pass through the blocks' place");
    __shared__ __align__(16) char lds[2 * S::BLOCK];
    __shared__ float factor_lds[S::PASS];
    __shared__ uint32_t arrival_lds;
    __shared__ double freq_lds[D / 2];
    PagedArgs p = paged_args_first();
    PagedItem t;
    const double freq = paged_frequency(p);
    PagedPiece piece = paged_find(p, R, t);
    if ((int)threadIdx.x < D / 2) freq_lds[threadIdx.x] = freq;
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lq = lane & 31, lh = lane >> 5;
  while (piece.start < piece.end) {
    const PagedPart part = paged_part(p, t, piece);
    if (part.none) break;
    const int row0 = t.tile * R, row = row0 + 32 * wave + lq, token = paged_div(row, p->d_group);
    uint64_t ticket_seen = 0;
    if (!part.whole && threadIdx.x == 0) ticket_seen = __hip_atomic_load(paged_ticket(p, t), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // ---- queries: through LDS into the waves that own them
    v8h q[KS], q_rest[REST ? KS : 1];
    float factor = 0.f;
    if (part.key_first < part.key_end) {                   // (rows that see no key are zeros without it)
        Queries queries[R / S::PASS];
#pragma unroll
        for (int pass = 0; pass < R / S::PASS; ++pass) queries[pass].request(p, t, row0 + pass * S::PASS);
#pragma unroll
        for (int pass = 0; pass < R / S::PASS; ++pass) {
            if (pass > 0) __syncthreads();
            if (queries[pass].rope) {
                queries[pass].turn_angles(p, t, freq_lds, (v2f*)(lds + ANGLES_AT));
                __syncthreads();
            }
            queries[pass].template stage<REST>(p, row0 + pass * S::PASS, (const v2f*)(lds + ANGLES_AT), lds, lds + S::PASS * Queries::ROW, factor_lds);
            __syncthreads();
            if (32 * wave / S::PASS == pass) {
                const char* const mine = lds + (32 * wave % S::PASS + lq) * Queries::ROW + 16 * lh;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    q[ks] = *(const v8h*)(mine + 32 * ks);
                    if (REST) q_rest[REST ? ks : 0] = *(const v8h*)(mine + S::PASS * Queries::ROW + 32 * ks);
                }
                factor = factor_lds[32 * wave % S::PASS + lq];
            }
        }
    }
    // ---- where the keys come from
    const char* const k_head = p->k + t.hk * p->k_sh;
    const char* const v_head = p->v + t.hk * p->v_sh;
    const int32_t* const table = p->table + t.z * p->bt_sb;
    const PagedInts table_s = (PagedInts)table;
    const PagedFloats k_scale = (PagedFloats)(p->k_scale + t.hk * p->ks_sh), v_scale = (PagedFloats)(p->v_scale + t.hk * p->vs_sh);
    const int64_t k_sp = p->k_sp, v_sp = p->v_sp, ks_sp = p->ks_sp, vs_sp = p->vs_sp;
    const int k_sn = p->k_sn, v_sn = p->v_sn, page_log2 = p->page_log2, num_pages = p->num_pages, last_column = p->table_width - 1;
    const int page_mask = (1 << page_log2) - 1, most = part.key_end;
    auto column = [&](int key) __attribute__((always_inline)) { const int c = key >> page_log2; return c < last_column ? c : last_column; };
    // Table entries are requested two blocks ahead of the bytes and the scales that they lead to.  Nothing here is conditional: behind the last block the
    // last column's page is read again, so that the compiler can count what is under way.
    int k_id[UNITS], v_id[UNITS];                          // of a thread's own keys, where a block has several pages
    int s_id[ONE ? 1 : G];                                 // of the block's granules (scalars)
    auto look = [&](int key0) __attribute__((always_inline)) {
        if (ONE) return;
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = (int)threadIdx.x + i * THREADS;
            k_id[i] = table[column(key0 + u / (D / 16))];
            v_id[i] = table[column(key0 + 4 * (u / NB))];
        }
    };
    auto look_scalar = [&](int key0) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < (ONE ? 1 : G); ++g) s_id[g] = table_s[column(key0 + 16 * g)];
    };
    auto fetch = [&](int key0, int one_id, PrefillBytes<D>& b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = (int)threadIdx.x + i * THREADS, kk = u / (D / 16), vk = 4 * (u / NB);
            const int kid = ONE ? one_id : k_id[i], vid = ONE ? one_id : v_id[i];
            const char* const kp = k_head + ((unsigned)kid < (unsigned)num_pages ? kid : 0) * k_sp + (ONE ? (key0 & page_mask) * k_sn : 0);
            const char* const vp = v_head + ((unsigned)vid < (unsigned)num_pages ? vid : 0) * v_sp + (ONE ? (key0 & page_mask) * v_sn : 0);
            b.k[i] = *(const v4i*)(kp + (uint32_t)((ONE ? kk : (key0 + kk) & page_mask) * k_sn + 16 * (u % (D / 16))));
#pragma unroll
            for (int j = 0; j < 4; ++j) b.v[i][j] = *(const uint32_t*)(vp + (uint32_t)(((ONE ? vk : (key0 + vk) & page_mask) + j) * v_sn + 4 * (u % NB)));
        }
    };
    auto store = [&](const PrefillBytes<D>& b, char* block) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = (int)threadIdx.x + i * THREADS;
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) i8x4_to_f16((uint32_t)b.k[i][j], w[2 * j], w[2 * j + 1]);
            char* const kd = block + (u / (D / 16)) * S::K_ROW + 32 * (u % (D / 16));
            *(v4i*)kd = (v4i){(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
            *(v4i*)(kd + 16) = (v4i){(int)w[4], (int)w[5], (int)w[6], (int)w[7]};
            const int four = u / NB;                       // which four keys: 4 (2 j + h) of 16 t
            char* const vd = block + S::K_BYTES + (u % NB) * S::V_ROW + 32 * (four >> 2) + 16 * (four & 1) + 8 * ((four >> 1) & 1);
            auto quad = [&](auto bt) __attribute__((always_inline)) {
                constexpr int B = decltype(bt)::value;
                *(v2i*)(vd + B * NB * S::V_ROW) = (v2i){(int)i8_pair_to_f16<B>(b.v[i][0], b.v[i][1]), (int)i8_pair_to_f16<B>(b.v[i][2], b.v[i][3])};
            };
            static_for<4>(quad);
        }
    };
    // scales of a block, and whether the table names its pages (scalars, by the entries in s_id)
    struct Scales { float k[G], v[G]; bool has[G]; };
    auto scales_of = [&](int key0, Scales& s) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int id = s_id[ONE ? 0 : g];
            s.has[g] = (unsigned)id < (unsigned)num_pages && key0 + 16 * g < most;
            if (ONE && g > 0) {
                s.k[g] = s.k[0]; s.v[g] = s.v[0];
                continue;
            }
            const int at = (unsigned)id < (unsigned)num_pages ? id : 0;
            s.k[g] = k_scale[at * ks_sp];
            s.v[g] = v_scale[at * vs_sp];
        }
    };
    const int seen = paged_token_keys(p, t, token), least = paged_token_keys(p, t, t.first_token);
    v16f acc[DTILES];
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
    float m = -INFINITY, l = 0.f, v_unit = 0.f, v_peak = 0.f;      // v_unit: of the accumulators, from the first scale of values on
    bool far = false;                                      // the wave's: some row's maximum is past kPrefillFar
    int key0 = part.key_first;
    PrefillBytes<D> even, odd;
    Scales scales;
    int id_next = 0;                                       // (ONE) the page of the block behind the next one
    if (key0 < most) {
        look_scalar(key0);
        look(key0);
        fetch(key0, s_id[0], even);
        scales_of(key0, scales);
        look_scalar(key0 + 64);
        look(key0 + 64);
        fetch(key0 + 64, s_id[0], odd);
        look(key0 + 128);
        if (ONE) id_next = table_s[column(key0 + 128)];
    }
    if (!part.whole) paged_open_ticket(p, paged_ticket(p, t), ticket_seen);
    __syncthreads();                                       // (the queries have been read)
    if (key0 < most) store(even, lds);
    __syncthreads();
    auto block = [&](const char* now, char* then, PrefillBytes<D>& next, PrefillBytes<D>& after) __attribute__((always_inline)) {
        // `next` holds the bytes of the block behind this one, `after` takes those of the one behind that
        fetch(key0 + 128, id_next, after);
        const Scales sc = scales;
        scales_of(key0 + 64, scales);
        if (ONE) s_id[0] = id_next;
        else look_scalar(key0 + 128);
        look(key0 + 192);
        if (ONE) id_next = table_s[column(key0 + 192)];
        store(next, then);
        // The matrix pipe waits for no LDS read: four fragments are under way while the products of four others run.
        v16f s[2];
        v8h kf[2][4];
        const char* const kl = now + lq * S::K_ROW + 16 * lh;
        auto read_k = [&](int quad, v8h (&f)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = *(const v8h*)(kl + 32 * (quad / (KS / 4)) * S::K_ROW + 32 * (4 * (quad % (KS / 4)) + i));
        };
        read_k(0, kf[0]);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
#pragma unroll
        for (int quad = 0; quad < KS / 2; ++quad) {
            if (quad + 1 < KS / 2) read_k(quad + 1, kf[(quad + 1) % 2]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int half = quad / (KS / 4), ks = 4 * (quad % (KS / 4)) + i;
                s[half] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[quad % 2][i], q[ks], s[half], 0, 0, 0);
                if (REST) s[half] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[quad % 2][i], q_rest[REST ? ks : 0], s[half], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // ---- hidden keys
        bool masked = key0 + 64 > least;
#pragma unroll
        for (int g = 0; g < G; ++g) masked = masked || !sc.has[g];
        if (masked) {
            const int last = seen - key0 - 4 * lh;           // of the lane's keys: 16 g + 8 j + i is hidden from here on
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int end = sc.has[g] ? last : 0;
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const int e = 8 * (g % 2) + r;
                    s[g / 2][e] = 16 * g + 8 * (r / 4) + r % 4 < end ? s[g / 2][e] : -INFINITY;
                }
            }
        }
        // ---- V's unit: the page's scale, or the largest of the block's
        float v_top = sc.has[0] ? sc.v[0] : 0.f;
        if (!ONE) {
#pragma unroll
            for (int g = 1; g < G; ++g) v_top = fmaxf(v_top, sc.has[g] ? sc.v[g] : 0.f);
        }
        v_top = v_top < 0x1p-120f ? 0.f : v_top;             // (its reciprocal would be none; the append leaves none under 2^-100)
        v_peak = fmaxf(v_peak, v_top);
        if (v_top > 2.f * v_unit || v_top < 0x1p-4f * v_unit) {      // (P, within 2^-4 .. 2 of its own size, has 11 bits down to p = 2^-18)
            const float unit = fmaxf(fmaxf(v_top, v_peak * 0x1p-60f), 0x1p-100f), scale = v_unit / unit;
            v_unit = unit;
#pragma unroll
            for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[dt][r] *= scale;
        }
        // (a ratio under 2^-100, of pages of zeros beside large values, say, counts as that: its reciprocal would be none)
        const float v_ratio = v_top > 0.f ? fmaxf(v_top * __builtin_amdgcn_rcpf(v_unit), 0x1p-100f) : 1.f, v_log = __builtin_amdgcn_logf(v_ratio), v_back = __builtin_amdgcn_rcpf(v_ratio);
        // ---- softmax
        float f[G];
#pragma unroll
        for (int g = 0; g < G; ++g) f[g] = fmaxf(factor * (ONE ? sc.k[0] : sc.k[g]), 0x1p-126f);      // (never zero: hidden keys are -infinity times it)
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float raw = -INFINITY;
#pragma unroll
            for (int r = 0; r < 8; ++r) raw = fmaxf(raw, s[g / 2][8 * (g % 2) + r]);
            top = fmaxf(top, raw * f[g]);
        }
        top = half_pair_max(top);
        if (__any(top - m > kPrefillSlack)) {                // (the difference is exact where it matters, m + 6 is not)
            const float grown = fmaxf(m, top), alpha = grown == -INFINITY ? 1.f : fast_exp2(m - grown);
            m = grown;
            far = __any(m > kPrefillFar || (m < -kPrefillFar && m > -INFINITY));
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[dt][r] *= alpha;
        }
        // The exponent is one multiply-add of the score.  Far from zero its rounding, and that of the products which the maximum was taken of, would grow past
        // what fp16 has room for: there the scores become differences from the maximum first, by the same products.
        const float base = m == -INFINITY ? 0.f : m;
        if (__builtin_expect(far, 0)) {
#pragma clang fp contract(off)
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int r = 0; r < 8; ++r) s[g / 2][8 * (g % 2) + r] = s[g / 2][8 * (g % 2) + r] * f[g] - base;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) f[g] = far ? 1.f : f[g];      // (chosen here and not in the branch: head_dim 256, 2 x 512 tokens over 30720 keys, 2060 -> 1729 us)
        const float frame = (far ? 0.f : base) - kPrefillShift - v_log;
        float sum = 0.f;
        v8h pf[4];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const float rel = ONE || v_top <= 0.f ? 1.f : (sc.has[g] ? sc.v[g] : 0.f) * __builtin_amdgcn_rcpf(v_top);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float e = fast_exp2(fmaf(s[g / 2][8 * (g % 2) + r], f[g], -frame));
                sum += e;
                if (!ONE) e *= rel;
                pf[g][r] = (_Float16)e;
            }
        }
        l = fmaf(sum, v_back, l);
        // ---- O^T += V^T P^T
        if (v_top > 0.f) {
            v8h vf[2][4];
            const char* const vl = now + S::K_BYTES + lq * S::V_ROW + 16 * lh;
            auto read_v = [&](int dt, v8h (&f)[4]) __attribute__((always_inline)) {
#pragma unroll
                for (int g = 0; g < 4; ++g) f[g] = *(const v8h*)(vl + 32 * dt * S::V_ROW + 32 * g);
            };
            read_v(0, vf[0]);
#pragma unroll
            for (int dt = 0; dt < DTILES; ++dt) {
                if (dt + 1 < DTILES) read_v(dt + 1, vf[(dt + 1) % 2]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int g = 0; g < 4; ++g) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[dt % 2][g], pf[g], acc[dt], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        key0 += 64;
        __syncthreads();
    };
    while (key0 < most) {
        block(lds, lds + S::BLOCK, odd, even);
        if (key0 >= most) break;
        block(lds + S::BLOCK, lds, even, odd);
    }
    p = paged_args();
    l = half_pair_sum(l);
    // ---- a lane's values: columns 4 (8 a + 4 lh + i) + b of its row, b = 0 .. 3 from as many tiles
    auto value = [&](int a, int i) __attribute__((always_inline)) {
        v4f x;
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = acc[(b * NB + 8 * a) / 32][4 * ((b * NB / 8 + a) % 4) + i];
        return x;
    };
    bool done = part.whole;
    float weight = v_unit;                                 // of the accumulators
    if (!part.whole) {
        const PagedParts mine(p, R, D, (int)part.slot);
#pragma unroll
        for (int a = 0; a < D / 32; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i) mine.put((uint32_t)(32 * wave), D, 4 * (64 * (4 * a + i) + lane), value(a, i) * (v_unit * kPartUnit));      // (a wave's stores: 1 KB each)
        if (lh == 0) mine.put_stats((uint32_t)(32 * wave + lq), m, l);
        if (paged_last_arrival(p, paged_ticket(p, t), &arrival_lds, part.pieces)) {
            // the pieces in their order, each wave its own rows in its own layout
            typedef unsigned v2u __attribute__((ext_vector_type(2)));
            done = true;
            weight = 1.f / kPartUnit;
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
            for (int k = 0; k < part.pieces; ++k) {
                const int slot = 2 * (part.one + k) + (k == 0 && !part.first_is_first);
                const BufferRsrc o = __builtin_amdgcn_make_buffer_rsrc(p->parts + (int64_t)slot * R * D, 0, R * D * 4, 0x00020000);
                const BufferRsrc st = __builtin_amdgcn_make_buffer_rsrc(p->part_stats + (int64_t)slot * R * 2, 0, R * 8, 0x00020000);
                const uint32_t r0 = (uint32_t)(32 * wave + lq);
                const v2u ml = __builtin_amdgcn_raw_buffer_load_b64(st, r0 * 8u, 0, kSplitAux);
                const float mk = __builtin_bit_cast(float, (unsigned)ml[0]), top = fmaxf(m, mk), base = top == -INFINITY ? 0.f : top;
                const float alpha = fast_exp2(m - base), w = fast_exp2(mk - base);
                l = l * alpha + w * __builtin_bit_cast(float, (unsigned)ml[1]);
                m = top;
#pragma unroll
                for (int a0 = 0; a0 < D / 32; a0 += 2) {
                    v4f x[2][4];
#pragma unroll
                    for (int a = a0; a < a0 + 2; ++a)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            x[a - a0][i] = __builtin_bit_cast(v4f, __builtin_amdgcn_raw_buffer_load_b128(o, ((uint32_t)(32 * wave * D) + 4u * (uint32_t)(64 * (4 * a + i) + lane)) * 4u, 0, kSplitAux));
#pragma unroll
                    for (int a = a0; a < a0 + 2; ++a)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                const int dt = (b * NB + 8 * a) / 32, r = 4 * ((b * NB / 8 + a) % 4) + i;
                                acc[dt][r] = alpha * acc[dt][r] + w * x[a - a0][i][b];
                            }
                    asm volatile("" ::: "memory");         // (these before the next ones are requested: room for all of a row is not there)
                }
            }
        }
    }
    if (done && row < p->rows) {
        const bool empty = m == -INFINITY || token >= t.m;
        const float inv = empty ? 0.f : weight / l;
        const int head = t.hk * p->group + row - token * p->group;
        char* const dst = p->out + t.z * p->o_sb + head * p->o_sh + token * p->o_sn + 32 * lh;
#pragma unroll
        for (int a = 0; a < D / 32; ++a)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v4f x = value(a, i) * inv;
                if (token >= t.m) x = (v4f){0.f, 0.f, 0.f, 0.f};
                store_out4<DT>(dst + 64 * a + 8 * i, x);
            }
        if (p->lse != nullptr && lh == 0)
            p->lse[((int64_t)t.z * p->heads + head) * p->seqlen + token] = token >= t.m ? -INFINITY : m + __builtin_log2f(l) - kPrefillShift;      // (as in intfa_paged_decode.h)
    }
    if (!paged_next(p, R, t, piece)) break;
    __syncthreads();
  }
}

template <int D> int launch_paged_prefill(const PagedParams& p, const PagedSel& sel, hipStream_t stream) {
    const dim3 grid((unsigned)p.grid), threads(PrefillShape<D>::THREADS);
#define INTFA_CALL(DT, REST) do { \
        if (sel.one_page) hipLaunchKernelGGL((paged_prefill_kernel<D, DT, REST, true>), grid, threads, 0, stream, p); \
        else hipLaunchKernelGGL((paged_prefill_kernel<D, DT, REST, false>), grid, threads, 0, stream, p); } while (0)
    if (sel.io_dt == 1) INTFA_CALL(1, false); else if (D < 256 && p.rope.freqs != nullptr) INTFA_CALL(0, (D < 256)); else INTFA_CALL(0, false);
#undef INTFA_CALL
    return (int)hipGetLastError();
}

}  // namespace intfa
