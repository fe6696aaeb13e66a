// Attention over a paged cache of latent vectors (absorbed queries): keys are the whole rows of the cache, values their latent part, for all heads.
//
// A workgroup takes a tile of 32 or 64 query rows and a range of keys in blocks of 64, which come into a ring of four LDS stages by asynchronous copies, as int8, once.
// Of its eight waves four form scores and weights (one a SIMD), and four multiply the weights of the block before with its values, so that one half's
// exponentials run under the other's products.
//   S^T = K Q^T    in int8.  A query row is held as whole steps of 1/32512 of its largest element, in two bytes: two products, whose sums 256 hi + lo are exact in
//                  32 bits (512 x 128 x 32640 < 2^31).  That takes the time of one fp16 product, leaves the keys as they are, and halves what is read from LDS.
//   O^T = V^T P^T  in fp16: P has a range that eight bits have not.  V's bytes are read transposed (ds_read_b64_tr_b8) and converted exactly; each wave has a quarter of
//                  the columns for all rows, so that no byte is converted twice.  P goes through LDS in the operand's own layout.
// A token's value scale s goes into the exponent: rows follow the maximum of t = score + log2 s, P = 2^(t - frame), and the sum of weights is that of P / s.  Whatever the
// scales' sizes, P is within fp16 and the accumulators are plain sums of int8 numbers times P; the output is their quotient.
// Measured, latent part 512 and rotary part 64: 16 heads of 256 requests over 4096 tokens 101 us with the merge, 6.1 TB/s (memory; the same pages over and over would be 86);
// 128 heads of 32 requests 54 us and 10 of merging, 670 TFLOP/s without it (4560 clocks a block of 64 rows, where products take 2176 and vector instructions 1840: two waves a SIMD, in order, hide little of either
// under the other).  Tiles of 32 rows are for few rows, and where there is little work (make_plan): 16 of their rows cost what 32 do in the values' product, which is not what bounds few rows.
#pragma once
#include "intfa_latent_host.h"
#include "intfa_paged_device.h"

namespace intfa {

typedef const __attribute__((address_space(4))) LatentParams* LatentArgs;
__device__ __forceinline__ LatentArgs latent_args() {
    LatentArgs p = (LatentArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// P = 2^(t - m + kLatentShift), and up to 2^kLatentSlack more before a row's m follows: at most 2^15, and 11 bits down to 2^-25 of the row's largest.
constexpr float kLatentShift = 11.f, kLatentSlack = 4.f;
// Scales enter scores as 2^-20 of themselves and the query's step as 2^20 of itself: products of up to 2^31 with scales of up to 2^117 fit.
constexpr float kScoreUnit = 0x1p-20f;
// Weights are summed as 2^-18 of themselves: a term P / s is at most 2^97 (of s = 2^-100), and 2^30 keys fit; a row's largest is at least 2^-124 (its frame goes by another key, of s = 2^117),
// where fp32 still has steps of 2^-25 of it.
constexpr float kWeightLog = 18.f, kWeightUnit = 0x1p-18f;
// P / s is P times a key's 1 / s, short of keys that lie so far under the row's frame, for their scale alone, that P leaves fp32 and P / s does not.  Where no scale that an item
// has met is over this, those have weights of less than 2^-33 of the row's largest; from the first larger one on (latent vectors of 2000 and more) a second exponential, of the
// score alone, takes the place of the product.
constexpr float kLargeScale = 16.f;
constexpr float kQuerySteps = 32512.f;         // 127 * 256: the high byte of a step count rounds to at most 127

// What the scale of a token on a page that the table does not name is read from
static __device__ const float kHiddenScale[32] = {-1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1, -1};

// Sums of weights follow their row's frame, which the scales alone may move by 2^217.  A factor 2^d of one exponential ends at 2^-126: where it goes further than kOneFactor, it
// is taken in two.  (Seldom: what checks for it does so for a wave, and for several factors at a time.)
constexpr float kOneFactor = -125.f;
__device__ __forceinline__ float add_moved(float sum, float a, float d) {
    const bool far = d < kOneFactor;
    return fmaf(fast_exp2(far ? kOneFactor : d), a * fast_exp2(far ? d - kOneFactor : 0.f), sum);
}
// sum + 2^x, down to fp32's last place (the exponential itself ends at 2^-126)
__device__ __forceinline__ float add_exp2(float sum, float x) {
    const float e = fast_exp2(0.5f * x);
    return fmaf(e, e, sum);
}
__device__ __forceinline__ float log2_of_weights(float sum) { return sum < 0x1p100f ? __builtin_log2f(sum * (1.f / kWeightUnit)) : __builtin_log2f(sum) + kWeightLog; }

template <int DC, int DR, int ROWS> struct LatentShape {
    static constexpr int ROW = DC + DR, UNITS = ROW / 16, LATENT_UNITS = DC / 16, KEYS = 64, THREADS = 512;
    static constexpr int RG = ROWS / 32, KG = 4 / RG;          // groups of 32 rows; waves that share a group's keys
    static constexpr int STAGE = KEYS * ROW, STAGES = 4;
    static constexpr int WHOLE = UNITS / 4, HALF = UNITS % 4 / 2;      // asynchronous copies of a wave and stage, of 64 and of 32 lanes: its 16 rows
    static constexpr int COPIES = WHOLE + HALF + 1;            // ... and their scales
    static_assert(UNITS % 4 == 0 || UNITS % 4 == 2, "");
    // The first blocks come into the first stages while the queries' bytes are in the last one or two.  The angles are behind the tiles, or, of 64 wide rows, in the second stage.
    static constexpr int QUERY_BYTES = ROWS * 2 * ROW, QUERY_AT = (STAGES - (QUERY_BYTES + STAGE - 1) / STAGE) * STAGE, QUERY_END = QUERY_AT + QUERY_BYTES, ANGLES = ROWS * (DR / 2) * 8;
    static constexpr bool ANGLES_IN = ROWS == 64 && DC == 512;
    static_assert(!ANGLES_IN || ANGLES <= STAGE, "");
    static_assert(QUERY_AT >= (ROWS == 32 ? 3 : 2) * STAGE, "copies of the first steps would meet the queries");
    static constexpr int TILES_END = STAGES * STAGE > QUERY_END ? STAGES * STAGE : QUERY_END, ANGLES_AT = ANGLES_IN ? STAGE : TILES_END;
    static constexpr int P_AT = ANGLES_IN ? TILES_END : TILES_END + ANGLES, P_BYTES = ROWS * KEYS * 2;
    static constexpr int SCALES_AT = P_AT + P_BYTES, SCALE_STAGE = KEYS * 8;
    static constexpr int ALPHA_AT = SCALES_AT + STAGES * SCALE_STAGE;      // [2][ROWS] factor of a row's accumulators, by the block's parity; then what the waves tell each other
    static constexpr int TOPS_AT = ALPHA_AT + 2 * ROWS * 4;                    // [KG][ROWS]
    static constexpr int FLAGS_AT = TOPS_AT + KG * ROWS * 4;               // [4]
    static constexpr int FREQS_AT = FLAGS_AT + 16, LDS = FREQS_AT + (DR / 2) * 8;
    static_assert(LDS <= 160 * 1024, "");
    static constexpr int CT = DC / 32, NT = CT / 4;            // column tiles of 32; of a wave
    // Where unit u of sixteen bytes of row m lies in its row.  Bank by bank: rows are 16 (rotary part of 64) or 8 words (of 32) past a multiple of 64, or such multiples that as few
    // consecutive rows meet; reads take one unit of sixteen consecutive rows (keys), or two neighbouring ones of rows 0 - 3 and 8 - 11 (+ 4) (values).
    static __device__ __forceinline__ int place(int u, int m) {
        if (DR == 64) return u ^ ((m >> 2) & 3);
        const int b = (m >> 3) & 1;
        return u ^ (u < LATENT_UNITS && LATENT_UNITS >= 16 ? 9 * b : b);
    }
};

__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// A wave's copies of a stage: N times 64 x 16 bytes from base + each lane's offset to consecutive KB of LDS from `lds` on (the last one of 32 lanes, if HALF), without a register on the
// way.  (As the copies of intfa_device.h: M0 is nobody else's.  One statement, which counts M0 on: with one each, the compiler keeps a scalar for every place of every stage, in lanes
// of vector registers.)  NT: past the caches, for rows that one workgroup alone reads (256 x 16 heads over 4096 tokens 117 -> 104 us, 5.9 TB/s; but 32 x 128 heads, whose two tiles of
// rows share them, 66 -> 70).
#define INTFA_COPY(o, nt) "\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tglobal_load_lds_dwordx4 " o ", %1" nt
#define INTFA_COPIES(nt) \
    if constexpr (N == 1) asm volatile(INTFA_FIRST(nt) :: "s"(lds), "s"(base), "v"(o[0]) : "memory"); \
    else if constexpr (N == 2) asm volatile(INTFA_FIRST(nt) INTFA_COPY("%3", nt) :: "s"(lds), "s"(base), "v"(o[0]), "v"(o[1]) : "memory", "scc"); \
    else if constexpr (N == 3) asm volatile(INTFA_FIRST(nt) INTFA_COPY("%3", nt) INTFA_COPY("%4", nt) :: "s"(lds), "s"(base), "v"(o[0]), "v"(o[1]), "v"(o[2]) : "memory", "scc"); \
    else if constexpr (N == 4) \
        asm volatile(INTFA_FIRST(nt) INTFA_COPY("%3", nt) INTFA_COPY("%4", nt) INTFA_COPY("%5", nt) :: "s"(lds), "s"(base), "v"(o[0]), "v"(o[1]), "v"(o[2]), "v"(o[3]) : "memory", "scc"); \
    else if constexpr (N == 5) \
        asm volatile(INTFA_FIRST(nt) INTFA_COPY("%3", nt) INTFA_COPY("%4", nt) INTFA_COPY("%5", nt) INTFA_COPY("%6", nt) \
                     :: "s"(lds), "s"(base), "v"(o[0]), "v"(o[1]), "v"(o[2]), "v"(o[3]), "v"(o[4]) : "memory", "scc"); \
    else if constexpr (N == 8) \
        asm volatile(INTFA_FIRST(nt) INTFA_COPY("%3", nt) INTFA_COPY("%4", nt) INTFA_COPY("%5", nt) INTFA_COPY("%6", nt) INTFA_COPY("%7", nt) INTFA_COPY("%8", nt) INTFA_COPY("%9", nt) \
                     :: "s"(lds), "s"(base), "v"(o[0]), "v"(o[1]), "v"(o[2]), "v"(o[3]), "v"(o[4]), "v"(o[5]), "v"(o[6]), "v"(o[7]) : "memory", "scc"); \
    else \
        asm volatile(INTFA_FIRST(nt) INTFA_COPY("%3", nt) INTFA_COPY("%4", nt) INTFA_COPY("%5", nt) INTFA_COPY("%6", nt) INTFA_COPY("%7", nt) INTFA_COPY("%8", nt) INTFA_COPY("%9", nt) INTFA_COPY("%10", nt) \
                     :: "s"(lds), "s"(base), "v"(o[0]), "v"(o[1]), "v"(o[2]), "v"(o[3]), "v"(o[4]), "v"(o[5]), "v"(o[6]), "v"(o[7]), "v"(o[8]) : "memory", "scc")
#define INTFA_FIRST(nt) "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %1" nt
template <bool NT, int N> __device__ __forceinline__ void copy_rows(const char* base, const uint32_t (&o)[N], uint32_t lds) {
    static_assert((N >= 1 && N <= 5) || N == 8 || N == 9, "");
    if constexpr (NT) { INTFA_COPIES(" nt"); } else { INTFA_COPIES(""); }
}
#undef INTFA_COPY
#undef INTFA_FIRST
#undef INTFA_COPIES
// 64 x 16 bytes and 64 x 4 alone
__device__ __forceinline__ void copy_units(const char* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "s"(lds), "v"(off), "s"(base) : "memory");
}
// 64 x 16 bytes to lds + at.  how: 0 none, 1 so, 2 past the caches.  (The branches are the statement's own: among the products, a branch of the compiler's costs it its schedule.)
__device__ __forceinline__ void copy_units_if(int how, const char* base, uint32_t off, uint32_t lds, int at) {
    asm volatile("s_cmp_eq_u32 %4, 0\n\ts_cbranch_scc1 .Lskip_copy%=\n\ts_add_u32 m0, %0, %3\n\ts_cmp_eq_u32 %4, 1\n\ts_cbranch_scc1 .Lcached_copy%=\n\t"
                 "global_load_lds_dwordx4 %1, %2 nt\n\ts_branch .Lskip_copy%=\n.Lcached_copy%=:\n\tglobal_load_lds_dwordx4 %1, %2\n.Lskip_copy%=:"
                 :: "s"(lds), "v"(off), "s"(base), "i"(at), "s"(how) : "memory", "scc");
}
__device__ __forceinline__ void copy_words(const char* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" :: "s"(lds), "v"(off), "s"(base) : "memory");
}
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" :: "i"(N) : "memory"); }

// Eight step counts x * steps, rounded, as their high bytes and what is left of them (-128 .. 127) as low bytes
__device__ __forceinline__ void split_steps(const float (&x)[8], float steps, v2i& hi, v2i& lo) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(uint32_t, fmaf(x[4 * w + i], steps, 12582912.f + 128.f));      // count + 128 in the low 16 bits
        hi[w] = (int)(__builtin_amdgcn_perm(u[1], u[0], 0x0c0c0501u) | __builtin_amdgcn_perm(u[3], u[2], 0x05010c0cu));
        lo[w] = (int)((__builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u) | __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu)) ^ 0x80808080u);
    }
}

// A tile's query rows on their way: all threads take part, 512 / ROWS of them a row, each with units of eight elements.  Their bytes go to LDS, from where the scoring waves take them
// as operands.  (Formed by the lanes that hold them, from rows copied to LDS, the code was 1300 instructions of straight line, read from memory in each launch: 64 rows of 576 elements
// took 42 000 clocks until their first product, and 13 000 so.)
template <int DC, int DR, int DT, int ROWS> struct LatentQueries {
    typedef LatentShape<DC, DR, ROWS> S;
    static constexpr int T = S::THREADS / ROWS, N = DC / 8 / T, RU = DR / 8;
    static_assert(RU <= T && DC % (8 * T) == 0, "");
    v4i x[N], rope, other;
    int row, unit, token;
    __device__ __forceinline__ void load(LatentArgs p, const PagedItem& t, int row0, int tid) {
        const auto& d = p->deal;
        row = tid / T;
        unit = tid % T;
        const int r = row0 + row < d.rows ? row0 + row : d.rows - 1;
        token = paged_div(r, d.d_group);
        const int head = r - token * d.group, u = unit % RU;
        const char* const latent = d.q + t.z * d.q_sb + head * d.q_sh + token * d.q_sn + 16 * unit;
        const char* const rotary = p->q_rope + t.z * p->qr_sb + head * p->qr_sh + token * p->qr_sn;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = *(const v4i*)(latent + 16 * T * i);
        rope = *(const v4i*)(rotary + 16 * u);
        other = rope;
        if (d.rope.freqs != nullptr && !d.rope.interleaved) {
            const int half = d.rope.pairs / 8;
            other = *(const v4i*)(rotary + 16 * (u >= 2 * half ? u : u >= half ? u - half : u + half));
        }
    }
    // angles: (cos, sin) of the pairs, of the tokens from first_token on.  The row's factor: of the integer sums times kScoreUnit * scale; NaN for a row that holds no number.
    __device__ __forceinline__ void form(LatentArgs p, char* lds, const v2f* angles, int first_token, float* factors) {
        const auto& d = p->deal;
        const int u = unit % RU, pairs = d.rope.freqs != nullptr ? d.rope.pairs : 0;
        float turned[8];
        unpack8<DT>(rope, turned);
        if (8 * u < 2 * pairs) {               // (pairs are a multiple of eight: eight elements turn alike)
            const bool second = 8 * u >= pairs;
            const v2f* const mine = angles + (token - first_token) * pairs;
            if (d.rope.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; ++i) rope_turn(turned[2 * i], turned[2 * i + 1], mine[4 * u + i][0], mine[4 * u + i][1]);
            } else {
                float y[8];
                unpack8<DT>(other, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const v2f a = mine[8 * u - (second ? pairs : 0) + i];
                    turned[i] = turned[i] * a[0] + y[i] * (second ? a[1] : -a[1]);
                }
            }
        }
        // (magnitudes of numbers are ordered as their bits are)
        typedef unsigned short v2us __attribute__((ext_vector_type(2)));
        v2us most = {0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(v2us, x[i][w] & 0x7fff7fff));
        float y[8];
        unpack8<DT>((v4i){__builtin_bit_cast(int, most), 0, 0, 0}, y);
        uint32_t top = __builtin_bit_cast(uint32_t, y[0]), other_top = __builtin_bit_cast(uint32_t, y[1]);
        top = top > other_top ? top : other_top;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t a = __builtin_bit_cast(uint32_t, turned[i]) & 0x7fffffffu;
            top = top > a ? top : a;
        }
#pragma unroll
        for (int w = 1; w < T; w <<= 1) {
            const uint32_t a = (uint32_t)__shfl_xor((int)top, w);
            top = top > a ? top : a;
        }
        const float size = fmaxf(__builtin_bit_cast(float, top), 0x1p-100f);      // (a row under it: its scores are nothing)
        const float steps = copysignf(kQuerySteps / size, d.qk_scale_log2);
        if (unit == 0) factors[row] = top < 0x7f800000u ? size * (1.f / kQuerySteps) * (fabsf(d.qk_scale_log2) * (1.f / kScoreUnit)) : __builtin_nanf("");
        char* const to = lds + S::QUERY_AT + row * S::ROW;
        auto put = [&](int at, const float (&e)[8]) __attribute__((always_inline)) {       // at: unit of eight
            v2i hi, lo;
            split_steps(e, steps, hi, lo);
            char* const dst = to + 16 * S::place(at / 2, row) + 8 * (at & 1);
            *(v2i*)dst = hi;
            *(v2i*)(dst + ROWS * S::ROW) = lo;
        };
#pragma unroll
        for (int i = 0; i < N; ++i) {
            unpack8<DT>(x[i], y);
            put(unit + T * i, y);
        }
        if (unit < RU) put(DC / 8 + unit, turned);
    }
};

// A lane's scales of one key: of scores (latent and rotary part, times kScoreUnit), log2 of the value's, and its reciprocal times kWeightUnit
struct LatentScale { float c, r, log, inv; };
__device__ __forceinline__ LatentScale latent_scale(float c, float r, bool beyond) {
    LatentScale s;
    const bool hidden = beyond || c < 0.f;
    const float v = fmaxf(c, 0x1p-100f);
    s.c = hidden ? 0.f : c * kScoreUnit;
    s.r = hidden ? 0.f : r * kScoreUnit;
    s.log = hidden ? -INFINITY : __builtin_amdgcn_logf(v);
    s.inv = hidden ? 0.f : kWeightUnit * __builtin_amdgcn_rcpf(v);
    return s;
}

// What takes log2 of the value's scale out of an exponent again, and the weights' unit in (0 for a hidden key: its exponent is -infinity)
__device__ __forceinline__ float less_log(float c, bool beyond) { return beyond || c < 0.f ? 0.f : -__builtin_amdgcn_logf(fmaxf(c, 0x1p-100f)) - kWeightLog; }

// Scales that come as lanes of a register (scale_lane_key), in the instruction that uses them: c = f * scale, c += scale of the lane's i-th key.  (Hand-written as fmac_lane_scale:
// the compiler takes sixteen copies of the register first, which have no room here.)
__device__ __forceinline__ float mul_lane_scale(float f, float scales, int i) {
    float c;
    asm("v_mul_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "=v"(c) : "v"(scales), "v"(f), "i"(i));
    return c;
}
__device__ __forceinline__ float add_lane_scale(float f, float scales, int i) {
    float c;
    asm("v_add_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "=v"(c) : "v"(scales), "v"(f), "i"(i));
    return c;
}
__device__ __forceinline__ void fmac_lane_scale_f(float& c, float scales, float f, int i) {
    asm("v_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "+v"(c) : "v"(scales), "v"(f), "i"(i));
}
// (f: of an exponential just ahead, which needs a wait state to its first reader; the compiler does not see a reader here)
__device__ __forceinline__ void fmac_lane_scale_exp(float& c, float scales, float f, int i) {
    asm("s_nop 0\n\tv_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "+v"(c) : "v"(scales), "v"(f), "i"(i));
}

// QT: tiles of 16 rows that the scores of a tile of 32 are formed for (the second one may be empty)
template <int DC, int DR, int DT, int ROWS, int QT>
__global__ void __launch_bounds__(512, 2) latent_attn_kernel(const LatentParams) {
    typedef LatentShape<DC, DR, ROWS> S;
    constexpr int RG = S::RG, KG = S::KG, NT = S::NT, KEYS = S::KEYS, STAGES = S::STAGES;
    constexpr bool SMALL = ROWS == 32;         // scores in tiles of 16 keys by 16 rows: a wave has 16 keys of a block; else of 32 by 32
    constexpr int STEP = SMALL ? 64 : 32;
    static_assert(SMALL || (QT == 1 && RG == 2), "");
    // The copies are the scoring waves' with few rows, which would wait for half of their time else (256 x 16 heads over 4096 tokens 106 us with the others' copies, 100 so), and
    // the others' with 64, among their products.
    constexpr bool SCORES_COPY = SMALL;
    constexpr int KC = DC / STEP, KR = (DR + STEP - 1) / STEP, KS = KC + KR;      // steps of the score's products: latent part, rotary part
    typedef LatentQueries<DC, DR, DT, ROWS> Queries;
    __shared__ __align__(16) char lds[S::LDS];
    LatentArgs p = latent_args();
    PagedArgs deal = paged_args_first();
    PagedItem t;
    const double freq = paged_frequency(deal);
    PagedPiece piece = paged_find(deal, ROWS, t);
    if ((int)threadIdx.x < DR / 2) ((double*)(lds + S::FREQS_AT))[threadIdx.x] = freq;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) & 3;      // (of its half)
    const bool scoring = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) < 4;
    const int rg = SMALL ? 0 : wave % RG, kg = SMALL ? wave : wave / RG;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    float* const tops = (float*)(lds + S::TOPS_AT);
    float* const alphas = (float*)(lds + S::ALPHA_AT);
    int* const flags = (int*)(lds + S::FLAGS_AT);
    v4i open = {0, 0, 0, 0};
    __syncthreads();
  while (piece.start < piece.end) {
    int tid = (int)threadIdx.x;
    asm volatile("" : "+v"(tid));              // (the lanes' many places are found again for each item: held beside each other from the kernel's start, they spill)
    const int lane = tid & 63, lq = lane & 31, lh = lane >> 5, x16 = lane & 15, c16 = lane >> 4;
    const PagedPart part = paged_part(deal, t, piece);
    if (part.none) break;
    const int row0 = t.tile * ROWS, most = part.key_end, key_first = part.key_first;
    const int blocks = most > key_first ? (most - key_first + KEYS - 1) / KEYS : 0;
    // Reads of rows of the tiles as operands: a fragment's place is one of two lane addresses and a constant (the permutation flips low bits of the unit's number, and for a
    // rotary part of 32 bit 3 as well).
    struct RowAt { int at[2], rope; };
    auto row_at = [&](int r, int unit) __attribute__((always_inline)) {
        return RowAt{{r * S::ROW + 16 * S::place(unit, r), r * S::ROW + 16 * S::place(unit + (DR == 32 ? 8 : 2), r)}, r * S::ROW + 16 * S::place(S::LATENT_UNITS + unit, r)};
    };
    auto fragment_at = [&](const RowAt& w, int k) __attribute__((always_inline)) {
        constexpr int UPF = SMALL ? 4 : 2;     // units of a fragment
        if (DR == 64) return SMALL ? w.at[0] + 64 * k : w.at[k & 1] + 64 * (k >> 1);
        if (k >= KC) return w.rope + 16 * UPF * (k - KC);
        const int bit = DR == 32 && S::LATENT_UNITS >= 16 ? UPF * k >> 3 & 1 : 0;
        return w.at[bit] + 16 * (UPF * k - 8 * bit);
    };
    // ======== copies: wave w of a half copies rows 16 w .. 16 w + 15 of every block
    const int k_sn = deal->k_sn;
    auto offset_of = [&](int i) __attribute__((always_inline)) {
        const int unit = 64 * i + lane, r = unit / S::UNITS < 16 ? unit / S::UNITS : 15, u = unit % S::UNITS;
        return (uint32_t)(r * k_sn + 16 * S::place(u, r));      // (the permutation is its own inverse)
    };
    uint32_t copy_off[S::WHOLE], copy_half = S::HALF ? offset_of(S::WHOLE) : 0u;
#pragma unroll
    for (int i = 0; i < S::WHOLE; ++i) copy_off[i] = offset_of(i);
    const uint32_t scale_off = (uint32_t)(((lane & 31) >> 1) * (int)deal->ks_sh * 4 + (lane & 1) * 4);
    // (what a copy needs of the arguments, held: loaded anew for each one, they are a chain of trips to the scalar cache)
    PagedInts table = (PagedInts)(deal->table + t.z * deal->bt_sb);
    const char* all_rows = deal->k;
    const float* all_scales = deal->k_scale;
    int64_t k_sp = deal->k_sp, ks_sp = deal->ks_sp;
    int page_log2 = deal->page_log2, last_column = deal->table_width - 1, num_pages = deal->num_pages, ks_sh = (int)deal->ks_sh;
    asm volatile("" : "+s"(table), "+s"(all_rows), "+s"(all_scales), "+s"(k_sp), "+s"(ks_sp), "+s"(page_log2), "+s"(last_column), "+s"(num_pages), "+s"(ks_sh));
    const int page_mask = (1 << page_log2) - 1;
    const bool streams = deal->tiles == 1;     // (nobody else reads these keys)
    auto look = [&](int block) __attribute__((always_inline)) {
        const int column = (key_first + KEYS * block + 16 * wave) >> page_log2;
        return table[column < last_column ? column : last_column];      // (behind the last key the table may hold anything)
    };
    struct BlockCopy { const char* rows; const char* scales; uint32_t to, scales_to; bool named; };
    auto block_copy = [&](int block, int id) __attribute__((always_inline)) {
        BlockCopy c;
        c.named = (unsigned)id < (unsigned)num_pages;
        const int at = c.named ? id : 0, row = (key_first + KEYS * block + 16 * wave) & page_mask, stage = block % STAGES;
        c.rows = all_rows + at * k_sp + row * k_sn;
        c.to = lds0 + (uint32_t)(stage * S::STAGE + wave * 16 * S::ROW);
        c.scales = c.named ? (const char*)(all_scales + at * ks_sp + row * ks_sh) : (const char*)kHiddenScale;
        c.scales_to = lds0 + (uint32_t)(S::SCALES_AT + stage * S::SCALE_STAGE + wave * 128);
        return c;
    };
    auto copy_rest = [&](const BlockCopy& c) __attribute__((always_inline)) {      // what is not copied 64 lanes at a time
        if (S::HALF && lane < 32) copy_units(c.rows, copy_half, c.to + 1024u * S::WHOLE);
        if (lane < 32) copy_words(c.scales, c.named ? scale_off : (uint32_t)lane * 4, c.scales_to);
    };
    constexpr int FIRST = (S::WHOLE + 1) / 2;
    auto copy_some = [&](const BlockCopy& c, auto second) __attribute__((always_inline)) {      // half of the whole ones
        constexpr int AT = decltype(second)::value ? FIRST : 0, N = decltype(second)::value ? S::WHOLE - FIRST : FIRST;
        uint32_t off[N];
#pragma unroll
        for (int i = 0; i < N; ++i) off[i] = copy_off[AT + i];
        if (streams) copy_rows<true>(c.rows, off, c.to + 1024u * AT);
        else copy_rows<false>(c.rows, off, c.to + 1024u * AT);
    };
    auto copy = [&](int block, int id) __attribute__((always_inline)) {
        const BlockCopy c = block_copy(block, id);
        if (streams) copy_rows<true>(c.rows, copy_off, c.to);
        else copy_rows<false>(c.rows, copy_off, c.to);
        copy_rest(c);
    };
    // ======== the queries, by all waves, while the first blocks come
    const bool early = blocks > 1 && (!S::ANGLES_IN || deal->rope.freqs == nullptr);      // (nothing else is in the second stage)
    {
        Queries queries;
        if (blocks > 0) {
            queries.load(p, t, row0, tid);
            if (SCORES_COPY ? scoring : !scoring) {
                copy(0, look(0));
                if (early) copy(1, look(1));
            }
            const int first_token = paged_div(row0, deal->d_group);
            if (deal->rope.freqs != nullptr) {     // the angles of the tile's tokens, each once
                const int last_row = row0 + ROWS < deal->rows ? row0 + ROWS - 1 : deal->rows - 1, pairs = deal->rope.pairs;
                const int angles = (paged_div(last_row, deal->d_group) - first_token + 1) * pairs;
                for (int i = tid; i < angles; i += S::THREADS) {
                    const int token = paged_div(i, deal->d_pairs), pair = i - token * pairs;
                    float c, s;
                    rope_angle(((const double*)(lds + S::FREQS_AT))[pair], t.n - t.m + first_token + token, deal->rope.magnitude, c, s);
                    ((v2f*)(lds + S::ANGLES_AT))[i] = (v2f){c, s};
                }
                lds_barrier();
            }
            queries.form(p, lds, (const v2f*)(lds + S::ANGLES_AT), first_token, alphas);
        }
        if (SCORES_COPY ? scoring : !scoring) {
            if (early) wait_copies<S::COPIES>(); else wait_copies<0>();
        }
        lds_barrier();                         // queries and first block are there
    }
    if (scoring) {
        // ======== scores and weights
        v4i query_hi[QT][KS], query_lo[QT][KS];
        float factor[QT];
        int seen[QT];
        const int least = paged_token_keys(deal, t, t.first_token);
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const int r = SMALL ? 16 * q + x16 : 32 * rg + lq, row = row0 + r < deal->rows ? row0 + r : deal->rows - 1, token = paged_div(row, deal->d_group);
            const RowAt at = row_at(r, SMALL ? c16 : lh);
            seen[q] = paged_token_keys(deal, t, token);
            factor[q] = alphas[r];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const bool in = DR % STEP == 0 || k < KC || c16 < DR / 16;      // (else the row's last step reaches behind it)
                query_hi[q][k] = *(const v4i*)(lds + S::QUERY_AT + fragment_at(at, k));
                query_lo[q][k] = *(const v4i*)(lds + S::QUERY_AT + ROWS * S::ROW + fragment_at(at, k));
                if (!in) query_hi[q][k] = query_lo[q][k] = (v4i){0, 0, 0, 0};
            }
        }
        const RowAt key_at = row_at(SMALL ? 16 * wave + x16 : 32 * kg + lq, SMALL ? c16 : lh);
        float m[QT], l[QT];
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            m[q] = -INFINITY;
            l[q] = 0.f;
        }
        if constexpr (!SMALL)
        {
            // A step forms the scores of block i + 1 while it takes the exponentials of block i: the first fragments' products run while the rows' maxima are settled, and with each of
            // the others come one or two of a lane's sixteen weights.
            constexpr int AHEAD = 3, EARLY = KC / 8 > 1 ? KC / 8 : 1;      // fragments ahead of the products; of the latent part ahead of the weights
            static_assert(KC >= 4, "");
            float s[16], inv = 0.f, e_last = 0.f;
            bool large = false;                // (of all waves alike)
            uint32_t w[4];
            auto element = [&](int j, float frame, int ln) __attribute__((always_inline)) {
                const float e = fast_exp2(s[j] - frame);
                fmac_lane_scale_exp(l[0], inv, e, j);
                if (j & 1) w[j % 8 / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){e_last, e}, v2h));
                else e_last = e;
                if (j % 8 == 7) *(v4i*)(lds + S::P_AT + ((rg * 4 + 2 * kg + j / 8) * 64 + ln) * 16) = (v4i){(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
            };
            // scores of block `next` (QK) beside the weights of the block before it (E)
            auto step = [&](auto qk_tag, auto e_tag, int next, int parity) __attribute__((always_inline)) {
                constexpr bool QK = decltype(qk_tag)::value, E = decltype(e_tag)::value;
                int ln = lane;
                asm volatile("" : "+v"(ln));   // (places that follow from it are found again in each step: kept, they push operands out of the registers)
                const int lq = ln & 31, lh = ln >> 5;
                const int tile = (next % STAGES) * S::STAGE, key0 = key_first + KEYS * next;
                v4i f[4];
                v16i hi, lo;
                auto fetch = [&](int k) __attribute__((always_inline)) {
                    if (QK && k < KS) f[k % 4] = *(const v4i*)(lds + tile + fragment_at(key_at, k));
                };
                auto product = [&](int k) __attribute__((always_inline)) {
                    fetch(k + AHEAD);
                    if (!QK) return;
                    const bool first = k == 0 || k == KC;
                    hi = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[k % 4], query_hi[0][k], first ? (v16i){0} : hi, 0, 0, 0);
                    lo = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[k % 4], query_lo[0][k], first ? (v16i){0} : lo, 0, 0, 0);
                };
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) fetch(k);
                float theirs[2];
                if (E) {                       // the rows' maxima: of the two waves that share a row's keys
                    theirs[0] = tops[32 * rg + lq];
                    theirs[1] = tops[ROWS + 32 * rg + lq];
                }
#pragma unroll
                for (int k = 0; k < EARLY; ++k) {
                    product(k);
                    __builtin_amdgcn_sched_barrier(0);
                }
                float frame = 0.f;
                if (E) {
                    const float top = fmaxf(theirs[0], theirs[1]);
                    const bool grows = top - m[0] > kLatentSlack, follow = __any(grows);      // (rows that do not need it stay: what a row gets does not depend on the others)
                    if (follow) {
                        const float alpha = grows ? fast_exp2(m[0] - top) : 1.f;
                        const float d = grows && l[0] != 0.f ? m[0] - top : 0.f, was = l[0];
                        m[0] = grows ? top : m[0];
                        l[0] *= alpha;
                        if (__builtin_expect(__any(d < kOneFactor), 0)) l[0] = add_moved(0.f, was, d);
                        if (kg == 0 && lh == 0) alphas[parity * ROWS + 32 * rg + lq] = alpha;
                    }
                    if (kg == 0 && ln == 0) flags[2 * parity + rg] = follow;
                    frame = (m[0] == -INFINITY ? 0.f : m[0]) - kLatentShift;
                    if (__builtin_expect(large, 0)) {      // (the scales of the block: its stage is written two blocks later)
                        const int key = 32 * kg + (int)scale_lane_key(ln);
                        float take = less_log(*(const float*)(lds + S::SCALES_AT + ((next + STAGES - 1) % STAGES) * S::SCALE_STAGE + 8 * key), key0 - KEYS + key >= most);
                        asm volatile("s_nop 1" : "+v"(take));
#pragma unroll
                        for (int i = 0; i < 16; ++i) l[0] = add_exp2(l[0], add_lane_scale(s[i] - frame, take, i));
                    }
                    lds_barrier();             // A: P of the block before has been read
                }
#pragma unroll
                for (int k = EARLY; k < KC; ++k) {
                    product(k);
                    if (E) {
#pragma unroll
                        for (int j = 16 * (k - EARLY) / (KC - EARLY); j < 16 * (k - EARLY + 1) / (KC - EARLY); ++j) element(j, frame, ln);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (QK) {
                    const v2f two = *(const v2f*)(lds + S::SCALES_AT + (next % STAGES) * S::SCALE_STAGE + 8 * (32 * kg + (int)scale_lane_key(ln)));
                    LatentScale sc = latent_scale(two[0], two[1], key0 + 32 * kg + (int)scale_lane_key(ln) >= most);
                    large = large || __any(*(const float*)(lds + S::SCALES_AT + (next % STAGES) * S::SCALE_STAGE + 8 * ln) > kLargeScale && key0 + ln < most);
                    inv = large ? 0.f : sc.inv;
                    asm volatile("s_nop 1" : "+v"(sc.c), "+v"(sc.r), "+v"(sc.log), "+v"(inv));      // (two wait states to other lanes' reads)
                    wait_for_product(hi);
                    wait_for_product(lo);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = mul_lane_scale((float)(hi[i] * 256 + lo[i]), sc.c, i);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = KC; k < KS; ++k) product(k);
                    wait_for_product(hi);
                    wait_for_product(lo);
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        fmac_lane_scale_f(s[i], sc.r, (float)(hi[i] * 256 + lo[i]), i);
                        s[i] = add_lane_scale(s[i] * factor[0], sc.log, i);
                    }
                    if (key0 + KEYS > least) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[i] = key0 + 32 * kg + 8 * (i / 4) + 4 * lh + i % 4 < seen[0] ? s[i] : -INFINITY;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
                    top = half_pair_max(top);
                    if (lh == 0) tops[kg * ROWS + 32 * rg + lq] = top;
                }
            };
            constexpr BoolTag<false> F{};
            constexpr BoolTag<true> T{};
            if (blocks > 0) step(T, F, 0, 0);
#pragma clang loop unroll(disable)
            for (int i = 0; i + 1 < blocks; ++i) {
                lds_barrier();                 // B: the next block is there
                step(T, T, i + 1, i & 1);
            }
            if (blocks > 0) {
                lds_barrier();
                step(F, T, blocks, (blocks - 1) & 1);
            }
        }
        else {
        int id_next = look(2);
        bool large = false;                    // (of all waves alike)
        for (int block = 0; block < blocks; ++block) {
            const bool more = block + 2 < blocks;
            const BlockCopy next = block_copy(block + 2, id_next);
            if (more) id_next = look(block + 3);
            const int key0 = key_first + KEYS * block, tile = (block % STAGES) * S::STAGE;
            const float* const scales = (const float*)(lds + S::SCALES_AT + (block % STAGES) * S::SCALE_STAGE);
            // ---- scores, as t = score + log2 of the value's scale
            constexpr int PER = 4;             // a lane's keys
            float s[QT][PER];
            // (lane i of a row of sixteen has the scales of the row's i-th key, from where all of the row take them)
            const int tile_key = 16 * wave, lane_key = tile_key + 4 * c16 + (x16 & 3);
            const v2f two = *(const v2f*)(scales + 2 * lane_key);
            // the rotary part first, then the latent one, two fragments ahead of the products
            auto fragment = [&](int i) __attribute__((always_inline)) {
                const int k = i < KS - KC ? KC + i : i - (KS - KC);
                return *(const v4i*)(lds + tile + fragment_at(key_at, k));
            };
            v4i hi[QT], lo[QT];
            auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int q = 0; q < QT; ++q)
#pragma unroll
                    for (int i = 0; i < PER; ++i) hi[q][i] = lo[q][i] = 0;
            };
            v4i f[4];
            f[0] = fragment(0);
            f[1] = fragment(1);
            LatentScale sc = latent_scale(two[0], two[1], key0 + lane_key >= most);
            large = large || __any(scales[2 * lane] > kLargeScale && key0 + lane < most);
            sc.inv = large ? 0.f : sc.inv;
            clear();
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                if (i + 2 < KS) f[(i + 2) % 4] = fragment(i + 2);
                const int k = i < KS - KC ? KC + i : i - (KS - KC);
                if (i == KS - KC) {
#pragma unroll
                    for (int q = 0; q < QT; ++q)
#pragma unroll
                        for (int e = 0; e < PER; ++e) s[q][e] = (float)(hi[q][e] * 256 + lo[q][e]) * lane_scale(sc.r, e);
                    clear();
                }
#pragma unroll
                for (int q = 0; q < QT; ++q) {
                    hi[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[i % 4], query_hi[q][k], hi[q], 0, 0, 0);
                    lo[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f[i % 4], query_lo[q][k], lo[q], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            float top[QT];
#pragma unroll
            for (int q = 0; q < QT; ++q) {
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    s[q][i] = ((float)(hi[q][i] * 256 + lo[q][i]) * lane_scale(sc.c, i) + s[q][i]) * factor[q] + lane_scale(sc.log, i);
                if (key0 + KEYS > least) {
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        const int key = key0 + tile_key + 4 * c16 + i;
                        s[q][i] = key < seen[q] ? s[q][i] : -INFINITY;
                    }
                }
                // ---- the rows' maxima: of the lanes that share a row, and of the waves that share its keys
                top[q] = -INFINITY;
#pragma unroll
                for (int i = 0; i < PER; ++i) top[q] = fmaxf(top[q], s[q][i]);
                top[q] = reduce_row_lanes(top[q], [](float a, float b) { return fmaxf(a, b); });
                if (c16 == 0) tops[kg * ROWS + 16 * q + x16] = top[q];
            }
            if (more) copy_some(next, BoolTag<false>{});
            lds_barrier();                     // A: the maxima are there, and P of the block before has been read
            bool grows[QT], any = false;
#pragma unroll
            for (int q = 0; q < QT; ++q) {
#pragma unroll
                for (int k = 0; k < KG; ++k) top[q] = fmaxf(top[q], tops[k * ROWS + 16 * q + x16]);
                grows[q] = top[q] - m[q] > kLatentSlack;
                any = any || grows[q];
            }
            const bool follow = __any(any);    // (of all waves alike; rows that do not need it stay: what a row gets does not depend on the others)
            if (follow) {
#pragma unroll
                for (int q = 0; q < QT; ++q) {
                    const float alpha = grows[q] ? fast_exp2(m[q] - top[q]) : 1.f;
                    const float d = grows[q] && l[q] != 0.f ? m[q] - top[q] : 0.f, was = l[q];
                    m[q] = grows[q] ? top[q] : m[q];
                    l[q] *= alpha;
                    if (__builtin_expect(__any(d < kOneFactor), 0)) l[q] = add_moved(0.f, was, d);
                    if (kg == 0 && c16 == 0) alphas[16 * q + x16] = alpha;
                }
            }
            if (kg == 0 && lane == 0) flags[rg] = follow;
            // ---- P, in the layout of the second product's operand: lane (row, h) has keys 16 t + 8 j + 4 h + i of step t at byte 8 j + 2 i of its sixteen
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                const float frame = (m[q] == -INFINITY ? 0.f : m[q]) - kLatentShift;
                if (__builtin_expect(large, 0)) {
                    const float take = less_log(two[0], key0 + lane_key >= most);
#pragma unroll
                    for (int i = 0; i < PER; ++i) l[q] = add_exp2(l[q], s[q][i] - frame + lane_scale(take, i));
                }
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    s[q][i] = fast_exp2(s[q][i] - frame);
                    l[q] += s[q][i] * lane_scale(sc.inv, i);
                }
                uint32_t w[PER / 2];
#pragma unroll
                for (int h = 0; h < PER / 2; ++h) w[h] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){s[q][2 * h], s[q][2 * h + 1]}, v2h));
                *(v2i*)(lds + S::P_AT + (64 * wave + 16 * q + x16 + 32 * (c16 & 1)) * 16 + 8 * (c16 >> 1)) = (v2i){(int)w[0], (int)w[1]};
            }
            if (more) {
                copy_some(next, BoolTag<true>{});
                copy_rest(next);
                wait_copies<S::COPIES>();
            } else wait_copies<0>();
            lds_barrier();                     // B: P is there, and so is the next block
        }
        }
        lds_barrier();                         // (the other half's last block)
        lds_barrier();
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            if constexpr (SMALL) l[q] = reduce_row_lanes(l[q], [](float a, float b) { return a + b; });
            else l[q] = half_pair_sum(l[q]);
            if (SMALL ? c16 == 0 : lh == 0) {
                const int r = SMALL ? 16 * q + x16 : 32 * rg + lq;
                tops[kg * ROWS + r] = l[q];
                if (kg == 0) alphas[r] = m[q];
            }
        }
        lds_barrier();
    } else {
        // ======== copies, and the values' product
        int id_next = look(2);
        int value_at[2];
        {
            const int j = x16 >> 1, value_row = 8 * (j >> 2) + 4 * lh + (j & 3), u = 2 * NT * wave + (c16 & 1);
            value_at[0] = value_row * S::ROW + 16 * S::place(u, value_row) + 8 * (x16 & 1);
            value_at[1] = value_row * S::ROW + 16 * S::place(u ^ 2, value_row) + 8 * (x16 & 1);
        }
        // (the tile's units 2 (NT w + ct) + ..: their bit 1 is that of ct where a wave has several tiles)
        auto value_offset = [&](int ct) __attribute__((always_inline)) { return DR == 64 ? value_at[ct & 1] + 64 * (ct >> 1) : value_at[0] + 32 * ct; };
        v16f acc[RG][NT];
#pragma unroll
        for (int g = 0; g < RG; ++g)
#pragma unroll
            for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[g][ct][r] = 0.f;
        if (!SMALL && blocks > 1 && !early) copy(1, look(1));
        for (int i = 0; i <= blocks; ++i) {
            if (!SMALL) {
                wait_copies<0>();
                lds_barrier();                 // B: the scores' next block, P of block i - 1 and its factors are there
            }
            auto copy_next = [&]() __attribute__((always_inline)) {
                if (i + 2 < blocks) {
                    copy(i + 2, id_next);
                    id_next = look(i + 3);
                }
            };
            const int tile = ((i + STAGES - 1) % STAGES) * S::STAGE, parity = SMALL ? 0 : (i & 1) ^ 1;      // of block i - 1
            v8h pf[KEYS / 16][RG];
            float alpha[RG];
            bool follow[RG];
            const bool more = !SMALL && i > 0 && i + 2 < blocks;
            int wanted = __builtin_amdgcn_readfirstlane(!more ? 0 : streams ? 2 : 1);
            asm volatile("" : "+s"(wanted));
            BlockCopy next{};
            // (values two steps ahead of their products; a copy of block i + 2 behind each column tile's products)
            v2i vb[2][NT];
            auto fetch = [&](int step) __attribute__((always_inline)) {
#pragma unroll
                for (int ct = 0; ct < NT; ++ct)
                    vb[step % 2][ct] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)INTFA_LDS(lds + tile + value_offset(ct) + 16 * step * S::ROW));
            };
            // Products of step `step`, the conversion of the next column tile's values between them: half of it in the shadow of each product (all of it ahead of both, and
            // the copies in a row ahead of them: 4790 clocks a block for 4560).
            uint32_t vf[2][4];
            auto convert = [&](int at, int half) __attribute__((always_inline)) {
                i8x4_to_f16((uint32_t)vb[at / NT % 2][at % NT][half], vf[at % 2][2 * half], vf[at % 2][2 * half + 1]);
            };
            auto product = [&](int step) __attribute__((always_inline)) {
#pragma unroll
                for (int ct = 0; ct < NT; ++ct) {
                    const int at = NT * step + ct;
                    const v8h v = __builtin_bit_cast(v8h, (v4i){(int)vf[at % 2][0], (int)vf[at % 2][1], (int)vf[at % 2][2], (int)vf[at % 2][3]});
#pragma unroll
                    for (int g = 0; g < RG; ++g) {
                        acc[g][ct] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pf[step][g], acc[g][ct], 0, 0, 0);
                        if (g == 0 && !SMALL && at < S::WHOLE) copy_units_if(wanted, next.rows, copy_off[at < S::WHOLE ? at : 0], next.to, 1024 * at);
                        if (at + 1 < NT * (KEYS / 16)) {
                            if (RG == 1) convert(at + 1, 0);
                            convert(at + 1, RG == 1 ? 1 : g);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if (step + 2 < KEYS / 16) fetch(step + 2);
            };
            if (i > 0) {
#pragma unroll
                for (int step = 0; step < KEYS / 16; ++step)
#pragma unroll
                    for (int g = 0; g < RG; ++g) pf[step][g] = *(const v8h*)(lds + S::P_AT + ((g * 4 + step) * 64 + lane) * 16);
#pragma unroll
                for (int g = 0; g < RG; ++g) {
                    follow[g] = flags[2 * parity + g] != 0;
                    alpha[g] = alphas[parity * ROWS + 32 * g + lq];
                }
                fetch(0);
                fetch(1);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!SMALL) {
                if (more) {
                    next = block_copy(i + 2, id_next);
                    id_next = look(i + 3);
                    copy_rest(next);
                }
                lds_barrier();                 // A: P has been read
            }
            if (i > 0) {
                // accumulators follow the maxima
#pragma unroll
                for (int g = 0; g < RG; ++g)
                    if (__builtin_amdgcn_readfirstlane((int)follow[g])) {
#pragma unroll
                        for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                            for (int r = 0; r < 16; ++r) acc[g][ct][r] *= alpha[g];
                    }
                convert(0, 0);
                convert(0, 1);
                product(0);
                product(1);
                if (!SMALL) {
                    product(2);
                    product(3);
                }
            } else if (!SMALL) copy_next();
            if (SMALL) lds_barrier();          // A
            if (SMALL && i > 0) {
                product(2);
                product(3);
            }
            if (SMALL) lds_barrier();          // B
        }
        lds_barrier();                         // (the rows' sums are there)
        p = latent_args();
#pragma unroll
        for (int g = 0; g < RG; ++g) {
            const int r = 32 * g + lq, row = row0 + r;
            if (row >= p->deal.rows) continue;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < KG; ++k) sum += tops[k * ROWS + r];
            const float top = alphas[r];
            if (part.whole) {
                const int token = paged_div(row, p->deal.d_group), head = row - token * p->deal.group;
                const bool empty = top == -INFINITY || token >= t.m;
                const float weight = empty ? 0.f : kWeightUnit / sum;
                // (through LDS: a lane has eight bytes of each of its units, and 32 rows are as many lines)
#pragma unroll
                for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        v4f o = {acc[g][ct][4 * k], acc[g][ct][4 * k + 1], acc[g][ct][4 * k + 2], acc[g][ct][4 * k + 3]};
                        o *= weight;
                        if (token >= t.m) o = (v4f){0.f, 0.f, 0.f, 0.f};
                        store_out4<DT>(lds + r * (2 * DC) + 16 * ((4 * (NT * wave + ct) + k) ^ (r & 15)) + 8 * lh, o);
                    }
                if (p->deal.lse != nullptr && wave == 0 && lh == 0)
                    p->deal.lse[((int64_t)t.z * p->deal.heads + head) * p->deal.seqlen + token] =
                        token >= t.m ? -INFINITY : (top == -INFINITY ? 0.f : top) - kLatentShift + log2_of_weights(sum);
            } else {
                float* const slot = p->deal.parts + (int64_t)part.slot * ROWS * DC;
#pragma unroll
                for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *(v4f*)(slot + (((g * S::CT + NT * wave + ct) * 4 + k) * 64 + lane) * 4) = (v4f){acc[g][ct][4 * k], acc[g][ct][4 * k + 1], acc[g][ct][4 * k + 2], acc[g][ct][4 * k + 3]};
                if (wave == 0 && lh == 0) *(v2f*)(p->deal.part_stats + ((int64_t)part.slot * ROWS + r) * 2) = (v2f){top, sum};
            }
        }
    }
    if (part.whole) {
        lds_barrier();
        for (int i = tid; i < ROWS * (DC / 8); i += S::THREADS) {
            const int r = i / (DC / 8), u = i % (DC / 8), row = row0 + r;
            if (row >= p->deal.rows) break;
            const int token = paged_div(row, p->deal.d_group), head = row - token * p->deal.group;
            *(v4i*)(p->deal.out + t.z * p->deal.o_sb + head * p->deal.o_sh + token * p->deal.o_sn + 16 * u) = *(const v4i*)(lds + r * (2 * DC) + 16 * (u ^ (r & 15)));
        }
    }
    if (!part.whole && part.one == (int)blockIdx.x) open = (v4i){part.pieces, t.z, t.tile, (int)part.slot};
    if (!paged_next(deal, ROWS, t, piece)) break;
    lds_barrier();
  }
    if (threadIdx.x == 0) latent_args()->open_items[blockIdx.x] = open;
}

// Pieces first, first + step .. of an item: a lane's Q groups of four columns (1024 bytes apart) of the weighted sums, the row's maximum and sum of weights.  PER: pieces under way at a time.
template <int Q, int PER> __device__ __forceinline__ void latent_gather(const float* parts, const float* stats, int64_t slot0, int64_t slot_bytes, int rows, int pieces, int first, int step,
                                                                        v4f (&acc)[Q], float& top, float& sum) {
    for (int j0 = first; j0 < pieces; j0 += PER * step) {
        v4f x[PER][Q];
        v2f st[PER];
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int j = j0 + u * step;
            st[u] = (v2f){-INFINITY, 0.f};
            if (j >= pieces) continue;
            // the pieces: the first in its workgroup's own slot, the others first items of theirs
            const int64_t slot = j == 0 ? slot0 : 2 * ((slot0 >> 1) + j);
            st[u] = *(const v2f*)(stats + slot * rows * 2);
#pragma unroll
            for (int k = 0; k < Q; ++k) x[u][k] = *(const v4f*)((const char*)parts + slot * slot_bytes + 1024 * k);
        }
        float grown = top;
#pragma unroll
        for (int u = 0; u < PER; ++u) grown = fmaxf(grown, st[u][0]);
        const float frame = grown == -INFINITY ? 0.f : grown, a = fast_exp2(top - frame), was = sum, moved = sum != 0.f ? top - frame : 0.f;
        float furthest = moved;
#pragma unroll
        for (int k = 0; k < Q; ++k) acc[k] *= a;
        sum *= a;
        top = grown;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            if (j0 + u * step >= pieces) continue;
            const float w = fast_exp2(st[u][0] - frame);
            furthest = fminf(furthest, st[u][0] - frame);
#pragma unroll
            for (int k = 0; k < Q; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[k][i] = fmaf(w, x[u][k][i], acc[k][i]);
            sum = fmaf(w, st[u][1], sum);
        }
        if (__builtin_expect(__any(furthest < kOneFactor), 0)) {
            sum = add_moved(0.f, was, moved);
#pragma unroll
            for (int u = 0; u < PER; ++u) sum = add_moved(sum, st[u][1], st[u][0] - frame);
        }
    }
}
// The items that lie in several pieces, a launch later.  A slice is 32 rows by 32 columns; a wave takes one, or, of an item of many pieces, eight waves share a quarter of one, an eighth of
// the pieces each, and the first joins theirs.  The workgroups deal the open items' slices among themselves (a grid over all items would be mostly workgroups without work).  Bound by a
// chain of four trips to memory, about 4 us, and by what the parts are: 128 heads of 32 requests 33 MB in 9.6 us; one request of 256 pieces, 8 MB, 8.5 (in whole slices 14.5).
template <int DC, int DT, int ROWS>
__global__ void __launch_bounds__(512) latent_merge_kernel(const LatentParams) {
    constexpr int SLICES = ROWS / 32 * (DC / 32), MANY = 8, WAVES = 8;
    constexpr int SETS = (SLICES + WAVES - 1) / WAVES;         // of slices, an eight of waves each
    __shared__ v4f joined[WAVES][64];
    __shared__ v2f joined_stats[WAVES][64];
    __shared__ v4i items[kComputeUnits];       // the open items
    __shared__ int first[kComputeUnits + 1], count;      // their first unit of work
    LatentArgs p = latent_args();
    const auto& d = p->deal;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (wave == 0) {
        int found = 0, units = 0;
        v4i all[kComputeUnits / 64];           // (one trip for all of them)
#pragma unroll
        for (int i = 0; i < kComputeUnits / 64; ++i) all[i] = p->open_items[64 * i + lane < d.grid ? 64 * i + lane : 0];
#pragma unroll
        for (int i = 0; i < kComputeUnits / 64; ++i) {
            const v4i item = all[i];
            const int pieces = 64 * i + lane < d.grid ? item[0] : 0, mine = pieces == 0 ? 0 : pieces > MANY ? 4 * SLICES : SETS;
            int upto = mine;
#pragma unroll
            for (int w = 1; w < 64; w <<= 1) {
                const int o = __shfl_up(upto, w);
                if (lane >= w) upto += o;
            }
            const uint64_t open = __ballot(pieces != 0);
            const int at = found + __popcll(open & ((1ull << lane) - 1));
            if (pieces != 0) {
                items[at] = item;
                first[at] = units + upto - mine;
            }
            found += __popcll(open);
            units += __shfl(upto, 63);
        }
        if (lane == 0) {
            count = found;
            first[found] = units;
        }
    }
    __syncthreads();
    const int found = count, total = first[found];
    for (int unit = (int)blockIdx.x; unit < total; unit += (int)gridDim.x) {
        int lo = 0, hi = found;                // the item that has it: first[lo] <= unit < first[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= unit) lo = mid; else hi = mid;
        }
        const v4i item = items[lo];
        const int pieces = __builtin_amdgcn_readfirstlane(item[0]), z = __builtin_amdgcn_readfirstlane(item[1]), tile = __builtin_amdgcn_readfirstlane(item[2]);
        const int part = unit - __builtin_amdgcn_readfirstlane(first[lo]);
        const bool share = pieces > MANY;      // the waves share a quarter of a slice
        const int slice = share ? part / 4 : part * WAVES + wave, quarter = share ? part % 4 : 0, g = slice / (DC / 32), ct = slice % (DC / 32);
        const int r = 32 * g + (lane & 31), row = tile * ROWS + r;
        const bool valid = row < d.rows && slice < SLICES;
        const int token = paged_div(valid ? row : 0, d.d_group), head = (valid ? row : 0) - token * d.group;
        const int64_t slot0 = __builtin_amdgcn_readfirstlane(item[3]);
        const float* const parts = d.parts + ((slice * 4 + quarter) * 64 + lane) * 4;
        const float* const stats = d.part_stats + r * 2;
        v4f acc[4];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = (v4f){0.f, 0.f, 0.f, 0.f};
        if (share) {
            v4f one[1] = {acc[0]};
            if (valid) latent_gather<1, MANY>(parts, stats, slot0, (int64_t)ROWS * DC * 4, ROWS, pieces, wave, WAVES, one, top, sum);
            joined[wave][lane] = one[0];
            joined_stats[wave][lane] = (v2f){top, sum};
            __syncthreads();
            if (wave == 0) {
                v2f st[WAVES];
                float grown = -INFINITY;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    st[w] = joined_stats[w][lane];
                    grown = fmaxf(grown, st[w][0]);
                }
                const float frame = grown == -INFINITY ? 0.f : grown;
                float furthest = 0.f;
                sum = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float a = fast_exp2(st[w][0] - frame);
                    const v4f x = joined[w][lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[0][i] = fmaf(a, x[i], acc[0][i]);
                    sum = fmaf(a, st[w][1], sum);
                    furthest = fminf(furthest, st[w][0] - frame);
                }
                if (__builtin_expect(__any(furthest < kOneFactor), 0)) {
                    sum = 0.f;
#pragma unroll
                    for (int w = 0; w < WAVES; ++w) sum = add_moved(sum, st[w][1], st[w][0] - frame);
                }
                top = grown;
            }
            __syncthreads();
        } else if (valid) latent_gather<4, MANY / 2>(parts, stats, slot0, (int64_t)ROWS * DC * 4, ROWS, pieces, 0, 1, acc, top, sum);
        if (valid && (!share || wave == 0)) {
            int m = d.seqlen;
            if (d.seqlens_q != nullptr) {
                const int n = d.seqlens_q[z];
                m = n < 0 ? 0 : n < m ? n : m;
            }
            const bool beyond = token >= m;
            const float weight = beyond || top == -INFINITY ? 0.f : kWeightUnit / sum;
            char* const dst = d.out + z * d.o_sb + head * d.o_sh + token * d.o_sn + 2 * (32 * ct + 4 * (lane >> 5) + 8 * quarter);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v4f o = acc[k] * weight;
                if (beyond) o = (v4f){0.f, 0.f, 0.f, 0.f};
                if (k == 0 || !share) store_out4<DT>(dst + 16 * k, o);
            }
            if (d.lse != nullptr && ct == 0 && quarter == 0 && lane < 32)
                d.lse[((int64_t)z * d.heads + head) * d.seqlen + token] = beyond ? -INFINITY : (top == -INFINITY ? 0.f : top) - kLatentShift + log2_of_weights(sum);
        }
    }
}

template <int DC, int DR, int DT, int ROWS, int QT> int launch_latent_rows(const LatentParams& p, hipStream_t stream) {
    hipLaunchKernelGGL((latent_attn_kernel<DC, DR, DT, ROWS, QT>), dim3((unsigned)p.deal.grid), dim3(512), 0, stream, p);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
    // (an item of few pieces is SLICES / 8 units of work, one of nine or more 4 SLICES)
    constexpr int SLICES = ROWS / 32 * (DC / 32);
    const int units = p.deal.grid * SLICES / 8 + 4 * SLICES;
    hipLaunchKernelGGL((latent_merge_kernel<DC, DT, ROWS>), dim3((unsigned)(units < 2 * kComputeUnits ? units : 2 * kComputeUnits)), dim3(512), 0, stream, p);
    return (int)hipGetLastError();
}
template <int DC, int DR, int DT> int launch_latent(const LatentParams& p, int rows, hipStream_t stream) {
    if (rows == 64) return launch_latent_rows<DC, DR, DT, 64, 1>(p, stream);
    return p.deal.rows <= 16 ? launch_latent_rows<DC, DR, DT, 32, 1>(p, stream) : launch_latent_rows<DC, DR, DT, 32, 2>(p, stream);
}

}  // namespace intfa
