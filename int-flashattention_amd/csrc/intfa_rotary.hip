// Rotary positions, and the append of rotated keys and of values to a paged int8 cache.  See include/intfa.h for the formulas.
#include "intfa_paged_host.h"

using namespace intfa;

namespace {

// ---- rotary
struct RotaryParams {
    const char* x; char* out;
    int64_t x_sb, x_sh, x_sn, o_sb, o_sh, o_sn;      // bytes
    const int32_t* positions;
    int64_t pos_sb, pos_sn;
    int32_t per_row, first;
    RopeArgs rope;
    int32_t heads, seqlen, units, heads_each;        // units of sixteen elements per row; heads per thread
    int64_t threads;                                 // batch * seqlen * units
    FastDiv d_units, d_seqlen;
    float sign;
};

// A thread takes one unit of one token and turns it in heads_each heads by the same eight angles, kRotaryHeads of them under way at a time.  Bound by memory
// once a thread has a few heads (an angle costs as much as a dozen turned pairs); each line is touched once, so loads and stores pass by the caches.
constexpr int kRotaryHeads = 4;
template <int DT, bool MANY> __global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
    constexpr int N = MANY ? kRotaryHeads : 1;
    const int64_t lin = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (lin >= p.threads) return;
    const int token = fast_div((int)lin, p.d_units), u = (int)lin - token * p.units;
    const int b = fast_div(token, p.d_seqlen), n = token - b * p.seqlen;
    int first, second;
    const bool turns = 8 * u < p.rope.pairs, interleaved = p.rope.interleaved != 0;
    rope_unit(u, p.rope.pairs, interleaved, first, second);
    const int h0 = (int)blockIdx.y * p.heads_each, h1 = h0 + p.heads_each < p.heads ? h0 + p.heads_each : p.heads;
    const char* const src = p.x + b * p.x_sb + n * p.x_sn;
    char* const dst = p.out + b * p.o_sb + n * p.o_sn;
    v4i raw[N][2];
    auto request = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const char* const at = src + (h + k < h1 ? h + k : h1 - 1) * p.x_sh;
            raw[k][0] = __builtin_nontemporal_load((const v4i*)(at + 2 * first));
            raw[k][1] = __builtin_nontemporal_load((const v4i*)(at + 2 * second));
        }
    };
    request(h0);
    float c[8], s[8];
    if (turns) {
        const double position = p.positions == nullptr ? (double)(p.first + n)
                                : p.per_row           ? (double)p.positions[b * p.pos_sb + n * p.pos_sn]
                                                      : (double)p.positions[b * p.pos_sb] + n;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            rope_angle(p.rope.freqs[8 * u + i], position, p.rope.magnitude, c[i], s[i]);
            s[i] *= p.sign;
        }
    }
    for (int h = h0; h < h1; h += N) {
        v4i y[N][2];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            y[k][0] = raw[k][0];
            y[k][1] = raw[k][1];
            if (turns) {
                float x[16];
                unpack8<DT>(raw[k][0], x);
                unpack8<DT>(raw[k][1], x + 8);
                rope_turn_unit(x, c, s, interleaved);
                y[k][0] = pack8<DT>(x);
                y[k][1] = pack8<DT>(x + 8);
            }
        }
        if (h + N < h1) request(h + N);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (h + k >= h1) break;
            char* const at = dst + (h + k) * p.o_sh;
            __builtin_nontemporal_store(y[k][0], (v4i*)(at + 2 * first));
            __builtin_nontemporal_store(y[k][1], (v4i*)(at + 2 * second));
        }
    }
}

// ---- append to pages
struct PagedSide {
    const char* src; char* cache; float* scale;
    int64_t n_sb, n_sh, n_sn;            // bytes
    int64_t c_sp, c_sh, c_sn;            // bytes
    int64_t s_sp, s_sh;                  // elements
};
struct PagedAppendParams {
    PagedSide k, v;
    const int32_t* table; int64_t bt_sb;
    const int32_t* seqlens_k; const int32_t* seqlens_new;
    RopeArgs rope;
    int32_t heads, seqlen_new, page_log2, num_pages, table_width, units;      // units: of sixteen elements per row
    int32_t slots, head_groups, heads_each;      // pages that a sequence may reach; groups of heads_each heads
    FastDiv d_slots, d_head_groups;
};

constexpr float kLeastScale = 0x1p-100f;

__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;      // (false for NaN too)
}
// rint(x / scale) within +-127, 0 for NaN, as a byte
__device__ __forceinline__ uint32_t quantise(float x, float scale) {
    const float q = rintf(x / scale);
    return (uint32_t)(q >= 127.f ? 127 : q <= -127.f ? -127 : q == q ? (int)q : 0) & 0xffu;
}
// Four of them for finite x with |x| <= 127 scale (to rounding).  The quotient is the correctly rounded one, by Markstein's correction of the product with
// the reciprocal (short of divisors whose significand is all ones, where it may be its neighbour); adding 1.5 * 2^23 rounds it to an integer
// in the low byte.  NaN gives 0: its low byte is.
__device__ __forceinline__ uint32_t quantise4(const float* x, float scale, float reciprocal) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = x[i] * reciprocal, e = __builtin_fmaf(-q, scale, x[i]);
        b[i] = __builtin_bit_cast(uint32_t, __builtin_fmaf(e, reciprocal, q) + 12582912.0f);
    }
    return __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
}

// One workgroup per page slot of a sequence, K or V, and group of heads.  A page's scale needs all its new rows before the first is stored: a thread holds up
// to HELD units of sixteen elements in registers in between (rows past that are read and turned a second time), and turns the same rows of all its
// heads by the same angles, which take longer to form than all the rest.  The next head's rows are requested ahead of this one's work.
// WAVES = 1, for few new rows: no wave waits for another.
template <int DT, int WAVES, int HELD> __global__ void __launch_bounds__(64 * WAVES) paged_append_kernel(const PagedAppendParams p) {
    constexpr int THREADS = 64 * WAVES;
    __shared__ float red[2][WAVES];
    const int zs = fast_div((int)blockIdx.x, p.d_head_groups), group = (int)blockIdx.x - zs * p.head_groups;
    const int z = fast_div(zs, p.d_slots), slot = zs - z * p.slots;
    const bool is_v = blockIdx.y != 0;            // (keys first: they have angles to form.  In turn with the values, whole prompts 23.4 -> 25.2 us)
    const PagedSide& side = is_v ? p.v : p.k;
    const int page = 1 << p.page_log2;
    int held = p.seqlens_k[z], fresh = p.seqlen_new;
    held = held < 0 ? 0 : held;
    if (p.seqlens_new != nullptr) {
        const int m = p.seqlens_new[z];
        fresh = m < 0 ? 0 : m < fresh ? m : fresh;
    }
    const int column = (held >> p.page_log2) + slot;
    if (column >= p.table_width) return;
    const int64_t start = (int64_t)column << p.page_log2;                       // position of the page's first row
    const int row0 = start < held ? (int)(held - start) : 0;                    // rows [row0, row1) are new
    const int64_t past = (int64_t)held + fresh - start;
    const int row1 = past < page ? (int)past : page;
    if (row1 <= row0) return;
    const int id = p.table[z * p.bt_sb + column];
    const int h0 = group * p.heads_each, h1 = h0 + p.heads_each < p.heads ? h0 + p.heads_each : p.heads;
    const char* const src0 = side.src + z * side.n_sb + (start + row0 - held) * side.n_sn;
    const bool rope = !is_v && p.rope.freqs != nullptr, interleaved = p.rope.interleaved != 0;
    const int pairs = rope ? p.rope.pairs : 0, units = (row1 - row0) * p.units, units_log2 = __builtin_ctz(p.units);
    // the thread's units: their rows, places and angles
    int row[HELD], first[HELD], second[HELD];
    v4i raw[HELD][2];
    auto request = [&](int h) __attribute__((always_inline)) {
        const char* const src = src0 + h * side.n_sh;
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            raw[k][0] = raw[k][1] = (v4i){0, 0, 0, 0};
            if ((int)threadIdx.x + k * THREADS < units) {
                raw[k][0] = __builtin_nontemporal_load((const v4i*)(src + row[k] * side.n_sn + 2 * first[k]));
                raw[k][1] = __builtin_nontemporal_load((const v4i*)(src + row[k] * side.n_sn + 2 * second[k]));
            }
        }
    };
    float c[HELD][8], s[HELD][8];
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int i = (int)threadIdx.x + k * THREADS;
        row[k] = i >> units_log2;
        rope_unit(i & (p.units - 1), pairs, interleaved, first[k], second[k]);
    }
    request(h0);
    if ((unsigned)id >= (unsigned)p.num_pages) return;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int i = (int)threadIdx.x + k * THREADS, u = i & (p.units - 1);
        if (8 * u < pairs && i < units) {
#pragma unroll
            for (int j = 0; j < 8; ++j) rope_angle(p.rope.freqs[8 * u + j], (int)(start + row0 + row[k]), p.rope.magnitude, c[k][j], s[k][j]);
        }
    }
    // a unit past the held ones
    auto read = [&](const char* src, int i, float (&x)[16], int& r, int& one, int& two) __attribute__((always_inline)) {
        r = i >> units_log2;
        const int u = i & (p.units - 1);
        rope_unit(u, pairs, interleaved, one, two);
        unpack8<DT>(*(const v4i*)(src + r * side.n_sn + 2 * one), x);
        unpack8<DT>(*(const v4i*)(src + r * side.n_sn + 2 * two), x + 8);
        if (8 * u < pairs) {
            float cc[8], ss[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) rope_angle(p.rope.freqs[8 * u + j], (int)(start + row0 + r), p.rope.magnitude, cc[j], ss[j]);
            rope_turn_unit(x, cc, ss, interleaved);
        }
    };
    for (int h = h0; h < h1; ++h) {
        const char* const src = src0 + h * side.n_sh;
        char* const dst = side.cache + id * side.c_sp + h * side.c_sh;
        float* const scale_at = side.scale + id * side.s_sp + h * side.s_sh;
        const float before = row0 > 0 ? *scale_at : 0.f;
        float x[HELD][16], top = 0.f;
#pragma unroll
        for (int k = 0; k < HELD; ++k) {
            unpack8<DT>(raw[k][0], x[k]);
            unpack8<DT>(raw[k][1], x[k] + 8);
            if (8 * (((int)threadIdx.x + k * THREADS) & (p.units - 1)) < pairs && (int)threadIdx.x + k * THREADS < units) rope_turn_unit(x[k], c[k], s[k], interleaved);
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(x[k][j]));      // (no NaN gets through)
        }
        if (h + 1 < h1) request(h + 1);
        for (int i = (int)threadIdx.x + HELD * THREADS; i < units; i += THREADS) {
            float y[16];
            int r, one, two;
            read(src, i, y, r, one, two);
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(y[j]));
        }
        auto of_all = [&](float v) __attribute__((always_inline)) {
            for (int m = 32; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
            if (WAVES > 1) {
                float* const r = red[h & 1];
                if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WAVES; ++w) v = fmaxf(v, r[w]);
            }
            return v;
        };
        top = of_all(top);
        const bool infinite = top > 3.402823466e38f;      // some value is: it does not count, and quotients need their bounds
        if (infinite) {
            top = 0.f;
#pragma unroll
            for (int k = 0; k < HELD; ++k)
#pragma unroll
                for (int j = 0; j < 16; ++j) top = fmaxf(top, finite_magnitude(x[k][j]));
            for (int i = (int)threadIdx.x + HELD * THREADS; i < units; i += THREADS) {
                float y[16];
                int r, one, two;
                read(src, i, y, r, one, two);
#pragma unroll
                for (int j = 0; j < 16; ++j) top = fmaxf(top, finite_magnitude(y[j]));
            }
            if (WAVES > 1) __syncthreads();
            top = of_all(top);
        }
        const float scale = fmaxf(fmaxf(top / 127.0f, kLeastScale), before), reciprocal = 1.0f / scale;
        if (scale != before) {
            const float ratio = before / scale;
            for (int i = threadIdx.x; i < row0 * p.units; i += THREADS) {
                v4i* const at = (v4i*)(dst + (i >> units_log2) * side.c_sn + 16 * (i & (p.units - 1)));
                v4i w = *at;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t r = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) r |= ((uint32_t)(int)rintf((float)(int8_t)((uint32_t)w[k] >> (8 * j)) * ratio) & 0xffu) << (8 * j);
                    w[k] = (int)r;
                }
                *at = w;
            }
        }
        auto put = [&](const float (&y)[16], int r, int one, int two) __attribute__((always_inline)) {
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                q[j] = !infinite ? quantise4(y + 4 * j, scale, reciprocal)
                                 : quantise(y[4 * j], scale) | quantise(y[4 * j + 1], scale) << 8 | quantise(y[4 * j + 2], scale) << 16 | quantise(y[4 * j + 3], scale) << 24;
            char* const d = dst + (row0 + r) * side.c_sn;
            if (two == one + 8) {
                *(v4i*)(d + one) = (v4i){(int)q[0], (int)q[1], (int)q[2], (int)q[3]};
            } else {
                *(v2i*)(d + one) = (v2i){(int)q[0], (int)q[1]};
                *(v2i*)(d + two) = (v2i){(int)q[2], (int)q[3]};
            }
        };
#pragma unroll
        for (int k = 0; k < HELD; ++k)
            if ((int)threadIdx.x + k * THREADS < units) put(x[k], row[k], first[k], second[k]);
        for (int i = (int)threadIdx.x + HELD * THREADS; i < units; i += THREADS) {
            float y[16];
            int r, one, two;
            read(src, i, y, r, one, two);
            put(y, r, one, two);
        }
        if (threadIdx.x == 0) *scale_at = scale;      // (`before` has been read by every thread: what it decides comes after the barrier)
    }
}

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1u)) == 0; }
bool strides16(int64_t a, int64_t b, int64_t c) { return a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }      // of 16-bit elements

}  // namespace

extern "C" {

int intfa_rotary(const intfa_rotary_params* p, void* stream) {
    if (p == nullptr || p->x == nullptr || p->out == nullptr || p->rope.freqs == nullptr) return INTFA_ERR_NULL;
    if (p->batch <= 0 || p->heads <= 0) return INTFA_ERR_SHAPE;
    if (p->seqlen <= 0) return INTFA_ERR_SEQLEN;
    const int d = p->head_dim;
    if (d != 16 && d != 32 && d != 64 && d != 128 && d != 256) return INTFA_ERR_HEAD_DIM;
    if (p->dtype != INTFA_F16 && p->dtype != INTFA_BF16) return INTFA_ERR_DTYPE;
    if (!rope_valid(&p->rope, d)) return INTFA_ERR_ROPE;
    if (!aligned(p->x, 16) || !aligned(p->out, 16) || !aligned(p->rope.freqs, 8) || !aligned(p->positions, 4) ||
        !strides16(p->x_stride_b, p->x_stride_h, p->x_stride_n) || !strides16(p->o_stride_b, p->o_stride_h, p->o_stride_n)) return INTFA_ERR_ALIGN;
    if (p->positions == nullptr && (int64_t)p->position_first + p->seqlen > 1ll << 31) return INTFA_ERR_SHAPE;      // positions are 32-bit numbers
    RotaryParams rp{};
    rp.units = d / 16;
    rp.threads = size_product((int64_t)p->batch * p->seqlen, rp.units);
    if (rp.threads >= (1ll << 31) - 256 || p->heads > 65535) return INTFA_ERR_SHAPE;
    rp.x = (const char*)p->x; rp.out = (char*)p->out;
    rp.x_sb = p->x_stride_b * 2; rp.x_sh = p->x_stride_h * 2; rp.x_sn = p->x_stride_n * 2;
    rp.o_sb = p->o_stride_b * 2; rp.o_sh = p->o_stride_h * 2; rp.o_sn = p->o_stride_n * 2;
    rp.positions = p->positions; rp.pos_sb = p->pos_stride_b; rp.pos_sn = p->pos_stride_n;
    rp.per_row = p->positions_per_row; rp.first = p->position_first;
    rp.rope = {p->rope.freqs, p->rope.pairs, p->rope.interleaved, p->rope.magnitude};
    rp.heads = p->heads; rp.seqlen = p->seqlen;
    rp.d_units = make_fast_div(rp.units); rp.d_seqlen = make_fast_div(p->seqlen);
    rp.sign = p->inverse ? -1.0f : 1.0f;
    // Heads per thread: as many as leave a workgroup per compute unit, up to eight.  (4 x 4096 tokens, 32 heads of 128, us: one 59, four 47.7, eight 46.3, sixteen 46.0)
    const int blocks = (int)((rp.threads + 255) / 256);
    rp.heads_each = 1;
    while (rp.heads_each < 8 && rp.heads_each < p->heads && (int64_t)blocks * p->heads >= 2ll * rp.heads_each * kComputeUnits) rp.heads_each *= 2;
    const dim3 grid(blocks, (p->heads + rp.heads_each - 1) / rp.heads_each);
#define INTFA_CALL(DT) do { \
        if (rp.heads_each >= kRotaryHeads) hipLaunchKernelGGL((rotary_kernel<DT, true>), grid, dim3(256), 0, (hipStream_t)stream, rp); \
        else hipLaunchKernelGGL((rotary_kernel<DT, false>), grid, dim3(256), 0, (hipStream_t)stream, rp); } while (0)
    if (p->dtype == INTFA_F16) INTFA_CALL(0); else INTFA_CALL(1);
#undef INTFA_CALL
    return (int)hipGetLastError();
}

int intfa_paged_append_int8(const intfa_paged_append_params* p, void* stream) {
    if (p == nullptr || p->k_new == nullptr || p->v_new == nullptr || p->seqlens_k == nullptr) return INTFA_ERR_NULL;
    const intfa_paged_cache& c = p->cache;
    const int rc = paged_cache_check(&c);
    if (rc != INTFA_OK) return rc;
    if (p->batch <= 0) return INTFA_ERR_SHAPE;
    if (p->seqlen_new <= 0 || p->seqlen_new > 1 << 30) return INTFA_ERR_SEQLEN;
    if (p->dtype != INTFA_F16 && p->dtype != INTFA_BF16) return INTFA_ERR_DTYPE;
    if (p->rope.freqs != nullptr && !rope_valid(&p->rope, c.head_dim)) return INTFA_ERR_ROPE;
    if (!aligned(p->k_new, 16) || !aligned(p->v_new, 16) || !aligned(p->seqlens_k, 4) || !aligned(p->seqlens_new, 4) || !aligned(p->rope.freqs, 8) ||
        !strides16(p->kn_stride_b, p->kn_stride_h, p->kn_stride_n) || !strides16(p->vn_stride_b, p->vn_stride_h, p->vn_stride_n)) return INTFA_ERR_ALIGN;
    PagedAppendParams ap{};
    ap.k = {(const char*)p->k_new, (char*)c.k, c.k_scale, p->kn_stride_b * 2, p->kn_stride_h * 2, p->kn_stride_n * 2,
            c.k_stride_p, c.k_stride_h, c.k_stride_n, c.ks_stride_p, c.ks_stride_h};
    ap.v = {(const char*)p->v_new, (char*)c.v, c.v_scale, p->vn_stride_b * 2, p->vn_stride_h * 2, p->vn_stride_n * 2,
            c.v_stride_p, c.v_stride_h, c.v_stride_n, c.vs_stride_p, c.vs_stride_h};
    ap.table = c.block_table; ap.bt_sb = c.bt_stride_b;
    ap.seqlens_k = p->seqlens_k; ap.seqlens_new = p->seqlens_new;
    ap.rope = {p->rope.freqs, p->rope.pairs, p->rope.interleaved, p->rope.magnitude};
    ap.heads = c.heads_kv; ap.seqlen_new = p->seqlen_new;
    ap.page_log2 = __builtin_ctz((unsigned)c.page_size); ap.num_pages = c.num_pages; ap.table_width = c.table_width;
    ap.units = c.head_dim / 16;
    ap.slots = (p->seqlen_new + c.page_size - 2) / c.page_size + 1;
    ap.slots = ap.slots < c.table_width ? ap.slots : c.table_width;
    // Heads per workgroup: as many as leave a workgroup for keys and one for values per compute unit.  (Prompts of 4 x 4096 tokens, 8 heads of 128, pages of 64, us:
    // one head a workgroup 34.9, two 28.4, four 26.4, eight 23.4; one token of 64 sequences each, two heads instead of one 5.3 -> 7.3.)
    const int64_t pages = (int64_t)p->batch * ap.slots;
    const int rows = p->seqlen_new < c.page_size ? p->seqlen_new : c.page_size, units = rows * ap.units;
    ap.heads_each = 1;
    while (units > 64 && ap.heads_each < 8 && ap.heads_each < c.heads_kv && size_product(pages, c.heads_kv) >= 2ll * ap.heads_each * kComputeUnits) ap.heads_each *= 2;
    ap.head_groups = (c.heads_kv + ap.heads_each - 1) / ap.heads_each;
    const int threads = units <= 64 ? 64 : 512;
    if (size_product(size_product(pages, ap.head_groups), threads) >= 1ll << 32) return INTFA_ERR_SHAPE;      // (threads of a launch are numbered in 32 bits)
    ap.d_slots = make_fast_div(ap.slots); ap.d_head_groups = make_fast_div(ap.head_groups);
    const dim3 g((unsigned)(pages * ap.head_groups), 2);
#define INTFA_CALL(DT) do { \
        if (units <= 64) hipLaunchKernelGGL((paged_append_kernel<DT, 1, 1>), g, dim3(threads), 0, (hipStream_t)stream, ap); \
        else if (units <= 512) hipLaunchKernelGGL((paged_append_kernel<DT, 8, 1>), g, dim3(threads), 0, (hipStream_t)stream, ap); \
        else hipLaunchKernelGGL((paged_append_kernel<DT, 8, 2>), g, dim3(threads), 0, (hipStream_t)stream, ap); } while (0)
    if (p->dtype == INTFA_F16) INTFA_CALL(0); else INTFA_CALL(1);
#undef INTFA_CALL
    return (int)hipGetLastError();
}

}  // extern "C"
