// The append of new tokens to a latent cache: norm, rotation, rounding to int8.  See include/intfa.h for the formulas.
#include "intfa_latent_host.h"
#include "intfa_quantise.h"

using namespace intfa;

namespace {

struct LatentAppendParams {
    const char* c; const char* k; const char* weight;
    int64_t c_sb, c_sn, k_sb, k_sn;                  // bytes
    char* rows; float* scale;
    int64_t r_sp, s_sp;                              // bytes, elements
    int32_t r_sn, s_sn;
    const int32_t* table; int64_t bt_sb;
    const int32_t* seqlens_k; const int32_t* seqlens_new;
    RopeArgs rope;
    float eps;
    int32_t tokens, seqlen_new, page_log2, num_pages, table_width;
    FastDiv d_seqlen;
};

// Where a token goes: false if nowhere.
struct LatentPlace { int64_t position; char* row; float* scale; int z, i; };
__device__ __forceinline__ bool latent_place(const LatentAppendParams& p, int token, LatentPlace& a) {
    const bool real = token < p.tokens;
    token = real ? token : p.tokens - 1;
    a.z = fast_div(token, p.d_seqlen);
    a.i = token - a.z * p.seqlen_new;
    const int held = p.seqlens_k[a.z], fresh = p.seqlens_new != nullptr ? p.seqlens_new[a.z] : p.seqlen_new;
    a.position = (int64_t)(held < 0 ? 0 : held) + a.i;
    const int64_t column = a.position >> p.page_log2;
    const int id = p.table[a.z * p.bt_sb + (column < p.table_width ? column : p.table_width - 1)];
    const int at = (int)a.position & ((1 << p.page_log2) - 1);
    const bool named = (unsigned)id < (unsigned)p.num_pages;
    a.row = p.rows + (named ? id : 0) * p.r_sp + at * p.r_sn;
    a.scale = p.scale + (named ? id : 0) * p.s_sp + at * p.s_sn;
    return real && a.i < fresh && column < p.table_width && named;
}

template <int LANES> __device__ __forceinline__ float over_lanes_max(float v) {
#pragma unroll
    for (int w = 1; w < LANES; w <<= 1) v = fmaxf(v, __shfl_xor(v, w));
    return v;
}
template <int LANES> __device__ __forceinline__ float over_lanes_sum(float v) {
#pragma unroll
    for (int w = 1; w < LANES; w <<= 1) v += __shfl_xor(v, w);
    return v;
}

// A wave takes T tokens, nothing of it waits for another wave: DC / 8 lanes a token for the latent part, eight elements each, and DR / 2 for the rotary one, a pair each, since
// an angle costs as much as all of a lane's other work (eight angles a lane: four prompts of 4096 tokens 20 us of angles alone).
template <int DT, int DC, int DR> __global__ void __launch_bounds__(256) latent_append_kernel(const LatentAppendParams p) {
    constexpr int LL = DC / 8, RL = DR / 2, LT = 64 / LL, RT = 64 / RL, T = LT > RT ? LT : RT, LP = T / LT, RP = T / RT;
    const int lane = threadIdx.x & 63, first = ((int)blockIdx.x * 4 + ((int)threadIdx.x >> 6)) * T;
    if (first >= p.tokens) return;
    // everything is requested before the first is used
    LatentPlace at[LP], rat[RP];
    bool put[LP], rput[RP];
    v4i raw[LP];
    uint16_t pair[RP][2];
    const int col = lane % LL * 8, j = lane % RL;
    const bool turns = p.rope.freqs != nullptr && j < p.rope.pairs;
    const int one = turns && !p.rope.interleaved ? j : 2 * j, two = turns && !p.rope.interleaved ? p.rope.pairs + j : 2 * j + 1;
#pragma unroll
    for (int k = 0; k < LP; ++k) {
        put[k] = latent_place(p, first + k * LT + lane / LL, at[k]);
        raw[k] = __builtin_nontemporal_load((const v4i*)(p.c + at[k].z * p.c_sb + at[k].i * p.c_sn + 2 * col));
    }
#pragma unroll
    for (int k = 0; k < RP; ++k) {
        rput[k] = latent_place(p, first + k * RT + lane / RL, rat[k]);
        const char* const src = p.k + rat[k].z * p.k_sb + rat[k].i * p.k_sn;
        pair[k][0] = *(const uint16_t*)(src + 2 * one);
        pair[k][1] = *(const uint16_t*)(src + 2 * two);
    }
    const double freq = turns ? p.rope.freqs[j] : 0.0;
    float weight[8];
    if (p.weight != nullptr) unpack8<DT>(*(const v4i*)(p.weight + 2 * col), weight);
#pragma unroll
    for (int k = 0; k < LP; ++k) {
        float x[8];
        unpack8<DT>(raw[k], x);
        if (p.weight != nullptr) {
            // The squares are those of x / 2^e, 2^e the size of the row's largest element: they stay in range whatever the row's size.  (e from -40, under which
            // eps is all there is; 126 for a row with an infinity, which thereby becomes one of zeros, as its formula has it)
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t a = __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu;
                top = top > a ? top : a;
            }
#pragma unroll
            for (int w = 1; w < LL; w <<= 1) {
                const uint32_t a = (uint32_t)__shfl_xor((int)top, w);
                top = top > a ? top : a;
            }
            int e = (int)(top >> 23) - 127;
            e = e < -40 ? -40 : e > 126 ? 126 : e;
            const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] *= down;
                sum = fmaf(x[i], x[i], sum);
            }
            sum = over_lanes_sum<LL>(sum);
            const float r = 1.0f / sqrtf(sum * (1.0f / DC) + p.eps * down * down);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * r * weight[i];
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
        top = over_lanes_max<LL>(top);
        const bool infinite = top > 3.402823466e38f;         // (of the token's lanes alike)
        if (__any(infinite)) {
            float finite = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) finite = fmaxf(finite, finite_magnitude(x[i]));
            finite = over_lanes_max<LL>(finite);
            top = finite;
        }
        const float scale = fmaxf(top / 127.0f, kLeastScale), reciprocal = 1.0f / scale;
        if (put[k]) {
            uint32_t q[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float* const y = x + 4 * h;
                q[h] = !infinite ? quantise4(y, scale, reciprocal)
                                 : quantise(y[0], scale) | quantise(y[1], scale) << 8 | quantise(y[2], scale) << 16 | quantise(y[3], scale) << 24;
            }
            *(v2i*)(at[k].row + col) = (v2i){(int)q[0], (int)q[1]};
            if (col == 0) at[k].scale[0] = scale;
        }
    }
#pragma unroll
    for (int k = 0; k < RP; ++k) {
        auto wide = [](uint16_t w) __attribute__((always_inline)) {
            return DT == 0 ? (float)__builtin_bit_cast(_Float16, w) : __builtin_bit_cast(float, (uint32_t)w << 16);
        };
        float a = wide(pair[k][0]), b = wide(pair[k][1]);
        if (turns) {
            float c, s;
            rope_angle(freq, (double)rat[k].position, p.rope.magnitude, c, s);
            rope_turn(a, b, c, s);
        }
        const float top = over_lanes_max<RL>(fmaxf(finite_magnitude(a), finite_magnitude(b))), scale = fmaxf(top / 127.0f, kLeastScale);
        if (rput[k]) {
            rat[k].row[DC + one] = (char)quantise(a, scale);
            rat[k].row[DC + two] = (char)quantise(b, scale);
            if (j == 0) rat[k].scale[1] = scale;
        }
    }
}

template <int DT> void launch(const LatentAppendParams& p, int dc, int dr, hipStream_t stream) {
    const int each = dc == 128 || dr == 32 ? 4 : 2;          // tokens of a wave (T above)
    const dim3 grid((unsigned)((p.tokens + 4 * each - 1) / (4 * each)));
#define INTFA_CALL(DC) do { \
        if (dr == 64) hipLaunchKernelGGL((latent_append_kernel<DT, DC, 64>), grid, dim3(256), 0, stream, p); \
        else hipLaunchKernelGGL((latent_append_kernel<DT, DC, 32>), grid, dim3(256), 0, stream, p); } while (0)
    if (dc == 512) INTFA_CALL(512); else if (dc == 256) INTFA_CALL(256); else INTFA_CALL(128);
#undef INTFA_CALL
}

}  // namespace

extern "C" {

int intfa_latent_append_int8(const intfa_latent_append_params* p, void* stream) {
    if (p == nullptr || p->c_new == nullptr || p->k_new == nullptr || p->seqlens_k == nullptr) return INTFA_ERR_NULL;
    const intfa_latent_cache& c = p->cache;
    const int rc = latent_cache_check(&c);
    if (rc != INTFA_OK) return rc;
    if (p->batch <= 0) return INTFA_ERR_SHAPE;
    if (p->seqlen_new <= 0 || p->seqlen_new > 1 << 30) return INTFA_ERR_SEQLEN;
    if (p->dtype != INTFA_F16 && p->dtype != INTFA_BF16) return INTFA_ERR_DTYPE;
    if (p->rope.freqs != nullptr && !rope_valid(&p->rope, c.rope_dim)) return INTFA_ERR_ROPE;
    if (!aligned_to(p->c_new, 16) || !aligned_to(p->k_new, 16) || p->cn_stride_b % 8 || p->cn_stride_n % 8 || p->kn_stride_b % 8 || p->kn_stride_n % 8 ||
        !aligned_to(p->norm_weight, 16) || !aligned_to(p->seqlens_k, 4) || !aligned_to(p->seqlens_new, 4) || !aligned_to(p->rope.freqs, 8)) return INTFA_ERR_ALIGN;
    if (p->norm_weight != nullptr && (!(p->norm_eps > 0.f) || p->norm_eps > 3.402823466e38f)) return INTFA_ERR_SHAPE;
    const int64_t tokens = size_product(p->batch, p->seqlen_new);
    if (tokens > 1ll << 30) return INTFA_ERR_SHAPE;          // (tokens are 32-bit numbers, and so are the threads of a launch)
    LatentAppendParams ap{};
    if (size_product(tokens, 64) >= 1ll << 32) return INTFA_ERR_SHAPE;
    ap.c = (const char*)p->c_new; ap.k = (const char*)p->k_new; ap.weight = (const char*)p->norm_weight;
    ap.c_sb = p->cn_stride_b * 2; ap.c_sn = p->cn_stride_n * 2; ap.k_sb = p->kn_stride_b * 2; ap.k_sn = p->kn_stride_n * 2;
    ap.rows = (char*)c.rows; ap.scale = c.scale; ap.r_sp = c.r_stride_p; ap.s_sp = c.s_stride_p; ap.r_sn = (int32_t)c.r_stride_n; ap.s_sn = (int32_t)c.s_stride_n;
    ap.table = c.block_table; ap.bt_sb = c.bt_stride_b; ap.seqlens_k = p->seqlens_k; ap.seqlens_new = p->seqlens_new;
    ap.rope = {p->rope.freqs, p->rope.freqs != nullptr ? p->rope.pairs : 0, p->rope.interleaved, p->rope.magnitude};
    ap.eps = p->norm_eps;
    ap.tokens = (int32_t)tokens; ap.seqlen_new = p->seqlen_new;
    ap.page_log2 = __builtin_ctz((unsigned)c.page_size); ap.num_pages = c.num_pages; ap.table_width = c.table_width;
    ap.d_seqlen = make_fast_div(p->seqlen_new);
    if (p->dtype == INTFA_F16) launch<0>(ap, c.latent_dim, c.rope_dim, (hipStream_t)stream); else launch<1>(ap, c.latent_dim, c.rope_dim, (hipStream_t)stream);
    return (int)hipGetLastError();
}

}  // extern "C"
