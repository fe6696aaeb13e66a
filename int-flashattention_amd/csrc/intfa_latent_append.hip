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
    int32_t least_e;                                 // the least power of two that a row counts as for its norm
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

// f over the 8 or 16 neighbouring lanes of a token, for all of them: by the rows' own permutations (neighbours, pairs, halves of eight, mirrored)
template <int LANES, typename T, typename F> __device__ __forceinline__ T over_lanes(T v, F f) {
    static_assert(LANES == 8 || LANES == 16, "");
    auto moved = [&](auto ctrl) __attribute__((always_inline)) { return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true)); };
    v = f(v, moved(std::integral_constant<int, 0xb1>()));
    v = f(v, moved(std::integral_constant<int, 0x4e>()));
    v = f(v, moved(std::integral_constant<int, 0x141>()));
    if (LANES == 16) v = f(v, moved(std::integral_constant<int, 0x140>()));
    return v;
}
template <int LANES> __device__ __forceinline__ float over_lanes_max(float v) { return over_lanes<LANES>(v, [](float a, float b) { return fmaxf(a, b); }); }
template <int LANES> __device__ __forceinline__ float over_lanes_sum(float v) { return over_lanes<LANES>(v, [](float a, float b) { return a + b; }); }

// N values of a token's lane, all N * LANES of them, to int8: the scale, and the bytes four a word
template <int N, int LANES> __device__ __forceinline__ float to_bytes(const float (&x)[N], uint32_t (&q)[N / 4]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(x[i]));
    top = over_lanes_max<LANES>(top);
    const bool infinite = top > 3.402823466e38f;             // (of the token's lanes alike)
    if (__any(infinite)) {
        float finite = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) finite = fmaxf(finite, finite_magnitude(x[i]));
        top = over_lanes_max<LANES>(finite);
    }
    const float scale = fmaxf(top / 127.0f, kLeastScale), reciprocal = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) q[i] = quantise4(x + 4 * i, scale, reciprocal);
    if (infinite) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) q[i] = quantise(x[4 * i], scale) | quantise(x[4 * i + 1], scale) << 8 | quantise(x[4 * i + 2], scale) << 16 | quantise(x[4 * i + 3], scale) << 24;
    }
    return scale;
}

// A wave takes 64 / L tokens, nothing of it waits for another wave: L lanes a token, with units of sixteen elements of the latent part and some pairs of the rotary one.  Bound by its
// arithmetic: with more lanes a token (64, and 32 for the rotary part) what a token costs once - its place, the norm's root, the divisions, the sums over its lanes - was more than what
// its elements cost (16384 tokens of 512 + 64 16.2 us, and 11.9 so, 28.6 MB; 65536 tokens 24.5, 4.7 TB/s; one token 3.4).
template <int DT, int DC, int DR> __global__ void __launch_bounds__(256) latent_append_kernel(const LatentAppendParams p) {
    constexpr int L = DC == 512 ? 16 : 8, T = 64 / L, E = DC / L, U = E / 16, P = DR / 2 / L;
    const int lane = threadIdx.x & 63, l = lane % L, first = ((int)blockIdx.x * 4 + ((int)threadIdx.x >> 6)) * T;
    if (first >= p.tokens) return;
    // everything is requested before the first is used
    LatentPlace at;
    const bool put = latent_place(p, first + lane / L, at);
    const char* const c = p.c + at.z * p.c_sb + at.i * p.c_sn;
    const char* const k = p.k + at.z * p.k_sb + at.i * p.k_sn;
    v4i raw[2 * U], raw_weight[2 * U];
#pragma unroll
    for (int u = 0; u < 2 * U; ++u) raw[u] = *(const v4i*)(c + 2 * (16 * (l + L * (u / 2)) + 8 * (u & 1)));
    uint16_t pair[P][2];
    double freq[P];
    int one[P], two[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int j = l + L * i;
        const bool turns = p.rope.freqs != nullptr && j < p.rope.pairs;
        one[i] = turns && !p.rope.interleaved ? j : 2 * j;
        two[i] = turns && !p.rope.interleaved ? p.rope.pairs + j : 2 * j + 1;
        pair[i][0] = *(const uint16_t*)(k + 2 * one[i]);
        pair[i][1] = *(const uint16_t*)(k + 2 * two[i]);
        freq[i] = turns ? p.rope.freqs[j] : 0.0;
    }
    if (p.weight != nullptr) {
#pragma unroll
        for (int u = 0; u < 2 * U; ++u) raw_weight[u] = *(const v4i*)(p.weight + 2 * (16 * (l + L * (u / 2)) + 8 * (u & 1)));
    }
    // ---- the rotary part
    {
        float y[2 * P < 4 ? 4 : 2 * P];
#pragma unroll
        for (int i = 2 * P; i < 4; ++i) y[i] = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            auto wide = [](uint16_t w) __attribute__((always_inline)) {
                return DT == 0 ? (float)__builtin_bit_cast(_Float16, w) : __builtin_bit_cast(float, (uint32_t)w << 16);
            };
            float a = wide(pair[i][0]), b = wide(pair[i][1]);
            if (p.rope.freqs != nullptr) {
                float cosine, sine;
                rope_angle(freq[i], (double)at.position, p.rope.magnitude, cosine, sine);
                float ta = a, tb = b;
                rope_turn(ta, tb, cosine, sine);
                const bool turns = l + L * i < p.rope.pairs;
                a = turns ? ta : a;
                b = turns ? tb : b;
            }
            y[2 * i] = a;
            y[2 * i + 1] = b;
        }
        uint32_t q[sizeof(y) / 16];
        const float scale = to_bytes<sizeof(y) / 4, L>(y, q);
        if (put) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                at.row[DC + one[i]] = (char)(q[i / 2] >> (16 * (i & 1)));
                at.row[DC + two[i]] = (char)(q[i / 2] >> (16 * (i & 1) + 8));
            }
            if (l == 0) at.scale[1] = scale;
        }
    }
    // ---- the latent part
    float x[E];
#pragma unroll
    for (int u = 0; u < 2 * U; ++u) unpack8<DT>(raw[u], x + 8 * u);
    if (p.weight != nullptr) {
        // The squares are those of x / 2^e, 2^e the size of the row's largest element: they stay in range whatever the row's size.  (e from -40, or from 2^-50 of eps' root, under which
        // eps is all there is and eps / 4^e would leave fp32; 126 for a row with an infinity, which thereby becomes one of zeros, as its formula has it)
        typedef unsigned short v2us __attribute__((ext_vector_type(2)));
        v2us most = {0, 0};                    // (magnitudes of 16-bit numbers are ordered as their bits are)
#pragma unroll
        for (int u = 0; u < 2 * U; ++u)
#pragma unroll
            for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(v2us, raw[u][w] & 0x7fff7fff));
        float two_tops[8];
        unpack8<DT>((v4i){__builtin_bit_cast(int, most), 0, 0, 0}, two_tops);
        uint32_t top = __builtin_bit_cast(uint32_t, two_tops[0]), other = __builtin_bit_cast(uint32_t, two_tops[1]);
        top = over_lanes<L>(top > other ? top : other, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        int e = (int)(top >> 23) - 127;
        e = e < p.least_e ? p.least_e : e > 126 ? 126 : e;
        const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            x[i] *= down;
            sum = fmaf(x[i], x[i], sum);
        }
        sum = over_lanes_sum<L>(sum);
        const float r = 1.0f / sqrtf(sum * (1.0f / DC) + p.eps * down * down);
#pragma unroll
        for (int u = 0; u < 2 * U; ++u) {
            float weight[8];
            unpack8<DT>(raw_weight[u], weight);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[8 * u + i] = x[8 * u + i] * r * weight[i];
        }
    }
    uint32_t q[E / 4];
    const float scale = to_bytes<E, L>(x, q);
    if (put) {
#pragma unroll
        for (int u = 0; u < U; ++u) *(v4i*)(at.row + 16 * (l + L * u)) = (v4i){(int)q[4 * u], (int)q[4 * u + 1], (int)q[4 * u + 2], (int)q[4 * u + 3]};
        if (l == 0) at.scale[0] = scale;
    }
}

constexpr int kAppendThreads = 256;
int64_t append_groups(int64_t tokens, int dc) {
    const int each = 4 * (dc == 512 ? 4 : 8);  // tokens of a workgroup: of its waves, T each
    return tokens / each + (tokens % each != 0);
}
template <int DT> void launch(const LatentAppendParams& p, int dc, int dr, hipStream_t stream) {
    const dim3 grid((unsigned)append_groups(p.tokens, dc));
#define INTFA_CALL(DC) do { \
        if (dr == 64) hipLaunchKernelGGL((latent_append_kernel<DT, DC, 64>), grid, dim3(kAppendThreads), 0, stream, p); \
        else hipLaunchKernelGGL((latent_append_kernel<DT, DC, 32>), grid, dim3(kAppendThreads), 0, stream, p); } while (0)
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
    // (tokens are 32-bit numbers, and so are the threads of a launch)
    if (tokens > 1ll << 30 || append_groups(tokens, c.latent_dim) * kAppendThreads >= 1ll << 32) return INTFA_ERR_SHAPE;
    LatentAppendParams ap{};
    ap.c = (const char*)p->c_new; ap.k = (const char*)p->k_new; ap.weight = (const char*)p->norm_weight;
    ap.c_sb = p->cn_stride_b * 2; ap.c_sn = p->cn_stride_n * 2; ap.k_sb = p->kn_stride_b * 2; ap.k_sn = p->kn_stride_n * 2;
    ap.rows = (char*)c.rows; ap.scale = c.scale; ap.r_sp = c.r_stride_p; ap.s_sp = c.s_stride_p; ap.r_sn = (int32_t)c.r_stride_n; ap.s_sn = (int32_t)c.s_stride_n;
    ap.table = c.block_table; ap.bt_sb = c.bt_stride_b; ap.seqlens_k = p->seqlens_k; ap.seqlens_new = p->seqlens_new;
    ap.rope = {p->rope.freqs, p->rope.freqs != nullptr ? p->rope.pairs : 0, p->rope.interleaved, p->rope.magnitude};
    ap.eps = p->norm_eps;
    const int root = p->norm_weight != nullptr ? ((int)(__builtin_bit_cast(uint32_t, p->norm_eps) >> 23) - 127) / 2 : 0;
    ap.least_e = root - 50 > -40 ? root - 50 : -40;
    ap.tokens = (int32_t)tokens; ap.seqlen_new = p->seqlen_new;
    ap.page_log2 = __builtin_ctz((unsigned)c.page_size); ap.num_pages = c.num_pages; ap.table_width = c.table_width;
    ap.d_seqlen = make_fast_div(p->seqlen_new);
    if (p->dtype == INTFA_F16) launch<0>(ap, c.latent_dim, c.rope_dim, (hipStream_t)stream); else launch<1>(ap, c.latent_dim, c.rope_dim, (hipStream_t)stream);
    return (int)hipGetLastError();
}

}  // extern "C"
