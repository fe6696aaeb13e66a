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
#include "intfa_paged_host.h"
#include "intfa_splitkv.h"

namespace intfa {

// The kernel's own argument block; its fields are scalar loads, made where they are used: paged_args() gives a pointer that the compiler takes for
// a new one (a hundred fields and what follows from them held from the prologue to the end would not fit the scalar registers).
typedef const __attribute__((address_space(4))) PagedParams* PagedArgs;
__device__ __forceinline__ PagedArgs paged_args() {
    PagedArgs p = (PagedArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
// The same at the start of a kernel, with all lines of the block requested at once: it is cold in each launch, and the prologue's first dozen reads of it
// would each be a trip to memory of their own.
__device__ __forceinline__ PagedArgs paged_args_first() {
    PagedArgs p = (PagedArgs)__builtin_amdgcn_kernarg_segment_ptr();
    typedef const __attribute__((address_space(4))) int* Words;
    const Words w = (Words)p;
    static_assert((sizeof(PagedParams) - 1) / 64 == 5, "the statement names a word of each line");
    asm("" : "+s"(p) : "s"(w[0]), "s"(w[16]), "s"(w[32]), "s"(w[48]), "s"(w[64]), "s"(w[80]));
    return p;
}

constexpr int kPagedWaves = 4;
constexpr float kPShift = 14.f;       // P is held as 2^14 p: fp16 keeps its 11 bits down to p = 2^-28, times the ratio of two pages' scales

// Four int8 of a word as fp16
__device__ __forceinline__ void i8x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    const v2h bias = {(_Float16)-1152.f, (_Float16)-1152.f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + bias);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + bias);
}
// Byte `b` of two words as a pair of fp16
template <int B> __device__ __forceinline__ uint32_t i8_pair_to_f16(uint32_t first, uint32_t second) {
    const uint32_t u = __builtin_amdgcn_perm(second, first, 0x0c000c00u | (uint32_t)(4 + B) << 16 | (uint32_t)B) ^ 0x64806480u;
    const v2h bias = {(_Float16)-1152.f, (_Float16)-1152.f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, u) + bias);
}

__device__ __forceinline__ int paged_div(int n, const __attribute__((address_space(4))) FastDiv& d) { return fast_div(n, FastDiv{d.m, d.s}); }

// (scalar loads of device memory that nothing in the launch writes)
typedef const __attribute__((address_space(4))) int32_t* PagedInts;
typedef const __attribute__((address_space(4))) float* PagedFloats;

// ---- who works on what
// The keys of all sequences, K/V heads and row tiles (the items, in that order) are one line of units of 2^unit_log2 keys, at least one per item, and
// every workgroup takes an equal piece of it: whatever the lengths, all compute units end together.  An item that lies in several pieces is merged
// by the workgroup that finishes its part last.  Each item has kPagedLead units without keys ahead of its own: beginning an item and ending one take a
// workgroup about as long as their keys would (8 us, where a unit takes 4 with the whole card reading), and without them the workgroups that have parts
// of two items came in last (ragged batch of 16, 512 workgroups of 5.3 units: 42 -> 47 us).
struct PagedItem { int z, hk, tile, n, m, units; };      // n: keys of the sequence, m: its new tokens, units: of each of its items, with the lead
__device__ __forceinline__ int paged_keys(PagedArgs p, int z) {
    const int most = p->table_width << p->page_log2, n = p->seqlens_k[z];
    return n < 0 ? 0 : n < most ? n : most;
}
__device__ __forceinline__ int paged_units(PagedArgs p, int n) {
    const int u = (n + (1 << p->unit_log2) - 1) >> p->unit_log2;
    return (u > 1 ? u : 1) + kPagedLead;
}
__device__ __forceinline__ void paged_sequence(PagedArgs p, int z, PagedItem& t) {
    const int most = p->table_width << p->page_log2, n = ((PagedInts)p->seqlens_k)[z];
    t.z = z;
    t.n = n < 0 ? 0 : n < most ? n : most;
    t.units = paged_units(p, t.n);
    t.m = p->seqlen;
    if (p->seqlens_q != nullptr) {
        const int m = ((PagedInts)p->seqlens_q)[z];
        t.m = m < 0 ? 0 : m < t.m ? m : t.m;
    }
}
// Finds this workgroup's piece [first, end) of the line, and the item that `first` lies in: it begins at unit `start`.  The line is cut for `grid`
// workgroups, those of the launch or as many as there are units: none of them has an empty piece (first == end: not one of them).  The host
// keeps the number of units times that of workgroups below 2^32.
// (Every wave finds it for itself, without LDS: sequences are dealt to the lanes in runs, of one up to 64 sequences, and a scan gives the total and
// every run's place.)
__device__ __forceinline__ uint32_t paged_find(PagedArgs p, PagedItem& t, uint32_t& first, uint32_t& end, uint32_t& start, uint32_t& grid) {
    const int per = p->heads_kv * p->tiles, run = (p->batch + 63) / 64, lane = threadIdx.x & 63, z0 = lane * run;
    uint32_t mine = 0;
    for (int z = z0; z < z0 + run && z < p->batch; ++z) mine += (uint32_t)paged_units(p, paged_keys(p, z)) * (uint32_t)per;
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)upto, d);
        if (lane >= d) upto += o;
    }
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    grid = (uint32_t)p->grid < total ? (uint32_t)p->grid : total;
    first = end = 0;
    if (blockIdx.x >= grid) return total;
    first = (uint32_t)blockIdx.x * total / grid;
    end = ((uint32_t)blockIdx.x + 1) * total / grid;
    // the lane whose run holds `first`, and the sequence in it
    const int holder = __builtin_ctzll(__ballot(first < upto));
    uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), holder);
    int z = holder * run;
    paged_sequence(p, z, t);
    while (first >= at + (uint32_t)(t.units * per)) {
        at += (uint32_t)(t.units * per);
        paged_sequence(p, ++z, t);
    }
    const uint32_t item = (first - at) / (uint32_t)t.units;
    start = at + item * (uint32_t)t.units;
    t.hk = paged_div((int)item, p->d_tiles);
    t.tile = (int)item - t.hk * p->tiles;
    return total;
}
// The workgroup that has unit u of a line of `total`.
__device__ __forceinline__ int paged_owner(uint32_t u, uint32_t total, uint32_t grid) { return (int)(((u + 1) * grid - 1) / total); }

// Keys that token i of the sequence sees: the first so many.
__device__ __forceinline__ int paged_token_keys(PagedArgs p, const PagedItem& t, int i) {
    const int seen = t.n - t.m + i + 1;
    return !p->causal || seen > t.n ? t.n : seen < 0 ? 0 : seen;
}

// The rows of a tile on their way to LDS: requested first, ahead of the cache's (loads come back in order), then turned and stored.  A row is D / 16
// units of sixteen elements, a lane each.
template <int D, int DT, int R, int THREADS> struct PagedQueries {
    static constexpr int U = D / 16, N = (R * U + THREADS - 1) / THREADS, ROW = 2 * D + 16;      // ROW: bytes in LDS (16 more: sixteen rows in sixteen banks)
    v4i x[N][2];
    double freq;
    int first_token, tokens;
    bool rope, interleaved;
    int pairs;
    __device__ __forceinline__ void request(PagedArgs p, const PagedItem& t, int row0) {
        rope = p->rope.freqs != nullptr;
        interleaved = p->rope.interleaved != 0;
        pairs = rope ? p->rope.pairs : 0;
        const int row_last = row0 + R < p->rows ? row0 + R - 1 : p->rows - 1;
        first_token = paged_div(row0, p->d_group);
        tokens = paged_div(row_last, p->d_group) - first_token + 1;
        freq = 0.0;
        if ((int)threadIdx.x < pairs) freq = p->rope.freqs[threadIdx.x];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = (int)threadIdx.x + k * THREADS, r = i / U, u = i % U, row = row0 + r, token = paged_div(row, p->d_group);
            int first, second;
            rope_unit(u, pairs, interleaved, first, second);
            x[k][0] = x[k][1] = (v4i){0, 0, 0, 0};
            if (i < R * U && row < p->rows) {
                const char* src = p->q + t.z * p->q_sb + (t.hk * p->group + row - token * p->group) * p->q_sh + token * p->q_sn;
                x[k][0] = *(const v4i*)(src + 2 * first);
                x[k][1] = *(const v4i*)(src + 2 * second);
            }
        }
    }
    // The angles of the tile's tokens, each once: angles[token * pairs + pair] = (cos, sin).  Threads beyond the pairs take further tokens.
    __device__ __forceinline__ void turn_angles(PagedArgs p, const PagedItem& t, v2f* angles) const {
        const float magnitude = p->rope.magnitude;
        const int position = t.n - t.m + first_token;
        for (int i = threadIdx.x; i < tokens * pairs; i += THREADS) {
            const int token = i / pairs, pair = i - token * pairs;
            float c, s;
            rope_angle(pair == (int)threadIdx.x ? freq : p->rope.freqs[pair], position + token, magnitude, c, s);
            angles[i] = (v2f){c, s};
        }
    }
    // To LDS as fp16 with a power of two of the row's own taken out (`factor` gets it back, with the softmax's scale in base 2): the row's largest element
    // is brought to 2^8, so that neither the range of bf16 nor a rotation leaves fp16's, and what lies under fp16's smallest step is 2^-32 of it.
    // 16-bit queries are held exactly that way; rotated ones are not 16-bit numbers, and what their rounding leaves goes to q_rest for a second product
    // (22 bits; one alone would put 2^-12 of each |q k| into the scores, more than P's rounding does to the result).
    __device__ __forceinline__ void stage(PagedArgs p, int row0, const v2f* angles, char* q_lds, char* q_rest, float* factor) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int i = (int)threadIdx.x + k * THREADS, r = i / U, u = i % U;
            if (R * U % THREADS != 0 && i >= R * U) continue;
            int first, second;
            rope_unit(u, pairs, interleaved, first, second);
            float y[16];
            unpack8<DT>(x[k][0], y);
            unpack8<DT>(x[k][1], y + 8);
            if (8 * u < pairs) {
                int token = paged_div(row0 + r, p->d_group) - first_token;
                token = token < tokens ? token : tokens - 1;
                float c[8], s[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const v2f a = angles[token * pairs + 8 * u + j];
                    c[j] = a[0];
                    s[j] = a[1];
                }
                rope_turn_unit(y, c, s, interleaved);
            }
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint32_t a = __builtin_bit_cast(uint32_t, y[j]) & 0x7fffffffu;
                top = top > a ? top : a;
            }
#pragma unroll
            for (int w = 1; w < U; w <<= 1) {
                const uint32_t a = (uint32_t)__shfl_xor((int)top, w);
                top = top > a ? top : a;
            }
            int e = (int)(top >> 23) - 127;
            e = e < -100 ? -100 : e > 100 ? 100 : e;
            const float down = __builtin_bit_cast(float, (uint32_t)(127 + 8 - e) << 23);
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                h[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){y[2 * j] * down, y[2 * j + 1] * down}, v2h));
            *(v4i*)(q_lds + r * ROW + 2 * first) = (v4i){(int)h[0], (int)h[1], (int)h[2], (int)h[3]};
            *(v4i*)(q_lds + r * ROW + 2 * second) = (v4i){(int)h[4], (int)h[5], (int)h[6], (int)h[7]};
            if (rope) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const v2f near = __builtin_convertvector(__builtin_bit_cast(v2h, h[j]), v2f);
                    h[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){y[2 * j] * down - near[0], y[2 * j + 1] * down - near[1]}, v2h));
                }
                *(v4i*)(q_rest + r * ROW + 2 * first) = (v4i){(int)h[0], (int)h[1], (int)h[2], (int)h[3]};
                *(v4i*)(q_rest + r * ROW + 2 * second) = (v4i){(int)h[4], (int)h[5], (int)h[6], (int)h[7]};
            }
            if (u == 0) factor[r] = __builtin_bit_cast(float, (uint32_t)(127 + e - 8) << 23) * p->qk_scale_log2;
        }
    }
};

// ---- partial results: a slot of R rows for a workgroup's first item (2 g) and one for its last (2 g + 1), the only ones that it can have parts of.
// Written and read past the XCDs' L2s, which are not coherent with each other (see intfa_splitkv.h).
struct PagedParts {
    BufferRsrc o, s;
    __device__ __forceinline__ PagedParts(PagedArgs p, int R, int D, int slot) {
        o = __builtin_amdgcn_make_buffer_rsrc(p->parts + (int64_t)slot * R * D, 0, R * D * 4, 0x00020000);
        s = __builtin_amdgcn_make_buffer_rsrc(p->part_stats + (int64_t)slot * R * 2, 0, R * 8, 0x00020000);
    }
    __device__ __forceinline__ void put(uint32_t row, int D, int col, v4f x) const {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, x), o, (row * (uint32_t)D + (uint32_t)col) * 4u, 0, kSplitAux);
    }
    __device__ __forceinline__ void put_stats(uint32_t row, float m, float l) const {
        typedef unsigned v2u __attribute__((ext_vector_type(2)));
        __builtin_amdgcn_raw_buffer_store_b64((v2u){__builtin_bit_cast(unsigned, m), __builtin_bit_cast(unsigned, l)}, s, row * 8u, 0, kSplitAux);
    }
};

// An item's ticket: the launch's epoch (upper 48 bits) and its arrivals so far.  The word is not cleared: every piece looks at it when it starts, and one
// that finds another epoch's exchanges it for (epoch, 0) before its own arrival (a word exchanged by another since then is left alone).  The last
// arrival leaves zero behind, so that the replays of a captured graph, whose epoch is a constant, find none of their own.
__device__ __forceinline__ uint64_t* paged_ticket(PagedArgs p, const PagedItem& t) {
    return p->ticket + (int64_t)((t.z * p->heads_kv + t.hk) * p->tiles + t.tile) * kTicketStride;
}
__device__ __forceinline__ void paged_open_ticket(PagedArgs p, uint64_t* word, uint64_t seen) {
    if (threadIdx.x == 0 && (seen ^ p->epoch) >= 1u << 16)
        __hip_atomic_compare_exchange_strong(word, &seen, p->epoch, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// True for the last of `pieces` arrivals.
__device__ __forceinline__ bool paged_last_arrival(PagedArgs p, uint64_t* word, uint32_t* lds, int pieces) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this wave's part has reached the point of coherence
    __syncthreads();
    if (threadIdx.x == 0) {
        const bool last = __hip_atomic_fetch_add(word, (uint64_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (p->epoch | (uint64_t)(pieces - 1));
        if (last) __hip_atomic_store(word, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *lds = last;
    }
    __syncthreads();
    const bool last = __builtin_amdgcn_readfirstlane((int)*lds) != 0;
    if (last) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    return last;
}

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
        auto add = [&](auto many) __attribute__((always_inline)) {      // (so many loads under way together: each takes a microsecond)
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
        store_out4<DT>(p->out + t.z * p->o_sb + head * p->o_sh + token * p->o_sn + col * 2, acc * (empty ? 0.f : 1.f / l));
        if (p->lse != nullptr && col == 0)
            p->lse[((int64_t)t.z * p->heads + head) * p->seqlen + token] = empty ? -INFINITY : m + __builtin_log2f(l) - kPShift;
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
    PagedArgs p = paged_args_first();
    PagedItem t;
    uint32_t first, end, start, grid;
    const uint32_t total = paged_find(p, t, first, end, start, grid);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), x = lane & 15, c = lane >> 4;
  for (uint32_t at = first; at < end;) {
    const int row0 = t.tile * R;
    // this workgroup's part of the item: keys key_first .. most - 1
    const uint32_t item_end = start + (uint32_t)t.units;
    if (end <= start + (uint32_t)kPagedLead) break;        // (no key of the last item)
    const bool whole = at <= start + (uint32_t)kPagedLead && item_end <= end;
    const int key_first = (at - start > (uint32_t)kPagedLead ? (int)(at - start) - kPagedLead : 0) << p->unit_log2;
    uint64_t ticket_seen = 0;
    if (!whole && threadIdx.x == 0) ticket_seen = __hip_atomic_load(paged_ticket(p, t), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    Queries queries;
    queries.request(p, t, row0);
    const bool rope = queries.rope;
    // (a row past the last one or a token past the sequence's new ones counts like the others here; what it gives is not used)
    int last_token = queries.first_token + queries.tokens - 1;
    last_token = last_token < t.m ? last_token : t.m - 1;
    int most = queries.first_token < t.m ? paged_token_keys(p, t, last_token) : 0;
    const int least = paged_token_keys(p, t, queries.first_token);
    if (item_end > end) {
        const int limit = (int)(end - start - (uint32_t)kPagedLead) << p->unit_log2;
        most = most < limit ? most : limit;
    }
    // the first keys are on their way while the queries are staged
    PagedStream<D, ONE> stream(p, t, most, x, c);
    PagedStep<D> now;
    int key0 = key_first + wave * STEP;
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
        queries.turn_angles(p, t, (v2f*)o_lds);
        __syncthreads();
    }
    queries.stage(p, row0, (const v2f*)o_lds, q_lds, q_rest, factor_lds);
    if (!whole) paged_open_ticket(p, paged_ticket(p, t), ticket_seen);
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
        float v_top = 0x1p-120f;
#pragma unroll
        for (int g = 0; g < G; ++g) v_top = fmaxf(v_top, now.has[g] ? fabsf(now.vs[g]) : 0.f);
        const float v_inv = __builtin_amdgcn_rcpf(v_top);
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
            const float m_new = fmaxf(m[rt], top), frame = (m_new == -INFINITY ? 0.f : m_new) - kPShift;
            alpha[rt] = m_new == -INFINITY ? 1.f : fast_exp2(m[rt] - m_new);
            m[rt] = m_new;
            float sum = 0.f;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[g][i] = fast_exp2(s[g][i] - frame);
                    sum += s[g][i];
                    s[g][i] *= v_rel[g];
                }
            l[rt] = l[rt] * alpha[rt] + sum;
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
                for (int i = 0; i < 4; ++i) o[rt][j][i] = fmaf(a[i], v_top, o[rt][j][i]);
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
        const int r = (int)threadIdx.x / 16, part = (int)threadIdx.x % 16, row = row0 + 16 * rt + r;      // D / 16 columns of one row
        static_assert(THREADS == 256, "a thread per row and sixteenth of it");
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, m_lds[w * R + 16 * rt + r]);
        const int token = paged_div(row, p->d_group);
        const bool empty = top == -INFINITY || (whole && token >= t.m);
        float sum = 0.f, weight[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            weight[w] = empty ? 0.f : fast_exp2(m_lds[w * R + 16 * rt + r] - top);
            sum += weight[w] * l_lds[w * R + 16 * rt + r];
        }
        const int head = t.hk * p->group + row - token * p->group;
        if (row < p->rows) {
            if (whole) {
                const float inv = empty ? 0.f : 1.f / sum;
                char* const dst = p->out + t.z * p->o_sb + head * p->o_sh + token * p->o_sn + part * DT16 * 2;
#pragma unroll
                for (int j = 0; j < DT16; j += 4) {
                    v4f a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < W; ++w) a += weight[w] * *(const v4f*)(o_lds + (w * 16 + r) * O_ROW + part * DT16 + j);
                    store_out4<DT>(dst + j * 2, a * inv);
                }
                if (p->lse != nullptr && part == 0)
                    p->lse[((int64_t)t.z * p->heads + head) * p->seqlen + token] = empty ? -INFINITY : top + __builtin_log2f(sum) - kPShift;
            } else {
                const PagedParts mine(p, R, D, 2 * (int)blockIdx.x + (at != first));
#pragma unroll
                for (int j = 0; j < DT16; j += 4) {
                    v4f a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < W; ++w) a += weight[w] * *(const v4f*)(o_lds + (w * 16 + r) * O_ROW + part * DT16 + j);
                    mine.put((uint32_t)(16 * rt + r), D, part * DT16 + j, a);
                }
                if (part == 0) mine.put_stats((uint32_t)(16 * rt + r), top, sum);
            }
        }
    }
    if (!whole) {
        const int one = paged_owner(start + (uint32_t)kPagedLead, total, grid), last = paged_owner(item_end - 1, total, grid);
        if (paged_last_arrival(p, paged_ticket(p, t), &arrival_lds, last - one + 1))
            paged_merge<D, DT, R, THREADS>(p, t, row0, one, last - one + 1, (uint32_t)one * total / grid >= start, o_lds);
    }
    // ---- the next item of the line
    at = item_end;
    if (at >= end) break;
    start = at;
    if (++t.tile == p->tiles) {
        t.tile = 0;
        if (++t.hk == p->heads_kv) {
            t.hk = 0;
            paged_sequence(p, t.z + 1, t);
        }
    }
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
