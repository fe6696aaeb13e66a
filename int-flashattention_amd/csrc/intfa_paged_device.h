// What the attention kernels over a paged int8 cache share: how the work is dealt, the queries on their way into the products, partial results.
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
// The work is a line: the row tiles of all sequences, each with all K/V heads (an item: one tile and head), and each item's keys as units of
// 2^unit_log2, at least one.  Every workgroup takes an equal piece of the line: whatever the lengths and the mask, all compute units end together.  An
// item that lies in several pieces is merged by the workgroup that finishes its part last.  Ahead of its own units each item has `lead`
// without keys: beginning an item and ending one take a workgroup about as long as their keys would (decode-shaped: 8 us, where a unit takes 4 with the whole
// card reading), and without them the workgroups that have parts of two items came in last (ragged batch of 16, 512 workgroups of 5.3 units: 42 -> 47 us).
struct PagedItem {
    int z, tile, hk;
    int n, m;              // keys of the sequence, and its new tokens
    int first_token;       // of the tile
    int most;              // keys that some row of the tile sees: the first so many
    int units;             // with the lead
};
// Keys that a tile's rows see: those of its last token.  rows: of a tile.
__device__ __forceinline__ int paged_seen(PagedArgs p, int n, int m, int tile, int rows, int& first_token) {
    const int row = tile * rows;
    first_token = paged_div(row, p->d_group);
    if (first_token >= m) return 0;
    int last = paged_div(row + rows < p->rows ? row + rows - 1 : p->rows - 1, p->d_group);
    last = last < m ? last : m - 1;
    const int seen = n - m + last + 1;
    return !p->causal ? n : seen < 0 ? 0 : seen;
}
__device__ __forceinline__ int paged_units(PagedArgs p, int keys) {
    const int u = (keys + (1 << p->unit_log2) - 1) >> p->unit_log2;
    return (u > 1 ? u : 1) + p->lead;
}
// The tile `pair` of the line's order (sequence, tile).
template <typename Ints> __device__ __forceinline__ void paged_pair(PagedArgs p, int pair, int rows, PagedItem& t) {
    t.z = paged_div(pair, p->d_tiles);
    t.tile = pair - t.z * p->tiles;
    const int most = p->table_width << p->page_log2, n = ((Ints)p->seqlens_k)[t.z];
    t.n = n < 0 ? 0 : n < most ? n : most;
    t.m = p->seqlen;
    if (p->seqlens_q != nullptr) {
        const int m = ((Ints)p->seqlens_q)[t.z];
        t.m = m < 0 ? 0 : m < t.m ? m : t.m;
    }
    t.most = paged_seen(p, t.n, t.m, t.tile, rows, t.first_token);
    t.units = paged_units(p, t.most);
}
// A workgroup's piece [first, end) of the line, and the item that it is at: the item begins at unit `start`.  The line is cut for `grid` workgroups, those
// of the launch or as many as there are units: none of them has an empty piece (first == end: not one of them).  The host keeps the number of units times
// that of workgroups below 2^32.
struct PagedPiece { uint32_t total, grid, first, end, start; };
// (Every wave finds it for itself, without LDS: tiles are dealt to the lanes in runs, of one up to 64 tiles, and a scan gives the total and every
// run's place.)
__device__ __forceinline__ PagedPiece paged_find(PagedArgs p, int rows, PagedItem& t) {
    const uint32_t per = (uint32_t)p->heads_kv;
    const int pairs = p->batch * p->tiles, run = (pairs + 63) / 64, lane = threadIdx.x & 63, pair0 = lane * run;
    uint32_t mine = 0;
    for (int k = pair0; k < pair0 + run && k < pairs; ++k) {
        PagedItem other;
        paged_pair<const int32_t*>(p, k, rows, other);
        mine += (uint32_t)other.units * per;
    }
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)upto, d);
        if (lane >= d) upto += o;
    }
    PagedPiece w;
    w.total = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    w.grid = (uint32_t)p->grid < w.total ? (uint32_t)p->grid : w.total;
    w.first = w.end = w.start = 0;
    if (blockIdx.x >= w.grid) return w;
    w.first = (uint32_t)blockIdx.x * w.total / w.grid;
    w.end = ((uint32_t)blockIdx.x + 1) * w.total / w.grid;
    // the lane whose run holds `first`, and the tile in it
    const int holder = __builtin_ctzll(__ballot(w.first < upto));
    uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), holder);
    int pair = holder * run;
    paged_pair<PagedInts>(p, pair, rows, t);
    while (w.first >= at + (uint32_t)t.units * per) {
        at += (uint32_t)t.units * per;
        paged_pair<PagedInts>(p, ++pair, rows, t);
    }
    t.hk = (int)((w.first - at) / (uint32_t)t.units);
    w.start = at + (uint32_t)(t.hk * t.units);
    return w;
}
// The item behind t, if the piece reaches it.
__device__ __forceinline__ bool paged_next(PagedArgs p, int rows, PagedItem& t, PagedPiece& w) {
    w.start += (uint32_t)t.units;
    if (w.start >= w.end) return false;
    if (++t.hk == p->heads_kv) {
        t.hk = 0;
        paged_pair<PagedInts>(p, t.z * p->tiles + t.tile + 1, rows, t);
    }
    return true;
}
// A workgroup's part of an item.
struct PagedPart { int key_first, key_end; bool none, whole; int one, pieces; bool first_is_first; uint32_t slot; };
__device__ __forceinline__ PagedPart paged_part(PagedArgs p, const PagedItem& t, const PagedPiece& w) {
    const uint32_t keys = w.start + (uint32_t)p->lead, item_end = w.start + (uint32_t)t.units;
    PagedPart a;
    a.none = w.end <= keys;                                // (the piece ends in the item's lead)
    a.whole = w.first <= keys && item_end <= w.end;
    a.key_first = w.first > keys ? (int)(w.first - keys) << p->unit_log2 : 0;
    a.key_end = t.most;
    if (item_end > w.end && !a.none) {
        const int limit = (int)(w.end - keys) << p->unit_log2;
        a.key_end = a.key_end < limit ? a.key_end : limit;
    }
    auto owner = [&](uint32_t unit) __attribute__((always_inline)) { return (int)(((unit + 1) * w.grid - 1) / w.total); };
    a.one = owner(keys);
    a.pieces = owner(item_end - 1) - a.one + 1;
    a.first_is_first = (uint32_t)a.one * w.total / w.grid >= w.start;
    a.slot = 2 * blockIdx.x + (w.start > w.first);         // (the piece's first item, or its last)
    return a;
}

// Keys that token i of the sequence sees: the first so many.
__device__ __forceinline__ int paged_token_keys(PagedArgs p, const PagedItem& t, int i) {
    const int seen = t.n - t.m + i + 1;
    return !p->causal || seen > t.n ? t.n : seen < 0 ? 0 : seen;
}

// The frequencies to LDS, once per workgroup: requested at the kernel's start, stored when its own place in the line is known.
__device__ __forceinline__ double paged_frequency(PagedArgs p) {
    return p->rope.freqs != nullptr && (int)threadIdx.x < p->rope.pairs ? p->rope.freqs[threadIdx.x] : 0.0;
}

// The rows of a tile on their way to LDS: requested first, ahead of the cache's (loads come back in order), then turned and stored.  A row is D / 16
// units of sixteen elements, a lane each.
template <int D, int DT, int R, int THREADS> struct PagedQueries {
    static constexpr int U = D / 16, N = (R * U + THREADS - 1) / THREADS, ROW = 2 * D + 16;      // ROW: bytes in LDS (16 more: sixteen rows in sixteen banks)
    v4i x[N][2];
    int first_token, tokens;
    bool rope, interleaved;
    int pairs;
    __device__ __forceinline__ void request(PagedArgs p, const PagedItem& t, int row0) {
        rope = p->rope.freqs != nullptr;
        interleaved = p->rope.interleaved != 0;
        pairs = rope ? p->rope.pairs : 0;
        const int row_last = row0 + R < p->rows ? row0 + R - 1 : p->rows - 1;
        first_token = paged_div(row0 < p->rows ? row0 : p->rows - 1, p->d_group);
        tokens = paged_div(row_last, p->d_group) - first_token + 1;
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
    // The angles of the tile's tokens, each once: angles[token * pairs + pair] = (cos, sin).  freqs: a copy in LDS (from memory each further token's
    // frequency was a trip of its own: 3 us a pass of 64 rows).
    __device__ __forceinline__ void turn_angles(PagedArgs p, const PagedItem& t, const double* freqs, v2f* angles) const {
        const float magnitude = p->rope.magnitude;
        const int position = t.n - t.m + first_token;
        for (int i = threadIdx.x; i < tokens * pairs; i += THREADS) {
            const int token = paged_div(i, p->d_pairs), pair = i - token * pairs;
            float c, s;
            rope_angle(freqs[pair], position + token, magnitude, c, s);
            angles[i] = (v2f){c, s};
        }
    }
    // To LDS as fp16 with a power of two of the row's own taken out (`factor` gets it back, with the softmax's scale in base 2): the row's largest element
    // is brought to 2^8, so that neither the range of bf16 nor a rotation leaves fp16's at the upper end.  Elements from 2^-22 of the largest one on are held
    // exactly, smaller ones in steps of 2^-32 of it (a row of less than 2^-100 is brought to less than 2^8: its scores are nothing, whatever the scale of its keys).
    // Rotated queries are not 16-bit numbers, and what their rounding leaves goes to q_rest for a second product
    // (22 bits; one alone would put 2^-12 of each |q k| into the scores, more than P's rounding does to the result).  Without REST they stay rounded to 11 bits.
    template <bool REST> __device__ __forceinline__ void stage(PagedArgs p, int row0, const v2f* angles, char* q_lds, char* q_rest, float* factor) const {
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
            e = e < -100 ? -100 : e;                       // (the factor below stays a normal number; 128, of a row that is none, leaves one too)
            const float down = copysignf(__builtin_bit_cast(float, (uint32_t)(127 + 8 - e) << 23), p->qk_scale_log2);
            uint32_t h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                h[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){y[2 * j] * down, y[2 * j + 1] * down}, v2h));
            *(v4i*)(q_lds + r * ROW + 2 * first) = (v4i){(int)h[0], (int)h[1], (int)h[2], (int)h[3]};
            *(v4i*)(q_lds + r * ROW + 2 * second) = (v4i){(int)h[4], (int)h[5], (int)h[6], (int)h[7]};
            if (REST && rope) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const v2f near = __builtin_convertvector(__builtin_bit_cast(v2h, h[j]), v2f);
                    h[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){y[2 * j] * down - near[0], y[2 * j + 1] * down - near[1]}, v2h));
                }
                *(v4i*)(q_rest + r * ROW + 2 * first) = (v4i){(int)h[0], (int)h[1], (int)h[2], (int)h[3]};
                *(v4i*)(q_rest + r * ROW + 2 * second) = (v4i){(int)h[4], (int)h[5], (int)h[6], (int)h[7]};
            }
            if (u == 0) factor[r] = __builtin_bit_cast(float, (uint32_t)(127 + e - 8) << 23) * fabsf(p->qk_scale_log2);
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
    return p->ticket + (int64_t)((t.z * p->tiles + t.tile) * p->heads_kv + t.hk) * kTicketStride;
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

}  // namespace intfa
