// The pages of a cache: copies, and the bookkeeping of who holds which.  See include/intfa.h.
//
// Counts, table and lengths stay on the device.  What has an order (free pages are dealt by their index, sequences served by theirs) is done by one workgroup, which
// walks the counts 16384 at a time; it leaves the pages to copy as a list, and a second launch copies them with the whole card.  Bound by latency: the walk
// takes about 2 us per 16384 counts.  The copies move 16 bytes a lane, four at a time.
// Measured: a reservation for 256 sequences 10 us, a fork of 224 of 95 columns 7, frees 3, the books of a compaction of 12000 pages 8, copies of 4000 pages of 37 KB 52 us (5.8 TB/s).
#include "intfa_paged_host.h"

using namespace intfa;

namespace {

constexpr int kPoolsEach = 96;                 // pools of a launch (the argument block holds them)
// Bytes of a page that a workgroup copies at a time: at most so many, a page's chunks alike (4000 pages of 36864 + 512 bytes: 67 us with chunks of 16384 and what is left, 62 with
// equal ones, 57 without the hint that passes the caches).  A pool's small page goes with the chunk ahead of it, up to four in a row (57 -> 52 us, 5.8 TB/s; a workgroup of its own for 512
// bytes costs what one for 12288 does, and 48 of them in one workgroup would be 48 trips).
constexpr int kChunk = 16384, kSmall = 1024, kFollowing = 4;
constexpr int kWalk = 1024;                    // threads that keep the books
constexpr int kLeastBlocks = 4 * kComputeUnits;

struct PoolArgs {
    char* data[kPoolsEach];
    int64_t stride[kPoolsEach], bytes[kPoolsEach];
    int32_t first[kPoolsEach + 1];             // chunk at which each pool begins within a page (one that follows another's last chunk: where that ends)
    int32_t width[kPoolsEach];                 // bytes of a lane's access
    int32_t chunk[kPoolsEach];                 // bytes of a chunk
    int32_t pools, num_pages;
    FastDiv d_chunks;
};
struct MoveArgs {
    const int32_t* src; const int32_t* dst;
    const int32_t* count;                      // on the device, or nullptr: n of them
    int32_t n;
    // compaction: the table's entries follow
    int32_t* table; const int32_t* new_index; int64_t bt_sb;
    int32_t batch, table_width;
};

template <typename W> __device__ __forceinline__ void copy_chunk(const char* src, char* dst, int64_t bytes) {
    constexpr int B = sizeof(W), MANY = 4;
    const int n = (int)(bytes / B);
    for (int i0 = threadIdx.x; i0 < n; i0 += 256 * MANY) {
        W w[MANY];
#pragma unroll
        for (int k = 0; k < MANY; ++k)
            if (i0 + 256 * k < n) w[k] = ((const W*)src)[i0 + 256 * k];
#pragma unroll
        for (int k = 0; k < MANY; ++k)
            if (i0 + 256 * k < n) ((W*)dst)[i0 + 256 * k] = w[k];
    }
}

__global__ void __launch_bounds__(256) pages_move_kernel(const PoolArgs a, const MoveArgs m) {
    const int count = m.count != nullptr ? *m.count : m.n, chunks = a.first[a.pools];
    const int64_t work = (int64_t)count * chunks;
    for (int64_t i = blockIdx.x; i < work; i += gridDim.x) {
        const int pair = work < 1ll << 31 ? fast_div((int)i, a.d_chunks) : (int)(i / chunks), chunk = (int)(i - (int64_t)pair * chunks);
        const int src = m.src[pair], dst = m.dst[pair];
        if ((unsigned)src >= (unsigned)a.num_pages || (unsigned)dst >= (unsigned)a.num_pages || src == dst) continue;
        int p = 0;
        while (chunk >= a.first[p + 1]) ++p;
        int64_t at = (int64_t)(chunk - a.first[p]) * a.chunk[p];
        do {
            const int64_t left = a.bytes[p] - at, bytes = left < a.chunk[p] ? left : a.chunk[p];
            const char* const from = a.data[p] + src * a.stride[p] + at;
            char* const to = a.data[p] + dst * a.stride[p] + at;
            if (a.width[p] == 16) copy_chunk<v4i>(from, to, bytes);
            else if (a.width[p] == 4) copy_chunk<int32_t>(from, to, bytes);
            else copy_chunk<int8_t>(from, to, bytes);
            at = 0;
            ++p;
        } while (p < a.pools && chunk + 1 == a.first[p] && a.first[p] == a.first[p + 1]);      // (small pools behind this chunk)
    }
    if (m.table == nullptr) return;
    const int64_t entries = (int64_t)m.batch * m.table_width;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
        const int64_t z = i / m.table_width;
        int32_t* const at = m.table + z * m.bt_sb + (i - z * m.table_width);
        const int id = *at;
        if ((unsigned)id < (unsigned)a.num_pages) *at = m.new_index[id];
    }
}

// ---- books
// Exclusive sum over the workgroup in thread order, and its total.
__device__ __forceinline__ int scan_all(int mine, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    __syncthreads();                           // (the words of the scan before have been read)
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWalk / 64; ++w) {
        const int v = lds[w];
        before += w < wave ? v : 0;
        total += v;
    }
    return before + upto - mine;
}
// The counts that a thread has of a stretch of the pool (behind the last page: 0 or 1 as `pad` says)
constexpr int kEach = 16, kStretch = kEach * kWalk;
typedef int32_t Four __attribute__((ext_vector_type(4), aligned(4)));
struct Counts { int32_t r[kEach]; };
__device__ __forceinline__ Counts load_counts(const int32_t* refs, int at, int pages, int pad) {
    Counts c;
    if (at + kEach <= pages) {
#pragma unroll
        for (int k = 0; k < kEach / 4; ++k) {
            const Four f = *(const Four*)(refs + at + 4 * k);
#pragma unroll
            for (int i = 0; i < 4; ++i) c.r[4 * k + i] = f[i];
        }
    } else {
#pragma unroll
        for (int k = 0; k < kEach; ++k) c.r[k] = at + k < pages ? refs[at + k] : pad;
    }
    return c;
}

// Which of them are in use, a bit each: what is done page by page is done for the bits that are set (with a test of every page, a compaction's walk was 660 vector instructions a wave
// of the one compute unit that has it, 9.2 us for 12000 pages)
__device__ __forceinline__ uint32_t used_bits(const Counts& c) {
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) bits |= c.r[k] > 0 ? 1u << k : 0u;
    return bits;
}

struct CompactArgs { int32_t* refs; int32_t* new_index; int32_t* src; int32_t* dst; int32_t* count; int32_t num_pages; };

__global__ void __launch_bounds__(kWalk) pages_compact_kernel(const CompactArgs a) {
    __shared__ int lds[kWalk / 64];
    const int pages = a.num_pages;
    int mine, used;
    const Counts first = load_counts(a.refs, kEach * (int)threadIdx.x, pages, 0);      // (what is in use of them is kept for the walk: most pools are no longer)
    const uint32_t first_bits = used_bits(first);
    mine = __popc(first_bits);
    for (int at0 = kStretch; at0 < pages; at0 += kStretch) mine += __popc(used_bits(load_counts(a.refs, at0 + kEach * (int)threadIdx.x, pages, 0)));
    scan_all(mine, lds, used);
    // the used pages from place `used` onward, and the free places before it: as many of both
    int from = 0, to = 0;
    for (int at0 = 0; at0 < pages; at0 += kStretch) {
        const int at = at0 + kEach * (int)threadIdx.x;
        const uint32_t bits = at0 == 0 ? first_bits : used_bits(load_counts(a.refs, at, pages, 0));
        const int split = used - at;           // pages of the thread before place `used`
        const uint32_t before_bits = split <= 0 ? 0u : split >= kEach ? (1u << kEach) - 1 : (1u << split) - 1;
        uint32_t moves = bits & ~before_bits, places = ~bits & before_bits;      // (used is at most the pages' number: none behind the last one is a place)
        // (at most 16384 of either: both in one word)
        int both;
        const int before = scan_all(__popc(moves) | __popc(places) << 16, lds, both);
        int f = from + (before & 0xffff), t = to + (before >> 16);
        for (; moves != 0; moves &= moves - 1) a.src[f++] = at + __builtin_ctz(moves);
        for (; places != 0; places &= places - 1) a.dst[t++] = at + __builtin_ctz(places);
        // (those that move get theirs below)
        if (at + kEach <= pages) {
#pragma unroll
            for (int k = 0; k < kEach; k += 4) {
                Four index;
#pragma unroll
                for (int i = 0; i < 4; ++i) index[i] = bits >> (k + i) & 1 ? at + k + i : -1;
                *(Four*)(a.new_index + at + k) = index;
            }
        } else {
            for (int k = 0; k < kEach && at + k < pages; ++k) a.new_index[at + k] = bits >> k & 1 ? at + k : -1;
        }
        from += both & 0xffff;
        to += both >> 16;
    }
    __threadfence_block();
    __syncthreads();
    // (no page is both: several at a time, each of whose reads would otherwise wait for the stores of the one before)
    constexpr int MANY = 4;
    for (int i0 = threadIdx.x; i0 < from; i0 += MANY * kWalk) {
        int s[MANY], d[MANY], count[MANY];
#pragma unroll
        for (int k = 0; k < MANY; ++k) {
            const int i = i0 + k * kWalk < from ? i0 + k * kWalk : i0;
            s[k] = a.src[i];
            d[k] = a.dst[i];
        }
#pragma unroll
        for (int k = 0; k < MANY; ++k) count[k] = a.refs[s[k]];
#pragma unroll
        for (int k = 0; k < MANY; ++k) {
            if (i0 + k * kWalk >= from) break;
            a.new_index[s[k]] = d[k];
            a.refs[d[k]] = count[k];
            a.refs[s[k]] = 0;
        }
    }
    if (threadIdx.x == 0) *a.count = from;
}

struct TableArgs {
    int32_t* refs; int32_t* table; int64_t bt_sb; int32_t* lens;
    int32_t num_pages, page_log2, table_width, batch;
};

__global__ void __launch_bounds__(256) pages_free_kernel(const TableArgs a, const int32_t* sequences, const int32_t* keep) {
    const int z = sequences[blockIdx.y];
    if ((unsigned)z >= (unsigned)a.batch) return;
    int kept = keep != nullptr ? keep[blockIdx.y] : 0;
    const int held = a.lens[z];                // (it may be shortened by another pair of the same sequence: that one takes what is more then)
    kept = kept < held ? kept : held;
    kept = kept < 0 ? 0 : kept;
    const int column = (int)blockIdx.x * 256 + (int)threadIdx.x;
    if (column == 0) atomicMin(a.lens + z, kept);
    // (an entry is taken by one thread, however often the sequence is listed)
    if (column < a.table_width && (int64_t)column << a.page_log2 >= kept) {
        const int id = atomicExch(a.table + z * a.bt_sb + column, -1);
        if ((unsigned)id < (unsigned)a.num_pages) atomicSub(a.refs + id, 1);
    }
}

// A workgroup takes some columns of all pairs: it reads the parents' entries to LDS before it writes the children's.  Of equal children the last pair counts: each child's last pair
// stands in a table of `slots` places (a power of two, 3 / 2 of the pairs or more), found by the child's number.  (Looked for by each entry among the pairs behind its own, 224 pairs of
// 95 columns took 47 us.)
__global__ void __launch_bounds__(256) pages_fork_kernel(const TableArgs a, const int32_t* parents, const int32_t* children, int n, int columns, int slots) {
    extern __shared__ int32_t fork_lds[];
    int32_t* const child = fork_lds;           // [n]: -1: left out
    int32_t* const entry = child + n;          // [n][columns]; the last workgroup's: the lengths
    int32_t* const parent = entry + n * columns;      // [n], and then
    int32_t* const last = parent;              // [slots]: a child's last pair, or -1
    const int column0 = (int)blockIdx.x * columns;
    const bool lengths = blockIdx.x == gridDim.x - 1;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int c = children[i], p = parents[i];
        const bool ok = (unsigned)c < (unsigned)a.batch && (unsigned)p < (unsigned)a.batch;
        child[i] = ok ? c : -1;
        parent[i] = ok ? p : 0;
    }
    __syncthreads();
    const int wide = lengths ? 1 : columns;
    for (int i = threadIdx.x; i < n * wide; i += 256) {
        const int k = i / wide, column = column0 + i - k * wide;
        entry[i] = lengths ? a.lens[parent[k]] : column < a.table_width ? a.table[parent[k] * a.bt_sb + column] : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < slots; i += 256) last[i] = -1;
    __syncthreads();
    // (linear probing: ends, since there are more places than children)
    auto place = [&](int c) __attribute__((always_inline)) { return (int)((uint32_t)c * 2654435769u >> 16) & (slots - 1); };
    for (int i = threadIdx.x; i < n; i += 256) {
        const int c = child[i];
        if (c < 0) continue;
        int at = place(c);
        while (true) {
            const int was = atomicCAS(last + at, -1, i);
            if (was == -1) break;
            if (child[was] == c) {             // (a place stays its child's)
                atomicMax(last + at, i);
                break;
            }
            at = (at + 1) & (slots - 1);
        }
    }
    __syncthreads();
    uint32_t out = 0;                          // (of up to 4096 pairs a thread has sixteen)
    for (int i = threadIdx.x; i < n; i += 256) {
        const int c = child[i];
        if (c < 0) continue;
        int at = place(c);
        while (child[last[at]] != c) at = (at + 1) & (slots - 1);
        if (last[at] != i) out |= 1u << (i >> 8);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256)
        if (out >> (i >> 8) & 1) child[i] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < n * wide; i += 256) {
        const int k = i / wide, column = column0 + i - k * wide, c = child[k];
        if (c < 0) continue;
        if (lengths) {
            a.lens[c] = entry[i];
        } else if (column < a.table_width) {
            int32_t* const at = a.table + c * a.bt_sb + column;
            const int was = *at, now = entry[i];
            if (was == now) continue;
            if ((unsigned)now < (unsigned)a.num_pages) atomicAdd(a.refs + now, 1);
            if ((unsigned)was < (unsigned)a.num_pages) atomicSub(a.refs + was, 1);
            *at = now;
        }
    }
}

struct ReserveArgs {
    TableArgs t;
    const int32_t* fresh; int32_t fresh_all;
    int32_t* granted;
    int32_t* free_list; int32_t* src; int32_t* dst; int32_t* count;      // src, dst: as long as the free list
    int32_t* reached; int32_t* last;           // [pages]: of a page that is held more than once, the entries that a call reaches, and the last of them
};

// The columns that a sequence's fresh tokens reach: [first, end), end at most the table's width.
struct Span { int held, fresh, first, end; };
__device__ __forceinline__ Span reserve_span(const ReserveArgs& a, int z) {
    Span s;
    s.held = a.t.lens[z];
    s.held = s.held < 0 ? 0 : s.held;
    s.fresh = a.fresh != nullptr ? a.fresh[z] : a.fresh_all;
    s.fresh = s.fresh < 0 ? 0 : s.fresh;
    const int64_t last = ((int64_t)s.held + s.fresh + (1ll << a.t.page_log2) - 1) >> a.t.page_log2;
    s.first = s.held >> a.t.page_log2;
    s.first = s.first < a.t.table_width ? s.first : a.t.table_width;
    s.end = s.fresh == 0 ? s.first : last < a.t.table_width ? (int)last : a.t.table_width;
    return s;
}

// Every sequence needs so many pages: those that it lacks, and copies of those that others hold; of all that want a copy of a page in this call, the last takes none if nobody else is
// left.  The page that forked sequences share is that of their first column, which holds their last tokens: who is the last there is found among the first columns, in LDS.  Where
// a later column is shared too (sequences forked after a reservation ahead), the entries that the call reaches are counted page by page in memory, and what the sequences need is
// counted again (256 sequences in groups of four, three columns ahead: 31 us).  (A thread keeps what it knows of its first sequence; of batches over 1024 it reads the others' again.
// Columns behind the first are its own work too while they are few, and a wave's where they are kLong or more: a trip to memory each, one after the other, a prompt of 16384 tokens
// on pages of 16 took 400 us, and 17 so.)
constexpr int kLong = 6;
__global__ void __launch_bounds__(kWalk) pages_reserve_kernel(const ReserveArgs a) {
    extern __shared__ __align__(16) int32_t head_lds[];      // [batch]: the shared page of a sequence's first column, or -1
    int32_t* const plan_lds = head_lds + a.t.batch;      // [batch]: what becomes of its first column
    enum { kLacks, kKeep, kCopy, kLeft, kNone };      // (left: kept if all that share it and come earlier get their copies, else kNone)
    __shared__ int lds[kWalk / 64];
    __shared__ int long_z[kWalk], long_count[kWalk], longs;      // sequences of many columns, and what is counted of them
    __shared__ int moves_lds, deep_lds;
    const int pages = a.t.num_pages, Z = a.t.batch, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) moves_lds = longs = deep_lds = 0;
    const Counts stretch = load_counts(a.t.refs, kEach * (int)threadIdx.x, pages, 1);      // (asked for ahead of their use)
    Span own = {0, 0, 0, 0};
    int own_head = -1, own_holders = 0;
    for (int z = threadIdx.x; z < Z; z += kWalk) {
        const Span s = reserve_span(a, z);
        int head = -1, holders = 0, plan = kLacks;
        if (s.first < s.end) {
            const int id = a.t.table[z * a.t.bt_sb + s.first];
            if ((unsigned)id < (unsigned)pages) {
                holders = a.t.refs[id];
                plan = kKeep;
                if (holders > 1) head = id;
            }
        }
        head_lds[z] = head;
        plan_lds[z] = plan;
        if (z < kWalk) {
            own = s;
            own_head = head;
            own_holders = holders;
        }
    }
    __syncthreads();
    auto cell = [&](int z, int c) __attribute__((always_inline)) { return z * a.t.table_width + c; };      // (below 2^31)
    // f(z, c, id) for the entries that are reached and name pages which others hold too
    auto each_shared = [&](auto f) __attribute__((always_inline)) {
        for (int z0 = 0; z0 < Z; z0 += kWalk) {
            const int z = z0 + (int)threadIdx.x;
            if (z < Z) {
                const Span s = z < kWalk ? own : reserve_span(a, z);
                if (s.end - s.first >= kLong) long_z[atomicAdd(&longs, 1)] = z;
                else
                    for (int c = s.first; c < s.end; ++c) {
                        const int id = a.t.table[z * a.t.bt_sb + c];
                        if ((unsigned)id < (unsigned)pages && a.t.refs[id] > 1) f(z, c, id);
                    }
            }
            __syncthreads();
            for (int i = wave; i < longs; i += kWalk / 64) {
                const int zl = long_z[i];
                const Span s = reserve_span(a, zl);
                for (int c = s.first + lane; c < s.end; c += 64) {
                    const int id = a.t.table[zl * a.t.bt_sb + c];
                    if ((unsigned)id < (unsigned)pages && a.t.refs[id] > 1) f(zl, c, id);
                }
            }
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) longs = 0;
            __syncthreads();
        }
    };
    // An entry that names a page which others hold too: by it alone in the end?  (Known where the entries have been counted; both ways of the code below are of their own, for
    // the sake of the usual one, which has no such entries behind the first columns: 2048 sequences 55 us, and 60 with the question in it.)
    auto kept = [&](auto counted, int z, int c, int id) __attribute__((always_inline)) {
        return decltype(counted)::value && __hip_atomic_load(a.last + id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == cell(z, c) &&
               __hip_atomic_load(a.reached + id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.t.refs[id];
    };
    // needs, in the order of the sequences: granted[z] holds the pages that were dealt before it until its own are
    int dealt = 0;
    auto count_needs = [&](auto counted) __attribute__((always_inline)) {
        for (int z0 = 0; z0 < Z; z0 += kWalk) {
            const int z = z0 + (int)threadIdx.x;
            int needs = 0;
            if (z < Z) {
                const Span s = z < kWalk ? own : reserve_span(a, z);
                const int head = z < kWalk ? own_head : head_lds[z];
                if (decltype(counted)::value && head >= 0) plan_lds[z] = kept(counted, z, s.first, head) ? kLeft : kCopy;
                else if (head >= 0) {
                    const int holders = z < kWalk ? own_holders : a.t.refs[head];
                    int before = 0, o = 0;
#pragma unroll 8
                    for (; o + 4 <= z; o += 4) {
                        const v4i h = *(const v4i*)(head_lds + o);
                        before += (h[0] == head) + (h[1] == head) + (h[2] == head) + (h[3] == head);
                    }
                    for (; o < z; ++o) before += head_lds[o] == head;
                    plan_lds[z] = holders - before > 1 ? kCopy : before > 0 ? kLeft : kKeep;
                }
                needs = s.first < s.end && (plan_lds[z] == kLacks || plan_lds[z] == kCopy);
                if (s.end - s.first >= kLong) long_z[atomicAdd(&longs, 1)] = z;
                else
                    for (int c = s.first + 1; c < s.end; ++c) {
                        const int id = a.t.table[z * a.t.bt_sb + c];
                        const bool named = (unsigned)id < (unsigned)pages, shared = named && a.t.refs[id] > 1;
                        if (shared) deep_lds = 1;
                        needs += !named || (shared && !kept(counted, z, c, id));
                    }
            }
            __syncthreads();
            if (longs > 0) {
                for (int i = wave; i < longs; i += kWalk / 64) {
                    const int zl = long_z[i];
                    const Span s = reserve_span(a, zl);
                    int count = 0;
                    for (int c0 = s.first + 1; c0 < s.end; c0 += 64) {
                        bool takes = false;
                        if (c0 + lane < s.end) {
                            const int id = a.t.table[zl * a.t.bt_sb + c0 + lane];
                            const bool named = (unsigned)id < (unsigned)pages, shared = named && a.t.refs[id] > 1;
                            if (shared) deep_lds = 1;
                            takes = !named || (shared && !kept(counted, zl, c0 + lane, id));
                        }
                        count += __popcll(__ballot(takes));
                    }
                    if (lane == 0) long_count[zl - z0] = count;
                }
                __syncthreads();
                const Span s = z >= Z ? Span{0, 0, 0, 0} : z < kWalk ? own : reserve_span(a, z);
                if (s.end - s.first >= kLong) needs += long_count[threadIdx.x];
                __syncthreads();
                if (threadIdx.x == 0) longs = 0;
            }
            int total;
            const int ahead = scan_all(needs, lds, total);
            if (z < Z) a.granted[z] = dealt + ahead;
            dealt += total;
        }
    };
    count_needs(std::false_type());
    __syncthreads();
    const bool deep = deep_lds != 0;
    if (__builtin_expect(deep, 0)) {
        each_shared([&](int, int, int id) __attribute__((always_inline)) {
            __hip_atomic_store(a.reached + id, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(a.last + id, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        });
        each_shared([&](int z, int c, int id) __attribute__((always_inline)) {
            atomicAdd(a.reached + id, 1);
            atomicMax(a.last + id, cell(z, c));
        });
        dealt = 0;
        count_needs(std::true_type());
    }
    // as many free pages, in their order
    int found = 0;
    for (int at0 = 0; at0 < pages && found < dealt; at0 += kStretch) {
        const int at = at0 + kEach * (int)threadIdx.x;
        uint32_t free = (1u << kEach) - 1 & ~used_bits(at0 == 0 ? stretch : load_counts(a.t.refs, at, pages, 1));
        int total, f = found + scan_all(__popc(free), lds, total);
        for (; free != 0 && f < dealt; free &= free - 1) a.free_list[f++] = at + __builtin_ctz(free);
        found += total;
    }
    found = found < dealt ? found : dealt;
    __threadfence_block();
    __syncthreads();
    // (the table's entry at `column`, which names `id`, becomes `page`)
    auto give = [&](int z, int column, int id, bool copy, int page) __attribute__((always_inline)) {
        a.t.refs[page] = 1;
        if (copy) {
            const int m = atomicAdd(&moves_lds, 1);
            a.src[m] = id;
            a.dst[m] = page;
        }
        a.t.table[z * a.t.bt_sb + column] = page;
    };
    auto grant = [&](int z, const Span& s, int room) __attribute__((always_inline)) {      // columns before `room` can be written
        const int64_t places = ((int64_t)room << a.t.page_log2) - s.held;
        a.granted[z] = places <= 0 ? 0 : places < s.fresh ? (int)places : s.fresh;
    };
    auto deal = [&](auto counted) __attribute__((always_inline)) {
        for (int z0 = 0; z0 < Z; z0 += kWalk) {
            const int z = z0 + (int)threadIdx.x;
            if (z < Z) {
                const Span s = z < kWalk ? own : reserve_span(a, z);
                int rank = a.granted[z], plan = plan_lds[z];
                if (plan == kLeft && rank > found) plan = kNone;
                const bool many = s.end - s.first >= kLong;
                int room = plan == kNone ? s.first : many ? s.first + 1 : s.end;
                for (int c = s.first; c < room; ++c) {
                    const int id = a.t.table[z * a.t.bt_sb + c];
                    const bool named = (unsigned)id < (unsigned)pages;
                    bool copy = named && (c == s.first ? plan == kCopy : a.t.refs[id] > 1);      // (counts that are over 0 change behind the barrier below)
                    if (copy && c != s.first && kept(counted, z, c, id)) {
                        copy = false;
                        if (rank > found) {        // (another could not leave)
                            room = c;
                            break;
                        }
                    }
                    if (named && !copy) continue;
                    if (rank >= found) {
                        room = c;
                        break;
                    }
                    give(z, c, id, copy, a.free_list[rank++]);
                }
                if (many && room > s.first) {
                    long_z[atomicAdd(&longs, 1)] = z;
                    long_count[threadIdx.x] = rank;
                } else grant(z, s, room);
            }
            __syncthreads();
            for (int i = wave; i < longs; i += kWalk / 64) {
                const int zl = long_z[i];
                const Span s = reserve_span(a, zl);
                int rank = long_count[zl - z0], room = s.end;
                for (int c0 = s.first + 1; c0 < s.end && room == s.end; c0 += 64) {
                    const int c = c0 + lane, id = c < s.end ? a.t.table[zl * a.t.bt_sb + c] : -1;
                    const bool named = (unsigned)id < (unsigned)pages, shared = named && a.t.refs[id] > 1, left = shared && kept(counted, zl, c, id), copy = shared && !left;
                    const bool takes = c < s.end && (!named || copy);
                    const uint64_t all = __ballot(takes);
                    const int mine = rank + __popcll(all & ((1ull << lane) - 1));
                    if (takes && mine < found) give(zl, c, id, copy, a.free_list[mine]);
                    const uint64_t out = __ballot((takes && mine >= found) || (left && mine > found));
                    if (out != 0) room = c0 + __builtin_ctzll(out);
                    rank += __popcll(all);
                }
                if (lane == 0) grant(zl, s, room);
            }
            __syncthreads();
            if (threadIdx.x == 0) longs = 0;
            __syncthreads();
        }
    };
    if (__builtin_expect(deep, 0)) deal(std::true_type());
    else deal(std::false_type());
    __threadfence_block();
    __syncthreads();
    for (int m = threadIdx.x; m < moves_lds; m += kWalk) atomicSub(a.t.refs + a.src[m], 1);
    if (threadIdx.x == 0) *a.count = moves_lds;
}

// ---- host
int check_pools(const intfa_page_pool* pools, int32_t n, int32_t num_pages) {
    if (n < 0 || n > INTFA_MAX_POOLS || (n > 0 && pools == nullptr)) return INTFA_ERR_POOL;
    for (int i = 0; i < n; ++i) {
        if (pools[i].data == nullptr) return INTFA_ERR_NULL;
        if (pools[i].page_bytes <= 0 || pools[i].page_bytes > 1ll << 40) return INTFA_ERR_POOL;
        if (num_pages > 1 && pools[i].page_stride < pools[i].page_bytes && -pools[i].page_stride < pools[i].page_bytes) return INTFA_ERR_POOL;      // (pages that overlap)
    }
    return INTFA_OK;
}
int check_table(const intfa_page_table* t, bool lens, bool page) {
    if (t == nullptr || t->refs == nullptr || t->block_table == nullptr || (lens && t->seqlens_k == nullptr)) return INTFA_ERR_NULL;
    if (t->num_pages <= 0 || t->num_pages >= 1 << 30 || t->table_width <= 0 || t->table_width >= 1 << 30) return INTFA_ERR_PAGE;
    if (t->batch <= 0 || (t->batch > 1 && t->bt_stride_b < t->table_width && -t->bt_stride_b < t->table_width)) return INTFA_ERR_SHAPE;      // (rows that overlap)
    if (page && (t->page_size < 16 || t->page_size > 256 || (t->page_size & (t->page_size - 1)))) return INTFA_ERR_PAGE;
    if ((reinterpret_cast<uintptr_t>(t->refs) | reinterpret_cast<uintptr_t>(t->block_table) | reinterpret_cast<uintptr_t>(t->seqlens_k)) & 3u) return INTFA_ERR_ALIGN;
    return INTFA_OK;
}
TableArgs table_args(const intfa_page_table* t) {
    return {t->refs, t->block_table, t->bt_stride_b, t->seqlens_k, t->num_pages, t->page_size > 0 ? __builtin_ctz((unsigned)t->page_size) : 0, t->table_width, t->batch};
}
// The copies of the list in all pools, kPoolsEach of them a launch; the table follows in the last one.  most: of the list.
int launch_moves(const intfa_page_pool* pools, int num_pools, int num_pages, MoveArgs m, int most, hipStream_t stream) {
    int32_t* const table = m.table;
    for (int at = 0; at < num_pools || (at == 0 && table != nullptr); at += kPoolsEach) {
        PoolArgs a{};
        a.pools = num_pools - at < kPoolsEach ? num_pools - at : kPoolsEach;
        a.num_pages = num_pages;
        int64_t chunks = 0;
        int following = 0;
        for (int i = 0; i < a.pools; ++i) {
            const intfa_page_pool& p = pools[at + i];
            a.data[i] = (char*)p.data; a.stride[i] = p.page_stride; a.bytes[i] = p.page_bytes;
            const uint64_t all = (uint64_t)reinterpret_cast<uintptr_t>(p.data) | (uint64_t)p.page_stride | (uint64_t)p.page_bytes;
            a.width[i] = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
            a.first[i] = (int32_t)chunks;
            const int64_t parts = (p.page_bytes + kChunk - 1) / kChunk;
            a.chunk[i] = (int32_t)(((p.page_bytes + parts - 1) / parts + 15) / 16 * 16);
            const bool follows = p.page_bytes <= kSmall && i > 0 && following < kFollowing;
            following = follows ? following + 1 : 0;
            chunks += follows ? 0 : parts;
            if (chunks >= 1ll << 31) return INTFA_ERR_POOL;
        }
        a.first[a.pools] = (int32_t)chunks;
        a.d_chunks = make_fast_div(chunks > 0 ? (int)chunks : 1);
        m.table = at + kPoolsEach >= num_pools ? table : nullptr;
        const int64_t work = size_product(most, chunks), entries = m.table != nullptr ? ((int64_t)m.batch * m.table_width + 255) / 256 : 0;
        // Workgroups: one a chunk while that is few, and not so many that those which find the list short cost more than the list
        int64_t grid = work > entries ? work : entries;
        grid = grid < 1 ? 1 : grid < 8 * kLeastBlocks ? grid : 8 * kLeastBlocks;
        hipLaunchKernelGGL(pages_move_kernel, dim3((unsigned)grid), dim3(256), 0, stream, a, m);
        const int rc = (int)hipGetLastError();
        if (rc != 0) return rc;
    }
    return INTFA_OK;
}
int64_t reserve_most(const intfa_page_table* t) {       // pages that a call can deal at most
    const int64_t entries = size_product(t->batch, t->table_width);
    return entries < t->num_pages ? entries : t->num_pages;
}
size_t reserve_bytes(const intfa_page_table* t) { return 16 + 12 * (size_t)reserve_most(t) + 8 * (size_t)t->num_pages; }

}  // namespace

extern "C" {

int intfa_pages_copy(const intfa_page_pool* pools, int32_t num_pools, int32_t num_pages, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
    if (num_pools <= 0) return INTFA_ERR_POOL;
    const int rc = check_pools(pools, num_pools, num_pages);
    if (rc != INTFA_OK) return rc;
    if (src == nullptr || dst == nullptr) return INTFA_ERR_NULL;
    if (num_pages <= 0) return INTFA_ERR_PAGE;
    if (n <= 0) return INTFA_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 3u) return INTFA_ERR_ALIGN;
    MoveArgs m{};
    m.src = src; m.dst = dst; m.n = n;
    return launch_moves(pools, num_pools, num_pages, m, n, (hipStream_t)stream);
}

int intfa_pages_fork(const intfa_page_table* t, const int32_t* parents, const int32_t* children, int32_t n, void* stream) {
    const int rc = check_table(t, true, false);
    if (rc != INTFA_OK) return rc;
    if (parents == nullptr || children == nullptr) return INTFA_ERR_NULL;
    if (n <= 0 || n > 4096) return INTFA_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(children)) & 3u) return INTFA_ERR_ALIGN;
    // Columns of a workgroup: 1024 entries in four rounds, or one column
    const int columns = n >= 1024 ? 1 : 1024 / n < 64 ? 1024 / n : 64;
    const unsigned groups = (unsigned)((t->table_width + columns - 1) / columns);
    if ((groups + 1ll) * 256 >= 1ll << 32) return INTFA_ERR_SHAPE;
    int slots = 64;
    while (2 * slots < 3 * n) slots *= 2;
    const size_t words = (size_t)(1 + columns) * n + slots;      // (slots: n or more; 64 KB at the most)
    hipLaunchKernelGGL(pages_fork_kernel, dim3(groups + 1), dim3(256), words * 4, (hipStream_t)stream, table_args(t), parents, children, n, columns, slots);
    return (int)hipGetLastError();
}

int intfa_pages_free(const intfa_page_table* t, const int32_t* sequences, const int32_t* keep, int32_t n, void* stream) {
    const int rc = check_table(t, true, true);
    if (rc != INTFA_OK) return rc;
    if (sequences == nullptr) return INTFA_ERR_NULL;
    if (n <= 0 || n > 65535) return INTFA_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(sequences) | reinterpret_cast<uintptr_t>(keep)) & 3u) return INTFA_ERR_ALIGN;
    const unsigned groups = (unsigned)((t->table_width + 255) / 256);
    if (size_product((int64_t)groups * 256, n) >= 1ll << 32) return INTFA_ERR_SHAPE;
    hipLaunchKernelGGL(pages_free_kernel, dim3(groups, (unsigned)n), dim3(256), 0, (hipStream_t)stream, table_args(t), sequences, keep);
    return (int)hipGetLastError();
}

size_t intfa_pages_reserve_workspace_bytes(const intfa_page_table* t) {
    return check_table(t, true, true) == INTFA_OK ? reserve_bytes(t) : 0;
}

int intfa_pages_reserve(const intfa_page_table* t, const intfa_page_pool* pools, int32_t num_pools, const int32_t* fresh, int32_t fresh_all, int32_t* granted,
                        void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_table(t, true, true);
    if (rc != INTFA_OK) return rc;
    rc = check_pools(pools, num_pools, t->num_pages);
    if (rc != INTFA_OK) return rc;
    if (granted == nullptr) return INTFA_ERR_NULL;
    if (t->batch > 8192 || size_product(t->batch, t->table_width) >= 1ll << 31) return INTFA_ERR_SHAPE;
    if ((reinterpret_cast<uintptr_t>(fresh) | reinterpret_cast<uintptr_t>(granted)) & 3u) return INTFA_ERR_ALIGN;
    const int64_t most = reserve_most(t);
    if (workspace == nullptr || workspace_bytes < reserve_bytes(t) || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return INTFA_ERR_WORKSPACE;
    int32_t* const words = (int32_t*)workspace;
    ReserveArgs a{table_args(t), fresh, fresh_all, granted, words + 4, words + 4 + most, words + 4 + 2 * most, words, words + 4 + 3 * most, words + 4 + 3 * most + t->num_pages};
    hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(kWalk), (size_t)t->batch * 8, (hipStream_t)stream, a);
    rc = (int)hipGetLastError();
    if (rc != 0 || num_pools == 0) return rc;
    MoveArgs m{};
    m.src = a.src; m.dst = a.dst; m.count = a.count;
    return launch_moves(pools, num_pools, t->num_pages, m, (int)most < t->batch ? (int)most : t->batch, (hipStream_t)stream);
}

size_t intfa_pages_compact_workspace_bytes(const intfa_page_table* t) {
    return check_table(t, false, false) == INTFA_OK ? 16 + 8 * (size_t)t->num_pages : 0;
}

int intfa_pages_compact(const intfa_page_table* t, const intfa_page_pool* pools, int32_t num_pools, int32_t* new_index, void* workspace, size_t workspace_bytes,
                        void* stream) {
    int rc = check_table(t, false, false);
    if (rc != INTFA_OK) return rc;
    rc = check_pools(pools, num_pools, t->num_pages);
    if (rc != INTFA_OK) return rc;
    if (new_index == nullptr) return INTFA_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(new_index) & 3u) return INTFA_ERR_ALIGN;
    if (workspace == nullptr || workspace_bytes < 16 + 8 * (size_t)t->num_pages || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return INTFA_ERR_WORKSPACE;
    int32_t* const words = (int32_t*)workspace;
    const CompactArgs a{t->refs, new_index, words + 4, words + 4 + t->num_pages, words, t->num_pages};
    hipLaunchKernelGGL(pages_compact_kernel, dim3(1), dim3(kWalk), 0, (hipStream_t)stream, a);
    rc = (int)hipGetLastError();
    if (rc != 0) return rc;
    MoveArgs m{};
    m.src = a.src; m.dst = a.dst; m.count = a.count;
    m.table = t->block_table; m.new_index = new_index; m.bt_sb = t->bt_stride_b; m.batch = t->batch; m.table_width = t->table_width;
    return launch_moves(pools, num_pools, t->num_pages, m, t->num_pages / 2 + 1, (hipStream_t)stream);
}

}  // extern "C"
