// Sums of looked-up rows of a table, and the table's gradient by sorted places.
//
//   out[r] = scale sum_i table[index[r][i]],   table_grad[v] = scale sum over the places (r, i) of v of grad[r]
//
// The gradient is a sum by entry without atomics: the places are sorted by entry (stable, so that a sum has one
// order), runs of equal entries are added up from the sorted list, and what of a run lies in several chunks of the list
// is joined in the chunks' order.
//
// Rows: 200000 lists of 40 over 1280 entries of 64 f32 57 us; 84 MB cross the memory, but 2.05 GB the LDS that holds the
// table, at 36 TB/s (from the caches 78 us).  The LDS is at work for 40% of that, half of it on bank conflicts, the vector units for
// 48%: neither is full, the rest waits for lists and sums.  32 rows of 256 bf16: a call's 8.5 us.
// Gradient: 262144 places of 50021 entries, 256 columns, bf16 to f32 87 us: sort 32, sums 43 (185 MB at 4.3 TB/s), join and zeros 12.
// 65536 lists of 40 over 1280 entries of 64 f32 110 us: sort 46 (2.6M keys, scattered stores), sums 58 (671 MB of rows at 11.6 TB/s from
// the second-level caches), join and parts 13 (the parts under the profiler, where a kernel takes longer than among others).  Up
// to 512 places one launch, up to 8192 three.
#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

// A vector of a row, from column c on.  kWhole: all rows are whole vectors of columns next to each other.  Else its values are loaded
// one by one where it does not lie whole in its row, without a branch between them (behind the end the last column again): guarded, each
// was waited for.
template <class T, bool kWhole>
__device__ __forceinline__ Pack<T> load_columns(const T* row, int64_t cs, uint32_t c, uint32_t dim) {
    constexpr int V = Pack<T>::V;
    Pack<T> p;
    if (kWhole || (cs == 1 && c + V <= dim)) {
        p.w = ((const Loose<T>*)(row + c))->w;
    } else {
        float x[V];
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = to_f32(row[(int64_t)min(c + v, dim - 1) * cs]);
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = c + v < dim ? x[v] : 0.0f;
        p.set(x);
    }
    return p;
}

// ---- rows -----------------------------------------------------------------------------------
struct Lookup {
    const int32_t* index;   // [rows][list]
    uint64_t rows;
    uint32_t entries, dim, list;
    float scale;
};
// Four indices of a row's list, from i on; `entries` where it ends.
__device__ __forceinline__ void load_indices(const Lookup& L, const int32_t* ix, uint32_t i, uint32_t (&e)[4]) {
    typedef int32_t Quad __attribute__((ext_vector_type(4), aligned(4)));
    if (i + 4 <= L.list) {
        const Quad q = *(const Quad*)(ix + i);
#pragma unroll
        for (int u = 0; u < 4; ++u) e[u] = (uint32_t)q[u];
    } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) e[u] = i + u < L.list ? (uint32_t)ix[i + u] : L.entries;
    }
}
// A group of `lanes` lanes takes a row of the output, a vector a lane, four rows of the table on their way at a time.
template <class T, bool kWhole>
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ table, int64_t rs, int64_t cs, Lookup L,
                                                     T* __restrict__ out, uint32_t lanes) {
    constexpr int V = Pack<T>::V;
    const uint32_t tiles = (L.dim + lanes * V - 1) / (lanes * V), per = 256 / lanes;
    const uint64_t jobs = (L.rows + per - 1) / per * tiles;
    for (uint64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        const uint64_t row = job / tiles * per + threadIdx.x / lanes;
        const uint32_t c = ((uint32_t)(job % tiles) * lanes + threadIdx.x % lanes) * V;
        if (row >= L.rows || c >= L.dim) continue;
        const int32_t* ix = L.index + row * L.list;
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        uint32_t next[4];
        load_indices(L, ix, 0, next);
        for (uint32_t i = 0; i < L.list; i += 4) {
            uint32_t e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) e[u] = next[u];
            if (i + 4 < L.list) load_indices(L, ix, i + 4, next);
            Pack<T> p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                // (without a branch: what is no entry reads the first and drops it)
                p[u] = load_columns<T, kWhole>(table + (int64_t)(e[u] < L.entries ? e[u] : 0) * rs, cs, c, L.dim);
                if (e[u] >= L.entries) p[u].w = Words{};
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] += p[u].get(v);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] *= L.scale;
        store_pack<T, true>(out + row * L.dim, 1, c, L.dim, acc);
    }
}
// Long lists over few entries: a workgroup holds `lanes` vectors of every entry in LDS and takes a part of the rows.
constexpr uint32_t kLdsThreads = 1024, kLdsBytes = 163840;   // (one workgroup a CU)
template <class T>
__global__ __launch_bounds__(kLdsThreads) void lookup_lds_kernel(const T* __restrict__ table, int64_t rs, Lookup L, T* __restrict__ out,
                                                                 uint32_t lanes, uint32_t tiles, uint64_t part) {
    constexpr int V = Pack<T>::V;
    extern __shared__ Words held[];   // [entries + 1][lanes]; the last is 0, for what is no entry
    const uint32_t c0 = blockIdx.x % tiles * lanes * V, lane = threadIdx.x % lanes, c = c0 + lane * V;
    const int shift = 31 - __builtin_clz(lanes);
    if (threadIdx.x < lanes) held[L.entries * lanes + threadIdx.x] = Words{};
    for (uint32_t i = threadIdx.x; i < L.entries * lanes; i += kLdsThreads) {
        const uint32_t at = c0 + i % lanes * V;
        held[i] = at < L.dim ? load_columns<T, false>(table + (int64_t)(i / lanes) * rs, 1, at, L.dim).w : Words{};
    }
    __syncthreads();
    const uint64_t from = blockIdx.x / tiles * part, to = min(L.rows, from + part);
    if (c >= L.dim) return;
    for (uint64_t row = from + threadIdx.x / lanes; row < to; row += kLdsThreads / lanes) {
        const int32_t* ix = L.index + row * L.list;
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        uint32_t next[4];
        load_indices(L, ix, 0, next);
        for (uint32_t i = 0; i < L.list; i += 4) {
            uint32_t e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) e[u] = next[u];
            load_indices(L, ix, i + 4 < L.list ? i + 4 : i, next);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const Pack<T> p{held[(min(e[u], L.entries) << shift) + lane]};
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] += p.get(v);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] *= L.scale;
        store_pack<T, true>(out + row * L.dim, 1, c, L.dim, acc);
    }
}

// ---- sort -----------------------------------------------------------------------------------
// What is summed up comes as (entry, row), sorted by entry and stable by place.  A place without an entry sorts behind all, as
// `entries`.
struct Sort {
    const int32_t* index;
    uint32_t n, entries, list;
    uint32_t blocks, digits;   // of a pass by digits; digits a power of two
    int shift, bits;
    uint32_t segs, seg_blocks; // parts of the places that are sorted by themselves, and a part's blocks
    uint8_t* mark;             // [segs][entries]: cleared here, set where an entry's sum is taken
};
constexpr uint32_t kNoEntry = ~0u;   // (in the sorted list)
__device__ __forceinline__ u64 sorted_key(const Sort& S, uint32_t seg, uint32_t entry, uint32_t place) {
    return (u64)(entry < S.entries ? seg * S.entries + entry : kNoEntry) << 32 | place / S.list;
}
__device__ __forceinline__ uint32_t place_entry(const Sort& S, uint32_t i) { return min((uint32_t)S.index[i], S.entries); }
__device__ __forceinline__ void clear_marks(const Sort& S, uint32_t block, uint32_t blocks) {
    for (uint64_t v = (uint64_t)block * blockDim.x + threadIdx.x; v < (uint64_t)S.segs * S.entries; v += (uint64_t)blocks * blockDim.x) S.mark[v] = 0;
}

// Few places: a workgroup takes 64 of them and counts, over all places, those ahead of each; a wave a sixteenth of them.
constexpr uint32_t kRankMost = 8192, kRankWaves = 16;
template <class O>
__global__ __launch_bounds__(64 * kRankWaves) void rank_kernel(Sort S, u64* __restrict__ out, O* __restrict__ grad, uint64_t cells) {
    __shared__ uint32_t entry[kRankMost];
    __shared__ uint32_t ahead[kRankWaves][64];
    const uint32_t blocks = (S.n + 63) / 64;
    if (blockIdx.x >= blocks) {   // the whole gradient is cleared: few of its entries occur, and are written over
        constexpr uint32_t V = 16 / sizeof(O);
        typedef uint32_t Unaligned __attribute__((ext_vector_type(4), aligned(2)));
        for (uint64_t i = ((uint64_t)(blockIdx.x - blocks) * blockDim.x + threadIdx.x) * V; i < cells; i += (uint64_t)(gridDim.x - blocks) * blockDim.x * V) {
            if (i + V <= cells) __builtin_nontemporal_store(Words{}, (Unaligned*)(grad + i));
            else
                for (uint64_t j = i; j < cells; ++j) grad[j] = from_f32<O>(0.0f);
        }
        return;
    }
    const uint32_t n64 = (S.n + 63) / 64 * 64;   // (sixteenths of whole vectors; what lies behind the places is behind all)
#pragma unroll
    for (uint32_t r = 0; r < kRankMost / 64 / kRankWaves; ++r) {
        const uint32_t i = r * 64 * kRankWaves + threadIdx.x;
        if (i < n64) entry[i] = i < S.n ? place_entry(S, i) : ~0u;
    }
    __syncthreads();
    const uint32_t wave = threadIdx.x / 64, lane = lane_id(), at = blockIdx.x * 64 + lane;
    const uint32_t mine = at < S.n ? entry[at] : ~0u;
    const uint32_t from = wave * (n64 / kRankWaves), to = from + n64 / kRankWaves;
    // places before this workgroup's go ahead of an equal one, those behind it do not
    uint32_t count = 0;
    const uint32_t own0 = min(max(blockIdx.x * 64, from), to), own1 = min(max(min(blockIdx.x * 64 + 64, n64), from), to);
    typedef uint32_t Quad __attribute__((ext_vector_type(4)));
    const Quad* q = (const Quad*)entry;
#pragma unroll 4
    for (uint32_t i = from / 4; i < own0 / 4; ++i) {
        const Quad e = q[i];
        count += (e[0] <= mine) + (e[1] <= mine) + (e[2] <= mine) + (e[3] <= mine);
    }
    for (uint32_t i = own0; i < own1; ++i) count += entry[i] < mine || (entry[i] == mine && i < at);
#pragma unroll 4
    for (uint32_t i = own1 / 4; i < to / 4; ++i) {
        const Quad e = q[i];
        count += (e[0] < mine) + (e[1] < mine) + (e[2] < mine) + (e[3] < mine);
    }
    ahead[wave][lane] = count;
    __syncthreads();
    if (wave == 0 && at < S.n) {
        uint32_t place = 0;
#pragma unroll
        for (uint32_t w = 0; w < kRankWaves; ++w) place += ahead[w][lane];
        out[place] = sorted_key(S, 0, mine, at);
    }
}

// Many places: radix sort of (entry, place), least significant digits first, of up to 11 bits.  A workgroup ranks
// 256 ROUNDS keys, held in registers; the last pass writes rows for places.
constexpr uint32_t kMaxDigitBits = 11;
template <bool kFirst>
__device__ __forceinline__ u64 sort_key(const u64* in, const Sort& S, uint32_t i) {
    return kFirst ? (u64)place_entry(S, i) << 32 | i : in[i];
}
__device__ __forceinline__ uint32_t digit_of(u64 key, const Sort& S) { return (uint32_t)(key >> 32 >> S.shift) & (S.digits - 1); }
// The block of the places that this workgroup takes (S.blocks and more: none): a part's blocks on one die, so that its stores
// to scattered places meet in that die's cache.
__device__ __forceinline__ uint32_t sort_block(const Sort& S) {
    return S.segs == 1 ? blockIdx.x : blockIdx.x % S.segs * S.seg_blocks + blockIdx.x / S.segs;
}
// Keys of every digit in every block: counts [block][digit].
template <bool kFirst, int ROUNDS>
__global__ __launch_bounds__(256) void sort_count_kernel(const u64* __restrict__ in, Sort S, uint32_t* __restrict__ counts) {
    __shared__ uint32_t count[1 << kMaxDigitBits];
    if (kFirst) clear_marks(S, blockIdx.x, gridDim.x);
    const uint32_t block = sort_block(S);
    if (block >= S.blocks) return;
    for (uint32_t d = threadIdx.x; d < S.digits; d += 256) count[d] = 0;
    uint32_t digit[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = (block * ROUNDS + r) * 256 + threadIdx.x;
        digit[r] = i < S.n ? digit_of(sort_key<kFirst>(in, S, i), S) : ~0u;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (digit[r] != ~0u) atomicAdd(&count[digit[r]], 1u);
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < S.digits; d += 256) counts[(uint64_t)block * S.digits + d] = count[d];
}
// For every part and digit the running sum over the blocks, in place, and its total.  A workgroup takes 64 digits, its
// waves some of the blocks each.
constexpr uint32_t kScanWaves = 16;
__global__ __launch_bounds__(1024) void sort_scan_kernel(Sort S, uint32_t* __restrict__ counts, uint32_t* __restrict__ totals) {
    __shared__ uint32_t part[kScanWaves][64];
    const uint32_t wave = threadIdx.x / 64, lane = lane_id(), d = blockIdx.x * 64 + lane;
    const uint32_t first = blockIdx.y * S.seg_blocks, end = min(S.blocks, first + S.seg_blocks);
    const uint32_t each = (S.seg_blocks + kScanWaves - 1) / kScanWaves, b0 = min(end, first + wave * each), b1 = min(end, b0 + each);
    uint32_t sum = 0;
    if (d < S.digits) {
#pragma unroll 8
        for (uint32_t b = b0; b < b1; ++b) sum += counts[(uint64_t)b * S.digits + d];
    }
    part[wave][lane] = sum;
    __syncthreads();
    uint32_t at = 0;
    for (uint32_t w = 0; w < wave; ++w) at += part[w][lane];
    if (d >= S.digits) return;
    for (uint32_t b = b0; b < b1; b += 8) {
        uint32_t c[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) c[j] = b + j < b1 ? counts[(uint64_t)(b + j) * S.digits + d] : 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            if (b + j < b1) counts[(uint64_t)(b + j) * S.digits + d] = at;
            at += c[j];
        }
    }
    if (wave == kScanWaves - 1) totals[blockIdx.y * S.digits + d] = at;
}
// Keys to their places: the digits below, then the blocks before, then the waves before, then the rounds before, then the lanes
// before.  Without `totals` the counts are as they were counted, and few blocks': each adds them up for itself.
template <bool kFirst, bool kLast, int ROUNDS>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const u64* __restrict__ in, Sort S, const uint32_t* __restrict__ counts,
                                                           const uint32_t* __restrict__ totals, u64* __restrict__ out) {
    __shared__ uint32_t at[4][1 << kMaxDigitBits];
    __shared__ uint32_t sums[4];
    const uint32_t block = sort_block(S), seg = block / S.seg_blocks;
    if (block >= S.blocks) return;
    const uint32_t wave = threadIdx.x / 64, lane = lane_id(), from = (block * 4 + wave) * ROUNDS * 64;
    u64 key[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = from + r * 64 + lane;
        key[r] = i < S.n ? sort_key<kFirst>(in, S, i) : 0;
    }
    for (uint32_t i = threadIdx.x; i < 4 * S.digits; i += 256) at[i / S.digits][i % S.digits] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (from + r * 64 + lane < S.n) atomicAdd(&at[wave][digit_of(key[r], S)], 1u);
    // digits in ascending order by threads: each takes a run of them
    constexpr uint32_t kRun = (1u << kMaxDigitBits) / 256;
    const uint32_t run = (S.digits + 255) / 256, d0 = threadIdx.x * run;
    uint32_t total[kRun], before[kRun], mine = 0;
#pragma unroll
    for (uint32_t j = 0; j < kRun; ++j) {
        const uint32_t d = d0 + j;
        total[j] = before[j] = 0;
        if (j >= run || d >= S.digits) continue;
        if (totals) {
            total[j] = totals[seg * S.digits + d];
            before[j] = counts[(uint64_t)block * S.digits + d];
        } else {
#pragma unroll 8
            for (uint32_t b = 0; b < S.blocks; ++b) {
                const uint32_t c = counts[(uint64_t)b * S.digits + d];
                total[j] += c;
                before[j] += b < block ? c : 0;
            }
        }
        mine += total[j];
    }
    const uint32_t upto = wave_scan(mine, Add(), 0u);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint32_t base = seg * S.seg_blocks * ROUNDS * 256 + upto - mine;   // (a part keeps its places)
    for (uint32_t w = 0; w < wave; ++w) base += sums[w];
#pragma unroll
    for (uint32_t j = 0; j < kRun; ++j) {
        const uint32_t d = d0 + j;
        if (j >= run || d >= S.digits) continue;
        uint32_t a = base + before[j];
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            const uint32_t c = at[w][d];
            at[w][d] = a;
            a += c;
        }
        base += total[j];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const uint32_t i = from + r * 64 + lane, d = digit_of(key[r], S);
        const bool have = i < S.n;
        u64 same = __ballot(have);
        for (int b = 0; b < S.bits; ++b) {
            const u64 set = __ballot(d >> b & 1);
            same &= d >> b & 1 ? set : ~set;
        }
        if (have) {
            const uint32_t place = at[wave][d] + (uint32_t)__popcll(same & ((1ull << lane) - 1));
            out[place] = kLast ? sorted_key(S, seg, (uint32_t)(key[r] >> 32), (uint32_t)key[r]) : key[r];
        }
        wave_fence();
        if (have && (same >> lane) == 1) at[wave][d] += (uint32_t)__popcll(same);   // (the last of the equal ones)
        wave_fence();
    }
}

// ---- sums -----------------------------------------------------------------------------------
constexpr uint32_t kSumThreads = 512;
struct Table {
    const u64* sorted;   // (entry, row); kNoEntry, or more than the entries: none
    uint32_t n, entries, dim;  // (entries: of all parts of the places)
    uint32_t lanes, places;    // of a group: lanes that hold a row's vectors, and places that it adds up
    uint32_t chunk, chunks;    // places of a workgroup
    bool by_chiplet;           // an eighth of the chunks, one after another, to each of the chip's eight dies
    float scale;
    float* part;         // [chunks][2][dim]: of the first run, where it began before; of the last, where it goes on
    uint8_t* mark;       // null: what does not occur is 0 already
};
__device__ __forceinline__ uint32_t entry_at(const Table& B, uint32_t i) { return (uint32_t)(B.sorted[i] >> 32); }

// V values from column c on, in the output's type.
template <class O, int V>
__device__ __forceinline__ void store_values(O* row, uint32_t c, uint32_t dim, const float (&y)[V]) {
    constexpr int N = V * (int)sizeof(O) / 4;   // words
    typedef uint32_t Some __attribute__((ext_vector_type(N), aligned(sizeof(O))));
    if (c + V <= dim) {
        Some w;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(O) == 4)
                w[i] = __builtin_bit_cast(uint32_t, y[i]);
            else
                w[i] = (uint32_t)__builtin_bit_cast(uint16_t, from_f32<O>(y[2 * i])) |
                       (uint32_t)__builtin_bit_cast(uint16_t, from_f32<O>(y[2 * i + 1])) << 16;
        }
        *(Some*)(row + c) = w;
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (c + v < dim) row[c + v] = from_f32<O>(y[v]);
    }
}

// Few places in one workgroup: each thread counts those ahead of its own, among them the ones of the waves before with the same entry.
constexpr uint32_t kAllMost = kSumThreads;
__device__ __forceinline__ void sort_all(const Sort& S, uint32_t* entry, u64* list) {
    const uint32_t n4 = (S.n + 3) / 4 * 4, t = threadIdx.x, wave0 = t / 64 * 64, wave1 = min(wave0 + 64, n4);
    const uint32_t mine = t < S.n ? place_entry(S, t) : ~0u;
    entry[t] = mine;
    __syncthreads();
    typedef uint32_t Quad __attribute__((ext_vector_type(4)));
    const Quad* q = (const Quad*)entry;
    uint32_t ahead = 0;
    if (wave0 < n4) {
#pragma unroll 4
        for (uint32_t i = 0; i < wave0 / 4; ++i) {
            const Quad e = q[i];
            ahead += (e[0] <= mine) + (e[1] <= mine) + (e[2] <= mine) + (e[3] <= mine);
        }
        for (uint32_t i = wave0; i < wave1; ++i) ahead += entry[i] < mine || (entry[i] == mine && i < t);
#pragma unroll 4
        for (uint32_t i = wave1 / 4; i < n4 / 4; ++i) {
            const Quad e = q[i];
            ahead += (e[0] < mine) + (e[1] < mine) + (e[2] < mine) + (e[3] < mine);
        }
        if (t < S.n) list[ahead] = sorted_key(S, 0, mine, t);
    }
    __syncthreads();
}
// Entries that a workgroup clears at a time: about 64 KB of them, for enough workgroups.
template <class O>
__host__ __device__ inline uint32_t zero_rows(uint32_t dim, uint32_t most) {
    const uint32_t rows = 65536 / (uint32_t)sizeof(O) / dim;
    return rows < 8 ? 8 : rows < most ? rows : most;
}
// The entries that do not occur among few places: `blocks` workgroups.
template <class O>
__device__ __forceinline__ void zero_rest(const Sort& S, uint32_t dim, uint32_t block, uint32_t blocks, uint32_t* occurs, O* out) {
    constexpr uint32_t V = 16 / sizeof(O);
    const uint32_t vecs = (dim + V - 1) / V, mine = threadIdx.x < S.n ? place_entry(S, threadIdx.x) : ~0u;
    const uint32_t most = zero_rows<O>(dim, kSumThreads);
    for (uint64_t row0 = (uint64_t)block * most; row0 < S.entries; row0 += (uint64_t)blocks * most) {
        __syncthreads();
        occurs[threadIdx.x] = 0;
        __syncthreads();
        if (mine < S.entries && mine >= row0 && mine - row0 < most) occurs[mine - row0] = 1;
        __syncthreads();
        const uint32_t rows = (uint32_t)min((uint64_t)most, S.entries - row0);
        float z[V] = {};
        for (uint32_t j = threadIdx.x; j < rows * vecs; j += kSumThreads) {
            const uint32_t r = j / vecs;
            if (!occurs[r]) store_pack<O, true>(out + (row0 + r) * dim, 1, j % vecs * V, dim, z);
        }
    }
}

// A group of lanes takes `places` of the list, eight rows on their way at a time, and writes the runs that lie within them.
// What of a run lies in several groups goes to LDS and is added up, in the groups' order, by the group in which it begins; what lies
// in several workgroups, by join_kernel.
enum { kHead = 1, kHeadEnds = 2, kTail = 4 };   // the first run began before; and ends here; the last begins here and goes on
// kAll: all places are one chunk, which the workgroup sorts by itself; behind the workgroups of the columns come those of the entries that do not
// occur.
template <class T, class O, bool kWhole, bool kAll>
__global__ __launch_bounds__(kSumThreads) void table_sum_kernel(const T* __restrict__ grad, int64_t rs, int64_t cs, Table B,
                                                                Sort S, O* __restrict__ out) {
    constexpr int V = Pack<T>::V, kFly = 8;
    __shared__ float slot[kSumThreads * V];   // heads [group][column]
    __shared__ uint32_t flags[kSumThreads];
    const uint32_t width = B.lanes * V, tiles = (B.dim + width - 1) / width, per = kSumThreads / B.lanes;
    const uint32_t group = threadIdx.x / B.lanes, in = threadIdx.x % B.lanes;
    __shared__ u64 list[kAll ? kAllMost : 1];
    if constexpr (kAll) {
        if (blockIdx.x >= tiles) return zero_rest<O>(S, B.dim, blockIdx.x - tiles, gridDim.x - tiles, (uint32_t*)list, out);
        static_assert(kAllMost <= kSumThreads * V, "entries in the heads' place");
        sort_all(S, (uint32_t*)slot, list);
        B.sorted = list;
    }
    const uint32_t eighth = (B.chunks + 7) / 8;
    for (uint64_t job = blockIdx.x; job < (kAll ? (uint64_t)tiles : (uint64_t)eighth * 8 * tiles); job += kAll ? tiles : gridDim.x) {
        const uint32_t chunk = B.by_chiplet ? (uint32_t)(job % 8) * eighth + (uint32_t)(job / 8 / tiles) : (uint32_t)(job / tiles);
        if (chunk >= B.chunks) continue;
        const uint32_t c0 = (uint32_t)((B.by_chiplet ? job / 8 : job) % tiles) * width, c = c0 + in * V;
        const uint32_t column = c < B.dim ? c : 0;   // (a lane behind the row reads its beginning)
        const uint32_t from = min(B.n, chunk * B.chunk + group * B.places), to = min(B.n, from + B.places);
        uint32_t cur = kNoEntry, flag = 0;
        bool before = false;
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        auto keep = [&] {
#pragma unroll
            for (int v = 0; v < V; ++v) slot[threadIdx.x * V + v] = acc[v];
        };
        auto finish = [&] {   // the run of cur ends within the group
            if (before) {
                keep();
                flag |= kHead | kHeadEnds;
            } else if (cur < B.entries && c < B.dim) {
                float y[V];
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = acc[v] * B.scale;
                store_values<O, V>(out + (uint64_t)cur * B.dim, c, B.dim, y);
                if (!kAll && c == 0 && B.mark) B.mark[cur] = 1;
            }
        };
        if (from < to) {
            cur = entry_at(B, from);
            before = from > 0 && cur < B.entries && entry_at(B, from - 1) == cur;
            for (uint32_t i0 = from; i0 < to; i0 += kFly) {
                uint32_t e[kFly];
                Pack<T> p[kFly];
#pragma unroll
                for (int u = 0; u < kFly; ++u) {
                    const u64 key = B.sorted[min(i0 + u, to - 1)];
                    e[u] = i0 + u < to ? (uint32_t)(key >> 32) : kNoEntry;
                    p[u] = load_columns<T, kWhole>(grad + (int64_t)(uint32_t)key * rs, cs, column, B.dim);   // (without a branch)
                    if (e[u] >= B.entries) p[u].w = Words{};
                }
#pragma unroll
                for (int u = 0; u < kFly; ++u) {
                    if (i0 + u < to && e[u] != cur) {
                        finish();
                        before = false;
                        cur = e[u];
#pragma unroll
                        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
                    }
#pragma unroll
                    for (int v = 0; v < V; ++v) acc[v] += p[u].get(v);
                }
            }
            const bool after = cur < B.entries && to < B.n && entry_at(B, to) == cur;
            if (!after) {
                finish();
            } else {
                if (before) keep();
                flag |= before ? kHead : kTail;   // (a tail stays in acc)
            }
        }
        if (in == 0) flags[group] = flag;
        __syncthreads();
        // a run's parts, by the group in which it begins, or by the first where it began before the chunk
        const bool tails = flag & kTail, heads = group == 0 && (flag & kHead);
        if ((tails || heads) && c < B.dim) {
            if (tails && heads) {   // (a head that ends here, before the tail)
                float y[V];
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = slot[threadIdx.x * V + v];
                store_values<float, V>(B.part + (uint64_t)chunk * 2 * B.dim, c, B.dim, y);
            } else if (heads) {
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] = slot[threadIdx.x * V + v];
            }
            uint32_t last = tails ? 0u : flag, a = group + 1;
            while (!(last & kHeadEnds) && a < per && (flags[a] & kHead)) {
                last = flags[a];
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] += slot[(a * B.lanes + in) * V + v];
                ++a;
            }
            if (!(last & kHeadEnds) || !tails) {   // past this workgroup, or from before it
                float* p = B.part + ((uint64_t)chunk * 2 + tails) * B.dim;
                store_values<float, V>(p, c, B.dim, acc);
            } else {
                float y[V];
#pragma unroll
                for (int v = 0; v < V; ++v) y[v] = acc[v] * B.scale;
                store_values<O, V>(out + (uint64_t)cur * B.dim, c, B.dim, y);
            }
            if (!kAll && c == 0 && tails && B.mark) B.mark[cur] = 1;
        }
        __syncthreads();
    }
}

// Runs of several workgroups, by that of the chunk in which they begin; and the entries that do not occur.
template <class O>
__global__ __launch_bounds__(256) void table_join_kernel(Table B, uint32_t join_blocks, O* __restrict__ out) {
    __shared__ uint32_t list[256], count;
    __shared__ float sum[4][64];
    const uint32_t wave = threadIdx.x / 64, lane = lane_id();
    if (blockIdx.x >= join_blocks) {
        constexpr uint32_t V = 16 / sizeof(O);
        const uint32_t vecs = (B.dim + V - 1) / V;
        const uint32_t most = zero_rows<O>(B.dim, 256);
        for (uint64_t row0 = (uint64_t)(blockIdx.x - join_blocks) * most; row0 < B.entries;
             row0 += (uint64_t)(gridDim.x - join_blocks) * most) {
            __syncthreads();
            if (threadIdx.x == 0) count = 0;
            __syncthreads();
            const uint64_t row = row0 + threadIdx.x;
            if (threadIdx.x < most && row < B.entries && (!B.n || !B.mark[row])) list[atomicAdd(&count, 1u)] = threadIdx.x;   // (their order does not matter)
            __syncthreads();
            float z[V] = {};
            for (uint32_t j = threadIdx.x; j < count * vecs; j += 256)
                store_pack<O, true>(out + (row0 + list[j / vecs]) * B.dim, 1, (uint32_t)(j % vecs) * V, B.dim, z);
        }
        return;
    }
    for (uint32_t chunk = blockIdx.x; chunk + 1 < B.chunks; chunk += join_blocks) {
        const uint32_t from = chunk * B.chunk, next = from + B.chunk, e = entry_at(B, next - 1);
        if (e >= B.entries || entry_at(B, next) != e) continue;
        if (from > 0 && entry_at(B, from) == e && entry_at(B, from - 1) == e) continue;   // began before
        // the last chunk that the run reaches
        __syncthreads();
        if (threadIdx.x == 0) count = B.chunks - 1;
        __syncthreads();
        for (uint32_t c0 = chunk + 1;; c0 += 256) {
            const uint32_t c = c0 + threadIdx.x;
            const bool ends = c < B.chunks && (c == B.chunks - 1 || entry_at(B, (c + 1) * B.chunk) != e);
            if (ends) atomicMin(&count, c);
            if (__syncthreads_or(ends) || c0 + 256 >= B.chunks) break;
        }
        __syncthreads();
        const uint32_t upto = count, behind = upto - chunk;   // chunks behind the first
        const uint32_t each = (behind + 3) / 4;
        const uint32_t a = chunk + 1 + min(behind, wave * each), b = min(upto + 1, a + each);
        for (uint32_t c0 = 0; c0 < B.dim; c0 += 64) {
            const uint32_t c = c0 + lane;
            float s = 0.0f;
            if (c < B.dim) {
                if (wave == 0) s = B.part[((uint64_t)chunk * 2 + 1) * B.dim + c];
#pragma unroll 8
                for (uint32_t q = a; q < b; ++q) s += B.part[(uint64_t)q * 2 * B.dim + c];
            }
            sum[wave][lane] = s;
            __syncthreads();
            if (wave == 0 && c < B.dim)
                out[(uint64_t)e * B.dim + c] = from_f32<O>((((sum[0][lane] + sum[1][lane]) + sum[2][lane]) + sum[3][lane]) * B.scale);
            __syncthreads();
        }
    }
}

// The parts' sums together.
template <class O>
__global__ __launch_bounds__(256) void table_parts_kernel(const float* __restrict__ sums, const uint8_t* __restrict__ mark, uint32_t segs,
                                                          uint32_t entries, uint32_t dim, float scale, O* __restrict__ out) {
    const uint64_t all = (uint64_t)entries * dim;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
        const uint32_t e = (uint32_t)(i / dim);
        float sum = 0.0f;
        for (uint32_t s = 0; s < segs; ++s)
            if (mark[(uint64_t)s * entries + e]) sum += sums[s * all + i];
        out[i] = from_f32<O>(sum * scale);
    }
}

// ---- host -----------------------------------------------------------------------------------
// Long lists read a row's gradient many times.  Where all rows pass a die's 4 MB of second-level cache and the entries are few, the places are
// sorted and added up in eight parts, one a die, whose rows are fewer; the parts' sums are added then.
constexpr uint32_t kParts = 8;
struct Layout {
    uint32_t n, passes, bits, rounds, blocks;
    uint32_t lanes, places, chunk, chunks;
    uint32_t segs, seg_blocks;
    uint64_t keys, counts, totals, mark, part, sums, bytes;   // offsets; keys: two arrays
};
Layout layout(uint64_t rows, uint32_t list, uint32_t entries, uint32_t dim, uint32_t vec) {
    Layout L{};
    L.n = (uint32_t)(rows * list);
    uint32_t bits = 1;
    while (entries >> bits) ++bits;   // keys are 0 .. entries
    L.passes = L.n <= kRankMost ? 0 : (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    L.bits = L.passes ? (bits + L.passes - 1) / L.passes : 0;
    L.rounds = L.n <= 1u << 19 ? 4 : 16;
    L.blocks = (L.n + L.rounds * 256 - 1) / (L.rounds * 256);
    const uint64_t cells = (uint64_t)entries * dim;
    const bool parted = L.passes && list >= 8 && rows * dim * (16 / vec) > 4u << 20 && (uint64_t)entries * kParts * 16 <= L.n && cells <= 1u << 20;
    L.segs = parted ? kParts : 1;
    L.seg_blocks = std::max(1u, (L.blocks + L.segs - 1) / L.segs);
    L.lanes = 1;
    while (L.lanes < 64 && L.lanes * vec < dim) L.lanes *= 2;
    // few places in one chunk: fewer lanes a group, so that eight places are a group's, one after another
    while (L.n <= kAllMost && L.lanes > 8 && kSumThreads / L.lanes * 8 < L.n) L.lanes /= 2;
    // workgroups that fill the chip about once (1024 of 512 threads): several rounds wait for the last one's few
    const uint64_t tiles = (dim + L.lanes * vec - 1) / (L.lanes * vec), per = kSumThreads / L.lanes;
    L.places = (uint32_t)std::min<uint64_t>(32, std::max<uint64_t>(8, (L.n <= 1u << 17 ? 256 : 512) / per));
    while (L.places < 128 && (uint64_t)L.n * tiles > 1024 * per * L.places) L.places *= 2;
    if (L.n <= kAllMost) L.places = (uint32_t)std::max<uint64_t>(1, (L.n + per - 1) / per);   // one chunk
    L.chunk = L.places * (kSumThreads / L.lanes);
    L.chunks = (L.n + L.chunk - 1) / L.chunk;
    if (L.n <= kAllMost) return L;   // (no workspace)
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t p = at;
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    L.keys = take((L.passes > 1 ? 16 : 8) * (uint64_t)L.n);
    L.counts = take(L.passes ? 4ull * L.blocks << L.bits : 0);
    L.totals = take(L.passes ? (4ull << L.bits) * L.segs : 0);
    L.mark = take(L.passes ? (uint64_t)entries * L.segs : 0);
    L.sums = take(L.segs > 1 ? 4 * cells * L.segs : 0);
    L.part = take(8ull * L.chunks * dim);
    L.bytes = at;
    return L;
}

template <class O>
uint32_t zero_blocks(uint32_t entries, uint32_t dim, uint32_t most) {
    const uint32_t rows = zero_rows<O>(dim, most);
    return std::min<uint32_t>((entries + rows - 1) / rows, 1u << 14);
}
template <class T, class O>
int launch_sums(const void* grad, int64_t rs, int64_t cs, const Table& B, const Sort& S, void* out, hipStream_t st) {
    const uint32_t tiles = (B.dim + B.lanes * Pack<T>::V - 1) / (B.lanes * Pack<T>::V);
    const bool whole = cs == 1 && B.dim % Pack<T>::V == 0;
    if (S.n && S.n <= kAllMost) {
        const unsigned grid = tiles + zero_blocks<O>(S.entries, B.dim, kSumThreads);
        if (whole) table_sum_kernel<T, O, true, true><<<grid, kSumThreads, 0, st>>>((const T*)grad, rs, cs, B, S, (O*)out);
        else table_sum_kernel<T, O, false, true><<<grid, kSumThreads, 0, st>>>((const T*)grad, rs, cs, B, S, (O*)out);
        CLS_TRY(hipGetLastError());
        return CBH_OK;
    }
    if (B.n) {
        const unsigned grid = row_grid((uint64_t)(B.chunks + 7) / 8 * 8 * tiles);
        if (whole) table_sum_kernel<T, O, true, false><<<grid, kSumThreads, 0, st>>>((const T*)grad, rs, cs, B, S, (O*)out);
        else table_sum_kernel<T, O, false, false><<<grid, kSumThreads, 0, st>>>((const T*)grad, rs, cs, B, S, (O*)out);
        CLS_TRY(hipGetLastError());
    }
    const uint32_t join = B.chunks > 1 ? std::min<uint32_t>(B.chunks - 1, 1u << 14) : 0;
    const uint32_t zero = B.by_chiplet || (B.n && !B.mark) ? 0 : zero_blocks<O>(B.entries, B.dim, 256);
    if (join + zero == 0) return CBH_OK;
    table_join_kernel<O><<<join + zero, 256, 0, st>>>(B, join, (O*)out);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}
template <class O>
int launch_parts(const Layout& L, char* ws, uint32_t entries, uint32_t dim, float scale, void* out, hipStream_t st) {
    const unsigned grid = (unsigned)std::min<uint64_t>(((uint64_t)entries * dim + 255) / 256, 4096);
    table_parts_kernel<O><<<grid, 256, 0, st>>>((const float*)(ws + L.sums), (const uint8_t*)(ws + L.mark), L.segs, entries, dim, scale, (O*)out);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}
template <class T>
int launch_sums(const void* grad, int64_t rs, int64_t cs, const Table& B, const Sort& S, void* out, int32_t type, hipStream_t st) {
    switch (type) {
        case CBH_TYPE_F32: return launch_sums<T, float>(grad, rs, cs, B, S, out, st);
        case CBH_TYPE_F16: return launch_sums<T, _Float16>(grad, rs, cs, B, S, out, st);
        default: return launch_sums<T, bf16_t>(grad, rs, cs, B, S, out, st);
    }
}

// Counts of so few blocks are added up by every block of the scatter, without a launch for them.
constexpr uint32_t kOwnScan = 32;
template <int ROUNDS>
int sort_by_digits(Sort S, const Layout& L, char* ws, u64** sorted, hipStream_t st) {
    u64* a = (u64*)(ws + L.keys);
    u64* b = a + L.n;
    const u64* in = nullptr;
    const unsigned grid = L.segs * L.seg_blocks;   // (one part: the blocks)
    uint32_t* counts = (uint32_t*)(ws + L.counts);
    uint32_t* totals = L.blocks <= kOwnScan && L.segs == 1 ? nullptr : (uint32_t*)(ws + L.totals);
    for (uint32_t p = 0; p < L.passes; ++p) {
        S.shift = (int)(p * L.bits);
        const bool first = p == 0, last = p + 1 == L.passes;
        if (first) sort_count_kernel<true, ROUNDS><<<grid, 256, 0, st>>>(in, S, counts);
        else sort_count_kernel<false, ROUNDS><<<grid, 256, 0, st>>>(in, S, counts);
        CLS_TRY(hipGetLastError());
        if (totals) {
            sort_scan_kernel<<<dim3((S.digits + 63) / 64, S.segs), 64 * kScanWaves, 0, st>>>(S, counts, totals);
            CLS_TRY(hipGetLastError());
        }
#define SCATTER(F, L_) sort_scatter_kernel<F, L_, ROUNDS><<<grid, 256, 0, st>>>(in, S, counts, totals, a)
        if (first) last ? SCATTER(true, true) : SCATTER(true, false);
        else last ? SCATTER(false, true) : SCATTER(false, false);
#undef SCATTER
        CLS_TRY(hipGetLastError());
        *sorted = a;
        in = a;
        std::swap(a, b);
    }
    return CBH_OK;
}
// Few places: sorted by one launch, which clears the gradient too.
template <class O>
int rank_places(const Sort& S, u64* sorted, void* out, uint32_t dim, hipStream_t st) {
    const uint64_t cells = (uint64_t)S.entries * dim, each = 64 * kRankWaves * (16 / sizeof(O)) * 4;
    const unsigned clear = (unsigned)std::min<uint64_t>((cells + each - 1) / each, 2048);
    rank_kernel<O><<<(S.n + 63) / 64 + clear, 64 * kRankWaves, 0, st>>>(S, sorted, (O*)out, cells);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

int check_index(const int32_t* index, uint64_t rows, uint32_t list, uint32_t entries, uint32_t dim) {
    if (entries < 1 || entries >= 1u << 31) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "entries must be in 1 .. 2^31 - 1");
    if (dim < 1 || dim > kMaxClasses) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "dim must be in 1 .. 2^24");
    if (list < 1) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "a list holds at least one index");
    if (rows > 0x7FFFFFFFull || rows * list > 0x7FFFFFFFull)
        return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "rows times list must be below 2^31");
    if (rows && !index) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "index is null");
    if ((uintptr_t)index % 4) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "index is not aligned to 4");
    return CBH_OK;
}
int check_matrix(const void* p, int32_t type, const char* what, uint64_t rows, uint32_t dim, int64_t rs, int64_t cs) {
    if (type != CBH_TYPE_F32 && type != CBH_TYPE_F16 && type != CBH_TYPE_BF16)
        return cbh_internal_fail(CBH_ERR_UNSUPPORTED, std::string(what) + " is f32, f16 or bf16");
    if (rows && !p) return cbh_internal_fail(CBH_ERR_INVALID_ARG, std::string(what) + " is null");
    if ((uintptr_t)p % type_bytes(type)) return cbh_internal_fail(CBH_ERR_INVALID_ARG, std::string(what) + " is not aligned to its type");
    const double lim = 4.0e18 / (double)type_bytes(type);
    if (std::abs((double)rs) * (double)rows + std::abs((double)cs) * (double)dim > lim)
        return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "strides pass the address range");
    return CBH_OK;
}
int check_scale(double scale) {
    return std::abs(scale) <= 3.4e38 ? CBH_OK : cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "scale must be a finite f32");
}

template <class T>
int run_lookup(const void* table, int64_t rs, int64_t cs, const Lookup& L, void* out, hipStream_t st) {
    constexpr uint32_t V = Pack<T>::V;
    uint32_t lanes = 1;
    while (lanes < 64 && lanes * V < L.dim) lanes *= 2;
    // In LDS: lists long enough that an entry is read often, and 64 bytes of every entry in it, or its whole row.  Of less, each list is
    // read by many workgroups, and rows are written in pieces of lines that lanes do not share.  By LDS and from the caches, us: 400000
    // lists of 8 f32, 2500 entries of 64 columns (64 bytes held) 34 and 37, 4000 of 64 (32 bytes) 134 and 37, 9000 of 64 (16 bytes) 254
    // and 40; 200000 lists of 40, 1280 of 64, 58 and 78.
    // Less of a row pays where the caches' way is slow.  Rows that are no whole vectors are read value by value: 400000 lists of 8 over
    // 9000 entries, 16 bytes of 30 bf16 64 and 108, of 255 723 and 484, of 5 f32 14 and 33, of 13 38 and 35; 100000 lists of 40 over 5200
    // entries of 255 bf16 195 and 389; over 4000 of 70 f32 (32 bytes) 106 and 137, 5200 of 255 (16 bytes) 300 and 357, 9000 of 30 100
    // and 53.  And a large table is not in the second level: 60000 lists of 40 over 9000 entries of 1000 f32 702 and 849, 100000 over
    // 9000 of 256 287 and 316; in it, 5200 of 256, 284 and 183.
    uint32_t held = lanes;
    while (held > 1 && (L.entries + 1ull) * held * 16 > kLdsBytes) held /= 2;
    const bool lists_long = L.list >= 32;
    // of a row's vectors, one that is enough
    const uint32_t share = L.dim % V == 0 ? 1 : lists_long && (V == 8 || held >= 2) ? 64 : V == 8 ? 8 : 2;
    const bool pays = held >= 4 || lanes <= held * share || (lists_long && (uint64_t)L.entries * L.dim * sizeof(T) > 8u << 20);
    if (cs == 1 && L.list >= 8 && L.rows * L.list >= 256ull * L.entries && pays && (L.entries + 1ull) * held * 16 <= kLdsBytes) {
        const uint32_t tiles = (L.dim + held * V - 1) / (held * V);
        const uint64_t least = kLdsThreads / held;   // rows of one round
        const uint64_t parts = std::max<uint64_t>(1, std::min<uint64_t>((256 + tiles - 1) / tiles, (L.rows + 2 * least - 1) / (2 * least)));
        const uint64_t part = (L.rows + parts - 1) / parts;
        const size_t lds = (L.entries + 1) * (size_t)held * 16;
        if (lds > 65536) CLS_TRY(hipFuncSetAttribute((const void*)lookup_lds_kernel<T>, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes));
        lookup_lds_kernel<T><<<(unsigned)((L.rows + part - 1) / part * tiles), kLdsThreads, lds, st>>>((const T*)table, rs, L, (T*)out, held, tiles, part);
        CLS_TRY(hipGetLastError());
        return CBH_OK;
    }
    const uint32_t tiles = (L.dim + lanes * V - 1) / (lanes * V), per = 256 / lanes;
    const unsigned grid = row_grid((L.rows + per - 1) / per * tiles);
    if (cs == 1 && L.dim % V == 0) lookup_kernel<T, true><<<grid, 256, 0, st>>>((const T*)table, rs, cs, L, (T*)out, lanes);
    else lookup_kernel<T, false><<<grid, 256, 0, st>>>((const T*)table, rs, cs, L, (T*)out, lanes);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

}  // namespace

extern "C" int cbh_lookup_rows(const void* table, int32_t type, uint32_t entries, uint32_t dim, int64_t row_stride,
                               int64_t column_stride, const int32_t* index, uint64_t rows, uint32_t list, double scale, void* out,
                               void* stream) {
    try {
        int rc = check_index(index, rows, list, entries, dim);
        if (rc == CBH_OK) rc = check_matrix(table, type, "the table", entries, dim, row_stride, column_stride);
        if (rc == CBH_OK) rc = check_matrix(out, type, "out", rows, dim, dim, 1);
        if (rc == CBH_OK) rc = check_scale(scale);
        if (rc != CBH_OK || rows == 0) return rc;
        hipStream_t st = (hipStream_t)stream;
        const Lookup L{index, rows, entries, dim, list, (float)scale};
#define RUN(T) run_lookup<T>(table, row_stride, column_stride, L, out, st)
        switch (type) {
            case CBH_TYPE_F32: return RUN(float);
            case CBH_TYPE_F16: return RUN(_Float16);
            default: return RUN(bf16_t);
        }
#undef RUN
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}

extern "C" uint64_t cbh_lookup_gradients_workspace(uint64_t rows, uint32_t list, uint32_t entries, uint32_t dim) {
    if (rows > 0x7FFFFFFFull || rows * list > 0x7FFFFFFFull || entries < 1 || entries >= 1u << 31 || dim > kMaxClasses) return 0;
    return std::max(layout(rows, list, entries, dim, 4).bytes, layout(rows, list, entries, dim, 8).bytes);
}

extern "C" int cbh_lookup_gradients(const void* grad, int32_t type, uint64_t rows, uint32_t dim, int64_t row_stride,
                                    int64_t column_stride, const int32_t* index, uint32_t list, uint32_t entries, double scale,
                                    void* table_grad, int32_t grad_type, void* workspace, uint64_t workspace_bytes, void* stream) {
    try {
        int rc = check_index(index, rows, list, entries, dim);
        if (rc == CBH_OK) rc = check_matrix(grad, type, "the gradient", rows, dim, row_stride, column_stride);
        if (rc == CBH_OK) rc = check_matrix(table_grad, grad_type, "the table's gradient", entries, dim, dim, 1);
        if (rc == CBH_OK) rc = check_scale(scale);
        if (rc != CBH_OK) return rc;
        const uint64_t need = cbh_lookup_gradients_workspace(rows, list, entries, dim);
        if (need > workspace_bytes || (need && (!workspace || (uintptr_t)workspace % 16)))
            return cbh_internal_fail(CBH_ERR_LENGTH_MISMATCH, "the workspace needs " + std::to_string(need) +
                                                                  " bytes, aligned to 16");
        const Layout L = layout(rows, list, entries, dim, 16 / (uint32_t)type_bytes(type));
        hipStream_t st = (hipStream_t)stream;
        char* ws = (char*)workspace;
        u64* sorted = nullptr;
        const Sort S{index, L.n, entries, list, L.blocks, 1u << L.bits, 0, (int)L.bits, L.segs, L.seg_blocks, (uint8_t*)(ws + L.mark)};
        if (L.n > kAllMost) {
            sorted = (u64*)(ws + L.keys);
            if (L.passes) rc = L.rounds == 4 ? sort_by_digits<4>(S, L, ws, &sorted, st) : sort_by_digits<16>(S, L, ws, &sorted, st);
            else if (grad_type == CBH_TYPE_F32) rc = rank_places<float>(S, sorted, table_grad, dim, st);
            else rc = rank_places<_Float16>(S, sorted, table_grad, dim, st);   // (0 is the same in both 16-bit types)
            if (rc != CBH_OK) return rc;
        }
        const bool parted = L.segs > 1;
        const Table B{sorted,  L.n,      L.segs * entries, dim,    L.lanes,        L.places, L.chunk,
                      L.chunks, parted, parted ? 1.0f : (float)scale, (float*)(ws + L.part), L.passes ? (uint8_t*)(ws + L.mark) : nullptr};
        void* sums = parted ? (void*)(ws + L.sums) : table_grad;
        const int32_t sum_type = parted ? CBH_TYPE_F32 : grad_type;
        switch (type) {
            case CBH_TYPE_F32: rc = launch_sums<float>(grad, row_stride, column_stride, B, S, sums, sum_type, st); break;
            case CBH_TYPE_F16: rc = launch_sums<_Float16>(grad, row_stride, column_stride, B, S, sums, sum_type, st); break;
            default: rc = launch_sums<bf16_t>(grad, row_stride, column_stride, B, S, sums, sum_type, st);
        }
        if (rc != CBH_OK || !parted) return rc;
        switch (grad_type) {
            case CBH_TYPE_F32: return launch_parts<float>(L, ws, entries, dim, (float)scale, table_grad, st);
            case CBH_TYPE_F16: return launch_parts<_Float16>(L, ws, entries, dim, (float)scale, table_grad, st);
            default: return launch_parts<bf16_t>(L, ws, entries, dim, (float)scale, table_grad, st);
        }
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}
