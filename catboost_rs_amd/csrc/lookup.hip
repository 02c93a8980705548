// Sums of looked-up rows of a table, and the table's gradient by sorted places.
//
//   out[r] = scale sum_i table[index[r][i]],   table_grad[v] = scale sum over the places (r, i) of v of grad[r]
//
// The gradient is a sum by entry without atomics: the places are sorted by entry (stable, so that a sum has one
// order), runs of equal entries are added up from the sorted list, and what of a run lies in several chunks of the list
// is joined in the chunks' order.
#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

// ---- rows -----------------------------------------------------------------------------------
// A thread takes a vector of a row of the output.
template <class T, bool kUnit>
__global__ __launch_bounds__(256) void lookup_kernel(const T* __restrict__ table, uint32_t entries, uint32_t dim, int64_t rs,
                                                     int64_t cs, const int32_t* __restrict__ index, uint64_t rows, uint32_t list,
                                                     float scale, T* __restrict__ out, uint32_t vecs) {
    constexpr int V = Pack<T>::V;
    const uint64_t jobs = rows * vecs;
    for (uint64_t job = (uint64_t)blockIdx.x * 256 + threadIdx.x; job < jobs; job += (uint64_t)gridDim.x * 256) {
        const uint64_t row = job / vecs;
        const uint32_t c = (uint32_t)(job % vecs) * V;
        const int32_t* ix = index + row * list;
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        for (uint32_t i = 0; i < list; ++i) {
            const uint32_t e = (uint32_t)ix[i];
            if (e >= entries) continue;
            float x[V];
            load_pack<T, kUnit>(table + (int64_t)e * rs, cs, c, dim, 0.0f, x);
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] += x[v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] *= scale;
        store_pack<T, true>(out + row * dim, 1, c, dim, acc);
    }
}

// ---- sort -----------------------------------------------------------------------------------
// Stable radix sort of (entry, place), least significant digits first, of up to 11 bits.  A workgroup ranks 4096 keys.
constexpr uint32_t kSortKeys = 4096, kSortWaves = 4, kMaxDigitBits = 11, kWaveKeys = kSortKeys / kSortWaves;
struct Sort {
    uint32_t n, entries;      // keys; a place without an entry sorts behind all, as `entries`
    uint32_t blocks, digits;  // of a pass; digits a power of two
    int shift, bits;
};
__device__ __forceinline__ u64 first_key(const int32_t* index, uint32_t i, uint32_t entries) {
    return (u64)min((uint32_t)index[i], entries) << 32 | i;
}
template <bool kFirst>
__device__ __forceinline__ u64 sort_key(const void* in, uint32_t i, uint32_t entries) {
    return kFirst ? first_key((const int32_t*)in, i, entries) : ((const u64*)in)[i];
}
template <bool kFirst>
__device__ __forceinline__ void count_digits(const void* in, const Sort& S, uint32_t from, uint32_t to, uint32_t* count) {
    for (uint32_t i = from + lane_id(); i < to; i += 64)
        atomicAdd(&count[(uint32_t)(sort_key<kFirst>(in, i, S.entries) >> 32 >> S.shift) & (S.digits - 1)], 1u);
}
// Keys of every digit in every block: counts [block][digit].  The first pass clears the marks of entries that occur.
template <bool kFirst>
__global__ __launch_bounds__(256) void sort_count_kernel(const void* __restrict__ in, Sort S, uint32_t* __restrict__ counts,
                                                         uint8_t* __restrict__ mark) {
    __shared__ uint32_t count[1 << kMaxDigitBits];
    if (kFirst)
        for (uint64_t v = (uint64_t)blockIdx.x * 256 + threadIdx.x; v < S.entries; v += (uint64_t)gridDim.x * 256) mark[v] = 0;
    for (uint32_t d = threadIdx.x; d < S.digits; d += 256) count[d] = 0;
    __syncthreads();
    const uint32_t wave = threadIdx.x / 64, from = blockIdx.x * kSortKeys + wave * kWaveKeys;
    if (from < S.n) count_digits<kFirst>(in, S, from, min(S.n, from + kWaveKeys), count);
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < S.digits; d += 256) counts[(uint64_t)blockIdx.x * S.digits + d] = count[d];
}
// For every digit the running sum over the blocks, in place, and its total.  A workgroup takes 64 digits, its waves
// a quarter of the blocks each.
__global__ __launch_bounds__(256) void sort_scan_kernel(Sort S, uint32_t* __restrict__ counts, uint32_t* __restrict__ totals) {
    __shared__ uint32_t part[4][64];
    const uint32_t wave = threadIdx.x / 64, lane = lane_id(), d = blockIdx.x * 64 + lane;
    const uint32_t each = (S.blocks + 3) / 4, b0 = min(S.blocks, wave * each), b1 = min(S.blocks, b0 + each);
    uint32_t sum = 0;
    if (d < S.digits)
        for (uint32_t b = b0; b < b1; ++b) sum += counts[(uint64_t)b * S.digits + d];
    part[wave][lane] = sum;
    __syncthreads();
    uint32_t at = 0;
    for (uint32_t w = 0; w < wave; ++w) at += part[w][lane];
    if (d >= S.digits) return;
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t c = counts[(uint64_t)b * S.digits + d];
        counts[(uint64_t)b * S.digits + d] = at;
        at += c;
    }
    if (wave == 3) totals[d] = at;
}
// Keys to their places: the digits below, then the blocks before, then the waves before, then the rounds before, then the lanes
// before.  The last pass marks the entries that occur.
template <bool kFirst, bool kLast>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const void* __restrict__ in, Sort S, const uint32_t* __restrict__ counts,
                                                           const uint32_t* __restrict__ totals, u64* __restrict__ out,
                                                           uint8_t* __restrict__ mark) {
    __shared__ uint32_t at[kSortWaves][1 << kMaxDigitBits];
    __shared__ uint32_t sums[4];
    const uint32_t wave = threadIdx.x / 64, lane = lane_id(), from = blockIdx.x * kSortKeys + wave * kWaveKeys;
    for (uint32_t i = threadIdx.x; i < kSortWaves * S.digits; i += 256) at[i / S.digits][i % S.digits] = 0;
    __syncthreads();
    const uint32_t to = from < S.n ? min(S.n, from + kWaveKeys) : from;
    count_digits<kFirst>(in, S, from, to, at[wave]);
    __syncthreads();
    // digits in ascending order by threads: each takes a run of them
    const uint32_t run = (S.digits + 255) / 256, d0 = threadIdx.x * run;
    uint32_t mine = 0;
    for (uint32_t d = d0; d < min(S.digits, d0 + run); ++d) mine += totals[d];
    const uint32_t upto = wave_scan(mine, Add(), 0u);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint32_t base = upto - mine;
    for (uint32_t w = 0; w < wave; ++w) base += sums[w];
    for (uint32_t d = d0; d < min(S.digits, d0 + run); ++d) {
        uint32_t a = base + counts[(uint64_t)blockIdx.x * S.digits + d];
#pragma unroll
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            const uint32_t c = at[w][d];
            at[w][d] = a;
            a += c;
        }
        base += totals[d];
    }
    __syncthreads();
    for (uint32_t i0 = from; i0 < to; i0 += 64) {
        const uint32_t i = i0 + lane;
        const bool have = i < to;
        const u64 key = have ? sort_key<kFirst>(in, i, S.entries) : 0;
        const uint32_t d = (uint32_t)(key >> 32 >> S.shift) & (S.digits - 1);
        u64 same = __ballot(have);
        for (int b = 0; b < S.bits; ++b) {
            const u64 set = __ballot(d >> b & 1);
            same &= d >> b & 1 ? set : ~set;
        }
        if (have) {
            const uint32_t ahead = (uint32_t)__popcll(same & ((1ull << lane) - 1));
            out[at[wave][d] + ahead] = key;
            if (kLast && (uint32_t)(key >> 32) < S.entries) mark[key >> 32] = 1;
        }
        wave_fence();
        if (have && (same >> lane) == 1) at[wave][d] += (uint32_t)__popcll(same);   // (the last of the equal ones)
        wave_fence();
    }
}

// ---- sums -----------------------------------------------------------------------------------
struct Table {
    const u64* sorted;   // (entry, place)
    uint32_t n, entries, dim, list, chunk, chunks;
    float scale;
    float* part;         // [chunks][2][dim]: of the first run, where it began before; of the last, where it goes on
};
__device__ __forceinline__ uint32_t entry_at(const Table& B, uint32_t i) { return (uint32_t)(B.sorted[i] >> 32); }

// A group of `lanes` lanes takes a chunk of the list and its vectors of the rows.
template <class T, class O, bool kUnit>
__global__ __launch_bounds__(256) void table_sum_kernel(const T* __restrict__ grad, int64_t rs, int64_t cs, Table B, uint32_t lanes,
                                                        O* __restrict__ out) {
    constexpr int V = Pack<T>::V;
    const uint32_t tiles = (B.dim + lanes * V - 1) / (lanes * V), per = 256 / lanes;
    const uint64_t groups = ((uint64_t)B.chunks + per - 1) / per;
    for (uint64_t job = blockIdx.x; job < groups * tiles; job += gridDim.x) {
        const uint32_t chunk = (uint32_t)(job / tiles) * per + threadIdx.x / lanes;
        const uint32_t c = ((uint32_t)(job % tiles) * lanes + threadIdx.x % lanes) * V;
        if (chunk >= B.chunks || c >= B.dim) continue;
        const uint32_t from = chunk * B.chunk, to = min(B.n, from + B.chunk);
        uint32_t cur = entry_at(B, from);
        bool before = from > 0 && entry_at(B, from - 1) == cur;
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        auto flush = [&](bool after) {
            if (cur >= B.entries) return;
            if (before || after) {
                float* p = B.part + ((uint64_t)chunk * 2 + !before) * B.dim;
                store_pack<float, true>(p, 1, c, B.dim, *(const float(*)[4])&acc[0]);
                if constexpr (V == 8)
                    if (c + 4 < B.dim) store_pack<float, true>(p, 1, c + 4, B.dim, *(const float(*)[4])&acc[4]);
            } else {
                O* o = out + (uint64_t)cur * B.dim;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (c + v < B.dim) o[c + v] = from_f32<O>(acc[v] * B.scale);
            }
        };
        for (uint32_t i = from; i < to; ++i) {
            const u64 key = B.sorted[i];
            const uint32_t e = (uint32_t)(key >> 32);
            if (e != cur) {
                flush(false);
                before = false;
                cur = e;
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] = 0.0f;
            }
            if (e >= B.entries) break;   // (sorted behind all)
            float x[V];
            load_pack<T, kUnit>(grad + (int64_t)((uint32_t)key / B.list) * rs, cs, c, B.dim, 0.0f, x);
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] += x[v];
        }
        flush(to < B.n && entry_at(B, to) == cur);
    }
}

// Runs of several chunks, by the workgroup of the chunk in which they begin; and the entries that do not occur.
constexpr uint32_t kJoinWaves = 4;
template <class O>
__global__ __launch_bounds__(256) void table_join_kernel(Table B, const uint8_t* __restrict__ mark, uint32_t join_blocks,
                                                         O* __restrict__ out) {
    if (blockIdx.x >= join_blocks) {
        const uint64_t all = (uint64_t)B.entries * B.dim, step = (uint64_t)(gridDim.x - join_blocks) * 256;
        for (uint64_t i = (uint64_t)(blockIdx.x - join_blocks) * 256 + threadIdx.x; i < all; i += step)
            if (!mark || !mark[i / B.dim]) out[i] = from_f32<O>(0.0f);
        return;
    }
    __shared__ uint32_t last;
    __shared__ float sum[kJoinWaves][64];
    const uint32_t wave = threadIdx.x / 64, lane = lane_id();
    for (uint32_t chunk = blockIdx.x; chunk + 1 < B.chunks; chunk += join_blocks) {
        const uint32_t from = chunk * B.chunk, next = from + B.chunk, e = entry_at(B, next - 1);
        if (e >= B.entries || entry_at(B, next) != e) continue;
        if (from > 0 && entry_at(B, from) == e && entry_at(B, from - 1) == e) continue;   // began before
        // the last chunk that the run reaches
        __syncthreads();
        if (threadIdx.x == 0) last = B.chunks - 1;
        __syncthreads();
        for (uint32_t c0 = chunk + 1;; c0 += 256) {
            const uint32_t c = c0 + threadIdx.x;
            const bool ends = c < B.chunks && (c == B.chunks - 1 || entry_at(B, (c + 1) * B.chunk) != e);
            if (ends) atomicMin(&last, c);
            if (__syncthreads_or(ends) || c0 + 256 >= B.chunks) break;
        }
        __syncthreads();
        const uint32_t upto = last, count = upto - chunk;   // chunks behind the first
        const uint32_t each = (count + kJoinWaves - 1) / kJoinWaves;
        const uint32_t a = chunk + 1 + min(count, wave * each), b = min(upto + 1, a + each);
        for (uint32_t c0 = 0; c0 < B.dim; c0 += 64) {
            const uint32_t c = c0 + lane;
            float s = 0.0f;
            if (c < B.dim) {
                if (wave == 0) s = B.part[((uint64_t)chunk * 2 + 1) * B.dim + c];
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

// ---- host -----------------------------------------------------------------------------------
struct Layout {
    uint32_t n, passes, bits, blocks, chunk, chunks;
    uint64_t keys, counts, totals, mark, part, bytes;   // offsets; keys: two arrays
};
Layout layout(uint64_t rows, uint32_t list, uint32_t entries, uint32_t dim) {
    Layout L{};
    L.n = (uint32_t)(rows * list);
    uint32_t bits = 1;
    while (entries >> bits) ++bits;   // keys are 0 .. entries
    L.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    L.bits = (bits + L.passes - 1) / L.passes;
    L.blocks = (L.n + kSortKeys - 1) / kSortKeys;
    L.chunk = L.n <= 1u << 14 ? 16 : L.n <= 1u << 18 ? 32 : 64;
    L.chunks = (L.n + L.chunk - 1) / L.chunk;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t p = at;
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    L.keys = take(16 * (uint64_t)L.n);
    L.counts = take(4ull * L.blocks << L.bits);
    L.totals = take(4ull << L.bits);
    L.mark = take(entries);
    L.part = take(8ull * L.chunks * dim);
    L.bytes = at;
    return L;
}

template <class T, class O>
int launch_sums(const void* grad, int64_t rs, int64_t cs, const Table& B, const uint8_t* mark, void* out, hipStream_t st) {
    constexpr uint32_t V = Pack<T>::V;
    uint32_t lanes = 1;
    while (lanes < 64 && lanes * V < B.dim) lanes *= 2;
    const uint32_t tiles = (B.dim + lanes * V - 1) / (lanes * V), per = 256 / lanes;
    if (B.chunks) {
        const unsigned grid = row_grid(((uint64_t)B.chunks + per - 1) / per * tiles);
        if (cs == 1) table_sum_kernel<T, O, true><<<grid, 256, 0, st>>>((const T*)grad, rs, cs, B, lanes, (O*)out);
        else table_sum_kernel<T, O, false><<<grid, 256, 0, st>>>((const T*)grad, rs, cs, B, lanes, (O*)out);
        CLS_TRY(hipGetLastError());
    }
    const uint32_t join = std::min<uint32_t>(B.chunks, 1u << 16);
    const uint32_t zero = (uint32_t)std::min<uint64_t>(((uint64_t)B.entries * B.dim + 1023) / 1024, 4096);
    table_join_kernel<O><<<join + zero, 256, 0, st>>>(B, mark, join, (O*)out);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}
template <class T>
int launch_sums(const void* grad, int64_t rs, int64_t cs, const Table& B, const uint8_t* mark, void* out, int32_t type,
                hipStream_t st) {
    switch (type) {
        case CBH_TYPE_F32: return launch_sums<T, float>(grad, rs, cs, B, mark, out, st);
        case CBH_TYPE_F16: return launch_sums<T, _Float16>(grad, rs, cs, B, mark, out, st);
        default: return launch_sums<T, bf16_t>(grad, rs, cs, B, mark, out, st);
    }
}

int sort_places(const int32_t* index, uint32_t entries, const Layout& L, char* ws, u64** sorted, hipStream_t st) {
    Sort S{L.n, entries, L.blocks, 1u << L.bits, 0, (int)L.bits};
    u64* a = (u64*)(ws + L.keys);
    u64* b = a + L.n;
    uint32_t *counts = (uint32_t*)(ws + L.counts), *totals = (uint32_t*)(ws + L.totals);
    uint8_t* mark = (uint8_t*)(ws + L.mark);
    const unsigned scan = (S.digits + 63) / 64;
    const void* in = index;
    for (uint32_t p = 0; p < L.passes; ++p) {
        S.shift = (int)(p * L.bits);
        const bool first = p == 0, last = p + 1 == L.passes;
        if (first) sort_count_kernel<true><<<L.blocks, 256, 0, st>>>(in, S, counts, mark);
        else sort_count_kernel<false><<<L.blocks, 256, 0, st>>>(in, S, counts, mark);
        CLS_TRY(hipGetLastError());
        sort_scan_kernel<<<scan, 256, 0, st>>>(S, counts, totals);
        CLS_TRY(hipGetLastError());
#define SCATTER(F, L_) sort_scatter_kernel<F, L_><<<L.blocks, 256, 0, st>>>(in, S, counts, totals, a, mark)
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
int run_lookup(const void* table, uint32_t entries, uint32_t dim, int64_t rs, int64_t cs, const int32_t* index, uint64_t rows,
               uint32_t list, double scale, void* out, hipStream_t st) {
    const uint32_t vecs = (dim + Pack<T>::V - 1) / Pack<T>::V;
    const unsigned grid = row_grid((rows * vecs + 255) / 256);
    if (cs == 1) lookup_kernel<T, true><<<grid, 256, 0, st>>>((const T*)table, entries, dim, rs, cs, index, rows, list, (float)scale, (T*)out, vecs);
    else lookup_kernel<T, false><<<grid, 256, 0, st>>>((const T*)table, entries, dim, rs, cs, index, rows, list, (float)scale, (T*)out, vecs);
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
#define RUN(T) run_lookup<T>(table, entries, dim, row_stride, column_stride, index, rows, list, scale, out, st)
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
    return layout(rows, list, entries, dim).bytes;
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
        const Layout L = layout(rows, list, entries, dim);
        if (L.bytes > workspace_bytes || !workspace || (uintptr_t)workspace % 16)
            return cbh_internal_fail(CBH_ERR_LENGTH_MISMATCH, "the workspace needs " + std::to_string(L.bytes) +
                                                                  " bytes, aligned to 16");
        hipStream_t st = (hipStream_t)stream;
        char* ws = (char*)workspace;
        u64* sorted = (u64*)(ws + L.keys);
        if (L.n) {
            rc = sort_places(index, entries, L, ws, &sorted, st);
            if (rc != CBH_OK) return rc;
        }
        const Table B{sorted, L.n, entries, dim, list, L.chunk, L.chunks, (float)scale, (float*)(ws + L.part)};
        const uint8_t* mark = L.n ? (const uint8_t*)(ws + L.mark) : nullptr;   // (no rows: no entry occurs)
        switch (type) {
            case CBH_TYPE_F32: return launch_sums<float>(grad, row_stride, column_stride, B, mark, table_grad, grad_type, st);
            case CBH_TYPE_F16: return launch_sums<_Float16>(grad, row_stride, column_stride, B, mark, table_grad, grad_type, st);
            default: return launch_sums<bf16_t>(grad, row_stride, column_stride, B, mark, table_grad, grad_type, st);
        }
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}
