// Top classes: the k largest scores of a row, ties to the lowest class, and the row's
// log-sum-exp at a temperature, in one pass over the scores.
//
//   values[r][i], index[r][i]   the i-th largest score of row r and its class
//   lse[r] = log sum_j exp(x_rj / temperature)
//
// What has to be read is the scores; a row's candidates live in LDS.  A wave keeps those of its
// scores that can still be among the k largest (`Candidates`); a score is compared with the bound as an
// f32 in a register, so that most scores cost one comparison beside the log-sum-exp's
// subtraction, exponential and sum.
#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

constexpr uint32_t kMaxTop = 1024;
constexpr int kUnroll = 4;   // 16-byte loads a thread has in flight

// One wave's candidates, CAP of them in LDS: the keys above `bound` that it has met.  Full, the wave
// keeps the k largest and raises the bound to the smallest of them.
template <int CAP>
struct Candidates {
    u64* keys;
    uint32_t count;   // wave-uniform
    u64 bound;        // keys at or below it are not among the k largest
    float fbound;     // no score below it passes (NaN: all pass)
    __device__ __forceinline__ void set_bound(u64 b) {
        if (b > bound) {
            bound = b;
            fbound = key_score((uint32_t)(b >> 32));
        }
    }
    __device__ __forceinline__ void compact(uint32_t k) {
        constexpr int R = CAP / 64;
        wave_fence();
        const uint32_t l = lane_id();
        u64 key[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t i = r * 64 + l;
            key[r] = i < count ? keys[i] : 0;
        }
        u64 kth = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const u64 t = kth | (1ull << bit);
            uint32_t c = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) c += (uint32_t)__popcll(__ballot(key[r] >= t));
            if (c >= k) kth = t;
            if (c == k) break;
        }
        uint32_t kept = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const u64 b = __ballot(key[r] >= kth);
            if (key[r] >= kth) keys[kept + (uint32_t)__popcll(b & ((1ull << l) - 1))] = key[r];
            kept += (uint32_t)__popcll(b);
        }
        count = kept;
        wave_fence();
        set_bound(kth - 1);   // (the smallest kept key is in; a key equal to it does not come again)
    }
    // x: this lane's score of class cls, or no score
    __device__ __forceinline__ void offer(float x, uint32_t cls, bool have, uint32_t k) {
        const u64 key = rank_key(x, cls);
        bool in = have && key > bound;
        u64 b = __ballot(in);
        if (!b) return;
        if (count + (uint32_t)__popcll(b) > (uint32_t)CAP) {
            compact(k);
            in = in && key > bound;
            b = __ballot(in);
        }
        if (in) keys[count + (uint32_t)__popcll(b & ((1ull << lane_id()) - 1))] = key;
        count += (uint32_t)__popcll(b);
    }
};

// A row's log-sum-exp from its (m, s).  A row of +inf has NaN in s (+inf - +inf), as one of NaN; which it is is known when the
// row's largest are ranked: a NaN is among them, and its thread then writes NaN in place of +inf.  (The
// log-sum-exp is written first and its registers are free from there: written last, by the thread that knows the
// largest, it took top_groups_kernel to 97 registers and a wave a SIMD less, 167 against 155 us.)
__device__ __forceinline__ float row_lse(float m, double s, double inv_t) {
    return m == INFINITY ? INFINITY : (float)((double)m * inv_t + log(s));
}
// The `got` keys of best, the largest first, and NaN to lse if there is one.
template <int THREADS>
__device__ __forceinline__ void write_ranked(const u64* best, uint32_t got, float* values, int32_t* index, float* lse) {
    for (uint32_t i = threadIdx.x; i < got; i += THREADS) {
        const u64 key = best[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < got; ++j) rank += best[j] > key;
        const float x = key_score((uint32_t)(key >> 32));
        values[rank] = x;
        index[rank] = (int32_t)~(uint32_t)key;
        if (x != x) *lse = x;
    }
}

// Short rows, and a k that is large beside the row: candidates are taken in the pass itself (4 x 1000 f32, k 5:
// 6.8 us, latency).
// A workgroup takes a row, or one of the `parts` segments of `seg` classes of a row (few rows of many
// classes), whose k largest keys and (m, s) go to the workspace for merge_kernel.
template <class T, bool kUnit, int THREADS, int CAP>
__global__ __launch_bounds__(THREADS) void top_kernel(Rows<T> X, uint32_t k, float c, double inv_t, uint32_t parts,
                                                      uint32_t seg, float* __restrict__ values,
                                                      int32_t* __restrict__ index, float* __restrict__ lse,
                                                      u64* __restrict__ part_keys, PartSum* __restrict__ part_ms) {
    constexpr int V = Pack<T>::V, W = THREADS / 64, KMAX = CAP / 2;
    constexpr uint32_t kTile = THREADS * V * kUnroll;
    __shared__ u64 cand[W][CAP];
    __shared__ u64 best[KMAX];
    __shared__ uint32_t vmax[THREADS * kUnroll];
    __shared__ CountLds lds;
    __shared__ uint32_t counts[W], nbest;
    __shared__ float tmp_f[W];
    __shared__ double tmp_d[W];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    auto cand_at = [&](uint32_t i) -> u64 { return i % CAP < counts[i / CAP] ? cand[i / CAP][i % CAP] : 0; };

    for (uint64_t job = blockIdx.x; job < X.rows * parts; job += gridDim.x) {
        const uint64_t row = job / parts;
        const uint32_t first = (uint32_t)(job % parts) * seg, n = min(X.classes - first, seg);
        const T* x0 = X.data + (int64_t)row * X.rs + (int64_t)first * X.cs;
        Candidates<CAP> C{cand[wave], 0, 0, key_score(0)};
        Running run;
        for (uint32_t base = 0; base < n; base += kTile) {
            float x[kUnroll][V];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                load_pack<T, kUnit>(x0, X.cs, base + (u * THREADS + threadIdx.x) * V, n, -INFINITY, x[u]);
            float vm[kUnroll], tm = -INFINITY;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                vm[u] = x[u][0];
#pragma unroll
                for (int v = 1; v < V; ++v) vm[u] = fmaxf(vm[u], x[u][v]);
                tm = fmaxf(tm, vm[u]);
            }
            run.raise(tm, c);
            run.add(x, c);
            if (base == 0) {
                // the first bound: k of the tile's vectors hold a score that reaches the k-th largest of
                // their maxima
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const uint32_t i = (u * THREADS + threadIdx.x);
                    vmax[i] = i * V < n ? order_key(vm[u]) : 0;
                }
                __syncthreads();
                const uint32_t vecs = min((uint32_t)(THREADS * kUnroll), (n + V - 1) / V);
                if (k <= vecs)
                    C.set_bound(kth_of<THREADS>([&](uint32_t i) { return (u64)vmax[i]; }, vecs, k, &lds) << 32);
            } else if (base == kTile || base == 3 * kTile) {
                // the candidates of the first tiles give a better one
                if ((threadIdx.x & 63) == 0) counts[wave] = C.count;
                __syncthreads();
                uint32_t total = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) total += counts[w];
                if (total >= k) {
                    const u64 kth = kth_of<THREADS>(cand_at, W * CAP, k, &lds);
                    C.set_bound(kth - 1);
                }
                __syncthreads();
            }
            // vectors that hold a score at the bound or above (NaN: somewhere in this thread's scores) are
            // read again, score by score
            uint32_t vecs = 0;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) vecs |= (uint32_t)!(vm[u] < C.fbound) << u;
            if (run.s != run.s) vecs = (1u << kUnroll) - 1;
            while (__any(vecs != 0)) {
                const uint32_t u = vecs ? (uint32_t)__builtin_ctz(vecs) : 0;
                const uint32_t i0 = base + (u * THREADS + threadIdx.x) * V;
                float y[V];
                load_pack<T, kUnit>(x0, X.cs, i0, vecs ? n : 0, -INFINITY, y);
                uint32_t hits = 0;
#pragma unroll
                for (int v = 0; v < V; ++v) hits |= (uint32_t)(i0 + v < n && !(y[v] < C.fbound)) << v;
                if (!vecs) hits = 0;
                while (__any(hits != 0)) {
                    const uint32_t v = hits ? (uint32_t)__builtin_ctz(hits) : 0;
                    float z = y[0];
#pragma unroll
                    for (int q = 1; q < V; ++q) z = v == (uint32_t)q ? y[q] : z;
                    C.offer(z, first + i0 + v, hits != 0, k);
                    hits &= hits - 1;
                }
                vecs &= vecs - 1;
            }
        }
        if ((threadIdx.x & 63) == 0) counts[wave] = C.count;
        if (threadIdx.x == 0) nbest = 0;
        float m;
        double s;
        __syncthreads();
        block_running<THREADS>(run, c, m, s, tmp_f, tmp_d);
        if (threadIdx.x == 0) {
            if (parts == 1) lse[row] = row_lse(m, s, inv_t);
            else part_ms[job] = PartSum{s, m};
        }
        uint32_t total = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) total += counts[w];
        u64 kth = 1;
        if (total > k) kth = kth_of<THREADS>(cand_at, W * CAP, k, &lds);
        for (uint32_t i = threadIdx.x; i < W * CAP; i += THREADS) {
            const u64 key = cand_at(i);
            if (key >= kth) best[atomicAdd(&nbest, 1u)] = key;
        }
        __syncthreads();
        const uint32_t got = nbest;   // k, or all of a segment of fewer
        if (parts == 1)
            write_ranked<THREADS>(best, got, values + row * k, index + row * k, lse + row);
        else
            for (uint32_t i = threadIdx.x; i < k; i += THREADS) part_keys[job * k + i] = i < got ? best[i] : 0;
        __syncthreads();
    }
}

// Long rows and a k that is small beside them.  The pass over the scores takes nothing but the log-sum-exp
// and the largest of every group of 32 classes, kept in LDS.  The k-th largest of those maxima is a bound that at least k scores reach and hardly more (a k of a
// quarter of the groups: 1.15 k of normal scores); the groups that reach it, which the caches still hold for the
// most part, are read again and offered to the candidates.
// 4096 x 65536 bf16, k 64: 159 us, 537 MB at 3.4 TB/s (a copy: 5.2); 777 x 50021 f32, k 20: 38 us, 155 MB at
// 4.1 TB/s.  Bound by the vector instructions of the pass (8.5 a score, 4 of them the exponential's quarter rate: 58
// us of the first case) and by the row's end, barriers and LDS that four workgroups a CU hide in part.  With
// candidates taken in the pass itself (top_kernel) the cases took 285 and 48 us.
constexpr uint32_t kMaxGroupSegs = 64;
template <class T, bool kUnit, int THREADS, int CAP>
__global__ __launch_bounds__(THREADS) void top_groups_kernel(Rows<T> X, uint32_t k, float c, double inv_t,
                                                             uint32_t parts, uint32_t seg, float* __restrict__ values,
                                                             int32_t* __restrict__ index, float* __restrict__ lse,
                                                             u64* __restrict__ part_keys,
                                                             PartSum* __restrict__ part_ms) {
    constexpr int V = Pack<T>::V, U = kGroup / V, W = THREADS / 64, KMAX = CAP / 2;
    extern __shared__ uint32_t groups[];
    __shared__ u64 cand[W][CAP];
    __shared__ u64 best[KMAX];
    __shared__ CountLds lds;
    __shared__ uint32_t counts[W], nbest;
    __shared__ float tmp_f[W];
    __shared__ double tmp_d[W];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = lane_id();
    auto cand_at = [&](uint32_t i) -> u64 { return i % CAP < counts[i / CAP] ? cand[i / CAP][i % CAP] : 0; };

    for (uint64_t job = blockIdx.x; job < X.rows * parts; job += gridDim.x) {
        const uint64_t row = job / parts;
        const uint32_t first = (uint32_t)(job % parts) * seg, n = min(X.classes - first, seg);
        const T* x0 = X.data + (int64_t)row * X.rs + (int64_t)first * X.cs;
        const uint32_t n_segs = (n + kSeg - 1) / kSeg;
        Running run;
        for (uint32_t s = wave; s < n_segs; s += W) {
            float x[U][V], vm[U], gm = -INFINITY;
            load_tile<T, kUnit>(x0, X.cs, s * kSeg, n, -INFINITY, x);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int v = 0; v < V; ++v) vm[u] = v ? fmaxf(vm[u], x[u][v]) : x[u][v];
#pragma unroll
            for (int u = 0; u < U; ++u) gm = fmaxf(gm, vm[u]);
            run.raise(gm, c);
            run.add(x, c);
            const uint32_t g = s * 64 + group_of<V>(lane);
            uint32_t key = order_key(group_max<V>(vm, lane, MaxF()));
            if (__any(run.s != run.s)) {   // since a NaN, which is the largest of its group, or +inf
                uint32_t keys[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    keys[u] = 0;
#pragma unroll
                    for (int v = 0; v < V; ++v) keys[u] = max(keys[u], order_key(x[u][v]));
                }
                key = group_max<V>(keys, lane, MaxU());
            }
            groups[g] = g * kGroup < n ? key : 0;
        }
        __syncthreads();
        const uint32_t bound = (uint32_t)kth_of<THREADS>([&](uint32_t i) { return (u64)groups[i]; }, n_segs * 64, k, &lds);
        Candidates<CAP> C{cand[wave], 0, 0, key_score(0)};
        C.set_bound((u64)bound << 32);
        for (uint32_t s = wave; s < n_segs; s += W) {
            u64 hit = __ballot(groups[s * 64 + lane] >= bound);
            while (hit) {   // two groups at a time, a class a lane
                const uint32_t a = (uint32_t)__builtin_ctzll(hit);
                hit &= hit - 1;
                const uint32_t b = hit ? (uint32_t)__builtin_ctzll(hit) : 64;
                hit &= hit - 1;
                const uint32_t ln = lane < kGroup ? a : b, q = lane % kGroup;
                const uint32_t i = s * kSeg + ln * kGroup + q;
                const bool have = ln < 64 && i < n;
                const float x = have ? to_f32(x0[kUnit ? (int64_t)i : (int64_t)i * X.cs]) : -INFINITY;
                C.offer(x, first + i, have, k);
            }
        }
        if ((threadIdx.x & 63) == 0) counts[wave] = C.count;
        if (threadIdx.x == 0) nbest = 0;
        float m;
        double sum;
        __syncthreads();
        block_running<THREADS>(run, c, m, sum, tmp_f, tmp_d);
        if (threadIdx.x == 0) {
            if (parts == 1) lse[row] = row_lse(m, sum, inv_t);
            else part_ms[job] = PartSum{sum, m};
        }
        uint32_t total = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) total += counts[w];
        u64 kth = 1;
        if (total > k) kth = kth_of<THREADS>(cand_at, W * CAP, k, &lds);
        for (uint32_t i = threadIdx.x; i < W * CAP; i += THREADS) {
            const u64 key = cand_at(i);
            if (key >= kth) best[atomicAdd(&nbest, 1u)] = key;
        }
        __syncthreads();
        if (parts == 1)
            write_ranked<THREADS>(best, k, values + row * k, index + row * k, lse + row);
        else
            for (uint32_t i = threadIdx.x; i < k; i += THREADS) part_keys[job * k + i] = best[i];
        __syncthreads();
    }
}

// The segments of a row together.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void merge_kernel(const u64* __restrict__ part_keys,
                                                        const PartSum* __restrict__ part_ms, uint32_t parts, uint32_t k,
                                                        float c, double inv_t, float* __restrict__ values,
                                                        int32_t* __restrict__ index, float* __restrict__ lse) {
    __shared__ u64 best[kMaxTop];
    __shared__ CountLds lds;
    __shared__ uint32_t nbest;
    __shared__ float tmp_f[THREADS / 64];
    __shared__ double tmp_d[THREADS / 64];
    const uint64_t row = blockIdx.x;
    const u64* keys = part_keys + row * parts * k;
    if (threadIdx.x == 0) nbest = 0;
    Running run;
    for (uint32_t p = threadIdx.x; p < parts; p += THREADS) {
        const PartSum ms = part_ms[row * parts + p];
        run.join(ms.m, ms.s, c);
    }
    float m;
    double s;
    __syncthreads();
    block_running<THREADS>(run, c, m, s, tmp_f, tmp_d);
    if (threadIdx.x == 0) lse[row] = row_lse(m, s, inv_t);
    const u64 kth = kth_of<THREADS>([&](uint32_t i) { return keys[i]; }, parts * k, k, &lds);
    for (uint32_t i = threadIdx.x; i < parts * k; i += THREADS) {
        const u64 key = keys[i];
        if (key != 0 && key >= kth) best[atomicAdd(&nbest, 1u)] = key;
    }
    __syncthreads();
    write_ranked<THREADS>(best, k, values + row * k, index + row * k, lse + row);
}

// Few classes: a row a thread, its scores in registers; a score's place is the count of those ahead.  1M x 10 f32, k 3: 35 us
// class-major, 36 by rows, 68 MB at 1.9 TB/s; 500k x 32, k 5: 67 and 77 us.  Bound by the comparisons of all pairs, whose masks
// do not fit the scalar registers (116 put aside at 16 places, 696 at 32), and by stores to scattered places.
template <class T, int NMAX>
__global__ __launch_bounds__(256) void top_few_kernel(Rows<T> X, uint32_t k, float c, double inv_t,
                                                      float* __restrict__ values, int32_t* __restrict__ index,
                                                      float* __restrict__ lse) {
    const uint32_t n = X.classes;
    for (uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x; row < X.rows; row += (uint64_t)gridDim.x * 256) {
        const T* x0 = X.data + (int64_t)row * X.rs;
        float x[NMAX];
        uint32_t key[NMAX], rank[NMAX];
        Running run;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) {
            x[i] = (uint32_t)i < n ? to_f32(x0[(int64_t)i * X.cs]) : -INFINITY;
            key[i] = (uint32_t)i < n ? order_key(x[i]) : 0;
            rank[i] = 0;
            run.m = fmaxf(run.m, x[i]);
        }
#pragma unroll
        for (int i = 0; i < NMAX; ++i) run.add_one(x[i], c);
        float z = row_lse(run.m, run.s, inv_t);
        if (run.m == INFINITY) {   // (beside a NaN: it)
#pragma unroll
            for (int i = 0; i < NMAX; ++i) z = x[i] != x[i] ? x[i] : z;
        }
        lse[row] = z;
#pragma unroll
        for (int i = 0; i < NMAX; ++i)
#pragma unroll
            for (int j = 0; j < i; ++j) {
                const bool ahead = key[j] >= key[i];
                rank[i] += ahead;
                rank[j] += !ahead;
            }
#pragma unroll
        for (int i = 0; i < NMAX; ++i)
            if ((uint32_t)i < n && rank[i] < k) {
                values[row * k + rank[i]] = key_score(key[i]);
                index[row * k + rank[i]] = i;
            }
    }
}

// Segments of a row: one, unless the rows alone leave CUs idle and a row is long.
constexpr uint32_t kMinSeg = 16384, kMaxSeg = kMaxGroupSegs * kSeg;
uint32_t plan_parts(uint64_t rows, uint32_t classes) {
    uint32_t parts = (classes + kMaxSeg - 1) / kMaxSeg;
    if (rows > 0 && rows < 512 && classes >= 2 * kMinSeg)
        parts = std::max(parts, (uint32_t)std::min<uint64_t>((512 + rows - 1) / rows, classes / kMinSeg));
    return parts;
}

template <class T, bool kUnit>
int launch_top(const Rows<T>& X, uint32_t k, double t, float* values, int32_t* index, float* lse, uint32_t parts,
               void* workspace, hipStream_t st) {
    const float c = (float)(1.4426950408889634 / t);
    const double it = 1.0 / t;
    const uint32_t n = X.classes;
    if (n <= 32) {
        const unsigned grid = row_grid((X.rows + 255) / 256);
        if (n <= 8) top_few_kernel<T, 8><<<grid, 256, 0, st>>>(X, k, c, it, values, index, lse);
        else if (n <= 16) top_few_kernel<T, 16><<<grid, 256, 0, st>>>(X, k, c, it, values, index, lse);
        else top_few_kernel<T, 32><<<grid, 256, 0, st>>>(X, k, c, it, values, index, lse);
        CLS_TRY(hipGetLastError());
        return CBH_OK;
    }
    const uint32_t seg = (n + parts - 1) / parts;
    u64* pk = (u64*)workspace;
    PartSum* pm = parts > 1 ? (PartSum*)(pk + X.rows * parts * k) : nullptr;
    const unsigned grid = row_grid(X.rows * parts);
    // by groups where k is at most a quarter of the shortest segment's
    const uint32_t shortest = n - seg * (parts - 1);
    if (n > 2048 && k * 4 <= shortest / kGroup && seg <= kMaxGroupSegs * kSeg) {
        const size_t lds = sizeof(uint32_t) * 64 * ((seg + kSeg - 1) / kSeg);
        if (k <= 128) top_groups_kernel<T, kUnit, 256, 256><<<grid, 256, lds, st>>>(X, k, c, it, parts, seg, values, index, lse, pk, pm);
        else top_groups_kernel<T, kUnit, 256, 2048><<<grid, 256, lds, st>>>(X, k, c, it, parts, seg, values, index, lse, pk, pm);
    } else
#define TOP(TH, CAP) top_kernel<T, kUnit, TH, CAP><<<grid, TH, 0, st>>>(X, k, c, it, parts, seg, values, index, lse, pk, pm)
    if (n <= 2048) {
        if (k <= 128) TOP(64, 256);
        else if (k <= 256) TOP(64, 512);
        else TOP(64, 2048);
    } else {
        if (k <= 128) TOP(256, 256);
        else if (k <= 256) TOP(256, 512);
        else TOP(256, 2048);
    }
#undef TOP
    CLS_TRY(hipGetLastError());
    if (parts > 1) {
        merge_kernel<256><<<(unsigned)X.rows, 256, 0, st>>>(pk, pm, parts, k, c, it, values, index, lse);
        CLS_TRY(hipGetLastError());
    }
    return CBH_OK;
}

template <class T>
int run_top(const void* scores, uint64_t rows, uint32_t classes, int64_t rs, int64_t cs, uint32_t k, double t,
            float* values, int32_t* index, float* lse, uint32_t parts, void* workspace, hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, classes, rs, cs};
    return cs == 1 ? launch_top<T, true>(X, k, t, values, index, lse, parts, workspace, st)
                   : launch_top<T, false>(X, k, t, values, index, lse, parts, workspace, st);
}

}  // namespace

extern "C" uint64_t cbh_top_classes_workspace(uint64_t rows, uint32_t classes, uint32_t k) {
    const uint32_t parts = plan_parts(rows, classes);
    return parts == 1 ? 0 : rows * parts * (8 * (uint64_t)k + sizeof(PartSum));
}

extern "C" int cbh_top_classes(const void* scores, int32_t type, uint64_t rows, uint32_t classes, int64_t row_stride,
                               int64_t class_stride, uint32_t k, double temperature, float* values, int32_t* index,
                               float* lse, void* workspace, uint64_t workspace_bytes, void* stream) {
    try {
        const int rc = check_scores(scores, type, rows, classes, row_stride, class_stride);
        if (rc != CBH_OK) return rc;
        if (k < 1 || k > classes || k > kMaxTop)
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "k must be in 1 .. min(classes, 1024)");
        if (!good_temperature(temperature))
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, kBadTemperature);
        if (rows == 0) return CBH_OK;
        if (!values || !index || !lse) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "outputs are null");
        const uint64_t need = cbh_top_classes_workspace(rows, classes, k);
        if (need > workspace_bytes || (need && (!workspace || (uintptr_t)workspace % 8)))
            return cbh_internal_fail(CBH_ERR_LENGTH_MISMATCH, "the workspace needs " + std::to_string(need) +
                                                                  " bytes, aligned to 8");
        const uint32_t parts = plan_parts(rows, classes);
        hipStream_t st = (hipStream_t)stream;
        switch (type) {
            case CBH_TYPE_F32:
                return run_top<float>(scores, rows, classes, row_stride, class_stride, k, temperature, values, index,
                                      lse, parts, workspace, st);
            case CBH_TYPE_F16:
                return run_top<_Float16>(scores, rows, classes, row_stride, class_stride, k, temperature, values,
                                         index, lse, parts, workspace, st);
            default:
                return run_top<bf16_t>(scores, rows, classes, row_stride, class_stride, k, temperature, values, index,
                                       lse, parts, workspace, st);
        }
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}
