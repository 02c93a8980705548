// Log probabilities of short rows: up to 64 classes by a thread a row, up to 2048 in the registers of a
// wave's lanes or of some of them.  A row is read once, its maximum is known before its exponentials.
//
// 1M x 10 f32 class-major, one entry, k 3: 30 us, 88 MB at 2.9 TB/s.  Without a k 16 us, near the memory's rate: what a k adds is the
// comparisons of all pairs, a choice among all classes and an f64 log probability for each place, and stores of 4 bytes, 4 k apart.
// 20000 x 1000 f32 without a k 19 us, k 5 42; 35431 x 70 bf16 13, k 5 30: the call itself costs 13.  With a k bound by vector
// instructions: the descent over the keys' bits, and the ranking.
#include "class_logprobs.hpp"

namespace {
using namespace cbh::cls;

// Few classes: a row a thread, its scores in registers.  Up to 32: a score's place is the count of those ahead; up to 64, for which
// there are too many pairs (rows next to each other): the largest one after another.
template <class T, int NMAX, bool kWhole, bool kTop>
__global__ __launch_bounds__(256) void logprobs_few_kernel(Rows<T> X, Asked A) {
    constexpr bool kEach = NMAX <= 8;   // (so few classes: the log probability of each, once)
    const uint32_t n = X.classes;
    for (uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x; row < X.rows; row += (uint64_t)gridDim.x * 256) {
        const T* x0 = X.data + (int64_t)row * X.rs;
        const uint32_t* words = A.allowed + (int64_t)row * A.allowed_stride;
        const uint32_t low = A.allowed ? words[0] : ~0u, high = NMAX > 32 && A.allowed && n > 32 ? words[1] : ~0u;
        uint32_t own = ~0u;
        if constexpr (!kEach) own = given_class<T>(A, row, 0);
        const float own_score = given_score(A, X, row, own);
        float x[NMAX];
        RunningStat run;
        load_few<T, NMAX, kWhole>(x0, X.cs, n, x);
#pragma unroll
        for (int i = 0; i < NMAX; ++i) x[i] = (i < 32 ? low : high) >> (i & 31) & 1 ? x[i] : -INFINITY;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) run.m = fmaxf(run.m, x[i]);
#pragma unroll
        for (int i = 0; i < NMAX; ++i) run.add_one(x[i], A.c);
        const RowStat q = row_stat(run);
        write_stats(A, row, run, q);
        if constexpr (!kEach) {
            write_given(A, X, row, q, 0, 1, own, own_score);
        } else if (A.logprob) {   // four indices on their way at a time
            float lp[NMAX];
#pragma unroll
            for (int i = 0; i < NMAX; ++i) lp[i] = log_prob(x[i], q, A.it);
            for (uint32_t i0 = 0; i0 < A.n_given; i0 += 4) {
                uint32_t j[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) j[u] = given_class<T>(A, row, i0 + u);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (i0 + u >= A.n_given) break;
                    float y = 0.0f;
#pragma unroll
                    for (int i = 0; i < NMAX; ++i) y = j[u] == (uint32_t)i ? lp[i] : y;
                    A.logprob[row * A.n_given + i0 + u] = j[u] >= n ? 0.0f : y;
                }
            }
        }
        if constexpr (kTop && NMAX > 32) {
            uint32_t key[NMAX];
#pragma unroll
            for (int i = 0; i < NMAX; ++i) key[i] = (uint32_t)i < n ? order_key(x[i]) : 0;
            for (uint32_t r = 0; r < A.k; ++r) {
                uint32_t most = 0;
                int32_t at = 0;
#pragma unroll
                for (int i = 0; i < NMAX; ++i) {
                    at = key[i] > most ? i : at;
                    most = max(key[i], most);
                }
#pragma unroll
                for (int i = 0; i < NMAX; ++i) key[i] = i == at ? 0 : key[i];
                const float y = key_score(most);
                A.top_logprob[row * A.k + r] = log_prob(y, q, A.it);
                A.top_index[row * A.k + r] = y == -INFINITY ? -1 : at;
            }
        } else if constexpr (kTop) {
            uint32_t key[NMAX], rank[NMAX];
#pragma unroll
            for (int i = 0; i < NMAX; ++i) {
                key[i] = (uint32_t)i < n ? order_key(x[i]) : 0;
                rank[i] = 0;
            }
#pragma unroll
            for (int i = 0; i < NMAX; ++i)
#pragma unroll
                for (int j = 0; j < i; ++j) {
                    const bool ahead = key[j] >= key[i];
                    rank[i] += ahead;
                    rank[j] += !ahead;
                }
            for (uint32_t r = 0; r < A.k; ++r) {
                float y = 0.0f;
                int32_t at = -1;
#pragma unroll
                for (int i = 0; i < NMAX; ++i) {
                    y = rank[i] == r ? x[i] : y;
                    at = rank[i] == r ? i : at;
                }
                A.top_logprob[row * A.k + r] = log_prob(y, q, A.it);
                A.top_index[row * A.k + r] = y == -INFINITY ? -1 : at;
            }
        }
    }
}

// The largest bound that k of a wave's keys reach, the highest bits first, from the one in which they differ on (0: no key; at least k
// are not 0); it may end below the k-th largest where exactly k are at the bound or above.
template <int N>
__device__ __forceinline__ uint32_t wave_kth(const uint32_t (&key)[N], uint32_t k) {
    uint32_t hi = key[0], lo = key[0] - 1;   // (0 is no key: the largest here)
#pragma unroll
    for (int r = 1; r < N; ++r) {
        hi = max(hi, key[r]);
        lo = min(lo, key[r] - 1);
    }
    hi = wave_reduce(hi, MaxU());
    lo = ~wave_reduce(~lo, MaxU()) + 1;
    const int bits = hi > lo ? 32 - __builtin_clz(hi ^ lo) : 0;
    uint32_t bound = bits == 32 ? 0 : hi >> bits << bits;
    for (int b = bits - 1; b >= 0; --b) {
        const uint32_t t = bound | 1u << b;
        uint32_t c = 0;
#pragma unroll
        for (int r = 0; r < N; ++r) c += (uint32_t)__popcll(__ballot(key[r] >= t));
        if (c >= k) bound = t;
        if (c == k) break;
    }
    return bound;
}

// Rows of up to 2048 classes in the registers of G lanes, 64 for the largest classes.  Those: the k-th largest of the vectors'
// maxima, where there are at least 4 k, is a bound that k classes reach, else that of all classes; those that reach it are
// listed in LDS and take the places that the count of larger ones gives.
template <class T, int G, int R, bool kVec, int CAP>
__global__ __launch_bounds__(256) void logprobs_short_kernel(Rows<T> X, Asked A) {
    constexpr int V = kWide<T, kVec>;
    __shared__ u64 cand[4][CAP ? CAP : 1];
    const uint32_t l = threadIdx.x % G, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), n = X.classes;
    for (uint64_t first = (uint64_t)blockIdx.x * (256 / G); first < X.rows; first += (uint64_t)gridDim.x * (256 / G)) {
        const uint64_t mine = first + threadIdx.x / G, row = min(mine, X.rows - 1);
        const bool there = mine < X.rows;   // (the same in a wave where G = 64)
        const uint32_t* words = A.allowed ? A.allowed + (int64_t)row * A.allowed_stride : nullptr;
        float x[R][V], lm = -INFINITY, se = 0.0f, sy = 0.0f;
        load_short<T, G, R, kVec>(X.data + (int64_t)row * X.rs, X.cs, l, n, words, x);
        const uint32_t own = given_class<T>(A, row, l);
        const float own_score = given_score(A, X, row, own);
#pragma unroll
        for (int u = 0; u < R; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) lm = fmaxf(lm, x[u][v]);
        RunningStat run;
        run.m = fmaxf(kLowest, group_reduce<G>(lm, MaxF()));
#pragma unroll
        for (int u = 0; u < R; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float e, ey;
                run.weigh(x[u][v], A.c, e, ey);
                se += e;
                sy += ey;
            }
        run.s = group_reduce<G>((double)se, Add());
        run.t = group_reduce<G>((double)sy, Add());
        const RowStat q = row_stat(run);
        if (there && l == 0) write_stats(A, row, run, q);
        if (there) write_given(A, X, row, q, l, G, own, own_score);
        if constexpr (CAP > 0) {
            static_assert(G == 64, "a row a wave");
            if (!there) continue;
            float bound;   // k classes reach it (NaN: all do)
            if (kVec && A.k <= 8 && n >= 32 * V) {   // of the lanes' maxima, a NaN left out: the smallest of the k largest
                uint32_t larger = 0;
#pragma unroll 16
                for (int j = 0; j < 64; ++j) larger += read_lane(lm, j) > lm;
                bound = -wave_reduce(larger < A.k ? -lm : -INFINITY, MaxF());
            } else {
                uint32_t key[R * V], most[R];
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    most[u] = 0;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        key[u * V + v] = (u * G + l) * V + v < n ? order_key(x[u][v]) : 0;
                        most[u] = max(most[u], key[u * V + v]);
                    }
                }
                bound = key_score(A.k * 4 <= n / V ? wave_kth(most, A.k) : wave_kth(key, A.k));
            }
            uint32_t count = 0;
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const uint32_t i = (u * G + l) * V + v;
                    const bool in = i < n && !(x[u][v] < bound);
                    const u64 b = __ballot(in);
                    if (b == 0) continue;
                    const uint32_t at = count + (uint32_t)__popcll(b & ((1ull << l) - 1));
                    if (in && at < (uint32_t)CAP) cand[wave][at] = rank_key(x[u][v], i);
                    count += (uint32_t)__popcll(b);
                }
            if (count > (uint32_t)CAP) {   // many equal ones: class by class, and only the k largest kept as the list fills
                Candidates<CAP> C{cand[wave], 0, 0, key_score(0)};
                wave_fence();
#pragma unroll 1
                for (uint32_t i0 = 0; i0 < n; i0 += 64) {
                    const uint32_t i = i0 + l;
                    float y = -INFINITY;
                    if (i < n && !(words && !is_allowed(words, i))) y = to_f32(X.data[(int64_t)row * X.rs + (int64_t)i * X.cs]);
                    C.offer(y, i, i < n, A.k);
                }
                count = C.count;
            }
            wave_fence();
            for (uint32_t i = l; i < count; i += 64) {
                const u64 key = cand[wave][i];
                uint32_t rank = 0;
                for (uint32_t j = 0; j < count; ++j) rank += cand[wave][j] > key;
                if (rank >= A.k) continue;
                const float y = key_score((uint32_t)(key >> 32));
                A.top_logprob[row * A.k + rank] = log_prob(y, q, A.it);
                A.top_index[row * A.k + rank] = y == -INFINITY ? -1 : (int32_t)~(uint32_t)key;
            }
            wave_fence();
        }
    }
}
template <class T, int G, int R, bool kVec>
void launch_short(const Rows<T>& X, const Asked& A, hipStream_t st) {
    const unsigned grid = row_grid((X.rows + 256 / G - 1) / (256 / G));
    if constexpr (G == 64) {
        if (A.k) {
            if (A.k <= 128) logprobs_short_kernel<T, G, R, kVec, 256><<<grid, 256, 0, st>>>(X, A);
            else logprobs_short_kernel<T, G, R, kVec, 1152><<<grid, 256, 0, st>>>(X, A);
            return;
        }
    }
    logprobs_short_kernel<T, G, R, kVec, 0><<<grid, 256, 0, st>>>(X, A);
}
template <class T>
int run_short(const Rows<T>& X, const Asked& A, hipStream_t st) {
    constexpr uint32_t V = Pack<T>::V;
    const uint32_t n = X.classes;
    // by vectors where they fill the lanes: half of them, or a part of the wave's for the sums alone
    if (X.cs == 1 && (n > 32 * V || !A.k)) {
        constexpr uint32_t least = 32 / V;   // (lanes: from 17 classes on)
        if (n <= least * V) launch_short<T, (int)least, 1, true>(X, A, st);
        else if (n <= 8 * V) launch_short<T, 8, 1, true>(X, A, st);
        else if (n <= 16 * V) launch_short<T, 16, 1, true>(X, A, st);
        else if (n <= 32 * V) launch_short<T, 32, 1, true>(X, A, st);
        else if (n <= 64 * V) launch_short<T, 64, 1, true>(X, A, st);
        else if (n <= 128 * V) launch_short<T, 64, 2, true>(X, A, st);
        else if (n <= 256 * V) launch_short<T, 64, 4, true>(X, A, st);
        else launch_short<T, 64, 32 / V, true>(X, A, st);
    } else {
        if (n <= 64) launch_short<T, 64, 1, false>(X, A, st);
        else if (n <= 128) launch_short<T, 64, 2, false>(X, A, st);
        else if (n <= 256) launch_short<T, 64, 4, false>(X, A, st);
        else if (n <= 512) launch_short<T, 64, 8, false>(X, A, st);
        else launch_short<T, 64, 32, false>(X, A, st);
    }
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

}  // namespace

namespace cbh {
namespace cls {
template <class T>
int run_short_rows(const Rows<T>& X, const Asked& A, hipStream_t st) {
    const uint32_t n = X.classes;
    const uint64_t rows = X.rows;
    const int64_t rs = X.rs, cs = X.cs;
    // (by rows and without a k, from 17 classes on a group of lanes reads them better)
    if (n <= 64 && (n <= 32 || (rs == 1 && cs != 1)) && !(cs == 1 && n > 16 && !A.k)) {
        const unsigned grid = row_grid((rows + 255) / 256);
#define FEW_(N, UNIT) (A.k ? logprobs_few_kernel<T, N, UNIT, true><<<grid, 256, 0, st>>>(X, A) \
                           : logprobs_few_kernel<T, N, UNIT, false><<<grid, 256, 0, st>>>(X, A))
#define FEW(N) (cs == 1 && n % Pack<T>::V == 0 ? FEW_(N, true) : FEW_(N, false))
        if (n <= 4) FEW(4);
        else if (n <= 8) FEW(8);
        else if (n <= 12) FEW(12);
        else if (n <= 16) FEW(16);
        else if (n <= 32) FEW(32);
        else FEW_(64, false);
#undef FEW
#undef FEW_
        CLS_TRY(hipGetLastError());
        return CBH_OK;
    }
    return run_short(X, A, st);
}
template int run_short_rows(const Rows<float>&, const Asked&, hipStream_t);
template int run_short_rows(const Rows<_Float16>&, const Asked&, hipStream_t);
template int run_short_rows(const Rows<bf16_t>&, const Asked&, hipStream_t);
}  // namespace cls
}  // namespace cbh
