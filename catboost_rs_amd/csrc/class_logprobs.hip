// Log probabilities of given classes, entropy and the most probable classes, in one pass over the
// scores; and the gradient of a function of them, in another.
//
// With d_j = (x_j - m) / t over the allowed classes, m the largest score:
//   Z = sum e^d_j,  E = -sum e^d_j d_j / Z,  logprob of c = d_c - log Z,  entropy = log Z + E
//   grad_j = (sum of g_i of j's entries - p_j (G + h (d_j + E))) / t,  p_j = e^d_j / Z,  G = sum of all g_i
// log Z and E are both at least 0: the entropy is no difference, and log p_j + entropy = d_j + E holds for
// a row of nearly equal scores too, where either is a small difference of large numbers.
#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

constexpr uint32_t kMaxTop = 1024, kMaxGiven = 1024;
constexpr double kLn2 = 0.6931471805599453;
constexpr float kFar = -200.0f;   // 2^y is 0 in f32 from -150 down: a y of less, -inf too, has no part in the sums

// The running sums of a softmax with those of its entropy: s = sum 2^y, t = sum 2^y y, y = (x - m) c.
struct RunningStat : Running {
    double t = 0.0;
    __device__ __forceinline__ void raise(float to, float c) {
        if (to > m) {
            const float y = fmaxf((m - to) * c, -1e30f);   // (finite: 0 times it is 0)
            const double f = (double)exp2_fast(y);
            t = f * (t + (double)y * s);
            s *= f;
            m = to;
        }
    }
    __device__ __forceinline__ void weigh(float x, float c, float& e, float& ey) const {
        const float y = (x - m) * c;
        e = exp2_fast(y);   // (NaN stays)
        ey = e * fmaxf(y, kFar);
    }
    // (sums of a tile side by side, then together, then in f64)
    template <int U, int V>
    __device__ __forceinline__ void add(const float (&x)[U][V], float c) {
        float e[V], ey[V];
#pragma unroll
        for (int v = 0; v < V; ++v) weigh(x[0][v], c, e[v], ey[v]);
#pragma unroll
        for (int u = 1; u < U; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float a, b;
                weigh(x[u][v], c, a, b);
                e[v] += a;
                ey[v] += b;
            }
#pragma unroll
        for (int o = V / 2; o > 0; o /= 2)
#pragma unroll
            for (int v = 0; v < o; ++v) {
                e[v] += e[v + o];
                ey[v] += ey[v + o];
            }
        s += (double)e[0];
        t += (double)ey[0];
    }
    __device__ __forceinline__ void add_one(float x, float c) {
        float e, ey;
        weigh(x, c, e, ey);
        s += (double)e;
        t += (double)ey;
    }
    __device__ __forceinline__ void join(float m2, double s2, double t2, float c) {
        raise(m2, c);
        const float y = fmaxf((m2 - m) * c, -1e30f);
        const double f = (double)exp2_fast(y);
        s += s2 * f;
        t += f * (t2 + (double)y * s2);
    }
};
struct PartStat {   // of a part of a row, between launches
    double s, t;
    float m, none;
};
// Those of a workgroup's threads together, in a fixed order; every thread gets them.  One barrier; tmp: one a wave.
template <int THREADS>
__device__ __forceinline__ void block_stat(RunningStat& r, float c, PartStat* tmp) {
    r.raise(wave_reduce(r.m, MaxF()), c);
    r.s = wave_reduce(r.s, Add());
    r.t = wave_reduce(r.t, Add());
    if (THREADS == 64) return;
    if (lane_id() == 0) tmp[threadIdx.x / 64] = PartStat{r.s, r.t, r.m, 0.0f};
    __syncthreads();
    r = RunningStat();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) r.join(tmp[w].m, tmp[w].s, tmp[w].t, c);
}

struct Asked {   // what is asked of every row, and where it goes
    const int32_t* given;
    const uint32_t* allowed;   // nullable
    int64_t allowed_stride;
    uint32_t n_given, k;
    float c;      // log2(e) / t
    double it;    // 1 / t
    float *logprob, *entropy, *stats, *top_logprob;
    int32_t* top_index;
};
__device__ __forceinline__ bool is_allowed(const uint32_t* words, uint32_t j) { return words[j >> 5] >> (j & 31) & 1; }

// A tile's scores, -inf where a class is not allowed; `words` are those from the tile's row segment on.
template <class T, bool kUnit, bool kMask>
__device__ __forceinline__ void load_allowed(const T* row, int64_t cs, const uint32_t* words, uint32_t base, uint32_t n,
                                             float (&x)[kPacks<T>][Pack<T>::V]) {
    constexpr int V = Pack<T>::V, U = kPacks<T>;
    const uint32_t lane = lane_id();
    uint32_t bits[U];
    if constexpr (kMask) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t i = base + (u * 64 + lane) * V;
            bits[u] = i < n ? words[i >> 5] >> (i & 31) : 0;
        }
    }
    load_tile<T, kUnit>(row, cs, base, n, -INFINITY, x);
    if constexpr (kMask) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) x[u][v] = bits[u] >> v & 1 ? x[u][v] : -INFINITY;
    }
}

// What is written of a row from its sums: the statistics by one thread, given classes by all.
struct RowStat {
    double m, log_z;   // (f64: logprob is rounded once)
    bool none;         // a row of -inf alone
};
__device__ __forceinline__ RowStat row_stat(const RunningStat& r) {
    RowStat q;
    q.none = r.s == 0.0;
    q.m = (double)r.m;
    q.log_z = q.none ? 0.0 : log(r.s);
    return q;
}
__device__ __forceinline__ float log_prob(float x, const RowStat& q, double it) {
    return x == -INFINITY && q.log_z == q.log_z ? x : (float)(((double)x - q.m) * it - q.log_z);
}
__device__ __forceinline__ void write_stats(const Asked& A, uint64_t row, const RunningStat& r, const RowStat& q) {
    const double e = q.none ? 0.0 : -r.t / r.s * kLn2, nan = r.s - r.s;   // (nan: 0 of a finite sum)
    if (A.entropy) A.entropy[row] = (float)(q.log_z + e);
    if (A.stats) {
        A.stats[row * 3] = q.none ? -INFINITY : (float)(q.m + nan);
        A.stats[row * 3 + 1] = q.none ? -INFINITY : (float)q.log_z;
        A.stats[row * 3 + 2] = (float)e;
    }
}
// The log probabilities of a row's entries from, from + step, ...; the first of them by a score that was read before.
template <class T>
__device__ __forceinline__ uint32_t given_class(const Asked& A, uint64_t row, uint32_t i) {
    return A.logprob && i < A.n_given ? (uint32_t)A.given[row * A.n_given + i] : ~0u;
}
template <class T>
__device__ __forceinline__ float given_score(const Asked& A, const Rows<T>& X, uint64_t row, uint32_t j) {
    if (j >= X.classes) return 0.0f;
    const float x = to_f32(X.data[(int64_t)row * X.rs + (int64_t)j * X.cs]);
    return A.allowed && !is_allowed(A.allowed + (int64_t)row * A.allowed_stride, j) ? -INFINITY : x;
}
template <class T>
__device__ __forceinline__ void write_given(const Asked& A, const Rows<T>& X, uint64_t row, const RowStat& q, uint32_t from,
                                            uint32_t step, uint32_t j, float x) {
    if (!A.logprob) return;
    for (uint32_t i = from; i < A.n_given; i += step) {
        if (i != from) {
            j = given_class<T>(A, row, i);
            x = given_score(A, X, row, j);
        }
        A.logprob[row * A.n_given + i] = j < X.classes ? log_prob(x, q, A.it) : 0.0f;
    }
}
// The k largest of the `got` keys of best (0: none), the largest first.
template <int THREADS>
__device__ __forceinline__ void write_top(const Asked& A, uint64_t row, const u64* best, uint32_t got, const RowStat& q) {
    for (uint32_t i = threadIdx.x; i < got; i += THREADS) {
        const u64 key = best[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < got; ++j) rank += best[j] > key;
        if (key == 0 || rank >= A.k) continue;
        const float x = key_score((uint32_t)(key >> 32));
        A.top_logprob[row * A.k + rank] = log_prob(x, q, A.it);
        A.top_index[row * A.k + rank] = x == -INFINITY ? -1 : (int32_t)~(uint32_t)key;
    }
}

// Keys of a segment that are kept beside its k largest: as many as reach the bound are mostly, and need no selection.
constexpr uint32_t kSpare = 64;
constexpr uint32_t kRanked = 384;   // keys of a row that are ranked among one another without a selection

// A workgroup takes a row, or one of the `parts` segments of a row (few rows of many classes).  Sums and k largest keys
// go to the workspace for finish_kernel, but for whole rows without the latter.  (With the epilogue in this kernel too, whose addresses and
// f64 values do not fit beside the selection's, it took 165 registers and 4096 x 8192 bf16, k 64: 108 us.)  How the largest are found:
//   kNone     k = 0
//   kGroups   a bound from the maxima of every 32 classes, kept in LDS; the groups that reach it are read again
//   kVectors  the same of every 4 or 8 classes, a vector
//   kWhole    digits of the keys of all classes, read again for every digit (a k that is large beside the row)
enum Select { kNone, kGroups, kVectors, kWhole };
template <class T, bool kUnit, bool kMask, int THREADS, Select kSel, int CAP>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(Rows<T> X, Asked A, uint32_t parts, uint32_t seg,
                                                           PartStat* __restrict__ part_stat, u64* __restrict__ part_keys) {
    constexpr int V = Pack<T>::V, U = kPacks<T>, W = THREADS / 64, KMAX = kSel == kWhole ? (int)kMaxTop : CAP / 2 + (int)kSpare;
    extern __shared__ uint32_t groups[];
    constexpr bool kBound = kSel == kGroups || kSel == kVectors;
    __shared__ u64 cand[kBound ? W : 1][kBound ? CAP : 1];
    __shared__ u64 best[kSel == kNone ? 1 : KMAX];
    __shared__ CountLds lds;
    __shared__ uint32_t counts[W], nbest;
    __shared__ PartStat tmp[W];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = lane_id();

    for (uint64_t job = blockIdx.x; job < X.rows * parts; job += gridDim.x) {
        const uint64_t row = job / parts;
        const uint32_t first = (uint32_t)(job % parts) * seg, n = min(X.classes - first, seg);
        const T* x0 = X.data + (int64_t)row * X.rs + (int64_t)first * X.cs;
        const uint32_t* words = kMask ? A.allowed + (int64_t)row * A.allowed_stride + first / 32 : nullptr;
        auto score = [&](uint32_t i) {
            const float x = to_f32(x0[kUnit ? (int64_t)i : (int64_t)i * X.cs]);
            return kMask && !is_allowed(words, i) ? -INFINITY : x;
        };
        auto vector_key = [&](uint32_t i) {   // the largest key of the classes from i on
            uint32_t key = 0;
            for (uint32_t j = i; j < min(i + V, n); ++j) key = max(key, order_key(score(j)));
            return key;
        };
        const uint32_t n_segs = (n + kSeg - 1) / kSeg;
        RunningStat run;
        uint32_t own = ~0u;
        if constexpr (kSel == kNone) own = parts == 1 ? given_class<T>(A, row, threadIdx.x) : ~0u;
        for (uint32_t s = wave; s < n_segs; s += W) {
            float x[U][V], vm[U], gm = -INFINITY;
            load_allowed<T, kUnit, kMask>(x0, X.cs, words, s * kSeg, n, x);
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int v = 0; v < V; ++v) vm[u] = v ? fmaxf(vm[u], x[u][v]) : x[u][v];
                gm = fmaxf(gm, vm[u]);
            }
            run.raise(gm, A.c);
            run.add(x, A.c);
            if constexpr (kSel == kGroups) {
                const uint32_t g = s * 64 + group_of<V>(lane);
                uint32_t key = order_key(group_max<V>(vm, lane, MaxF()));
                // since a NaN, which is the largest of its group, or +inf (the tile is read again: kept until here, its scores
                // took the kernel from 103 to 165 registers)
                if (__any(run.s != run.s)) {
                    uint32_t keys[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) keys[u] = vector_key(s * kSeg + (u * 64 + lane) * V);
                    key = group_max<V>(keys, lane, MaxU());
                }
                groups[g] = g * kGroup < n ? key : 0;
            } else if constexpr (kSel == kVectors) {
                const bool nan = __any(run.s != run.s);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t i = s * kSeg + (u * 64 + lane) * V;
                    groups[(s * U + u) * 64 + lane] = i >= n ? 0 : nan ? vector_key(i) : order_key(vm[u]);
                }
            }
        }
        if (kSel != kNone && threadIdx.x == 0) nbest = 0;
        if (kSel != kNone && THREADS == 64) __syncthreads();
        if (kSel == kNone && parts == 1) {
            const float own_score = given_score(A, X, row, own);
            block_stat<THREADS>(run, A.c, tmp);
            const RowStat q = row_stat(run);
            if (threadIdx.x == 0) write_stats(A, row, run, q);
            write_given(A, X, row, q, threadIdx.x, THREADS, own, own_score);
        } else {
            block_stat<THREADS>(run, A.c, tmp);
            if (threadIdx.x == 0) part_stat[job] = PartStat{run.s, run.t, run.m, 0.0f};
        }
        if constexpr (kBound) {
            const uint32_t n_groups = n_segs * (kSel == kGroups ? 64 : 64 * U);
            const uint32_t bound = (uint32_t)kth_of<THREADS>([&](uint32_t i) { return (u64)groups[i]; }, n_groups, A.k, &lds);
            Candidates<CAP> C{cand[wave], 0, 0, key_score(0)};
            C.set_bound((u64)bound << 32);
            for (uint32_t s = wave; s < n_segs; s += W) {
                if constexpr (kSel == kVectors) {
                    for (int u = 0; u < U; ++u) {
                        const bool hit = groups[(s * U + u) * 64 + lane] >= bound;
                        if (!__any(hit)) continue;
                        const uint32_t i = s * kSeg + (u * 64 + lane) * V;
                        for (int v = 0; v < V; ++v) {
                            const bool have = hit && i + v < n;
                            const float x = have ? score(i + v) : -INFINITY;
                            if (__any(have && !(x < C.fbound))) C.offer(x, first + i + v, have, A.k);
                        }
                    }
                    continue;
                }
                u64 hit = __ballot(groups[s * 64 + lane] >= bound);
                while (hit) {   // two groups at a time, a class a lane
                    const uint32_t a = (uint32_t)__builtin_ctzll(hit);
                    hit &= hit - 1;
                    const uint32_t b = hit ? (uint32_t)__builtin_ctzll(hit) : 64;
                    hit &= hit - 1;
                    const uint32_t ln = lane < kGroup ? a : b, i = s * kSeg + ln * kGroup + lane % kGroup;
                    const bool have = ln < 64 && i < n;
                    C.offer(have ? score(i) : -INFINITY, first + i, have, A.k);
                }
            }
            if (lane == 0) counts[wave] = C.count;
            __syncthreads();
            auto cand_at = [&](uint32_t i) -> u64 { return i % CAP < counts[i / CAP] ? cand[i / CAP][i % CAP] : 0; };
            uint32_t total = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) total += counts[w];
            u64 kth = 1;
            if (total > A.k + kSpare) kth = kth_of<THREADS>(cand_at, W * CAP, A.k, &lds);
            for (uint32_t i = threadIdx.x; i < W * CAP; i += THREADS) {
                const u64 key = cand_at(i);
                if (key >= kth) best[atomicAdd(&nbest, 1u)] = key;
            }
        } else if constexpr (kSel == kWhole) {
            const uint32_t want = min(A.k, n);
            auto key_at = [&](uint32_t i) { return rank_key(score(i), first + i); };
            const u64 kth = kth_of<THREADS>(key_at, n, want, &lds);
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const u64 key = key_at(i);
                if (key >= kth) best[atomicAdd(&nbest, 1u)] = key;
            }
        }
        if constexpr (kSel != kNone) {
            __syncthreads();
            const uint32_t got = nbest;
            const uint32_t slots = A.k + kSpare;
            for (uint32_t i = threadIdx.x; i < slots; i += THREADS) part_keys[job * slots + i] = i < got ? best[i] : 0;
        }
        __syncthreads();
    }
}

// What is written of a row, from its sums and largest keys, or from those of its segments.
template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void finish_kernel(Rows<T> X, Asked A, uint32_t parts, const PartStat* __restrict__ part_stat,
                                                         const u64* __restrict__ part_keys) {
    __shared__ u64 best[kMaxTop + kSpare];
    __shared__ CountLds lds;
    __shared__ uint32_t nbest;
    __shared__ PartStat tmp[THREADS / 64];
    const uint32_t slots = A.k + kSpare;
    for (uint64_t row = blockIdx.x; row < X.rows; row += gridDim.x) {
        const u64* keys = part_keys + row * parts * slots;
        uint32_t got = A.k;
        if (threadIdx.x == 0) nbest = 0;
        RunningStat run;
        const uint32_t own = given_class<T>(A, row, threadIdx.x);
        const float own_score = given_score(A, X, row, own);
        for (uint32_t p = threadIdx.x; p < parts; p += THREADS) {
            const PartStat ps = part_stat[row * parts + p];
            run.join(ps.m, ps.s, ps.t, A.c);
        }
        __syncthreads();
        if (A.k) {   // (their order does not matter: a key's place is the count of larger ones)
            for (uint32_t i = threadIdx.x; i < parts * slots; i += THREADS) {
                const u64 key = keys[i];
                if (key == 0) continue;
                const uint32_t at = atomicAdd(&nbest, 1u);
                if (at < kMaxTop + kSpare) best[at] = key;
            }
            __syncthreads();
            got = nbest;
            if (got > A.k && got > kRanked) {
                const bool here = got <= kMaxTop + kSpare;
                const uint32_t n = here ? got : parts * slots;
                auto key_at = [&](uint32_t i) { return here ? best[i] : keys[i]; };
                const u64 kth = kth_of<THREADS>(key_at, n, A.k, &lds);
                // (in place: a round's keys are read before any of it is written, and none lands behind what was read)
                if (threadIdx.x == 0) nbest = 0;
                for (uint32_t i0 = 0; i0 < n; i0 += THREADS) {
                    const uint32_t i = i0 + threadIdx.x;
                    const u64 key = i < n ? key_at(i) : 0;
                    __syncthreads();
                    if (key != 0 && key >= kth) best[atomicAdd(&nbest, 1u)] = key;
                    __syncthreads();
                }
                got = A.k;
            }
        }
        block_stat<THREADS>(run, A.c, tmp);
        const RowStat q = row_stat(run);
        if (threadIdx.x == 0) write_stats(A, row, run, q);
        write_given(A, X, row, q, threadIdx.x, THREADS, own, own_score);
        if (A.k) write_top<THREADS>(A, row, best, got, q);
        __syncthreads();
    }
}

// A row of at most NMAX classes in a thread's registers; kWhole: whole vectors of classes next to each other.
template <class T, int NMAX, bool kWhole>
__device__ __forceinline__ void load_few(const T* row, int64_t cs, uint32_t n, float (&x)[NMAX]) {
    constexpr int V = kWhole && Pack<T>::V <= NMAX ? Pack<T>::V : 1;
#pragma unroll
    for (int j = 0; j < NMAX; j += V) {
        if constexpr (V > 1) {
            Pack<T> p;
            if ((uint32_t)j < n) p.w = ((const Loose<T>*)(row + j))->w;
#pragma unroll
            for (int v = 0; v < V; ++v) x[j + v] = (uint32_t)j < n ? p.get(v) : -INFINITY;
        } else {
            x[j] = (uint32_t)j < n ? to_f32(row[(int64_t)j * cs]) : -INFINITY;
        }
    }
}

// Few classes: a row a thread, its scores in registers.  Up to 32: a score's place is the count of those ahead; up to 64, for which
// there are too many pairs (rows next to each other): the largest one after another.
template <class T, int NMAX, bool kWhole, bool kTop>
__global__ __launch_bounds__(256) void logprobs_few_kernel(Rows<T> X, Asked A) {
    const uint32_t n = X.classes;
    for (uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x; row < X.rows; row += (uint64_t)gridDim.x * 256) {
        const T* x0 = X.data + (int64_t)row * X.rs;
        const uint32_t* words = A.allowed + (int64_t)row * A.allowed_stride;
        const uint32_t low = A.allowed ? words[0] : ~0u, high = NMAX > 32 && A.allowed && n > 32 ? words[1] : ~0u;
        const uint32_t own = given_class<T>(A, row, 0);
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
        write_given(A, X, row, q, 0, 1, own, given_score(A, X, row, own));
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

// ---- short rows -------------------------------------------------------------------------------
// Over the G lanes of a group; every lane gets it.
template <int G, class V, class Op>
__device__ __forceinline__ V group_reduce(V v, Op op) {
    if constexpr (G >= 2) v = op(v, dpp_move<0xB1, 0xf>(v, v));     // lanes 1 0 3 2
    if constexpr (G >= 4) v = op(v, dpp_move<0x4E, 0xf>(v, v));     // lanes 2 3 0 1
    if constexpr (G >= 8) v = op(v, dpp_move<0x141, 0xf>(v, v));    // mirrored within 8
    if constexpr (G >= 16) v = op(v, dpp_move<0x140, 0xf>(v, v));   // mirrored within 16
    if constexpr (G >= 32) v = op(v, __shfl_xor(v, 16));
    if constexpr (G >= 64) v = op(v, __shfl_xor(v, 32));
    return v;
}
// A lane's scores of a row of at most G R V classes: vector u of lane l holds the classes from (u G + l) V on (kVec), or one
// class, (u G + l).
template <class T, bool kVec>
constexpr int kWide = kVec ? Pack<T>::V : 1;
template <class T, int G, int R, bool kVec>
__device__ __forceinline__ void load_short(const T* row, int64_t cs, uint32_t l, uint32_t n, const uint32_t* words,
                                           float (&x)[R][kWide<T, kVec>]) {
    constexpr int V = kWide<T, kVec>;
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const uint32_t i = (u * G + l) * V;
        if constexpr (kVec) load_pack<T, true>(row, 1, i, n, -INFINITY, x[u]);
        else x[u][0] = i < n ? to_f32(row[(int64_t)i * cs]) : -INFINITY;
    }
    if (words) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const uint32_t i = (u * G + l) * V, bits = i < n ? words[i >> 5] >> (i & 31) : 0;
#pragma unroll
            for (int v = 0; v < V; ++v) x[u][v] = bits >> v & 1 ? x[u][v] : -INFINITY;
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
constexpr uint32_t kShort = 2048;
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
        if (n <= 4 * V) launch_short<T, 4, 1, true>(X, A, st);
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

// Segments of a row: one, unless the rows alone leave CUs idle and a row is long.  They start at a multiple of 32
// classes, a word of the allowed ones.
constexpr uint32_t kMinSeg = 16384, kMaxGroupSegs = 64;
struct Plan {
    uint32_t parts, seg;
};
Plan plan_parts(uint64_t rows, uint32_t classes) {
    uint32_t parts = (classes + kMaxGroupSegs * kSeg - 1) / (kMaxGroupSegs * kSeg);
    if (rows > 0 && rows < 512 && classes >= 2 * kMinSeg)
        parts = std::max(parts, (uint32_t)std::min<uint64_t>((512 + rows - 1) / rows, classes / kMinSeg));
    const uint32_t seg = ((classes + parts - 1) / parts + 31) / 32 * 32;
    return Plan{(classes + seg - 1) / seg, seg};
}

// Rows enough to fill the chip are taken by workgroups of one wave, whose barriers cost nothing; long rows whose largest are
// asked for are not (4096 x 8192 bf16, k 5: 34 against 43 us; 4096 x 65536: 178 against 136).
constexpr uint64_t kManyRows = 2048;
constexpr uint32_t kWaveRow = 16384;
template <class T, bool kUnit, bool kMask>
int launch_rows(const Rows<T>& X, const Asked& A, const Plan& P, void* workspace, hipStream_t st) {
    const uint32_t n = X.classes, k = A.k, seg = P.seg;
    PartStat* ps = (PartStat*)workspace;
    u64* pk = (u64*)(ps + X.rows * P.parts);   // (neither is touched for whole rows without a k, which have no workspace)
    const unsigned grid = row_grid(X.rows * P.parts);
    const uint32_t shortest = n - seg * (P.parts - 1);
    const bool many = X.rows * P.parts >= kManyRows && (k == 0 || seg <= kWaveRow);
#define RUN(SEL, CAP, LDS)                                                                                              \
    (many ? logprobs_kernel<T, kUnit, kMask, 64, SEL, CAP><<<grid, 64, LDS, st>>>(X, A, P.parts, seg, ps, pk) \
          : logprobs_kernel<T, kUnit, kMask, 256, SEL, CAP><<<grid, 256, LDS, st>>>(X, A, P.parts, seg, ps, pk))
    // by groups, or vectors, where k is at most a quarter of the shortest segment's
    const size_t lds = sizeof(uint32_t) * 64 * ((seg + kSeg - 1) / kSeg);
    constexpr uint32_t V = Pack<T>::V;
    const size_t lds_v = sizeof(uint32_t) * (kSeg / V) * ((seg + kSeg - 1) / kSeg);
    if (k == 0) {
        RUN(kNone, 2, 0);
    } else if (k * 4 <= shortest / kGroup) {
        if (k <= 128) RUN(kGroups, 256, lds);
        else RUN(kGroups, 2048, lds);
    } else if (k * 4 <= shortest / V && lds_v <= 65536) {
        if (k <= 128) RUN(kVectors, 256, lds_v);
        else RUN(kVectors, 2048, lds_v);
    } else {
        RUN(kWhole, 2, 0);
    }
#undef RUN
    CLS_TRY(hipGetLastError());
    if (P.parts > 1 || k) {
        if (P.parts == 1 && k <= 256) finish_kernel<T, 64><<<row_grid(X.rows), 64, 0, st>>>(X, A, 1, ps, pk);
        else finish_kernel<T, 256><<<row_grid(X.rows), 256, 0, st>>>(X, A, P.parts, ps, pk);
        CLS_TRY(hipGetLastError());
    }
    return CBH_OK;
}

template <class T>
int run_logprobs(const void* scores, uint64_t rows, uint32_t n, int64_t rs, int64_t cs, const Asked& A, void* workspace,
                 hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, n, rs, cs};
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
    if (n <= kShort) return run_short(X, A, st);
    const Plan P = plan_parts(rows, n);
    if (cs == 1) return A.allowed ? launch_rows<T, true, true>(X, A, P, workspace, st) : launch_rows<T, true, false>(X, A, P, workspace, st);
    return A.allowed ? launch_rows<T, false, true>(X, A, P, workspace, st) : launch_rows<T, false, false>(X, A, P, workspace, st);
}

// ---- gradient -------------------------------------------------------------------------------
struct Upstream {
    const int32_t* given;
    const float* logprob_grad;
    const float* entropy_grad;   // nullable
    const float* stats;
    const uint32_t* allowed;     // nullable
    int64_t allowed_stride;
    uint32_t n_given;
    float c;
    double it;
};
// The factors of a row: grad_j = 2^y (a + b y), y = (x_j - m) c, beside the entries' own.
struct RowFactors {
    float m, a, b;
    double log_z, far, G, h;
    bool zero;   // all derivatives are 0
};
__device__ __forceinline__ float clamp_finite(double v) {   // (2^y = 0 times it is 0)
    return v != v ? (float)v : (float)fmin(fmax(v, -3.4e38), 3.4e38);
}
__device__ __forceinline__ RowFactors row_factors(const Upstream& P, uint64_t row, double G, bool any) {
    RowFactors f;
    const float* s = P.stats + row * 3;
    f.h = P.entropy_grad ? (double)P.entropy_grad[row] : 0.0;
    f.zero = !any && f.h == 0.0;
    f.G = G;
    const bool none = s[1] == -INFINITY;   // a row of -inf alone: no class has a probability
    f.m = none ? 0.0f : s[0];
    f.log_z = (double)s[1];
    f.far = (double)s[2];
    const double r = none ? 0.0 : -P.it * exp_f64(-f.log_z);
    f.a = none ? 0.0f : clamp_finite(r * (f.G + f.h * f.far));
    f.b = none ? 0.0f : clamp_finite(r * f.h * kLn2);
    return f;
}
__device__ __forceinline__ float grad_of(float x, const RowFactors& f, float c) {
    const float y = (x - f.m) * c;
    return exp2_fast(y) * (f.a + f.b * fmaxf(y, kFar));
}
// That of a class with entries whose derivatives add up to g.
__device__ __forceinline__ float grad_of_given(float x, double g, const RowFactors& f, double it) {
    const double d = ((double)x - (double)f.m) * it, p = f.log_z == -INFINITY ? 0.0 : exp_f64(d - f.log_z);
    return (float)(it * (g - (p == 0.0 ? 0.0 : p * (f.G + f.h * (d + f.far)))));
}

// A wave takes a segment of a row; classes with entries are written over.
constexpr uint32_t kGradSeg = 4 * kSeg;
template <class T, bool kUnit, bool kMask>
__global__ __launch_bounds__(256) void logprob_grad_kernel(Rows<T> X, Upstream P, T* __restrict__ grad, int64_t grs,
                                                           int64_t gcs, uint32_t segs) {
    constexpr int V = Pack<T>::V, U = kPacks<T>;
    const uint32_t lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    for (uint64_t job = (uint64_t)blockIdx.x * 4 + wave; job < X.rows * segs; job += (uint64_t)gridDim.x * 4) {
        const uint64_t row = job / segs;
        const uint32_t first = (uint32_t)(job % segs) * kGradSeg, n = min(X.classes - first, kGradSeg);
        const T* x0 = X.data + (int64_t)row * X.rs + (int64_t)first * X.cs;
        T* g0 = grad + (int64_t)row * grs + (int64_t)first * gcs;
        const uint32_t* words = kMask ? P.allowed + (int64_t)row * P.allowed_stride + first / 32 : nullptr;
        const int32_t* given = P.given + row * P.n_given;
        const float* g = P.logprob_grad + row * P.n_given;
        double G = 0.0;
        bool some = false;
        for (uint32_t i = lane; i < P.n_given; i += 64)
            if ((uint32_t)given[i] < X.classes) {
                G += (double)g[i];
                some |= g[i] != 0.0f;
            }
        G = wave_reduce(G, Add());
        const RowFactors f = row_factors(P, row, G, __any(some));
        for (uint32_t base = 0; base < n; base += kSeg) {
            float x[U][V];
            uint32_t bits[U];
            if (!f.zero) load_tile<T, kUnit>(x0, X.cs, base, n, -INFINITY, x);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = base + (u * 64 + lane) * V;
                if constexpr (kMask) bits[u] = i < n ? words[i >> 5] >> (i & 31) : 0;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    x[u][v] = f.zero ? 0.0f : grad_of(x[u][v], f, P.c);
                    if constexpr (kMask) x[u][v] = bits[u] >> v & 1 ? x[u][v] : 0.0f;
                }
                if (i < n) store_pack<T, kUnit>(g0, gcs, i, n, x[u]);
            }
        }
        if (f.zero) continue;
        __threadfence_block();   // (the stores above are done)
        for (uint32_t i = lane; i < P.n_given; i += 64) {
            const uint32_t j = (uint32_t)given[i];
            if (j >= X.classes || j < first || j - first >= n) continue;
            if (kMask && !is_allowed(words, j - first)) continue;
            double sum = 0.0;
            bool again = false;   // (the first of a class's entries writes)
            for (uint32_t e = 0; e < P.n_given; ++e)
                if ((uint32_t)given[e] == j) {
                    sum += (double)g[e];
                    again |= e < i;
                }
            if (again) continue;
            const float x = to_f32(x0[kUnit ? (int64_t)(j - first) : (int64_t)(j - first) * X.cs]);
            g0[kUnit ? (int64_t)(j - first) : (int64_t)(j - first) * gcs] = from_f32<T>(grad_of_given(x, sum, f, P.it));
        }
    }
}

// Rows of up to 2048 classes in the registers of G lanes.  Lists of more than kShortGiven entries go the other ways: the owner of a
// class goes through the whole list for it.
constexpr uint32_t kShortGiven = 8;
template <class T, int G, int R>
__global__ __launch_bounds__(256) void logprob_grad_short_kernel(Rows<T> X, Upstream P, T* __restrict__ grad, int64_t grs) {
    constexpr int V = Pack<T>::V;
    const uint32_t l = threadIdx.x % G, n = X.classes;
    for (uint64_t first = (uint64_t)blockIdx.x * (256 / G); first < X.rows; first += (uint64_t)gridDim.x * (256 / G)) {
        const uint64_t mine = first + threadIdx.x / G, row = min(mine, X.rows - 1);
        const uint32_t* words = P.allowed ? P.allowed + (int64_t)row * P.allowed_stride : nullptr;
        const int32_t* given = P.given + row * P.n_given;
        const float* g = P.logprob_grad + row * P.n_given;
        const T* x0 = X.data + (int64_t)row * X.rs;
        float x[R][V];
        load_short<T, G, R, true>(x0, 1, l, n, nullptr, x);
        double sum = 0.0;
        bool some = false;
        for (uint32_t i = 0; i < P.n_given; ++i)
            if ((uint32_t)given[i] < n) {
                sum += (double)g[i];
                some |= g[i] != 0.0f;
            }
        const RowFactors f = row_factors(P, row, sum, some);
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const uint32_t i = (u * G + l) * V, bits = words && i < n ? words[i >> 5] >> (i & 31) : ~0u;
#pragma unroll
            for (int v = 0; v < V; ++v) x[u][v] = f.zero || !(bits >> v & 1) ? 0.0f : grad_of(x[u][v], f, P.c);
        }
        if (!f.zero)
            for (uint32_t i = 0; i < P.n_given; ++i) {
                const uint32_t j = (uint32_t)given[i];
                if (j >= n || j / V % G != l || (words && !is_allowed(words, j))) continue;
                double own = 0.0;
                for (uint32_t e = 0; e < P.n_given; ++e) own += (uint32_t)given[e] == j ? (double)g[e] : 0.0;
                const float y = grad_of_given(to_f32(x0[j]), own, f, P.it);
#pragma unroll
                for (int u = 0; u < R; ++u)
#pragma unroll
                    for (int v = 0; v < V; ++v) x[u][v] = (u * G + l) * V + v == j ? y : x[u][v];
            }
        if (mine >= X.rows) continue;
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const uint32_t i = (u * G + l) * V;
            if (i < n) store_pack<T, true>(grad + (int64_t)row * grs, 1, i, n, x[u]);
        }
    }
}

// Few classes, and rows next to each other: a thread takes up to NMAX classes of a row, in registers.  The
// f64 of a row's factors and entries is a thread's, not a group of lanes': 1M x 10 f32 by rows takes 42 us by groups.
template <class T, int NMAX, bool kWhole>
__global__ __launch_bounds__(256) void logprob_grad_few_kernel(Rows<T> X, Upstream P, T* __restrict__ grad, int64_t grs,
                                                               int64_t gcs, uint32_t segs) {
    const uint64_t blocks = (X.rows + 255) / 256;
    for (uint64_t job = blockIdx.x; job < blocks * segs; job += gridDim.x) {
        const uint64_t row = job % blocks * 256 + threadIdx.x;
        if (row >= X.rows) continue;
        const uint32_t first = (uint32_t)(job / blocks) * NMAX, n = min(X.classes - first, (uint32_t)NMAX);
        const T* x0 = X.data + (int64_t)row * X.rs + (int64_t)first * X.cs;
        T* g0 = grad + (int64_t)row * grs + (int64_t)first * gcs;
        const uint32_t bits = P.allowed ? P.allowed[(int64_t)row * P.allowed_stride + first / 32] >> first % 32 : ~0u;
        const int32_t* given = P.given + row * P.n_given;
        const float* g = P.logprob_grad + row * P.n_given;
        float x[NMAX];
        load_few<T, NMAX, kWhole>(x0, X.cs, n, x);
        double G = 0.0;
        bool some = false;
        for (uint32_t i = 0; i < P.n_given; ++i)
            if ((uint32_t)given[i] < X.classes) {
                G += (double)g[i];
                some |= g[i] != 0.0f;
            }
        const RowFactors f = row_factors(P, row, G, some);
        float y[NMAX];
#pragma unroll
        for (int j = 0; j < NMAX; ++j) y[j] = f.zero || !(bits >> j & 1) ? 0.0f : grad_of(x[j], f, P.c);
        uint32_t done = f.zero ? ~0u : ~bits;
        for (uint32_t i = 0; i < P.n_given; ++i) {
            const uint32_t j = (uint32_t)given[i] - first;
            if ((uint32_t)given[i] >= X.classes || j >= n || (done >> j & 1)) continue;
            done |= 1u << j;
            double sum = 0.0;
            for (uint32_t e = i; e < P.n_given; ++e) sum += (uint32_t)given[e] - first == j ? (double)g[e] : 0.0;
            float at = 0.0f;
#pragma unroll
            for (int q = 0; q < NMAX; ++q) at = (uint32_t)q == j ? x[q] : at;
            at = grad_of_given(at, sum, f, P.it);
#pragma unroll
            for (int q = 0; q < NMAX; ++q) y[q] = (uint32_t)q == j ? at : y[q];
        }
        constexpr int V = kWhole && Pack<T>::V <= NMAX ? Pack<T>::V : 1;
#pragma unroll
        for (int j = 0; j < NMAX; j += V) {
            if constexpr (V > 1) {
                float part[V];
#pragma unroll
                for (int v = 0; v < V; ++v) part[v] = y[j + v];
                if ((uint32_t)j < n) store_pack<T, true>(g0, 1, j, n, part);
            } else {
                if ((uint32_t)j < n) g0[(int64_t)j * gcs] = from_f32<T>(y[j]);
            }
        }
    }
}

template <class T>
int run_grad(const void* scores, uint64_t rows, uint32_t n, int64_t rs, int64_t cs, const Upstream& P, void* grad,
             int64_t grs, int64_t gcs, hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, n, rs, cs};
    T* g = (T*)grad;
    constexpr uint32_t V = Pack<T>::V;
    const bool unit = cs == 1 && gcs == 1, lanes = unit && n <= kShort && P.n_given <= kShortGiven;
    if (!(lanes && n > 16) && (n <= 32 || (rs == 1 && grs == 1 && cs != 1))) {
        const unsigned grid = row_grid((rows + 255) / 256 * ((n + 31) / 32));
#define RUN(N) (unit && n % V == 0 ? logprob_grad_few_kernel<T, N, true><<<grid, 256, 0, st>>>(X, P, g, grs, gcs, (n + 31) / 32) \
                     : logprob_grad_few_kernel<T, N, false><<<grid, 256, 0, st>>>(X, P, g, grs, gcs, (n + 31) / 32))
        if (n <= 4) RUN(4);
        else if (n <= 8) RUN(8);
        else if (n <= 16) RUN(16);
        else RUN(32);
#undef RUN
    } else if (lanes) {
#define RUN(G, R) logprob_grad_short_kernel<T, G, R><<<row_grid((rows + 256 / G - 1) / (256 / G)), 256, 0, st>>>(X, P, g, grs)
        if (n <= 4 * V) RUN(4, 1);
        else if (n <= 8 * V) RUN(8, 1);
        else if (n <= 16 * V) RUN(16, 1);
        else if (n <= 32 * V) RUN(32, 1);
        else if (n <= 64 * V) RUN(64, 1);
        else if (n <= 128 * V) RUN(64, 2);
        else if (n <= 256 * V) RUN(64, 4);
        else RUN(64, (int)(32 / V));
#undef RUN
    } else {
        const uint32_t segs = (n + kGradSeg - 1) / kGradSeg;
        const unsigned grid = row_grid((rows * segs + 3) / 4);
#define RUN(UNIT, MASK) logprob_grad_kernel<T, UNIT, MASK><<<grid, 256, 0, st>>>(X, P, g, grs, gcs, segs)
        if (unit) P.allowed ? RUN(true, true) : RUN(true, false);
        else P.allowed ? RUN(false, true) : RUN(false, false);
#undef RUN
    }
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

// What both ask of the given and allowed classes.
int check_lists(const void* given, uint32_t n_given, uint64_t rows, uint32_t classes, const uint32_t* allowed,
                int64_t allowed_stride) {
    if (n_given > kMaxGiven) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "at most 1024 given classes a row");
    if (rows && n_given && !given) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "given is null");
    if (allowed) {
        if ((uintptr_t)allowed % 4) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "allowed is not aligned to 4");
        if (allowed_stride != 0 && allowed_stride < (int64_t)((classes + 31) / 32))
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "allowed_stride is 0 or at least ceil(classes / 32)");
        if ((double)allowed_stride * (double)rows > 1.0e18)
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "strides pass the address range");
    }
    return CBH_OK;
}

}  // namespace

extern "C" uint64_t cbh_class_logprobs_workspace(uint64_t rows, uint32_t classes, uint32_t k) {
    if (classes <= kShort) return 0;
    const Plan P = plan_parts(rows, classes);
    return P.parts == 1 && k == 0 ? 0 : rows * P.parts * (8 * (uint64_t)(k ? k + kSpare : 0) + sizeof(PartStat));
}

extern "C" int cbh_class_logprobs(const void* scores, int32_t type, uint64_t rows, uint32_t classes, int64_t row_stride,
                                  int64_t class_stride, const int32_t* given, uint32_t n_given, double temperature,
                                  const uint32_t* allowed, int64_t allowed_stride, uint32_t k, float* logprob,
                                  float* entropy, float* stats, float* top_logprob, int32_t* top_index, void* workspace,
                                  uint64_t workspace_bytes, void* stream) {
    try {
        int rc = check_scores(scores, type, rows, classes, row_stride, class_stride);
        if (rc != CBH_OK) return rc;
        rc = check_lists(given, n_given, rows, classes, allowed, allowed_stride);
        if (rc != CBH_OK) return rc;
        if (k > classes || k > kMaxTop)
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "k must be in 0 .. min(classes, 1024)");
        if (!good_temperature(temperature)) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, kBadTemperature);
        if (rows == 0) return CBH_OK;
        if (k && (!top_logprob || !top_index))
            return cbh_internal_fail(CBH_ERR_INVALID_ARG, "outputs of the top classes are null");
        const uint64_t need = cbh_class_logprobs_workspace(rows, classes, k);
        if (need > workspace_bytes || (need && (!workspace || (uintptr_t)workspace % 8)))
            return cbh_internal_fail(CBH_ERR_LENGTH_MISMATCH, "the workspace needs " + std::to_string(need) +
                                                                  " bytes, aligned to 8");
        const Asked A{given,  allowed, allowed_stride, n_given, k, (float)(1.4426950408889634 / temperature), 1.0 / temperature,
                      logprob, entropy, stats, top_logprob, top_index};
        hipStream_t st = (hipStream_t)stream;
        switch (type) {
            case CBH_TYPE_F32: return run_logprobs<float>(scores, rows, classes, row_stride, class_stride, A, workspace, st);
            case CBH_TYPE_F16: return run_logprobs<_Float16>(scores, rows, classes, row_stride, class_stride, A, workspace, st);
            default: return run_logprobs<bf16_t>(scores, rows, classes, row_stride, class_stride, A, workspace, st);
        }
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}

extern "C" int cbh_logprob_gradients(const void* scores, int32_t type, uint64_t rows, uint32_t classes,
                                     int64_t row_stride, int64_t class_stride, const int32_t* given, uint32_t n_given,
                                     const float* logprob_grad, const float* entropy_grad, const float* stats,
                                     double temperature, const uint32_t* allowed, int64_t allowed_stride, void* grad,
                                     int64_t grad_row_stride, int64_t grad_class_stride, void* stream) {
    try {
        int rc = check_scores(scores, type, rows, classes, row_stride, class_stride);
        if (rc != CBH_OK) return rc;
        rc = check_lists(given, n_given, rows, classes, allowed, allowed_stride);
        if (rc != CBH_OK) return rc;
        if (!good_temperature(temperature)) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, kBadTemperature);
        if (rows == 0) return CBH_OK;
        if (n_given && !logprob_grad) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "logprob_grad is null");
        if (!stats || !grad) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "stats or grad is null");
        rc = check_scores(grad, type, rows, classes, grad_row_stride, grad_class_stride);
        if (rc != CBH_OK) return rc;
        const Upstream P{given, logprob_grad, entropy_grad, stats, allowed, allowed_stride, n_given,
                         (float)(1.4426950408889634 / temperature), 1.0 / temperature};
        hipStream_t st = (hipStream_t)stream;
#define RUN(T) run_grad<T>(scores, rows, classes, row_stride, class_stride, P, grad, grad_row_stride, grad_class_stride, st)
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
