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
template <int THREADS>
__device__ __forceinline__ void block_stat(RunningStat& r, float c, float* tmp_f, double* tmp_d) {
    const float m = block_reduce<THREADS>(r.m, MaxF(), tmp_f);
    r.raise(m, c);
    double v[2] = {r.s, r.t};
    block_sums<THREADS>(v, tmp_d);
    r.s = v[0];
    r.t = v[1];
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
template <class T>
__device__ __forceinline__ void write_given(const Asked& A, const Rows<T>& X, uint64_t row, const RowStat& q, uint32_t from,
                                            uint32_t step) {
    if (!A.logprob) return;
    const uint32_t* words = A.allowed ? A.allowed + (int64_t)row * A.allowed_stride : nullptr;
    for (uint32_t i = from; i < A.n_given; i += step) {
        const uint32_t j = (uint32_t)A.given[row * A.n_given + i];
        float lp = 0.0f;
        if (j < X.classes) {
            float x = to_f32(X.data[(int64_t)row * X.rs + (int64_t)j * X.cs]);
            if (words && !is_allowed(words, j)) x = -INFINITY;
            lp = log_prob(x, q, A.it);
        }
        A.logprob[row * A.n_given + i] = lp;
    }
}
// The `got` keys of best, the largest first.
template <int THREADS>
__device__ __forceinline__ void write_top(const Asked& A, uint64_t row, const u64* best, uint32_t got, const RowStat& q) {
    for (uint32_t i = threadIdx.x; i < got; i += THREADS) {
        const u64 key = best[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < got; ++j) rank += best[j] > key;
        const float x = key_score((uint32_t)(key >> 32));
        A.top_logprob[row * A.k + rank] = log_prob(x, q, A.it);
        A.top_index[row * A.k + rank] = x == -INFINITY ? -1 : (int32_t)~(uint32_t)key;
    }
}

// A workgroup takes a row, or one of the `parts` segments of a row (few rows of many classes), whose sums and
// k largest keys go to the workspace for join_kernel.  How the largest are found:
//   kNone    k = 0
//   kGroups  a bound from the maxima of every 32 classes, kept in LDS; the groups that reach it are read again
//   kWhole   digits of the keys of all classes, read again for every digit (a k that is large beside the row)
enum Select { kNone, kGroups, kWhole };
template <class T, bool kUnit, bool kMask, int THREADS, Select kSel, int CAP>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(Rows<T> X, Asked A, uint32_t parts, uint32_t seg,
                                                           PartStat* __restrict__ part_stat, u64* __restrict__ part_keys) {
    constexpr int V = Pack<T>::V, U = kPacks<T>, W = THREADS / 64, KMAX = kSel == kWhole ? (int)kMaxTop : CAP / 2;
    extern __shared__ uint32_t groups[];
    __shared__ u64 cand[kSel == kGroups ? W : 1][kSel == kGroups ? CAP : 1];
    __shared__ u64 best[kSel == kNone ? 1 : KMAX];
    __shared__ CountLds lds;
    __shared__ uint32_t counts[W], nbest;
    __shared__ float tmp_f[W];
    __shared__ double tmp_d[W * 2];
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
        const uint32_t n_segs = (n + kSeg - 1) / kSeg;
        RunningStat run;
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
        }
        if (kSel != kNone && threadIdx.x == 0) nbest = 0;
        __syncthreads();
        block_stat<THREADS>(run, A.c, tmp_f, tmp_d);
        const RowStat q = row_stat(run);
        if (parts == 1) {
            if (threadIdx.x == 0) write_stats(A, row, run, q);
            write_given(A, X, row, q, threadIdx.x, THREADS);
        } else if (threadIdx.x == 0) {
            part_stat[job] = PartStat{run.s, run.t, run.m, 0.0f};
        }
        if constexpr (kSel == kGroups) {
            const uint32_t bound =
                (uint32_t)kth_of<THREADS>([&](uint32_t i) { return (u64)groups[i]; }, n_segs * 64, A.k, &lds);
            Candidates<CAP> C{cand[wave], 0, 0, key_score(0)};
            C.set_bound((u64)bound << 32);
            for (uint32_t s = wave; s < n_segs; s += W) {
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
            if (total > A.k) kth = kth_of<THREADS>(cand_at, W * CAP, A.k, &lds);
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
            if (parts == 1) write_top<THREADS>(A, row, best, got, q);
            else
                for (uint32_t i = threadIdx.x; i < A.k; i += THREADS) part_keys[job * A.k + i] = i < got ? best[i] : 0;
        }
        __syncthreads();
    }
}

// The segments of a row together.
template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void join_kernel(Rows<T> X, Asked A, uint32_t parts, const PartStat* __restrict__ part_stat,
                                                       const u64* __restrict__ part_keys) {
    __shared__ u64 best[kMaxTop];
    __shared__ CountLds lds;
    __shared__ uint32_t nbest;
    __shared__ float tmp_f[THREADS / 64];
    __shared__ double tmp_d[THREADS / 64 * 2];
    for (uint64_t row = blockIdx.x; row < X.rows; row += gridDim.x) {
        const u64* keys = part_keys + row * parts * A.k;
        if (threadIdx.x == 0) nbest = 0;
        RunningStat run;
        for (uint32_t p = threadIdx.x; p < parts; p += THREADS) {
            const PartStat ps = part_stat[row * parts + p];
            run.join(ps.m, ps.s, ps.t, A.c);
        }
        __syncthreads();
        block_stat<THREADS>(run, A.c, tmp_f, tmp_d);
        const RowStat q = row_stat(run);
        if (threadIdx.x == 0) write_stats(A, row, run, q);
        write_given(A, X, row, q, threadIdx.x, THREADS);
        if (A.k) {
            const u64 kth = kth_of<THREADS>([&](uint32_t i) { return keys[i]; }, parts * A.k, A.k, &lds);
            for (uint32_t i = threadIdx.x; i < parts * A.k; i += THREADS) {
                const u64 key = keys[i];
                if (key != 0 && key >= kth) best[atomicAdd(&nbest, 1u)] = key;
            }
            __syncthreads();
            write_top<THREADS>(A, row, best, nbest, q);
        }
        __syncthreads();
    }
}

// Few classes: a row a thread, its scores in registers; a score's place is the count of those ahead.
template <class T, int NMAX, bool kTop>
__global__ __launch_bounds__(256) void logprobs_few_kernel(Rows<T> X, Asked A) {
    const uint32_t n = X.classes;
    for (uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x; row < X.rows; row += (uint64_t)gridDim.x * 256) {
        const T* x0 = X.data + (int64_t)row * X.rs;
        const uint32_t bits = A.allowed ? A.allowed[(int64_t)row * A.allowed_stride] : ~0u;
        float x[NMAX];
        RunningStat run;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) {
            x[i] = (uint32_t)i < n ? to_f32(x0[(int64_t)i * X.cs]) : -INFINITY;
            if (!(bits >> i & 1)) x[i] = -INFINITY;
            run.m = fmaxf(run.m, x[i]);
        }
#pragma unroll
        for (int i = 0; i < NMAX; ++i) run.add_one(x[i], A.c);
        const RowStat q = row_stat(run);
        write_stats(A, row, run, q);
        write_given(A, X, row, q, 0, 1);
        if constexpr (kTop) {
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
#pragma unroll
            for (int i = 0; i < NMAX; ++i)
                if ((uint32_t)i < n && rank[i] < A.k) {
                    A.top_logprob[row * A.k + rank[i]] = log_prob(key_score(key[i]), q, A.it);
                    A.top_index[row * A.k + rank[i]] = x[i] == -INFINITY ? -1 : i;
                }
        }
    }
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

template <class T, bool kUnit, bool kMask>
int launch_rows(const Rows<T>& X, const Asked& A, const Plan& P, void* workspace, hipStream_t st) {
    const uint32_t n = X.classes, k = A.k, seg = P.seg;
    PartStat* ps = P.parts > 1 ? (PartStat*)workspace : nullptr;
    u64* pk = P.parts > 1 ? (u64*)(ps + X.rows * P.parts) : nullptr;
    const unsigned grid = row_grid(X.rows * P.parts);
    const uint32_t shortest = n - seg * (P.parts - 1);
#define RUN(TH, SEL, CAP, LDS) logprobs_kernel<T, kUnit, kMask, TH, SEL, CAP><<<grid, TH, LDS, st>>>(X, A, P.parts, seg, ps, pk)
    // by groups where k is at most a quarter of the shortest segment's
    const size_t lds = sizeof(uint32_t) * 64 * ((seg + kSeg - 1) / kSeg);
    if (n <= 2048) {
        if (k == 0) RUN(64, kNone, 2, 0);
        else RUN(64, kWhole, 2, 0);
    } else if (k == 0) {
        RUN(256, kNone, 2, 0);
    } else if (k * 4 <= shortest / kGroup) {
        if (k <= 128) RUN(256, kGroups, 256, lds);
        else RUN(256, kGroups, 2048, lds);
    } else {
        RUN(256, kWhole, 2, 0);
    }
#undef RUN
    CLS_TRY(hipGetLastError());
    if (P.parts > 1) {
        join_kernel<T, 256><<<row_grid(X.rows), 256, 0, st>>>(X, A, P.parts, ps, pk);
        CLS_TRY(hipGetLastError());
    }
    return CBH_OK;
}

template <class T>
int run_logprobs(const void* scores, uint64_t rows, uint32_t n, int64_t rs, int64_t cs, const Asked& A, void* workspace,
                 hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, n, rs, cs};
    if (n <= 32) {
        const unsigned grid = row_grid((rows + 255) / 256);
#define FEW(N) (A.k ? logprobs_few_kernel<T, N, true><<<grid, 256, 0, st>>>(X, A) \
                    : logprobs_few_kernel<T, N, false><<<grid, 256, 0, st>>>(X, A))
        if (n <= 8) FEW(8);
        else if (n <= 16) FEW(16);
        else FEW(32);
#undef FEW
        CLS_TRY(hipGetLastError());
        return CBH_OK;
    }
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
    const double r = none ? 0.0 : -P.it * exp(-f.log_z);
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

// Few classes, and rows next to each other: a thread takes `seg` classes of a row.
template <class T, bool kMask>
__global__ __launch_bounds__(256) void logprob_grad_few_kernel(Rows<T> X, Upstream P, T* __restrict__ grad, int64_t grs,
                                                               int64_t gcs, uint32_t segs, uint32_t seg) {
    const uint64_t blocks = (X.rows + 255) / 256;
    for (uint64_t job = blockIdx.x; job < blocks * segs; job += gridDim.x) {
        const uint64_t row = job % blocks * 256 + threadIdx.x;
        if (row >= X.rows) continue;
        const uint32_t first = (uint32_t)(job / blocks) * seg, end = min(X.classes, first + seg);
        const T* x0 = X.data + (int64_t)row * X.rs;
        T* g0 = grad + (int64_t)row * grs;
        const uint32_t* words = kMask ? P.allowed + (int64_t)row * P.allowed_stride : nullptr;
        const int32_t* given = P.given + row * P.n_given;
        const float* g = P.logprob_grad + row * P.n_given;
        double G = 0.0;
        bool some = false;
        for (uint32_t i = 0; i < P.n_given; ++i)
            if ((uint32_t)given[i] < X.classes) {
                G += (double)g[i];
                some |= g[i] != 0.0f;
            }
        const RowFactors f = row_factors(P, row, G, some);
        for (uint32_t j = first; j < end; ++j) {
            float v = 0.0f;
            if (!f.zero && !(kMask && !is_allowed(words, j))) v = grad_of(to_f32(x0[(int64_t)j * X.cs]), f, P.c);
            g0[(int64_t)j * gcs] = from_f32<T>(v);
        }
        if (f.zero) continue;
        for (uint32_t i = 0; i < P.n_given; ++i) {
            const uint32_t j = (uint32_t)given[i];
            if (j < first || j >= end || (kMask && !is_allowed(words, j))) continue;
            double sum = 0.0;
            for (uint32_t e = 0; e < P.n_given; ++e) sum += (uint32_t)given[e] == j ? (double)g[e] : 0.0;
            g0[(int64_t)j * gcs] = from_f32<T>(grad_of_given(to_f32(x0[(int64_t)j * X.cs]), sum, f, P.it));
        }
    }
}

template <class T>
int run_grad(const void* scores, uint64_t rows, uint32_t n, int64_t rs, int64_t cs, const Upstream& P, void* grad,
             int64_t grs, int64_t gcs, hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, n, rs, cs};
    T* g = (T*)grad;
    if (n <= 32 || (rs == 1 && grs == 1 && cs != 1)) {
        const uint32_t seg = 32, segs = (n + seg - 1) / seg;
        const unsigned grid = row_grid((rows + 255) / 256 * segs);
        if (P.allowed) logprob_grad_few_kernel<T, true><<<grid, 256, 0, st>>>(X, P, g, grs, gcs, segs, seg);
        else logprob_grad_few_kernel<T, false><<<grid, 256, 0, st>>>(X, P, g, grs, gcs, segs, seg);
    } else {
        const uint32_t segs = (n + kGradSeg - 1) / kGradSeg;
        const unsigned grid = row_grid((rows * segs + 3) / 4);
        const bool unit = cs == 1 && gcs == 1;
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
    if (classes <= 32) return 0;
    const Plan P = plan_parts(rows, classes);
    return P.parts == 1 ? 0 : rows * P.parts * (8 * (uint64_t)k + sizeof(PartStat));
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
