// Shared parts of log probabilities (class_logprobs.hip, class_logprobs_short.hip) and their gradient
// (class_logprob_grad.hip).
#pragma once
#include "class_scores.hpp"

namespace cbh {
namespace cls {

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

// The allowed bits of a tile's vectors: a word a lane, and each vector's from the lane that has it (a load for every vector instead
// took 4096 x 65536 bf16 from 104 to 139 us).
template <class T>
__device__ __forceinline__ void tile_bits(const uint32_t* words, uint32_t base, uint32_t n, uint32_t (&bits)[kPacks<T>]) {
    constexpr uint32_t V = Pack<T>::V;
    const uint32_t lane = lane_id(), at = base / 32 + lane, word = at < (n + 31) / 32 ? words[at] : 0;
#pragma unroll
    for (int u = 0; u < kPacks<T>; ++u) bits[u] = (uint32_t)__shfl((int)word, (int)((u * 64 + lane) * V / 32)) >> lane * V % 32;
}

// A tile's scores, -inf where a class is not allowed; `words` are those from the tile's row segment on.
template <class T, bool kUnit, bool kMask>
__device__ __forceinline__ void load_allowed(const T* row, int64_t cs, const uint32_t* words, uint32_t base, uint32_t n,
                                             float (&x)[kPacks<T>][Pack<T>::V]) {
    constexpr int V = Pack<T>::V, U = kPacks<T>;
    uint32_t bits[U];
    if constexpr (kMask) tile_bits<T>(words, base, n, bits);
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

constexpr uint32_t kShort = 2048;
// Rows of up to kShort classes (class_logprobs_short.hip).
template <class T>
int run_short_rows(const Rows<T>& X, const Asked& A, hipStream_t st);

// What both ask of the given and allowed classes.
inline int check_lists(const void* given, uint32_t n_given, uint64_t rows, uint32_t classes, const uint32_t* allowed,
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

}  // namespace cls
}  // namespace cbh
