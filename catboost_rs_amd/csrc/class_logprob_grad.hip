// The gradient by the scores of a function of the log probabilities and the entropy, in one pass over the scores.
//
//   grad_j = (sum of g_i of j's entries - p_j (G + h (d_j + E))) / t,  p_j = e^d_j / Z,  G = sum of all g_i
// with the forward pass's m, log Z and E of the row.  A class with entries is f64: its gradient is a difference of nearly equal
// numbers where the row is sure of it.  Read and written once: 4096 x 65536 bf16 with entropy 191 us, 1.07 GB at 5.6 TB/s, the memory's rate.
#include "class_logprobs.hpp"

namespace {
using namespace cbh::cls;

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
// The factors of a row: grad_j = 2^y (a + b y), y = (x_j - m) c, beside the entries' own.  Up to kWidest a and b are f32: their sum is
// finite then, and 0 times it is 0.  Beyond (derivatives over a small temperature: 1 / t reaches 1e38) what a class has may still be
// a number of f32, or 0: the row is `wide`, and each of its classes f64.
constexpr double kWidest = 1e30;
struct RowFactors {
    float m, a, b;
    double log_z, far, G, h;
    bool zero;   // all derivatives are 0
    bool wide;
};
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
    const double a = none ? 0.0 : r * (f.G + f.h * f.far), b = none ? 0.0 : r * f.h * kLn2;
    f.a = (float)a;
    f.b = (float)b;
    f.wide = !f.zero && (fabs(a) > kWidest || fabs(b) > kWidest);
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

// A wave takes a segment of a row; classes with entries, or all of a wide row, are written over.
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
            if constexpr (kMask) tile_bits<T>(words, base, n, bits);
            if (!f.zero) load_tile<T, kUnit>(x0, X.cs, base, n, -INFINITY, x);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = base + (u * 64 + lane) * V;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    x[u][v] = f.zero || f.wide ? 0.0f : grad_of(x[u][v], f, P.c);
                    if constexpr (kMask) x[u][v] = bits[u] >> v & 1 ? x[u][v] : 0.0f;
                }
                if (i < n) store_pack<T, kUnit>(g0, gcs, i, n, x[u]);
            }
        }
        if (f.zero) continue;
        __threadfence_block();   // (the stores above are done)
        for (uint32_t i = lane; i < (f.wide ? n : P.n_given); i += 64) {
            const uint32_t j = f.wide ? first + i : (uint32_t)given[i];
            if (j >= X.classes || j < first || j - first >= n) continue;
            if (kMask && !is_allowed(words, j - first)) continue;
            double sum = 0.0;
            bool again = false;   // (the first of a class's entries writes)
            for (uint32_t e = 0; e < P.n_given; ++e)
                if ((uint32_t)given[e] == j) {
                    sum += (double)g[e];
                    again |= e < i;
                }
            if (again && !f.wide) continue;
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
            for (int v = 0; v < V; ++v) x[u][v] = f.zero || f.wide || !(bits >> v & 1) ? 0.0f : grad_of(x[u][v], f, P.c);
        }
        if (!f.zero)
            for (uint32_t i = 0; i < (f.wide ? n : P.n_given); ++i) {
                const uint32_t j = f.wide ? i : (uint32_t)given[i];
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
// f64 of a row's factors and entries is a thread's, not a group of lanes'.  1M rows by rows, by a thread and by groups of lanes, us: 8
// classes f32 22 and 40, 10 42 and 42, 16 86 and 39, 16 bf16 24 and 28; with 8 entries a row 53 and 234, 143 and 239, 167 and 228, 135 and 184.
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
        // (few enough classes: a sum of entries for each, and the list is read once)
        constexpr bool kSums = NMAX <= 8;
        double G = 0.0, own[kSums ? NMAX : 1] = {};
        bool some = false;
        uint32_t listed = 0;
        for (uint32_t i = 0; i < P.n_given; ++i) {
            const uint32_t j = (uint32_t)given[i];
            if (j >= X.classes) continue;
            const float gi = g[i];
            G += (double)gi;
            some |= gi != 0.0f;
            if constexpr (kSums) {
                listed |= 1u << j;
#pragma unroll
                for (int q = 0; q < NMAX; ++q) own[q] += j == (uint32_t)q ? (double)gi : 0.0;
            }
        }
        const RowFactors f = row_factors(P, row, G, some);
        float y[NMAX];
#pragma unroll
        for (int j = 0; j < NMAX; ++j) y[j] = f.zero || f.wide || !(bits >> j & 1) ? 0.0f : grad_of(x[j], f, P.c);
        if constexpr (kSums) {
            if (f.wide) listed = ~0u;
#pragma unroll
            for (int j = 0; j < NMAX; ++j)
                if (!f.zero && (listed & bits) >> j & 1) y[j] = grad_of_given(x[j], own[j], f, P.it);
        } else {
            uint32_t done = f.zero ? ~0u : ~bits;
            for (uint32_t i = 0; i < (f.wide ? n : P.n_given); ++i) {
                const uint32_t c = f.wide ? first + i : (uint32_t)given[i], j = c - first;
                if (c >= X.classes || j >= n || (done >> j & 1)) continue;
                done |= 1u << j;
                double sum = 0.0;
                for (uint32_t e = f.wide ? 0 : i; e < P.n_given; ++e) sum += (uint32_t)given[e] - first == j ? (double)g[e] : 0.0;
                float at = 0.0f;
#pragma unroll
                for (int q = 0; q < NMAX; ++q) at = (uint32_t)q == j ? x[q] : at;
                at = grad_of_given(at, sum, f, P.it);
#pragma unroll
                for (int q = 0; q < NMAX; ++q) y[q] = (uint32_t)q == j ? at : y[q];
            }
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
        constexpr uint32_t least = 32 / V;   // (lanes: from 17 classes on)
        if (n <= least * V) RUN((int)least, 1);
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

}  // namespace

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
