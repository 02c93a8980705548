// Distillation from a teacher's top classes: the loss and the gradient of a student's scores.
//
// With p = softmax(x / t), the teacher's probabilities q of its listed classes and `rest` what they
// leave to the others (one bucket):
//   loss = w t^2 [ sum_l q_l (log q_l - log p_l) + rest (log rest - log sum_others p) ]
//   grad = w t [ p_j H - q_j ] (listed),  w t p_j (H - rest / sum_others p) (others),  H = sum q + rest
// The others' softmax mass is summed over the others themselves (the listed classes are marked in
// an LDS bit mask and read as -inf), never as the difference 1 - listed, and relative to the others' own
// largest score m: a student that is sure of its answer leaves the others a mass that such a difference would
// lose, and that no number relative to the row's largest score M holds (e^((m - M) / t) is 0 in f32 from a gap of 87
// temperatures on, in f64 from 745).  With s the others' sum of e^((x - m) / t) and S all classes' of e^((x - M) / t):
//   sum_others p = s e^((m - M) / t) / S,  p_j (H - rest / sum_others p) = e^((x_j - m) / t) (H e^((m - M) / t) / S - rest / s)
// What belongs to the listed classes is f64: their gradient is a difference of nearly equal probabilities.
#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

constexpr uint32_t kMaxList = 1024;
// Rows from 256 KB on are taken by 512 threads, one workgroup a CU: with four of 256 threads a CU the rows that are
// under way pass the 256 MB of the last cache, and the second read comes from HBM (1500 x 100003 f32: 320 against
// 372 us; 4096 x 65536 bf16, 128 KB a row: 349 against 278).
constexpr size_t kWideRow = (size_t)1 << 18;
constexpr uint32_t kMaxSeg = 1u << 18;   // classes a workgroup takes: their marks are 32 KB of LDS

struct Lists {   // the teacher's, and what weighs the rows
    const float* scores;     // [rows][k]
    const int32_t* index;
    const float* lse;        // nullable
    const float* weight;     // nullable
    uint32_t k;
};
template <class T>
struct Grad {
    T* data;   // nullable
    int64_t rs, cs;
};

// Sums over a row's list, and the factors of its outputs.
struct RowSums {
    double held, entropy;   // sum q, sum q log q
    uint32_t listed;        // valid entries
    double base, base_log;  // log q = (u / t - base) - base_log
};
struct Outcome {
    double loss;
    float others;          // gradient of an other class: 2^((x - m) c) * others, m the largest of them
    double whole, inv_s;   // of a listed one: wt (2^((x - M) c) * inv_s * whole - q)
};

__device__ __forceinline__ double row_rest(const RowSums& r, bool has_lse, uint32_t n) {
    return has_lse && r.listed < n ? fmax(0.0, 1.0 - r.held) : 0.0;
}
// q log q and q log p, 0 where q is
__device__ __forceinline__ double times_log(double q, double l) { return q == 0.0 ? 0.0 : q * l; }
// gap: (m - M) / t; s_others: the others' sum at m; s_listed: the listed classes' at M; cross: sum q (x - M) / t.  t, w as
// in the loss.
__device__ __forceinline__ Outcome outcome(const RowSums& r, double rest, double gap, double s_others, double s_listed,
                                           double cross, double t, double w) {
    Outcome o;
    const double fade = s_others == 0.0 ? 0.0 : exp_f64(gap), S = s_others * fade + s_listed;
    const double share = s_others > 0.0 ? rest / s_others : 0.0, log_s = log(S);
    o.whole = r.held + rest;
    o.inv_s = S > 0.0 ? 1.0 / S : S == 0.0 ? 0.0 : S;   // (NaN stays)
    o.others = (float)(w * t * (o.whole * o.inv_s * fade - share));
    // sum q log p; a row without a score above -inf gives its classes no probability
    const double lin = S == 0.0 ? (r.held > 0.0 ? -(double)INFINITY : 0.0) : cross - times_log(r.held, log_s);
    double loss = r.entropy - lin;
    if (rest > 0.0) loss += s_others == 0.0 ? (double)INFINITY : rest * (log(rest / s_others) - gap + log_s);
    o.loss = w * t * t * loss;
    return o;
}
// (the list's own log-sum-exp stays in two parts: next to the lowest f32 one number would lose the logarithm; an entry
// of -inf has no mass beside a log-sum-exp of -inf either)
__device__ __forceinline__ double log_q(double ut, const RowSums& r) {
    return ut == -(double)INFINITY ? ut : (ut - r.base) - r.base_log;
}

// Two passes over a row, the second from the last cache while the rows under way fit it, one of them writing.
// 4096 x 65536 bf16, k 64: 269 us, 1.07 GB of reads and writes at 4.0 TB/s (a copy: 5.2); 1500 x 100003 f32, k 20: 297
// us, 1.2 GB at 4.0 TB/s.  Bound by memory and the second read.  Holding a row's tiles in registers between the
// passes was built and spilled (the f32 forms of a tile are twice its registers): not kept.
// A workgroup takes a row (kPhase 0), or a segment of one (few rows of many classes): phase 1 leaves the
// segment's (m, s) of its others, phase 2 reads all of the row's and writes its part of the gradient.
template <class T, bool kUnit, int THREADS, int LE /* list entries a thread */, int kPhase>
__global__ __launch_bounds__(THREADS) void distill_kernel(Rows<T> X, Lists L, float c, double it, double t,
                                                          uint32_t parts, uint32_t seg, float* __restrict__ loss,
                                                          Grad<T> G, PartSum* __restrict__ part_ms) {
    constexpr int V = Pack<T>::V, U = kPacks<T>, W = THREADS / 64;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = lane_id();
    extern __shared__ uint32_t mark[];   // a bit a class of the segment
    __shared__ float tmp_f[W];
    __shared__ double tmp_d[W * 5];
    const uint32_t words = (min(seg, X.classes) + 31) / 32;

    for (uint64_t job = blockIdx.x; job < X.rows * parts; job += gridDim.x) {
        const uint64_t row = job / parts;
        const uint32_t first = (uint32_t)(job % parts) * seg, n = min(X.classes - first, seg);
        const T* x0 = X.data + (int64_t)row * X.rs + (int64_t)first * X.cs;
        T* g0 = G.data ? G.data + (int64_t)row * G.rs + (int64_t)first * G.cs : nullptr;
        const float* u = L.scores + row * L.k;
        const int32_t* ix = L.index + row * L.k;
        const double w = L.weight ? (double)L.weight[row] : 1.0;
        if (w == 0.0) {   // (uniform: the whole workgroup)
            if (kPhase != 1) {
                if (loss && first == 0 && threadIdx.x == 0) loss[row] = 0.0f;
                if (g0) {
                    float z[V];
#pragma unroll
                    for (int v = 0; v < V; ++v) z[v] = 0.0f;
                    for (uint32_t i = threadIdx.x * V; i < n; i += THREADS * V) store_pack<T, kUnit>(g0, G.cs, i, n, z);
                }
            }
            continue;
        }
        // the list, once: the teacher's log probabilities and the student's scores stay in registers
        uint32_t cls[LE];   // (a class past all: no entry)
        float xl[LE];
        double lq[LE];
        const T* xr = X.data + (int64_t)row * X.rs;
#pragma unroll
        for (int e = 0; e < LE; ++e) {
            const uint32_t i = e * THREADS + threadIdx.x;
            cls[e] = i < L.k ? (uint32_t)ix[i] : ~0u;
            if (cls[e] >= X.classes) cls[e] = ~0u;
            lq[e] = cls[e] != ~0u ? (double)u[i] * it : -INFINITY;
            xl[e] = cls[e] != ~0u ? to_f32(xr[(int64_t)cls[e] * X.cs]) : -INFINITY;
        }
        Running run;
        if (kPhase != 2) {
            for (uint32_t i = threadIdx.x; i < words; i += THREADS) mark[i] = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < LE; ++e) {
                const uint32_t j = cls[e] - first;
                if (cls[e] != ~0u && j < n) atomicOr(&mark[j >> 5], 1u << (j & 31));
            }
            __syncthreads();
            for (uint32_t base = wave * kSeg; base < n; base += W * kSeg) {
                float x[U][V], tm = -INFINITY;
                load_tile<T, kUnit>(x0, X.cs, base, n, -INFINITY, x);
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const uint32_t i = base + (q * 64 + lane) * V;
                    const uint32_t bits = i < n ? mark[i >> 5] >> (i & 31) : 0;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        x[q][v] = bits >> v & 1 ? -INFINITY : x[q][v];
                        tm = fmaxf(tm, x[q][v]);
                    }
                }
                run.raise(tm, c);
                run.add(x, c);
            }
        } else {
            for (uint32_t p = threadIdx.x; p < parts; p += THREADS) {
                const PartSum ms = part_ms[row * parts + p];
                run.join(ms.m, ms.s, c);
            }
        }
        float mo;
        double so;
        block_running<THREADS>(run, c, mo, so, tmp_f, tmp_d);
        if (kPhase == 1) {
            if (threadIdx.x == 0) part_ms[job] = PartSum{so, mo};
            continue;
        }
        float lmax = kLowest;
        double umax = -INFINITY;
#pragma unroll
        for (int e = 0; e < LE; ++e) {
            lmax = fmaxf(lmax, xl[e]);
            umax = fmax(umax, lq[e]);
        }
        const float M = fmaxf(mo, block_reduce<THREADS>(lmax, MaxF(), tmp_f));
        RowSums r{};
        if (L.lse) {
            r.base = (double)L.lse[row];
        } else {
            r.base = umax = block_reduce<THREADS>(umax, MaxF(), tmp_d);
            double s[1] = {0.0};
#pragma unroll
            for (int e = 0; e < LE; ++e) s[0] += lq[e] == -INFINITY ? 0.0 : exp_f64(lq[e] - umax);   // (no entry: -inf)
            block_sums<THREADS>(s, tmp_d);
            r.base_log = log(s[0]);
        }
        // sums over the list: q, q log q, the student's exponentials, q (x - M) / t, entries
        double s[5] = {};
        double el[LE];
#pragma unroll
        for (int e = 0; e < LE; ++e) {
            el[e] = 0.0;
            if (cls[e] == ~0u) continue;
            const double l = log_q(lq[e], r), q = exp_f64(l), d = ((double)xl[e] - (double)M) * it;
            el[e] = exp_f64(d);
            lq[e] = q;   // (from here on: q)
            s[0] += q;
            s[1] += times_log(q, l);
            s[2] += el[e];
            s[3] += times_log(q, d);
            s[4] += 1.0;
        }
        block_sums<THREADS>(s, tmp_d);
        r.held = s[0];
        r.entropy = s[1];
        r.listed = (uint32_t)s[4];
        const double rest = row_rest(r, L.lse != nullptr, X.classes);
        const Outcome o = outcome(r, rest, ((double)mo - (double)M) * it, so, s[2], s[3], t, w);
        if (loss && first == 0 && threadIdx.x == 0) loss[row] = (float)o.loss;
        if (g0) {
            for (uint32_t base = wave * kSeg; base < n; base += W * kSeg) {
                float x[U][V];
                load_tile<T, kUnit>(x0, X.cs, base, n, -INFINITY, x);
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const uint32_t i = base + (q * 64 + lane) * V;
#pragma unroll
                    for (int v = 0; v < V; ++v) x[q][v] = exp2_fast((x[q][v] - mo) * c) * o.others;
                    if (i < n) store_pack<T, kUnit>(g0, G.cs, i, n, x[q]);
                }
            }
            __syncthreads();   // the listed classes are written over
#pragma unroll
            for (int e = 0; e < LE; ++e) {
                const uint32_t j = cls[e] - first;
                if (cls[e] == ~0u || j >= n) continue;
                g0[(int64_t)j * G.cs] = from_f32<T>((float)(w * t * (el[e] * o.inv_s * o.whole - lq[e])));
            }
        }
        __syncthreads();
    }
}

// Few classes: a row a thread, its scores in registers, the listed classes a bit mask.  1M x 10 f32, k 3, class-major:
// 39 us, 112 MB at 2.9 TB/s; bound by the f64 exponentials and logarithms of the lists, their loads, and scalar registers
// that do not fit (108 put aside at 12 classes and 4 entries, 286 at 32).
// Lists of up to KM entries are held in registers as well (KM 0: read again in every step; k 3 that way 59 us).
template <class T, int NMAX, int KM>
__global__ __launch_bounds__(256) void distill_few_kernel(Rows<T> X, Lists L, float c, double it, double t,
                                                          float* __restrict__ loss, Grad<T> G) {
    const uint32_t n = X.classes;
    for (uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x; row < X.rows; row += (uint64_t)gridDim.x * 256) {
        const T* x0 = X.data + (int64_t)row * X.rs;
        T* g0 = G.data ? G.data + (int64_t)row * G.rs : nullptr;
        const double w = L.weight ? (double)L.weight[row] : 1.0;
        if (w == 0.0) {
            if (loss) loss[row] = 0.0f;
            if (g0)
                for (uint32_t j = 0; j < n; ++j) g0[(int64_t)j * G.cs] = from_f32<T>(0.0f);
            continue;
        }
        const float* u = L.scores + row * L.k;
        const int32_t* ix = L.index + row * L.k;
        struct Entry {   // of the list: class (n and more: none), teacher's score / t, then the student's, q, e^(x - M)
            uint32_t cls;
            double ut;
            float x;
            double q, e;
        };
        Entry kept[KM ? KM : 1];
        if constexpr (KM > 0) {
#pragma unroll
            for (int i = 0; i < KM; ++i) {
                const uint32_t at = min((uint32_t)i, L.k - 1);
                kept[i].cls = (uint32_t)i < L.k ? (uint32_t)ix[at] : ~0u;
                kept[i].ut = (double)u[at] * it;
            }
        }
        float x[NMAX], M = kLowest, mo = kLowest;
#pragma unroll
        for (int j = 0; j < NMAX; ++j) x[j] = (uint32_t)j < n ? to_f32(x0[(int64_t)j * X.cs]) : -INFINITY;
        if constexpr (KM > 0) {
#pragma unroll
            for (int i = 0; i < KM; ++i) {
                kept[i].x = -INFINITY;
#pragma unroll
                for (int j = 0; j < NMAX; ++j) kept[i].x = kept[i].cls == (uint32_t)j ? x[j] : kept[i].x;
            }
        }
        auto each = [&](auto f) {
            if constexpr (KM > 0) {
#pragma unroll
                for (int i = 0; i < KM; ++i)
                    if (kept[i].cls < n) f(kept[i]);
            } else {
                for (uint32_t i = 0; i < L.k; ++i) {
                    Entry en;
                    en.cls = (uint32_t)ix[i];
                    if (en.cls >= n) continue;
                    en.ut = (double)u[i] * it;
                    en.x = to_f32(x0[(int64_t)en.cls * X.cs]);
                    f(en);
                }
            }
        };
        uint32_t mask = 0;
        double umax = -INFINITY;
        each([&](Entry& en) {
            mask |= 1u << en.cls;
            umax = fmax(umax, en.ut);
        });
        RowSums r{};
        r.listed = (uint32_t)__popc(mask);
        if (L.lse) {
            r.base = (double)L.lse[row];
        } else {
            double s = 0.0;
            each([&](Entry& en) { s += en.ut == -INFINITY ? 0.0 : exp_f64(en.ut - umax); });
            r.base = umax;
            r.base_log = log(s);
        }
#pragma unroll
        for (int j = 0; j < NMAX; ++j) {
            M = fmaxf(M, x[j]);
            mo = fmaxf(mo, mask >> j & 1 ? -INFINITY : x[j]);
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < NMAX; ++j) {
            const float e = exp2_fast((x[j] - mo) * c);
            s += mask >> j & 1 ? 0.0f : e;
        }
        auto weigh = [&](Entry& en) {
            en.q = exp_f64(log_q(en.ut, r));
            en.e = exp_f64(((double)en.x - (double)M) * it);
        };
        double sl = 0.0, cross = 0.0;   // sum q (x - M) / t
        each([&](Entry& en) {
            weigh(en);
            sl += en.e;
            r.held += en.q;
            r.entropy += times_log(en.q, log_q(en.ut, r));
            cross += times_log(en.q, ((double)en.x - (double)M) * it);
        });
        const double rest = row_rest(r, L.lse != nullptr, n);
        const Outcome o = outcome(r, rest, ((double)mo - (double)M) * it, (double)s, sl, cross, t, w);
        if (loss) loss[row] = (float)o.loss;
        if (g0) {
#pragma unroll
            for (int j = 0; j < NMAX; ++j)
                if ((uint32_t)j < n && !(mask >> j & 1))
                    g0[(int64_t)j * G.cs] = from_f32<T>(exp2_fast((x[j] - mo) * c) * o.others);
            each([&](Entry& en) {
                if constexpr (KM == 0) weigh(en);
                g0[(int64_t)en.cls * G.cs] = from_f32<T>((float)(w * t * (en.e * o.inv_s * o.whole - en.q)));
            });
        }
    }
}

constexpr uint32_t kMinSeg = 16384;
uint32_t plan_parts(uint64_t rows, uint32_t classes) {
    uint32_t parts = (classes + kMaxSeg - 1) / kMaxSeg;
    if (rows > 0 && rows < 512 && classes >= 2 * kMinSeg)
        parts = std::max(parts, (uint32_t)std::min<uint64_t>((512 + rows - 1) / rows, classes / kMinSeg));
    return parts;
}
// Segments start at a multiple of 32 classes: a vector's marks lie in one word.
uint32_t segment(uint32_t classes, uint32_t parts) { return ((classes + parts - 1) / parts + 31) / 32 * 32; }

template <class T, bool kUnit, int THREADS, int LE>
int launch_rows(const Rows<T>& X, const Lists& L, float c, double t, uint32_t parts, float* loss, const Grad<T>& G,
                void* workspace, hipStream_t st) {
    const uint32_t seg = segment(X.classes, parts);
    const unsigned grid = row_grid(X.rows * parts);
    const size_t lds = 4 * (size_t)((std::min(seg, X.classes) + 31) / 32);
    PartSum* ms = (PartSum*)workspace;
    const double it = 1.0 / t;
    if (parts == 1) {
        distill_kernel<T, kUnit, THREADS, LE, 0><<<grid, THREADS, lds, st>>>(X, L, c, it, t, 1, seg, loss, G, ms);
    } else {
        distill_kernel<T, kUnit, THREADS, LE, 1><<<grid, THREADS, lds, st>>>(X, L, c, it, t, parts, seg, loss, G, ms);
        CLS_TRY(hipGetLastError());
        distill_kernel<T, kUnit, THREADS, LE, 2><<<grid, THREADS, 0, st>>>(X, L, c, it, t, parts, seg, loss, G, ms);
    }
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

template <class T>
int run_distill(const void* scores, uint64_t rows, uint32_t n, int64_t rs, int64_t cs, const Lists& L, double t,
                uint32_t parts, float* loss, void* grad, int64_t grs, int64_t gcs, void* workspace, hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, n, rs, cs};
    const Grad<T> G{(T*)grad, grs, gcs};
    const float c = (float)(1.4426950408889634 / t);
    if (n <= 32) {
        const unsigned grid = row_grid((rows + 255) / 256);
        const double it = 1.0 / t;
#define FEW(N) (L.k <= 4 ? distill_few_kernel<T, N, 4><<<grid, 256, 0, st>>>(X, L, c, it, t, loss, G) \
                         : distill_few_kernel<T, N, 0><<<grid, 256, 0, st>>>(X, L, c, it, t, loss, G))
        if (n <= 4) FEW(4);
        else if (n <= 8) FEW(8);
        else if (n <= 12) FEW(12);
        else if (n <= 16) FEW(16);
        else FEW(32);
#undef FEW
        CLS_TRY(hipGetLastError());
        return CBH_OK;
    }
    const bool unit = cs == 1 && (!grad || gcs == 1);
#define ROWS(TH, LE) (unit ? launch_rows<T, true, TH, LE>(X, L, c, t, parts, loss, G, workspace, st) \
                           : launch_rows<T, false, TH, LE>(X, L, c, t, parts, loss, G, workspace, st))
    if (n <= 2048) return L.k <= 64 ? ROWS(64, 1) : L.k <= 256 ? ROWS(64, 4) : ROWS(64, 16);
    if (n * sizeof(T) < kWideRow) return L.k <= 256 ? ROWS(256, 1) : ROWS(256, 4);
    return L.k <= 512 ? ROWS(512, 1) : ROWS(512, 2);
#undef ROWS
}

}  // namespace

extern "C" uint64_t cbh_distill_gradients_workspace(uint64_t rows, uint32_t classes) {
    const uint32_t parts = plan_parts(rows, classes);
    return parts <= 1 ? 0 : rows * parts * sizeof(PartSum);
}

extern "C" int cbh_distill_gradients(const void* scores, int32_t type, uint64_t rows, uint32_t classes,
                                     int64_t row_stride, int64_t class_stride, const float* top_scores,
                                     const int32_t* top_index, uint32_t k, const float* top_lse, double temperature,
                                     const float* weight, float* loss, void* grad, int64_t grad_row_stride,
                                     int64_t grad_class_stride, void* workspace, uint64_t workspace_bytes,
                                     void* stream) {
    try {
        int rc = check_scores(scores, type, rows, classes, row_stride, class_stride);
        if (rc != CBH_OK) return rc;
        if (k < 1 || k > kMaxList) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "k must be in 1 .. 1024");
        if (!good_temperature(temperature))
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, kBadTemperature);
        if (rows == 0) return CBH_OK;
        if (!top_scores || !top_index) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "the teacher's lists are null");
        if (!loss && !grad) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "loss and grad are both null");
        if (grad) {
            rc = check_scores(grad, type, rows, classes, grad_row_stride, grad_class_stride);
            if (rc != CBH_OK) return rc;
        }
        const uint64_t need = cbh_distill_gradients_workspace(rows, classes);
        if (need > workspace_bytes || (need && (!workspace || (uintptr_t)workspace % 8)))
            return cbh_internal_fail(CBH_ERR_LENGTH_MISMATCH, "the workspace needs " + std::to_string(need) +
                                                                  " bytes, aligned to 8");
        const uint32_t parts = plan_parts(rows, classes);
        const Lists L{top_scores, top_index, top_lse, weight, k};
        hipStream_t st = (hipStream_t)stream;
#define RUN(T) run_distill<T>(scores, rows, classes, row_stride, class_stride, L, temperature, parts, loss, grad, \
                              grad_row_stride, grad_class_stride, workspace, st)
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
