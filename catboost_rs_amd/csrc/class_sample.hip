// One class drawn from every row of scores, from a given uniform number, after the cuts of a
// temperature, the top k classes, the nucleus of mass p and a smallest weight.
//
// The classes are ordered by score (largest first, the lowest class first among equal ones); every
// cut keeps a prefix of that order, so together they keep the classes above a score and the first
// few of those at it (`Cut`).  The weight of a class, exp((x - max) / t), is an integer in units of 2^-S:
// sums of masses are exact, equal whatever the order they are taken in, and the running mass
// that the draw compares with u times the total cannot disagree with that total.
#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

struct Settings {
    const double* uniform;
    double t, p, min_p;
    uint32_t k;
    const float *t_rows, *p_rows, *min_p_rows;   // nullable
    const int32_t* k_rows;
    const uint32_t* allowed;   // nullable
    int64_t allowed_stride;
};
struct Row {   // a row's settings
    double u, rt, p, min_p;
    uint32_t k;    // 0: all
    bool greedy;
    const uint32_t* allowed;
};
__device__ __forceinline__ Row settings(const Settings& S, uint64_t row, uint32_t n) {
    Row r;
    r.u = S.uniform[row];
    const double t = S.t_rows ? (double)S.t_rows[row] : S.t;
    r.greedy = !(t > 0.0);
    r.rt = 1.0 / t;
    r.p = S.p_rows ? (double)S.p_rows[row] : S.p;
    r.min_p = S.min_p_rows ? (double)S.min_p_rows[row] : S.min_p;
    const uint32_t k = S.k_rows ? (uint32_t)max(S.k_rows[row], 0) : S.k;
    r.k = k >= n ? 0 : k;
    r.allowed = S.allowed ? S.allowed + (int64_t)row * S.allowed_stride : nullptr;
    return r;
}

// Keys: 0 for a class that is not drawn (-inf, NaN, not allowed), else ordered as the scores.
__device__ __forceinline__ uint32_t class_key(float x, bool allowed) {
    return allowed && x > -INFINITY ? order_key(x) : 0;
}
// The weight of a score in [0, 1], and its mass in units of 2^-S: S <= 51, the product with 2^S is
// rounded to an integer by the addition of 2^52.
__device__ __forceinline__ double weight_of(float x, float m, double rt) {
    return x == m ? 1.0 : exp(((double)x - (double)m) * rt);
}
__device__ __forceinline__ u64 mass_of(double w, double unit) {
    return __builtin_bit_cast(u64, __builtin_fma(w, unit, 4503599627370496.0)) - 0x4330000000000000ull;
}
// floor(u total), below total
__device__ __forceinline__ u64 target_of(double u, u64 total) {
    const double d = u * (double)total;
    const u64 v = d > 0.0 ? (u64)d : 0;
    return v < total ? v : total - 1;
}
// the least mass that a nucleus holds: classes stay while the mass ahead is below it
__device__ __forceinline__ u64 nucleus_of(double p, u64 total) {
    const double d = ceil(p * (double)total);
    const u64 v = d > 0.0 ? (u64)d : 0;
    return v < 1 ? 1 : v > total ? total : v;
}

struct Cut {   // kept: classes with a larger key, and the first `ties` with this one
    uint32_t key, ties;
    u64 mass;   // kept mass
};

// A workgroup a row.
template <class T, int THREADS>
struct Walk {
    static constexpr int W = THREADS / 64;
    const T* x0;
    int64_t cs;
    uint32_t n;
    Row r;
    float m;
    double unit;
    __device__ __forceinline__ float score(uint32_t i) const { return to_f32(x0[(int64_t)i * cs]); }
    __device__ __forceinline__ uint32_t key(uint32_t i, float x) const {
        return class_key(x, !r.allowed || (r.allowed[i >> 5] >> (i & 31) & 1));
    }
    __device__ __forceinline__ u64 mass(float x) const { return mass_of(weight_of(x, m, r.rt), unit); }

    // The shortest prefix of the order that holds `count` classes (by_mass false) or a mass of `want`;
    // keys below `floor` are no candidates.  By bytes of the key from the top.
    __device__ Cut select(bool by_mass, u64 want, uint32_t floor, uint32_t* hist, u64* hist_mass) const {
        uint32_t prefix = 0;
        u64 above = 0, above_mass = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t b = threadIdx.x; b < 256; b += THREADS) {
                hist[b] = 0;
                hist_mass[b] = 0;
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                const float x = score(i);
                const uint32_t q = key(i, x);
                if (q == 0 || q < floor || (shift < 24 && (q >> (shift + 8)) != prefix)) continue;
                atomicAdd(&hist[q >> shift & 255], 1u);
                atomicAdd(&hist_mass[q >> shift & 255], mass(x));
            }
            __syncthreads();
            uint32_t bin;
            if (by_mass) {
                const Found<u64> f = find_bin(hist_mass, want - above_mass);
                bin = f.bin;
                above_mass += f.above;
            } else {
                const Found<uint32_t> f = find_bin(hist, (uint32_t)(want - above));
                bin = f.bin;
                above += f.above;
                u64 m = 0;
                for (uint32_t b = lane_id(); b < 256; b += 64) m += b > bin ? hist_mass[b] : 0;
                above_mass += wave_reduce(m, Add());
            }
            prefix = prefix << 8 | bin;
            if (shift == 0) {
                const uint32_t ties = hist[bin];
                const u64 each = ties ? hist_mass[bin] / ties : 0;
                u64 need = want - (by_mass ? above_mass : above);
                if (by_mass) need = each ? (need + each - 1) / each : ties;
                Cut c;
                c.key = prefix;
                c.ties = (uint32_t)(need < ties ? need : ties);
                c.mass = above_mass + (u64)c.ties * each;
                __syncthreads();
                return c;
            }
            __syncthreads();
        }
        return Cut{};
    }
};

template <class T, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_kernel(Rows<T> X, Settings S, double unit,
                                                         int32_t* __restrict__ index, float* __restrict__ logprob) {
    constexpr int W = THREADS / 64;
    __shared__ uint32_t hist[256];
    __shared__ u64 hist_mass[256];
    __shared__ u64 tmp_u[W], wave_mass[W];
    __shared__ uint32_t wave_ties[W];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = lane_id();
    const uint32_t n = X.classes;
    for (uint64_t row = blockIdx.x; row < X.rows; row += gridDim.x) {
        Walk<T, THREADS> K{X.data + (int64_t)row * X.rs, X.cs, n, settings(S, row, n), 0.0f, unit};
        u64 top = 0;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
            const uint32_t q = K.key(i, K.score(i));
            const u64 key = q ? ((u64)q << 32) | (uint32_t)~i : 0;
            top = key > top ? key : top;
        }
        top = block_reduce<THREADS>(top, [](u64 a, u64 b) { return a > b ? a : b; }, tmp_u);
        if (top == 0 || K.r.greedy) {
            if (threadIdx.x == 0) {
                index[row] = top ? (int32_t)~(uint32_t)top : -1;
                if (logprob) logprob[row] = top ? 0.0f : -INFINITY;
            }
            continue;
        }
        K.m = key_score((uint32_t)(top >> 32));
        u64 total = 0;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
            const float x = K.score(i);
            if (K.key(i, x)) total += K.mass(x);
        }
        total = block_reduce<THREADS>(total, Add(), tmp_u);
        Cut cut{0, 0, total};
        if (K.r.min_p > 1.0) {
            cut = Cut{(uint32_t)(top >> 32), 1, mass_of(1.0, unit)};
        } else {
            if (K.r.k) cut = K.select(false, K.r.k, 0, hist, hist_mass);
            if (K.r.p < 1.0) cut = K.select(true, nucleus_of(K.r.p, cut.mass), cut.key, hist, hist_mass);
        }
        // wave w holds the classes [w per, (w + 1) per), lanes side by side
        const uint32_t per = ((n + W - 1) / W + 63) / 64 * 64;
        const uint32_t a = wave * per, b = min(n, a + per);
        uint32_t ties = 0;
        for (uint32_t i = a + lane; i < b; i += 64) {
            const uint32_t q = K.key(i, K.score(i));
            ties += q != 0 && q == cut.key;
        }
        ties = wave_reduce(ties, Add());
        if (lane == 0) wave_ties[wave] = ties;
        __syncthreads();
        uint32_t ties_before = 0;
        for (uint32_t v = 0; v < wave; ++v) ties_before += wave_ties[v];
        // the kept mass of class i (no class at b and beyond); `seen` counts the ties passed
        auto kept = [&](uint32_t i, uint32_t& seen) -> u64 {
            const float x = i < b ? K.score(i) : 0.0f;
            const uint32_t q = i < b ? K.key(i, x) : 0;
            const bool tie = q != 0 && q == cut.key;
            const u64 t = __ballot(tie);
            bool in = q > cut.key || (tie && seen + (uint32_t)__popcll(t & ((1ull << lane) - 1)) < cut.ties);
            seen += (uint32_t)__popcll(t);
            if (!in) return 0;
            const double w = weight_of(x, K.m, K.r.rt);
            return !(w < K.r.min_p) || K.r.min_p > 1.0 ? mass_of(w, unit) : 0;
        };
        u64 mine = 0;
        uint32_t seen = ties_before;
        for (uint32_t i = a; i < b; i += 64) mine += kept(i + lane, seen);
        mine = wave_reduce(mine, Add());
        if (lane == 0) wave_mass[wave] = mine;
        __syncthreads();
        u64 sum = 0, before = 0;
        for (uint32_t v = 0; v < W; ++v) {
            if (v == wave) before = sum;
            sum += wave_mass[v];
        }
        const u64 target = target_of(K.r.u, sum);
        if (target >= before && target < before + mine) {
            seen = ties_before;
            for (uint32_t i = a; i < b; i += 64) {
                u64 c = kept(i + lane, seen);
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const u64 v = __shfl_up(c, o);
                    if (lane >= (uint32_t)o) c += v;
                }
                const u64 hit = __ballot(before + c > target);
                if (hit) {
                    const uint32_t j = i + (uint32_t)__builtin_ctzll(hit);
                    if (lane == 0) {
                        index[row] = (int32_t)j;
                        if (logprob)
                            logprob[row] = (float)(((double)K.score(j) - (double)K.m) * K.r.rt - log((double)total / unit));
                    }
                    break;
                }
                before += __shfl(c, 63);
            }
        }
        __syncthreads();
    }
}

// Masses are sums of at most n weights of 1.
double unit_of(uint32_t n) {
    int b = 0;
    while ((1ull << b) < n) ++b;
    return std::ldexp(1.0, std::min(51, 62 - b));
}

template <class T>
int run_sample(const void* scores, uint64_t rows, uint32_t n, int64_t rs, int64_t cs, const Settings& S, int32_t* index,
               float* logprob, hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, n, rs, cs};
    const double unit = unit_of(n);
    if (n <= 2048) sample_kernel<T, 64><<<row_grid(rows), 64, 0, st>>>(X, S, unit, index, logprob);
    else sample_kernel<T, 1024><<<row_grid(rows), 1024, 0, st>>>(X, S, unit, index, logprob);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

}  // namespace

extern "C" uint64_t cbh_sample_classes_workspace(uint64_t rows, uint32_t classes) { return 0; }

extern "C" int cbh_sample_classes(const void* scores, int32_t type, uint64_t rows, uint32_t classes,
                                  int64_t row_stride, int64_t class_stride, const double* uniform, double temperature,
                                  const float* temperature_rows, uint32_t top_k, const int32_t* top_k_rows,
                                  double top_p, const float* top_p_rows, double min_p, const float* min_p_rows,
                                  const uint32_t* allowed, int64_t allowed_stride, int32_t* index, float* logprob,
                                  void* workspace, uint64_t workspace_bytes, void* stream) {
    try {
        const int rc = check_scores(scores, type, rows, classes, row_stride, class_stride);
        if (rc != CBH_OK) return rc;
        if (rows == 0) return CBH_OK;
        if (!uniform || !index) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "uniform and index are required");
        if (allowed && (uintptr_t)allowed % 4) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "allowed is not aligned to 4");
        if (allowed && allowed_stride != 0 && std::abs(allowed_stride) < ((int64_t)classes + 31) / 32)
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "allowed_stride must be 0 or at least ceil(classes / 32)");
        const uint64_t need = cbh_sample_classes_workspace(rows, classes);
        if (need > workspace_bytes || (need && (!workspace || (uintptr_t)workspace % 8)))
            return cbh_internal_fail(CBH_ERR_LENGTH_MISMATCH, "the workspace needs " + std::to_string(need) +
                                                                  " bytes, aligned to 8");
        const Settings S{uniform, temperature, top_p, min_p, top_k, temperature_rows, top_p_rows, min_p_rows,
                         top_k_rows, allowed, allowed_stride};
        hipStream_t st = (hipStream_t)stream;
        switch (type) {
            case CBH_TYPE_F32:
                return run_sample<float>(scores, rows, classes, row_stride, class_stride, S, index, logprob, st);
            case CBH_TYPE_F16:
                return run_sample<_Float16>(scores, rows, classes, row_stride, class_stride, S, index, logprob, st);
            default:
                return run_sample<bf16_t>(scores, rows, classes, row_stride, class_stride, S, index, logprob, st);
        }
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}
