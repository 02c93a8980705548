// One AdamW step over many tensors, in place, with states in 32 or 8 bits.
//
//   g = grad gs;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - m lr / (1 - b1^s) / (sqrt(v) / sqrt(1 - b2^s) + eps)
//
// Every value is read and written once: 60M f32 values with 8-bit states and bf16 gradients 165 us, 840 MB at 5.1 TB/s, a copy's rate; what
// it computes (a correctly rounded root and division, the hash, the codes: about 100 instructions a value) hides behind that.  It does not
// where weights have 16 bits too: 152 us, 600 MB at 4.0 TB/s.  150 tensors of 4M values: launches of 14 us (the 76 largest) and 8 us, and
// 90 us of a call from Python, which looks at 150 gradients, weights and their states.  8-bit states are m and sqrt(v) as e4m3 codes
// over a power of two that a block of 256 values shares: a wave takes a block, four values a lane.  sqrt(v), not v: the codes reach from
// 448 down to 2^-9, 18 binades, which are 36 of v.
#include <vector>

#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

constexpr uint32_t kBlock = 256;      // values that share a scale: a wave's
constexpr uint32_t kBlocks = 4;       // blocks a wave has in flight
constexpr uint32_t kTile = kBlock * kBlocks * 4;   // values of a workgroup's step

// Tensors of a launch: their addresses are kernel arguments (4 KB at most with the settings).
template <bool kSmall, bool kCopy>
struct Batch {
    static constexpr uint32_t N = kCopy ? 44 : kSmall ? 56 : 76;
    void* param[N];
    const void* grad[N];
    void* m[N];
    void* v[N];
    float* m_scale[kSmall ? N : 1];
    float* v_scale[kSmall ? N : 1];
    void* copy[kCopy ? N : 1];
    uint64_t n[N];
    uint32_t tiles[N];   // of this tensor and those before
    uint32_t number[N];
    uint32_t count;
    int32_t copy_type;
};
struct Factors {
    float decay, rate, root;   // 1 - lr wd, lr / (1 - b1^s), 1 / sqrt(1 - b2^s)
};
struct Step {
    double lr, beta1, beta2, weight_decay;
    float b1, a1, b2, a2, eps;   // a = 1 - b
    Factors f;
    uint32_t key;   // mix(seed ^ mix(step))
    uint32_t seed;
    const int64_t* step;
    const float* lr_device;
    const float* grad_scale;
    const int32_t* skip;
    int64_t step_host;
};

// b^s by squaring: the same on the host and on the device.
__host__ __device__ inline double power(double b, int64_t s) {
    double r = 1.0;
    for (; s > 0; s >>= 1) {
        if (s & 1) r *= b;
        b *= b;
    }
    return r;
}
__host__ __device__ inline Factors factors(double lr, double weight_decay, double beta1, double beta2, int64_t s) {
    return Factors{(float)(1.0 - lr * weight_decay), (float)(lr / (1.0 - power(beta1, s))),
                   (float)(1.0 / sqrt(1.0 - power(beta2, s)))};
}
// (the factors: the halves of Knuth's multiplier for 64 bits, 6364136223846793005)
__host__ __device__ inline uint32_t mix(uint32_t x) {
    x = (x ^ x >> 16) * 0x5851F42Du;
    x = (x ^ x >> 15) * 0x4C957F2Du;
    return x ^ x >> 16;
}

// ---- e4m3 --------------------------------------------------------------------------------------
// |x| times the block's inverse scale (at most 448), rounded up or down by 16 random bits.  Normal values: the bits that an f32
// has below the code's carry into it; below 2^-6: a multiple of 2^-9.  What comes out has a code, which the conversion
// then finds (NaN stays NaN).
__device__ __forceinline__ float round_code(float x, float inv, uint32_t random, bool least) {
    const float y = fabsf(x) * inv;
    const float small = truncf(y * 512.0f + (float)random * 0x1p-16f);
    const float large = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, y) + (random << 4)) & 0xFFF00000u);
    float c = y < 0x1p-6f ? (least ? fmaxf(small, 1.0f) : small) * 0x1p-9f : large;
    if (!(y > 0.0f)) c = 0.0f;
    if (!(fabsf(x) < INFINITY)) c = NAN;
    return c;
}
// The power of two that takes the block's largest finite value into (224, 448]; 0 below 2^-100.
__device__ __forceinline__ float block_scale(float largest) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, largest);
    const uint32_t e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000);
    return largest < 0x1p-100f ? 0.0f : __builtin_bit_cast(float, e << 23);
}
// Of a power of two, or 0 for 0.
__device__ __forceinline__ float inverse(float s) {
    return s > 0.0f ? __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, s)) : 0.0f;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.0f;
}

// ---- four values of a lane -----------------------------------------------------------------------
template <class T>
struct Words4 {   // four values in words
    static constexpr int N = (int)sizeof(T);
    typedef uint32_t Type __attribute__((ext_vector_type(N)));
    struct __attribute__((packed, aligned(sizeof(T)))) Any {
        Type w;
    };
};
template <>
struct Words4<uint8_t> {
    typedef uint32_t Type;
    struct __attribute__((packed, aligned(1))) Any {
        uint32_t w;
    };
};
template <class T>
struct Four {
    typename Words4<T>::Type w;
    __device__ __forceinline__ float get(int k) const {
        if constexpr (sizeof(T) == 4) {
            const uint32_t word = w[k];   // (the cast of a vector's element itself takes the first)
            return __builtin_bit_cast(float, word);
        } else if constexpr (sizeof(T) == 1) {
            return k == 0   ? __builtin_amdgcn_cvt_f32_fp8((int)w, 0)
                   : k == 1 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 1)
                   : k == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 2)
                            : __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
        } else {
            const uint32_t word = w[k / 2];
            if constexpr (__is_same(T, bf16_t)) return __builtin_bit_cast(float, k % 2 ? word & 0xFFFF0000u : word << 16);
            else return (float)__builtin_bit_cast(_Float16, (uint16_t)(word >> (k % 2 * 16)));
        }
    }
    // (8 bits: values that have a code)
    __device__ __forceinline__ void set(const float (&x)[4]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = __builtin_bit_cast(uint32_t, x[k]);
        } else if constexpr (sizeof(T) == 1) {
            int q = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
            w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], q, true);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k += 2)
                w[k / 2] = (uint32_t)__builtin_bit_cast(uint16_t, from_f32<T>(x[k])) |
                           (uint32_t)__builtin_bit_cast(uint16_t, from_f32<T>(x[k + 1])) << 16;
        }
    }
    // (kWhole: all four are there)
    template <bool kWhole>
    __device__ __forceinline__ void load(const T* p, uint64_t i, uint64_t n) {
        if constexpr (kWhole) {
            w = ((const typename Words4<T>::Any*)(p + i))->w;
        } else {
            T t[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = i + k < n ? p[i + k] : T{};
            w = __builtin_bit_cast(typename Words4<T>::Type, t);
        }
    }
    template <bool kWhole>
    __device__ __forceinline__ void store(T* p, uint64_t i, uint64_t n) const {
        if constexpr (kWhole) {
            ((typename Words4<T>::Any*)(p + i))->w = w;
        } else {
            struct Values {
                T v[4];
            };
            const Values t = __builtin_bit_cast(Values, w);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) p[i + k] = t.v[k];
        }
    }
};

// A wave's blocks: all loads under way before the first is waited for.
template <class P, class G, bool kSmall, bool kCopy, bool kWhole, int BLOCKS>
__device__ __forceinline__ void step_blocks(const Batch<kSmall, kCopy>& B, const Step& S, uint32_t t, uint64_t block0, uint64_t n) {
    using State = typename std::conditional<kSmall, uint8_t, float>::type;
    const uint32_t lane = lane_id();
    P* p = (P*)B.param[t];
    const G* g = (const G*)B.grad[t];
    State *m = (State*)B.m[t], *v = (State*)B.v[t];
    Four<P> qp[BLOCKS];
    Four<G> qg[BLOCKS];
    Four<State> qm[BLOCKS], qv[BLOCKS];
    float ms[BLOCKS], vs[BLOCKS];
#pragma unroll
    for (uint32_t b = 0; b < BLOCKS; ++b) {
        const uint64_t i = (block0 + b) * kBlock + lane * 4;
        qp[b].template load<kWhole>(p, i, n);
        qg[b].template load<kWhole>(g, i, n);
        qm[b].template load<kWhole>(m, i, n);
        qv[b].template load<kWhole>(v, i, n);
        if constexpr (kSmall) {
            ms[b] = B.m_scale[t][block0 + b];
            vs[b] = B.v_scale[t][block0 + b];
        }
    }
    Factors f = S.f;
    uint32_t key = S.key;
    if (S.step || S.lr_device) {
        const int64_t s = S.step ? *S.step : S.step_host;
        f = factors(S.lr_device ? (double)*S.lr_device : S.lr, S.weight_decay, S.beta1, S.beta2, s);
        key = mix(S.seed ^ mix((uint32_t)s));
    }
    key += B.number[t] * 0x9E3779B9u;
    const float gs = S.grad_scale ? *S.grad_scale : 1.0f;
#pragma unroll
    for (uint32_t b = 0; b < BLOCKS; ++b) {
        const uint64_t i = (block0 + b) * kBlock + lane * 4;
        float nm[4], nv[4], root[4], np[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float gk = qg[b].get(k);
            if (S.grad_scale) gk = gk * gs;
            float om = qm[b].get(k), ov = qv[b].get(k);
            if constexpr (kSmall) {
                om = om * ms[b];
                ov = ov * vs[b];
                ov = ov * ov;
            }
            nm[k] = om * S.b1 + gk * S.a1;
            nv[k] = ov * S.b2 + gk * gk * S.a2;
            root[k] = sqrtf(nv[k]);
            np[k] = qp[b].get(k) * f.decay - nm[k] * f.rate / (root[k] * f.root + S.eps);
        }
        qp[b].set(np);
        qp[b].template store<kWhole>(p, i, n);
        if constexpr (kCopy) {
            auto copy = [&](auto type) {
                Four<decltype(type)> q;
                q.set(np);
                q.template store<kWhole>((decltype(type)*)B.copy[t], i, n);
            };
            if (B.copy_type == CBH_TYPE_F32) copy(float{});
            else if (B.copy_type == CBH_TYPE_F16) copy(_Float16{});
            else copy(bf16_t{});
        }
        if constexpr (kSmall) {
            float lm = 0.0f, lv = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (kWhole || i + k < n) {
                    lm = fmaxf(lm, finite_abs(nm[k]));
                    lv = fmaxf(lv, finite_abs(root[k]));
                }
            const float sm = block_scale(wave_reduce(lm, MaxF())), sv = block_scale(wave_reduce(lv, MaxF()));
            const float im = inverse(sm), iv = inverse(sv);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t r = mix((uint32_t)(i + k) + key);
                nm[k] = copysignf(round_code(nm[k], im, r & 0xFFFF, false), nm[k]);
                nv[k] = round_code(root[k], iv, r >> 16, true);
            }
            if (lane == 0) {
                B.m_scale[t][block0 + b] = sm;
                B.v_scale[t][block0 + b] = sv;
            }
        }
        qm[b].set(nm);
        qv[b].set(nv);
        qm[b].template store<kWhole>(m, i, n);
        qv[b].template store<kWhole>(v, i, n);
    }
}

template <class P, class G, bool kSmall, bool kCopy>
__global__ __launch_bounds__(256) void adamw_kernel(Batch<kSmall, kCopy> B, Step S) {
    if (S.skip && *S.skip != 0) return;
    // the tensor of this tile (uniform)
    uint32_t t = 0;
    for (uint32_t hi = B.count - 1; t < hi;) {
        const uint32_t mid = (t + hi) / 2;
        if (blockIdx.x < B.tiles[mid]) hi = mid;
        else t = mid + 1;
    }
    const uint64_t n = B.n[t], tile = blockIdx.x - (t ? B.tiles[t - 1] : 0);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint64_t block0 = tile * (kTile / kBlock) + wave * kBlocks;
    if ((block0 + kBlocks) * kBlock <= n) {
        step_blocks<P, G, kSmall, kCopy, true, kBlocks>(B, S, t, block0, n);
    } else {   // the end of a tensor
#pragma unroll 1
        for (uint32_t b = 0; b < kBlocks && (block0 + b) * kBlock < n; ++b)
            step_blocks<P, G, kSmall, kCopy, false, 1>(B, S, t, block0 + b, n);
    }
}

// ---- host -----------------------------------------------------------------------------------
struct Run {   // tensors of one launch's types: collected until a launch is full
    const cbh_adamw_tensor* tensors;
    uint32_t count;
    const cbh_adamw_tensor& first;
    const Step& S;
    hipStream_t st;
    std::vector<char>& done;
};
template <class P, class G, bool kSmall, bool kCopy>
hipError_t launch_all(const Run& R) {
    Batch<kSmall, kCopy> B;
    B.count = 0;
    B.copy_type = R.first.copy_type;
    auto flush = [&] {
        if (!B.count) return hipSuccess;
        adamw_kernel<P, G, kSmall, kCopy><<<B.tiles[B.count - 1], 256, 0, R.st>>>(B, R.S);
        B.count = 0;
        return hipGetLastError();
    };
    for (uint32_t j = (uint32_t)(&R.first - R.tensors); j < R.count; ++j) {
        const cbh_adamw_tensor& t = R.tensors[j];
        if (R.done[j] || t.n == 0 || t.param_type != R.first.param_type || t.grad_type != R.first.grad_type || !t.copy != !kCopy ||
            (kCopy && t.copy_type != R.first.copy_type))
            continue;
        R.done[j] = 1;
        // (a launch holds fewer than 2^32 threads; a longer tensor takes several)
        constexpr uint64_t kMost = 1ull << 22;
        const uint64_t all = (t.n + kTile - 1) / kTile;
        for (uint64_t at = 0; at < all; at += kMost) {
            const uint64_t tiles = std::min(kMost, all - at), off = at * kTile;
            if (B.count == B.N || (B.count && B.tiles[B.count - 1] + tiles > kMost)) {
                const hipError_t e = flush();
                if (e != hipSuccess) return e;
            }
            const uint32_t c = B.count++;
            const size_t s = kSmall ? 1 : 4;
            B.param[c] = (char*)t.param + off * sizeof(P);
            B.grad[c] = (const char*)t.grad + off * sizeof(G);
            B.m[c] = (char*)t.exp_avg + off * s;
            B.v[c] = (char*)t.exp_avg_sq + off * s;
            if constexpr (kSmall) {
                B.m_scale[c] = t.exp_avg_scale + off / kBlock;
                B.v_scale[c] = t.exp_avg_sq_scale + off / kBlock;
            }
            if constexpr (kCopy) B.copy[c] = (char*)t.copy + off * type_bytes(t.copy_type);
            B.n[c] = std::min<uint64_t>(t.n - off, tiles * kTile);
            B.tiles[c] = (c ? B.tiles[c - 1] : 0) + (uint32_t)tiles;
            B.number[c] = t.number;   // (a value's place counts modulo 2^32, which divides off)
        }
    }
    return flush();
}
template <class P, class G>
hipError_t launch_all(const Run& R, int32_t state) {
    if (state == CBH_STATE_F8) return R.first.copy ? launch_all<P, G, true, true>(R) : launch_all<P, G, true, false>(R);
    return R.first.copy ? launch_all<P, G, false, true>(R) : launch_all<P, G, false, false>(R);
}
template <class P>
hipError_t launch_all(const Run& R, int32_t state) {
    return R.first.grad_type == CBH_TYPE_F32   ? launch_all<P, float>(R, state)
           : R.first.grad_type == CBH_TYPE_F16 ? launch_all<P, _Float16>(R, state)
                                               : launch_all<P, bf16_t>(R, state);
}

bool is_type(int32_t t) { return t == CBH_TYPE_F32 || t == CBH_TYPE_F16 || t == CBH_TYPE_BF16; }
int invalid(const char* what) { return cbh_internal_fail(CBH_ERR_INVALID_ARG, what); }

struct Span {
    uintptr_t from, to;
};
int check_tensor(const cbh_adamw_tensor& t, int32_t state, std::vector<Span>& written) {
    if (t.n == 0) return CBH_OK;
    if (t.n > 1ull << 40) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "more than 2^40 values of a tensor");
    if (!is_type(t.param_type) || !is_type(t.grad_type) || (t.copy && !is_type(t.copy_type)))
        return cbh_internal_fail(CBH_ERR_UNSUPPORTED, "parameters, gradients and copies are f32, f16 or bf16");
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return invalid("a tensor's address is null");
    if (state == CBH_STATE_F8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return invalid("a state's scales are null");
    const size_t s = state == CBH_STATE_F8 ? 1 : 4;
    if ((uintptr_t)t.param % type_bytes(t.param_type) || (uintptr_t)t.grad % type_bytes(t.grad_type) ||
        (uintptr_t)t.exp_avg % s || (uintptr_t)t.exp_avg_sq % s || (t.copy && (uintptr_t)t.copy % type_bytes(t.copy_type)))
        return invalid("a tensor is not aligned to its type");
    auto span = [&](const void* p, size_t bytes) { written.push_back({(uintptr_t)p, (uintptr_t)p + bytes}); };
    span(t.param, t.n * type_bytes(t.param_type));
    span(t.exp_avg, t.n * s);
    span(t.exp_avg_sq, t.n * s);
    if (state == CBH_STATE_F8) {
        if ((uintptr_t)t.exp_avg_scale % 4 || (uintptr_t)t.exp_avg_sq_scale % 4) return invalid("a state's scales are not aligned to 4");
        span(t.exp_avg_scale, (t.n + kBlock - 1) / kBlock * 4);
        span(t.exp_avg_sq_scale, (t.n + kBlock - 1) / kBlock * 4);
    }
    if (t.copy) span(t.copy, t.n * type_bytes(t.copy_type));
    return CBH_OK;
}

}  // namespace

extern "C" int cbh_adamw_step(const cbh_adamw_tensor* tensors, uint32_t count, const cbh_adamw_settings* settings, void* stream) {
    try {
        if (!settings || (count && !tensors)) return invalid("tensors or settings are null");
        const cbh_adamw_settings& A = *settings;
        if (A.state != CBH_STATE_F32 && A.state != CBH_STATE_F8)
            return cbh_internal_fail(CBH_ERR_UNSUPPORTED, "states are of 32 bits or of 8");
        if (!(A.beta1 >= 0.0 && A.beta1 < 1.0 && A.beta2 >= 0.0 && A.beta2 < 1.0))
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "betas must be in [0, 1)");
        if (!(A.eps >= 0.0 && A.eps <= 3.4e38) || !(std::abs(A.weight_decay) <= 3.4e38) || (!A.lr_device && !(std::abs(A.lr) <= 3.4e38)))
            return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "lr, eps and weight_decay must be finite");
        if (!A.step_device && A.step < 1) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "steps count from 1");
        if ((uintptr_t)A.step_device % 8 || (uintptr_t)A.lr_device % 4 || (uintptr_t)A.grad_scale % 4 || (uintptr_t)A.skip % 4)
            return invalid("a setting's address is not aligned to its type");
        std::vector<Span> written;
        written.reserve(count * 6);
        for (uint32_t i = 0; i < count; ++i) {
            const int rc = check_tensor(tensors[i], A.state, written);
            if (rc != CBH_OK) return rc;
        }
        std::sort(written.begin(), written.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
        for (size_t i = 1; i < written.size(); ++i)
            if (written[i].from < written[i - 1].to) return invalid("tensors that are written overlap");
        for (uint32_t i = 0; i < count; ++i) {
            if (tensors[i].n == 0) continue;
            const uintptr_t from = (uintptr_t)tensors[i].grad, to = from + tensors[i].n * type_bytes(tensors[i].grad_type);
            const auto next = std::lower_bound(written.begin(), written.end(), to, [](const Span& a, uintptr_t at) { return a.from < at; });
            if (next != written.begin() && next[-1].to > from) return invalid("a gradient overlaps a tensor that is written");
        }

        Step S{};
        S.lr = A.lr, S.beta1 = A.beta1, S.beta2 = A.beta2, S.weight_decay = A.weight_decay;
        S.b1 = (float)A.beta1, S.a1 = (float)(1.0 - A.beta1), S.b2 = (float)A.beta2, S.a2 = (float)(1.0 - A.beta2);
        S.eps = (float)A.eps;
        S.seed = A.seed;
        S.step = A.step_device, S.lr_device = A.lr_device, S.grad_scale = A.grad_scale, S.skip = A.skip;
        S.step_host = A.step;
        S.f = factors(A.lr, A.weight_decay, A.beta1, A.beta2, A.step);
        S.key = mix(A.seed ^ mix((uint32_t)A.step));
        // tensors of the same types share launches
        std::vector<char> done(count, 0);
        for (uint32_t i = 0; i < count; ++i) {
            if (done[i] || tensors[i].n == 0) continue;
            const Run R{tensors, count, tensors[i], S, (hipStream_t)stream, done};
            const int32_t type = tensors[i].param_type;
            CLS_TRY(type == CBH_TYPE_F32   ? launch_all<float>(R, A.state)
                    : type == CBH_TYPE_F16 ? launch_all<_Float16>(R, A.state)
                                           : launch_all<bf16_t>(R, A.state));
        }
        return CBH_OK;
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}
