// One AdamW step over many tensors, in place, with states in 32 or 8 bits.
//
//   g = grad gs;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - m lr / (1 - b1^s) / (sqrt(v) / sqrt(1 - b2^s) + eps)
//
// Every value is read and written once.  8-bit states are m and sqrt(v) as e4m3 codes over a power of two that a
// block of 256 values shares: a wave takes a block, four values a lane.  sqrt(v), not v: the codes reach from 448 down to 2^-9, 18
// binades, which are 36 of v.
#include <vector>

#include "class_scores.hpp"

namespace {
using namespace cbh::cls;

constexpr uint32_t kBlock = 256;      // values that share a scale: a wave's
constexpr uint32_t kBlocks = 4;       // blocks a wave has in flight
constexpr uint32_t kTile = kBlock * kBlocks * 4;   // values of a workgroup's step
constexpr uint32_t kBatch = 44;       // tensors of a launch: their addresses are kernel arguments (4 KB at most)

struct Batch {
    void* param[kBatch];
    const void* grad[kBatch];
    void* m[kBatch];
    void* v[kBatch];
    float* m_scale[kBatch];
    float* v_scale[kBatch];
    void* copy[kBatch];
    uint64_t n[kBatch];
    uint64_t tiles[kBatch];   // of this tensor and those before
    uint32_t number[kBatch];
    uint32_t count;
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
__host__ __device__ inline uint32_t mix(uint32_t x) {
    x = (x ^ x >> 16) * 0x5851F42Du;
    x = (x ^ x >> 15) * 0x4C957F2Du;
    return x ^ x >> 16;
}

// ---- e4m3 --------------------------------------------------------------------------------------
__device__ __forceinline__ float from_code(uint32_t c) {
    const uint32_t u = c & 0x7F;
    // normal codes are the top bits of an f32 with another exponent bias; below, multiples of 2^-9
    float x = u >= 8 ? __builtin_bit_cast(float, (u + (120u << 3)) << 20) : (float)u * 0x1p-9f;
    x = u == 0x7F ? NAN : x;
    return c & 0x80 ? -x : x;
}
// |x| times the block's inverse scale (at most 448), rounded up or down by 16 random bits.
__device__ __forceinline__ uint32_t to_code(float x, float inv, uint32_t random, bool least) {
    const float y = fabsf(x) * inv;
    uint32_t c;
    if (y < 0x1p-6f) c = (uint32_t)(y * 512.0f + (float)random * 0x1p-16f);
    else c = ((__builtin_bit_cast(uint32_t, y) + (random << 4)) >> 20) - (120u << 3);
    if (least) c = x > 0.0f ? max(c, 1u) : c;
    c = y > 0.0f ? c : 0;
    if (!(fabsf(x) < INFINITY)) c = 0x7F;
    return c | (x < 0.0f ? 0x80u : 0u);
}
// The power of two that takes the block's largest finite value into (224, 448]; 0 below 2^-100.
__device__ __forceinline__ float block_scale(float largest) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, largest);
    const uint32_t e = (bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000);
    return largest < 0x1p-100f ? 0.0f : __builtin_bit_cast(float, e << 23);
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.0f;
}

// ---- four values of a lane -----------------------------------------------------------------------
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T v[4];
};
template <class T>
__device__ __forceinline__ void load4(const T* p, uint64_t i, uint64_t n, Four<T>& q) {
    if (i + 4 <= n) {
        q = *(const Four<T>*)(p + i);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) q.v[k] = i + k < n ? p[i + k] : T{};
    }
}
template <class T>
__device__ __forceinline__ void store4(T* p, uint64_t i, uint64_t n, const Four<T>& q) {
    if (i + 4 <= n) {
        *(Four<T>*)(p + i) = q;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k < n) p[i + k] = q.v[k];
    }
}
template <class T>
__device__ __forceinline__ void store_copy(void* copy, uint64_t i, uint64_t n, const float (&x)[4]) {
    Four<T> q;
#pragma unroll
    for (int k = 0; k < 4; ++k) q.v[k] = from_f32<T>(x[k]);
    store4((T*)copy, i, n, q);
}

template <class P, class G, bool kSmall>
__global__ __launch_bounds__(256) void adamw_kernel(Batch B, Step S, int32_t copy_type) {
    using State = typename std::conditional<kSmall, uint8_t, float>::type;
    if (S.skip && *S.skip != 0) return;
    // the tensor of this tile (uniform)
    uint32_t t = 0;
    for (uint32_t hi = B.count - 1; t < hi;) {
        const uint32_t mid = (t + hi) / 2;
        if (blockIdx.x < B.tiles[mid]) hi = mid;
        else t = mid + 1;
    }
    const uint64_t n = B.n[t], tile = blockIdx.x - (t ? B.tiles[t - 1] : 0);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = lane_id();
    const uint64_t block0 = tile * (kTile / kBlock) + wave * kBlocks;
    P* p = (P*)B.param[t];
    const G* g = (const G*)B.grad[t];
    State *m = (State*)B.m[t], *v = (State*)B.v[t];
    Four<P> qp[kBlocks];
    Four<G> qg[kBlocks];
    Four<State> qm[kBlocks], qv[kBlocks];
    float ms[kBlocks], vs[kBlocks];
#pragma unroll
    for (uint32_t b = 0; b < kBlocks; ++b) {
        const uint64_t i = (block0 + b) * kBlock + lane * 4;
        load4(p, i, n, qp[b]);
        load4(g, i, n, qg[b]);
        load4(m, i, n, qm[b]);
        load4(v, i, n, qv[b]);
        if constexpr (kSmall) {
            const bool have = (block0 + b) * kBlock < n;
            ms[b] = have ? B.m_scale[t][block0 + b] : 0.0f;
            vs[b] = have ? B.v_scale[t][block0 + b] : 0.0f;
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
    for (uint32_t b = 0; b < kBlocks; ++b) {
        const uint64_t i = (block0 + b) * kBlock + lane * 4;
        if ((block0 + b) * kBlock >= n) break;
        float nm[4], nv[4], root[4], np[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float gk = to_f32(qg[b].v[k]);
            if (S.grad_scale) gk = gk * gs;
            float om, ov;
            if constexpr (kSmall) {
                om = from_code(qm[b].v[k]) * ms[b];
                ov = from_code(qv[b].v[k]) * vs[b];
                ov = ov * ov;
            } else {
                om = qm[b].v[k];
                ov = qv[b].v[k];
            }
            nm[k] = om * S.b1 + gk * S.a1;
            nv[k] = ov * S.b2 + gk * gk * S.a2;
            root[k] = sqrtf(nv[k]);
            np[k] = to_f32(qp[b].v[k]) * f.decay - nm[k] * f.rate / (root[k] * f.root + S.eps);
            qp[b].v[k] = from_f32<P>(np[k]);
        }
        store4(p, i, n, qp[b]);
        if (B.copy[t]) {
            if (copy_type == CBH_TYPE_F32) store_copy<float>(B.copy[t], i, n, np);
            else if (copy_type == CBH_TYPE_F16) store_copy<_Float16>(B.copy[t], i, n, np);
            else store_copy<bf16_t>(B.copy[t], i, n, np);
        }
        if constexpr (kSmall) {
            float lm = 0.0f, lv = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) {
                    lm = fmaxf(lm, finite_abs(nm[k]));
                    lv = fmaxf(lv, finite_abs(root[k]));
                }
            const float sm = block_scale(wave_reduce(lm, MaxF())), sv = block_scale(wave_reduce(lv, MaxF()));
            const float im = sm > 0.0f ? 1.0f / sm : 0.0f, iv = sv > 0.0f ? 1.0f / sv : 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t r = mix((uint32_t)(i + k) + key);
                qm[b].v[k] = (uint8_t)to_code(nm[k], im, r & 0xFFFF, false);
                qv[b].v[k] = (uint8_t)to_code(root[k], iv, r >> 16, true);
            }
            if (lane == 0) {
                B.m_scale[t][block0 + b] = sm;
                B.v_scale[t][block0 + b] = sv;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                qm[b].v[k] = nm[k];
                qv[b].v[k] = nv[k];
            }
        }
        store4(m, i, n, qm[b]);
        store4(v, i, n, qv[b]);
    }
}

// ---- host -----------------------------------------------------------------------------------
using Launch = void (*)(const Batch&, const Step&, int32_t, unsigned, hipStream_t);
template <class P, class G, bool kSmall>
void launch(const Batch& B, const Step& S, int32_t copy_type, unsigned grid, hipStream_t st) {
    adamw_kernel<P, G, kSmall><<<grid, 256, 0, st>>>(B, S, copy_type);
}
template <class P, class G>
Launch pick(int32_t state) {
    return state == CBH_STATE_F8 ? launch<P, G, true> : launch<P, G, false>;
}
template <class P>
Launch pick(int32_t grad, int32_t state) {
    return grad == CBH_TYPE_F32 ? pick<P, float>(state) : grad == CBH_TYPE_F16 ? pick<P, _Float16>(state) : pick<P, bf16_t>(state);
}
Launch pick(int32_t param, int32_t grad, int32_t state) {
    return param == CBH_TYPE_F32 ? pick<float>(grad, state)
                                 : param == CBH_TYPE_F16 ? pick<_Float16>(grad, state) : pick<bf16_t>(grad, state);
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
            const cbh_adamw_tensor& a = tensors[i];
            const int32_t copy_type = a.copy ? a.copy_type : CBH_TYPE_F32;
            const Launch run = pick(a.param_type, a.grad_type, A.state);
            Batch B;
            B.count = 0;
            auto flush = [&] {
                if (!B.count) return hipSuccess;
                run(B, S, copy_type, (unsigned)B.tiles[B.count - 1], (hipStream_t)stream);
                B.count = 0;
                return hipGetLastError();
            };
            for (uint32_t j = i; j < count; ++j) {
                const cbh_adamw_tensor& t = tensors[j];
                if (done[j] || t.n == 0 || t.param_type != a.param_type || t.grad_type != a.grad_type ||
                    (t.copy ? t.copy_type : copy_type) != copy_type)
                    continue;
                done[j] = 1;
                // (a launch holds fewer than 2^32 threads; a longer tensor takes several)
                constexpr uint64_t kMost = 1ull << 22;
                const uint64_t all = (t.n + kTile - 1) / kTile;
                for (uint64_t at = 0; at < all; at += kMost) {
                    const uint64_t tiles = std::min(kMost, all - at), off = at * kTile;
                    if (B.count == kBatch || (B.count && B.tiles[B.count - 1] + tiles > kMost)) CLS_TRY(flush());
                    const uint32_t c = B.count++;
                    B.param[c] = (char*)t.param + off * type_bytes(t.param_type);
                    B.grad[c] = (const char*)t.grad + off * type_bytes(t.grad_type);
                    const size_t s = A.state == CBH_STATE_F8 ? 1 : 4;
                    B.m[c] = (char*)t.exp_avg + off * s;
                    B.v[c] = (char*)t.exp_avg_sq + off * s;
                    B.m_scale[c] = t.exp_avg_scale ? t.exp_avg_scale + off / kBlock : nullptr;
                    B.v_scale[c] = t.exp_avg_sq_scale ? t.exp_avg_sq_scale + off / kBlock : nullptr;
                    B.copy[c] = t.copy ? (char*)t.copy + off * type_bytes(t.copy_type) : nullptr;
                    B.n[c] = std::min<uint64_t>(t.n - off, tiles * kTile);
                    B.tiles[c] = (c ? B.tiles[c - 1] : 0) + tiles;
                    B.number[c] = t.number;   // (a value's place counts modulo 2^32, which divides off)
                }
            }
            CLS_TRY(flush());
        }
        return CBH_OK;
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}
