// Shared parts of the operators on class scores (class_top.hip, class_distill.hip,
// class_sample.hip): reading rows of scores in any of the three types and any strides, keys
// that order scores, and sums over a wave or a workgroup.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/cbhip.h"

int cbh_internal_fail(int code, const std::string& msg);  // session.hip

namespace cbh {
namespace cls {

typedef unsigned long long u64;

constexpr float kLowest = -3.402823466e38f;   // the lowest finite f32
constexpr uint32_t kMaxClasses = 1u << 24;

// ---- element types: f32, IEEE half, bfloat16 ------------------------------------------------
struct bf16_t {
    uint16_t bits;
};
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __builtin_bit_cast(float, (uint32_t)x.bits << 16); }
template <class T>
__device__ __forceinline__ T from_f32(float x);   // round to nearest even
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float x) { return (_Float16)x; }
template <>
__device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) {
    return __builtin_bit_cast(bf16_t, (__bf16)x);
}

// One vector load or store moves 16 bytes; the address needs the element's alignment only (rows of odd
// length start anywhere).
// A vector stays in its four words until a score of it is used: as separate 16-bit values the compiler gives each
// a register.
typedef uint32_t Words __attribute__((ext_vector_type(4)));
template <class T>
struct Pack {
    static constexpr int V = 16 / (int)sizeof(T);
    Words w;
    __device__ __forceinline__ float get(int v) const {
        const uint32_t word = w[v * (int)sizeof(T) / 4];
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, word);
        else if constexpr (__is_same(T, bf16_t)) return __builtin_bit_cast(float, v % 2 ? word & 0xFFFF0000u : word << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)(word >> (v % 2 * 16)));
    }
    __device__ __forceinline__ void set(const float (&x)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int v = 0; v < V; ++v) w[v] = __builtin_bit_cast(uint32_t, x[v]);
        } else {
#pragma unroll
            for (int v = 0; v < V; v += 2)
                w[v / 2] = (uint32_t)__builtin_bit_cast(uint16_t, from_f32<T>(x[v])) |
                           (uint32_t)__builtin_bit_cast(uint16_t, from_f32<T>(x[v + 1])) << 16;
        }
    }
};
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    Words w;
};

// Scores as the kernels take them.
template <class T>
struct Rows {
    const T* data;
    uint64_t rows;
    uint32_t classes;
    int64_t rs, cs;   // strides in elements
};

// The V scores from class i on, as f32; classes at n and beyond read as `fill`.
template <class T, bool kUnit>
__device__ __forceinline__ void load_pack(const T* row, int64_t cs, uint32_t i, uint32_t n, float fill,
                                          float (&x)[Pack<T>::V]) {
    constexpr int V = Pack<T>::V;
    if (kUnit && i + V <= n) {
        const Pack<T> p{((const Loose<T>*)(row + i))->w};
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = p.get(v);
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            x[v] = i + (uint32_t)v < n ? to_f32(row[kUnit ? (int64_t)(i + v) : (int64_t)(i + v) * cs]) : fill;
    }
}
// A wave's 2048 classes from `base` on (a multiple of 2048, the same in all lanes): vector u of a lane holds
// the classes from base + (u 64 + lane) V on.  The loads of a whole tile are all under way before the first is
// waited for (guarded one by one, each was waited for in its branch: 203 against 175 us for the top classes of
// 4096 x 65536 bf16).
constexpr uint32_t kSeg = 2048, kGroup = 32;   // classes of a wave's tile, and of a lane in it
template <class T>
constexpr int kPacks = (int)kGroup / Pack<T>::V;
template <class T, bool kUnit>
__device__ __forceinline__ void load_tile(const T* row, int64_t cs, uint32_t base, uint32_t n, float fill,
                                          Pack<T> (&p)[kPacks<T>]) {
    constexpr int V = Pack<T>::V, U = kPacks<T>;
    const uint32_t lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    if (kUnit && base + kSeg <= n) {
        const Loose<T>* at = (const Loose<T>*)(row + base + lane * V);
#pragma unroll
        for (int u = 0; u < U; ++u) p[u].w = at[u * 64].w;
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[V];
            load_pack<T, kUnit>(row, cs, base + (u * 64 + lane) * V, n, fill, x);
            p[u].set(x);
        }
    }
}
template <class T, bool kUnit>
__device__ __forceinline__ void load_tile(const T* row, int64_t cs, uint32_t base, uint32_t n, float fill,
                                          float (&x)[kPacks<T>][Pack<T>::V]) {
    Pack<T> p[kPacks<T>];
    load_tile<T, kUnit>(row, cs, base, n, fill, p);
#pragma unroll
    for (int u = 0; u < kPacks<T>; ++u)
#pragma unroll
        for (int v = 0; v < Pack<T>::V; ++v) x[u][v] = p[u].get(v);
}
template <class T, bool kUnit>
__device__ __forceinline__ void store_pack(T* row, int64_t cs, uint32_t i, uint32_t n, const float (&x)[Pack<T>::V]) {
    constexpr int V = Pack<T>::V;
    if (kUnit && i + V <= n) {
        Pack<T> p;
        p.set(x);
        // (past the caches: nobody reads a gradient before the pass ends, and the rows' second read shares them)
        typedef uint32_t Unaligned __attribute__((ext_vector_type(4), aligned(2)));
        __builtin_nontemporal_store(p.w, (Unaligned*)(row + i));
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (i + (uint32_t)v < n) row[kUnit ? (int64_t)(i + v) : (int64_t)(i + v) * cs] = from_f32<T>(x[v]);
    }
}

// ---- order of scores ------------------------------------------------------------------------
// A u32 that orders as the score does: -0 and +0 alike, NaN (of either sign) above +inf.
__device__ __forceinline__ uint32_t order_key(float x) {
    x = x + 0.0f;   // -0 -> +0
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    u = x != x ? 0x7FC00000u : u;
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// Larger for the larger score, and for the lower class among equal ones; never 0.
__device__ __forceinline__ u64 rank_key(float x, uint32_t cls) { return ((u64)order_key(x) << 32) | (uint32_t)~cls; }

// ---- waves and workgroups -------------------------------------------------------------------
__device__ __forceinline__ uint32_t lane_id() { return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }

// What the lanes of a wave have written to LDS is seen by its other lanes.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A value from another lane by a data-parallel-primitive move (a register access, where a shuffle is a round
// trip through LDS); lanes without a source get `none`.
template <int kCtrl, int kRows, class V>
__device__ __forceinline__ V dpp_move(V v, V none) {
    static_assert(sizeof(V) == 4 || sizeof(V) == 8, "moved in words of 32 bits");
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v),
                                                                 kCtrl, kRows, 0xf, false));
    } else {
        const u64 a = __builtin_bit_cast(u64, v), b = __builtin_bit_cast(u64, none);
        const uint32_t lo = __builtin_amdgcn_update_dpp((int)(uint32_t)b, (int)(uint32_t)a, kCtrl, kRows, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp((int)(b >> 32), (int)(a >> 32), kCtrl, kRows, 0xf, false);
        return __builtin_bit_cast(V, (u64)hi << 32 | lo);
    }
}
// Inclusive scan over the lanes, `none` the operation's neutral value: rows of 16 lanes, then across them.
template <class V, class Op>
__device__ __forceinline__ V wave_scan(V v, Op op, V none) {
    v = op(dpp_move<0x111, 0xf>(v, none), v);   // from 1, 2, 4, 8 lanes below, within the row
    v = op(dpp_move<0x112, 0xf>(v, none), v);
    v = op(dpp_move<0x114, 0xf>(v, none), v);
    v = op(dpp_move<0x118, 0xf>(v, none), v);
    v = op(dpp_move<0x142, 0xa>(v, none), v);   // lane 15 of the row below to rows 1 and 3
    v = op(dpp_move<0x143, 0xc>(v, none), v);   // lane 31 to rows 2 and 3
    return v;
}
// (of a wave-uniform lane)
template <class V>
__device__ __forceinline__ V read_lane(V v, int lane) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        const u64 a = __builtin_bit_cast(u64, v);
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)a, lane);
        const uint32_t hi = __builtin_amdgcn_readlane((int)(a >> 32), lane);
        return __builtin_bit_cast(V, (u64)hi << 32 | lo);
    }
}
template <class V, class Op>
__device__ __forceinline__ V wave_reduce(V v, Op op) {
    return read_lane(wave_scan(v, op, op.template none<V>()), 63);
}
// Reduction over a workgroup, in a fixed order; every thread gets it.  `tmp` holds a value a wave; the
// call ends with a barrier after which tmp may be used again.
template <int THREADS, class V, class Op>
__device__ __forceinline__ V block_reduce(V v, Op op, V* tmp) {
    v = wave_reduce(v, op);
    if (THREADS == 64) return v;
    if (lane_id() == 0) tmp[threadIdx.x / 64] = v;
    __syncthreads();
    V r = tmp[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) r = op(r, tmp[w]);
    __syncthreads();
    return r;
}
struct Add {
    template <class V>
    __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
    template <class V>
    __device__ __forceinline__ V none() const { return V(0); }
};
struct MaxF {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return fmax(a, b); }
    template <class V>
    __device__ __forceinline__ V none() const { return -(V)INFINITY; }
};
struct MaxU {
    template <class V>
    __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
    template <class V>
    __device__ __forceinline__ V none() const { return V(0); }
};
struct MinU {
    template <class V>
    __device__ __forceinline__ V operator()(V a, V b) const { return a < b ? a : b; }
    template <class V>
    __device__ __forceinline__ V none() const { return ~V(0); }
};

// The largest of 32 classes next to each other (a group), from the maxima of a lane's vectors: vector u of 32 / V
// lanes side by side is a group.  Lane l gets that of group group_of<V>(l) of the tile, which holds the classes
// [32 g, 32 g + 32): what is read again of a group is one run of memory.
template <int V>
__device__ __forceinline__ uint32_t group_of(uint32_t lane) {
    constexpr uint32_t L = kGroup / V;
    return lane % L * (64 / L) + lane / L;
}
template <int V, class K, class Op>
__device__ __forceinline__ K group_max(const K (&vm)[kGroup / V], uint32_t lane, Op op) {
    constexpr int L = (int)kGroup / V;   // lanes of a group, and vectors of a lane
    K out = vm[0];
#pragma unroll
    for (int u = 0; u < L; ++u) {
        K k = vm[u];
        k = op(k, dpp_move<0xB1, 0xf>(k, k));                    // lanes 1 0 3 2
        k = op(k, dpp_move<0x4E, 0xf>(k, k));                    // lanes 2 3 0 1
        if constexpr (L == 8) k = op(k, dpp_move<0x141, 0xf>(k, k));   // mirrored within 8
        out = lane % L == (uint32_t)u ? k : out;
    }
    return out;
}

// Where a sum over 256 bins in LDS, taken from bin 255 down, reaches `want`: the bin, what lies above it
// and what it holds (the lowest non-zero place if the sum stays below).  Every wave finds it by itself: lane l
// holds bins 255 - 4 l .. 252 - 4 l.  (Walked bin by bin with wave-uniform 64-bit sums, hipcc 7.2 selected
// the next sum by a stale condition code.)
template <class V>
struct Found {
    uint32_t bin;
    V above, inside;
};
template <class V>
__device__ __forceinline__ Found<V> find_bin(const V* hist, V want) {
    const uint32_t l = lane_id();
    V c[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        c[j] = hist[255 - 4 * l - j];
        sum += c[j];
    }
    const V upto = wave_scan(sum, Add(), V(0));
    V above = upto - sum, inside = c[0];
    uint32_t b = 255 - 4 * l;
    const u64 cross = __ballot(upto >= want);
    const int at = cross ? __builtin_ctzll(cross) : 63;
#pragma unroll
    for (int j = 1; j < 4; ++j)
        if (above + inside < want) {
            above += inside;
            inside = c[j];
            --b;
        }
    return Found<V>{read_lane(b, at), read_lane(above, at), read_lane(inside, at)};
}

struct CountLds {
    u64 tmp[16], top[16];
    uint32_t count[256];
};
struct SelectLds : CountLds {
    u64 mass[256];   // (digits; or the entries of a short list)
    u64 rank[128], weight[128];
    uint32_t place[128];
};
// The bits of a rank's distance that are known before the digit at `shift`: from here up.
__device__ __forceinline__ int prefix_shift(int shift, int bits) {
    return shift == max(0, bits - 8) ? bits : shift == 0 ? (bits % 8 ? bits % 8 : 8) : shift + 8;
}
struct Crossing {
    u64 from;    // ranks from here on are in the prefix
    u64 last;    // and the lowest of them that may be there: the crossing entry's is in [from, last]
};

// Entries have ranks and weights: 1, or their mass (ranks are then all different).  Taken from the largest rank down, where do
// the weights reach `want` (at most their sum)?  By digits of 8 bits of the ranks' distance from the lowest one, from
// the highest bit that it has (the ranks of a list share their leading bits: as digits, every one of their atomics
// would meet in one cell); done as soon as one entry is left, or (kWhole) the ones left are all needed.
template <int THREADS, bool kMass, bool kWhole, class ForEach, class Lds>
__device__ __forceinline__ Crossing select(ForEach for_each, u64 want, Lds* lds) {
    u64 lo = ~0ull, hi = 0;
    for_each([&](u64 rank, u64) {
        lo = rank < lo ? rank : lo;
        hi = rank > hi ? rank : hi;
    });
    lo = ~wave_reduce(~lo, MaxU());
    hi = wave_reduce(hi, MaxU());
    if (THREADS > 64) {
        if (lane_id() == 0) {
            lds->tmp[threadIdx.x / 64] = lo;
            lds->top[threadIdx.x / 64] = hi;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) {
            lo = lds->tmp[w] < lo ? lds->tmp[w] : lo;
            hi = lds->top[w] > hi ? lds->top[w] : hi;
        }
    }
    const int bits = hi > lo ? 64 - __builtin_clzll(hi - lo) : 0;
    u64 prefix = 0;
    for (int shift = max(0, bits - 8); ; shift = max(0, shift - 8)) {
        // (the last digit may repeat bits of the one before: those are equal among the entries left)
        const int known = prefix_shift(shift, bits);
        for (uint32_t b = threadIdx.x; b < 256; b += THREADS) {
            lds->count[b] = 0;
            if constexpr (kMass) lds->mass[b] = 0;
        }
        __syncthreads();
        for_each([&](u64 rank, u64 mass) {
            const u64 d = rank - lo;
            if (known < bits && (d >> known) != (prefix >> known)) return;
            atomicAdd(&lds->count[d >> shift & 255], 1u);
            if constexpr (kMass) atomicAdd(&lds->mass[d >> shift & 255], mass);
        });
        __syncthreads();
        bool done;
        if constexpr (kMass) {
            const Found<u64> f = find_bin(lds->mass, want);
            prefix = (prefix & ~(255ull << shift)) | (u64)f.bin << shift;
            want -= f.above;
            done = lds->count[f.bin] <= 1 || (kWhole && f.inside == want);
        } else {
            const Found<uint32_t> f = find_bin(lds->count, (uint32_t)want);
            prefix = (prefix & ~(255ull << shift)) | (u64)f.bin << shift;
            want -= f.above;
            done = f.inside <= 1 || (kWhole && f.inside == want);
        }
        done = __builtin_amdgcn_readfirstlane((uint32_t)done) != 0 || shift == 0;
        __syncthreads();
        if (done) return Crossing{lo + prefix, lo + (prefix | ((1ull << shift) - 1))};
    }
}

// A bound that the k largest of the keys get(0 .. n - 1) reach and, unless there are equal ones, no others (0: no key;
// at least k are not 0).
template <int THREADS, class Get, class Lds>
__device__ __forceinline__ u64 kth_of(Get get, uint32_t n, uint32_t k, Lds* lds) {
    return select<THREADS, false, true>(
               [&](auto f) {
                   for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                       const u64 key = get(i);
                       if (key) f(key, 0);
                   }
               },
               k, lds)
        .from;
}

// (2^f - 1) / f for |f| <= 1/2 as a polynomial of degree 8, lowest term first: it meets the function in the Chebyshev
// points of the interval; 1 + f q(f) is 2^f within 2^-44, and exactly 1 at 0.
#define CBH_EXP2_TERMS                                                                            \
    0.6931471805599453, 0.2402265069581299, 0.055504108664760424,                   \
        0.009618129159402558, 0.0013333558179043112, 0.00015403455852453838,           \
        1.525268684626772e-05, 1.3255224878668817e-06, 1.0203121063391729e-07
// e^z within 2^-43, for what is held in f64 (half the instructions of exp()); 0 from -760 down, NaN stays.
__device__ __forceinline__ double exp_f64(double z) {
    const double q[9] = {CBH_EXP2_TERMS};
    double y = z * 1.4426950408889634;
    y = y < -1100.0 ? -1100.0 : y;
    const double k = rint(y), f = y - k;
    double p = q[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) p = __builtin_fma(p, f, q[i]);
    return ldexp(__builtin_fma(p, f, 1.0), (int)k);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Sums of N values at once.  tmp: N values a wave.
template <int THREADS, int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double* tmp) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_reduce(v[i], Add());
    if (THREADS == 64) return;
    if (lane_id() == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) tmp[threadIdx.x / 64 * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) v[i] += tmp[w * N + i];
    }
    __syncthreads();
}

// A running softmax denominator: sum over the scores seen of 2^((x - m) c), c = log2(e) / temperature.
// m starts at the lowest finite value, so that a score of -inf adds 0 and a row of nothing else
// keeps s = 0; a NaN, or a score of +inf (inf - inf), leaves NaN in s.  The difference is taken before
// the product: the product's rounding then counts against x - m, which is small for the scores
// that matter, and not against x.
// Sums of a tile's scores are taken side by side and then together, and added up in f64: beside a largest
// weight of 1, each f32 addition in a row of many would lose up to 2^-25.
struct Running {
    float m = kLowest;
    double s = 0.0;
    __device__ __forceinline__ void raise(float to, float c) {
        if (to > m) {
            s *= (double)exp2_fast((m - to) * c);
            m = to;
        }
    }
    template <int U, int V>
    __device__ __forceinline__ void add(const float (&x)[U][V], float c) {
        float e[V];
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = exp2_fast((x[0][v] - m) * c);
#pragma unroll
        for (int u = 1; u < U; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) e[v] += exp2_fast((x[u][v] - m) * c);
#pragma unroll
        for (int o = V / 2; o > 0; o /= 2)
#pragma unroll
            for (int v = 0; v < o; ++v) e[v] += e[v + o];
        s += (double)e[0];
    }
    __device__ __forceinline__ void add_one(float x, float c) { s += (double)exp2_fast((x - m) * c); }
    __device__ __forceinline__ void join(float m2, double s2, float c) {
        raise(m2, c);
        s += s2 * (double)exp2_fast((m2 - m) * c);
    }
};
// That of a part of a row, between launches: the sum stays in f64 (rounded to f32, what the other classes add to a
// largest weight of 1 would lose up to 2^-25 a part).
struct PartSum {
    double s;
    float m;
};
// (m, s) pairs of several threads together: the largest m, and the sums in f64.
template <int THREADS>
__device__ __forceinline__ void block_running(Running r, float c, float& m, double& s, float* tmp_f, double* tmp_d) {
    m = block_reduce<THREADS>(r.m, MaxF(), tmp_f);
    s = block_reduce<THREADS>(r.s * (double)exp2_fast((r.m - m) * c), Add(), tmp_d);
}

// ---- host -----------------------------------------------------------------------------------
#define CLS_TRY(expr)                                                                            \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess)                                                                    \
            return cbh_internal_fail(CBH_ERR_DEVICE, std::string(#expr ": ") + hipGetErrorString(e_)); \
    } while (0)

inline size_t type_bytes(int32_t type) { return type == CBH_TYPE_F32 ? 4 : 2; }

// What every operator asks of its scores.
inline int check_scores(const void* scores, int32_t type, uint64_t rows, uint32_t classes, int64_t row_stride,
                        int64_t class_stride) {
    if (type != CBH_TYPE_F32 && type != CBH_TYPE_F16 && type != CBH_TYPE_BF16)
        return cbh_internal_fail(CBH_ERR_UNSUPPORTED, "scores are f32, f16 or bf16");
    if (rows > 0x7FFFFFFFull) return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "more than 2^31 - 1 rows");
    if (classes == 0 || classes > kMaxClasses)
        return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "classes must be in 1 .. 2^24");
    if (rows && !scores) return cbh_internal_fail(CBH_ERR_INVALID_ARG, "scores are null");
    if ((uintptr_t)scores % type_bytes(type))
        return cbh_internal_fail(CBH_ERR_INVALID_ARG, "scores are not aligned to their type");
    const double lim = 4.0e18 / (double)type_bytes(type);
    if (std::abs((double)row_stride) * (double)rows + std::abs((double)class_stride) * (double)classes > lim)
        return cbh_internal_fail(CBH_ERR_OUT_OF_RANGE, "strides pass the address range");
    return CBH_OK;
}
// The exponent of a score, (x - m) log2(e) / t, is taken in f32: log2(e) / t is finite and normal there from 1e-38 on,
// and up to 1e36 a difference that leaves f32 has no weight (e^-340).
inline bool good_temperature(double t) { return t >= 1e-38 && t <= 1e36; }
constexpr const char* kBadTemperature = "temperature must be in 1e-38 .. 1e36";

// The grid of a kernel whose workgroups walk over the rows: a launch holds fewer than 2^32 threads.
inline unsigned row_grid(uint64_t blocks) { return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>(blocks, 1u << 20)); }

}  // namespace cls
}  // namespace cbh
