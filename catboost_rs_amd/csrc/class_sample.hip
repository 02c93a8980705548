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
    r.rt = fmin(1.0 / t, 1e308);   // (finite: the largest score's own exponent is 0 times it)
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
// The mass of a score: 2^((x - m) c) in units of 2^-S, rounded to an integer by the addition of 2^52
// (S <= 51).  -inf and NaN have none (the maximum with a number drops NaN).  m is finite.
struct Masses {
    double m, c;   // largest score, log2(e) / temperature
    double big;    // 1.5 2^52 + S
    double q[9];
    // The polynomial's coefficients are held in scalar registers (the compiler's own choice is 18 vector registers).
    __device__ __forceinline__ Masses(double m, double c, int S) : m(m), c(c), big(6755399441055744.0 + S) {
        const double k[9] = {CBH_EXP2_TERMS};
#pragma unroll
        for (int i = 0; i < 9; ++i) {
            q[i] = k[i];
            asm("" : "+s"(q[i]));
        }
    }
    __device__ __forceinline__ double exp2_part(double f) const {
        double p = q[8];
#pragma unroll
        for (int i = 7; i >= 0; --i) p = __builtin_fma(p, f, q[i]);
        return __builtin_fma(p, f, 1.0);
    }
    __device__ __forceinline__ u64 raw(float x) const {   // the mass plus kRaw
        // (the difference first: beside scores next to the lowest f32 the product's rounding would be more than it)
        const double y = fmax(((double)x - m) * c, -120.0);   // no mass below -53
        // y rounded to an integer k, and k + S in the low word of the sum: it goes to the exponent of a
        // number in [0.7, 1.5]
        const double t = y + big, k = t - big;
        const uint32_t e = (uint32_t)__builtin_bit_cast(u64, t);
        const u64 p = __builtin_bit_cast(u64, exp2_part(y - k)) + ((u64)e << 52);
        return __builtin_bit_cast(u64, __builtin_bit_cast(double, p) + 4503599627370496.0);
    }
    // sums of masses against the largest's
    __device__ __forceinline__ double log_of(u64 total) const { return log((double)total / (double)(*this)((float)m)); }
    // the mass of a weight of min_p (0 and NaN: none; 1: the largest's own)
    __device__ __forceinline__ u64 least(double min_p) const {
        const u64 one = (*this)((float)m);
        if (!(min_p > 0.0)) return 0;
        const double v = ceil(min_p * (double)one);
        return v < (double)one ? (u64)v : one;
    }
    static constexpr u64 kRaw = 0x4330000000000000ull;
    __device__ __forceinline__ u64 operator()(float x) const { return raw(x) - kRaw; }
};
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

// ---- entries in registers ----------------------------------------------------------------------
// Exclusive prefix sum over the workgroup, in thread order, and the sum of all.
template <int THREADS>
__device__ __forceinline__ u64 block_scan(u64 v, u64& all, u64* tmp) {
    const uint32_t lane = lane_id(), wave = threadIdx.x / 64;
    const u64 upto = wave_scan(v, Add(), u64(0));
    if (THREADS == 64) {
        all = read_lane(upto, 63);
        return upto - v;
    }
    if (lane == 63) tmp[wave] = upto;
    __syncthreads();
    u64 before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        before += (uint32_t)w < wave ? tmp[w] : 0;
        sum += tmp[w];
    }
    __syncthreads();
    all = sum;
    return before + upto - v;
}

// What a row's answer is written through.
struct Out {
    int32_t* index;
    float* logprob;
    __device__ __forceinline__ void put(uint64_t row, uint32_t cls, double lp) const {
        index[row] = (int32_t)cls;
        if (logprob) logprob[row] = (float)lp;
    }
    __device__ __forceinline__ void empty(uint64_t row) const {
        index[row] = -1;
        if (logprob) logprob[row] = -INFINITY;
    }
};

// Entries of a row in registers: cut them, and draw.  Entry e of a thread has order key key[e] (0: none) and
// class idx[e].
template <int THREADS, int E>
struct Entries {
    uint32_t key[E], idx[E];
    u64 mass[E];
    __device__ __forceinline__ u64 rank(int e) const { return ((u64)key[e] << 32) | (uint32_t)~idx[e]; }
    __device__ __forceinline__ void keep_from(Crossing c) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (rank(e) < c.from) key[e] = 0;
    }
    __device__ void cut_count(uint32_t k, SelectLds* lds, u64* tmp) {
        uint32_t have = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) have += key[e] != 0;
        if (block_reduce<THREADS>((u64)have, Add(), tmp) <= k) return;
        keep_from(select<THREADS, false, true>(
            [&](auto f) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (key[e]) f(rank(e), 0);
            },
            k, lds));
    }
    __device__ __forceinline__ void weigh(const Masses& M) {
#pragma unroll
        for (int e = 0; e < E; ++e) mass[e] = key[e] ? M(key_score(key[e])) : 0;
    }
    __device__ __forceinline__ u64 sum(u64* tmp) const {
        u64 s = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += key[e] ? mass[e] : 0;
        return block_reduce<THREADS>(s, Add(), tmp);
    }
    // the shortest prefix of the order with a mass of `want` stays
    __device__ void cut_mass(u64 want, SelectLds* lds) {
        keep_from(select<THREADS, true, true>(
            [&](auto f) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (key[e] && mass[e]) f(rank(e), mass[e]);
            },
            want, lds));
    }
    __device__ __forceinline__ void drop_below(u64 least) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (mass[e] < least) key[e] = 0;
    }
};

// ---- few classes: a row a thread ---------------------------------------------------------------
// Scores and masses in registers.  A nucleus needs the mass ahead of every class: the pairs of classes, in
// f64 (with S = 46 and at most 32 classes every sum is an integer below 2^53 and exact), each pair a
// comparison and two multiply-adds with 0 or 1.
// 1M x 10 f32, top_p 0.9, class-major: 35 us, 56 MB at 1.6 TB/s; bound by f64 instructions (the masses, and
// the pairs of 10 places; 46 us with 12) and by scalar registers that do not fit: the pairs' comparisons are masks in
// pairs of them, and each that the compiler puts aside costs vector instructions (119 at 10 places, 1133 at 32:
// 500k x 32 271 us).  A wave a row took 3.2 ms.
constexpr int kFewShift = 46;
template <class T, int NMAX>
__global__ __launch_bounds__(256) void sample_few_kernel(Rows<T> X, Settings S, Out out) {
    const uint32_t n = X.classes;
    for (uint64_t row = (uint64_t)blockIdx.x * 256 + threadIdx.x; row < X.rows; row += (uint64_t)gridDim.x * 256) {
        const Row r = settings(S, row, n);
        const T* x0 = X.data + (int64_t)row * X.rs;
        const uint32_t bits = r.allowed ? r.allowed[0] : ~0u;
        float x[NMAX], m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) {
            x[i] = (uint32_t)i < n ? to_f32(x0[(int64_t)i * X.cs]) : -INFINITY;
            x[i] = bits >> i & 1 && x[i] == x[i] ? x[i] : -INFINITY;
            m = fmaxf(m, x[i]);
        }
        int first = -1;
#pragma unroll
        for (int i = NMAX - 1; i >= 0; --i) first = x[i] == m ? i : first;
        if (m == -INFINITY) {
            out.empty(row);
            continue;
        }
        if (r.greedy) {
            out.put(row, first, 0.0);
            continue;
        }
        const bool inf = m == INFINITY;
        const Masses M{inf ? 0.0 : (double)m, r.rt * 1.4426950408889634, kFewShift};
        double w[NMAX], total = 0.0;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) {
            if (inf) x[i] = x[i] == m ? 0.0f : -INFINITY;
            w[i] = __builtin_bit_cast(double, M.raw(x[i])) - 4503599627370496.0;
            total += w[i];
        }
        uint32_t kept = ~0u;   // a bit a class
        if (r.min_p > 1.0) {
            kept = 1u << first;
        } else if (r.k || r.p < 1.0) {
            double ahead[NMAX], whole = total;
            uint32_t place[NMAX];
#pragma unroll
            for (int i = 0; i < NMAX; ++i) {
                ahead[i] = 0.0;
                place[i] = 0;
            }
            const bool count = r.k != 0;
#pragma unroll
            for (int i = 1; i < NMAX; ++i)
#pragma unroll
                for (int j = 0; j < i; ++j) {
                    const bool a = x[j] >= x[i];   // j is ahead of i
                    ahead[i] = __builtin_fma(w[j], a ? 1.0 : 0.0, ahead[i]);
                    ahead[j] = __builtin_fma(w[i], a ? 0.0 : 1.0, ahead[j]);
                    if (count) {
                        place[i] += a;
                        place[j] += !a;
                    }
                }
            if (count) {
                whole = 0.0;
#pragma unroll
                for (int i = 0; i < NMAX; ++i) {
                    const bool in = place[i] < r.k;
                    whole += in ? w[i] : 0.0;
                    kept = in ? kept : kept & ~(1u << i);
                }
            }
            if (r.p < 1.0) {
                const double want = r.p * whole;
#pragma unroll
                for (int i = 0; i < NMAX; ++i) kept = ahead[i] < want ? kept : kept & ~(1u << i);
                kept |= 1u << first;
            }
        }
        const double least = r.min_p > 0.0 && r.min_p <= 1.0 ? r.min_p * 70368744177664.0 : 0.0;
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) {
            w[i] = kept >> i & 1 && w[i] >= least ? w[i] : 0.0;
            sum += w[i];
        }
        const double target = r.u > 0.0 ? r.u * sum : 0.0;   // (NaN: 0)
        int at = first;
        double run = 0.0;
        bool open = true;
        float xs = m;
#pragma unroll
        for (int i = 0; i < NMAX; ++i) {
            run += w[i];
            if (open && w[i] > 0.0) {   // the last class with mass, unless the running mass passes the target before
                at = i;
                xs = x[i];
                open = !(run > target);
            }
        }
        out.put(row, at, (inf ? 0.0 : ((double)xs - (double)m) * r.rt) - log(total * 0x1p-46));
    }
}

// ---- rows that fit the registers of a workgroup -----------------------------------------------
// 33 to 2048 classes, in one launch; bound by the latency of the selection's rounds.
// Thread t holds classes [t E, (t + 1) E).
template <class T, bool kUnit, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_short_kernel(Rows<T> X, Settings S, int shift, Out out) {
    constexpr int E = 8, V = Pack<T>::V, W = THREADS / 64;
    __shared__ SelectLds lds;
    __shared__ u64 tmp[W];
    const uint32_t n = X.classes, i0 = threadIdx.x * E;
    for (uint64_t row = blockIdx.x; row < X.rows; row += gridDim.x) {
        const Row r = settings(S, row, n);
        const T* x0 = X.data + (int64_t)row * X.rs;
        float x[E];
#pragma unroll
        for (int q = 0; q < E / V; ++q)
            load_pack<T, kUnit>(x0, X.cs, i0 + q * V, n, -INFINITY, *(float(*)[V])&x[q * V]);
        const uint32_t bits = r.allowed && i0 < n ? r.allowed[i0 >> 5] >> (i0 & 31) : ~0u;
        Entries<THREADS, E> L;
        u64 top = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            L.idx[e] = i0 + e;
            L.key[e] = class_key(x[e], bits >> e & 1);
            const u64 k = L.key[e] ? L.rank(e) : 0;
            top = k > top ? k : top;
        }
        top = block_reduce<THREADS>(top, MaxU(), tmp);
        if (top == 0) {
            if (threadIdx.x == 0) out.empty(row);
            continue;
        }
        const uint32_t first = ~(uint32_t)top;
        const float m = key_score((uint32_t)(top >> 32));
        if (r.greedy) {
            if (threadIdx.x == 0) out.put(row, first, 0.0);
            continue;
        }
        // (beside +inf nothing has mass: the classes of +inf become 0, the others -inf)
        const bool inf = m == INFINITY;
        const Masses M{inf ? 0.0 : (double)m, r.rt * 1.4426950408889634, shift};
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float y = !inf ? key_score(L.key[e]) : L.key[e] == (uint32_t)(top >> 32) ? 0.0f : -INFINITY;
            L.mass[e] = L.key[e] ? M(y) : 0;
        }
        const u64 total = L.sum(tmp);
        if (r.min_p > 1.0) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (L.idx[e] != first) L.key[e] = 0;
        } else {
            if (r.k) L.cut_count(r.k, &lds, tmp);
            if (r.p < 1.0) L.cut_mass(nucleus_of(r.p, r.k ? L.sum(tmp) : total), &lds);
            L.drop_below(M.least(r.min_p));
        }
        u64 mine = 0, all;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += L.key[e] ? L.mass[e] : 0;
        u64 before = block_scan<THREADS>(mine, all, tmp);
        const u64 target = target_of(r.u, all);
        if (target >= before && target - before < mine) {
            uint32_t cls = first;
            float xs = m;
            bool found = false;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const u64 w = L.key[e] ? L.mass[e] : 0;
                if (!found && target - before < w) {
                    found = true;
                    cls = L.idx[e];
                    xs = key_score(L.key[e]);
                }
                before += w;
            }
            out.put(row, cls, (inf ? 0.0 : ((double)xs - (double)m) * r.rt) - M.log_of(total));
        }
        __syncthreads();
    }
}

// ---- long rows --------------------------------------------------------------------------------
// A wave takes 2048 classes at a time (a segment), in groups of 32.  Which classes can be kept is found from the maxima of the groups (few of many: top_k), or from a
// histogram of counts or masses over the distance from the largest score; those, or those of the one
// bin in which the cut lies, are listed, and the list cut exactly in registers.  Kept masses of the
// bins above a nucleus's last are summed by segments, and the draw looks through one of them.
constexpr uint32_t kGroupSegs = 128, kMostByGroups = 1024, kListCap = 8192, kShortList = 128;
constexpr uint32_t kBins = 1024, kBinsPad = kBins + kBins / 16;
// The bins reach from the largest score to a little below the lowest of a sample (the first class of every lane's
// tile, 64 of 2048), 32 nats at most and where the sample holds no class (all of them masked): 32 bins a nat, and more of
// them for the rows of a narrow range, whose nucleus is wide: one bin then holds hundreds of classes and not
// thousands, which the list has to take.
constexpr float kMostNats = 32.0f;
__device__ __forceinline__ uint32_t bin_at(uint32_t b) { return b + (b >> 4); }   // (its place in LDS)

enum Mode : uint32_t { kGreedy, kWhole, kList, kNucleus };   // (kWhole: a least weight above 1 as well)

template <class T, bool kUnit, int THREADS>
struct Long {
    static constexpr int V = Pack<T>::V, U = kGroup / V, W = THREADS / 64;
    static constexpr int E = THREADS == 1024 ? 8 : 2048 / THREADS, CAP = THREADS * E;   // a list's entries in registers
    const T* x0;
    int64_t cs;
    uint32_t n;
    Row r;
    int S;
    uint32_t lane, wave;

    __device__ __forceinline__ Long(const Rows<T>& X, const Settings& St, uint64_t row, int shift)
        : x0(X.data + (int64_t)row * X.rs), cs(X.cs), n(X.classes), r(settings(St, row, X.classes)), S(shift),
          lane(lane_id()), wave(__builtin_amdgcn_readfirstlane(threadIdx.x / 64)) {}

    __device__ __forceinline__ uint32_t at(uint32_t seg, int u, uint32_t ln) const { return seg * kSeg + (u * 64 + ln) * V; }
    // classes that are not allowed read as -inf
    __device__ __forceinline__ void load(uint32_t i, float (&x)[V]) const {
        load_pack<T, kUnit>(x0, cs, i, n, -INFINITY, x);
        if (r.allowed && i < n) {
            const uint32_t bits = r.allowed[i >> 5] >> (i & 31);
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = bits >> v & 1 ? x[v] : -INFINITY;
        }
    }
    struct Tile {   // a segment's scores in their type; vector u becomes f32 where it is used
        Pack<T> p[U];
        uint32_t bits[U];
        bool masked;
        __device__ __forceinline__ void get(int u, float (&x)[V]) const {
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = p[u].get(v);
            if (masked) {
#pragma unroll
                for (int v = 0; v < V; ++v) x[v] = bits[u] >> v & 1 ? x[v] : -INFINITY;
            }
        }
    };
    __device__ __forceinline__ void load(uint32_t seg, Tile& t) const {
        t.masked = r.allowed != nullptr;
        if (t.masked) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = at(seg, u, lane);
                t.bits[u] = i < n ? r.allowed[i >> 5] >> (i & 31) : 0;
            }
        }
        load_tile<T, kUnit>(x0, cs, seg * kSeg, n, -INFINITY, t.p);
    }
    __device__ __forceinline__ float score(uint32_t i) const {
        const uint32_t j = min(i, n - 1);   // (a load that waits for no branch)
        const float x = to_f32(x0[kUnit ? (int64_t)j : (int64_t)j * cs]);
        const uint32_t bits = r.allowed ? r.allowed[j >> 5] >> (j & 31) : 1;
        return i < n && (bits & 1) ? x : -INFINITY;
    }
    __device__ __forceinline__ Mode mode() const {
        return r.greedy ? kGreedy : r.min_p > 1.0 ? kWhole : r.k ? kList : r.p < 1.0 ? kNucleus : kWhole;
    }
    // top_k from the groups' maxes: a quarter of them at most, so that few classes beside the k largest reach
    // the k-th of the maxima; 2^18 classes at most (32 KB of maxima)
    __host__ __device__ static bool by_groups_of(uint32_t k, uint32_t segs) {
        return segs <= kGroupSegs && k <= segs * 16 && k <= kMostByGroups;
    }
    __device__ __forceinline__ bool by_groups(uint32_t segs) const { return by_groups_of(r.k, segs); }

    // Largest score of the segments [s0, s1) and the segment it was first met in, per thread; into `groups`
    // (nullable) every group's largest as an order key (0: nothing to draw); with `sums` the running softmax
    // denominator: what a top_k row's log probability takes of the classes that are cut.  Its exponentials are f32 (off by
    // 3 |d| 2^-24 + 2^-23, d = (x - max) / t, the sum f64): the pass stays bound by memory with them, at 24 us for 256 x
    // 131072 f32, where f64 masses, which need the maximum first, take a pass of 27 to 34 us more.
    __device__ __forceinline__ void scan(uint32_t s0, uint32_t s1, uint32_t* groups, bool sums, float c,
                                         float& best, uint32_t& best_seg, float& low, Running& run) const {
        best = -INFINITY;
        low = INFINITY;
        best_seg = s0;
        for (uint32_t seg = s0 + wave; seg < s1; seg += W) {
            Tile t;
            load(seg, t);
            float x[U][V], vm[U], gm = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) t.get(u, x[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                vm[u] = -INFINITY;   // (NaN is no class)
#pragma unroll
                for (int v = 0; v < V; ++v) vm[u] = fmaxf(vm[u], x[u][v]);
                gm = fmaxf(gm, vm[u]);
            }
            if (gm > best) {
                best = gm;
                best_seg = seg;
            }
            if (x[0][0] > -INFINITY) low = fminf(low, x[0][0]);
            if (groups) {
                const float g = group_max<V>(vm, lane, MaxF());
                groups[(seg - s0) * 64 + group_of<V>(lane)] = g > -INFINITY ? order_key(g) : 0;
            }
            if (sums) {
                run.raise(gm, c);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int v = 0; v < V; ++v) x[u][v] = x[u][v] == x[u][v] ? x[u][v] : -INFINITY;   // (NaN is no class)
                run.add(x, c);
            }
        }
    }
    // The first class at the score m, of the threads that have met it in best_seg; n if there is none.
    __device__ __forceinline__ uint32_t first_at(float m, float best, uint32_t best_seg) const {
        if (!(best == m) || m == -INFINITY) return 0xFFFFFFFFu;
        uint32_t first = 0xFFFFFFFFu;
#pragma unroll 1
        for (int u = U - 1; u >= 0; --u) {
            float x[V];
            const uint32_t i = at(best_seg, u, lane);
            load(i, x);
#pragma unroll
            for (int v = V - 1; v >= 0; --v) first = x[v] == m ? i + v : first;
        }
        return first;
    }

    // Rows that slow() takes whatever their settings: those of +inf, and those whose cut goes by bins or by f32
    // exponentials at a temperature beyond [1e-30, 1e36], whose reciprocal's products leave f32 (an infinite scale of
    // the bins puts the largest score, at distance 0, into the last).  Masses are f64 at any temperature.
    __device__ __forceinline__ bool whole_row(float m, Mode mode) const {
        return m == INFINITY || (mode != kWhole && !(r.rt >= 1e-36 && r.rt <= 1e30));
    }

    // ---- bins: monotone in the score, the largest in bin 0 (whole_row() keeps the scale finite) ----
    float bm, bscale;
    __device__ __forceinline__ void set_bins(float m, float low) {
        bm = m;
        const float range = low < INFINITY ? fminf((m - low) * (float)r.rt * 1.25f + 1.0f, kMostNats) : kMostNats;
        bscale = (float)(r.rt * (double)((float)kBins / range));
    }
    __device__ __forceinline__ uint32_t bin(float x) const {
        const float z = (bm - x) * bscale;
        return z < (float)(kBins - 1) ? (uint32_t)z : kBins - 1;   // (NaN: the last)
    }
    // Histogram of the segments' counts or masses, added into `hist` in LDS (padded).
    template <bool kMass>
    __device__ __forceinline__ void histogram(uint32_t s0, uint32_t s1, const Masses& M, u64* hist) const {
        for (uint32_t seg = s0 + wave; seg < s1; seg += W) {
            Tile t;
            load(seg, t);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[V];
                t.get(u, x);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float y = x[v];
                    if (kMass) {
                        const u64 w = M(y);
                        if (w) atomicAdd(&hist[bin_at(bin(y))], w);
                    } else if (y > -INFINITY) {
                        atomicAdd((uint32_t*)&hist[bin_at(bin(y))], 1u);
                    }
                    if (v % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (four masses at a time: registers)
                }
            }
        }
    }
    // Masses of the segments, of the classes of at least `least`; the mass of all classes, per thread.
    template <bool kLeast>
    __device__ __forceinline__ u64 weigh_segments(uint32_t s0, uint32_t s1, const Masses& M, u64 least, u64* segs) const {
        u64 all = 0;
        for (uint32_t seg = s0 + wave; seg < s1; seg += W) {
            Tile t;
            load(seg, t);
            u64 sum = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[V];
                t.get(u, x);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (kLeast) {
                        const u64 w = M(x[v]);
                        all += w;
                        sum += w >= least ? w : 0;
                    } else {
                        sum += M.raw(x[v]);
                    }
                    if (v % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (!kLeast) {
                sum -= kGroup * Masses::kRaw;
                all += sum;
            }
            sum = wave_reduce(sum, Add());
            if (lane == 0) segs[seg] = sum;
        }
        return all;
    }
    __device__ __forceinline__ u64 weigh(uint32_t s0, uint32_t s1, const Masses& M, u64 least, u64* segs) const {
        return least ? weigh_segments<true>(s0, s1, M, least, segs) : weigh_segments<false>(s0, s1, M, 0, segs);
    }
    // The lowest score whose bin is at most b (bins are monotone): the order keys' range is cut into 64 by the lanes.
    __device__ __forceinline__ float lowest_of(uint32_t b) const {
        uint32_t lo = order_key(-INFINITY), hi = order_key(bm);   // (bin(lo) is above b, or lo is it; bin(hi) = 0)
        while (hi - lo > 1) {
            const uint32_t step = (hi - lo + 63) / 64, probe = min(hi, lo + step * (lane + 1));   // (the last is hi)
            const u64 yes = __ballot(probe == hi || bin(key_score(probe)) <= b);   // (hi is one: the range shrinks)
            const uint32_t at = yes ? (uint32_t)__builtin_ctzll(yes) : 63;
            hi = min(hi, lo + step * (at + 1));
            lo = lo + step * at;
        }
        return key_score(hi);
    }
    // The scores of the bins at the cut: [from, above); with `all`, all from there up.
    __device__ __forceinline__ void cut_scores(uint32_t cut, bool all, float& from, float& above) const {
        from = cut == kBins - 1 ? kLowest : lowest_of(cut);   // (the last bin takes all that is left)
        above = all || cut == 0 ? INFINITY : lowest_of(cut - 1);
    }
    // Entries of a wave's staging area in LDS.
    static constexpr uint32_t kStage = 256;
    // The classes of scores in [from, above) go to the list (at most cap; count goes on); with kSum the masses of
    // those above go to their segments.
    template <bool kSum>
    __device__ __forceinline__ void collect(uint32_t s0, uint32_t s1, const Masses& M, float from, float above, u64 least,
                                            u64* segs, u64* list, uint32_t* count, uint32_t cap, u64* stage) const {
        stage += wave * kStage;
        uint32_t staged = 0;
        auto flush = [&]() {
            wave_fence();
            uint32_t base = 0;
            if (lane == 0) base = atomicAdd(count, staged);
            base = __builtin_amdgcn_readfirstlane(base);
            for (uint32_t i = lane; i < staged; i += 64)
                if (base + i < cap) list[base + i] = stage[i];
            wave_fence();
            staged = 0;
        };
        for (uint32_t seg = s0 + wave; seg < s1; seg += W) {
            u64 sum = 0;
            Tile t;
            load(seg, t);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[V];
                t.get(u, x);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (kSum) {
                        const u64 w = M(x[v] >= above ? x[v] : -INFINITY);
                        sum += w >= least ? w : 0;
                    }
                    const bool in = x[v] >= from && x[v] < above;
                    const u64 who = __ballot(in);
                    if (who) {
                        if (in) stage[staged + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0u))] =
                            rank_key(x[v], at(seg, u, lane) + v);
                        staged += (uint32_t)__popcll(who);
                        if (staged > kStage - 64) flush();
                    }
                    if (v % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (kSum) {
                sum = wave_reduce(sum, Add());
                if (lane == 0) segs[seg] = sum;
            }
        }
        if (staged) flush();
    }
    // Classes that reach the bound, of the groups listed in hits (count[1] of them; written without a barrier since),
    // go to the list (count[0]); half a wave reads a group.
    __device__ __forceinline__ void gather(uint32_t bound, u64* list, uint32_t* count, const uint16_t* hits) const {
        __syncthreads();
        const uint32_t n_hits = count[1], q = threadIdx.x % kGroup;
        constexpr int D = 8;   // groups a half wave has under way
        for (uint32_t h0 = threadIdx.x / kGroup; h0 < n_hits; h0 += THREADS / kGroup * D) {
            float x[D];
            uint32_t i[D];
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const uint32_t h = h0 + d * (THREADS / kGroup), g = h < n_hits ? hits[h] : 0;
                i[d] = h < n_hits ? g * kGroup + q : n;
                x[d] = score(i[d]);
            }
#pragma unroll
            for (int d = 0; d < D; ++d)
                if (x[d] > -INFINITY && order_key(x[d]) >= bound) {
                    const uint32_t at = atomicAdd(&count[0], 1u);
                    if (at < (uint32_t)CAP) list[at] = rank_key(x[d], i[d]);
                }
        }
    }
    __device__ __forceinline__ void read_list(Entries<THREADS, E>& L, const u64* list, uint32_t count) const {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t i = e * THREADS + threadIdx.x;
            const u64 k = i < count ? list[i] : 0;
            L.key[e] = (uint32_t)(k >> 32);
            L.idx[e] = ~(uint32_t)k;
        }
    }

    // ---- the last steps ----
    // A list that holds every class that may be kept: top_k, top_p, min_p, and the draw.
    __device__ void finish_list(const u64* list, uint32_t count, const Masses& M, double log_z, uint64_t row, SelectLds* lds,
                                u64* tmp, const Out& out) const {
        if (count <= min(kShortList, (uint32_t)THREADS)) {
            finish_short(list, count, M, log_z, row, lds, tmp, out);
            return;
        }
        Entries<THREADS, E> L;
        read_list(L, list, count);
        L.cut_count(r.k, lds, tmp);
        L.weigh(M);
        if (r.p < 1.0) L.cut_mass(nucleus_of(r.p, L.sum(tmp)), lds);
        L.drop_below(M.least(r.min_p));
        const u64 want = target_of(r.u, L.sum(tmp)) + 1;
        const Crossing c = select<THREADS, true, false>(
            [&](auto f) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (L.key[e] && L.mass[e]) f((uint32_t)~L.idx[e], L.mass[e]);
            },
            want, lds);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (L.key[e] && L.mass[e] && (uint32_t)~L.idx[e] >= c.from && (uint32_t)~L.idx[e] <= c.last)
                out.put(row, L.idx[e], ((double)key_score(L.key[e]) - M.m) * r.rt - log_z);
    }
    // The same for up to 128 classes: every entry counts those ahead of it, and later the mass of the classes
    // before it; several threads share an entry's counting.
    __device__ void finish_short(const u64* list, uint32_t count, const Masses& M, double log_z, uint64_t row, SelectLds* lds,
                                 u64* tmp, const Out& out) const {
        const uint32_t t = threadIdx.x;
        const uint32_t slots = (count + 63) / 64 * 64, shares = (uint32_t)THREADS / slots, share = t / slots, e = t % slots;
        const uint32_t each = ((slots + shares - 1) / shares + 7) / 8 * 8;   // (of the entries, by eights)
        const uint32_t j0 = min(slots, share * each), j1 = share < shares ? min(slots, j0 + each) : j0;
        for (uint32_t i = t; i < slots; i += THREADS) {
            lds->mass[i] = i < count ? list[i] : 0;
            lds->place[i] = 0;
        }
        __syncthreads();
        const u64 key = lds->mass[e];
        uint32_t place = 0;
        for (uint32_t j = j0; j < j1; j += 8)
#pragma unroll
            for (int q = 0; q < 8; ++q) place += lds->mass[j + q] > key;
        if (j0 < j1 && e < count) atomicAdd(&lds->place[e], place);
        __syncthreads();
        if (t < count) lds->rank[lds->place[t]] = key;   // (t < slots: e is t)
        __syncthreads();
        const uint32_t kept = min(count, r.k);
        const u64 rank = t < kept ? lds->rank[t] : 0;
        const float x = key_score((uint32_t)(rank >> 32));
        u64 w = t < kept ? M(x) : 0, all;
        const u64 ahead = block_scan<THREADS>(w, all, tmp);
        if (r.p < 1.0 && ahead >= nucleus_of(r.p, all)) w = 0;
        if (w < M.least(r.min_p)) w = 0;
        const u64 sum = block_reduce<THREADS>(w, Add(), tmp);
        // before the draw's class lie the classes whose masses come to no more than the target
        for (uint32_t i = t; i < slots; i += THREADS) lds->mass[i] = 0;
        __syncthreads();
        u64 mine = t < kept ? w : 0;
        if (t < slots) {
            lds->rank[t] = t < kept ? rank : 0;
            lds->weight[t] = mine;
        }
        __syncthreads();
        const uint32_t cls = (uint32_t)lds->rank[e];   // (~class: larger for a class before)
        u64 before = 0;
        for (uint32_t j = j0; j < j1; j += 8)
#pragma unroll
            for (int q = 0; q < 8; ++q) before += (uint32_t)lds->rank[j + q] > cls ? lds->weight[j + q] : 0;
        if (j0 < j1 && e < kept) atomicAdd(&lds->mass[e], before);
        __syncthreads();
        if (mine) {
            const u64 target = target_of(r.u, sum);
            before = lds->mass[t];
            if (target >= before && target - before < mine) out.put(row, ~(uint32_t)rank, ((double)x - M.m) * r.rt - log_z);
        }
        __syncthreads();
    }
    // Segments' kept masses (and a nucleus's cut): the segment of the draw, then its class.
    __device__ void finish_segments(const u64* segs, uint32_t n_segs, const Masses& M, uint32_t cut, u64 from, u64 least,
                                    u64 total, uint64_t row, u64* tmp, u64* pick, const Out& out) const {
        const uint32_t per = (n_segs + THREADS - 1) / THREADS, a = min(n_segs, threadIdx.x * per), b = min(n_segs, a + per);
        u64 mine = 0, all;
        for (uint32_t s = a; s < b; ++s) mine += segs[s];
        u64 before = block_scan<THREADS>(mine, all, tmp);
        const u64 target = target_of(r.u, all);
        if (target >= before && target - before < mine) {
            uint32_t s = a;
            while (target - before >= segs[s]) before += segs[s++];
            pick[0] = s;
            pick[1] = before;
        }
        __syncthreads();
        const uint32_t seg = (uint32_t)pick[0];
        const u64 base = pick[1];
        constexpr int Q = kSeg / THREADS;
        u64 w[Q];
        mine = 0;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const uint32_t i = seg * kSeg + threadIdx.x * Q + q;
            const float x = score(i);
            bool in = x > -INFINITY;
            if (cut < kBins) {
                const uint32_t bi = bin(x);
                in = in && (bi < cut || (bi == cut && rank_key(x, i) >= from));
            }
            w[q] = in ? M(x) : 0;
            w[q] = w[q] >= least ? w[q] : 0;
            mine += w[q];
        }
        before = base + block_scan<THREADS>(mine, all, tmp);
        if (target >= before && target - before < mine) {
            bool found = false;
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                if (!found && target - before < w[q]) {
                    found = true;
                    const uint32_t i = seg * kSeg + threadIdx.x * Q + q;
                    out.put(row, i, ((double)score(i) - M.m) * r.rt - M.log_of(total));
                }
                before += w[q];
            }
        }
    }
    // Any row, by selection over the whole of it, read again for every digit: rows of +inf or of far temperatures
    // (whole_row()), and those whose cut needs more classes than a list holds: a nucleus that ends among so many of
    // one bin (equal scores, or few of the bins' sample allowed), a top_k and what shares its last bin beyond 8192 (2048 in
    // rows of 2049 to 8192 classes).  256 x 131072 f32: top_k 5000 126 us, 8000 138, 9000 700, 100000 706; 256 x 6000: top_k
    // 2000 28 us, 2100 84.
    __device__ void slow(uint32_t top_key, uint32_t first, uint64_t row, SelectLds* lds, u64* tmp, u64* pick, const Out& out) const {
        const float m = key_score(top_key);
        const bool inf = m == INFINITY;
        const Masses M{inf ? 0.0 : (double)m, r.rt * 1.4426950408889634, S};
        auto mass = [&](float x) -> u64 { return M(!inf ? x : x == m ? 0.0f : -INFINITY); };
        auto key_at = [&](uint32_t i) { return class_key(score(i), true); };
        u64 total = 0;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS)
            if (key_at(i)) total += mass(score(i));
        total = block_reduce<THREADS>(total, Add(), tmp);
        if (r.min_p > 1.0) {
            if (threadIdx.x == 0) out.put(row, first, -M.log_of(total));
            __syncthreads();
            return;
        }
        u64 from = 0;   // ranks below it are cut
        u64 have = 0, kept = total;
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) have += key_at(i) != 0;
        have = block_reduce<THREADS>(have, Add(), tmp);
        if (r.k && have > r.k) {
            const Crossing c = select<THREADS, false, true>(
                [&](auto f) {
                    for (uint32_t i = threadIdx.x; i < n; i += THREADS)
                        if (key_at(i)) f(rank_key(score(i), i), 0);
                },
                r.k, lds);
            from = c.from;
            kept = 0;
            for (uint32_t i = threadIdx.x; i < n; i += THREADS)
                if (key_at(i) && rank_key(score(i), i) >= from) kept += mass(score(i));
            kept = block_reduce<THREADS>(kept, Add(), tmp);
        }
        if (r.p < 1.0) {
            const Crossing c = select<THREADS, true, true>(
                [&](auto f) {
                    for (uint32_t i = threadIdx.x; i < n; i += THREADS)
                        if (key_at(i) && rank_key(score(i), i) >= from) {
                            const u64 w = mass(score(i));
                            if (w) f(rank_key(score(i), i), w);
                        }
                },
                nucleus_of(r.p, kept), lds);
            from = c.from > from ? c.from : from;
        }
        const u64 least = M.least(r.min_p);
        // thread t holds the classes [t per, (t + 1) per)
        const uint32_t per = (n + THREADS - 1) / THREADS, a = min(n, threadIdx.x * per), b = min(n, a + per);
        auto weight = [&](uint32_t i) -> u64 {
            const float x = score(i);
            if (!class_key(x, true) || rank_key(x, i) < from) return 0;
            const u64 w = mass(x);
            return w >= least ? w : 0;
        };
        u64 mine = 0, all;
        for (uint32_t i = a; i < b; ++i) mine += weight(i);
        u64 before = block_scan<THREADS>(mine, all, tmp);
        const u64 target = target_of(r.u, all);
        if (target >= before && target - before < mine) {
            uint32_t i = a;
            for (u64 w; target - before >= (w = weight(i)); ++i) before += w;
            out.put(row, i, (inf ? 0.0 : ((double)score(i) - (double)m) * r.rt) - M.log_of(total));
        }
        __syncthreads();
    }
};

// Where the weights of the bins, from bin 0 on, reach `want`; every wave by itself.
template <class Get>
__device__ __forceinline__ Found<u64> find_cut(Get get, u64 want) {
    const uint32_t l = lane_id();
    u64 sum = 0;
    for (uint32_t j = 0; j < kBins / 64; ++j) sum += get(l * (kBins / 64) + j);
    const u64 upto = wave_scan(sum, Add(), u64(0));
    u64 above = upto - sum, inside = 0;
    uint32_t b = l * (kBins / 64);
    const u64 cross = __ballot(upto >= want);
    const int at = cross ? __builtin_ctzll(cross) : 63;
    bool open = true;
    for (uint32_t j = 0; j < kBins / 64; ++j) {
        const u64 c = get(l * (kBins / 64) + j);
        if (open) {
            b = l * (kBins / 64) + j;
            inside = c;
            if (above + c >= want) open = false;
            else if (j + 1 < kBins / 64) above += c;
        }
    }
    return Found<u64>{read_lane(b, at), read_lane(above, at), read_lane(inside, at)};
}

// Up to 8192 classes: a workgroup a row, all steps in one launch.
template <class T, bool kUnit, int THREADS>
__global__ __launch_bounds__(THREADS) void sample_long_kernel(Rows<T> X, Settings S, int shift, Out out) {
    typedef Long<T, kUnit, THREADS> L;
    constexpr int W = THREADS / 64;
    extern __shared__ u64 pool[];   // list, or segments' masses behind it; groups
    __shared__ u64 hist[kBinsPad];
    __shared__ SelectLds lds;
    __shared__ u64 tmp[W], pick[2];
    __shared__ float tmp_f[W];
    __shared__ double tmp_d[W];
    __shared__ uint32_t counts[2];
    uint32_t& count = counts[0];
    __shared__ u64 stage[W * L::kStage];
    const uint32_t n_segs = (X.classes + kSeg - 1) / kSeg;
    u64* list = pool;
    u64* segs = pool + L::CAP;
    uint32_t* groups = (uint32_t*)(segs + n_segs);
    uint16_t* hits = (uint16_t*)(groups + n_segs * 64);
    for (uint64_t row = blockIdx.x; row < X.rows; row += gridDim.x) {
        L R(X, S, row, shift);
        const Mode mode = R.mode();
        const float c = (float)(R.r.rt * 1.4426950408889634);
        const bool by_groups = mode == kList && R.by_groups(n_segs);
        float best, low;
        uint32_t best_seg;
        Running run;
        R.scan(0, n_segs, by_groups ? groups : nullptr, mode == kList, c, best, best_seg, low, run);
        for (uint32_t b = threadIdx.x; b < kBinsPad; b += THREADS) hist[b] = 0;
        if (threadIdx.x < 2) counts[threadIdx.x] = 0;
        const float m = block_reduce<THREADS>(best, MaxF(), tmp_f);
        __syncthreads();
        if (m == -INFINITY) {
            if (threadIdx.x == 0) out.empty(row);
            continue;
        }
        bool slow = R.whole_row(m, mode);
        uint32_t first = 0;
        if (R.r.greedy || R.r.min_p > 1.0) {
            first = (uint32_t)block_reduce<THREADS>((u64)R.first_at(m, best, best_seg), MinU(), tmp);
            if (R.r.greedy) {
                if (threadIdx.x == 0) out.put(row, first, 0.0);
                continue;
            }
        }
        const Masses M{(double)m, R.r.rt * 1.4426950408889634, shift};
        R.set_bins(m, -block_reduce<THREADS>(-low, MaxF(), tmp_f));
        if (!slow && mode == kWhole) {
            const u64 least = M.least(R.r.min_p);
            u64 z = R.weigh(0, n_segs, M, R.r.min_p > 1.0 ? 0 : least, segs);
            z = block_reduce<THREADS>(z, Add(), tmp);
            __syncthreads();
            if (R.r.min_p > 1.0) {
                if (threadIdx.x == 0) out.put(row, first, -M.log_of(z));
            } else {
                R.finish_segments(segs, n_segs, M, kBins, 0, least, z, row, tmp, pick, out);
            }
        } else if (!slow && mode == kNucleus) {
            R.template histogram<true>(0, n_segs, M, hist);
            __syncthreads();
            u64 z = 0;
            for (uint32_t b = threadIdx.x; b < kBins; b += THREADS) z += hist[bin_at(b)];
            z = block_reduce<THREADS>(z, Add(), tmp);
            const u64 want = nucleus_of(R.r.p, z), least = M.least(R.r.min_p);
            const Found<u64> f = find_cut([&](uint32_t b) { return hist[bin_at(b)]; }, want);
            float from, above;
            R.cut_scores(f.bin, false, from, above);
            R.template collect<true>(0, n_segs, M, from, above, least, segs, list, &count, L::CAP, stage);
            __syncthreads();
            if (count > (uint32_t)L::CAP) {
                slow = true;
            } else {
                Entries<THREADS, 8> E;
                R.read_list(E, list, count);
                E.weigh(M);
                const Crossing x = select<THREADS, true, true>(
                    [&](auto g) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (E.key[e] && E.mass[e]) g(E.rank(e), E.mass[e]);
                    },
                    want - f.above, &lds);
                E.keep_from(x);
                E.drop_below(least);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (E.key[e] && E.mass[e]) atomicAdd(&segs[E.idx[e] / kSeg], E.mass[e]);
                __syncthreads();
                R.finish_segments(segs, n_segs, M, f.bin, x.from, least, z, row, tmp, pick, out);
            }
        } else if (!slow) {
            float mr;
            double sr;
            block_running<THREADS>(run, c, mr, sr, tmp_f, tmp_d);
            const double log_z = log(sr);
            bool listed = false;
            if (by_groups) {
                u64 have = 0;
                for (uint32_t g = threadIdx.x; g < n_segs * 64; g += THREADS) have += groups[g] != 0;
                have = block_reduce<THREADS>(have, Add(), tmp);
                if (have >= R.r.k) {
                    const u64 kth = kth_of<THREADS>([&](uint32_t i) { return (u64)groups[i]; }, n_segs * 64, R.r.k, &lds);
                    for (uint32_t g = threadIdx.x; g < n_segs * 64; g += THREADS)
                        if (groups[g] != 0 && groups[g] >= (uint32_t)kth) hits[atomicAdd(&counts[1], 1u)] = (uint16_t)g;
                    R.gather((uint32_t)kth, list, counts, hits);
                    __syncthreads();
                    listed = count <= (uint32_t)L::CAP;
                    __syncthreads();
                }
            }
            if (!listed) {
                if (threadIdx.x == 0) count = 0;
                R.template histogram<false>(0, n_segs, M, hist);
                __syncthreads();
                u64 have = 0;
                for (uint32_t b = threadIdx.x; b < kBins; b += THREADS) have += hist[bin_at(b)];
                have = block_reduce<THREADS>(have, Add(), tmp);
                const Found<u64> f = find_cut([&](uint32_t b) { return hist[bin_at(b)]; }, have < R.r.k ? have : (u64)R.r.k);
                if (f.above + f.inside > (u64)L::CAP) {
                    slow = true;
                } else {
                    float from, above;
                    R.cut_scores(f.bin, true, from, above);
                    R.template collect<false>(0, n_segs, M, from, above, 0, nullptr, list, &count, L::CAP, stage);
                    __syncthreads();
                }
            }
            if (!slow) R.finish_list(list, count, M, log_z, row, &lds, tmp, out);
        }
        if (slow) R.slow(order_key(m), first, row, &lds, tmp, pick, out);
        __syncthreads();
    }
}

// Rows of more than 8192 classes: the steps as launches of their own, `parts` workgroups a row, so that a few
// rows fill the CUs and every step has the registers it needs (all steps in one launch of 1024 threads spilled
// 110 registers: 256 x 131072 f32 with settings a row took 189 to 287 us).  Between the launches, per row:
struct Top {      // of a part: its largest score (order key) over ~(its first class); the softmax denominator; a low score
    u64 key;
    double s;
    float m, low;
};
struct Step {     // where the cut lies
    u64 total, above;   // mass of all classes; weight of the bins before the cut's
    uint32_t bin, state;
    float m, from, up_to;   // the largest score; the scores that are listed
    uint32_t unused;
};
enum State : uint32_t { kNone, kCut, kOverflow };
struct Space {    // the workspace of a chunk of rows
    Top* tops;          // [rows][parts1]
    uint32_t* groups;   // [rows][64 segs], nullable
    u64* hist;          // [rows][parts2][kBins]
    u64* segs;          // [rows][n_segs]
    u64* list;          // [rows][kListCap]
    uint32_t* count;    // [rows]
    Step* steps;        // [rows]
    u64* totals;        // [rows][parts2]
    uint32_t parts1, per1, parts2, per2, n_segs;   // parts of a row and segments a part: of the scan, of the rest
};

template <int THREADS>
__device__ __forceinline__ u64 row_top(const Space& P, uint64_t row, u64* tmp, float& low) {
    u64 top = 0;
    low = INFINITY;
    for (uint32_t p = threadIdx.x; p < P.parts1; p += THREADS) {
        const u64 k = P.tops[row * P.parts1 + p].key;
        top = k > top ? k : top;
        low = fminf(low, P.tops[row * P.parts1 + p].low);
    }
    low = -block_reduce<THREADS>(-low, MaxF(), (float*)tmp);
    return block_reduce<THREADS>(top, MaxU(), tmp);
}

template <class T, bool kUnit>
__global__ __launch_bounds__(256) void scan_kernel(Rows<T> X, Settings S, int shift, Space P) {
    constexpr int THREADS = 256;
    __shared__ float tmp_f[4];
    __shared__ double tmp_d[4];
    __shared__ u64 tmp[4];
    const uint64_t row = blockIdx.x / P.parts1;
    const uint32_t part = blockIdx.x % P.parts1, s0 = part * P.per1, s1 = min(P.n_segs, s0 + P.per1);
    Long<T, kUnit, THREADS> R(X, S, row, shift);
    const Mode mode = R.mode();
    const float c = (float)(R.r.rt * 1.4426950408889634);
    float best, low;
    uint32_t best_seg;
    Running run;
    R.scan(s0, s1, mode == kList && R.by_groups(P.n_segs) ? P.groups + row * P.n_segs * 64 + s0 * 64 : nullptr, mode == kList,
           c, best, best_seg, low, run);
    low = -block_reduce<THREADS>(-low, MaxF(), tmp_f);
    const float m = block_reduce<THREADS>(best, MaxF(), tmp_f);
    u64 first = 0xFFFFFFFFu;
    if (R.r.greedy || R.r.min_p > 1.0)
        first = block_reduce<THREADS>((u64)R.first_at(m, best, best_seg), MinU(), tmp);
    float rm = 0.0f;
    double rs = 0.0;
    if (mode == kList) block_running<THREADS>(run, c, rm, rs, tmp_f, tmp_d);
    if (threadIdx.x == 0) {
        P.tops[row * P.parts1 + part] = Top{m == -INFINITY ? 0 : (u64)order_key(m) << 32 | (uint32_t)~first, rs, rm, low};
        if (part == 0) P.count[row] = 0;
    }
}

// Masses of the segments, or the part's histogram of masses or counts.  Bound by f64 instructions (21 a mass; 512 x
// 65537 bf16, masses of the whole rows: 34 us, 70% of the vector issue slots) and, for histograms, by LDS
// atomics (64 x 200001 f16: 24 us; 256 x 131072 f32: 27 us of counts, 41 of masses).
template <class T, bool kUnit>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 3 : 4) void weigh_kernel(Rows<T> X, Settings S, int shift, Space P) {
    constexpr int THREADS = 256;
    __shared__ u64 hist[kBinsPad];
    __shared__ u64 tmp[THREADS / 64];
    const uint64_t row = blockIdx.x / P.parts2;
    const uint32_t part = blockIdx.x % P.parts2, s0 = part * P.per2, s1 = min(P.n_segs, s0 + P.per2);
    Long<T, kUnit, THREADS> R(X, S, row, shift);
    const Mode mode = R.mode();
    if (mode == kGreedy || (mode == kList && P.groups && R.by_groups(P.n_segs))) return;
    float low;
    const u64 top = row_top<THREADS>(P, row, tmp, low);
    const float m = key_score((uint32_t)(top >> 32));
    if (top == 0 || R.whole_row(m, mode)) return;
    const Masses M{(double)m, R.r.rt * 1.4426950408889634, shift};
    if (mode == kWhole) {
        u64 all = R.weigh(s0, s1, M, R.r.min_p > 1.0 ? 0 : M.least(R.r.min_p), P.segs + row * P.n_segs);
        all = block_reduce<THREADS>(all, Add(), tmp);
        if (threadIdx.x == 0) P.totals[row * P.parts2 + part] = all;
        return;
    }
    for (uint32_t b = threadIdx.x; b < kBinsPad; b += THREADS) hist[b] = 0;
    __syncthreads();
    R.set_bins(m, low);
    if (mode == kNucleus) R.template histogram<true>(s0, s1, M, hist);
    else R.template histogram<false>(s0, s1, M, hist);
    __syncthreads();
    u64* to = P.hist + (row * P.parts2 + part) * kBins;
    for (uint32_t b = threadIdx.x; b < kBins; b += THREADS) to[b] = hist[bin_at(b)];
}

// The bin of the cut, once a row (by each of a row's workgroups in the pass after, it took longer than the pass).
template <class T, bool kUnit>
__global__ __launch_bounds__(1024) void cut_kernel(Rows<T> X, Settings S, int shift, Space P) {
    constexpr int THREADS = 1024;
    __shared__ u64 hist[kBinsPad];
    __shared__ u64 tmp[THREADS / 64];
    const uint64_t row = blockIdx.x;
    Long<T, kUnit, THREADS> R(X, S, row, shift);
    const Mode mode = R.mode();
    float low;
    const u64 top = row_top<THREADS>(P, row, tmp, low);
    const float m = key_score((uint32_t)(top >> 32));
    const bool list = mode == kList && !(P.groups && R.by_groups(P.n_segs));
    if ((mode != kNucleus && !list) || top == 0 || R.whole_row(m, mode)) {
        if (threadIdx.x == 0) P.steps[row].state = kNone;
        return;
    }
    R.set_bins(m, low);
    u64 total = 0;
    static_assert(THREADS == kBins, "a bin a thread");
#pragma unroll 8
    for (uint32_t p = 0; p < P.parts2; ++p) total += P.hist[(row * P.parts2 + p) * kBins + threadIdx.x];
    hist[bin_at(threadIdx.x)] = total;
    total = block_reduce<THREADS>(total, Add(), tmp);
    __syncthreads();
    const u64 want = !list ? nucleus_of(R.r.p, total) : total < R.r.k ? total : (u64)R.r.k;
    const Found<u64> f = find_cut([&](uint32_t b) { return hist[bin_at(b)]; }, want);
    const bool over = list && f.above + f.inside > kListCap;
    Step step{total, f.above, f.bin, over ? kOverflow : kCut, m, 0.0f, 0.0f, 0};
    R.cut_scores(f.bin, list, step.from, step.up_to);
    if (threadIdx.x == 0) P.steps[row] = step;
}

// The classes of the cut's bin (top_k: and of those before), and the segments' masses before it.  64 x 200001 f16: 34
// us; 256 x 131072 f32: 44 us with masses, 31 without; bound by f64 instructions and the lists' ballots.
template <class T, bool kUnit>
__global__ __launch_bounds__(256, 4) void collect_kernel(Rows<T> X, Settings S, int shift, Space P) {
    constexpr int THREADS = 256;
    __shared__ u64 stage[THREADS / 64 * Long<T, kUnit, THREADS>::kStage];
    const uint64_t row = blockIdx.x / P.parts2;
    const Step step = P.steps[row];
    if (step.state != kCut) return;
    const uint32_t part = blockIdx.x % P.parts2, s0 = part * P.per2, s1 = min(P.n_segs, s0 + P.per2);
    Long<T, kUnit, THREADS> R(X, S, row, shift);
    const Masses M{(double)step.m, R.r.rt * 1.4426950408889634, shift};
    u64* list = P.list + row * kListCap;
    if (R.mode() == kNucleus)
        R.template collect<true>(s0, s1, M, step.from, step.up_to, M.least(R.r.min_p), P.segs + row * P.n_segs, list,
                                 &P.count[row], kListCap, stage);
    else
        R.template collect<false>(s0, s1, M, step.from, step.up_to, 0, nullptr, list, &P.count[row], kListCap, stage);
}

// Rows whose cut needs no pass over the row: nothing allowed, the largest score, the whole row, and a small top_k
// from the maxima of the groups.  512 threads: what these steps wait for is barriers and LDS, and 8 waves
// wait less than 16 (1 x 131072 bf16, top_k 50: 15 us; whole rows 7).
template <class T, bool kUnit>
__global__ __launch_bounds__(512) void draw_direct_kernel(Rows<T> X, Settings S, int shift, Out out, Space P) {
    constexpr int THREADS = 512, W = THREADS / 64;
    typedef Long<T, kUnit, THREADS> L;
    __shared__ u64 list[L::CAP];
    __shared__ uint16_t hits[kGroupSegs * 64];
    __shared__ SelectLds lds;
    __shared__ u64 tmp[W], pick[2];
    __shared__ float tmp_f[W];
    __shared__ double tmp_d[W];
    __shared__ uint32_t count[2];
    const uint64_t row = blockIdx.x;
    L R(X, S, row, shift);
    const Mode mode = R.mode();
    const bool by_groups = mode == kList && R.by_groups(P.n_segs);
    constexpr int kGroupsEach = (int)(kGroupSegs * 64 / THREADS);
    uint32_t groups[kGroupsEach];   // (under way while the rest of the row's state is read)
#pragma unroll
    for (int j = 0; j < kGroupsEach; ++j) {
        const uint32_t g = j * THREADS + threadIdx.x;
        groups[j] = by_groups && g < P.n_segs * 64 ? P.groups[row * P.n_segs * 64 + g] : 0;
    }
    float low;
    const u64 top = row_top<THREADS>(P, row, tmp, low);
    if (top == 0) {
        if (threadIdx.x == 0) out.empty(row);
        return;
    }
    const float m = key_score((uint32_t)(top >> 32)), c = (float)(R.r.rt * 1.4426950408889634);
    const uint32_t first = ~(uint32_t)top;
    if (mode == kGreedy) {
        if (threadIdx.x == 0) out.put(row, first, 0.0);
        return;
    }
    if (mode != kWhole && !by_groups) return;
    if (R.whole_row(m, mode)) {
        R.slow((uint32_t)(top >> 32), first, row, &lds, tmp, pick, out);
        return;
    }
    const Masses M{(double)m, R.r.rt * 1.4426950408889634, shift};
    if (mode == kWhole) {
        u64 total = 0;
        for (uint32_t p = threadIdx.x; p < P.parts2; p += THREADS) total += P.totals[row * P.parts2 + p];
        total = block_reduce<THREADS>(total, Add(), tmp);
        if (R.r.min_p > 1.0) {
            if (threadIdx.x == 0) out.put(row, first, -M.log_of(total));
            return;
        }
        R.finish_segments(P.segs + row * P.n_segs, P.n_segs, M, kBins, 0, M.least(R.r.min_p), total, row, tmp, pick, out);
        return;
    }
    Running run;
    for (uint32_t p = threadIdx.x; p < P.parts1; p += THREADS) {
        const Top t = P.tops[row * P.parts1 + p];
        run.join(t.m, t.s, c);
    }
    float mr;
    double sr;
    block_running<THREADS>(run, c, mr, sr, tmp_f, tmp_d);
    const double log_z = log(sr);
    u64 have = 0;
#pragma unroll
    for (int j = 0; j < kGroupsEach; ++j) have += groups[j] != 0;
    if (threadIdx.x < 2) count[threadIdx.x] = 0;
    have = block_reduce<THREADS>(have, Add(), tmp);
    u64 kth = 0;   // (fewer groups than k: all that is allowed is listed)
    if (have >= R.r.k)
        kth = select<THREADS, false, true>(
                  [&](auto f) {
#pragma unroll
                      for (int j = 0; j < kGroupsEach; ++j)
                          if (groups[j]) f((u64)groups[j], 0);
                  },
                  R.r.k, &lds)
                  .from;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kGroupsEach; ++j)
        if (groups[j] != 0 && groups[j] >= (uint32_t)kth) hits[atomicAdd(&count[1], 1u)] = (uint16_t)(j * THREADS + threadIdx.x);
    R.gather((uint32_t)kth, list, count, hits);
    __syncthreads();
    const bool slow = count[0] > (uint32_t)L::CAP;
    if (!slow) R.finish_list(list, count[0], M, log_z, row, &lds, tmp, out);
    else R.slow((uint32_t)(top >> 32), first, row, &lds, tmp, pick, out);
}

// The others, a workgroup a row: the exact cut, and the draw (64 x 200001 f16 nucleus: 20 us; lists of 5000: 29 us).
// Bound by barriers and LDS.
template <class T, bool kUnit>
__global__ __launch_bounds__(1024) void draw_kernel(Rows<T> X, Settings S, int shift, Out out, Space P) {
    constexpr int THREADS = 1024, W = THREADS / 64;
    typedef Long<T, kUnit, THREADS> L;
    extern __shared__ u64 pool[];   // its segments' masses
    __shared__ SelectLds lds;
    __shared__ u64 tmp[W], pick[2];
    __shared__ float tmp_f[W];
    __shared__ double tmp_d[W];
    const uint64_t row = blockIdx.x;
    L R(X, S, row, shift);
    const Mode mode = R.mode();
    float low;
    const u64 top = row_top<THREADS>(P, row, tmp, low);
    const float m = key_score((uint32_t)(top >> 32));
    if (top == 0 || mode == kGreedy || mode == kWhole || (mode == kList && P.groups && R.by_groups(P.n_segs))) return;
    const uint32_t first = ~(uint32_t)top;
    const Masses M{(double)m, R.r.rt * 1.4426950408889634, shift};
    bool slow = R.whole_row(m, mode);
    if (!slow && mode == kNucleus) {
        const Step step = P.steps[row];
        const uint32_t n_list = P.count[row];
        const u64 least = M.least(R.r.min_p);
        slow = n_list > kListCap;
        if (!slow) {
            for (uint32_t s = threadIdx.x; s < P.n_segs; s += THREADS) pool[s] = P.segs[row * P.n_segs + s];
            Entries<THREADS, L::E> E;
            R.read_list(E, P.list + row * kListCap, n_list);
            E.weigh(M);
            __syncthreads();
            const Crossing x = select<THREADS, true, true>(
                [&](auto g) {
#pragma unroll
                    for (int e = 0; e < L::E; ++e)
                        if (E.key[e] && E.mass[e]) g(E.rank(e), E.mass[e]);
                },
                nucleus_of(R.r.p, step.total) - step.above, &lds);
            E.keep_from(x);
            E.drop_below(least);
#pragma unroll
            for (int e = 0; e < L::E; ++e)
                if (E.key[e] && E.mass[e]) atomicAdd(&pool[E.idx[e] / kSeg], E.mass[e]);
            __syncthreads();
            R.set_bins(m, low);
            R.finish_segments(pool, P.n_segs, M, step.bin, x.from, least, step.total, row, tmp, pick, out);
            return;
        }
    }
    if (!slow && mode == kList) {
        Running run;
        for (uint32_t p = threadIdx.x; p < P.parts1; p += THREADS) {
            const Top t = P.tops[row * P.parts1 + p];
            run.join(t.m, t.s, (float)(R.r.rt * 1.4426950408889634));
        }
        float mr;
        double sr;
        block_running<THREADS>(run, (float)(R.r.rt * 1.4426950408889634), mr, sr, tmp_f, tmp_d);
        const double log_z = log(sr);
        slow = P.steps[row].state == kOverflow;
        if (!slow) R.finish_list(P.list + row * kListCap, P.count[row], M, log_z, row, &lds, tmp, out);
    }
    if (slow) R.slow((uint32_t)(top >> 32), first, row, &lds, tmp, pick, out);
}

// Masses are sums of at most n weights of 1: they stay below 2^63.
int shift_of(uint32_t n) {
    int b = 0;
    while ((1ull << b) < n) ++b;
    return std::min(51, 62 - b);
}

template <class T, bool kUnit>
int launch_mid(const Rows<T>& X, const Settings& S, int shift, const Out& out, hipStream_t st) {
    typedef Long<T, kUnit, 256> L;
    const size_t n_segs = (X.classes + kSeg - 1) / kSeg;
    const size_t lds = sizeof(u64) * (L::CAP + n_segs) + (sizeof(uint32_t) + sizeof(uint16_t)) * 64 * n_segs;
    sample_long_kernel<T, kUnit, 256><<<row_grid(X.rows), 256, lds, st>>>(X, S, shift, out);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

// Long rows in chunks (the workspace stays below 64 MB up to 2^18 classes), each of at least 4 million scores.
constexpr uint64_t kChunkRows = 512;
constexpr uint32_t kMidClasses = 8192;
size_t align64(size_t v) { return (v + 63) & ~(size_t)63; }
// Parts of a row: the scan's workgroups of 4 waves take a tile each where the rows are few, 8 tiles where
// they fill the chip; the others (8 waves) likewise, with histograms to pay for.
Space plan(uint64_t rows, uint32_t n, unsigned char* base, size_t* bytes) {
    Space P{};
    P.n_segs = (n + kSeg - 1) / kSeg;
    auto split = [&](uint64_t wgs, uint32_t waves, uint32_t& parts, uint32_t& per) {
        const uint64_t want = std::max<uint64_t>(1, wgs / rows);
        per = (uint32_t)((P.n_segs + want - 1) / want + waves - 1) / waves * waves;
        parts = (P.n_segs + per - 1) / per;
    };
    split(2048, 4, P.parts1, P.per1);
    split(1024, 4, P.parts2, P.per2);
    size_t at = 0;
    auto take = [&](size_t size) {
        const size_t a = at;
        at += align64(size);
        return base ? base + a : nullptr;
    };
    P.tops = (Top*)take(sizeof(Top) * rows * P.parts1);
    P.groups = (uint32_t*)take(P.n_segs <= kGroupSegs ? sizeof(uint32_t) * 64 * P.n_segs * rows : 0);
    if (P.n_segs > kGroupSegs) P.groups = nullptr;
    P.hist = (u64*)take(sizeof(u64) * kBins * P.parts2 * rows);
    P.segs = (u64*)take(sizeof(u64) * P.n_segs * rows);
    P.list = (u64*)take(sizeof(u64) * kListCap * rows);
    P.count = (uint32_t*)take(sizeof(uint32_t) * rows);
    P.steps = (Step*)take(sizeof(Step) * rows);
    P.totals = (u64*)take(sizeof(u64) * P.parts2 * rows);
    *bytes = at;
    return P;
}

template <class T, bool kUnit>
int launch_split(const Rows<T>& X, const Settings& S, int shift, const Out& out, void* workspace, hipStream_t st) {
    // what the settings can ask for (settings a row: anything)
    const bool all_greedy = !S.t_rows && !(S.t > 0.0), any_list = S.k_rows || (S.k && S.k < X.classes);
    const bool all_list = !S.k_rows && any_list && !(S.min_p_rows || S.min_p > 1.0);
    const uint32_t n_segs = (X.classes + kSeg - 1) / kSeg;
    const bool list_by_groups = all_list && Long<T, kUnit, 512>::by_groups_of(S.k, n_segs);
    const bool any_cut = S.k_rows || S.p_rows || S.p < 1.0 || any_list;
    for (uint64_t r0 = 0; r0 < X.rows; r0 += kChunkRows) {
        const uint64_t m = std::min(kChunkRows, X.rows - r0);
        size_t bytes = 0;
        const Space P = plan(m, X.classes, (unsigned char*)workspace, &bytes);
        Rows<T> C = X;
        C.data += (int64_t)r0 * X.rs;
        C.rows = m;
        Settings Q = S;
        Q.uniform += r0;
        if (Q.t_rows) Q.t_rows += r0;
        if (Q.k_rows) Q.k_rows += r0;
        if (Q.p_rows) Q.p_rows += r0;
        if (Q.min_p_rows) Q.min_p_rows += r0;
        if (Q.allowed) Q.allowed += (int64_t)r0 * Q.allowed_stride;
        const Out o{out.index + r0, out.logprob ? out.logprob + r0 : nullptr};
        scan_kernel<T, kUnit><<<(unsigned)(m * P.parts1), 256, 0, st>>>(C, Q, shift, P);
        CLS_TRY(hipGetLastError());
        if (!all_greedy && !list_by_groups) {
            weigh_kernel<T, kUnit><<<(unsigned)(m * P.parts2), 256, 0, st>>>(C, Q, shift, P);
            CLS_TRY(hipGetLastError());
            if (any_cut) {
                cut_kernel<T, kUnit><<<(unsigned)m, 1024, 0, st>>>(C, Q, shift, P);
                CLS_TRY(hipGetLastError());
                collect_kernel<T, kUnit><<<(unsigned)(m * P.parts2), 256, 0, st>>>(C, Q, shift, P);
                CLS_TRY(hipGetLastError());
            }
        }
        draw_direct_kernel<T, kUnit><<<(unsigned)m, 512, 0, st>>>(C, Q, shift, o, P);
        CLS_TRY(hipGetLastError());
        if (all_greedy || !any_cut || list_by_groups) continue;
        const size_t lds = sizeof(u64) * P.n_segs;
        if (lds > 32 * 1024)
            CLS_TRY(hipFuncSetAttribute((const void*)draw_kernel<T, kUnit>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        draw_kernel<T, kUnit><<<(unsigned)m, 1024, lds, st>>>(C, Q, shift, o, P);
        CLS_TRY(hipGetLastError());
    }
    return CBH_OK;
}

template <class T, bool kUnit>
int launch_sample(const Rows<T>& X, const Settings& S, const Out& out, void* workspace, hipStream_t st) {
    const uint32_t n = X.classes;
    const int shift = shift_of(n);
    if (n <= 32) {
        const unsigned grid = row_grid((X.rows + 255) / 256);
        // (the pairs grow with the square: places in twos up to 12, then in fours and eights)
        if (n <= 4) sample_few_kernel<T, 4><<<grid, 256, 0, st>>>(X, S, out);
        else if (n <= 6) sample_few_kernel<T, 6><<<grid, 256, 0, st>>>(X, S, out);
        else if (n <= 8) sample_few_kernel<T, 8><<<grid, 256, 0, st>>>(X, S, out);
        else if (n <= 10) sample_few_kernel<T, 10><<<grid, 256, 0, st>>>(X, S, out);
        else if (n <= 12) sample_few_kernel<T, 12><<<grid, 256, 0, st>>>(X, S, out);
        else if (n <= 16) sample_few_kernel<T, 16><<<grid, 256, 0, st>>>(X, S, out);
        else if (n <= 24) sample_few_kernel<T, 24><<<grid, 256, 0, st>>>(X, S, out);
        else sample_few_kernel<T, 32><<<grid, 256, 0, st>>>(X, S, out);
    } else if (n <= 512) sample_short_kernel<T, kUnit, 64><<<row_grid(X.rows), 64, 0, st>>>(X, S, shift, out);
    else if (n <= 2048) sample_short_kernel<T, kUnit, 256><<<row_grid(X.rows), 256, 0, st>>>(X, S, shift, out);
    else if (n <= kMidClasses) return launch_mid<T, kUnit>(X, S, shift, out, st);
    else return launch_split<T, kUnit>(X, S, shift, out, workspace, st);
    CLS_TRY(hipGetLastError());
    return CBH_OK;
}

template <class T>
int run_sample(const void* scores, uint64_t rows, uint32_t n, int64_t rs, int64_t cs, const Settings& S, int32_t* index,
               float* logprob, void* workspace, hipStream_t st) {
    const Rows<T> X{(const T*)scores, rows, n, rs, cs};
    const Out out{index, logprob};
    return cs == 1 ? launch_sample<T, true>(X, S, out, workspace, st) : launch_sample<T, false>(X, S, out, workspace, st);
}

}  // namespace

extern "C" uint64_t cbh_sample_classes_workspace(uint64_t rows, uint32_t classes) {
    if (rows == 0 || classes <= kMidClasses || classes > kMaxClasses) return 0;   // (more is refused)
    // a last chunk of fewer rows has more parts a row, and at most as many in all as a full one may have
    size_t most = 0, bytes = 0;
    (void)plan(std::min(rows, kChunkRows), classes, nullptr, &most);
    if (rows > kChunkRows && rows % kChunkRows) {
        (void)plan(rows % kChunkRows, classes, nullptr, &bytes);
        most = std::max(most, bytes);
    }
    return most;
}

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
                return run_sample<float>(scores, rows, classes, row_stride, class_stride, S, index, logprob, workspace, st);
            case CBH_TYPE_F16:
                return run_sample<_Float16>(scores, rows, classes, row_stride, class_stride, S, index, logprob, workspace, st);
            default:
                return run_sample<bf16_t>(scores, rows, classes, row_stride, class_stride, S, index, logprob, workspace, st);
        }
    } catch (const std::exception& e) {
        return cbh_internal_fail(CBH_ERR_DEVICE, e.what());
    }
}
