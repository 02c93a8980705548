// Log probabilities of given classes, entropy and the most probable classes, in one pass over the scores.
//
// With d_j = (x_j - m) / t over the allowed classes, m the largest score:
//   Z = sum e^d_j,  E = -sum e^d_j d_j / Z,  logprob of c = d_c - log Z,  entropy = log Z + E
// log Z and E are both at least 0: the entropy is no difference of large numbers, and log p_j + entropy = d_j + E holds
// for a row of nearly equal scores too.  The sums run along with the running maximum: when it rises from m to m',
// sum e^d d becomes e^((m - m') / t) (sum e^d d + (m - m') / t sum e^d).
//
// What has to be read is the scores.  Without a k: 4096 x 65536 bf16 99 us, 537 MB at 5.4 TB/s, the memory's rate.  With one, bound by the
// row's end, a selection of dependent steps in LDS that four workgroups a CU hide in part: 4096 x 65536 bf16, k 5:
// 128 us; 777 x 50021 f32 with allowed classes, four entries and k 20: 50 us, 155 MB at 3.1 TB/s, on 777 workgroups.
#include "class_logprobs.hpp"

namespace {
using namespace cbh::cls;

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
            for (uint32_t i0 = threadIdx.x; i0 < parts * slots; i0 += 4 * THREADS) {
                u64 key[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) key[u] = i0 + u * THREADS < parts * slots ? keys[i0 + u * THREADS] : 0;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (key[u] == 0) continue;
                    const uint32_t at = atomicAdd(&nbest, 1u);
                    if (at < kMaxTop + kSpare) best[at] = key[u];
                }
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

// Segments of a row: one, unless the rows alone leave CUs idle and a row is long.  They start at a multiple of 32
// classes, a word of the allowed ones.
constexpr uint32_t kMinSeg = 8192, kMaxGroupSegs = 64;   // (12 x 238819 bf16, k 20: 27 us; segments of 16384 44, of 4096 28)
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
#define RUN_BY(THREADS, SEL, CAP, LDS) logprobs_kernel<T, kUnit, kMask, THREADS, SEL, CAP><<<grid, THREADS, LDS, st>>>(X, A, P.parts, seg, ps, pk)
#define RUN(SEL, CAP, LDS) (many ? RUN_BY(64, SEL, CAP, LDS) : RUN_BY(256, SEL, CAP, LDS))
    // by groups, or vectors, where k is at most a quarter of the shortest segment's
    const size_t lds = sizeof(uint32_t) * 64 * ((seg + kSeg - 1) / kSeg);
    constexpr uint32_t V = Pack<T>::V;
    const size_t lds_v = sizeof(uint32_t) * (kSeg / V) * ((seg + kSeg - 1) / kSeg);
    if (k == 0) {
        RUN(kNone, 2, 0);
    } else if (k * 4 <= shortest / kGroup) {
        // (a k of more than 128 is a quarter of the groups of rows beyond kWaveRow only)
        if (k <= 128) RUN(kGroups, 256, lds);
        else if (k <= 256) RUN_BY(256, kGroups, 512, lds);
        else RUN_BY(256, kGroups, 2048, lds);
    } else if (k * 4 <= shortest / V && lds_v <= 65536) {
        if (k <= 128) RUN(kVectors, 256, lds_v);
        else if (k <= 256) RUN(kVectors, 512, lds_v);
        else RUN(kVectors, 2048, lds_v);
    } else {
        RUN(kWhole, 2, 0);
    }
#undef RUN
#undef RUN_BY
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
    if (n <= kShort) return run_short_rows(X, A, st);
    const Plan P = plan_parts(rows, n);
    if (cs == 1) return A.allowed ? launch_rows<T, true, true>(X, A, P, workspace, st) : launch_rows<T, true, false>(X, A, P, workspace, st);
    return A.allowed ? launch_rows<T, false, true>(X, A, P, workspace, st) : launch_rows<T, false, false>(X, A, P, workspace, st);
}

}  // namespace

extern "C" uint64_t cbh_class_logprobs_workspace(uint64_t rows, uint32_t classes, uint32_t k) {
    if (classes <= kShort || classes > kMaxClasses) return 0;   // (more is refused)
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
