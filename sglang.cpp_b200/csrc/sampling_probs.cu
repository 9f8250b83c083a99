// The probabilities that a row of logits is sampled with: temperature, then the top_k largest, then the top_p of those.
//
//     w_i = exp((x_i - max x) / T),   p_i = w_i / (sum of the kept w) for kept i, 0 elsewhere
// Kept are the top_k largest (equal ones by index) and of those, in descending order, the entries whose running sum, their own
// weight included, stays within top_p times the sum of all top_k (never without the first).  T at most 1e-6: one-hot at the first
// maximum.
//
// A logit is one of 65536 bf16 patterns, and its weight is a function of the pattern: where a row is cut follows from the COUNTS of
// the patterns and one fp64 weight for each that occurs, which puts the borders where 64-bit sums do (fp32 weights summed entry
// by entry are off by 1e-7 of the sum, more than many an entry's weight).  Counted are the patterns of 2^-24 <= |x| < 2^8, 8192 of
// them; the few entries outside are added up one by one in fp64, by class (above, between, below).  Where a border falls among those
// it is found by bisection of the patterns instead, 16 rounds of counts or sums over the whole row.
//
// A CTA, or where rows are few a cluster of them, owns a row and goes over it from memory once and once or twice more, mostly from L2.
//     no filter:       sums under a running maximum; results.
//     top_k <= 256:    the lanes' maxima; of every warp's 32 the r-th largest, r = ceil(top_k / warps of the row): the smallest of these
//                      has top_k entries at or above it.  All such entries (some hundreds) are listed, from the threads whose maximum
//                      reaches it, sorted, weighed and cut; the results are zeros but for what is kept.
//     other filters:   maximum and counts; results.  In a cluster the counters meet by ranges of patterns: CTA r adds up all CTAs'
//                      counts of the r-th range from the top, weighs them, and the sums of the ranges before decide in which
//                      thread's patterns the cut falls.
// What bounds it: no filter, HBM (512 rows of 128256, 6 bytes per entry: 85 us, 0.71 of the copy bandwidth; of the 131 MB
// that are read twice, 82 come from memory again).
// The others wait for one another's meetings, sorts and counts, an atomic per entry in shared memory (320 rows of 151936: 65 us
// without filters, 77 with top_k 40, 133 to 138 with top_p 0.9; DRAM at 31 percent with all kinds mixed).  CTAs of 256 threads, five on an
// SM, so that one's loads and stores lie under another's sorting (at top_p 0.9 160 us with four, 141 with five, 155 with six,
// whose registers do not suffice).
// Far from these: a mask that leaves fewer entries than top_k, whose border is found by bisection (20 of 151936, top_k 40: 320 rows 710
// us, with top_p 1730; 8 rows 123 and 384); rows of an odd length, read 2 and written 4 bytes at a time (320 of 151935: 123 us
// without filters, 124 with top_k 40, 171 with top_p).
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 1 << 24;
constexpr int kPerSm = 5;                   // CTAs on an SM at once ...
constexpr int kMostPerSm = 16;              // ... and all in all, as far as clusters make them more
constexpr int kList = 2048;                 // entries that can be listed
constexpr int kBins = 8192;                 // counted patterns: half of them positive
constexpr int kHalf = kBins / 2;
constexpr uint32_t kLowMagnitude = 0x3380;  // 2^-24
static_assert(kLowMagnitude + kHalf == 0x4380, "2^8");

struct ProbsParams {
    float* out;
    const __nv_bfloat16* logits;
    int64_t ld;
    int rows, vocab, slice, cluster;
    const float* temperatures;
    const int32_t* top_k;
    const float* top_p;
};

// bf16 patterns of a value (which is one), in the order of the values.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t bits = __float_as_uint(x) >> 16;
    return (bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    const uint32_t bits = (key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu);
    return __uint_as_float(bits << 16);
}
constexpr uint32_t kLowestKey = 0x007fu;     // -inf
// Its place among the counted patterns in ascending order; outside [0, kBins): not counted.
__device__ __forceinline__ int bin_of(float x) {
    const uint32_t bits = __float_as_uint(x) >> 16;
    const int m = static_cast<int>(bits & 0x7fffu) - static_cast<int>(kLowMagnitude);
    if (static_cast<uint32_t>(m) >= static_cast<uint32_t>(kHalf)) return -1;
    return (bits & 0x8000u) ? kHalf - 1 - m : kHalf + m;
}
__device__ __forceinline__ float value_of_bin(int bin) {
    const uint32_t bits = bin >= kHalf ? kLowMagnitude + (bin - kHalf) : 0x8000u | (kLowMagnitude + (kHalf - 1 - bin));
    return __uint_as_float(bits << 16);
}

// Entries that are not counted: 0 above all that are, 1 between the positive and the negative, 2 below.
constexpr int kClasses = 3;

struct Meet {   // each CTA's copy: what the CTAs of a row tell one another
    float top[kMaxCluster];                  // the share's maximum
    int first[kMaxCluster];                  // where it is first
    float from[kMaxCluster];                 // its part of the top_k entries, by number, is at least this
    int listed[kMaxCluster];
    double sum[kMaxCluster];                 // weights: of the share under its maximum (no filters), of the CTA's range of patterns
    int count[kMaxCluster];                  // entries in that range
    int out_count[kMaxCluster][kClasses];
    double out_sum[kMaxCluster][kClasses];
    int equal[kMaxCluster];                  // entries of the share that equal the last kept value
    int turn_count[2][kMaxCluster];          // bisection, in turns
    double turn_sum[2][kMaxCluster];
    float value[2];                          // last kept value after top_k, after top_p ...
    int ties[2];                             // ... how many of it are kept ...
    double kept[2];                          // ... and the sum of the kept
    unsigned long long cut;                  // the last entry of the sorted list that is kept
};

__device__ __forceinline__ uint32_t remote(const void* p, int r) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(r));
    return a;
}
__device__ __forceinline__ void tell(const int* p, int ctas, int v) {
    for (int r = 0; r < ctas; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, r)), "r"(v) : "memory");
}
__device__ __forceinline__ void tell(const float* p, int ctas, float v) {
    for (int r = 0; r < ctas; ++r) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(p, r)), "f"(v) : "memory");
}
__device__ __forceinline__ void tell(const double* p, int ctas, double v) {
    for (int r = 0; r < ctas; ++r) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote(p, r)), "d"(v) : "memory");
}
__device__ __forceinline__ void tell(const unsigned long long* p, int ctas, unsigned long long v) {
    for (int r = 0; r < ctas; ++r) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, r)), "l"(v) : "memory");
}
__device__ __forceinline__ void meet_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The weight that decides: a is at most top, per_t = log2(e) / T.
__device__ __noinline__ double weight64(float a, float top, double per_t) {
    if (a == top) return 1.0;   // (also where both are infinite)
    if (a == -INFINITY) return 0.0;
    const double e = (static_cast<double>(a) - static_cast<double>(top)) * per_t;
    return e < -200.0 ? 0.0 : exp2(e);
}

// The weight of a, and by what factor the weight of a - step is smaller.
__device__ __noinline__ double2 weight_and_ratio(float a, float top, double per_t, float step) {
    const double e = (static_cast<double>(a) - static_cast<double>(top)) * per_t, d = -static_cast<double>(step) * per_t;
    const double w = exp2(e), ratio = exp2(d);
    return make_double2(a == top ? 1.0 : e >= -200.0 ? w : 0.0, ratio);
}

// Are exponents of the form a s - max s good enough in fp32?  Not where the second term is infinite or its rounding more than a half
// (nor, then, with a temperature of 0 or infinity).
__device__ __forceinline__ bool fp32_does(float top, float s) { return fabsf(top * s) < 4e6f && s > 1e-30f && s < 1e30f; }

// A logit: a NaN as -inf, one kind of zero.
__device__ __forceinline__ float clean(float x) { return fmaxf(x + 0.f, -INFINITY); }

// Two entries, a NaN as -inf.
__device__ __forceinline__ uint32_t number_or_low(uint32_t w) {
    uint32_t low = 0xff80ff80u;
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&w), *reinterpret_cast<__nv_bfloat162*>(&low));
    return *reinterpret_cast<const uint32_t*>(&m);
}
// The largest of eight entries (two at a time; a NaN loses against a number).
__device__ __forceinline__ float largest_of(const uint4& a) {
    auto pair = [](uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); };
    const __nv_bfloat162 m = __hmax2(__hmax2(pair(a.x), pair(a.y)), __hmax2(pair(a.z), pair(a.w)));
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&m);
    return fmaxf(fmaxf(bf16_lo(w), bf16_hi(w)) + 0.f, -INFINITY);
}

// ALIGNED: rows of both sides are read and written 16 bytes at a time; else entry by entry, neighbours by neighbouring threads.
template <bool FILTERS, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, kPerSm)
sampling_probs_kernel(const ProbsParams p) {
    __shared__ __align__(16) int hist[FILTERS ? kBins : 4];
    __shared__ Meet meet;
    __shared__ double s_d[kWarps];
    __shared__ float s_f[kWarps];
    __shared__ int s_i[kWarps], s_cut;
    __shared__ int s_count[kClasses], s_listed, s_owners;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = p.cluster, rank = static_cast<int>(blockIdx.x) % C, row = static_cast<int>(blockIdx.x) / C;
    const int begin = min(rank * p.slice, p.vocab), n = min(p.slice, p.vocab - begin);
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (waited for ahead of the first remote store)
    pdl_launch_dependents();
    pdl_wait_prior();
    const __nv_bfloat16* x = p.logits + static_cast<int64_t>(row) * p.ld + begin;
    float* out = p.out + static_cast<int64_t>(row) * p.vocab + begin;
    const float T = p.temperatures[row];
    const bool greedy = !(T > 1.0000001e-6f);
    int K = FILTERS && p.top_k != nullptr ? p.top_k[row] : 0;
    if (K < 1 || K > p.vocab) K = p.vocab;
    const float P = FILTERS && p.top_p != nullptr ? p.top_p[row] : 1.f;
    const bool want_k = K < p.vocab, want_p = P < 1.f;
    const bool filter = FILTERS && !greedy && (want_k || want_p);
    const double per_t = 1.4426950408889634 / static_cast<double>(T);
    const float s_hi = static_cast<float>(per_t);

    // eight(their patterns, the first one's place) or one(entry, place) for all of the share, a round's loads ahead of its work.
    auto all_of = [&](auto eight, auto one) {
        if (ALIGNED) {
            constexpr int kRound = 4;
            const int vectors = n >> 3;
            for (int v0 = tid; v0 < vectors; v0 += kRound * kThreads) {
                uint4 a[kRound];
#pragma unroll
                for (int j = 0; j < kRound; ++j)
                    if (v0 + j * kThreads < vectors) a[j] = __ldg(reinterpret_cast<const uint4*>(x) + v0 + j * kThreads);
#pragma unroll
                for (int j = 0; j < kRound; ++j) {
                    if (v0 + j * kThreads >= vectors) break;
                    eight(a[j], (v0 + j * kThreads) * 8);
                }
            }
            if (const int i = vectors * 8 + tid; i < n) one(clean(__bfloat162float(x[i])), i);
        } else {
            constexpr int kRound = 8;
            for (int i0 = tid; i0 < n; i0 += kRound * kThreads) {
                float a[kRound];
#pragma unroll
                for (int j = 0; j < kRound; ++j) a[j] = i0 + j * kThreads < n ? clean(__bfloat162float(x[i0 + j * kThreads])) : -INFINITY;
#pragma unroll
                for (int j = 0; j < kRound; ++j) {
                    if (i0 + j * kThreads >= n) break;
                    one(a[j], i0 + j * kThreads);
                }
            }
        }
    };
    // f(eight neighbouring entries, or one; how many; the first one's place); eight of which none reaches the bound go to else_f instead.
    auto each_from = [&](float bound, auto f, auto else_f) {
        all_of(
            [&](const uint4& a, int at) {
                if (bound > -INFINITY && largest_of(a) < bound) {
                    else_f(at);
                    return;
                }
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = clean((e & 1) ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]));
                f(y, std::integral_constant<int, 8>{}, at);
            },
            [&](float a, int at) {
                const float y[1] = {a};
                f(y, std::integral_constant<int, 1>{}, at);
            });
    };
    auto each = [&](auto f) { each_from(-INFINITY, f, [](int) {}); };
    // This thread's largest entry.
    auto largest = [&]() {
        float top = -INFINITY;
        all_of([&](const uint4& a, int) { top = fmaxf(top, largest_of(a)); }, [&](float a, int) { top = fmaxf(top, a); });
        return top;
    };
    // Eight neighbouring results, whole sectors at once where rows begin with one (halves of them: 20 percent of the time).
    const bool sectors = ALIGNED && reinterpret_cast<uintptr_t>(out) % 32 == 0;
    auto store8 = [&](const float (&z)[8], int at) {
        if (sectors) {
            asm volatile("st.global.cs.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + at), "f"(z[0]), "f"(z[1]), "f"(z[2]), "f"(z[3]),
                         "f"(z[4]), "f"(z[5]), "f"(z[6]), "f"(z[7])
                         : "memory");
        } else {
            __stcs(reinterpret_cast<float4*>(out + at), make_float4(z[0], z[1], z[2], z[3]));
            __stcs(reinterpret_cast<float4*>(out + at) + 1, make_float4(z[4], z[5], z[6], z[7]));
        }
    };
    // value(entry, place) to the results.
    auto store_from = [&](float bound, auto value) {   // (entries below the bound: 0)
        each_from(bound, [&](const auto& y, auto count, int at) {
            if constexpr (count() == 8) {
                float z[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = value(y[e], at + e);
                store8(z, at);
            } else {
                __stcs(out + at, value(y[0], at));
            }
        }, [&](int at) {
            const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            store8(z, at);
        });
    };
    auto store = [&](auto value) { store_from(-INFINITY, value); };

    if (FILTERS && tid == 0) {
        meet.value[0] = meet.value[1] = -INFINITY;
        meet.ties[0] = meet.ties[1] = 0x7fffffff;
        s_cut = 0x7fffffff;
        s_listed = s_owners = 0;
    }
    bool met = false;   // the first wait for the cluster is done
    auto meet_first = [&]() {
        if (!met) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        met = true;
    };
    if constexpr (FILTERS) {
        if (filter && want_k && K <= kThreads) {
            // ---- a bound that top_k entries reach ----
            float top = largest();
            const float own_top = top;
            const int r = (K + kWarps * C - 1) / (kWarps * C);
            float sorted = top;   // of the lanes, the largest first
#pragma unroll
            for (int size = 2; size <= 32; size *= 2)
#pragma unroll
                for (int o = size / 2; o > 0; o /= 2) {
                    const float other = __shfl_xor_sync(0xffffffffu, sorted, o);
                    const bool down = (lane & size) == 0 || size == 32, low = (lane & o) == 0;
                    sorted = low == down ? fmaxf(sorted, other) : fminf(sorted, other);
                }
            const float reach = __shfl_sync(0xffffffffu, sorted, r - 1);
            top = __shfl_sync(0xffffffffu, sorted, 0);
            if (lane == 0) {
                s_f[warp] = reach;
                s_d[warp] = top;
            }
            __syncthreads();
            float from = INFINITY;
            for (int w = 0; w < kWarps; ++w) {
                from = fminf(from, s_f[w]);
                top = fmaxf(top, static_cast<float>(s_d[w]));
            }
            meet_first();
            if (tid == 0) {
                tell(&meet.top[rank], C, top);
                tell(&meet.from[rank], C, from);
            }
            meet_all();
            float xmax = -INFINITY;
            for (int i = 0; i < C; ++i) {
                from = fminf(from, meet.from[i]);
                xmax = fmaxf(xmax, meet.top[i]);
            }
            // ---- the entries that reach it, by value and place in one word, the larger value and the earlier place the smaller word ----
            uint64_t* list = reinterpret_cast<uint64_t*>(hist) + kList;   // this share's; all of them sorted ahead of it
            uint64_t* all = reinterpret_cast<uint64_t*>(hist);
            auto take = [&](const auto& y, auto count, int at) {
#pragma unroll
                for (int e = 0; e < count(); ++e)
                    if (y[e] >= from) {
                        const int i = atomicAdd(&s_listed, 1);
                        if (i < kList) list[i] = static_cast<uint64_t>(0xffffu - key_of(y[e])) << 32 | static_cast<uint32_t>(begin + at + e);
                    }
            };
            // They lie with the threads whose maximum reaches it: where these are few, all go over those threads' entries together (a
            // round over everything took 8.6 us of a CTA's 31).
            int* owner = hist;   // (ahead of the list)
            if (ALIGNED && own_top >= from && from > -INFINITY) owner[atomicAdd(&s_owners, 1)] = tid;
            __syncthreads();
            if (from > -INFINITY) {
                if (ALIGNED && s_owners * 2 <= kThreads) {
                    constexpr int kRound = 4;
                    const int vectors = n >> 3, each_has = (vectors + kThreads - 1) / kThreads, items = s_owners * each_has;
                    for (int i0 = tid; i0 < items; i0 += kRound * kThreads) {
                        uint4 a[kRound];
                        int v[kRound];
#pragma unroll
                        for (int j = 0; j < kRound; ++j) {
                            const int i = i0 + j * kThreads, o = i / each_has;
                            v[j] = i < items ? owner[o] + (i - o * each_has) * kThreads : vectors;
                            if (v[j] < vectors) a[j] = __ldg(reinterpret_cast<const uint4*>(x) + v[j]);
                        }
#pragma unroll
                        for (int j = 0; j < kRound; ++j) {
                            if (v[j] >= vectors || largest_of(a[j]) < from) continue;
                            const uint32_t w[4] = {a[j].x, a[j].y, a[j].z, a[j].w};
                            float y[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[e] = clean((e & 1) ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]));
                            take(y, std::integral_constant<int, 8>{}, v[j] * 8);
                        }
                    }
                    if (const int i = vectors * 8 + tid; i < n) {
                        const float y[1] = {clean(__bfloat162float(x[i]))};
                        take(y, std::integral_constant<int, 1>{}, i);
                    }
                } else {
                    each_from(from, take, [](int) {});
                }
            }
            __syncthreads();
            if (tid == 0) tell(&meet.listed[rank], C, from > -INFINITY ? s_listed : kList + 1);
            meet_all();
            int total = 0;
            for (int i = 0; i < C; ++i) total += min(meet.listed[i], kList + 1);
            if (total <= kList) {
                // Zeros everywhere, while the first CTA sorts all the lists.  (Every CTA sorting them: 64 rows of 128256 28.4 us, so 24.7; 320
                // of 151936 79.3 and 76.6; but 6 of 32000 12.1 and 12.6.)
                if (ALIGNED) {
                    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    for (int v = tid; v < n >> 3; v += kThreads) store8(z, v * 8);
                }
                for (int i = (ALIGNED ? n & ~7 : 0) + tid; i < n; i += kThreads) __stcs(out + i, 0.f);
                if (rank == 0) {
                    int size = 32;
                    while (size < total) size *= 2;
                    for (int i = tid; i < size; i += kThreads) {
                        uint64_t word = ~0ull;
                        int at = i, who = 0;
                        while (who < C - 1 && at >= meet.listed[who]) at -= meet.listed[who++];
                        if (i < total) {
                            if (C == 1) word = list[i];
                            else asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(word) : "r"(remote(list + at, who)));
                        }
                        all[i] = word;
                    }
                    __syncthreads();
                    // (Thread i's pair lies in the 64 words of its warp as long as they are at most 32 apart: no need to wait for other
                    // warps.)
                    for (int run = 2; run <= size; run *= 2) {
                        if (run > 64) __syncthreads();
                        for (int o = run / 2; o > 0; o /= 2) {
                            for (int i = tid; i < size / 2; i += kThreads) {
                                const int a = 2 * i - (i & (o - 1)), b = a + o;
                                const uint64_t wa = all[a], wb = all[b];
                                if ((wa > wb) == ((a & run) == 0)) {
                                    all[a] = wb;
                                    all[b] = wa;
                                }
                            }
                            if (o > 32) __syncthreads();
                            else __syncwarp();
                        }
                    }
                    __syncthreads();
                    // ---- weights of the first top_k, and how many of them stay ----
                    const uint64_t word = all[tid];   // (at least 32; behind them whatever is there is not used)
                    const bool there = tid < K && tid < total;
                    const double w = there ? weight64(value_of(0xffffu - static_cast<uint32_t>(word >> 32)), xmax, per_t) : 0.0;
                    double upto = w;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double d = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += d;
                    }
                    if (lane == 31) s_d[warp] = upto;
                    __syncthreads();
                    double sum = 0.0, ahead = 0.0;
                    for (int i = 0; i < kWarps; ++i) {
                        if (i == warp) ahead = sum;
                        sum += s_d[i];
                    }
                    upto += ahead;
                    const bool stays = there && w > 0.0 && (!want_p || tid == 0 || upto <= fmax(static_cast<double>(P), 0.0) * sum);
                    const uint32_t ends = __ballot_sync(0xffffffffu, !stays);
                    if (lane == 0) s_i[warp] = ends != 0 ? warp * 32 + __ffs(ends) - 1 : kThreads;
                    __syncthreads();
                    int stay = kThreads;
                    for (int i = 0; i < kWarps; ++i) stay = min(stay, s_i[i]);
                    double kept = warp_sum(tid < stay ? w : 0.0);
                    if (lane == 0) s_d[warp] = kept;
                    __syncthreads();
                    kept = 0.0;
                    for (int i = 0; i < kWarps; ++i) kept += s_d[i];
                    if (tid == 0) {
                        tell(&meet.kept[0], C, kept);
                        tell(&meet.cut, C, all[max(stay - 1, 0)]);
                    }
                }
                meet_all();   // (also: the zeros of this CTA are ahead of what is kept, and nothing remote is touched behind this)
                const double kept = meet.kept[0];
                for (int i = tid; i < min(s_listed, kList); i += kThreads) {
                    const uint64_t word = list[i];
                    if (word <= meet.cut)
                        out[static_cast<int>(word & 0xffffffffu) - begin] =
                            static_cast<float>(weight64(value_of(0xffffu - static_cast<uint32_t>(word >> 32)), xmax, per_t) / kept);
                }
                return;
            }
            // (too many: counted like the others.  The lists have been read by nobody.)
        }
    }
    // ---- the maximum; without filters also the sum under a running one, with them the counts ----
    float top = -INFINITY, part = 0.f, at = -INFINITY;
    bool outside = false;
    if (FILTERS && filter) {
        for (int i = tid; i < kBins / 4; i += kThreads) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
        if (tid < kClasses) s_count[tid] = 0;
        __syncthreads();
        auto count_one = [&](uint32_t bits) {   // (patterns outside may be a NaN's: looked at again below)
            const int m = static_cast<int>(bits & 0x7fffu) - static_cast<int>(kLowMagnitude);
            const int bin = kHalf + (m ^ (static_cast<int>(bits << 16) >> 31));
            if (static_cast<uint32_t>(m) < static_cast<uint32_t>(kHalf)) atomicAdd(&hist[bin], 1);
            else outside = true;
        };
        all_of(
            [&](const uint4& a, int) {
                top = fmaxf(top, largest_of(a));
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    count_one(w[e] & 0xffffu);
                    count_one(w[e] >> 16);
                }
            },
            [&](float a, int) {
                top = fmaxf(top, a);
                count_one(__float_as_uint(a) >> 16);
            });
    } else if (greedy) {
        top = largest();
    } else {
        // 2^(y s - at), at = s times the maximum so far.  Where that is below -2^30 there is nothing but a mask's low numbers so far, which
        // are nothing beside a maximum that fp32 does for: as its own reference at would be off by more than an exponent's range.
        constexpr float kLowest = -1073741824.f;
        all_of(
            [&](const uint4& a, int) {
                const float here = largest_of(a);
                if (here > top) {
                    const float now = fmaxf(here * s_hi, kLowest);
                    part *= exp2f(at - now);   // (the first time: nothing)
                    top = here;
                    at = now;
                }
                const uint32_t w[4] = {number_or_low(a.x), number_or_low(a.y), number_or_low(a.z), number_or_low(a.w)};
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += ex2_approx(fmaf((e & 1) ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]), s_hi, -at));
                if (top > -INFINITY) part += sum;
            },
            [&](float a, int) {
                if (a > top) {
                    const float now = fmaxf(a * s_hi, kLowest);
                    part *= exp2f(at - now);
                    top = a;
                    at = now;
                }
                if (top > -INFINITY) part += ex2_approx(fmaf(a, s_hi, -at));
            });
    }
    const float my_top = top;
    top = warp_max(top);
    if (lane == 0) s_f[warp] = top;
    outside = __syncthreads_or(outside);
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_f[w]);
    const bool odd = !fp32_does(top, s_hi);
    if (!greedy && !filter) {   // this share's sum under its maximum
        double sum = 0.0;
        if (odd) each([&](const auto& y, auto count, int) {
            for (int e = 0; e < count(); ++e) sum += weight64(y[e], top, per_t);
        });
        else if (my_top > -INFINITY) sum = static_cast<double>(part) * exp2(static_cast<double>(at) - static_cast<double>(top) * s_hi);
        sum = warp_sum(sum);
        if (lane == 0) s_d[warp] = sum;
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < kWarps; ++w) sum += s_d[w];
        meet_first();
        if (tid == 0) tell(&meet.sum[rank], C, sum);
    } else {
        meet_first();
    }
    if (tid == 0) tell(&meet.top[rank], C, top);
    meet_all();   // also: everyone's counters are complete
    float xmax = -INFINITY;
    for (int r = 0; r < C; ++r) xmax = fmaxf(xmax, meet.top[r]);

    if (greedy) {   // one-hot at the first maximum of all shares
        int at = 0x7fffffff;
        each([&](const auto& y, auto count, int place) {
#pragma unroll
            for (int e = 0; e < count(); ++e)
                if (y[e] == xmax) at = min(at, begin + place + e);
        });
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) s_i[warp] = at;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) at = min(at, s_i[w]);
        if (tid == 0) tell(&meet.first[rank], C, at);
        meet_all();
        int first = 0x7fffffff;
        for (int r = 0; r < C; ++r) first = min(first, meet.first[r]);
        store([&](float, int place) { return begin + place == first ? 1.f : 0.f; });
        return;
    }
    if (xmax == -INFINITY) {   // nothing but -inf and NaN
        store([](float, int) { return 0.f; });
        return;
    }

    // Weights.  fp64 for the sums that decide; for the results fp32: 2^(a s - c) with c = max s rounded, whose rounding, the same for all,
    // is part of the factor behind it.  s is rounded too: an entry 2^e below the largest is off by |e| 2^-23 of itself.
    const float c = xmax * s_hi;
    const bool plain = fp32_does(xmax, s_hi);
    // Results of the entries above or at `bound` for which keeps(entry, place); 0 elsewhere.
    auto finish = [&](double kept, float bound, auto keeps) {
        if (plain) {
            const float factor = static_cast<float>(exp2(static_cast<double>(c) - static_cast<double>(xmax) * s_hi) / kept);
            store_from(bound, [&](float a, int place) { return keeps(a, place) ? ex2_approx(fmaf(a, s_hi, -c)) * factor : 0.f; });
        } else {
            store_from(bound, [&](float a, int place) { return keeps(a, place) ? static_cast<float>(weight64(a, xmax, per_t) / kept) : 0.f; });
        }
    };

    if (!filter) {
        double sum = 0.0;
        for (int r = 0; r < C; ++r)
            sum += plain ? meet.sum[r] * exp2((static_cast<double>(meet.top[r]) - static_cast<double>(xmax)) * s_hi)
                         : meet.sum[r] * weight64(meet.top[r], xmax, per_t);
        finish(sum, -INFINITY, [](float, int) { return true; });
        return;
    }
    if constexpr (FILTERS) {
        // ---- entries that are not counted ----
        double out_sum[kClasses] = {0.0, 0.0, 0.0};
        if (outside) {   // (a round of its own: one row in hundreds has any, but every one with a mask: 320 rows at top_p 0.9 133 us, so 164)
            int out_count[kClasses] = {0, 0, 0};
            each([&](const auto& y, auto count, int) {
#pragma unroll
                for (int e = 0; e < count(); ++e) {
                    if (bin_of(y[e]) >= 0) continue;
                    const double w = weight64(y[e], xmax, per_t);
                    const int c = y[e] >= 256.f ? 0 : y[e] <= -256.f ? 2 : 1;
#pragma unroll
                    for (int i = 0; i < kClasses; ++i)
                        if (i == c) {
                            out_sum[i] += w;
                            ++out_count[i];
                        }
                }
            });
#pragma unroll
            for (int c = 0; c < kClasses; ++c) {
                const double sum = warp_sum(out_sum[c]);
                const int count = __reduce_add_sync(0xffffffffu, out_count[c]);
                if (lane == 0) {
                    s_d[warp] = sum;
                    atomicAdd(&s_count[c], count);
                }
                __syncthreads();
                out_sum[c] = 0.0;
                for (int w = 0; w < kWarps; ++w) out_sum[c] += s_d[w];
                __syncthreads();
            }
        }
        if (tid < kClasses) {
            tell(&meet.out_count[rank][tid], C, outside ? s_count[tid] : 0);
            tell(&meet.out_sum[rank][tid], C, tid == 0 ? out_sum[0] : tid == 1 ? out_sum[1] : out_sum[2]);
        }
        // ---- this CTA's range of patterns, a run of them per thread, from the top down ----
        const int bins = kBins / C / kThreads;   // 4 .. 32
        const int bin_top = kBins - 1 - (rank * kThreads + tid) * bins;
        int my_count = 0;
        double my_sum = 0.0;
        // Four patterns at a time, the CTAs' counts in one load each: their counts and weights in descending order.  (Four lie in one
        // binade: their values are a step apart and their weights a factor.  A load and an exponential for each took 21 us of a CTA's 67.)
        auto four = [&](int top, int (&c)[4]) {
            int4 v = make_int4(0, 0, 0, 0);
            if (C == 1) {
                v = *reinterpret_cast<const int4*>(&hist[top - 3]);
            } else {
#pragma unroll
                for (int r = 0; r < kMaxCluster; ++r) {
                    int4 u = make_int4(0, 0, 0, 0);
                    if (r < C)
                        asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                                     : "r"(remote(&hist[top - 3], r)));
                    v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                }
            }
            c[0] = v.w, c[1] = v.z, c[2] = v.y, c[3] = v.x;
            return (v.x | v.y | v.z | v.w) != 0;
        };
        auto weights = [&](int top, double (&w)[4]) {
            int k = 0;   // (those above the maximum do not occur)
            while (k < 3 && value_of_bin(top - k) > xmax) ++k;
            const double2 f = weight_and_ratio(value_of_bin(top - k), xmax, per_t, value_of_bin(top) - value_of_bin(top - 1));
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = i < k ? 0.0 : i == k ? f.x : w[i - 1] * f.y;
        };
#pragma unroll 1
        for (int i = 0; i < bins; i += 4) {
            int c[4];
            if (!four(bin_top - i, c)) continue;
            double w[4];
            weights(bin_top - i, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                my_count += c[k];
                my_sum += c[k] * w[k];
            }
        }
        // Counts and sums of the threads before this one.  `lower` of a thread is `upper` of the one before it to the last bit, so
        // that exactly one thread's run holds a border.
        int incl = my_count;
        double upper = my_sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int c = __shfl_up_sync(0xffffffffu, incl, o);
            const double d = __shfl_up_sync(0xffffffffu, upper, o);
            if (lane >= o) {
                incl += c;
                upper += d;
            }
        }
        double lower = __shfl_up_sync(0xffffffffu, upper, 1);
        if (lane == 0) lower = 0.0;
        if (lane == 31) {
            s_i[warp] = incl;
            s_d[warp] = upper;
        }
        __syncthreads();
        int warp_count = 0, cta_count = 0;
        double warp_before = 0.0, cta_sum = 0.0;
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) {
                warp_count = cta_count;
                warp_before = cta_sum;
            }
            cta_count += s_i[w];
            cta_sum += s_d[w];
        }
        if (tid == 0) {
            tell(&meet.count[rank], C, cta_count);
            tell(&meet.sum[rank], C, cta_sum);
        }
        meet_all();
        // In descending order: class 0, positive patterns, class 1, negative patterns, class 2.  A run of patterns has one sign, a
        // CTA's range has too unless it is all of them.
        const bool negative = bin_top < kHalf;
        int class_count[kClasses] = {0, 0, 0};
        double class_sum[kClasses] = {0.0, 0.0, 0.0};
        int above = warp_count + incl - my_count, counted = 0;
        double range_sum = 0.0, counted_sum = 0.0;
        for (int r = 0; r < C; ++r) {
#pragma unroll
            for (int c = 0; c < kClasses; ++c) {
                class_count[c] += meet.out_count[r][c];
                class_sum[c] += meet.out_sum[r][c];
            }
            if (r < rank) above += meet.count[r];
            if (r == rank) range_sum = counted_sum;
            counted += meet.count[r];
            counted_sum += meet.sum[r];
        }
        const double head = class_sum[0] + (negative ? class_sum[1] : 0.0);
        above += class_count[0] + (negative ? class_count[1] : 0);
        lower = head + (range_sum + (warp_before + lower));
        upper = head + (range_sum + (warp_before + upper));
        double kept = (class_sum[0] + class_sum[1]) + counted_sum + class_sum[2];
        float last = -INFINITY;      // kept: entries above it, and of it the first `ties`
        int ties = 0x7fffffff;
        bool missed = false;         // a border is not among the counted patterns
        // ---- top_k: the thread whose run holds the K-th largest ----
        if (want_k) {
            if (above < K && K <= above + my_count) {
                int c_run = above;
                double s_run = lower;
                bool found = false;
#pragma unroll 1
                for (int i = 0; i < bins && !found; i += 4) {
                    int c[4];
                    if (!four(bin_top - i, c)) continue;
                    double w[4];
                    weights(bin_top - i, w);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (!found && K <= c_run + c[k]) {
                            tell(&meet.value[0], C, value_of_bin(bin_top - i - k));
                            tell(&meet.ties[0], C, K - c_run);
                            tell(&meet.kept[0], C, s_run + (K - c_run) * w[k]);
                            found = true;
                        }
                        c_run += c[k];
                        s_run += c[k] * w[k];
                    }
                }
            }
            meet_all();
            missed = meet.ties[0] == 0x7fffffff;
            last = meet.value[0];
            ties = meet.ties[0];
            if (!missed) kept = meet.kept[0];
        }
        // ---- top_p of those ----
        const double share = fmax(static_cast<double>(P), 0.0);
        if (want_p && !missed) {
            const double budget = share * kept;
            if (my_count > 0 && value_of_bin(bin_top) >= last && (lower <= budget || above == 0) && upper > budget) {
                int c_run = above;
                double s_run = lower;
                bool found = false;
#pragma unroll 1
                for (int i = 0; i < bins && !found; i += 4) {
                    int c[4];
                    if (!four(bin_top - i, c)) continue;
                    double w[4];
                    weights(bin_top - i, w);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float a = value_of_bin(bin_top - i - k);
                        if (found || a < last || c[k] == 0) continue;
                        if (a == last) c[k] = min(c[k], ties);
                        if (s_run + c[k] * w[k] > budget) {
                            const double fit = fmin(fmax(floor((budget - s_run) / w[k]), 0.0), static_cast<double>(c[k]));
                            int j = static_cast<int>(fit);
                            if (c_run == 0 && j == 0) j = 1;
                            tell(&meet.value[1], C, a);
                            tell(&meet.ties[1], C, j);
                            tell(&meet.kept[1], C, s_run + j * w[k]);
                            found = true;
                        }
                        c_run += c[k];
                        s_run += c[k] * w[k];
                    }
                }
            }
            meet_all();
            // Not found: the border is in a class, or rounding has left none (then all of the top_k stay).
            if (meet.ties[1] != 0x7fffffff) {
                last = meet.value[1];
                ties = meet.ties[1];
                kept = meet.kept[1];
            } else {
                const bool in_class = (class_count[0] > 0 && budget < class_sum[0]) || (class_count[1] > 0) || (class_count[2] > 0);
                missed = in_class;
            }
        }
        if (missed) {
            // ---- bisection of the patterns: the last one with at least K entries at or above it; then the last one whose sum at or
            //      above it, within those, exceeds the budget ----
            int turn = 0;
            auto all_counts = [&](int count) {
                count = __reduce_add_sync(0xffffffffu, count);
                __syncthreads();
                if (lane == 0) s_i[warp] = count;
                __syncthreads();
                count = 0;
                for (int w = 0; w < kWarps; ++w) count += s_i[w];
                if (tid == 0) tell(&meet.turn_count[turn & 1][rank], C, count);
                meet_all();
                count = 0;
                for (int r = 0; r < C; ++r) count += meet.turn_count[turn & 1][r];
                ++turn;
                return count;
            };
            auto all_sums = [&](double sum) {
                sum = warp_sum(sum);
                __syncthreads();
                if (lane == 0) s_d[warp] = sum;
                __syncthreads();
                sum = 0.0;
                for (int w = 0; w < kWarps; ++w) sum += s_d[w];
                if (tid == 0) tell(&meet.turn_sum[turn & 1][rank], C, sum);
                meet_all();
                sum = 0.0;
                for (int r = 0; r < C; ++r) sum += meet.turn_sum[turn & 1][r];
                ++turn;
                return sum;
            };
            auto count_from = [&](uint32_t key) {   // entries at or above a pattern
                int count = 0;
                for (int i = tid; i < n; i += kThreads) count += key_of(clean(__bfloat162float(x[i]))) >= key ? 1 : 0;
                return all_counts(count);
            };
            last = -INFINITY;
            ties = 0x7fffffff;
            if (want_k) {
                uint32_t lo = 0, hi = 0x10000u;   // (there are at least K at or above lo, fewer at or above hi)
                while (hi - lo > 1) {
                    const uint32_t mid = (lo + hi) >> 1;
                    if (count_from(mid) >= K) lo = mid; else hi = mid;
                }
                last = value_of(lo);
                ties = K - count_from(lo + 1);
            }
            const float floor_value = last;
            const int floor_ties = ties;
            auto sum_from = [&](uint32_t key) {     // within the top_k
                const float from = key <= 0xffffu ? value_of(key) : INFINITY;
                double sum = 0.0;
                for (int i = tid; i < n; i += kThreads) {
                    const float a = clean(__bfloat162float(x[i]));
                    if (key <= 0xffffu && a >= from && a > floor_value) sum += weight64(a, xmax, per_t);
                }
                sum = all_sums(sum);
                if (floor_ties != 0x7fffffff && key <= 0xffffu && floor_value >= from) sum += floor_ties * weight64(floor_value, xmax, per_t);
                return sum;
            };
            kept = sum_from(kLowestKey);
            if (want_p) {
                const double budget = share * kept;
                uint32_t lo = kLowestKey, hi = key_of(xmax) + 1;   // (the sum from lo exceeds the budget, the one from hi does not)
                if (kept > budget) {
                    while (hi - lo > 1) {
                        const uint32_t mid = (lo + hi) >> 1;
                        if (sum_from(mid) > budget) lo = mid; else hi = mid;
                    }
                    const float a = value_of(lo);
                    const double before = sum_from(lo + 1), w = weight64(a, xmax, per_t);
                    int j = static_cast<int>(fmin(fmax(floor((budget - before) / w), 0.0), 2147483646.0));
                    if (a == xmax && j == 0) j = 1;
                    const int there = a == floor_value ? floor_ties : count_from(lo) - count_from(lo + 1);
                    last = a;
                    ties = min(j, there);
                    kept = before + ties * w;
                }
            }
        }
        // ---- of the last kept value, the first `ties` by index: those of the shares before this one first ----
        {
            const int bin = bin_of(last);   // (counted, or found by bisection: then by counting)
            int count = 0;
            if (bin >= 0 && !missed) {
                if (tid == 0) tell(&meet.equal[rank], C, hist[bin]);
            } else {
                each([&](const auto& y, auto c, int) {
#pragma unroll
                    for (int e = 0; e < c(); ++e) count += y[e] == last ? 1 : 0;
                });
                count = __reduce_add_sync(0xffffffffu, count);
                __syncthreads();
                if (lane == 0) s_i[warp] = count;
                __syncthreads();
                if (tid == 0) {
                    count = 0;
                    for (int w = 0; w < kWarps; ++w) count += s_i[w];
                    tell(&meet.equal[rank], C, count);
                }
            }
            meet_all();   // (nothing remote is touched behind this)
        }
        int before = 0;
        for (int r = 0; r < rank; ++r) before += meet.equal[r];
        const int room = max(ties - before, 0);
        if (room > 0 && room < meet.equal[rank]) {
            // Some of this share's do not fit: the first that does not.  By blocks of as many entries as there are bits where the counters
            // were.
            constexpr int kBlock = kBins * 32;
            int passed = 0;   // equal entries of the blocks before
            for (int base = 0; base < n; base += kBlock) {
                const int words = min(kBins, (n - base + 31) / 32), mine_words = (words + kThreads - 1) / kThreads;
                __syncthreads();
                for (int i = tid; i < words; i += kThreads) hist[i] = 0;
                __syncthreads();
                each_from(last, [&](const auto& y, auto c, int at) {
#pragma unroll
                    for (int e = 0; e < c(); ++e)
                        if (y[e] == last && at + e >= base && at + e - base < kBlock)
                            atomicOr(&hist[(at + e - base) >> 5], 1 << ((at + e - base) & 31));
                }, [](int) {});
                __syncthreads();
                int mine = 0;
                for (int i = tid * mine_words; i < min((tid + 1) * mine_words, words); ++i) mine += __popc(hist[i]);
                int to = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int c = __shfl_up_sync(0xffffffffu, to, o);
                    if (lane >= o) to += c;
                }
                if (lane == 31) s_i[warp] = to;
                __syncthreads();
                int total = 0;
                for (int w = 0; w < kWarps; ++w) {
                    if (w < warp) to += s_i[w];
                    total += s_i[w];
                }
                int from = passed + to - mine;
                if (from <= room && room < passed + to)
                    for (int i = tid * mine_words; i < min((tid + 1) * mine_words, words); ++i) {
                        const int here = __popc(hist[i]);
                        if (from <= room && room < from + here) s_cut = base + i * 32 + __fns(hist[i], 0, room - from + 1);
                        from += here;
                    }
                passed += total;
            }
            __syncthreads();
        }
        const int cut = room > 0 ? s_cut : 0;
        finish(kept, last, [&](float a, int place) { return a > last || (a == last && place < cut); });
    }
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_sampling_probs(float* out, const void* logits, int64_t ld, int rows, int vocab, const float* temperatures,
                        const int32_t* top_k, const float* top_p, b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(rows >= 0 && vocab > 0 && ld >= vocab, "sampling_probs: bad shape");
    if (vocab > kMaxVocab) {
        set_last_error("sampling_probs: vocab %d is above %d", vocab, kMaxVocab);
        return B200_ERR_UNSUPPORTED;
    }
    B200_CHECK_ARG(rows <= (1 << 27), "sampling_probs: too many rows");
    if (rows == 0) return B200_OK;
    B200_CHECK_ARG(out && logits && temperatures, "sampling_probs: NULL tensor");
    const bool filters = top_k != nullptr || top_p != nullptr;
    const bool aligned = (reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) % 16 == 0 && ld % 8 == 0 && vocab % 4 == 0;
    // CTAs per row: one, and more while that makes no more than 16 for an SM, three rounds of them, so that the SMs stay full to the end
    // (320 rows of 151936, filters mixed: up to 4 for an SM 164 us, 8: 130, 16: 109, 36: 133; 512 rows without filters 98, 92, 85, 96),
    // and while shares are large enough to pay for the CTAs' meetings: 64 entries a thread, or 32 where no row lists its largest (8 rows
    // of 32000: 8.3 us at 64 and 6.3 at 32 without filters, 28.7 and 24.6 with top_p, but 14.4 and 16.5 for 64 rows with top_k 40).
    int cluster = 1;
    const int least = kThreads * (top_k != nullptr ? 64 : 32);
    while (cluster < kMaxCluster && static_cast<int64_t>(rows) * cluster * 2 <= kMostPerSm * sm_count() && vocab / cluster > least) cluster *= 2;
    ProbsParams p = {out, static_cast<const __nv_bfloat16*>(logits), ld, rows, vocab, div_ceil(div_ceil(vocab, cluster), 8) * 8, cluster,
                     temperatures, top_k, top_p};
    auto kernel = filters ? (aligned ? sampling_probs_kernel<true, true> : sampling_probs_kernel<true, false>)
                          : (aligned ? sampling_probs_kernel<false, true> : sampling_probs_kernel<false, false>);
    B200_CHECK_CUDA(launch_kernel(kernel, dim3(static_cast<unsigned>(rows) * cluster), dim3(kThreads), 0, static_cast<cudaStream_t>(stream),
                                  dim3(cluster, 1, 1), p));
    return B200_OK;
}

}  // extern "C"
