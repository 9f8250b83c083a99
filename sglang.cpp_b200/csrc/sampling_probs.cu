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
// A cluster of CTAs owns a row and keeps it in registers: read once, written once.  The counters meet by ranges of patterns: CTA r adds
// up all CTAs' counts of the r-th range from the top, weighs them, and the sums of the ranges before decide in which thread's
// patterns the cut falls.  Bound by HBM, 6 bytes per entry; with filters also by the counting, an atomic per entry in shared
// memory.  CTAs of 512 threads, two on an SM, so that one's loads and stores lie under the other's meetings.
#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxVectors = 10;             // of 8 entries, per thread
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
    double sum[kMaxCluster];                 // weights: of the share (no filters), of the CTA's range of patterns
    int count[kMaxCluster];                  // entries in that range
    int out_count[kMaxCluster][kClasses];
    double out_sum[kMaxCluster][kClasses];
    int equal[kMaxCluster];                  // entries of the share that equal the last kept value
    int turn_count[2][kMaxCluster];          // bisection, in turns
    double turn_sum[2][kMaxCluster];
    float value[2];                          // last kept value after top_k, after top_p ...
    int ties[2];                             // ... how many of it are kept ...
    double kept[2];                          // ... and the sum of the kept
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

// A logit: a NaN as -inf, one kind of zero.
__device__ __forceinline__ float clean(float x) { return fmaxf(x + 0.f, -INFINITY); }

// VECTORS: of 8 entries per thread.  ALIGNED: rows of both sides are read and written 16 bytes at a time; else entry by entry, neighbours
// by neighbouring threads.
template <int VECTORS, bool FILTERS, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, VECTORS <= 5 ? 2 : 1)
sampling_probs_kernel(const ProbsParams p) {
    constexpr int N = VECTORS * 8;
    __shared__ __align__(16) int hist[FILTERS ? kBins : 4];
    __shared__ Meet meet;
    __shared__ double s_d[kWarps];
    __shared__ int s_i[kWarps], s_cut;
    __shared__ int s_count[kClasses];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = p.cluster, rank = static_cast<int>(blockIdx.x) % C, row = static_cast<int>(blockIdx.x) / C;
    const int begin = min(rank * p.slice, p.vocab), n = min(p.slice, p.vocab - begin);
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (waited for ahead of the first remote store)
    pdl_launch_dependents();
    pdl_wait_prior();
    const __nv_bfloat16* x = p.logits + static_cast<int64_t>(row) * p.ld + begin;
    float* out = p.out + static_cast<int64_t>(row) * p.vocab + begin;
    // Entry e of this thread's vector j is entry ... of the share.
    auto place = [&](int i) { return ALIGNED ? ((i >> 3) * kThreads + tid) * 8 + (i & 7) : i * kThreads + tid; };

    // ---- the share, in registers, two entries to one; what lies behind the row as -inf ----
    uint32_t raw[N / 2];
    if (ALIGNED) {
#pragma unroll
        for (int j = 0; j < VECTORS; ++j) {
            const int at = (j * kThreads + tid) * 8;
            uint4 a = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
            if (at + 8 <= n) a = __ldg(reinterpret_cast<const uint4*>(x + at));
            raw[j * 4] = a.x, raw[j * 4 + 1] = a.y, raw[j * 4 + 2] = a.z, raw[j * 4 + 3] = a.w;
        }
#pragma unroll
        for (int j = 0; j < VECTORS; ++j) {
            const int at = (j * kThreads + tid) * 8;
            if (at < n && at + 8 > n) {   // the row's last entries
                for (int e = 0; e < n - at; ++e) {
                    const uint32_t bits = __bfloat16_as_ushort(x[at + e]);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k == e >> 1) raw[j * 4 + k] = (e & 1) ? (raw[j * 4 + k] & 0xffffu) | bits << 16 : (raw[j * 4 + k] & 0xffff0000u) | bits;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint32_t lo = place(i) < n ? __bfloat16_as_ushort(x[place(i)]) : 0xff80u;
            const uint32_t hi = place(i + 1) < n ? __bfloat16_as_ushort(x[place(i + 1)]) : 0xff80u;
            raw[i >> 1] = hi << 16 | lo;
        }
    }
    auto entry = [&](int i) { return clean((i & 1) ? bf16_hi(raw[i >> 1]) : bf16_lo(raw[i >> 1])); };
    const float T = p.temperatures[row];
    const bool greedy = !(T > 1.0000001e-6f);
    int K = FILTERS && p.top_k != nullptr ? p.top_k[row] : 0;
    if (K < 1 || K > p.vocab) K = p.vocab;
    const float P = FILTERS && p.top_p != nullptr ? p.top_p[row] : 1.f;
    const bool want_k = K < p.vocab, want_p = P < 1.f;
    const bool filter = FILTERS && !greedy && (want_k || want_p);
    if (FILTERS && filter) {
        for (int i = tid; i < kBins / 4; i += kThreads) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
        if (tid < kClasses) s_count[tid] = 0;
        __syncthreads();
    }
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, entry(i));
    bool outside = false;
    if (FILTERS && filter) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int bin = bin_of(entry(i));
            if (bin >= 0) atomicAdd(&hist[bin], 1);
            else if (place(i) < n) outside = true;
        }
    }
    top = warp_max(top);
    if (lane == 0) s_d[warp] = top;
    if (tid == 0) {
        meet.value[0] = meet.value[1] = -INFINITY;
        meet.ties[0] = meet.ties[1] = 0x7fffffff;
        s_cut = 0x7fffffff;
    }
    outside = __syncthreads_or(outside);
    top = -INFINITY;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, static_cast<float>(s_d[w]));
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0) tell(&meet.top[rank], C, top);
    meet_all();   // also: everyone's counters are complete
    float xmax = -INFINITY;
    for (int r = 0; r < C; ++r) xmax = fmaxf(xmax, meet.top[r]);

    auto store = [&](auto value) {   // value(i) to entry i
        if (ALIGNED) {
#pragma unroll
            for (int j = 0; j < VECTORS; ++j) {
                const int at = (j * kThreads + tid) * 8;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = value(j * 8 + e);
                if (at + 8 <= n) {
                    reinterpret_cast<float4*>(out + at)[0] = make_float4(y[0], y[1], y[2], y[3]);
                    reinterpret_cast<float4*>(out + at)[1] = make_float4(y[4], y[5], y[6], y[7]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (at + e < n) out[at + e] = y[e];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (place(i) < n) out[place(i)] = value(i);
        }
    };

    if (greedy) {   // one-hot at the first maximum of all shares
        int at = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (entry(i) == xmax) at = min(at, begin + place(i));
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) s_i[warp] = at;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) at = min(at, s_i[w]);
        if (tid == 0) tell(&meet.first[rank], C, at);
        meet_all();
        int first = 0x7fffffff;
        for (int r = 0; r < C; ++r) first = min(first, meet.first[r]);
        store([&](int i) { return begin + place(i) == first ? 1.f : 0.f; });
        return;
    }
    if (xmax == -INFINITY) {   // nothing but -inf and NaN
        store([](int) { return 0.f; });
        return;
    }

    // Weights.  fp64 for the sums that decide; for the entries fp32, with what the exponent (x - max) log2(e) / T loses when it is
    // rounded put back as a factor 2^lost = 1 + lost ln 2, so that a far tail keeps its digits.
    const double per_t = 1.4426950408889634 / static_cast<double>(T);
    const float s_hi = static_cast<float>(per_t), s_lo = static_cast<float>(per_t - static_cast<double>(s_hi));
    const bool plain = xmax < INFINITY && s_hi > 1e-30f && s_hi < 1e30f;   // no infinities but -inf, whose exponent is -inf
    auto weight = [&](float a) -> float {
        const float d = a - xmax, hi = d * s_hi;
        float y;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(hi));
        const float lost = fmaf(d, s_lo, fmaf(d, s_hi, -hi));
        if (plain) return hi < -126.f ? 0.f : fmaf(y, lost * 0.693147182f, y);
        return static_cast<float>(weight64(a, xmax, per_t));
    };

    if (!filter) {
        float w[N];   // (where there are filters too, registers are short: weights are formed a second time)
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                w[i + e] = weight(entry(i + e));
                part += w[i + e];
            }
            sum += part;
        }
        sum = warp_sum(sum);
        if (lane == 0) s_d[warp] = sum;
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < kWarps; ++w) sum += s_d[w];
        if (tid == 0) tell(&meet.sum[rank], C, sum);
        meet_all();
        sum = 0.0;
        for (int r = 0; r < C; ++r) sum += meet.sum[r];
        const float inv = static_cast<float>(1.0 / sum);
        if (FILTERS) store([&](int i) { return weight(entry(i)) * inv; });
        else store([&](int i) { return w[i] * inv; });
        return;
    }
    if constexpr (FILTERS) {
        // ---- entries that are not counted ----
        double out_sum[kClasses] = {0.0, 0.0, 0.0};
        if (outside) {
#pragma unroll 1
            for (int c = 0; c < kClasses; ++c) {
                double sum = 0.0;
                int count = 0;
                for (int i = tid; i < n; i += kThreads) {
                    const float a = clean(__bfloat162float(x[i]));
                    if (bin_of(a) >= 0 || c != (a >= 256.f ? 0 : a <= -256.f ? 2 : 1)) continue;
                    sum += weight64(a, xmax, per_t);
                    ++count;
                }
                sum = warp_sum(sum);
                count = __reduce_add_sync(0xffffffffu, count);
                if (lane == 0) {
                    s_d[warp] = sum;
                    atomicAdd(&s_count[c], count);
                }
                __syncthreads();
                for (int w = 0; w < kWarps; ++w) out_sum[c] += s_d[w];
                __syncthreads();
            }
        }
        if (tid < kClasses) {
            tell(&meet.out_count[rank][tid], C, outside ? s_count[tid] : 0);
            tell(&meet.out_sum[rank][tid], C, tid == 0 ? out_sum[0] : tid == 1 ? out_sum[1] : out_sum[2]);
        }
        // ---- this CTA's range of patterns, a run of them per thread, from the top down ----
        const int each = kBins / C / kThreads;   // 2 .. 16
        const int bin_top = kBins - 1 - (rank * kThreads + tid) * each;
        int my_count = 0;
        double my_sum = 0.0;
        auto count_of = [&](int bin) {
            int c[kMaxCluster], sum = 0;
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) {
                c[r] = 0;
                if (r < C) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(c[r]) : "r"(remote(&hist[bin], r)));
            }
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) sum += c[r];
            return sum;
        };
#pragma unroll 1
        for (int i = 0; i < each; ++i) {
            const int c = count_of(bin_top - i);
            if (c == 0) continue;
            my_count += c;
            my_sum += c * weight64(value_of_bin(bin_top - i), xmax, per_t);
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
#pragma unroll 1
                for (int i = 0; i < each; ++i) {
                    const int c = count_of(bin_top - i);
                    if (c == 0) continue;
                    const float a = value_of_bin(bin_top - i);
                    const double w = weight64(a, xmax, per_t);
                    if (K <= c_run + c) {
                        tell(&meet.value[0], C, a);
                        tell(&meet.ties[0], C, K - c_run);
                        tell(&meet.kept[0], C, s_run + (K - c_run) * w);
                        break;
                    }
                    c_run += c;
                    s_run += c * w;
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
#pragma unroll 1
                for (int i = 0; i < each; ++i) {
                    const float a = value_of_bin(bin_top - i);
                    int c = count_of(bin_top - i);
                    if (a < last) break;
                    if (c == 0) continue;
                    if (a == last) c = min(c, ties);
                    const double w = weight64(a, xmax, per_t);
                    if (s_run + c * w > budget) {
                        const double fit = fmin(fmax(floor((budget - s_run) / w), 0.0), static_cast<double>(c));
                        int j = static_cast<int>(fit);
                        if (c_run == 0 && j == 0) j = 1;
                        tell(&meet.value[1], C, a);
                        tell(&meet.ties[1], C, j);
                        tell(&meet.kept[1], C, s_run + j * w);
                        break;
                    }
                    c_run += c;
                    s_run += c * w;
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
            int count = 0;
#pragma unroll
            for (int i = 0; i < N; ++i) count += place(i) < n && entry(i) == last ? 1 : 0;
            count = __reduce_add_sync(0xffffffffu, count);
            __syncthreads();
            if (lane == 0) s_i[warp] = count;
            __syncthreads();
            if (tid == 0) {
                count = 0;
                for (int w = 0; w < kWarps; ++w) count += s_i[w];
                tell(&meet.equal[rank], C, count);
            }
            meet_all();   // (nothing remote is touched behind this)
        }
        int before = 0;
        for (int r = 0; r < rank; ++r) before += meet.equal[r];
        const int room = max(ties - before, 0);
        if (room < meet.equal[rank]) {
            // Some of this share's do not fit.  A bit per entry, where the counters were: the first that does not.
            constexpr int kWords = (N * kThreads + 31) / 32, kEach = (kWords + kThreads - 1) / kThreads;
            static_assert(kWords <= kBins, "");
            for (int i = tid; i < kWords; i += kThreads) hist[i] = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (place(i) < n && entry(i) == last) atomicOr(&hist[place(i) >> 5], 1 << (place(i) & 31));
            __syncthreads();
            int mine = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (tid * kEach + i < kWords) mine += __popc(hist[tid * kEach + i]);
            int to = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int c = __shfl_up_sync(0xffffffffu, to, o);
                if (lane >= o) to += c;
            }
            if (lane == 31) s_i[warp] = to;
            __syncthreads();
            for (int w = 0; w < warp; ++w) to += s_i[w];
            int from = to - mine;
            if (from <= room && room < to)
                for (int i = 0; i < kEach; ++i) {
                    const int word = hist[tid * kEach + i], here = __popc(word);
                    if (from <= room && room < from + here) s_cut = (tid * kEach + i) * 32 + __fns(word, 0, room - from + 1);
                    from += here;
                }
            __syncthreads();
        }
        const int cut = s_cut;
        const float inv = static_cast<float>(1.0 / kept);
        store([&](int i) {
            const float a = entry(i);
            return a > last || (a == last && place(i) < cut) ? weight(a) * inv : 0.f;
        });
    }
}

template <int VECTORS>
auto kernel_for(bool filters, bool aligned) {
    return filters ? (aligned ? sampling_probs_kernel<VECTORS, true, true> : sampling_probs_kernel<VECTORS, true, false>)
                   : (aligned ? sampling_probs_kernel<VECTORS, false, true> : sampling_probs_kernel<VECTORS, false, false>);
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_sampling_probs(float* out, const void* logits, int64_t ld, int rows, int vocab, const float* temperatures,
                        const int32_t* top_k, const float* top_p, b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(rows >= 0 && vocab > 0 && ld >= vocab, "sampling_probs: bad shape");
    constexpr int most = kMaxCluster * kThreads * kMaxVectors * 8;
    if (vocab > most) {
        set_last_error("sampling_probs: vocab %d is above %d", vocab, most);
        return B200_ERR_UNSUPPORTED;
    }
    B200_CHECK_ARG(rows <= (1 << 27), "sampling_probs: too many rows");
    if (rows == 0) return B200_OK;
    B200_CHECK_ARG(out && logits && temperatures, "sampling_probs: NULL tensor");
    const bool filters = top_k != nullptr || top_p != nullptr;
    const bool aligned = (reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) % 16 == 0 && ld % 8 == 0 && vocab % 4 == 0;
    // CTAs per row: as few as hold it at five vectors a thread, and more while rows are few and shares large.
    int cluster = 1;
    while (cluster < kMaxCluster && vocab > cluster * kThreads * 5 * 8) cluster *= 2;
    while (cluster < kMaxCluster && static_cast<int64_t>(rows) * cluster * 2 <= 2 * sm_count() && vocab / cluster > kThreads * 8) cluster *= 2;
    const int vectors = div_ceil(vocab, cluster * kThreads * 8);
    ProbsParams p = {out, static_cast<const __nv_bfloat16*>(logits), ld, rows, vocab, div_ceil(div_ceil(vocab, cluster), 8) * 8, cluster,
                     temperatures, top_k, top_p};
    auto kernel = vectors <= 1 ? kernel_for<1>(filters, aligned) : vectors <= 2 ? kernel_for<2>(filters, aligned)
                : vectors <= 3 ? kernel_for<3>(filters, aligned) : vectors <= 4 ? kernel_for<4>(filters, aligned)
                : vectors <= 5 ? kernel_for<5>(filters, aligned) : kernel_for<kMaxVectors>(filters, aligned);
    B200_CHECK_CUDA(launch_kernel(kernel, dim3(static_cast<unsigned>(rows) * cluster), dim3(kThreads), 0, static_cast<cudaStream_t>(stream),
                                  dim3(cluster, 1, 1), p));
    return B200_OK;
}

}  // extern "C"
