// The probabilities that a row of logits is sampled with: temperature, then the top_k largest, then the top_p of those.
//
//     w_i = exp((x_i - max x) / T),   p_i = w_i / (sum of the kept w) for kept i, 0 elsewhere
// Kept are the top_k largest (equal ones by index) and of those, in descending order, the entries whose running sum, their own
// weight included, stays within top_p times the sum of all top_k (never without the first).  T at most 1e-6: one-hot at the first
// maximum.
//
// A logit is one of 65536 bf16 patterns, and its weight is a function of the pattern: where a row is cut follows from the COUNTS of
// the patterns and one fp64 weight for each that occurs, which puts the borders where 64-bit sums do (fp32 weights summed entry
// by entry are off by 1e-7 of the sum, more than many an entry's weight).
//
// A cluster of CTAs owns a row; each keeps its share of the entries in shared memory (read once from HBM) and counts them at full
// resolution, two 16-bit counters to a word.  The counters meet by ranges of patterns: CTA r adds up all CTAs' counts of the
// r-th range from the top, weighs them, and the sums of the ranges before decide in which thread's patterns the cut falls.
// Bound by HBM (6 bytes per entry) without filters, by the counting (an atomic per entry in shared memory) with them.
#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 40960;      // entries per CTA: their counters of 16 bits cannot overflow
constexpr int kKeys = 65536;
constexpr uint32_t kLowest = 0x007fu; // the key of -inf

struct ProbsParams {
    float* out;
    const __nv_bfloat16* logits;
    int64_t ld;
    int rows, vocab, slice, cluster;
    const float* temperatures;
    const int32_t* top_k;
    const float* top_p;
};

// Keys order like the values: both zeros have one, a NaN counts as -inf.
__device__ __forceinline__ uint32_t key_of(uint32_t bits) {
    if ((bits & 0x7fffu) > 0x7f80u) return kLowest;
    if (bits == 0x8000u) bits = 0u;
    return (bits & 0x8000u) ? (~bits & 0xffffu) : (bits | 0x8000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    const uint32_t bits = (key & 0x8000u) ? (key & 0x7fffu) : (~key & 0xffffu);
    return __uint_as_float(bits << 16);
}

struct Meet {              // each CTA's copy: what the CTAs of a row tell one another
    uint32_t top[kMaxCluster];       // largest key of a CTA's share
    int first[kMaxCluster];          // where it is first
    double sum[kMaxCluster];         // weights: of the CTA's share (no filters) or of its range of keys
    uint32_t count[kMaxCluster];     // entries in its range of keys
    uint32_t equal[kMaxCluster];     // entries of its share at the last kept key
    double kept[2];                  // sum of the top_k, of the kept
    uint32_t key[2];                 // last kept key after top_k, after top_p ...
    uint32_t ties[2];                // ... and how many of it are kept
};

__device__ __forceinline__ uint32_t remote(const void* p, int r) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(r));
    return a;
}
__device__ __forceinline__ void tell(const uint32_t* p, int ctas, uint32_t v) {
    for (int r = 0; r < ctas; ++r) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, r)), "r"(v) : "memory");
}
__device__ __forceinline__ void tell(const double* p, int ctas, double v) {
    for (int r = 0; r < ctas; ++r) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote(p, r)), "d"(v) : "memory");
}
__device__ __forceinline__ void meet_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <bool FILTERS>
__global__ void __launch_bounds__(kThreads)
sampling_probs_kernel(const ProbsParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t* hist = reinterpret_cast<uint32_t*>(smem);                                        // FILTERS: key k in half k & 1 of word k >> 1
    uint16_t* share = reinterpret_cast<uint16_t*>(smem + (FILTERS ? kKeys * 2 : 0));   // this CTA's logits
    __shared__ Meet meet;
    __shared__ uint32_t s_u[kWarps];
    __shared__ double s_d[kWarps];
    __shared__ int s_cut;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = p.cluster, rank = static_cast<int>(blockIdx.x) % C, row = static_cast<int>(blockIdx.x) / C;
    const int begin = min(rank * p.slice, p.vocab), n = min(p.slice, p.vocab - begin);
    if (FILTERS)
        for (int i = tid; i < kKeys / 8; i += kThreads) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (waited for ahead of the first remote store)
    pdl_launch_dependents();
    pdl_wait_prior();
    const __nv_bfloat16* x = p.logits + static_cast<int64_t>(row) * p.ld + begin;
    const float T = p.temperatures[row];
    const bool greedy = !(T > 1.0000001e-6f);
    int K = FILTERS && p.top_k != nullptr ? p.top_k[row] : 0;
    if (K < 1 || K > p.vocab) K = p.vocab;
    float P = FILTERS && p.top_p != nullptr ? p.top_p[row] : 1.f;
    const bool want_k = K < p.vocab, want_p = P < 1.f;
    const bool count = FILTERS && !greedy && (want_k || want_p);
    if (FILTERS) __syncthreads();

    // ---- the share: into shared memory, counted on the way ----
    uint32_t top = 0;
    auto take = [&](uint32_t bits) {
        const uint32_t k = key_of(bits);
        top = max(top, k);
        if (count) atomicAdd(&hist[k >> 1], (k & 1) ? 0x10000u : 1u);
    };
    if ((reinterpret_cast<uintptr_t>(x) & 15) == 0) {
        const int vecs = n >> 3;
        for (int v = tid; v < vecs; v += kThreads) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(x) + v);
            reinterpret_cast<uint4*>(share)[v] = a;
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) take((w[j >> 1] >> ((j & 1) * 16)) & 0xffffu);
        }
        for (int i = vecs * 8 + tid; i < n; i += kThreads) take(share[i] = __bfloat16_as_ushort(x[i]));
    } else {
        for (int i = tid; i < n; i += kThreads) take(share[i] = __bfloat16_as_ushort(x[i]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_u[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, s_u[lane]);
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid == 0) {
        tell(&meet.top[rank], C, top);
        meet.key[0] = meet.key[1] = 0;
        meet.ties[0] = meet.ties[1] = 0;
        s_cut = 0x7fffffff;
    }
    meet_all();   // also: everyone's counters are complete
    uint32_t best = 0;
    for (int r = 0; r < C; ++r) best = max(best, meet.top[r]);
    const float xmax = value_of(best);
    float* out = p.out + static_cast<int64_t>(row) * p.vocab + begin;

    if (greedy) {
        // one-hot at the first maximum of all shares
        int at = 0x7fffffff;
        for (int i = tid; i < n; i += kThreads)
            if (key_of(share[i]) == best) at = min(at, begin + i);
        at = __reduce_min_sync(0xffffffffu, at);
        if (lane == 0) s_u[warp] = static_cast<uint32_t>(at);
        __syncthreads();
        at = static_cast<int>(__reduce_min_sync(0xffffffffu, s_u[lane]));
        if (tid == 0) tell(reinterpret_cast<uint32_t*>(&meet.first[rank]), C, static_cast<uint32_t>(at));
        meet_all();
        int first = 0x7fffffff;
        for (int r = 0; r < C; ++r) first = min(first, meet.first[r]);
        for (int i = tid; i < n; i += kThreads) out[i] = begin + i == first ? 1.f : 0.f;
        return;
    }

    // Weights.  fp64 for the sums that decide; for the entries fp32 with the exponent (x - max) log2(e) / T in two words, so that a far
    // tail keeps its digits.
    const double per_t = 1.4426950408889634 / static_cast<double>(T);
    const float s_hi = static_cast<float>(per_t), s_lo = static_cast<float>(per_t - static_cast<double>(s_hi));
    auto weight64 = [&](uint32_t k) -> double {
        if (k == best) return 1.0;
        if (k <= kLowest) return 0.0;
        const double e = (static_cast<double>(value_of(k)) - static_cast<double>(xmax)) * per_t;
        return e < -200.0 ? 0.0 : exp2(e);
    };
    auto weight = [&](uint32_t k) -> float {
        if (k == best) return 1.f;
        if (k <= kLowest) return 0.f;
        const float d = value_of(k) - xmax, hi = d * s_hi;
        const float lo = fmaf(d, s_lo, fmaf(d, s_hi, -hi));
        const float whole = rintf(hi);
        return hi < -200.f ? 0.f : exp2f(whole) * exp2f((hi - whole) + lo);
    };
    if (best <= kLowest) {   // nothing but -inf and NaN
        for (int i = tid; i < n; i += kThreads) out[i] = 0.f;
        return;
    }

    uint32_t last_key = 0;   // kept: keys above it, and of it the entries before s_cut
    double kept;
    if (!count) {
        double sum = 0.0;
        {
            float part = 0.f;
            int taken = 0;
            for (int i = tid; i < n; i += kThreads) {
                part += weight(key_of(share[i]));
                if (++taken == 16) {
                    sum += part;
                    part = 0.f;
                    taken = 0;
                }
            }
            sum += part;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_d[warp] = sum;
        __syncthreads();
        sum = s_d[lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (tid == 0) tell(&meet.sum[rank], C, sum);
        meet_all();
        kept = 0.0;
        for (int r = 0; r < C; ++r) kept += meet.sum[r];
    } else {
        // ---- this CTA's range of keys, a run of them per thread, from the top down ----
        const int range = kKeys / C, each = range / kThreads;   // 8 .. 64 keys per thread
        const int key_top = kKeys - 1 - rank * range - tid * each;
        uint32_t my_count = 0;
        double my_sum = 0.0;
        auto count_of = [&](int k) -> uint32_t {
            uint32_t c = 0;
            for (int r = 0; r < C; ++r) {
                uint32_t w;
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(remote(&hist[k >> 1], r)));
                c += (k & 1) ? w >> 16 : w & 0xffffu;
            }
            return c;
        };
        for (int i = 0; i < each; ++i) {
            const uint32_t c = count_of(key_top - i);
            if (c == 0) continue;
            my_count += c;
            my_sum += c * weight64(static_cast<uint32_t>(key_top - i));
        }
        // Counts and sums of the threads before this one.  `lower` of a thread is `upper` of the one before it to the last bit, so
        // that exactly one thread's run holds a border.
        uint32_t incl = my_count;
        double upper = my_sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t c = __shfl_up_sync(0xffffffffu, incl, o);
            const double d = __shfl_up_sync(0xffffffffu, upper, o);
            if (lane >= o) {
                incl += c;
                upper += d;
            }
        }
        double lower = __shfl_up_sync(0xffffffffu, upper, 1);
        if (lane == 0) lower = 0.0;
        __syncthreads();
        if (lane == 31) {
            s_u[warp] = incl;
            s_d[warp] = upper;
        }
        __syncthreads();
        uint32_t warp_count = 0, cta_count = 0;
        double warp_sum = 0.0, cta_sum = 0.0;
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) {
                warp_count = cta_count;
                warp_sum = cta_sum;
            }
            cta_count += s_u[w];
            cta_sum += s_d[w];
        }
        if (tid == 0) {
            tell(&meet.count[rank], C, cta_count);
            tell(&meet.sum[rank], C, cta_sum);
        }
        meet_all();
        uint32_t above = warp_count + incl - my_count;   // entries with larger keys
        double range_sum = 0.0, all_sum = 0.0;
        for (int r = 0; r < C; ++r) {
            if (r < rank) above += meet.count[r];
            if (r == rank) range_sum = all_sum;
            all_sum += meet.sum[r];
        }
        lower = range_sum + (warp_sum + lower);
        upper = range_sum + (warp_sum + upper);
        kept = all_sum;
        uint32_t ties = 0xffffffffu;
        // ---- top_k: the thread whose run holds the K-th largest ----
        if (want_k) {
            if (above < static_cast<uint32_t>(K) && static_cast<uint32_t>(K) <= above + my_count) {
                uint32_t c_run = above;
                double s_run = lower;
                for (int i = 0; i < each; ++i) {
                    const uint32_t k = key_top - i, c = count_of(key_top - i);
                    if (c == 0) continue;
                    const double w = weight64(k);
                    if (c_run + c >= static_cast<uint32_t>(K)) {
                        tell(&meet.key[0], C, k);
                        tell(&meet.ties[0], C, K - c_run);
                        tell(&meet.kept[0], C, s_run + (K - c_run) * w);
                        break;
                    }
                    c_run += c;
                    s_run += c * w;
                }
            }
            meet_all();
            last_key = meet.key[0];
            ties = meet.ties[0];
            kept = meet.kept[0];
        }
        // ---- top_p of those ----
        if (want_p) {
            const double budget = fmax(static_cast<double>(P), 0.0) * kept;
            if (tid == 0) {   // (rounding may leave no run that exceeds the budget: then all of them stay)
                meet.key[1] = last_key;
                meet.ties[1] = ties;
                meet.kept[1] = kept;
            }
            meet_all();
            const bool holds_first = above == 0 && my_count > 0;
            if (my_count > 0 && static_cast<uint32_t>(key_top) >= last_key && (lower <= budget || holds_first) && upper > budget) {
                uint32_t c_run = above;
                double s_run = lower;
                for (int i = 0; i < each; ++i) {
                    const uint32_t k = key_top - i;
                    uint32_t c = count_of(key_top - i);
                    if (k < last_key) break;
                    if (c == 0) continue;
                    if (k == last_key) c = min(c, ties);
                    const double w = weight64(k);
                    if (s_run + c * w > budget) {
                        double fit = floor((budget - s_run) / w);
                        fit = fmin(fmax(fit, 0.0), static_cast<double>(c));
                        uint32_t j = static_cast<uint32_t>(fit);
                        if (c_run == 0 && j == 0) j = 1;
                        tell(&meet.key[1], C, k);
                        tell(&meet.ties[1], C, j);
                        tell(&meet.kept[1], C, s_run + j * w);
                        break;
                    }
                    c_run += c;
                    s_run += c * w;
                }
            }
            meet_all();
            last_key = meet.key[1];
            ties = meet.ties[1];
            kept = meet.kept[1];
        }
        // ---- of the last kept key, the first `ties` by index: those of the shares before this one first ----
        if (tid == 0) {
            const uint32_t w = hist[last_key >> 1];
            tell(&meet.equal[rank], C, (last_key & 1) ? w >> 16 : w & 0xffffu);
        }
        meet_all();   // (nothing remote is touched behind this)
        uint32_t before = 0;
        for (int r = 0; r < rank; ++r) before += meet.equal[r];
        const uint32_t room = ties > before ? ties - before : 0;
        if (room < meet.equal[rank]) {   // some of this share's do not fit: find the first that does not
            const int run = (n + kThreads - 1) / kThreads, i0 = min(tid * run, n), i1 = min(i0 + run, n);
            uint32_t mine = 0;
            for (int i = i0; i < i1; ++i) mine += key_of(share[i]) == last_key ? 1u : 0u;
            uint32_t to = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t c = __shfl_up_sync(0xffffffffu, to, o);
                if (lane >= o) to += c;
            }
            __syncthreads();
            if (lane == 31) s_u[warp] = to;
            __syncthreads();
            for (int w = 0; w < warp; ++w) to += s_u[w];
            uint32_t from = to - mine;
            if (mine > 0 && from <= room && room < to)
                for (int i = i0; i < i1; ++i)
                    if (key_of(share[i]) == last_key && from++ == room) s_cut = i;
        }
        __syncthreads();
    }
    const int cut = s_cut;
    const float inv = static_cast<float>(1.0 / kept);
    for (int i = tid; i < n; i += kThreads) {
        const uint32_t k = key_of(share[i]);
        out[i] = k > last_key || (k == last_key && i < cut) ? weight(k) * inv : 0.f;
    }
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_sampling_probs(float* out, const void* logits, int64_t ld, int rows, int vocab, const float* temperatures,
                        const int32_t* top_k, const float* top_p, b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(rows >= 0 && vocab > 0 && ld >= vocab, "sampling_probs: bad shape");
    if (vocab > kMaxCluster * kMaxSlice) {
        set_last_error("sampling_probs: vocab %d is above %d", vocab, kMaxCluster * kMaxSlice);
        return B200_ERR_UNSUPPORTED;
    }
    B200_CHECK_ARG(rows <= (1 << 27), "sampling_probs: too many rows");
    if (rows == 0) return B200_OK;
    B200_CHECK_ARG(out && logits && temperatures, "sampling_probs: NULL tensor");
    const bool filters = top_k != nullptr || top_p != nullptr;
    // CTAs per row: as many as its shares need, and more while rows are few and shares large.
    int cluster = 1;
    while (vocab > cluster * kMaxSlice) cluster *= 2;
    while (cluster < kMaxCluster && static_cast<int64_t>(rows) * cluster * 2 <= sm_count() && vocab / cluster > 8192) cluster *= 2;
    ProbsParams p = {out, static_cast<const __nv_bfloat16*>(logits), ld, rows, vocab, div_ceil(div_ceil(vocab, cluster), 8) * 8, cluster,
                     temperatures, top_k, top_p};
    const int smem = p.slice * 2 + (filters ? kKeys * 2 : 0);
    auto kernel = filters ? sampling_probs_kernel<true> : sampling_probs_kernel<false>;
    B200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    B200_CHECK_CUDA(launch_kernel(kernel, dim3(static_cast<unsigned>(rows) * cluster), dim3(kThreads), smem,
                                  static_cast<cudaStream_t>(stream), dim3(cluster, 1, 1), p));
    return B200_OK;
}

}  // extern "C"
