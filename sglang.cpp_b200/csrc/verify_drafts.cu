// Which drafted tokens the target's probabilities accept, and the token that follows them (speculative sampling).
//
// A request with drafts x_1 .. x_n, drawn from q_1 .. q_n, has target rows p_0 .. p_n (p_i: what follows the first i drafts).
// Draft i stands if those before it do and u_i q_i(x_i) < p_{i-1}(x_i), with u_i uniform in [0, 1): probability min(1, p / q).
// The token behind the a accepted ones is drawn from max(p_a - q_{a+1}, 0), or from p_n where all stand; together that is a draw
// from the target's own distribution.  The draw is the inverse of the summed probabilities in index order: the first index whose
// running sum exceeds u * (sum of all).
//
// Drafts are tested in fp64, where a product of two fp32 numbers is exact.  A row's sum is right to 1e-13 or so (fp64, but for what the
// rounding of sixteen differences left out, which is added up in fp32: 2^-45 of them), so that a border is missed by no more
// than that.  Sums are formed in a fixed order: equal calls, equal tokens.
//
// Bound by HBM: one row of p, and one of q where a draft was refused, 8 bytes per vocabulary entry and request, read once; the
// other rows are looked at in one place each.  A cluster of CTAs shares a row: every warp sums a run of consecutive entries in
// rounds of 512 (their loads before their sums), the CTAs exchange their sums, and the warp in whose run the target lies finds
// the round by the sums that its lanes kept and reads that round once more.  64 requests of up to five drafts, 151936 entries (55 MB):
// 18.5 us from L2, 24.6 from memory, of which 6 are the launch and the three trips to the drafts' probabilities, 10 to 12 the row's
// sums, 4 the exchange and the entry.  (All sums first and a stretch of neighbours per lane for the entry: 31.7.)
#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kMaxThreads = 1024, kMaxPerSm = 4;   // an SM's threads are shared by one, two or four CTAs
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kEach = 16;            // entries of a lane in a round
constexpr int kRound = 32 * kEach;

struct VerifyParams {
    int32_t *tokens, *accepted;
    const float *target, *draft;
    int64_t target_ld, draft_ld;
    const int32_t *draft_tokens, *draft_indptr;
    const float *accept, *draw;
    int batch, total, most, vocab, cluster;
    int* status;
};

// What an entry counts for: nothing unless it is a positive number.
__device__ __forceinline__ float entry(float p) { return fminf(fmaxf(p, 0.f), 3.402823466e38f); }   // (a NaN is 0: the other of the two)
__device__ __forceinline__ float unit_interval(float u) { return u > 0.f ? fminf(u, 0.99999994f) : 0.f; }

__global__ void __launch_bounds__(kMaxThreads)
verify_drafts_kernel(const VerifyParams p) {
    __shared__ double s_sum[kMaxWarps], s_cta[kMaxCluster];
    __shared__ int s_accepted;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int C = p.cluster, rank = static_cast<int>(blockIdx.x) % C, b = static_cast<int>(blockIdx.x) / C;
    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // (waited for ahead of the first remote store)
    pdl_launch_dependents();
    pdl_wait_prior();

    const int start = min(max(p.draft_indptr[b], 0), p.total);
    const int n = min(min(max(p.draft_indptr[b + 1], start), p.total) - start, p.most);
    const float* target = p.target + static_cast<int64_t>(start + b) * p.target_ld;   // the request's first row
    // ---- the drafts, 32 at a time ----
    if (warp == 0) {
        int a = 0;
        for (int base = 0; base < n; base += 32) {
            const int j = base + lane;
            bool refused = false;
            if (j < n) {
                const int x = p.draft_tokens[start + j];
                const bool known = x >= 0 && x < p.vocab;
                if (!known && rank == 0) atomicExch(&p.status[kStatusBadIndex], bad_index_word(x));
                const double px = known ? entry(target[j * p.target_ld + x]) : 0.0;
                const double qx = p.draft == nullptr ? 1.0 : known ? entry(p.draft[(start + j) * p.draft_ld + x]) : 0.0;
                refused = !(unit_interval(p.accept[start + j]) * qx < px);
            }
            const uint32_t first = __ballot_sync(0xffffffffu, refused);
            a = first != 0 ? base + __ffs(first) - 1 : min(base + 32, n);
            if (first != 0) break;
        }
        if (lane == 0) s_accepted = a;
    }
    __syncthreads();
    const int a = s_accepted;
    if (rank == 0)
        for (int j = threadIdx.x; j <= p.most; j += blockDim.x)
            if (j != a) p.tokens[static_cast<int64_t>(b) * (p.most + 1) + j] = j < a ? p.draft_tokens[start + j] : -1;
    if (rank == 0 && threadIdx.x == 0) p.accepted[b] = a;

    // ---- the row to draw from: this warp's run of it ----
    const float* prow = target + a * p.target_ld;
    const bool refused = a < n;
    const float* qrow = refused && p.draft != nullptr ? p.draft + (start + a) * p.draft_ld : nullptr;
    const int without = refused && p.draft == nullptr ? p.draft_tokens[start + a] : -1;   // a draft that was certain
    const int run = (p.vocab + C * warps * kRound - 1) / (C * warps * kRound) * kRound;
    const int first = static_cast<int>(min(static_cast<int64_t>(rank * warps + warp) * run, static_cast<int64_t>(p.vocab)));
    const int last = first + min(run, p.vocab - first);
    const int per = (run / kRound + 31) / 32, part = per * kRound;   // a part: rounds, entries whose sum one lane keeps
    bool rest = refused;   // p - q; or p, where no entry of p exceeds q
    auto weigh = [&](float x, float y, int i) -> double {
        const float px = entry(x);
        if (!rest) return px;
        if (qrow == nullptr) return i == without ? fmaxf(px - 1.f, 0.f) : px;
        return fmax(static_cast<double>(px) - static_cast<double>(entry(y)), 0.0);
    };
    // Sums of a lane's entries of a round.  p - q is taken as the rounded fp32 difference and what its rounding left out (an fp32
    // number too, as p >= q >= 0), and the small parts are summed in fp32: sixteen of them are off by 2^-20 of theirs, 2^-45 of
    // the difference, and a conversion to fp64 per entry is saved (they run at a quarter of fp64's rate).
    auto difference = [&](const float (&x)[kEach], const float (&y)[kEach]) {
        double sum = 0.0;
        float small = 0.f;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const float px = entry(x[k]), qx = entry(y[k]), d = px - qx;
            if (d > 0.f) small += (px - d) - qx;
            sum += fmaxf(d, 0.f);
        }
        return sum + small;
    };
    auto plain = [&](const float (&x)[kEach], int base, bool aligned) {   // p, less the draft that was certain
        double sum = 0.0;
        const int skip = rest && without >= base && without < base + kRound ? without - base : -1;
        const int at = aligned ? skip / 128 * 4 + skip % 4 : skip / 32, of = aligned ? skip % 128 / 4 : skip % 32;
        const bool here = skip >= 0 && lane == of;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const float px = entry(x[k]);
            sum += here && k == at ? fmaxf(px - 1.f, 0.f) : px;
        }
        return sum;
    };
    // Sum of this warp's run, the same in every lane; kept: lane c's, of the run's c-th part.
    double kept = 0.0;
    auto sum_run = [&]() {
        const bool both = rest && qrow != nullptr;
        const bool aligned = ((reinterpret_cast<uintptr_t>(prow) | (both ? reinterpret_cast<uintptr_t>(qrow) : 0) | (p.vocab & 3)) & 15) == 0;
        auto fetch = [&](float (&x)[kEach], const float* row, int round) {
            const int base = first + round * kRound;
            if (aligned) {
#pragma unroll
                for (int k = 0; k < kEach / 4; ++k) {
                    const int i = base + k * 128 + lane * 4;
                    reinterpret_cast<float4*>(x)[k] = i < last ? __ldg(reinterpret_cast<const float4*>(row + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            } else {
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    const int i = base + k * 32 + lane;
                    x[k] = i < last ? __ldg(row + i) : 0.f;
                }
            }
        };
        double all = 0.0, sum = 0.0;
        kept = 0.0;
        const int rounds = (last - first + kRound - 1) / kRound;
        auto add = [&](double w, int round) {
            sum += w;
            if ((round + 1) % per != 0 && round + 1 < rounds) return;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == round / per) kept = sum;
            all += sum;
            sum = 0.0;
        };
        for (int r = 0; r < rounds; ++r) {
            float x[kEach], y[kEach];
            fetch(x, prow, r);
            if (both) fetch(y, qrow, r);
            add(both ? difference(x, y) : plain(x, first + r * kRound, aligned), r);
        }
        return all;
    };
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    double total = 0.0, before = 0.0, upto_end = 0.0;   // of the row, of the runs before this warp's, with this one
    for (int pass = 0; pass < 2; ++pass) {
        const double sum = sum_run();
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        double cta = 0.0, ahead = 0.0, with = 0.0;
        for (int w = 0; w < warps; ++w) {
            if (w == warp) ahead = cta;
            cta += s_sum[w];
            if (w == warp) with = cta;
        }
        if (C > 1) {
            if (threadIdx.x < static_cast<unsigned>(C)) {
                uint32_t at;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&s_cta[rank])), "r"(threadIdx.x));
                asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(cta) : "memory");
            }
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else {
            if (threadIdx.x == 0) s_cta[0] = cta;
            __syncthreads();
        }
        total = 0.0;
        for (int r = 0; r < C; ++r) {
            // (One run's end is the next one's beginning to the last bit, so that exactly one of them holds the goal.)
            if (r == rank) before = total + ahead, upto_end = total + with;
            total += s_cta[r];
        }
        if (total > 0.0 || !rest) break;   // (the same in every CTA of the cluster)
        rest = false;
        if (C > 1) {   // everyone has read the sums before the next ones arrive
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else {
            __syncthreads();
        }
    }
    int32_t* out = p.tokens + static_cast<int64_t>(b) * (p.most + 1) + a;
    if (!(total > 0.0)) {
        if (rank == 0 && threadIdx.x == 0) *out = 0;   // a row without a positive number
        return;
    }
    const double goal = unit_interval(p.draw[b]) * total;
    if (goal < before || goal >= upto_end) return;
    // The part of the run, by the sums that the lanes kept; then that part once more, neighbouring entries in a lane.  (The sums
    // are formed in another order than before: the last bits may put the goal behind the part's last entry.)
    auto scan = [&](double w) {   // sums up to and with each lane's
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double t = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += t;
        }
        return w;
    };
    auto choose = [&](double own, double ahead, double& upto) {   // the first lane whose sum passes the goal, or -1
        upto = scan(own);
        return __ffs(__ballot_sync(0xffffffffu, own > 0.0 && ahead + upto > goal)) - 1;
    };
    double upto;
    int chosen = choose(kept, before, upto);
    if (chosen < 0) chosen = 31 - __clz(__ballot_sync(0xffffffffu, kept > 0.0));
    double ahead = before + __shfl_sync(0xffffffffu, upto, chosen) - __shfl_sync(0xffffffffu, kept, chosen);
    const int from = first + chosen * part, to = min(from + part, last);
    int pick = -1;   // the last positive entry so far, until one passes the goal
    for (int base = from; base < to; base += kRound) {
        double w[kEach], own = 0.0;
        const int at = base + lane * kEach;
        float x[kEach], y[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            x[k] = at + k < to ? __ldg(prow + at + k) : 0.f;
            y[k] = rest && qrow != nullptr && at + k < to ? __ldg(qrow + at + k) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < kEach; ++k) own += w[k] = weigh(x[k], y[k], at + k);
        const int hit = choose(own, ahead, upto);
        const uint32_t positive = __ballot_sync(0xffffffffu, own > 0.0);
        const int who = hit >= 0 ? hit : 31 - __clz(positive);
        if (who >= 0) {
            double sum = ahead + upto - own;
            int mine = -1;
            bool passed = false;
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                sum += w[k];
                if (w[k] > 0.0 && !passed) mine = at + k, passed = hit >= 0 && sum > goal;
            }
            pick = __shfl_sync(0xffffffffu, mine, who);
        }
        if (hit >= 0) break;
        ahead += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) *out = pick;
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_verify_drafts(int32_t* tokens, int32_t* accepted, const float* target_probs, int64_t target_ld, const float* draft_probs,
                       int64_t draft_ld, const int32_t* draft_tokens, const int32_t* draft_indptr, const float* accept_uniform,
                       const float* draw_uniform, int batch, int total_drafts, int max_drafts, int vocab, b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(batch >= 0 && total_drafts >= 0 && max_drafts >= 0 && vocab > 0, "verify_drafts: bad shape");
    B200_CHECK_ARG(batch <= (1 << 24) && vocab <= (1 << 30) && max_drafts <= (1 << 20), "verify_drafts: too large");
    B200_CHECK_ARG(target_ld >= vocab && (draft_probs == nullptr || draft_ld >= vocab), "verify_drafts: row stride below vocab");
    if (batch == 0) return B200_OK;
    B200_CHECK_ARG(tokens && accepted && target_probs && draft_indptr && draw_uniform, "verify_drafts: NULL tensor");
    B200_CHECK_ARG(total_drafts == 0 || (draft_tokens && accept_uniform), "verify_drafts: NULL tensor");
    int err = B200_OK;
    int* status = device_status_words(&err);
    if (err != B200_OK) return err;
    // CTAs per row: enough to fill the device, and no fewer than 4096 entries each (1024 or 16384 make no difference from 8192 entries
    // and 1 request on).  Their threads: all that an SM has room for.  (200 requests of 50001 entries: 20.5 us with up to four CTAs on an SM,
    // 22.6 with two, 26.7 with one.)
    const int64_t sms = sm_count();
    int cluster = 1, threads = kMaxThreads;
    while (cluster < kMaxCluster && static_cast<int64_t>(batch) * 2 * cluster <= kMaxPerSm * sms && vocab / (2 * cluster) >= 4096) cluster *= 2;
    while (threads > kMaxThreads / kMaxPerSm && static_cast<int64_t>(batch) * cluster * threads > sms * kMaxThreads) threads /= 2;
    VerifyParams p = {tokens,       accepted,       target_probs, draft_probs, target_ld,    draft_ld, draft_tokens, draft_indptr,
                      accept_uniform, draw_uniform, batch,        total_drafts, max_drafts, vocab,    cluster,      status};
    B200_CHECK_CUDA(launch_kernel(verify_drafts_kernel, dim3(static_cast<unsigned>(batch) * cluster), dim3(threads), 0,
                                  static_cast<cudaStream_t>(stream), dim3(cluster, 1, 1), p));
    return B200_OK;
}

}  // extern "C"
