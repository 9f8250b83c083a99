// Causal attention over whole prompts that lie behind one another, without a cache, on the tcgen05 tensor cores.
//
// For row i of a sequence, head h and its key / value head g = h / G, G = q_heads / kv_heads:
//   s_j = scale q_i . k_j  (j <= i),  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log sum_j exp(s_j - m).
//
// An item is (sequence, KV head, block of 2 x QB query tokens), QB = 128 / G: two tiles of 128 rows, each row a (token, head of the group)
// pair, that share every K/V tile of 128 keys.  Per query tile and K/V tile:
//     S = Q K^T            128 x 128 x d, accumulator in TMEM
//     softmax              one thread per row takes its 128 scores to registers, keeps a reference maximum and the sum, and writes
//                          the probabilities to TMEM as bf16
//     O += P V             P the A operand from TMEM, V MN-major from the layout that TMA delivers, O in TMEM for the whole row
// The reference is the maximum of a row's first tile, and moves only where a later tile's probabilities add up to more than 2^24 (sum and
// division use the same reference: exact; weights and sums are floating-point numbers, as right for 2^24 as for 1).  Tiles behind the first
// therefore need no maximum: they are exponentiated at once, and once more in the rare case that the sum says so.
//
// A CTA per SM walks over items, the longest of all sequences and heads first, in turns that change direction.  Roles: warp 0 finds the
// items and fetches Q and K, warp 2 V, one thread of warp 1 issues S, one of warp 3 P V, warps 4-7 and 8-11 are the softmax of the two tiles,
// warps 12-15 write results.  Each goes on to its next item by itself, so that an item's results are written while the next one's first products
// run.
//
// Keys behind a row are masked as scores; as values they meet weights of 0, which is right for numbers only.  Rows behind a sequence
// become zeros in shared memory.  Sums of weights of 2^24 a tile and more also leave the range of numbers with values from 2^79 on, whose mean
// does not.  So where a row's result is no number, values are looked through at the end, and if one that the row does not see or a large one may be to
// blame, the row is summed up once more from what it sees, by weights that add up to 1, a thread per row (16 / 8 heads, one block behind 8000 keys: 58 ms,
// behind 1024 7.1; values of all keys looked through and nothing found: 1.1 ms a call of 8000).  Rows that no value can make numbers are left: a NaN among
// their scores, columns whose first value that all see is one (2 x 8000 tokens of NaN throughout 528 -> 0.8 ms).  It is rare, and code that ran it faster would stand
// in the way of the rest.
//
// What bounds it: for long prompts products and exponentials, 2048 cycles each per K/V tile and pair of query tiles (68 % of the tensor pipe, 68 % of
// the units for exponentials), and power: 2 x 8000 tokens of 32 / 8 heads run at 1.16 to 1.17 PFLOP/s one behind another, up to 1.34 with idle time between; the library's products at 1.43 sustained.
// For short ones the chain of an item's steps (first copies, S, softmax, P V, results) with half of either pipe idle.  What cost most on the
// way there was code: roles that run side by side share small instruction caches, and cold code ran at 5 cycles per instruction and more.
// The steps (us, replays; 64 texts of 1 to 700 tokens, 32 / 8 heads / 7 of 333 to 2100, 24 / 8 heads of 64 / 2 of 7900 to 8192, 32 / 8):
//     a warp per row and head, without tensor cores                                       13348 / 7672 / 154089
//     tensor cores; the softmax warps write results, the tiles take turns at exponentials   315 / 107 / 1171
//     without turns                                                                         228 / 89 / 983
//     masks 32 keys at a time, results in a loop, V looked through only if need be          166 / 70 / 930
//     results by warps of their own; no maximum behind the first tile                       187 / 78 / 938
//     ... waits of a few instructions, loops over the two tiles (132 -> 80 KB of code)      143 / 58 / 856
//     halves of a tile that no row of a warp sees left out                                  139 to 141 / 54 to 62 / 874 to 891
// Tried and left: an item's rows on their way to L2 ahead of it (no faster, 8 % slower with all of them); masked tiles 32 keys at a time in loops of
// their own (single tokens 88 -> 76, but 2 x 8000 tokens 846 -> 943); quarters instead of halves left out (2 x 8000 856 -> 910); results 32
// columns at a time (registers spill: 143 -> 211).
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"
#include "tensormap.cuh"

namespace b200 {
namespace {

constexpr int kMaxDim = 128, kMaxBatch = 1024, kMaxGroup = 128;
constexpr int kTile = 128;                  // keys per K/V tile and rows per query tile
constexpr int kThreads = 512;               // warpgroups: copies and issue, softmax of either query tile, output
// The first and the last one leave registers to the others; 512 x 128 are launched.
constexpr int kFewRegs = 72, kSoftmaxRegs = 184;
static_assert(128 * (2 * kFewRegs + 2 * kSoftmaxRegs) <= kThreads * 128, "");
constexpr uint32_t kAtomBytes = 128 * 128;  // 128 rows x 64 bf16 under the 128-byte swizzle
constexpr uint32_t kStageBytes = 32 * 64;   // a warp's output rows, 32 columns
constexpr int kAgain = 2048;                // query tiles of a CTA that are noted one by one
constexpr float kMostSum = 1 << 24;         // the reference moves where a row's probabilities of a tile add up to more
constexpr float kFar = 1 << 14;              // the scaled reference is rounded before it is subtracted: by 2^-11 here, beyond 2^31 weights overflow or vanish
constexpr uint32_t kLargeBits = (127 + 80) << 7;   // of bf16 2^80: kMostSum of at most 2^21 tiles times smaller values stay below 2^125

// Sizes by the padded head dimension.
template <int DP>
struct Shape {
    static constexpr int kHalves = DP / 64;
    static constexpr int kKSlots = DP == 128 ? 2 : 3, kVSlots = kKSlots;
    static constexpr uint32_t kSlotBytes = kHalves * kAtomBytes;
    static constexpr uint32_t kQOff = 0, kKOff = 2 * kSlotBytes, kVOff = kKOff + kKSlots * kSlotBytes;
    static constexpr uint32_t kStageOff = kVOff + kVSlots * kSlotBytes;
    static constexpr uint32_t kSmemBytes = kStageOff + 4 * kStageBytes;
    // TMEM columns: S (128, of both tiles in turn where O takes 256), P0, P1 (64 each), O0, O1
    static constexpr bool kSharedS = DP == 128;
    static constexpr uint32_t kColS1 = kSharedS ? 0 : 128, kColP = kSharedS ? 128 : 256, kColO = kColP + 128;
};

// A wait for the phase of that parity in few instructions (the kernel has some thirty, and its roles share the SM's small instruction caches):
// the hardware sleeps some 4 us per test, and the tests are counted: two seconds.  False: reported, and nothing more is waited for.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int* status, int site) {
    const uint32_t addr = smem_u32(bar);
#pragma unroll 1
    for (int i = 0; i < (1 << 19); ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "}\n"
            : "=r"(done)
            : "r"(addr), "r"(parity & 1u)
            : "memory");
        if (done) return true;
    }
    atomicExch(&status[kStatusTimeout], site);
    return false;
}
// The same for a whole warp whose lanes go on together.
__device__ __forceinline__ bool wait_phase_warp(uint64_t* bar, uint32_t parity, int* status, int site) {
    return __all_sync(0xffffffffu, wait_phase(bar, parity, status, site)) != 0;
}

struct PromptParams {
    __nv_bfloat16* out;
    float* lse;
    const __nv_bfloat16 *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    const int32_t* indptr;
    int tokens, batch, q_heads, kv_heads, dim;
    int group, group_inverse;   // 65536 / group, rounded up: r / group = r * group_inverse >> 16 for r <= 128
    int span;                   // query tokens of an item
    float scale_log2;
    int* status;
};

struct PromptMaps {
    CUtensorMap q, k, v;
};

struct Item {
    int first, len;       // row and length of the sequence (len < 0: no more items)
    int t0, head;         // first query token in it, KV head
    int tiles[2];         // K/V tiles of each query tile (0: it has no rows)
    int keys[2];          // keys of its last one that some row sees, to a multiple of 16
    // keys of tile kt that are multiplied with values
    __device__ __forceinline__ int reach(int kt) const {
        return max(kt + 1 < tiles[0] ? kTile : kt + 1 == tiles[0] ? keys[0] : 0, kt + 1 < tiles[1] ? kTile : kt + 1 == tiles[1] ? keys[1] : 0);
    }
};

// The items of a CTA in turn.  Those of one KV head in order: blocks that are far down their sequences first; the CTAs take them one after another,
// in turns that change direction, so that each gets long ones and short ones.  A whole warp calls.
struct Walk {
    const int *indptr, *blocks;
    int batch, kv_heads, span, half, total, ctas, me;
    int place, above, upto;       // at_least(place + 1), at_least(place): items only come nearer to the beginnings

    // items of a KV head whose block is the j-th of its sequence or a later one
    __device__ __forceinline__ int at_least(int j) const {
        int n = 0;
#pragma unroll 1
        for (int s = threadIdx.x & 31; s < batch; s += 32) n += max(blocks[s] - j, 0);
        return __reduce_add_sync(0xffffffffu, n);
    }
    __device__ __forceinline__ Walk(const PromptParams& p, const int* indptr_, const int* blocks_, int half_)
        : indptr(indptr_), blocks(blocks_), batch(p.batch), kv_heads(p.kv_heads), span(p.span), half(half_), ctas(gridDim.x), me(blockIdx.x) {
        int most = 0;
#pragma unroll 1
        for (int s = threadIdx.x & 31; s < batch; s += 32) most = max(most, blocks[s]);
        place = __reduce_max_sync(0xffffffffu, most);
        above = upto = 0;
        total = at_least(0) * kv_heads;
    }
    // The n-th (n not falling).
    __device__ __forceinline__ void find(int n, Item* it) {
        const int lane = threadIdx.x & 31, index = n * ctas + ((n & 1) != 0 ? ctas - 1 - me : me);
        if (index >= total) {
            if (lane == 0) it->len = -1;
        } else {
            const int k = index / kv_heads;
            while (upto <= k) {
                above = upto;
                upto = at_least(--place);
            }
            int rank = k - above;                       // that one of the sequences with a block there
#pragma unroll 1
            for (int base = 0; base < batch; base += 32) {
                const bool has = base + lane < batch && blocks[base + lane] > place;
                const uint32_t all = __ballot_sync(0xffffffffu, has);
                if (rank < __popc(all)) {
                    if (has && __popc(all & ((1u << lane) - 1u)) == rank) {
                        const int first = indptr[base + lane], len = indptr[base + lane + 1] - first, t0 = place * span;
                        it->first = first;
                        it->len = len;
                        it->t0 = t0;
                        it->head = index - k * kv_heads;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int from = t0 + i * half, to = min(min(from + half, t0 + span), len), tiles = from < to ? (to + kTile - 1) / kTile : 0;
                            it->tiles[i] = tiles;
                            it->keys[i] = (to - (tiles - 1) * kTile + 15) & ~15;
                        }
                    }
                    break;
                }
                rank -= __popc(all);
            }
        }
        __syncwarp();
    }
};

// A warp's rows of a query tile once more, from the keys that each row sees and no others and with weights that add up to 1, where a row is no number
// and its keys need not be to blame: a value that is no number among those of tokens [first, end) may have met the weight 0 of a row before it,
// and values from 2^79 on the sum of all weights, which only then are divided by it.  If there are neither, nothing is done (the rows are
// what their own values make them).  tok, h: the row's token and head of the group.
__device__ __noinline__ void sum_up_again(const PromptParams& p, int seq_first, int kv_head, int first, int end, int tok, int h, bool store) {
    const int lane = threadIdx.x & 31, vectors = p.dim >> 3, keys = 32 / vectors, sub = lane / vectors, column = (lane - sub * vectors) * 8;
    const __nv_bfloat16* v = p.v + static_cast<int64_t>(seq_first) * p.v_st + kv_head * p.v_sh;
    const __nv_bfloat16* k = p.k + static_cast<int64_t>(seq_first) * p.k_st + kv_head * p.k_sh;
    // Two numbers at a time: exponents and fractions as integers, 0x7f80 and more for no numbers, which 0x80 more make negative before `first`.
    // Columns in which `first`, which all rows see, is NaN: they are NaN whatever else there is.
    const bool looks = sub < keys;
    const uint4 x0 = looks ? *reinterpret_cast<const uint4*>(v + first * p.v_st + column) : make_uint4(0, 0, 0, 0);
    auto mask_of = [&](uint32_t w) { return looks ? __vcmpleu2(w & 0x7fff7fffu, 0x7f807f80u) & 0x7fff7fffu : 0u; };
    const uint4 mask = make_uint4(mask_of(x0.x), mask_of(x0.y), mask_of(x0.z), mask_of(x0.w));
    if (!__any_sync(0xffffffffu, (mask.x | mask.y | mask.z | mask.w) != 0)) return;
    bool found = false;
#pragma unroll 1
    for (int last = end - 1; last >= 0 && !__any_sync(0xffffffffu, found); last -= 8 * keys) {
        uint32_t most = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int key = last - u * keys - sub;
            if (!looks || key < 0) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(v + key * p.v_st + column);
            const uint32_t seen = key < first ? 0x00800080u : 0u;
            most = __vmaxs2(__vmaxs2(most, (x.x & mask.x) + seen), (x.y & mask.y) + seen);
            most = __vmaxs2(__vmaxs2(most, (x.z & mask.z) + seen), (x.w & mask.w) + seen);
        }
        found = (most & 0xffffu) >= kLargeBits || most >> 16 >= kLargeBits;
    }
    if (!__any_sync(0xffffffffu, found)) return;
    const int64_t row = seq_first + tok, head = kv_head * p.group + h;
    const __nv_bfloat16* q = p.q + row * p.q_st + head * p.q_sh;
    auto score = [&](int key) {
        float s = 0.f;
#pragma unroll 4
        for (int d = 0; d < p.dim; d += 8) {
            const Vec8 a = load8(q + d), b = load8(k + key * p.k_st + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(a.v[e], b.v[e], s);
        }
        return __fmul_rn(s, p.scale_log2);   // (the same number in both passes, whatever is made of it)
    };
    float m = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int key = 0; key <= tok; ++key) {
        const float s = score(key), now = fmaxf(m, s);
        sum = now > -INFINITY ? fmaf(sum, exp2f(m - now), exp2f(s - now)) : s == -INFINITY ? sum : s;   // (a score that is no number makes the sum none)
        m = now;
    }
    const float inv = sum > 0.f ? 1.f / sum : sum;
#pragma unroll 1
    for (int c = 0; c < p.dim; c += 64) {
        float o[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) o[i] = 0.f;
#pragma unroll 1
        for (int key = 0; key <= tok; ++key) {
            const float w = m == -INFINITY ? inv : exp2f(score(key) - m) * inv;
#pragma unroll
            for (int e = 0; e < 64; e += 8) {
                if (c + e >= p.dim) break;
                const Vec8 x = load8(v + key * p.v_st + c + e);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[e + i] = fmaf(w, x.v[i], o[e + i]);
            }
        }
#pragma unroll
        for (int e = 0; e < 64; e += 8) {
            if (!store || c + e >= p.dim) break;
            Vec8 x;
#pragma unroll
            for (int i = 0; i < 8; ++i) x.v[i] = o[e + i];
            store8(p.out + (row * p.q_heads + head) * p.dim + c + e, x);
        }
    }
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
prompt_attention_kernel(const __grid_constant__ PromptMaps maps, const __grid_constant__ PromptParams p) {
    using X = Shape<DP>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_indptr[kMaxBatch + 1];
    __shared__ int s_blocks[kMaxBatch];               // items per KV head of a sequence
    __shared__ Item s_item[2], s_redo[8];
    __shared__ __align__(8) uint64_t item_full[2], item_empty[2];
    __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[X::kKSlots], k_empty[X::kKSlots], v_full[X::kVSlots], v_empty[X::kVSlots];
    __shared__ __align__(8) uint64_t v_ready[X::kVSlots];   // a tile's rows behind the sequence have become zeros
    __shared__ __align__(8) uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];
    __shared__ __align__(8) uint64_t rows_full[2][2], o_free[2];   // reference and sum of a tile's rows are there (items in turn); O has been read
    __shared__ float2 s_rows[2][2][kTile];
    __shared__ uint32_t s_again[kAgain / 32 + 1];   // query tiles whose rows are not all numbers, a bit each; the last word: of later items
    __shared__ __align__(8) uint64_t drain[2];
    __shared__ uint32_t tmem_base_slot;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int G = p.group;
    auto token_of = [&](int r) { return r * p.group_inverse >> 16; };   // of a tile's row
    const int QB = token_of(kTile);

    if (tid == 0) {
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&item_full[i]), 1);
            mbar_init(smem_u32(&item_empty[i]), 4 + 8 + 4);
            mbar_init(smem_u32(&q_full[i]), 1);
            mbar_init(smem_u32(&q_empty[i]), 1);
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_free[i]), 4);
            mbar_init(smem_u32(&p_full[i]), 4);
            mbar_init(smem_u32(&pv_done[i]), 1);
            mbar_init(smem_u32(&drain[i]), 1);
            mbar_init(smem_u32(&rows_full[i][0]), 4);
            mbar_init(smem_u32(&rows_full[i][1]), 4);
            mbar_init(smem_u32(&o_free[i]), 4);
        }
        for (int s = 0; s < X::kKSlots; ++s) {
            mbar_init(smem_u32(&k_full[s]), 1);
            mbar_init(smem_u32(&k_empty[s]), 1);
        }
        for (int s = 0; s < X::kVSlots; ++s) {
            mbar_init(smem_u32(&v_full[s]), 1);
            mbar_init(smem_u32(&v_empty[s]), 1);
            mbar_init(smem_u32(&v_ready[s]), 1);
        }
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    pdl_launch_dependents();
    pdl_wait_prior();
    for (int i = tid; i <= kAgain / 32; i += kThreads) s_again[i] = 0;
    bool odd = false;
    for (int s = tid; s < p.batch; s += kThreads) {
        const int a = p.indptr[s], b = p.indptr[s + 1];
        odd = odd || a < 0 || b < a || b > p.tokens;
        s_indptr[s] = a;
        if (s == p.batch - 1) s_indptr[p.batch] = b;
        s_blocks[s] = (max(b - a, 0) + p.span - 1) / p.span;
    }
    if (QB * G < kTile) {   // rows of a query tile that no copy ever writes
        for (uint32_t a = tid * 16; a < 2 * X::kSlotBytes; a += kThreads * 16)
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(smem_base + X::kQOff + a), "r"(0u) : "memory");
        fence_proxy_async_smem();
    }
    if (__syncthreads_or(odd)) {
        if (blockIdx.x == 0 && tid == 0) atomicExch(&p.status[kStatusBadIndex], bad_index_word(p.tokens));
        return;
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));

    if (warp == 0) {
        // ================= items, Q and K =================
        Walk walk(p, s_indptr, s_blocks, QB);
        uint32_t slot = 0, phase = 1, uses[2] = {0, 0}, loads = 0;
        bool ok = true;
        const bool leader = lane == 0;
        auto publish = [&](int n) {
            if (!wait_phase_warp(&item_empty[n & 1], static_cast<uint32_t>(n >> 1 & 1) ^ 1u, p.status, 371)) return false;
            walk.find(n, &s_item[n & 1]);
            if (lane == 0) mbar_arrive(smem_u32(&item_full[n & 1]));
            return true;
        };
        ok = publish(0);
        for (int n = 0; ok; ++n) {
            const Item* it = &s_item[n & 1];
            const int first = it->first, head = it->head, t0 = it->t0, tiles0 = it->tiles[0], tiles1 = it->tiles[1];
            const bool end = it->len < 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&item_empty[n & 1]));
            if (end) break;
            auto load_q = [&](int i) {
                ok = ok && wait_phase_warp(&q_empty[i], (uses[i] & 1u) ^ 1u, p.status, 372);
                ++uses[i];
                if (ok && leader) {
                    const uint32_t bar = smem_u32(&q_full[i]), dst = smem_base + X::kQOff + i * X::kSlotBytes;
                    mbar_arrive_expect_tx(bar, static_cast<uint32_t>(X::kHalves * QB * G * 128));
                    for (int c = 0; c < X::kHalves; ++c) tma_load_3d(dst + c * kAtomBytes, &maps.q, c * 64, head * G, first + t0 + i * QB, bar);
                }
            };
            const int ntiles = max(tiles0, tiles1);
            load_q(0);
            for (int kt = 0; kt < ntiles && ok; ++kt) {
                ok = wait_phase_warp(&k_empty[slot], phase, p.status, 373);
                if (!ok) break;
                if (leader) {
                    const uint32_t bar = smem_u32(&k_full[slot]), dst = smem_base + X::kKOff + slot * X::kSlotBytes;
                    mbar_arrive_expect_tx(bar, X::kSlotBytes);
                    for (int c = 0; c < X::kHalves; ++c) tma_load_3d(dst + c * kAtomBytes, &maps.k, c * 64, head, first + kt * kTile, bar);
                }
                ++loads;
                if (++slot == X::kKSlots) {
                    slot = 0;
                    phase ^= 1;
                }
                if (kt == 0) {
                    if (tiles1 > 0) load_q(1);
                    ok = ok && publish(n + 1);   // (while the copies are under way)
                }
            }
        }
        // The block ends when nothing of it is under way: the releases of the last tiles, or the copies themselves.
        for (uint32_t s = 0; s < X::kKSlots; ++s) {
            const uint32_t at = (slot + s) % X::kKSlots, turns = loads / X::kKSlots + (at < loads % X::kKSlots ? 1 : 0);
            if (turns > 0) wait_phase_warp(ok ? &k_empty[at] : &k_full[at], (turns - 1) & 1u, p.status, 374);
        }
        for (int i = 0; i < 2; ++i)
            if (uses[i] > 0) wait_phase_warp(ok ? &q_empty[i] : &q_full[i], (uses[i] - 1) & 1u, p.status, 374);
    } else if (warp == 2) {
        // ================= V =================
        uint32_t slot = 0, phase = 1, loads = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
            ok = wait_phase_warp(&item_full[n & 1], static_cast<uint32_t>(n >> 1 & 1), p.status, 375);
            if (!ok) break;
            const Item it = s_item[n & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&item_empty[n & 1]));
            if (it.len < 0) break;
            const int ntiles = max(it.tiles[0], it.tiles[1]);
            for (int kt = 0; kt < ntiles; ++kt) {
                ok = wait_phase_warp(&v_empty[slot], phase, p.status, 376);
                if (!ok) break;
                const uint32_t bar = smem_u32(&v_full[slot]), dst = smem_base + X::kVOff + slot * X::kSlotBytes;
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, X::kSlotBytes);
                    for (int c = 0; c < X::kHalves; ++c) tma_load_3d(dst + c * kAtomBytes, &maps.v, c * 64, it.head, it.first + kt * kTile, bar);
                }
                ++loads;
                const int rows = it.len - kt * kTile, reach = it.reach(kt);
                if (kt == ntiles - 1 && rows < reach) {
                    ok = wait_phase_warp(&v_full[slot], phase ^ 1u, p.status, 377);
                    if (!ok) break;
                    for (int c = 0; c < X::kHalves; ++c)
                        for (int row = rows + (lane >> 3); row < reach; row += 4)
                            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(dst + c * kAtomBytes + row * 128 + (lane & 7) * 16), "r"(0u) : "memory");
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&v_ready[slot]));
                }
                if (++slot == X::kVSlots) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            if (!ok) break;
        }
        for (uint32_t s = 0; s < X::kVSlots; ++s) {
            const uint32_t turns = loads / X::kVSlots + (s < loads % X::kVSlots ? 1 : 0);
            if (turns > 0) wait_phase_warp(ok ? &v_empty[s] : &v_full[s], (turns - 1) & 1u, p.status, 374);
        }
    } else if (warp == 1) {
        // ================= issuer of S_i = Q_i K^T =================
        if (elect_one()) {
            const uint64_t q_desc = kmajor_sw128_desc(smem_base + X::kQOff), k_desc = kmajor_sw128_desc(smem_base + X::kKOff);
            const int steps = (p.dim + 15) >> 4;
            // (phases: a bit per query tile)
            uint32_t slot = 0, phase = 0, q_phase = 0, made = 0, last = 0;
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int site) { ok = ok && wait_phase(bar, parity, p.status, site); };
            for (int n = 0; ok; ++n) {
                const Item* it = &s_item[n & 1];
                wait(&item_full[n & 1], static_cast<uint32_t>(n >> 1), 378);
                if (!ok || it->len < 0) break;
                const int tiles0 = it->tiles[0], tiles1 = it->tiles[1], keys0 = it->keys[0], keys1 = it->keys[1];
                mbar_arrive(smem_u32(&item_empty[n & 1]));
                const int ntiles = max(tiles0, tiles1);
#pragma unroll 1
                for (int kt = 0; kt < ntiles && ok; ++kt) {
                    const uint64_t k = k_desc + slot * (X::kSlotBytes >> 4);
                    wait(&k_full[slot], phase, 379);
#pragma unroll 1
                    for (uint32_t i = 0; i < 2; ++i) {
                        const int tiles = i == 0 ? tiles0 : tiles1;
                        if (kt >= tiles) continue;
                        if (kt == 0) {
                            wait(&q_full[i], q_phase >> i, 380);
                            q_phase ^= 1u << i;
                        }
                        // the columns' last scores have to have been read
                        if (!X::kSharedS) last = i;
                        wait(&s_free[last], (made >> last) ^ 1u, 381);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t idesc = idesc_bf16_m128(kt == tiles - 1 ? (i == 0 ? keys0 : keys1) : kTile);
                        const uint64_t a = q_desc + i * (X::kSlotBytes >> 4);
                        const uint32_t d = tmem_base + i * X::kColS1;
#pragma unroll
                        for (int ks = 0; ks < DP / 16; ++ks)
                            if (ks < steps)
                                tc_mma_bf16(d, a + (((ks >> 2) * kAtomBytes + (ks & 3) * 32) >> 4), k + (((ks >> 2) * kAtomBytes + (ks & 3) * 32) >> 4), idesc,
                                            ks > 0 ? 1u : 0u);
                        tc_commit(smem_u32(&s_full[i]));
                        if (kt == tiles - 1) tc_commit(smem_u32(&q_empty[i]));
                        made ^= 1u << i;
                        last = i;
                    }
                    if (!ok) break;
                    tc_commit(smem_u32(&k_empty[slot]));
                    if (++slot == X::kKSlots) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok) {   // products under way end before the block does
                tc_commit(smem_u32(&drain[0]));
                wait_phase(&drain[0], 0, p.status, 374);
            }
        }
    } else if (warp == 3) {
        // ================= issuer of O_i += P_i V =================
        if (elect_one()) {
            const uint32_t idesc = idesc_bf16_128xn((p.dim + 15) & ~15, true);
            const uint64_t v_desc = mnmajor_sw128_desc(smem_base + X::kVOff);
            uint32_t slot = 0, phase = 0, p_phase = 0, o_phase = 0, looked = 0;   // (a bit per query tile; of the last: per slot)
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int site) { ok = ok && wait_phase(bar, parity, p.status, site); };
            for (int n = 0; ok; ++n) {
                const Item* it = &s_item[n & 1];
                wait(&item_full[n & 1], static_cast<uint32_t>(n >> 1), 378);
                if (!ok || it->len < 0) break;
                const int tiles0 = it->tiles[0], tiles1 = it->tiles[1], keys0 = it->keys[0], keys1 = it->keys[1];
                const int ntiles = max(tiles0, tiles1);
                const bool tail = it->len - (ntiles - 1) * kTile < it->reach(ntiles - 1);
                mbar_arrive(smem_u32(&item_empty[n & 1]));
#pragma unroll 1
                for (int kt = 0; kt < ntiles && ok; ++kt) {
                    const uint64_t v = v_desc + slot * (X::kSlotBytes >> 4);
                    wait(&v_full[slot], phase, 382);
                    if (tail && kt == ntiles - 1) {
                        wait(&v_ready[slot], looked >> slot, 383);
                        looked ^= 1u << slot;
                    }
#pragma unroll 1
                    for (uint32_t i = 0; i < 2; ++i) {
                        const int tiles = i == 0 ? tiles0 : tiles1;
                        if (kt >= tiles) continue;
                        if (kt == 0) {
                            wait(&o_free[i], (o_phase >> i) ^ 1u, 385);   // (of the item before)
                            o_phase ^= 1u << i;
                        }
                        wait(&p_full[i], p_phase >> i, 384);
                        p_phase ^= 1u << i;
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t prob = tmem_base + X::kColP + i * 64u, d = tmem_base + X::kColO + i * DP;
                        const int keys = kt == tiles - 1 ? (i == 0 ? keys0 : keys1) : kTile;
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)   // keys ks*16 .. +15: eight packed columns
                            if (ks * 16 < keys) tc_mma_bf16_ts(d, prob + static_cast<uint32_t>(ks * 8), v + (ks * 2048 >> 4), idesc, (kt > 0 || ks > 0) ? 1u : 0u);
                        tc_commit(smem_u32(&pv_done[i]));
                    }
                    if (!ok) break;
                    tc_commit(smem_u32(&v_empty[slot]));
                    if (++slot == X::kVSlots) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok) {
                tc_commit(smem_u32(&drain[1]));
                wait_phase(&drain[1], 0, p.status, 374);
            }
        }
    } else if (warp < 12) {
        // ================= softmax =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int tile = (warp >> 2) - 1;         // query tile of this warp
        const int qtr = warp & 3;                 // TMEM lane quarter this warp may read
        const int r = qtr * 32 + lane;            // query row = TMEM lane
        const int r_tok = token_of(r);
        const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(qtr * 32) << 16);
        const uint32_t s_addr = lane_addr + (tile == 1 ? X::kColS1 : 0u);
        const uint32_t p_addr = lane_addr + X::kColP + static_cast<uint32_t>(tile) * 64u;
        const uint32_t o_addr = lane_addr + X::kColO + static_cast<uint32_t>(tile) * DP;
        const float sc = p.scale_log2;
        uint32_t uses = 0, items = 0;             // K/V tiles of this query tile so far, items with rows in it
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
            if (ok && !wait_phase_warp(bar, parity, p.status, site)) ok = false;
        };

        for (int n = 0; ok; ++n) {
            wait(&item_full[n & 1], static_cast<uint32_t>(n >> 1), 386);
            if (!ok) break;
            const int len = s_item[n & 1].len, t0 = s_item[n & 1].t0, mine = s_item[n & 1].tiles[tile], keys16 = s_item[n & 1].keys[tile];
            __syncwarp();
            if (len < 0) break;
            if (lane == 0) mbar_arrive(smem_u32(&item_empty[n & 1]));
            const int limit = min(t0 + tile * QB + r_tok, len - 1);   // last visible key of this row
            float m_ref = -INFINITY;   // what the exponentials refer to, in units of the raw scores
            float l_run = 0.f;
            for (int kt = 0; kt < mine; ++kt, ++uses) {
                wait(&s_full[tile], uses, 387);
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s[c]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_free[tile]));
                const int seen = limit + 1 - kt * kTile;      // keys of the tile that the row sees
                bool half_only = false;   // no row sees the second half of the keys
                if (__any_sync(0xffffffffu, seen < kTile)) {
                    half_only = __all_sync(0xffffffffu, seen <= kTile / 2);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (__all_sync(0xffffffffu, seen >= c * 32 + 32) || (c >= 2 && half_only)) continue;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (c * 32 + i >= seen) s[c][i] = 0xff800000u;
                    }
                }
                if (uses > 0) wait(&pv_done[tile], uses - 1, 388);   // the last product has read P and added to O
                tc_fence_after();
                float tile_sum;
                bool move = kt == 0;
#pragma unroll 1
                for (;;) {
                    if (move) {
                        // The reference moves to the row's maximum; O and the sum shrink by the same factor.  (TMEM accesses are warp-wide: a
                        // warp rescales all of its rows, by 1 where nothing has moved.)
                        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (c == 2 && half_only) break;   // (scores of nobody's)
#pragma unroll
                            for (int i = 0; i < 32; i += 2)
                                m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
                        }
                        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                        float alpha = 1.f;
                        if (mx > m_ref) {
                            if (m_ref != -INFINITY) alpha = ex2_approx((m_ref - mx) * sc);
                            m_ref = mx;
                        }
                        if (kt > 0) {
                            l_run *= alpha;
                            tmem_st_wait();
#pragma unroll 1
                            for (int c = 0; c < DP / 4; ++c) {   // (rare: few registers beside the scores)
                                uint32_t ov[4];
                                asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                                             : "=r"(ov[0]), "=r"(ov[1]), "=r"(ov[2]), "=r"(ov[3]) : "r"(o_addr + c * 4) : "memory");
                                tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 4; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                                asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};"
                                             ::"r"(o_addr + c * 4), "r"(ov[0]), "r"(ov[1]), "r"(ov[2]), "r"(ov[3]) : "memory");
                            }
                        }
                    }
                    float mb = m_ref == -INFINITY ? INFINITY : m_ref * sc;   // (no key seen yet: probabilities 0)
                    if (move) {
                        const bool far = fabsf(mb) > kFar && fabsf(m_ref) < INFINITY;
                        if (__any_sync(0xffffffffu, far)) {   // (rare) differences of the raw scores instead, which are exact where they matter
                            const float2 to = make_float2(far ? -m_ref : 0.f, far ? -m_ref : 0.f);
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
#pragma unroll
                                for (int i = 0; i < 32; i += 2) {
                                    const float2 d = add2(make_float2(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), to);
                                    s[c][i] = __float_as_uint(d.x);
                                    s[c][i + 1] = __float_as_uint(d.y);
                                }
                            }
                            if (far) mb = 0.f;
                        }
                    }
                    const float2 sc2 = make_float2(sc, sc), mb2 = make_float2(-mb, -mb);
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t packed[16];
                        if (c == 2 && half_only) {
                            if (kt + 1 < mine || keys16 > kTile / 2) {
#pragma unroll
                                for (int i = 0; i < 16; ++i) packed[i] = 0;
                                tmem_st_32x32b_x16(p_addr + 32, packed);
                                tmem_st_32x32b_x16(p_addr + 48, packed);
                            }
                            break;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 e = fma2(make_float2(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), sc2, mb2);
                            const float2 pr = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                            sum = add2(sum, pr);
                            packed[i >> 1] = pack_bf16(pr.x, pr.y);
                        }
                        tmem_st_32x32b_x16(p_addr + c * 16, packed);
                    }
                    tile_sum = sum.x + sum.y;
                    if (move || !__any_sync(0xffffffffu, tile_sum > kMostSum || fabsf(mb) > kFar)) break;
                    move = true;
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[tile]));
                l_run += tile_sum;
            }
            if (mine > 0) {
                s_rows[tile][items & 1][r] = make_float2(m_ref, l_run);
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&rows_full[tile][items & 1]));
                ++items;
            }
        }
        // ---- rows that are no numbers, once more where that is not their own keys' doing (behind the last output) ----
        asm volatile("bar.sync 1, 384;" ::: "memory");
        bool any = false;
#pragma unroll 1
        for (int i = lane; i <= kAgain / 32; i += 32) any = any || s_again[i] != 0;
        if (__any_sync(0xffffffffu, any) && ok) {
            Walk walk(p, s_indptr, s_blocks, QB);
#pragma unroll 1
            for (int n = 0;; ++n) {
                const uint32_t noted = n < kAgain / 2 ? s_again[n >> 4] >> (2 * n & 31) & 3u : s_again[kAgain / 32] != 0 ? 3u : 0u;
                if (noted == 0 && n < kAgain / 2 && n * walk.ctas < walk.total) continue;
                Item* it = &s_redo[warp - 4];
                walk.find(n, it);
                if (it->len < 0) break;
                const int first = it->t0 + tile * QB, rows = min(min(QB, it->t0 + p.span - first), it->len - first);
                if ((noted >> tile & 1u) != 0 && rows > 0)
                    sum_up_again(p, it->first, it->head, first, min(it->len, first + 2 * kTile), first + min(r_tok, rows - 1), r - r_tok * G, r_tok < rows);
                __syncwarp();
            }
        }
    } else {
        // ================= output: O / sum =================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        const int qtr = warp & 3;
        const int r = qtr * 32 + lane;
        const int r_tok = token_of(r), r_head = r - r_tok * G;
        const uint32_t stage = smem_base + X::kStageOff + static_cast<uint32_t>(qtr) * kStageBytes;
        uint32_t uses = 0, items = 0;             // their parities, a bit per query tile; of the second: two bits each
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
            if (ok && !wait_phase_warp(bar, parity & 1u, p.status, site)) ok = false;
        };
        for (int n = 0; ok; ++n) {
            wait(&item_full[n & 1], static_cast<uint32_t>(n >> 1), 386);
            if (!ok) break;
            const Item it = s_item[n & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&item_empty[n & 1]));
            if (it.len < 0) break;
#pragma unroll 1
            for (int tile = 0; tile < 2; ++tile) {
                const int tiles = tile == 0 ? it.tiles[0] : it.tiles[1];
                if (tiles == 0) continue;
                uses ^= static_cast<uint32_t>(tiles & 1) << tile;
                const uint32_t turn = items >> (2 * tile) & 3u;
                items = (items & ~(3u << (2 * tile))) | ((turn + 1) & 3u) << (2 * tile);
                const int first = it.t0 + tile * QB;                                        // token of the sequence
                const int rows = min(min(QB, it.t0 + p.span - first), it.len - first);     // tokens of this tile
                // four lanes write the 64 bytes of 32 columns of a row
                int to[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row2 = qtr * 32 + i * 8 + (lane >> 2), tok2 = token_of(row2);
                    to[i] = tok2 < rows ? (it.first + first + tok2) * p.q_heads + it.head * G + row2 - tok2 * G : -1;
                }
                wait(&rows_full[tile][turn & 1], turn >> 1, 389);
                const float2 ml = s_rows[tile][turn & 1][r];
                const float inv = ml.y > 0.f ? __frcp_rn(ml.y) : ml.y;      // (a sum that is no number makes the row none)
                if (ok && r_tok < rows && p.lse != nullptr)
                    p.lse[(it.first + first + r_tok) * p.q_heads + it.head * G + r_head] = (ml.x * p.scale_log2 + log2f(ml.y)) * 0.6931471805599453f;
                wait(&pv_done[tile], (uses >> tile) ^ 1u, 390);
                tc_fence_after();
                const uint32_t o_addr = tmem_base + (static_cast<uint32_t>(qtr * 32) << 16) + X::kColO + static_cast<uint32_t>(tile) * DP;
                float2 odd = make_float2(0.f, 0.f);   // 0 as long as all are numbers
                const bool may_be = r_tok < rows && ml.y - ml.y == 0.f;   // (a sum that is no number: the row's own keys)
#pragma unroll 1
                for (int c = 0; c * 32 < p.dim; ++c) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t ov[16];
                        tmem_ld_32x32b_x16(o_addr + c * 32 + half * 16, ov);
                        tmem_ld_wait();
                        if (half == 1 && c * 32 + 32 >= p.dim) {   // the next item's products may have it
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(smem_u32(&o_free[tile]));
                        }
                        if (half == 0 || c * 32 + 16 < p.dim) {
#pragma unroll
                            for (int i = 0; i < 16; i += 2)
                                odd = fma2(make_float2(__uint_as_float(ov[i]), __uint_as_float(ov[i + 1])), make_float2(0.f, 0.f), odd);
                        }
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                w[i] = pack_bf16(__uint_as_float(ov[j * 8 + 2 * i]) * inv, __uint_as_float(ov[j * 8 + 2 * i + 1]) * inv);
                            const uint32_t a = stage + lane * 64 + (((half * 2 + j) ^ (lane >> 1 & 3)) << 4);
                            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                        }
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a = stage + (i * 8 + (lane >> 2)) * 64 + (((lane & 3) ^ (lane >> 3 & 3)) << 4);
                        uint4 w;
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(a) : "memory");
                        if (ok && to[i] >= 0 && c * 32 + (lane & 3) * 8 < p.dim)
                            *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(to[i]) * p.dim + c * 32 + (lane & 3) * 8) = w;
                    }
                    __syncwarp();
                }
                if (__any_sync(0xffffffffu, may_be && !(odd.x == 0.f && odd.y == 0.f)) && lane == 0) {
                    const int at = min(2 * n + tile, kAgain);
                    atomicOr(&s_again[at >> 5], 1u << (at & 31));
                }
            }
        }
        asm volatile("bar.arrive 1, 384;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, 512);
}

// [tokens, heads, dim] with strides, copied in boxes of 64 elements x `heads_box` heads x `tokens_box` tokens.
int make_rows_tmap(CUtensorMap* out, const void* base, int dim, int heads, int tokens, int64_t st, int64_t sh, int heads_box, int tokens_box) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) {
        set_last_error("cuTensorMapEncodeTiled is not available from this driver");
        return B200_ERR_CUDA;
    }
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(st) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(heads_box), static_cast<cuuint32_t>(tokens_box)};
    const cuuint32_t es[3] = {1, 1, 1};
    const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_error("cuTensorMapEncodeTiled (prompt rows) failed with CUresult %d", static_cast<int>(r));
        return B200_ERR_CUDA;
    }
    return B200_OK;
}

template <int DP>
int launch_prompt(const PromptMaps& maps, const PromptParams& p, int grid, cudaStream_t stream) {
    const int smem = Shape<DP>::kSmemBytes + 1024;
    static std::atomic<uint64_t> asked{0};
    B200_CHECK_CUDA(allow_smem(asked, reinterpret_cast<const void*>(prompt_attention_kernel<DP>), smem));
    B200_CHECK_CUDA(launch_kernel(prompt_attention_kernel<DP>, dim3(grid), dim3(kThreads), smem, stream, dim3(1, 1, 1), maps, p));
    return B200_OK;
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_attention_prompt(const b200_prompt_attention_args* a, b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(a != nullptr, "attention_prompt: NULL arguments");
    B200_CHECK_ARG(a->tokens >= 0 && a->batch >= 0 && a->batch <= kMaxBatch, "attention_prompt: batch must be in [0, %d], tokens not negative", kMaxBatch);
    B200_CHECK_ARG(a->head_dim >= 8 && a->head_dim <= kMaxDim && a->head_dim % 8 == 0, "attention_prompt: head_dim must be a multiple of 8 up to %d", kMaxDim);
    B200_CHECK_ARG(a->kv_heads >= 1 && a->q_heads >= 1 && a->q_heads % a->kv_heads == 0 && a->q_heads / a->kv_heads <= kMaxGroup,
                   "attention_prompt: q_heads must be a multiple of kv_heads with group size <= %d", kMaxGroup);
    const int64_t strides[6] = {a->q_stride_token, a->q_stride_head, a->k_stride_token, a->k_stride_head, a->v_stride_token, a->v_stride_head};
    for (int64_t s : strides)
        B200_CHECK_ARG(s > 0 && s % 8 == 0 && s < (1ll << 38), "attention_prompt: strides must be positive multiples of 8");
    B200_CHECK_ARG(a->sm_scale > 0.f && a->sm_scale <= 1e30f, "attention_prompt: sm_scale must be a positive number");
    B200_CHECK_ARG(static_cast<int64_t>(a->tokens) * a->q_heads <= (1 << 28), "attention_prompt: too many query rows");
    if (a->batch == 0 || a->tokens == 0) return B200_OK;
    B200_CHECK_ARG(a->out && a->q && a->k && a->v && a->indptr, "attention_prompt: NULL tensor");
    for (const void* t : {static_cast<const void*>(a->out), a->q, a->k, a->v})
        B200_CHECK_ARG(reinterpret_cast<uintptr_t>(t) % 16 == 0, "attention_prompt: out, q, k and v must be 16-byte aligned");
    int err = B200_OK;
    PromptParams p;
    p.status = device_status_words(&err);
    if (err != B200_OK) return err;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.lse = a->lse;
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.k = static_cast<const __nv_bfloat16*>(a->k);
    p.v = static_cast<const __nv_bfloat16*>(a->v);
    p.q_st = a->q_stride_token;
    p.q_sh = a->q_stride_head;
    p.k_st = a->k_stride_token;
    p.k_sh = a->k_stride_head;
    p.v_st = a->v_stride_token;
    p.v_sh = a->v_stride_head;
    p.indptr = a->indptr;
    p.tokens = a->tokens;
    p.batch = a->batch;
    p.q_heads = a->q_heads;
    p.kv_heads = a->kv_heads;
    p.dim = a->head_dim;
    p.group = a->q_heads / a->kv_heads;
    p.group_inverse = (65536 + p.group - 1) / p.group;
    p.scale_log2 = a->sm_scale * 1.4426950408889634f;
    const int QB = kTile / p.group, sms = sm_count();
    // Where there is hardly an item per SM, an item is one query tile: its K/V tiles take two thirds of the time of a pair's (16 / 8 heads: 1 x 500
    // tokens 18.6 us, so 14.3; 1 x 1000 22.5, 18.6; 4 x 300 14.0, 12.5; beyond: 3 x 700 of 16 / 2 heads 20.1, 22.5; 1 x 4000 of 8 / 1 59.5, 74.6).
    auto items_of = [&](int span) { return static_cast<int64_t>(a->tokens / span + a->batch) * a->kv_heads; };   // at most
    p.span = 2 * items_of(2 * QB) <= sms + sms / 2 ? QB : 2 * QB;
    const int grid = static_cast<int>(min(items_of(p.span), static_cast<int64_t>(sms)));
    PromptMaps maps;
    err = make_rows_tmap(&maps.q, a->q, p.dim, p.q_heads, p.tokens, a->q_stride_token, a->q_stride_head, p.group, QB);
    if (err == B200_OK) err = make_rows_tmap(&maps.k, a->k, p.dim, p.kv_heads, p.tokens, a->k_stride_token, a->k_stride_head, 1, kTile);
    if (err == B200_OK) err = make_rows_tmap(&maps.v, a->v, p.dim, p.kv_heads, p.tokens, a->v_stride_token, a->v_stride_head, 1, kTile);
    if (err != B200_OK) return err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p.dim <= 64 ? launch_prompt<64>(maps, p, grid, s) : launch_prompt<128>(maps, p, grid, s);
}

}  // extern "C"
