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
// The reference is moved only where a row's maximum has outgrown it by 2^8 (sum and division use the same reference: exact), so that a
// tile behind the first is exponentiated with the reference as it stands while its maximum is found beside, and once more in the rare
// case that the reference has to move.
//
// A CTA per SM walks over items, the longest of all sequences and heads first, in turns that change direction.  Roles: warp 0 finds the
// items and fetches Q and K, warp 2 V, one thread of warp 1 issues S, one of warp 3 P V, warps 4-7 and 8-11 are the softmax of the two tiles.
// Each goes on to its next item by itself, so that an item's output is written while the next one's first products run.
//
// Keys behind a row are masked as scores; as values they meet weights of 0, which is right for numbers only.  Warp 2 therefore looks
// through the tiles that some row of the item does not see in full: rows behind the sequence become zeros, and an infinity or NaN
// becomes 0 and is added in the end to the rows that see it.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"
#include "tensormap.cuh"

namespace b200 {
namespace {

constexpr int kMaxDim = 128, kMaxBatch = 1024, kMaxGroup = 128;
constexpr int kTile = 128;                  // keys per K/V tile and rows per query tile
constexpr int kThreads = 384;
// The first warpgroup leaves its registers to the others; 384 x 168 are launched.
constexpr int kIssueRegs = 72, kSoftmaxRegs = 216;
static_assert(128 * (kIssueRegs + 2 * kSoftmaxRegs) <= kThreads * 168, "");
constexpr uint32_t kAtomBytes = 128 * 128;  // 128 rows x 64 bf16 under the 128-byte swizzle
constexpr uint32_t kStageBytes = 32 * 64;   // a warp's output rows, 32 columns at a time
constexpr float kLazyLog2 = 8.0f;           // the reference maximum moves when the true one is 2^8 ahead
constexpr int kOddTiles = 2;                // K/V tiles of an item that some of its rows do not see in full

// Sizes by the padded head dimension.
template <int DP>
struct Shape {
    static constexpr int kHalves = DP / 64;
    static constexpr int kKSlots = DP == 128 ? 2 : 3, kVSlots = kKSlots;
    static constexpr uint32_t kSlotBytes = kHalves * kAtomBytes;
    static constexpr uint32_t kQOff = 0, kKOff = 2 * kSlotBytes, kVOff = kKOff + kKSlots * kSlotBytes;
    static constexpr uint32_t kStageOff = kVOff + kVSlots * kSlotBytes;
    static constexpr uint32_t kSmemBytes = kStageOff + 8 * kStageBytes;
    // TMEM columns: S (128, of both tiles in turn where O takes 256), P0, P1 (64 each), O0, O1
    static constexpr bool kSharedS = DP == 128;
    static constexpr uint32_t kColS1 = kSharedS ? 0 : 128, kColP = kSharedS ? 128 : 256, kColO = kColP + 128;
};

struct PromptParams {
    __nv_bfloat16* out;
    float* lse;
    const __nv_bfloat16* v;
    int64_t v_st, v_sh;
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
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
prompt_attention_kernel(const __grid_constant__ PromptMaps maps, const PromptParams p) {
    using X = Shape<DP>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_indptr[kMaxBatch + 1];
    __shared__ int s_blocks[kMaxBatch];               // items per KV head of a sequence
    __shared__ Item s_item[2];
    __shared__ uint32_t s_odd[2][kOddTiles][4];       // keys whose values are not all numbers, by item and tile
    __shared__ __align__(8) uint64_t item_full[2], item_empty[2];
    __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[X::kKSlots], k_empty[X::kKSlots], v_full[X::kVSlots], v_empty[X::kVSlots];
    __shared__ __align__(8) uint64_t v_ready[X::kVSlots];   // a tile that not all rows see has been looked through
    __shared__ __align__(8) uint64_t odd_done[2];           // ... all of an item's
    __shared__ __align__(8) uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];
    __shared__ __align__(8) uint64_t turn[2][4];      // a softmax warp of tile i lets its neighbour of the other tile exponentiate
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
            mbar_init(smem_u32(&item_empty[i]), 3 + 8);
            mbar_init(smem_u32(&q_full[i]), 1);
            mbar_init(smem_u32(&q_empty[i]), 1);
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_free[i]), 4);
            mbar_init(smem_u32(&p_full[i]), 4);
            mbar_init(smem_u32(&pv_done[i]), 1);
            mbar_init(smem_u32(&drain[i]), 1);
            mbar_init(smem_u32(&odd_done[i]), 1);
            for (int q = 0; q < 4; ++q) mbar_init(smem_u32(&turn[i][q]), 1);
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
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));

    if (warp == 0) {
        // ================= items, Q and K =================
        // The items of one KV head in order: those that end a sequence's longest row of blocks first.  Of items at place j or later in their
        // sequences there are at_least(j).
        auto at_least = [&](int j) {
            int n = 0;
            for (int s = lane; s < p.batch; s += 32) n += max(s_blocks[s] - j, 0);
            return __reduce_add_sync(0xffffffffu, n);
        };
        int most = 0;
        for (int s = lane; s < p.batch; s += 32) most = max(most, s_blocks[s]);
        int level = __reduce_max_sync(0xffffffffu, most);   // (items come in falling order)
        const int total = at_least(0) * p.kv_heads;
        const int ctas = static_cast<int>(gridDim.x), me = static_cast<int>(blockIdx.x);
        uint32_t slot = 0, phase = 1, uses[2] = {0, 0}, loads = 0;
        bool ok = true;
        const bool leader = lane == 0;
        for (int n = 0; ok; ++n) {
            const int index = n * ctas + ((n & 1) != 0 ? ctas - 1 - me : me);
            const bool any = index < total;
            Item it;
            it.len = -1;
            int ntiles = 0;
            if (any) {
                const int k = index / p.kv_heads;
                int lo = 0, hi = level;                     // at_least(lo) > k >= at_least(hi)
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (at_least(mid) > k) lo = mid; else hi = mid;
                }
                level = hi;
                int rank = k - at_least(hi), seq = 0;       // of the sequences with a block at place lo, that one
                for (int base = 0; base < p.batch; base += 32) {
                    const uint32_t has = __ballot_sync(0xffffffffu, base + lane < p.batch && s_blocks[base + lane] > lo);
                    const int c = __popc(has);
                    if (rank < c) {
                        seq = base + __fns(has, 0, rank + 1);
                        break;
                    }
                    rank -= c;
                }
                it.first = s_indptr[seq];
                it.len = s_indptr[seq + 1] - it.first;
                it.t0 = lo * p.span;
                it.head = index - k * p.kv_heads;
                for (int i = 0; i < 2; ++i) {
                    const int from = it.t0 + i * QB, to = min(min(from + QB, it.t0 + p.span), it.len);
                    it.tiles[i] = from < to ? (to + kTile - 1) / kTile : 0;
                }
                ntiles = max(it.tiles[0], it.tiles[1]);
            }
            ok = mbar_wait_warp(smem_u32(&item_empty[n & 1]), static_cast<uint32_t>(n >> 1 & 1) ^ 1u, p.status, 371);
            if (leader) {
                s_item[n & 1] = it;
                mbar_arrive(smem_u32(&item_full[n & 1]));
            }
            if (!any || !ok) break;
            auto load_q = [&](int i) {
                if (it.tiles[i] == 0) return;
                ok = ok && mbar_wait_warp(smem_u32(&q_empty[i]), (uses[i] & 1u) ^ 1u, p.status, 372);
                ++uses[i];
                if (ok && leader) {
                    const uint32_t bar = smem_u32(&q_full[i]), dst = smem_base + X::kQOff + i * X::kSlotBytes;
                    mbar_arrive_expect_tx(bar, static_cast<uint32_t>(X::kHalves * QB * G * 128));
                    for (int c = 0; c < X::kHalves; ++c) tma_load_3d(dst + c * kAtomBytes, &maps.q, c * 64, it.head * G, it.first + it.t0 + i * QB, bar);
                }
            };
            load_q(0);
            for (int kt = 0; kt < ntiles && ok; ++kt) {
                ok = mbar_wait_warp(smem_u32(&k_empty[slot]), phase, p.status, 373);
                if (!ok) break;
                if (leader) {
                    const uint32_t bar = smem_u32(&k_full[slot]), dst = smem_base + X::kKOff + slot * X::kSlotBytes;
                    mbar_arrive_expect_tx(bar, X::kSlotBytes);
                    for (int c = 0; c < X::kHalves; ++c) tma_load_3d(dst + c * kAtomBytes, &maps.k, c * 64, it.head, it.first + kt * kTile, bar);
                }
                ++loads;
                if (++slot == X::kKSlots) {
                    slot = 0;
                    phase ^= 1;
                }
                if (kt == 0) load_q(1);
            }
        }
        // The block ends when nothing of it is under way: the releases of the last tiles, or the copies themselves.
        for (uint32_t s = 0; s < X::kKSlots; ++s) {
            const uint32_t at = (slot + s) % X::kKSlots, turns = loads / X::kKSlots + (at < loads % X::kKSlots ? 1 : 0);
            if (turns > 0) mbar_wait_warp(smem_u32(ok ? &k_empty[at] : &k_full[at]), (turns - 1) & 1u, p.status, 374);
        }
        for (int i = 0; i < 2; ++i)
            if (uses[i] > 0) mbar_wait_warp(smem_u32(ok ? &q_empty[i] : &q_full[i]), (uses[i] - 1) & 1u, p.status, 374);
    } else if (warp == 2) {
        // ================= V =================
        uint32_t slot = 0, phase = 1, loads = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
            ok = mbar_wait_warp(smem_u32(&item_full[n & 1]), static_cast<uint32_t>(n >> 1 & 1), p.status, 375);
            if (!ok) break;
            const Item it = s_item[n & 1];
            if (it.len < 0) break;
            if (lane < 4 * kOddTiles) s_odd[n & 1][lane >> 2][lane & 3] = 0;
            __syncwarp();
            const int ntiles = max(it.tiles[0], it.tiles[1]), partly = it.t0 / kTile;
            for (int kt = 0; kt < ntiles; ++kt) {
                ok = mbar_wait_warp(smem_u32(&v_empty[slot]), phase, p.status, 376);
                if (!ok) break;
                const uint32_t bar = smem_u32(&v_full[slot]), dst = smem_base + X::kVOff + slot * X::kSlotBytes;
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, X::kSlotBytes);
                    for (int c = 0; c < X::kHalves; ++c) tma_load_3d(dst + c * kAtomBytes, &maps.v, c * 64, it.head, it.first + kt * kTile, bar);
                }
                ++loads;
                if (kt >= partly) {
                    ok = mbar_wait_warp(bar, phase ^ 1u, p.status, 377);
                    if (!ok) break;
                    const int rows = min(kTile, it.len - kt * kTile);
#pragma unroll 1
                    for (int c = 0; c < X::kHalves; ++c) {
#pragma unroll 4
                        for (int i = 0; i < 32; ++i) {      // four rows at a time, 16 bytes per lane
                            const int row = i * 4 + (lane >> 3);
                            const uint32_t a = dst + c * kAtomBytes + i * 512 + lane * 16;
                            uint32_t x[4];
                            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a) : "memory");
                            uint32_t bad = 0;                // an exponent of all ones: the top bit of its half
                            for (int k = 0; k < 4; ++k) bad |= (x[k] & 0x7f807f80u) + 0x00800080u;
                            if (row >= rows) {
                                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0u) : "memory");
                            } else if ((bad & 0x80008000u) != 0) {
                                for (int k = 0; k < 4; ++k) {
                                    const uint32_t b = (x[k] & 0x7f807f80u) + 0x00800080u;
                                    if ((b & 0x8000u) != 0) x[k] &= 0xffff0000u;
                                    if ((b & 0x80000000u) != 0) x[k] &= 0x0000ffffu;
                                }
                                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
                                atomicOr(&s_odd[n & 1][kt - partly][row >> 5], 1u << (row & 31));
                            }
                        }
                    }
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
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&odd_done[n & 1]));
                mbar_arrive(smem_u32(&item_empty[n & 1]));
            }
        }
        for (uint32_t s = 0; s < X::kVSlots; ++s) {
            const uint32_t turns = loads / X::kVSlots + (s < loads % X::kVSlots ? 1 : 0);
            if (turns > 0) mbar_wait_warp(smem_u32(ok ? &v_empty[s] : &v_full[s]), (turns - 1) & 1u, p.status, 374);
        }
    } else if (warp == 1) {
        // ================= issuer of S_i = Q_i K^T =================
        if (elect_one()) {
            const uint32_t idesc = idesc_bf16_128x128(false);
            const uint64_t q_desc = kmajor_sw128_desc(smem_base + X::kQOff), k_desc = kmajor_sw128_desc(smem_base + X::kKOff);
            const int steps = (p.dim + 15) >> 4;
            uint32_t slot = 0, phase = 0, uses[2] = {0, 0}, heads[2] = {0, 0};
            int last = -1;               // the tile whose scores were made last
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
                if (ok && !mbar_wait_mostly_ready(smem_u32(bar), parity & 1u, p.status, site)) ok = false;
            };
            for (int n = 0; ok; ++n) {
                wait(&item_full[n & 1], static_cast<uint32_t>(n >> 1), 378);
                if (!ok) break;
                const int t[2] = {s_item[n & 1].tiles[0], s_item[n & 1].tiles[1]}, len = s_item[n & 1].len;
                if (len < 0) break;
                mbar_arrive(smem_u32(&item_empty[n & 1]));
                const int ntiles = max(t[0], t[1]);
                for (int kt = 0; kt < ntiles && ok; ++kt) {
                    const uint64_t k = k_desc + slot * (X::kSlotBytes >> 4);
                    wait(&k_full[slot], phase, 379);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (kt >= t[i]) continue;
                        if (kt == 0) wait(&q_full[i], heads[i]++, 380);
                        // the columns' last scores have to have been read
                        if (X::kSharedS) {
                            if (last >= 0) wait(&s_free[last], uses[last] - 1, 381);
                        } else if (uses[i] > 0) {
                            wait(&s_free[i], uses[i] - 1, 381);
                        }
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t a = q_desc + static_cast<uint32_t>(i) * (X::kSlotBytes >> 4);
#pragma unroll
                        for (int ks = 0; ks < DP / 16; ++ks)
                            if (ks < steps)
                                tc_mma_bf16(tmem_base + (i == 1 ? X::kColS1 : 0u), a + (((ks >> 2) * kAtomBytes + (ks & 3) * 32) >> 4),
                                            k + (((ks >> 2) * kAtomBytes + (ks & 3) * 32) >> 4), idesc, ks > 0 ? 1u : 0u);
                        tc_commit(smem_u32(&s_full[i]));
                        if (kt == t[i] - 1) tc_commit(smem_u32(&q_empty[i]));
                        ++uses[i];
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
                mbar_wait_bounded(smem_u32(&drain[0]), 0, p.status, 374);
            }
        }
    } else if (warp == 3) {
        // ================= issuer of O_i += P_i V =================
        if (elect_one()) {
            const uint32_t idesc = idesc_bf16_128xn((p.dim + 15) & ~15, true);
            const uint64_t v_desc = mnmajor_sw128_desc(smem_base + X::kVOff);
            uint32_t slot = 0, phase = 0, uses[2] = {0, 0}, looked = 0;
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
                if (ok && !mbar_wait_mostly_ready(smem_u32(bar), parity & 1u, p.status, site)) ok = false;
            };
            for (int n = 0; ok; ++n) {
                wait(&item_full[n & 1], static_cast<uint32_t>(n >> 1), 378);
                if (!ok) break;
                const int t[2] = {s_item[n & 1].tiles[0], s_item[n & 1].tiles[1]}, len = s_item[n & 1].len, partly = s_item[n & 1].t0 / kTile;
                if (len < 0) break;
                mbar_arrive(smem_u32(&item_empty[n & 1]));
                const int ntiles = max(t[0], t[1]);
                for (int kt = 0; kt < ntiles && ok; ++kt) {
                    const uint64_t v = v_desc + slot * (X::kSlotBytes >> 4);
                    wait(&v_full[slot], phase, 382);
                    if (kt >= partly) {
                        wait(&v_ready[slot], looked >> slot, 383);
                        looked ^= 1u << slot;   // (its phase, a bit per slot)
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (kt >= t[i]) continue;
                        wait(&p_full[i], uses[i], 384);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t prob = tmem_base + X::kColP + static_cast<uint32_t>(i) * 64u;
                        const uint32_t d = tmem_base + X::kColO + static_cast<uint32_t>(i) * DP;
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)   // keys ks*16 .. +15: eight packed columns
                            tc_mma_bf16_ts(d, prob + static_cast<uint32_t>(ks * 8), v + (ks * 2048 >> 4), idesc, (kt > 0 || ks > 0) ? 1u : 0u);
                        tc_commit(smem_u32(&pv_done[i]));
                        ++uses[i];
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
                mbar_wait_bounded(smem_u32(&drain[1]), 0, p.status, 374);
            }
        }
    } else {
        // ================= softmax / output rows =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int tile = (warp >> 2) - 1;         // query tile of this warp
        const int qtr = warp & 3;                 // TMEM lane quarter this warp may read
        const int r = qtr * 32 + lane;            // query row = TMEM lane
        const int r_tok = token_of(r), r_head = r - r_tok * G;
        const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(qtr * 32) << 16);
        const uint32_t s_addr = lane_addr + (tile == 1 ? X::kColS1 : 0u);
        const uint32_t p_addr = lane_addr + X::kColP + static_cast<uint32_t>(tile) * 64u;
        const uint32_t o_addr = lane_addr + X::kColO + static_cast<uint32_t>(tile) * DP;
        const uint32_t stage = smem_base + X::kStageOff + static_cast<uint32_t>(warp - 4) * kStageBytes;
        const float sc = p.scale_log2;
        uint32_t uses = 0;                        // K/V tiles of this query tile so far
        uint32_t turns = 0;                       // ... in which both tiles took part
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
            if (ok && !__all_sync(0xffffffffu, mbar_wait_mostly_ready(smem_u32(bar), parity & 1u, p.status, site))) ok = false;
        };
        auto low_bits = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };

        for (int n = 0; ok; ++n) {
            wait(&item_full[n & 1], static_cast<uint32_t>(n >> 1), 385);
            if (!ok) break;
            const Item it = s_item[n & 1];
            if (it.len < 0) break;
            const int mine = it.tiles[tile], both = min(it.tiles[0], it.tiles[1]);
            const int tok = it.t0 + tile * QB + r_tok;
            const int limit = min(tok, it.len - 1);   // last visible key of this row
            float m_ref = -INFINITY;   // the maximum the exponentials refer to, in units of the raw scores
            float l_run = 0.f;
            for (int kt = 0; kt < mine; ++kt, ++uses) {
                wait(&s_full[tile], uses, 386);
                tc_fence_after();
                const int k0 = kt * kTile;
                const bool need_mask = __any_sync(0xffffffffu, k0 + kTile - 1 > limit);
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s[c]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_free[tile]));
                // the neighbour's exponentials first, the last product has read P and added to O
                if (kt < both && (tile == 1 || turns > 0)) wait(&turn[tile ^ 1][qtr], tile == 1 ? turns : turns - 1, 387);
                if (kt > 0) wait(&pv_done[tile], uses - 1, 388);
                tc_fence_after();
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                uint32_t seen[4];   // of a masked tile: which of each 32 keys the row sees
                float2 sum;
                // MODE 0: no masks; 1: masks; 2: no masks, and the maximum beside
                auto probabilities = [&](auto mode) {
                    const float mb = m_ref == -INFINITY ? INFINITY : m_ref * sc;   // (no key seen yet: probabilities 0)
                    const float2 sc2 = make_float2(sc, sc), mb2 = make_float2(-mb, -mb);
                    sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t packed[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float a = __uint_as_float(s[c][i]), b = __uint_as_float(s[c][i + 1]);
                            const float2 e = fma2(make_float2(a, b), sc2, mb2);
                            float2 pr = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                            if (mode == 1) {
                                if ((seen[c] >> i & 1) == 0) pr.x = 0.f;
                                if ((seen[c] >> (i + 1) & 1) == 0) pr.y = 0.f;
                            }
                            if (mode == 2) m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], a, b);
                            sum = add2(sum, pr);
                            packed[i >> 1] = pack_bf16(pr.x, pr.y);
                        }
                        tmem_st_32x32b_x16(p_addr + c * 16, packed);
                    }
                };
                // Moves the reference where the row's maximum has outgrown it; O and the sum shrink by the same factor.  (TMEM accesses are
                // warp-wide: a warp rescales all of its rows, by 1 where nothing moved.)
                auto outgrown = [&](float mx) { return mx != -INFINITY && (m_ref == -INFINITY || (mx - m_ref) * sc > kLazyLog2); };
                auto move_reference = [&](float mx) {
                    float alpha = 1.f;
                    if (outgrown(mx)) {
                        if (m_ref != -INFINITY) alpha = ex2_approx((m_ref - mx) * sc);
                        m_ref = mx;
                    }
                    if (__any_sync(0xffffffffu, alpha != 1.f)) {
                        l_run *= alpha;
#pragma unroll
                        for (int c = 0; c < DP / 16; ++c) {
                            uint32_t ov[16];
                            tmem_ld_32x32b_x16(o_addr + c * 16, ov);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                            tmem_st_32x32b_x16(o_addr + c * 16, ov);
                        }
                    }
                };
                auto highest = [&]() { return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])); };
                if (need_mask) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        seen[c] = low_bits(limit + 1 - k0 - c * 32);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            m4[i & 3] = fmaxf(m4[i & 3], (seen[c] >> i & 1) != 0 ? __uint_as_float(s[c][i]) : -INFINITY);
                    }
                    move_reference(highest());
                    probabilities(std::integral_constant<int, 1>{});
                } else {
                    if (kt == 0) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; i += 2)
                                m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
                        m_ref = highest();
                    }
                    probabilities(std::integral_constant<int, 2>{});
                    const float mx = highest();
                    if (__any_sync(0xffffffffu, outgrown(mx))) {
                        move_reference(mx);
                        probabilities(std::integral_constant<int, 0>{});
                    }
                }
                if (kt < both) {
                    if (lane == 0) mbar_arrive(smem_u32(&turn[tile][qtr]));
                    ++turns;
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full[tile]));
                l_run += sum.x + sum.y;
            }
            if (mine > 0) {
                // ---- the last product, then O / sum ----
                wait(&odd_done[n & 1], static_cast<uint32_t>(n >> 1), 389);
                wait(&pv_done[tile], uses - 1, 390);
                tc_fence_after();
                const float inv = l_run > 0.f ? 1.f / l_run : l_run;      // (a sum that is no number makes the row none)
                const int partly = it.t0 / kTile;
                uint32_t any_odd = 0;
#pragma unroll
                for (int k = 0; k < 4 * kOddTiles; ++k) any_odd |= s_odd[n & 1][k >> 2][k & 3];
                const bool store = ok && r_tok < QB && tok < it.len && tok < it.t0 + p.span;
                const int64_t row0 = static_cast<int64_t>(it.first) + it.t0 + tile * QB;
                const int head0 = it.head * G;
                if (store && p.lse != nullptr)
                    p.lse[(row0 + r_tok) * p.q_heads + head0 + r_head] = (m_ref * sc + log2f(l_run)) * 0.6931471805599453f;
#pragma unroll 1
                for (int c = 0; c < DP / 32; ++c) {
                    if (c * 32 >= p.dim) break;
                    uint32_t ov[32];
                    tmem_ld_32x32b_x32(o_addr + c * 32, ov);
                    tmem_ld_wait();
                    if (any_odd != 0) {   // (rare: values of visible keys that are no numbers)
#pragma unroll 1
                        for (int k = 0; k < 4 * kOddTiles; ++k) {
                            for (uint32_t bits = s_odd[n & 1][k >> 2][k & 3]; bits != 0; bits &= bits - 1) {
                                const int key = (partly + (k >> 2)) * kTile + (k & 3) * 32 + __ffs(bits) - 1;
                                if (key > limit) continue;
                                const __nv_bfloat16* v = p.v + static_cast<int64_t>(it.first + key) * p.v_st + it.head * p.v_sh + c * 32;
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float x = c * 32 + i < p.dim ? __bfloat162float(v[i]) : 0.f;
                                    if (!isfinite(x)) ov[i] = __float_as_uint(__uint_as_float(ov[i]) + x);
                                }
                            }
                        }
                        __syncwarp();
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            w[i] = pack_bf16(__uint_as_float(ov[j * 8 + 2 * i]) * inv, __uint_as_float(ov[j * 8 + 2 * i + 1]) * inv);
                        const uint32_t a = stage + lane * 64 + ((j ^ (lane >> 1 & 3)) << 4);
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
                    }
                    __syncwarp();
                    // four lanes write the 64 bytes of a row
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = i * 8 + (lane >> 2), row2 = qtr * 32 + rr, tok2 = token_of(row2), j = lane & 3;
                        const uint32_t a = stage + rr * 64 + ((j ^ (rr >> 1 & 3)) << 4);
                        uint4 w;
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(a) : "memory");
                        const int t = it.t0 + tile * QB + tok2;
                        if (ok && tok2 < QB && t < it.len && t < it.t0 + p.span && c * 32 + j * 8 < p.dim)
                            *reinterpret_cast<uint4*>(p.out + ((row0 + tok2) * p.q_heads + head0 + row2 - tok2 * G) * p.dim + c * 32 + j * 8) = w;
                    }
                    __syncwarp();
                }
                tc_fence_before();
            } else {
                wait(&odd_done[n & 1], static_cast<uint32_t>(n >> 1), 389);   // (so that this warp is never two of its phases behind)
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&item_empty[n & 1]));
        }
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
    B200_CHECK_CUDA(cudaFuncSetAttribute(prompt_attention_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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
    p.v = static_cast<const __nv_bfloat16*>(a->v);
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
    const int QB = kTile / p.group;
    p.span = 2 * QB;
    const int64_t items = static_cast<int64_t>(a->tokens / p.span + a->batch) * a->kv_heads;   // at most
    const int grid = static_cast<int>(items < sm_count() ? items : sm_count());
    PromptMaps maps;
    err = make_rows_tmap(&maps.q, a->q, p.dim, p.q_heads, p.tokens, a->q_stride_token, a->q_stride_head, p.group, QB);
    if (err == B200_OK) err = make_rows_tmap(&maps.k, a->k, p.dim, p.kv_heads, p.tokens, a->k_stride_token, a->k_stride_head, 1, kTile);
    if (err == B200_OK) err = make_rows_tmap(&maps.v, a->v, p.dim, p.kv_heads, p.tokens, a->v_stride_token, a->v_stride_head, 1, kTile);
    if (err != B200_OK) return err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p.dim <= 64 ? launch_prompt<64>(maps, p, grid, s) : launch_prompt<128>(maps, p, grid, s);
}

}  // extern "C"
