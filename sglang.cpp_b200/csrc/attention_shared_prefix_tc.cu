// The prefixes of attention over a shared prefix on the tcgen05 tensor cores: groups with more query rows than a warp's tile or two
// (attention_shared_prefix.cu has the formulas, the other parts and the kernel that joins them).
//
// All query rows of a group that read one KV head are one matrix, [tokens * heads per KV head, 128], in blocks of up to 256 rows; no
// row of a prefix is masked.  A unit is (group, KV head, block).  A unit's K/V tiles of 128 keys are cut into equal chunks, a CTA
// each; where there are too many units for that, the tiles of all units form one sequence that is cut into equal contiguous runs
// (shared_prefix_plan.cu).  Runs cross from unit to unit, which costs 5 to 14 us of queries, first scores, last products and
// results.  Per tile
//     S = Q K^T     128 x 128 x 128 into TMEM; a thread per row takes its 128 scores to registers
//     P = 2^(S - m) bf16 into TMEM, the A operand of      O += P V      128 x 128 x 128, accumulated in TMEM
// with the reference m moved (and O rescaled) only when the true maximum is 2^8 ahead of it.  Two chains of S, softmax and P V take
// turns on the tensor core, so that one chain's softmax runs under the other's products:
//     a block of more rows than a chain's 128: a chain per half, both on the same tiles;
//     a block of up to 128 rows:     both on the same rows, one on the even, one on the odd tiles of the run, their sums joined at
//                                    its end (in TMEM both have a row in the same lane).
// Roles: warp 0 copies K tiles, warp 2 V tiles, one thread of warp 1 issues S, one of warp 3 issues P V, warps 4-7 and 8-11 are the
// chains' softmax.  Every role walks the same items; the rings and the chains go on across them, so the next item's tiles are under
// way while one is finished.  Barriers are tested by parity: whoever tests one knows that the phase before it is over (the rings
// are filled and emptied in order, and a chain's barriers alternate between its two sides).
// A tile of two chains (16.8 MFLOP) takes 1.65 to 1.9 us, 0.8 to 0.9 of the rate of large library products, whose power limit it
// meets as well; a tile of one chain 0.85.  In pages of fewer than eight slots a tile is 128 copies of four half rows and takes 3.1 us.
// The softmax is bound by its instructions: an eighth of the exponentials on the FMA pipe cost 12 percent.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "shared_prefix.cuh"
#include "tcgen05.cuh"
#include "tensormap.cuh"

namespace b200 {
namespace {

constexpr int kD = 128;
constexpr int kTile = 128;                  // keys per K/V tile, rows per chain
constexpr int kThreads = 384;
// The first warpgroup leaves its registers to the others; 384 x 168 are launched.
constexpr int kIssueRegs = 72, kSoftmaxRegs = 216;
static_assert(128 * (kIssueRegs + 2 * kSoftmaxRegs) <= kThreads * 168, "");
constexpr uint32_t kAtomBytes = 128 * 128;  // 128 rows x 64 bf16
constexpr uint32_t kKVOff = 4 * kAtomBytes; // behind 2 tiles of queries of 2 atoms each
constexpr uint32_t kSlotBytes = 2 * kAtomBytes;
constexpr int kKSlots = 2, kVSlots = 3, kSlots = kKSlots + kVSlots;   // a ring of tiles each
constexpr uint32_t kSmemBytes = kKVOff + kSlots * kSlotBytes;
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256;  // TMEM columns: S (128, both chains in turn), P (64 each), O (128 each)
constexpr float kLazyLog2 = 8.0f;

// How K and V tiles are copied ([0] K, [1] V), into 16 groups of 8 keys, each both halves of the head dimension.
struct SharedKvMaps {
    CUtensorMap q;         // half rows of a chain's tokens, all heads of a KV head
    CUtensorMap rows[2];   // half rows of single keys, four to a copy: any slots
    CUtensorMap page[2];   // whole rows of min(page, 128) keys from a slot that 8 divides
    CUtensorMap tile[2];   // whole rows of 128 keys: tiles whose pages are consecutive slots
    int whole_pages, whole_tiles;   // are the latter two there?
    int kpc;                        // keys of a page in a tile
};

// Half rows of four slots, one behind the other in shared memory.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const void* tmap, int column, int r0, int r1, int r2, int r3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(column), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void softmax_bar() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_tc_kernel(const __grid_constant__ SharedKvMaps maps, const SharedPrefixParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full[kSlots];    // slots of K tiles, then of V tiles
    __shared__ __align__(8) uint64_t empty[kSlots];
    __shared__ __align__(8) uint64_t q_full, q_empty; // an item's queries are in shared memory, have been multiplied
    __shared__ __align__(8) uint64_t s_full[2];       // per chain: S is in TMEM
    __shared__ __align__(8) uint64_t s_free[2];       // ... and has been read from there (4 warp arrivals)
    __shared__ __align__(8) uint64_t p_full[2];       // per chain: P is in TMEM (4 warp arrivals)
    __shared__ __align__(8) uint64_t pv_done[2];      // per chain: O += P V has completed
    __shared__ uint32_t tmem_base_slot;
    __shared__ float2 s_ml[kTile];                    // second chain's statistics, where both have the same rows

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int G = p.group;
    const int QB = kTile / G;   // query tokens of a chain
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&maps.q);
        for (int kv = 0; kv < 2; ++kv) {
            if (maps.kpc < 8) tma_prefetch_desc(&maps.rows[kv]);
            if (maps.whole_pages) tma_prefetch_desc(&maps.page[kv]);
            if (maps.whole_tiles) tma_prefetch_desc(&maps.tile[kv]);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(smem_u32(&full[s]), 1);
            mbar_init(smem_u32(&empty[s]), 1);
        }
        mbar_init(smem_u32(&q_full), 1);
        mbar_init(smem_u32(&q_empty), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_free[i]), 4);
            mbar_init(smem_u32(&p_full[i]), 4);
            mbar_init(smem_u32(&pv_done[i]), 1);
        }
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_slot;

    // This CTA's items, known once the plan is there (every role asks by itself: the softmax warps have something to do before).
    int2 items;
    int ntiles = 0;   // of all of them
    auto get_items = [&]() {
        pdl_wait_prior();
        pdl_launch_dependents();
        items = p.plan.tc_of[blockIdx.x];
    };
    auto get_item = [&](int i) {
        const int4* src = reinterpret_cast<const int4*>(p.plan.tc + i);
        const int4 a = src[0], b = src[1];
        TcItem it;
        it.h = a.x, it.tok0 = a.y, it.ntok = a.z, it.keys = a.w, it.t0 = b.x, it.t1 = b.y, it.table = b.z;
        return it;
    };

    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 0 || warp == 2) {
        // ================= producers: K tiles, V tiles =================
        get_items();
        const int kv = warp >> 1, kpc = maps.kpc;
        const uint32_t ring = kv == 0 ? 0 : kKSlots, ring_end = kv == 0 ? kKSlots : kSlots;
        uint32_t slot = ring, phase = 1;   // (the first waits are for slots that nobody has used)
        bool failed = false;
        for (int i = items.x; i < items.y && !failed; ++i) {
            const TcItem it = get_item(i);
            const int32_t* pt_row = p.page_table + static_cast<int64_t>(it.table) * p.pt_stride;
            // This lane's slots, fetched a tile ahead (the table's trip to L2 would stand between a slot's release and its copy): of keys
            // lane * 4 .. + 3 where pages are smaller than a group of 8, else of the first keys of pages lane and lane + 32 ...
            const bool small = kpc < 8;
            int next[4];
            auto fetch_slots = [&](int kt) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = kt * kTile + (small ? lane * 4 + i : (i * 32 + lane) * kpc);
                    next[i] = key < it.keys && (small || (i * 32 + lane) * kpc < kTile) ? pt_row[key] : 0;
                }
            };
            fetch_slots(it.t0);
            if (kv == 0) {   // the queries: rows (token, head) of each chain, in two halves
                if (i > items.x && !__all_sync(0xffffffffu, mbar_wait_mostly_ready(smem_u32(&q_empty), (i - items.x - 1) & 1, p.status, 341))) {
                    failed = true;
                    break;
                }
                const int chains = it.ntok > QB ? 2 : 1;
                const uint32_t bar = smem_u32(&q_full);
                if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(chains * QB * G) * kD * 2u);
                __syncwarp();
                if (lane < 2 * chains)
                    tma_load_3d(smem_base + lane * kAtomBytes, &maps.q, (lane & 1) * 64, it.h * G, it.tok0 + (lane >> 1) * QB, bar);
            }
            for (int kt = it.t0; kt < it.t1; ++kt) {
                // A tile whose pages are consecutive slots is one copy; so is a page, unless it is smaller than a group of 8 or starts
                // inside one: then every four keys are.
                const int keys = min(kTile, it.keys - kt * kTile), n = small ? 0 : (keys + kpc - 1) / kpc;
                const int span = small ? 1 : kpc;   // slots that a table entry stands for here
                bool whole = keys == kTile && maps.whole_tiles, pages = !small;
                int sl[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sl[i] = next[i];
                    if (sl[i] < 0 || static_cast<int64_t>(sl[i]) + span > p.num_slots) {
                        atomicExch(&p.status[kStatusBadIndex], bad_index_word(sl[i]));
                        sl[i] = 0;
                    }
                    if ((sl[i] & 7) != 0) pages = false;
                }
                const int first = __shfl_sync(0xffffffffu, sl[0], 0);
                if ((first & 7) != 0) whole = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = small ? lane * 4 + i : (i * 32 + lane) * kpc;
                    if (key < kTile && sl[i] != first + key) whole = false;
                }
                whole = __all_sync(0xffffffffu, whole);
                pages = __all_sync(0xffffffffu, pages) && (maps.whole_pages || whole);
                if (kt + 1 < it.t1) fetch_slots(kt + 1);
                if (!__all_sync(0xffffffffu, mbar_wait_mostly_ready(smem_u32(&empty[slot]), phase, p.status, 331))) {
                    failed = true;
                    break;
                }
                const uint32_t bar = smem_u32(&full[slot]), base = smem_base + kKVOff + slot * kSlotBytes;
                if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(whole || !pages ? kTile : n * kpc) * kD * 2u);
                __syncwarp();
                if (whole) {
                    if (lane == 0) tma_load_5d(base, &maps.tile[kv], 0, 0, 0, first >> 3, it.h, bar);
                } else if (pages) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int copy = i * 32 + lane;
                        if (copy < n) tma_load_5d(base + copy * kpc * (kD * 2), &maps.page[kv], 0, 0, 0, sl[i] >> 3, it.h, bar);
                    }
                } else {
                    if (!small) {   // pages that start inside a group: their keys' slots
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = kt * kTile + lane * 4 + i;
                            sl[i] = key < it.keys ? pt_row[key] : 0;
                            if (sl[i] < 0 || sl[i] >= p.num_slots) sl[i] = 0;
                        }
                    }
                    // (keys behind the prefix: slot 0's, of which nothing is used)
                    const uint32_t dst = base + (lane >> 1) * 2048 + (lane & 1) * 512;
                    tma_gather4(dst, &maps.rows[kv], it.h * kD, sl[0], sl[1], sl[2], sl[3], bar);
                    tma_gather4(dst + 1024, &maps.rows[kv], it.h * kD + 64, sl[0], sl[1], sl[2], sl[3], bar);
                }
                if (++slot == ring_end) {
                    slot = ring;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        // ================= issuer of S = Q K^T =================
        if (elect_one()) {
            const uint32_t idesc = idesc_bf16_128x128(false);
            const uint64_t q_desc = kmajor_sw128_desc(smem_base);
            const uint64_t k_desc = grouped_keys_desc(smem_base + kKVOff, 0);
            get_items();
            for (int i = items.x; i < items.y; ++i) {
                const TcItem it = get_item(i);
                ntiles += it.t1 - it.t0;
            }
            uint32_t slot = 0, phase = 0;
            uint32_t uses[2] = {0, 0};   // of each chain so far
            int last = -1, tile = 0;     // the chain of the last scores; tiles so far
            bool failed = false;
            auto wait = [&](uint32_t bar, uint32_t parity, int site) {
                if (!failed && !mbar_wait_mostly_ready(bar, parity, p.status, site)) failed = true;
            };
            auto scores = [&](int chain, uint64_t a, uint64_t k) {
                // both chains use the same columns: the last scores have to have been read
                if (last >= 0) wait(smem_u32(&s_free[last]), (uses[last] - 1) & 1u, 338);
                if (failed) return;
                tc_fence_after();
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    tc_mma_bf16(tmem_base + kColS, a + (((ks >> 2) * kAtomBytes + (ks & 3) * 32) >> 4),
                                k + (((ks >> 2) * 1024 + (ks & 3) * 32) >> 4), idesc, ks > 0 ? 1u : 0u);
                tc_commit(smem_u32(&s_full[chain]));
                last = chain;
                ++uses[chain];
            };
            for (int i = items.x; i < items.y && !failed; ++i) {
                const TcItem it = get_item(i);
                const bool two = it.ntok > QB;
                wait(smem_u32(&q_full), static_cast<uint32_t>(i - items.x) & 1u, 339);
                for (int kt = it.t0; kt < it.t1 && !failed; ++kt, ++tile) {
                    const uint64_t k = k_desc + slot * (kSlotBytes >> 4);
                    wait(smem_u32(&full[slot]), phase, 332);
                    if (two) {
                        scores(0, q_desc, k);
                        scores(1, q_desc + (2 * kAtomBytes >> 4), k);
                    } else if (((kt - it.t0) & 1) == 0) {
                        scores(0, q_desc, k);
                    } else {
                        scores(1, q_desc, k);
                    }
                    if (failed) break;
                    // (a slot that is not filled again is not handed back: the arrival could be under way when the block ends)
                    if (tile + kKSlots < ntiles) tc_commit(smem_u32(&empty[slot]));
                    if (++slot == kKSlots) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
                if (!failed && i + 1 < items.y) tc_commit(smem_u32(&q_empty));
            }
        }
    } else if (warp == 3) {
        // ================= issuer of O += P V =================
        if (elect_one()) {
            const uint32_t idesc = idesc_bf16_128x128(true);
            const uint64_t v_desc = grouped_keys_desc(smem_base + kKVOff, 1024);
            get_items();
            for (int i = items.x; i < items.y; ++i) {
                const TcItem it = get_item(i);
                ntiles += it.t1 - it.t0;
            }
            uint32_t slot = kKSlots, phase = 0;
            uint32_t uses[2] = {0, 0};
            int tile = 0;
            bool failed = false;
            auto wait = [&](uint32_t bar, uint32_t parity, int site) {
                if (!failed && !mbar_wait_mostly_ready(bar, parity, p.status, site)) failed = true;
            };
            auto add = [&](int chain, uint64_t v, bool first) {
                wait(smem_u32(&p_full[chain]), uses[chain] & 1u, 333);
                if (failed) return;
                tc_fence_after();
                const uint32_t prob = tmem_base + kColP + static_cast<uint32_t>(chain) * 64u;
                const uint32_t d = tmem_base + kColO + static_cast<uint32_t>(chain) * 128u;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)   // keys ks*16 .. +15: eight packed columns
                    tc_mma_bf16_ts(d, prob + static_cast<uint32_t>(ks * 8), v + (ks * 4096 >> 4), idesc, !first || ks > 0 ? 1u : 0u);
                tc_commit(smem_u32(&pv_done[chain]));
                ++uses[chain];
            };
            for (int i = items.x; i < items.y && !failed; ++i) {
                const TcItem it = get_item(i);
                const bool two = it.ntok > QB;
                for (int kt = it.t0; kt < it.t1 && !failed; ++kt, ++tile) {
                    const uint64_t v = v_desc + slot * (kSlotBytes >> 4);
                    wait(smem_u32(&full[slot]), phase, 336);
                    if (two) {
                        add(0, v, kt == it.t0);
                        add(1, v, kt == it.t0);
                    } else if (((kt - it.t0) & 1) == 0) {
                        add(0, v, kt == it.t0);
                    } else {
                        add(1, v, kt == it.t0 + 1);
                    }
                    if (failed) break;
                    if (tile + kVSlots < ntiles) tc_commit(smem_u32(&empty[slot]));
                    if (++slot == kSlots) {
                        slot = kKSlots;
                        phase ^= 1;
                    }
                }
            }
        }
    } else {
        // ================= softmax, and the rows' results =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int chain = (warp >> 2) - 1;
        const int qtr = warp & 3;                 // TMEM lane quarter this warp may read
        const int r = qtr * 32 + lane;            // row = TMEM lane
        const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(qtr * 32) << 16);
        const uint32_t s_addr = lane_addr + kColS;
        const uint32_t p_addr = lane_addr + kColP + static_cast<uint32_t>(chain) * 64u;
        const uint32_t o_addr = lane_addr + kColO + static_cast<uint32_t>(chain) * 128u;
        const float sc = p.scale_log2;
        uint32_t uses = 0;
        int tiles_before = 0;
        bool failed = false;
        // The first round of all is made on whatever TMEM holds and undone, while the plan and the first copies are under way: it brings
        // the loop's instructions, which the first tile waited 4 us for otherwise.
        TcItem it = {};
        it.t0 = it.t1 = 0;
        items = make_int2(0, 1);
        for (int i = -1; i < items.y; ++i) {
            if (i >= 0) it = get_item(i);
            const bool real = i >= 0, two = it.ntok > QB;
            float m_ref = -INFINITY, l_run = 0.f;
            const int step = two ? 1 : 2;
            bool any = false;   // has this chain had a tile of the item?
            for (int kt = real ? it.t0 + (two ? 0 : chain) : -1; kt < it.t1; kt += step) {
                if (real && !failed && !mbar_wait_mostly_ready(smem_u32(&s_full[chain]), uses & 1u, p.status, 334)) failed = true;
                tc_fence_after();
                const int valid = it.keys - kt * kTile;   // keys of the tile that belong to the prefix
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s[c]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (real && lane == 0) mbar_arrive(smem_u32(&s_free[chain]));
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (valid < kTile) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (c * 32 + i >= valid) s[c][i] = 0xff800000u;   // -inf
                            m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(s[c][i]));
                        }
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
                }
                const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                // this chain's product before has read P and has added to O
                if (any && !failed && !mbar_wait_mostly_ready(smem_u32(&pv_done[chain]), (uses - 1) & 1u, p.status, 337)) failed = true;
                tc_fence_after();
                float alpha = 1.f;
                if (mx != -INFINITY && (m_ref == -INFINITY || (mx - m_ref) * sc > kLazyLog2)) {
                    if (m_ref != -INFINITY) alpha = ex2_approx((m_ref - mx) * sc);
                    m_ref = mx;
                }
                if (__any_sync(0xffffffffu, alpha != 1.f)) {
                    l_run *= alpha;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t ov[16];
                        tmem_ld_32x32b_x16(o_addr + c * 16, ov);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                        tmem_st_32x32b_x16(o_addr + c * 16, ov);
                    }
                }
                const float mb = m_ref == -INFINITY ? INFINITY : m_ref * sc;
                float2 sum = make_float2(0.f, 0.f);
                const float2 sc2 = make_float2(sc, sc), mb2 = make_float2(-mb, -mb);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 e = fma2(make_float2(__uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1])), sc2, mb2);
                        const float2 pr = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                        sum = add2(sum, pr);
                        packed[i >> 1] = pack_bf16(pr.x, pr.y);
                    }
                    tmem_st_32x32b_x16(p_addr + c * 16, packed);
                }
                if (real && valid < kTile) {
                    // Values behind the prefix (of the page, or what the slot held before) must be numbers: their weights are 0.
                    const int j = tiles_before + kt - it.t0;
                    const uint32_t slot = kKSlots + static_cast<uint32_t>(j % kVSlots);
                    if (!failed && !mbar_wait_mostly_ready(smem_u32(&full[slot]), static_cast<uint32_t>(j / kVSlots) & 1u, p.status, 340))
                        failed = true;
                    const uint32_t base = smem_base + kKVOff + slot * kSlotBytes;
                    for (int i = r; i < (kTile - valid) * 16; i += kTile) {
                        const int key = valid + (i >> 4), at = i & 15;
                        const uint32_t a = base + (key >> 3) * 2048 + (at >> 3) * 1024 + (key & 7) * 128 + (at & 7) * 16;
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0u) : "memory");
                    }
                    fence_proxy_async_smem();
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (!real) break;
                if (lane == 0) mbar_arrive(smem_u32(&p_full[chain]));
                l_run += sum.x + sum.y;
                any = true;
                ++uses;
            }
            if (!real) {
                get_items();
                i = items.x - 1;
                continue;
            }
            tiles_before += it.t1 - it.t0;
            if (any && !failed && !mbar_wait_mostly_ready(smem_u32(&pv_done[chain]), (uses - 1) & 1u, p.status, 335)) failed = true;
            __syncwarp();
            tc_fence_after();
            // ---- the rows' sums and statistics (maximum in the exponent's units) ----
            float m = m_ref == -INFINITY ? -INFINITY : m_ref * sc, l = l_run, mine = 1.f, other = 0.f;
            bool join = false;
            if (!two) {
                if (chain == 1) s_ml[r] = make_float2(any ? m : -INFINITY, any ? l : 0.f);
                tc_fence_before();
                softmax_bar();   // the second chain's sums are complete and its statistics are there
                tc_fence_after();
                join = chain == 0 && it.t1 - it.t0 > 1;
                if (join) {
                    const float2 b = s_ml[r];
                    const float top = fmaxf(m, b.x), ref = top == -INFINITY ? 0.f : top;
                    mine = ex2_approx(m - ref);
                    other = ex2_approx(b.x - ref);
                    l = l * mine + b.y * other;
                    m = top;
                }
            }
            if (two || chain == 0) {
                const int tok = r / G + (two ? chain * QB : 0);
                const bool store = r < QB * G && tok < it.ntok;
                const int64_t at = p.tc_base + static_cast<int64_t>(i) * (2 * kTile) + (two ? chain * kTile : 0) + r;
                float* dst = p.ws_o + at * kD;
#pragma unroll 1
                for (int c = 0; c < 8; ++c) {
                    uint32_t a[16], b[16];
                    tmem_ld_32x32b_x16(o_addr + c * 16, a);
                    if (join) tmem_ld_32x32b_x16(o_addr + 128 + c * 16, b);
                    tmem_ld_wait();
                    if (join) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            a[j] = __float_as_uint(__uint_as_float(a[j]) * mine + __uint_as_float(b[j]) * other);
                    }
                    if (store) {
#pragma unroll
                        for (int j = 0; j < 16; j += 8)   // a sector per store
                            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + c * 16 + j), "r"(a[j]), "r"(a[j + 1]),
                                         "r"(a[j + 2]), "r"(a[j + 3]), "r"(a[j + 4]), "r"(a[j + 5]), "r"(a[j + 6]), "r"(a[j + 7])
                                         : "memory");
                    }
                }
                if (store) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(m, failed ? 0.f : l);
            }
            tc_fence_before();
            softmax_bar();   // the item's queries and sums have been read
            tc_fence_after();
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, 512);
}

}  // namespace

int make_shared_query_tmap(CUtensorMap* out, const SharedPrefixParams& p, int heads, int tokens) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) {
        set_last_error("cuTensorMapEncodeTiled is not available from this driver");
        return B200_ERR_CUDA;
    }
    const cuuint64_t dims[3] = {kD, static_cast<cuuint64_t>(p.q_heads), static_cast<cuuint64_t>(p.tokens)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.q_sh) * 2, static_cast<cuuint64_t>(p.q_st) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(heads), static_cast<cuuint32_t>(tokens)};
    const cuuint32_t es[3] = {1, 1, 1};
    CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(p.q), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_last_error("cuTensorMapEncodeTiled (queries) failed with CUresult %d", static_cast<int>(r));
        return B200_ERR_CUDA;
    }
    return B200_OK;
}

int launch_shared_prefix_tc(const SharedPrefixParams& p, const void* k_cache, const void* v_cache, int page_size, cudaStream_t stream) {
    SharedKvMaps maps = {};
    int err = make_shared_query_tmap(&maps.q, p, p.group, kTile / p.group);
    if (err != B200_OK) return err;
    maps.kpc = page_size < kTile ? page_size : kTile;
    maps.whole_pages = maps.kpc >= 8 && p.num_slots >= 8 ? 1 : 0;
    maps.whole_tiles = p.num_slots >= kTile ? 1 : 0;
    for (int kv = 0; kv < 2; ++kv) {
        const void* cache = kv == 0 ? k_cache : v_cache;
        const uint64_t width = static_cast<uint64_t>(p.kv_heads) * kD;
        err = make_tmap_2d_bf16_sw128(&maps.rows[kv], cache, width, static_cast<uint64_t>(p.num_slots), width * 2, 64, 1);
        if (err == B200_OK && maps.whole_pages) err = make_kv_groups_tmap(&maps.page[kv], cache, p.num_slots, p.kv_heads, maps.kpc);
        if (err == B200_OK && maps.whole_tiles) err = make_kv_groups_tmap(&maps.tile[kv], cache, p.num_slots, p.kv_heads, kTile);
        if (err != B200_OK) return err;
    }
    const int smem = kSmemBytes + 1024;
    B200_CHECK_CUDA(cudaFuncSetAttribute(shared_prefix_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    B200_CHECK_CUDA(launch_kernel(shared_prefix_tc_kernel, dim3(p.ctas), dim3(kThreads), smem, stream, dim3(1, 1, 1), maps, p));
    return B200_OK;
}

}  // namespace b200
