// Attention of a batch whose requests share long prefixes: the keys and values of a prefix are read once for all query rows of
// its group, a request's own keys for its own rows, and the parts are joined by their softmax statistics.
//
// For query row r (token i of request b, head h; limit = len_b - rows_b + i) and a set of keys K
//     m = max s_j,   l = sum 2^(s_j - m),   o = sum 2^(s_j - m) v_j     over j in K, j <= limit,   s_j = scale log2(e) q . k_j
// and the parts of a row join exactly: M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.  Everything up to the output is fp32 but
// the probabilities, which are rounded to bf16 as the other attention kernels here do (their products run on the tensor cores).
//
// Rows kernel (bound by HBM): an item is a run of stages of a group's prefix or of what a request has of its own, for a tile of up to
// 8 * NT of its rows, (token, head of the KV head's group) pairs.  Items are cut by shared_prefix_plan.cu; a CTA takes the next one that
// nobody has taken (which CTA does an item changes no result): short ones two ahead, since their description, slots and first copies
// are three trips to memory, long ones with the last copies of the one before, so that late CTAs find some (taken with the first
// copies: 48 drafted requests behind 16001 keys 80 us, so 74.5).  A stage is 128 (key, KV head) rows of K and of V, copied by 3-D TMA
// boxes of whole pages, a warp for each half of K and of V; eight warps each own 16 keys of one KV head in it and multiply with
// mma.sync: S^T = K Q^T and O^T = V^T P^T, so that the rows are the products' short side (eight of them; with the rows on the long side a
// step of one token and two heads per KV head filled 2 of 16).  64 KB of a stage, with all CTAs at work, take one 1.07 us from L2 and
// 1.39 us from memory (7.0 TB/s; copies 6.5), with two eights of rows 1.47; 128 requests of 1 row with up to 2048 keys of their own
// behind 32768 shared ones: 668 MB in 142 us with the tensor-core kernel beside it, 0.72 of the copy bandwidth.
//
// Few launches, no wait between them that is not needed: the kernels are launched early (programmatic dependent launches), the
// rows kernel does not wait for the tensor-core kernel, whose SMs its last CTAs take over, and the merge finds its parts ahead of
// its wait.
#include "common.cuh"
#include "kernels.h"
#include "shared_prefix.cuh"
#include "tensormap.cuh"

namespace b200 {
namespace {

constexpr int kD = 128;
constexpr int kConsumerWarps = 8;
constexpr int kProducerWarps = 4;                    // K lo, K hi, V lo, V hi
constexpr int kThreads = (kConsumerWarps + kProducerWarps) * 32;
constexpr int kStageRows = 128;
constexpr uint32_t kHalfBytes = kStageRows * 128;    // 64 of the 128 elements of every row
constexpr uint32_t kStageBytes = 4 * kHalfBytes;
constexpr uint32_t kItems = 4;                       // places for items that have been taken
constexpr int kSmallPage = 8;                        // pages of fewer slots are copied slot by slot (of 4: 40.7 us, 40.9 by pages)
// Warps of a CTA of the merge, w of them for a row.  (With a warp per row as many as join a row of many parts: 158 requests, two of them
// behind 26298 keys, 97 us with four, 86 with eight, 83 with sixteen, which cost others 2 to 5 percent.)
constexpr int merge_warps(int w) { return w < 2 ? 8 : w; }
// Rows of a group above which its prefix may be the tensor-core kernel's (shared_prefix_plan.cu has the rest of the rule).  Up to 16 the
// rows kernel is no slower: 4 requests of 4 heads per KV head behind 300, 2000 and 32768 keys 14.9, 16.4 and 45.1 us, there 20.5, 20.5
// and 43.1; 16 requests behind 4096 keys 37 and 22.6.
constexpr int kTcRows = 16;

constexpr int kStages = 3;   // in the ring, beside the queries of 8 * NT rows of every KV head
// Values of keys behind limit0 that hold an infinity or NaN: weight times value for the rows that see the key, then zeros in
// the key's place.  Weights x and sums o as the products' registers hold them.
template <int NT, typename Addr>
__device__ __forceinline__ void add_odd_values(uint32_t base, int key0, int valid, int limit0, const int (&limit)[NT][2],
                                               const float (&x)[NT][4], float (&o)[NT][8][4], const Addr& value_addr) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t odd = 0;
    for (int i = lane; i < 16 * 16; i += 32) {
        const int j = i >> 4;
        if (j >= valid || key0 + j <= limit0) continue;
        uint32_t v[4];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(value_addr(base, j, i & 15)));
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if ((v[k] & 0x7f80u) == 0x7f80u || (v[k] & 0x7f800000u) == 0x7f800000u) odd |= 1u << j;
    }
    odd = __reduce_or_sync(0xffffffffu, odd);
    if (odd == 0) return;
#pragma unroll 1
    for (int j = 0; j < 16; ++j) {
        if ((odd >> j & 1) == 0) continue;
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                const float w = round_bf16(__shfl_sync(0xffffffffu, (j & 8) ? x[m][2 + rr] : x[m][rr], (j & 7) << 2 | t));
                if (key0 + j <= limit[m][rr]) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {   // of the values, elements i * 8 + g
                        uint32_t v;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(value_addr(base, j, i) + (g >> 1) * 4u));
                        o[m][i >> 1][(i & 1) * 2 + rr] += w * ((g & 1) ? bf16_hi(v) : bf16_lo(v));
                    }
                }
                __syncwarp();
            }
        if (lane < 16) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(value_addr(base, j, lane)), "r"(0u) : "memory");
    }
    fence_proxy_async_smem();
    __syncwarp();
}
// An 8 x 8 matrix of 16-bit elements, rows to columns.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <int NT, bool SMALL>
__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                          const __grid_constant__ CUtensorMap tmap_q, const SharedPrefixParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kStages];
    __shared__ __align__(8) uint64_t empty_bar[kStages];
    __shared__ __align__(8) uint64_t item_full[kItems], item_empty[kItems], query_full, query_empty;
    __shared__ RowsItem s_item[kItems];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    // Large pages: K lo, K hi, V lo, V hi in swizzled rows of 128 bytes.  Small ones: K and V of a slot in one piece, all heads, 16 bytes
    // further apart than they are long, which spreads eight keys over all banks.
    const uint32_t slot_bytes = static_cast<uint32_t>(p.kv_heads) * kD * 2 + 16;
    const uint32_t values_at = SMALL ? static_cast<uint32_t>(p.stage_keys) * slot_bytes : 2 * kHalfBytes;
    const uint32_t stage_bytes = SMALL ? 2 * values_at : kStageBytes;
    const uint32_t query_base = smem_base + (kStages * stage_bytes + 127u & ~127u);
    const int Hkv = p.kv_heads, G = p.group, SK = p.stage_keys;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), kProducerWarps);
            mbar_init(smem_u32(&empty_bar[s]), kConsumerWarps);
        }
        mbar_init(smem_u32(&query_full), 1);
        mbar_init(smem_u32(&query_empty), kConsumerWarps);
        for (uint32_t i = 0; i < kItems; ++i) {
            mbar_init(smem_u32(&item_full[i]), 1);
            mbar_init(smem_u32(&item_empty[i]), kConsumerWarps + kProducerWarps);
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
        tma_prefetch_desc(&tmap_q);
    }
    __syncthreads();
    // Behind the tensor-core kernel nothing here waits for what that writes, and the plan is complete: it has waited for it.  The wait
    // is made up for at the end, since the kernel that joins the parts waits for this one alone.  (What other kernels wrote is read
    // from L2 here: the plan, the page table, and by copies queries, keys and values.)
    if (!p.with_tc) pdl_wait_prior();
    pdl_launch_dependents();
    // Item number `turn` of this CTA, for the whole warp; a slot of -1 ends it.
    auto get_item = [&](uint32_t turn) {
        RowsItem it;
        it.slot = -1;
        const uint32_t at = turn % kItems;
        if (!mbar_wait_warp(smem_u32(&item_full[at]), turn / kItems & 1u, p.status, 223)) return it;
        it = s_item[at];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&item_empty[at]));
        return it;
    };
    // By one lane of the first producer warp: items are handed on one or two ahead of the one whose copies are made (long and short
    // ones: an item's description, its pages' slots and its first copies are three trips to memory, which short ones do not cover).
    const int count = __ldcg(&p.plan.head->rows_items);
    const uint32_t lead = static_cast<uint32_t>(__ldcg(&p.plan.head->rows_lead));
    auto hand_on = [&](uint32_t turn, int taken) {
        const uint32_t at = turn % kItems;
        RowsItem it;
        it.slot = -1;
        if (taken < count) {
            static_assert(sizeof(RowsItem) % 16 == 0, "read in 16-byte loads");
#pragma unroll
            for (unsigned i = 0; i < sizeof(RowsItem) / 16; ++i)
                reinterpret_cast<int4*>(&it)[i] = __ldcg(reinterpret_cast<const int4*>(p.plan.rows + taken) + i);
        }
        if (!mbar_wait_bounded(smem_u32(&item_empty[at]), (turn / kItems & 1u) ^ 1u, p.status, 224)) return;
        s_item[at] = it;
        mbar_arrive(smem_u32(&item_full[at]));
    };
    uint32_t it_count = 0;
    bool failed = false;

    if (warp >= kConsumerWarps) {
        // ================= producers =================
        const int which = warp - kConsumerWarps;
        const uint32_t copy_bytes = static_cast<uint32_t>(p.kpc) * Hkv * 128u;
        const uint64_t once = l2_policy_evict_first();
        const void* map = which < 2 ? &tmap_k : &tmap_v;
        const bool leads = which == 0 && lane == 0;
        if (leads) {
            const bool first = static_cast<int>(blockIdx.x) < __ldcg(&p.plan.head->rows_first);
            if (first) hand_on(0, static_cast<int>(blockIdx.x));
            for (uint32_t i = first ? 1 : 0; i < lead; ++i) hand_on(i, atomicAdd(&p.plan.head->next, 1));
        }
        __syncwarp();
        auto copies_of = [&](const RowsItem& it, int st) { return (min(SK, it.hi - it.start - st * SK) + p.kpc - 1) / p.kpc; };
        // Pages of fewer than 8 slots: a slot's row of all heads by one plain copy, by two warps for K and two for V, every other key each.
        // (Tensor copies of a slot or two take 17 ns each whatever their size: stages of pages of one slot 2.2 us.  16 bytes per lane,
        // by cp.async: 2.5 us, the instructions that form 4096 addresses.)
        const int span = SMALL ? 1 : p.kpc;   // slots that a table entry stands for here
        const __nv_bfloat16* cache = which < 2 ? p.k_cache : p.v_cache;
        int next[4];   // this lane's slots of a stage's copies, fetched a stage ahead
        auto fetch_slots = [&](const RowsItem& it, int st) {
            const int32_t* row = p.page_table + static_cast<int64_t>(it.table) * p.pt_stride + it.start + st * SK;
            const int n = SMALL ? min(SK, it.hi - it.start - st * SK) : copies_of(it, st);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int copy = c * 32 + lane;
                next[c] = copy < n ? __ldcg(row + copy * span) : 0;
            }
        };
        RowsItem it = get_item(0);
        if (it.slot >= 0) fetch_slots(it, it.s_begin);
        for (uint32_t turn = 0; it.slot >= 0 && !failed; ++turn) {
            if (which == 3) {   // the queries, when the consumers have taken the last item's to registers
                if (!mbar_wait_warp(smem_u32(&query_empty), (turn & 1u) ^ 1u, p.status, 226)) break;
                const uint32_t half = static_cast<uint32_t>(p.row_tokens * p.q_heads) * 128u, bar = smem_u32(&query_full);
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, 2 * half);
                    for (int i = 0; i < 2; ++i)
                        tma_load_3d(query_base + i * (half + 1023u & ~1023u), &tmap_q, i * 64, 0, it.tok0 + it.tile * p.row_tokens, bar);
                }
                __syncwarp();
            }
            RowsItem after;
            after.slot = -1;
            const int take_at = lead > 1 ? it.s_begin : max(it.s_end - 1, it.s_begin);
            for (int st = it.s_begin; st < it.s_end; ++st, ++it_count) {
                const int n = copies_of(it, st);
                int sl[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    sl[c] = next[c];
                    if (sl[c] < 0 || static_cast<int64_t>(sl[c]) + span > p.num_slots) {
                        atomicExch(&p.status[kStatusBadIndex], bad_index_word(sl[c]));
                        sl[c] = 0;
                    }
                }
                if (st + 1 < it.s_end) fetch_slots(it, st + 1);
                const uint32_t slot = it_count % kStages;
                if (!mbar_wait_warp(smem_u32(&empty_bar[slot]), ((it_count / kStages) & 1u) ^ 1u, p.status, 221)) {
                    failed = true;
                    break;
                }
                const uint32_t bar = smem_u32(&full_bar[slot]);
                if (SMALL) {
                    const uint32_t base = smem_base + slot * stage_bytes + (which >> 1) * values_at, bytes = slot_bytes - 16;
                    const int keys = min(SK, it.hi - it.start - st * SK);
                    if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>((keys + 1 - (which & 1)) >> 1) * bytes);
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int key = c * 32 + lane;
                        if (key < keys && (key & 1) == (which & 1))
                            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                             base + static_cast<uint32_t>(key) * slot_bytes),
                                         "l"(cache + static_cast<int64_t>(sl[c]) * Hkv * kD), "r"(bytes), "r"(bar)
                                         : "memory");
                    }
                } else {
                    if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(n) * copy_bytes);
                    __syncwarp();
                    const uint32_t base = smem_base + slot * stage_bytes + which * kHalfBytes;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int copy = c * 32 + lane;
                        if (copy >= n) continue;
                        if (it.reread) tma_load_3d(base + copy * copy_bytes, map, (which & 1) * 64, sl[c], 0, bar);
                        else tma_load_3d_hint(base + copy * copy_bytes, map, (which & 1) * 64, sl[c], 0, bar, once);
                    }
                }
                if (st == take_at) {
                    if (leads) hand_on(turn + lead, atomicAdd(&p.plan.head->next, 1));
                    __syncwarp();
                    after = get_item(turn + 1);
                }
                if (st + 1 == it.s_end && after.slot >= 0) fetch_slots(after, after.s_begin);
            }
            it = after;
        }
        if (p.with_tc) pdl_wait_prior();
        return;
    }

    // ================= consumers =================
    const int h = warp % Hkv, kg = warp / Hkv, KG = kConsumerWarps / Hkv;
    const int g = lane >> 2, t = lane & 3;
    const int mi = lane >> 3, r8 = lane & 7;
    // Row of key j of this warp's 16 inside a half tile: a copy of kpc keys lands as [head][key] rows.
    auto tile_row = [&](int j) -> uint32_t {
        const int js = kg * 16 + j;
        return static_cast<uint32_t>((js & ~(p.kpc - 1)) * Hkv + h * p.kpc + (js & (p.kpc - 1)));
    };
    // 16 bytes of that key and head.
    auto key_addr = [&](uint32_t base, int j, int c16) -> uint32_t {
        if (SMALL) return base + static_cast<uint32_t>(kg * 16 + j) * slot_bytes + static_cast<uint32_t>(h * 16 + c16) * 16u;
        return swz128(base + (c16 >> 3) * kHalfBytes + tile_row(j) * 128u, c16 & 7);
    };
    auto value_addr = [&](uint32_t base, int j, int c16) { return key_addr(base + values_at, j, c16); };
    const int QT = p.row_tokens;   // query tokens of a row tile
    // Queries lie as [token][head] in shared memory: the rows of this lane's addresses (row r8 of each eight), and the tokens of its
    // products' columns.
    uint32_t query_row[NT];
    int row_tok[NT][2];
#pragma unroll
    for (int m = 0; m < NT; ++m) {
        const int r = m * 8 + r8, tok = min(r / G, QT - 1);
        query_row[m] = query_base + static_cast<uint32_t>(tok * p.q_heads + h * G + min(r - tok * G, G - 1)) * 128u;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) row_tok[m][rr] = (m * 8 + 2 * t + rr) / G;
    }
    const uint32_t query_half = static_cast<uint32_t>(QT * p.q_heads + 7 & ~7) * 128u;
    for (uint32_t turn = 0;; ++turn) {
        const RowsItem un = get_item(turn);
        if (un.slot < 0) break;
        const int rows = min(un.ntok - un.tile * QT, QT) * G;   // of this tile, at least one
        // Query fragments (columns are rows of the tile), and the last key that each of this lane's rows sees.
        uint32_t qb[NT][8][2];
        int limit[NT][2];
        if (!failed && !mbar_wait_warp(smem_u32(&query_full), turn & 1u, p.status, 225)) failed = true;
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
            for (int ks = 0; ks < 8; ks += 2) {   // four 8 x 8 matrices: 32 elements of the head dimension
                const int c16 = ks * 2 + mi;
                ldmatrix_x4(swz128(query_row[m] + (c16 >> 3) * query_half, c16 & 7), qb[m][ks][0], qb[m][ks][1], qb[m][ks + 1][0], qb[m][ks + 1][1]);
            }
        mbar_release_stage(smem_u32(&query_empty), lane);
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
            for (int rr = 0; rr < 2; ++rr)
                limit[m][rr] = m * 8 + 2 * t + rr < rows ? min(un.limit0 + un.tile * QT + row_tok[m][rr], un.hi - 1) : -1;
        float mx[NT][2], l[NT][2], o[NT][8][4];
#pragma unroll
        for (int m = 0; m < NT; ++m) {
            mx[m][0] = mx[m][1] = -INFINITY;
            l[m][0] = l[m][1] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[m][i][0] = o[m][i][1] = o[m][i][2] = o[m][i][3] = 0.f;
        }
        for (int st = un.s_begin; st < un.s_end; ++st, ++it_count) {
            const uint32_t slot = it_count % kStages;
            if (!failed && !mbar_wait_warp(smem_u32(&full_bar[slot]), (it_count / kStages) & 1u, p.status, 222)) failed = true;
            const int key0 = un.start + st * SK + kg * 16;
            const int skip = un.lo - key0, valid = un.hi - key0;   // keys [skip, valid) of the 16 belong to the unit
            if (!failed && valid > 0 && skip < 16) {
                const uint32_t base = smem_base + slot * stage_bytes;
                if (valid < 16 || skip > 0) {
                    // Rows outside the unit hold whatever the page (or an earlier stage) has there: 0 * NaN would stay.
                    for (int i = lane; i < 16 * 16; i += 32) {
                        const int j = i >> 4;
                        if (j < valid && j >= skip) continue;
                        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(value_addr(base, j, i & 15)), "r"(0u) : "memory");
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                // ---- S^T = K Q^T: keys g and g + 8, rows 2 t and 2 t + 1 of every eight ----
                float x[NT][4];
#pragma unroll
                for (int m = 0; m < NT; ++m) x[m][0] = x[m][1] = x[m][2] = x[m][3] = 0.f;
                {
                    const int j = (mi & 1) * 8 + r8;
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        uint32_t ka[4];
                        ldmatrix_x4(key_addr(base, j, ks * 2 + (mi >> 1)), ka[0], ka[1], ka[2], ka[3]);
#pragma unroll
                        for (int m = 0; m < NT; ++m) mma_bf16_16816(x[m], ka, qb[m][ks][0], qb[m][ks][1]);
                    }
                }
                // ---- softmax, with the running maximum ----
                uint32_t pb[NT][2];
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    float top[2];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + g + (e >> 1) * 8;
                        x[m][e] = key >= un.lo && key <= limit[m][e & 1] ? x[m][e] * p.scale_log2 : -INFINITY;
                    }
#pragma unroll
                    for (int rr = 0; rr < 2; ++rr) {
                        top[rr] = fmaxf(x[m][rr], x[m][2 + rr]);
#pragma unroll
                        for (int d = 4; d < 32; d *= 2) top[rr] = fmaxf(top[rr], __shfl_xor_sync(0xffffffffu, top[rr], d));
                        const float now = fmaxf(mx[m][rr], top[rr]);
                        const float ref = now == -INFINITY ? 0.f : now;   // no key seen yet: every weight is 2^-inf = 0
                        const float shrink = exp2f(mx[m][rr] - ref);
                        mx[m][rr] = now;
                        x[m][rr] = exp2f(x[m][rr] - ref);
                        x[m][2 + rr] = exp2f(x[m][2 + rr] - ref);
                        l[m][rr] = l[m][rr] * shrink + (x[m][rr] + x[m][2 + rr]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            o[m][i][rr] *= shrink;
                            o[m][i][2 + rr] *= shrink;
                        }
                    }
                    pb[m][0] = transpose_8x8(pack_bf16(x[m][0], x[m][1]));
                    pb[m][1] = transpose_8x8(pack_bf16(x[m][2], x[m][3]));
                }
                // Keys that later rows see and earlier ones do not: an infinity or NaN in their values must not reach the earlier
                // rows as 0 times it.  Such keys are added by hand for the rows that see them.
                if (un.ntok > 1 && un.limit0 + 1 < key0 + min(valid, 16)) add_odd_values<NT>(base, key0, valid, un.limit0, limit, x, o, value_addr);
                // ---- O^T += V^T P^T ----
                {
                    const int j = (mi >> 1) * 8 + r8;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint32_t va[4];
                        ldmatrix_x4_trans(value_addr(base, j, i * 2 + (mi & 1)), va[0], va[1], va[2], va[3]);
#pragma unroll
                        for (int m = 0; m < NT; ++m) mma_bf16_16816(o[m][i], va, pb[m][0], pb[m][1]);
                    }
                }
            }
            mbar_release_stage(smem_u32(&empty_bar[slot]), lane);
        }
        // ---- the part's statistics and sums ----
        const int64_t part = ((static_cast<int64_t>(un.slot) * KG + kg) * Hkv + h) * (8 * NT);
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                float sum = l[m][rr];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const int r = m * 8 + 2 * t + rr;
                if (r >= rows) continue;
                float* dst = p.ws_o + (part + r) * kD + g;
#pragma unroll
                for (int i = 0; i < 16; ++i) dst[i * 8] = o[m][i >> 1][(i & 1) * 2 + rr];
                if (g == 0) *reinterpret_cast<float2*>(p.ws_ml + (part + r) * 2) = make_float2(mx[m][rr], sum);
            }
    }
    if (p.with_tc) pdl_wait_prior();
}

// Parts of a row: `count` of them, the first at `first`, `step` rows apart.
struct Parts {
    int64_t first, step;
    int count;
};

// Where a row's parts are: of the group's prefix, and of the request's own keys.  The plan stands before the parts do: the kernel
// ahead of the merge is launched behind the end of the plan's, and the merge behind that launch.  (Found ahead of the wait: 0.9 us of
// divisions and a trip to L2 while the last parts are formed.)
struct RowParts {
    Parts pre, own;
    bool owned, many;
    __device__ __forceinline__ int64_t at(int i) const { return i < pre.count ? pre.first + i * pre.step : own.first + (i - pre.count) * own.step; }
};
__device__ __forceinline__ RowParts find_parts(const SharedPrefixParams& p, int tok, int head) {
    JoinItem j;
    static_assert(sizeof(JoinItem) % 16 == 0, "read in 16-byte loads");
#pragma unroll
    for (unsigned i = 0; i < sizeof(JoinItem) / 16; ++i)
        reinterpret_cast<int4*>(&j)[i] = __ldcg(reinterpret_cast<const int4*>(p.plan.join + tok) + i);
    const int tc_per = __ldcg(&p.plan.head->tc_per), tc_chunked = __ldcg(&p.plan.head->tc_chunked);
    const int h = head / p.group, hh = head - h * p.group, KG = kConsumerWarps / p.kv_heads;
    auto parts_of = [&](int first, int pieces, int t) {   // of token t of the unit
        const int tile = t / p.row_tokens, r = (t - tile * p.row_tokens) * p.group + hh;
        return Parts{(static_cast<int64_t>(first + tile * pieces) * KG * p.kv_heads + h) * p.tile_rows + r,
                     static_cast<int64_t>(p.kv_heads) * p.tile_rows, pieces * KG};
    };
    const Parts own = parts_of(j.own_first, j.own_pieces, j.own_t);
    const int t = j.pre_t;
    Parts pre = parts_of(j.pre_first, j.pre_pieces, t);
    const int half = kSharedTcTile / p.group, block = t / (2 * half);   // tokens of a chain
    if (block < j.tc_blocks) {
        const int unit = h * j.tc_blocks + block, in_block = t - block * 2 * half, chain = in_block >= half ? 1 : 0;
        const int from = j.tc_first + unit * j.tc_tiles, chunks = (j.tc_tiles + tc_per - 1) / tc_per;
        const int c0 = tc_chunked ? j.tc_cta + unit * chunks : from / tc_per;
        pre.count = tc_chunked ? chunks : (from + j.tc_tiles - 1) / tc_per - c0 + 1;
        pre.first = p.tc_base + static_cast<int64_t>(j.tc_unit + unit + c0) * (2 * kSharedTcTile) + chain * kSharedTcTile +
                    (in_block - chain * half) * p.group + hh;
        pre.step = 2 * kSharedTcTile;
    }
    return RowParts{pre, own, j.owned != 0, j.many != 0};
}

// Joins the parts of a row by W warps, this one those of number `share` and every W-th behind it.  Bound by the trips to L2: where the
// parts are, then their statistics and the first of their sums, then the other sums.
template <int W>
__device__ __forceinline__ void join_row(const SharedPrefixParams& p, int tok, int head, int share, bool waited, float2* s_ml, float4 (*s_acc)[32]) {
    const int lane = threadIdx.x & 31;
    const RowParts parts = find_parts(p, tok, head);
    if (!waited) pdl_wait_prior();   // (by every CTA: what follows this kernel waits for it alone)
    if (!parts.owned) return;
    const int n = parts.pre.count + parts.own.count;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float M = -INFINITY, L = 0.f;
    constexpr int kAhead = 8;   // sums that are requested at a time, the first together with the statistics
    const int mine = (n - share + W - 1) / W;
    for (int base = 0; base < mine; base += 32) {
        const int m = min(32, mine - base);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < m) ml = __ldcg(reinterpret_cast<const float2*>(p.ws_ml) + parts.at((base + lane) * W + share));
        float4 x[kAhead];
        auto fetch = [&](int from) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                x[i] = from + i < m ? __ldcg(reinterpret_cast<const float4*>(p.ws_o + parts.at((base + from + i) * W + share) * kD) + lane)
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        fetch(0);
        const float Mn = fmaxf(M, warp_max(ml.x));
        const float ref = Mn == -INFINITY ? 0.f : Mn;
        const float shrink = exp2f(M - ref), w = exp2f(ml.x - ref);
        M = Mn;
        L = L * shrink + warp_sum(w * ml.y);
        acc.x *= shrink, acc.y *= shrink, acc.z *= shrink, acc.w *= shrink;
        for (int from = 0; from < m; from += kAhead) {
            if (from > 0) fetch(from);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, from + i);
                if (from + i < m) acc.x += x[i].x * wi, acc.y += x[i].y * wi, acc.z += x[i].z * wi, acc.w += x[i].w * wi;
            }
        }
    }
    if (waited) __syncthreads();   // (the last row's have been read)
    s_acc[share][lane] = acc;
    if (lane == 0) s_ml[share] = make_float2(M, L);
    __syncthreads();
    if (share > 0) return;
#pragma unroll
    for (int i = 1; i < W; ++i) M = fmaxf(M, s_ml[i].x);
    const float ref = M == -INFINITY ? 0.f : M;
    L = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float w = exp2f(s_ml[i].x - ref);
        const float4 y = s_acc[i][lane];
        L += w * s_ml[i].y;
        acc.x += y.x * w, acc.y += y.y * w, acc.z += y.z * w, acc.w += y.w * w;
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;   // a row that sees no key: zeros
    uint2 packed;
    packed.x = pack_bf16(acc.x * inv, acc.y * inv);
    packed.y = pack_bf16(acc.z * inv, acc.w * inv);
    reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(tok) * p.q_heads + head) * kD)[lane] = packed;
}

// ... of two rows, neighbouring heads of a token, by half a warp each: 8 elements of the head dimension per lane.  (A warp each: 48 drafted
// requests of 5376 rows 75.5 us, so 72.4; 256 requests behind 50 keys 34.8 and 32.0.)
__device__ __forceinline__ void join_two(const SharedPrefixParams& p, int tok, int pair) {
    const int lane = threadIdx.x & 15, head = pair * 2 + (threadIdx.x >> 4 & 1);
    const RowParts parts = find_parts(p, tok, min(head, p.q_heads - 1));
    pdl_wait_prior();
    if (!parts.owned || parts.many) return;   // (the same for both)
    const int n = parts.pre.count + parts.own.count, most = __reduce_max_sync(0xffffffffu, n);
    float4 acc[2] = {};
    float M = -INFINITY, L = 0.f;
    constexpr int kAhead = 4;
    for (int base = 0; base < most; base += 16) {
        const int m = min(16, n - base);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < m) ml = __ldcg(reinterpret_cast<const float2*>(p.ws_ml) + parts.at(base + lane));
        float4 x[kAhead][2];
        auto fetch = [&](int from) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                x[i][0] = x[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (from + i >= m) continue;
                const float4* src = reinterpret_cast<const float4*>(p.ws_o + parts.at(base + from + i) * kD) + lane;
                x[i][0] = __ldcg(src);
                x[i][1] = __ldcg(src + 16);
            }
        };
        fetch(0);
        float top = ml.x;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float Mn = fmaxf(M, top);
        const float ref = Mn == -INFINITY ? 0.f : Mn;
        const float shrink = exp2f(M - ref), w = exp2f(ml.x - ref);
        M = Mn;
        float sum = w * ml.y;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        L = L * shrink + sum;
#pragma unroll
        for (int e = 0; e < 2; ++e) acc[e].x *= shrink, acc[e].y *= shrink, acc[e].z *= shrink, acc[e].w *= shrink;
        for (int from = 0; from < min(16, most - base); from += kAhead) {
            if (from > 0) fetch(from);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, from + i, 16);
                if (from + i >= m) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    acc[e].x += x[i][e].x * wi, acc[e].y += x[i][e].y * wi, acc[e].z += x[i][e].z * wi, acc[e].w += x[i][e].w * wi;
            }
        }
    }
    if (head >= p.q_heads) return;
    const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        uint2 packed;
        packed.x = pack_bf16(acc[e].x * inv, acc[e].y * inv);
        packed.y = pack_bf16(acc[e].z * inv, acc[e].w * inv);
        reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(tok) * p.q_heads + head) * kD)[lane + e * 16] = packed;
    }
}

// Rows that no request owns stay as they were.  Many rows (W = 1): half a warp each, but those of dozens of parts by the grid's first
// CTAs, a CTA each (with all alike, two requests behind 26298 keys kept 158 others waiting for 60 us).
template <int W>
__global__ void __launch_bounds__(merge_warps(W) * 32)
shared_prefix_merge_kernel(const SharedPrefixParams p, int first_ctas) {
    constexpr int kWarps = merge_warps(W);
    __shared__ float2 s_ml[kWarps];
    __shared__ float4 s_acc[kWarps][32];
    const int warp = threadIdx.x >> 5;
    pdl_launch_dependents();
    if constexpr (W > 1) {
        join_row<W>(p, static_cast<int>(blockIdx.x) / p.q_heads, static_cast<int>(blockIdx.x) % p.q_heads, warp, false, s_ml, s_acc);
    } else {
        const int cta = static_cast<int>(blockIdx.x) - first_ctas, pairs = (p.q_heads + 1) / 2;
        if (cta >= 0) {
            const int id = cta * kWarps + warp, tok = id / pairs;
            if (tok < p.tokens) join_two(p, tok, id - tok * pairs);
            else pdl_wait_prior();
        } else {
            const int rows = __ldcg(&p.plan.head->many) * p.q_heads;
            pdl_wait_prior();
            for (int i = blockIdx.x; i < rows; i += first_ctas)
                join_row<kWarps>(p, __ldcg(p.plan.many + i / p.q_heads), i % p.q_heads, warp, true, s_ml, s_acc);
        }
    }
}

int64_t round256(int64_t n) { return (n + 255) & ~int64_t(255); }

// Eights of rows of a row tile: as few as hold what a request brings on average, or a group whose prefix is read here.  (64 requests of
// 8 rows and up to 1000 keys each: 38.5 us with one, 42.4 with two; of 12 rows: 59.6 and 46.3.)
int row_eights(int64_t tokens, int64_t batch, int64_t groups, int64_t group) {
    int64_t rows = div_ceil64(tokens * group, batch);
    if (groups > 0 && tokens * group <= kTcRows * groups) rows = div_ceil64(tokens * group, groups);
    if (rows < group) rows = group;
    return rows <= 8 ? 1 : 2;
}

// Where the pieces of the workspace begin, in bytes; partial rows ahead of the tensor-core kernel's.
struct SharedLayout {
    int64_t slots, tc_slots, rows, tc_of, rows_items, tc_items, join, many, ml, o, bytes;
};
SharedLayout shared_layout(int64_t tokens, int64_t batch, int64_t groups, int q_heads, int kv_heads, int nt) {
    const int64_t group = q_heads / kv_heads, rows = tokens * group, kg = kConsumerWarps / kv_heads, ctas = sm_count();
    SharedLayout x;
    // row tiles: at most one more than full ones per unit, and every row is in two units; items: one more than full ones per tile
    x.slots = kSharedPieces * ctas + 2 * (tokens / (8 * nt / group)) + batch + groups;
    x.rows = x.slots * kg * kv_heads * 8 * nt;
    // units of the tensor-core kernel: the same of groups that have more than kTcRows rows
    const int64_t tc_groups = groups < rows / (kTcRows + 1) ? groups : rows / (kTcRows + 1);
    x.tc_slots = rows > kTcRows && groups > 0 ? ctas + kv_heads * (tokens / (2 * (kSharedTcTile / group)) + tc_groups) : 0;
    const int64_t part_rows = x.rows + x.tc_slots * (2 * kSharedTcTile);
    x.tc_of = round256(sizeof(PlanHead));
    x.rows_items = x.tc_of + round256(ctas * sizeof(int2));
    x.tc_items = x.rows_items + round256(x.slots * sizeof(RowsItem));
    x.join = x.tc_items + round256(x.tc_slots * sizeof(TcItem));
    x.many = x.join + round256(tokens * sizeof(JoinItem));
    x.ml = x.many + round256(tokens * sizeof(int));
    x.o = x.ml + round256(part_rows * 8);
    x.bytes = x.o + part_rows * kD * 4;
    return x;
}

// Launches of a call after its first may begin before the one ahead of them has ended.
struct FollowOn {
    const bool was = pdl_launches_enabled();
    FollowOn() { set_pdl_launches(true); }
    ~FollowOn() { set_pdl_launches(was); }
};

template <int NT>
int launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq, const SharedPrefixParams& p, cudaStream_t stream) {
    const int stage = kStageBytes + (p.small ? 2 * p.stage_keys * 16 : 0);
    const int smem = (kStages * stage + 127 & ~127) + NT * 8 * p.kv_heads * kD * 2 + 1024;
    auto kernel = p.small ? shared_prefix_rows_kernel<NT, true> : shared_prefix_rows_kernel<NT, false>;
    B200_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    B200_CHECK_CUDA(launch_kernel(kernel, dim3(p.ctas), dim3(kThreads), smem, stream, dim3(1, 1, 1), tk, tv, tq, p));
    return B200_OK;
}

// Warps per row: sixteen as long as there is a row per SM, whose registers hold one such CTA (128 rows of 8 KV heads behind 304, 4096 and
// 32768 keys 13.4, 16.4 and 42.3 us, with four 13.6, 20.7 and 56.1; 160 rows 16.3, 21.0 and 43.0, with four 14.0, 20.4 and 40.0; 256 rows
// 17.7, 22.2 and 44.7, with four 14.2, 18.9 and 40.8).  Four up to three and a half rows per SM (512 rows 18.4, 19.7 and 42.2, with half a
// warp 17.7, 21.1 and 43.7; 64 requests of 16 heads behind 2051 keys 30.8 and 28.8); half a warp for all others.
int launch_merge(const SharedPrefixParams& p, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(p.tokens) * p.q_heads, sms = sm_count();
    const int w = rows <= sms ? 16 : rows * 2 <= sms * 7 ? 4 : 1;
    auto kernel = w == 16 ? shared_prefix_merge_kernel<16> : w == 4 ? shared_prefix_merge_kernel<4> : shared_prefix_merge_kernel<1>;
    const int first = w > 1 ? 0 : sm_count();
    const int64_t ctas = w > 1 ? rows : div_ceil64(static_cast<int64_t>(p.tokens) * div_ceil(p.q_heads, 2), merge_warps(w));
    B200_CHECK_CUDA(launch_kernel(kernel, dim3(first + static_cast<unsigned>(ctas)), dim3(merge_warps(w) * 32), 0, stream, dim3(1, 1, 1), p, first));
    return B200_OK;
}

}  // namespace
}  // namespace b200

extern "C" {

int64_t b200_attention_shared_prefix_workspace_bytes(int max_tokens, int max_batch, int q_heads, int kv_heads, int head_dim) {
    using namespace b200;
    if (max_tokens <= 0 || max_batch <= 0 || max_batch > kSharedMaxBatch || q_heads <= 0 || head_dim != kD) return -1;
    if (kv_heads < 1 || kv_heads > 8 || 8 % kv_heads != 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > 16) return -1;
    if (static_cast<int64_t>(max_tokens) * q_heads > (1 << 28)) return -1;
    int64_t most = 0;
    for (int nt = q_heads / kv_heads <= 8 ? 1 : 2; nt <= 2; ++nt) {
        const int64_t bytes = shared_layout(max_tokens, max_batch, max_batch, q_heads, kv_heads, nt).bytes;
        if (bytes > most) most = bytes;
    }
    return most + 256;
}

int b200_attention_shared_prefix(const b200_shared_prefix_args* a, b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(a != nullptr, "attention_shared_prefix: NULL arguments");
    B200_CHECK_ARG(a->head_dim == kD, "attention_shared_prefix: head_dim must be 128");
    B200_CHECK_ARG(a->tokens >= 0 && a->batch >= 0 && a->batch <= kSharedMaxBatch, "attention_shared_prefix: batch must be in [0, 1024]");
    B200_CHECK_ARG(a->groups >= 0 && a->groups <= a->batch, "attention_shared_prefix: groups must be in [0, batch]");
    B200_CHECK_ARG(a->kv_heads >= 1 && a->kv_heads <= 8 && 8 % a->kv_heads == 0,
                   "attention_shared_prefix: kv_heads (per rank) must be 1, 2, 4 or 8");
    B200_CHECK_ARG(a->q_heads >= 1 && a->q_heads % a->kv_heads == 0 && a->q_heads / a->kv_heads <= 16,
                   "attention_shared_prefix: q_heads must be a multiple of kv_heads with group size <= 16");
    B200_CHECK_ARG(a->page_size >= 1 && (a->page_size & (a->page_size - 1)) == 0,
                   "attention_shared_prefix: page_size must be a power of two");
    B200_CHECK_ARG(a->q_stride_token % 8 == 0 && a->q_stride_head % 8 == 0 && a->q_stride_token > 0 && a->q_stride_head > 0 &&
                       a->q_stride_token < (1ll << 38) && a->q_stride_head < (1ll << 38),
                   "attention_shared_prefix: q strides must be positive multiples of 8");
    B200_CHECK_ARG(a->num_slots > 0 && a->num_slots <= 0x7fffffff, "attention_shared_prefix: num_slots must be in [1, 2^31)");
    B200_CHECK_ARG(a->page_table_stride > 0 && a->page_table_stride <= (1 << 29),
                   "attention_shared_prefix: page_table_stride must be in [1, 2^29]");
    B200_CHECK_ARG(a->sm_scale > 0.f && a->sm_scale <= 1e30f, "attention_shared_prefix: sm_scale must be a positive number");
    B200_CHECK_ARG(static_cast<int64_t>(a->tokens) * a->q_heads <= (1 << 28), "attention_shared_prefix: too many query rows");
    if (a->batch == 0 || a->tokens == 0) return B200_OK;
    B200_CHECK_ARG(a->out && a->q && a->k_cache && a->v_cache && a->page_table && a->table_idx && a->seq_lens && a->qo_indptr &&
                       a->workspace && (a->groups == 0 || (a->group_indptr && a->prefix_lens)),
                   "attention_shared_prefix: NULL tensor");
    B200_CHECK_ARG(reinterpret_cast<uintptr_t>(a->out) % 8 == 0 && reinterpret_cast<uintptr_t>(a->q) % 16 == 0,
                   "attention_shared_prefix: out must be 8-byte and q 16-byte aligned");
    int err = B200_OK;
    int* status = device_status_words(&err);
    if (err != B200_OK) return err;

    SharedPrefixParams p = {};
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.q_st = a->q_stride_token;
    p.q_sh = a->q_stride_head;
    p.page_table = a->page_table;
    p.pt_stride = a->page_table_stride;
    p.table_idx = a->table_idx;
    p.seq_lens = a->seq_lens;
    p.qo_indptr = a->qo_indptr;
    p.group_indptr = a->group_indptr;
    p.prefix_lens = a->prefix_lens;
    p.tokens = a->tokens;
    p.batch = a->batch;
    p.groups = a->groups;
    p.q_heads = a->q_heads;
    p.kv_heads = a->kv_heads;
    p.group = a->q_heads / a->kv_heads;
    p.stage_keys = kStageRows / a->kv_heads;
    p.small = a->page_size < kSmallPage;
    p.kpc = !p.small && a->page_size < p.stage_keys ? a->page_size : p.stage_keys;
    p.align = p.small ? 1 : p.kpc;
    p.k_cache = static_cast<const __nv_bfloat16*>(a->k_cache);
    p.v_cache = static_cast<const __nv_bfloat16*>(a->v_cache);
    p.num_slots = a->num_slots;
    p.scale_log2 = a->sm_scale * 1.4426950408889634f;
    p.status = status;
    const int nt = row_eights(a->tokens, a->batch, a->groups, p.group);
    const SharedLayout x = shared_layout(a->tokens, a->batch, a->groups, a->q_heads, a->kv_heads, nt);
    if (a->workspace_bytes < x.bytes + 256) {
        set_last_error("attention_shared_prefix: workspace of %lld bytes is too small (need %lld)",
                       static_cast<long long>(a->workspace_bytes), static_cast<long long>(x.bytes + 256));
        return B200_ERR_INVALID_ARGUMENT;
    }
    uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(a->workspace) + 255) & ~uintptr_t(255));
    p.plan.head = reinterpret_cast<PlanHead*>(ws);
    p.plan.tc_of = reinterpret_cast<int2*>(ws + x.tc_of);
    p.plan.rows = reinterpret_cast<RowsItem*>(ws + x.rows_items);
    p.plan.tc = reinterpret_cast<TcItem*>(ws + x.tc_items);
    p.plan.join = reinterpret_cast<JoinItem*>(ws + x.join);
    p.plan.many = reinterpret_cast<int*>(ws + x.many);
    p.parts = kConsumerWarps / p.kv_heads;
    p.ws_ml = reinterpret_cast<float*>(ws + x.ml);
    p.ws_o = reinterpret_cast<float*>(ws + x.o);
    p.tc_base = x.rows;
    p.max_slots = static_cast<int>(x.slots);
    p.tc_slots = static_cast<int>(x.tc_slots);
    p.tile_rows = 8 * nt;
    p.row_tokens = p.tile_rows / p.group;
    p.tc_rows = kTcRows;
    // (a group has more rows than that only if all have)
    p.with_tc = a->groups > 0 && static_cast<int64_t>(a->tokens) * p.group > kTcRows;
    p.ctas = sm_count();
    CUtensorMap tk, tv, tq;
    err = make_shared_query_tmap(&tq, p, p.q_heads, p.row_tokens);
    if (err != B200_OK) return err;
    err = make_kv_tmap(&tk, a->k_cache, a->num_slots, a->kv_heads, a->page_size);
    if (err != B200_OK) return err;
    err = make_kv_tmap(&tv, a->v_cache, a->num_slots, a->kv_heads, a->page_size);
    if (err != B200_OK) return err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    err = launch_shared_prefix_plan(p, s);
    if (err != B200_OK) return err;
    FollowOn follow;
    if (p.with_tc) {
        err = launch_shared_prefix_tc(p, a->k_cache, a->v_cache, a->page_size, s);
        if (err != B200_OK) return err;
    }
    err = nt == 1 ? launch_rows<1>(tk, tv, tq, p, s) : launch_rows<2>(tk, tv, tq, p, s);
    if (err != B200_OK) return err;
    return launch_merge(p, s);
}

}  // extern "C"
