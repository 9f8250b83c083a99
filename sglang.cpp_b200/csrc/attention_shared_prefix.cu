// Attention of a batch whose requests share long prefixes: the keys and values of a prefix are read once for all query rows of
// its group, a request's own keys for its own rows, and the parts are joined by their softmax statistics.
//
// For query row r (token i of request b, head h; limit = len_b - rows_b + i) and a set of keys K
//     m = max s_j,   l = sum 2^(s_j - m),   o = sum 2^(s_j - m) v_j     over j in K, j <= limit,   s_j = scale log2(e) q . k_j
// and the parts of a row join exactly: M = max m, out = sum 2^(m - M) o / sum 2^(m - M) l.  Everything up to the output is fp32 but
// the probabilities, which are rounded to bf16 as the other attention kernels here do (their products run on the tensor cores).
//
// Rows kernel (bound by HBM): a unit is a group's prefix or what a request has of its own; its rows are (token, head of the KV
// head's group) pairs, in tiles of 16.  The stages of all tiles of all units form one sequence that is cut into equal
// contiguous runs, one per CTA, from the lengths on the device: no host plan, so a captured call follows new lengths.  A stage is
// 128 (key, KV head) rows of K and of V, copied by 3-D TMA boxes of whole pages; eight warps each own 16 keys of one KV head in it
// and multiply with mma.sync.
#include "common.cuh"
#include "kernels.h"
#include "shared_prefix.cuh"
#include "tensormap.cuh"

namespace b200 {
namespace {

constexpr int kD = 128;
constexpr int kConsumerWarps = 8;
constexpr int kThreads = (kConsumerWarps + 1) * 32;
constexpr int kStageRows = 128;
constexpr uint32_t kHalfBytes = kStageRows * 128;    // 64 of the 128 elements of every row
constexpr uint32_t kStageBytes = 4 * kHalfBytes;     // K lo, K hi, V lo, V hi
constexpr int kStages = 3;
constexpr int kSlotTab = 1024;
constexpr int RT = 16;                               // query rows of a tile
constexpr int kMinStagesPerCta = 2;
constexpr int kMergeWarps = 4;
constexpr int kTcRows = 32;
constexpr int kNoLimit = 0x3fffffff;
constexpr int kMaxUnits = 2 * kSharedMaxBatch;

struct Unit {
    int tok0, ntok;    // query tokens
    int lo, hi;        // keys [lo, hi) ...
    int start;         // ... read from here: the beginning of lo's copy
    int limit0;        // token i sees keys up to limit0 + i
    int table;         // page-table row
};

struct Item {
    Unit unit;
    int tile, s_begin, s_end, slot;
    bool reread;       // other tiles of rows read the same keys
};

// Values of keys behind limit0 that hold an infinity or NaN: weight times value for the rows that see the key, then zeros in
// the key's place.  Weights x and sums o as the products' registers hold them.
template <typename Addr>
__device__ __forceinline__ void add_odd_values(uint32_t base, int key0, int valid, int limit0, const int (&limit)[2],
                                               const float (&x)[8], float (&o)[16][4], const Addr& value_addr) {
    const int lane = threadIdx.x & 31, t = lane & 3;
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
        for (int rr = 0; rr < 2; ++rr) {
            const float even = (j & 8) ? x[4 + 2 * rr] : x[2 * rr], next = (j & 8) ? x[5 + 2 * rr] : x[1 + 2 * rr];
            const float w = round_bf16(__shfl_sync(0xffffffffu, (j & 1) ? next : even, (lane & ~3) | (j & 7) >> 1));
            if (key0 + j <= limit[rr]) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    uint32_t v;
                    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(value_addr(base, j, i) + 4u * t));
                    o[i][2 * rr] += w * bf16_lo(v);
                    o[i][2 * rr + 1] += w * bf16_hi(v);
                }
            }
            __syncwarp();
        }
        if (lane < 16) asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(value_addr(base, j, lane)), "r"(0u) : "memory");
    }
    fence_proxy_async_smem();
    __syncwarp();
}

__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                          const SharedPrefixParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kStages];
    __shared__ __align__(8) uint64_t empty_bar[kStages];
    __shared__ int s_stage[kMaxUnits + 1], s_tile[kMaxUnits + 1];
    __shared__ int s_bound[kSharedMaxBatch + 1], s_prefix[kSharedMaxBatch];
    __shared__ int s_slot_tab[kSlotTab];
    __shared__ int2 s_warp[kThreads / 32];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int Hkv = p.kv_heads, G = p.group, SK = p.stage_keys;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&full_bar[s]), 1);
            mbar_init(smem_u32(&empty_bar[s]), kConsumerWarps);
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
    }
    // Behind the tensor-core kernel nothing here waits for what it writes, and what came before it is complete: it has waited.  The
    // wait is made up for at the end, since the kernel that joins the parts waits for this one alone.
    if (!p.after_tc) pdl_wait_prior();
    pdl_launch_dependents();

    // ---- units, tiles and stages ----
    shared_prefixes(p, s_bound, s_prefix);
    auto unit_of = [&](int u) {
        Unit x;
        int b = u - p.groups;
        if (b < 0) {
            b = min(s_bound[u], p.batch - 1);
            x.tok0 = shared_row(p, s_bound[u]);
            x.ntok = max(shared_row(p, s_bound[u + 1]) - x.tok0, 0);
            x.lo = 0;
            x.hi = s_prefix[u];
            x.limit0 = kNoLimit;
        } else {
            const int g = shared_group_of(s_bound, p.groups, b);
            const int len = shared_len(p, b);
            x.tok0 = shared_row(p, b);
            x.ntok = max(shared_row(p, b + 1) - x.tok0, 0);
            x.lo = g >= 0 ? s_prefix[g] : 0;
            x.hi = len;
            x.limit0 = len - x.ntok;
        }
        x.table = p.table_idx[b];
        x.start = x.lo & ~(p.kpc - 1);
        return x;
    };
    const int U = p.groups + p.batch;
    {
        auto size_of = [&](int u) {
            const Unit x = unit_of(u);
            const int stages = (max(x.hi - x.start, 0) + SK - 1) / SK, tiles = stages > 0 && (u >= p.groups || x.ntok * G <= p.tc_rows) ? (x.ntok * G + RT - 1) / RT : 0;
            return make_int2(tiles * stages, tiles);
        };
        const int each = (U + kThreads - 1) / kThreads;
        const int u0 = min(static_cast<int>(threadIdx.x) * each, U), u1 = min(u0 + each, U);
        int2 mine = make_int2(0, 0);
        for (int u = u0; u < u1; ++u) {
            const int2 n = size_of(u);
            mine.x += n.x;
            mine.y += n.y;
        }
        int2 incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, incl.x, o), b = __shfl_up_sync(0xffffffffu, incl.y, o);
            if (lane >= o) {
                incl.x += a;
                incl.y += b;
            }
        }
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        int2 at = make_int2(incl.x - mine.x, incl.y - mine.y);
        for (int w = 0; w < warp; ++w) {
            at.x += s_warp[w].x;
            at.y += s_warp[w].y;
        }
        for (int u = u0; u < u1; ++u) {
            s_stage[u] = at.x;
            s_tile[u] = at.y;
            const int2 n = size_of(u);
            at.x += n.x;
            at.y += n.y;
        }
        if (threadIdx.x == kThreads - 1) {
            s_stage[U] = at.x;
            s_tile[U] = at.y;
        }
    }
    __syncthreads();
    const int total = s_stage[U];
    const int per = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), kMinStagesPerCta);
    // Partial results lie at tile + CTA.  The host has made room for `tokens` rows; an index array whose requests overlap asks for
    // more, and is reported instead.
    const bool fits = static_cast<int>(gridDim.x) + s_tile[U] <= p.max_slots;
    if (blockIdx.x == 0) {
        for (int u = threadIdx.x; u <= U; u += kThreads) {
            p.plan.stage[u] = s_stage[u];
            p.plan.tile[u] = s_tile[u];
        }
        for (int g = threadIdx.x; g < p.groups; g += kThreads) p.plan.prefix[g] = s_prefix[g];
        for (int b = threadIdx.x; b < p.batch; b += kThreads) p.plan.group_of[b] = shared_group_of(s_bound, p.groups, b);
        if (threadIdx.x == 0) {
            p.plan.per[0] = fits ? per : 0;
            if (!fits) atomicExch(&p.status[kStatusBadIndex], p.tokens + 1);
        }
    }
    if (!fits) {
        if (p.after_tc) pdl_wait_prior();
        return;
    }
    const int g_begin = min(static_cast<int>(blockIdx.x) * per, total);
    const int g_end = min(total, g_begin + per);

    // The item that starts at stage gpos < g_end of the sequence.
    auto locate = [&](int gpos) {
        int lo = 0, hi = U;   // the last unit that does not begin behind gpos (units without stages are skipped)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_stage[mid] <= gpos) lo = mid; else hi = mid;
        }
        Item it;
        it.unit = unit_of(lo);
        const int off = gpos - s_stage[lo], tiles = s_tile[lo + 1] - s_tile[lo];
        const int stages = (s_stage[lo + 1] - s_stage[lo]) / tiles;
        it.tile = off / stages;
        it.s_begin = off - it.tile * stages;
        it.s_end = min(stages, it.s_begin + (g_end - gpos));
        it.slot = s_tile[lo] + it.tile + static_cast<int>(blockIdx.x);
        it.reread = tiles > 1;
        return it;
    };
    uint32_t it_count = 0;
    bool failed = false;

    if (warp == kConsumerWarps) {
        // ================= producer =================
        const uint32_t copy_bytes = static_cast<uint32_t>(p.kpc) * Hkv * 128u;
        const uint64_t once = l2_policy_evict_first();
        for (int gpos = g_begin; gpos < g_end && !failed;) {
            const Item it = locate(gpos);
            gpos += it.s_end - it.s_begin;
            const int32_t* row = p.page_table + static_cast<int64_t>(it.unit.table) * p.pt_stride;
            const int first_key = it.unit.start + it.s_begin * SK;
            const int copies = (min(it.unit.hi, it.unit.start + it.s_end * SK) - first_key + p.kpc - 1) / p.kpc;
            __syncwarp();
            for (int c = lane; c < min(copies, kSlotTab); c += 32) s_slot_tab[c] = row[first_key + c * p.kpc];
            __syncwarp();
            for (int st = it.s_begin; st < it.s_end; ++st, ++it_count) {
                const uint32_t slot = it_count % kStages;
                if (!mbar_wait_warp(smem_u32(&empty_bar[slot]), ((it_count / kStages) & 1u) ^ 1u, p.status, 221)) {
                    failed = true;
                    break;
                }
                const int k0 = it.unit.start + st * SK;
                const int n = (min(SK, it.unit.hi - k0) + p.kpc - 1) / p.kpc;
                const uint32_t bar = smem_u32(&full_bar[slot]);
                if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(n) * 4u * copy_bytes);
                __syncwarp();
                const uint32_t base = smem_base + slot * kStageBytes;
                for (int ci = lane; ci < n * 4; ci += 32) {
                    const int copy = ci >> 2, which = ci & 3;
                    const int tab = (k0 - first_key) / p.kpc + copy;
                    int64_t sl = tab < kSlotTab ? s_slot_tab[tab] : row[k0 + copy * p.kpc];
                    if (sl < 0 || sl + p.kpc > p.num_slots) {
                        atomicExch(&p.status[kStatusBadIndex], static_cast<int>(sl) + 1);
                        sl = 0;
                    }
                    const uint32_t dst = base + which * kHalfBytes + copy * copy_bytes;
                    const void* map = which < 2 ? &tmap_k : &tmap_v;
                    if (it.reread) tma_load_3d(dst, map, (which & 1) * 64, static_cast<int>(sl), 0, bar);
                    else tma_load_3d_hint(dst, map, (which & 1) * 64, static_cast<int>(sl), 0, bar, once);
                }
            }
        }
        if (p.after_tc) pdl_wait_prior();
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
    auto value_addr = [&](uint32_t base, int j, int c16) { return swz128(base + (2 + (c16 >> 3)) * kHalfBytes + tile_row(j) * 128u, c16 & 7); };
    for (int gpos = g_begin; gpos < g_end;) {
        const Item it = locate(gpos);
        gpos += it.s_end - it.s_begin;
        const Unit& un = it.unit;
        const int rows = un.ntok * G - it.tile * RT;   // of this tile, at least one
        // Query fragments and the last key that a row sees.
        uint32_t qa[8][4];
        int limit[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            const bool there = rr * 8 + g < rows;
            const int r = it.tile * RT + rr * 8 + g, tok = there ? r / G : 0;
            limit[rr] = there ? min(un.limit0 + tok, un.hi - 1) : -1;
            const __nv_bfloat16* q = p.q + (un.tok0 + tok) * p.q_st + (h * G + (there ? r - tok * G : 0)) * p.q_sh;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                qa[ks][rr] = there ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 2 * t) : 0u;
                qa[ks][2 + rr] = there ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + 2 * t + 8) : 0u;
            }
        }
        float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[16][4];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        for (int st = it.s_begin; st < it.s_end; ++st, ++it_count) {
            const uint32_t slot = it_count % kStages;
            if (!failed && !mbar_wait_warp(smem_u32(&full_bar[slot]), (it_count / kStages) & 1u, p.status, 222)) failed = true;
            const int key0 = un.start + st * SK + kg * 16;
            const int skip = un.lo - key0, valid = un.hi - key0;   // keys [skip, valid) of the 16 belong to the unit
            if (!failed && valid > 0 && skip < 16) {
                const uint32_t base = smem_base + slot * kStageBytes;
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
                // ---- S = Q K^T ----
                float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
                {
                    const uint32_t rowoff = tile_row((mi >> 1) * 8 + r8) * 128u;
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        const int c16 = ks * 2 + (mi & 1);
                        uint32_t b00, b01, b10, b11;
                        ldmatrix_x4(swz128(base + (c16 >> 3) * kHalfBytes + rowoff, c16 & 7), b00, b01, b10, b11);
                        mma_bf16_16816(s0, qa[ks], b00, b01);
                        mma_bf16_16816(s1, qa[ks], b10, b11);
                    }
                }
                // ---- softmax, with the running maximum ----
                float x[8], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key0 + (e >> 2) * 8 + 2 * t + (e & 1), rr = e >> 1 & 1;
                    x[e] = key >= un.lo && key <= limit[rr] ? (e < 4 ? s0[e] : s1[e - 4]) * p.scale_log2 : -INFINITY;
                    top[rr] = fmaxf(top[rr], x[e]);
                }
#pragma unroll
                for (int rr = 0; rr < 2; ++rr) {
                    top[rr] = fmaxf(top[rr], __shfl_xor_sync(0xffffffffu, top[rr], 1));
                    top[rr] = fmaxf(top[rr], __shfl_xor_sync(0xffffffffu, top[rr], 2));
                    const float now = fmaxf(mx[rr], top[rr]);
                    const float ref = now == -INFINITY ? 0.f : now;   // no key seen yet: every weight is 2^-inf = 0
                    const float shrink = exp2f(mx[rr] - ref);
                    mx[rr] = now;
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if ((e >> 1 & 1) == rr) {
                            x[e] = exp2f(x[e] - ref);
                            sum += x[e];
                        }
                    l[rr] = l[rr] * shrink + sum;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        o[i][2 * rr] *= shrink;
                        o[i][2 * rr + 1] *= shrink;
                    }
                }
                const uint32_t pa[4] = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
                // Keys that later rows see and earlier ones do not: an infinity or NaN in their values must not reach the earlier
                // rows as 0 times it.  Such keys are added by hand for the rows that see them.
                if (un.ntok > 1 && un.limit0 + 1 < key0 + min(valid, 16)) add_odd_values(base, key0, valid, un.limit0, limit, x, o, value_addr);
                // ---- O += P V ----
                {
                    const int j = (mi & 1) * 8 + r8;
#pragma unroll
                    for (int np = 0; np < 8; ++np) {
                        uint32_t v0, v1, v2, v3;
                        ldmatrix_x4_trans(value_addr(base, j, np * 2 + (mi >> 1)), v0, v1, v2, v3);
                        mma_bf16_16816(o[2 * np], pa, v0, v1);
                        mma_bf16_16816(o[2 * np + 1], pa, v2, v3);
                    }
                }
            }
            mbar_release_stage(smem_u32(&empty_bar[slot]), lane);
        }
        // ---- the part's statistics and sums ----
        const int64_t part = (static_cast<int64_t>(it.slot) * KG + kg) * Hkv + h;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            float sum = l[rr];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if (rr * 8 + g >= rows) continue;
            const int64_t at = part * RT + rr * 8 + g;
            float* dst = p.ws_o + at * kD + 2 * t;
#pragma unroll
            for (int i = 0; i < 16; ++i) *reinterpret_cast<float2*>(dst + i * 8) = make_float2(o[i][2 * rr], o[i][2 * rr + 1]);
            if (t == 0) *reinterpret_cast<float2*>(p.ws_ml + at * 2) = make_float2(mx[rr], sum);
        }
    }
    if (p.after_tc) pdl_wait_prior();
}

// Parts of a row: `count` of them, the first at `first`, `step` rows apart.
struct Parts {
    int64_t first, step;
    int count;
};

// Joins the parts of every row.  One warp per (token, head), tokens of a request in turn; rows that no request owns stay as they
// were.  Bound by the trips to L2: lengths, statistics, sums.
__global__ void __launch_bounds__(kMergeWarps * 32)
shared_prefix_merge_kernel(const SharedPrefixParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = static_cast<int>(blockIdx.x) * kMergeWarps + warp;
    const int b = static_cast<int>(blockIdx.y);
    pdl_launch_dependents();
    pdl_wait_prior();
    const int per = p.plan.per[0];
    const int tc_per = p.after_tc ? p.plan.per[1] : 0;
    if (head >= p.q_heads || per <= 0 || (p.after_tc && tc_per <= 0)) return;
    const int h = head / p.group, KG = kConsumerWarps / p.kv_heads;
    const int row0 = shared_row(p, b), row1 = shared_row(p, b + 1);
    const int grp = p.plan.group_of[b];
    const int own_first = p.plan.stage[p.groups + b], own_stages = p.plan.stage[p.groups + b + 1] - own_first;
    const int own_tile = p.plan.tile[p.groups + b], own_tiles = p.plan.tile[p.groups + b + 1] - own_tile;
    int pre_first = 0, pre_stages = 0, pre_tile = 0, pre_tiles = 0, pre_row = 0;
    int tc_first = 0, tc_unit = 0, tc_units = 0, tc_tiles = 0, tc_cta = 0;
    const bool chunked = p.after_tc && p.plan.per[2] != 0;
    if (grp >= 0) {
        if (p.after_tc) {
            tc_first = p.plan.tc_first[grp];
            tc_unit = p.plan.tc_unit[grp];
            tc_cta = p.plan.tc_cta[grp];
            tc_units = p.plan.tc_unit[grp + 1] - tc_unit;
            tc_tiles = tc_units > 0 ? (p.plan.tc_first[grp + 1] - tc_first) / tc_units : 0;
        }
        pre_first = p.plan.stage[grp];
        pre_stages = p.plan.stage[grp + 1] - pre_first;
        pre_tile = p.plan.tile[grp];
        pre_tiles = p.plan.tile[grp + 1] - pre_tile;
        pre_row = shared_row(p, shared_bound(p, grp));
    }
    auto parts_of = [&](int first, int stages, int tile, int tiles, int r) {
        Parts x = {0, static_cast<int64_t>(p.kv_heads) * RT, 0};
        const int mine = r / RT;
        if (r < 0 || mine >= tiles) return x;
        const int n = stages / tiles, from = first + mine * n, c0 = from / per;
        x.count = ((from + n - 1) / per - c0 + 1) * KG;
        x.first = (static_cast<int64_t>(tile + mine + c0) * KG * p.kv_heads + h) * RT + r % RT;
        return x;
    };
    for (int tok = row0 + static_cast<int>(blockIdx.z); tok < row1; tok += static_cast<int>(gridDim.z)) {
        const int hh = head - h * p.group;
        Parts pre = parts_of(pre_first, pre_stages, pre_tile, pre_tiles, (tok - pre_row) * p.group + hh);
        const Parts own = parts_of(own_first, own_stages, own_tile, own_tiles, (tok - row0) * p.group + hh);
        const int t = tok - pre_row, half = 128 / p.group, block = t / (2 * half);   // tokens of a chain
        if (tc_units > 0 && t >= 0 && block < tc_units / p.kv_heads) {
            const int unit = h * (tc_units / p.kv_heads) + block, from = tc_first + unit * tc_tiles;
            const int in_block = t - block * 2 * half, chain = in_block >= half ? 1 : 0;
            const int chunks = (tc_tiles + tc_per - 1) / tc_per;
            const int c0 = chunked ? tc_cta + unit * chunks : from / tc_per;
            pre.count = chunked ? chunks : (from + tc_tiles - 1) / tc_per - c0 + 1;
            pre.first = p.tc_base + static_cast<int64_t>(tc_unit + unit + c0) * 256 + chain * 128 + (in_block - chain * half) * p.group + hh;
            pre.step = 256;
        }
        const int n = pre.count + own.count;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float M = -INFINITY, L = 0.f;
        for (int base = 0; base < n; base += 32) {
            const int i = base + lane;
            int64_t at = 0;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (i < n) {
                at = i < pre.count ? pre.first + i * pre.step : own.first + (i - pre.count) * own.step;
                ml = __ldcg(reinterpret_cast<const float2*>(p.ws_ml) + at);
            }
            const float Mn = fmaxf(M, warp_max(ml.x));
            const float ref = Mn == -INFINITY ? 0.f : Mn;
            const float shrink = exp2f(M - ref), w = exp2f(ml.x - ref);
            M = Mn;
            L = L * shrink + warp_sum(w * ml.y);
            acc.x *= shrink, acc.y *= shrink, acc.z *= shrink, acc.w *= shrink;
            const int m = min(32, n - base);
#pragma unroll 4
            for (int j = 0; j < m; ++j) {
                const float wj = __shfl_sync(0xffffffffu, w, j);
                const int64_t aj = __shfl_sync(0xffffffffu, at, j);
                const float4 x = __ldcg(reinterpret_cast<const float4*>(p.ws_o + aj * kD) + lane);
                acc.x += x.x * wj, acc.y += x.y * wj, acc.z += x.z * wj, acc.w += x.w * wj;
            }
        }
        const float inv = L > 0.f ? 1.f / L : 0.f;   // a row that sees no key: zeros
        uint2 packed;
        packed.x = pack_bf16(acc.x * inv, acc.y * inv);
        packed.y = pack_bf16(acc.z * inv, acc.w * inv);
        reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(tok) * p.q_heads + head) * kD)[lane] = packed;
    }
}

int64_t round256(int64_t n) { return (n + 255) & ~int64_t(255); }

// Where the pieces of the workspace begin, in bytes.
struct SharedLayout {
    int64_t slots, tc_slots, rows, plan, ml, o, bytes;   // rows: of the rows kernel's parts, ahead of the tensor-core kernel's
};
SharedLayout shared_layout(int64_t tokens, int64_t batch, int64_t groups, int q_heads, int kv_heads) {
    const int64_t rows = tokens * (q_heads / kv_heads), kg = kConsumerWarps / kv_heads;
    SharedLayout x;
    // tiles: at most one more than full ones per unit, and every row is in two units
    x.slots = sm_count() + 2 * (rows / RT) + batch + groups;
    x.rows = x.slots * kg * kv_heads * RT;
    // units of the tensor-core kernel: the same of groups that have more than kTcRows rows
    const int64_t tc_groups = groups < rows / (kTcRows + 1) ? groups : rows / (kTcRows + 1);
    x.tc_slots = rows > kTcRows ? sm_count() + kv_heads * (tokens / (2 * (128 / (q_heads / kv_heads))) + tc_groups) : 0;
    const int64_t part_rows = x.rows + x.tc_slots * 256;
    x.plan = 0;
    x.ml = round256((4 + 2 * (groups + batch + 1) + groups + batch + 3 * (groups + 1)) * 4);
    x.o = x.ml + round256(part_rows * 8);
    x.bytes = x.o + part_rows * kD * 4;
    return x;
}

// Launches of a call after its first may begin before the one ahead of them has ended.
struct FollowOn {
    const bool was = pdl_launches_enabled();
    explicit FollowOn(bool on) { set_pdl_launches(was || on); }
    ~FollowOn() { set_pdl_launches(was); }
};

}  // namespace
}  // namespace b200

extern "C" {

int64_t b200_attention_shared_prefix_workspace_bytes(int max_tokens, int max_batch, int q_heads, int kv_heads, int head_dim) {
    using namespace b200;
    if (max_tokens <= 0 || max_batch <= 0 || max_batch > kSharedMaxBatch || q_heads <= 0 || head_dim != kD) return -1;
    if (kv_heads < 1 || kv_heads > 8 || 8 % kv_heads != 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > 16) return -1;
    if (static_cast<int64_t>(max_tokens) * q_heads > (1 << 28)) return -1;
    return shared_layout(max_tokens, max_batch, max_batch, q_heads, kv_heads).bytes + 256;
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
    B200_CHECK_ARG(a->q_stride_token % 2 == 0 && a->q_stride_head % 2 == 0, "attention_shared_prefix: q strides must be even");
    B200_CHECK_ARG(a->num_slots > 0 && a->num_slots <= 0x7fffffff, "attention_shared_prefix: num_slots must be in [1, 2^31)");
    B200_CHECK_ARG(a->page_table_stride > 0 && a->page_table_stride <= (1 << 29),
                   "attention_shared_prefix: page_table_stride must be in [1, 2^29]");
    B200_CHECK_ARG(a->sm_scale > 0.f && a->sm_scale <= 1e30f, "attention_shared_prefix: sm_scale must be a positive number");
    B200_CHECK_ARG(static_cast<int64_t>(a->tokens) * a->q_heads <= (1 << 28), "attention_shared_prefix: too many query rows");
    if (a->batch == 0 || a->tokens == 0) return B200_OK;
    B200_CHECK_ARG(a->out && a->q && a->k_cache && a->v_cache && a->page_table && a->table_idx && a->seq_lens && a->qo_indptr &&
                       a->workspace && (a->groups == 0 || (a->group_indptr && a->prefix_lens)),
                   "attention_shared_prefix: NULL tensor");
    B200_CHECK_ARG(reinterpret_cast<uintptr_t>(a->out) % 8 == 0 && reinterpret_cast<uintptr_t>(a->q) % 4 == 0,
                   "attention_shared_prefix: out must be 8-byte and q 4-byte aligned");
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
    p.kpc = a->page_size < p.stage_keys ? a->page_size : p.stage_keys;
    p.num_slots = a->num_slots;
    p.scale_log2 = a->sm_scale * 1.4426950408889634f;
    p.status = status;
    const SharedLayout x = shared_layout(a->tokens, a->batch, a->groups, a->q_heads, a->kv_heads);
    if (a->workspace_bytes < x.bytes + 256) {
        set_last_error("attention_shared_prefix: workspace of %lld bytes is too small (need %lld)",
                       static_cast<long long>(a->workspace_bytes), static_cast<long long>(x.bytes + 256));
        return B200_ERR_INVALID_ARGUMENT;
    }
    uint8_t* ws = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(a->workspace) + 255) & ~uintptr_t(255));
    int* ints = reinterpret_cast<int*>(ws + x.plan);
    p.plan.per = ints;
    p.plan.stage = ints + 4;
    p.plan.tile = p.plan.stage + a->groups + a->batch + 1;
    p.plan.prefix = p.plan.tile + a->groups + a->batch + 1;
    p.plan.group_of = p.plan.prefix + a->groups;
    p.ws_ml = reinterpret_cast<float*>(ws + x.ml);
    p.ws_o = reinterpret_cast<float*>(ws + x.o);
    p.max_slots = static_cast<int>(x.slots);
    p.plan.tc_first = p.plan.group_of + a->batch;
    p.plan.tc_unit = p.plan.tc_first + a->groups + 1;
    p.plan.tc_cta = p.plan.tc_unit + a->groups + 1;
    // Queries are copied by tensor maps there.
    const bool aligned = reinterpret_cast<uintptr_t>(a->q) % 16 == 0 && a->q_stride_token % 8 == 0 && a->q_stride_head % 8 == 0 &&
                         a->q_stride_token > 0 && a->q_stride_head > 0;
    p.tc_rows = aligned ? kTcRows : 0x7fffffff;
    p.tc_slots = static_cast<int>(x.tc_slots);
    p.tc_base = x.rows;
    // (a group has more rows than that only if all have)
    p.after_tc = a->groups > 0 && static_cast<int64_t>(a->tokens) * p.group > p.tc_rows;
    CUtensorMap tk, tv;
    err = make_kv_tmap(&tk, a->k_cache, a->num_slots, a->kv_heads, a->page_size);
    if (err != B200_OK) return err;
    err = make_kv_tmap(&tv, a->v_cache, a->num_slots, a->kv_heads, a->page_size);
    if (err != B200_OK) return err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int grid = sm_count();
    if (p.after_tc) {
        err = launch_shared_prefix_tc(p, a->k_cache, a->v_cache, a->page_size, s);
        if (err != B200_OK) return err;
    }
    FollowOn follow(p.after_tc);
    const int smem = kStages * kStageBytes + 1024;
    B200_CHECK_CUDA(cudaFuncSetAttribute(shared_prefix_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    B200_CHECK_CUDA(launch_kernel(shared_prefix_rows_kernel, dim3(grid), dim3(kThreads), smem, s, dim3(1, 1, 1), tk, tv, p));
    FollowOn merge(true);
    const int turns = div_ceil(a->tokens, a->batch) < 64 ? div_ceil(a->tokens, a->batch) : 64;
    B200_CHECK_CUDA(launch_kernel(shared_prefix_merge_kernel, dim3(div_ceil(a->q_heads, kMergeWarps), a->batch, turns),
                                  dim3(kMergeWarps * 32), 0, s, dim3(1, 1, 1), p));
    return B200_OK;
}

}  // extern "C"
