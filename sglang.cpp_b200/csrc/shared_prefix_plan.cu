// Attention over a shared prefix: how the work of a call is cut into items (attention_shared_prefix.cu has the formulas).
//
// Lengths are known on the device alone, so that a captured call follows them.  One CTA counts, for every unit, row tiles x stages
// (rows kernel) or KV heads x blocks x key tiles (tensor-core kernel), adds these up over the units, and writes one item after the
// other where the kernels' CTAs find them; they in turn begin with one load.  (Every CTA counting for itself: 2.5 to 4.5 us ahead of
// each of the two kernels, and five dependent loads per item.)
//
// The tensor-core kernel is bound by products and exponentials, the rows kernel by HBM, and a CTA of either fills an SM.  Both
// therefore run at once on different SMs: with chunks of `per` tiles the first takes so many CTAs, the rows kernel's first CTAs begin
// on the SMs left over, and the others where the chunks end.  `per` is chosen for the earliest end by the times measured for a tile, a
// stage and all SMs' stages, and the early CTAs' share of the stages is larger by what they can do in the meantime.
#include "common.cuh"
#include "kernels.h"
#include "shared_prefix.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 1024;
constexpr int kMaxUnits = 2 * kSharedMaxBatch;
constexpr int kMinStages = 2, kMinTiles = 2;   // per CTA
// Nanoseconds: a tile of two chains' rows, one of a single chain's, the rest of a chunk; a stage of a CTA among few, of all at once.
constexpr int kTileTwo = 1650, kTileOne = 850, kChunk = 7000, kStageAlone = 930, kStageAll = 1450;

struct Unit {
    int tok0, ntok, lo, hi, start, limit0, table;
};

__global__ void __launch_bounds__(kThreads)
shared_prefix_plan_kernel(const SharedPrefixParams p) {
    __shared__ int s_bound[kSharedMaxBatch + 1], s_prefix[kSharedMaxBatch];
    __shared__ int s_stage[kMaxUnits + 1], s_tile[kMaxUnits + 1];               // before a unit, in the rows kernel
    __shared__ int s_first[kSharedMaxBatch + 1], s_unit[kSharedMaxBatch + 1];   // tiles and units before a group, in the other
    __shared__ int4 s_warp[kThreads / 32];
    __shared__ PlanHead s_head;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.group, Hkv = p.kv_heads, SK = p.stage_keys, QB = kSharedTcTile / G, U = p.groups + p.batch, ctas = p.ctas;
    pdl_launch_dependents();
    pdl_wait_prior();

    // Bounds hold whatever the arrays say.
    auto row_of = [&](int b) { return min(max(p.qo_indptr[b], 0), p.tokens); };
    auto len_of = [&](int b) { return static_cast<int>(min(static_cast<int64_t>(max(p.seq_lens[b], 0)), p.pt_stride)); };
    auto group_of = [&](int b) {   // -1: none
        if (p.groups == 0 || b < s_bound[0] || b >= s_bound[p.groups]) return -1;
        int lo = 0, hi = p.groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_bound[mid] <= b) lo = mid; else hi = mid;
        }
        return lo;
    };
    // ---- the keys that are read once for a group: those that its caller names, as far as they lie before every query row of its
    //      requests; none for a request that shares with nobody ----
    if (tid <= p.groups) s_bound[tid] = p.groups > 0 ? min(max(p.group_indptr[tid], 0), p.batch) : 0;
    if (tid == 0 && p.groups == kThreads) s_bound[kThreads] = min(max(p.group_indptr[kThreads], 0), p.batch);
    int row = 0, row_end = 0, len = 0;   // of request tid
    if (tid < p.batch) {
        row = row_of(tid);
        row_end = row_of(tid + 1);
        len = len_of(tid);
    }
    const int named = tid < p.groups ? max(p.prefix_lens[tid], 0) : 0;
    __syncthreads();
    if (tid < p.groups) s_prefix[tid] = s_bound[tid + 1] - s_bound[tid] > 1 ? named : 0;
    __syncthreads();
    const int grp = tid < p.batch ? group_of(tid) : -1;
    if (grp >= 0 && row_end > row) atomicMin(&s_prefix[grp], max(len - (row_end - row), 0));
    __syncthreads();

    // ---- sizes, and their sums: x stages, y row tiles; z key tiles, w units of the tensor-core kernel ----
    auto unit_of = [&](int u) {
        Unit x;
        int b = u - p.groups;
        if (b < 0) {
            b = min(s_bound[u], p.batch - 1);
            x.tok0 = row_of(s_bound[u]);
            x.ntok = max(row_of(s_bound[u + 1]) - x.tok0, 0);
            x.lo = 0;
            x.hi = s_prefix[u];
            x.limit0 = 0x3fffffff;
        } else {
            const int g = group_of(b), n = len_of(b);
            x.tok0 = row_of(b);
            x.ntok = max(row_of(b + 1) - x.tok0, 0);
            x.lo = g >= 0 ? s_prefix[g] : 0;
            x.hi = n;
            x.limit0 = n - x.ntok;
        }
        x.table = p.table_idx[b];
        x.start = x.lo & ~(p.kpc - 1);
        return x;
    };
    auto sizes_of = [&](int u) {
        const Unit x = unit_of(u);
        const bool tc = u < p.groups && x.ntok * G > p.tc_rows;
        const int stages = tc ? 0 : (max(x.hi - x.start, 0) + SK - 1) / SK, tiles = stages > 0 ? (x.ntok * G + kSharedRowTile - 1) / kSharedRowTile : 0;
        const int units = tc && x.hi > 0 ? Hkv * ((x.ntok + 2 * QB - 1) / (2 * QB)) : 0;
        return make_int4(tiles * stages, tiles, units * ((x.hi + kSharedTcTile - 1) / kSharedTcTile), units);
    };
    const int each = (U + kThreads - 1) / kThreads, u0 = min(tid * each, U), u1 = min(u0 + each, U);
    int4 n[2];   // at most 2 units per thread
#pragma unroll
    for (int i = 0; i < 2; ++i) n[i] = u0 + i < u1 ? sizes_of(u0 + i) : make_int4(0, 0, 0, 0);
    const int4 mine = make_int4(n[0].x + n[1].x, n[0].y + n[1].y, n[0].z + n[1].z, n[0].w + n[1].w);
    int4 at = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, at.x, o), y = __shfl_up_sync(0xffffffffu, at.y, o);
        const int z = __shfl_up_sync(0xffffffffu, at.z, o), w = __shfl_up_sync(0xffffffffu, at.w, o);
        if (lane >= o) at.x += x, at.y += y, at.z += z, at.w += w;
    }
    if (lane == 31) s_warp[warp] = at;
    __syncthreads();
    at.x -= mine.x, at.y -= mine.y, at.z -= mine.z, at.w -= mine.w;
    {
        int4 before = lane < warp ? s_warp[lane] : make_int4(0, 0, 0, 0);
        at.x += __reduce_add_sync(0xffffffffu, before.x);
        at.y += __reduce_add_sync(0xffffffffu, before.y);
        at.z += __reduce_add_sync(0xffffffffu, before.z);
        at.w += __reduce_add_sync(0xffffffffu, before.w);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = u0 + i;
        if (u < u1) {
            s_stage[u] = at.x;
            s_tile[u] = at.y;
            if (u < p.groups) {
                s_first[u] = at.z;
                s_unit[u] = at.w;
            }
            at.x += n[i].x, at.y += n[i].y, at.z += n[i].z, at.w += n[i].w;
        }
    }
    if (tid == kThreads - 1) {
        s_stage[U] = at.x;
        s_tile[U] = at.y;
        s_first[p.groups] = at.z;
        s_unit[p.groups] = at.w;
    }
    __syncthreads();
    const int stages = s_stage[U], tiles = s_tile[U], tc_tiles = s_first[p.groups], units = s_unit[p.groups];

    // ---- chunks of the tensor-core kernel, and the rows kernel's shares ----
    if (warp == 0) {
        bool two = false;   // does any block take two chains?
        for (int g = lane; g < p.groups; g += 32)
            if (s_unit[g + 1] > s_unit[g] && row_of(s_bound[g + 1]) - row_of(s_bound[g]) > QB) two = true;
        const int tile_ns = __any_sync(0xffffffffu, two) ? kTileTwo : kTileOne;
        PlanHead h = {};
        h.fits = ctas + tiles <= p.max_slots && (units == 0 || ctas + units <= p.tc_slots);
        h.tc_chunked = units > 0 && 2 * units <= ctas;
        int chunks = 0, busy = 0;   // CTAs of the tensor-core kernel, and for how long
        if (h.tc_chunked) {
            // A lane per candidate, from an equal share for every CTA to a CTA per unit.
            int longest = 0;
            for (int g = 0; g < p.groups; ++g)
                if (s_unit[g + 1] > s_unit[g]) longest = max(longest, (s_prefix[g] + kSharedTcTile - 1) / kSharedTcTile);
            const int least = max((tc_tiles + ctas - 1) / ctas, kMinTiles);
            longest = max(longest, least);
            const float ratio = powf(static_cast<float>(longest) / static_cast<float>(least), lane / 31.f);
            const int per = lane == 31 ? longest : min(static_cast<int>(least * ratio + 0.5f), longest);
            int count = 0;
            for (int g = 0; g < p.groups; ++g) {
                const int k = s_unit[g + 1] - s_unit[g];
                if (k > 0) count += k * (((s_prefix[g] + kSharedTcTile - 1) / kSharedTcTile + per - 1) / per);
            }
            const int64_t time = static_cast<int64_t>(per) * tile_ns + kChunk;
            const int64_t done = min(static_cast<int64_t>(ctas - count) * (time / kStageAlone), static_cast<int64_t>(stages));
            int64_t cost = count <= ctas ? time + (stages - done) * kStageAll / ctas : INT64_MAX / 2;
            int best = lane;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const int64_t other = __shfl_xor_sync(0xffffffffu, cost, o);
                const int whose = __shfl_xor_sync(0xffffffffu, best, o);
                if (other < cost || (other == cost && whose < best)) {
                    cost = other;
                    best = whose;
                }
            }
            h.tc_per = __shfl_sync(0xffffffffu, per, best);
            chunks = __shfl_sync(0xffffffffu, count, best);
            busy = static_cast<int>(min(static_cast<int64_t>(h.tc_per) * tile_ns + kChunk, static_cast<int64_t>(1) << 30));
        } else if (units > 0) {
            h.tc_per = max((tc_tiles + ctas - 1) / ctas, kMinTiles);
            chunks = (tc_tiles + h.tc_per - 1) / h.tc_per;
            busy = static_cast<int>(min(static_cast<int64_t>(h.tc_per) * tile_ns + 2 * kChunk, static_cast<int64_t>(1) << 30));
        }
        // stages = early * (late + ahead) + (ctas - early) * late
        h.early = chunks < ctas ? ctas - chunks : 0;
        const int ahead = units > 0 ? busy / kStageAlone : 0;
        const int64_t left = stages - static_cast<int64_t>(h.early) * ahead;
        if (left > 0) {
            h.late_stages = max(static_cast<int>((left + ctas - 1) / ctas), kMinStages);
            h.early_stages = h.late_stages + ahead;
        } else {
            h.early_stages = h.early > 0 ? max((stages + h.early - 1) / h.early, kMinStages) : kMinStages;
            h.late_stages = kMinStages;   // (nothing is left for them)
        }
        if (lane == 0) {
            s_head = h;
            *p.plan.head = h;
            if (!h.fits) atomicExch(&p.status[kStatusBadIndex], p.tokens + 1);
        }
    }
    __syncthreads();
    const PlanHead h = s_head;

    // ---- items of the rows kernel: a thread per CTA ----
    if (tid < ctas) {
        const int64_t early_end = static_cast<int64_t>(h.early) * h.early_stages;
        const int64_t from = tid < h.early ? static_cast<int64_t>(tid) * h.early_stages
                                           : early_end + static_cast<int64_t>(tid - h.early) * h.late_stages;
        const int begin = static_cast<int>(min(from, static_cast<int64_t>(stages)));
        const int end = min(begin + (tid < h.early ? h.early_stages : h.late_stages), stages);
        int2 items = make_int2(0, 0);
        if (h.fits && begin < end) {
            int lo = 0, hi = U;   // the last unit that does not begin behind `begin` (units without stages are skipped)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_stage[mid] <= begin) lo = mid; else hi = mid;
            }
            Unit x = unit_of(lo);
            int per_tile = (s_stage[lo + 1] - s_stage[lo]) / (s_tile[lo + 1] - s_tile[lo]);
            int tile = (begin - s_stage[lo]) / per_tile;
            items = make_int2(s_tile[lo] + tile + tid, s_tile[lo] + tile + tid);
            for (int pos = begin; pos < end;) {
                const int first = s_stage[lo] + tile * per_tile;
                RowsItem it;
                it.tok0 = x.tok0, it.ntok = x.ntok, it.lo = x.lo, it.hi = x.hi, it.start = x.start, it.limit0 = x.limit0, it.table = x.table;
                it.tile = tile;
                it.s_begin = pos - first;
                it.s_end = min(per_tile, end - first);
                it.reread = s_tile[lo + 1] - s_tile[lo] > 1;
                it.pad = 0;
                p.plan.rows[items.y++] = it;
                pos = first + it.s_end;
                if (++tile == s_tile[lo + 1] - s_tile[lo] && pos < end) {
                    do ++lo; while (s_tile[lo + 1] == s_tile[lo]);
                    x = unit_of(lo);
                    per_tile = (s_stage[lo + 1] - s_stage[lo]) / (s_tile[lo + 1] - s_tile[lo]);
                    tile = 0;
                }
            }
        }
        p.plan.rows_of[tid] = items;
    }
    // ---- items of the tensor-core kernel: a thread per CTA, from the other end of the block ----
    const int cta = kThreads - 1 - tid;
    if (p.with_tc && cta < ctas) {
        int begin = 0, end = 0;
        if (h.tc_chunked) {
            int before = 0;
            for (int g = 0; g < p.groups && before <= cta; ++g) {
                const int k = s_unit[g + 1] - s_unit[g];
                if (k == 0) continue;
                const int of_unit = (s_prefix[g] + kSharedTcTile - 1) / kSharedTcTile, chunk = (of_unit + h.tc_per - 1) / h.tc_per;
                if (cta < before + k * chunk) {
                    const int unit = (cta - before) / chunk, t = (cta - before - unit * chunk) * h.tc_per;
                    begin = s_first[g] + unit * of_unit + t;
                    end = s_first[g] + unit * of_unit + min(t + h.tc_per, of_unit);
                    break;
                }
                before += k * chunk;
            }
        } else {
            begin = static_cast<int>(min(static_cast<int64_t>(cta) * h.tc_per, static_cast<int64_t>(tc_tiles)));
            end = min(begin + h.tc_per, tc_tiles);
        }
        int2 items = make_int2(0, 0);
        if (h.fits && begin < end) {
            int lo = 0, hi = p.groups;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_first[mid] <= begin) lo = mid; else hi = mid;
            }
            for (int pos = begin, first_item = 1; pos < end;) {
                while (pos >= s_first[lo + 1]) ++lo;
                const int of_unit = (s_prefix[lo] + kSharedTcTile - 1) / kSharedTcTile, off = pos - s_first[lo], unit = off / of_unit;
                const int blocks = (s_unit[lo + 1] - s_unit[lo]) / Hkv;
                TcItem it;
                it.h = unit / blocks;
                it.tok0 = row_of(s_bound[lo]) + (unit - it.h * blocks) * 2 * QB;
                it.ntok = min(row_of(s_bound[lo + 1]) - it.tok0, 2 * QB);
                it.keys = s_prefix[lo];
                it.t0 = off - unit * of_unit;
                it.t1 = min(of_unit, it.t0 + end - pos);
                it.table = p.table_idx[min(s_bound[lo], p.batch - 1)];
                it.pad = 0;
                const int slot = s_unit[lo] + unit + cta;
                if (first_item) items.x = slot;
                first_item = 0;
                items.y = slot + 1;
                p.plan.tc[slot] = it;
                pos += it.t1 - it.t0;
            }
        }
        p.plan.tc_of[cta] = items;
    }
    // ---- where each request's parts will be ----
    if (tid < p.batch) {
        JoinItem j = {};
        const int u = p.groups + tid;
        j.row0 = row;
        j.row1 = row_end;
        j.own_tile = s_tile[u];
        j.own_tiles = s_tile[u + 1] - s_tile[u];
        j.own_first = s_stage[u];
        j.own_stages = j.own_tiles > 0 ? (s_stage[u + 1] - s_stage[u]) / j.own_tiles : 0;
        if (grp >= 0) {
            j.pre_row0 = row_of(s_bound[grp]);
            j.pre_tile = s_tile[grp];
            j.pre_tiles = s_tile[grp + 1] - s_tile[grp];
            j.pre_first = s_stage[grp];
            j.pre_stages = j.pre_tiles > 0 ? (s_stage[grp + 1] - s_stage[grp]) / j.pre_tiles : 0;
            const int k = s_unit[grp + 1] - s_unit[grp];
            if (k > 0) {
                j.tc_unit = s_unit[grp];
                j.tc_blocks = k / Hkv;
                j.tc_first = s_first[grp];
                j.tc_tiles = (s_prefix[grp] + kSharedTcTile - 1) / kSharedTcTile;
                for (int g = 0; h.tc_chunked && g < grp; ++g) {
                    const int kk = s_unit[g + 1] - s_unit[g];
                    if (kk > 0) j.tc_cta += kk * (((s_prefix[g] + kSharedTcTile - 1) / kSharedTcTile + h.tc_per - 1) / h.tc_per);
                }
            }
        }
        p.plan.join[tid] = j;
    }
}

}  // namespace

int launch_shared_prefix_plan(const SharedPrefixParams& p, cudaStream_t stream) {
    B200_CHECK_CUDA(launch_kernel(shared_prefix_plan_kernel, dim3(1), dim3(kThreads), 0, stream, dim3(1, 1, 1), p));
    return B200_OK;
}

}  // namespace b200
