// Attention over a shared prefix: how the work of a call is cut into items (attention_shared_prefix.cu has the formulas).
//
// Lengths are known on the device alone, so that a captured call follows them.  One CTA, a thread per request and per group (no more
// warps than that takes: 32 of them for 64 requests cost 2 us), counts row tiles and stages (rows kernel) or KV heads x blocks and
// key tiles (tensor-core kernel), adds these up, and writes the items that the kernels begin with one load.  Bound by its trips to memory
// and barriers: 3.5 us for 4 requests, 4.2 for 64, 6 for 48 of 168 rows, 9 for 158 of 474.  (Every CTA counting for itself: 2.5 to
// 4.5 us ahead of each of the two kernels, and five dependent loads per item.)
//
// The tensor-core kernel is bound by products and exponentials, the rows kernel by HBM, and a CTA of either fills an SM.  Both
// therefore run at once on different SMs: with chunks of `per` tiles the first takes so many CTAs, the rows kernel's first CTAs begin
// on the SMs left over, the others where chunks have ended, and each takes the next item that nobody has taken.  `per` is chosen for
// the earliest end by the times measured for a tile, a stage and all SMs' stages.
#include "common.cuh"
#include "kernels.h"
#include "shared_prefix.cuh"

namespace b200 {
namespace {

constexpr int kMaxThreads = 1024, kMinThreads = 256;
static_assert(kMaxThreads >= kSharedMaxBatch, "a thread per request");
constexpr int kMaxUnits = 2 * kSharedMaxBatch;
constexpr int kMinTiles = 2;                   // per item
constexpr int kLarge = 1 << 19;                // stages or tiles of a unit that are added up in 64 bits
// Groups of up to kTcAlways rows are the tensor-core kernel's only where they are that many stages per CTA: 8 requests of 4 heads per KV
// head behind 300 keys (0.5 stages) 18.5 us without and 21.3 with it, behind 4096 (7) 28.7 and 22.6, behind 32768 106 and 46.8.
constexpr int kTcAlways = 32, kTcWorth = 6;
// Microseconds: a tile of two chains' rows, one of a single chain's, one of small pages (128 copies), the rest of a chunk; a stage of a
// CTA among few, and of all at once.
// (kTileSmall as large as kTileOne: 105 requests in pages of four tokens 150 us, so 105.  kTileTwo 1.65 to 1.9 where the memory has
// little else to do; 128 requests behind 32768 keys 145 to 149 us with 1.8, 141 to 146 with 2.0; kStageAlone 1.0 instead 142 to 145.)
constexpr float kTileTwo = 2.0f, kTileOne = 0.85f, kTileSmall = 3.1f, kChunk = 5.f, kStageAlone = 1.2f, kStageAll = 1.45f;

// A warp's sum of numbers that add up to less than 2^54: 32 of 27 bits are a 32-bit sum.
__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
    const uint32_t low = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v) & 0x7ffffffu);
    const uint32_t high = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v >> 27));
    return (static_cast<int64_t>(high) << 27) + low;
}

__global__ void __launch_bounds__(kMaxThreads, 1)
shared_prefix_plan_kernel(const SharedPrefixParams p) {
    __shared__ int s_row[kSharedMaxBatch + 1], s_len[kSharedMaxBatch], s_table[kSharedMaxBatch];
    __shared__ short s_group[kSharedMaxBatch];                                  // of a request, -1: none
    __shared__ int s_bound[kSharedMaxBatch + 1], s_prefix[kSharedMaxBatch];
    __shared__ int s_first[kMaxUnits + 1];                                      // items before a unit, in the rows kernel
    __shared__ int s_tc[kSharedMaxBatch + 1], s_unit[kSharedMaxBatch + 1];      // tiles and units before a group, in the other
    __shared__ short s_pieces[kMaxUnits];                                       // items of a row tile of a unit, in the rows kernel
    __shared__ int s_cta[kSharedMaxBatch + 1];                                  // chunks before a group, in the other
    __shared__ int4 s_warp[32], s_open[32];
    __shared__ int s_per, s_chunks;   // tiles per chunk, chunks
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, threads = static_cast<int>(blockDim.x);
    const int G = p.group, Hkv = p.kv_heads, SK = p.stage_keys, QB = kSharedTcTile / G, QT = p.row_tokens, U = p.groups + p.batch, ctas = p.ctas;
    pdl_launch_dependents();
    pdl_wait_prior();

    // ---- lengths.  Index arrays that decrease, or name rows or requests that there are not, ask for nothing that could be answered ----
    int row = 0, row_end = 0, len = 0, named = 0;
    bool odd = false;
    if (tid < p.batch) {
        row = p.qo_indptr[tid];
        row_end = p.qo_indptr[tid + 1];
        odd = row < 0 || row_end < row || row_end > p.tokens;
        row = min(max(row, 0), p.tokens);
        row_end = min(max(row_end, 0), p.tokens);
        len = static_cast<int>(min(static_cast<int64_t>(max(p.seq_lens[tid], 0)), p.pt_stride));
        s_table[tid] = p.table_idx[tid];
        s_row[tid] = row;
        s_len[tid] = len;
        if (tid == p.batch - 1) s_row[p.batch] = row_end;
    }
    if (tid < p.groups) {
        const int first = p.group_indptr[tid], end = p.group_indptr[tid + 1];
        odd = odd || first < 0 || end < first || end > p.batch;
        s_bound[tid] = min(max(first, 0), p.batch);
        named = max(p.prefix_lens[tid], 0);
        if (tid == p.groups - 1) s_bound[p.groups] = min(max(end, 0), p.batch);
    }
    odd = __syncthreads_or(odd);
    // The keys that are read once for a group: those that its caller names, as far as they lie before every query row of its
    // requests; none for a request that shares with nobody.
    if (tid < p.groups) s_prefix[tid] = s_bound[tid + 1] - s_bound[tid] > 1 ? named : 0;
    int grp = -1;
    if (tid < p.batch && p.groups > 0 && tid >= s_bound[0] && tid < s_bound[p.groups]) {
        int lo = 0, hi = p.groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_bound[mid] <= tid) lo = mid; else hi = mid;
        }
        grp = lo;
    }
    if (tid < p.batch) s_group[tid] = static_cast<short>(grp);
    __syncthreads();
    const int ntok = max(row_end - row, 0);
    if (grp >= 0 && ntok > 0) atomicMin(&s_prefix[grp], max(len - ntok, 0));
    __syncthreads();

    // ---- sizes ----
    auto start_of = [&](int lo) { return lo & ~(p.align - 1); };
    auto stages_of = [&](int lo, int hi) { return (max(hi - start_of(lo), 0) + SK - 1) / SK; };
    // a group's prefix: row tiles and stages of the rows kernel, or units and key tiles of the other; or both ways, where that is
    // still open
    int g_tiles = 0, g_stages = 0, g_units = 0, g_tc = 0;
    bool two = false, open = false;
    if (tid < p.groups && s_prefix[tid] > 0) {
        const int n = max(s_row[s_bound[tid + 1]] - s_row[s_bound[tid]], 0);
        open = n * G > p.tc_rows && n * G <= kTcAlways;
        if (n * G > p.tc_rows) {
            g_units = Hkv * ((n + 2 * QB - 1) / (2 * QB));
            g_tc = (s_prefix[tid] + kSharedTcTile - 1) / kSharedTcTile;
            two = n > QB;
        }
        if (n > 0 && n * G <= kTcAlways) {
            g_tiles = (n + QT - 1) / QT;
            g_stages = stages_of(0, s_prefix[tid]);
        }
    }
    // a request's own keys
    const int lo = grp >= 0 ? s_prefix[grp] : 0;
    int b_stages = 0, b_tiles = 0;
    if (tid < p.batch && ntok > 0 && len > lo) {
        b_stages = stages_of(lo, len);
        b_tiles = (ntok + QT - 1) / QT;
    }
    // sums over all: stages, key tiles, units, longest prefix; what is open apart.  (2048 units of up to kLarge are a 32-bit sum.)
    auto counted = [](int tiles, int each) { return static_cast<int>(min(shared_unit_work(tiles, each), static_cast<int64_t>(kLarge))); };
    const int g_work = counted(g_tiles, g_stages), g_tc_work = counted(g_units, g_tc);
    int4 sum = make_int4((open ? 0 : g_work) + counted(b_tiles, b_stages), open ? 0 : g_tc_work, open ? 0 : g_units, open ? 0 : g_tc);
    int4 also = open ? make_int4(g_work, g_tc_work, g_units, g_tc) : make_int4(0, 0, 0, 0);
    auto add_up = [](int4 v) {
        return make_int4(__reduce_add_sync(0xffffffffu, v.x), __reduce_add_sync(0xffffffffu, v.y), __reduce_add_sync(0xffffffffu, v.z),
                         __reduce_max_sync(0xffffffffu, v.w));
    };
    sum = add_up(sum);
    also = add_up(also);
    if (lane == 0) {
        s_warp[warp] = sum;
        s_open[warp] = also;
    }
    const bool any_two = __syncthreads_or(two);
    sum = add_up(lane < threads >> 5 ? s_warp[lane] : make_int4(0, 0, 0, 0));
    also = add_up(lane < threads >> 5 ? s_open[lane] : make_int4(0, 0, 0, 0));
    const bool by_tc = also.x > kTcWorth * ctas;
    if (open) {
        if (by_tc) g_tiles = g_stages = 0;
        else g_units = g_tc = 0;
    }
    int64_t stages = sum.x + (by_tc ? 0 : also.x), all_tiles = sum.y + (by_tc ? also.y : 0);
    const int units = sum.z + (by_tc ? also.z : 0), longest = by_tc ? max(sum.w, also.w) : sum.w;
    if (stages >= kLarge || all_tiles >= kLarge) {   // (the same in every thread; otherwise no unit has so many)
        __syncthreads();   // (the sums have been read)
        stages = warp_sum64(shared_unit_work(g_tiles, g_stages) + shared_unit_work(b_tiles, b_stages));
        all_tiles = warp_sum64(shared_unit_work(g_units, g_tc));
        longlong2* s_large = reinterpret_cast<longlong2*>(s_open);
        if (lane == 0) s_large[warp] = make_longlong2(stages, all_tiles);
        __syncthreads();
        const longlong2 part = lane < threads >> 5 ? s_large[lane] : make_longlong2(0, 0);
        stages = warp_sum64(part.x);
        all_tiles = warp_sum64(part.y);
    }
    // (Tiles are numbered in 32 bits: so many, a quarter of a minute's work, are refused.)
    const bool countable = all_tiles < 0x40000000;
    const int tc_tiles = countable ? static_cast<int>(all_tiles) : 0;
    const int piece = shared_stages_per_item(stages, ctas);
    const int g_pieces = (g_stages + piece - 1) / piece, b_pieces = (b_stages + piece - 1) / piece;

    // ---- sums over what comes before: x the groups' items, y the requests'; z key tiles, w units ----
    int4 at = make_int4(g_tiles * g_pieces, b_tiles * b_pieces, g_units * g_tc, g_units);
    const int4 mine = at;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, at.x, o), y = __shfl_up_sync(0xffffffffu, at.y, o);
        const int z = __shfl_up_sync(0xffffffffu, at.z, o), w = __shfl_up_sync(0xffffffffu, at.w, o);
        if (lane >= o) at.x += x, at.y += y, at.z += z, at.w += w;
    }
    __syncthreads();   // (the sums have been read)
    if (lane == 31) s_warp[warp] = at;
    __syncthreads();
    const int4 part = lane < threads >> 5 ? s_warp[lane] : make_int4(0, 0, 0, 0);
    const int4 ahead = lane < warp ? part : make_int4(0, 0, 0, 0);
    const int g_items = __reduce_add_sync(0xffffffffu, part.x), items = g_items + __reduce_add_sync(0xffffffffu, part.y);
    at.x += __reduce_add_sync(0xffffffffu, ahead.x) - mine.x;
    at.y += __reduce_add_sync(0xffffffffu, ahead.y) - mine.y + g_items;
    at.z += __reduce_add_sync(0xffffffffu, ahead.z) - mine.z;
    at.w += __reduce_add_sync(0xffffffffu, ahead.w) - mine.w;
    if (tid < p.groups) {
        s_first[tid] = at.x;
        s_tc[tid] = at.z;
        s_unit[tid] = at.w;
        s_pieces[tid] = static_cast<short>(g_pieces);   // (kSharedPieces * ctas and one at most)
    }
    if (tid < p.batch) {
        s_first[p.groups + tid] = at.y;
        s_pieces[p.groups + tid] = static_cast<short>(b_pieces);
    }
    if (tid == 0) {
        s_first[U] = items;
        s_tc[p.groups] = tc_tiles;
        s_unit[p.groups] = units;
    }
    __syncthreads();
    const bool fits = !odd && countable && items <= p.max_slots && (units == 0 || ctas + units <= p.tc_slots);

    // tiles of a unit, and units per KV head, of a group in the tensor-core kernel
    const int kv_shift = 31 - __clz(Hkv);
    auto tiles_of = [&](int g) { return (s_prefix[g] + kSharedTcTile - 1) / kSharedTcTile; };
    auto blocks_of = [&](int g) { return (s_unit[g + 1] - s_unit[g]) >> kv_shift; };

    // ---- chunks of the tensor-core kernel: a lane per candidate, from an equal share for every CTA to a CTA per unit ----
    const bool chunked = units > 0 && 2 * units <= ctas;
    if (warp == 0) {
        const int least = max((tc_tiles + ctas - 1) / ctas, kMinTiles), most = max(longest, least);
        int per = least, chunks = 0;
        if (chunked) {
            per = lane == 31 ? most : min(static_cast<int>(least * exp2f(log2f(static_cast<float>(most) / least) * (lane / 31.f)) + 0.5f), most);
            int count = 0;
            for (int g = 0; g < p.groups; ++g) {
                const int k = s_unit[g + 1] - s_unit[g];
                if (k > 0) count += k * ((tiles_of(g) + per - 1) / per);
            }
            const float time = per * (p.small ? kTileSmall : any_two ? kTileTwo : kTileOne) + kChunk;
            const float left = fmaxf(stages - (ctas - count) * (time * (1.f / kStageAlone)), 0.f);
            float cost = count <= ctas ? time + left * (kStageAll / ctas) : 3e38f;
            int best = lane;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float other = __shfl_xor_sync(0xffffffffu, cost, o);
                const int whose = __shfl_xor_sync(0xffffffffu, best, o);
                if (other < cost || (other == cost && whose < best)) {
                    cost = other;
                    best = whose;
                }
            }
            per = __shfl_sync(0xffffffffu, per, best);
            chunks = __shfl_sync(0xffffffffu, count, best);
            int before = 0;
            for (int base = 0; base < p.groups; base += 32) {
                const int g = base + lane, mine = g < p.groups ? (s_unit[g + 1] - s_unit[g]) * ((tiles_of(g) + per - 1) / per) : 0;
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += x;
                }
                if (g < p.groups) s_cta[g] = before + upto - mine;
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (lane == 0) s_cta[p.groups] = before;
        }
        if (lane == 0) {
            s_per = per;
            s_chunks = chunks;
            PlanHead h = {};
            h.fits = fits;
            h.rows_items = fits ? items : 0;
            // CTAs that find an SM free begin with the item of their own number.
            h.rows_first = chunked || units == 0 ? max(ctas - s_chunks, 0) : 0;
            h.next = min(h.rows_first, h.rows_items);
            h.rows_lead = piece < kSharedLongPiece && items > 2 * ctas ? 2 : 1;
            h.tc_per = per;
            h.tc_chunked = chunked;
            *p.plan.head = h;
            if (!fits) atomicExch(&p.status[kStatusBadIndex], p.tokens + 1);
        }
    }
    // ---- items of the rows kernel (by all warps but that one) ----
    if (warp > 0 && fits) {
        for (int i = tid - 32; i < items; i += threads - 32) {
            int u = 0, hi = U;   // the last unit that does not begin behind item i (units without items are skipped)
            while (hi - u > 1) {
                const int mid = (u + hi) >> 1;
                if (s_first[mid] <= i) u = mid; else hi = mid;
            }
            RowsItem it;
            int b = u - p.groups;
            if (b < 0) {
                b = s_bound[u];
                it.tok0 = s_row[b];
                it.ntok = s_row[s_bound[u + 1]] - it.tok0;
                it.lo = 0;
                it.hi = s_prefix[u];
                it.limit0 = 0x3fffffff;
            } else {
                const int g = s_group[b];
                it.tok0 = s_row[b];
                it.ntok = s_row[b + 1] - it.tok0;
                it.lo = g >= 0 ? s_prefix[g] : 0;
                it.hi = s_len[b];
                it.limit0 = it.hi - it.ntok;
            }
            it.table = s_table[b];
            it.start = start_of(it.lo);
            const int pieces = s_pieces[u], off = i - s_first[u];
            it.tile = off / pieces;
            it.s_begin = (off - it.tile * pieces) * piece;
            it.s_end = min(it.s_begin + piece, stages_of(it.lo, it.hi));
            it.reread = it.ntok > QT;
            it.slot = i;
            p.plan.rows[i] = it;
        }
    }
    __syncthreads();
    const int per = s_per;
    // ---- items of the tensor-core kernel: a thread per CTA, from the end of the block ----
    const int cta = threads - 1 - tid;
    if (p.with_tc && cta < ctas) {
        int begin = 0, end = 0;
        if (chunked) {
            if (cta < s_cta[p.groups]) {
                int g = 0, hi = p.groups;   // the last group that does not begin behind it (those without chunks are skipped)
                while (hi - g > 1) {
                    const int mid = (g + hi) >> 1;
                    if (s_cta[mid] <= cta) g = mid; else hi = mid;
                }
                const int of_unit = tiles_of(g), chunk = (of_unit + per - 1) / per, unit = (cta - s_cta[g]) / chunk;
                const int t = (cta - s_cta[g] - unit * chunk) * per;
                begin = s_tc[g] + unit * of_unit + t;
                end = s_tc[g] + unit * of_unit + min(t + per, of_unit);
            }
        } else if (units > 0) {
            begin = static_cast<int>(min(static_cast<int64_t>(cta) * per, static_cast<int64_t>(tc_tiles)));
            end = min(begin + per, tc_tiles);
        }
        int2 of = make_int2(0, 0);
        if (fits && begin < end) {
            int g = 0, hi = p.groups;
            while (hi - g > 1) {
                const int mid = (g + hi) >> 1;
                if (s_tc[mid] <= begin) g = mid; else hi = mid;
            }
            bool first = true;
            for (int pos = begin; pos < end;) {
                while (pos >= s_tc[g + 1]) ++g;
                const int of_unit = tiles_of(g), off = pos - s_tc[g], unit = off / of_unit;
                TcItem it;
                it.h = unit / blocks_of(g);
                it.tok0 = s_row[s_bound[g]] + (unit - it.h * blocks_of(g)) * 2 * QB;
                it.ntok = min(s_row[s_bound[g + 1]] - it.tok0, 2 * QB);
                it.keys = s_prefix[g];
                it.t0 = off - unit * of_unit;
                it.t1 = min(of_unit, it.t0 + end - pos);
                it.table = s_table[s_bound[g]];
                it.pad = 0;
                const int slot = s_unit[g] + unit + cta;
                if (first) of.x = slot;
                first = false;
                of.y = slot + 1;
                p.plan.tc[slot] = it;
                pos += it.t1 - it.t0;
            }
        }
        p.plan.tc_of[cta] = of;
    }
    // ---- where each row's parts will be ----
    for (int tok = tid; tok < p.tokens; tok += threads) {
        JoinItem j = {};
        if (fits && tok >= s_row[0] && tok < s_row[p.batch]) {
            int b = 0, hi = p.batch;   // the last request that does not begin behind it: the one that owns it
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (s_row[mid] <= tok) b = mid; else hi = mid;
            }
            const int u = p.groups + b, g = s_group[b];
            j.owned = 1;
            j.own_t = tok - s_row[b];
            j.own_first = s_first[u];
            j.own_pieces = s_pieces[u];
            if (g >= 0) {
                j.pre_t = tok - s_row[s_bound[g]];
                if (blocks_of(g) > 0) {
                    j.tc_unit = s_unit[g];
                    j.tc_blocks = blocks_of(g);
                    j.tc_first = s_tc[g];
                    j.tc_tiles = tiles_of(g);
                    if (chunked) j.tc_cta = s_cta[g];
                } else if (s_first[g + 1] > s_first[g]) {
                    j.pre_first = s_first[g];
                    j.pre_pieces = s_pieces[g];
                }
            }
            j.many = (j.own_pieces + j.pre_pieces) * p.parts + (j.tc_blocks > 0 ? (j.tc_tiles + per - 1) / per : 0) > kSharedMany;
            if (j.many != 0) p.plan.many[atomicAdd(&p.plan.head->many, 1)] = tok;
        }
        p.plan.join[tok] = j;
    }
}

}  // namespace

int launch_shared_prefix_plan(const SharedPrefixParams& p, cudaStream_t stream) {
    int threads = kMinThreads;
    while (threads < p.batch || threads < p.ctas) threads *= 2;
    B200_CHECK_CUDA(launch_kernel(shared_prefix_plan_kernel, dim3(1), dim3(threads), 0, stream, dim3(1, 1, 1), p));
    return B200_OK;
}

}  // namespace b200
